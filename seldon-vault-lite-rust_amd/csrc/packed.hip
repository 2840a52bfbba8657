// Positions of packed documents over (time, height, width) and the rotation of
// queries and keys by them. Both move bytes and little else.
#include <algorithm>

#include "dev_common.hpp"
#include "packed.hpp"

namespace svl {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

// ---- axis positions -----------------------------------------------------------

// A workgroup writes 1024 tokens, a thread finds four. The table's entries that
// the workgroup's tokens lie in are brought to LDS in one round of loads (at most
// 1025: every segment has a token) and searched there; a search in HBM would be
// ten or more dependent loads. The positions go out through LDS too, so that a
// wave's stores are 1 KB in a row. Two million tokens of video: 8.2 us (9.6
// with 48 bytes a thread stored as three pieces); bytes alone would be 4.
__global__ __launch_bounds__(256) void axis_positions_kernel(const PositionSegment *seg,
                                                             const int32_t *block_seg,
                                                             int64_t tokens, int32_t *pos) {
    __shared__ PositionSegment table[POSITION_BLOCK + 1];
    __shared__ i32x4 out[3 * POSITION_BLOCK / 4];
    const int first = block_seg[blockIdx.x], last = block_seg[blockIdx.x + 1];
    const int n = last - first + 1;
    for (int i = threadIdx.x; i < n; i += 256) table[i] = seg[first + i];
    __syncthreads();
    const int64_t block0 = (int64_t)blockIdx.x * POSITION_BLOCK, t0 = block0 + 4 * threadIdx.x;
    int lo = 0, hi = n - 1;  // the last entry that begins at or before t0
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (table[mid].begin <= t0) lo = mid;
        else hi = mid - 1;
    }
    int32_t v[12];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t t = t0 + i;
        if (lo + 1 < n && table[lo + 1].begin <= t) ++lo;  // segments have tokens: one step is enough
        const PositionSegment s = table[lo];
        const uint32_t local = (uint32_t)(t - s.begin);
        if (s.area == 0) {
            v[3 * i] = v[3 * i + 1] = v[3 * i + 2] = s.start + (int32_t)local;
        } else {
            const uint32_t frame = local / (uint32_t)s.area, in = local - frame * (uint32_t)s.area;
            const uint32_t row = in / (uint32_t)s.cols, col = in - row * (uint32_t)s.cols;
            v[3 * i] = s.start + (int32_t)frame * s.step;
            v[3 * i + 1] = s.start + (int32_t)row;
            v[3 * i + 2] = s.start + (int32_t)col;
        }
    }
#pragma unroll
    for (int i = 0; i < 3; ++i)
        out[3 * threadIdx.x + i] = i32x4{v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
    __syncthreads();
    int32_t *p = pos + 3 * block0;
    const int count = 3 * (int)min((int64_t)POSITION_BLOCK, tokens - block0);
    const bool whole = ((uintptr_t)pos & 15) == 0;
#pragma unroll
    for (int i = threadIdx.x; i < 3 * POSITION_BLOCK / 4; i += 256) {
        const i32x4 x = out[i];
        if (whole && 4 * i + 4 <= count) {
            *(i32x4 *)(p + 4 * i) = x;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (4 * i + e < count) p[4 * i + e] = x[e];
        }
    }
}

hipError_t launch_axis_positions(const PositionSegment *seg, const int32_t *block_seg,
                                 int64_t tokens, int32_t *pos, hipStream_t s) {
    if (tokens <= 0) return hipSuccess;
    const unsigned blocks = (unsigned)((tokens + POSITION_BLOCK - 1) / POSITION_BLOCK);
    hipLaunchKernelGGL(axis_positions_kernel, dim3(blocks), dim3(256), 0, s, seg, block_seg, tokens,
                       pos);
    return hipGetLastError();
}

// ---- rotation -------------------------------------------------------------------

template <class T, int W>
struct Row;
template <>
struct Row<float, 1> { typedef float type; };
template <>
struct Row<float, 4> { typedef f32x4 type; };
template <>
struct Row<__bf16, 1> { typedef __bf16 type; };
template <>
struct Row<__bf16, 4> { typedef bf16x4 type; };
template <>
struct Row<__bf16, 8> { typedef bf16x8 type; };

template <class T, int W>
__device__ __forceinline__ void load_row(const T *p, float (&x)[W]) {
    const auto v = *(const typename Row<T, W>::type *)p;
    if constexpr (W == 1) {
        x[0] = (float)v;
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i) x[i] = (float)v[i];
    }
}

template <class T, int W>
__device__ __forceinline__ void store_row(T *p, const float (&x)[W]) {
    typename Row<T, W>::type v;
    if constexpr (W == 1) {
        v = (T)x[0];
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = (T)x[i];
    }
    *(typename Row<T, W>::type *)p = v;
}

// (cos, sin) of token t's pair j: a 64-bit product, its fraction of a turn to
// sincospi. The product of a 32-bit position and a 24-bit frequency is exact to
// 2^-53, so the fraction of 2^31 turns still has 22 bits.
__device__ __forceinline__ float2 turn_of(const RopeAxesArgs &a, int64_t t, int j) {
    const double turns = (double)a.pos[t * a.axes + a.axis[j]] * (double)a.inv_freq[j] *
                         0.15915494309189535;  // 1 / (2 pi)
    const float f = (float)(turns - rint(turns));
    float s, c;
    sincospif(2.f * f, &s, &c);
    return make_float2(c, s);
}

// A workgroup takes R * 256 / TT tokens at a time, TT threads for R of them
// (TT = 1 << shift), and goes on to the next ones in steps of the grid. What a thread does is the
// same for every token: up to U units of W pairs (or of copied columns) of some
// head of queries or keys, whose addresses it finds once. Per token it issues
// their loads, finds the turns of some of the token's pairs for all heads, in
// LDS, and rotates.
// Bytes bound it: 18688 tokens, 4 float heads of 256 take 26 us, 5.8 TB/s (26-28
// with one wave a token that finds its addresses for every unit). W is 16 bytes;
// rows off that alignment go value by value, with more tokens in flight.
template <class T, int W, bool ADJACENT, int U, int R>
__global__ __launch_bounds__(256) void rope_axes_kernel(RopeAxesArgs a, int shift) {
    extern __shared__ float2 turn_s[];  // [2][R * 256 / TT][pairs]
    const int tt = 1 << shift, many = 256 >> shift;
    const int group = (int)threadIdx.x >> shift, lane = (int)threadIdx.x & (tt - 1);
    const int units = a.pairs / W, copies = a.copied / W, each = units + copies;
    const int total = (a.heads[0] + a.heads[1]) * each;
    struct Unit {
        const T *in;
        T *out;
        int64_t in_tok, out_tok;
        int far, pair;  // second column's distance, first pair; pair < 0: copied columns
    };
    auto find = [&](int i) {
        Unit x{};
        const int hh = i / each, u = i - hh * each;
        const int which = hh >= a.heads[0];
        const int h = hh - (which ? a.heads[0] : 0);
        const int c = u < units ? a.col[u * W] : 2 * a.pairs + (u - units) * W;
        x.in = (const T *)a.in[which] + h * a.in_head[which] + c;
        x.out = (T *)a.out[which] + h * a.out_head[which] + c;
        x.in_tok = a.in_tok[which];
        x.out_tok = a.out_tok[which];
        x.pair = u < units ? u * W : -1;
        x.far = u >= units ? 0 : ADJACENT ? W : a.partner[u * W] - c;
        return x;
    };
    auto load = [&](const Unit &w, int64_t t, float (&x)[W], float (&y)[W]) {
        load_row<T, W>(w.in + t * w.in_tok, x);
        if (w.pair >= 0) load_row<T, W>(w.in + t * w.in_tok + w.far, y);
    };
    auto finish = [&](const Unit &w, int64_t t, const float2 *turn, float (&x)[W], float (&y)[W]) {
        T *out = w.out + t * w.out_tok;
        if (w.pair >= 0) {
#pragma unroll
            for (int e = 0; e < W; ++e) {
                const float2 cs = turn[w.pair + e];
                // adjacent: element pairs of the 2 W values x, y in a row
                constexpr bool ROW = ADJACENT && W > 1;
                float &p = !ROW ? x[e] : e < W / 2 ? x[(2 * e) % W] : y[(2 * e) % W];
                float &q = !ROW ? y[e] : e < W / 2 ? x[(2 * e + 1) % W] : y[(2 * e + 1) % W];
                const float np = p * cs.x - q * cs.y, nq = q * cs.x + p * cs.y;
                p = np;
                q = nq;
            }
            store_row<T, W>(out + w.far, y);
        }
        store_row<T, W>(out, x);
    };
    Unit mine[U];
#pragma unroll
    for (int n = 0; n < U; ++n)
        if (lane + n * tt < total) mine[n] = find(lane + n * tt);
    int buffer = 0;
    const int64_t step = (int64_t)many * R;
    for (int64_t t0 = blockIdx.x * step; t0 < a.tokens; t0 += gridDim.x * step) {
        float2 *turn = turn_s + (buffer * many + group) * R * a.pairs;
        float x[R][U][W], y[R][U][W];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int n = 0; n < U; ++n) {
                const int64_t t = t0 + r * many + group;
                if (t < a.tokens && lane + n * tt < total) load(mine[n], t, x[r][n], y[r][n]);
            }
        for (int i = lane; i < R * a.pairs; i += tt) {
            const int r = i / a.pairs, j = i - r * a.pairs;
            const int64_t t = t0 + r * many + group;
            if (t >= a.tokens) break;
            turn[i] = turn_of(a, t, j);
        }
        __syncthreads();  // the other buffer is read no more, too
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t t = t0 + r * many + group;
            if (t >= a.tokens) break;
#pragma unroll
            for (int n = 0; n < U; ++n)
                if (lane + n * tt < total) finish(mine[n], t, turn + r * a.pairs, x[r][n], y[r][n]);
            for (int i = lane + U * tt; i < total; i += tt) {
                const Unit w = find(i);
                load(w, t, x[r][0], y[r][0]);
                finish(w, t, turn + r * a.pairs, x[r][0], y[r][0]);
            }
        }
        buffer ^= 1;
    }
}

// Threads a token: as few as leave each at most two units (of up to 256), so
// that a workgroup's tokens fill it; U to match.
template <class T, int W, bool ADJACENT>
static hipError_t launch_rope_form(const RopeAxesArgs &a, hipStream_t s) {
    const int64_t total = (int64_t)(a.heads[0] + a.heads[1]) * (a.pairs / W + a.copied / W);
    const int shift = total <= 128 ? 6 : total <= 256 ? 7 : 8, many = 256 >> shift;
    constexpr int R = W > 1 ? 1 : 4;  // tokens in flight
    const int64_t rounds = (a.tokens + many * R - 1) / (many * R);
    const dim3 grid((unsigned)std::min<int64_t>(rounds, 2048)), block(256);
    const size_t lds = (size_t)2 * many * R * std::max(a.pairs, 1) * sizeof(float2);
    if (total <= (1 << shift))
        hipLaunchKernelGGL((rope_axes_kernel<T, W, ADJACENT, 1, R>), grid, block, lds, s, a, shift);
    else
        hipLaunchKernelGGL((rope_axes_kernel<T, W, ADJACENT, 2, R>), grid, block, lds, s, a, shift);
    return hipGetLastError();
}

template <class T, int W>
static hipError_t launch_rope_width(const RopeAxesArgs &a, bool adjacent, hipStream_t s) {
    return adjacent ? launch_rope_form<T, W, true>(a, s) : launch_rope_form<T, W, false>(a, s);
}

// Rows in whole 16-byte chunks, whatever the pairs' layout: a thread takes a chunk
// of a head row, C values, for R tokens at a time; the rows also go to LDS, where
// it finds its values' partners (at places that are the same for every token),
// beside the turns, one of (cos, +-sin) a column. A column that is only copied
// has the turn (1, -0) and a zero for its partner, which leave it as it is.
// Workgroups of grid.y share a token's heads, as many as 256 threads hold.
// For pairs that come in runs of less than 16 bytes: 36864 tokens, 24 bfloat16
// heads of 64 with axes of 10 pairs take 45 us, 5.0 TB/s (78 us as units of two
// pairs, 92 with one token in flight); where runs are longer the units are as
// fast and start sooner (17 tokens, 4 heads of 256: 4.7 us, 7.3 by rows).
template <class T, int R>
__global__ __launch_bounds__(256) void rope_rows_kernel(RopeAxesArgs a, int heads_each, int many) {
    constexpr int C = 16 / sizeof(T);
    typedef typename Row<T, C>::type Chunk;
    extern __shared__ char rope_s[];
    const int chunks = a.hd / C;                   // of a head row
    const int heads = a.heads[0] + a.heads[1];
    const int h0 = blockIdx.y * heads_each, here = min(heads_each, heads - h0);
    const int used = chunks * here;                // threads a token, `many` tokens side by side
    const int group = (int)threadIdx.x / used, lane = (int)threadIdx.x - group * used;
    const bool mine = group < many;
    const int hh = h0 + lane / chunks, col = (lane % chunks) * C;
    const int which = hh >= a.heads[0], h = hh - (which ? a.heads[0] : 0);
    const T *in = (const T *)a.in[which] + h * a.in_head[which] + col;
    T *out = (T *)a.out[which] + h * a.out_head[which] + col;
    const int64_t in_tok = a.in_tok[which], out_tok = a.out_tok[which];
    // a token's part of LDS: the heads' rows, a chunk of zeros, the turns
    const int zero_at = chunks * heads_each * 16, turns_at = zero_at + 16;
    const int each = turns_at + a.hd * 8, step = many * R;
    char *mine_s = rope_s + group * R * each;         // of the first buffer
    // partners' bytes from the token's part
    int partner[C];
    {
        int *of = (int *)rope_s;
        for (int c = threadIdx.x; c < a.hd; c += 256) of[c] = -1;
        __syncthreads();
        for (int j = threadIdx.x; j < a.pairs; j += 256) {
            of[a.col[j]] = a.partner[j];
            of[a.partner[j]] = a.col[j];
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < C; ++e) {
            const int v = of[col + e];
            partner[e] = v < 0 ? zero_at : (lane / chunks * a.hd + v) * (int)sizeof(T);
        }
        __syncthreads();
    }
    for (int i = threadIdx.x; i < 2 * step; i += 256) *(f32x4 *)(rope_s + i * each + zero_at) = f32x4{0.f, 0.f, 0.f, 0.f};
    const int rest = a.hd - 2 * a.pairs;           // columns without a turn
    for (int i = threadIdx.x; i < 2 * step * rest; i += 256)
        *(float2 *)(rope_s + i / rest * each + turns_at + (2 * a.pairs + i % rest) * 8) =
            make_float2(1.f, -0.f);
    int buffer = 0;
    for (int64_t t0 = (int64_t)blockIdx.x * step; t0 < a.tokens; t0 += (int64_t)gridDim.x * step) {
        char *part = mine_s + buffer * step * each;
        Chunk x[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t t = t0 + r * many + group;
            if (mine && t < a.tokens) x[r] = *(const Chunk *)(in + t * in_tok);
        }
        if (mine)
            for (int i = lane; i < R * a.pairs; i += used) {
                const int r = i / a.pairs, j = i - r * a.pairs;
                const int64_t t = t0 + r * many + group;
                if (t >= a.tokens) break;
                const float2 cs = turn_of(a, t, j);
                float2 *turn = (float2 *)(part + r * each + turns_at);
                turn[a.col[j]] = make_float2(cs.x, -cs.y);
                turn[a.partner[j]] = cs;
            }
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (mine) *(Chunk *)(part + r * each + lane * 16) = x[r];
        __syncthreads();  // the other buffer is read no more, too
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t t = t0 + r * many + group;
            if (!mine || t >= a.tokens) break;
            const f32x4 *turn = (const f32x4 *)(part + r * each + turns_at + col * 8);
            Chunk y;
#pragma unroll
            for (int e = 0; e < C; e += 2) {
                const f32x4 cs = turn[e / 2];
                const float p0 = (float)*(const T *)(part + r * each + partner[e]);
                const float p1 = (float)*(const T *)(part + r * each + partner[e + 1]);
                y[e] = (T)(p0 * cs.y + (float)x[r][e] * cs.x);
                y[e + 1] = (T)(p1 * cs.w + (float)x[r][e + 1] * cs.z);
            }
            *(Chunk *)(out + t * out_tok) = y;
        }
        buffer ^= 1;
    }
}

template <class T, int R>
static hipError_t launch_rope_rows(const RopeAxesArgs &a, hipStream_t s) {
    const int chunks = a.hd * (int)sizeof(T) / 16, heads = a.heads[0] + a.heads[1];
    const int each = std::min(heads, 256 / chunks);
    const int part = chunks * each * 16 + 16 + a.hd * 8;  // LDS a token: at most 12 KB
    const int many = std::min(256 / (chunks * each), std::max(48 * 1024 / (2 * R * part), 1));
    const int64_t rounds = (a.tokens + many * R - 1) / (many * R);
    const int groups = (heads + each - 1) / each;
    const dim3 grid((unsigned)std::min<int64_t>(rounds, std::max(8192 / groups, 1)), (unsigned)groups);
    const size_t lds = (size_t)2 * R * many * part;
    hipLaunchKernelGGL((rope_rows_kernel<T, R>), grid, dim3(256), lds, s, a, each, many);
    return hipGetLastError();
}

hipError_t launch_rope_axes(const RopeAxesArgs &a, bool bf16, bool adjacent, RopeForm form,
                            hipStream_t s) {
    if (a.tokens <= 0 || a.heads[0] + a.heads[1] <= 0) return hipSuccess;
    switch (form) {
        case ROPE_CHUNKS:
            return bf16 ? launch_rope_width<__bf16, 8>(a, adjacent, s)
                        : launch_rope_width<float, 4>(a, adjacent, s);
        case ROPE_ROWS:
            return bf16 ? launch_rope_rows<__bf16, 2>(a, s) : launch_rope_rows<float, 2>(a, s);
        case ROPE_SINGLE:
            return bf16 ? launch_rope_width<__bf16, 1>(a, adjacent, s)
                        : launch_rope_width<float, 1>(a, adjacent, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace svl
