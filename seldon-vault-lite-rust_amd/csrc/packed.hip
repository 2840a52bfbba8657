// Positions of packed documents over (time, height, width) and the rotation of
// queries and keys by them. Both move bytes and little else.
#include "dev_common.hpp"
#include "packed.hpp"

namespace svl {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

// ---- axis positions -----------------------------------------------------------

// A workgroup writes 1024 tokens, a thread four (48 bytes, three 16-byte
// stores). The table's entries that the workgroup's tokens lie in are brought
// to LDS in one round of loads (at most 1025: every segment has a token) and
// searched there; a search in HBM would be ten or more dependent loads.
__global__ __launch_bounds__(256) void axis_positions_kernel(const PositionSegment *seg,
                                                             const int32_t *block_seg,
                                                             int64_t tokens, int32_t *pos) {
    __shared__ PositionSegment table[POSITION_BLOCK + 1];
    const int first = block_seg[blockIdx.x], last = block_seg[blockIdx.x + 1];
    const int n = last - first + 1;
    for (int i = threadIdx.x; i < n; i += 256) table[i] = seg[first + i];
    __syncthreads();
    const int64_t t0 = (int64_t)blockIdx.x * POSITION_BLOCK + 4 * threadIdx.x;
    if (t0 >= tokens) return;
    int lo = 0, hi = n - 1;  // the last entry that begins at or before t0
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (table[mid].begin <= t0) lo = mid;
        else hi = mid - 1;
    }
    int32_t v[12];
    const int count = (int)min((int64_t)4, tokens - t0);
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
    int32_t *p = pos + 3 * t0;
    if (count == 4 && ((uintptr_t)pos & 15) == 0) {
#pragma unroll
        for (int i = 0; i < 3; ++i)
            *(i32x4 *)(p + 4 * i) = i32x4{v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
    } else {
#pragma unroll
        for (int i = 0; i < 12; ++i)
            if (i < 3 * count) p[i] = v[i];
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
struct Row<float, 2> { typedef float type __attribute__((ext_vector_type(2))); };
template <>
struct Row<float, 4> { typedef f32x4 type; };
template <>
struct Row<__bf16, 1> { typedef __bf16 type; };
template <>
struct Row<__bf16, 2> { typedef bf16x2 type; };
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

// A wave takes a token: its lanes first find the turns of the token's pairs
// once (one pair a lane, 64-bit product, the fraction of a turn to sincospi),
// then all heads of queries and keys, a unit of W pairs a lane, read them from
// LDS. The product of a 32-bit position and a 24-bit frequency is exact to
// 2^-53, so the fraction of 2^31 turns still has 22 bits.
template <class T, int W, bool ADJACENT>
__global__ __launch_bounds__(256) void rope_axes_kernel(RopeAxesArgs a) {
    __shared__ float2 turn[4][ROPE_MAX_PAIRS];
    const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
    const int64_t t = (int64_t)blockIdx.x * 4 + wave;
    const bool live = t < a.tokens;
    if (live)
        for (int j = lane; j < a.pairs; j += 64) {
            const double turns = (double)a.pos[t * a.axes + a.axis[j]] * (double)a.inv_freq[j] *
                                 0.15915494309189535;  // 1 / (2 pi)
            const float f = (float)(turns - rint(turns));
            float s, c;
            sincospif(2.f * f, &s, &c);
            turn[wave][j] = make_float2(c, s);
        }
    __syncthreads();
    if (!live) return;
    const int units = a.pairs / W, copies = a.copied / W, each = units + copies;
    const int total = (a.heads[0] + a.heads[1]) * each;
    for (int i = lane; i < total; i += 64) {
        const int hh = i / each, u = i - hh * each;
        const int which = hh >= a.heads[0];
        const int h = hh - (which ? a.heads[0] : 0);
        const T *in = (const T *)a.in[which] + t * a.in_tok[which] + h * a.in_head[which];
        T *out = (T *)a.out[which] + t * a.out_tok[which] + h * a.out_head[which];
        float x[W], y[W];
        if (u >= units) {
            const int c = 2 * a.pairs + (u - units) * W;
            load_row<T, W>(in + c, x);
            store_row<T, W>(out + c, x);
            continue;
        }
        const int j = u * W;
        const int c0 = a.col[j], c1 = ADJACENT ? c0 + W : a.partner[j];
        load_row<T, W>(in + c0, x);
        load_row<T, W>(in + c1, y);
        if constexpr (ADJACENT && W > 1) {
#pragma unroll
            for (int e = 0; e < W; ++e) {
                const float2 cs = turn[wave][j + e];
                float &p = e < W / 2 ? x[(2 * e) % W] : y[(2 * e) % W];
                float &q = e < W / 2 ? x[(2 * e + 1) % W] : y[(2 * e + 1) % W];
                const float np = p * cs.x - q * cs.y, nq = q * cs.x + p * cs.y;
                p = np;
                q = nq;
            }
        } else {
#pragma unroll
            for (int e = 0; e < W; ++e) {
                const float2 cs = turn[wave][j + e];
                const float p = x[e], q = y[e];
                x[e] = p * cs.x - q * cs.y;
                y[e] = q * cs.x + p * cs.y;
            }
        }
        store_row<T, W>(out + c0, x);
        store_row<T, W>(out + c1, y);
    }
}

template <class T, int W>
static hipError_t launch_rope_width(const RopeAxesArgs &a, bool adjacent, hipStream_t s) {
    const dim3 grid((unsigned)((a.tokens + 3) / 4));
    if (adjacent) hipLaunchKernelGGL((rope_axes_kernel<T, W, true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((rope_axes_kernel<T, W, false>), grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

hipError_t launch_rope_axes(const RopeAxesArgs &a, bool bf16, bool adjacent, int width,
                            hipStream_t s) {
    if (a.tokens <= 0 || a.heads[0] + a.heads[1] <= 0) return hipSuccess;
    switch (width) {
        case 8: return bf16 ? launch_rope_width<__bf16, 8>(a, adjacent, s) : hipErrorInvalidValue;
        case 4: return bf16 ? launch_rope_width<__bf16, 4>(a, adjacent, s)
                            : launch_rope_width<float, 4>(a, adjacent, s);
        case 2: return bf16 ? launch_rope_width<__bf16, 2>(a, adjacent, s)
                            : launch_rope_width<float, 2>(a, adjacent, s);
        case 1: return bf16 ? launch_rope_width<__bf16, 1>(a, adjacent, s)
                            : launch_rope_width<float, 1>(a, adjacent, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace svl
