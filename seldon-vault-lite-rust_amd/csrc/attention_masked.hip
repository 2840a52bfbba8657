// Attention over packed documents with causal, window and prefix masks, a
// score cap and a distance bias (svl_masked_attention).
#include <algorithm>

#include "dev_common.hpp"
#include "packed.hpp"

namespace svl {

constexpr float LOG2E = 1.4426950408889634f;

// One query vector of a piece of work by a whole wave, any head dim up to
// 64 * NPER: lanes hold dims lane, lane + 64, ...; only visible keys are
// visited, in order, with the running maximum and sum of the softmax. The
// kernel of large head dims, and what the tile kernel turns to where a tile
// holds non-finite values that only some of its queries may see.
template <class T, int NPER>
__device__ void masked_row(const MaskedArgs &a, const AttnWork &w, int vec, int tile_keys,
                           float *out_part, float *ml_part) {
    const int lane = threadIdx.x & 63;
    const int G = a.heads / a.kv_heads;
    const int qi = vec / G, head = w.kvh * G + (vec - qi * G);
    const int64_t qrow = (int64_t)w.q_row + qi;
    const int64_t p = (int64_t)qi + w.k_len - w.q_len;
    int64_t lo = 0, hi = w.k_len - 1;
    if (a.causal) hi = min(hi, p);
    if (a.window >= 0) {
        lo = max(lo, p - a.window);
        hi = min(hi, p + a.window);
    }
    const T *q = (const T *)a.q + qrow * a.q_tok + head * a.q_head;
    float qv[NPER], acc[NPER];
#pragma unroll
    for (int e = 0; e < NPER; ++e) {
        const int d = lane + 64 * e;
        qv[e] = d < a.hd ? (float)q[d] * a.scale : 0.f;
        acc[e] = 0.f;
    }
    const float slope = a.slopes ? a.slopes[head] : 0.f;
    float m = -INFINITY, l = 0.f;
    for (int part = 0; part < 2; ++part) {
        // tiles t0 .. t1 of the prefix, then of the rest
        const int ta = part ? max(w.t0, w.pre_tiles) : w.t0;
        const int tb = part ? w.t1 : min(w.t1, w.pre_tiles);
        const int64_t first = part ? w.main_key + (int64_t)(ta - w.pre_tiles) * tile_keys
                                   : (int64_t)ta * tile_keys;
        const int64_t last = min((int64_t)w.k_len, first + (int64_t)(tb - ta) * tile_keys);
        for (int64_t key = first; key < last; ++key) {
            if (key >= w.prefix) {  // on to the next visible one
                if (key < lo) key = lo;
                if (key > hi || key >= last) break;
            }
            const T *k = (const T *)a.k + (w.k_row + key) * a.k_tok + w.kvh * a.k_head;
            const T *v = (const T *)a.v + (w.k_row + key) * a.v_tok + w.kvh * a.v_head;
            float s = 0.f;
#pragma unroll
            for (int e = 0; e < NPER; ++e) {
                const int d = lane + 64 * e;
                if (d < a.hd) s += qv[e] * (float)k[d];
            }
            s = wave_sum(s);
            if (a.cap > 0.f) s = a.cap * tanhf(s / a.cap);
            if (a.slopes) s -= slope * fabsf((float)(p - key));
            const float mn = fmaxf(m, s);
            const float base = mn == -INFINITY ? 0.f : mn;
            const float scale = expf(m - base), pr = expf(s - base);
            l = l * scale + pr;
            m = mn;
#pragma unroll
            for (int e = 0; e < NPER; ++e) {
                const int d = lane + 64 * e;
                if (d < a.hd) acc[e] = acc[e] * scale + pr * (float)v[d];
            }
        }
    }
    if (out_part) {
#pragma unroll
        for (int e = 0; e < NPER; ++e) out_part[lane + 64 * e] = acc[e];
        if (lane == 0) {
            ml_part[0] = m * LOG2E;
            ml_part[1] = l;
        }
        return;
    }
    T *out = (T *)a.out + qrow * a.o_tok + head * a.o_head;
#pragma unroll
    for (int e = 0; e < NPER; ++e) {
        const int d = lane + 64 * e;
        if (d < a.hd) out[d] = (T)(l == 0.f ? 0.f : acc[e] / l);
    }
    if (a.lse && lane == 0)
        a.lse[qrow * a.heads + head] = l == 0.f ? -INFINITY : m + logf(l);
}

constexpr int ROW_KEYS = 64;  // keys that a tile of the row kernel's plans stands for

template <class T>
__global__ __launch_bounds__(256) void masked_rows_kernel(MaskedArgs a, int vectors) {
    const AttnWork w = a.work[blockIdx.x];
    const int nvec = w.q_len * (a.heads / a.kv_heads);
    for (int i = uniform((int)threadIdx.x >> 6); i < vectors && w.v0 + i < nvec; i += 4)
        masked_row<T, 16>(a, w, w.v0 + i, ROW_KEYS, nullptr, nullptr);
}

// ---- tiles on the matrix cores ---------------------------------------------------

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4_raw __attribute__((vector_size(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// Row r of a tile holds its 16-byte chunks in another order, so that the rows
// that one LDS instruction reads at one column lie in different banks (a tile
// row is 128 bytes at 64 dims, else a multiple of the banks' 256). Scores read
// 16 bytes of 32 rows at one chunk; values are read transposed, 64 bytes of
// four rows.
template <int D>
__device__ __forceinline__ int key_swizzle(int r) { return D == 64 ? (r >> 1) & 7 : r & 15; }
template <int D>
__device__ __forceinline__ int value_swizzle(int r) {
    return D == 64 ? ((r >> 1) & 1) << 2 : (r & 3) << 2;
}

// x = high + middle + low, bfloat16 each, two values at a time (packed, the
// first below). Each part is the rest's nearest bfloat16, so the rest is at most
// 2^-8 of it and the three hold all 24 bits of x. Infinities and NaN stay in the
// high part (as do magnitudes above the largest bfloat16, 0.996 of the largest
// float: they become infinities).
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
}
template <bool FINITE>
__device__ __forceinline__ void split3(float a, float b, uint32_t (&p)[3]) {
    p[0] = pack_bf16(a, b);
    float ra = a - __uint_as_float(p[0] << 16), rb = b - __uint_as_float(p[0] & 0xffff0000u);
    if constexpr (!FINITE) {
        ra = isfinite(ra) ? ra : 0.f;
        rb = isfinite(rb) ? rb : 0.f;
    }
    p[1] = pack_bf16(ra, rb);
    p[2] = pack_bf16(ra - __uint_as_float(p[1] << 16), rb - __uint_as_float(p[1] & 0xffff0000u));
}

// A tile's way from HBM to LDS: fetch() starts it, commit() ends it.
//  * FROM_ROWS: whole 16-byte chunks of bfloat16 rows, by DMA.
//  * FROM_PIECES: bfloat16 rows of any alignment, through registers.
//  * FROM_PLANES: tiles that masked_planes_kernel has laid out, P planes of
//    them as they lie in LDS, by DMA.
enum TileSource { FROM_ROWS, FROM_PIECES, FROM_PLANES };

template <class T, int P, int D, int KT, int THREADS, TileSource FROM, int (*SWIZZLE)(int)>
struct TileCopy {
    static constexpr int EACH = (FROM == FROM_PLANES ? P : 1) * KT * D / 8 / THREADS;  // chunks of a thread
    static_assert(KT * D / 8 % THREADS == 0, "tile");
    static constexpr int OUT = (int)0x80000000;  // an offset out of range: reads zero
    __bf16 reg[FROM == FROM_PIECES ? EACH * 8 : 1];
    // Offsets are kept where there is room, else found anew for each tile (at
    // 256 dims the registers are worth more than the few instructions).
    static constexpr bool KEPT = FROM == FROM_ROWS && D < 256;
    int kept[KEPT ? EACH : 1];

    __device__ __forceinline__ static int offset(int i, int lane, int ld, int hd) {
        const int c = ((int)threadIdx.x >> 6) * (64 * EACH) + 64 * i + lane;
        if constexpr (FROM == FROM_PLANES) return c * 16;
        const int r = c / (D / 8), dim = 8 * ((c % (D / 8)) ^ SWIZZLE(r));
        return FROM == FROM_PIECES || dim < hd ? (r * ld + dim) * 2 : OUT;
    }
    __device__ __forceinline__ void init(int ld, int hd) {
        if constexpr (KEPT) {
#pragma unroll
            for (int i = 0; i < EACH; ++i) kept[i] = offset(i, (int)threadIdx.x & 63, ld, hd);
        }
    }

    // chunk that this thread moves i-th: a wave's DMA fills 1 KB of LDS in a row
    __device__ __forceinline__ static int place(int i) {
        return ((int)threadIdx.x >> 6) * (64 * EACH) + 64 * i + ((int)threadIdx.x & 63);
    }
    // rows: rows of the tile that exist
    __device__ __forceinline__ void fetch(const void *base, int ld, int hd, int rows, __bf16 *lds) {
        const int bytes = FROM == FROM_PLANES ? P * KT * D * 2 : ((rows - 1) * ld + hd) * 2;
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
            uniform((char *)base), (short)0, uniform(bytes), 0x00020000);
        const int wave = uniform((int)threadIdx.x >> 6);
        int lane = (int)threadIdx.x & 63;
        if constexpr (!KEPT) asm volatile("" : "+v"(lane));
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            int off;
            if constexpr (KEPT) off = kept[i];
            else off = offset(i, lane, ld, hd);
            if constexpr (FROM == FROM_PIECES) {
                const int c = wave * (64 * EACH) + 64 * i + lane, r = c / (D / 8);
                const int dim = 8 * ((c % (D / 8)) ^ SWIZZLE(r));
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    reg[8 * i + e] = __builtin_bit_cast(
                        __bf16, __builtin_amdgcn_raw_buffer_load_b16(
                                    rs, dim + e < hd ? off + 2 * e : OUT, 0, 0));
            } else {
                __builtin_amdgcn_raw_ptr_buffer_load_lds(
                    rs, (__attribute__((address_space(3))) void *)(lds + (wave * EACH + i) * 512),
                    16, off, 0, 0, 0);
            }
        }
    }
    __device__ __forceinline__ void commit(__bf16 *lds) {
        if constexpr (FROM != FROM_PIECES) {
            wait_vmcnt<0>();
        } else {
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                bf16x8 v;
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = reg[8 * i + e];
                *(bf16x8 *)(lds + place(i) * 8) = v;
            }
        }
    }
    // Whether this thread's part of a landed tile holds a non-finite value (of
    // three planes the first tells).
    __device__ __forceinline__ static bool non_finite(const __bf16 *lds) {
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            if (place(i) * 8 >= KT * D) continue;
            const u32x4 v = *(const u32x4 *)(lds + place(i) * 8);
#pragma unroll
            for (int e = 0; e < 4; ++e) any |= (v[e] & 0x7fff7fffu) + 0x00800080u;
        }
        return (any & 0x80008000u) != 0;
    }
};

// Keys and values as tiles of KT rows in the order of LDS, keys and dims past the
// end zero: float ones in three planes, one for each bfloat16 part, and bfloat16
// ones of head dims that are no whole chunks. Done once a call: splitting floats
// in every workgroup that reads them was a third of the vector work of the tile
// kernel (64 documents of 64-512 tokens, 3 heads of 256: 214 us against 181 + 17),
// and rows of 100 bfloat16 values read one by one took 1296 us against
// 371 (4 x 4096 tokens, 8 heads).
template <class T, int P, int D, int KT>
__global__ __launch_bounds__(256) void masked_planes_kernel(MaskedArgs a) {
    const AttnTiles w = a.tiles[blockIdx.x];
    const bool values = blockIdx.y != 0;
    const int64_t ld = values ? a.v_tok : a.k_tok;
    const T *base = (const T *)(values ? a.v : a.k) + (int64_t)w.k_row * ld +
                    w.kvh * (values ? a.v_head : a.k_head);
    __bf16 *out = (__bf16 *)a.planes + ((int64_t)blockIdx.x * 2 + values) * (P * KT * D);
    for (int c = threadIdx.x; c < KT * D / 8; c += 256) {
        const int r = c / (D / 8);
        const int dim = 8 * ((c % (D / 8)) ^ (values ? value_swizzle<D>(r) : key_swizzle<D>(r)));
        T x[8];
        const T *row = base + r * ld + dim;
        if (P == 3 && r < w.rows && a.whole && dim + 8 <= a.hd) {
            __builtin_memcpy(x, __builtin_assume_aligned(row, 16), sizeof x);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = r < w.rows && dim + e < a.hd ? row[e] : (T)0.f;
        }
        u32x4 pl[P];
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            if constexpr (P == 1) {
                pl[0][e / 2] = __builtin_bit_cast(uint32_t, bf16x2{x[e], x[e + 1]});
            } else {
                uint32_t y[3];
                split3<false>(x[e], x[e + 1], y);
#pragma unroll
                for (int p = 0; p < P; ++p) pl[p][e / 2] = y[p];
            }
        }
#pragma unroll
        for (int p = 0; p < P; ++p) *(u32x4 *)(out + p * KT * D + c * 8) = pl[p];
    }
}

// Four keys x 16 dims of bfloat16 read transposed (a lane's 8-byte piece: key
// (lane % 16) / 4 of the four, dims 4 (lane % 4) ..): the lane receives dim
// lane % 16 of the four keys.
__device__ __forceinline__ bf16x4 read_transposed_bf16(const __bf16 *p) {
    return __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
                                          (__attribute__((address_space(3))) bf16x4_raw *)p));
}

__device__ __forceinline__ float other_half_max(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float other_half_sum(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// Max / sum over the four 16-lane groups of a wave.
__device__ __forceinline__ float group_max4(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return other_half_max(fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1])));
}
__device__ __forceinline__ float group_sum4(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return other_half_sum(__uint_as_float(a[0]) + __uint_as_float(a[1]));
}

// tanh(y) / y = 1 + q P(q), q = y^2: a Chebyshev fit of P on [0, 0.56^2], error
// of tanh 6e-9.
constexpr float TANH_C0 = -0.33333331f, TANH_C1 = 0.13333082f, TANH_C2 = -0.053903349f,
                TANH_C3 = 0.021272749f, TANH_C4 = -0.006542542f;

// cap tanh(x / cap) log2(e) from the raw product: to2x = 2 log2(e) scale / cap
// takes it to the exponent of e^(2 x / cap), capl = cap log2(e).
// tanh y = 1 - 2 / (e^2y + 1) loses the low bits of a small y (an absolute
// error of 2^-24), which bfloat16 scores do without and float scores take from
// the series above below 0.55.
__device__ __forceinline__ float capped(float s, float to2x, float capl) {
    const float z = s * to2x;
    const float r = __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(z) + 1.f);
    const float y = z * 0.34657359028f;  // ln 2 / 2
    const float q = y * y;
    float p = __builtin_fmaf(q, TANH_C4, TANH_C3);
    p = __builtin_fmaf(q, p, TANH_C2);
    p = __builtin_fmaf(q, p, TANH_C1);
    p = __builtin_fmaf(q, p, TANH_C0);
    return fabsf(y) < 0.55f ? capl * __builtin_fmaf(y * q, p, y) : __builtin_fmaf(r, -2.f * capl, capl);
}

// A workgroup takes WAVES / DS * 32 query vectors of one document and KV head:
// the heads that share a KV head are vectors beside each other, so a tile of
// keys serves all of them. Keys stream through LDS in tiles of KT.
//  * S^T = K Q^T on 32x32x16 MFMAs, queries in registers: a lane holds 16 of
//    a block's 32 keys for one query, so that maximum and sum are a lane's own
//    but for one exchange with lane ^ 32.
//  * O^T += V^T P^T: the score registers 8 u .. 8 u + 7 are the B operand of
//    step u as they stand (keys 16 u + 4 h + 0..3 and + 8, h = lane / 32), and V
//    is read transposed in the same order.
//  * The running maximum moves only when some query's weights of a tile add up
//    to more than MOST_SUM, so outputs are rarely rescaled and most tiles look
//    for no maximum at all.
//  * STAGES = 2: a tile's K and V come in under the whole tile before, one
//    barrier a tile. STAGES = 1, where LDS holds no more: V(t) comes in under
//    the scores of tile t, K(t + 1) under its softmax and P V; two barriers.
//    STAGES = 0: K and V in turn in one buffer (512 float dims).
//  * DS = 2: two waves share 32 queries, each with half of the dims of scores
//    (summed through LDS) and output, where one wave's registers would leave a
//    SIMD to a single wave (float rows: three parts of every query; 256 dims
//    311 us with one wave, 214 us with two).
// P = 1: bfloat16 operands; weights are rounded to bfloat16 for the product
// with V (a relative 2^-8 of each, the output's own step). LSE: their sum is
// taken before, so that the lse keeps its 32 bits, else of the rounded ones.
// P = 3: float operands as three bfloat16 parts; of the nine products the six
// above 2^-24 are taken, the five small ones in an accumulator of their own.
constexpr float MOST_SUM = 16384.f;

template <class T, int P, int D, int KT, int WAVES, int DS, int STAGES, TileSource FROM, bool CAP,
          bool LSE, int MINW>
__global__ __launch_bounds__(64 * WAVES, MINW) void masked_tile_kernel(MaskedArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int DW = D / DS;  // dims of a wave
    constexpr int NB = DW / 16, NT = DW / 32, NK = KT / 32, VECTORS = 32 * WAVES / DS;
    // one object a stage, chosen at compile time: the compiler then sees that
    // the DMA into one does not touch the reads of the other
    __shared__ __bf16 K0[P * KT * D], V0[STAGES > 0 ? P * KT * D : 8];
    __shared__ __bf16 K1[STAGES > 1 ? P * KT * D : 8], V1[STAGES > 1 ? P * KT * D : 8];
    __shared__ f32x4 Sx[DS > 1 ? WAVES * NK * 4 * 64 : 1];  // the waves' parts of the scores
    __shared__ int dirty;  // 1 + the tile whose values hold a non-finite one
    const AttnWork w = a.work[blockIdx.x];
    const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
    const int l32 = lane & 31, h = lane >> 5;
    const int G = a.heads / a.kv_heads;
    const int nvec = w.q_len * G;
    const int dim0 = (wave % DS) * DW;
    const int wv0 = w.v0 + wave / DS * 32;     // this wave's first vector
    const bool some = wv0 < nvec;              // ... and whether it has any
    const int vec = min(wv0 + l32, nvec - 1);
    const bool valid = wv0 + l32 < nvec;
    const int qi = vec / G, head = w.kvh * G + (vec - qi * G);
    const int shift = w.k_len - w.q_len;
    const int p = qi + shift;
    const int p_lo = min(wv0, nvec - 1) / G + shift, p_hi = min(wv0 + 31, nvec - 1) / G + shift;
    const int wg_lo = w.v0 / G + shift, wg_hi = min(w.v0 + VECTORS - 1, nvec - 1) / G + shift;

    // a query's keys besides the prefix: lo .. hi
    auto first_key = [&](int pos) { return a.window >= 0 ? (int)max((int64_t)pos - a.window, (int64_t)0) : 0; };
    auto last_key = [&](int pos) {
        int64_t k = w.k_len - 1;
        if (a.causal) k = min(k, (int64_t)pos);
        if (a.window >= 0) k = min(k, (int64_t)pos + a.window);
        return (int)max(k, (int64_t)-1);
    };
    const int lo = first_key(p);
    const uint32_t span = (uint32_t)max(last_key(p) - lo + 1, 0);  // keys from lo on
    // the wave's: any of its queries, all of them; and all of the workgroup's
    const int any_lo = first_key(p_lo), any_hi = last_key(p_hi);
    const int all_lo = first_key(p_hi), all_hi = last_key(p_lo);
    const int wg_all_lo = first_key(wg_hi), wg_all_hi = last_key(wg_lo);

    // scores: sign of the scale into the queries, its size into the exponent
    const float size = fabsf(a.scale);
    bf16x8 q[P][NB];
    {
        const T *row = (const T *)a.q + (int64_t)(w.q_row + qi) * a.q_tok + head * a.q_head;
        const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int d = dim0 + 16 * b + 8 * h;
            T x[8];
            if (a.whole) {
                constexpr int N = 16 / sizeof(T);
#pragma unroll
                for (int i = 0; i < 8; i += N) {
                    u32x4 v = {0, 0, 0, 0};
                    if (d + i < a.hd) v = *(const u32x4 *)(row + d + i);
                    __builtin_memcpy(&x[i], &v, 16);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = d + i < a.hd ? row[d + i] : (T)0.f;
            }
            u32x4 pl[P];
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                if constexpr (P == 1) {
                    pl[0][e / 2] = __builtin_bit_cast(uint32_t, bf16x2{x[e], x[e + 1]});
                } else {
                    uint32_t y[3];
                    split3<false>(x[e], x[e + 1], y);
#pragma unroll
                    for (int i = 0; i < P; ++i) pl[i][e / 2] = y[i];
                }
            }
#pragma unroll
            for (int i = 0; i < P; ++i) {
#pragma unroll
                for (int e = 0; e < 4; ++e) pl[i][e] ^= flip;
                q[i][b] = __builtin_bit_cast(bf16x8, pl[i]);
            }
        }
    }
    const float to_log2 = size * LOG2E;
    const float to2x = CAP ? fminf(2.f * LOG2E * size / a.cap, 3e38f) : 0.f, capl = a.cap * LOG2E;
    const float slope = a.slopes ? a.slopes[head] * LOG2E : 0.f;

    f32x16 o[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[t][r] = 0.f;
    float m_ref = -INFINITY, l_run = 0.f;

    const int ldk = (int)a.k_tok, ldv = (int)a.v_tok;
    const __bf16 *kbase = FROM == FROM_PLANES ? (const __bf16 *)a.planes + (int64_t)w.tile0 * (2 * P * KT * D)
                                              : (const __bf16 *)a.k + w.k_row * a.k_tok + w.kvh * a.k_head;
    const __bf16 *vbase = FROM == FROM_PLANES ? kbase + P * KT * D
                                              : (const __bf16 *)a.v + w.k_row * a.v_tok + w.kvh * a.v_head;
    TileCopy<T, P, D, KT, 64 * WAVES, FROM, key_swizzle<D>> kc;
    TileCopy<T, P, D, KT, 64 * WAVES, FROM, value_swizzle<D>> vc;
    kc.init(ldk, a.hd);
    vc.init(ldv, a.hd);
    auto key_of = [&](int t) { return t < w.pre_tiles ? t * KT : w.main_key + (t - w.pre_tiles) * KT; };
    auto fetch_k = [&](int k0, __bf16 *to) {
        kc.fetch(FROM == FROM_PLANES ? kbase + (int64_t)k0 * (2 * P * D) : kbase + (int64_t)k0 * ldk,
                 ldk, a.hd, min(KT, w.k_len - k0), to);
    };
    auto fetch_v = [&](int k0, __bf16 *to) {
        vc.fetch(FROM == FROM_PLANES ? vbase + (int64_t)k0 * (2 * P * D) : vbase + (int64_t)k0 * ldv,
                 ldv, a.hd, min(KT, w.k_len - k0), to);
    };
    // Lane addresses, in bytes: K row l32 of a block at chunk h, V row
    // (lane % 16) / 4 of four at its chunk of a 32-dim tile. Rows start at
    // multiples of D, so another chunk (a multiple of 2 or 4 further before the
    // swizzle) is an exclusive or of the offset; it is done as each fragment is
    // read (kept in registers, the addresses would spill).
    int koff = l32 * D * 2 + (((dim0 / 8 + h) ^ key_swizzle<D>(l32)) << 4);
    const int vr = 4 * h + ((lane & 15) >> 2);
    int voff = vr * D * 2 +
               (((dim0 / 8 + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ value_swizzle<D>(vr)) << 4) +
               8 * (lane & 1);

    f32x16 s[NK];
    auto scores = [&](const __bf16 *Ks) {
#pragma unroll
        for (int kb = 0; kb < NK; ++kb) {
            f32x16 big, rest;
#pragma unroll
            for (int r = 0; r < 16; ++r) big[r] = rest[r] = 0.f;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const __bf16 *at = (const __bf16 *)((const char *)Ks + (koff ^ (32 * b)));
                bf16x8 k[P];
#pragma unroll
                for (int i = 0; i < P; ++i) k[i] = *(const bf16x8 *)(at + i * KT * D + kb * 32 * D);
                big = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[0], q[0][b], big, 0, 0, 0);
                if constexpr (P == 3) {
                    rest = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[2], q[0][b], rest, 0, 0, 0);
                    rest = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[0], q[P - 1][b], rest, 0, 0, 0);
                    rest = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[1], q[P / 2][b], rest, 0, 0, 0);
                    rest = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[1], q[0][b], rest, 0, 0, 0);
                    rest = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[0], q[P / 2][b], rest, 0, 0, 0);
                }
            }
            if constexpr (P == 3) {
                // an infinite score is what its high parts give (the others' products
                // with it may be 0 * inf)
#pragma unroll
                for (int r = 0; r < 16; ++r) big[r] += isfinite(big[r]) ? rest[r] : 0.f;
            }
            s[kb] = big;
            if constexpr (DS > 1) {
#pragma unroll
                for (int r = 0; r < 16; r += 4)
                    Sx[((wave * NK + kb) * 4 + r / 4) * 64 + lane] =
                        f32x4{big[r], big[r + 1], big[r + 2], big[r + 3]};
            }
        }
    };
    bf16x8 pr[P][NK][2];  // the tile's weights
    auto weigh = [&](int k0, bool all) {
        if constexpr (DS > 1) {
#pragma unroll
            for (int kb = 0; kb < NK; ++kb)
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const f32x4 x = Sx[(((wave ^ 1) * NK + kb) * 4 + r / 4) * 64 + lane];
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[kb][r + e] += x[e];
                }
        }
        // scores in log2 units are s * mul + add
        float mul = to_log2, add = 0.f;
        // A capped score is capl - 2 capl r, r = 1 / (e^2y + 1): without a bias
        // r stays, and the line goes into the exponent's.
        const bool falling = CAP && P == 1 && !a.slopes;
        if (falling) {
            mul = -2.f * capl;
            add = capl;
        }
        if (CAP || a.slopes || !all) {
#pragma unroll
            for (int kb = 0; kb < NK; ++kb)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    if constexpr (CAP && P == 1)
                        s[kb][r] = __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(s[kb][r] * to2x) + 1.f);
                    else if constexpr (CAP)
                        s[kb][r] = capped(s[kb][r], to2x, capl);
                    else
                        s[kb][r] *= to_log2;
                }
            if (!falling) mul = 1.f;
            if (a.slopes) {
                const float d0 = (float)(p - k0 - 4 * h);
#pragma unroll
                for (int kb = 0; kb < NK; ++kb)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        if constexpr (CAP && P == 1) s[kb][r] = __builtin_fmaf(s[kb][r], -2.f * capl, capl);
                        s[kb][r] = __builtin_fmaf(
                            -slope, fabsf(d0 - (float)(32 * kb + 8 * (r >> 2) + (r & 3))), s[kb][r]);
                    }
            }
            if (!all) {
                const float hidden = falling ? INFINITY : -INFINITY;
#pragma unroll
                for (int kb = 0; kb < NK; ++kb)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        // key - lo as an unsigned number is at most hi - lo inside
                        const int key = k0 + 4 * h + 32 * kb + 8 * (r >> 2) + (r & 3);
                        const bool vis = (key < w.prefix) | ((uint32_t)(key - lo) < span);
                        s[kb][r] = vis ? s[kb][r] : hidden;
                    }
            }
        }
        auto exponentials = [&]() {  // the weights, and this lane's sum of them
            const float base = add - (m_ref == -INFINITY ? 0.f : m_ref);
            float psum = 0.f;
#pragma unroll
            for (int kb = 0; kb < NK; ++kb)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    float e[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][8 * u + i], mul, base));
                        if constexpr (LSE || P == 3) psum += e[i];
                    }
                    if constexpr (P == 1) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) pr[0][kb][u][i] = (__bf16)e[i];
                        if constexpr (!LSE) {
#pragma unroll
                            for (int i = 0; i < 8; i += 2)
                                psum = __builtin_amdgcn_fdot2_f32_bf16(
                                    bf16x2{pr[0][kb][u][i], pr[0][kb][u][i + 1]},
                                    bf16x2{(__bf16)1.f, (__bf16)1.f}, psum, false);
                        }
                    } else {
                        u32x4 pl[P];
#pragma unroll
                        for (int i = 0; i < 8; i += 2) {
                            uint32_t x[3];
                            split3<true>(e[i], e[i + 1], x);
#pragma unroll
                            for (int j = 0; j < P; ++j) pl[j][i / 2] = x[j];
                        }
#pragma unroll
                        for (int j = 0; j < P; ++j) pr[j][kb][u] = __builtin_bit_cast(bf16x8, pl[j]);
                    }
                }
            return psum;
        };
        // With the maximum of before, where there is one: weights that have not
        // grown too large need no new one.
        bool renew = __ballot(m_ref == -INFINITY) != 0;
        float psum = 0.f;
        if (!renew) {
            psum = exponentials();
            renew = __ballot(!(psum <= MOST_SUM)) != 0;
        }
        if (renew) {
            float most = -INFINITY, least = INFINITY;
#pragma unroll
            for (int kb = 0; kb < NK; ++kb)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    most = fmaxf(most, s[kb][r]);
                    if constexpr (CAP && P == 1) least = fminf(least, s[kb][r]);
                }
            const float m_new = fmaxf(m_ref, other_half_max(falling ? __builtin_fmaf(least, mul, add) : most * mul));
            const float alpha = m_ref == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_ref - m_new);
            l_run *= alpha;
#pragma unroll
            for (int d = 0; d < NT; ++d) o[d] = o[d] * alpha;
            m_ref = m_new;
            psum = exponentials();
        }
        l_run += psum;
    };
    auto gather = [&](const __bf16 *Vs) {  // weights times values
#pragma unroll
        for (int d = 0; d < NT; ++d) {
            const __bf16 *tile = (const __bf16 *)((const char *)Vs + (voff ^ (64 * d)));
            f32x16 rest;
            if constexpr (P == 3) {
#pragma unroll
                for (int r = 0; r < 16; ++r) rest[r] = 0.f;
            }
#pragma unroll
            for (int kb = 0; kb < NK; ++kb)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    bf16x8 v[P];
#pragma unroll
                    for (int i = 0; i < P; ++i) {
                        const __bf16 *at = tile + i * KT * D + (32 * kb + 16 * u) * D;
                        v[i] = __builtin_shufflevector(read_transposed_bf16(at),
                                                       read_transposed_bf16(at + 8 * D), 0, 1, 2,
                                                       3, 4, 5, 6, 7);
                    }
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v[0], pr[0][kb][u], o[d], 0, 0, 0);
                    if constexpr (P == 3) {
                        rest = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v[2], pr[0][kb][u], rest, 0, 0, 0);
                        rest = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v[0], pr[P - 1][kb][u], rest, 0, 0, 0);
                        rest = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v[1], pr[P / 2][kb][u], rest, 0, 0, 0);
                        rest = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v[1], pr[0][kb][u], rest, 0, 0, 0);
                        rest = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v[0], pr[P / 2][kb][u], rest, 0, 0, 0);
                    }
                }
            if constexpr (P == 3) o[d] = o[d] + rest;
        }
    };

    if (threadIdx.x == 0) dirty = 0;
    __syncthreads();
    bool redo = false;
    // V(t) has landed in the thread's part: whether values that are hidden from
    // some of the workgroup's queries are finite. They must not reach those
    // queries through a product 0 * inf.
    auto inspect = [&](const __bf16 *Vs, int t, int k0) {
        const bool mixed = !(k0 + KT <= w.prefix ||
                             (k0 >= wg_all_lo && min(k0 + KT, w.k_len) - 1 <= wg_all_hi));
        if (mixed && __ballot(vc.non_finite(Vs)) != 0 && lane == 0) dirty = t + 1;
        return mixed;
    };
    // after a barrier: true where they are not, and the rows are to be redone
    auto spoilt = [&](bool mixed, int t) {
        redo = mixed && uniform(*(volatile int *)&dirty) == t + 1;
        return redo;
    };
    auto sees = [&](int k0) { return some && (k0 < w.prefix || (k0 <= any_hi && k0 + KT > any_lo)); };
    auto sees_all = [&](int k0) {
        return k0 + KT <= w.prefix || (k0 >= all_lo && k0 + KT - 1 <= all_hi);
    };
    if constexpr (STAGES == 2) {
        auto step = [&](int t, __bf16 *Ks, __bf16 *Vs, __bf16 *Kn, __bf16 *Vn) {
            const int k0 = key_of(t);
            asm volatile("" : "+v"(koff), "+v"(voff));  // no hoisting of what follows from them
            kc.commit(Ks);
            vc.commit(Vs);
            const bool mixed = inspect(Vs, t, k0);
            __syncthreads();  // tile t has landed; no wave reads tile t - 1 any more
            if (spoilt(mixed, t)) return;
            if (t + 1 < w.t1) {
                fetch_k(key_of(t + 1), Kn);
                fetch_v(key_of(t + 1), Vn);
            }
            const bool seen = sees(k0);
            if (seen) scores(Ks);
            if constexpr (DS > 1) __syncthreads();  // the other wave's part of the scores
            if (seen) {
                weigh(k0, sees_all(k0));
                gather(Vs);
            }
        };
        if (w.t0 < w.t1) {
            fetch_k(key_of(w.t0), K0);
            fetch_v(key_of(w.t0), V0);
        }
        for (int t = w.t0; t < w.t1; t += 2) {
            step(t, K0, V0, K1, V1);
            if (redo || t + 1 >= w.t1) break;
            step(t + 1, K1, V1, K0, V0);
            if (redo) break;
        }
    } else if constexpr (STAGES == 0) {
        for (int t = w.t0; t < w.t1; ++t) {
            const int k0 = key_of(t);
            asm volatile("" : "+v"(koff), "+v"(voff));
            fetch_k(k0, K0);
            kc.commit(K0);
            __syncthreads();
            const bool seen = sees(k0);
            if (seen) scores(K0);
            __syncthreads();  // no wave reads K any more
            fetch_v(k0, K0);
            if (seen) weigh(k0, sees_all(k0));
            vc.commit(K0);
            const bool mixed = inspect(K0, t, k0);
            __syncthreads();
            if (spoilt(mixed, t)) break;
            if (seen) gather(K0);
            __syncthreads();  // nor V
        }
    } else {
        if (w.t0 < w.t1) {
            fetch_k(key_of(w.t0), K0);
            kc.commit(K0);
        }
        __syncthreads();
        for (int t = w.t0; t < w.t1; ++t) {
            const int k0 = key_of(t);
            asm volatile("" : "+v"(koff), "+v"(voff));
            fetch_v(k0, V0);
            const bool seen = sees(k0);
            if (seen) scores(K0);
            vc.commit(V0);
            const bool mixed = inspect(V0, t, k0);
            __syncthreads();  // V has landed; no wave reads K any more
            if (spoilt(mixed, t)) break;
            if (t + 1 < w.t1) fetch_k(key_of(t + 1), K0);
            if (seen) {
                weigh(k0, sees_all(k0));
                gather(V0);
            }
            if (t + 1 < w.t1) kc.commit(K0);
            __syncthreads();  // K has landed; no wave reads V any more
        }
    }

    l_run = other_half_sum(l_run);
    float *part = w.slot < 0 ? nullptr : a.partial + w.slot * masked_slot(VECTORS, D);
    if (redo) {
        for (int i = wave; i < VECTORS && w.v0 + i < nvec; i += WAVES)
            masked_row<T, D / 64>(a, w, w.v0 + i, KT, part ? part + i * D : nullptr,
                                  part ? part + VECTORS * D + 2 * i : nullptr);
        return;
    }
    if (!valid) return;
    const int local = wave / DS * 32 + l32;
    if (part) {
#pragma unroll
        for (int d = 0; d < NT; ++d)
#pragma unroll
            for (int r = 0; r < 16; r += 4)
                *(f32x4 *)(part + local * D + dim0 + 32 * d + 2 * r + 4 * h) =
                    f32x4{o[d][r], o[d][r + 1], o[d][r + 2], o[d][r + 3]};
        if (h == 0 && dim0 == 0) {
            part[VECTORS * D + 2 * local] = m_ref;
            part[VECTORS * D + 2 * local + 1] = l_run;
        }
        return;
    }
    if (l_run == 0.f) {  // nothing seen (or scores of -inf alone, whose 0 * v may be NaN)
#pragma unroll
        for (int d = 0; d < NT; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
    }
    const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
    const int64_t qrow = (int64_t)w.q_row + qi;
    T *row = (T *)a.out + qrow * a.o_tok + head * a.o_head;
#pragma unroll
    for (int d = 0; d < NT; ++d)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int dim = dim0 + 32 * d + 2 * r + 4 * h;
            typename Row<T, 4>::type y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = (T)(o[d][r + e] * inv);
            if (a.whole) {
                if (dim < a.hd) *(typename Row<T, 4>::type *)(row + dim) = y;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (dim + e < a.hd) row[dim + e] = y[e];
            }
        }
    if (a.lse && h == 0 && dim0 == 0)
        a.lse[qrow * a.heads + head] =
            l_run == 0.f ? -INFINITY : (m_ref + __builtin_amdgcn_logf(l_run)) * 0.6931471805599453f;
#endif
}

// Keys of a tile of the kernel of few queries.
constexpr int few_keys(int dim) { return 8192 / dim; }
constexpr int FEW_PARTS = 8;

// ---- few float queries over many keys ---------------------------------------------

// Up to NV query vectors of a document and KV head against a range of
// keys: the bytes of K and V bound it, and with so few queries a matrix tile
// would be mostly empty (and three parts of every key more work than the key
// itself). 16 lanes take a key, E = D / 16 dims each, so a wave loads four
// keys at once straight into registers and sums a score with four lane
// exchanges; the keys of a 16-lane group keep a softmax state of their own, and
// groups and waves are joined at the end. A group's keys of a tile, two of 256
// dims, four of 128 or eight of 64, are loaded together.
template <class T, int D, int NV, bool WHOLE>
__global__ __launch_bounds__(256, 2) void masked_few_kernel(MaskedArgs a) {
    constexpr int E = D / 16, KT = few_keys(D), KG = KT / 16;
    __shared__ float out_s[4][NV][D];
    __shared__ float ml_s[4][NV][2];
    const AttnWork w = a.work[blockIdx.x];
    const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
    const int l16 = lane & 15, g = lane >> 4;
    const int G = a.heads / a.kv_heads;
    const int nvec = min(w.q_len * G - w.v0, NV);
    const int shift = w.k_len - w.q_len;
    // dims of a lane: 4 from every 64
    float q[NV][E], o[NV][E], m[NV], l[NV], slope[NV];
    int pos[NV], lo[NV], hi[NV];
    auto load = [&](const T *row, float (&x)[E]) {
#pragma unroll
        for (int c = 0; c < E; c += 4) {
            const int d = 16 * c + 4 * l16;
            if constexpr (WHOLE) {
                typename Row<T, 4>::type v = {};
                if (d < a.hd) v = *(const typename Row<T, 4>::type *)(row + d);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[c + e] = (float)v[e];
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[c + e] = d + e < a.hd ? (float)row[d + e] : 0.f;
            }
        }
    };
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int vec = w.v0 + min(v, nvec - 1);
        const int qi = vec / G, head = w.kvh * G + (vec - qi * G);
        load((const T *)a.q + (int64_t)(w.q_row + qi) * a.q_tok + head * a.q_head, q[v]);
        const int p = qi + shift;
        pos[v] = p;
        lo[v] = a.window >= 0 ? (int)max((int64_t)p - a.window, (int64_t)0) : 0;
        int64_t last = w.k_len - 1;
        if (a.causal) last = min(last, (int64_t)p);
        if (a.window >= 0) last = min(last, (int64_t)p + a.window);
        hi[v] = (int)max(last, (int64_t)-1);
        slope[v] = a.slopes ? a.slopes[head] * LOG2E : 0.f;
        m[v] = -INFINITY;
        l[v] = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            q[v][e] *= a.scale * (a.cap > 0.f ? 1.f : LOG2E);
            o[v][e] = 0.f;
        }
    }
    const T *kbase = (const T *)a.k + w.k_row * a.k_tok + w.kvh * a.k_head;
    const T *vbase = (const T *)a.v + w.k_row * a.v_tok + w.kvh * a.v_head;
    const float to2x = a.cap > 0.f ? fminf(2.f * LOG2E / a.cap, 3e38f) : 0.f, capl = a.cap * LOG2E;
    for (int t = w.t0; t < w.t1; ++t) {
        const int k0 = (t < w.pre_tiles ? t * KT : w.main_key + (t - w.pre_tiles) * KT) + 4 * KG * wave + g;
        float k[KG][E], v[KG][E], s[KG][NV];
#pragma unroll
        for (int i = 0; i < KG; ++i) {  // keys past the end: the last one, hidden below
            const int64_t key = min(k0 + 4 * i, w.k_len - 1);
            load(kbase + key * a.k_tok, k[i]);
        }
#pragma unroll
        for (int i = 0; i < KG; ++i) {
            const int64_t key = min(k0 + 4 * i, w.k_len - 1);
            load(vbase + key * a.v_tok, v[i]);
        }
#pragma unroll
        for (int i = 0; i < KG; ++i)
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                s[i][j] = -INFINITY;
                if (j >= nvec) continue;
                float x = 0.f;
#pragma unroll
                for (int e = 0; e < E; ++e) x = __builtin_fmaf(q[j][e], k[i][e], x);
                x = group_reduce<16, false>(x);
                if (a.cap > 0.f) x = capped(x, to2x, capl);
                const int key = k0 + 4 * i;
                if (a.slopes) x -= slope[j] * fabsf((float)(pos[j] - key));
                const bool vis = key < w.k_len && (key < w.prefix || (key >= lo[j] && key <= hi[j]));
                s[i][j] = vis ? x : -INFINITY;
            }
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if (j >= nvec) continue;
            float top = m[j];
#pragma unroll
            for (int i = 0; i < KG; ++i) top = fmaxf(top, s[i][j]);
            const float base = top == -INFINITY ? 0.f : top;
            const float f = __builtin_amdgcn_exp2f(m[j] - base);
            m[j] = top;
            l[j] *= f;
#pragma unroll
            for (int e = 0; e < E; ++e) o[j][e] *= f;
#pragma unroll
            for (int i = 0; i < KG; ++i) {
                const float p = __builtin_amdgcn_exp2f(s[i][j] - base);
                l[j] += p;
                // a hidden key's value may be anything
                const bool vis = s[i][j] != -INFINITY;
#pragma unroll
                for (int e = 0; e < E; ++e) o[j][e] += vis ? p * v[i][e] : 0.f;
            }
        }
    }
    // the wave's four groups, then the four waves
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const float top = group_max4(m[j]);
        const float f = __builtin_amdgcn_exp2f(m[j] - (top == -INFINITY ? 0.f : top));
        const float sum = group_sum4(l[j] * f);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float x = group_sum4(o[j][e] * f);
            if (g == 0) out_s[wave][j][16 * (e & ~3) + 4 * l16 + (e & 3)] = x;
        }
        if (lane == 0) {
            ml_s[wave][j][0] = top;
            ml_s[wave][j][1] = sum;
        }
    }
    __syncthreads();
    for (int j = wave; j < nvec; j += 4) {
        float top = -INFINITY, sum = 0.f, f[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, ml_s[i][j][0]);
        const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[i] = __builtin_amdgcn_exp2f(ml_s[i][j][0] - base);
            sum += f[i] * ml_s[i][j][1];
        }
        const int vec = w.v0 + j, qi = vec / G, head = w.kvh * G + (vec - qi * G);
        const int64_t qrow = (int64_t)w.q_row + qi;
        T *row = (T *)a.out + qrow * a.o_tok + head * a.o_head;
        float *part = w.slot < 0 ? nullptr : a.partial + w.slot * masked_slot(NV, D);
#pragma unroll
        for (int e = 0; e < D / 64; ++e) {
            const int d = lane + 64 * e;
            float x = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) x += f[i] * out_s[i][j][d];
            if (part) part[j * D + d] = x;
            else if (d < a.hd) row[d] = (T)(sum == 0.f ? 0.f : x / sum);
        }
        if (lane == 0) {
            if (part) {
                part[NV * D + 2 * j] = top;
                part[NV * D + 2 * j + 1] = sum;
            } else if (a.lse) {
                a.lse[qrow * a.heads + head] =
                    sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
            }
        }
    }
}

// Joins the parts of split work: 2^(m - max m) of each part's output and sum.
// A workgroup takes 32 dims of a vector. The parts' weights are found once, in
// LDS; then eight lanes (four dims each) read a part, 32 parts at once and eight
// rounds of them in flight: what it takes is a few dependent loads.
template <class T>
__global__ __launch_bounds__(256) void masked_join_kernel(MaskedArgs a, MaskedShape shape) {
    __shared__ float f_s[MASKED_MOST_PARTS];
    __shared__ f32x4 acc_s[4][8];
    __shared__ float red_s[2][4];
    const AttnJoin w = a.join[blockIdx.x];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int l8 = threadIdx.x & 7, group = threadIdx.x >> 3;
    const int G = a.heads / a.kv_heads;
    const int local = blockIdx.y, vec = w.v0 + local, dim = blockIdx.z * 32 + 4 * l8;
    if (vec >= w.q_len * G) return;
    const int qi = vec / G, head = w.kvh * G + (vec - qi * G);
    const int64_t slot = masked_slot(shape.vectors, shape.dim);
    const float *part = a.partial + w.slot * slot;
    const float *ml = part + shape.vectors * shape.dim + 2 * local;
    float m[MASKED_MOST_PARTS / 256], l[MASKED_MOST_PARTS / 256], top = -INFINITY;
#pragma unroll
    for (int r = 0; r < MASKED_MOST_PARTS / 256; ++r) {
        const int i = threadIdx.x + 256 * r;
        m[r] = i < w.parts ? ml[i * slot] : -INFINITY;
        l[r] = i < w.parts ? ml[i * slot + 1] : 0.f;
        top = fmaxf(top, m[r]);
    }
    top = wave_max(top);
    if (lane == 0) red_s[0][wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red_s[0][0], red_s[0][1]), fmaxf(red_s[0][2], red_s[0][3]));
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
#pragma unroll
    for (int r = 0; r < MASKED_MOST_PARTS / 256; ++r) {
        const float f = __builtin_amdgcn_exp2f(m[r] - base);
        f_s[threadIdx.x + 256 * r] = f;
        sum += f * l[r];
    }
    sum = wave_sum(sum);
    if (lane == 0) red_s[1][wave] = sum;
    __syncthreads();
    sum = (red_s[1][0] + red_s[1][1]) + (red_s[1][2] + red_s[1][3]);
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int i = group; i < w.parts; i += 32)
        acc = acc + *(const f32x4 *)(part + i * slot + local * shape.dim + dim) * f_s[i];
#pragma unroll
    for (int e = 0; e < 4; ++e) {  // the wave's eight groups
        acc[e] += dpp_mov<0x128>(acc[e]);  // row_ror 8: the other half of 16 lanes
        acc[e] = group_sum4(acc[e]);
    }
    if (lane < 8) acc_s[wave][l8] = acc;
    __syncthreads();
    if (threadIdx.x >= 8) return;
    acc = (acc_s[0][l8] + acc_s[1][l8]) + (acc_s[2][l8] + acc_s[3][l8]);
    const int64_t qrow = (int64_t)w.q_row + qi;
    T *row = (T *)a.out + qrow * a.o_tok + head * a.o_head;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (dim + e < a.hd) row[dim + e] = (T)(sum == 0.f ? 0.f : acc[e] / sum);
    if (a.lse && dim == 0)
        a.lse[qrow * a.heads + head] =
            sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
}

// The same for at most FEW_PARTS parts of many vectors: D / 4 lanes take a
// vector's dims and go over the parts.
template <class T>
__global__ __launch_bounds__(256) void masked_join_few_kernel(MaskedArgs a, MaskedShape shape) {
    const AttnJoin w = a.join[blockIdx.x];
    const int lanes = shape.dim / 4, each = 256 / lanes;
    const int local = blockIdx.y * each + (int)threadIdx.x / lanes, vec = w.v0 + local;
    const int dim = (int)threadIdx.x % lanes * 4;
    const int G = a.heads / a.kv_heads;
    if (local >= shape.vectors || vec >= w.q_len * G) return;
    const int qi = vec / G, head = w.kvh * G + (vec - qi * G);
    const int64_t slot = masked_slot(shape.vectors, shape.dim);
    const float *part = a.partial + w.slot * slot;
    const float *ml = part + shape.vectors * shape.dim + 2 * local;
    float m[FEW_PARTS], l[FEW_PARTS], top = -INFINITY, sum = 0.f;
    f32x4 x[FEW_PARTS], acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < FEW_PARTS; ++i) {
        const bool in = i < w.parts;
        m[i] = in ? ml[i * slot] : -INFINITY;
        l[i] = in ? ml[i * slot + 1] : 0.f;
        x[i] = in ? *(const f32x4 *)(part + i * slot + local * shape.dim + dim) : acc;
        top = fmaxf(top, m[i]);
    }
    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int i = 0; i < FEW_PARTS; ++i) {
        const float f = __builtin_amdgcn_exp2f(m[i] - base);
        sum += f * l[i];
        acc = acc + x[i] * f;
    }
    const int64_t qrow = (int64_t)w.q_row + qi;
    T *row = (T *)a.out + qrow * a.o_tok + head * a.o_head;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (dim + e < a.hd) row[dim + e] = (T)(sum == 0.f ? 0.f : acc[e] / sum);
    if (a.lse && dim == 0)
        a.lse[qrow * a.heads + head] =
            sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
}

// What a batch is run by:
//  * head dims above 512: a wave a query.
//  * up to eight float queries of a document and KV head (four of 512 dims): straight from
//    registers (a matrix tile of them took 756 us for 200003 keys, 82 this way);
//    bfloat16 ones are as fast as the bytes on the matrix cores, 32 to a
//    workgroup of one wave (4 queries of 128 dims over 2000-8192 keys of 64
//    requests: 128 us, 358 from registers, where the vector work is the bound).
//  * else 128 queries to a workgroup. Tiles of 32 keys leave room for a third
//    workgroup a CU at 128 dims (prefix mask 1139 -> 1111 us), of 64 for a
//    fourth at 64 dims (1264 us with tiles of 32, 1137).
MaskedShape masked_shape(bool bf16, int hd, int64_t most) {
    if (hd > 512) return {0, 16, ROW_KEYS, 0, 2048, 16};
    const int dim = hd <= 64 ? 64 : hd <= 128 ? 128 : hd <= 256 ? 256 : 512;
    if (bf16) {
        const int planes = hd % 8 ? 1 : 0;
        if (most <= 32) return {dim, 32, dim >= 256 ? 32 : 64, planes, dim == 512 ? 512 : 1280, 1};
        return {dim, 128, dim == 64 ? 64 : 32, planes, dim == 64 ? 1024 : dim == 128 ? 768 : dim == 256 ? 512 : 256, 8};
    }
    // (a workgroup's registers hold 8, 4 or 2 of them; the rest of 8 are a second group's)
    if (most <= (dim == 512 ? 4 : 8)) {
        const int held = dim == 512 ? 2 : dim == 256 ? 4 : 8;
        return {dim, most <= 1 ? 1 : std::min(held, most <= 4 ? 4 : 8), few_keys(dim), 0, 512, 1};
    }
    return {dim, dim == 512 ? 64 : 128, 32, 3, dim == 64 ? 512 : 256, 8};
}

template <class T, int P, int D, int KT, int WAVES, int DS, int STAGES, TileSource FROM, int MINW,
          bool CAP>
static hipError_t launch_tiles_capped(const MaskedArgs &a, hipStream_t s) {
    const dim3 grid((unsigned)a.n_work), block(64 * WAVES);
    // The sum of rounded weights costs half as much and is what the rounded
    // products are to be divided by, but no lse; it is worth a kernel of its own
    // where vector work bounds it (video 1197 -> 1168 us), not where keys' bytes do.
    constexpr bool ROUNDED = P == 1 && WAVES / DS > 1 && FROM == FROM_ROWS;
    if (ROUNDED && !a.lse)
        hipLaunchKernelGGL((masked_tile_kernel<T, P, D, KT, WAVES, DS, STAGES, FROM, CAP, !ROUNDED, MINW>),
                           grid, block, 0, s, a);
    else
        hipLaunchKernelGGL((masked_tile_kernel<T, P, D, KT, WAVES, DS, STAGES, FROM, CAP, true, MINW>),
                           grid, block, 0, s, a);
    return hipGetLastError();
}

template <class T, int P, int D, int KT, int WAVES, int DS, int STAGES, TileSource FROM, int MINW>
static hipError_t launch_tiles(const MaskedArgs &a, hipStream_t s) {
    return a.cap > 0.f
               ? launch_tiles_capped<T, P, D, KT, WAVES, DS, STAGES, FROM, MINW, true>(a, s)
               : launch_tiles_capped<T, P, D, KT, WAVES, DS, STAGES, FROM, MINW, false>(a, s);
}

template <TileSource FROM>
static hipError_t launch_bf16(const MaskedArgs &a, const MaskedShape &shape, hipStream_t s) {
    const bool few = shape.vectors == 32;
    switch (shape.dim) {
        case 64:
            return few ? launch_tiles<__bf16, 1, 64, 64, 1, 1, 2, FROM, 1>(a, s)
                       : launch_tiles<__bf16, 1, 64, 64, 4, 1, 2, FROM, 4>(a, s);
        case 128:
            return few ? launch_tiles<__bf16, 1, 128, 64, 1, 1, 2, FROM, 1>(a, s)
                       : launch_tiles<__bf16, 1, 128, 32, 4, 1, 2, FROM, 3>(a, s);
        case 256:
            // (one stage: 64 x 2000-8192 keys, 3 heads: 78 us, 85 with two, of which a CU
            // holds two workgroups)
            return few ? launch_tiles<__bf16, 1, 256, 32, 1, 1, 1, FROM, 1>(a, s)
                       : launch_tiles<__bf16, 1, 256, 32, 4, 1, 2, FROM, 2>(a, s);
        case 512:
            return few ? launch_tiles<__bf16, 1, 512, 32, 2, 2, 1, FROM, 1>(a, s)
                       : launch_tiles<__bf16, 1, 512, 32, 8, 2, 1, FROM, 2>(a, s);
    }
    return hipErrorInvalidValue;
}

template <int D, int NV>
static hipError_t launch_few(const MaskedArgs &a, hipStream_t s) {
    const dim3 grid((unsigned)a.n_work), block(256);
    if (a.whole) hipLaunchKernelGGL((masked_few_kernel<float, D, NV, true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((masked_few_kernel<float, D, NV, false>), grid, block, 0, s, a);
    return hipGetLastError();
}

template <class T, int P, int D, int KT>
static hipError_t launch_planes(const MaskedArgs &a, hipStream_t s) {
    if (a.n_tiles > 0)
        hipLaunchKernelGGL((masked_planes_kernel<T, P, D, KT>), dim3((unsigned)a.n_tiles, 2), dim3(256),
                           0, s, a);
    return hipGetLastError();
}

static hipError_t launch_float(const MaskedArgs &a, const MaskedShape &shape, hipStream_t s) {
    if (shape.planes == 0) switch (shape.dim * 16 + shape.vectors) {
        case 64 * 16 + 1: return launch_few<64, 1>(a, s);
        case 64 * 16 + 4: return launch_few<64, 4>(a, s);
        case 64 * 16 + 8: return launch_few<64, 8>(a, s);
        case 128 * 16 + 1: return launch_few<128, 1>(a, s);
        case 128 * 16 + 4: return launch_few<128, 4>(a, s);
        case 128 * 16 + 8: return launch_few<128, 8>(a, s);
        case 256 * 16 + 1: return launch_few<256, 1>(a, s);
        case 256 * 16 + 4: return launch_few<256, 4>(a, s);
        case 512 * 16 + 1: return launch_few<512, 1>(a, s);
        case 512 * 16 + 2: return launch_few<512, 2>(a, s);
        default: return hipErrorInvalidValue;
    }
    switch (shape.dim) {
        case 64: return launch_tiles<float, 3, 64, 32, 4, 1, 2, FROM_PLANES, 2>(a, s);
        case 128: return launch_tiles<float, 3, 128, 32, 8, 2, 2, FROM_PLANES, 2>(a, s);
        case 256: return launch_tiles<float, 3, 256, 32, 8, 2, 1, FROM_PLANES, 2>(a, s);
        case 512: return launch_tiles<float, 3, 512, 32, 4, 2, 0, FROM_PLANES, 1>(a, s);
    }
    return hipErrorInvalidValue;
}

static hipError_t launch_planes_of(const MaskedArgs &a, bool bf16, const MaskedShape &shape,
                                   hipStream_t s) {
    if (!bf16) switch (shape.dim) {
        case 64: return launch_planes<float, 3, 64, 32>(a, s);
        case 128: return launch_planes<float, 3, 128, 32>(a, s);
        case 256: return launch_planes<float, 3, 256, 32>(a, s);
        case 512: return launch_planes<float, 3, 512, 32>(a, s);
        default: return hipErrorInvalidValue;
    }
    switch (shape.dim * 64 + shape.keys) {
        case 64 * 64 + 64: return launch_planes<__bf16, 1, 64, 64>(a, s);
        case 128 * 64 + 64: return launch_planes<__bf16, 1, 128, 64>(a, s);
        case 128 * 64 + 32: return launch_planes<__bf16, 1, 128, 32>(a, s);
        case 256 * 64 + 32: return launch_planes<__bf16, 1, 256, 32>(a, s);
        case 512 * 64 + 32: return launch_planes<__bf16, 1, 512, 32>(a, s);
    }
    return hipErrorInvalidValue;
}

template <class T>
static hipError_t launch_rows(const MaskedArgs &a, int vectors, hipStream_t s) {
    const dim3 grid((unsigned)a.n_work), block(256);
    hipLaunchKernelGGL(masked_rows_kernel<T>, grid, block, 0, s, a, vectors);
    return hipGetLastError();
}

hipError_t launch_masked_attention(MaskedArgs a, bool bf16, const MaskedShape &shape,
                                   hipStream_t s) {
    if (a.n_work <= 0) return hipSuccess;
    if (shape.dim == 0) return bf16 ? launch_rows<__bf16>(a, shape.vectors, s)
                                    : launch_rows<float>(a, shape.vectors, s);
    // whole 16-byte chunks at 16-byte addresses
    const int64_t size = bf16 ? 2 : 4, n = 16 / size;
    a.whole = a.hd % n == 0;
    for (const void *p : {a.q, a.k, a.v, (const void *)a.out}) a.whole = a.whole && (uintptr_t)p % 16 == 0;
    for (int64_t st : {a.q_tok, a.q_head, a.k_tok, a.k_head, a.v_tok, a.v_head, a.o_tok, a.o_head})
        a.whole = a.whole && st % n == 0;
    hipError_t e = shape.planes > 0 ? launch_planes_of(a, bf16, shape, s) : hipSuccess;
    if (e != hipSuccess) return e;
    e = !bf16             ? launch_float(a, shape, s)
        : shape.planes > 0 ? launch_bf16<FROM_PLANES>(a, shape, s)
        : a.whole          ? launch_bf16<FROM_ROWS>(a, shape, s)
                           : launch_bf16<FROM_PIECES>(a, shape, s);
    if (e != hipSuccess || a.n_join == 0) return e;
    const unsigned joins = (unsigned)a.n_join, vectors = (unsigned)a.join_vectors;
    // (the other kernel's workgroup for each 32 dims of a vector takes 80 us for some 4 parts of 200
    // groups of 128 queries, which this one joins in a few; a thousand parts want its 32 readers)
    if (a.join_parts <= FEW_PARTS) {
        const unsigned each = 1024u / (unsigned)shape.dim;
        const dim3 grid(joins, (vectors + each - 1) / each), block(256);
        if (bf16) hipLaunchKernelGGL(masked_join_few_kernel<__bf16>, grid, block, 0, s, a, shape);
        else hipLaunchKernelGGL(masked_join_few_kernel<float>, grid, block, 0, s, a, shape);
    } else {
        const dim3 grid(joins, vectors, (unsigned)(shape.dim / 32)), block(256);
        if (bf16) hipLaunchKernelGGL(masked_join_kernel<__bf16>, grid, block, 0, s, a, shape);
        else hipLaunchKernelGGL(masked_join_kernel<float>, grid, block, 0, s, a, shape);
    }
    return hipGetLastError();
}

}  // namespace svl
