// Attention over packed documents with causal, window and prefix masks, a
// score cap and a distance bias (svl_masked_attention).
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

// A tile's way from HBM to LDS: fetch() starts it, commit() ends it. `P`
// planes of KT rows of D bfloat16 in LDS. Whole 16-byte chunks of bfloat16 rows
// go there by DMA; rows of another alignment and float rows go through
// registers (float ones are split on the way).
template <class T, int P, int D, int KT, int THREADS, bool WHOLE, int (*SWIZZLE)(int)>
struct TileCopy {
    static constexpr int CHUNKS = KT * D / 8;          // of eight values
    static constexpr int EACH = CHUNKS / THREADS;
    static constexpr bool DMA = WHOLE && P == 1;
    static_assert(CHUNKS % THREADS == 0, "tile");
    static constexpr int OUT = (int)0x80000000;        // an offset out of range: reads zero
    T reg[DMA ? 1 : EACH * 8];

    // chunk that this thread moves i-th: a wave's DMA fills 1 KB of LDS in a row
    __device__ __forceinline__ static int place(int i) {
        return ((int)threadIdx.x >> 6) * (64 * EACH) + 64 * i + ((int)threadIdx.x & 63);
    }
    // rows: rows of the tile that exist
    __device__ __forceinline__ void fetch(const T *base, int ld, int hd, int rows, __bf16 *lds) {
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
            (void *)uniform((T *)base), (short)0, uniform(((rows - 1) * ld + hd) * (int)sizeof(T)),
            0x00020000);
        const int wave = uniform((int)threadIdx.x >> 6);
        // found anew for each tile: the registers are worth more than the few
        // instructions
        int lane = (int)threadIdx.x & 63;
        asm volatile("" : "+v"(lane));
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int c = wave * (64 * EACH) + 64 * i + lane;
            const int r = c / (D / 8), dim = 8 * ((c % (D / 8)) ^ SWIZZLE(r));
            const int off = (r * ld + dim) * (int)sizeof(T);
            if constexpr (DMA) {
                __builtin_amdgcn_raw_ptr_buffer_load_lds(
                    rs, (__attribute__((address_space(3))) void *)(lds + (wave * EACH + i) * 512),
                    16, dim < hd ? off : OUT, 0, 0, 0);
            } else if constexpr (WHOLE) {  // float
#pragma unroll
                for (int q = 0; q < 8; q += 4) {
                    const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(
                        rs, dim + q < hd ? off + 4 * q : OUT, 0, 0);
#pragma unroll
                    for (int e = 0; e < 4; ++e) reg[8 * i + q + e] = __uint_as_float(v[e]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int o = dim + e < hd ? off + e * (int)sizeof(T) : OUT;
                    if constexpr (sizeof(T) == 2)
                        reg[8 * i + e] = __builtin_bit_cast(
                            __bf16, __builtin_amdgcn_raw_buffer_load_b16(rs, o, 0, 0));
                    else
                        reg[8 * i + e] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, o, 0, 0));
                }
            }
        }
    }
    __device__ __forceinline__ void commit(__bf16 *lds) {
        if constexpr (DMA) {
            wait_vmcnt<0>();
        } else {
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                u32x4 pl[P];
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    if constexpr (P == 1) {
                        pl[0][e / 2] = __builtin_bit_cast(uint32_t, bf16x2{reg[8 * i + e], reg[8 * i + e + 1]});
                    } else {
                        uint32_t x[3];
                        split3<false>(reg[8 * i + e], reg[8 * i + e + 1], x);
#pragma unroll
                        for (int p = 0; p < P; ++p) pl[p][e / 2] = x[p];
                    }
                }
#pragma unroll
                for (int p = 0; p < P; ++p) *(u32x4 *)(lds + p * KT * D + place(i) * 8) = pl[p];
            }
        }
    }
    // Whether this thread's part of a landed tile holds a non-finite value
    // (high parts tell).
    __device__ __forceinline__ bool non_finite(const __bf16 *lds) const {
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const u32x4 v = *(const u32x4 *)(lds + place(i) * 8);
#pragma unroll
            for (int e = 0; e < 4; ++e) any |= (v[e] & 0x7fff7fffu) + 0x00800080u;
        }
        return (any & 0x80008000u) != 0;
    }
};

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

// tanh(y) / y = 1 + q P(q), q = y^2: a Chebyshev fit of P on [0, 0.56^2], error
// of tanh 6e-9.
constexpr float TANH_C0 = -0.33333331f, TANH_C1 = 0.13333082f, TANH_C2 = -0.053903349f,
                TANH_C3 = 0.021272749f, TANH_C4 = -0.006542542f;

// cap tanh(x / cap) log2(e) from the raw product: to2x = 2 log2(e) scale / cap
// takes it to the exponent of e^(2 x / cap), capl = cap log2(e).
// tanh y = 1 - 2 / (e^2y + 1) loses the low bits of a small y (an absolute
// error of 2^-24): float scores take the series y + y^3 P(y^2) below 0.55
// (Chebyshev fit of tanh(y) / y, error 4e-8 there).
template <bool EXACT>
__device__ __forceinline__ float capped(float s, float to2x, float capl) {
    const float z = s * to2x;
    const float r = __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(z) + 1.f);
    float t = __builtin_fmaf(r, -2.f * capl, capl);
    if constexpr (EXACT) {
        const float y = z * 0.34657359028f;  // ln 2 / 2
        const float q = y * y;
        float p = __builtin_fmaf(q, TANH_C4, TANH_C3);
        p = __builtin_fmaf(q, p, TANH_C2);
        p = __builtin_fmaf(q, p, TANH_C1);
        p = __builtin_fmaf(q, p, TANH_C0);
        const float small = capl * __builtin_fmaf(y * q, p, y);
        t = fabsf(y) < 0.55f ? small : t;
    }
    return t;
}

// A workgroup takes WAVES * 32 query vectors of one document and KV head: the
// heads that share a KV head are vectors beside each other, so a tile of keys
// serves all of them. Keys stream through LDS in tiles of KT.
//  * S^T = K Q^T on 32x32x16 MFMAs, queries in registers: a lane holds 16 of
//    a block's 32 keys for one query, so that maximum and sum are a lane's own
//    but for one exchange with lane ^ 32.
//  * O^T += V^T P^T: the score registers 8 u .. 8 u + 7 are the B operand of
//    step u as they stand (keys 16 u + 4 h + 0..3 and + 8, h = lane / 32), and V
//    is read transposed in the same order.
//  * The running maximum moves only when a query's grows by more than 2^8, so
//    outputs are rarely rescaled.
//  * One LDS buffer each for K and V: V(t) comes in under the scores of tile
//    t, K(t + 1) under its softmax and P V; two barriers a tile.
// P = 1: bfloat16 operands; weights are rounded to bfloat16 for the product
// with V (a relative 2^-8 of each, the output's own step); their sum is taken
// before, so that the lse keeps its 32 bits.
// P = 3: float operands as three bfloat16 parts; of the nine products the six
// above 2^-24 are taken, the five small ones in an accumulator of their own.
template <class T, int P, int D, int KT, int WAVES, bool WHOLE, bool CAP, int MINB>
__global__ __launch_bounds__(64 * WAVES, MINB) void masked_tile_kernel(MaskedArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int NB = D / 16, NT = D / 32, NK = KT / 32;
    __shared__ __bf16 Ks[P * KT * D];
    __shared__ __bf16 Vs[P * KT * D];
    __shared__ int dirty;  // 1 + the tile whose values hold a non-finite one
    const AttnWork w = a.work[blockIdx.x];
    const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
    const int l32 = lane & 31, h = lane >> 5;
    const int G = a.heads / a.kv_heads;
    const int nvec = w.q_len * G;
    const int wv0 = w.v0 + wave * 32;          // this wave's first vector
    const bool some = wv0 < nvec;              // ... and whether it has any
    const int vec = min(wv0 + l32, nvec - 1);
    const bool valid = wv0 + l32 < nvec;
    const int qi = vec / G, head = w.kvh * G + (vec - qi * G);
    const int shift = w.k_len - w.q_len;
    const int p = qi + shift;
    const int p_lo = min(wv0, nvec - 1) / G + shift, p_hi = min(wv0 + 31, nvec - 1) / G + shift;
    const int wg_lo = w.v0 / G + shift, wg_hi = min(w.v0 + 32 * WAVES - 1, nvec - 1) / G + shift;

    // a query's keys besides the prefix: lo .. hi
    auto first_key = [&](int pos) { return a.window >= 0 ? (int)max((int64_t)pos - a.window, (int64_t)0) : 0; };
    auto last_key = [&](int pos) {
        int64_t k = w.k_len - 1;
        if (a.causal) k = min(k, (int64_t)pos);
        if (a.window >= 0) k = min(k, (int64_t)pos + a.window);
        return (int)max(k, (int64_t)-1);
    };
    const int lo = first_key(p), hi = last_key(p);

    // scores: sign of the scale into the queries, its size into the exponent
    const float size = fabsf(a.scale);
    bf16x8 q[P][NB];
    {
        const T *row = (const T *)a.q + (int64_t)(w.q_row + qi) * a.q_tok + head * a.q_head;
        const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int d = 16 * b + 8 * h;
            T x[8];
            if constexpr (WHOLE) {
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
    const float to2x = CAP ? 2.f * LOG2E * size / a.cap : 0.f, capl = a.cap * LOG2E;
    const float slope = a.slopes ? a.slopes[head] * LOG2E : 0.f;

    f32x16 o[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[t][r] = 0.f;
    float m_ref = -INFINITY, l_run = 0.f;

    const int ldk = (int)a.k_tok, ldv = (int)a.v_tok;
    const T *kbase = (const T *)a.k + w.k_row * a.k_tok + w.kvh * a.k_head;
    const T *vbase = (const T *)a.v + w.k_row * a.v_tok + w.kvh * a.v_head;
    TileCopy<T, P, D, KT, 64 * WAVES, WHOLE, key_swizzle<D>> kc;
    TileCopy<T, P, D, KT, 64 * WAVES, WHOLE, value_swizzle<D>> vc;
    auto key_of = [&](int t) { return t < w.pre_tiles ? t * KT : w.main_key + (t - w.pre_tiles) * KT; };
    auto fetch_k = [&](int k0) {
        kc.fetch(kbase + (int64_t)k0 * ldk, ldk, a.hd, min(KT, w.k_len - k0), Ks);
    };
    auto fetch_v = [&](int k0) {
        vc.fetch(vbase + (int64_t)k0 * ldv, ldv, a.hd, min(KT, w.k_len - k0), Vs);
    };
    // Lane addresses, in elements: K row l32 of a block at chunk h, V row
    // (lane % 16) / 4 of four at its chunk of a 32-dim tile. Rows start at
    // multiples of D, so another chunk (a multiple of 2 or 4 further before the
    // swizzle) is an exclusive or of the offset; it is done as each fragment is
    // read (kept in registers, the addresses would spill).
    int koff = l32 * D + ((h ^ key_swizzle<D>(l32)) << 3);
    const int vr = 4 * h + ((lane & 15) >> 2);
    int voff = vr * D + (((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ value_swizzle<D>(vr)) << 3) +
               4 * (lane & 1);

    if (threadIdx.x == 0) dirty = 0;
    bool redo = false;
    if (w.t0 < w.t1) {
        fetch_k(key_of(w.t0));
        kc.commit(Ks);
    }
    __syncthreads();
    for (int t = w.t0; t < w.t1; ++t) {
        const int k0 = key_of(t);
        asm volatile("" : "+v"(koff), "+v"(voff));  // no hoisting of what follows from them
        fetch_v(k0);
        // what of the tile this wave's queries see
        const bool in_prefix = k0 < w.prefix;
        const bool seen = some && (in_prefix || (k0 <= last_key(p_hi) && k0 + KT > first_key(p_lo)));
        const bool all = k0 + KT <= w.prefix ||
                         (k0 >= first_key(p_hi) && k0 + KT - 1 <= last_key(p_lo));
        f32x16 s[NK];
        if (seen) {
#pragma unroll
            for (int kb = 0; kb < NK; ++kb) {
                f32x16 big, rest;
#pragma unroll
                for (int r = 0; r < 16; ++r) big[r] = rest[r] = 0.f;
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const __bf16 *at = Ks + (koff ^ (16 * b));
                    bf16x8 k[P];
#pragma unroll
                    for (int i = 0; i < P; ++i)
                        k[i] = *(const bf16x8 *)(at + i * KT * D + kb * 32 * D);
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
            }
        }
        vc.commit(Vs);
        // Values hidden from some of the workgroup's queries must not reach them
        // through a product 0 * inf.
        const bool mixed = !(k0 + KT <= w.prefix ||
                             (k0 >= first_key(wg_hi) &&
                              min(k0 + KT, w.k_len) - 1 <= last_key(wg_lo)));
        if (mixed && __ballot(vc.non_finite(Vs)) != 0 && lane == 0) dirty = t + 1;
        __syncthreads();  // V has landed; no wave reads K any more
        if (mixed && uniform(*(volatile int *)&dirty) == t + 1) {
            redo = true;
            break;
        }
        if (t + 1 < w.t1) fetch_k(key_of(t + 1));
        if (seen) {
            float tmax = -INFINITY;
            auto score = [&](int kb, int r) {  // log2 units
                float x = CAP ? capped<P == 3>(s[kb][r], to2x, capl) : s[kb][r] * to_log2;
                return x;
            };
            if (CAP || a.slopes || !all) {
                const float d0 = (float)(p - k0 - 4 * h);
#pragma unroll
                for (int kb = 0; kb < NK; ++kb)
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[kb][r] = score(kb, r);
                if (a.slopes) {
#pragma unroll
                    for (int kb = 0; kb < NK; ++kb)
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            s[kb][r] = __builtin_fmaf(
                                -slope, fabsf(d0 - (float)(32 * kb + 8 * (r >> 2) + (r & 3))), s[kb][r]);
                }
                if (!all) {
#pragma unroll
                    for (int kb = 0; kb < NK; ++kb)
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const int key = k0 + 32 * kb + 8 * (r >> 2) + 4 * h + (r & 3);
                            s[kb][r] = key < w.prefix || (key >= lo && key <= hi) ? s[kb][r] : -INFINITY;
                        }
                }
#pragma unroll
                for (int kb = 0; kb < NK; ++kb)
#pragma unroll
                    for (int r = 0; r < 16; ++r) tmax = fmaxf(tmax, s[kb][r]);
            } else {
#pragma unroll
                for (int kb = 0; kb < NK; ++kb)
#pragma unroll
                    for (int r = 0; r < 16; ++r) tmax = fmaxf(tmax, s[kb][r]);
                tmax *= to_log2;
            }
            const float mul = CAP || a.slopes || !all ? 1.f : to_log2;
            tmax = other_half_max(tmax);
            const bool grow = tmax > m_ref + 8.f;
            if (__ballot(grow)) {
                const float m_new = grow ? tmax : m_ref;
                const float alpha = m_ref == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_ref - m_new);
                l_run *= alpha;
#pragma unroll
                for (int d = 0; d < NT; ++d) o[d] = o[d] * alpha;
                m_ref = m_new;
            }
            const float base = m_ref == -INFINITY ? 0.f : -m_ref;
            bf16x8 pr[P][NK][2];
            float psum = 0.f;
#pragma unroll
            for (int kb = 0; kb < NK; ++kb)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    float e[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][8 * u + i], mul, base));
                    if constexpr (P == 1) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            psum += e[i];
                            pr[0][kb][u][i] = (__bf16)e[i];
                        }
                    } else {
                        u32x4 pl[P];
#pragma unroll
                        for (int i = 0; i < 8; i += 2) {
                            uint32_t x[3];
                            psum += e[i];
                            psum += e[i + 1];
                            split3<true>(e[i], e[i + 1], x);
#pragma unroll
                            for (int j = 0; j < P; ++j) pl[j][i / 2] = x[j];
                        }
#pragma unroll
                        for (int j = 0; j < P; ++j) pr[j][kb][u] = __builtin_bit_cast(bf16x8, pl[j]);
                    }
                }
            l_run += other_half_sum(psum);
#pragma unroll
            for (int d = 0; d < NT; ++d) {
                const __bf16 *tile = Vs + (voff ^ (32 * d));
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
        }
        if (t + 1 < w.t1) kc.commit(Ks);
        __syncthreads();  // K has landed; no wave reads V any more
    }

    float *part = w.slot < 0 ? nullptr : a.partial + (int64_t)w.slot * (32 * WAVES * (D + 2));
    if (redo) {
        for (int i = wave * 32; i < wave * 32 + 32 && w.v0 + i < nvec; ++i)
            masked_row<T, D / 64>(a, w, w.v0 + i, KT, part ? part + i * D : nullptr,
                                  part ? part + 32 * WAVES * D + 2 * i : nullptr);
        return;
    }
    if (!valid) return;
    const int local = wave * 32 + l32;
    if (part) {
#pragma unroll
        for (int d = 0; d < NT; ++d)
#pragma unroll
            for (int r = 0; r < 16; r += 4)
                *(f32x4 *)(part + local * D + 32 * d + 2 * r + 4 * h) =
                    f32x4{o[d][r], o[d][r + 1], o[d][r + 2], o[d][r + 3]};
        if (h == 0) {
            part[32 * WAVES * D + 2 * local] = m_ref;
            part[32 * WAVES * D + 2 * local + 1] = l_run;
        }
        return;
    }
    const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
    const int64_t qrow = (int64_t)w.q_row + qi;
    T *row = (T *)a.out + qrow * a.o_tok + head * a.o_head;
#pragma unroll
    for (int d = 0; d < NT; ++d)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int dim = 32 * d + 2 * r + 4 * h;
            typename Row<T, 4>::type y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = (T)(l_run == 0.f ? 0.f : o[d][r + e] * inv);
            if constexpr (WHOLE) {
                if (dim < a.hd) *(typename Row<T, 4>::type *)(row + dim) = y;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (dim + e < a.hd) row[dim + e] = y[e];
            }
        }
    if (a.lse && h == 0)
        a.lse[qrow * a.heads + head] =
            l_run == 0.f ? -INFINITY : (m_ref + __builtin_amdgcn_logf(l_run)) * 0.6931471805599453f;
#endif
}

// Joins the parts of split work: a wave per vector, 2^(m - max m) of each
// part's output and sum.
template <class T>
__global__ __launch_bounds__(256) void masked_join_kernel(MaskedArgs a, MaskedShape shape) {
    const AttnJoin w = a.join[blockIdx.x];
    const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
    const int G = a.heads / a.kv_heads;
    const int local = blockIdx.y * 4 + wave;
    const int vec = w.v0 + local;
    if (local >= shape.vectors || vec >= w.q_len * G) return;
    const int qi = vec / G, head = w.kvh * G + (vec - qi * G);
    const int64_t slot = (int64_t)shape.vectors * (shape.dim + 2);  // masked_slot
    const float *part = a.partial + w.slot * slot;
    const float *ml = part + shape.vectors * shape.dim + 2 * local;
    float top = -INFINITY;
    for (int i = lane; i < w.parts; i += 64) top = fmaxf(top, ml[i * slot]);
    top = wave_max(top);
    const float base = top == -INFINITY ? 0.f : top;
    float acc[4] = {0.f, 0.f, 0.f, 0.f}, l = 0.f;
    for (int i = 0; i < w.parts; ++i) {
        const float f = __builtin_amdgcn_exp2f(ml[i * slot] - base);
        l += f * ml[i * slot + 1];
        const float *src = part + i * slot + local * shape.dim;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int d = lane + 64 * e;
            if (d < a.hd) acc[e] += f * src[d];
        }
    }
    const int64_t qrow = (int64_t)w.q_row + qi;
    T *row = (T *)a.out + qrow * a.o_tok + head * a.o_head;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int d = lane + 64 * e;
        if (d < a.hd) row[d] = (T)(l == 0.f ? 0.f : acc[e] / l);
    }
    if (a.lse && lane == 0)
        a.lse[qrow * a.heads + head] =
            l == 0.f ? -INFINITY : (top + log2f(l)) * 0.6931471805599453f;
}

MaskedShape masked_shape(bool bf16, int hd, int64_t most) {
    if (hd > 256) return {0, 16, ROW_KEYS};
    const int dim = hd <= 64 ? 64 : hd <= 128 ? 128 : 256;
    if (bf16) return {dim, most <= 32 ? 32 : 128, dim == 256 ? 32 : 64};
    return {dim, 128, dim == 64 ? 64 : 32};
}

template <class T>
static hipError_t launch_rows(const MaskedArgs &a, int vectors, hipStream_t s) {
    const dim3 grid((unsigned)a.n_work), block(256);
    hipLaunchKernelGGL(masked_rows_kernel<T>, grid, block, 0, s, a, vectors);
    return hipGetLastError();
}

template <class T, int P, int D, int KT, int WAVES, bool WHOLE, int MINB>
static hipError_t launch_tiles(const MaskedArgs &a, hipStream_t s) {
    const dim3 grid((unsigned)a.n_work), block(64 * WAVES);
    if (a.cap > 0.f) hipLaunchKernelGGL((masked_tile_kernel<T, P, D, KT, WAVES, WHOLE, true, MINB>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((masked_tile_kernel<T, P, D, KT, WAVES, WHOLE, false, MINB>), grid, block, 0, s, a);
    return hipGetLastError();
}

template <bool WHOLE>
static hipError_t launch_tiles_of(const MaskedArgs &a, bool bf16, const MaskedShape &shape,
                                  hipStream_t s) {
    if (bf16 && shape.vectors == 32) {
        switch (shape.dim) {
            case 64: return launch_tiles<__bf16, 1, 64, 64, 1, WHOLE, 1>(a, s);
            case 128: return launch_tiles<__bf16, 1, 128, 64, 1, WHOLE, 1>(a, s);
            case 256: return launch_tiles<__bf16, 1, 256, 32, 1, WHOLE, 1>(a, s);
        }
    } else if (bf16) {
        switch (shape.dim) {
            case 64: return launch_tiles<__bf16, 1, 64, 64, 4, WHOLE, 3>(a, s);
            case 128: return launch_tiles<__bf16, 1, 128, 64, 4, WHOLE, 2>(a, s);
            case 256: return launch_tiles<__bf16, 1, 256, 32, 4, WHOLE, 2>(a, s);
        }
    } else {
        switch (shape.dim) {
            case 64: return launch_tiles<float, 3, 64, 64, 4, WHOLE, 2>(a, s);
            case 128: return launch_tiles<float, 3, 128, 32, 4, WHOLE, 1>(a, s);
            case 256: return launch_tiles<float, 3, 256, 32, 4, WHOLE, 1>(a, s);
        }
    }
    return hipErrorInvalidValue;
}

hipError_t launch_masked_attention(const MaskedArgs &a, bool bf16, const MaskedShape &shape,
                                   hipStream_t s) {
    if (a.n_work <= 0) return hipSuccess;
    if (shape.dim == 0) return bf16 ? launch_rows<__bf16>(a, shape.vectors, s)
                                    : launch_rows<float>(a, shape.vectors, s);
    // whole 16-byte chunks at 16-byte addresses
    const int64_t size = bf16 ? 2 : 4, n = 16 / size;
    bool whole = a.hd % n == 0;
    for (const void *p : {a.q, a.k, a.v, (const void *)a.out}) whole = whole && (uintptr_t)p % 16 == 0;
    for (int64_t st : {a.q_tok, a.q_head, a.k_tok, a.k_head, a.v_tok, a.v_head, a.o_tok, a.o_head})
        whole = whole && st % n == 0;
    const hipError_t e = whole ? launch_tiles_of<true>(a, bf16, shape, s)
                               : launch_tiles_of<false>(a, bf16, shape, s);
    if (e != hipSuccess || a.n_join == 0) return e;
    const dim3 grid((unsigned)a.n_join, (unsigned)(shape.vectors / 4)), block(256);
    if (bf16) hipLaunchKernelGGL(masked_join_kernel<__bf16>, grid, block, 0, s, a, shape);
    else hipLaunchKernelGGL(masked_join_kernel<float>, grid, block, 0, s, a, shape);
    return hipGetLastError();
}

}  // namespace svl
