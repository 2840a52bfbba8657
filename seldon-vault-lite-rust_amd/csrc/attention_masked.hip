// Attention over packed documents with causal, window and prefix masks, a
// score cap and a distance bias (svl_masked_attention).
#include "dev_common.hpp"
#include "packed.hpp"

namespace svl {

constexpr float LOG2E = 1.4426950408889634f;

// One wave per query vector, any head dim up to 64 * NPER: lanes hold dims
// lane, lane + 64, ...; only visible keys are visited, in order, with the
// running maximum and sum of the softmax.
template <class T, int NPER>
__global__ __launch_bounds__(256) void masked_rows_kernel(MaskedArgs a) {
    const AttnWork w = a.work[blockIdx.x];
    const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
    const int G = a.heads / a.kv_heads;
    const int64_t nvec = (int64_t)w.q_len * G;
    for (int i = wave; i < 128; i += 4) {
        const int64_t vec = w.v0 + i;
        if (vec >= nvec) return;
        const int qi = (int)(vec / G), head = w.kvh * G + (int)(vec - (int64_t)qi * G);
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
            const int64_t k0 = part ? max(lo, (int64_t)w.prefix) : 0;
            const int64_t k1 = part ? hi : (int64_t)w.prefix - 1;
            for (int64_t key = k0; key <= k1; ++key) {
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
        T *out = (T *)a.out + qrow * a.o_tok + head * a.o_head;
#pragma unroll
        for (int e = 0; e < NPER; ++e) {
            const int d = lane + 64 * e;
            if (d < a.hd) out[d] = (T)(l == 0.f ? 0.f : acc[e] / l);
        }
        if (a.lse && lane == 0)
            a.lse[qrow * a.heads + head] = l == 0.f ? -INFINITY : m + logf(l);
    }
}

MaskedShape masked_shape(bool bf16, int hd) { return {128, 64, 0}; }

template <class T>
static hipError_t launch_rows(const MaskedArgs &a, hipStream_t s) {
    const dim3 grid((unsigned)a.n_work), block(256);
    if (a.hd <= 64) hipLaunchKernelGGL((masked_rows_kernel<T, 1>), grid, block, 0, s, a);
    else if (a.hd <= 256) hipLaunchKernelGGL((masked_rows_kernel<T, 4>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((masked_rows_kernel<T, 16>), grid, block, 0, s, a);
    return hipGetLastError();
}

hipError_t launch_masked_attention(const MaskedArgs &a, bool bf16, const MaskedShape &shape,
                                   hipStream_t s) {
    if (a.n_work <= 0) return hipSuccess;
    return bf16 ? launch_rows<__bf16>(a, s) : launch_rows<float>(a, s);
}

}  // namespace svl
