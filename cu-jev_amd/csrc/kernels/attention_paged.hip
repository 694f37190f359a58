/* Attention over a paged K/V cache for gfx950.
 *
 * Row (n, h) of sequence b, at position p, sees the keys j <= p of b's pages
 * and, with a window W, of those only j > p - W and the first S (sinks):
 *   out = sigmoid(gate) sum_j 2^(q.k_j) v_j / sum_j 2^(q.k_j). */
#include "paged.h"

namespace CUJEV_KNS {
namespace {

/* One wave per (row, q-head): lane j takes key j of a page for the scores, dims
 * 4 lane .. + 3 for the output; running maximum and sum in fp32. */
template <bool E4M3>
__global__ __launch_bounds__(64) void attention_paged_kernel(
    const bf16 *__restrict__ q, const bf16 *__restrict__ gate, int gts, int ghs,
    const void *__restrict__ kp, const void *__restrict__ vp, const float *__restrict__ ks,
    const float *__restrict__ vs, int num_pages, const int32_t *__restrict__ q_start,
    const int32_t *__restrict__ kv_len, const int32_t *__restrict__ page_table, int max_pages,
    int B, int N, int Hq, int Hkv, int window, int sinks, bf16 *__restrict__ out) {
    const int n = blockIdx.x / Hq, h = blockIdx.x % Hq, kh = h / (Hq / Hkv), lane = threadIdx.x;
    __shared__ float qs[PD], pr[PG];
    const int b = find_seq(q_start, B, n);
    if (b < 0)
        return;
    const Seq s = load_seq(q_start, kv_len, b, N, max_pages);
    if ((unsigned)(n - s.q0) >= (unsigned)s.ql)
        return;
    const int pos = s.p0 + n - s.q0;
    for (int e = 0; e < 4; e++)
        qs[4 * lane + e] = bf2f(q[((size_t)n * Hq + h) * PD + 4 * lane + e]);
    __syncthreads();
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    const int hi = min(pos, s.kv - 1), lo = window ? max(pos - window + 1, 0) : 0;
    for (int t = 0; t <= hi / PG && hi >= 0; t++) {
        const int j = t * PG + lane;
        const bool seen = j <= hi && (j >= lo || j < sinks);
        const int page = page_table[(size_t)b * max_pages + t];
        if (!__any(seen) || page < 0 || page >= num_pages)
            continue;
        const size_t head = (size_t)page * Hkv + kh;
        float x = 0.f;
        for (int d = 0; d < PD; d++) {
            const size_t at = head * PSLICE + (size_t)lane * PD + d;
            float kv;
            if constexpr (E4M3)
                kv = bf2f(unpack_e4m3<false>(((const uint8_t *)kp)[at], 1.f)[0]);
            else
                kv = bf2f(((const bf16 *)kp)[at]);
            x += qs[d] * kv;
        }
        if constexpr (E4M3)
            x *= ks[head * PG + lane];
        x = seen ? x : -INFINITY;
        const float mn = fmaxf(m, wave_max(x)), a = fast_exp2(m - mn), p = fast_exp2(x - mn);
        m = mn;
        l = l * a + wave_sum(p);
        __syncthreads();
        pr[lane] = p;
        __syncthreads();
        for (int e = 0; e < 4; e++) {
            o[e] *= a;
            for (int i = 0; i < PG; i++) {
                const size_t at = head * PSLICE + (size_t)(4 * lane + e) * PG + i;
                float v;
                if constexpr (E4M3)
                    v = bf2f(unpack_e4m3<false>(((const uint8_t *)vp)[at], 1.f)[0]) *
                        vs[head * PG + i];
                else
                    v = bf2f(((const bf16 *)vp)[at]);
                o[e] += pr[i] > 0.f ? pr[i] * v : 0.f;
            }
        }
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
    for (int e = 0; e < 4; e++) {
        float g = 1.f;
        if (gate)
            g = sigmoid_f(bf2f(gate[(size_t)n * gts + (size_t)h * ghs + 4 * lane + e]));
        out[((size_t)n * Hq + h) * PD + 4 * lane + e] = f2bf(o[e] * inv * g);
    }
}

} // namespace
} // namespace CUJEV_KNS
using namespace CUJEV_KNS;

extern "C" size_t cujev_attention_paged_ws_bytes(int N, int B, int max_q, int max_kv, int Hq,
                                                 int Hkv, int window, int sinks, int type) {
    return 0;
}

extern "C" hipError_t k_attention_paged(const bf16_t *q, const bf16_t *gate, int gate_tok_stride,
                                        int gate_head_stride, const cujev_kv_pages *pages,
                                        const cujev_paged_seqs *seqs, int N, int max_q, int max_kv,
                                        int Hq, int window, int sinks, bf16_t *out, void *ws,
                                        size_t ws_bytes, hipStream_t stream) {
    if (N <= 0 || seqs->B <= 0)
        return hipSuccess;
    if ((long long)N * Hq > 0x7fffffff)
        return hipErrorInvalidValue;
#define LAUNCH(T)                                                                                 \
    hipLaunchKernelGGL(attention_paged_kernel<T>, dim3((unsigned)(N * Hq)), dim3(64), 0, stream,  \
                       (const bf16 *)q, (const bf16 *)gate, gate_tok_stride, gate_head_stride,    \
                       pages->k, pages->vt, pages->k_scale, pages->v_scale, pages->num_pages,     \
                       seqs->q_start, seqs->kv_len, seqs->page_table, seqs->max_pages, seqs->B,   \
                       N, Hq, pages->Hkv, window, sinks, (bf16 *)out)
    if (pages->type == CUJEV_KV_E4M3)
        LAUNCH(true);
    else
        LAUNCH(false);
#undef LAUNCH
    return hipGetLastError();
}
