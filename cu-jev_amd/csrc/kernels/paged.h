/* Device helpers of the paged K/V cache (paged.hip, attention_paged.hip).
 *
 * A page holds 64 tokens of every kv-head: K [Hkv][64][256] and V transposed
 * [Hkv][256][64], bf16 or e4m3 with one fp32 scale per token and kv-head. 64
 * tokens are one key tile of the attention, so a tile has one page id, one
 * base address (64-bit) and offsets that fit 15 bits however long the pool. */
#pragma once
#include "common.h"
#include "kernels.h"
#include "paged_index.h"

namespace CUJEV_KNS {
namespace {

static_assert(PG == CUJEV_KV_PAGE, "one definition of a page");

constexpr int PD = 256;                /* head dim */
constexpr int PSLICE = PG * PD;        /* elements of one head's K or V^T in a page */

DEV pg_seq load_seq(const int32_t *q_start, const int32_t *kv_len, int b, int N, int max_q,
                    int max_kv) {
    return pg_clean_seq(q_start[b], q_start[b + 1], kv_len[b], N, max_q, max_kv);
}

/* The sequences of rows n0 .. n0 + TOK - 1, row n0 + t in lane t: the last b
 * with q_start[b] <= n, -1 for a row before the first or behind the last
 * sequence. One load of 64 starts a step. */
template <int TOK> DEV int find_seqs(const int32_t *q_start, int B, int n0) {
    const int lane = threadIdx.x & 63;
    int before[TOK] = {}; /* starts <= n among q_start[0 .. B] */
    for (int b0 = 0; b0 <= B; b0 += 64) {
        const int v = q_start[min(b0 + lane, B)];
        int c = 0;
#pragma unroll
        for (int t = 0; t < TOK; t++) {
            c = __popcll(__ballot(b0 + lane <= B && v <= n0 + t));
            before[t] += c;
        }
        if (c < 64)
            break;
    }
    int b = before[0];
#pragma unroll
    for (int t = 1; t < TOK; t++)
        b = lane == t ? before[t] : b;
    return b == 0 || b > B ? -1 : b - 1;
}

/* Work item `item` of a launch whose sequence b has count(b, s) of them, in
 * order: the sequence, and the item's number in it (-1: no such item). */
template <typename F>
DEV int find_item(const int32_t *q_start, const int32_t *kv_len, int B, int N, int max_q,
                  int max_kv, int item, F count, pg_seq *s, int *local) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int b0 = 0; b0 < B; b0 += 64) {
        const int b = min(b0 + lane, B - 1);
        const pg_seq mine = load_seq(q_start, kv_len, b, N, max_q, max_kv);
        const int own = b0 + lane < B ? count(mine) : 0;
        int sum = own; /* inclusive sum over the lanes */
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(sum, o, 64);
            sum += lane >= o ? v : 0;
        }
        const uint64_t past = __ballot(before + sum > item);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            s->q0 = __builtin_amdgcn_readlane(mine.q0, l);
            s->ql = __builtin_amdgcn_readlane(mine.ql, l);
            s->kv = __builtin_amdgcn_readlane(mine.kv, l);
            s->p0 = __builtin_amdgcn_readlane(mine.p0, l);
            *local = item - before - __builtin_amdgcn_readlane(sum - own, l);
            return b0 + l;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
    }
    return -1;
}

/* Scale of a row whose largest magnitude is a: 2^e, e the least integer with
 * a <= 448 * 2^e, in [-100, 120]. A power of two loses nothing against a /
 * 448 but where values fall below e4m3's range (its precision is relative),
 * and makes x / scale and stored * scale exact, the latter also in bf16: a
 * row is rounded once, and every reader sees the same values. From the bits:
 * a = 1.m * 2^(x - 127), and 448 = 1.75 * 2^8. */
DEV int e4m3_exp(float a) {
    const uint32_t u = __float_as_uint(a);
    const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffff) > 0x600000 ? 1 : 0);
    return min(max(e, -100), 120);
}
DEV float exp2_int(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

/* Four values, already divided by their scales, to four e4m3 bytes (nearest
 * even; NaN and infinity become NaN). */
DEV uint32_t pack_e4m3(float a, float b, float c, float d) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}
/* Two e4m3 bytes (of the low or high half) times 2^k, exact in bf16. */
template <bool HIGH> DEV bf16x2 unpack_e4m3(uint32_t v, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v, scale, HIGH);
}

} // namespace
} // namespace CUJEV_KNS
