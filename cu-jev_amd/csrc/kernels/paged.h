/* Device helpers of the paged K/V cache (paged.hip, attention_paged.hip).
 *
 * A page holds 64 tokens of every kv-head: K [Hkv][64][256] and V transposed
 * [Hkv][256][64], bf16 or e4m3 with one fp32 scale per token and kv-head. 64
 * tokens are one key tile of the attention, so a tile has one page id, one
 * base address (64-bit) and offsets that fit 15 bits however long the pool. */
#pragma once
#include <type_traits>

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

DEV pg_seq seq_at(const pg_seq &s, int l) { /* lane l's */
    auto of = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
    return {of(s.q0), of(s.ql), of(s.kv), of(s.p0)};
}

/* f over the lanes with the same number in each of the wave's four rows of 16 */
template <class F> DEV float fold_rows(float x, F f) {
    const uint32_t u = __float_as_uint(x);
    auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const uint32_t v = __float_as_uint(f(__uint_as_float(a[0]), __uint_as_float(a[1])));
    a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return f(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
/* Inclusive sum over the lanes below: 6 DPP adds (through LDS they took 6 trips) */
template <int ctrl, int rows> DEV int dpp_or_0(int v) {
    return __builtin_amdgcn_update_dpp(0, v, ctrl, rows, 0xf, true);
}
DEV int wave_scan(int v) {
    v += dpp_or_0<0x111, 0xf>(v); /* row_shr 1, 2, 4, 8 */
    v += dpp_or_0<0x112, 0xf>(v);
    v += dpp_or_0<0x114, 0xf>(v);
    v += dpp_or_0<0x118, 0xf>(v);
    v += dpp_or_0<0x142, 0xa>(v); /* row_bcast 15, 31 */
    v += dpp_or_0<0x143, 0xc>(v);
    return v;
}
DEV int last_lane(int v) { return __builtin_amdgcn_readlane(v, 63); }
/* f over the 16 lanes of each row of the wave, as a butterfly from 8 down to 1 (a
 * rotation by o meets what lane ^ o has, once the larger strides are done), and over
 * the wave, from 32 down */
template <int ctrl> DEV float dpp(float x) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(
        0, (int)__float_as_uint(x), ctrl, 0xf, 0xf, true));
}
template <class F> DEV float fold_row(float x, F f) {
    x = f(x, dpp<0x128>(x)); /* row_ror 8, 4, 2, 1 */
    x = f(x, dpp<0x124>(x));
    x = f(x, dpp<0x122>(x));
    return f(x, dpp<0x121>(x));
}
template <class F> DEV float fold_wave(float x, F f) {
    const uint32_t u = __float_as_uint(x);
    auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t v = __float_as_uint(f(__uint_as_float(a[0]), __uint_as_float(a[1])));
    a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return fold_row(f(__uint_as_float(a[0]), __uint_as_float(a[1])), f);
}

/* fold_wave of doubles, dword by dword */
template <class F> DEV double fold_wave(double x, F f) {
    union Two {
        double d;
        uint32_t u[2];
    };
    auto swap = [&](auto swapped) {
        Two p, q, v{x};
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const auto a = swapped(v.u[i]);
            p.u[i] = a[0], q.u[i] = a[1];
        }
        x = f(p.d, q.d);
    };
    auto turn = [&](auto ctrl) {
        Two p, v{x};
#pragma unroll
        for (int i = 0; i < 2; i++)
            p.u[i] = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v.u[i], decltype(ctrl)::value,
                                                           0xf, 0xf, true);
        x = f(x, p.d);
    };
    swap([](uint32_t v) { return __builtin_amdgcn_permlane32_swap(v, v, false, false); });
    swap([](uint32_t v) { return __builtin_amdgcn_permlane16_swap(v, v, false, false); });
    turn(std::integral_constant<int, 0x128>{});
    turn(std::integral_constant<int, 0x124>{});
    turn(std::integral_constant<int, 0x122>{});
    turn(std::integral_constant<int, 0x121>{});
    return x;
}
/* d towards zero, the last bit set where that lost something: rounding this again
 * to fewer bits rounds d once */
DEV float to_odd(double d) {
    const float f = (float)d;
    uint32_t u = __float_as_uint(f);
    if ((double)f != d) {
        u -= fabs((double)f) > fabs(d);
        u |= 1;
    }
    return d != d ? f : __uint_as_float(u);
}

/* The sequences of rows n0 .. n0 + TOK - 1, row n0 + t in lane t: the last b
 * with q_start[b] <= n, -1 for a row before the first or behind the last
 * sequence. Up to 64 sequences' starts and lengths come in one go; of more, 64
 * starts spread over those that are left narrow them down to 64 first. */
template <int TOK>
DEV int find_seqs(const int32_t *q_start, const int32_t *kv_len, int B, int N, int max_kv, int n0,
                  pg_seq *s) {
    const int lane = threadIdx.x & 63;
    const pg_seq mine = load_seq(q_start, kv_len, min(lane, B - 1), N, N, max_kv);
    int from = 0; /* starts before it are <= n0 */
    for (int len = B + 1; len > 64;) {
        const int stride = (len + 63) / 64;
        const int v = q_start[min(from + lane * stride, B)];
        const int c = __popcll(__ballot(lane * stride < len && v <= n0));
        from += max(c - 1, 0) * stride;
        len = min(len - max(c - 1, 0) * stride, stride);
    }
    int before[TOK]; /* starts <= n among q_start[0 .. B] */
#pragma unroll
    for (int t = 0; t < TOK; t++)
        before[t] = from;
    for (int b0 = from; b0 <= B; b0 += 64) {
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
    b = b > B ? -1 : b - 1;
    const int l = max(b, 0) & 63; /* outside a branch: its loads stay with the starts' */
    *s = {__shfl(mine.q0, l, 64), __shfl(mine.ql, l, 64), __shfl(mine.kv, l, 64),
          __shfl(mine.p0, l, 64)};
    if (B > 64)
        *s = load_seq(q_start, kv_len, max(b, 0), N, N, max_kv);
    return b;
}

/* Work item `item` of a launch whose sequence b has count(b, s) of them, in
 * order: the sequence, and the item's number in it (-1: no such item). J
 * sequences a lane, 64 J a step. */
template <int J, typename F>
DEV int find_item_among(const int32_t *q_start, const int32_t *kv_len, int B, int N, int max_q,
                        int max_kv, int item, F count, pg_seq *s, int *local) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int b0 = 0; b0 < B; b0 += 64 * J) {
        pg_seq mine[J];
        int own[J], sum = 0;
#pragma unroll
        for (int j = 0; j < J; j++)
            mine[j] = load_seq(q_start, kv_len, min(b0 + J * lane + j, B - 1), N, max_q, max_kv);
#pragma unroll
        for (int j = 0; j < J; j++)
            sum += own[j] = b0 + J * lane + j < B ? count(mine[j]) : 0;
        const int to = before + wave_scan(sum);
        const uint64_t past = __ballot(to > item);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            int at = __builtin_amdgcn_readlane(to - sum, l), b = 0;
#pragma unroll
            for (int j = 0; j < J; j++) {
                const int here = __builtin_amdgcn_readlane(own[j], l);
                if (item >= at && item < at + here) {
                    *s = seq_at(mine[j], l);
                    *local = item - at;
                    b = b0 + J * l + j;
                }
                at += here;
            }
            return b;
        }
        before = last_lane(to);
    }
    return -1;
}
template <typename F>
DEV int find_item(const int32_t *q_start, const int32_t *kv_len, int B, int N, int max_q,
                  int max_kv, int item, F count, pg_seq *s, int *local) {
    return B > 64 ? find_item_among<4>(q_start, kv_len, B, N, max_q, max_kv, item, count, s, local)
                  : find_item_among<1>(q_start, kv_len, B, N, max_q, max_kv, item, count, s, local);
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
DEV int e4m3_exp(double a) { /* the same from a double */
    const uint64_t u = __builtin_bit_cast(uint64_t, a), low = (1ull << 52) - 1;
    const int e = (int)(u >> 52) - 1023 - 8 + ((u & low) > (3ull << 50) ? 1 : 0);
    return min(max(e, -100), 120);
}
DEV float exp2_int(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

/* Four values, already divided by their scales, to four e4m3 bytes (nearest
 * even; NaN and infinity become NaN). */
DEV uint32_t pack_e4m3(float a, float b, float c, float d) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}
/* Value i of four e4m3 bytes */
DEV float e4m3_of(uint32_t v, int i) {
    return i < 2 ? __builtin_amdgcn_cvt_pk_f32_fp8(v, false)[i & 1]
                 : __builtin_amdgcn_cvt_pk_f32_fp8(v, true)[i & 1];
}
/* Two e4m3 bytes (of the low or high half) times 2^k, exact in bf16. */
template <bool HIGH> DEV bf16x2 unpack_e4m3(uint32_t v, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v, scale, HIGH);
}

} // namespace
} // namespace CUJEV_KNS
