/* The paged K/V cache of gfx950: new tokens into pages (norm, RoPE, e4m3
 * quantisation), and pages back into a state's contiguous caches. The
 * reference has one contiguous bf16 cache per state (src/engine/model.h:60-72)
 * and neither operator. */
#include "paged.h"

namespace CUJEV_KNS {
namespace {

/* ---- new tokens into pages ---------------------------------------------------
 * Three kinds of wave in one launch. A row wave normalises TOK tokens' rows of one
 * q-head or K head, lane l holding dims 4l .. 4l + 3, as attn_prep does:
 *   y = x rsqrt(mean x^2 + eps) w, RoPE (dim i with i + rot/2, lane l with
 *   l ^ rot/8), q times q_scale.
 * A V wave takes the tokens of one aligned group of 16 positions and one
 * kv-head: the group's V^T rows are whole 16-byte (e4m3) or 32-byte pieces, so
 * the transpose needs neither LDS nor another wave's data: lane l holds 16
 * tokens of dims 4l .. 4l + 3 and stores one piece per dim. A page's four groups
 * are a wave's, or waves' on one XCD, whose L2 gathers their lines of V^T. With
 * V_ROWS V's tokens are row waves, too, and store single elements.
 *
 * 8 sequences of up to 700 tokens, e4m3: 15.5 us a call (16.0 traced) for 62 MB, 4.0
 * TB/s; reductions through LDS, rope loads by all lanes and a page's groups on other
 * XCDs took 25. 64 of one token: 6.3 us, a chain of loads: arguments, lengths, page
 * ids, stores; bf16 5.2. Four tokens a wave, two of e4m3 keys: their rounding needs
 * the registers. A wave a workgroup: 1024 tokens bf16 take 8.6 us so, 10.6 with four. */
constexpr int PREP_TOK = 4;
/* V by rows as well, a token's 256 values as single elements, where there are many
 * sequences of a token or so each: 1024 x 1 e4m3 26 us, 38 by groups, each of which
 * has to find its sequence among all; 1024 x 3 bf16 63 and 84; but 256 x 4 20.0 and
 * 18.7, and 64 x 1 bf16 6.6 and 5.5. */
constexpr int PREP_V_ROWS = 3, PREP_V_SEQS = 64;
/* V by groups, a wave each where they are few or most of a page's are there (kernel of
 * 16 x 48 e4m3 7.5 us, 11.2 with a wave a page; of 8 x 700 16.4 and 17.6), a wave a
 * page otherwise, which starts fewer that have nothing to do (64 x 48 16.7 and 19.5). */
constexpr int PREP_V_FEW = 1024, PREP_V_WHOLE = 128;
/* A K row's lane in doubles, rounded to e4m3 once: the bytes, and the scale 2^*e */
DEV uint32_t k_row_exact(const bf16 *src, const float2 *rope, const float *w, bool rotates,
                         bool first, int half_lanes, float eps, int *e) {
    const bf16x4 raw = *(const bf16x4 *)src;
    double y[4], ss = 0., most = 0.;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        y[i] = bf2f(raw[i]);
        ss = __builtin_fma(y[i], y[i], ss);
    }
    ss = fold_wave(ss, [](double p, double q) { return p + q; });
    const double a = ss * (1. / 256.) + (double)eps;
    double rinv = __builtin_amdgcn_rsq(a); /* about 2^-26 off: Newton twice */
    if (a > 0. && a < (double)INFINITY) {
        rinv *= __builtin_fma(-.5 * a * rinv, rinv, 1.5);
        rinv *= __builtin_fma(-.5 * a * rinv, rinv, 1.5);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        y[i] *= rinv * w[i];
        const float2 cs = rope[rotates ? i : 0];
        const double o = __shfl_xor(y[i], half_lanes, 64) * cs.y;
        y[i] = rotates ? __builtin_fma(y[i], (double)cs.x, first ? -o : o) : y[i];
        most = fmax(most, fabs(y[i]));
    }
    most = fold_wave(most, [](double p, double q) { return fmax(p, q); });
    *e = e4m3_exp(most);
    const double inv = exp2_int(-*e);
    return pack_e4m3(to_odd(y[0] * inv), to_odd(y[1] * inv), to_odd(y[2] * inv),
                     to_odd(y[3] * inv));
}

struct Prep {
    const bf16 *proj;
    int ps;
    const float *qw, *kw;
    const int32_t *pos, *q_start, *kv_len, *page_table;
    int max_pages, B, N, Hq, Hkv, rot;
    const float2 *rope;
    int npos;
    float eps, q_scale;
    bf16 *q_out;
    void *k_pages, *vt_pages;
    float *k_scale, *v_scale;
    int num_pages, k_blocks, v_blocks;
    bool v_spread; /* a wave a group of V, or a page */
};
enum { ROW_Q, ROW_K, ROW_V };

/* A wave for tokens n0 .. n0 + TOK - 1 of one head */
template <int KIND, int TOK, bool E4M3> DEV void row_wave(const Prep &c, int head, int n0) {
    constexpr bool is_k = KIND == ROW_K;
    const int lane = threadIdx.x & 63, N = c.N, rot = c.rot;
    const float *w = is_k ? c.kw : c.qw;
    /* K's heads, then V's, follow q's and the gates' */
    const int at0 = KIND == ROW_Q ? head * 512 : c.Hq * 512 + (is_k ? head : c.Hkv + head) * 256;
    const bf16 *src = c.proj + at0 + 4 * lane;
    const int half_lanes = rot / 8;
    const bool rotates = lane < 2 * half_lanes, first = lane < half_lanes;
    const int fi0 = rotates ? (first ? 4 * lane : 4 * lane - rot / 2) : 0;
    /* every load before any arithmetic, token indices clamped */
    bf16x4 raw[TOK];
#pragma unroll
    for (int t = 0; t < TOK; t++)
        raw[t] = *(const bf16x4 *)(src + (size_t)min(n0 + t, N - 1) * c.ps);
    const float4 wl = *(const float4 *)(w + 4 * lane);
    const int pos_lane = min(max(c.pos[min(n0 + (lane & (TOK - 1)), N - 1)], 0), c.npos - 1);
    /* The tokens' sequences, then (K) their slots, token t in lane t: one
     * chain of loads for all of them. at: the K row in the pool, -1: none */
    pg_seq s;
    int b = find_seqs<TOK>(c.q_start, c.kv_len, c.B, N, c.max_pages * PG, n0, &s);
    float4 rc[TOK][2] = {};
    if (rotates) { /* 16 lanes' loads or fewer: by all 64 they cost more than x's */
#pragma unroll
        for (int t = 0; t < TOK; t++) {
            const float4 *r = (const float4 *)(
                c.rope + (size_t)__builtin_amdgcn_readlane(pos_lane, t) * (rot / 2) + fi0);
            rc[t][0] = r[0];
            rc[t][1] = r[1];
        }
    }
    if (n0 + lane >= N)
        b = -1;
    long long at = b;
    if (KIND != ROW_Q) {
        const int p = s.p0 + (n0 + lane - s.q0);
        const bool in = b >= 0 && (unsigned)(n0 + lane - s.q0) < (unsigned)s.ql && p >= 0 &&
                        p < s.kv;
        const int page = c.page_table[(size_t)max(b, 0) * c.max_pages + (in ? p / PG : 0)];
        at = in && page >= 0 && page < c.num_pages
                 ? ((long long)page * c.Hkv + head) * PG + p % PG
                 : -1;
    }
    auto row_of = [&](int t) {
        return (long long)(uint32_t)__builtin_amdgcn_readlane((int)at, t) |
               (long long)__builtin_amdgcn_readlane((int)(at >> 32), t) << 32;
    };
    if constexpr (KIND == ROW_V) {
#pragma unroll
        for (int t = 0; t < TOK; t++) {
            const long long row = row_of(t);
            if (row < 0)
                continue;
            const size_t to = (size_t)(row / PG) * PSLICE + (size_t)4 * lane * PG + row % PG;
            if constexpr (E4M3) {
                float v[4], amax = 0.f;
#pragma unroll
                for (int d = 0; d < 4; d++) {
                    v[d] = bf2f(raw[t][d]);
                    amax = fmaxf(amax, fabsf(v[d]));
                }
                amax = fold_wave(amax, [](float p, float q) { return fmaxf(p, q); });
                const int e = e4m3_exp(amax);
                const float inv = exp2_int(-e);
                const uint32_t out =
                    pack_e4m3(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
#pragma unroll
                for (int d = 0; d < 4; d++)
                    ((uint8_t *)c.vt_pages)[to + d * PG] = (uint8_t)(out >> (8 * d));
                if (lane == 0)
                    c.v_scale[row] = exp2_int(e);
            } else {
#pragma unroll
                for (int d = 0; d < 4; d++)
                    ((bf16 *)c.vt_pages)[to + d * PG] = raw[t][d];
            }
        }
        return;
    }
    float x[TOK][4], ss[TOK];
#pragma unroll
    for (int t = 0; t < TOK; t++) {
        ss[t] = 0.f;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            x[t][e] = bf2f(raw[t][e]);
            ss[t] += x[t][e] * x[t][e];
        }
    }
#pragma unroll
    for (int t = 0; t < TOK; t++)
        ss[t] = fold_wave(ss[t], [](float p, float q) { return p + q; });
    const float we[4] = {wl.x, wl.y, wl.z, wl.w};
#pragma unroll
    for (int t = 0; t < TOK; t++) {
        const float rinv = rsqrtf(ss[t] * (1.f / 256.f) + c.eps);
        const float cz[8] = {rc[t][0].x, rc[t][0].y, rc[t][0].z, rc[t][0].w,
                             rc[t][1].x, rc[t][1].y, rc[t][1].z, rc[t][1].w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float y = x[t][e] * rinv * we[e];
            /* rounded as attn_prep rounds: the same bits reach both caches */
            const float o = __shfl_xor(y, half_lanes, 64) * cz[2 * e + 1];
            x[t][e] = rotates ? __builtin_fmaf(y, cz[2 * e], first ? -o : o) : y;
        }
    }
    uint32_t again = 0; /* tokens */
#pragma unroll
    for (int t = 0; t < TOK; t++) {
        const long long row = row_of(t);
        if (row < 0) /* no sequence's row, or no slot */
            continue;
        if constexpr (E4M3 && is_k) {
            float amax = 0.f;
#pragma unroll
            for (int e = 0; e < 4; e++)
                amax = fmaxf(amax, fabsf(x[t][e]));
            amax = fold_wave(amax, [](float p, float q) { return fmaxf(p, q); });
            const int e = e4m3_exp(amax);
            const float inv = exp2_int(-e);
            const uint32_t out =
                pack_e4m3(x[t][0] * inv, x[t][1] * inv, x[t][2] * inv, x[t][3] * inv);
            /* Close to a tie, or to the next scale, float's errors (about ten
             * roundings, of values up to amax sqrt 2 where they rotate) can lead a
             * value to the other side, a whole step of 2^-3; one or two of 5
             * million did. Such a row, one of 30 or so, again in doubles. */
            constexpr float NEAR = 0x1p-20f;
            const float top = amax * inv;
            bool close = top > 448.f * (1.f - NEAR) || top < 224.f * (1.f + NEAR);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float v = fabsf(x[t][i] * inv), r = fabsf(e4m3_of(out, i));
                const float step = __uint_as_float(
                    max(__float_as_uint(v) & 0x7f800000u, (127u - 6) << 23) - (3u << 23));
                close |= .5f * step - fabsf(v - r) < NEAR * (rotates ? 2.f * top : v);
            }
            again |= __any(close) ? 1u << t : 0u;
            ((uint32_t *)c.k_pages)[row * 64 + lane] = out;
            if (lane == 0)
                c.k_scale[row] = exp2_int(e);
            continue;
        }
        const float f = is_k ? 1.f : c.q_scale;
        const bf16x4 o = {f2bf(x[t][0] * f), f2bf(x[t][1] * f), f2bf(x[t][2] * f),
                          f2bf(x[t][3] * f)};
        if constexpr (!is_k) {
            *(bf16x4 *)(c.q_out + ((size_t)(n0 + t) * c.Hq + head) * 256 + 4 * lane) = o;
        } else {
            *(bf16x4 *)((bf16 *)c.k_pages + row * 256 + 4 * lane) = o;
        }
    }
#pragma unroll 1
    while (E4M3 && is_k && again) { /* a loop: unrolled, it took registers from the others */
        const int t = __ffs(again) - 1;
        again &= again - 1;
        const long long row = row_of(t);
        int e;
        const uint32_t out = k_row_exact(
            src + (size_t)(n0 + t) * c.ps,
            c.rope + (size_t)__builtin_amdgcn_readlane(pos_lane, t) * (rot / 2) + fi0,
            w + 4 * lane, rotates, first, half_lanes, c.eps, &e);
        ((uint32_t *)c.k_pages)[row * 64 + lane] = out;
        if (lane == 0)
            c.k_scale[row] = exp2_int(e);
    }
}

/* V of groups g0 .. g1 - 1 of 16 positions of a page: of number `unit` / Hkv among
 * those that the new tokens touch */
template <bool E4M3> DEV void v_groups(const Prep &c, int unit, int g0, int g1) {
    const int lane = threadIdx.x & 63, kh = unit % c.Hkv;
    pg_seq s;
    int i;
    const int b = find_item(
        c.q_start, c.kv_len, c.B, c.N, c.N, c.max_pages * PG, unit / c.Hkv,
        [](const pg_seq &q) { return pg_v_pages(q); }, &s, &i);
    if (b < 0)
        return;
    const int at = pg_new_lo(s) / PG + i;          /* the page's number in the sequence */
    const int page = c.page_table[(size_t)b * c.max_pages + at];
    if (page < 0 || page >= c.num_pages)
        return;
#pragma unroll 1
    for (int group = g0; group < g1; group++) {
        const int base = at * PG + group * VTOK; /* the group's first position */
        if (base + VTOK <= pg_new_lo(s) || base >= pg_new_hi(s))
            continue;
        const int lo = max(pg_new_lo(s), base), hi = min(pg_new_hi(s), base + VTOK);
        const bf16 *src = c.proj + c.Hq * 512 + c.Hkv * 256 + kh * 256 + 4 * lane;
        bf16x4 v[VTOK];
#pragma unroll
        for (int t = 0; t < VTOK; t++) {
            const int p = min(max(base + t, lo), hi - 1);
            v[t] = *(const bf16x4 *)(src + (size_t)(s.q0 + p - s.p0) * c.ps);
        }
        const size_t head = (size_t)page * c.Hkv + kh;
        const int col = base % PG;
        const bool whole = hi - lo == VTOK;
        if constexpr (E4M3) {
            /* max of each token over the wave: lanes that meet exchange the halves
             * they give up (16 -> 8 -> 4 -> 2 -> 1 tokens a lane), so lane l ends
             * with token l >> 2 */
            float m[VTOK];
#pragma unroll
            for (int t = 0; t < VTOK; t++)
                m[t] = fmaxf(fmaxf(fabsf(bf2f(v[t][0])), fabsf(bf2f(v[t][1]))),
                             fmaxf(fabsf(bf2f(v[t][2])), fabsf(bf2f(v[t][3]))));
            auto meet = [](float p, float q, bool by32) {
                const uint32_t u = __float_as_uint(p), v = __float_as_uint(q);
                const auto a = by32 ? __builtin_amdgcn_permlane32_swap(u, v, false, false)
                                    : __builtin_amdgcn_permlane16_swap(u, v, false, false);
                return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
            };
#pragma unroll
            for (int t = 0; t < 8; t++)
                m[t] = meet(m[t], m[t + 8], true);
#pragma unroll
            for (int t = 0; t < 4; t++)
                m[t] = meet(m[t], m[t + 4], false);
#pragma unroll
            for (int t = 0; t < 2; t++) /* row_ror 8 */
                m[t] = fmaxf(lane & 8 ? m[t + 2] : m[t], dpp<0x128>(lane & 8 ? m[t] : m[t + 2]));
            /* row_half_mirror: lane ^ 7, in the other four as lane ^ 4 is */
            m[0] = fmaxf(lane & 4 ? m[1] : m[0], dpp<0x141>(lane & 4 ? m[0] : m[1]));
            m[0] = fmaxf(m[0], dpp<0x4e>(m[0])); /* quad_perm, lane ^ 2, lane ^ 1 */
            m[0] = fmaxf(m[0], dpp<0xb1>(m[0]));
            const int e = e4m3_exp(m[0]), tok = lane >> 2;
            if ((lane & 3) == 0 && base + tok >= lo && base + tok < hi)
                c.v_scale[head * PG + col + tok] = exp2_int(e);
            float inv[VTOK];
#pragma unroll
            for (int t = 0; t < VTOK; t++)
                inv[t] = exp2_int(-__builtin_amdgcn_readlane(e, 4 * t));
            uint8_t *dst = (uint8_t *)c.vt_pages + head * PSLICE + (size_t)4 * lane * PG + col;
#pragma unroll
            for (int d = 0; d < 4; d++) {
                u32x4 q;
#pragma unroll
                for (int w = 0; w < 4; w++)
                    q[w] = pack_e4m3(bf2f(v[4 * w][d]) * inv[4 * w],
                                     bf2f(v[4 * w + 1][d]) * inv[4 * w + 1],
                                     bf2f(v[4 * w + 2][d]) * inv[4 * w + 2],
                                     bf2f(v[4 * w + 3][d]) * inv[4 * w + 3]);
                if (whole) {
                    *(u32x4 *)(dst + d * PG) = q;
                } else {
#pragma unroll
                    for (int t = 0; t < VTOK; t++)
                        if (base + t >= lo && base + t < hi)
                            dst[d * PG + t] = (uint8_t)(q[t >> 2] >> (8 * (t & 3)));
                }
            }
        } else {
            bf16 *dst = (bf16 *)c.vt_pages + head * PSLICE + (size_t)4 * lane * PG + col;
#pragma unroll
            for (int d = 0; d < 4; d++) {
                if (whole) {
#pragma unroll
                    for (int w = 0; w < 2; w++) {
                        bf16x8 q;
#pragma unroll
                        for (int t = 0; t < 8; t++)
                            q[t] = v[8 * w + t][d];
                        *(bf16x8 *)(dst + d * PG + 8 * w) = q;
                    }
                } else {
#pragma unroll
                    for (int t = 0; t < VTOK; t++)
                        if (base + t >= lo && base + t < hi)
                            dst[d * PG + t] = v[t][d];
                }
            }
        }
    }
}

template <int n> using is = std::integral_constant<int, n>;
template <bool E4M3, bool V_ROWS>
__global__ __launch_bounds__(64) void prep_paged_kernel(Prep c) {
    int block = blockIdx.x;
    auto rows = [&](auto kind, auto tok, int heads) {
        const int n0 = block / heads * decltype(tok)::value;
        if (n0 < c.N)
            row_wave<decltype(kind)::value, decltype(tok)::value, E4M3>(c, block % heads, n0);
    };
    /* The longest first (8 x 700 e4m3 1.7 us less than with q's rows first) */
    if (block < c.v_blocks) {
        if constexpr (V_ROWS) {
            return rows(is<ROW_V>{}, is<PREP_TOK>{}, c.Hkv);
        } else {
            /* a page's groups on one XCD: block b runs on b % 8 */
            const int group = block / 8 % 4;
            return c.v_spread ? v_groups<E4M3>(c, block / 32 * 8 + block % 8, group, group + 1)
                              : v_groups<E4M3>(c, block, 0, 4);
        }
    }
    block -= c.v_blocks;
    if (block < c.k_blocks)
        return rows(is<ROW_K>{}, is<E4M3 ? PREP_TOK / 2 : PREP_TOK>{}, c.Hkv);
    block -= c.k_blocks;
    rows(is<ROW_Q>{}, is<PREP_TOK>{}, c.Hq);
}

/* ---- pages back into a state's caches -----------------------------------------
 * One workgroup per (sequence, page, kv-head, K or V^T): 64 rows of 512 bytes
 * or 256 rows of 128 out, 16 values a thread and step. A page id outside the
 * pool reads as zeros; columns from kv_len on stay as they were. 8192 keys of 4
 * kv-heads from e4m3: 10.4 us a call for 50 MB, 4.9 TB/s. */
template <bool E4M3>
__global__ __launch_bounds__(256) void page_read_kernel(
    const void *__restrict__ k_pages, const void *__restrict__ vt_pages,
    const float *__restrict__ k_scale, const float *__restrict__ v_scale, int num_pages,
    const int32_t *__restrict__ page_table, int max_pages, const int32_t *__restrict__ kv_len,
    int max_kv, int Hkv, bf16 *__restrict__ kc, bf16 *__restrict__ vtc, int stride) {
    const int j = blockIdx.x >> 1, b = blockIdx.z, kh = blockIdx.y, tid = threadIdx.x;
    const int page = page_table[(size_t)b * max_pages + j]; /* beside kv_len's load */
    const int kv = min(max(kv_len[b], 0), max_kv), left = kv - j * PG; /* tokens of this page */
    if (left <= 0)
        return;
    const bool ok = page >= 0 && page < num_pages;
    const size_t head = (size_t)(ok ? page : 0) * Hkv + kh;
    const size_t out = ((size_t)b * Hkv + kh) * PD * (size_t)stride;
    if ((blockIdx.x & 1) == 0) { /* K: 16 dims a thread, 16 rows a step */
        bf16 *dst = kc + out + (size_t)j * PG * PD;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int row = 16 * i + (tid >> 4), at = row * PD + (tid & 15) * 16;
            bf16x8 r[2] = {};
            if constexpr (E4M3) {
                const u32x4 v = *(const u32x4 *)((const uint8_t *)k_pages + head * PSLICE + at);
                const float sc = k_scale[head * PG + row];
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    const bf16x2 a = unpack_e4m3<false>(v[w], sc), c = unpack_e4m3<true>(v[w], sc);
                    r[w >> 1][4 * (w & 1)] = a[0], r[w >> 1][4 * (w & 1) + 1] = a[1];
                    r[w >> 1][4 * (w & 1) + 2] = c[0], r[w >> 1][4 * (w & 1) + 3] = c[1];
                }
            } else {
                const bf16x8 *v = (const bf16x8 *)((const bf16 *)k_pages + head * PSLICE + at);
                r[0] = v[0], r[1] = v[1];
            }
            if (!ok)
                r[0] = r[1] = bf16x8{};
            if (row < left) {
                *(bf16x8 *)(dst + at) = r[0];
                *(bf16x8 *)(dst + at + 8) = r[1];
            }
        }
        return;
    }
    /* V^T: 16 tokens a thread, 64 rows a step */
    const int t0 = (tid & 3) * 16;
    float sc[16];
    if constexpr (E4M3) {
#pragma unroll
        for (int t = 0; t < 16; t += 4) {
            const float4 s4 = *(const float4 *)(v_scale + head * PG + t0 + t);
            sc[t] = s4.x, sc[t + 1] = s4.y, sc[t + 2] = s4.z, sc[t + 3] = s4.w;
        }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int d = 64 * i + (tid >> 2);
        bf16x8 r[2] = {};
        if constexpr (E4M3) {
            const u32x4 v =
                *(const u32x4 *)((const uint8_t *)vt_pages + head * PSLICE + d * PG + t0);
#pragma unroll
            for (int t = 0; t < 16; t++) {
                const bf16x2 p = t & 2 ? unpack_e4m3<true>(v[t >> 2], 1.f)
                                       : unpack_e4m3<false>(v[t >> 2], 1.f);
                r[t >> 3][t & 7] = f2bf(bf2f(p[t & 1]) * sc[t]);
            }
        } else {
            const bf16 *at = (const bf16 *)vt_pages + head * PSLICE + d * PG + t0;
            const bf16x8 *v = (const bf16x8 *)at;
            r[0] = v[0], r[1] = v[1];
        }
        if (!ok)
            r[0] = r[1] = bf16x8{};
        bf16 *dst = vtc + out + (size_t)d * stride + j * PG + t0;
        if (t0 + 16 <= left) {
            *(bf16x8 *)dst = r[0];
            *(bf16x8 *)(dst + 8) = r[1];
        } else {
#pragma unroll
            for (int t = 0; t < 16; t++)
                if (t0 + t < left)
                    dst[t] = r[t >> 3][t & 7];
        }
    }
}

} // namespace
} // namespace CUJEV_KNS
using namespace CUJEV_KNS;

extern "C" int cujev_kv_pages_ok(const cujev_kv_pages *p) {
    const uintptr_t at = (uintptr_t)p->k | (uintptr_t)p->vt;
    if (!p->k || !p->vt || (at & 15) || p->num_pages <= 0 || p->Hkv <= 0 ||
        (p->type != CUJEV_KV_BF16 && p->type != CUJEV_KV_E4M3))
        return 0;
    return p->type == CUJEV_KV_BF16 ||
           (p->k_scale && p->v_scale && !(((uintptr_t)p->k_scale | (uintptr_t)p->v_scale) & 15));
}

extern "C" hipError_t k_attn_prep_paged(const bf16_t *proj, int proj_stride, const float *q_norm_w,
                                        const float *k_norm_w, const int32_t *pos,
                                        const cujev_paged_seqs *seqs, int N, int Hq, int rot,
                                        const float *rope_table, int npos, float eps,
                                        float q_scale, bf16_t *q_out, const cujev_kv_pages *pages,
                                        hipStream_t stream) {
    const int Hkv = pages->Hkv, B = seqs->B;
    if (N <= 0 || B <= 0)
        return hipSuccess;
    const bool v_rows = B > PREP_V_SEQS && N <= PREP_V_ROWS * (long long)B;
    const bool e4m3 = pages->type == CUJEV_KV_E4M3;
    auto row_blocks = [&](int tok, int heads) {
        return (long long)CEIL_DIV(N, tok) * heads;
    };
    const long long v_pages = N < N / PG + 2ll * B ? N : N / PG + 2ll * B;
    const bool v_spread = v_pages * Hkv * 4 <= PREP_V_FEW || N >= PREP_V_WHOLE * (long long)B;
    const long long k_blocks = row_blocks(e4m3 ? PREP_TOK / 2 : PREP_TOK, Hkv);
    const long long v_blocks = v_rows ? row_blocks(PREP_TOK, Hkv)
                               : v_spread ? CEIL_DIV(v_pages * Hkv, 8) * 32
                                          : v_pages * Hkv;
    const long long blocks = k_blocks + v_blocks + row_blocks(PREP_TOK, Hq);
    if (blocks * 64 > PG_MOST_ITEMS)
        return hipErrorInvalidValue;
    const Prep c = {(const bf16 *)proj, proj_stride, q_norm_w, k_norm_w, pos, seqs->q_start,
                    seqs->kv_len, seqs->page_table, seqs->max_pages, B, N, Hq, Hkv, rot,
                    (const float2 *)rope_table, npos, eps, q_scale, (bf16 *)q_out, pages->k,
                    pages->vt, pages->k_scale, pages->v_scale, pages->num_pages, (int)k_blocks,
                    (int)v_blocks, v_spread};
#define LAUNCH(T, V)                                                                              \
    hipLaunchKernelGGL((prep_paged_kernel<T, V>), dim3((unsigned)blocks), dim3(64), 0, stream, c)
    if (e4m3 && v_rows)
        LAUNCH(true, true);
    else if (e4m3)
        LAUNCH(true, false);
    else if (v_rows)
        LAUNCH(false, true);
    else
        LAUNCH(false, false);
#undef LAUNCH
    return hipGetLastError();
}

extern "C" hipError_t k_kv_page_read(const cujev_kv_pages *pages, const cujev_paged_seqs *seqs,
                                     int max_kv, bf16_t *k_cache, bf16_t *vt_cache,
                                     int cache_stride, hipStream_t stream) {
    if (seqs->B <= 0 || max_kv <= 0)
        return hipSuccess;
    const int n = CEIL_DIV(max_kv, PG);
    if (n > seqs->max_pages || seqs->B > 65535 || pages->Hkv > 65535)
        return hipErrorInvalidValue;
    const dim3 grid(2u * n, (unsigned)pages->Hkv, (unsigned)seqs->B);
#define LAUNCH(T)                                                                                 \
    hipLaunchKernelGGL(page_read_kernel<T>, grid, dim3(256), 0, stream, pages->k, pages->vt,      \
                       pages->k_scale, pages->v_scale, pages->num_pages, seqs->page_table,        \
                       seqs->max_pages, seqs->kv_len, max_kv, pages->Hkv, (bf16 *)k_cache,        \
                       (bf16 *)vt_cache, cache_stride)
    if (pages->type == CUJEV_KV_E4M3)
        LAUNCH(true);
    else
        LAUNCH(false);
#undef LAUNCH
    return hipGetLastError();
}
