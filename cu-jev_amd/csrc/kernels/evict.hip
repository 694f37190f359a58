/* Eviction from the paged K/V cache on gfx950: the weight that attention has given
 * each key, the positions worth keeping, and their move to the front. The reference
 * has one contiguous cache per state that only grows (src/engine/model.h:60-72). */
#include "paged.h"

namespace CUJEV_KNS {
namespace {
/* ---- attention weights by key --------------------------------------------------
 *   w[j] = prev[j] + sum over the call's rows (n, h) that see key j of 2^(q.k_j - lse)
 * with the attention's own lse, so that one product with K gives p whole: no second
 * pass, and no sum that crosses workgroups. S^T = K Q^T on v_mfma_f32_32x32x16_bf16,
 * keys on M: a lane has p of one row and 16 keys of each block of 32, and adds them up
 * over the packed rows (token, q-head); lanes are summed once, at the end, in a fixed
 * order. Two forms:
 *   up to 128 rows  Q stays in LDS, a wave streams pages of K past it (weigh_few)
 *   more            K stays in registers, Q streams through LDS (weigh_many) */
struct Weigh {
    const bf16 *q;
    const float *lse;
    const void *k;
    const float *ks;
    int num_pages;
    const int32_t *q_start, *kv_len, *page_table;
    int max_pages, B, N, max_q, max_kv, Hq, Hkv, G, rG;
    int blocks; /* workgroups of a sequence and kv-head (many rows: of each split) */
    int splits; /* many rows: parts of a block's rows, each with a place in parts if over 1 */
    const float *prev;
    float *w, *parts; /* [splits][B][Hkv][blocks * 256] */
};
/* Rows of 512 bytes of Q by DMA into LDS, two a load; piece p of row r lies in slot
 * p ^ (r & 15), so that 16 lanes' operands hit 16 bank groups. src: q of the token that
 * row 0 minus `rest` is the first of; rows past `most` repeat it. */
DEV void q_rows(const Weigh &c, __amdgpu_buffer_rsrc_t src, unsigned char *to, int first, int rest,
                int most) {
    const int id = lane_again(), at = first + (id >> 5); /* worked out each time, not kept */
    const int row = rest + min(at, most), tok = row * c.rG >> 16;
    const uint32_t off = (tok * c.Hq + row - tok * c.G) * PD * 2;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(src, (lds_ptr)(to + first * 512), 16,
                                             off + (((id & 31) ^ (at & 15)) << 4), 0, 0, 0);
}
/* Where a lane finds its operand of step ks: the address of step 0's, in the buffer at
 * `buf`, and the bits to flip. From the buffer's address each time: kept, 16 of them
 * went to scratch memory. e4m3's steps take 16 dims of K in turn from a load's 16 bytes. */
template <bool E4M3> DEV uint32_t q_lane(uint32_t buf, int row, int h) {
    return buf + row * 512 + (((E4M3 ? 2 * h : h) ^ (row & 15)) << 4);
}
template <bool E4M3> constexpr uint32_t q_step(int ks) {
    return (E4M3 ? 4 * (ks >> 1) + (ks & 1) : 2 * ks) << 4;
}
/* K of a page's keys, the first `keys` of them: what is past those reads as 0 */
template <bool E4M3> DEV __amdgpu_buffer_rsrc_t k_rows(const Weigh &c, size_t slice, int keys) {
    constexpr int ROW = PD * (E4M3 ? 1 : 2);
    const int bytes = __builtin_amdgcn_readfirstlane(min(max(keys, 0), PG) * ROW);
    return make_rsrc((const char *)c.k + slice * PG * ROW, bytes);
}
/* Sums over the 32 lanes of a half, of pairs a, b: in rows 0, 2 of 16 lanes a's, in 1, 3 b's */
DEV float sum_rows(float a, float b) {
    const auto s =
        __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return fold_row(__uint_as_float(s[0]) + __uint_as_float(s[1]),
                    [](float p, float q) { return p + q; });
}
/* key of accumulator v of a block, lane half h */
DEV int key_at(int v, int h) { return 8 * (v >> 2) + 4 * h + (v & 3); }

constexpr int WEIGH_FEW = 128; /* rows */
/* A wave a page, up to this many: 64 sequences' token on 4096 bf16 keys 98 us, 5.5 TB/s,
 * so, 106 with two pages a wave, the next on its way, 113 with four; e4m3 55 (4.9 TB/s), 62
 * and 67; 512 on 1024 188 and 196 with two */
constexpr int WEIGH_WAVES = 1 << 20;

/* Few rows: bound by K's bytes. Each of a workgroup's four waves takes a page of the
 * sequence and kv-head, all 32 KiB of it on the way at once (and beyond WEIGH_WAVES every
 * blocks * 4-th page), and works on it 32 keys at a time. RB blocks of 32 rows. */
template <bool E4M3, int RB>
__global__ __launch_bounds__(256, 2) void weigh_few_kernel(Weigh c) {
    constexpr int ROW = PD * (E4M3 ? 1 : 2), NL = E4M3 ? 8 : 16; /* loads of 32 keys */
    __shared__ __attribute__((aligned(1024))) unsigned char smem[RB * 16384];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int col = lane & 31, h = lane >> 5;
    const int kh = blockIdx.x % c.Hkv, at = blockIdx.x / c.Hkv;
    const int b = at / c.blocks, stride = c.blocks * 4;
    int tile = (at % c.blocks) * 4 + wave;
    const pg_seq s = load_seq(c.q_start, c.kv_len, b, c.N, c.max_q, c.max_kv);
    const int tiles = pg_div_up(s.kv, PG);
    if (s.ql <= 0 || (at % c.blocks) * 4 >= tiles)
        return;
    /* the page ids of 64 of the wave's tiles, one a lane */
    int ids = -1, ids0 = tile;
    auto page_of = [&](int t) {
        if (t == ids0 || t - ids0 >= 64 * stride) {
            ids0 = t;
            const int mine = t + lane * stride;
            ids = mine < tiles ? c.page_table[(size_t)b * c.max_pages + mine] : -1;
            ids = ids < c.num_pages ? ids : -1;
        }
        return __builtin_amdgcn_readlane(ids, (t - ids0) / stride);
    };
    const int nrows = s.ql * c.G;
    const __amdgpu_buffer_rsrc_t qsrc =
        make_rsrc(c.q + ((size_t)s.q0 * c.Hq + kh * c.G) * PD, 0x7fffffff);
#pragma unroll
    for (int i = 0; i < RB * 4; i++)
        q_rows(c, qsrc, smem, (i * 4 + wave) * 2, 0, nrows - 1);
    /* this lane's rows: lse (+inf: none, or it sees nothing), and the last key each sees */
    float lse[RB];
    int last[RB];
#pragma unroll
    for (int r = 0; r < RB; r++) {
        const int row = min(32 * r + col, nrows - 1), tok = row * c.rG >> 16;
        const float x = c.lse[(size_t)(s.q0 + tok) * c.Hq + kh * c.G + row - tok * c.G];
        lse[r] = 32 * r + col < nrows && x != -INFINITY ? x : INFINITY;
        last[r] = s.p0 + tok;
    }
    u32x4 raw[2][NL];
    float sc[2] = {1.f, 1.f};
    auto load = [&](int half, int page, int t) { /* of tile t */
        const size_t slice = (size_t)max(page, 0) * c.Hkv + kh;
        const int keys = page < 0 ? 0 : s.kv - t * PG;
        const __amdgpu_buffer_rsrc_t src = k_rows<E4M3>(c, slice, keys);
#pragma unroll
        for (int n = 0; n < NL; n++)
            raw[half][n] = buf_load16(src, col * ROW + h * 16, half * 32 * ROW + n * 32);
        if constexpr (E4M3) {
            const float x = c.ks[slice * PG + 32 * half + col];
            sc[half] = 32 * half + col < keys ? x : 1.f;
        }
    };
    int page = page_of(tile);
    load(0, page, tile);
    load(1, page, tile);
    /* Q is there (all waves' part of it) */
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    while (tile < tiles) {
        const int next = tile + stride, next_page = next < tiles ? page_of(next) : -1;
        unroll_for<2>([&](auto ih) {
            constexpr int half = decltype(ih)::value;
            const int key0 = tile * PG + 32 * half;
            /* after the sums lane 16 r + v (v < 8) is left with accumulator v + 8 (r & 1) */
            const int mine = key_at((lane & 7) + (lane >> 4 & 1) * 8, h);
            const size_t to = ((size_t)max(page, 0) * c.Hkv + kh) * PG + 32 * half + mine;
            const bool own = !(lane & 8) && page >= 0 && key0 + mine < s.kv;
            const bool add = own && c.prev && key0 + mine < s.p0;
            float before = 0.f;
            if (add)
                before = c.prev[to];
            float sum[16] = {};
#pragma unroll
            for (int r = 0; r < RB; r++) {
                if (32 * r >= nrows) /* uniform */
                    break;
                const uint32_t q0 = q_lane<E4M3>(r * 16384, col, h);
                floatx16 x = {};
#pragma unroll
                for (int ks = 0; ks < 16; ks++) {
                    const bf16x8 q = *(const bf16x8 *)(smem + (q0 ^ q_step<E4M3>(ks)));
                    bf16x8 k;
                    if constexpr (E4M3) {
                        const u32x4 v = raw[half][ks >> 1];
                        k = ks & 1 ? widen(v[2], v[3], sc[half]) : widen(v[0], v[1], sc[half]);
                    } else {
                        k = __builtin_bit_cast(bf16x8, raw[half][ks]);
                    }
                    x = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k, q, x, 0, 0, 0);
                }
                if (key0 + 31 <= s.p0) { /* uniform: all rows see them all */
#pragma unroll
                    for (int v = 0; v < 16; v++)
                        sum[v] += fast_exp2(x[v] - lse[r]);
                } else {
                    const int seen = last[r] - key0 - 4 * h;
#pragma unroll
                    for (int v = 0; v < 16; v++) {
                        const float p = fast_exp2(x[v] - lse[r]);
                        sum[v] += key_at(v, 0) <= seen ? p : 0.f;
                    }
                }
            }
            if (next < tiles)
                load(half, next_page, next);
            float all = 0.f;
#pragma unroll
            for (int v = 0; v < 8; v++) {
                const float y = sum_rows(sum[v], sum[v + 8]);
                all = (lane & 7) == v ? y : all;
            }
            if (own)
                c.w[to] = all + before;
        });
        tile = next, page = next_page;
    }
}

/* Many rows: bound by the matrix cores. A workgroup holds four pages of a kv-head's K in
 * registers, a wave 64 keys as the A operands of v_mfma_f32_16x16x32_bf16, and streams
 * packed rows through LDS, 16 for each of its two row groups a step: a Q operand feeds
 * four products, and LDS holds four steps, of which three are on their way. Few blocks
 * of keys share their rows out among several workgroups, whose sums weigh_sum_kernel
 * adds up. Half a step's products go beside the exponentials of the half before. 4096
 * tokens on 8192 keys, 16 / 4 heads, bf16, call after call: 202 us with the sums' 4.8,
 * 1.02 PFLOP/s, 75 % of a large library product's rate in the same loop (1.37). */
constexpr int WEIGH_KG = 4, WEIGH_AHEAD = 4, WEIGH_GROUPS = 1024, WEIGH_STEPS = 4;
template <bool E4M3> DEV void weigh_many(const Weigh &c) {
    constexpr int KG = WEIGH_KG, STEP = 32; /* rows a step, in two halves */
    constexpr int QB = STEP * PD * 2;       /* bytes of a step's Q */
    constexpr int NB = WEIGH_AHEAD;         /* steps that LDS holds */
    constexpr int NL = QB / (KG * 1024);    /* a wave's loads of a step */
    constexpr int ROW = PD * (E4M3 ? 1 : 2);
    constexpr int QD = 3; /* Q operand reads ahead */
    /* Q of NB steps, their lse, and at the end the sums: one array, since of several the
     * compiler waits for all loads to any of them before it reads one */
    constexpr int LSE = NB * QB;
    __shared__ __attribute__((aligned(1024))) unsigned char smem[LSE + NB * STEP * 4];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int col = lane & 15, g = lane >> 4;
    /* where the kv-heads divide the 8 XCDs, an XCD's workgroups read the same rows; the
     * blocks of the most rows, a sequence's first, start first */
    int kh, kb, b, split;
    {
        const int per = 8 % c.Hkv == 0 ? 8 / c.Hkv : 1, items = c.blocks * c.splits;
        const int all = pg_div_up(items, per) * per * c.Hkv;
        b = blockIdx.x / all;
        int at = blockIdx.x % all;
        if (8 % c.Hkv == 0) {
            kh = (at & 7) / per;
            at = (at >> 3) * per + (at & 7) % per;
        } else {
            kh = at % c.Hkv;
            at = at / c.Hkv;
        }
        kb = at / c.splits;
        split = at % c.splits;
    }
    const pg_seq s = load_seq(c.q_start, c.kv_len, b, c.N, c.max_q, c.max_kv);
    const int k0 = kb * KG * PG; /* the workgroup's first key */
    if (s.ql <= 0 || k0 >= s.kv || kb >= c.blocks)
        return;
    const int key0 = k0 + wave * PG; /* the wave's */
    int page = -1;
    if (key0 < s.kv) {
        page = __builtin_amdgcn_readfirstlane(c.page_table[(size_t)b * c.max_pages + key0 / PG]);
        page = page >= 0 && page < c.num_pages ? page : -1;
    }
    const size_t slice = (size_t)max(page, 0) * c.Hkv + kh;

    /* Rows: the tokens from position k0 on, and all behind it; the last ones first, so that
     * the workgroups of a kv-head, whatever their first, read the same ones at a time. A
     * step has as many whole tokens as fit: where a lane's rows lie in its Q is the same
     * in all steps. Past the last token Q and lse read as 0. */
    const int t_first = max(k0 - s.p0, 0), toks = STEP / c.G;
    const int all_steps = pg_div_up(s.ql - t_first, toks);
    const int n0 = (int)((long long)all_steps * split / c.splits);
    const int steps = (int)((long long)all_steps * (split + 1) / c.splits);
    auto part = [&](int k) { /* key0 + k's place among this split's sums */
        return c.parts + (((size_t)split * c.B + b) * c.Hkv + kh) * c.blocks * (KG * PG) + key0 + k;
    };
    if (n0 == steps) { /* uniform: fewer steps than splits, and none is this one's */
        *part(lane) = 0.f;
        return;
    }
    uint32_t qoff[NL];
#pragma unroll
    for (int i = 0; i < NL; i++) {
        const int at = (i * KG + wave) * 2 + (lane >> 5), tok = at * c.rG >> 16;
        qoff[i] = tok < toks ? (tok * c.Hq + at - tok * c.G) * PD * 2 +
                                   (((lane & 31) ^ (at & 15)) << 4)
                             : 0x7ffffff0u; /* no row: it reads as 0 */
    }
    /* the most that a descriptor spans: below qoff of no row */
    constexpr size_t SPAN = 0x7fff0000;
    /* from step `steps` on the first tokens again: what a wait counts stays the same */
    auto first_tok = [&](int n) { return max(s.ql - (n + 1) * toks, t_first); };
    auto issue = [&](int n) {
        const int i0 = first_tok(n);
        const size_t from = (size_t)(s.q0 + i0) * c.Hq + kh * c.G;
        const size_t left = (size_t)(s.ql - i0) * c.Hq - kh * c.G;
        const int bytes = (int)min(left * PD * 2, SPAN);
        const __amdgpu_buffer_rsrc_t src =
            make_rsrc(c.q + from * PD, __builtin_amdgcn_readfirstlane(bytes));
#pragma unroll
        for (int i = 0; i < NL; i++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                src, (lds_ptr)(smem + n % NB * QB + (i * KG + wave) * 1024), 16, qoff[i], 0, 0, 0);
        const int at = lane_again(); /* worked out each time, not kept: registers */
        if (wave == 0 && at < STEP) {
            const int lbytes = (int)min(left * 4, SPAN), tok = at * c.rG >> 16;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                make_rsrc(c.lse + from, __builtin_amdgcn_readfirstlane(lbytes)),
                (lds_ptr)(smem + LSE + n % NB * (STEP * 4)), 4,
                (tok * c.Hq + at - tok * c.G) * 4, 0, 0, 0);
        }
    };
#pragma unroll
    for (int i = 0; i < NB - 1; i++)
        issue(n0 + i);
    bf16x8 kf[4][8];
    {
        const int keys = page < 0 ? 0 : s.kv - key0;
        const __amdgpu_buffer_rsrc_t src = k_rows<E4M3>(c, slice, keys);
        const uint32_t voff = col * ROW + g * 16;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (E4M3) {
                u32x4 raw[4];
#pragma unroll
                for (int n = 0; n < 4; n++)
                    raw[n] = buf_load16(src, voff, i * 16 * ROW + n * 64);
                const float x = c.ks[slice * PG + 16 * i + col];
                const float sc = 16 * i + col < keys ? x : 1.f;
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    kf[i][2 * n] = widen(raw[n][0], raw[n][1], sc);
                    kf[i][2 * n + 1] = widen(raw[n][2], raw[n][3], sc);
                }
            } else {
#pragma unroll
                for (int n = 0; n < 8; n++)
                    kf[i][n] =
                        __builtin_bit_cast(bf16x8, buf_load16(src, voff, i * 16 * ROW + n * 64));
            }
        }
    }
    float sum[4][4] = {};
    floatx4 xa[4] = {}, xb[4] = {};
    /* this lane's operand of row col of a step, the k-steps' bits flipped */
    const uint32_t q_row = col * 512 + (((E4M3 ? 2 * g : g) ^ col) << 4);
    bf16x8 ring[QD];
    /* operand j of a step: k-step j % 8 of half j / 8 */
    auto q_at = [&](uint32_t q0, int j) {
        const int ks = j & 7;
        const uint32_t bits = (E4M3 ? 8 * (ks >> 1) + (ks & 1) : 4 * ks) << 4;
        return __builtin_bit_cast(
            bf16x8, lds_read16((lds_u8 *)smem, (q0 ^ bits) + (j >> 3) * (16 * PD * 2)));
    };
    /* Products of a half of step n into x; beside(ks) goes between the k-steps */
    auto products = [&](auto ih, uint32_t q0, floatx4 (&x)[4], auto beside) {
        constexpr int half = decltype(ih)::value;
        unroll_for<8>([&](auto iks) {
            constexpr int ks = decltype(iks)::value, j = 8 * half + ks;
            const bf16x8 q = ring[j % QD];
            if constexpr (j + QD < 16)
                ring[j % QD] = q_at(q0, j + QD);
#pragma unroll
            for (int i = 0; i < 4; i++)
                x[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[i][ks], q,
                                                               ks ? x[i] : floatx4{}, 0, 0, 0);
            beside(iks);
            __builtin_amdgcn_sched_barrier(0); /* no more operands at a time: registers */
        });
    };
    int my_tok[2]; /* of this lane's row of each half */
#pragma unroll
    for (int i = 0; i < 2; i++)
        my_tok[i] = 16 * i + col < toks * c.G ? (16 * i + col) * c.rG >> 16 : 0x7fffffff;
    /* a half that is done: its lane's lse (+inf: no row, or it sees nothing), the last key
     * that the row sees, from key0 + 4 g on, and whether all rows see all the wave's keys */
    struct Row {
        float lse;
        int seen;
        bool whole;
    };
    auto row_of = [&](int n, int half) {
        const float l =
            *(lds_f32)((lds_u8 *)smem + LSE + n % NB * (STEP * 4) + half * 64 + col * 4);
        const int tok = my_tok[half];
        const int i0 = first_tok(n); /* the last step's tokens end where the others began */
        const bool there = tok < s.ql - n * toks - i0;
        Row r;
        r.lse = there && l != -INFINITY ? l : INFINITY;
        r.whole = s.p0 + i0 >= key0 + PG - 1;
        r.seen = r.whole ? PG : s.p0 + i0 + min(tok, STEP) - key0 - 4 * g;
        return r;
    };
    /* The difference before the power: 2^x times 2^-lse would be a product added at once, but
     * either may leave fp32's range where the weight does not */
    auto add_whole = [&](const floatx4 (&x)[4], float lse, int m) {
        sum[m >> 2][m & 3] += fast_exp2(x[m >> 2][m & 3] - lse);
    };
    auto add = [&](const floatx4 (&x)[4], const Row &r) {
#pragma unroll
        for (int m = 0; m < 16; m++) {
            const float p = fast_exp2(x[m >> 2][m & 3] - r.lse);
            sum[m >> 2][m & 3] += 16 * (m >> 2) + (m & 3) <= r.seen ? p : 0.f;
        }
    };
    /* a half's products into y, and beside them what x has of the half before */
    auto turn = [&](auto ih, uint32_t q0, floatx4 (&y)[4], const floatx4 (&x)[4], const Row &r) {
        if (r.whole) {
            products(ih, q0, y, [&](auto iks) {
                constexpr int ks = decltype(iks)::value;
                add_whole(x, r.lse, 2 * ks);
                add_whole(x, r.lse, 2 * ks + 1);
            });
        } else {
            add(x, r);
            products(ih, q0, y, [](auto) {});
        }
    };
    Row before{INFINITY, 0, true}; /* ahead of the first half: nothing */
    for (int n = n0; n < steps; n++) {
        /* step n's Q is there, and that of n - 1 read: its place takes step n + NB - 1's */
        if (wave == 0)
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NB - 2) * (NL + 1)) : "memory");
        else
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NB - 2) * NL) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const uint32_t q0 = n % NB * QB + q_row;
#pragma unroll
        for (int j = 0; j < QD; j++)
            ring[j] = q_at(q0, j);
        issue(n + NB - 1);
        const Row r = row_of(n, 0);
        turn(template_int<0>{}, q0, xa, xb, before);
        before = row_of(n, 1);
        turn(template_int<1>{}, q0, xb, xa, r);
    }
    add(xb, before);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    /* over the 16 rows' lanes: lane 16 g + m is left with block m >> 2, number m & 3 */
    const int id = lane_again();
    float mine = 0.f;
#pragma unroll
    for (int m = 0; m < 16; m++) {
        const float y = fold_row(sum[m >> 2][m & 3], [](float p, float q) { return p + q; });
        mine = (id & 15) == m ? y : mine;
    }
    /* and left with key l of the wave's in lane l */
    mine = __shfl(mine, (id >> 2 & 3) * 16 + (id >> 4) * 4 + (id & 3), 64);
    {
        if (c.splits > 1) {
            *part(id) = mine;
        } else if (page >= 0 && key0 + id < s.kv) {
            const size_t to = slice * PG + id;
            if (c.prev && key0 + id < s.p0)
                mine += c.prev[to];
            c.w[to] = mine;
        }
    }
}

template <bool E4M3> __global__ __launch_bounds__(256, 2) void weigh_many_kernel(Weigh c) {
    weigh_many<E4M3>(c);
}

/* The splits' sums of a key, in order: a thread a key */
__global__ __launch_bounds__(256) void weigh_sum_kernel(Weigh c) {
    const int kh = blockIdx.x % c.Hkv, at = blockIdx.x / c.Hkv;
    const int b = at / c.blocks, key = at % c.blocks * 256 + threadIdx.x;
    const pg_seq s = load_seq(c.q_start, c.kv_len, b, c.N, c.max_q, c.max_kv);
    if (s.ql <= 0 || key >= s.kv)
        return;
    const int page = c.page_table[(size_t)b * c.max_pages + key / PG];
    if (page < 0 || page >= c.num_pages)
        return;
    const size_t all = (size_t)c.B * c.Hkv * c.blocks * 256;
    const float *from = c.parts + ((size_t)b * c.Hkv + kh) * c.blocks * 256 + key;
    const size_t to = ((size_t)page * c.Hkv + kh) * PG + key % PG;
    float x = c.prev && key < s.p0 ? c.prev[to] : 0.f;
    float sum = 0.f;
    for (int i = 0; i < c.splits; i += 8) { /* loads of 8 at a time */
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; j++)
            v[j] = from[min(i + j, c.splits - 1) * all];
#pragma unroll
        for (int j = 0; j < 8; j++)
            sum += i + j < c.splits ? v[j] : 0.f;
    }
    c.w[to] = x + sum;
}
static_assert(WEIGH_KG * PG == 256, "a thread a key of a block");

/* ---- positions to keep ------------------------------------------------------------
 * A workgroup per sequence and kv-head. The weights' order is that of 32-bit integers
 * (ordered()); the least one kept is found by its digits of 11, 11 and 10 bits from the
 * top, each by a histogram in LDS of what has the digits before. Then positions are
 * counted in order: heavier ones, and of its equals the first. A chain of loads, LDS and
 * barriers: 1 x 8192 keys 12 us, 64 sequences of up to 4096, a workgroup a CU, 9.5. */
constexpr int SEL_T = 1024;
struct Select {
    const float *w;
    int num_pages;
    const int32_t *page_table;
    int max_pages;
    const int32_t *kv_len;
    int max_kv, Hkv, budget, sinks, recent;
    int32_t *keep;
    int max_keep;
    int32_t *keep_len;
};
/* NaN above all, -0 as 0; 0 is below every weight */
DEV uint32_t ordered(float x) {
    const uint32_t u = __float_as_uint(x);
    if ((u & 0x7fffffffu) > 0x7f800000u)
        return ~0u;
    if ((u & 0x7fffffffu) == 0)
        return 0x80000000u;
    return u >> 31 ? ~u : u | 0x80000000u;
}
/* exclusive sum over the workgroup, and its total */
DEV int block_scan(int v, int *scratch, int *total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int to = wave_scan(v);
    __syncthreads();
    if (lane == 63)
        scratch[wave] = to;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < SEL_T / 64; i++) {
        const int x = scratch[i];
        before += i < wave ? x : 0;
        all += x;
    }
    *total = all;
    return before + to - v;
}

/* E tiles of SEL_T positions at a time, a thread's weights in registers: all there are, or
 * read again for each pass over them */
template <int E> __global__ __launch_bounds__(SEL_T) void select_kernel(Select c) {
    constexpr int SPAN = E * SEL_T, WAVES = SEL_T / 64;
    /* each pass's own: no barrier for their reuse */
    __shared__ int hist[3][2048], sums[3][WAVES], found[3][3];
    __shared__ int scratch[WAVES], counts[E * WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int kh = blockIdx.x % c.Hkv, b = blockIdx.x / c.Hkv;
    const int kv = min(max(c.kv_len[b], 0), c.max_kv), n = min(kv, c.budget);
    int32_t *keep = c.keep + (size_t)blockIdx.x * c.max_keep;
    if (kh == 0 && tid == 0)
        c.keep_len[b] = n;
    if (kv <= c.budget) {
        for (int i = tid; i < n; i += SEL_T)
            keep[i] = i;
        return;
    }
    const int lo = c.sinks, hi = kv - c.recent; /* the positions to choose among */
    const int want = n - c.sinks - c.recent;
    for (int i = tid; i < 2048; i += SEL_T)
        hist[0][i] = hist[1][i] = hist[2][i] = 0;
    uint32_t u[E];
    auto load = [&](int from) {
        int page[E];
#pragma unroll
        for (int e = 0; e < E; e++) {
            const int j = min(from + e * SEL_T + tid, kv - 1);
            page[e] = c.page_table[(size_t)b * c.max_pages + j / PG];
        }
#pragma unroll
        for (int e = 0; e < E; e++) {
            const int j = min(from + e * SEL_T + tid, kv - 1);
            const bool there = page[e] >= 0 && page[e] < c.num_pages;
            const float x = c.w[((size_t)(there ? page[e] : 0) * c.Hkv + kh) * PG + j % PG];
            u[e] = there ? ordered(x) : 0u;
        }
    };
    load(0);
    const bool again = kv > SPAN;
    /* the least kept: digits `top` so far under `mask`; ties: how many of its equals, `every`
     * one there is or not */
    uint32_t top = 0, mask = 0;
    int ties = want;
    bool every = want == 0;
    __syncthreads(); /* the histograms are clear */
    for (int pass = 0; want > 0 && pass < 3; pass++) {
        const int bits = pass < 2 ? 11 : 10, shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        for (int from = 0; from < kv; from += SPAN) {
            if (again)
                load(from);
#pragma unroll
            for (int e = 0; e < E; e++) {
                const int j = from + e * SEL_T + tid;
                const bool in = j >= lo && j < hi && (u[e] & mask) == top;
                const int digit = u[e] >> shift & ((1u << bits) - 1);
                /* the first lane's digit by one add: many weights may be the same */
                const uint64_t live = __ballot(in);
                if (!live)
                    continue;
                const int l = __ffsll((unsigned long long)live) - 1;
                const int d = __builtin_amdgcn_readlane(digit, l);
                const uint64_t same = __ballot(in && digit == d);
                if (lane == l)
                    atomicAdd(&hist[pass][d], __popcll(same));
                if (in && digit != d)
                    atomicAdd(&hist[pass][digit], 1);
            }
        }
        __syncthreads();
        /* from the top: two digits a thread */
        const int d1 = 2047 - 2 * tid, c1 = hist[pass][d1], c0 = hist[pass][d1 - 1];
        const int to = wave_scan(c1 + c0);
        if (lane == 63)
            sums[pass][wave] = to;
        __syncthreads();
        int above = to - c1 - c0;
#pragma unroll
        for (int i = 0; i < WAVES; i++)
            above += i < wave ? sums[pass][i] : 0;
        if (above < ties && above + c1 + c0 >= ties) {
            const bool first = above + c1 >= ties;
            found[pass][0] = first ? d1 : d1 - 1;
            found[pass][1] = ties - above - (first ? 0 : c1);
            found[pass][2] = first ? c1 : c0;
        }
        __syncthreads();
        top |= (uint32_t)found[pass][0] << shift;
        mask |= ((1u << bits) - 1) << shift;
        ties = found[pass][1];
        every = found[pass][2] == ties;
        if (every) /* all with these digits are kept, whatever the rest are */
            break;
    }
    /* In order, tile by tile and wave by wave: each wave's count of each tile to LDS, their
     * sums up to each in its place, and a lane's own by the lanes below. First of the least
     * kept one's equals, then of all that are kept. */
    auto ranks = [&](auto flag, int before, int (&rank)[E]) {
        uint64_t bal[E];
#pragma unroll
        for (int e = 0; e < E; e++) {
            bal[e] = __ballot(flag(e));
            if (lane == 0)
                counts[e * WAVES + wave] = __popcll(bal[e]);
        }
        __syncthreads();
        const int own = tid < E * WAVES ? counts[tid] : 0;
        int all;
        const int to = block_scan(own, scratch, &all);
        if (tid < E * WAVES)
            counts[tid] = to;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < E; e++)
            rank[e] = before + counts[e * WAVES + wave] +
                      __builtin_amdgcn_mbcnt_hi((uint32_t)(bal[e] >> 32),
                                                __builtin_amdgcn_mbcnt_lo((uint32_t)bal[e], 0));
        __syncthreads(); /* the counts are read */
        return before + all;
    };
    int kept = 0, equal = 0;
    for (int from = 0; from < kv; from += SPAN) {
        if (again)
            load(from);
        auto at = [&](int e) { return from + e * SEL_T + tid; };
        auto mid = [&](int e) { return at(e) >= lo && at(e) < hi && want > 0; };
        int rank[E] = {};
        if (!every)
            equal = ranks([&](int e) { return mid(e) && (u[e] & mask) == top; }, equal, rank);
        bool yes[E];
#pragma unroll
        for (int e = 0; e < E; e++)
            yes[e] = at(e) < kv &&
                     (at(e) < lo || at(e) >= hi ||
                      (mid(e) && ((u[e] & mask) > top ||
                                  ((u[e] & mask) == top && (every || rank[e] < ties)))));
        kept = ranks([&](int e) { return yes[e]; }, kept, rank);
#pragma unroll
        for (int e = 0; e < E; e++)
            if (yes[e] && rank[e] < n)
                keep[rank[e]] = at(e);
    }
}

/* ---- kept positions to the front -----------------------------------------------------
 * Slot dst + i takes what position keep[i] has: rows of K by lines of 128 bytes, V^T by
 * rows of dims, an element a slot, and scales and weights. In place a workgroup does its
 * lines or rows of a sequence and kv-head from the front to the back: positions ascend
 * and none is before the slot it goes to, so that all reads of a step are of slots that
 * no step before has written, and those of the step itself are done before its writes.
 * Bound by lines where few of a page are kept: 16 sequences of up to 4096 keys (41972) to
 * 1024 each, bf16, other pages, 43 us (the least of 20 33) for 187 MB, since all of V^T's
 * lines of 128 bytes are read for a quarter or more of each. In place one sequence of 8192
 * to 2048 takes 28, a chain of list, page ids, loads and stores a step. */
constexpr int KEEP_STEP = 256; /* slots a step, 64 a wave (K) or each wave all (V^T) */
constexpr int KEEP_VR = 8;     /* rows of V^T a wave */
struct Keep {
    void *k, *vt;
    float *ks, *vs, *w;
    int num_pages, Hkv;
    const int32_t *from, *to;
    int from_pages, to_pages;
    const int32_t *keep;
    int heads, max_keep; /* heads of keep: 1 or Hkv */
    const int32_t *dst, *keep_len;
    int units, steps, per; /* workgroups a sequence and head; steps in all, and of one */
};
/* where slot i's value comes from and goes to: (page Hkv + kh) PG + slot, -1: nowhere */
struct Move {
    long long src, dst;
};
DEV Move move_of(const Keep &c, int b, int kh, int n, int dst0, int i) {
    Move m{-1, -1};
    if (i >= n)
        return m;
    const int p = c.keep[((size_t)b * c.heads + (c.heads > 1 ? kh : 0)) * c.max_keep + i];
    const long long d = (long long)dst0 + i;
    if (p < 0 || p >= c.from_pages * PG || d < 0 || d >= (long long)c.to_pages * PG)
        return m;
    const int ps = c.from[(size_t)b * c.from_pages + p / PG];
    const int pd = c.to[(size_t)b * c.to_pages + (int)d / PG];
    if (ps < 0 || ps >= c.num_pages || pd < 0 || pd >= c.num_pages)
        return m;
    m.src = ((long long)ps * c.Hkv + kh) * PG + p % PG;
    m.dst = ((long long)pd * c.Hkv + kh) * PG + (int)d % PG;
    if (m.src == m.dst)
        m.dst = -1;
    return m;
}
DEV long long shfl(long long x, int l) {
    return (long long)(uint32_t)__shfl((int)x, l, 64) |
           (long long)__shfl((int)(x >> 32), l, 64) << 32;
}

template <bool E4M3> __global__ __launch_bounds__(256) void keep_kernel(Keep c) {
    typedef std::conditional_t<E4M3, uint8_t, uint16_t> elem;
    constexpr int LINES = PD * sizeof(elem) / 128; /* of a K row */
    constexpr int VBLOCKS = PD / (4 * KEEP_VR);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    int at = blockIdx.x;
    const int unit = at % c.units;
    at /= c.units;
    const int kh = at % c.Hkv;
    at /= c.Hkv;
    const int groups = pg_div_up(c.steps, c.per), group = at % groups, b = at / groups;
    const int n = min(max(c.keep_len[b], 0), c.max_keep), dst0 = c.dst ? c.dst[b] : 0;
    const int s0 = group * c.per, s1 = min(min(s0 + c.per, c.steps), pg_div_up(n, KEEP_STEP));
    if (unit < LINES) { /* K */
        for (int s = s0; s < s1; s++) {
            const Move m = move_of(c, b, kh, n, dst0, s * KEEP_STEP + 64 * wave + lane);
            u32x4 v[8];
            long long to[8];
            const int piece = unit * 128 + (lane & 7) * 16;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int l = 8 * i + (lane >> 3);
                const long long src = shfl(m.src, l);
                to[i] = shfl(m.dst, l);
                v[i] = *(const u32x4 *)((const char *)c.k +
                                        max(src, 0ll) * (long long)(PD * sizeof(elem)) + piece);
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads(); /* all waves' reads of the step */
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (to[i] >= 0)
                    *(u32x4 *)((char *)c.k + to[i] * (long long)(PD * sizeof(elem)) + piece) = v[i];
        }
        return;
    }
    if (unit < LINES + VBLOCKS) { /* V^T: the wave's own rows, no other's */
        const int d0 = ((unit - LINES) * 4 + wave) * KEEP_VR;
        elem *vt = (elem *)c.vt;
        for (int s = s0; s < s1; s++) {
            elem v[4][KEEP_VR];
            long long to[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const Move m = move_of(c, b, kh, n, dst0, s * KEEP_STEP + 64 * i + lane);
                const long long src = max(m.src, 0ll);
                to[i] = m.dst;
                const elem *p = vt + (src / PG) * PSLICE + d0 * PG + src % PG;
#pragma unroll
                for (int r = 0; r < KEEP_VR; r++)
                    v[i][r] = p[r * PG];
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (to[i] < 0)
                    continue;
                elem *p = vt + (to[i] / PG) * PSLICE + d0 * PG + to[i] % PG;
#pragma unroll
                for (int r = 0; r < KEEP_VR; r++)
                    p[r * PG] = v[i][r];
            }
        }
        return;
    }
    /* scales and weights: a wave each */
    float *x = wave == 0 ? c.w : wave == 1 ? c.ks : wave == 2 ? c.vs : nullptr;
    if (!x)
        return;
    for (int s = s0; s < s1; s++) {
        float v[4];
        long long to[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const Move m = move_of(c, b, kh, n, dst0, s * KEEP_STEP + 64 * i + lane);
            to[i] = m.dst;
            v[i] = x[max(m.src, 0ll)];
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (to[i] >= 0)
                x[to[i]] = v[i];
    }
}

} // namespace
} // namespace CUJEV_KNS
using namespace CUJEV_KNS;

/* How many rows: splits of a block's, so that the chip has WEIGH_GROUPS workgroups of them
 * (blocks of a prompt differ in rows: several each even out), of WEIGH_STEPS steps at
 * least. */
static int weigh_splits(long long units, int max_q, int G) {
    const int steps = pg_div_up(max_q, 32 / G);
    const long long n = pg_min((int)((WEIGH_GROUPS + units - 1) / units), steps / WEIGH_STEPS);
    return n > 1 ? (int)n : 1;
}
extern "C" size_t cujev_kv_weights_ws_bytes(int N, int B, int max_q, int max_kv, int Hq, int Hkv) {
    const long long mq = pg_min(max_q, N);
    if (mq <= 0 || B <= 0 || max_kv <= 0 || mq * (Hq / Hkv) <= WEIGH_FEW)
        return 0;
    /* of fewer units than WEIGH_GROUPS, splits times units are below twice as many */
    return (size_t)2 * WEIGH_GROUPS * 256 * sizeof(float);
}

extern "C" hipError_t k_kv_weights(const bf16_t *q, const float *lse, const cujev_kv_pages *pages,
                                   const cujev_paged_seqs *seqs, int N, int max_q, int max_kv,
                                   int Hq, const float *prev, float *weights, void *ws,
                                   size_t ws_bytes, hipStream_t stream) {
    const int Hkv = pages->Hkv, B = seqs->B, G = Hq / Hkv, tiles = pg_div_up(max_kv, PG);
    const int mq = pg_min(max_q, N);
    if (B <= 0 || mq <= 0 || tiles <= 0)
        return hipSuccess;
    if ((long long)B * tiles > (1ll << 40) / Hkv) /* tables beyond any memory */
        return hipErrorInvalidValue;
    const bool e4m3 = pages->type == CUJEV_KV_E4M3;
    const long long rows = (long long)mq * G;
    Weigh c = {(const bf16 *)q, lse, pages->k, pages->k_scale, pages->num_pages,
               seqs->q_start, seqs->kv_len, seqs->page_table, seqs->max_pages, B, N, max_q,
               max_kv, Hq, Hkv, G, pg_div_up(65536, G), 0, 1, prev, weights, (float *)ws};
    if (rows <= WEIGH_FEW) {
        const long long all = (long long)B * tiles * Hkv;
        const int pages_each = (int)((all + WEIGH_WAVES - 1) / WEIGH_WAVES);
        c.blocks = pg_div_up(tiles, 4 * pages_each);
        const long long grid = (long long)c.blocks * Hkv * B;
        if (grid * 256 > PG_MOST_ITEMS)
            return hipErrorInvalidValue;
        const dim3 g((unsigned)grid), t(256);
        auto launch = [&](auto ie) {
            constexpr bool E = decltype(ie)::value;
            if (rows <= 32)
                hipLaunchKernelGGL((weigh_few_kernel<E, 1>), g, t, 0, stream, c);
            else if (rows <= 64)
                hipLaunchKernelGGL((weigh_few_kernel<E, 2>), g, t, 0, stream, c);
            else
                hipLaunchKernelGGL((weigh_few_kernel<E, 4>), g, t, 0, stream, c);
        };
        if (e4m3)
            launch(std::true_type{});
        else
            launch(std::false_type{});
        return hipGetLastError();
    }
    c.blocks = pg_div_up(tiles, WEIGH_KG);
    const long long units = (long long)B * c.blocks * Hkv;
    if (units * 256 > PG_MOST_ITEMS)
        return hipErrorInvalidValue;
    c.splits = units < WEIGH_GROUPS ? weigh_splits(units, mq, G) : 1;
    if (c.splits > 1 && ws_bytes < (size_t)units * c.splits * 256 * sizeof(float))
        return hipErrorInvalidValue;
    const int per = 8 % Hkv == 0 ? 8 / Hkv : 1;
    const long long grid = (long long)pg_div_up(c.blocks * c.splits, per) * per * Hkv * B;
    if (grid * 256 > PG_MOST_ITEMS)
        return hipErrorInvalidValue;
    const dim3 g((unsigned)grid), t(256);
    if (e4m3)
        hipLaunchKernelGGL((weigh_many_kernel<true>), g, t, 0, stream, c);
    else
        hipLaunchKernelGGL((weigh_many_kernel<false>), g, t, 0, stream, c);
    if (c.splits > 1)
        hipLaunchKernelGGL(weigh_sum_kernel, dim3((unsigned)units), dim3(256), 0, stream, c);
    return hipGetLastError();
}

extern "C" hipError_t k_kv_select(const float *weights, int num_pages, int Hkv,
                                  const cujev_paged_seqs *seqs, int max_kv, int budget, int sinks,
                                  int recent, int32_t *keep, int max_keep, int32_t *keep_len,
                                  hipStream_t stream) {
    if (seqs->B <= 0)
        return hipSuccess;
    const long long grid = (long long)seqs->B * Hkv;
    if (grid * SEL_T > PG_MOST_ITEMS)
        return hipErrorInvalidValue;
    const Select c = {weights, num_pages, seqs->page_table, seqs->max_pages, seqs->kv_len, max_kv,
                      Hkv, budget, sinks, recent, keep, max_keep, keep_len};
#define LAUNCH(E)                                                                                 \
    hipLaunchKernelGGL((select_kernel<E>), dim3((unsigned)grid), dim3(SEL_T), 0, stream, c)
    if (max_kv <= 4 * SEL_T)
        LAUNCH(4);
    else if (max_kv <= 8 * SEL_T)
        LAUNCH(8);
    else
        LAUNCH(16);
#undef LAUNCH
    return hipGetLastError();
}

extern "C" hipError_t k_kv_keep(const cujev_kv_pages *pages, float *weights,
                                const cujev_paged_seqs *seqs, const int32_t *to_table,
                                int to_pages, const int32_t *keep, int keep_heads, int max_keep,
                                const int32_t *dst, const int32_t *keep_len, hipStream_t stream) {
    if (seqs->B <= 0 || max_keep <= 0)
        return hipSuccess;
    const bool e4m3 = pages->type == CUJEV_KV_E4M3;
    const int lines = PD * (e4m3 ? 1 : 2) / 128;
    const int units = lines + PD / (4 * KEEP_VR) + (weights || e4m3 ? 1 : 0);
    const int steps = pg_div_up(max_keep, KEEP_STEP), per = to_table ? 1 : steps;
    const long long groups = pg_div_up(steps, per);
    const long long each = groups * units * pages->Hkv;
    if (each > PG_MOST_ITEMS / 256 || each * seqs->B > PG_MOST_ITEMS / 256)
        return hipErrorInvalidValue;
    const Keep c = {pages->k, pages->vt, pages->k_scale, pages->v_scale, weights,
                    pages->num_pages, pages->Hkv, seqs->page_table,
                    to_table ? to_table : seqs->page_table, seqs->max_pages,
                    to_table ? to_pages : seqs->max_pages, keep, keep_heads, max_keep, dst,
                    keep_len, units, steps, per};
    const dim3 grid((unsigned)(each * seqs->B));
    if (e4m3)
        hipLaunchKernelGGL(keep_kernel<true>, grid, dim3(256), 0, stream, c);
    else
        hipLaunchKernelGGL(keep_kernel<false>, grid, dim3(256), 0, stream, c);
    return hipGetLastError();
}
