/* Attention over a paged K/V cache for gfx950.
 *
 * Row (n, h) of sequence b, at position p, sees the keys j <= p of b's pages
 * and, with a window W, of those only j > p - W and the first S (sinks):
 *   out = sigmoid(gate) sum_j 2^(q.k_j) v_j / sum_j 2^(q.k_j).
 *
 * The rows of one sequence that share a kv-head, ql new tokens x G q-heads, are
 * packed (row r = token r / G, head r % G), so any G fills the same tiles.
 * Both kernels below run S^T = K Q^T and O^T += V^T P^T on matrix
 * instructions, keys (or dims) on the M side and rows on N: a lane holds
 * scores of one row, and feeding K's rows in the right order makes its score
 * accumulators exactly the P operand of the next product. e4m3 pages become
 * bf16 operands in registers, exactly: K's scale is the conversion's, V's (one
 * per key, the summed index) multiplies p before its rounding, which a power
 * of two does not change.
 *
 * Scores, maxima, l and O are fp32. p is rounded to bf16, the operand that the
 * matrix instructions take (l sums it before), as the contiguous attention rounds
 * it: with the result's rounding 2.1e-3 to 2.3e-3 of the result (RMS), 1.65e-3 by
 * the latter alone. */
#include "paged.h"

#include <type_traits>

namespace CUJEV_KNS {
namespace {

DEV void lds_write16(unsigned char *base, uint32_t off, u32x4 v) { *(u32x4 *)(base + off) = v; }


/* x of lane i of this lane's 16 (DPP row broadcast) */
template <int i> DEV float row_lane(float x) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(
        0, (int)__float_as_uint(x), 0x150 + i, 0xf, 0xf, false));
}
/* x, or -inf where the key is hidden. On the bits: hidden scores may be NaN. */
DEV float hide(bool seen, float x) {
    return __uint_as_float(seen ? __float_as_uint(x) : 0xff800000u);
}

/* v_mfma_f32_32x32x16_bf16 by hand, so that O and Q stay in accumulation registers
 * and the scores in ordinary ones; with the builtin the compiler moved Q's operands
 * over before each MFMA. What it leaves to the code around it: two wait states
 * between a VALU write of an operand and the MFMA (NOP), and 18 between an MFMA and
 * a read of its result by anything but the next MFMA on it (settle()). Operands from
 * LDS are waited for as for any instruction. */
#define MFMA "v_mfma_f32_32x32x16_bf16 "
template <bool NOP> DEV void mfma_first(floatx16 &s, bf16x8 a, bf16x8 q) {
    if constexpr (NOP)
        asm volatile("s_nop 1\n\t" MFMA "%0, %1, %2, 0" : "=&v"(s) : "v"(a), "a"(q));
    else
        asm volatile(MFMA "%0, %1, %2, 0" : "=&v"(s) : "v"(a), "a"(q));
}
template <bool NOP> DEV void mfma_score(floatx16 &s, bf16x8 a, bf16x8 q) {
    if constexpr (NOP)
        asm volatile("s_nop 1\n\t" MFMA "%0, %1, %2, %0" : "+v"(s) : "v"(a), "a"(q));
    else
        asm volatile(MFMA "%0, %1, %2, %0" : "+v"(s) : "v"(a), "a"(q));
}
template <bool NOP> DEV void mfma_out(floatx16 &o, bf16x8 a, bf16x8 p) {
    if constexpr (NOP)
        asm volatile("s_nop 1\n\t" MFMA "%0, %1, %2, %0" : "+a"(o) : "v"(a), "v"(p));
    else
        asm volatile(MFMA "%0, %1, %2, %0" : "+a"(o) : "v"(a), "v"(p));
}
DEV void mfma_zero(floatx16 &o, bf16x8 none) { /* none: zeros */
    asm volatile("s_nop 1\n\t" MFMA "%0, %1, %1, 0" : "=a"(o) : "v"(none));
}
#undef MFMA
/* before O is read or written by anything but mfma_out, and after */
DEV void settle(floatx16 (&o)[4]) {
    asm volatile("s_nop 15\n\ts_nop 7" : "+a"(o[0]), "+a"(o[1]), "+a"(o[2]), "+a"(o[3]));
}

/* keys hi at most, and past lo or a sink (without branches) */
DEV bool key_seen(int j, int hi, int lo, int sinks) { return (j <= hi) & ((j > lo) | (j < sinks)); }
/* the same of keys j .. j + N - 1, a bit each (0 <= j <= PG_MOST_KEYS, hi >= -PG_MOST and
 * lo >= -1, so that no difference leaves an int) */
template <int N> DEV uint32_t keys_seen(int j, int hi, int lo, int sinks) {
    auto below = [&](int x) { return (1u << min(max(x - j, 0), N)) - 1; }; /* keys < x */
    return below(hi + 1) & (~below(lo + 1) | below(sinks));
}
/* Bit `bit` to all of a word; x, or -inf where it says hidden */
template <int bit> DEV uint32_t spread_bit(uint32_t bits) {
    return (uint32_t)((int)(bits << (31 - bit)) >> 31);
}
/* four bits to a byte each, two to two bytes each */
DEV uint32_t bytes_by(uint32_t bits) { return ((bits & 15) * 0x204081u & 0x1010101u) * 0xffu; }
template <int bit> DEV uint32_t halves_by(uint32_t bits) {
    return (spread_bit<bit>(bits) & 0xffffu) | (spread_bit<bit + 1>(bits) & 0xffff0000u);
}
template <int bit> DEV float hide_by(uint32_t bits, float x) {
    const uint32_t m = spread_bit<bit>(bits);
    return __uint_as_float((__float_as_uint(x) & m) | (0xff800000u & ~m));
}

/* What the kernels and the merge share.
 *
 * The work of a kv-head is its units, tiles of packed rows of a sequence. So that
 * all parts of a call finish together however uneven its sequences are, each
 * workgroup works out the same plan from q_start and kv_len: what all units have
 * to do, over what the chip runs at once, gives the size of a share
 * (paged_index.h). A unit that several shares work on keeps, in a slot for each,
 * unnormalised o, l and the softmax's reference mu of its rows, for the merge. */
struct Call {
    const bf16 *q, *gate;
    int gts, ghs;
    const void *k, *vt;
    const float *ks, *vs;
    int num_pages;
    const int32_t *q_start, *kv_len, *page_table;
    int max_pages, B, N, max_q, max_kv, Hq, Hkv, G, window, sinks;
    /* the same for lists of tiles and the plan: 0 where no window ends behind key 0 of
     * the call's max_kv. A row past max_kv keys (of a longer sequence) has a mask
     * all the same. */
    int list_window, list_sinks;
    int rG; /* r / G = r * rG >> 16 for r < 4096 (an integer division is 30 instructions) */
    /* LSE and TREE calls: [N][words], bit j of row n: it sees its sequence's new token j;
     * log2 of sum 2^(q.k), [N][Hq], -inf where there is none (NULL: not asked for) */
    const uint64_t *tree;
    int words;
    float *lse;
    bf16 *out;
    float *po, *pl, *pmu;
    /* for the merge: few rows {first piece, parts} of each sequence, many rows
     * {sequence, unit, parts (0: not a unit's first), 0} of each part */
    int32_t *info;
    pg_plan plan;
};
DEV pg_seq seq_of(const Call &c, int b) {
    return load_seq(c.q_start, c.kv_len, b, c.N, c.max_q, c.max_kv);
}
DEV int page_id(const Call &c, int b, const pg_tiles &t, int i) {
    const int page = c.page_table[(size_t)b * c.max_pages + pg_tile_page(t, i)];
    return page >= 0 && page < c.num_pages ? page : -1;
}

/* What a call asks for: causal rows; the same with lse; rows of a tree of drafted tokens.
 * Kinds of their own, so that the first one's code stays what it is. */
enum { CAUSAL, LSE, TREE };
/* TREE: the keys k0 .. k0 + 63 that the row with these words sees by its tree, first key
 * lowest: all before the sequence's first new token (at p0), then as the bits say. Both
 * words are loaded, whichever count: conditional loads came one after the other. */
DEV uint64_t tree_keys(const uint64_t *row, int words, int k0, int p0) {
    const int at = k0 - p0, i = at >> 6, sh = at & 63; /* i -1: the tile that p0 is in */
    uint64_t lo = row[min(max(i, 0), words - 1)], hi = row[min(max(i + 1, 0), words - 1)];
    lo = i < 0 ? ~0ull : i < words ? lo : 0;
    hi = i < -1 ? ~0ull : i + 1 < words ? hi : 0;
    return sh ? lo >> sh | hi << (64 - sh) : lo;
}
/* the same of a sequence of up to 64 new tokens, from its row's first word */
DEV uint64_t tree_keys(uint64_t word, int k0, int p0) {
    const int at = k0 - p0;
    return at <= -64 ? ~0ull
           : at < 0  ? word << -at | ((1ull << -at) - 1)
                     : at < 64 ? word >> at : 0;
}
template <class F> DEV uint64_t each_half(uint64_t x, F f) {
    return (uint64_t)f((uint32_t)(x >> 32)) << 32 | f((uint32_t)x);
}
/* or over the lanes of each row of 16; over the wave */
template <int ctrl> DEV uint32_t or_dpp(uint32_t v) {
    return v | (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, 0xf, 0xf, true);
}
DEV uint32_t or_row(uint32_t v) { /* row_ror 8, 4, 2, 1 */
    return or_dpp<0x121>(or_dpp<0x122>(or_dpp<0x124>(or_dpp<0x128>(v))));
}
DEV uint64_t or_row(uint64_t x) {
    return each_half(x, [](uint32_t v) { return or_row(v); });
}
DEV uint64_t or_wave(uint64_t x) {
    return or_row(each_half(x, [](uint32_t v) {
        auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        const uint32_t u = a[0] | a[1];
        a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
        return (uint32_t)(a[0] | a[1]);
    }));
}
/* log2 of l 2^mu; -inf for a row that has seen no key */
DEV float lse_of(float l, float mu) { return l > 0.f ? mu + __builtin_amdgcn_logf(l) : -INFINITY; }

/* The unit that share `target` of a kv-head belongs to (few rows: the one that piece
 * `target` begins in): its sequence (b -1: there is none), its number in it, its parts,
 * the first one's number (few rows: its piece's), which of them `target` is. */
struct Where {
    pg_seq s;
    int b, unit, parts, first, part;
    int begin, own, size; /* few rows: the unit on the line, tiles a piece */
};
/* many rows: w's unit, parts and first from its sequence, whose parts begin at `have` */
DEV void set_part(const Call &c, Where &w, int target, int have, int share) {
    const int whole = pg_short_units(w.s, c.G, c.list_window, w.own, share), at = target - have;
    w.parts = at < whole ? 1 : pg_nshare(w.own, share);
    w.unit = at < whole ? at : whole + (at - whole) / w.parts;
    w.first = at < whole ? target : have + whole + (w.unit - whole) * w.parts;
}
/* J sequences a lane, 64 J a step: what all have, then where target lies */
template <int RT_, int J> DEV Where locate_among(const Call &c, int target) {
    constexpr bool FEWR = RT_ == PG_FEW;
    const int lane = threadIdx.x & 63;
    pg_seq s[J];
    int units[J], n[J];
    auto read = [&](int b0) {
#pragma unroll
        for (int j = 0; j < J; j++)
            s[j] = seq_of(c, min(b0 + J * lane + j, c.B - 1));
#pragma unroll
        for (int j = 0; j < J; j++) {
            units[j] = b0 + J * lane + j < c.B ? pg_units(s[j], c.G, RT_) : 0;
            n[j] = units[j] ? pg_longest(s[j], c.G, RT_, c.list_window, c.list_sinks) : 0;
        }
    };
    auto parts_of = [&](int j, int share) {
        return units[j] ? pg_parts(s[j], c.G, c.list_window, n[j], share) : 0;
    };
    if constexpr (J == 1) /* the only step */
        read(0);
    int size = PG_MOST;
    if (FEWR || c.plan.goal > 0) {
        int U = 0, longest = 0;
        unsigned T = 0;
        for (int b0 = 0; b0 < c.B; b0 += 64 * J) {
            if constexpr (J > 1)
                read(b0);
#pragma unroll
            for (int j = 0; j < J; j++) {
                T += FEWR || J > 1 ? (unsigned)units[j] * (unsigned)n[j]
                                   : pg_all_tiles(s[j], c.G, c.list_window, n[j]) * (units[j] > 0);
                U += units[j];
                longest = max(longest, n[j]);
            }
        }
        T = (unsigned)last_lane(wave_scan((int)T));
        U = last_lane(wave_scan(U));
        if constexpr (FEWR) {
            size = pg_few_share(c.plan, U, T);
        } else if (pg_splits(c.plan, U)) {
            size = pg_share_first(c.plan, U, T, J > 1);
            if constexpr (J == 1)
                while (last_lane(wave_scan(parts_of(0, size))) > c.plan.goal)
                    size = pg_share_next(size);
            longest = (int)fold_wave((float)longest, [](float p, float q) {
                return fmaxf(p, q); /* below 2^24 tiles: exact */
            });
            size = pg_share_last(size, __builtin_amdgcn_readfirstlane(longest));
        }
    }
    Where w;
    w.b = -1;
    const int item = FEWR ? target * size : target; /* a tile of the line, or a part */
    int before = 0;
    for (int b0 = 0; b0 < c.B; b0 += 64 * J) {
        if constexpr (J > 1)
            read(b0);
        int own[J], sum = 0;
#pragma unroll
        for (int j = 0; j < J; j++)
            sum += own[j] = FEWR ? units[j] * n[j] : parts_of(j, size);
        const int to = before + wave_scan(sum);
        const uint64_t past = __ballot(to > item);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            int at = __builtin_amdgcn_readlane(to - sum, l), have = 0;
            w.b = 0;
#pragma unroll
            for (int j = 0; j < J; j++) {
                const int here = __builtin_amdgcn_readlane(own[j], l);
                if (item >= at && item < at + here) {
                    w.s = seq_at(s[j], l);
                    w.b = b0 + J * l + j;
                    w.own = __builtin_amdgcn_readlane(n[j], l);
                    have = at;
                }
                at += here;
            }
            if constexpr (FEWR) {
                w.unit = 0, w.begin = have, w.size = size;
                w.first = have / size;
                w.parts = (have + w.own - 1) / size - w.first + 1;
            } else {
                set_part(c, w, target, have, size);
            }
            w.part = target - w.first;
            return w;
        }
        before = last_lane(to);
    }
    return w;
}
template <int RT_> DEV Where locate(const Call &c, int target) {
    constexpr bool FEWR = RT_ == PG_FEW;
    if (c.B > 64)
        return locate_among<RT_, 4>(c, target);
    if (c.B > 1)
        return locate_among<RT_, 1>(c, target);
    /* one sequence: no scan */
    Where w;
    w.b = -1, w.begin = 0;
    w.s = seq_of(c, 0);
    const int units = pg_units(w.s, c.G, RT_);
    const int n = pg_longest(w.s, c.G, RT_, c.list_window, c.list_sinks);
    if (units == 0)
        return w;
    if constexpr (FEWR) {
        w.size = pg_few_share(c.plan, 1, (unsigned)n);
        w.own = n;
        w.parts = (n - 1) / w.size + 1;
    } else {
        int share = PG_MOST;
        if (pg_splits(c.plan, units)) {
            share = pg_share_first(c.plan, units, pg_all_tiles(w.s, c.G, c.list_window, n), false);
            while (pg_parts(w.s, c.G, c.list_window, n, share) > c.plan.goal)
                share = pg_share_next(share);
            share = pg_share_last(share, n);
        }
        w.own = n;
        set_part(c, w, target, 0, share);
        w.part = target - w.first;
        w.b = w.unit < units ? 0 : -1;
        return w;
    }
    w.unit = target / w.parts;
    w.first = w.unit * w.parts;
    w.part = target - w.first;
    w.b = w.unit < units ? 0 : -1;
    return w;
}
/* The slot of part `at` of a kv-head */
DEV size_t slot_of(const Call &c, int kh, int at) { return (size_t)kh * c.plan.slots + at; }

/* ---- few rows: up to 16 packed rows of a sequence and kv-head ------------------
 * Bound by the K/V bytes, so that what counts is that every wave of the chip
 * streams all the time. The key tiles of all units of a kv-head are one line, cut
 * into equal pieces; a wave takes a piece, or the part of it that lies in one unit,
 * and waits for no other. K and V^T go from memory into registers as the operands
 * of v_mfma_f32_16x16x32_bf16, 16 bytes a lane and whole 128-byte lines within 16
 * loads (half a line of V^T at a time, 32 keys of bf16, read each line twice: 157 us
 * against 126 for 64 sequences of 2560 keys), in two sets of 16 registers' worth:
 *   e4m3  K of tile i + 1 is in flight during the softmax and the products with
 *         V^T, V^T during the scores
 *   bf16  a set holds 32 keys of K, then 128 dims of V^T; each goes out when the
 *         other's products begin
 * All loads are unconditional (past the end the last tile's again), so a wait for
 * one set's counts the other's in flight and not more; in 256 registers two waves
 * share a SIMD. Q waits in LDS: read again each tile, it leaves the registers to
 * loads.
 *
 * 64 sequences' tokens on up to 4096 keys, e4m3: 63 us for 320 MB (5.1 TB/s), and 5
 * for the merge; bf16 114 for 628 (5.5), and 5. A call of one tile takes 7.5 us, a
 * chain of loads: arguments, lengths, page ids, K, gates. */
constexpr int FEW = PG_FEW;

template <bool E4M3, int KIND>
__global__ __launch_bounds__(64, 2) void attention_few_kernel(Call c) {
    constexpr uint32_t EB = E4M3 ? 1 : 2, SLICE = PSLICE * EB;
    __shared__ bf16x8 sq[8 * 64];
    const int kh = blockIdx.x % c.Hkv;
    Where w = locate<FEW>(c, blockIdx.x / c.Hkv);
    /* the units that the piece lies in */
    while (w.b >= 0) {
        const int lane = lane_again(), m = lane & 15, g = lane >> 4;
        const pg_seq s = w.s;
        const int b = w.b, rows = min(s.ql * c.G, FEW);
        const pg_tiles list = pg_tile_list(s, 0, s.ql - 1, c.list_window, c.list_sinks);
        /* tiles [i0, i1) of the unit's; a unit without a key has one that is not there */
        const int cut = (w.first + w.part) * w.size - w.begin;
        const int i0 = max(cut, 0), i1 = min(min(cut + w.size, w.own), list.ntl);
        /* the ids of 64 tiles of the list are in a lane each */
        int ids = i0 < i1 ? page_id(c, b, list, min(i0 + lane, list.ntl - 1)) : -1, ids0 = i0;

        /* this lane's row (column of S^T and O^T) */
        const int row = min(m, rows - 1), tok = row * c.rG >> 16, head = kh * c.G + row - tok * c.G;
        const int hi = KIND == TREE ? s.kv - 1 : min(s.p0 + tok, s.kv - 1);
        const int lo = pg_low(s.p0 + tok, c.window);
        const int own_lo = pg_low(s.p0, c.window); /* of the first row: below, no row's key */
        bf16x8 *const qf = sq + lane;
        {
            const bf16 *qp = c.q + ((size_t)(s.q0 + tok) * c.Hq + head) * PD;
#pragma unroll
            for (int ks = 0; ks < 8; ks++) /* dims as K's loads below */
                qf[64 * ks] = *(const bf16x8 *)(qp + (E4M3 ? 64 * (ks >> 1) + 16 * g + 8 * (ks & 1)
                                                           : 32 * ks + 8 * g));
        }

        /* Row m of score block kb is key key0 + kkey(kb): lane g then holds, in
         * accumulators v = 4 kb .. + 3, the keys key_of(v) that its V^T loads bring. */
        const int key0 = (E4M3 ? 16 : 8) * (m >> 2) + (m & 3), keyg = (E4M3 ? 16 : 8) * g;
        auto kkey = [](int kb) { return E4M3 ? 4 * kb : 4 * (kb & 1) + 32 * (kb >> 1); };
        auto key_of = [&](int v) { return keyg + (E4M3 ? v : (v & 7) + 32 * (v >> 3)); };
        const uint32_t kvoff = key0 * PD * EB + 16 * g, vvoff = m * PG * EB + 16 * g;

        u32x4 ra[16] = {}, rb[16] = {}; /* e4m3: K, V^T; bf16: the first half of each, the second */
        float ksc[4] = {}, vsc = 1.f;
        auto rsrc = [&](const void *p, int page) {
            return make_rsrc((const char *)p + ((size_t)max(page, 0) * c.Hkv + kh) * SLICE, SLICE);
        };
        auto scale = [&](const float *p, int page, int key) { /* without a 64-bit address a lane */
            const __amdgpu_buffer_rsrc_t src =
                make_rsrc(p + ((size_t)max(page, 0) * c.Hkv + kh) * PG, PG * 4);
            return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(src, key * 4, 0, 0));
        };
        /* K: e4m3 all score blocks, bf16 blocks 2 part and 2 part + 1 */
        auto load_k = [&](u32x4 (&r)[16], int page, int part) {
            const __amdgpu_buffer_rsrc_t src = rsrc(c.k, page);
#pragma unroll
            for (int k = 0; k < (E4M3 ? 4 : 2); k++)
#pragma unroll
                for (int i = 0; i < (E4M3 ? 4 : 8); i++) /* the halves of a line in turn */
                    r[i * (E4M3 ? 4 : 2) + k] =
                        buf_load16(src, kvoff, kkey((E4M3 ? 0 : 2 * part) + k) * PD * EB + 64 * i);
            if constexpr (E4M3) {
#pragma unroll
                for (int kb = 0; kb < 4; kb++)
                    ksc[kb] = scale(c.ks, page, key0 + 4 * kb);
            }
        };
        /* V^T: e4m3 all 16 rows of 16 dims, bf16 8 of them, two halves of 32 keys each */
        auto load_v = [&](u32x4 (&r)[16], int page, int part) {
            const __amdgpu_buffer_rsrc_t src = rsrc(c.vt, page);
#pragma unroll
            for (int i = 0; i < 16; i++)
                r[i] = E4M3 ? buf_load16(src, vvoff + (i & 1) * 1024, (i >> 1) * 2048)
                            : buf_load16(src, vvoff + (i & 1) * 64, (8 * part + (i >> 1)) * 2048);
            if constexpr (E4M3) /* of key keyg + m, in lane m of the 16 that need all 16 */
                vsc = scale(c.vs, page, keyg + m);
        };
        /* tile t (past the last: it again): its page, -1 if it is not there */
        auto page_of = [&](int t) {
            t = min(t, i1 - 1);
            if (t - ids0 >= 64) {
                ids0 = t;
                ids = page_id(c, b, list, min(t + lane, list.ntl - 1));
            }
            return __builtin_amdgcn_readlane(ids, t - ids0);
        };

        floatx4 o[16];
#pragma unroll
        for (int t = 0; t < 16; t++)
            o[t] = floatx4{};
        float mrun = -INFINITY, lrun = 0.f;
        int next = -1;
        if (i0 < i1) {
            next = page_of(i0);
            load_k(ra, next, 0);
            if constexpr (!E4M3)
                load_k(rb, next, 1);
        }
        for (int i = i0; i < i1; i++) {
            const int page = next, k0 = pg_tile_page(list, i) * PG;
            const bool there = page >= 0;
            if constexpr (E4M3)
                load_v(rb, page, 0);
            next = page_of(i + 1);

            asm volatile("" ::: "memory"); /* Q is read here, not kept */
            floatx4 x[4];
            if constexpr (E4M3) {
#pragma unroll
                for (int ks = 0; ks < 8; ks++) {
                    const bf16x8 q = qf[64 * ks];
#pragma unroll
                    for (int kb = 0; kb < 4; kb++) {
                        const u32x4 v = ra[(ks >> 1) * 4 + kb];
                        x[kb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                            ks & 1 ? widen(v[2], v[3], ksc[kb]) : widen(v[0], v[1], ksc[kb]), q,
                            ks == 0 ? floatx4{} : x[kb], 0, 0, 0);
                    }
                }
                load_k(ra, next, 0);
            } else {
                auto scores = [&](u32x4 (&r)[16], int part) {
#pragma unroll
                    for (int ks = 0; ks < 8; ks++) {
                        const bf16x8 q = qf[64 * ks];
#pragma unroll
                        for (int k = 0; k < 2; k++)
                            x[2 * part + k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                                __builtin_bit_cast(bf16x8, r[2 * ks + k]), q,
                                ks == 0 ? floatx4{} : x[2 * part + k], 0, 0, 0);
                    }
                };
                scores(ra, 0);
                load_v(ra, page, 0);
                scores(rb, 1);
                load_v(rb, page, 1);
            }

            /* bits to keep of V^T values: those of no key of this call, whatever they
             * are, meet p = 0 */
            u32x4 keep[E4M3 ? 1 : 2];
            bool foreign = false;
            uint32_t tbits = 0;
            if (!there || !pg_tile_whole(k0, s.p0 - (KIND == TREE), s.p0 + s.ql - 1, s.kv, c.window,
                                         c.sinks)) {
                const int top = there ? s.kv - 1 : -1;
                if constexpr (KIND == TREE) {
                    /* bit v of the low half: this lane's row sees key key_of(v); of the
                     * high half: some row does. Lane and row are worked out again: kept,
                     * they went to scratch memory. */
                    const int id = lane_again(), of = min(id & 15, rows - 1) * c.rG >> 16;
                    uint64_t m64 = tree_keys(c.tree[(size_t)(s.q0 + of) * c.words], k0, s.p0);
                    const int left = top + 1 - k0; /* keys of the tile, 64 at most count */
                    m64 &= left >= PG ? ~0ull : left <= 0 ? 0ull : (1ull << left) - 1;
                    m64 >>= (E4M3 ? 16 : 8) * (id >> 4);
                    tbits = E4M3 ? (uint32_t)m64 & 0xffffu
                                 : ((uint32_t)m64 & 0xffu) | ((uint32_t)(m64 >> 32) & 0xffu) << 8;
                    tbits |= (uint32_t)or_row(tbits) << 16;
                    unroll_for<16>([&](auto iv) {
                        constexpr int v = decltype(iv)::value;
                        x[v >> 2][v & 3] = hide_by<v>(tbits, x[v >> 2][v & 3]);
                    });
                } else {
#pragma unroll
                    for (int v = 0; v < 16; v++)
                        x[v >> 2][v & 3] = hide(
                            key_seen(k0 + key_of(v), min(hi, top), lo, c.sinks), x[v >> 2][v & 3]);
                }
                foreign = KIND == TREE || !there ||
                          pg_tile_foreign(k0, s.p0, s.kv, c.window, c.sinks);
                if (foreign) {
#pragma unroll
                    for (int h = 0; h < (E4M3 ? 1 : 2); h++)
#pragma unroll
                        for (int d = 0; d < 4; d++) {
                            uint32_t k = 0;
#pragma unroll
                            for (int e = 0; e < (E4M3 ? 4 : 2); e++) {
                                const int v = E4M3 ? 4 * d + e : 8 * h + 2 * d + e;
                                const bool some =
                                    KIND == TREE ? tbits >> (16 + v) & 1
                                                 : key_seen(k0 + key_of(v), top, own_lo, c.sinks);
                                k |= some
                                         ? (E4M3 ? 0xffu << (8 * e) : 0xffffu << (16 * e))
                                         : 0u;
                            }
                            keep[h][d] = k;
                        }
                    vsc = __uint_as_float(
                        (KIND == TREE ? tbits >> (16 + (lane_again() & 15)) & 1
                                      : key_seen(k0 + keyg + m, top, own_lo, c.sinks))
                            ? __float_as_uint(vsc)
                            : 0u);
                }
            }
            float mx = -INFINITY;
#pragma unroll
            for (int v = 0; v < 16; v++)
                mx = fmaxf(mx, x[v >> 2][v & 3]);
            mx = fold_rows(mx, [](float a, float b) { return fmaxf(a, b); });
            const float mnew = fmaxf(mrun, mx);
            const float ref = mnew == -INFINITY ? 0.f : mnew; /* no key yet: p = 2^-inf = 0 */
            if (__any(mnew != mrun)) {
                const float a = fast_exp2(mrun - ref);
                lrun *= a;
#pragma unroll
                for (int t = 0; t < 16; t++)
                    o[t] *= a;
            }
            mrun = mnew;
            bf16x8 p[2];
            unroll_for<16>([&](auto iv) {
                constexpr int v = decltype(iv)::value;
                float pv = fast_exp2(x[v >> 2][v & 3] - ref);
                lrun += pv;
                if constexpr (E4M3)
                    pv *= row_lane<v>(vsc);
                p[v >> 3][v & 7] = f2bf(pv);
            });
            if constexpr (E4M3) {
                if (foreign) {
#pragma unroll
                    for (int t = 0; t < 16; t++)
                        rb[t] &= keep[0];
                }
#pragma unroll
                for (int t = 0; t < 16; t++) {
                    o[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(rb[t][0], rb[t][1], 1.f),
                                                                   p[0], o[t], 0, 0, 0);
                    o[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(rb[t][2], rb[t][3], 1.f),
                                                                   p[1], o[t], 0, 0, 0);
                }
            } else {
                auto values = [&](u32x4 (&r)[16], int part) {
                    if (foreign) {
#pragma unroll
                        for (int j = 0; j < 16; j++)
                            r[j] &= keep[j & 1];
                    }
#pragma unroll
                    for (int j = 0; j < 16; j++)
                        o[8 * part + (j >> 1)] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                            __builtin_bit_cast(bf16x8, r[j]), p[j & 1],
                            o[8 * part + (j >> 1)], 0, 0, 0);
                };
                values(ra, 0);
                load_k(ra, next, 0);
                values(rb, 1);
                load_k(rb, next, 1);
            }
        }
        lrun = fold_rows(lrun, [](float a, float b) { return a + b; });
        if (w.part == 0 && kh == 0 && c.plan.slots > 0 && lane_again() == 0)
            ((int2 *)c.info)[b] = int2{w.first, w.parts};

        /* lane (m, g) holds dims 16 t + 4 g .. + 3 of row m. Both are worked out again:
         * kept over the loop they went to scratch memory. */
        const int id = lane_again(), r = id & 15, d0 = id >> 4 << 2;
        if (w.parts > 1) {
            const size_t slot = slot_of(c, kh, pg_few_slot(w.first, w.part));
            if (r < rows) {
#pragma unroll
                for (int t = 0; t < 16; t++)
                    *(floatx4 *)(c.po + (slot * FEW + r) * PD + 16 * t + d0) = o[t];
                if (d0 == 0) {
                    c.pl[slot * FEW + r] = lrun;
                    c.pmu[slot * FEW + r] = mrun == -INFINITY ? 0.f : mrun;
                }
            }
        } else if (r < rows) {
            const float inv = lrun > 0.f ? 1.f / lrun : 0.f;
            const int tk = r * c.rG >> 16, n = s.q0 + tk, hd = kh * c.G + r - tk * c.G;
            if constexpr (KIND != CAUSAL) {
                if (c.lse && d0 == 0)
                    c.lse[(size_t)n * c.Hq + hd] = lse_of(lrun, mrun);
            }
            bf16x4 gv[16] = {};
            if (c.gate) {
                const bf16 *gp = c.gate + (size_t)n * c.gts + (size_t)hd * c.ghs + d0;
#pragma unroll
                for (int t = 0; t < 16; t++)
                    gv[t] = *(const bf16x4 *)(gp + 16 * t);
            }
#pragma unroll
            for (int t = 0; t < 16; t++) {
                bf16x4 res;
#pragma unroll
                for (int e = 0; e < 4; e++)
                    res[e] = f2bf(o[t][e] * inv * (c.gate ? sigmoid_f(bf2f(gv[t][e])) : 1.f));
                *(bf16x4 *)(c.out + ((size_t)n * c.Hq + hd) * PD + 16 * t + d0) = res;
            }
        }
        /* on to the next unit, if the piece goes on after this one */
        w.begin += w.own, w.first = w.begin / w.size, w.part = 0;
        w.b = -1;
        for (int b0 = cut + w.size <= w.own ? c.B : b + 1; b0 < c.B; b0 += 64) {
            const int at = lane_again();
            const pg_seq t = seq_of(c, min(b0 + at, c.B - 1));
            const uint64_t any = __ballot(b0 + at < c.B && pg_units(t, c.G, FEW) > 0);
            if (any) {
                const int l = __ffsll((unsigned long long)any) - 1;
                w.s = seq_at(t, l);
                w.b = b0 + l;
                w.own = pg_longest(w.s, c.G, FEW, c.list_window, c.list_sinks);
                w.parts = (w.begin + w.own - 1) / w.size - w.first + 1;
                break;
            }
        }
    }
}

/* ---- a middling number of rows of a draft tree: units of up to 64 ----------------------
 * Bound by the K/V bytes as few rows are, but O of 64 rows is four waves' registers. So four
 * waves, one a SIMD, share RB blocks of 16 rows (RG such groups): wave i scores the 16 keys i
 * of a tile against them, and after P has gone through LDS takes dims 64 i .. + 63 of O^T.
 * Each element of a tile is read (and e4m3 widened) once a group so; with the rows shared
 * out, once by every wave, 64 sequences' 16 tokens on up to 4096 e4m3 keys took 119 us.
 * Tiles come to LDS by loads (buffer_load ... lds), K and V^T in rings of NB buffers each.
 * One barrier a tile: between two, O^T of a tile and the scores of the next one are worked
 * on side by side, and P of the next one is written. That needs the softmax's reference
 * before the waves have compared their maxima: it stays what it was unless a score is more
 * than MID_OVER above it (then the waves do compare, with two barriers more; each unit's
 * first tile, and few others). The same with three barriers, scores before O^T: 64 sequences'
 * 16 tokens on 4096 keys each 138 us e4m3 and 204 bf16, so 118 and 193 (5.6 TB/s).
 * The line of key tiles is cut and merged as for few rows. */
template <bool E4M3, int RB, int RG> struct Mid {
    static constexpr int T = PSLICE * (E4M3 ? 1 : 2); /* bytes of a K or V^T tile */
    static constexpr int NB = E4M3 ? 4 : 2;
    static constexpr int V = NB * T, SK = 2 * NB * T, SV = SK + NB * 256;
    /* P, rows of 128 bytes; a float of each row and wave */
    static constexpr int P = SK + (E4M3 ? 2 * NB * 256 : 0), PB = RG * RB * 16 * 128;
    static constexpr int STAT = P + 2 * PB, FLAG = STAT + RG * RB * 16 * 16, BYTES = FLAG + 16;
};
typedef const __attribute__((address_space(3))) floatx4 *lds_f32x4;
typedef const __attribute__((address_space(3))) int *lds_i32;
/* A tile moves the softmax's reference where a score is more than this above it: p is up to
 * 2^8, far from fp32's and bf16's ends, and rounds as it does below 1 */
constexpr float MID_OVER = 8.f;

/* The unit on the line that piece `target` begins in */
DEV Where locate_mid(const Call &c, int target, int &over) {
    const int lane = threadIdx.x & 63;
    pg_seq s;
    int n = 0, units = 0; /* of sequence b0 + lane */
    auto read = [&](int b0) {
        s = seq_of(c, min(b0 + lane, c.B - 1));
        units = b0 + lane < c.B ? pg_units(s, c.G, PG_MID) : 0;
        n = units ? pg_longest(s, c.G, PG_LINE, 0, 0) : 0;
    };
    int T = 0, U = 0;
    for (int b0 = 0; b0 < c.B; b0 += 64) {
        read(b0);
        T += units * n;
        U += units;
    }
    T = last_lane(wave_scan(T)), U = last_lane(wave_scan(U));
    over = pg_mid_over(c.plan, (unsigned)T);
    Where w;
    w.b = -1;
    w.size = pg_mid_share(c.plan, (unsigned)T + (unsigned)U * over);
    const int item = target * w.size;
    int before = 0;
    for (int b0 = 0; b0 < c.B; b0 += 64) {
        if (c.B > 64)
            read(b0);
        const int own = units * (n + over), to = before + wave_scan(own);
        const uint64_t past = __ballot(to > item);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            const int have = __builtin_amdgcn_readlane(to - own, l);
            w.s = seq_at(s, l);
            w.b = b0 + l;
            w.own = __builtin_amdgcn_readlane(n, l);
            w.unit = (item - have) / (w.own + over);
            w.begin = have + w.unit * (w.own + over) + over;
            w.first = w.begin / w.size;
            w.parts = (w.begin + w.own - 1) / w.size - w.first + 1;
            w.part = target - w.first;
            return w;
        }
        before = last_lane(to);
    }
    return w;
}

template <bool E4M3, int RB, int RG> DEV void attend_mid(const Call &c, unsigned char *smem) {
    typedef Mid<E4M3, RB, RG> M;
    constexpr int NW = 4 * RG, NB = M::NB, T = M::T, L = T / (NW * 1024); /* a wave's loads */
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int wq = wave & 3, rg = wave >> 2; /* keys or dims; rows */
    const int m = lane & 15, g = lane >> 4, kh = blockIdx.x % c.Hkv;
    lds_u8 *lds = (lds_u8 *)smem;
    int over;
    Where w = locate_mid(c, blockIdx.x / c.Hkv, over);
    if (w.b < 0)
        return;
    /* A unit, or the part of it in the piece: rows r0 .. r0 + rows - 1 of tokens i_first .. i_last,
     * the first from its head `rest` on; its tiles i0 .. i0 + ntl - 1 */
    pg_seq s;
    int b, rows, i_first, rest, i_last, cut, i0, ntl, ids, ids0;
    auto id_at = [&](int i) {
        const int page = c.page_table[(size_t)b * c.max_pages + min(i0 + i, (s.kv - 1) / PG)];
        return page >= 0 && page < c.num_pages ? page : -1;
    };
    auto set_unit = [&] {
        s = w.s, b = w.b;
        const int r0 = w.unit * PG_MID;
        rows = min(s.ql * c.G - r0, 16 * RB * RG);
        i_first = r0 / c.G, rest = r0 - i_first * c.G;
        i_last = i_first + ((rest + rows - 1) * c.rG >> 16);
        cut = (w.first + w.part) * w.size - w.begin;
        i0 = max(cut, 0);
        ntl = min(min(cut + w.size, w.own), pg_tile_list(s, 0, s.ql - 1, 0, 0).ntl) - i0;
        ids = ntl > 0 ? id_at(lane) : -1, ids0 = 0;
    };
    auto page_of = [&](int t) { /* of tile t from i0 on; past the last, it again */
        t = max(min(t, ntl - 1), 0);
        if (t - ids0 >= 64) {
            ids0 = t;
            ids = id_at(t + lane);
        }
        return __builtin_amdgcn_readlane(ids, t - ids0);
    };
    /* this lane's rows */
    auto row_of = [&](int rb) { return 16 * (rg * RB + rb) + m; };
    auto after = [&](int rb) { /* tokens after i_first */
        return (rest + min(row_of(rb), rows - 1)) * c.rG >> 16;
    };
    auto tok_of = [&](int rb) { return i_first + after(rb); };
    auto head_of = [&](int rb) {
        return kh * c.G + rest + min(row_of(rb), rows - 1) - after(rb) * c.G;
    };
    auto row_words = [&](int tok) { return c.tree + (size_t)(s.q0 + tok) * c.words; };
    bf16x8 qf[RB][8];
    /* the tree's words of this lane's rows, and of all the unit's tokens together: of up to 64
     * new tokens the first is all there is */
    uint64_t word[RB], any_word;
    int pg[NB + 1]; /* pages of tiles i .. i + NB */
    /* Tiles: KiB j NW + wave of a tile is a wave's load j, 2 K rows or 8 V^T rows (e4m3
     * 4 and 16). Pieces of 16 bytes are swizzled, in the address, so that 16 lanes'
     * operands hit 16 bank groups: K's piece p of key k in slot p ^ (k & 15), V^T's of
     * row d in p ^ (d / 2 & 7) (e4m3 d / 4 & 3), P's of row r in p ^ (r / 2 & 7). */
    auto slice = [&](int page) { return (size_t)max(page, 0) * c.Hkv + kh; };
    auto issue_k = [&](int t, int page) {
        const __amdgpu_buffer_rsrc_t src = make_rsrc((const char *)c.k + slice(page) * T, T);
#pragma unroll
        for (int j = 0; j < L; j++) {
            const int kib = j * NW + wave, key = E4M3 ? 4 * kib + g : 2 * kib + (lane >> 5);
            const uint32_t off = E4M3 ? g * 256 + ((m ^ (key & 15)) << 4)
                                      : (lane >> 5) * 512 + (((lane & 31) ^ (key & 15)) << 4);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                src, (lds_ptr)(smem + t % NB * T + kib * 1024), 16, off, kib * 1024, 0, 0);
        }
        if (E4M3 && wave < 2) /* both operands' scales: V's multiply p */
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                make_rsrc((wave ? c.vs : c.ks) + slice(page) * PG, 256),
                (lds_ptr)(smem + (wave ? M::SV : M::SK) + t % NB * 256), 4, lane * 4, 0, 0, 0);
    };
    auto issue_v = [&](int t, int page) {
        const __amdgpu_buffer_rsrc_t src = make_rsrc((const char *)c.vt + slice(page) * T, T);
#pragma unroll
        for (int j = 0; j < L; j++) {
            const int kib = j * NW + wave;
            const int d = E4M3 ? 16 * kib + (lane >> 2) : 8 * kib + (lane >> 3);
            const uint32_t off = E4M3 ? (lane >> 2) * 64 + (((lane & 3) ^ (d >> 2 & 3)) << 4)
                                      : (lane >> 3) * 128 + (((lane & 7) ^ (d >> 1 & 7)) << 4);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                src, (lds_ptr)(smem + M::V + t % NB * T + kib * 1024), 16, off, kib * 1024, 0,
                0);
        }
    };
    /* all but the newest `nk` of K's groups of loads and `nv` of V^T's are there, and all
     * waves as far; what is issued past the last tile keeps the count */
    auto meet = [&](auto nk, auto nv) {
        constexpr int n = (decltype(nk)::value + decltype(nv)::value) * L;
        if (E4M3 && wave < 2)
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(n + decltype(nk)::value)
                         : "memory");
        else
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(n) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    const uint32_t ka = (16 * wq + m) * (T / PG) + ((g ^ m) << 4);
    const uint32_t va = M::V + (64 * wq + m) * (T / PD) +
                        ((E4M3 ? g ^ (m >> 2) : g ^ (m >> 1)) << 4);
    /* P of row m of a block: written 4 keys, 16 wq + 4 g on, read 8 at a time */
    const uint32_t pr = M::P + (rg * RB * 16 + m) * 128;
    const uint32_t pw = pr + (((2 * wq + (g >> 1)) ^ (m >> 1)) << 4) + (g & 1) * 8;
    const uint32_t stat = M::STAT + (rg * RB * 16 + m) * 16;
    /* What a unit needs first, all of it on its way at once: Q, then tiles */
    auto begin = [&] {
#pragma unroll
        for (int rb = 0; rb < RB; rb++) {
            const bf16 *qp = c.q + ((size_t)(s.q0 + tok_of(rb)) * c.Hq + head_of(rb)) * PD;
#pragma unroll
            for (int ks = 0; ks < 8; ks++) /* dims as K's pieces below */
                qf[rb][ks] = *(const bf16x8 *)(qp + (E4M3 ? 64 * (ks >> 1) + 16 * g + 8 * (ks & 1)
                                                          : 32 * ks + 8 * g));
            word[rb] = *row_words(tok_of(rb));
        }
        any_word = *row_words(min(i_first + lane, i_last));
#pragma unroll
        for (int t = 0; t <= NB; t++)
            pg[t] = page_of(t);
        issue_k(0, pg[0]);
#pragma unroll
        for (int t = 0; t < NB - 1; t++) {
            issue_k(t + 1, pg[t + 1]);
            issue_v(t, pg[t]);
        }
        if (threadIdx.x < 2)
            *(int *)(smem + M::FLAG + threadIdx.x * 4) = 0;
    };
    set_unit();
    begin();
    while (true) { /* the units that the piece lies in */
        floatx4 o[RB][4]; /* dims 64 wq + 16 t + 4 g .. + 3 of row m of block rb */
        float mrun[RB], lrun[RB];
#pragma unroll
        for (int rb = 0; rb < RB; rb++) {
            mrun[rb] = -INFINITY, lrun[rb] = 0.f;
#pragma unroll
            for (int t = 0; t < 4; t++)
                o[rb][t] = floatx4{};
        }
        floatx4 x[RB], vsc;      /* a tile's scores; e4m3: V's scales of the lane's keys */
        float ladd[RB];          /* its sums of p */
        bool foreign = false;    /* it has keys that not all rows see, */
        uint64_t any = ~0ull;    /* and those that some row does */
        /* What the scores of tile i need beside their products */
        auto begin_scores = [&](int i, int page) {
            const int k0 = (i0 + i) * PG;
            foreign = page < 0 || !pg_tile_whole(k0, s.p0 - 1, s.p0 + s.ql - 1, s.kv, 0, 0);
            if constexpr (E4M3)
                vsc = *(lds_f32x4)(lds + M::SV + i % NB * 256 + (16 * wq + 4 * g) * 4);
        };
        auto k_scale = [&](int i) {
            return E4M3 ? *(lds_f32)(lds + M::SK + i % NB * 256 + (16 * wq + m) * 4) : 1.f;
        };
        auto k_at = [&](int j, uint32_t kbuf) {
            return lds_read16(lds, (kbuf ^ ((j & 3) << 6)) + (j >> 2) * 256);
        };
        auto scores = [&](int j, u32x4 v, float ksc, floatx4 (&y)[RB]) { /* of step j */
#pragma unroll
            for (int rb = 0; rb < RB; rb++) {
                const floatx4 in = j ? y[rb] : floatx4{};
                if constexpr (E4M3) {
                    y[rb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(v[0], v[1], ksc),
                                                                    qf[rb][2 * j], in, 0, 0, 0);
                    y[rb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                        widen(v[2], v[3], ksc), qf[rb][2 * j + 1], y[rb], 0, 0, 0);
                } else {
                    y[rb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                        __builtin_bit_cast(bf16x8, v), qf[rb][j], in, 0, 0, 0);
                }
            }
        };
        auto flag_of = [&](int i) { /* i + 1 where the tile moves the reference */
            return __builtin_amdgcn_readfirstlane(*(lds_i32)(lds + M::FLAG + (i & 1) * 4));
        };
        /* P of tile i from x, by the reference as it is; rounded to bf16 for its product, as
         * in the other forms (off by 2^-8 of a term at most): a second product, of what the
         * rounding leaves, would add half to a tile's MFMAs, whose chain bounds it already */
        auto write_p = [&](int i) {
#pragma unroll
            for (int rb = 0; rb < RB; rb++) {
                const float ref = mrun[rb] == -INFINITY ? 0.f : mrun[rb]; /* no key yet: p = 0 */
                floatx4 p;
#pragma unroll
                for (int v = 0; v < 4; v++)
                    p[v] = fast_exp2(x[rb][v] - ref);
                ladd[rb] = (p[0] + p[1]) + (p[2] + p[3]);
                if constexpr (E4M3)
                    p *= vsc;
                *(bf16x4 *)(smem + pw + (i & 1) * M::PB + rb * 2048) =
                    bf16x4{f2bf(p[0]), f2bf(p[1]), f2bf(p[2]), f2bf(p[3])};
            }
        };
        auto end_scores = [&](int i, int page) {
            const int k0 = (i0 + i) * PG;
            if (foreign) {
                const int left = page >= 0 ? s.kv - k0 : 0; /* keys of the tile, 64 at most count */
                const uint64_t live = left >= PG ? ~0ull : left <= 0 ? 0ull : (1ull << left) - 1;
                any = live & tree_keys(any_word, k0, s.p0);
                if constexpr (E4M3) { /* scales of no key of the call: any bits */
                    const uint32_t some = (uint32_t)(any >> (16 * wq + 4 * g));
#pragma unroll
                    for (int v = 0; v < 4; v++)
                        vsc[v] = some >> v & 1 ? vsc[v] : 0.f;
                }
#pragma unroll
                for (int rb = 0; rb < RB; rb++) {
                    const uint64_t own = live & tree_keys(word[rb], k0, s.p0);
                    const uint32_t bits = (uint32_t)(own >> (16 * wq + 4 * g));
                    unroll_for<4>([&](auto iv) {
                        constexpr int v = decltype(iv)::value;
                        x[rb][v] = hide_by<v>(bits, x[rb][v]);
                    });
                }
            }
            bool over = false;
#pragma unroll
            for (int rb = 0; rb < RB; rb++)
                over |= fmaxf(fmaxf(x[rb][0], x[rb][1]), fmaxf(x[rb][2], x[rb][3])) >
                        mrun[rb] + MID_OVER;
            if (__any(over) && lane == 0)
                *(int *)(smem + M::FLAG + (i & 1) * 4) = i + 1;
            write_p(i);
        };
        if (ntl > 0) {
            /* Q is waited for here, where what was issued after it is known: in the loop the
             * compiler would wait for tiles of the next rounds with it */
#pragma unroll
            for (int rb = 0; rb < RB; rb++) {
                asm volatile("" : "+v"(word[rb]));
#pragma unroll
                for (int ks = 0; ks < 8; ks++)
                    asm volatile("" : "+v"(qf[rb][ks]));
            }
            any_word = or_wave(any_word);
            /* the first tile's scores */
            meet(template_int<NB - 1>{}, template_int<NB - 1>{});
            begin_scores(0, pg[0]);
            const float ksc = k_scale(0);
#pragma unroll
            for (int j = 0; j < (E4M3 ? 4 : 8); j++)
                scores(j, k_at(j, ka), ksc, x);
            end_scores(0, pg[0]);
            for (int i = 0; i < ntl; i++) {
                meet(template_int<NB - 2>{}, template_int<NB - 2>{});
                issue_k(i + NB, pg[NB]);
                issue_v(i + NB - 1, pg[NB - 1]);
                if (flag_of(i) == i + 1) { /* uniform */
                    /* the reference moves: to the maximum, and P is written again */
#pragma unroll
                    for (int rb = 0; rb < RB; rb++) {
                        float mx = fmaxf(fmaxf(x[rb][0], x[rb][1]), fmaxf(x[rb][2], x[rb][3]));
                        mx = fold_rows(mx, [](float a, float e) { return fmaxf(a, e); });
                        if (g == 0)
                            *(float *)(smem + stat + rb * 256 + wq * 4) = mx;
                    }
                    lds_barrier();
#pragma unroll
                    for (int rb = 0; rb < RB; rb++) {
                        const floatx4 all = *(lds_f32x4)(lds + stat + rb * 256);
                        const float mnew =
                            fmaxf(fmaxf(fmaxf(all[0], all[1]), fmaxf(all[2], all[3])), mrun[rb]);
                        const float a = fast_exp2(mrun[rb] - (mnew == -INFINITY ? 0.f : mnew));
                        lrun[rb] *= a;
#pragma unroll
                        for (int t = 0; t < 4; t++)
                            o[rb][t] *= a;
                        mrun[rb] = mnew;
                    }
                    write_p(i);
                    lds_barrier();
                }
#pragma unroll
                for (int rb = 0; rb < RB; rb++)
                    lrun[rb] += ladd[rb];
                bf16x8 p[RB][2];
#pragma unroll
                for (int rb = 0; rb < RB; rb++)
#pragma unroll
                    for (int st = 0; st < 2; st++) /* keys 32 st + 8 g on (e4m3 16 g + 8 st) */
                        p[rb][st] = __builtin_bit_cast(
                            bf16x8, lds_read16(lds, pr + (i & 1) * M::PB + rb * 2048 +
                                                        (((E4M3 ? 2 * g + st : 4 * st + g) ^
                                                          (m >> 1))
                                                         << 4)));
                /* O^T of tile i, dims 16 t on of the wave's, and scores of tile i + 1 between (past
                 * the last of that one again, for nothing): neither waits for the other's */
                const uint32_t vbuf = i % NB * T + va, kbuf = (i + 1) % NB * T + ka;
                floatx4 y[RB];
                const float ksc = k_scale(i + 1);
                auto products = [&](auto masked) {
                    u32x4 keep[2]; /* bits to keep of V^T: of keys of the call */
                    if constexpr (decltype(masked)::value) {
                        const uint32_t a = (uint32_t)(any >> ((E4M3 ? 16 : 8) * g));
                        const uint32_t e = (uint32_t)(any >> 32 >> (8 * g));
#pragma unroll
                        for (int d = 0; d < 4; d++) {
                            auto two = [&](uint32_t x2) {
                                return ((x2 >> (2 * d) & 1) ? 0xffffu : 0u) |
                                       ((x2 >> (2 * d + 1) & 1) ? 0xffff0000u : 0u);
                            };
                            keep[0][d] = E4M3 ? bytes_by(a >> (4 * d)) : two(a);
                            keep[1][d] = two(e);
                        }
                    }
                    /* operands of a quarter are read while the one before is worked on */
                    constexpr int KS = E4M3 ? 1 : 2;
                    u32x4 kr[2][KS], vr[2][KS];
                    auto read = [&](int t) {
#pragma unroll
                        for (int u = 0; u < KS; u++) {
                            kr[t & 1][u] = k_at(KS * t + u, kbuf);
                            vr[t & 1][u] = lds_read16(lds, (vbuf ^ (u << 6)) + t * (1024 * KS));
                        }
                    };
                    read(0);
                    unroll_for<4>([&](auto it) {
                        constexpr int t = decltype(it)::value;
                        if constexpr (t < 3)
                            read(t + 1);
                        __builtin_amdgcn_sched_barrier(0);
                        bf16x8 v[2];
                        if constexpr (E4M3) {
                            u32x4 raw = vr[t & 1][0];
                            if constexpr (decltype(masked)::value)
                                raw &= keep[0];
                            v[0] = widen(raw[0], raw[1], 1.f), v[1] = widen(raw[2], raw[3], 1.f);
                        } else {
#pragma unroll
                            for (int st = 0; st < 2; st++) {
                                u32x4 raw = vr[t & 1][st];
                                if constexpr (decltype(masked)::value)
                                    raw &= keep[st];
                                v[st] = __builtin_bit_cast(bf16x8, raw);
                            }
                        }
#pragma unroll
                        for (int u = 0; u < KS; u++)
                            scores(KS * t + u, kr[t & 1][u], ksc, y);
#pragma unroll
                        for (int rb = 0; rb < RB; rb++)
#pragma unroll
                            for (int st = 0; st < 2; st++)
                                o[rb][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                                    v[st], p[rb][st], o[rb][t], 0, 0, 0);
                    });
                };
                if (foreign)
                    products(std::true_type{});
                else
                    products(std::false_type{});
#pragma unroll
                for (int rb = 0; rb < RB; rb++)
                    x[rb] = y[rb];
                if (i + 1 < ntl) {
                    begin_scores(i + 1, pg[1]);
                    end_scores(i + 1, pg[1]);
                }
#pragma unroll
                for (int t = 0; t < NB; t++)
                    pg[t] = pg[t + 1];
                pg[NB] = page_of(i + 1 + NB);
            }
        }
        /* this unit's rows, and where they go */
        const int parts = w.parts, old_rows = rows;
        const size_t slot = slot_of(c, kh, pg_few_slot(w.first, w.part)) * c.plan.rt;
        int n[RB], head[RB];
#pragma unroll
        for (int rb = 0; rb < RB; rb++)
            n[rb] = s.q0 + tok_of(rb), head[rb] = head_of(rb);
        if (w.part == 0 && kh == 0 && c.plan.slots > 0 && threadIdx.x == 0)
            ((int2 *)c.info)[b * (c.plan.units / c.B) + w.unit] = int2{w.first, w.parts};
        /* on to the next unit, if the piece goes on after this one */
        bool more = cut + w.size > w.own + over;
        if (more) {
            w.begin += w.own + over, w.first = w.begin / w.size, w.part = 0;
            if (w.unit + 1 < pg_units(s, c.G, PG_MID)) {
                w.unit++;
            } else {
                more = false;
                for (int b0 = b + 1; b0 < c.B && !more; b0 += 64) {
                    const pg_seq t = seq_of(c, min(b0 + lane, c.B - 1));
                    const uint64_t some = __ballot(b0 + lane < c.B && t.ql > 0);
                    if (some) {
                        const int l = __ffsll((unsigned long long)some) - 1;
                        w.s = seq_at(t, l);
                        w.b = b0 + l;
                        w.unit = 0;
                        w.own = pg_longest(w.s, c.G, PG_LINE, 0, 0);
                        more = true;
                    }
                }
            }
            w.parts = (w.begin + w.own - 1) / w.size - w.first + 1;
        }
        if (more)
            set_unit();
        /* nothing is on its way, and all have read: the next unit's Q and tiles go out ahead of
         * what is left of this one */
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (more)
            begin();
#pragma unroll
        for (int rb = 0; rb < RB; rb++) { /* l of a row from the four waves' keys */
            const float l = fold_rows(lrun[rb], [](float a, float e) { return a + e; });
            if (g == 0)
                *(float *)(smem + stat + rb * 256 + wq * 4) = l;
        }
        lds_barrier();
        const int d0 = 64 * wq + 4 * g;
#pragma unroll
        for (int rb = 0; rb < RB; rb++) {
            const floatx4 all = *(lds_f32x4)(lds + stat + rb * 256);
            const float l = (all[0] + all[1]) + (all[2] + all[3]);
            const int r = row_of(rb);
            if (r >= old_rows)
                continue;
            if (parts > 1) {
#pragma unroll
                for (int t = 0; t < 4; t++)
                    *(floatx4 *)(c.po + (slot + r) * PD + d0 + 16 * t) = o[rb][t];
                if (d0 == 0) {
                    c.pl[slot + r] = l;
                    c.pmu[slot + r] = mrun[rb] == -INFINITY ? 0.f : mrun[rb];
                }
                continue;
            }
            const float inv = l > 0.f ? 1.f / l : 0.f;
            const size_t at = (size_t)n[rb] * c.Hq + head[rb];
            if (c.lse && d0 == 0)
                c.lse[at] = lse_of(l, mrun[rb]);
            bf16x4 gv[4] = {};
            if (c.gate) {
                const bf16 *gp = c.gate + (size_t)n[rb] * c.gts + (size_t)head[rb] * c.ghs + d0;
#pragma unroll
                for (int t = 0; t < 4; t++)
                    gv[t] = *(const bf16x4 *)(gp + 16 * t);
            }
#pragma unroll
            for (int t = 0; t < 4; t++) {
                bf16x4 res;
#pragma unroll
                for (int e = 0; e < 4; e++)
                    res[e] = f2bf(o[rb][t][e] * inv * (c.gate ? sigmoid_f(bf2f(gv[t][e])) : 1.f));
                *(bf16x4 *)(c.out + at * PD + d0 + 16 * t) = res;
            }
        }
        if (!more)
            break;
    }
}
template <bool E4M3, int RB, int RG>
__global__ __launch_bounds__(256 * RG) void attention_mid_kernel(Call c) {
    __shared__ __attribute__((aligned(1024))) unsigned char smem[Mid<E4M3, RB, RG>::BYTES];
    static_assert(sizeof(smem) <= 163840, "LDS of a CU");
    attend_mid<E4M3, RB, RG>(c, smem);
}

/* ---- many rows: tiles of 128 packed rows -----------------------------------------
 * One workgroup, 8 waves, two on each SIMD. Wave (i, j) computes the scores of
 * 32 rows (quarter i) against 32 keys of a tile (half j), and then O^T of the same
 * rows for 128 dims (half j); the pair (i, 0), (i, 1) exchanges its P, 2 KiB each
 * way per tile, through LDS. Half of a row's scores and half of its O per wave fit
 * 256 registers (O 64, Q 64), so that one wave's softmax, conversions and waits
 * run beside the other's MFMAs; one wave a SIMD (64 rows of it, half the operand
 * reads) issued a VALU instruction only every other slot.
 *
 * Per tile one barrier. Before it a wave runs the S^T MFMAs of tile i + 1 with the
 * second half of p of tile i, and leaves P of tile i in LDS; after it the PV MFMAs
 * of tile i, its own keys' first, with the mask, maximum and first half of p of
 * tile i + 1, while K of tile i + 3 and V^T of tile i + 1 go to the buffers that
 * were last read before the barrier.
 *
 * The softmax's reference mu of a row stays 0 while the scores are within 2^+-64
 * of it (mu cancels in o / l). A wave that leaves that range takes an integer
 * mu of its own for the tile and tells the other of its pair through the signs
 * of its P, which are otherwise 0: lane h = 0 sends the low and h = 1 the high
 * half of the float. Both then agree on the larger one and rescale. From then on
 * all of the wave's tiles go that way, half as long again: 4096 tokens on 8192 keys
 * with scores past 64 take 511 us instead of 363 (bf16), 633 instead of 391 (e4m3).
 *
 * 4096 tokens on 8192 keys: 363-371 us, 1.1 PFLOP/s, 80 % of the rate of a large
 * library product on the same card (1.41; bf16); e4m3 389-396, where the conversions
 * to bf16 fill the VALU beside the MFMAs. A workgroup spends 12 us outside its tiles:
 * 3.5 on lengths, page ids and the first K, 5 on the epilogue (the gates' 32768
 * sigmoids are 2 of them). */
constexpr int RT = PG_MANY;
constexpr float SHIFT_RANGE = 64.f;
/* With the reference 0, V far from 1 can lead p v out of fp32's range: p = 2^62 and V =
 * 2^70, or 2^-62 and 2^-70. So where a row's l ends beyond 2^+-32 its O is looked at, and
 * where that is above 2^96 or below 2^-64 the workgroup does its share once more with
 * the range 0: the reference is then the maximum and p at most 1, as it is for few
 * rows. V up to 2^80 so is safe with any scores and any number of keys. */
constexpr float LOST_L = 0x1p32f, LOST_HIGH = 0x1p96f, LOST_LOW = 0x1p-64f;

template <bool E4M3> struct Lay {
    static constexpr int T = PSLICE * (E4M3 ? 1 : 2); /* bytes of a K or V^T tile */
    static constexpr int V = 0, K = 2 * T, P = 4 * T, PBUF = 16384, SC = P + 2 * PBUF;
    /* e4m3: K scales of two tiles, V scales of four (read a tile later) */
    static constexpr int TILES = SC + (E4M3 ? 2 * 256 + 4 * 256 : 0);
    /* Q on its way to registers, 64 rows each: in P, and in V^T's second buffer (e4m3:
     * behind the scales) */
    static constexpr int Q0 = P, Q1 = E4M3 ? TILES : V + T, QEND = Q1 + RT / 2 * PD * 2;
    static constexpr int STAT = RT * PD * 4; /* l behind the staged O */
    static constexpr int ALL = TILES > QEND ? TILES : QEND;
    static constexpr int AGAIN = STAT + RT * 8, END = AGAIN + 8 * 4; /* a flag a wave */
    static constexpr int BYTES = ALL > END ? ALL : END;
};
static_assert(Lay<false>::BYTES <= 163840 && Lay<true>::BYTES <= 163840, "LDS of a CU");

/* 16-byte pieces of the tiles are XOR-swizzled so that the 16 lanes of a
 * ds_read_b128 phase hit 16 distinct bank groups. bf16: K rows of 512 bytes,
 * V^T rows of 128; e4m3: 256 and 64. */
template <bool E4M3> DEV int swz_k(int key) {
    return E4M3 ? (key & 3) | ((key >> 4) & 1) << 2 | ((key >> 2) & 1) << 3
                : ((key & 4) << 1) | ((key & 8) >> 1) | (key & 3);
}
template <bool E4M3> DEV int swz_v(int d) {
    return E4M3 ? (d >> 2) & 3 : (d & 7) ^ ((d >> 3) & 1);
}
/* key of MFMA row m of a 32-key block: score accumulator r of lane half h is
 * then key 16 (r >> 3) + 8 h + (r & 7) (bf16), 16 h + r (e4m3) */
template <bool E4M3> DEV int perm_row(int m) {
    return E4M3 ? 16 * ((m >> 2) & 1) + (m & 3) + 4 * (m >> 3)
                : (m & ~12) | ((m & 4) << 1) | ((m & 8) >> 1);
}

/* A workgroup's share, with a reference of 0 within the range; true: once more with none.
 * The second time is the first one's code again, and nothing but the range may be kept
 * for it: all of the 128 + 128 registers are taken. */
template <bool E4M3, int KIND>
DEV bool attend_many(const Call &c, unsigned char *smem, const float range) {
    typedef Lay<E4M3> L;
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid)); /* unknown: what goes by it is worked out each time */
    /* XCD-aware: where the kv-heads divide the 8 XCDs, an XCD's workgroups read
     * the same kv-head. The longest (last) tiles of a sequence start first. */
    int kh, at;
    if (8 % c.Hkv == 0) {
        const int per = 8 / c.Hkv, xcd = blockIdx.x & 7;
        kh = xcd / per;
        at = (blockIdx.x >> 3) * per + xcd % per;
    } else {
        kh = blockIdx.x % c.Hkv;
        at = blockIdx.x / c.Hkv;
    }
    if (at >= c.plan.shares)
        return false;
    const int target = c.plan.shares - 1 - at;
    const Where w = locate<RT>(c, target);
    if (kh == 0 && target < c.plan.slots && tid == 0)
        ((int4 *)c.info)[target] =
            int4{w.b, w.unit, w.b >= 0 && w.part == 0 ? w.parts : 0, 0};
    if (w.b < 0)
        return false;
    const pg_seq s = w.s;
    const int b = w.b, nshare = w.parts, share = w.part;
    const int r0 = w.unit * RT, nrows = min(s.ql * c.G - r0, RT);
    const int i0 = r0 / c.G, rest = r0 - i0 * c.G, i1 = i0 + ((rest + nrows - 1) * c.rG >> 16);
    const pg_tiles list =
        pg_tile_list(s, i0, KIND == TREE ? s.ql - 1 : i1, c.list_window, c.list_sinks);
    const int tb = pg_share_begin(list.ntl, share, nshare);
    const int ntl = pg_share_begin(list.ntl, share + 1, nshare) - tb;
    const size_t slot = slot_of(c, kh, w.first + share);

    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int wi = wave & 3, wj = wave >> 2, h = lane >> 5, col = lane & 31;

    /* page ids of the list, 64 entries in a lane each; the first ahead of Q's loads,
     * which a wait for them would wait for too */
    int ids = 0;
    if (ntl > 0)
        ids = page_id(c, b, list, min(tb + lane, list.ntl - 1));

    int hi, lo; /* of this lane's row; rows past the last repeat it */
    {
        const int tok = i0 + ((rest + min(32 * wi + col, nrows - 1)) * c.rG >> 16);
        hi = KIND == TREE ? s.kv - 1 : min(s.p0 + tok, s.kv - 1);
        lo = pg_low(s.p0 + tok, c.window);
    }
    /* TREE: all rows see the keys up to pmin, no other order of theirs is known */
    const int pmin = KIND == TREE ? s.p0 - 1 : s.p0 + i0, pmax = s.p0 + i1;
    /* of keys k0 .. k0 + 63, those that the row of token i sees, and that any row does */
    auto seen_by = [&](int k0, int i) {
        return tree_keys(c.tree + (size_t)(s.q0 + i) * c.words, c.words, k0, s.p0);
    };
    auto seen_by_any = [&](int k0) { /* tokens i0 .. i1, up to 128 */
        const int n = lane_again();
        return or_wave(seen_by(k0, min(i0 + n, i1)) | seen_by(k0, min(i0 + 64 + n, i1)));
    };

    /* ---- tile loads: memory -> LDS (buffer_load ... lds: lane l's 16 bytes land
     * at base + 16 l, so the swizzle is applied to the address). Load n of a wave is
     * KiB 8 n + wave of the tile: 2 K rows or 8 V^T rows (e4m3 4 and 16). ---- */
    constexpr int NL = L::T / 8192; /* loads of a wave, tile and operand */
    uint32_t kvoff, vvoff;
    if constexpr (E4M3) {
        kvoff = (lane >> 4) * 256 + (((lane & 15) ^ swz_k<true>(4 * wave + (lane >> 4))) << 4);
        vvoff = (lane >> 2) * 64 + (((lane & 3) ^ swz_v<true>(lane >> 2)) << 4);
    } else {
        kvoff = (lane >> 5) * 512 + (((lane & 31) ^ swz_k<false>(2 * wave + (lane >> 5))) << 4);
        vvoff = (lane >> 3) * 128 + (((lane & 7) ^ swz_v<false>(8 * wave + (lane >> 3))) << 4);
    }
    auto slice = [&](int page) { return (size_t)max(page, 0) * c.Hkv + kh; };
    auto k_rsrc = [&](int page) {
        return make_rsrc((const char *)c.k + slice(page) * L::T, L::T);
    };
    auto v_rsrc = [&](int page) {
        return make_rsrc((const char *)c.vt + slice(page) * L::T, L::T);
    };
    auto issue_k = [&](__amdgpu_buffer_rsrc_t r, int buf, int n) {
        const int at = 8192 * n + 1024 * wave;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr)(smem + L::K + buf * L::T + at), 16,
                                                 kvoff, at, 0, 0);
    };
    auto issue_v = [&](__amdgpu_buffer_rsrc_t r, int buf, int n) {
        const int at = 8192 * n + 1024 * wave;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr)(smem + L::V + buf * L::T + at), 16,
                                                 vvoff, at, 0, 0);
    };
    /* scales of tile t: wave 0 K's, wave 1 V's */
    auto issue_scales = [&](int page, int t) {
        if constexpr (E4M3) {
            if (wave < 2) {
                const float *src = (wave ? c.vs : c.ks) + slice(page) * PG;
                const int at = L::SC + (wave ? 512 + (t & 3) * 256 : (t & 1) * 256);
                __builtin_amdgcn_raw_ptr_buffer_load_lds(make_rsrc(src, 256),
                                                         (lds_ptr)(smem + at), 4, lane * 4, 0, 0,
                                                         0);
            }
        }
    };

    /* Q through LDS, as whole rows: lane by lane each load touched 32 lines, which
     * took 3 us. Wave (i, j) brings half j of the rows of quarter i, two a load;
     * piece p of row r lies in slot p ^ (r & 15). */
    lds_u8 *lds = (lds_u8 *)smem;
    const uint32_t qat = (wi & 2 ? L::Q1 : L::Q0) + (wi & 1) * 16384;
    auto issue_q = [&]() {
        const __amdgpu_buffer_rsrc_t r =
            make_rsrc(c.q + ((size_t)(s.q0 + i0) * c.Hq + kh * c.G) * PD, 0x7fffffff);
#pragma unroll
        for (int n = 0; n < 8; n++) {
            const int at = 16 * wj + 2 * n + h, row = rest + min(32 * wi + at, nrows - 1);
            const int tok = row * c.rG >> 16; /* after i0 */
            const uint32_t off = (tok * c.Hq + row - tok * c.G) * PD * 2;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                r, (lds_ptr)(smem + qat + (16 * wj + 2 * n) * 512), 16,
                off + ((col ^ (at & 15)) << 4), 0, 0, 0);
        }
    };
    bf16x8 qf[16]; /* Q^T operands of this wave's 32 rows */

    /* ---- per-lane LDS read addresses ---- */
    const int arow = perm_row<E4M3>(col);
    uint32_t ka[8];
#pragma unroll
    for (int p = 0; p < 8; p++)
        ka[p] = L::K + (32 * wj + arow) * (L::T / PG) +
                (((2 * p + h) ^ swz_k<E4M3>(32 * wj + arow)) << 4);
    /* V^T pieces of key half kb (0: this wave's own keys, 1: the other's) */
    uint32_t va[2][2];
#pragma unroll
    for (int kb = 0; kb < 2; kb++)
#pragma unroll
        for (int st = 0; st < 2; st++) {
            const int half = wj ^ kb;
            const int piece = E4M3 ? 2 * half + h : 4 * half + 2 * st + h;
            va[kb][st] = L::V + (128 * wj + col) * (L::T / PD) +
                         ((piece ^ swz_v<E4M3>(col)) << 4);
        }
    const uint32_t psend = L::P + wave * 2048 + lane * 16;
    const uint32_t precv = L::P + (wave ^ 4) * 2048 + lane * 16;

    auto page_of = [&](int t) { /* called with t = 0, 1, 2, ... < ntl */
        if ((t & 63) == 0 && t > 0)
            ids = page_id(c, b, list, min(tb + t + lane, list.ntl - 1));
        return __builtin_amdgcn_readlane(ids, t & 63);
    };

    floatx16 o[4]; /* zeros by MFMAs: constants were kept in 16 registers */
    {
        bf16x8 none = {};
        asm volatile("" : "+v"(none));
#pragma unroll
        for (int d = 0; d < 4; d++)
            mfma_zero(o[d], none);
    }
    /* of this lane's row: running maximum, l, the reference agreed on; of the
     * current tile: its p, their sum, the reference this wave wants */
    float mrun = -INFINITY, lrun = 0.f, mus = 0.f, mx = 0.f, ls = 0.f, mul = 0.f;
    bf16x8 pf[2], pn;
    float vsc = 1.f; /* e4m3: V's scale of key (lane & 15) of this half's 16 */
    bool moved = false;

    constexpr int QD = E4M3 ? 2 : 3;   /* K operand reads ahead */
    constexpr int NKR = E4M3 ? 8 : 16; /* K reads a tile */
    auto kaddr = [&](int n, int buf) {
        return (E4M3 ? ka[n] : ka[n & 7] + (n >> 3) * 256) + buf * L::T;
    };
    auto kscale = [&](int buf) {
        return E4M3 ? *(lds_f32)(lds + L::SC + buf * 256 + (32 * wj + arow) * 4) : 1.f;
    };
    auto score = [&](floatx16 &y, bf16x8 a, int ks) { /* k-step ks of S^T */
        if (ks == 0)
            mfma_first<E4M3>(y, a, qf[0]);
        else
            mfma_score<E4M3>(y, a, qf[ks]);
    };
    auto load_vsc = [&](int t) {
        if constexpr (E4M3)
            vsc = *(lds_f32)(lds + L::SC + 512 + (t & 3) * 256 +
                             (32 * wj + 16 * h + (lane & 15)) * 4);
    };
    /* hides what the rows of tile t's scores do not see */
    auto mask = [&](floatx16 &x, int t, bool there) {
        const int k0 = pg_tile_page(list, tb + t) * PG;
        if (there && pg_tile_whole(k0, pmin, pmax, s.kv, c.window, c.sinks))
            return;
        const int kb = k0 + 32 * wj + (E4M3 ? 16 : 8) * h;
        const int top = there ? s.kv - 1 : -1;
        uint32_t bits = keys_seen<E4M3 ? 16 : 24>(kb, min(hi, top), lo, c.sinks);
        if constexpr (KIND == TREE)
            bits &= (uint32_t)(seen_by(k0, i0 + ((rest + min(32 * wi + col, nrows - 1)) * c.rG >>
                                                 16)) >>
                               (kb - k0));
        unroll_for<16>([&](auto iv) {
            constexpr int r = decltype(iv)::value;
            x[r] = hide_by<E4M3 ? r : 16 * (r >> 3) + (r & 7)>(bits, x[r]);
        });
        if constexpr (E4M3) { /* a scale of no key of this call: any bits */
            bool some = key_seen(kb + (lane & 15), top, pg_low(pmin, c.window), c.sinks);
            if constexpr (KIND == TREE)
                some &= seen_by_any(k0) >> (kb - k0 + (lane & 15)) & 1;
            vsc = __uint_as_float(some ? __float_as_uint(vsc) : 0u);
        }
    };
    /* p of accumulators v, v + 1 into operand f */
    auto pair = [&](const floatx16 &x, bf16x8 &f, auto iv, float shift) {
        constexpr int v = decltype(iv)::value;
        float a = fast_exp2(x[v] - shift), e = fast_exp2(x[v + 1] - shift);
        ls += a + e;
        if constexpr (E4M3) {
            a *= row_lane<v>(vsc);
            e *= row_lane<v + 1>(vsc);
        }
        /* the empty asm keeps the pair in its place among the MFMAs */
        bf16x2 pk = {f2bf(a), f2bf(e)};
        asm volatile("" : "+v"(pk), "+v"(ls));
        f[v & 7] = pk[0];
        f[(v & 7) + 1] = pk[1];
    };
    /* the reference this wave wants for a tile whose maximum is known */
    auto want = [&]() {
        const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx),
                                                         false, false);
        mrun = fmaxf(mrun, fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])));
        /* a row without a key yet leaves the choice to the other wave */
        mul = mrun == -INFINITY           ? -INFINITY
              : fabsf(mrun - mus) > range ? ceilf(mrun)
                                          : mus;
        moved = __any(mul != 0.f);
    };

    int pg[4]; /* pages of tiles i .. i + 3 */
    u32x4 ring[QD];
    float ksc = 1.f;
    /* One tile. On entry x holds its masked scores, pn the first half of p for the
     * reference 0, and ring the first K operands of tile i + 1. The last tile
     * runs the same code: what it does for a next one (from stale buffers, and
     * loads of the last page again) reaches no result. A variant without it cost
     * the registers of a second set of accumulators where the two meet. */
    auto step = [&](int i, auto parity, floatx16 &x, floatx16 &y) {
        constexpr int PAR = decltype(parity)::value; /* i & 1 */
        const bool there = pg[0] >= 0;
        /* ---- S^T of tile i + 1 with the second half of p; its last two k-steps wait
         * for the barrier, to work while the reads behind it come back ---- */
        bf16x8 held[2] = {};
        unroll_for<16>([&](auto iks) {
            constexpr int ks = decltype(iks)::value;
            if constexpr (E4M3) {
                if constexpr ((ks & 1) == 0) {
                    const u32x4 w = ring[(ks >> 1) % QD];
                    if constexpr ((ks >> 1) + QD < NKR)
                        ring[(ks >> 1) % QD] = lds_read16(lds, kaddr((ks >> 1) + QD, PAR ^ 1));
                    held[0] = widen(w[0], w[1], ksc);
                    held[1] = widen(w[2], w[3], ksc);
                }
            } else {
                held[ks & 1] = __builtin_bit_cast(bf16x8, ring[ks % QD]);
                if constexpr (ks + QD < NKR)
                    ring[ks % QD] = lds_read16(lds, kaddr(ks + QD, PAR ^ 1));
            }
            if constexpr (ks < 14)
                score(y, held[ks & 1], ks);
            if constexpr (ks < 12 && ks % 3 == 1)
                pair(x, pf[1], template_int<8 + ks / 3 * 2>{}, 0.f);
            __builtin_amdgcn_sched_barrier(0);
        });
        pf[0] = pn;
        if (__builtin_expect(moved, 0)) {
            const float shift = mul == -INFINITY ? 0.f : mul;
            ls = 0.f;
            unroll_for<8>([&](auto iv) {
                constexpr int v = 2 * decltype(iv)::value;
                pair(x, pf[v >> 3], template_int<v>{}, shift);
            });
#pragma unroll
            for (int st = 0; st < 2; st++) {
                u32x4 w = __builtin_bit_cast(u32x4, pf[st]);
                const uint32_t u = __float_as_uint(mul) >> (16 * h + 8 * st);
#pragma unroll
                for (int e = 0; e < 4; e++)
                    w[e] |= ((u >> (2 * e)) & 1) << 15 | ((u >> (2 * e + 1)) & 1) << 31;
                pf[st] = __builtin_bit_cast(bf16x8, w);
            }
        }
#pragma unroll
        for (int st = 0; st < 2; st++)
            lds_write16(smem, psend + PAR * L::PBUF + st * 1024,
                        __builtin_bit_cast(u32x4, pf[st]));
        /* P is in LDS, this wave's reads of K are done, its tile loads have landed */
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");

        const int k0 = pg_tile_page(list, tb + i) * PG;
        if (!there || pg_tile_foreign(k0, pmin, s.kv, c.window, c.sinks) ||
            (KIND == TREE && k0 + PG > s.p0)) {
            /* values of no key of these rows meet p = 0: make them 0 */
            uint64_t any = ~0ull;
            if constexpr (KIND == TREE)
                any = seen_by_any(k0);
#pragma unroll 1
            for (int n = 0; n < L::T / 8192; n++) {
                const int at = (n * 512 + tid) * 16, d = at / (L::T / PD);
                const int piece = ((at >> 4) & (L::T / PD / 16 - 1)) ^ swz_v<E4M3>(d);
                u32x4 w = lds_read16(lds, L::V + PAR * L::T + at);
                const uint32_t bits =
                    there ? keys_seen<E4M3 ? 16 : 8>(k0 + (E4M3 ? 16 : 8) * piece, s.kv - 1,
                                                     pg_low(pmin, c.window), c.sinks) &
                                (uint32_t)(any >> ((E4M3 ? 16 : 8) * piece))
                          : 0u;
                unroll_for<4>([&](auto ie) {
                    constexpr int e = decltype(ie)::value;
                    if constexpr (E4M3)
                        w[e] &= bytes_by(bits >> (4 * e));
                    else
                        w[e] &= halves_by<2 * e>(bits);
                });
                lds_write16(smem, L::V + PAR * L::T + at, w);
            }
            lds_barrier();
        }

        /* ---- O^T += V^T P^T: own keys, then the other wave's; beside it the tile
         * loads, and the mask, maximum and first half of p of tile i + 1 ---- */
        constexpr int NVR = E4M3 ? 4 : 8; /* V^T reads of a key half */
        constexpr int VD = E4M3 ? 2 : 3;
        auto vaddr = [&](int n, int kb) { /* bf16: step-major, e4m3: both steps a read */
            return (E4M3 ? va[kb][0] + n * 32 * (L::T / PD)
                         : va[kb][n >> 2] + (n & 3) * 32 * (L::T / PD)) +
                   PAR * L::T;
        };
        u32x4 vring[VD], pw[2];
#pragma unroll
        for (int st = 0; st < 2; st++)
            pw[st] = lds_read16(lds, precv + PAR * L::PBUF + st * 1024);
#pragma unroll
        for (int n = 0; n < VD; n++)
            vring[n] = lds_read16(lds, vaddr(n, 0));
        __builtin_amdgcn_sched_barrier(0);
        score(y, held[0], 14);
        score(y, held[1], 15);
        __builtin_amdgcn_sched_barrier(0);
        const uint32_t signs = pw[0][0] | pw[0][1] | pw[0][2] | pw[0][3] | pw[1][0] | pw[1][1] |
                               pw[1][2] | pw[1][3];
        if (__builtin_expect(moved || __any((signs & 0x80008000u) != 0), 0)) {
            /* Both waves' references of a row are known: take the larger one. The
             * accumulators of y are not touched in here. */
            uint32_t u = 0;
#pragma unroll
            for (int st = 0; st < 2; st++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    u |= ((pw[st][e] >> 15) & 1) << (8 * st + 2 * e);
                    u |= (pw[st][e] >> 31) << (8 * st + 2 * e + 1);
                }
            const uint32_t v = __shfl_xor(u, 32, 64);
            const float mup = __uint_as_float(h ? u << 16 | v : v << 16 | u);
            float ref = fmaxf(mul, mup);
            ref = ref == -INFINITY ? mus : ref;
            /* it only falls while no key has counted, with o = l = 0 */
            const float fo = fast_exp2(fminf(mus - ref, 0.f));
            const float fm = fast_exp2(mul - ref), fp = fast_exp2(mup - ref);
            settle(o);
#pragma unroll
            for (int d = 0; d < 4; d++) { /* one at a time: 16 registers in passing */
                o[d] *= fo;
                asm volatile("" : "+a"(o[d]));
                __builtin_amdgcn_sched_barrier(0);
            }
            lrun *= fo;
            ls *= fm;
            mus = ref;
#pragma unroll
            for (int st = 0; st < 2; st++) {
                bf16x8 t = __builtin_bit_cast(bf16x8, pw[st] & 0x7fff7fffu);
                bf16x8 w = __builtin_bit_cast(
                    bf16x8, __builtin_bit_cast(u32x4, pf[st]) & 0x7fff7fffu);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    t[e] = f2bf(bf2f(t[e]) * fp);
                    w[e] = f2bf(bf2f(w[e]) * fm);
                }
                pw[st] = __builtin_bit_cast(u32x4, t);
                pf[st] = w;
                asm volatile("s_nop 1" : "+v"(pw[st]), "+v"(pf[st]));
            }
            settle(o);
        }
        lrun += ls;
        const __amdgpu_buffer_rsrc_t rk = k_rsrc(pg[3]), rv = v_rsrc(pg[1]);
        unroll_for<16>([&](auto ig) {
            constexpr int g = decltype(ig)::value;
            constexpr int PER = E4M3 ? 2 : 1; /* MFMAs a V^T read feeds */
            constexpr int n = g / PER, kb = n / NVR, half = g % PER;
            const u32x4 w = vring[n % VD];
            if constexpr (half == PER - 1 && n + VD < 2 * NVR)
                vring[n % VD] = lds_read16(lds, vaddr((n + VD) % NVR, (n + VD) / NVR));
            bf16x8 a;
            if constexpr (E4M3)
                a = half ? widen(w[2], w[3], 1.f) : widen(w[0], w[1], 1.f);
            else
                a = __builtin_bit_cast(bf16x8, w);
            constexpr int d = E4M3 ? n % NVR : n & 3, st = E4M3 ? half : n % NVR >> 2;
            mfma_out<E4M3>(o[d], a, kb ? __builtin_bit_cast(bf16x8, pw[st]) : pf[st]);
            if constexpr (g < NL) /* a tile load beside an MFMA */
                issue_v(rv, PAR ^ 1, g);
            else if constexpr (g < 2 * NL)
                issue_k(rk, PAR ^ 1, g - NL);
            if constexpr (g == 0)
                load_vsc(i + 1);
            if constexpr (g == 3) { /* y's last MFMA is four behind */
                asm volatile("" : "+v"(y));
                mask(y, i + 1, pg[1] >= 0);
                ls = 0.f;
                mx = fmaxf(y[0], y[1]);
            }
            if constexpr (g >= 4 && g < 11) {
                constexpr int v = 2 * (g - 3);
                mx = fmaxf(mx, fmaxf(y[v], y[v + 1]));
            }
            if constexpr (g >= 4 && g < 12 && (g & 1) == 1)
                pair(y, pn, template_int<g - 5>{}, 0.f);
            if constexpr (g == 12)
                want();
            if constexpr (g >= 16 - QD) /* K of tile i + 2 is there since the barrier */
                ring[g - 16 + QD] = lds_read16(lds, kaddr(g - 16 + QD, PAR));
            if constexpr (g == 15)
                ksc = kscale(PAR);
            __builtin_amdgcn_sched_barrier(0);
        });
        issue_scales(pg[3], i + 3);
        pg[0] = pg[1], pg[1] = pg[2], pg[2] = pg[3];
        if (i + 4 < ntl)
            pg[3] = page_of(i + 4);
    };

    if (ntl > 0) {
        floatx16 xa, xb;
#pragma unroll
        for (int t = 0; t < 4; t++)
            pg[t] = t < ntl ? page_of(t) : pg[t - 1];
        const __amdgpu_buffer_rsrc_t k_0 = k_rsrc(pg[0]), v_0 = v_rsrc(pg[0]), k_1 = k_rsrc(pg[1]);
#pragma unroll
        for (int n = 0; n < NL; n++)
            issue_k(k_0, 0, n);
        issue_scales(pg[0], 0);
        issue_q();
#pragma unroll
        for (int n = 0; n < NL; n++) {
            issue_k(k_1, 1, n);
            issue_v(v_0, 0, n);
        }
        issue_scales(pg[1], 1);
        /* Q and K of tile 0; what was issued after them is at least 2 NL loads */
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * NL) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
#pragma unroll
        for (int ks = 0; ks < 16; ks++) {
            const int piece = E4M3 ? 4 * (ks >> 1) + 2 * h + (ks & 1) : 2 * ks + h;
            qf[ks] = __builtin_bit_cast(
                bf16x8, lds_read16(lds, qat + col * 512 + ((piece ^ (col & 15)) << 4)));
        }
        ksc = kscale(0);
        unroll_for<2>([&](auto ib) { /* operands of 8 k-steps at a time */
            constexpr int part = decltype(ib)::value;
            u32x4 w[NKR / 2];
#pragma unroll
            for (int n = 0; n < NKR / 2; n++)
                w[n] = lds_read16(lds, kaddr(part * (NKR / 2) + n, 0));
            __builtin_amdgcn_sched_barrier(0);
            unroll_for<8>([&](auto ik) {
                constexpr int k = decltype(ik)::value;
                if constexpr (E4M3)
                    score(xa, k & 1 ? widen(w[k >> 1][2], w[k >> 1][3], ksc)
                                    : widen(w[k >> 1][0], w[k >> 1][1], ksc),
                          8 * part + k);
                else
                    score(xa, __builtin_bit_cast(bf16x8, w[k]), 8 * part + k);
            });
        });
        asm volatile("s_nop 15\n\ts_nop 7" : "+v"(xa));
        load_vsc(0);
        mask(xa, 0, pg[0] >= 0);
        mx = -INFINITY;
#pragma unroll
        for (int v = 0; v < 16; v++)
            mx = fmaxf(mx, xa[v]);
        unroll_for<4>([&](auto iv) { pair(xa, pn, template_int<2 * decltype(iv)::value>{}, 0.f); });
        want();
        /* K of tile 1 is there, and K buffer 0 free */
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        ksc = kscale(1);
#pragma unroll
        for (int n = 0; n < QD; n++)
            ring[n] = lds_read16(lds, kaddr(n, 1));
        const __amdgpu_buffer_rsrc_t k_2 = k_rsrc(pg[2]);
#pragma unroll
        for (int n = 0; n < NL; n++)
            issue_k(k_2, 0, n);
        issue_scales(pg[2], 2);
        for (int i = 0;;) {
            step(i, template_int<0>{}, xa, xb);
            if (++i == ntl)
                break;
            step(i, template_int<1>{}, xb, xa);
            if (++i == ntl)
                break;
        }
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    }

    /* ---- epilogue: l of a row from the pair's two halves; O / l (a share: O) as fp32
     * rows of 1 KiB through LDS, piece p of row r in slot p ^ (r & 31); then a wave
     * finishes 16 rows, their gates on the way since before O was staged. Where row
     * t's gate and output lie is worked out by lane t. ---- */
    settle(o);
    const bool whole = nshare == 1, gated = whole && c.gate;
    const int t0 = 16 * wave;
    size_t gat, oat;
    {
        const int r = rest + min(t0 + (lane & 15), nrows - 1), after = r * c.rG >> 16;
        const int tok = i0 + after, hd = r - after * c.G;
        gat = (size_t)(s.q0 + tok) * c.gts + (size_t)(kh * c.G + hd) * c.ghs;
        oat = whole ? ((size_t)(s.q0 + tok) * c.Hq + kh * c.G + hd) * PD
                    : (slot * RT + t0 + (lane & 15)) * PD;
    }
    auto of_row = [&](size_t x, int t) {
        return (size_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, t) |
               (size_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(x >> 32), t) << 32;
    };
    bf16x4 gv[16];
    if (gated) {
#pragma unroll
        for (int t = 0; t < 16; t++)
            gv[t] = *(const bf16x4 *)(c.gate + of_row(gat, t) + 4 * lane);
    }
    __syncthreads(); /* the tile buffers are idle */
    float *stat = (float *)(smem + L::STAT); /* [2][row] */
    const float lw = lrun + __shfl_xor(lrun, 32, 64);
    if (h == 0)
        stat[wj * RT + 32 * wi + col] = lw;
    __syncthreads();
    const float l = stat[32 * wi + col] + stat[RT + 32 * wi + col];
    const float inv = !whole ? 1.f : l > 0.f ? 1.f / l : 0.f;
    bool lost = false; /* see LOST_L */
    const bool large = l > LOST_L, small = l < 1.f / LOST_L && l > 0.f;
    if (__any(large || small)) {
        uint32_t most = 0;
#pragma unroll
        for (int d = 0; d < 4; d++) {
#pragma unroll
            for (int r = 0; r < 16; r++) /* on the bits: O may be NaN */
                most = max(most, __float_as_uint(o[d][r]) & 0x7fffffffu);
            asm volatile("" : "+a"(o[d])); /* read again below, not kept */
            __builtin_amdgcn_sched_barrier(0);
        }
        lost = (large && most > __float_as_uint(LOST_HIGH)) ||
               (small && most < __float_as_uint(LOST_LOW));
    }
    if constexpr (KIND != CAUSAL) {
        if (whole && c.lse && wj == 0 && h == 0 && 32 * wi + col < nrows) {
            const int r = rest + 32 * wi + col, after = r * c.rG >> 16;
            c.lse[(size_t)(s.q0 + i0 + after) * c.Hq + kh * c.G + r - after * c.G] =
                lse_of(l, mus);
        }
    }
    int *again = (int *)(smem + L::AGAIN);
    const int any_lost = __any(lost);
    if (lane == 0)
        again[wave] = any_lost;
    if (!whole && wj == 0 && h == 0) {
        c.pl[slot * RT + 32 * wi + col] = l;
        c.pmu[slot * RT + 32 * wi + col] = mus;
    }
#pragma unroll
    for (int d = 0; d < 4; d++) {
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const floatx4 v = {o[d][4 * q] * inv, o[d][4 * q + 1] * inv, o[d][4 * q + 2] * inv,
                               o[d][4 * q + 3] * inv};
            const int piece = 32 * wj + 8 * d + 2 * q + h;
            *(floatx4 *)(smem + (32 * wi + col) * 1024 + ((piece ^ col) << 4)) = v;
        }
        __builtin_amdgcn_sched_barrier(0);
    }
    __syncthreads();
    if (range > 0.f && __any(again[lane & 7])) {
        __syncthreads(); /* the flags are read, LDS is free */
        return true;
    }
#pragma unroll
    for (int half = 0; half < 2; half++) { /* no branch between the reads */
        floatx4 v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int row = t0 + 8 * half + i;
            v[i] = *(const floatx4 *)(smem + row * 1024 + ((lane ^ (row & 31)) << 4));
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int t = 8 * half + i;
            if (!whole) {
                if (t0 + t < nrows)
                    *(floatx4 *)(c.po + of_row(oat, t) + 4 * lane) = v[i];
                continue;
            }
            bf16x4 res;
#pragma unroll
            for (int e = 0; e < 4; e++)
                res[e] = f2bf(gated ? v[i][e] * sigmoid_f(bf2f(gv[t][e])) : v[i][e]);
            if (t0 + t < nrows)
                *(bf16x4 *)(c.out + of_row(oat, t) + 4 * lane) = res;
        }
    }
    return false;
}
template <bool E4M3, int KIND>
__global__ __launch_bounds__(512, 2) void attention_many_kernel(Call c) {
    __shared__ __attribute__((aligned(1024))) unsigned char smem[Lay<E4M3>::BYTES];
    /* c by an address that is unknown each time: known, the arguments were kept for the
     * second time, in more registers than there are. A copy: through the address they
     * were loaded where they are used, tile by tile (12 x 500 0.6 us more). */
    auto *args =
        (const __attribute__((address_space(4))) Call *)__builtin_amdgcn_kernarg_segment_ptr();
    float range = SHIFT_RANGE;
    for (;;) {
        asm volatile("" : "+s"(args));
        const Call a = *(const Call *)args;
        if (!attend_many<E4M3, KIND>(a, smem, range))
            break;
        range = 0.f;
    }
}

/* ---- merge of a unit's parts -----------------------------------------------------
 * o = sum 2^(mu_i - mu) o_i over the parts that saw keys, l likewise, mu the largest
 * of theirs; then / l and the gate. The loads of l and mu, a part a lane, and of the
 * first o go out together. */

/* Of few rows: a wave per row, o 16 parts at a time; or, ROW, a workgroup: a wave 64
 * dims, o 64 parts at a time, 4 a load. That is for few rows after many keys (4 rows
 * of 64 parts: 5.4 us, and 8.8 a wave per row); the starts of many workgroups cost
 * more than it gains (1024 rows of 4 parts: 5.6 and 4.8, 4096 of them 22 and 8). */
template <bool ROW, bool STATS, int RU = PG_FEW>
__global__ __launch_bounds__(256) void merge_few_kernel(Call c, int groups) {
    constexpr int STEP = ROW ? 64 : 16, PER = STEP / 16;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int group = blockIdx.x % groups, kh = blockIdx.x / groups % c.Hkv;
    const int u = blockIdx.x / groups / c.Hkv, r = ROW ? group : group * 4 + wave;
    /* RU rows a unit: of few rows a sequence is one */
    const int per = RU == FEW ? 1 : c.plan.units / c.B, b = u / per, r0 = (u - b * per) * RU;
    const pg_seq s = seq_of(c, b);
    const int2 info = ((const int2 *)c.info)[u]; /* of a unit with rows */
    if (r0 + r >= s.ql * c.G || info.y <= 1)
        return;
    const int first = info.x, parts = info.y;
    const size_t slot0 = slot_of(c, kh, 0);
    auto at = [&](int j) { return (slot0 + pg_few_slot(first, j)) * RU + r; };
    const int dim = ROW ? 64 * wave + 4 * (lane & 15) : 4 * lane, own = ROW ? lane >> 4 : 0;
    const int tok = RU == FEW ? r * c.rG >> 16 : (r0 + r) / c.G;
    const int n = s.q0 + tok, head = kh * c.G + r0 + r - tok * c.G;
    bf16x4 gv = {};
    if (c.gate)
        gv = *(const bf16x4 *)(c.gate + (size_t)n * c.gts + (size_t)head * c.ghs + dim);
    float mu = -INFINITY, l = 0.f;
    floatx4 acc = {};
    for (int j0 = 0; j0 < parts; j0 += 64) { /* more than 64 parts: in turns */
        const int cnt = min(parts - j0, 64);
        const size_t mine = at(j0 + min(lane, cnt - 1));
        const float pl = c.pl[mine], pm = c.pmu[mine];
        const float li = lane < cnt ? pl : 0.f, mi = li > 0.f ? pm : -INFINITY;
        float wi = 0.f;
        for (int k0 = 0; k0 < cnt; k0 += STEP) {
            floatx4 v[16];
#pragma unroll
            for (int k = 0; k < 16; k++)
                if (k0 + k * PER < cnt) /* uniform */
                    v[k] = *(const floatx4 *)(
                        c.po + at(j0 + min(k0 + k * PER + own, cnt - 1)) * PD + dim);
            if (k0 == 0) {
                const float next = fmaxf(mu, wave_max(mi));
                const float ref = next == -INFINITY ? 0.f : next, old = fast_exp2(mu - ref);
                wi = li > 0.f ? fast_exp2(mi - ref) : 0.f;
                mu = next;
                l = l * old + wave_sum(wi * li);
                acc *= old;
            }
#pragma unroll
            for (int k = 0; k < 16; k++) {
                if (k0 + k * PER >= cnt)
                    break;
                /* lanes from cnt on have weight 0 */
                const float f = ROW ? __shfl(wi, k * PER + own, 64)
                                    : __uint_as_float((uint32_t)__builtin_amdgcn_readlane(
                                          (int)__float_as_uint(wi), k0 + k));
                if (f > 0.f)
                    acc += v[k] * f;
            }
        }
    }
    if constexpr (ROW) {
#pragma unroll
        for (int e = 0; e < 4; e++)
            acc[e] = fold_rows(acc[e], [](float x, float y) { return x + y; });
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
    bf16x4 res;
#pragma unroll
    for (int e = 0; e < 4; e++)
        res[e] = f2bf(acc[e] * inv * (c.gate ? sigmoid_f(bf2f(gv[e])) : 1.f));
    if (!ROW || lane < 16)
        *(bf16x4 *)(c.out + ((size_t)n * c.Hq + head) * PD + dim) = res;
    if (STATS && c.lse && dim == 0 && (!ROW || lane < 16))
        c.lse[(size_t)n * c.Hq + head] = lse_of(l, mu);
}

/* Of many rows: a wave 4 rows, all at once (one after the other took 11.2 us instead
 * of 9.6 for 16 sequences' 40 tokens in 2 or 3 parts). l and mu: lane 16 i + j has row
 * i's of part j, 16 parts in turn; o 4 parts at a time. */
template <bool STATS> __global__ __launch_bounds__(256) void merge_many_kernel(Call c) {
    constexpr int R = 4, GROUPS = RT / (4 * R);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int group = blockIdx.x % GROUPS, kh = blockIdx.x / GROUPS % c.Hkv;
    const int part = blockIdx.x / GROUPS / c.Hkv; /* a unit's first: its merge */
    const int4 info = ((const int4 *)c.info)[part];
    const int parts = info.z, r0 = info.y * RT, t0 = (group * 4 + wave) * R;
    if (parts <= 1 || part + parts > c.plan.slots) /* more than any rising q_start has */
        return;
    const pg_seq s = seq_of(c, info.x);
    const int last = min(s.ql * c.G - r0, RT) - 1;
    if (t0 > last)
        return;
    const float *po[R]; /* part 0 of a row's o; past the last row it again */
    bf16 *out[R];
    bf16x4 gv[R] = {};
    const size_t slot = slot_of(c, kh, part);
#pragma unroll
    for (int i = 0; i < R; i++) {
        const int t = min(t0 + i, last), r = r0 + t, tok = r / c.G, head = kh * c.G + r % c.G;
        const size_t n = s.q0 + tok;
        po[i] = c.po + (slot * RT + t) * PD + 4 * lane;
        out[i] = c.out + (n * c.Hq + head) * PD + 4 * lane;
        if (c.gate)
            gv[i] = *(const bf16x4 *)(c.gate + n * c.gts + (size_t)head * c.ghs + 4 * lane);
    }
    const int own = min(t0 + (lane >> 4), last);
    float mu = -INFINITY, l = 0.f; /* of row lane >> 4 */
    floatx4 acc[R] = {};
    auto of = [&](float x, int at) {
        return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(x), at));
    };
    for (int j0 = 0; j0 < parts; j0 += 16) {
        const int cnt = min(parts - j0, 16);
        const size_t mine = (slot + j0 + min(lane & 15, cnt - 1)) * RT + own;
        const float pl = c.pl[mine], pm = c.pmu[mine];
        const float li = (lane & 15) < cnt ? pl : 0.f, mi = li > 0.f ? pm : -INFINITY;
        float wi = 0.f;
        for (int k0 = 0; k0 < cnt; k0 += 4) {
            floatx4 v[4][R];
#pragma unroll
            for (int k = 0; k < 4; k++) /* past the last part it again, with weight 0 */
#pragma unroll
                for (int i = 0; i < R; i++)
                    v[k][i] = *(const floatx4 *)(po[i] + (size_t)(j0 + min(k0 + k, cnt - 1)) *
                                                             (RT * PD));
            if (k0 == 0) {
                const float next =
                    fmaxf(mu, fold_row(mi, [](float x, float y) { return fmaxf(x, y); }));
                const float ref = next == -INFINITY ? 0.f : next, old = fast_exp2(mu - ref);
                wi = li > 0.f ? fast_exp2(mi - ref) : 0.f;
                mu = next;
                l = l * old + fold_row(wi * li, [](float x, float y) { return x + y; });
#pragma unroll
                for (int i = 0; i < R; i++)
                    acc[i] *= of(old, 16 * i);
            }
#pragma unroll
            for (int k = 0; k < 4; k++)
#pragma unroll
                for (int i = 0; i < R; i++) {
                    const float f = of(wi, 16 * i + k0 + k);
                    if (f > 0.f)
                        acc[i] += v[k][i] * f;
                }
        }
    }
#pragma unroll
    for (int i = 0; i < R; i++) {
        const float li = of(l, 16 * i), inv = li > 0.f ? 1.f / li : 0.f;
        bf16x4 res;
#pragma unroll
        for (int e = 0; e < 4; e++)
            res[e] = f2bf(acc[i][e] * inv * (c.gate ? sigmoid_f(bf2f(gv[i][e])) : 1.f));
        if (t0 + i <= last)
            *(bf16x4 *)out[i] = res;
        if (STATS && c.lse && lane == 0 && t0 + i <= last)
            c.lse[(size_t)(out[i] - c.out) / PD] = lse_of(li, of(mu, 16 * i));
    }
}

} // namespace
} // namespace CUJEV_KNS
using namespace CUJEV_KNS;

extern "C" size_t cujev_attention_paged_ws_bytes(int N, int B, int max_q, int max_kv, int Hq,
                                                 int Hkv, int window, int sinks, int type) {
    (void)type, (void)window, (void)sinks; /* enough for either type and any window */
    return pg_ws_causal(N, B, max_q, max_kv, Hq / Hkv, Hkv);
}
extern "C" size_t cujev_attention_paged_tree_ws_bytes(int N, int B, int max_q, int max_kv, int Hq,
                                                      int Hkv) {
    return pg_ws_most(N, B, max_q, max_kv, Hq / Hkv, Hkv);
}

/* The workspace, from c.po on: o, l and mu of the plan's slots, then info */
static void set_workspace(Call &c, int Hkv) {
    const size_t rows = (size_t)c.plan.slots * Hkv * c.plan.rt;
    c.pl = c.po + rows * PD, c.pmu = c.pl + rows, c.info = (int32_t *)(c.pmu + rows);
}

/* Draft trees of a middling number of rows */
static hipError_t attend_middling(Call c, int Hkv, bool e4m3, size_t ws_bytes,
                                  hipStream_t stream) {
    const pg_plan p = c.plan = pg_make_mid_plan(c.N, c.B, c.max_q, c.max_kv, c.G, Hkv);
    if (p.shares == 0)
        return hipSuccess;
    if (p.shares < 0 || pg_mid_ws_bytes(p, Hkv) > ws_bytes)
        return hipErrorInvalidValue;
    set_workspace(c, Hkv);
    const dim3 grid((unsigned)(p.shares * Hkv));
    auto attend = [&](auto ie, auto ig) {
        constexpr int RG = decltype(ig)::value;
        hipLaunchKernelGGL((attention_mid_kernel<decltype(ie)::value, 2, RG>), grid,
                           dim3(256 * RG), 0, stream, c);
    };
    auto by_rows = [&](auto ie) {
        if ((long long)pg_min(c.max_q, c.N) * c.G <= 32)
            attend(ie, template_int<1>{});
        else
            attend(ie, template_int<2>{});
    };
    if (e4m3)
        by_rows(std::true_type{});
    else
        by_rows(std::false_type{});
    if (p.slots > 0) {
        const bool row = pg_mid_by_row(p, Hkv);
        const int groups = row ? PG_MID : PG_MID / 4;
        const dim3 mgrid((unsigned)(pg_mid_merge_items(p, Hkv) / 256));
        auto merge = [&](auto ir) {
            hipLaunchKernelGGL((merge_few_kernel<decltype(ir)::value, true, PG_MID>), mgrid,
                               dim3(256), 0, stream, c, groups);
        };
        if (row)
            merge(std::true_type{});
        else
            merge(std::false_type{});
    }
    return hipGetLastError();
}

extern "C" hipError_t k_attention_paged(const bf16_t *q, const bf16_t *gate, int gate_tok_stride,
                                        int gate_head_stride, const cujev_kv_pages *pages,
                                        const cujev_paged_seqs *seqs, int N, int max_q, int max_kv,
                                        int Hq, int window, int sinks, const uint64_t *tree,
                                        int tree_words, bf16_t *out, float *lse, void *ws,
                                        size_t ws_bytes, hipStream_t stream) {
    const int Hkv = pages->Hkv, B = seqs->B, G = Hq / Hkv;
    const bool e4m3 = pages->type == CUJEV_KV_E4M3;
    const bool all = window >= max_kv; /* keys of a row, but behind max_kv */
    Call c = {(const bf16 *)q, (const bf16 *)gate, gate_tok_stride, gate_head_stride,
              pages->k, pages->vt, pages->k_scale, pages->v_scale, pages->num_pages,
              seqs->q_start, seqs->kv_len, seqs->page_table, seqs->max_pages, B, N,
              max_q, max_kv, Hq, Hkv, G, window, sinks,
              all ? 0 : window, all ? 0 : sinks, pg_div_up(65536, G), tree, tree_words, lse,
              (bf16 *)out, (float *)ws, nullptr, nullptr, nullptr, {}};
    if (tree && pg_takes_mid(N, B, max_q, max_kv, G, Hkv, ws_bytes))
        return attend_middling(c, Hkv, e4m3, ws_bytes, stream);
    const pg_plan p = c.plan = pg_make_plan(N, B, max_q, max_kv, G, Hkv, window, sinks);
    if (p.shares == 0)
        return hipSuccess;
    if (p.shares < 0 || pg_ws_bytes(p, Hkv) > ws_bytes)
        return hipErrorInvalidValue;
    set_workspace(c, Hkv);
    const bool few = p.rt == FEW;
    const int per = !few && 8 % Hkv == 0 ? 8 / Hkv : 1;
    const dim3 grid((unsigned)(pg_div_up(p.shares, per) * per * Hkv)); /* all parts */
    auto launch = [&](auto ie, auto ik) {
        constexpr bool E = decltype(ie)::value;
        constexpr int KIND = decltype(ik)::value;
        if (few)
            hipLaunchKernelGGL((attention_few_kernel<E, KIND>), grid, dim3(64), 0, stream, c);
        else
            hipLaunchKernelGGL((attention_many_kernel<E, KIND>), grid, dim3(512), 0, stream, c);
    };
    auto by_kind = [&](auto ie) {
        if (tree)
            launch(ie, template_int<TREE>{});
        else if (lse)
            launch(ie, template_int<LSE>{});
        else
            launch(ie, template_int<CAUSAL>{});
    };
    if (e4m3)
        by_kind(std::true_type{});
    else
        by_kind(std::false_type{});
    if (p.slots > 0) {
        const int rows = pg_min(max_q, N) * G;
        const bool row = pg_merge_by_row(p, rows, Hkv);
        const int groups = pg_merge_groups(p, rows, Hkv);
        const dim3 mgrid((unsigned)(pg_merge_items(p, rows, Hkv) / 256));
        auto merge = [&](auto stats) {
            constexpr bool S = decltype(stats)::value;
            if (row)
                hipLaunchKernelGGL((merge_few_kernel<true, S>), mgrid, dim3(256), 0, stream, c,
                                   groups);
            else if (few)
                hipLaunchKernelGGL((merge_few_kernel<false, S>), mgrid, dim3(256), 0, stream, c,
                                   groups);
            else
                hipLaunchKernelGGL((merge_many_kernel<S>), mgrid, dim3(256), 0, stream, c);
        };
        if (lse)
            merge(std::true_type{});
        else
            merge(std::false_type{});
    }
    return hipGetLastError();
}
