/* Eviction from the paged K/V cache on gfx950: the weight that attention has given
 * each key, the positions worth keeping, and their move to the front. The reference
 * has one contiguous cache per state that only grows (src/engine/model.h:60-72). */
#include "paged.h"

namespace CUJEV_KNS {
namespace {



/* ---- attention weights by key --------------------------------------------------
 *   w[j] = prev[j] + sum over the call's rows (n, h) that see key j of 2^(q.k_j - lse)
 * with the attention's own lse, so that one product with K gives p whole: no second
 * pass, and no sum that crosses workgroups. A workgroup holds KG pages of a kv-head's
 * K in registers, a wave 64 keys, as the A operand of v_mfma_f32_32x32x16_bf16, and
 * streams the packed rows (token, q-head) through LDS, 32 for each of its 8 / KG row
 * groups at a time. A lane then has p of one row and 32 keys and adds them up over
 * the rows; lanes and row groups are summed once, at the end, in a fixed order. */
struct Weigh {
    const bf16 *q;
    const float *lse;
    const void *k;
    const float *ks;
    int num_pages;
    const int32_t *q_start, *kv_len, *page_table;
    int max_pages, B, N, max_q, max_kv, Hq, Hkv, G, rG, blocks; /* of a sequence and head */
    const float *prev;
    float *w;
};

template <bool E4M3, int KG>
__global__ __launch_bounds__(512, 2) void weigh_kernel(Weigh c) {
    constexpr int RG = 8 / KG, STEP = 32 * RG;       /* rows a step */
    constexpr int QB = STEP * PD * 2;                /* bytes of a step's Q */
    constexpr int T = PSLICE * (E4M3 ? 1 : 2);       /* bytes of a K tile */
    constexpr int QD = 3;                            /* Q operand reads ahead */
    __shared__ __attribute__((aligned(1024))) unsigned char smem[2 * QB];
    __shared__ float part[RG][KG][64];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int kg = wave % KG, rg = wave / KG, col = lane & 31, h = lane >> 5;
    /* where the kv-heads divide the 8 XCDs, an XCD's workgroups read the same rows */
    int kh, kb, b;
    {
        const int per = 8 % c.Hkv == 0 ? 8 / c.Hkv : 1, all = pg_div_up(c.blocks, per) * per * c.Hkv;
        b = blockIdx.x / all;
        const int at = blockIdx.x % all;
        if (8 % c.Hkv == 0) {
            kh = (at & 7) / per;
            kb = (at >> 3) * per + (at & 7) % per;
        } else {
            kh = at % c.Hkv;
            kb = at / c.Hkv;
        }
    }
    const pg_seq s = load_seq(c.q_start, c.kv_len, b, c.N, c.max_q, c.max_kv);
    const int k0 = kb * KG * PG; /* the workgroup's first key */
    if (s.ql <= 0 || k0 >= s.kv)
        return;
    const int key0 = k0 + kg * PG; /* the wave's */
    int page = -1;
    if (key0 < s.kv) {
        page = c.page_table[(size_t)b * c.max_pages + key0 / PG];
        page = page >= 0 && page < c.num_pages ? page : -1;
    }
    const size_t slice = (size_t)max(page, 0) * c.Hkv + kh;

    /* rows: token t of the sequence sees key0 from position key0 on */
    const int t_first = max(k0 - s.p0, 0), nrows = s.ql * c.G;
    const int steps = pg_div_up(nrows - t_first * c.G, STEP);
    /* Q of step n: 2 rows a load, piece p of row r in slot p ^ (r & 15) */
    auto issue_q = [&](int n) {
        const int r0 = t_first * c.G + n * STEP, i0 = r0 / c.G, rest = r0 - i0 * c.G;
        const __amdgpu_buffer_rsrc_t src =
            make_rsrc(c.q + ((size_t)(s.q0 + i0) * c.Hq + kh * c.G) * PD, 0x7fffffff);
        const int id = lane_again(); /* addresses are worked out again, not kept */
#pragma unroll
        for (int i = 0; i < 2 * RG; i++) {
            const int at = (i * 8 + wave) * 2 + (id >> 5), row = rest + min(at, nrows - 1 - r0);
            const int tok = row * c.rG >> 16;
            const uint32_t off = (tok * c.Hq + row - tok * c.G) * PD * 2;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                src, (lds_ptr)(smem + (n & 1) * QB + (i * 8 + wave) * 1024), 16,
                off + (((id & 31) ^ (at & 15)) << 4), 0, 0, 0);
        }
    };
    /* this lane's row of step n: its lse (+inf where there is none, or it sees nothing), and
     * the last key that it sees */
    float lse;
    int last;
    auto row_of = [&](int n) {
        const int r0 = t_first * c.G + n * STEP, i0 = r0 / c.G, rest = r0 - i0 * c.G;
        const int at = 32 * rg + (lane_again() & 31), row = rest + min(at, nrows - 1 - r0);
        const int tok = row * c.rG >> 16;
        const float x = c.lse[(size_t)(s.q0 + i0 + tok) * c.Hq + kh * c.G + row - tok * c.G];
        lse = r0 + at < nrows && x != -INFINITY ? x : INFINITY;
        last = s.p0 + i0 + tok;
    };
    if (steps > 0)
        issue_q(0);
    bf16x8 kf[2][16];
    {
        const __amdgpu_buffer_rsrc_t src = make_rsrc((const char *)c.k + slice * T, T);
        const uint32_t voff = col * (T / PG) + h * 16;
        u32x4 raw[2][E4M3 ? 8 : 16];
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int n = 0; n < (E4M3 ? 8 : 16); n++)
                raw[i][n] = buf_load16(src, voff, i * (T / 2) + n * 32);
        float sc[2] = {1.f, 1.f};
        if constexpr (E4M3) {
#pragma unroll
            for (int i = 0; i < 2; i++)
                sc[i] = c.ks[slice * PG + 32 * i + col];
        }
        if (page < 0 || key0 + PG > s.kv) { /* slots of no key may hold anything */
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const bool there = page >= 0 && key0 + 32 * i + col < s.kv;
                sc[i] = there ? sc[i] : 1.f;
#pragma unroll
                for (int n = 0; n < (E4M3 ? 8 : 16); n++)
                    raw[i][n] &= there ? ~0u : 0u;
            }
        }
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int n = 0; n < (E4M3 ? 8 : 16); n++) {
                const u32x4 v = raw[i][n];
                if constexpr (E4M3) {
                    kf[i][2 * n] = widen(v[0], v[1], sc[i]);
                    kf[i][2 * n + 1] = widen(v[2], v[3], sc[i]);
                } else {
                    kf[i][n] = __builtin_bit_cast(bf16x8, v);
                }
            }
    }
    float sum[2][16] = {};
    for (int n = 0; n < steps; n++) {
        row_of(n);
        /* step n's Q is there, and the other buffer read */
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (n + 1 < steps)
            issue_q(n + 1);
        /* this lane's row and half of piece 0; the others by their bits, worked out from
         * the buffer's address each time: kept, 16 of them went to scratch memory */
        const uint32_t at0 = (n & 1) * QB + (32 * rg + col) * 512 +
                             (((E4M3 ? 2 * h : h) ^ (col & 15)) << 4);
        auto q_at = [&](int ks) {
            const uint32_t bits = (E4M3 ? 4 * (ks >> 1) + (ks & 1) : 2 * ks) << 4;
            return *(const bf16x8 *)(smem + (at0 ^ bits));
        };
        floatx16 x[2] = {};
        bf16x8 ring[QD];
#pragma unroll
        for (int ks = 0; ks < QD; ks++)
            ring[ks] = q_at(ks);
#pragma unroll
        for (int ks = 0; ks < 16; ks++) {
            const bf16x8 qv = ring[ks % QD];
            if (ks + QD < 16)
                ring[ks % QD] = q_at(ks + QD);
#pragma unroll
            for (int i = 0; i < 2; i++)
                x[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[i][ks], qv, x[i], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0); /* no more operands at a time: registers */
        }
        /* accumulator v of block i is key key0 + 32 i + 8 (v >> 2) + 4 h + (v & 3) */
        if (__all(last >= key0 + PG - 1)) {
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int v = 0; v < 16; v++)
                    sum[i][v] += fast_exp2(x[i][v] - lse);
        } else {
            const int seen = last - key0 - 4 * h;
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int v = 0; v < 16; v++) {
                    const float p = fast_exp2(x[i][v] - lse);
                    sum[i][v] += 32 * i + 8 * (v >> 2) + (v & 3) <= seen ? p : 0.f;
                }
        }
    }
    /* over the 32 rows' lanes: lane 16 r + v is left with block r & 1, half r >> 1, number v */
    float mine = 0.f;
#pragma unroll
    for (int v = 0; v < 16; v++) {
        const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(sum[0][v]),
                                                        __float_as_uint(sum[1][v]), false, false);
        const float t = fold_row(__uint_as_float(a[0]) + __uint_as_float(a[1]),
                                 [](float p, float q) { return p + q; });
        mine = (lane & 15) == v ? t : mine;
    }
    const int v = lane & 15, key = 32 * (lane >> 4 & 1) + 8 * (v >> 2) + 4 * h + (v & 3);
    part[rg][kg][key] = mine;
    __syncthreads();
    if (rg == 0 && page >= 0 && key0 + lane < s.kv) {
        float all = part[0][kg][lane];
#pragma unroll
        for (int i = 1; i < RG; i++)
            all += part[i][kg][lane];
        const size_t to = slice * PG + lane;
        if (c.prev && key0 + lane < s.p0)
            all += c.prev[to];
        c.w[to] = all;
    }
}

/* ---- positions to keep ------------------------------------------------------------
 * A workgroup per sequence and kv-head. The weights' order is that of 32-bit integers
 * (ordered()); the least one kept is found by its digits of 11, 11 and 10 bits from the
 * top, each by a histogram in LDS of what has the digits before. Then positions are
 * counted in order: heavier ones, and of its equals the first. */
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

/* E weights a thread in registers, or E 0: read again each time */
template <int E> __global__ __launch_bounds__(SEL_T) void select_kernel(Select c) {
    __shared__ int hist[2048], scratch[SEL_T / 64], found[2];
    const int tid = threadIdx.x, lane = tid & 63, kh = blockIdx.x % c.Hkv, b = blockIdx.x / c.Hkv;
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
    auto weight = [&](int j) -> uint32_t {
        const int page = c.page_table[(size_t)b * c.max_pages + j / PG];
        return page >= 0 && page < c.num_pages
                   ? ordered(c.w[((size_t)page * c.Hkv + kh) * PG + j % PG])
                   : 0u;
    };
    const int tiles = E ? E : pg_div_up(kv, SEL_T);
    uint32_t u[E ? E : 1];
    if constexpr (E > 0) {
#pragma unroll
        for (int e = 0; e < E; e++)
            u[e] = e * SEL_T + tid < kv ? weight(e * SEL_T + tid) : 0u;
    }
    auto each = [&](auto f) { /* f(position, weight) of this thread's positions in order */
        if constexpr (E > 0) {
#pragma unroll
            for (int e = 0; e < E; e++)
                f(e * SEL_T + tid, u[e]);
        } else {
            for (int e = 0; e < tiles; e++) {
                const int j = e * SEL_T + tid;
                f(j, j < kv ? weight(j) : 0u);
            }
        }
    };
    /* the least kept: digits `top` so far under `mask`; ties: how many of its equals */
    uint32_t top = 0, mask = 0;
    int ties = want;
    if (want > 0) {
        for (int shift = 21, bits = 11; shift >= 0; bits = shift == 10 ? 10 : 11, shift -= bits) {
            for (int i = tid; i < 2048; i += SEL_T)
                hist[i] = 0;
            __syncthreads();
            each([&](int j, uint32_t x) {
                const bool in = j >= lo && j < hi && (x & mask) == top;
                const int digit = x >> shift & ((1u << bits) - 1);
                /* the first lane's digit by one add: many weights may be the same */
                const uint64_t live = __ballot(in);
                if (!live)
                    return;
                const int l = __ffsll((unsigned long long)live) - 1;
                const int d = __builtin_amdgcn_readlane(digit, l);
                const uint64_t same = __ballot(in && digit == d);
                if (lane == l)
                    atomicAdd(&hist[d], __popcll(same));
                if (in && digit != d)
                    atomicAdd(&hist[digit], 1);
            });
            __syncthreads();
            /* from the top: two digits a thread */
            const int d1 = 2047 - 2 * tid, c1 = hist[d1], c0 = hist[d1 - 1];
            int all;
            const int above = block_scan(c1 + c0, scratch, &all);
            if (above < ties && above + c1 + c0 >= ties) {
                const bool first = above + c1 >= ties;
                found[0] = first ? d1 : d1 - 1;
                found[1] = ties - above - (first ? 0 : c1);
            }
            __syncthreads();
            top |= (uint32_t)found[0] << shift;
            mask |= ((1u << bits) - 1) << shift;
            ties = found[1];
            if (shift == 0)
                break;
        }
    }
    /* in order: which are kept, and where they go */
    int kept = 0, equal = 0;
    each([&](int j, uint32_t x) {
        const bool mid = j >= lo && j < hi && want > 0;
        const bool eq = mid && x == top;
        int all;
        const int rank = equal + block_scan(eq, scratch, &all);
        equal += all;
        const bool yes = j < kv && (j < lo || j >= hi || (mid && x > top) || (eq && rank < ties));
        const int at = kept + block_scan(yes, scratch, &all);
        kept += all;
        if (yes && at < n)
            keep[at] = j;
    });
}

/* ---- kept positions to the front -----------------------------------------------------
 * Slot dst + i takes what position keep[i] has: rows of K by lines of 128 bytes, V^T by
 * rows of dims, an element a slot, and scales and weights. In place a workgroup does its
 * lines or rows of a sequence and kv-head from the front to the back: positions ascend
 * and none is before the slot it goes to, so that all reads of a step are of slots that
 * no step before has written, and those of the step itself are done before its writes. */
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
    return (long long)(uint32_t)__shfl((int)x, l, 64) | (long long)__shfl((int)(x >> 32), l, 64) << 32;
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

extern "C" hipError_t k_kv_weights(const bf16_t *q, const float *lse, const cujev_kv_pages *pages,
                                   const cujev_paged_seqs *seqs, int N, int max_q, int max_kv,
                                   int Hq, const float *prev, float *weights,
                                   hipStream_t stream) {
    const int Hkv = pages->Hkv, B = seqs->B, G = Hq / Hkv, tiles = pg_div_up(max_kv, PG);
    if (N <= 0 || B <= 0 || max_q <= 0 || tiles <= 0)
        return hipSuccess;
    /* as many pages a workgroup as leave a workgroup for each CU */
    int kg = 8;
    while (kg > 2 && (long long)B * pg_div_up(tiles, kg) * Hkv < 256)
        kg /= 2;
    const int blocks = pg_div_up(tiles, kg), per = 8 % Hkv == 0 ? 8 / Hkv : 1;
    const long long grid = (long long)pg_div_up(blocks, per) * per * Hkv * B;
    if (grid * 512 > PG_MOST_ITEMS)
        return hipErrorInvalidValue;
    const Weigh c = {(const bf16 *)q, lse, pages->k, pages->k_scale, pages->num_pages,
                     seqs->q_start, seqs->kv_len, seqs->page_table, seqs->max_pages, B, N, max_q,
                     max_kv, Hq, Hkv, G, pg_div_up(65536, G), blocks, prev, weights};
#define LAUNCH(T, KG)                                                                             \
    hipLaunchKernelGGL((weigh_kernel<T, KG>), dim3((unsigned)grid), dim3(512), 0, stream, c)
    if (pages->type == CUJEV_KV_E4M3) {
        if (kg == 8)
            LAUNCH(true, 8);
        else if (kg == 4)
            LAUNCH(true, 4);
        else
            LAUNCH(true, 2);
    } else {
        if (kg == 8)
            LAUNCH(false, 8);
        else if (kg == 4)
            LAUNCH(false, 4);
        else
            LAUNCH(false, 2);
    }
#undef LAUNCH
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
    else if (max_kv <= 16 * SEL_T)
        LAUNCH(16);
    else
        LAUNCH(0);
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
