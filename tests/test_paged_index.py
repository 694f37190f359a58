"""Where the paged operators read and write, on the CPU: paged_index.h, which
the kernels index with, compiled for the host and checked against brute force
over random and extreme lengths, and over lengths no caller should pass."""
import pathlib
import subprocess

KERNELS = pathlib.Path(__file__).resolve().parent.parent / "cu-jev_amd" / "csrc" / "kernels"

CHECK = r"""
#include "paged_index.h"
#include <cstdio>
#include <cstdlib>
#include <set>
#include <vector>

static int bad;
#define NEED(c) do { if (!(c) && bad++ < 10) printf("line %d: %s\n", __LINE__, #c); } while (0)
static unsigned rs = 12345;
static int rnd(int lo, int hi) { rs = rs * 1664525u + 1013904223u; return lo + (int)((rs >> 4) % (unsigned)(hi - lo + 1)); }

static bool seen(int j, int hi, int lo, int S) { return j <= hi && (j > lo || j < S); }

int main() {
    /* any lengths at all stay inside the call */
    const int odd[] = {0, 1, -1, 5, 63, 64, 65, 200, 4096, PG_MOST, -PG_MOST, 0x7fffffff, (int)0x80000000};
    for (int q0 : odd) for (int q1 : odd) for (int kv : odd) for (int N : {0, 1, 64, 200, PG_MOST})
        for (int mq : {0, 1, 100, PG_MOST}) for (int mk : {0, 1, 64, 1000, PG_MOST_KEYS}) {
            const pg_seq s = pg_clean_seq(q0, q1, kv, N, mq, mk);
            NEED(s.q0 >= 0 && s.ql >= 0 && s.ql <= mq && (long long)s.q0 + s.ql <= N);
            NEED(s.kv >= 0 && s.kv <= mk && s.p0 >= -N);
            NEED(pg_new_lo(s) >= 0 && (pg_new_hi(s) <= s.kv));
            for (int w : {0, 1, 100, PG_MOST_KEYS}) for (int S : {0, 1, 64, 65, PG_MOST}) {
                if (s.ql == 0) continue;
                const pg_tiles t = pg_tile_list(s, 0, s.ql - 1, w, w ? S : 0);
                NEED(t.ntl >= 0 && t.nsk >= 0 && t.nsk <= t.ntl);
                if (t.ntl > 0) {
                    NEED(pg_tile_page(t, 0) >= 0);
                    NEED((long long)pg_tile_page(t, t.ntl - 1) * PG < s.kv);
                }
            }
        }
    /* lists, masks and bounds against brute force */
    for (int it = 0; it < 60000; it++) {
        const int ql = rnd(1, it % 3 ? 6 : 150), kvl = rnd(0, it % 5 ? 700 : 70), N = ql + rnd(0, 5), q0 = rnd(0, N - ql);
        const int max_kv = kvl + rnd(-20, 200) > 0 ? kvl + rnd(-20, 200) : 1, mk = max_kv < 1 ? 1 : max_kv;
        const int w = rnd(0, 2) ? rnd(1, 300) : 0, S = w && rnd(0, 1) ? rnd(0, 200) : 0;
        const pg_seq s = pg_clean_seq(q0, q0 + ql, kvl, N, N, mk);
        NEED(s.ql == ql && s.q0 == q0 && s.p0 == kvl - ql);
        const int i0 = rnd(0, ql - 1), i1 = rnd(i0, ql - 1 < i0 + 40 ? ql - 1 : i0 + 40);
        const pg_tiles t = pg_tile_list(s, i0, i1, w, S);
        const int pmin = s.p0 + i0, pmax = s.p0 + i1;
        std::set<int> visited;
        for (int i = 0; i < t.ntl; i++) {
            const int pg = pg_tile_page(t, i);
            NEED(pg >= 0 && pg * PG < s.kv && visited.insert(pg).second);
            NEED(i == 0 || pg > pg_tile_page(t, i - 1));
            bool whole = true, foreign = false;
            for (int j = pg * PG; j < pg * PG + PG; j++) {
                bool own = false;
                for (int p = pmin; p <= pmax; p++) {
                    const bool sees = j <= p && j < s.kv && (!w || j > p - w || j < S);
                    NEED(sees == seen(j, pg_min(p, s.kv - 1), pg_low(p, w), S));
                    whole &= sees, own |= sees;
                }
                NEED(!own || seen(j, s.kv - 1, pg_low(pmin, w), S));
                foreign |= !seen(j, s.kv - 1, pg_low(pmin, w), S);
            }
            NEED(!pg_tile_whole(pg * PG, pmin, pmax, s.kv, w, S) || whole);
            NEED(!foreign || pg_tile_foreign(pg * PG, pmin, s.kv, w, S));
            /* a tile with a scale or value to hide also takes the masked path */
            NEED(!pg_tile_foreign(pg * PG, pmin, s.kv, w, S) || !pg_tile_whole(pg * PG, pmin, pmax, s.kv, w, S));
        }
        for (int p = pmin; p <= pmax; p++) for (int j = 0; j < s.kv; j++)
            NEED(!seen(j, pg_min(p, s.kv - 1), pg_low(p, w), S) || visited.count(j / PG));
        NEED(t.ntl <= pg_max_tiles(i1 - i0 + 1, mk, w, S));
        NEED(t.ntl <= pg_max_tiles(i1 - i0 + 1 + rnd(0, 50), mk, w, S));
    }
    /* V groups: each new position in exactly one; the launch has enough */
    for (int it = 0; it < 20000; it++) {
        const int B = rnd(1, 8);
        int N = 0, groups = 0;
        std::vector<int> q, kv;
        for (int b = 0; b < B; b++) { q.push_back(rnd(0, it % 2 ? 3 : 90)); kv.push_back(rnd(0, 200)); N += q[b]; }
        int at = 0;
        for (int b = 0; b < B; b++) {
            const pg_seq s = pg_clean_seq(at, at + q[b], kv[b], N, N, 160);
            at += q[b];
            const int n = pg_v_pages(s);
            groups += n;
            std::set<int> seen;
            for (int i = 0; i < 4 * n; i++) { /* a page's four groups of positions */
                const int base = (pg_new_lo(s) / PG + i / 4) * PG + i % 4 * VTOK;
                if (base + VTOK <= pg_new_lo(s) || base >= pg_new_hi(s)) continue;
                const int lo = pg_max(pg_new_lo(s), base), hi = pg_min(pg_new_hi(s), base + VTOK);
                NEED(lo < hi && base % PG + VTOK <= PG && base < s.kv);
                for (int p = lo; p < hi; p++) {
                    NEED(seen.insert(p).second && p >= 0 && p < s.kv);
                    const int row = s.q0 + p - s.p0;
                    NEED(row >= s.q0 && row < s.q0 + s.ql && row < N);
                }
            }
            NEED((int)seen.size() == pg_max(pg_new_hi(s) - pg_new_lo(s), 0));
        }
        NEED(groups <= (N < N / PG + 2 * B ? N : N / PG + 2 * B));
    }
    /* the plan: shares tile each unit's list, and the launch and slots hold them */
    for (int it = 0; it < 30000; it++) {
        const int G = 1 << rnd(0, 4), Hkv = 1 << rnd(0, 3);
        const int B = it % 7 ? rnd(1, 12) : rnd(1, 600), top = it % 3 ? 1 << rnd(0, 13) : 20000;
        const int mq = it % 2 ? rnd(1, 3) : rnd(1, 300), w = rnd(0, 2) ? 0 : rnd(1, 2000), S = w ? rnd(0, 100) : 0;
        std::vector<int> q, kv;
        int N = rnd(0, 3), max_q = 0, max_kv = 1;
        for (int b = 0; b < B; b++) {
            q.push_back(rnd(0, 3) ? rnd(0, mq) : mq), kv.push_back(rnd(0, top));
            N += q[b], max_q = pg_max(max_q, q[b]), max_kv = pg_max(max_kv, kv[b]);
        }
        if (rnd(0, 1)) max_kv += rnd(0, 500);
        const pg_plan p = pg_make_plan(N, B, max_q, max_kv, G, Hkv, w, S);
        const int W = w >= max_kv ? 0 : w, SS = W ? S : 0;
        long long U = 0, T = 0, C = 0;
        int at = 0;
        std::vector<pg_seq> seqs;
        for (int b = 0; b < B; b++) {
            seqs.push_back(pg_clean_seq(at, at + q[b], kv[b], N, max_q, max_kv));
            at += q[b];
            const int u = max_q ? pg_units(seqs[b], G, p.rt) : 0;
            U += u, T += (long long)u * pg_longest(seqs[b], G, p.rt, W, SS);
        }
        if (max_q == 0) { NEED(p.shares == 0); continue; }
        NEED(p.rt == (max_q * G <= 16 ? 16 : 128) && U <= p.units);
        if (p.rt == 16) {
            if (U == 0) continue;
            const int size = pg_few_share(p, (int)U, (unsigned)T);
            int line = 0;
            std::vector<char> used(p.slots);
            for (int b = 0; b < B; b++) {
                if (pg_units(seqs[b], G, 16) == 0) continue;
                NEED(pg_units(seqs[b], G, 16) == 1);
                const int n = pg_longest(seqs[b], G, 16, W, SS);
                const pg_tiles t = pg_tile_list(seqs[b], 0, seqs[b].ql - 1, W, SS);
                NEED(t.ntl == n || t.ntl == 0);
                const int p0 = line / size, p1 = (line + n - 1) / size;
                NEED(B > 1 || p1 - p0 < 64);
                NEED(p1 < p.shares);
                for (int j = 0; p1 > p0 && j <= p1 - p0; j++) {
                    const int slot = pg_few_slot(p0, j);
                    NEED(slot < p.slots && !used[slot]);
                    if (slot < p.slots) used[slot] = 1;
                }
                line += n;
            }
            continue;
        }
        auto parts = [&](int share) {
            long long n = 0;
            for (int b = 0; b < B; b++) {
                const int u = pg_units(seqs[b], G, p.rt);
                n += u ? pg_parts(seqs[b], G, W, pg_longest(seqs[b], G, p.rt, W, SS), share) : 0;
            }
            return n;
        };
        int share = PG_MOST, longest = 0;
        for (int b = 0; b < B; b++)
            longest = pg_max(longest, pg_longest(seqs[b], G, p.rt, W, SS));
        if (pg_splits(p, (int)U) && U > 0) {
            const int sure = pg_share_first(p, (int)U, (unsigned)T, true);
            NEED(parts(sure) <= p.goal);
            unsigned all = 0;
            for (int b = 0; b < B; b++)
                if (pg_units(seqs[b], G, p.rt))
                    all += pg_all_tiles(seqs[b], G, W, pg_longest(seqs[b], G, p.rt, W, SS));
            NEED(all <= T + U);
            share = pg_share_first(p, (int)U, B > 64 ? (unsigned)T : all, B > 64);
            if (B <= 64)
                for (int tries = 0; parts(share) > p.goal; tries++) {
                    NEED(tries < 100);
                    share = pg_share_next(share);
                }
            share = pg_share_last(share, longest);
        }
        bool split = false;
        for (int b = 0; b < B; b++) {
            const int u = pg_units(seqs[b], G, p.rt), most = pg_longest(seqs[b], G, p.rt, W, SS);
            const int whole = u ? pg_short_units(seqs[b], G, W, most, share) : 0;
            NEED(whole >= 0 && whole <= u);
            long long own = 0;
            for (int k = 0; k < u; k++) {
                const int n = k < whole ? 1 : pg_nshare(most, share);
                own += n;
                split |= n > 1;
                const int r0 = k * p.rt, rows = pg_min(seqs[b].ql * G - r0, p.rt);
                NEED(rows > 0);
                const pg_tiles t = pg_tile_list(seqs[b], r0 / G, (r0 + rows - 1) / G, W, SS);
                NEED(k >= whole || share >= most || t.ntl <= share);
                NEED(pg_share_begin(t.ntl, 0, n) == 0 && pg_share_begin(t.ntl, n, n) == t.ntl);
                for (int i = 0; i < n && i < 70; i++)
                    NEED(pg_share_begin(t.ntl, i + 1, n) >= pg_share_begin(t.ntl, i, n));
            }
            NEED(u == 0 || own == pg_parts(seqs[b], G, W, most, share));
            C += own;
        }
        NEED(C <= p.shares && (!split || p.slots >= C));
    }
    {   /* the largest calls: nothing overflows */
        NEED(pg_make_plan(PG_MOST, 1, PG_MOST, PG_MOST_KEYS, 16, 1, 0, 0).shares == -1);
        NEED(pg_make_plan(PG_MOST, PG_MOST, 1, PG_MOST_KEYS, 16, 1, 0, 0).shares == -1);
        const pg_plan f = pg_make_plan(60, 60, 1, PG_MOST_KEYS, 16, 1, 0, 0);
        const pg_seq s = pg_clean_seq(0, 1, PG_MOST_KEYS, 60, 1, PG_MOST_KEYS);
        const int n = pg_longest(s, 16, 16, 0, 0);
        const int size = pg_few_share(f, 60, 60u * (unsigned)n);
        NEED(f.shares > 0 && (60ll * n - 1) / size < f.shares);
        NEED((f.goal + 1ll) * size < 0x7fffffff); /* where a piece ends */
    }
    printf("bad %d\n", bad);
    return bad != 0;
}
"""


def test_every_index_stays_inside(tmp_path):
    src, exe = tmp_path / "check.cpp", tmp_path / "check"
    src.write_text(CHECK)
    subprocess.run(["g++", "-O2", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover",
                    "-I", str(KERNELS), str(src), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout + run.stderr


WORKSPACE = r"""
#include "paged_index.h"
#include <cstdio>

static int bad;
#define NEED(c) do { if (!(c) && bad++ < 10) printf("line %d: %s\n", __LINE__, #c); } while (0)
static unsigned rs = 777;
static int rnd(int lo, int hi) { rs = rs * 1664525u + 1013904223u; return lo + (int)((rs >> 4) % (unsigned)(hi - lo + 1)); }
static int upto(int most) { return rnd(0, 3) ? rnd(0, most) : rnd(0, 1) ? most : rnd(0, most < 40 ? most : 40); }

int main() {
    for (int it = 0; it < 400000; it++) {
        const int G = rnd(1, 16), Hkv = it % 5 ? 1 << rnd(0, 4) : rnd(1, 300);
        const int N = rnd(0, it % 3 ? 300 : 9000), B = rnd(0, it % 4 ? 70 : 3000);
        const int mq = it % 2 ? rnd(0, 20) : rnd(0, 5000), mk = rnd(0, it % 3 ? 3000 : 70000);
        const size_t most = pg_ws_most(N, B, mq, mk, G, Hkv);
        const int n = upto(N), b = upto(B), q = upto(mq), k = upto(mk), w = rnd(0, 1) ? 0 : rnd(1, 4000);
        const pg_plan p = pg_make_plan(n, b, q, k, G, Hkv, w, w ? rnd(0, 200) : 0);
        if (p.shares < 0) continue; /* refused */
        NEED(pg_ws_bytes(p, Hkv) <= most);
        NEED(pg_ws_most(n, b, q, k, G, Hkv) <= most);
        NEED(Hkv > 256 || most <= (34u << 20) + 8ull * B);
    }
    /* a prompt that needs none, and what follows it */
    NEED(pg_ws_bytes(pg_make_plan(4096, 1, 4096, 8192, 4, 4, 0, 0), 4) == 0);
    NEED(pg_ws_bytes(pg_make_plan(512, 1, 512, 8192, 4, 4, 0, 0), 4) > 0);
    NEED(pg_ws_most(4096, 1, 4096, 8192, 4, 4) >= pg_ws_bytes(pg_make_plan(512, 1, 512, 8192, 4, 4, 0, 0), 4));
    NEED(pg_ws_most(4096, 1, 4096, 8192, 4, 4) >= pg_ws_bytes(pg_make_plan(1, 1, 1, 8192, 4, 4, 0, 0), 4));
    /* nothing to merge in one tile; the largest arguments */
    NEED(pg_ws_most(16, 16, 1, 64, 4, 4) == 0 && pg_ws_most(0, 4, 4, 4096, 4, 4) == 0);
    NEED(pg_ws_most(0x7fffffff, 0x7fffffff, 0x7fffffff, 0x7fffffff, 16, 1) < (80u << 20));
    printf("bad %d\n", bad);
    return bad != 0;
}
"""


def test_one_workspace_is_enough_for_every_smaller_call(tmp_path):
    src, exe = tmp_path / "ws.cpp", tmp_path / "ws"
    src.write_text(WORKSPACE)
    subprocess.run(["g++", "-O2", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover",
                    "-I", str(KERNELS), str(src), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout + run.stderr


MASKS = r"""
#include "paged_index.h"
#include <cstdio>
#include <initializer_list>

static int bad;
#define NEED(c) do { if (!(c) && bad++ < 10) printf("line %d: %s\n", __LINE__, #c); } while (0)

int main() {
    const int P[] = {-PG_MOST, -PG_MOST + 1, -64, -1, 0, 1, 63, 64, 129, 2000, PG_MOST_KEYS, 0x7ffffffe, 0x7fffffff};
    const int W[] = {0, 1, 2, 64, 65, 128, 1999, 2001, PG_MOST_KEYS, PG_MOST, 0x7ffffffe, 0x7fffffff};
    const int S[] = {0, 1, 64, 100, PG_MOST_KEYS, 0x7fffffff};
    const int KV[] = {1, 63, 64, 128, 500, 2048, PG_MOST_KEYS};
    for (int kv : KV) for (int w : W) for (int sinks : S) for (int p : P) for (int more : {0, 1, 40}) {
        const long long q = p + (long long)more;
        if (q > 0x7fffffff) continue;
        for (int k0 = 0; k0 < kv && k0 < 2200; k0 += PG) {
            bool whole = true, foreign = false;
            for (int j = k0; j < k0 + PG; j++) {
                /* the definition in 64 bits, of the rows at p and q and of any between */
                auto sees = [&](long long r) { return j <= r && j < kv && (w == 0 || j > r - w || j < sinks); };
                whole &= sees(p) && sees(q);
                const bool own = j < kv && (w == 0 || j > (long long)p - w || j < sinks);
                NEED(sees(p) == (j <= p && j < kv && (j > pg_low(p, w) || j < sinks)));
                NEED(own == (j < kv && (j > pg_low(p, w) || j < sinks)) || p < 0);
                foreign |= !own;
            }
            NEED(!pg_tile_whole(k0, p, (int)q, kv, w, sinks) || whole);
            NEED(!foreign || pg_tile_foreign(k0, p, kv, w, sinks) || p < 0);
        }
    }
    printf("bad %d\n", bad);
    return bad != 0;
}
"""


def test_masks_of_any_position_and_window(tmp_path):
    """Rows of sequences longer than the call's max_kv keep their window, however far."""
    src, exe = tmp_path / "masks.cpp", tmp_path / "masks"
    src.write_text(MASKS)
    subprocess.run(["g++", "-O2", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover",
                    "-I", str(KERNELS), str(src), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout + run.stderr


LENGTHS = r"""
#include "paged_index.h"
#include <cstdio>
#include <initializer_list>

static int bad;
#define NEED(c) do { if (!(c) && bad++ < 10) printf("line %d: %s\n", __LINE__, #c); } while (0)

int main() {
    for (int ql : {0, 1, 5, 64, 200}) for (int kv : {-7, 0, 1, 3, 64, 500, 0x7fffffff})
        for (int mq : {0, 1, 3, 64, 1000}) for (int mk : {1, 64, 400, PG_MOST_KEYS}) {
            const pg_seq s = pg_clean_seq(2, 2 + ql, kv, 1000, mq, mk);
            const int keys = kv < 0 ? 0 : kv;
            NEED(s.p0 == keys - ql && s.ql == (ql < mq ? ql : mq));
            /* a key is one of the call's where some computed row can see it, or the
             * sequence has no new token */
            const long long last = (long long)s.p0 + s.ql - 1;
            const long long want = last + 1 < 0 ? 0 : last + 1;
            NEED(s.kv == (want < mk ? want : mk));
            /* the plan of such lengths: no sum leaves an int */
            for (int G : {1, 4, 16}) for (int w : {0, 100}) {
                if (s.ql == 0) continue;
                const int n = pg_longest(s, G, PG_MANY, w, w ? 4 : 0);
                const int units = pg_units(s, G, PG_MANY), all = (int)pg_all_tiles(s, G, w, n);
                NEED(n >= 1 && all >= units && all <= units * n + units);
                for (int share : {1, 8, 100, PG_MOST})
                    NEED(pg_parts(s, G, w, n, share) >= units);
            }
        }
    printf("bad %d\n", bad);
    return bad != 0;
}
"""


def test_keys_end_with_the_last_computed_row(tmp_path):
    src, exe = tmp_path / "lens.cpp", tmp_path / "lens"
    src.write_text(LENGTHS)
    subprocess.run(["g++", "-O2", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover",
                    "-I", str(KERNELS), str(src), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout + run.stderr


LAUNCHES = r"""
#include "paged_index.h"
#include <cstdio>
#include <initializer_list>

static int bad;
#define NEED(c) do { if (!(c) && bad++ < 10) printf("line %d: %s\n", __LINE__, #c); } while (0)
static unsigned rs = 4242;
static int rnd(int lo, int hi) { rs = rs * 1664525u + 1013904223u; return lo + (int)((rs >> 4) % (unsigned)(hi - lo + 1)); }

int main() {
    int largest = 0;
    for (int it = 0; it < 300000; it++) {
        const int G = rnd(1, 16), Hkv = rnd(0, 3) ? 1 << rnd(0, 9) : rnd(1, 8192 / G);
        const int q = it % 2 ? rnd(1, 16) : rnd(1, 5000), k = 1 << rnd(0, 16);
        const int B = rnd(0, 1) ? (1 << 22) / Hkv + rnd(-2, 2) : 1 << rnd(0, 24);
        if (B < 1) continue;
        const long long n = (long long)B * q;
        const int N = n < PG_MOST ? (int)n : PG_MOST;
        const pg_plan p = pg_make_plan(N, B, q, k, G, Hkv, 0, 0);
        if (p.shares <= 0) continue;
        const int per = p.rt == PG_MANY && 8 % Hkv == 0 ? 8 / Hkv : 1;
        const long long grid = (long long)pg_div_up(p.shares, per) * per * Hkv;
        NEED(grid * (p.rt == PG_FEW ? 64 : 512) <= PG_MOST_ITEMS);
        if (p.slots <= 0) continue;
        const int rows = pg_min(q, N) * G;
        const int groups = pg_merge_groups(p, rows, Hkv);
        const long long merge = (long long)(p.rt == PG_FEW ? p.units : p.slots) * Hkv * groups;
        NEED(merge * 256 <= PG_MOST_ITEMS && merge * 256 == pg_merge_items(p, rows, Hkv));
        /* each row has a place in it */
        NEED(p.rt == PG_FEW ? groups * (pg_merge_by_row(p, rows, Hkv) ? 1 : 4) >= rows : groups * 16 == 128);
        largest += merge * 256 > PG_MOST_ITEMS - (1 << 20);
    }
    NEED(largest > 0); /* calls right below the bound were among them */
    /* as many units as there may be, where the merge has room for their rows */
    NEED(pg_make_plan(1 << 20, 1 << 20, 1, 4096, 4, 4, 0, 0).shares > 0);
    NEED(pg_make_plan(1 << 22, 1 << 20, 4, 4096, 4, 4, 0, 0).shares == -1);
    printf("bad %d\n", bad);
    return bad != 0;
}
"""


def test_launches_stay_within_their_bounds(tmp_path):
    src, exe = tmp_path / "grid.cpp", tmp_path / "grid"
    src.write_text(LAUNCHES)
    subprocess.run(["g++", "-O2", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover",
                    "-I", str(KERNELS), str(src), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout + run.stderr
