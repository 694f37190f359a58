"""Where draft trees of a middling number of rows are cut, on the CPU: the part of
paged_index.h that the kernels plan them with, compiled for the host and checked against
brute force: every tile of every unit is in one piece, parts have slots of their own in
the workspace, and the workspace that a query gives is enough for every smaller call."""
import pathlib
import subprocess

KERNELS = pathlib.Path(__file__).resolve().parent.parent / "cu-jev_amd" / "csrc" / "kernels"

CHECK = r"""
#include "paged_index.h"
#include <cstdio>
#include <set>
#include <vector>

static int bad;
#define NEED(c) do { if (!(c) && bad++ < 10) printf("line %d: %s\n", __LINE__, #c); } while (0)
static unsigned rs = 4321;
static int rnd(int lo, int hi) { rs = rs * 1664525u + 1013904223u; return lo + (int)((rs >> 4) % (unsigned)(hi - lo + 1)); }

static void pieces(int B, int G, int Hkv, int most_q, int most_kv, int loose) {
    std::vector<pg_seq> seqs;
    int N = 0, max_q = 0, max_kv = 0;
    std::vector<int> ql(B), kv(B);
    for (int b = 0; b < B; b++) {
        ql[b] = rnd(0, 4) ? rnd(1, most_q) : 0;
        kv[b] = rnd(0, 9) ? rnd(0, most_kv) : rnd(0, 3);
        N += ql[b];
        max_q = ql[b] > max_q ? ql[b] : max_q;
        max_kv = kv[b] > max_kv ? kv[b] : max_kv;
    }
    max_q += loose, max_kv += 100 * loose;
    if (!pg_is_mid(N, B, max_q, max_kv, G, Hkv)) return;
    const pg_plan p = pg_make_mid_plan(N, B, max_q, max_kv, G, Hkv);
    NEED(p.shares >= 0 && p.rt == PG_MID && p.units % B == 0);
    NEED(pg_mid_ws_bytes(p, Hkv) <= pg_ws_most(N, B, max_q, max_kv, G, Hkv));
    long long T = 0, U = 0;
    for (int b = 0, q0 = 0; b < B; q0 += ql[b++]) {
        seqs.push_back(pg_clean_seq(q0, q0 + ql[b], kv[b], N, max_q, max_kv));
        T += (long long)pg_units(seqs[b], G, PG_MID) * (ql[b] ? pg_longest(seqs[b], G, PG_LINE, 0, 0) : 0);
        U += pg_units(seqs[b], G, PG_MID);
    }
    const int over = pg_mid_over(p, (unsigned)T); /* what a unit counts for beside its tiles */
    const int size = pg_mid_share(p, (unsigned)T + (unsigned)U * over);
    NEED(size > over && (T + U * over + size - 1) / size <= p.shares); /* a workgroup for every piece */
    NEED((long long)p.shares * size < 0x7fffffff);
    std::set<int> slots, infos;
    long long begin = 0;
    for (int b = 0; b < B; b++) {
        const pg_seq &s = seqs[b];
        const int units = pg_units(s, G, PG_MID);
        NEED(units <= p.units / B);
        for (int u = 0; u < units; u++) {
            const int own = pg_longest(s, G, PG_LINE, 0, 0);
            NEED(own >= pg_tile_list(s, 0, s.ql - 1, 0, 0).ntl && own * PG <= pg_max(max_kv, 1) + PG);
            begin += over;
            const int first = (int)(begin / size), parts = (int)((begin + own - 1) / size) - first + 1;
            int covered = 0;
            for (int j = 0; j < parts; j++) {
                if (j > 0) /* what the piece's workgroup finds at the piece's start */
                    NEED((long long)(first + j) * size >= begin);
                else /* the start is in the unit, or the workgroup comes from one before */
                    NEED((long long)first * size <= begin && ((long long)first * size >= begin - over || begin > over));
                const int cut = (int)((first + (long long)j) * size - begin), i0 = pg_max(cut, 0);
                const int ntl = pg_min(cut + size, own) - i0;
                NEED(i0 == covered && ntl > 0);
                covered = i0 + ntl;
                NEED(first + j < p.shares);
                if (parts > 1) {
                    const int slot = pg_few_slot(first, j);
                    NEED(slot >= 0 && slot < p.slots && slots.insert(slot).second);
                }
            }
            NEED(covered == own);
            const int info = b * (p.units / B) + u;
            NEED(info < p.units && infos.insert(info).second);
            begin += own;
        }
    }
    NEED(begin == T + U * over);
    /* a piece's start is in some unit, whose first tile is in the piece, or in one before */
    begin = 0;
    for (int b = 0; b < B; b++)
        for (int u = 0; u < pg_units(seqs[b], G, PG_MID); u++) {
            const int own = pg_longest(seqs[b], G, PG_LINE, 0, 0);
            for (long long item = (begin + size - 1) / size * size; item < begin + over + own; item += size) {
                const int target = (int)(item / size), first = (int)((begin + over) / size);
                const int parts = (int)((begin + over + own - 1) / size) - first + 1;
                NEED(first <= target && target - first < parts);
            }
            begin += over + own;
        }
}

int main() {
    for (int it = 0; it < 30000; it++) {
        const int G = rnd(1, 16), Hkv = it % 7 ? 1 << rnd(0, 5) : rnd(1, 256);
        pieces(it % 5 ? rnd(1, 12) : rnd(1, 300), G, Hkv, it % 3 ? rnd(1, 64 / G + 1) : rnd(1, 200),
               rnd(1, it % 4 ? 900 : 30000), it % 6 ? 0 : rnd(1, 30));
    }
    /* the most that numbers on the line reach */
    for (long long B = 1; B <= PG_MOST; B *= 2) for (int kv : {64, 100000, PG_MOST_KEYS}) for (int G : {1, 16}) {
        const int N = B * 4 > PG_MOST ? PG_MOST : (int)(B * 4), mq = G == 16 ? 4 : 64;
        if (!pg_is_mid(N, (int)B, mq, kv, G, 1)) continue;
        const pg_plan p = pg_make_mid_plan(N, (int)B, mq, kv, G, 1);
        if (p.shares < 0) continue; /* refused */
        const long long T = (long long)p.units * ((kv + PG - 1) / PG);
        NEED(T <= PG_MOST);
        NEED((p.goal + 1ll) * pg_mid_share(p, (unsigned)(T + (long long)p.units * PG_MID_OVER)) < 0x7fffffff);
    }
    NEED(!pg_is_mid(1 << 22, 1 << 20, 4, PG_MOST_KEYS, 16, 1));
    /* one workspace for every smaller call */
    for (int it = 0; it < 300000; it++) {
        const int G = rnd(1, 16), Hkv = it % 5 ? 1 << rnd(0, 5) : rnd(1, 300);
        const int N = rnd(1, it % 3 ? 300 : 9000), B = rnd(1, it % 4 ? 70 : 3000);
        const int mq = it % 2 ? rnd(1, 64) : rnd(1, 1000), mk = rnd(1, it % 3 ? 5000 : 70000);
        const int n = rnd(1, N), b = rnd(1, B), q = rnd(1, mq), k = rnd(1, mk);
        if (!pg_is_mid(n, b, q, k, G, Hkv)) continue;
        const pg_plan p = pg_make_mid_plan(n, b, q, k, G, Hkv);
        NEED(p.shares < 0 || pg_mid_ws_bytes(p, Hkv) <= pg_ws_most(N, B, mq, mk, G, Hkv));
        NEED(p.shares * Hkv <= PG_MID_CHIP);
    }
    printf("bad %d\n", bad);
    return bad != 0;
}
"""


def test_every_tile_is_in_one_piece(tmp_path):
    src, exe = tmp_path / "check.cpp", tmp_path / "check"
    src.write_text(CHECK)
    subprocess.run(["g++", "-O2", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover",
                    "-I", str(KERNELS), str(src), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout + run.stderr
