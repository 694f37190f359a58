"""Workspace sizes of paged attention, on the CPU: callers without draft trees are not asked
for what trees take, and whatever the size, a tree's call fits in what it is given."""
import subprocess
from pathlib import Path

import pytest

pytest.importorskip("torch")

from cujev import ops  # noqa: E402
from test_paged_args import CAPACITY, FAKE  # noqa: E402
from test_paged_more_args import TREE, call  # noqa: E402

KERNELS = Path(__file__).resolve().parent.parent / "cu-jev_amd" / "csrc" / "kernels"


@pytest.mark.parametrize("N,B,max_q,max_kv,most", [
    # slots of 16 rows for pieces of two tiles; of 128 rows for none
    (64, 8, 8, 512, 64 * 16), (26, 1, 26, 530, 18 * 16), (896, 1, 896, 896, 28 * 16)])
def test_calls_without_trees_are_not_asked_for_more(N, B, max_q, max_kv, most):
    size = ops.attention_paged_ws_bytes(N, B, max_q, max_kv, 16, 4)
    assert 0 < size <= most * 4 * 258 * 4 + 8 * B
    assert size < ops.attention_paged_ws_bytes(N, B, max_q, max_kv, 16, 4, tree=True) < 35 << 20


def test_a_tree_is_refused_below_what_a_call_without_one_needs():
    need = ops.attention_paged_ws_bytes(64, 8, 4, 128, 8, 2)
    for ws, size in ((None, 0), (FAKE, 16), (FAKE + 8, need)):
        st, msg = call(TREE, N=64, B=8, max_q=4, ws=ws, ws_bytes=size)
        assert need > 0 and st == CAPACITY and "workspace" in msg


CHECK = r"""
#include "paged_index.h"
#include <cstdio>
static int bad;
#define NEED(c) do { if (!(c) && bad++ < 10) printf("line %d: %s\n", __LINE__, #c); } while (0)
static unsigned rs = 99;
static int rnd(int lo, int hi) { rs = rs * 1664525u + 1013904223u; return lo + (int)((rs >> 4) % (unsigned)(hi - lo + 1)); }

int main() {
    int small = 0;
    for (int it = 0; it < 400000; it++) {
        const int G = rnd(1, 16), Hkv = it % 5 ? 1 << rnd(0, 4) : rnd(1, 300);
        const int N = rnd(0, it % 3 ? 300 : 9000), B = rnd(0, it % 4 ? 70 : 3000);
        const int mq = it % 2 ? rnd(0, 64) : rnd(0, 5000), mk = rnd(0, it % 3 ? 3000 : 70000);
        const size_t causal = pg_ws_causal(N, B, mq, mk, G, Hkv), all = pg_ws_most(N, B, mq, mk, G, Hkv);
        NEED(causal <= all);
        small += causal < all;
        const int n = rnd(0, N), b = rnd(0, B), q = rnd(0, mq), k = rnd(0, mk), w = rnd(0, 1) ? 0 : rnd(1, 4000);
        const pg_plan p = pg_make_plan(n, b, q, k, G, Hkv, w, w ? rnd(0, 200) : 0);
        NEED(p.shares < 0 || pg_ws_bytes(p, Hkv) <= causal);
        NEED(pg_ws_causal(n, b, q, k, G, Hkv) <= causal);
        /* a tree: units of 64 rows with the larger size wherever they are the faster form,
         * and with the smaller one what fits */
        NEED(pg_takes_mid(n, b, q, k, G, Hkv, all) == pg_is_mid(n, b, q, k, G, Hkv));
        const pg_plan t = pg_make_plan(n, b, q, k, G, Hkv, 0, 0);
        const bool mid = pg_takes_mid(n, b, q, k, G, Hkv, causal);
        NEED(mid || t.shares < 0 || pg_ws_bytes(t, Hkv) <= causal);
        if (mid) NEED(pg_mid_ws_bytes(pg_make_mid_plan(n, b, q, k, G, Hkv), Hkv) <= causal);
    }
    NEED(small > 1000);
    printf("bad %d\n", bad);
    return bad != 0;
}
"""


def test_each_size_is_enough_for_its_calls(tmp_path):
    src, exe = tmp_path / "check.cpp", tmp_path / "check"
    src.write_text(CHECK)
    subprocess.run(["g++", "-O2", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover",
                    "-I", str(KERNELS), str(src), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout + run.stderr
