"""What the cases of test_gpu_paged_tree_long.py reach, on the CPU: the plan that the
launcher makes of each, from the same header compiled for the host."""
import pathlib
import subprocess

import pytest

pytest.importorskip("torch")

import test_gpu_paged_tree_long as long  # noqa: E402

KERNELS = pathlib.Path(__file__).resolve().parent.parent / "cu-jev_amd" / "csrc" / "kernels"
PLAN = r"""
#include "paged_index.h"
#include <cstdio>
#include <cstdlib>
int main(int argc, char **argv) { /* Hq Hkv {rows keys}... */
    const int Hkv = atoi(argv[2]), G = atoi(argv[1]) / Hkv, B = (argc - 3) / 2;
    int N = 2, max_q = 0, max_kv = 0; /* 2 rows of no sequence */
    for (int b = 0; b < B; b++) {
        const int q = atoi(argv[3 + 2 * b]), k = atoi(argv[4 + 2 * b]);
        N += q, max_q = pg_max(max_q, q), max_kv = pg_max(max_kv, k);
    }
    const pg_plan p = pg_make_mid_plan(N, B, max_q, max_kv, G, Hkv);
    unsigned T = 0, U = 0;
    for (int b = 0, q0 = 0; b < B; b++) {
        const int q = atoi(argv[3 + 2 * b]);
        const pg_seq s = pg_clean_seq(q0, q0 + q, atoi(argv[4 + 2 * b]), N, max_q, max_kv);
        T += pg_units(s, G, PG_MID) * pg_longest(s, G, PG_LINE, 0, 0), U += pg_units(s, G, PG_MID);
        q0 += q;
    }
    const int over = pg_mid_over(p, T);
    printf("%d %d %d %d\n", pg_is_mid(N, B, max_q, max_kv, G, Hkv), max_q * G, over,
           pg_mid_share(p, T + U * over));
}
"""
BUFFERS = 4  # the most tiles that LDS holds at a time


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    at = tmp_path_factory.mktemp("plan")
    (at / "plan.cpp").write_text(PLAN)
    subprocess.run(["g++", "-std=c++17", "-I", str(KERNELS), str(at / "plan.cpp"), "-o",
                    str(at / "plan")], check=True)

    def of(Hq, Hkv, lens):
        args = [Hq, Hkv, *(x for pair in lens for x in pair)]
        out = subprocess.run([str(at / "plan"), *map(str, args)], capture_output=True, text=True,
                             check=True).stdout
        mid, rows, over, size = map(int, out.split())
        return bool(mid), rows, over, size
    return of


def test_pieces_are_long(plan):
    for case in long.LONG + long.RISING:
        mid, _, over, size = plan(*case)
        assert mid and over > 0 and size > 2 * BUFFERS, case
    assert max(plan(*case)[3] for case in long.LONG) > 64 + 6


def test_both_forms_are_reached(plan):
    rows = [plan(*case)[1] for case in long.LONG + long.RISING]
    assert min(rows) <= 32 < max(rows) <= 64
    for case in long.SMALL:
        mid, rows, _, _ = plan(*case)
        assert mid and 16 < rows <= 32, case
