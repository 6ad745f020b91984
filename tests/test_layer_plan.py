"""CPU checks of the rule that gives the few-token layer and the mixture their kernels
(csrc/layer_plan.hpp, plain arithmetic, run by a host program): sizes of the GPU tests reach the
forms that they are there for."""
import os
import shutil
import subprocess

import pytest

import layer_sizes as sizes

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sushiblas_amd", "csrc")

PROGRAM = r"""
#include <stdio.h>
#include "layer_plan.hpp"

int main()
{
    char what;
    int a[6];
    while (scanf(" %c %d %d %d %d %d %d", &what, a, a + 1, a + 2, a + 3, a + 4, a + 5) == 7)
        if (what == 'l') {
            const sbx::Mx4LinearPlan p = sbx::mx4_linear_plan(a[0], a[1] != 0, a[2], a[3], a[4]);
            printf("%d %d %d %d %d %d\n", (int)p.form, p.tokens, p.tiles, p.blocks, p.waves, p.ahead);
        } else {
            const sbx::Mx4MoePlan p = sbx::mx4_moe_plan(a[0], a[1], a[2], a[3], a[4], a[5]);
            printf("%d %d %d %d %d %d %d %u %u %u\n", p.one, p.few, p.each, p.up, p.down, p.up_rows, p.down_rows,
                   p.chunks, p.up_tiles, p.down_tiles);
        }
    return 0;
}
"""


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no host C++ compiler")
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(PROGRAM)
    subprocess.run([cxx, "-std=c++17", "-O1", f"-I{CSRC}", "-o", str(d / "plan"), str(d / "plan.cpp")], check=True)

    def ask(what, cases):
        text = "\n".join(what + " " + " ".join(map(str, c)) for c in cases)
        res = subprocess.run([str(d / "plan")], input=text, stdout=subprocess.PIPE, text=True, check=True, timeout=60)
        return [tuple(map(int, line.split())) for line in res.stdout.splitlines()]
    return ask


def linear(plans, cases):
    return plans("l", [(p, int(mx8), m, n, k, 0) for p, mx8, m, n, k in cases])


def test_groups_under_way(plans):
    for cases, ahead in ((sizes.TWO_AHEAD, 2), (sizes.ONE_AHEAD, 1)):
        for mx8 in (False, True):
            got = linear(plans, [(1, mx8, *c) for c in cases])
            assert [g[0] for g in got] == [0] * len(cases) and [g[5] for g in got] == [ahead] * len(cases)
            assert [g[3:5] for g in got] == list(cases.values())
    assert all(g[5] == 1 for p in (2, 3) for g in linear(plans, [(p, False, *c) for c in sizes.TWO_AHEAD]))


def test_tiles(plans):
    assert [g[:3] for g in linear(plans, [(p, False, *c) for p, *c in sizes.TILES])] == [(0, *t) for t in sizes.TILES.values()]


def test_tall_weights(plans):
    assert all(g[0] == 1 for g in linear(plans, [(p, False, *c) for p, *c in sizes.TALL]))
    assert all(g[0] == 0 for g in linear(plans, [(1, False, *c) for _, *c in sizes.TALL]))


def test_few_terms(plans):
    got = linear(plans, [(1, False, 5, 40, 7), (1, True, 5, 40, 7), (3, False, 5, 40, 8), (2, True, 5, 40, 0)])
    assert [g[0] for g in got] == [2, 0, 0, 2]


def test_mixtures(plans):
    for pieces in (1, 2, 3):
        got = plans("m", [(pieces, *c) for c in sizes.ROWS])
        assert [(bool(g[5]), bool(g[6]), g[4]) for g in got] == list(sizes.ROWS.values())
        got = plans("m", [(pieces, t, 64, 64, e, k) for t, e, k in sizes.CHOICES])
        assert [g[2] for g in got] == list(sizes.CHOICES.values())
        assert [bool(g[0]) for g in got] == [t == 1 for t, _, _ in sizes.CHOICES]


def test_tiles_are_enough(plans):
    """However the choices fall: an expert's tiles are its tokens over their size, rounded up."""
    cases = [(p, t, 64, 64, e, k) for p in (1, 3) for t in (2, 7, 8, 9, 40, 64, 65, 200, 256) for e, k in
             ((1, 1), (3, 2), (8, 2), (16, 16), (64, 8), (512, 16))]
    for (_, t, _, _, e, k), g in zip(cases, plans("m", cases)):
        chunk = min(t, 64)
        for size, tiles in ((g[3], g[8]), (g[4], g[9])):
            # the most: as many experts as can have a token beyond whole tiles
            worst = max(sum(-(-n // size) for n in counts) for counts in _spreads(chunk, e, k, size))
            assert worst <= tiles <= chunk * k
        assert g[7] == -(-t // 64)


def _spreads(tokens, experts, topk, size):
    """Counts of tokens an expert that make many tiles: evenly, all on a few, one beyond whole tiles each."""
    total = tokens * topk
    yield [total // experts + (i < total % experts) for i in range(experts)]
    yield [tokens] * topk
    counts, left = [0] * experts, total
    for i in range(experts):
        counts[i] = min(1, left)
        left -= counts[i]
    while left > 0:
        before = left
        for i in range(experts):
            add = min(size, left, tokens - counts[i])
            counts[i] += add
            left -= add
        if left == before:
            break
    yield counts
