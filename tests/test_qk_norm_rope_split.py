"""How a head norm's warps are divided between q and k: by the units of work either has,
so that no warp has many times another's. On the host, from the kernels' own header."""

from __future__ import annotations

import subprocess

import pytest

from tests.conftest import ROOT

MAIN = """
#include <cstdio>
#include "gdr_qk_norm_rope.cuh"
int main() {
    long long tokens; int hq, hk, per, blocks;
    while (std::scanf("%lld %d %d %d %d", &tokens, &hq, &hk, &per, &blocks) == 5)
        std::printf("%u\\n", gdr::norm_rope_q_warps(8LL * blocks, hq, hk, per));
}
"""


@pytest.fixture(scope="module")
def q_warps(tmp_path_factory):
    d = tmp_path_factory.mktemp("split")
    (d / "main.cpp").write_text(MAIN)
    subprocess.run(["g++", "-std=c++17", "-I", str(ROOT / "bunsen_b200" / "csrc"),
                    "-I", "/usr/local/cuda/include", "-o", str(d / "main"), str(d / "main.cpp")],
                   check=True)

    def call(cases):
        text = "\n".join(" ".join(map(str, c)) for c in cases)
        out = subprocess.run([str(d / "main")], input=text, capture_output=True, text=True,
                             check=True)
        return [int(x) for x in out.stdout.split()]

    return call


def test_warps_follow_the_units(q_warps):
    """A unit is `per` heads of one token, rounded up for each token: the most units a warp
    has is the mean, times what an even division of whole warps allows, and one."""
    cases = [(tokens, hq, hk, per, blocks)
             for tokens in (1, 100, 32768) for hq, hk in ((16, 16), (32, 1), (31, 2), (28, 4), (1, 32),
                                                          (16, 4), (1, 1), (128, 1), (5, 3))
             for per in (1, 2, 4, 8, 16) for blocks in (1, 7, 296, 2368)]
    for (tokens, hq, hk, per, blocks), q in zip(cases, q_warps(cases)):
        warps, units = 8 * blocks, [-(-h // per) * tokens for h in (hq, hk)]
        assert 1 <= q <= warps - 1
        # A part's share of the warps loses less than one of them to rounding.
        for mine, n in zip(units, (q, warps - q)):
            fair = warps * mine / sum(units)
            assert n > fair - 1 and -(-mine // n) <= mine / max(fair - 1, 1) + 1
