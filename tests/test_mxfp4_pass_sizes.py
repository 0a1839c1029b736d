"""The rule for the pass size of an MXFP4 product, compiled for the host."""
import math
import os
import random
import subprocess

import pytest

from conftest import ROOT


def compiled(folder, name):
    """Lines of numbers in, lines of numbers out, by tests/c/<name>.cpp."""
    exe = folder / name
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-I", os.path.join(ROOT, "salt-core_b200", "csrc"),
                    os.path.join(ROOT, "tests", "c", name + ".cpp"), "-o", str(exe)], check=True)

    def run(sizes):
        out = subprocess.run([str(exe)], input="\n".join(" ".join(map(str, s)) for s in sizes), text=True, check=True, capture_output=True)
        return [tuple(map(float, line.split())) for line in out.stdout.splitlines()]
    return run


@pytest.fixture(scope="module")
def rule(tmp_path_factory):
    return compiled(tmp_path_factory.mktemp("passes"), "mxfp4_pass_sizes")


@pytest.fixture(scope="module")
def split(tmp_path_factory):
    return compiled(tmp_path_factory.mktemp("splits"), "mxfp4_splits")


def spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def test_the_choice_stays_near_the_least_estimate(rule):
    """Fewer and longer passes are taken for a little more time, never for more than 15 % above the least over all sizes: dense and
    grouped, one row tile to hundreds."""
    rng = random.Random(17)
    sizes = [(2134, 1, 4, 19, 148), (2361, 1, 3, 19, 148), (1176, 1, 13, 18, 148), (97, 1, 1, 32, 148), (300, 1, 1, 32, 148)]
    for _ in range(20000):
        sizes.append((spread(rng, 1, 100000), rng.choice([1, 1, 1, 2, 8, 31, 64, 256, 1024]), spread(rng, 1, 400), spread(rng, 1, 512),
                      rng.choice([148, 148, 132])))
    for size, (chosen, estimate, least) in zip(sizes, rule(sizes)):
        assert chosen % 32 == 0 and 32 <= chosen <= 224
        assert estimate <= 1.15 * least, (size, chosen)


def test_a_single_pass_where_it_is_as_good(rule):
    """37 rows of 2112 x 2816 and 4096 of 5120 x 5120: one pass instead of two, the longest instead of more."""
    assert [c for c, _, _ in rule([(37, 1, 17, 11, 148), (4096, 1, 40, 20, 148)])] == [64, 224]


def test_clusters_find_a_place_at_once(split):
    """Of blocks that fill an SM each, an SM count of 148 holds 74 clusters of two, 33 of four and 15 of eight at the same time; a unit
    that waits for a place doubles the call (16 units of 64 chunks: 13.4 us by clusters of eight, 9.4 by four).  Two a place where they
    share an SM."""
    held = {2: 74, 4: 33, 8: 15}
    sizes = [(u, c, h, 148) for u in range(1, 200) for c in (1, 5, 8, 11, 16, 19, 20, 32, 64, 160, 512) for h in (0, 4, 8)]
    for (units, chunks, half, _), (chosen,) in zip(sizes, split(sizes)):
        assert chosen in (1, 2, 4, 8)
        if chosen > 1:
            assert units <= held[chosen] * (2 if -(-chunks // chosen) <= half else 1), (units, chunks, half, chosen)


def test_clusters_where_they_pay(split):
    """One row of 4096 x 4096 by four blocks a unit, 37 rows of 2112 x 2816 by four, 15 units of 64 chunks by eight and 16 by four."""
    assert [int(c) for c, in split([(32, 16, 4, 148), (17, 11, 4, 148), (15, 64, 4, 148), (16, 64, 4, 148), (96, 20, 4, 148)])] == [4, 4, 8, 4, 1]
