"""Which tiles the workgroups of an experts' launch take and where their partial sums lie
(kadan_amd/csrc/mxfp4_plan.hpp's arithmetic, which the kernel uses, replayed on the host by
tests/cpp/experts_tiles_check.cpp)."""
import os
import random
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)


@pytest.fixture(scope="module")
def replay(tmp_path_factory):
    """replay([(path, m, experts, n, k, offsets), ..]) -> [(slices, partial tiles, reached, asked,
    wrong) or None, ..] on 256 compute units."""
    if not shutil.which("g++"):
        pytest.skip("no g++")
    exe = str(tmp_path_factory.mktemp("tiles") / "check")
    subprocess.run(["g++", "-O2", "-std=c++20", "-Wall", "-Werror", "-o", exe,
                    "-I", os.path.join(ROOT, "kadan_amd", "csrc"),
                    os.path.join(HERE, "cpp", "experts_tiles_check.cpp")], check=True)

    def ask(calls):
        text = "\n".join(" ".join(map(str, (*call[:5], *call[5]))) for call in calls)
        out = subprocess.run([exe, "256"], input=text, capture_output=True, text=True)
        assert out.returncode == 0, out.stdout[-200:]
        lines = out.stdout.splitlines()
        assert len(lines) == len(calls)
        return [None if line == "decode" else tuple(map(int, line.split())) for line in lines]

    return ask


# calls whose tiles are few and whose K is long, so that it is split: m, experts, n, k
SLICED = [("linear", 594, 6, 416, 5920), ("linear", 300, 16, 128, 8192),
          ("gated", 330, 3, 288, 3968), ("gated", 27, 7, 384, 2912),
          ("back", 330, 3, 3960, 288), ("back", 27, 7, 2904, 416),
          ("gated_back", 4, 28, 3392, 1024), ("gated_back", 594, 6, 5920, 416),
          ("gated_back", 40, 8, 5888, 1120)]
WHOLE = [("linear", 2048, 32, 2880, 2880), ("gated", 2048, 32, 2880, 2880),
         ("back", 700, 32, 2880, 2880), ("gated_back", 4096, 128, 768, 2048)]


def spread(rng, m, experts):
    """Offsets of m rows over the experts, some popular, some with none."""
    kind = rng.randrange(4)
    if kind == 0:
        of = [rng.randrange(experts)] * m
    elif kind == 1:
        of = [i % experts for i in range(m)]
    else:
        odds = [rng.random() ** 4 for _ in range(experts)]
        of = rng.choices(range(experts), odds, k=m)
    counts = [of.count(e) for e in range(experts)]
    return [sum(counts[:e]) for e in range(experts + 1)]


@pytest.mark.parametrize("call", SLICED + WHOLE)
def test_every_tile_and_slice_is_one_workgroups(replay, call):
    rng = random.Random(5)
    calls = [(*call, spread(rng, call[1], call[2])) for _ in range(30)]
    m, experts = call[1:3]
    calls.append((*call, [0] + [m // 2] * (experts - 1) + [m - 1]))  # rows of no expert
    for result in replay(calls):
        slices, partials, reached, asked, wrong = result
        assert asked and not wrong
        assert (slices > 1) == (call in SLICED) and reached <= partials


@pytest.mark.parametrize("call", SLICED)
def test_offsets_that_decrease_reach_no_partial_sums_but_the_workspaces(replay, call):
    """Such offsets may make more tiles than any spread of the rows does."""
    _, m, experts, _, _ = call
    rng = random.Random(6)
    bad = [[0, m] * experts, [m, 0] * experts, [0, m, m // 4] + [m] * experts]
    for _ in range(40):
        bad.append([rng.choice([-5, 0, m, m + 3, rng.randrange(m + 1)])
                    for _ in range(experts + 1)])
    for result in replay([(*call, offsets[:experts + 1]) for offsets in bad]):
        slices, partials, reached, _, _ = result
        assert slices > 1 and reached <= partials
