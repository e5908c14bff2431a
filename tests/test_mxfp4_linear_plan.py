"""Which kernel variants the MXFP4 products with an epilogue and the experts' products reach
(kadan_amd/csrc/mxfp4_plan.hpp, compiled for the host by tests/cpp/mxfp4_linear_plan_check.cpp),
that the GPU tests' sizes reach them all, and that a launch has workgroups for every tile."""
import math
import os
import random
import shutil
import subprocess

import pytest

import test_mxfp4_linear_gpu as sizes

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    """plan([call, ..]) -> [line, ..] on 256 compute units."""
    if not shutil.which("g++"):
        pytest.skip("no g++")
    exe = str(tmp_path_factory.mktemp("plan") / "check")
    subprocess.run(["g++", "-O2", "-std=c++20", "-Wall", "-Werror", "-o", exe,
                    "-I", os.path.join(ROOT, "kadan_amd", "csrc"),
                    os.path.join(HERE, "cpp", "mxfp4_linear_plan_check.cpp")], check=True)

    def ask(calls):
        text = "\n".join(" ".join(str(int(v)) if i else v for i, v in enumerate(call))
                         for call in calls)
        out = subprocess.run([exe, "256"], input=text, capture_output=True, text=True, check=True)
        lines = out.stdout.splitlines()
        assert len(lines) == len(calls)
        return lines

    return ask


def experts(path, cases, *flags):
    return [(path, m, e, n, k, *flags) for m, e, n, k, *_ in cases]


TESTED = {
    ("linear",): [("linear", *s) for s in sizes.LINEAR],
    ("back",): [("back", *s) for s in sizes.BACKWARD],
    ("experts", False, False): experts("experts", sizes.EXPERTS, False, False),
    ("experts", True, False): experts("experts", sizes.GATED, True, False),
    ("experts", True, True): experts("experts", sizes.GATED, True, True),
    ("experts_back", False): experts("experts_back", sizes.EXPERTS_BACKWARD, False),
    ("experts_back", True): experts("experts_back", sizes.GATED_BACKWARD, True),
}


@pytest.mark.parametrize("path", list(TESTED))
def test_every_variant_is_reached_by_a_tested_size(plan, path):
    name, flags = path[0], path[1:]
    tested = set(plan(TESTED[path]))
    rng = random.Random(11)

    def spread(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    calls = []
    for _ in range(60000):
        n, k = spread(1, 40000), 32 * spread(1, 512)
        if name == "back":
            n = 8 * max(1, n // 8)
        if name.startswith("experts"):
            calls.append((name, spread(1, 20000), spread(1, 256), 32 * max(1, n // 32), k, *flags))
        else:
            calls.append((name, spread(1, 4096), n, k))
    found = {}
    for call, variant in zip(calls, plan(calls)):
        found.setdefault(variant, call)
    assert not {v: call for v, call in found.items() if v not in tested}


@pytest.mark.parametrize("call,kernel", [
    (("experts", 4, 32, 2880, 2880, 1, 0), "experts decode 0"),      # a token gated
    (("experts", 8, 32, 2880, 2880, 1, 0), "experts gemm 1 0"),      # two
    (("experts", 8, 32, 2880, 2880, 0, 0), "experts decode 1"),      # their down projection
    (("experts", 16, 32, 2880, 2880, 0, 0), "experts gemm 1 0"),
    (("experts", 64, 8, 4096, 5632, 0, 0), "experts gemm 1 0"),      # eight rows an expert
    (("experts", 4, 32, 2880, 2880, 1, 1), "experts gemm 1 0"),      # kept: for a backward pass
    (("experts", 32768, 128, 768, 2048, 1, 1), "experts gemm 2 0"),
    (("experts", 594, 6, 416, 5920, 0, 0), "experts gemm 2 1"),      # few tiles, a long K
    (("experts_back", 4, 28, 3392, 1024, 1), "experts gemm 1 1"),
    (("experts_back", 594, 6, 5920, 416, 1), "experts gemm 2 1")])
def test_kernels_of_measured_sizes(plan, call, kernel):
    assert plan([call]) == [kernel]


def test_a_launch_has_workgroups_for_every_tile(plan):
    """However the rows are spread over the experts."""
    rng = random.Random(3)
    asked, needed = [], []
    for _ in range(4000):
        count, rows = rng.choice([1, 2, 3, 8, 100, 256]), rng.choice([16, 32, 64])
        kind = rng.randrange(4)
        if kind == 0:  # as many last tiles of a row as can be
            each = [rows * rng.randrange(3) + 1 for _ in range(count)]
        elif kind == 1:
            each = [0] * count
            each[rng.randrange(count)] = rng.randrange(1, 3000)
        else:
            each = [int(rng.expovariate(1 / 60) * rng.random()) for _ in range(count)]
        if not sum(each):
            each[0] = 1
        asked.append(("tiles", sum(each), count, rows))
        needed.append(sum(-(-c // rows) for c in each))
    most = [int(line) for line in plan(asked)]
    assert all(a >= b for a, b in zip(most, needed))
    assert any(a == b for a, b in zip(most, needed))
