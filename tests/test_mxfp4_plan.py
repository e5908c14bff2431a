"""Which kernel variants the MXFP4 dense calls reach (kadan_amd/csrc/mxfp4_plan.hpp, compiled
for the host by tests/cpp/mxfp4_plan_check.cpp), and that the GPU tests' sizes reach them all.
The choice is an estimate of times: a change of it must not drop a variant from the tests."""
import math
import os
import random
import shutil
import subprocess

import pytest

import test_mxfp4_dense_gpu as sizes

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    """plan([call, ..]) -> [variant, ..] on 256 compute units: ("decode", wide, staged, rows of
    16) or ("gemm", tiles, split, sliced)."""
    if not shutil.which("g++"):
        pytest.skip("no g++")
    exe = str(tmp_path_factory.mktemp("plan") / "check")
    subprocess.run(["g++", "-O2", "-std=c++20", "-Wall", "-Werror", "-o", exe,
                    "-I", os.path.join(ROOT, "kadan_amd", "csrc"),
                    os.path.join(HERE, "cpp", "mxfp4_plan_check.cpp")], check=True)

    def ask(calls):
        text = "\n".join(" ".join(map(str, call)) for call in calls)
        out = subprocess.run([exe, "256"], input=text, capture_output=True, text=True, check=True)
        lines = [line.split() for line in out.stdout.splitlines()]
        assert len(lines) == len(calls)
        return [(kind, int(a), int(b), int(c) if kind == "decode" else int(c) > 1)
                for kind, a, b, c, *_ in lines]

    return ask


def cross(path, lists, *flag):
    return [(path, *size, *flag) for size in lists]


TESTED = {
    ("product", 0): sizes.SIZES + sizes.TILES + sizes.WIDE,
    ("product", 1): sizes.SIZES + sizes.TILES_MXFP4 + sizes.WIDE_MXFP4,
    ("gated", 0): sizes.GATED + sizes.GATED_TILES + sizes.GATED_WIDE,
    ("gated", 1): sizes.GATED + sizes.GATED_TILES_KEPT,
    ("backward",): sizes.GATED + sizes.BACKWARD_TILES,
}


@pytest.mark.parametrize("path", list(TESTED))
def test_every_variant_is_reached_by_a_tested_size(plan, path):
    name, flag = path[0], path[1:]
    tested = set(plan(cross(name, TESTED[path], *flag)))
    rng = random.Random(5)

    def spread(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    calls = []
    for _ in range(150000):
        n = spread(1, 40000)
        if name != "product":
            n = 32 * max(1, n // 32)
        calls.append((name, spread(1, 4096), n, 32 * spread(1, 512), *flag))
    found = {}
    for call, variant in zip(calls, plan(calls)):
        found.setdefault(variant, call)
    assert {v[1] for v in found if v[0] == "gemm"} == {1, 2, 3, 4}
    assert not {v: call for v, call in found.items() if v not in tested}


@pytest.mark.parametrize("call,kernel", [
    (("product", 31, 131072, 512, 0), "gemm"), (("product", 17, 65536, 896, 0), "gemm"),
    (("product", 64, 65536, 896, 1), "gemm"), (("product", 31, 131072, 1984, 1), "gemm"),
    (("gated", 17, 65536, 512, 0), "gemm"), (("product", 32, 4096, 512, 0), "decode"),
    (("product", 64, 4096, 896, 1), "decode"), (("gated", 32, 4096, 512, 0), "decode"),
    (("product", 16, 14336, 512, 0), "decode")])
def test_rows_that_every_workgroup_reads_again_are_counted(plan, call, kernel):
    """More than 16 rows never pass through LDS, however short they are: over many workgroups
    their reading outweighs the weights'."""
    variant, = plan([call])
    assert variant[0] == kernel
    if call[1] > 16 and kernel == "decode":
        assert not variant[2]  # (not staged)
