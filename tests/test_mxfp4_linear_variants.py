"""That the sizes of test_mxfp4_linear_variants_gpu.py reach every kernel variant that a dense MXFP4
product with an epilogue, or its backward pass, can take."""
import math
import random

import pytest

import test_mxfp4_linear_variants_gpu as sizes
from test_mxfp4_linear_plan import plan  # noqa: F401  (a fixture)


@pytest.mark.parametrize("name,tested,sliced", [
    ("linear", sizes.LINEAR, sizes.SLICED), ("back", sizes.BACKWARD, sizes.SLICED_BACKWARD)])
def test_every_variant_is_among_the_sizes(plan, name, tested, sliced):  # noqa: F811
    rng = random.Random(12)

    def spread(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    calls = []
    for _ in range(60000):
        m, n, k = spread(1, 4096), spread(1, 20000), 32 * spread(1, 512)
        calls.append((name, m, 8 * max(1, n // 8) if name == "back" else n, k))
    found = set(plan(calls))
    reached = plan([(name, *s) for s in tested])
    assert found <= set(reached)
    assert all(line.startswith("gemm") and line.endswith(" 1")
               for line in plan([(name, *s) for s in sliced]))
    assert {line for line in found if line.startswith("gemm") and line.endswith(" 1")} <= set(
        plan([(name, *s) for s in sliced]))
