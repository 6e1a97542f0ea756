"""The rule that cuts the dense products into tiles, on the CPU (which counts 256 CUs): the sizes that the GPU tests
run reach every kernel that any size reaches, and every kernel that is built is reached."""
import ctypes
import math
import random

import pytest

from dense_variants import F32, FEW_ROWS, GLU, LINEAR, SHORT, VARIANTS, plans

OK, SHAPE, DTYPE, ARG = 0, 1, 3, 6


def sizes(count, seed):
    rng = random.Random(seed)

    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    for _ in range(count):
        n, k, m = log(1, 1 << 15), log(1, 1 << 15), log(1, 1 << 15)
        if rng.random() < 0.5:
            k, m = (k + 7) // 8 * 8, (m + 7) // 8 * 8
        yield n, k, m


@pytest.mark.parametrize("gated", [LINEAR, GLU])
@pytest.mark.parametrize("dtype", [F32, SHORT])
def test_tested_sizes_reach_every_kernel(built_lib, gated, dtype):
    def of(n, k, m):
        fills = k % 8 == 0 and m % 8 == 0
        return {(*p, fills) for p in plans(gated, dtype, n, k, m)}
    tested = set().union(*[of(*s) for s in VARIANTS[gated, dtype]])
    reached = set().union(*[of(*s) for s in sizes(8000, 7)])
    assert reached <= tested, sorted(reached - tested)


@pytest.mark.parametrize("gated", [LINEAR, GLU])
@pytest.mark.parametrize("dtype", [F32, SHORT])
def test_few_rows_sizes_run_the_few_rows_kernel(built_lib, gated, dtype):
    assert all(("forward", 0, False) in plans(gated, dtype, *s) for s in FEW_ROWS)


# what is built, by product: kinds of tiles, split and unsplit (0: the few-rows / few-tokens kernels, unsplit)
BUILT = {("forward", LINEAR): {F32: {1, 3, 4, 6}, SHORT: {1, 2, 3, 4, 6}},
         ("forward", GLU): {F32: {1, 3, 4}, SHORT: {1, 2, 3, 4}},
         ("input gradient", None): {F32: {1, 3, 4, 5, 6}, SHORT: {1, 2, 3, 4, 6}},
         ("weight gradient", None): {F32: {1, 3}, SHORT: {1, 2, 3}}}


@pytest.mark.parametrize("gated", [LINEAR, GLU])
@pytest.mark.parametrize("dtype", [F32, SHORT])
def test_every_kernel_that_is_built_is_reached(built_lib, gated, dtype):
    """And no other is asked for: a kind that is not built would launch nothing."""
    reached = set().union(*[plans(gated, dtype, *s) for s in VARIANTS[gated, dtype]])
    anywhere = reached.union(*[plans(gated, dtype, *s) for s in sizes(4000, 8)])
    for product in ("forward", "input gradient", "weight gradient"):
        kinds = BUILT.get((product, gated), BUILT.get((product, None)))[dtype]
        built = {(product, kind, split) for kind in kinds for split in (False, True)}
        if product != "input gradient":
            built.add((product, 0, False))
        assert {p for p in reached if p[0] == product} == built
        assert {p for p in anywhere if p[0] == product} == built


def test_plan_refusals(built_lib):
    from bcfft import _lib
    lib, a, b = _lib.load(), ctypes.c_int(), ctypes.c_int()

    def plan(op=0, product=0, n=4, k=64, m=32, dt=2, kind=a, slices=b):
        return lib.bcfft_dense_plan(op, product, n, k, m, dt, kind, slices)
    assert plan() == OK and (a.value, b.value) == (0, 1)
    for bad, status in ((dict(op=4), ARG), (dict(op=-1), ARG), (dict(product=1), ARG), (dict(op=2, product=2), ARG),
                        (dict(product=-1), ARG), (dict(n=0), SHAPE), (dict(k=0), SHAPE), (dict(m=1 << 21), SHAPE),
                        (dict(dt=9), DTYPE), (dict(kind=None), ARG), (dict(slices=None), ARG)):
        assert plan(**bad) == status, bad
