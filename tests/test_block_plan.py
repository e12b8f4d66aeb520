"""Which tiles block-scaled products run on (``csrc/block_plan.h``, compiled here as
plain C++): the sizes of ``test_gpu_block_tiles.py`` reach every form that any call
reaches, so that a change of the cost model cannot leave a kernel untested."""
import ctypes
import math
import random
import subprocess

import pytest

from tests.test_gpu_block_tiles import GATED, LAYER, LINEAR
from tokenfactory_amd.build import CSRC

CUS = 256
SHIM = """
#include "block_plan.h"
extern "C" void plan(int64_t m, int64_t n, int64_t k, int gated, int64_t cus, int64_t* out) {
  const int64_t kb = tfa::ceil_div(k, 128);
  const tfa::BlockPlan p = gated ? tfa::plan_gated(m, n, kb, cus)
                                 : tfa::plan_linear(m, n, 1, kb, false, cus);
  out[0] = p.shape.mt; out[1] = p.shape.wn; out[2] = p.full; out[3] = p.splits;
  out[4] = p.fused; out[5] = p.part; out[6] = gated && tfa::wide_gated(m);
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "shim.cpp").write_text(SHIM)
    lib = d / "shim.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", f"-I{CSRC}", "-o", str(lib),
                    str(d / "shim.cpp")], check=True)
    fn = ctypes.CDLL(str(lib)).plan
    fn.argtypes = [ctypes.c_int64] * 3 + [ctypes.c_int, ctypes.c_int64, ctypes.c_void_p]
    fn.restype = None

    def run(m, n, k, gated=False, cus=CUS):
        out = (ctypes.c_int64 * 7)()
        fn(m, n, k, gated, cus, out)
        return tuple(out)
    return run


def form(plan, m, n, k, gated=False):
    """The kernel (shape, fused, wide) and which of its workgroups there are: whole
    tiles, partials or both."""
    mt, wn, full, splits, fused, part, wide = plan(m, n, k, gated)
    kind = "fused" if fused else "whole" if not part else "both" if full else "partials"
    return gated, mt, wn, kind, bool(wide)


def covered(plan):
    return {form(plan, m, n, k) for m, n, k in LINEAR} | {
        form(plan, m, inter, hidden, True) for m, hidden, inter in GATED + LAYER}


def test_the_gpu_tests_reach_every_form(plan):
    rng, seen = random.Random(1), covered(plan)
    log = lambda a, b: int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))
    missing = {}
    for _ in range(150000):
        gated, m = rng.random() < 0.5, log(17, 16384)
        n, k = 16 * log(1, 2048), 16 * log(1, 2048)
        f = form(plan, m, n, k, gated)
        if f not in seen:
            missing.setdefault(f, (m, n, k))
    assert not missing


def test_every_shape_is_chosen(plan):
    """No shape of the tables is there for nothing."""
    seen = covered(plan)
    assert {f[1:3] for f in seen if not f[0]} == {(1, 2), (2, 2), (4, 2), (6, 2), (4, 4), (6, 4),
                                                  (8, 4)}
    assert {f[1:3] for f in seen if f[3] == "fused"} == {(2, 4), (4, 4), (6, 4), (8, 4)}
    assert {f[1:4] for f in seen if f[4]} == {(1, 2, "partials"), (2, 2, "partials"),
                                              (2, 4, "fused")}


@pytest.mark.parametrize("cus", [1, 64, 256, 304])
def test_plans_are_launches(plan, cus):
    """Whole and split tiles are all tiles, every split has two slices of K, and the
    partials have room in the workspace."""
    rng = random.Random(2)
    for _ in range(3000):
        gated, m = rng.random() < 0.5, rng.randint(17, 9000)
        n, k = 16 * rng.randint(1, 1200), 16 * rng.randint(1, 1200)
        mt, wn, full, splits, fused, part, wide = plan(m, n, k, gated, cus)
        bm, bn = 32 * mt, 128 if fused else 64 * wn
        tiles = -(-m // bm) * -(-n // bn) * (2 if gated and not fused else 1)
        assert 0 <= full <= tiles and 1 <= splits <= 16
        assert part == (0 if fused else (tiles - full) * splits * bm * bn)
        assert splits == 1 or (-(-k // 128)) // splits >= 2
        assert not wide or mt <= 2
        if gated and not fused:
            assert full == 0
        elif splits == 1:
            assert full == tiles


def test_partials_that_no_launch_finishes_are_not_planned(plan):
    """A launch has 2^32 threads, gated_finish_kernel 32 of them per row and block."""
    rng = random.Random(3)
    log = lambda a, b: int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))
    for m, n, k in [(8460377, 18144, 269168), (1 << 20, 20480, 65536)] + [
            (log(1 << 19, 1 << 24), 16 * log(64, 4096), 16 * log(1024, 1 << 16))
            for _ in range(20000)]:
        fused = plan(m, n, k, True)[4]
        assert fused or m * -(-n // 128) * 32 < 1 << 32, (m, n, k)
