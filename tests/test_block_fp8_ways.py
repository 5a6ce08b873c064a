"""Which kernels the sizes of the GPU tests reach: hdmoe_block_plan_get tells, without a device. A constant of the cost model that moves is no reason for
a way to run to go untested."""
import ctypes
import math
import random

import pytest

from comfyui_amd import _lib as L
from tests import test_gpu_block_fp8 as first
from tests import test_gpu_block_fp8_ways as second


def plan(gate_up, a_dtype, rows, E, K, N):
    a = L.BlockArgs()
    a.a_dtype, a.out_dtype = a_dtype, L.W_BF16
    if E:
        a.E, a.rows, a.K, a.N = E, rows, K, N
    else:
        a.rows_static, a.K_static, a.N_static = rows, K, N
    p = L.BlockPlan()
    L.check(L.lib.hdmoe_block_plan_get(ctypes.byref(a), gate_up, ctypes.byref(p)))
    return p


def way(p):
    return ("few rows", "low tiles", "high tiles")[p.kernel], p.tile_rows, p.strips, p.cast_inside, p.stages


def covered(gate_up, grouped):
    """(way, K) of every size in the lists."""
    old, new = (first.EVERY_GATE_UP, second.GATE_UP) if gate_up else (first.EVERY, second.LINEAR)
    sizes = [(rows, E, K, N) for rows, E, K, N in old] + [(sum(s), len(s) if many else 0, K, N) for s, many, K, N in new]
    return {(way(plan(gate_up, a, rows, E, K, N)), K) for rows, E, K, N in sizes if (E > 0) == grouped for a in (L.W_BF16, L.W_E4M3FN)}


def sample(rng, largest_k):
    spread = lambda lo, hi: int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))  # noqa: E731
    return spread(1, 20000), 16 * spread(1, largest_k // 16), 16 * spread(1, 512)


@pytest.mark.parametrize("gate_up", [0, 1])
@pytest.mark.parametrize("grouped", [False, True])
def test_every_way_to_run_is_tested(gate_up, grouped):
    rng, have, reached = random.Random(7), {w for w, _ in covered(gate_up, grouped)}, {}
    for _ in range(40000):
        rows, K, N = sample(rng, 16384)
        E = rng.choice((1, 2, 3, 4, 6, 8, 16, 32)) if grouped else 0
        a = rng.choice((L.W_BF16, L.W_E4M3FN))
        reached.setdefault(way(plan(gate_up, a, rows, E, K, N)), (a, rows, E, K, N))
    assert not {w: at for w, at in reached.items() if w not in have}


@pytest.mark.parametrize("gate_up", [0, 1])
@pytest.mark.parametrize("grouped", [False, True])
def test_tiles_of_a_single_block_of_k_are_tested(gate_up, grouped):
    """K up to 128, where the first K step is the last one too: in every form of the tile kernels that takes it."""
    rng, have, reached = random.Random(8), {w for w, K in covered(gate_up, grouped) if K <= 128}, {}
    for _ in range(40000):
        rows, K, N = sample(rng, 128)
        E = rng.choice((1, 3, 4, 8)) if grouped else 0
        w = way(plan(gate_up, L.W_E4M3FN, rows, E, K, N))
        if w[0] != "few rows":
            reached.setdefault(w, (rows, E, K, N))
    assert reached and not {w: at for w, at in reached.items() if w not in have}


def test_refusals():
    a, p = L.BlockArgs(), L.BlockPlan()
    f = L.lib.hdmoe_block_plan_get
    a.a_dtype = L.W_BF16
    assert f(None, 0, ctypes.byref(p)) == L.E_NULL and f(ctypes.byref(a), 0, None) == L.E_NULL
    assert f(ctypes.byref(a), 0, ctypes.byref(p)) == L.E_SHAPE                  # no rows
    a.E, a.rows, a.K, a.N = 2, 4, 128, 24
    assert f(ctypes.byref(a), 0, ctypes.byref(p)) == L.E_SHAPE
    a.N, a.E = 32, 33
    assert f(ctypes.byref(a), 0, ctypes.byref(p)) == L.E_SHAPE
    a.E, a.rows_static, a.K_static, a.N_static = 32, 4, 100, 128
    assert f(ctypes.byref(a), 0, ctypes.byref(p)) == L.E_SHAPE
    a.K_static = 112
    assert f(ctypes.byref(a), 0, ctypes.byref(p)) == 0 and p.tile_rows >= 16


def test_a_block_fits_its_cu():
    rng = random.Random(9)
    for _ in range(5000):
        rows, K, N = sample(rng, 16384)
        p = plan(rng.choice((0, 1)), rng.choice((L.W_BF16, L.W_E4M3FN)), rows, rng.choice((0, 1, 4, 8)), K, N)
        assert 0 < p.lds_bytes <= 163840


def test_blocks_fit_their_cu_together():
    """As many as the choice counts on: rings, and the rows that a block casts for itself, in 160 KiB."""
    rng, casting = random.Random(9), 0
    for _ in range(20000):
        rows, K, N = sample(rng, 16384)
        p = plan(rng.choice((0, 1)), rng.choice((L.W_BF16, L.W_E4M3FN)), rows, rng.choice((0, 1, 4, 8)), K, N)
        assert p.blocks_per_cu * p.lds_bytes <= 163840, (rows, K, N)
        casting += p.cast_inside
    assert casting > 1000
    two, one = plan(1, L.W_BF16, 2, 4, 2560, 6912), plan(1, L.W_BF16, 1, 4, 2560, 6912)
    assert (two.cast_inside, two.lds_bytes, two.blocks_per_cu) == (1, 87296, 1) and (one.lds_bytes, one.blocks_per_cu) == (80640, 2)


@pytest.mark.parametrize("a_dtype", [L.W_BF16, L.W_F16, L.W_E4M3FN])
def test_gate_up_has_exact_products_where_the_header_says(a_dtype):
    """Up to 64 rows in each group, with fp16 activations, and when asked. (A Linear has none, and no flag.)"""
    rng, p = random.Random(10), L.BlockPlan()
    few = many = 0
    for _ in range(4000):
        rows, K, N = sample(rng, 8192)
        a = L.BlockArgs()
        a.a_dtype, a.out_dtype = a_dtype, L.W_BF16
        form = rng.choice(("dense", "experts", "layer"))
        if form != "dense":
            a.E, a.rows, a.K, a.N = rng.choice((1, 2, 4, 32)), rows, K, N
        if form != "experts":
            a.rows_static, a.K_static, a.N_static = rows if form == "dense" else -(-rows // 2), K, 16 * rng.randint(1, 400)
        for exact in (0, 1):
            for fixed in (0, 1):
                a.exact, a.fixed_k_cut = exact, fixed
                L.check(L.lib.hdmoe_block_plan_get(ctypes.byref(a), 1, ctypes.byref(p)))
                if exact or a_dtype == L.W_F16 or (rows <= 64 and not fixed):
                    assert p.exact, (form, rows, K, N)
                    few += 1
                elif fixed:
                    assert not p.exact    # one kind at any size
                else:
                    many += not p.exact
                assert not (p.exact and p.kernel == 2)
        a.exact = a.fixed_k_cut = 0
        L.check(L.lib.hdmoe_block_plan_get(ctypes.byref(a), 0, ctypes.byref(p)))
        assert not p.exact
    assert few > 100 and (many > 100 or a_dtype == L.W_F16)
