"""Gradients of the balance loss where dp, what a token's scores enter the loss with, is the same for all of its experts: sum_e p[e] = 1, so there is nothing
to move, and the gradient is 0, not a rounding of it."""
import pytest
import torch

from tests import test_gpu_router

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]
SIZES = [(1, 1, 264, 2, 2, False), (1, 6, 2560, 4, 4, False), (5, 1, 128, 1, 1, False), (2, 17, 520, 16, 16, True), (3, 700, 2048, 8, 8, True), (1, 20000, 328, 3, 3, False)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("S,L,D,E,k,masked", SIZES)
def test_every_expert_chosen_by_every_token(dtype, S, L, D, E, k, masked):
    p = test_gpu_router.problem(S * 7 + L, S, L, D, E, k, dtype, masked, weights=False)
    _, _, scores, dx, dw = test_gpu_router.check(p)
    assert not dx.any() and not dw.any() and scores.any()
    p["dweight"] = torch.full((S * L, k), 0.625, device="cuda", dtype=dtype)        # the same for all of them as well
    _, _, _, dx, dw = test_gpu_router.check(p)
    assert not dx.any() and not dw.any()


@pytest.mark.parametrize("dtype", TYPES)
def test_what_all_scores_have_in_common_changes_nothing(dtype):
    """64 more on every score's gradient: multiples of a half, so that their differences are the same to the bit."""
    p = test_gpu_router.problem(3, 2, 90, 640, 6, 6, dtype)
    p["dloss"] = torch.zeros((), device="cuda")
    small = torch.randint(0, 100, p["dweight"].shape, generator=test_gpu_router.gen(4), device="cuda").to(dtype) / 2
    p["dweight"] = small
    want = test_gpu_router.check(p)
    p["dweight"] = small + 64
    got = test_gpu_router.call(p)
    assert want[3].any() and torch.equal(got[3], want[3]) and torch.equal(got[4], want[4])
