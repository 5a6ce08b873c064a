"""Sizes of adapters where a drawn index may name none at all, with one that does: whatever is multiplied at these widths and ranks is compared with 64 bits."""
import pytest
import torch

from tests.test_gpu_adapters import check, problem

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]


def used(requests, n, seed):
    """An index in which the first request has an adapter, and others may."""
    index = torch.randint(-1, n, (requests,), generator=torch.Generator().manual_seed(seed))
    index[0] = seed % n
    return index


def check_used(requests, per, K, N, n, R, dtype):
    p = problem(K + N + R, requests, per, K, N, n, R, dtype, used(requests, n, K + N + R))
    assert (p["index"] >= 0).any()
    out = check(p)
    assert not torch.equal(out, p["base"])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("requests,per,K,N,n,R", [
    (1, 1, 64, 64, 1, 8), (1, 1, 8, 8, 1, 1), (1, 1, 2560, 6912, 4, 16), (1, 3, 8, 8, 2, 1), (2, 1, 100, 36, 3, 64), (1, 2, 264, 520, 2, 40), (1, 130, 1, 1, 1, 1),
    (1, 600, 9, 2560, 2, 3), (2, 64, 640, 1088, 3, 64), (2, 65, 512, 256, 2, 72), (2, 300, 328, 136, 2, 136), (1, 511, 96, 640, 1, 256), (2, 4096, 264, 520, 2, 33)])
def test_sizes(dtype, requests, per, K, N, n, R):
    check_used(requests, per, K, N, n, R, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K,N", [(120, 128), (129, 255), (136, 1160), (1025, 511), (2048, 640)])
@pytest.mark.parametrize("requests,per,n,R", [(2, 300, 2, 40), (1, 900, 1, 88), (1, 600, 1, 256), (1, 40, 5, 104), (3, 50, 2, 72)])
def test_columns_that_end_inside_a_wave(dtype, K, N, requests, per, n, R):
    check_used(requests, per, K, N, n, R, dtype)
