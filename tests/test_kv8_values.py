"""Attention over the 8-bit KV cache: what a row's result may depend on, and how many bits it keeps."""
import pytest
import torch

from tests.kv8_bounds import attend, check
from tests.kv8_util import random_ref

BF, HF = torch.bfloat16, torch.float16


def _q(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


# tokens, query heads of one key head: 8, 16 and more rows
ROWS = [(4, 2, 64), (2, 8, 256), (4, 4, 128), (40, 2, 64), (24, 8, 256)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("T,H,D", ROWS)
@pytest.mark.parametrize("louder", [12, 24, 45, 100])
def test_loud_values_behind_the_mask(require_gpu, T, H, D, dtype, louder):
    """The last block's V scale is 2^louder of the others': tokens that do not see it keep all their bits, those that do are as loud."""
    n, block = 16 * 21, 16
    ref = random_ref(1, 1, 1, D, n, block, louder)
    ref.vs[0, 0, 0, -1] = 2.0 ** (louder - 9)
    q = _q((1, T, H, D), dtype, 3)
    lens = [n - 16 + T // 2] if T <= 16 else [n]  # the last block begins between the tokens
    got = ref.to_cache(lens).attend(0, q.cuda())
    want, tol = attend(ref, 0, q, lens)
    early = lens[0] - T + torch.arange(T) + 1 <= n - 16
    assert early.any() and not early.all()
    check(got[:, early], want[:, early], tol[:, early])
    if louder <= 12 or dtype == BF:  # the others' values are beyond fp16
        check(got, want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("T,H,D", ROWS)
@pytest.mark.parametrize("louder", [12, 24, 45, 100])
def test_loud_values_of_faint_keys(require_gpu, T, H, D, dtype, louder):
    """A block whose V scale is far above the others' and whose keys have next to no weight, first or last of the cache."""
    n, block = 16 * 21, 16
    for where in (0, -1):
        ref = random_ref(1, 1, 1, D, n, block, louder)
        ref.vs[0, 0, 0, where] = 2.0 ** (louder - 9)
        # one dimension drives the scores: the block's keys stand at -448 and the others near 0, times q = 1 and a scale of 2
        ref.k[0, 0, 0, :, 0] = 0
        ref.k[0, 0, 0].view(-1, block, D)[where, :, 0] = 0x7E | 0x80
        ref.ks[0, 0, 0] = 2.0 ** -8
        q = _q((1, T, H, D), dtype, 3) * 0.01
        q[..., 0] = (louder + 3) * 0.69314718 / (448 * 2.0 ** -8 * 2)  # p = 2^-(louder + 3) of the others'
        got = ref.to_cache([n]).attend(0, q.cuda(), scale=2.0, causal=False)
        want, tol = attend(ref, 0, q, [n], scale=2.0, causal=False)
        check(got, want, tol)
