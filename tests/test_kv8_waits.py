"""Attention over the 8-bit KV cache: a device wait that runs out (made on the host, no GPU fault) is seen in every row it served."""
import pytest
import torch

from tests.kv8_bounds import attend, check
from tests.kv8_util import random_ref

BF, HF = torch.bfloat16, torch.float16


@pytest.fixture
def hook():
    from flashact_b200 import _capi as C
    lib = C.load_library()
    yield lambda split: lib.fa_kv8_set_fault_injection(split, 1 << 16)
    lib.fa_kv8_set_fault_injection(-1, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("T,H,D", [(1, 8, 256), (3, 4, 64), (24, 8, 256), (40, 1, 96)])
@pytest.mark.parametrize("cap,long", [(128, 120), (1024, 968), (1 << 15, 30000)])
def test_a_wait_that_runs_out(require_gpu, hook, T, H, D, cap, long, dtype):
    """One split, splits joined in a cluster, splits joined by the merge: the scores of one split never come. Observations that have that
    split are NaN, whatever the other splits hold; one that does not need it is as before; so is the next call."""
    lens = [long, 50]
    ref = random_ref(2, 1, 1, D, cap, 128, 3)
    cache = ref.to_cache(lens)
    q = torch.randn(2, T, H, D, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    good = cache.attend(0, q)
    check(good, *attend(ref, 0, q.cpu(), lens))
    for split in (0, 1):
        hook(split)
        got = cache.attend(0, q)
        torch.cuda.synchronize()
        if split == 0 or long > 128:
            assert torch.isnan(got[0]).all()
        if split == 0:
            assert torch.isnan(got[1]).all()
        else:
            assert torch.equal(got[1], good[1])
        hook(-1)
        assert torch.equal(cache.attend(0, q), good)
