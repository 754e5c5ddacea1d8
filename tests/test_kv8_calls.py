"""Calls of the 8-bit KV cache and the NVFP4 linear layer at the edges of what their documentation allows."""
import pytest
import torch

BF, HF = torch.bfloat16, torch.float16


def _dev(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.gpu
def test_bind_of_tokens_that_lens_does_not_count_yet(require_gpu):
    """Lengths given to the bind are what is read: tokens appended and not yet advanced over are real."""
    from flashact_b200 import Kv8Cache
    from oracle import pi05_oracle as O
    from tests.pi05_util import engine_for
    c = O.make_case(seed=6, L=2, T=50, AD=32, Lp=120, B=2, num_steps=2)
    cache = Kv8Cache(2, 2, 1, 256, 120)
    for layer in range(2):
        cache.append(layer, c.k[:, layer, :, None].contiguous().cuda(), c.v[:, layer, :, None].contiguous().cuda())
    eng = engine_for(c)
    k, v = cache.read(120, lens=_dev([120, 90]))
    eng.bind_prefix_kv(k, v, [120, 90])
    want = eng.sample_actions(c.noise.cuda())
    for lens in ([0, 0], [50, 120]):
        cache.lens.copy_(_dev(lens))
        eng.bind_prefix_cache(cache, [120, 90])
        assert torch.equal(eng.sample_actions(c.noise.cuda()), want), lens
    eng.close()
