"""Attention over the 8-bit KV cache: what a row's result may depend on, and how many bits it keeps."""
import numpy as np
import pytest
import torch

from tests.kv8_bounds import P_REL, attend, check
from tests.kv8_util import random_ref

BF, HF = torch.bfloat16, torch.float16


def _q(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _e5m2(x):
    """The nearest E5M2 value (half up in magnitude) of f16 numbers, by their bits: the upper byte of an f16."""
    return ((x.view(np.uint16) + np.uint16(0x80)) & np.uint16(0xFF00)).view(np.float16)


@pytest.mark.parametrize("up", [1.0, 8.0])
def test_three_rounded_parts_hold_an_f16(up):
    """Every f16 up to 2^15.25: three E5M2 parts, each the rounding of what the parts before it left over (times `up` a part), are its value
    but for the last part's smallest steps; no part leaves the type; cut parts would lose two bits."""
    p = np.arange(1, 0x7C00, dtype=np.uint16).view(np.float16)
    p = p[p.astype(np.float64) <= 2.0 ** 15.25]
    rest, total, unit = p, np.zeros(p.shape), 1.0
    for _ in range(3):
        part = _e5m2(rest)
        assert np.isfinite(part).all() and np.abs(part.astype(np.float64)).max() <= 57344
        total += part.astype(np.float64) * unit
        left = rest.astype(np.float64) - part.astype(np.float64)
        rest, unit = (left * up).astype(np.float16), unit / up
        assert (rest.astype(np.float64) == left * up).all()  # the kernel's f16 subtraction loses nothing
    x = p.astype(np.float64)
    lost = np.abs(total - x)
    assert (lost <= 2.0 ** -17 / up ** 2).all()
    assert (lost[x >= 2.0 ** (-6 - 2 * np.log2(up))] == 0).all()
    cut = lambda y: (y.view(np.uint16) & np.uint16(0xFF00)).view(np.float16)  # noqa: E731
    a = cut(p)
    b = cut((x - a).astype(np.float16))
    c = _e5m2((x - a - b).astype(np.float16))
    big = x >= 1
    assert np.abs(x - a - b - c)[big].max() > 0 and (np.abs(x - a - b - c) / x)[big].max() > 3 * P_REL[BF]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("T,H,D", [(4, 2, 64), (2, 8, 256), (4, 4, 128), (40, 2, 64), (24, 8, 256), (30, 8, 96)])
@pytest.mark.parametrize("n", [2, 3, 5, 40])
def test_probabilities_keep_their_bits(require_gpu, T, H, D, dtype, n):
    """A few keys of unlike weight whose values have one sign, so that nothing hides behind cancellation: a part of P that went missing
    is 2^-7 (bf16) or 2^-11 (fp16) of the output."""
    ref = random_ref(4, 1, 1, D, 64, 16, n)
    ref.v &= 0x7F
    q = _q((4, T, H, D), dtype, n)
    want, tol = attend(ref, 0, q, [n] * 4, causal=False)
    check(ref.to_cache([n] * 4).attend(0, q.cuda(), causal=False), want, tol)


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


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("T,H,heads", [(2, 8, 1), (3, 3, 1), (1, 32, 2), (5, 6, 2), (16, 1, 1)])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("cap,lens", [(128, [100, 3]), (1024, [968, 301]), (1 << 15, [20000, 130])], ids=["one", "cluster", "merge"])
def test_nine_to_sixteen_rows(require_gpu, T, H, heads, D, cap, lens, dtype):
    """9 to 16 rows of a key head: one split, splits joined in a cluster and by the merge; prefix masks and padded queries."""
    assert 9 <= T * H // heads <= 16
    q_lens, prefix = [T, max(1, T - 1)], [7, lens[1]]
    ref = random_ref(2, 1, heads, D, cap, 128, D + T)
    q = _q((2, T, H, D), dtype, T)
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    got = ref.to_cache(lens).attend(0, q.cuda(), q_lens=dev(q_lens), prefix=dev(prefix)).cpu()
    want, tol = attend(ref, 0, q, lens, q_lens=q_lens, prefix=prefix)
    check(got, want, tol)
