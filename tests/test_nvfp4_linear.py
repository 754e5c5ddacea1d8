"""fa_nvfp4_linear against a 64-bit restatement."""
import ctypes

import pytest
import torch

BF, HF = torch.bfloat16, torch.float16
E2M1 = torch.tensor([0.0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)


def dequant(packed, bscale, tscale):
    c = torch.stack([packed & 15, packed >> 4], -1).flatten(-2).long()
    return E2M1.to(packed.device)[c] * bscale.view(torch.float8_e4m3fn).double().repeat_interleave(16, -1) * tscale.double()


def check_linear(y, x, packed, bscale, tscale, bias=None):
    """|y - exact| counts its roundings: half a step of y's type, and fp32 sums of K products, in K / 16 steps of the
    matrix instruction (which truncates: 2^-23 of the running sum each) and a few additions, of sum |x w|."""
    w = dequant(packed.view(-1, packed.shape[-1]), bscale.view(-1, bscale.shape[-1]), tscale.view(-1)[0])
    xd = x.double().view(-1, x.shape[-1])
    want, size = xd @ w.T, xd.abs() @ w.abs().T
    if bias is not None:
        want, size = want + bias.double(), size + bias.double().abs()
    u = torch.finfo(y.dtype).eps / 2
    tol = u * want.abs() + (1 + u) * (x.shape[-1] / 16 + 16) * 2.0 ** -23 * size + 2.0 ** -25
    d = (y.double().view(want.shape) - want).abs()
    assert (d <= tol).all(), (d / tol).max().item()


def test_refusals():
    from flashact_b200 import _capi as C
    from flashact_b200.build import build
    lib = C.load_library(build())

    def call(x=16, dt=1, M=1, K=64, ldx=64, w=16, bs=16, ts=16, bias=None, N=8, y=16, ldy=8):
        return lib.fa_nvfp4_linear(x, dt, M, K, ldx, w, bs, ts, bias, N, y, ldy, None)
    assert call(dt=0) == C.FA_ERR_UNSUPPORTED and call(M=17) == C.FA_ERR_UNSUPPORTED
    for kw in (dict(M=-1), dict(N=0), dict(K=0), dict(K=72, ldx=72), dict(M=2, ldx=56), dict(ldx=66), dict(M=2, ldy=7), dict(x=8),
               dict(w=12), dict(y=17), dict(ts=2), dict(bias=2)):
        assert call(**kw) == C.FA_ERR_INVALID, kw
    assert call(M=0) == C.FA_OK
    if not torch.cuda.is_available():
        assert call() == C.FA_ERR_CUDA
    assert ctypes.sizeof(C.FaKv8) == 4 * 8 + 6 * 4 and ctypes.sizeof(C.FaRows) == 32


def _case(M, N, K, dtype, seed, dev="cuda"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g).to(dtype)
    packed = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8)
    bs = torch.randint(0, 127, (N, K // 16), generator=g, dtype=torch.uint8)  # every finite scale, subnormals and 448 too
    ts = torch.tensor([3e-4])
    return [t.to(dev) for t in (x, packed, bs, ts)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("M,N,K", [(1, 1, 16), (1, 17, 48), (3, 16, 32), (8, 100, 1024), (9, 33, 1040), (16, 257, 2064),
                                   (1, 2560, 1024), (5, 10000, 128), (16, 9481, 160), (2, 19001, 4112), (16, 64, 16384),
                                   (7, 20000, 2048)])
def test_linear(require_gpu, M, N, K, dtype):
    from flashact_b200.quant import nvfp4_linear
    x, packed, bs, ts = _case(M, N, K, dtype, M + N + K)
    ts = ts / 100 if dtype == HF else ts  # results inside fp16
    bias = torch.randn(N, generator=torch.Generator().manual_seed(1)).cuda()
    y = nvfp4_linear(x, packed, bs, ts)
    check_linear(y, x, packed, bs, ts)
    check_linear(nvfp4_linear(x, packed, bs, ts, bias=bias), x, packed, bs, ts, bias)
    assert torch.equal(y, nvfp4_linear(x, packed, bs, ts))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF])
def test_linear_every_code_and_scale(require_gpu, dtype):
    """Each of the 16 codes times each finite block scale, alone: the result is the exact product, rounded once."""
    from flashact_b200.quant import nvfp4_linear
    N, K = 127, 256
    packed = torch.zeros(N, K // 2, dtype=torch.uint8)
    for c in range(16):
        packed[:, c * 8] = c  # code c at k = 16 c
    bs = torch.arange(127, dtype=torch.uint8)[:, None].repeat(1, 16)
    x = torch.zeros(16, K, dtype=dtype)
    x[torch.arange(16), torch.arange(16) * 16] = 1.0
    y = nvfp4_linear(x.cuda(), packed.cuda(), bs.cuda(), torch.ones(1, device="cuda"))
    want = E2M1[:, None] * bs[:, 0].view(torch.float8_e4m3fn).double()[None]
    assert torch.equal(y.cpu().double(), want)  # six bits: exact in both types


@pytest.mark.gpu
def test_linear_calls(require_gpu):
    """Leading dimensions, out, strided and misaligned x, misaligned codes, NaN and infinity, capture, a side stream."""
    from flashact_b200 import FlashActError
    from flashact_b200.quant import nvfp4_linear
    x, packed, bs, ts = _case(6, 100, 96, BF, 3)
    want = nvfp4_linear(x, packed, bs, ts)
    assert torch.equal(nvfp4_linear(x.view(2, 3, 96), packed, bs, ts).view(6, 100), want)
    out = torch.empty_like(want)
    assert nvfp4_linear(x, packed, bs, ts, out=out) is out and torch.equal(out, want)
    assert torch.equal(nvfp4_linear(x.t().contiguous().t(), packed, bs, ts), want)
    odd = torch.zeros(6 * 96 + 1, dtype=BF, device="cuda")
    odd[1:] = x.flatten()
    assert torch.equal(nvfp4_linear(odd[1:].view(6, 96), packed, bs, ts), want)
    raw = torch.zeros(packed.numel() + 8, dtype=torch.uint8, device="cuda")
    raw[8:] = packed.flatten()
    shifted = nvfp4_linear(x, raw[8:].view_as(packed), bs, ts)  # 8-byte aligned codes: the narrow loads
    check_linear(shifted, x, packed, bs, ts)
    assert nvfp4_linear(x[:0], packed, bs, ts).shape == (0, 100)
    x2 = x.clone()
    x2[2, 5], x2[3, 7] = float("nan"), float("inf")
    got = nvfp4_linear(x2, packed, bs, ts)
    assert torch.isnan(got[2]).all() and not torch.isfinite(got[3]).all()
    assert torch.equal(got[[0, 1, 4, 5]], want[[0, 1, 4, 5]])
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        y = nvfp4_linear(x, packed, bs, ts)
    x.mul_(2)
    g.replay()
    torch.cuda.synchronize()
    check_linear(y, x, packed, bs, ts)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    z = nvfp4_linear(x, packed, bs, ts, stream=side)
    side.synchronize()
    assert torch.equal(z, y)
    big = torch.zeros(17, 96, dtype=BF, device="cuda")
    for f in (lambda: nvfp4_linear(big, packed, bs, ts), lambda: nvfp4_linear(x.float(), packed, bs, ts),
              lambda: nvfp4_linear(x, packed[:, :40], bs, ts), lambda: nvfp4_linear(x, packed, bs[:50], ts),
              lambda: nvfp4_linear(x, packed, bs, ts.double()), lambda: nvfp4_linear(x.cpu(), packed, bs, ts),
              lambda: nvfp4_linear(x, packed, bs, ts, bias=ts), lambda: nvfp4_linear(x, packed, bs, ts, out=want[:3])):
        with pytest.raises((FlashActError, RuntimeError)):
            f()
