"""Calls of the 8-bit KV cache and the NVFP4 linear layer at the edges of what their documentation allows."""
import ctypes
import os
import subprocess
import sys
import threading
from types import SimpleNamespace

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


def test_bind_refuses_another_device():
    """Values are read, copied and bound on one stream of one device."""
    from flashact_b200 import FlashActError
    from flashact_b200.pi05 import bind_cache
    cache = SimpleNamespace(device=torch.device("cuda", 0), layers=2, heads=1, head_dim=256, batch=1, capacity=64, tensors=lambda: ())
    with pytest.raises(FlashActError, match="the engine is on cuda:1"):
        bind_cache(SimpleNamespace(device=1), None, cache, (2, 1, 256), [3], None)
    with pytest.raises(FlashActError, match="a stream of cuda:1"):
        bind_cache(SimpleNamespace(device=0), None, cache, (2, 1, 256), [3], SimpleNamespace(device_index=1))


@pytest.mark.gpu
def test_streams_of_another_device_are_refused(require_gpu):
    """They would not be the stream that the call then runs on."""
    from flashact_b200 import FlashActError, Kv8Cache
    from flashact_b200.quant import nvfp4_linear
    other = SimpleNamespace(device_index=1)
    c = Kv8Cache(1, 1, 1, 64, 64)
    k = torch.zeros(1, 1, 1, 64, dtype=BF, device="cuda")
    x, w, bs, ts = (torch.zeros(*n, dtype=t, device="cuda") for n, t in (((1, 64), BF), ((8, 32), torch.uint8), ((8, 4), torch.uint8),
                                                                        ((1,), torch.float32)))
    for f in (lambda: c.append(0, k, k, stream=other), lambda: c.attend(0, k, stream=other), lambda: c.read(1, stream=other),
              lambda: nvfp4_linear(x, w, bs, ts, stream=other)):
        with pytest.raises(FlashActError, match="a stream of cuda:1"):
            f()


@pytest.mark.gpu
def test_bind_on_a_side_stream(require_gpu):
    """Read and bound on the stream that is given, or on the current one where that is not the default."""
    from flashact_b200 import Kv8Cache
    from oracle import pi05_oracle as O
    from tests.pi05_util import engine_for
    c = O.make_case(seed=7, L=2, T=50, AD=32, Lp=64, B=1, num_steps=2)
    eng = engine_for(c)
    side = torch.cuda.Stream()
    got = []
    for how in (0, 1, 2):
        cache = Kv8Cache(1, 2, 1, 256, 64)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side if how else torch.cuda.current_stream()):
            for layer in range(2):
                cache.append(layer, c.k[:, layer, :, None].contiguous().cuda(), c.v[:, layer, :, None].contiguous().cuda())
            cache.advance(64)
            if how < 2:
                eng.bind_prefix_cache(cache)
        if how == 2:
            eng.bind_prefix_cache(cache, stream=side)
        torch.cuda.synchronize()
        got.append(eng.sample_actions(c.noise.cuda()))
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
    eng.close()


@pytest.mark.gpu
def test_advance_on_the_stream_of_the_appends(require_gpu):
    """A step on a side stream that is behind the current one: every layer appends at the same place, then the lengths move."""
    from flashact_b200 import Kv8Cache
    k = torch.randn(1, 5, 1, 64, generator=torch.Generator().manual_seed(0)).to(BF).cuda()
    here, there = Kv8Cache(1, 3, 1, 64, 64), Kv8Cache(1, 3, 1, 64, 64)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)  # some ms
    for c, s in ((here, None), (there, side)):
        for _ in range(2):
            for layer in range(3):
                c.append(layer, k, k, stream=s)
            c.advance(5, stream=s)
    torch.cuda.synchronize()
    assert here.lens.tolist() == there.lens.tolist() == [10]
    assert torch.equal(here.k, there.k) and torch.equal(here.v, there.v) and torch.equal(here.k_scale, there.k_scale)
    with pytest.raises(RuntimeError):
        here.advance(torch.ones(2, dtype=torch.int32, device="cuda"))
    assert here.lens.tolist() == [10]


@pytest.mark.gpu
def test_inputs_dropped_before_a_side_stream_has_run(require_gpu):
    """Temporaries handed to a call on another stream keep their memory until that stream is done with them."""
    from flashact_b200 import Kv8Cache
    from flashact_b200.quant import nvfp4_linear
    g = torch.Generator().manual_seed(2)
    k = torch.randn(2, 300, 2, 64, generator=g).to(BF).cuda()
    q = torch.randn(2, 40, 4, 64, generator=g).to(BF).cuda()
    x = torch.randn(16, 4096, generator=g).to(BF).cuda()
    w = [torch.randint(0, 256, (640, 2048), generator=g, dtype=torch.uint8).cuda(),
         torch.randint(0, 100, (640, 256), generator=g, dtype=torch.uint8).cuda(), torch.tensor([1e-4], device="cuda")]
    n = _dev([300, 200])
    want = Kv8Cache(2, 1, 2, 64, 512)
    want.append(0, k, k, count=n)
    want.advance(n)
    attended, linear = want.attend(0, q), nvfp4_linear(x, *w)
    side = torch.cuda.Stream()
    got = Kv8Cache(2, 1, 2, 64, 512)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(40_000_000)  # longer than the host needs for what follows
    # the clones are made on the current stream, which is idle: their values are there long before the side stream gets to them
    tmp = [t.clone() for t in (k, k, n, q, x, n)]
    torch.cuda.current_stream().synchronize()
    got.append(0, tmp[0], tmp[1], count=tmp[2], stream=side)
    got.advance(tmp[5], stream=side)
    a = got.attend(0, tmp[3], stream=side)
    y = nvfp4_linear(tmp[4], *w, stream=side)
    sizes = [(t.shape, t.dtype) for t in tmp]
    del tmp
    for shape, dt in sizes * 4:  # whoever asks next
        torch.full(shape, 1, dtype=dt, device="cuda")
    torch.cuda.synchronize()
    assert torch.equal(got.k, want.k) and torch.equal(got.v, want.v) and torch.equal(got.lens, want.lens)
    assert torch.equal(a, attended) and torch.equal(y, linear)


def test_one_workspace_for_several_calls():
    """The workspace of a large call need not do for a smaller one; the largest of what the calls ask for does for each of them."""
    from flashact_b200 import _capi as C
    from flashact_b200.build import build
    lib = C.load_library(build())
    c = C.FaKv8(16, 16, 16, 16, 1, 1, 1, 256, 1 << 14, 64)
    r = C.FaRows(16, 256, 256, 256)

    def need(tokens, max_len):
        n = ctypes.c_size_t()
        assert lib.fa_kv8_attention_workspace(ctypes.byref(c), tokens, 8, max_len, ctypes.byref(n)) == C.FA_OK
        return n.value

    def attend(tokens, max_len, ws):
        st = lib.fa_kv8_attention(ctypes.byref(c), 0, tokens, 8, ctypes.byref(r), C.FA_DT_BF16, 16, None, None, 1, 0.1, max_len,
                                  ctypes.byref(r), 16, ws, None)
        return st, lib.fa_last_error(None).decode()
    calls = [(t, n) for t in (1, 2, 16, 50, 256, 1024) for n in (0, 128, 1024, 9000)]
    needs = [need(*x) for x in calls]
    assert need(1024, 0) < need(1, 0)
    st, why = attend(1, 0, need(1024, 0))
    assert st == C.FA_ERR_INVALID and "workspace" in why
    for x in calls:
        st, why = attend(*x, max(needs))
        assert "workspace of" not in why  # whatever else these made-up pointers are refused for


@pytest.mark.gpu
def test_values_past_32_bits(require_gpu):
    """More than 2^32 codes in K and in V: what append wrote at the end of each head, found there by torch's own indexing, is the reference's; read
    gives it back, and attention weighs it against a million keys of zero."""
    from flashact_b200 import Kv8Cache
    from tests.kv8_util import codes, scale_of, values
    B, heads, D, cap = 3, 6, 256, 1 << 20
    c = Kv8Cache(B, 1, heads, D, cap, block=128)
    assert c.k.numel() > 1 << 32
    n = cap - 3
    g = torch.Generator().manual_seed(9)
    k, v = torch.randn(B, 2, heads, D, generator=g).to(BF), (torch.randn(B, 2, heads, D, generator=g) * 1000).to(BF)
    q = torch.randn(B, 1, heads, D, generator=g)
    q = (q + 1.3 * k.float().mean(1, keepdim=True)).to(BF)  # scores near log(cap), so that both sides count
    c.lens.fill_(n - 2)
    c.append(0, k.cuda(), v.cuda())
    c.advance(2)
    got = c.attend(0, q.cuda()).cpu().double()
    kk, vv = c.read(cap)
    assert (kk[:, 0, n - 130:n - 2] == 0).all() and (vv[:, 0, n:] == 0).all()
    for b in range(B):
        for h in range(heads):
            real = []
            for name, new, x in (("k", k, kk), ("v", v, vv)):
                x32 = new[b, :, h].float()
                s = scale_of(x32.abs().max().item())
                want = codes(x32, s)
                held = (c.k[b, 0, h, n - 2:n] if name == "k" else c.v[b, 0, h, :, n - 2:n].t()).cpu()
                assert torch.equal(held, want) and (c.k_scale if name == "k" else c.v_scale)[b, 0, h, -1].item() == s
                real.append(values(want) * s)
                assert torch.equal(x[b, 0, n - 2:n, h * D:(h + 1) * D].cpu().double(), real[-1])
            a = real[0] @ q[b, 0, h].double() / D ** 0.5
            p = torch.exp(a)
            p = p / (p.sum() + n - 2)
            o, spread = p @ real[1], p @ real[1].abs()
            big = (real[0].abs() @ q[b, 0, h].double().abs()).max().item() / D ** 0.5
            # roundings as in tests/kv8_bounds.py: output, products of P, scores and exponentials; the sum of a million ones in fp32, at most
            # 2^20 / 128 of them to a thread, is exact
            tol = 2.0 ** -8 * o.abs() + 1.01 * (2.0 ** -11 + 2 * ((D + 8) * 2.0 ** -23 * big + 2.0 ** -17 + 2.0 ** -20)) * spread
            assert p.min() > 1e-9 and ((got[b, 0, h] - o).abs() <= tol).all(), (b, h, p.tolist(), ((got[b, 0, h] - o).abs() / tol).max().item())


@pytest.mark.gpu
def test_linear_refuses_an_output_over_its_input(require_gpu):
    """Blocks write y while others read x. Columns beside each other in one buffer do not overlap."""
    from flashact_b200 import FlashActError, _capi as C
    from flashact_b200.quant import nvfp4_linear
    from tests.test_nvfp4_linear import check_linear
    lib = C.load_library()
    g = torch.Generator().manual_seed(5)
    w = (torch.randint(0, 256, (64, 32), generator=g, dtype=torch.uint8).cuda(),
         torch.randint(0, 100, (64, 4), generator=g, dtype=torch.uint8).cuda(), torch.tensor([1e-2], device="cuda"))
    x = torch.randn(4, 64, generator=g).to(BF).cuda()
    with pytest.raises(FlashActError, match="overlaps"):
        nvfp4_linear(x, *w, out=x)
    buf = torch.zeros(4, 128, dtype=BF, device="cuda")
    buf[:, :64] = x

    def call(y, N, ldy):
        return lib.fa_nvfp4_linear(buf.data_ptr(), C.FA_DT_BF16, 4, 64, 128, w[0].data_ptr(), w[1].data_ptr(), w[2].data_ptr(), None, N,
                                   buf.data_ptr() + 2 * y, ldy, torch.cuda.current_stream().cuda_stream)
    for y, N, ldy in ((0, 64, 128), (63, 64, 128), (64 + 3 * 128, 64, 64), (65, 64, 128), (10, 8, 128)):
        overlaps = any(y + j * ldy < i * 128 + 64 and i * 128 < y + j * ldy + N for i in range(4) for j in range(4))
        if overlaps:  # the others lie inside the buffer only where the next line says so
            assert call(y, N, ldy) == C.FA_ERR_INVALID, (y, N, ldy)
    assert call(64, 64, 128) == C.FA_OK
    check_linear(buf[:, 64:].contiguous(), x, *w)
    assert torch.equal(buf[:, :64], x)


def test_attention_refuses_output_rows_on_one_another():
    """An expanded output: all rows of it would be written to one place, in no order."""
    from flashact_b200 import _capi as C
    from flashact_b200.build import build
    lib = C.load_library(build())
    c = C.FaKv8(16, 16, 16, 16, 2, 1, 1, 64, 128, 64)
    q = C.FaRows(16, 512, 128, 64)

    def refused(tokens, heads, batch, token, head):
        o = C.FaRows(16, batch, token, head)
        st = lib.fa_kv8_attention(ctypes.byref(c), 0, tokens, heads, ctypes.byref(q), C.FA_DT_BF16, 16, None, None, 1, 0.1, 0,
                                  ctypes.byref(o), None, 0, None)
        return st == C.FA_ERR_INVALID and "stride of 0" in lib.fa_last_error(None).decode()
    assert refused(4, 2, 0, 128, 64) and refused(4, 2, 512, 0, 64) and refused(4, 2, 512, 128, 0)
    assert not refused(4, 2, 512, 128, 64) and not refused(1, 1, 64, 0, 0)


def test_scale_past_fp32_is_refused():
    """The kernels hold scale log2 e: a finite scale whose product is none would make every score infinite or NaN."""
    from flashact_b200 import _capi as C
    from flashact_b200.build import build
    lib = C.load_library(build())
    c = C.FaKv8(16, 16, 16, 16, 1, 1, 1, 64, 128, 64)
    r = C.FaRows(16, 64, 64, 64)

    def refused(scale):
        st = lib.fa_kv8_attention(ctypes.byref(c), 0, 1, 1, ctypes.byref(r), C.FA_DT_BF16, 16, None, None, 1, scale, 0,
                                  ctypes.byref(r), None, 0, None)
        return st == C.FA_ERR_INVALID and "finite" in lib.fa_last_error(None).decode()
    assert refused(2.9e38) and refused(-2.9e38) and refused(float("inf")) and refused(float("nan"))
    assert not refused(2.3e38) and not refused(-1.0) and not refused(0.0)


def test_lens_must_be_a_tensor():
    from flashact_b200 import FlashActError, Kv8Cache
    c = Kv8Cache.__new__(Kv8Cache)
    c._lens, c._lens_tensor = 16, "as it was"
    with pytest.raises(FlashActError):
        c.lens = None
    assert (c._lens, c.lens) == (16, "as it was")
    with pytest.raises(FlashActError):
        Kv8Cache.from_tensors(*[torch.zeros(()) for _ in range(4)])


@pytest.mark.gpu
def test_exact_max_len_of_each_step_is_not_kept(require_gpu):
    """A decoder that passes each step's length as max_len: what the cache remembers stays small."""
    from flashact_b200 import Kv8Cache
    c = Kv8Cache(1, 1, 1, 64, 512)
    q = torch.zeros(1, 1, 1, 64, dtype=BF, device="cuda")
    for n in range(1, 300):
        c.attend(0, q, max_len=n)
    assert len(c._ws) <= 64


def test_splits_fit_the_kernel_that_runs():
    """Two tokens of 8 query heads at head_dim 256 are blocks that fill an SM: four observations of a long cache are split into no more
    of them than there are SMs (148 where no device is), not into two to an SM."""
    from flashact_b200 import _capi as C
    from flashact_b200.build import build
    lib = C.load_library(build())
    n = ctypes.c_size_t()
    c = C.FaKv8(16, 16, 16, 16, 4, 1, 1, 256, 1 << 14, 64)
    assert lib.fa_kv8_attention_workspace(ctypes.byref(c), 2, 8, 0, ctypes.byref(n)) == C.FA_OK
    splits = n.value // (4 * 16 * (256 * 4 + 8))  # observations x rows x (sums, maximum and sum)
    assert 8 < splits and 4 * splits <= 148


FIRST = """
import torch
from flashact_b200 import Kv8Cache
from flashact_b200.quant import nvfp4_linear
BF = torch.bfloat16
c = Kv8Cache(2, 1, 1, 256, 1 << 14)
k = torch.randn(2, 300, 1, 256, device="cuda").to(BF)
q = [torch.randn(2, t, 8, 256, device="cuda").to(dt) for t in (1, 2, 40) for dt in (BF, torch.float16)]
x, w, bs, ts = torch.ones(1, 64, dtype=BF, device="cuda"), *(torch.zeros(8, n, dtype=torch.uint8, device="cuda") for n in (32, 4)), torch.ones(1, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):  # nothing of the library has run before
    c.append(0, k, k)
    c.advance(300)
    got = [c.attend(0, x) for x in q]
    v = c.read(300)
    y = nvfp4_linear(x, w, bs, ts)
g.replay()
torch.cuda.synchronize()
assert c.lens.tolist() == [300, 300]
assert all(torch.equal(a, c.attend(0, x)) for a, x in zip(got, q)) and torch.equal(v[0], c.read(300)[0]) and (y == 0).all()
print("captured first")
"""


@pytest.mark.gpu
def test_first_calls_of_a_process_may_be_captured(require_gpu):
    """Kernels are loaded, limits set and the device's room asked for inside the capture."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST], cwd=root, capture_output=True, text=True, timeout=300)
    assert "captured first" in r.stdout, r.stderr[-2000:]


@pytest.mark.gpu
def test_calls_from_several_threads(require_gpu):
    """Two caches, a thread and a stream each, long enough to overlap: the results of calls one after the other."""
    from flashact_b200 import Kv8Cache
    g = torch.Generator().manual_seed(8)
    work, want = [], []
    for n in (700, 9000):
        c = Kv8Cache(3, 1, 2, 128, 1 << 14)
        k = torch.randn(3, n, 2, 128, generator=g).to(BF).cuda()
        c.append(0, k, k)
        c.advance(n)
        qs = [torch.randn(3, t, 8, 128, generator=g).to(dt).cuda() for t in (1, 3, 30) for dt in (BF, HF)]
        work.append((c, qs))
        want.append([c.attend(0, q) for q in qs])
    torch.cuda.synchronize()
    bad = []

    def run(i):
        try:
            c, qs = work[i]
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(60):
                    got = [c.attend(0, q) for q in qs]
                torch.cuda.current_stream().synchronize()
                bad.extend(j for j, (a, b) in enumerate(zip(got, want[i])) if not torch.equal(a, b))
        except Exception as e:  # noqa: BLE001
            bad.append(e)
    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


@pytest.mark.gpu
def test_bind_with_the_same_lengths_may_be_captured(require_gpu):
    """Lengths that the host knows cost no copy to the device and no wait: a bind with those of the last one is launches alone."""
    from flashact_b200 import Kv8Cache
    from oracle import pi05_oracle as O
    from tests.pi05_util import engine_for
    c = O.make_case(seed=9, L=2, T=50, AD=32, Lp=64, B=2, num_steps=2)
    eng, cache = engine_for(c), Kv8Cache(2, 2, 1, 256, 64)

    def fill(scale):
        for layer in range(2):
            cache.append(layer, (c.k[:, layer, :, None] * scale).contiguous().cuda(), (c.v[:, layer, :, None] * scale).contiguous().cuda())
    fill(1.0)
    eng.bind_prefix_cache(cache, [64, 40])
    first = eng.sample_actions(c.noise.cuda())
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        eng.bind_prefix_cache(cache, [64, 40])
    fill(0.5)
    g.replay()
    got = eng.sample_actions(c.noise.cuda())
    eng.bind_prefix_cache(cache, [64, 40])
    assert torch.equal(got, eng.sample_actions(c.noise.cuda())) and not torch.equal(got, first)
    eng.close()
