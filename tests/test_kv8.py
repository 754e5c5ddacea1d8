"""The 8-bit KV cache: append, attention and read against 64-bit restatements (tests/kv8_util.py)."""
import ctypes

import pytest
import torch

from tests.kv8_util import Ref, attend, codes, random_ref, scale_of, values

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


# ------------------------------------------------------------------------------------------------ CPU
def test_scale_rule():
    for a in (0.0, 1e-40, 1.0, 448.0, 449.0, 447.9, 1.75, 1.76, 3e38, 448 * 2.0 ** -96, 450 * 2.0 ** -96):
        s = scale_of(a)
        assert a <= 448 * s and (s == 2.0 ** -96 or a > 224 * s)


def test_reference_append_keeps_values_on_a_larger_scale():
    r = Ref(1, 1, 1, 64, 32, 32)
    g = torch.Generator().manual_seed(0)
    a, b = torch.randn(1, 3, 1, 64, generator=g), torch.randn(1, 2, 1, 64, generator=g) * 100
    r.append(0, a, a, [0], [3])
    before = values(r.k[0, 0, 0, :3]) * r.ks[0, 0, 0, 0].item()
    r.append(0, b, b, [3], [2])
    after = values(r.k[0, 0, 0, :3]) * r.ks[0, 0, 0, 0].item()
    # a larger power of two only drops what becomes subnormal: half its step, 2^-10 scales
    assert ((after - before).abs() <= 2.0 ** -10 * r.ks[0, 0, 0, 0].item()).all()


def _desc(**kw):
    from flashact_b200 import _capi as C
    a = dict(k=16, v=16, k_scale=16, v_scale=16, batch=2, layers=2, heads=2, head_dim=64, capacity=128, block=32)
    a.update(kw)
    return C.FaKv8(*[a[n] for n, _ in C.FaKv8._fields_])


def _append(C, lib, c, layer=0, rows=1, dtype=0, ptr=16):
    r = C.FaRows(ptr, 64, 64, 64)
    return lib.fa_kv8_append(ctypes.byref(c), layer, rows, ctypes.byref(r), ctypes.byref(r), dtype, 16, None, None)


def _attend(C, lib, c, layer=0, tokens=1, heads=2, dtype=1, causal=1, prefix=None, scale=0.1, max_len=0, ws=1 << 40, ptr=16):
    r = C.FaRows(ptr, 64, 64, 64)
    return lib.fa_kv8_attention(ctypes.byref(c), layer, tokens, heads, ctypes.byref(r), dtype, 16, None, prefix, causal, scale,
                                max_len, ctypes.byref(r), 16, ws, None)


@pytest.mark.parametrize("kw,status", [
    (dict(head_dim=80), 5), (dict(head_dim=512), 5), (dict(block=8), 5), (dict(block=48), 5), (dict(capacity=100), 1),
    (dict(capacity=0), 1), (dict(batch=0), 1), (dict(heads=0), 1), (dict(layers=-1), 1), (dict(k=8), 1), (dict(v=24), 1),
    (dict(k_scale=2), 1), (dict(capacity=(1 << 30) + 32), 1), (dict(batch=70000), 1)])
def test_descriptor_refusals(kw, status):
    """Refused before any pointer is looked at, on every entry point."""
    from flashact_b200 import _capi as C
    from flashact_b200.build import build
    lib = C.load_library(build())
    c = _desc(**kw)
    n = ctypes.c_size_t()
    assert _append(C, lib, c) == status
    assert _attend(C, lib, c) == status
    assert lib.fa_kv8_attention_workspace(ctypes.byref(c), 1, 2, 0, ctypes.byref(n)) == status
    assert lib.fa_kv8_read(ctypes.byref(c), 16, 1, 16, 16, 1, None) == status
    assert lib.fa_last_error(None)


def test_call_refusals():
    from flashact_b200 import _capi as C
    from flashact_b200.build import build
    lib = C.load_library(build())
    c = _desc()
    for kw in (dict(layer=2), dict(layer=-1), dict(rows=-1), dict(dtype=3), dict(ptr=18)):
        assert _append(C, lib, c, **kw) == C.FA_ERR_INVALID, kw
    assert _append(C, lib, c, rows=0) == C.FA_OK  # nothing to do, nothing looked at
    for kw in (dict(layer=2), dict(tokens=-1), dict(heads=3), dict(heads=0), dict(max_len=129), dict(max_len=-1),
               dict(scale=float("nan")), dict(scale=float("inf")), dict(causal=0, prefix=16), dict(ptr=17),
               dict(tokens=1 << 25)):
        assert _attend(C, lib, c, **kw) == C.FA_ERR_INVALID, kw
    assert _attend(C, lib, c, dtype=0) == C.FA_ERR_UNSUPPORTED
    assert _attend(C, lib, c, tokens=0) == C.FA_OK
    big = _desc(capacity=1 << 20)
    n = ctypes.c_size_t()
    assert lib.fa_kv8_attention_workspace(ctypes.byref(big), 1, 2, 0, ctypes.byref(n)) == C.FA_OK and n.value > 0
    assert _attend(C, lib, big, ws=n.value - 1) == C.FA_ERR_INVALID
    assert lib.fa_kv8_attention_workspace(ctypes.byref(big), 1, 2, 0, None) == C.FA_ERR_INVALID
    assert lib.fa_kv8_read(ctypes.byref(c), 16, -1, 16, 16, 1, None) == C.FA_ERR_INVALID
    assert lib.fa_kv8_read(ctypes.byref(c), 16, 1, 8, 16, 1, None) == C.FA_ERR_INVALID
    assert lib.fa_kv8_read(ctypes.byref(c), 16, 1, 16, 16, 7, None) == C.FA_ERR_INVALID
    assert lib.fa_kv8_read(ctypes.byref(_desc(batch=300, layers=300)), 16, 1, 16, 16, 1, None) == C.FA_ERR_INVALID
    assert lib.fa_kv8_append(None, 0, 1, None, None, 0, None, None, None) == C.FA_ERR_INVALID
    if not torch.cuda.is_available():  # no device: an error, never a crash
        assert _append(C, lib, c) == C.FA_ERR_CUDA


def test_python_refuses_host_tensors():
    from flashact_b200 import FlashActError, Kv8Cache
    k = torch.zeros(1, 1, 1, 32, 64, dtype=torch.uint8)
    s = torch.zeros(1, 1, 1, 1)
    with pytest.raises(FlashActError):
        Kv8Cache.from_tensors(k, k.transpose(-1, -2).contiguous(), s, s)
    with pytest.raises(FlashActError):
        Kv8Cache(0, 1, 1, 64, 32)


# ------------------------------------------------------------------------------------------------ GPU
def _same(cache, ref):
    assert torch.equal(cache.k_scale.cpu(), ref.ks)
    assert torch.equal(cache.v_scale.cpu(), ref.vs)
    assert torch.equal(cache.k.cpu(), ref.k)
    assert torch.equal(cache.v.cpu().transpose(-1, -2), ref.v)


def _check(got, want, tol):
    d = (got.cpu().double() - want).abs()
    assert torch.isfinite(got).all()
    assert (d <= tol).all(), (d.max().item(), (d / tol).max().item())


def _q(shape, dtype, seed, loud=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * loud).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("D,block,heads,dtype", [(64, 16, 3, BF), (96, 32, 2, HF), (128, 64, 1, FP), (256, 128, 2, BF),
                                                 (256, 16, 1, FP), (64, 128, 1, HF)])
def test_append(require_gpu, D, block, heads, dtype):
    """Prompts, then tokens one by one and in ragged batches, louder and quieter, in two layers."""
    from flashact_b200 import Kv8Cache
    B, cap = 3, 3 * block
    cache, ref = Kv8Cache(B, 2, heads, D, cap, block=block), Ref(B, 2, heads, D, cap, block)
    assert (cache.capacity, cache.block) == (cap, block)
    g = torch.Generator().manual_seed(D + block)
    lens = [0] * B
    steps = [(block + 5, [block + 5, 1, 0], 1.0), (1, None, 1.0), (1, [1, 0, 1], 50.0), (7, [7, 3, 5], 1e-4),
             (1, None, 3000.0), (block, [block - 9, block, 2], 1.0)]
    for n, count, loud in steps:
        for layer in (1, 0):
            k, v = ((torch.randn(B, n, heads, D, generator=g) * loud).to(dtype) for _ in range(2))
            c = None if count is None else torch.tensor(count, dtype=torch.int32, device="cuda")
            for _ in range(2):  # the same rows at the same place again change nothing
                cache.append(layer, k.cuda(), v.cuda(), count=c)
            ref.append(layer, k, v, lens, count or [n] * B)
            _same(cache, ref)
        step = count or [n] * B
        lens = [a + b for a, b in zip(lens, step)]
        cache.advance(torch.tensor(step, dtype=torch.int32, device="cuda"))
    assert cache.lens.tolist() == lens


@pytest.mark.gpu
def test_append_edges(require_gpu):
    """NaN and infinities, zero rows, strided and misaligned rows, rows behind the capacity, negative counts."""
    from flashact_b200 import Kv8Cache
    B, H, D, cap = 2, 2, 64, 64
    cache, ref = Kv8Cache(B, 1, H, D, cap, block=32), Ref(B, 1, H, D, cap, 32)
    g = torch.Generator().manual_seed(3)
    k, v = torch.randn(B, 40, H, D, generator=g), torch.randn(B, 40, H, D, generator=g)
    k[0, 3, 0, 5], k[0, 4, 0, 6], v[1, 2, 1, 7], v[1, 33, 0, 0] = float("nan"), float("inf"), float("-inf"), float("nan")
    k[1, :32, 1] = 0.0
    v[0, 32:, 0] = 1e-35
    wide_k = torch.zeros(B, H, 40, D + 3)  # heads before tokens, rows of an odd pitch
    wide_k[..., 1:D + 1] = k.transpose(1, 2)
    cache.append(0, wide_k.cuda()[..., 1:D + 1].transpose(1, 2), v.cuda())
    ref.append(0, k, v, [0, 0], [40, 40])
    _same(cache, ref)
    assert ((cache.k & 127) < 127).all() and ((cache.v & 127) < 127).all()
    start = torch.tensor([50, -5], dtype=torch.int32, device="cuda")
    count = torch.tensor([40, -1], dtype=torch.int32, device="cuda")
    cache.append(0, k.cuda(), v.cuda(), start=start, count=count)
    ref.append(0, k, v, [50, 0], [14, 0])
    _same(cache, ref)
    far = torch.tensor([64, 1 << 30], dtype=torch.int32, device="cuda")
    cache.append(0, k.cuda(), v.cuda(), start=far)  # all of it behind the capacity
    _same(cache, ref)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("D,block,heads", [(64, 16, 2), (96, 32, 8), (256, 128, 1)])
def test_read(require_gpu, D, block, heads, dtype):
    B, L, cap = 2, 3, 256
    ref = random_ref(B, L, heads, D, cap, block, 5)
    lens, rows = [77, 140], 131
    ref.k[0, :, :, 77:], ref.v[0, :, :, 77:] = 0x7F, 0xFF  # NaN codes behind the length
    cache = ref.to_cache(lens)
    got = cache.read(rows, dtype=dtype)
    for layer in range(L):
        for x, want in zip(got, ref.real(layer)):
            want = torch.nan_to_num(want[:, :, :rows])
            for b in range(B):
                want[b, :, lens[b]:] = 0
            want = want.transpose(1, 2).flatten(2).to(dtype)  # [B][rows][heads * D]
            assert torch.equal(x[:, layer].cpu(), want)
    assert cache.read(0)[0].shape == (B, L, 0, heads * D)


CASES = [  # B, T, H, Hkv, D, lens, block, causal
    (1, 1, 8, 1, 256, [1], 64, True), (2, 1, 8, 1, 256, [0, 63], 64, True), (1, 1, 8, 1, 256, [968], 64, True),
    (3, 1, 4, 2, 128, [64, 65, 700], 16, True), (2, 3, 6, 6, 96, [3, 130], 32, True), (2, 1, 8, 8, 64, [200, 17], 128, True),
    (2, 5, 10, 2, 256, [5, 300], 128, True), (1, 30, 8, 8, 96, [493], 16, False), (2, 50, 8, 1, 256, [1018, 60], 64, False),
    (1, 33, 16, 2, 64, [1500], 32, True), (2, 17, 3, 1, 128, [40, 257], 64, True), (1, 1, 32, 8, 128, [5000], 128, True),
    (1, 2, 17, 1, 64, [90], 16, False), (1, 130, 4, 1, 128, [260], 32, True), (1, 260, 1, 1, 256, [400], 64, True)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c[:5])))
def test_attention(require_gpu, case, dtype):
    B, T, H, heads, D, lens, block, causal = case
    cap = -(-max(lens) // block) * block + block
    ref = random_ref(B, 2, heads, D, cap, block, T + D)
    for b in range(B):  # NaN codes and scales behind the length
        ref.k[b, :, :, lens[b]:], ref.v[b, :, :, lens[b]:] = 0x7F, 0xFF
        dead = -(-lens[b] // block)
        ref.ks[b, ..., dead:], ref.vs[b, ..., dead:] = float("nan"), float("inf")
    q = _q((B, T, H, D), dtype, 9)
    clean = random_ref(B, 2, heads, D, cap, block, T + D)
    cache = ref.to_cache(lens)
    want, tol = attend(clean, 1, q, lens, causal=causal)
    for max_len in (0, max(lens)):
        got = cache.attend(1, q.cuda(), causal=causal, max_len=max_len)
        _check(got, want, tol)
    assert torch.equal(got, cache.attend(1, q.cuda(), causal=causal, max_len=max(lens)))  # the same bits again


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF])
def test_attention_masks(require_gpu, dtype):
    """Prefix masks, padded queries, queries without a key, lengths above max_len, a scale of its own."""
    B, T, H, heads, D = 5, 20, 4, 2, 64
    lens, q_lens, prefix = [100, 20, 7, 0, 64], [20, 1, 12, 3, 0], [50, 500, 0, 5, 64]
    ref = random_ref(B, 1, heads, D, 128, 16, 1)
    cache, q = ref.to_cache(lens), _q((B, T, H, D), dtype, 2)
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    out = torch.full((B, T, H, D), 7.0, dtype=dtype, device="cuda")
    want, tol = attend(ref, 0, q, lens, prefix=prefix, q_lens=q_lens, scale=0.3)
    got = cache.attend(0, q.cuda(), prefix=dev(prefix), q_lens=dev(q_lens), scale=0.3, out=out)
    assert got is out
    for b in range(B):
        _check(got[b, :q_lens[b]], want[b, :q_lens[b]], tol[b, :q_lens[b]])
        assert (got[b, q_lens[b]:] == 7.0).all()
    # twelve queries over seven tokens: five of them stand before the first key
    assert (got[2, :5] == 0).all() and (got[2, 5] != 0).any()
    want, tol = attend(ref, 0, q, [min(n, 50) for n in lens], causal=False)
    _check(cache.attend(0, q.cuda(), causal=False, max_len=50), want, tol)
    want, tol = attend(ref, 0, q, [3] * B, causal=False)
    _check(cache.attend(0, q.cuda(), causal=False, lens=dev([3] * B)), want, tol)


def _workspace(tokens, q_heads, cap, max_len=0, **kw):
    from flashact_b200 import _capi as C
    from flashact_b200.build import build
    n = ctypes.c_size_t()
    c = _desc(capacity=cap, **kw)
    assert C.load_library(build()).fa_kv8_attention_workspace(ctypes.byref(c), tokens, q_heads, max_len, ctypes.byref(n)) == 0
    return n.value


def test_workspace_follows_the_splits():
    """More than eight splits of the keys go through the merge kernel and a workspace; up to eight are a cluster."""
    one = dict(batch=1, layers=1, heads=1, head_dim=64)
    assert _workspace(1, 4, 1 << 16, **one) > 0 and _workspace(40, 4, 1 << 16, **one) > 0
    assert _workspace(1, 4, 1 << 16, max_len=1024, **one) == 0
    assert _workspace(1, 64, 1 << 15, batch=64, layers=1, heads=8, head_dim=128) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("T,H,D", [(1, 4, 64), (3, 4, 96), (40, 4, 64), (33, 4, 256)])
def test_attention_many_splits(require_gpu, T, H, D, dtype):
    """A long cache of one key head: splits joined by the merge kernel, some of them without a key; the captured call follows
    the lengths into other numbers of splits."""
    cap, lens, q_lens = 1 << 15, [20000, 130, 0], [T, T, max(1, T - 2)]
    assert _workspace(T, H, cap, batch=3, layers=1, heads=1, head_dim=D) > 0
    ref = random_ref(3, 1, 1, D, cap, 128, D)
    cache, q = ref.to_cache(lens), _q((3, T, H, D), dtype, 3)
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    ql, prefix, qc = dev(q_lens), dev([40, 0, 7]), q.cuda()
    out = torch.zeros(3, T, H, D, dtype=dtype, device="cuda")
    cache.attend(0, qc, q_lens=ql, prefix=prefix, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cache.attend(0, qc, q_lens=ql, prefix=prefix, out=out)
    for now in (lens, [700, 20, 5000]):
        cache.lens.copy_(dev(now))
        out.fill_(5.0)
        g.replay()
        want, tol = attend(ref, 0, q, now, prefix=[40, 0, 7], q_lens=q_lens)
        for b in range(3):
            _check(out[b, :q_lens[b]], want[b, :q_lens[b]], tol[b, :q_lens[b]])
            assert (out[b, q_lens[b]:] == 5.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,D", [(1, 8, 256), (40, 8, 64)])
def test_attention_layouts(require_gpu, T, H, D):
    """Queries and outputs with heads before tokens, odd pitches and 2-byte alignment."""
    B, heads, lens = 2, 1, [70, 131]
    ref = random_ref(B, 1, heads, D, 160, 32, 4)
    cache, q = ref.to_cache(lens), _q((B, T, H, D), BF, 5)
    want, tol = attend(ref, 0, q, lens)
    wide = torch.zeros(B, H, T, D + 5, dtype=BF, device="cuda")
    wide[..., 3:D + 3] = q.cuda().transpose(1, 2)
    out = torch.full((B, H, T, D + 7), 3.0, dtype=BF, device="cuda")
    cache.attend(0, wide[..., 3:D + 3].transpose(1, 2), out=out[..., 1:D + 1].transpose(1, 2))
    _check(out[..., 1:D + 1].transpose(1, 2), want, tol)
    assert (out[..., 0] == 3).all() and (out[..., D + 1:] == 3).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 40])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_attention_extremes(require_gpu, T, dtype):
    """One key that takes everything; scores far apart; block scales far apart; queries near the type's ends."""
    heads, H, D, n = 1, 8, 128, 600
    ref = random_ref(1, 1, heads, D, 640, 32, 6)
    ref.ks[0, 0, 0] = torch.exp2(torch.arange(20).float() % 7 - 12)
    ref.vs[0, 0, 0] = torch.exp2((torch.arange(20) * 5 % 19).float() - 15)
    cache = ref.to_cache([n])
    for loud in (30.0, 1e-6, 200.0):
        q = _q((1, T, H, D), dtype, 7, loud)
        want, tol = attend(ref, 0, q, [n], scale=2.0)
        _check(cache.attend(0, q.cuda(), scale=2.0), want, tol)
    q = _q((1, T, H, D), dtype, 8)
    q[0, 0, 3] = float("nan")
    got = cache.attend(0, q.cuda())
    assert torch.isnan(got[0, 0, 3]).all()  # and nothing else is touched by it
    q[0, 0, 3] = 0
    want, tol = attend(ref, 0, q, [n])
    got[0, 0, 3] = cache.attend(0, q.cuda())[0, 0, 3]
    _check(got, want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 40])
def test_attention_sink(require_gpu, T):
    """A first key that holds half the weight and 4096 others that share the rest, none of which may be lost."""
    heads, H, D, n = 1, 8, 64, 4097
    ref = Ref(1, 1, heads, D, 4160, 64)
    ref.ks.fill_(1.0), ref.vs.fill_(1.0)
    one = codes(torch.ones(1), 1.0).item()
    ref.k[0, 0, 0, 0, 0], ref.v[0, 0, 0, 1:, 1], ref.v[0, 0, 0, 0, 0] = one, one, one
    q = torch.zeros(1, T, H, D, dtype=BF)
    for s in (8.0, 12.0, 16.0):  # exp(s) against 4096 times 1
        q[..., 0] = s
        want, tol = attend(ref, 0, q, [n], scale=1.0, causal=False)
        _check(ref.to_cache([n]).attend(0, q.cuda(), scale=1.0, causal=False), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 24])
def test_graphs_and_streams(require_gpu, T):
    """Captured steps follow lengths and contents that change between replays; two graphs replayed at once."""
    from flashact_b200 import Kv8Cache
    B, heads, H, D, cap = 2, 1, 8, 256, 2048
    refs = [random_ref(B, 1, heads, D, cap, 64, s) for s in (1, 2)]
    caches = [r.to_cache([500, 900]) for r in refs]
    q, k, v = _q((B, T, H, D), BF, 1).cuda(), _q((B, T, heads, D), BF, 2).cuda(), _q((B, T, heads, D), BF, 3).cuda()
    graphs, outs = [], []
    for c in caches:
        c.attend(0, q)
    torch.cuda.synchronize()
    for c in caches:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.append(0, k, v)
            c.advance(T)
            outs.append(c.attend(0, q))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in caches]
    lens = [500, 900]
    for _ in range(3):
        for g, s in zip(graphs, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for r in refs:
            r.append(0, k.cpu(), v.cpu(), lens, [T] * B)
        lens = [n + T for n in lens]
        for c, r, o in zip(caches, refs, outs):
            assert c.lens.tolist() == lens
            _same(c, r)
            _check(o, *attend(r, 0, q.cpu(), lens))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = caches[0].attend(0, q, stream=side)
    side.synchronize()
    assert torch.equal(got, outs[0])
    assert isinstance(caches[0], Kv8Cache)


@pytest.mark.gpu
def test_offsets_past_32_bits(require_gpu):
    """More than 2^32 codes in K and in V: the last observation's last head, at the end of a long cache."""
    from flashact_b200 import Kv8Cache
    B, heads, D, cap = 3, 6, 256, 1 << 20
    c = Kv8Cache(B, 1, heads, D, cap, block=128)
    assert c.k.numel() > 1 << 32
    n = cap - 3
    k, v = torch.zeros(B, 2, heads, D, dtype=BF, device="cuda"), _q((B, 2, heads, D), BF, 1).cuda()
    c.lens.fill_(n - 2)
    c.append(0, k, v * 1000)
    c.advance(2)
    q = _q((B, 1, heads, D), BF, 2).cuda()
    got = c.attend(0, q)  # every key is zero: the mean of all values
    kk, vv = c.read(cap)
    s = vv[:, 0, n - 2:n].double().sum(1).view(B, 1, heads, D)
    assert (vv[:, 0, n:] == 0).all() and (kk == 0).all()
    want = s / n
    # probabilities are equal and exact in f16; two values each: output rounding and fp32 sums
    assert ((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -18 * s.abs() / n + 1e-12).all()
    want = codes(v.float().cpu() * 0 + (v * 1000).float().cpu(), 1.0)  # values came back through the cache
    assert want.shape == (B, 2, heads, D) and s.abs().max() > 0


@pytest.mark.gpu
def test_python_refusals(require_gpu):
    from flashact_b200 import FlashActError, Kv8Cache
    c = Kv8Cache(2, 1, 2, 64, 100, block=32)
    assert c.capacity == 128
    q, k = torch.zeros(2, 1, 4, 64, dtype=BF, device="cuda"), torch.zeros(2, 1, 2, 64, dtype=BF, device="cuda")
    i = torch.zeros(2, dtype=torch.int32, device="cuda")
    bad = [lambda: c.attend(1, q), lambda: c.attend(0, q.float()), lambda: c.attend(0, q[:1]), lambda: c.attend(0, q[..., :32]),
           lambda: c.attend(0, q[:, :, :3]), lambda: c.attend(0, q.cpu()), lambda: c.attend(0, q, lens=i.long()),
           lambda: c.attend(0, q, prefix=i, causal=False), lambda: c.attend(0, q, max_len=129),
           lambda: c.attend(0, q, out=q.half()), lambda: c.attend(0, q, q_lens=i.cpu()), lambda: c.attend(0, q, scale=float("nan")),
           lambda: c.append(0, k, k.float()), lambda: c.append(2, k, k), lambda: c.append(0, k[:, :, :1], k[:, :, :1]),
           lambda: c.append(0, k, torch.cat([k, k], 1)), lambda: c.append(0, k.cpu(), k.cpu()), lambda: c.append(0, k, k, count=i[:1]),
           lambda: c.read(-1), lambda: c.read(1, dtype=torch.int8), lambda: Kv8Cache(1, 1, 1, 80, 32).attend(0, q[:1, :, :1]),
           lambda: Kv8Cache.from_tensors(c.k, c.k, c.k_scale, c.v_scale),
           lambda: Kv8Cache.from_tensors(c.k, c.v, c.k_scale[..., :3], c.v_scale)]
    for f in bad:
        with pytest.raises((FlashActError, RuntimeError)):
            f()
    assert c.attend(0, q[:, :0]).shape == (2, 0, 4, 64)
    c.append(0, k[:, :0], k[:, :0])


@pytest.mark.gpu
def test_engines_bind_a_cache(require_gpu):
    """pi0.5 and MolmoAct2 sample the same actions from a cache as from the values read out of it."""
    from flashact_b200 import FlashActError, Kv8Cache, MolmoAct2ActionExpert
    from oracle import molmoact2_oracle as M
    from oracle import pi05_oracle as O
    from tests.pi05_util import engine_for
    c = O.make_case(seed=5, L=2, T=50, AD=32, Lp=200, B=2, num_steps=2)
    cache = Kv8Cache(2, 2, 1, 256, 200)
    for layer in range(2):
        cache.append(layer, c.k[:, layer, :, None].contiguous().cuda(), c.v[:, layer, :, None].contiguous().cuda(),
                     count=torch.tensor([200, 150], dtype=torch.int32, device="cuda"))
    cache.advance(torch.tensor([200, 150], dtype=torch.int32, device="cuda"))
    eng = engine_for(c)
    k, v = cache.read(200)
    eng.bind_prefix_kv(k, v, [200, 150])
    want = eng.sample_actions(c.noise.cuda())
    for lens in (None, [200, 150]):
        eng.bind_prefix_cache(cache, lens)
        assert torch.equal(eng.sample_actions(c.noise.cuda()), want)
    with pytest.raises(FlashActError):
        eng.bind_prefix_cache(Kv8Cache(2, 3, 1, 256, 200))
    with pytest.raises(FlashActError):
        eng.bind_prefix_cache(cache, [200, 300])
    eng.close()
    m = M.make_case(seed=12, L=2, T=30, Lk=96, B=1, num_steps=2)
    eng = MolmoAct2ActionExpert(m.w, m.mods, m.mod_final, num_layers=m.L, horizon=m.T, action_dim=m.AD,
                                valid_action_dim=m.adim, max_context=m.Lk, max_batch=1, num_steps=m.num_steps,
                                device=0, rope_cos=m.rope_cos, rope_sin=m.rope_sin)
    cache = Kv8Cache(1, 2, 8, 96, 96, block=32)
    for layer in range(2):
        cache.append(layer, m.kctx[:, layer].view(1, 96, 8, 96).cuda(), m.vctx[:, layer].view(1, 96, 8, 96).cuda())
    cache.advance(96)
    k, v = cache.read(96)
    eng.bind_context(k, v, [96])
    want = eng.sample_actions(m.noise.cuda())
    eng.bind_context_cache(cache)
    assert torch.equal(eng.sample_actions(m.noise.cuda()), want)
    eng.close()


@pytest.mark.gpu
def test_quantised_layer_step(require_gpu):
    """One decode step of a quantised attention layer as it is used: NVFP4 projections, append, attention, output
    projection; each stage against 64 bits on the stage's own inputs."""
    from flashact_b200 import Kv8Cache
    from flashact_b200.quant import nvfp4_linear, quantize_nvfp4
    from tests.test_nvfp4_linear import check_linear
    B, H, D, W = 4, 8, 256, 1024
    g = torch.Generator().manual_seed(11)
    w = {n: quantize_nvfp4((torch.randn(1, o, i, generator=g) * 0.02).cuda())
         for n, o, i in (("q", H * D, W), ("k", D, W), ("v", D, W), ("o", W, H * D))}
    lin = lambda x, n: nvfp4_linear(x, w[n][0][0], w[n][1][0], w[n][2])  # noqa: E731
    cache, ref, lens = Kv8Cache(B, 1, 1, D, 256), Ref(B, 1, 1, D, 256, 64), [0] * B
    prompt = torch.randn(B, 100, 1, D, generator=g).to(BF)
    count = [100, 64, 63, 1]
    cache.append(0, prompt.cuda(), prompt.cuda(), count=torch.tensor(count, dtype=torch.int32, device="cuda"))
    cache.advance(torch.tensor(count, dtype=torch.int32, device="cuda"))
    ref.append(0, prompt, prompt, lens, count)
    lens = list(count)
    h = torch.randn(B, W, generator=g).to(BF).cuda()
    for _ in range(3):
        q, k, v = lin(h, "q"), lin(h, "k"), lin(h, "v")
        for x, n in ((q, "q"), (k, "k"), (v, "v")):
            check_linear(x, h, *w[n])
        cache.append(0, k.view(B, 1, 1, D), v.view(B, 1, 1, D))
        ref.append(0, k.view(B, 1, 1, D).cpu(), v.view(B, 1, 1, D).cpu(), lens, [1] * B)
        cache.advance(1)
        lens = [n + 1 for n in lens]
        _same(cache, ref)
        o = cache.attend(0, q.view(B, 1, H, D))
        _check(o, *attend(ref, 0, q.view(B, 1, H, D).cpu(), lens))
        y = lin(o.view(B, H * D), "o")
        check_linear(y, o.view(B, H * D), *w["o"])
        h = h + y


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,dim", [(1, 256), (2, 128), (20, 64), (20, 256), (150, 128)])
def test_padding_of_any_content_and_in_place(tokens, dim):
    """Query rows behind q_lens may hold NaN and infinities, and the output may be the queries: the same bits, and the padding
    as it was."""
    c = _filled(2, 1, dim, 300, tokens)
    lens = torch.tensor([300, 7 + tokens], dtype=torch.int32, device="cuda")
    qn = torch.tensor([(tokens + 1) // 2, tokens], dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(tokens)
    q = torch.randn(2, tokens, 4, dim, generator=g).to(BF).cuda()
    want = c.attend(0, q, lens=lens, q_lens=qn)
    bad = q.clone()
    bad[0, (tokens + 1) // 2:, ::2] = float("nan")
    bad[0, (tokens + 1) // 2:, 1::2] = float("inf")
    before = bad.clone()
    c.attend(0, bad, lens=lens, q_lens=qn, out=bad)
    real = (tokens + 1) // 2
    assert torch.equal(bad[0, :real], want[0, :real]) and torch.equal(bad[1], want[1])
    assert torch.equal(bad[0, real:].view(torch.int16), before[0, real:].view(torch.int16))


def _filled(batch, heads, dim, n, seed):
    from flashact_b200 import Kv8Cache
    c = Kv8Cache(batch, 1, heads, dim, 512)
    g = torch.Generator().manual_seed(100 + seed)
    k, v = (torch.randn(batch, n, heads, dim, generator=g).to(BF).cuda() for _ in range(2))
    c.append(0, k, v)
    c.advance(n)
    return c
