"""What is measured of the quantised serving operators: the 8-bit KV cache (append, attention, read) and the
NVFP4 linear layer. Each has a plain form in elementary torch operations, the framework's call (`own`), its work in
bytes and operations, and its result in 64 bits (`exact`).

The cache of one layer: K codes E4M3 [batch][heads][capacity][head_dim], V codes transposed
[batch][heads][head_dim][capacity], and a power-of-two fp32 scale for each block of tokens and head, for K and for V
[batch][heads][capacity / block]. A value is its code times its block's scale.
"""
import math

import numpy as np
import torch

own = False

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ----------------------------------------------------------------------------------------------- cases
def attend(name, batch, tokens, q_heads, heads, head_dim, max_len, block, dtype, mask, ragged):
    return {"name": name, "op": "attend", "batch": batch, "tokens": tokens, "q_heads": q_heads, "heads": heads,
            "head_dim": head_dim, "max_len": max_len, "block": block, "dtype": dtype, "mask": mask, "ragged": ragged}


def append(name, batch, tokens, heads, head_dim, at, block, dtype, ragged):
    return {"name": name, "op": "append", "batch": batch, "tokens": tokens, "heads": heads, "head_dim": head_dim,
            "at": at, "block": block, "dtype": dtype, "ragged": ragged}


def read(name, batch, layers, heads, head_dim, max_len, block, dtype, ragged):
    return {"name": name, "op": "read", "batch": batch, "layers": layers, "heads": heads, "head_dim": head_dim,
            "max_len": max_len, "block": block, "dtype": dtype, "ragged": ragged}


def linear(name, m, n, k, dtype, bias):
    return {"name": name, "op": "linear", "m": m, "n": n, "k": k, "dtype": dtype, "bias": bias}


def listed():
    return [
        # one text token of one robot's prompt against its image + text prefix: latency only
        attend("attend_token_bs1", 1, 1, 8, 1, 256, 968, 64, "bf16", "causal", False),
        # one token for each of 64 observations with six cameras, prefixes of different lengths
        attend("attend_token_bs64", 64, 1, 8, 1, 256, 1736, 64, "bf16", "causal", True),
        # the action suffix of 16 observations over its prefix, every token seeing every other
        attend("attend_suffix_bs16", 16, 50, 8, 1, 256, 1018, 64, "bf16", "full", False),
        # a chunk of a long prompt: 1024 tokens seen by all, the rest causal; fp16
        attend("attend_chunk_fp16", 4, 256, 8, 1, 256, 4096, 128, "fp16", "prefix", True),
        # a long context in grouped heads, one token each: the cache's bytes alone count
        attend("attend_long", 8, 1, 32, 8, 128, 32768, 128, "bf16", "causal", False),
        # one new token for each of 64 observations, in the middle of a block
        append("append_token_bs64", 64, 1, 1, 256, 1300, 64, "bf16", True),
        # 16 prompts at once, of different lengths in one padded batch
        append("append_prompt_bs16", 16, 1736, 8, 128, 0, 64, "bf16", True),
        # one observation's prefix of all 18 layers, for the action expert's bind
        read("read_bind_bs1", 1, 18, 1, 256, 968, 64, "bf16", False),
        # cross-attention contexts of 32 observations (8 heads of 96), six layers at a time
        read("read_context_bs32", 32, 6, 8, 96, 493, 16, "bf16", True),
        # a QKV projection of one token: the smallest call
        linear("linear_qkv_m1", 1, 2560, 1024, "bf16", False),
        # a gate/up projection of eight tokens
        linear("linear_gate_up_m8", 8, 32768, 2048, "bf16", False),
        # a wide MLP's matrix for sixteen tokens, with a bias
        linear("linear_wide_m16", 16, 28672, 8192, "fp16", True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "read", "linear", "linear"])
    if op == "linear":
        while True:
            c = linear("", _log(rng, 1, 16), _log(rng, 100, 32768), 16 * _log(rng, 4, 768),
                       rng.choice(["bf16", "fp16"]), rng.random() < 0.5)
            if c["n"] * c["k"] <= 28672 * 8192:
                break
    else:
        q_heads, heads, head_dim = rng.choice([(8, 1, 256), (8, 8, 96), (32, 8, 128), (16, 2, 64), (12, 4, 128),
                                               (10, 2, 256), (6, 6, 64)])
        block = rng.choice([16, 32, 64, 128])
        batch = _log(rng, 1, 64)
        if op == "attend":
            while True:
                tokens = rng.choice([1, 1, _log(rng, 2, 64), _log(rng, 16, 256)])
                c = attend("", batch, tokens, q_heads, heads, head_dim, max(tokens, _log(rng, 20, 32768)), block,
                           rng.choice(["bf16", "bf16", "fp16"]), rng.choice(["causal", "prefix", "full"]),
                           rng.random() < 0.7)
                w = work(c)
                if w["bytes"] <= 5e8 and w["flops"] <= 3e10:
                    break
        elif op == "append":
            while True:
                tokens = rng.choice([1, _log(rng, 2, 64), _log(rng, 64, 1736)])
                c = append("", batch, tokens, heads, head_dim, rng.choice([0, rng.randrange(1, 2000)]), block,
                           rng.choice(["bf16", "fp16", "fp32"]), rng.random() < 0.7)
                if work(c)["bytes"] <= 1.6e8:
                    break
        else:
            while True:
                c = read("", batch, _log(rng, 1, 36), heads, head_dim, _log(rng, 20, 2000), block,
                         rng.choice(["bf16", "bf16", "fp16", "fp32"]), rng.random() < 0.7)
                if work(c)["bytes"] <= 3.5e8:
                    break
    del c["name"]
    return c


def _spread(n, top, low):
    """n whole numbers from low to top, in no order: the lengths of a ragged batch, the same for every seed."""
    return [low + int((top - low) * ((0.999 + 0.618034 * i) % 1.0) + 0.5) for i in range(n)]


def _lens(c):
    if c["op"] == "append":  # (rows already there, new rows) of each observation
        at = [c["at"]] * c["batch"] if not c["ragged"] or not c["at"] else _spread(c["batch"], c["at"], c["at"] // 2)
        new = _spread(c["batch"], c["tokens"], (c["tokens"] + 1) // 2) if c["ragged"] else [c["tokens"]] * c["batch"]
        return at, new
    low = max(c.get("tokens", 1), c["max_len"] // 2)
    return _spread(c["batch"], c["max_len"], low) if c["ragged"] else [c["max_len"]] * c["batch"]


def _capacity(c):
    top = c["at"] + c["tokens"] if c["op"] == "append" else c["max_len"]
    return -(-top // c["block"]) * c["block"]


def _prefix(c, lens):
    """Keys that every query sees, whatever its own position."""
    return [n // 4 for n in lens] if c["mask"] == "prefix" else [0] * len(lens)


def work(c):
    if c["op"] == "linear":
        e = 2
        return {"bytes": c["n"] * (c["k"] // 2 + c["k"] // 16) + e * c["m"] * (c["k"] + c["n"])
                + 4 * c["n"] * bool(c["bias"]), "flops": 2 * c["m"] * c["n"] * c["k"]}
    e, hd = torch.finfo(DT[c["dtype"]]).bits // 8, c["heads"] * c["head_dim"]
    if c["op"] == "append":
        at, new = _lens(c)
        return {"bytes": sum(new) * hd * 2 * (e + 1) + sum(-(-(a + n) // c["block"]) - a // c["block"]
                                                           for a, n in zip(at, new)) * c["heads"] * 8,
                "flops": 4 * sum(new) * hd}
    lens = _lens(c)
    cache = sum(2 * n * hd + 8 * c["heads"] * -(-n // c["block"]) for n in lens)
    if c["op"] == "read":
        rows = c["batch"] * c["max_len"]
        return {"bytes": c["layers"] * (cache + 2 * rows * hd * e), "flops": 2 * c["layers"] * sum(lens) * hd}
    pairs = 0  # visible (query, key) pairs
    for n, p in zip(lens, _prefix(c, lens)):
        if c["mask"] == "full":
            pairs += c["tokens"] * n
        else:
            pairs += sum(max(n - c["tokens"] + i + 1, p) for i in range(c["tokens"]))
    return {"bytes": cache + 2 * e * c["batch"] * c["tokens"] * c["q_heads"] * c["head_dim"],
            "flops": 4 * pairs * c["q_heads"] * c["head_dim"]}


# ---------------------------------------------------------------------------------------------- inputs
def _scale_of(amax):
    """The smallest power of two that brings amax to at most 448, no smaller than 2^-96."""
    m, x = torch.frexp(amax)  # amax = m 2^x, m in [0.5, 1)
    e = torch.where(m <= 0.875, x - 9, x - 8)
    e = torch.where(amax > 0, e, -96).clamp(min=-96)
    return torch.ldexp(torch.ones_like(amax), e)


def _cache(g, c, shape, cap, lens):
    """Codes and scales of shape + [cap][head_dim] tokens: heads and blocks of different loudness, a few loud channels of
    K, as a trained model's; rows at and behind each observation's length are zero."""
    d, block, dev = c["head_dim"], c["block"], "cuda"
    live = torch.arange(cap, device=dev) < torch.tensor(lens, device=dev)[:, None]  # [batch][cap]
    live = live.view(live.shape[0], *[1] * (len(shape) - 1), cap, 1)
    made = []
    for loud in (True, False):
        x = torch.randn(*shape, cap, d, generator=g, device=dev)
        x *= torch.exp2(torch.randn(*shape, 1, 1, generator=g, device=dev))
        if loud:
            x *= 1 + 3 * (torch.rand(*shape, 1, d, generator=g, device=dev) < 0.03)
        x *= live
        s = _scale_of(x.view(*shape, cap // block, block * d).abs().amax(-1))
        x /= s.repeat_interleave(block, -1)[..., None]
        made.append((x.to(torch.float8_e4m3fn).view(torch.uint8), s))
    (k, ks), (v, vs) = made
    return k.contiguous(), v.transpose(-1, -2).contiguous(), ks.contiguous(), vs.contiguous()


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev, dt = "cuda", DT[c["dtype"]]
    if c["op"] == "linear":
        m, n, k = c["m"], c["n"], c["k"]
        s = {"x": torch.randn(m, k, generator=g, device=dev).to(dt),
             "codes": torch.randint(0, 256, (n, k // 2), generator=g, device=dev, dtype=torch.uint8),
             # block scales of weights N(0, 0.02): within a factor of a few of each other
             "bscale": (torch.exp2(torch.randn(n, k // 16, generator=g, device=dev) * 0.5) * 64)
             .to(torch.float8_e4m3fn).view(torch.uint8),
             "tscale": torch.rand(1, generator=g, device=dev) * 1e-4 + 1e-4,
             "bias": torch.randn(n, generator=g, device=dev) if c["bias"] else None}
        return {"case": c, **s}
    batch, heads, d, cap = c["batch"], c["heads"], c["head_dim"], _capacity(c)
    layers = c.get("layers", 1)
    lens = _lens(c)
    there = lens[0] if c["op"] == "append" else lens
    k, v, ks, vs = _cache(g, c, (batch, layers, heads), cap, there)
    s = {"case": c, "k": k, "v": v, "ks": ks, "vs": vs, "lens": torch.tensor(there, dtype=torch.int32, device=dev)}
    if own:
        from flashact_b200 import Kv8Cache
        s["cache"] = Kv8Cache.from_tensors(k, v, ks, vs, lens=s["lens"])
    if c["op"] == "append":
        for n in ("new_k", "new_v"):
            s[n] = torch.randn(batch, c["tokens"], heads, d, generator=g, device=dev).mul_(2).to(dt)
        s["count"] = torch.tensor(lens[1], dtype=torch.int32, device=dev) if c["ragged"] else None
    elif c["op"] == "attend":
        # queries that make a few keys matter: scores of a few units
        s["q"] = torch.randn(batch, c["tokens"], c["q_heads"], d, generator=g, device=dev).mul_(0.7).to(dt)
        s["prefix"] = (torch.tensor(_prefix(c, lens), dtype=torch.int32, device=dev)
                       if c["mask"] == "prefix" else None)
    return s


# ------------------------------------------------------------------------------------------------- run
def run(s):
    return RUN[s["case"]["op"]](s)


def _run_linear(s):
    if own:
        from flashact_b200.quant import nvfp4_linear
        return nvfp4_linear(s["x"], s["codes"], s["bscale"], s["tscale"], bias=s["bias"])
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=s["x"].device)
    codes = torch.stack([s["codes"] & 15, s["codes"] >> 4], -1).int().flatten(1)
    w = table[codes] * s["bscale"].view(torch.float8_e4m3fn).float().repeat_interleave(16, 1)
    y = (s["x"].float() @ w.t()) * s["tscale"]
    return (y if s["bias"] is None else y + s["bias"]).to(s["x"].dtype)


def _run_attend(s):
    c = s["case"]
    if own:
        return s["cache"].attend(0, s["q"], causal=c["mask"] != "full", prefix=s["prefix"], max_len=c["max_len"])
    n, block = c["max_len"], c["block"]
    value = lambda codes: codes.view(torch.float8_e4m3fn).float()  # noqa: E731
    ks, vs = (s[x][:, 0].repeat_interleave(block, -1)[..., :n, None] for x in ("ks", "vs"))
    k = value(s["k"][:, 0, :, :n]) * ks
    v = value(s["v"][:, 0, :, :, :n]).transpose(-1, -2) * vs
    b, t, h, d = s["q"].shape
    q = s["q"].float().view(b, t, c["heads"], h // c["heads"], d).permute(0, 2, 1, 3, 4).flatten(2, 3)
    score = (q @ k.transpose(-1, -2)) * d ** -0.5  # [b][heads][t * group][n]
    key, lens = torch.arange(n, device=k.device), s["lens"].long()
    see = (key < lens[:, None])[:, None, :].expand(b, t, n)
    if c["mask"] != "full":
        at = lens[:, None] - t + torch.arange(t, device=k.device)
        first = s["prefix"].long() if s["prefix"] is not None else torch.zeros_like(lens)
        see = see & ((key <= at[..., None]) | (key < first[:, None, None]))
    see = see.repeat_interleave(h // c["heads"], 1)[:, None]
    score = score.masked_fill(~see, -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    o = (p @ v) / p.sum(-1, keepdim=True)
    return o.view(b, c["heads"], t, h // c["heads"], d).permute(0, 2, 1, 3, 4).reshape(b, t, h, d).to(s["q"].dtype)


def _run_append(s):
    c = s["case"]
    if own:
        s["cache"].append(0, s["new_k"], s["new_v"], count=s["count"])
    else:
        _plain_append(s, c)
    return {"k": s["k"].view(torch.float8_e4m3fn), "v": s["v"].view(torch.float8_e4m3fn), "k_scale": s["ks"],
            "v_scale": s["vs"]}


def _plain_append(s, c):
    b, t, block, cap = c["batch"], c["tokens"], c["block"], _capacity(c)
    start = s["lens"].long()
    end = start + (s["count"].long() if s["count"] is not None else t)
    touched = (t + block - 2) // block + 1  # blocks that t rows can reach
    blk = start[:, None] // block + torch.arange(touched, device=start.device)
    pos = (blk[..., None] * block + torch.arange(block, device=start.device)).flatten(1)  # [b][touched * block]
    real = pos < cap
    pos_in, row = pos.clamp(max=cap - 1), torch.arange(b, device=start.device)[:, None]
    blk_in = blk.clamp(max=cap // block - 1)
    old, new = pos < start[:, None], (pos >= start[:, None]) & (pos < end[:, None])
    src = (pos - start[:, None]).clamp(0, t - 1)
    keep = real & (pos < end[:, None]) & (blk * block < end[:, None]).repeat_interleave(block, 1)
    for codes, scale, rows, vt in ((s["k"], s["ks"], s["new_k"], False), (s["v"], s["vs"], s["new_v"], True)):
        at = codes[:, 0].transpose(-1, -2) if vt else codes[:, 0]  # [b][heads][cap][d]
        was = at[row, :, pos_in]  # [b][p][heads][d]
        fresh = rows[row, src].float()
        amax = torch.where(new[..., None, None], fresh, 0).abs().view(b, touched, block, c["heads"], -1)
        need = _scale_of(amax.amax((2, 4)))  # [b][touched][heads]
        had = scale[:, 0].transpose(-1, -2)[row, blk_in]
        has_old = (blk * block < start[:, None])[..., None]
        now = torch.where(has_old, torch.maximum(had, need), need)
        spread = lambda x: x.repeat_interleave(block, 1)[..., None]  # noqa: E731
        held = was.view(torch.float8_e4m3fn).float() * (spread(had) / spread(now))
        value = torch.where(old[..., None, None], held, fresh / spread(now))
        out = torch.where(keep[..., None, None], value.to(torch.float8_e4m3fn).view(torch.uint8), was)
        i = keep.nonzero(as_tuple=True)
        at[i[0], :, pos_in[i]] = out[i]
        j = (blk * block < end[:, None]).nonzero(as_tuple=True)
        scale[:, 0].transpose(-1, -2)[j[0], blk_in[j]] = now[j]


def _run_read(s):
    c = s["case"]
    if own:
        return s["cache"].read(c["max_len"], dtype=DT[c["dtype"]])
    n = c["max_len"]
    live = (torch.arange(n, device=s["k"].device) < s["lens"][:, None])[:, None, None, :, None]
    out = []
    for codes, scale in ((s["k"], s["ks"]), (s["v"].transpose(-1, -2), s["vs"])):
        x = codes[:, :, :, :n].view(torch.float8_e4m3fn).float() * scale.repeat_interleave(c["block"], -1)[..., :n, None]
        x = torch.where(live, x, 0).to(DT[c["dtype"]])
        out.append(x.transpose(2, 3).flatten(3))  # [batch][layers][n][heads * head_dim]
    return tuple(out)


RUN = {"linear": _run_linear, "attend": _run_attend, "append": _run_append, "read": _run_read}


# ----------------------------------------------------------------------------------------------- exact
def _e4m3_values():
    """The 256 values of E4M3, from its definition: sign, 4 exponent bits (bias 7), 3 mantissa bits, no infinities."""
    got = []
    for code in range(256):
        e, m = code >> 3 & 15, code & 7
        x = math.ldexp(m, -9) if e == 0 else math.ldexp(8 + m, e - 10)
        got.append(math.nan if code & 127 == 127 else -x if code & 128 else x)
    return torch.tensor(got, dtype=torch.float64, device="cuda")


def exact(c, seed):
    s = prepare(c, seed)
    table = _e4m3_values()
    if c["op"] == "linear":
        fp4 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
        fp4 = torch.tensor(fp4 + [-x for x in fp4], dtype=torch.float64, device="cuda")
        y = torch.empty(c["m"], c["n"], dtype=torch.float64, device="cuda")
        x = s["x"].double()
        for i in range(0, c["n"], 4096):
            codes = s["codes"][i:i + 4096].long()
            w = torch.empty(codes.shape[0], c["k"], dtype=torch.float64, device="cuda")
            w[:, 0::2], w[:, 1::2] = fp4[codes % 16], fp4[codes // 16]
            w.view(-1, c["k"] // 16, 16).mul_(table[s["bscale"][i:i + 4096].long()][..., None])
            y[:, i:i + 4096] = x @ w.T
        y *= s["tscale"].double()
        return y if s["bias"] is None else y + s["bias"].double()
    if c["op"] == "append":
        return _exact_append(c, s, table)
    if c["op"] == "read":
        b, layers, heads, n, d = c["batch"], c["layers"], c["heads"], c["max_len"], c["head_dim"]
        out = [torch.zeros(b, layers, n, heads, d, dtype=torch.float64, device="cuda") for _ in range(2)]
        blk = torch.arange(n, device="cuda") // c["block"]
        for i, length in enumerate(s["lens"].tolist()):
            k = table[s["k"][i].long()][:, :, :n] * s["ks"][i].double()[..., blk, None]
            v = table[s["v"][i].long()][..., :n] * s["vs"][i].double()[..., None, blk]
            out[0][i, :, :length] = k.permute(0, 2, 1, 3)[:, :length]
            out[1][i, :, :length] = v.permute(0, 3, 1, 2)[:, :length]
        return tuple(x.flatten(3) for x in out)
    # softmax(q k / sqrt(d)) v, one observation and key head at a time
    b, t, h, d = s["q"].shape
    group = h // c["heads"]
    y = torch.zeros(b, t, h, d, dtype=torch.float64, device="cuda")
    prefix = _prefix(c, s["lens"].tolist())
    for i, n in enumerate(s["lens"].tolist()):
        j = torch.arange(n, device="cuda")
        seen = torch.ones(t, n, dtype=torch.bool, device="cuda")
        if c["mask"] != "full":
            seen = (j <= (n - t + torch.arange(t, device="cuda"))[:, None]) | (j < prefix[i])
        for kv in range(c["heads"]):
            k = table[s["k"][i, 0, kv, :n].long()] * s["ks"][i, 0, kv].double()[j // c["block"], None]
            v = table[s["v"][i, 0, kv, :, :n].long()] * s["vs"][i, 0, kv].double()[j // c["block"]]
            for r in range(kv * group, (kv + 1) * group):
                a = s["q"][i, :, r].double() @ k.T / math.sqrt(d)
                a[~seen] = -math.inf
                y[i, :, r] = torch.softmax(a, -1) @ v.T
    return y


def _nearest_code(x):
    """Codes of the E4M3 values nearest to x (|x| <= 448), ties to the even code; numpy, 64 bits."""
    grid = np.array([math.ldexp(m, -9) for m in range(8)] + [math.ldexp(8 + m, e - 10) for e in range(1, 16)
                                                             for m in range(8)])[:127]
    a = np.abs(x)
    i = np.clip(np.searchsorted(grid, a), 1, 126)
    low, high = grid[i - 1], grid[i]
    up = (a - low > high - a) | ((a - low == high - a) & (i % 2 == 0))
    return np.where(up, i, i - 1) + 128 * np.signbit(x)


def _exact_append(c, s, table):
    b, t, heads, block = c["batch"], c["tokens"], c["heads"], c["block"]
    if b * t * heads * c["head_dim"] > 1 << 25:
        return None
    values = table.cpu().numpy()
    start = s["lens"].tolist()
    count = s["count"].tolist() if s["count"] is not None else [t] * b
    out = {}
    for name, codes, scale, rows in (("k", s["k"], s["ks"], s["new_k"]), ("v", s["v"].transpose(-1, -2), s["vs"], s["new_v"])):
        got, sc = codes[:, 0].cpu().numpy().copy(), scale[:, 0].double().cpu().numpy().copy()  # [b][heads][cap][d]
        new = rows.double().cpu().numpy().transpose(0, 2, 1, 3)
        for i in range(b):
            first, end = start[i], start[i] + count[i]
            for n in range(first // block, -(-end // block)):
                lo, hi = max(first, n * block), min(end, (n + 1) * block)
                fresh = new[i, :, lo - first:hi - first]
                amax = np.abs(fresh).max((1, 2))
                need = np.array([2.0 ** max(-96, math.ceil(math.log2(a / 448))) if a > 0 else 2.0 ** -96 for a in amax])
                if n * block < first:  # rows that are there keep their values, on the larger scale
                    was = got[i, :, n * block:first]
                    need = np.maximum(need, sc[i, :, n])
                    got[i, :, n * block:first] = _nearest_code(values[was] * (sc[i, :, n] / need)[:, None, None])
                got[i, :, lo:hi] = _nearest_code(fresh / need[:, None, None])
                sc[i, :, n] = need
        x = values[got][:, None]
        out[name] = torch.from_numpy(x if name == "k" else x.swapaxes(-1, -2).copy())
        out[name + "_scale"] = torch.from_numpy(sc[:, None])
    return out
