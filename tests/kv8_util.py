"""64-bit restatements of the 8-bit KV cache's operators, on the CPU, and the tolerances of their tests."""
import math

import torch

F8 = torch.float8_e4m3fn


def scale_of(amax):
    """Smallest power of two s >= 2^-96 with amax <= 448 s."""
    s = 2.0 ** -96
    if amax > 448 * s:
        s = 2.0 ** math.ceil(math.log2(amax / 448))
        s = s * 2 if amax > 448 * s else s / 2 if amax <= 224 * s else s
    return s


def codes(x, s):
    """E4M3 codes (uint8) of x / s: nearest even, saturating, NaN as 0. x, s fp32."""
    y = torch.nan_to_num(x.double() / s, nan=0.0, posinf=448.0, neginf=-448.0).clamp(-448, 448)
    return y.float().to(F8).view(torch.uint8)  # x / 2^e is exact in fp32 but where it is far below the smallest code


def values(c):
    return c.view(F8).double()


class Ref:
    """A cache on the CPU: k, v codes [B][L][heads][cap][D] (v not transposed), scales fp32 [B][L][heads][blocks]."""

    def __init__(self, B, L, heads, D, cap, block):
        self.shape, self.block = (B, L, heads, cap, D), block
        self.k, self.v = (torch.zeros(self.shape, dtype=torch.uint8) for _ in range(2))
        self.ks, self.vs = (torch.full((B, L, heads, cap // block), 2.0 ** -96) for _ in range(2))

    def append(self, layer, k, v, start, count):
        cap, block = self.shape[3], self.block
        for c, s, new in ((self.k, self.ks, k), (self.v, self.vs, v)):
            for b in range(self.shape[0]):
                lo = min(max(start[b], 0), cap)
                hi = lo + min(max(count[b], 0), new.shape[1], cap - lo)
                for h in range(self.shape[2]):
                    for blk in range(lo // block, -(-hi // block)) if hi > lo else ():
                        i, j = max(lo, blk * block), min(hi, (blk + 1) * block)
                        x = new[b, i - lo:j - lo, h].float()
                        fin = torch.where(torch.isfinite(x), x, torch.zeros_like(x)).abs()
                        now, had = scale_of(fin.max().item()), s[b, layer, h, blk].item()
                        if i > blk * block:
                            now = max(now, had)
                            old = values(c[b, layer, h, blk * block:i]) * had
                            c[b, layer, h, blk * block:i] = codes(old.float(), now)
                        c[b, layer, h, i:j] = codes(x, now)
                        s[b, layer, h, blk] = now

    def to_cache(self, lens=None):
        from flashact_b200 import Kv8Cache
        return Kv8Cache.from_tensors(self.k.cuda(), self.v.transpose(-1, -2).contiguous().cuda(), self.ks.cuda(), self.vs.cuda(),
                                     lens=None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda"))

    def real(self, layer):
        blk = torch.arange(self.shape[3]) // self.block
        return (values(self.k[:, layer]) * self.ks[:, layer].double()[..., blk, None],
                values(self.v[:, layer]) * self.vs[:, layer].double()[..., blk, None])


def random_ref(B, L, heads, D, cap, block, seed):
    g = torch.Generator().manual_seed(seed)
    r = Ref(B, L, heads, D, cap, block)
    for c, s in ((r.k, r.ks), (r.v, r.vs)):
        x = torch.randn(r.shape, generator=g)
        c.copy_((x * 100).clamp(-448, 448).to(F8).view(torch.uint8))
        s.copy_(torch.exp2(torch.randint(-9, -5, s.shape, generator=g).float()))
    return r


def attend(ref, layer, q, lens, *, causal=True, prefix=None, q_lens=None, scale=None):
    """(out, tol): softmax(scale q K^T + mask) V in 64 bits and how far a result may be off, both [B][T][H][D].

    The tolerance counts roundings. Output: half a step of q's type, u |o|. Probabilities: rounded to eight bits
    (bf16 queries) or eleven (fp16) before the product, so each p_j is off by at most w p_j, and the output by
    w sum p |v| / sum p. Scores: fp32 sums of D products are off by at most (D + 8) 2^-23 of scale * sum |q k|
    (the matrix unit truncates), 2^x by 2^-21 of its result: p_j is off by that share, in numerator and sum.
    Smallest probabilities: up to 16 rows of a key head (few), P is held as p_j 2^12 vs_j / max vs in f16 (steps of 2^-24 at
    the small end, half of one is 2^-25) and from there in E5M2 parts, the third in units of 1/64 (steps of 2^-16, half of one
    is 2^-17 / 64 = 2^-23): together each is off by at most 2^-22 whatever its size, which is 2^-34 of the largest. More rows: p_j 2^14
    and parts in the same units: 2^-17 + 2^-25 < 2^-16, which is 2^-30 of the largest. The output is off by that times
    sum max vs |code_j| / sum 2^(s_j - max s), the sum being relative to a maximum no larger than the true one.
    Smallest query elements: parts of a row whose largest element is brought to [128, 256) end at E4M3's steps of 2^-9, half
    of one 2^-10, for few rows in units of 1/16: an element is off by 2^-17 (few: 2^-21) of the row's largest, and a score by
    that times sum |k|."""
    B, T, H, D = q.shape
    k, v = ref.real(layer)
    heads = k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    u = torch.finfo(q.dtype).eps / 2
    few = T * (H // heads) <= 16
    low_p, low_q = (2.0 ** -34, 2.0 ** -21) if few else (2.0 ** -30, 2.0 ** -17)
    w = 2.0 ** -8 if q.dtype == torch.bfloat16 else 2.0 ** -11
    out, tol = torch.zeros(B, T, H, D, dtype=torch.float64), torch.zeros(B, T, H, D, dtype=torch.float64)
    for b in range(B):
        n, nq = lens[b], T if q_lens is None else q_lens[b]
        for h in range(H):
            kk, vv = k[b, h * heads // H, :n], v[b, h * heads // H, :n]
            for t in range(nq):
                see = min(n, max(n - nq + t + 1, 0 if prefix is None else prefix[b], 0)) if causal else n
                if see == 0:
                    continue
                x = q[b, t, h].double()
                s = kk[:see] @ x * scale
                p = torch.softmax(s, 0)
                big = ((kk[:see].abs() @ x.abs()) * abs(scale)).max().item()
                out[b, t, h] = p @ vv[:see]
                floor = low_q * x.abs().max().item() * kk[:see].abs().sum(1).max().item() * abs(scale)
                spread = p @ vv[:see].abs()
                blk = -(-see // ref.block)
                faint = low_p * ref.vs[b, layer, h * heads // H, :blk].max().item() * p.max() * \
                    values(ref.v[b, layer, h * heads // H, :see]).abs().sum(0)  # 1 / sum 2^(s_j - max s) = the largest p
                tol[b, t, h] = u * out[b, t, h].abs() + (w * (1 + u) + 2 * ((D + 8) * 2.0 ** -23 * big + floor + 2.0 ** -20)) * spread + faint + 1e-30
    return out, tol
