"""Attention over the 8-bit KV cache in 64 bits, and how far a result may be off, by what a row itself sees."""
import torch

from tests.kv8_util import values

# Bits that the kernels keep of a probability times its V scale, and where they end, relative to the largest such product of the row
# (tests/test_kv8_values.py goes through the parts on the CPU).
#   P_REL: f16 holds eleven bits, and three E5M2 parts rounded to nearest hold all of them: half a step, 2^-11 of the product's leading power of
#          two. fp16 queries have a fourth part for what f16 lost, at most 2^-11, rounded to three bits: 2^-15.
#   p_abs: few rows: P holds the row's largest product at 2^11.25 or more; the third part's smallest step is 2^-16 / 64, the fourth's
#          2^-16 / 512, f16's own 2^-24; half of each: below 2^-22.6, under 2^-33 of the largest. More rows: the largest at 2^13.25 or more,
#          all parts in units of 1, half a step of 2^-16 for the third and for the fourth, f16's 2^-25: under 2^-29 of the largest.
P_REL = {torch.bfloat16: 2.0 ** -11, torch.float16: 2.0 ** -15}


def seen_by(lens, T, causal, prefix, q_lens):
    """Keys that each query token sees, -1 for padding: [B][T]."""
    out = torch.full((len(lens), T), -1, dtype=torch.long)
    for b, n in enumerate(lens):
        nq = T if q_lens is None else q_lens[b]
        for t in range(nq):
            out[b, t] = min(n, max(n - nq + t + 1, 0 if prefix is None else prefix[b], 0)) if causal else n
    return out


def attend(ref, layer, q, lens, *, causal=True, prefix=None, q_lens=None, scale=None):
    """(out, tol), both [B][T][H][D]; softmax(scale q K^T + mask) V of the cache `ref` (tests/kv8_util.py).

    The tolerance counts roundings, for each row by the keys that it sees alone. Output: half a step of q's type. Products p_j vs_j: P_REL and
    p_abs above. Scores: fp32 sums of D products off by (D + 8) 2^-23 of scale sum |q k| (the matrix unit truncates), queries given in parts off
    by 2^-17 of the row's largest element (few rows 2^-21), the exponential and the scales' logarithm by 2^-20 together: a share of p
    in numerator and sum."""
    B, T, H, D = q.shape
    k, v = ref.real(layer)
    heads = k.shape[1]
    group = H // heads
    scale = D ** -0.5 if scale is None else scale
    few = T * group <= 16
    p_rel = P_REL[q.dtype]
    p_abs, low_q = (2.0 ** -33, 2.0 ** -21) if few else (2.0 ** -29, 2.0 ** -17)
    u = torch.finfo(q.dtype).eps / 2
    see = seen_by(lens, T, causal, prefix, q_lens)
    out, tol = torch.zeros(B, T, H, D, dtype=torch.float64), torch.zeros(B, T, H, D, dtype=torch.float64)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        blk = torch.arange(n) // ref.block
        for h in range(heads):
            kk, vv = k[b, h, :n], v[b, h, :n]
            code, vs = values(ref.v[b, layer, h, :n]).abs(), ref.vs[b, layer, h].double()[blk]
            x = q[b, :, h * group:(h + 1) * group].double().transpose(0, 1)  # [group][T][D]
            mask = torch.arange(n) < see[b][:, None]
            live = (see[b] > 0)[None, :, None]
            s = (x @ kk.T * scale).masked_fill(~mask, -torch.inf)
            p = torch.softmax(s.masked_fill(~live, 0.0), -1) * mask
            big = (x.abs() @ kk.abs().T * abs(scale)).masked_fill(~mask, 0.0).amax(-1, keepdim=True)
            knorm = (kk.abs().sum(1) * mask).amax(-1)[None, :, None]
            floor = low_q * x.abs().amax(-1, keepdim=True) * knorm * abs(scale)
            o, spread = p @ vv, p @ vv.abs()
            faint = p_abs * (p * vs).amax(-1, keepdim=True) * (mask.double() @ code)
            e = u * o.abs() + (1 + u) * ((p_rel + 2 * ((D + 8) * 2.0 ** -23 * big + floor + 2.0 ** -20)) * spread + faint) + 1e-30
            out[b, :, h * group:(h + 1) * group] = (o * live).transpose(0, 1)
            tol[b, :, h * group:(h + 1) * group] = (e * live).transpose(0, 1)
    return out, tol


def check(got, want, tol):
    d = (got.cpu().double() - want).abs()
    assert torch.isfinite(got).all()
    assert (d <= tol).all(), (d.max().item(), (d / tol.clamp(min=1e-300)).max().item())
