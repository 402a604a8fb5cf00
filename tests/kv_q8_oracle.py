"""A cache in 8 bits from its definition, in 64 bits on the CPU."""
import math

import torch

MOST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def nearest(x: torch.Tensor, dtype) -> torch.Tensor:
    """Nearest code, ties to even."""
    if dtype == torch.int8:
        return torch.round(x)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def least_scale(top: float, dtype) -> float:
    return 2.0 ** max(-126, math.ceil(math.log2(top / MOST[dtype]))) if top > 0 else 2.0 ** -126


class Cache:
    """Codes [blocks, Hkv, bs, hd] and scales [blocks, Hkv] as float64."""

    def __init__(self, codes: torch.Tensor, scale: torch.Tensor):
        self.dtype, self.codes, self.scale = codes.dtype, codes.double().cpu(), scale.double().cpu()

    def write(self, x: torch.Tensor, slots: list[int]) -> None:
        _, kv, bs, hd = self.codes.shape
        x = x.double().cpu().view(-1, kv, hd)
        of: dict[int, list] = {}
        for row, s in enumerate(slots):
            if s >= 0:
                of.setdefault(s // bs, []).append((row, s % bs))
        for b, members in of.items():
            rows, places = [r for r, _ in members], [p for _, p in members]
            for h in range(kv):
                top, old = float(x[rows, h].abs().max()), float(self.scale[b, h])
                if not math.isfinite(top) or (0 not in places and math.isnan(old)):
                    self.scale[b, h] = math.nan
                    self.codes[b, h, places] = 0.0
                    continue
                f = least_scale(top, self.dtype)
                if 0 not in places:
                    if f > old:
                        self.codes[b, h] = nearest(self.codes[b, h] * (old / f), self.dtype)
                    f = max(f, old)
                self.codes[b, h, places] = nearest(x[rows, h] / f, self.dtype)
                self.scale[b, h] = f

    def tokens(self, slots) -> torch.Tensor:
        """Values [n, Hkv, hd] at ``slots``; zeros where negative."""
        _, kv, bs, hd = self.codes.shape
        s = torch.as_tensor(slots)
        t = s.clamp(min=0)
        v = self.codes[t // bs, :, t % bs] * self.scale[t // bs][..., None]
        return torch.where((s >= 0)[:, None, None], v, torch.zeros_like(v))


def attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, dtype=None):
    """``q`` [Hq, hd] over ``k``, ``v`` [n, Hkv, hd], all float64: the result [Hq, hd] and how far a kernel may be from it that
    takes products of exact operands into fp32 sums, rounds each weight to fp16 and the result to bf16; for codes of ``dtype`` int8
    one that first rounds a head's query to 16-bit whole numbers, the largest of which is at least 2^14."""
    Hq, hd = q.shape
    G, n = Hq // k.shape[1], k.shape[0]
    if n == 0:
        return torch.zeros_like(q), torch.zeros_like(q)
    k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    p = torch.softmax(torch.einsum("hd,nhd->hn", q, k) / math.sqrt(hd), -1)
    ref = torch.einsum("hn,nhd->hd", p, v)
    size = torch.einsum("hn,nhd->hd", p, v.abs())
    # a score is a sum of hd products, scaled: each of its hd + 4 roundings is within 2^-24 of the sum of magnitudes; the exponential
    # is good to 2^-21; numerator and denominator have both errors.  Sums over n keys: rounded n times in each of few orders, which
    # 2^-24 * n bounds.  A weight (at most 2^8 above the running reference, whose own is 1) below 2^-14 is rounded by 2^-25.
    score = (hd + 4) * 2.0 ** -24 * float((torch.einsum("hd,nhd->hn", q.abs(), k.abs()) / math.sqrt(hd)).max()) + 2.0 ** -21
    if dtype == torch.int8:
        # value i of a query is off by 1/2 where the largest is 2^14 or more, so by 2^-15 max|q|, and the score by the sum over i of
        # that times |k_i|
        score += 2.0 ** -15 * float((q.abs().amax(1)[:, None] * k.abs().sum(-1).T).max()) / math.sqrt(hd)
    weight = 2.0 ** -11 + 2 * score + 2 * n * 2.0 ** -24
    bound = 2.0 ** -8 * ref.abs() + 1.01 * weight * (size + ref.abs()) + 2.0 ** -25 * v.abs().sum(0)
    return ref, bound + 1e-30
