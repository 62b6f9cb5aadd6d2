"""Softmax attention in float64 and error bounds for it, for the tests of prompt and
shared-prefix attention."""

from __future__ import annotations

import torch


def unit(dtype) -> float:
    """Half a step of ``dtype`` relative to the value: the error of one rounding."""
    return torch.finfo(dtype).eps / 2


class Rows:
    """Attention of query rows ``q [n, Hq, D]`` over ``k``, ``v`` ``[m, H, D]`` where row i sees the first
    ``lims[i]`` keys: ``out``, ``lse`` (log2 units) and what their error bounds need."""

    def __init__(self, q, k, v, lims, scale):
        q, k, v = q.double(), k.double(), v.double()
        n, hq, d = q.shape
        m, h = k.shape[:2]
        gqa = hq // h
        ke, ve = k.repeat_interleave(gqa, 1), v.repeat_interleave(gqa, 1)  # [m, Hq, D]
        seen = torch.arange(m, device=q.device)[None] < torch.as_tensor(lims, device=q.device)[:, None]
        mask = seen[:, None, :]
        kt, vt = ke.permute(1, 2, 0).contiguous(), ve.permute(1, 0, 2).contiguous()
        qh = q.permute(1, 0, 2).contiguous()
        s = torch.matmul(qh, kt).permute(1, 0, 2) * scale  # [n, Hq, m]
        s = s.masked_fill(~mask, float("-inf"))
        top = s.amax(-1, keepdim=True) if m else s.new_full((n, hq, 1), float("-inf"))
        top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
        p = (s - top).exp().masked_fill(~mask, 0.0)
        tot = p.sum(-1, keepdim=True)
        w = torch.where(tot > 0, p / tot, torch.zeros_like(p)).permute(1, 0, 2).contiguous()
        self.out = torch.matmul(w, vt).permute(1, 0, 2)
        self.absv = torch.matmul(w, vt.abs()).permute(1, 0, 2)  # sum of weight x |value|
        self.lse = ((tot.log() + top) / torch.log(torch.tensor(2.0, dtype=torch.float64)))[..., 0]
        self.vmax = float(v.abs().max()) if m else 0.0
        self.sabs = float((torch.matmul(qh.abs(), kt.abs()) * abs(scale)).max()) if m else 0.0  # sum |q||k| x scale
        self.keys, self.d = m, d

    def score_error(self, operands: float = 0.0) -> float:
        """Bound of a score's absolute error: D products summed in float32, the scale, and
        ``operands`` of relative error in the products' factors."""
        return ((self.d + 8) * 2.0 ** -24 + operands) * self.sabs + 2.0 ** -22

    def bound(self, out_dtype, weight: float = 0.0, value: float = 0.0, operands: float = 0.0) -> torch.Tensor:
        """Bound of ``|out - exact|``: each weight within exp(2 ds) of its exact value (numerator
        and sum move by at most ds each), rounded to ``weight``, the values to ``value``; sums
        of at most ``keys`` float32 terms, numerator and denominator; the result rounded once."""
        ds = self.score_error(operands)
        rel = 2 * ds * (1 + ds) + weight + value + (self.keys + 64) * 2.0 ** -23 + 2.0 ** -20
        e = rel * self.absv
        return e + unit(out_dtype) * (self.out.abs() + e) + 1e-30

    def lse_bound(self, operands: float = 0.0) -> float:
        ds = self.score_error(operands)
        return 1.4427 * (ds * (1 + ds) + (self.keys + 64) * 2.0 ** -24) + 2.0 ** -20 * max(1.0, self.sabs)


def check(got, rows: Rows, **kw) -> None:
    d = (got.double() - rows.out).abs()
    b = rows.bound(got.dtype, **kw)
    worst = float((d / b).max())
    assert not torch.isnan(d).any() and worst <= 1.0, f"error {float(d.max())}, {worst} of its bound"
