"""The distribution operators of the LM head in 64 bits, with bounds on what the kernels may be off by.

Bounds. A logit's f32 accumulation adds d / 16 partial products one after the other, each addition
off by at most 2^-23 of a partial sum (<= sum |h w|); the softcap's exponential and reciprocal are
off by at most 2^-22 of the cap each, the change to base 2 and back by 2^-23 of the logit. Their sum
is ``delta``, the largest error of any logit of the row. From it:
  log-normaliser and log-probability   2 delta (one delta each) + 2^-22 (|z| + |log p| + 1)
  entropy                              sum p |log p + E| delta <= 2 E delta, + 2^-18 (E + 1) for the
                                       exponentials (2^-22 each) and the f32 sums
  dZ                                   its own rounding to bf16 (2^-8), and the relative error of p
                                       and of its factor (8 delta + 2^-18), of the magnitudes that
                                       enter it; and log p + E, which can cancel (to 0 where one token
                                       has all the mass), is off by the bounds of log p and of E,
                                       which p times the entropy's gradient carries into dZ. Logits kept
                                       in 16 bits are off by half a step, 24 ln2 / 65535, more (delta of
                                       dZ alone), and one more than 48 ln2 below the largest of its
                                       group has p up to 2^-48 of that one's. dH and dW
                                       sum these, and are rounded once more
"""

from __future__ import annotations

import torch


def _cap(x, c):
    return x if c is None else c * torch.tanh(x / c)


class Reference:
    def __init__(self, embed, hidden, softcap, kept=False):
        self.w, self.h, self.c = embed.double(), hidden.double(), softcap
        self.raw = self.h @ self.w.T
        self.z = _cap(self.raw, softcap)
        self.lse = torch.logsumexp(self.z, -1)
        self.logp = self.z - self.lse[:, None]
        self.p = self.logp.exp()
        self.entropy = -(self.p * self.logp).sum(-1)
        d = embed.shape[1]
        acc = (d / 16 + 4) * 2**-23 * (self.h.abs() @ self.w.abs().T).amax(-1)
        self.half_step = 24 * 0.6931471805599453 / 65535 if kept else 0.0
        self.floor = 2.0**-47 if kept else 0.0
        self.delta = acc + (2 * 2**-22 * softcap if softcap is not None else 0.0) + 2**-23 * self.z.abs().amax(-1)

    def picked(self, tokens):
        ok = (tokens >= 0) & (tokens < self.w.shape[0])
        return torch.where(ok, self.logp.gather(1, tokens.long() * ok), 0.0)

    def logp_bound(self, picked):
        return 2 * self.delta[:, None] + 2**-22 * (self.z.abs().amax(-1)[:, None] + picked.abs() + 1)

    def entropy_bound(self):
        return 2 * self.entropy * self.delta + 2**-18 * (self.entropy + 1)

    def grads(self, tokens, g, ge):
        """(dH, dW, bound of dH, bound of dW) for g [T, K] and ge [T] (None: no gradient)."""
        T, V = self.z.shape
        ok = (tokens >= 0) & (tokens < V)
        g = torch.zeros(tokens.shape, device=self.z.device, dtype=torch.float64) if g is None else g.double()
        g = torch.where(ok, g, 0.0)
        ge = torch.zeros(T, device=self.z.device, dtype=torch.float64) if ge is None else ge.double()
        hot = torch.zeros_like(self.z).scatter_add_(1, tokens.long() * ok, g)
        hot_abs = torch.zeros_like(self.z).scatter_add_(1, tokens.long() * ok, g.abs())
        G, G_abs = g.sum(-1, keepdim=True), g.abs().sum(-1, keepdim=True)
        slope = 1.0 if self.c is None else 1.0 - (self.z / self.c) ** 2
        E = self.entropy[:, None]
        dz = slope * (hot - self.p * (G + ge[:, None] * (self.logp + E)))
        # the slope itself is off by at most 4 * 2^-22 + 2 delta / c where it is near 0
        raw = hot_abs + self.p * (G_abs + ge[:, None].abs() * (self.logp.abs() + E))
        size = (slope + (0.0 if self.c is None else 2**-19)) * raw
        far = self.floor * (G_abs + ge[:, None].abs() * (40.0 + E))
        # p is off by delta + half a step of itself, log p by as much, and the slope, 1 - (z / c)^2, by
        # at most 2 / c of it whatever its own size
        off = (1.01 * 2**-8 + 8 * (self.delta[:, None] + self.half_step) + 2**-18) * size + far
        if self.c is not None:
            off = off + 2 / self.c * (self.delta[:, None] + self.half_step) * raw
        off = off + self.p * ge[:, None].abs() * (
            self.logp_bound(self.logp) + self.entropy_bound()[:, None] + self.half_step
        )
        # products and sums of the two gradient products in f32: far below the terms above
        bound = lambda ref, b: b + 1.01 * 2**-8 * ref.abs() + 1e-30  # noqa: E731
        dH, dW = dz @ self.w, dz.T @ self.h
        return dH, dW, bound(dH, off @ self.w.abs()), bound(dW, off.T @ self.h.abs())

    def order(self, k):
        key = torch.where(self.raw.isnan(), -torch.inf, self.raw)
        return key.sort(dim=-1, descending=True, stable=True).indices[:, :k]

    def draw(self, uniform, k, temperature, top_p):
        ids = self.order(k)
        best = self.z.gather(1, ids)
        w = ((best - best[:, :1]) / temperature).exp()
        upto = w.cumsum(-1)
        keep = upto - w < top_p * upto[:, -1:]
        keep[:, 0] = True
        kept = torch.where(keep, w, 0.0).cumsum(-1)
        place = (kept <= uniform.double()[:, None] * kept[:, -1:]).sum(-1)
        place = torch.minimum(place, keep.sum(-1) - 1)
        return ids.gather(1, place[:, None])[:, 0]


def within(got, ref, bound, what):
    got = got.detach()
    off = (got.double() - ref).abs()
    assert torch.isfinite(got).all(), what
    worst = float((off / bound).max()) if off.numel() else 0.0
    print(f"{what}: at most {worst:.3f} of its bound")
    assert worst <= 1.0, what
