"""The cache operators' definitions in 64 bits on the CPU, written for checking: dense
products, no blocks, no running maximum.  Everything is [B, H, T, D] (bhsd)."""

import math
from fractions import Fraction

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # half a step, relative
PI = Fraction(314159265358979323846264338327950288419716939937510582097494459, 10 ** 62)


def own_keep(B, Hq, Tq, Tk, lengths, mask, causal):
    keep = torch.ones((B, Hq, Tq, Tk), dtype=torch.bool)
    if lengths is not None:
        keep &= (torch.arange(Tk) < lengths.clamp(0, Tk).view(B, 1, 1, 1))
    if causal:
        keep &= torch.ones((Tq, Tk), dtype=torch.bool).tril()
    if mask is not None:
        keep &= mask
    return keep


class Attention:
    """All of one softmax over a prefix and own keys; p [B, Hq, Tq, Tp + Tk]."""

    def __init__(self, q, k, v, pk=None, pv=None, lengths=None, mask=None, score=None, scale=None, causal=False):
        B, Hq, Tq, D = q.shape
        Hk, Tk = k.shape[1], k.shape[2]
        G = Hq // Hk
        self.scale = D ** -0.5 if scale is None else scale
        self.G, self.Tp, self.Tk = G, 0 if pk is None else pk.shape[2], Tk
        keep = own_keep(B, Hq, Tq, Tk, lengths, mask, causal)
        # memory past the lengths may hold anything
        there = own_keep(B, 1, 1, Tk, lengths, None, False)[:, :, 0, :, None]
        k, v = (torch.where(there, x.double(), 0.0) for x in (k, v))
        if self.Tp:
            k = torch.cat([pk.double().expand(B, -1, -1, -1), k], 2)
            v = torch.cat([pv.double().expand(B, -1, -1, -1), v], 2)
            keep = torch.cat([torch.ones((B, Hq, Tq, self.Tp), dtype=torch.bool), keep], 3)
        self.q, self.k, self.v = q.double(), k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
        self.keep = keep
        s = self.q @ self.k.transpose(2, 3)
        size = (self.q.abs() @ self.k.abs().transpose(2, 3)).amax(3, keepdim=True)
        if score is not None:
            s[..., self.Tp:] += score.double()
        self.s = (s * self.scale).masked_fill(~keep, -math.inf)
        self.p = torch.softmax(self.s, 3)
        self.o = self.p @ self.v
        self.lse2 = torch.logsumexp(self.s, 3) / math.log(2)
        # What p may be off by of itself [B, Hq, Tq, 1]: s is a chain of D / 16 fp32 sums of the
        # logit's size, then rounded with its factor; 2^-13 for exp2, the lse and the joins.  (Scores so
        # large that they absorb the products leave no error: all such logits are equal.)
        top = self.s.masked_fill(~keep | torch.isinf(self.s), 0.0).abs().amax(3, keepdim=True)
        absorbed = top > abs(self.scale) * size * 2.0 ** 25
        self.off = 2.0 ** -13 + torch.where(absorbed, 0.0, (D / 16 + 3) * 2.0 ** -24 * (top + abs(self.scale) * size))

    def weights(self, before=None):
        """Sums of the own keys' probabilities [B, Hk, Tk]; dead rows add nothing."""
        B, Hq, Tq, _ = self.p.shape
        w = torch.nan_to_num(self.p, nan=0.0)[..., self.Tp:].sum(2).view(B, Hq // self.G, self.G, self.Tk).sum(2)
        return w if before is None else w + before.double()

    def _groups(self, x):
        """Summed over a group's heads."""
        B, Hq, T, D = x.shape
        return x.view(B, Hq // self.G, self.G, T, D).sum(2)

    def _split(self, x):
        """Own keys' part, prefix's part summed over the batch."""
        x = self._groups(x)
        return x[:, :, self.Tp:], x[:, :, :self.Tp].sum(0, keepdim=True)

    def grads(self, do):
        """dQ, dK, dV, dKp, dVp from the formulas."""
        do = do.double()
        delta = (do * self.o).sum(3, keepdim=True)
        ds = self.p * (do @ self.v.transpose(2, 3) - delta) * self.scale
        dk, dpk = self._split(ds.transpose(2, 3) @ self.q)
        dv, dpv = self._split(self.p.transpose(2, 3) @ do)
        return ds @ self.k, dk, dv, dpk, dpv

    def grad_bounds(self, do, dtype):
        """What each gradient may be off by, from the roundings on the way.

        P is off by self.off of itself; dP and Delta (O to 16 bits and a residual of 16 bits, fp32
        sums) by less than 2^-14 of sum |dO||V| and sum |dO||O|.  dS and P enter their products
        in two 16-bit parts, P of dV in one where no mask or score is given (half a step u);
        in fp16 the last part of a small value is subnormal (2^-25).  Then each output's own
        rounding, u of its value."""
        u = U[dtype]
        do = do.double()
        big = self.p * (do.abs() @ self.v.abs().transpose(2, 3) + (do.abs() * self.o.abs()).sum(3, keepdim=True))
        off = 2 * self.off + 2.0 ** -13
        ds = off * big * abs(self.scale)
        dp = (u + off) * self.p
        if dtype == torch.float16:
            ds = ds + 2.0 ** -25 * abs(self.scale) * self.keep
            dp = dp + 2.0 ** -25 * self.keep
        dk, dpk = self._split(ds.transpose(2, 3) @ self.q.abs())
        dv, dpv = self._split(dp.transpose(2, 3) @ do.abs())
        tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
        return [b + u * g.abs() + tiny for b, g in zip((ds @ self.k.abs(), dk, dv, dpk, dpv), self.grads(do))]

    def out_bound(self, dtype):
        """O: its own rounding; p's error (P is normalised by the sum of the same p: twice
        self.off less its constant part) and P in two parts (u^2, and 2^-18 for fp32 sums, exp2 and
        the joins' factors) against the largest |v|; in fp16 subnormal parts of small p."""
        u = U[dtype]
        vmax = self.v.abs().max().item() if self.v.numel() else 0.0
        b = u * self.o.abs() + (2 * (self.off - 2.0 ** -13) + u * u + 2.0 ** -18) * vmax
        if dtype == torch.float16:
            b = b + 2.0 ** -24 * (1 + self.v.abs().sum(2).max().item())
        return b

    def weights_bound(self, before=None):
        """Each p off by twice self.off of itself (itself, and the sum it is divided by), fp32 sums of
        at most 2^10 terms per lane, and the sum with what was there before."""
        p = torch.nan_to_num(self.p, nan=0.0)[..., self.Tp:]
        B, Hq, Tq, _ = p.shape
        off = (p * (2 * self.off + 2.0 ** -13)).sum(2).view(B, Hq // self.G, self.G, self.Tk).sum(2)
        w = self.weights()
        return off + 2.0 ** -23 * (w + (0.0 if before is None else before.double().abs())) + 1e-30


def evict(k, v, w, keep, recent, lengths):
    """Kept rows, weights and indices of [B, H, T, D] caches."""
    B, H, T, D = k.shape
    ko, vo = torch.zeros((B, H, keep, D), dtype=k.dtype), torch.zeros((B, H, keep, D), dtype=v.dtype)
    wo, idx = torch.zeros((B, H, keep)), torch.full((B, H, keep), -1, dtype=torch.int64)
    for b in range(B):
        n = T if lengths is None else max(0, min(T, int(lengths[b])))
        for h in range(H):
            rank = lambda j: (-math.inf if math.isnan(w[b, h, j]) else -float(w[b, h, j]), not math.isnan(w[b, h, j]), j)  # noqa: E731,B023
            last = max(0, n - recent)
            # NaN above +inf above the rest; ties to the lowest index
            order = sorted(range(last), key=rank)
            at = sorted(order[:max(0, min(keep, n) - (n - last))]) + list(range(last, n))
            m = len(at)
            idx[b, h, :m] = torch.tensor(at, dtype=torch.int64)
            ko[b, h, :m], vo[b, h, :m], wo[b, h, :m] = k[b, h, at], v[b, h, at], w[b, h, at]
    return ko, vo, wo, idx


def angles(positions, inv_freq, sections):
    """[B, T, pairs] in [-pi, pi], reduced in exact arithmetic."""
    A, B, T = positions.shape
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    freq = [Fraction(float(f)) for f in inv_freq]
    out = torch.empty((B, T, len(freq)), dtype=torch.float64)
    for b in range(B):
        for t in range(T):
            for i, f in enumerate(freq):
                x = int(positions[axis[i], b, t]) * f / (2 * PI)
                x -= round(x)
                out[b, t, i] = float(x * 2 * PI)
    return out


def turn(x, angle, interleaved, back=False):
    """x [B, H, T, D] turned by angle [B, T, pairs]."""
    x = x.double()
    R = 2 * angle.shape[2]
    c, s = angle.cos()[:, None], (-angle if back else angle).sin()[:, None]
    y = x.clone()
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., :R // 2], x[..., R // 2:R])
    ya, yb = a * c - b * s, b * c + a * s
    if interleaved:
        y[..., 0:R:2], y[..., 1:R:2] = ya, yb
    else:
        y[..., :R // 2], y[..., R // 2:R] = ya, yb
    return y


def turn_bound(x, y, angle, interleaved, dtype):
    """The output's own rounding, and the fp32 cosine, sine (3 2^-24 of a turn's reach with the
    angle's 2^-31 of a turn) and products against the pair's size: 2^-20 |pair|."""
    R = 2 * angle.shape[2]
    x = x.double().abs()
    size = torch.zeros_like(x)
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., :R // 2], x[..., R // 2:R])
    if interleaved:
        size[..., 0:R:2], size[..., 1:R:2] = a + b, a + b
    else:
        size[..., :R // 2], size[..., R // 2:R] = a + b, a + b
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    return U[dtype] * y.abs() + 2.0 ** -20 * size + tiny * (size > 0)
