"""The window operators in 64 bits, and how far a result may be from them."""

import math

import torch

U_BF16, U_F16 = 2.0 ** -8, 2.0 ** -11  # half a step, relative
# Scores: fp32 sums of at most 128 products that add up to at most 16 in magnitude (times the softmax scale) in the tests'
# data: 128 * 2^-24 * 16 = 2^-13 absolute, which is the relative error of a weight; as much again for the exponential's
# argument (|x| <= 2^6, rounded to 2^-18) and the approximate exponential (2^-22).
WEIGHT_NOISE = 2.0 ** -12


def visible(n_queries, n_keys, window, sinks, device):
    p = torch.arange(n_keys - n_queries, n_keys, device=device)[:, None]
    j = torch.arange(n_keys, device=device)[None]
    return (j <= p) & ((j > p - window) | (j < sinks))


def attend(q, k, v, see, scale):
    """q [Hq,T,D], k, v [Hkv,S,D], see [T,S] -> (output, sum of weight * |value|) [Hq,T,D] in 64 bits; a masked key is not there
    at all, whatever it holds."""
    g = q.size(0) // k.size(0)
    q, k, v = q.double(), k.double().repeat_interleave(g, 0), v.double().repeat_interleave(g, 0)
    if bool(see.all()):
        p = torch.softmax(q @ k.transpose(1, 2) * scale, -1)
        return p @ v, p @ v.abs()
    out, mag = torch.zeros_like(q), torch.zeros_like(q)
    some = see.any(0)
    k, v, see = k[:, some], v[:, some], see[:, some]
    s = (q @ k.transpose(1, 2) * scale).masked_fill(~see, -math.inf)
    p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0) if not bool(see.any(1).all()) else torch.softmax(s, -1)
    finite = bool(torch.isfinite(v).all())
    if finite:
        return p @ v, p @ v.abs()
    for t in range(q.size(1)):
        at = see[t]
        out[:, t] = (p[:, t, at].unsqueeze(1) @ v[:, at]).squeeze(1)
        mag[:, t] = (p[:, t, at].unsqueeze(1) @ v[:, at].abs()).squeeze(1)
    return out, mag


def prompt(q, k, v, window, sinks, scale=None, lengths=None):
    """(output, magnitude) [B,T,Hq,D]."""
    B, Hq, T, D = q.shape
    S = k.size(2)
    scale = 1 / math.sqrt(D) if scale is None else scale
    see = visible(T, S, window or S, sinks, q.device)
    out, mag = (torch.zeros(B, T, Hq, D, device=q.device, dtype=torch.float64) for _ in range(2))
    for b in range(B):
        n = S if lengths is None else int(lengths[b])
        t = max(n - (S - T), 0)
        if t:
            o, m = attend(q[b, :, :t], k[b, :, :n], v[b, :, :n], see[:t, :n], scale)
            out[b, :t], mag[b, :t] = o.transpose(0, 1), m.transpose(0, 1)
    return out, mag


def quantised(x):
    """What the 4-bit form of the rows holds (64 bits): by distance to the levels, ties to the even code."""
    g = x.double().reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    bad = ~torch.isfinite(g).all(-1, keepdim=True)
    g = torch.where(bad, torch.zeros_like(g), g)
    mant, expo = torch.frexp(g.abs().amax(-1, keepdim=True) / 6)
    s = torch.ldexp(torch.round(mant * 64), expo - 6)
    s = torch.where(s < 2.0 ** -126, torch.zeros_like(s), s)
    best, dist = torch.zeros_like(g), g.abs()
    for level in (1.0, 2.0, 4.0, 0.5, 1.5, 3.0, 6.0):  # even codes first
        d = (g.abs() - level * s).abs()
        near = d < dist
        best, dist = torch.where(near, level * s, best), torch.where(near, d, dist)
    best = torch.where(g < 0, -best, best)
    return torch.where(bad, torch.full_like(best, math.nan), best).reshape(x.shape)


class Cache:
    """The sequences' tokens as Python keeps them: everything that was ever written."""

    def __init__(self, batch, heads, dim, window, sinks, bits, device="cuda"):
        self.window, self.sinks, self.bits = window, sinks, bits
        self.k = [torch.zeros(heads, 0, dim, device=device, dtype=torch.float64) for _ in range(batch)]
        self.v = [t.clone() for t in self.k]

    def write(self, b, k, v, position):
        hold = quantised if self.bits == 4 else torch.Tensor.double
        for store, x in ((self.k, k), (self.v, v)):
            assert position <= store[b].size(1)
            store[b] = torch.cat([store[b][:, :position], hold(x), store[b][:, position + x.size(1):]], 1)

    def held(self, b, n):
        """(k, v) of the tokens that the last of n sees, in order."""
        at = torch.tensor([j for j in range(n) if j < self.sinks or j >= n - self.window], dtype=torch.long, device=self.k[b].device)
        return self.k[b][:, at], self.v[b][:, at]

    def attend(self, b, q, n, scale=None):
        """q [Hq,1,D] -> (output, magnitude) [Hq,D]."""
        if n <= 0:
            z = torch.zeros(q.size(0), q.size(2), device=q.device, dtype=torch.float64)
            return z, z
        k, v = self.held(b, n)
        o, m = attend(q, k, v, torch.ones(1, k.size(1), device=q.device, dtype=torch.bool), q.size(2) ** -0.5 if scale is None else scale)
        return o[:, 0], m[:, 0]


def assert_near(got, want, mag, bits=16, what=""):
    """Each weight is rounded once to bf16 (16 bits), or to f16 and again with its value's scale (4 bits), the result once to bf16."""
    got, want = got.double(), want.reshape(got.shape)
    mag = mag.reshape(got.shape)
    tol = (U_BF16 if bits == 16 else 2 * U_F16) * mag + WEIGHT_NOISE * mag + U_BF16 * want.abs() * (1 + 2.0 ** -6) + 1e-30
    same_nan = torch.isnan(got) == torch.isnan(want)
    assert bool(same_nan.all()), f"{what}: NaN in other places ({int((~same_nan).sum())})"
    fine = torch.isnan(want) | (got == want)
    worst = torch.where(fine, torch.zeros_like(want), (got - want).abs() / tol).nan_to_num(nan=math.inf).max().item() if got.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.2f} of the tolerance"


def heads_data(gen, batch, heads, rows, dim, device="cuda", scale=1.0):
    """[B,H,T,D] views of [B,T,H,D] storage, as projections write them."""
    x = torch.randn(batch, rows, heads, dim, device=device, generator=gen) * scale
    return x.bfloat16().transpose(1, 2)
