"""The operators of bndm_amd.tokens in 64 bits on the CPU, each with a bound on what storage in 16 (or 32) bits may do to it.

A value of type t is off by at most u = finfo(t).eps / 2 of itself when it is stored.  The bounds below follow one such error for each
value that the kernels store or hand to the matrix units (results, weights, their gradients, o and o2, the kept z), to first order, plus
SUMS = 2^-13 of the sum of magnitudes for what happens in 32 bits: a score of 128 products of magnitude up to about 10 is off by
128 * 2^-24 * 10 = 2^-13.7, and its exponential by as much relative; longer sums are split over registers and tiles."""
import math

import torch

SUMS = 2.0 ** -13


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    """what a stored value is off by where the type runs out of exponents"""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def assert_within(got, want, bound, what):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got - want).abs() <= bound)                    # (a NaN is bad)
    if bad.any():
        at = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} out of bounds, first at {at}: {got[at]} for {want[at]} +- {bound[at]}")


# ---------------------------------------------------------------------------------------------- linear
def act(name, z):
    """value, slope, and a bound of the second derivative"""
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s)), 0.5
    if name == "gelu":
        c = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        return z * c, c + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi), 0.8
    return z, torch.ones_like(z), 0.0


def linear(x, w, b, name, r, dtype):
    """-> y, bound"""
    x, w = x.double(), w.double()
    z, size = x @ w.t(), x.abs() @ w.abs().t()
    if b is not None:
        z, size = z + b.double(), size + b.double().abs()
    y, slope, _ = act(name, z)
    bound = SUMS * 1.13 * (size + 1e-3)                      # (no slope of either activation exceeds 1.13)
    if r is not None:
        y = y + r.double()
        bound = bound + SUMS * r.double().abs()
    return y, bound + unit(dtype) * y.abs() + smallest(dtype)


def linear_gradients(x, w, b, name, dy, dtype):
    """-> {name: (gradient, bound)} of x, w, b"""
    u = unit(dtype)
    x, w, dy = x.double(), w.double(), dy.double()
    z, size = x @ w.t(), x.abs() @ w.abs().t()
    if b is not None:
        z, size = z + b.double(), size + b.double().abs()
    _, slope, curve = act(name, z)
    dz = dy * slope
    # the kept z is rounded, then its slope taken
    off = dy.abs() * (curve * (u * z.abs() + SUMS * size) + (SUMS if name else 0.0))
    stored = off + (u * dz.abs() + smallest(dtype) if name else 0.0)
    out = {}
    for key, grad, mag, err in (("x", dz @ w, dz.abs() @ w.abs(), stored @ w.abs()), ("w", dz.t() @ x, dz.abs().t() @ x.abs(), stored.t() @ x.abs()),
                                ("b", dz.sum(0), dz.abs().sum(0), off.sum(0))):
        out[key] = (grad, err + SUMS * mag + u * (grad.abs() + err) + smallest(dtype))
    return out


# ---------------------------------------------------------------------------------------------- rotary
def rotary(x, positions, sections, base, interleaved, inverse=False):
    """-> y, bound"""
    d = x.shape[-1]
    f = torch.cat([float(base) ** (-torch.arange(s, dtype=torch.float64) / s) for s in sections])
    axis = torch.cat([torch.full((s,), i, dtype=torch.long) for i, s in enumerate(sections)])
    angle = (positions.double()[..., axis] * f)[..., None, :] * (-1 if inverse else 1)
    y = x.double()
    a, b = (y[..., 0::2], y[..., 1::2]) if interleaved else (y[..., : d // 2], y[..., d // 2 :])
    p, q = a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()
    size = (a.abs() + b.abs()) * 2.0 ** -21                  # sine, cosine, two products and a sum of 32 bits
    join = (lambda s, t: torch.stack((s, t), -1).flatten(-2)) if interleaved else (lambda s, t: torch.cat((s, t), -1))
    out = join(p, q)
    return out, join(size, size) + unit(x.dtype) * out.abs() + smallest(x.dtype)


# ---------------------------------------------------------------------------------------------- differential attention
def visible(nq, nk, lengths, causal, starts, batch):
    """[batch, 1, nq, nk]"""
    j, i = torch.arange(nk), torch.arange(nq)
    seen = torch.ones(batch, 1, nq, nk, dtype=torch.bool)
    if lengths is not None:
        seen &= j < torch.as_tensor(lengths)[:, None, None, None]
    if causal:
        first = torch.full((batch,), nk - nq) if starts is None else torch.as_tensor(starts)
        seen &= j <= (first[:, None, None, None] + i[:, None])
    return seen


def attention(q, k, v, lam, seen, scale=None, dout=None):
    """-> {"o": (value, bound), and with dout "q", "k", "v", "lam": (gradient, bound)}"""
    dtype = q.dtype
    u = unit(dtype)
    b, nq, maps, d = q.shape
    nk, per = k.shape[1], maps // 2 // v.shape[2]
    scale = d ** -0.5 if scale is None else scale
    q64 = q.double().transpose(1, 2)
    kept = seen.any(2, keepdim=True).transpose(2, 3) if seen.shape[2] else torch.zeros(b, 1, nk, 1, dtype=torch.bool)
    clean = lambda t: torch.where(kept, t.double().transpose(1, 2), torch.zeros((), dtype=torch.float64))   # unseen keys count for nothing
    wide = lambda t: t.unflatten(1, (-1, 2)).repeat_interleave(per, 1).flatten(1, 2)
    k64, v64 = wide(clean(k)), clean(v).repeat_interleave(per, 1)
    s = (q64 @ k64.transpose(-1, -2) * scale).masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True) if nk else torch.zeros(b, maps, nq, 1, dtype=torch.float64)
    e = torch.exp(s - torch.where(top.isfinite(), top, torch.zeros_like(top)))
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total > 0, total, torch.ones_like(total))
    p1, p2, l = p[:, 0::2], p[:, 1::2], lam.double()[:, None, None]
    w = p1 - l * p2
    o, o1, o2 = w @ v64, p1 @ v64, p2 @ v64
    tiny = smallest(dtype)
    # weights are rounded before they are divided by their sum, which is at least that of the largest, 1
    magnitude = (p1 + tiny) @ v64.abs() + l.abs() * ((p2 + tiny) @ v64.abs())
    out = {"o": (o.transpose(1, 2), ((u + SUMS) * magnitude + u * o.abs() + tiny).transpose(1, 2))}
    if dout is None:
        return out
    g = dout.double().transpose(1, 2)
    gv = g @ v64.transpose(-1, -2)
    mag_gv = g.abs() @ v64.abs().transpose(-1, -2)
    off_o = (u + SUMS) * magnitude + u * o.abs() + tiny
    off_o2 = (2 * u + SUMS) * ((p2 + tiny) @ v64.abs()) + tiny
    off_d2 = (g.abs() * off_o2).sum(-1, keepdim=True)
    off_d1 = (g.abs() * off_o).sum(-1, keepdim=True) + l.abs() * off_d2
    d1, d2 = (g * o1).sum(-1, keepdim=True), (g * o2).sum(-1, keepdim=True)
    ds1, ds2 = p1 * (gv - d1), -l * p2 * (gv - d2)
    off1 = p1 * (off_d1 + SUMS * (mag_gv + d1.abs())) + u * ds1.abs() + tiny
    off2 = l.abs() * p2 * (off_d2 + SUMS * (mag_gv + d2.abs())) + u * ds2.abs() + tiny
    ds, off = torch.stack((ds1, ds2), 2).flatten(1, 2), torch.stack((off1, off2), 2).flatten(1, 2)

    def shared(t, two):
        t = t.unflatten(1, (v.shape[2], per, 2)) if two else t.unflatten(1, (v.shape[2], per))
        return t.sum(2).flatten(1, 2) if two else t.sum(2)

    def add(key, grad, err, size):
        out[key] = (grad.transpose(1, 2), (err + SUMS * size + u * (grad.abs() + err) + tiny).transpose(1, 2))

    add("q", ds @ k64 * scale, off @ k64.abs() * scale, ds.abs() @ k64.abs() * scale)
    add("k", shared(ds.transpose(-1, -2) @ q64, True) * scale, shared(off.transpose(-1, -2) @ q64.abs(), True) * scale,
        shared(ds.abs().transpose(-1, -2) @ q64.abs(), True) * scale)
    off_w = u * w.abs() + SUMS * (p1 + l.abs() * p2) + tiny
    add("v", shared(w.transpose(-1, -2) @ g, False), shared(off_w.transpose(-1, -2) @ g.abs(), False),
        shared(w.abs().transpose(-1, -2) @ g.abs(), False))
    grad = -d2.sum((0, 2, 3))
    err = off_d2.sum((0, 2, 3)) + SUMS * d2.abs().sum((0, 2, 3))
    out["lam"] = (grad, err + unit(lam.dtype) * (grad.abs() + err) + smallest(lam.dtype))
    return out
