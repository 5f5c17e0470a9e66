"""GPU tests of what bndm_amd.tokens keeps between its 16-bit inputs and outputs: weights, statistics, gradients that cancel, values past
the types' ranges, memory that no query sees.

Bounds are worst cases to first order.  u = finfo(t).eps / 2 is what storing a value may take off it, relative to it; in 32 bits that is
E = 2^-24.  A sum of n products in 32 bits is off by n E of the sum of their magnitudes at most, whatever its order."""
import math

import pytest
import torch

from tests import tokens_reference as R

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
E = 2.0 ** -24


@pytest.fixture(scope="module")
def T():
    from bndm_amd import tokens
    return tokens


def normal(seed, *shape, dtype=F16, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype)


def on_gpu(values):
    return None if values is None else torch.tensor(values, dtype=torch.int32, device="cuda")


def attention_in_64_bits(q, k, v, lam, seen, dout=None, scale=None):
    """-> {name: (value, bound)} as R.attention, but the weights, the outputs and the sums of weights times their gradients are held in 32
    bits (weights, and dS on its way to dq, in two parts of 16): what is rounded to 16 bits is the results, the weights dv is formed of, and
    the dS that dk is."""
    dtype, u, tiny = q.dtype, R.unit(q.dtype), R.smallest(q.dtype)
    b, nq, maps, d = q.shape
    nk, hk, dv = v.shape[1:]
    per = maps // 2 // hk
    scale = d ** -0.5 if scale is None else scale
    wide = lambda t: t.unflatten(1, (hk, 2)).repeat_interleave(per, 1).flatten(1, 2)
    q64, k64 = q.double().transpose(1, 2), wide(k.double().transpose(1, 2))
    v64 = v.double().transpose(1, 2).repeat_interleave(per, 1)
    l = lam.double()[:, None, None]
    s = (q64 @ k64.transpose(-1, -2) * scale).masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top.isfinite(), top, torch.zeros_like(top))
    e = torch.exp(s - top)
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total > 0, total, torch.ones_like(total))
    # a score is a sum of d products; it meets the running maximum and the sum's logarithm, 8 roundings of numbers of that size with the
    # exponential's own; sums of nk weights, and as many again where a running maximum moves
    size = q64.abs() @ k64.abs().transpose(-1, -2) * scale
    off_p = (d * E * size + 8 * E * (1 + size.amax(-1, keepdim=True) + math.log(nk))) + 2 * nk * E
    p1, p2, e1, e2 = p[:, 0::2], p[:, 1::2], off_p[:, 0::2], off_p[:, 1::2]
    w = p1 - l * p2
    o = w @ v64
    # two parts of 16 bits leave u of u of a weight, and the least number of the type of a sum that is 1 at least
    part = lambda pm, em: ((pm * (em + (pm * em).sum(-1, keepdim=True) + u * u) + tiny * (pm > 0)) @ v64.abs()) + nk * E * (pm @ v64.abs())
    off_o = part(p1, e1) + l.abs() * part(p2, e2)
    out = {"o": (o.transpose(1, 2), (off_o + u * (o.abs() + off_o) + tiny).transpose(1, 2))}
    if dout is None:
        return out
    g = dout.double().transpose(1, 2)
    gv, mag = g @ v64.transpose(-1, -2), g.abs() @ v64.abs().transpose(-1, -2)
    ds, off, part_off, sums = [], [], [], []
    for pm, em, f in ((p1, e1, torch.ones_like(l)), (p2, e2, -l)):
        big = pm * em
        centre = (pm * gv).sum(-1, keepdim=True)
        # dP is a sum of dv products, D = sum P dP in 32 bits
        raw = dv * E * mag
        off_d = (pm * raw + big * (gv - centre).abs()).sum(-1, keepdim=True) + 2 * nk * E * (pm * gv.abs()).sum(-1, keepdim=True)
        sums.append((centre, off_d))
        x = pm * (gv - centre) * f
        ds.append(x)
        err = f.abs() * (pm * (raw + off_d + 4 * E * (gv.abs() + centre.abs())) + (em + (pm * em).sum(-1, keepdim=True)) * pm * (gv - centre).abs())
        off.append(err + u * x.abs() + tiny / scale * (pm > 0))
        part_off.append(err + u * u * x.abs() + tiny / scale * (pm > 0))
    ds, off, part_off = (torch.stack(t, 2).flatten(1, 2) for t in (ds, off, part_off))

    def shared(t, two):
        t = t.unflatten(1, (hk, per, 2)) if two else t.unflatten(1, (hk, per))
        return t.sum(2).flatten(1, 2) if two else t.sum(2)

    def add(key, grad, err, size, n):
        out[key] = (grad.transpose(1, 2), (err + n * E * size + u * (grad.abs() + err) + tiny).transpose(1, 2))

    add("q", ds @ k64 * scale, part_off @ k64.abs() * scale, ds.abs() @ k64.abs() * scale, nk)
    add("k", shared(ds.transpose(-1, -2) @ q64, True) * scale, shared(off.transpose(-1, -2) @ q64.abs(), True) * scale,
        shared(ds.abs().transpose(-1, -2) @ q64.abs(), True) * scale, nq * per)
    off_w = u * w.abs() + p1 * e1 + l.abs() * p2 * e2 + (p1 * (p1 * e1).sum(-1, keepdim=True) + l.abs() * p2 * (p2 * e2).sum(-1, keepdim=True)) + tiny * (p1 > 0)
    add("v", shared(w.transpose(-1, -2) @ g, False), shared(off_w.transpose(-1, -2) @ g.abs(), False), shared(w.abs().transpose(-1, -2) @ g.abs(), False), nq * per)
    (_, _), (d2, off_d2) = sums
    grad, err = -d2.sum((0, 2, 3)), off_d2.sum((0, 2, 3)) + nq * b * E * d2.abs().sum((0, 2, 3))
    out["lam"] = (grad, err + R.unit(lam.dtype) * (grad.abs() + err) + R.smallest(lam.dtype))
    return out


# ---------------------------------------------------------------------------------------------- gradients of peaked rows
@pytest.mark.parametrize("b,nq,nk,h,hk,d,dv,causal", [(1, 70, 513, 2, 1, 64, 128, False), (2, 40, 1030, 2, 2, 64, 128, False), (1, 600, 600, 2, 1, 64, 128, True),
                                                      (1, 33, 2000, 1, 1, 128, 256, False), (2, 130, 700, 2, 1, 32, 64, False), (1, 64, 200, 2, 1, 64, 128, False),
                                                      (2, 5, 1500, 4, 2, 24, 40, True)])
@pytest.mark.parametrize("std", [1.0, 4.0, 6.0])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_gradients_of_peaked_rows(T, b, nq, nk, h, hk, d, dv, causal, std, dtype):
    """Few keys have nearly all of a row's weight: dP - D cancels there, and what D is off by is all that is left.  So D must not come from
    outputs that were rounded to 16 bits."""
    q, k = normal(1, b, nq, 2 * h, d, dtype=dtype, std=std ** 0.5), normal(2, b, nk, 2 * hk, d, dtype=dtype, std=std ** 0.5)
    v, g = normal(3, b, nk, hk, dv, dtype=dtype), normal(4, b, nq, h, dv, dtype=dtype)
    lam = torch.rand(h, generator=torch.Generator().manual_seed(5)) + 0.1
    leaves = [t.cuda().requires_grad_() for t in (q, k, v, lam)]
    o = T.differential_attention(*leaves, causal=causal)
    want = attention_in_64_bits(q, k, v, lam, R.visible(nq, nk, None, causal, None, b), g)
    for name, got in zip(("q", "k", "v", "lam"), torch.autograd.grad(o, leaves, g.cuda())):
        R.assert_within(got, *want[name], "d" + name)


@pytest.mark.parametrize("b,nq,nk,h,hk,d,causal", [(1, 70, 60, 2, 1, 64, False), (2, 40, 530, 2, 2, 8, False), (1, 200, 200, 2, 1, 32, True), (2, 33, 20, 1, 1, 128, False)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_gradients_of_keys_with_a_common_part(T, b, nq, nk, h, hk, d, causal, dtype):
    """A row's dS adds up to 0: what all keys have in common (a projection's bias) goes out of dq, and what dS was rounded by, times that, does not."""
    q, v, g = normal(1, b, nq, 2 * h, d, dtype=dtype), normal(3, b, nk, hk, 2 * d, dtype=dtype), normal(4, b, nq, h, 2 * d, dtype=dtype)
    k = (normal(2, b, nk, 2 * hk, d, dtype=F32) + 6 * normal(5, d, dtype=F32)).to(dtype)
    lam = torch.full((h,), 0.5)
    leaves = [t.cuda().requires_grad_() for t in (q, k, v, lam)]
    o = T.differential_attention(*leaves, causal=causal, scale=0.25 * d ** -0.5)
    want = attention_in_64_bits(q, k, v, lam, R.visible(nq, nk, None, causal, None, b), g, scale=0.25 * d ** -0.5)
    for name, got in zip(("q", "k", "v", "lam"), torch.autograd.grad(o, leaves, g.cuda())):
        R.assert_within(got, *want[name], "d" + name)


# ---------------------------------------------------------------------------------------------- outputs of maps that cancel
@pytest.mark.parametrize("b,nq,nk,h,hk,d,dv", [(1, 200, 2100, 2, 1, 64, 128), (1, 40, 300, 2, 2, 128, 256), (2, 130, 130, 2, 1, 32, 64), (2, 33, 1000, 1, 1, 64, 128),
                                               (2, 1, 3000, 4, 1, 64, 128), (1, 300, 70, 1, 1, 8, 16)])
@pytest.mark.parametrize("std", [0.3, 1.0])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_outputs_of_maps_that_cancel(T, b, nq, nk, h, hk, d, dv, std, dtype):
    """Both maps' common part goes out of the difference, what the weights were rounded by does not: at lam = 0.9 and nearly flat weights the
    output is a fifth of either map's.  It is as exact as its own rounding for few queries and for many."""
    q, k = normal(1, b, nq, 2 * h, d, dtype=dtype, std=std ** 0.5), normal(2, b, nk, 2 * hk, d, dtype=dtype, std=std ** 0.5)
    v = normal(3, b, nk, hk, dv, dtype=dtype)
    lam = torch.full((h,), 0.9)
    o = T.differential_attention(*(t.cuda() for t in (q, k, v, lam)))
    R.assert_within(o, *attention_in_64_bits(q, k, v, lam, R.visible(nq, nk, None, False, None, b))["o"], "o")


# ---------------------------------------------------------------------------------------------- a kept z past the range of f16
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("m,k,n", [(20, 64, 40), (300, 520, 264), (33, 5, 77)])
def test_linear_gradients_past_the_range_of_f16(T, act, m, k, n):
    """x W^T + b of -70000 and +100000, which f16 does not hold: slopes there are 0 and 1"""
    x, w, dy = normal(1, m, k), normal(2, n, k, std=k ** -0.5), normal(3, m, n)
    low, high = 3, n - 2                                     # columns
    w[low], w[high] = 0, 0
    w[low, 0], w[high, 0] = -35000.0, 50000.0
    x[:, 0] = 0
    x[5, 0] = 2.0
    dy[:, low] *= 0.25                                       # (other rows' slopes there are about a half: their dx stays in range)
    dy[:, high] *= 0.25
    b = normal(4, n, std=0.1)
    leaves = [t.cuda().requires_grad_() for t in (x, w, b)]
    y = T.linear(*leaves, activation=act)
    assert float(y[5, low]) == 0 and float(y[5, high]) == math.inf
    got = torch.autograd.grad(y, leaves, dy.cuda())
    z = x.double() @ w.double().t() + b.double()
    _, slope, curve = R.act(act, z)
    slope[5, low], slope[5, high] = 0, 1
    dz = dy.double() * slope
    # the kept z is rounded, then its slope taken, where that is neither 0 nor 1
    u, sums = R.unit(F16), 2 * max(m, n, k) * E
    off = dy.double().abs() * (curve * torch.where(z.abs() < 100, z.abs(), torch.zeros_like(z)) * (u + sums) + 2.0 ** -17) + u * dz.abs() + R.smallest(F16)
    off[5, low] = 0
    off[5, high] = u * abs(float(dy[5, high]))
    for name, g, want, size, err in (("x", got[0], dz @ w.double(), dz.abs() @ w.double().abs(), off @ w.double().abs()),
                                     ("w", got[1], dz.t() @ x.double(), dz.abs().t() @ x.double().abs(), off.t() @ x.double().abs()),
                                     ("b", got[2], dz.sum(0), dz.abs().sum(0), off.sum(0))):
        R.assert_within(g, want, err + sums * size + u * (want.abs() + err) + R.smallest(F16), "d" + name)


# ---------------------------------------------------------------------------------------------- gradients of weights past the range of f16
def test_weight_gradients_past_the_range_of_f16(T):
    """dS reaches past 65504, scale dS does not"""
    b, nq, nk, h, d, dv = 1, 6, 3, 2, 64, 128
    q, k = normal(1, b, nq, 2 * h, d, std=0.25), normal(2, b, nk, 2 * h, d, std=0.25)
    v, g = normal(3, b, nk, h, dv, std=250.0), normal(4, b, nq, h, dv, std=200.0)
    lam = torch.tensor([0.4, 0.8])
    want = attention_in_64_bits(q, k, v, lam, R.visible(nq, nk, None, False, None, b), g)
    assert all(float(want[name][0].abs().max()) < 65504 for name in "qkv")
    leaves = [t.cuda().requires_grad_() for t in (q, k, v, lam)]
    o = T.differential_attention(*leaves)
    for name, got in zip(("q", "k", "v", "lam"), torch.autograd.grad(o, leaves, g.cuda())):
        R.assert_within(got, *want[name], "d" + name)


@pytest.mark.parametrize("nq,nk,hk,d,causal", [(40, 300, 1, 64, False), (200, 200, 2, 32, True), (33, 70, 2, 128, False)])
def test_gradients_follow_the_factor_of_the_loss(T, nq, nk, hk, d, causal):
    """A loss times a power of two: every gradient times that, bit for bit, but for what f16 cannot hold of the gradients themselves.  dS, a
    thousandth of them, is not what runs out of digits first."""
    b, h = 2, 2
    q, k, v = normal(1, b, nq, 2 * h, d), normal(2, b, nk, 2 * hk, d), normal(3, b, nk, hk, 2 * d)
    g = normal(4, b, nq, h, 2 * d)
    g = torch.where(g.abs() < 0.01, torch.full_like(g, 0.01), g)       # (none leaves f16's normal range below)
    leaves = [t.cuda().requires_grad_() for t in (q, k, v, torch.tensor([0.4, 1.8]))]
    grads = lambda factor: torch.autograd.grad(T.differential_attention(*leaves, causal=causal), leaves, (g * factor).cuda())
    one = grads(1.0)
    for factor in (2.0 ** -6, 2.0 ** 8):
        for name, a, c in zip(("q", "k", "v", "lam"), grads(factor), one):
            want = c.double() * factor
            least = R.smallest(F16) * max(1.0, factor) if a.dtype == F16 else 0.0
            assert ((a.double() - want).abs() <= least).all(), name


# ---------------------------------------------------------------------------------------------- memory that no query sees
@pytest.mark.parametrize("nq,nk,starts,hk,d", [(1, 700, [30, 600], 1, 64), (3, 3000, [1000, 0], 2, 64), (40, 500, [0, 100], 2, 32), (130, 900, [0, 333], 1, 64),
                                               (70, 300, [5, 100], 2, 128), (128, 400, [0, 0], 1, 64), (5, 40, [-9, 2], 1, 64)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_keys_that_no_query_sees_are_not_read(T, nq, nk, starts, hk, d, dtype):
    """a store of keys whose memory past the last query's place was never written, and no kv_lengths"""
    b, h = 2, 2
    q, k = normal(1, b, nq, 2 * h, d, dtype=dtype), normal(2, b, nk, 2 * hk, d, dtype=dtype)
    v, g = normal(3, b, nk, hk, 2 * d, dtype=dtype), normal(4, b, nq, h, 2 * d, dtype=dtype)
    lam = torch.tensor([0.4, 0.8])
    seen = R.visible(nq, nk, None, True, starts, b)
    want = R.attention(q, k, v, lam, seen, dout=g)
    for bad in (math.nan, math.inf, -math.inf):
        k2, v2 = k.clone(), v.clone()
        for i, s in enumerate(starts):
            k2[i, max(0, s + nq):] = bad
            v2[i, max(0, s + nq):] = bad
        leaves = [t.cuda().requires_grad_() for t in (q, k2, v2, lam)]
        o = T.differential_attention(*leaves, causal=True, q_start=on_gpu(starts))
        R.assert_within(o, *want["o"], f"o beside {bad}")
        R.assert_within(T.differential_attention(*(t.detach() for t in leaves), causal=True, q_start=on_gpu(starts)), *want["o"], "o")
        for name, got in zip(("q", "k", "v", "lam"), torch.autograd.grad(o, leaves, g.cuda())):
            R.assert_within(got, *want[name], f"d{name} beside {bad}")


# ---------------------------------------------------------------------------------------------- rows that lie far apart
def test_linear_rows_far_apart(T):
    """the last token of each long sequence: rows 2^23 elements apart; gradients that arrive so"""
    h = torch.zeros(6, (1 << 23) + 24, dtype=F16, device="cuda")
    for m, k, n in ((6, 512, 72), (6, 517, 72), (5, 24, 300)):
        for start in (0, 3):
            x, w, b = normal(1, m, k), normal(2, n, k, std=k ** -0.5), normal(3, n)
            h[:m, start : start + k] = x.cuda()
            rows = h[:m, start : start + k]
            y = T.linear(rows, w.cuda(), b.cuda())
            R.assert_within(y, *R.linear(x, w, b, None, None, F16), "y")
            leaves = [rows.detach().requires_grad_(), w.cuda().requires_grad_(), b.cuda().requires_grad_()]
            y = T.linear(*leaves, activation="silu")
            dy = normal(4, m, n)
            far = torch.zeros(m, (1 << 22) + 8, dtype=F16, device="cuda")[:, 1 : 1 + n].copy_(dy)
            got = torch.autograd.grad(y, leaves, far)
            for name, g in zip("xwb", got):
                R.assert_within(g, *R.linear_gradients(x, w, b, "silu", dy, F16)[name], "d" + name)
    tiles = torch.zeros(150, 1 << 23, dtype=F16, device="cuda")[:, 8:2056]          # as many rows as the large tiles take
    x, w = normal(5, 150, 2048), normal(6, 264, 2048, std=0.02)
    tiles.copy_(x)
    R.assert_within(T.linear(tiles, w.cuda()), *R.linear(x, w, None, None, None, F16), "y")


# ---------------------------------------------------------------------------------------------- sums in 32 bits
@pytest.mark.parametrize("m,k,n", [(5, 8192, 40), (40, 4100, 72), (130, 8192, 264), (2056, 2048, 264), (257, 515, 300), (100, 7, 70), (4104, 264, 2312)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_linear_sums_of_whole_numbers(T, m, k, n, dtype):
    """Whole numbers up to 3: every sum is one below 2^24, which 32 bits hold exactly and fewer do not, so that the result is the rounded sum,
    bit for bit; gradients likewise."""
    g = torch.Generator().manual_seed(m)
    whole = lambda *shape: torch.randint(-3, 4, shape, generator=g).to(dtype).cuda()
    x, w, b, r, dy = whole(m, k).requires_grad_(), whole(n, k).requires_grad_(), whole(n).requires_grad_(), whole(m, n), whole(m, n)
    y = T.linear(x, w, b, residual=r)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    wide = lambda t: t.detach().double().cpu()
    X, W, D = wide(x), wide(w), wide(dy)
    for got, want in ((y, X @ W.t() + wide(b) + wide(r)), (dx, D @ W), (dw, D.t() @ X), (db, D.sum(0))):
        assert torch.equal(got.cpu(), want.to(dtype))
