"""GPU tests of bndm_amd.tokens against the operators in 64 bits (tests/tokens_reference.py, where the bounds are derived)."""
import math

import pytest
import torch

from tests import tokens_reference as R

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def T():
    from bndm_amd import tokens
    return tokens


def normal(seed, *shape, dtype=F16, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype)


# ---------------------------------------------------------------------------------------------- linear
SIZES = [(1, 8, 8), (1, 512, 1000), (5, 64, 24), (64, 512, 512), (130, 72, 136), (37, 515, 77), (3, 1, 1), (300, 200, 264), (129, 128, 1), (1000, 40, 130),
         (65, 640, 24), (33, 523, 40), (200, 5, 70), (200, 70, 3), (7, 131, 140), (100, 3, 5), (100, 8192, 72), (100, 4099, 70), (8200, 40, 72),                # long sums, in parts
         (9000, 5, 200), (5003, 139, 300), (1003, 4099, 300),                                        # many rows, unaligned
         (300, 600, 520), (1003, 515, 515), (2, 4100, 2056), (40, 1030, 9000),                         # few rows at a time, 16, 32 and 64 of them
         (4104, 136, 2312), (4104, 2312, 136), (136, 2312, 4104)]                                      # large tiles, with edges


@pytest.mark.parametrize("m,k,n", SIZES)
@pytest.mark.parametrize("act,bias,residual,dtype", [(None, False, False, F16), ("silu", True, False, BF16), ("gelu", True, True, F16), (None, True, True, BF16)])
def test_linear(T, m, k, n, act, bias, residual, dtype):
    x, w = normal(1, m, k, dtype=dtype), normal(2, n, k, dtype=dtype, std=k ** -0.5)
    b = normal(3, n, dtype=dtype) if bias else None
    r = normal(4, m, n, dtype=dtype) if residual else None
    dev = lambda t: None if t is None else t.cuda()
    y = T.linear(dev(x), dev(w), dev(b), activation=act, residual=dev(r))
    assert y.dtype == dtype and y.is_contiguous()
    R.assert_within(y, *R.linear(x, w, b, act, r, dtype), "y")


@pytest.mark.parametrize("m,k,n", SIZES)
@pytest.mark.parametrize("act,bias,dtype", [("silu", True, F16), ("gelu", False, BF16), (None, True, BF16)])
def test_linear_gradients(T, m, k, n, act, bias, dtype):
    x, w = normal(1, m, k, dtype=dtype), normal(2, n, k, dtype=dtype, std=k ** -0.5)
    b = normal(3, n, dtype=dtype) if bias else None
    r, dy = normal(4, m, n, dtype=dtype), normal(5, m, n, dtype=dtype)
    leaves = [t.cuda().requires_grad_() for t in (x, w, b, r) if t is not None]
    y = T.linear(leaves[0], leaves[1], leaves[2] if bias else None, activation=act, residual=leaves[-1])
    R.assert_within(y, *R.linear(x, w, b, act, r, dtype), "y")
    grads = torch.autograd.grad(y, leaves, dy.cuda())
    want = R.linear_gradients(x, w, b, act, dy, dtype)
    for key, g in zip(("x", "w", "b") if bias else ("x", "w"), grads):
        R.assert_within(g, *want[key], "d" + key)
    assert torch.equal(grads[-1].cpu(), dy)


def test_linear_takes_rows_as_they_lie(T):
    """slices of wider rows, rows that start off 16 bytes, a transposed weight, leading axes, a repeated row, one row of a matrix"""
    wide = normal(1, 50, 160).cuda()
    w = normal(2, 96, 64, std=0.125).cuda()
    r = normal(3, 50, 200).cuda()
    for x in (wide[:, :64], wide[:, 8:72], wide[:, 3:67], wide[3:4, 5:69], wide[7, :64].expand(50, 64), wide[:, ::2][:, :64]):
        for weight in (w, w.t().contiguous().t()):
            for res in (None, r[: x.shape[0], 5:101]):
                y = T.linear(x, weight, residual=res)
                R.assert_within(y, *R.linear(x.cpu(), w.cpu(), None, None, None if res is None else res.cpu(), F16), "y")
    x = normal(4, 2, 3, 5, 64).cuda()
    y = T.linear(x, w)
    assert y.shape == (2, 3, 5, 96)
    R.assert_within(y.reshape(30, 96), *R.linear(x.cpu().reshape(30, 64), w.cpu(), None, None, None, F16), "y")
    assert T.linear(x[:0], w).shape == (0, 3, 5, 96)


def test_linear_gradients_of_broadcast_and_strided_inputs(T):
    x, w, b = normal(1, 64), normal(2, 40, 64, std=0.125), normal(3, 40)
    leaves = [t.cuda().requires_grad_() for t in (x, w, b)]
    rows = leaves[0].expand(20, 64)                          # one row for all: its gradient is the sum
    y = T.linear(rows, leaves[1], leaves[2], activation="silu")
    got = torch.autograd.grad(y.sum(), leaves)               # (the gradient that comes in is one number, repeated)
    ref = [t.double().requires_grad_() for t in (x, w, b)]
    z = ref[0].expand(20, 64) @ ref[1].t() + ref[2]
    want = torch.autograd.grad((z * torch.sigmoid(z)).sum(), ref)
    bounds = R.linear_gradients(x.expand(20, 64), w, b, "silu", torch.ones(20, 40), F16)
    R.assert_within(got[1], want[1], bounds["w"][1], "dw")
    R.assert_within(got[2], want[2], bounds["b"][1], "db")
    R.assert_within(got[0], want[0], bounds["x"][1].sum(0) + 20 * 2.0 ** -11 * want[0].abs(), "dx")   # 20 rows added up in 16 bits
    x = torch.zeros(0, 64, dtype=F16, device="cuda", requires_grad=True)
    y = T.linear(x, leaves[1], leaves[2], activation="gelu")
    dx, dw, db = torch.autograd.grad(y, (x, leaves[1], leaves[2]), torch.empty_like(y))
    assert dx.shape == (0, 64) and not dw.any() and not db.any()


# ---------------------------------------------------------------------------------------------- rotary
@pytest.mark.parametrize("b,n,h,hk,d,sections,interleaved,dtype", [
    (1, 1, 1, 1, 2, (1,), False, F32), (2, 7, 3, 1, 30, (5, 5, 5), False, F16), (2, 7, 3, 1, 30, (5, 5, 5), True, BF16),
    (3, 65, 8, 2, 64, (16, 16), False, BF16), (3, 65, 8, 2, 64, (12, 10, 10), True, F16), (2, 300, 2, 2, 96, (48,), False, F32),
    (2, 300, 2, 2, 40, (10, 5, 5), True, F32), (1, 5000, 1, 1, 256, (32, 32, 32, 32), False, F16), (64, 1, 16, 4, 72, (0, 18, 18), False, BF16),
    (2, 9, 5, 3, 24, (6, 6), True, F32), (2, 9, 5, 3, 24, (6, 6), False, F32)])
@pytest.mark.parametrize("kind", ["int32", "int64", "float32"])
def test_rotary(T, b, n, h, hk, d, sections, interleaved, dtype, kind):
    g = torch.Generator().manual_seed(n)
    shape = (b, n, len(sections)) if kind != "int32" else (n, len(sections))
    positions = torch.randint(-3, 1_000_000, shape, generator=g).to(getattr(torch, kind))
    q, k = normal(1, b, n, h, d, dtype=dtype), normal(2, b, n, hk, d, dtype=dtype)
    dq, dk = normal(3, b, n, h, d, dtype=dtype), normal(4, b, n, hk, d, dtype=dtype)
    lq, lk = q.cuda().requires_grad_(), k.cuda().requires_grad_()
    oq, ok = T.rotary(lq, lk, positions.cuda(), sections, interleaved=interleaved)
    gq, gk = torch.autograd.grad((oq, ok), (lq, lk), (dq.cuda(), dk.cuda()))
    for got, x, inverse in ((oq, q, False), (ok, k, False), (gq, dq, True), (gk, dk, True)):
        R.assert_within(got, *R.rotary(x, positions, sections, 10000.0, interleaved, inverse), "inverse" if inverse else "forward")
    assert torch.equal(T.rotary(lq.detach(), None, positions.cuda(), sections, interleaved=interleaved), oq)


def test_rotary_takes_heads_as_they_lie(T):
    """slices of a packed projection, heads before tokens, odd starts, repeated heads, strided positions; a base of its own"""
    packed = normal(1, 2, 33, 7 * 48).cuda()
    positions = torch.randint(0, 500, (2, 33, 6), dtype=torch.int32).cuda()[..., ::3]
    q, k = packed[..., : 4 * 48].unflatten(-1, (4, 48)), packed[..., 4 * 48 : 6 * 48].unflatten(-1, (2, 48))
    cases = [(q, k), (packed[..., 1 : 1 + 4 * 48].unflatten(-1, (4, 48)), packed[..., 4 * 48 + 4 : 6 * 48 + 4].unflatten(-1, (2, 48))),
             (q.transpose(1, 2).contiguous().transpose(1, 2), k[:, :, :1].expand(2, 33, 3, 48)),
             (packed[..., ::2][..., : 3 * 48].unflatten(-1, (3, 48)), k)]
    for a, b in cases:
        for interleaved in (False, True):
            oa, ob = T.rotary(a, b, positions, (12, 12), base=500.0, interleaved=interleaved)
            R.assert_within(oa, *R.rotary(a.cpu(), positions.cpu(), (12, 12), 500.0, interleaved), "q")
            R.assert_within(ob, *R.rotary(b.cpu(), positions.cpu(), (12, 12), 500.0, interleaved), "k")
    assert T.rotary(q[:0], k[:0], positions[:0], (12, 12))[0].shape == (0, 33, 4, 48)


def test_rotary_gradient_of_one_output(T):
    q, k = normal(1, 2, 5, 4, 32).cuda().requires_grad_(), normal(2, 2, 5, 1, 32).cuda().requires_grad_()
    positions = torch.arange(10, dtype=torch.int32).reshape(5, 2).cuda()
    oq, ok = T.rotary(q, k, positions, (8, 8))
    g = normal(3, 2, 5, 1, 32).cuda()
    gq, gk = torch.autograd.grad(ok, (q, k), g, allow_unused=True)
    assert gq is None
    R.assert_within(gk, *R.rotary(g.cpu(), positions.cpu(), (8, 8), 10000.0, False, True), "dk")


# ---------------------------------------------------------------------------------------------- differential attention
def attention_inputs(b, nq, nk, h, hk, d, dv, dtype, lam_dtype=None):
    return (normal(1, b, nq, 2 * h, d, dtype=dtype), normal(2, b, nk, 2 * hk, d, dtype=dtype), normal(3, b, nk, hk, dv, dtype=dtype),
            (torch.rand(h, generator=torch.Generator().manual_seed(4)) + 0.1).to(lam_dtype or dtype), normal(5, b, nq, h, dv, dtype=dtype))


CASES = [
    # b, nq, nk, h, hk, d, dv, causal, starts, lengths, dtype
    (1, 1, 1, 1, 1, 8, 16, False, None, None, F16),
    (2, 3, 1, 2, 1, 64, 128, False, None, None, F16),
    (2, 16, 16, 4, 4, 8, 16, False, None, None, F16),
    (1, 33, 65, 3, 1, 40, 80, False, None, None, BF16),
    (3, 130, 130, 2, 2, 64, 128, True, None, [130, 0, 71], F16),
    (2, 200, 333, 4, 2, 64, 128, True, None, None, BF16),
    (2, 300, 90, 2, 1, 64, 128, True, None, [90, 1], F16),           # most rows see nothing, one sequence has one key
    (2, 129, 257, 2, 2, 128, 256, True, [64, -5], [200, 257], F16),
    (1, 100, 100, 2, 1, 128, 256, False, None, [99], BF16),
    (2, 70, 70, 3, 3, 24, 48, True, [0, 0], [70, 33], BF16),
    (2, 40, 129, 2, 1, 72, 64, False, None, [129, 64], F16),          # values narrower than 2 D, and wider
    (1, 40, 64, 2, 2, 16, 200, False, None, None, F16),
    (4, 1, 1000, 8, 2, 64, 128, True, [999, 0, -1, 500], [1000, 1, 300, 501], BF16),
    (2, 1, 5000, 4, 1, 64, 128, False, None, [5000, 2000], F16),
    (3, 2, 700, 16, 1, 32, 64, True, None, None, F16),
    (2, 5, 3000, 6, 3, 128, 256, True, [2995, 1], [3000, 6], BF16),
    (1, 128, 4100, 1, 1, 64, 128, False, None, None, F16),
    (2, 4, 0, 2, 1, 64, 128, False, None, None, F16),
    (2, 4, 9, 2, 1, 64, 128, False, None, [0, 0], F16),
]


def on_gpu(values):
    return None if values is None else torch.tensor(values, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("b,nq,nk,h,hk,d,dv,causal,starts,lengths,dtype", CASES)
def test_attention(T, b, nq, nk, h, hk, d, dv, causal, starts, lengths, dtype):
    q, k, v, lam, _ = attention_inputs(b, nq, nk, h, hk, d, dv, dtype)
    o = T.differential_attention(*(t.cuda() for t in (q, k, v, lam)), causal=causal, q_start=on_gpu(starts), kv_lengths=on_gpu(lengths))
    assert o.dtype == dtype and o.is_contiguous()
    R.assert_within(o, *R.attention(q, k, v, lam, R.visible(nq, nk, lengths, causal, starts, b))["o"], "o")


@pytest.mark.parametrize("lam_dtype", [None, F32])
@pytest.mark.parametrize("b,nq,nk,h,hk,d,dv,causal,starts,lengths,dtype", CASES)
def test_attention_gradients(T, b, nq, nk, h, hk, d, dv, causal, starts, lengths, dtype, lam_dtype):
    q, k, v, lam, dout = attention_inputs(b, nq, nk, h, hk, d, dv, dtype, lam_dtype)
    leaves = [t.cuda().requires_grad_() for t in (q, k, v, lam)]
    o = T.differential_attention(*leaves, causal=causal, q_start=on_gpu(starts), kv_lengths=on_gpu(lengths))
    grads = torch.autograd.grad(o, leaves, dout.cuda())
    seen = R.visible(nq, nk, lengths, causal, starts, b)
    want = R.attention(q, k, v, lam, seen, dout=dout)
    R.assert_within(o, *want["o"], "o")
    for name, g, leaf in zip(("q", "k", "v", "lam"), grads, leaves):
        assert g.dtype == leaf.dtype
        R.assert_within(g, *want[name], "d" + name)
    if nk:
        hidden = ~seen.any(2)[:, 0]                          # keys that no query sees
        assert not grads[1][hidden.cuda()].any() and not grads[2][hidden.cuda()].any()
    few = (seen.sum(-1) < 2)[:, 0].cuda()                    # no key, or one, whose weight is 1 whatever the score
    assert not grads[0][few].any()


def test_attention_does_not_read_past_a_sequence(T):
    q, k, v, lam, dout = attention_inputs(3, 20, 300, 2, 1, 64, 128, F16)
    lengths = [300, 130, 0]
    seen = R.visible(20, 300, lengths, False, None, 3)
    want = R.attention(q, k, v, lam, seen, dout=dout)
    for bad in (math.nan, math.inf, -math.inf, -65504.0):
        k2, v2 = k.clone(), v.clone()
        for b, n in enumerate(lengths):
            k2[b, n:] = bad
            v2[b, n:] = bad
        leaves = [t.cuda().requires_grad_() for t in (q, k2, v2, lam)]
        o = T.differential_attention(*leaves, kv_lengths=on_gpu(lengths))
        R.assert_within(o, *want["o"], "o")
        R.assert_within(T.differential_attention(*(t.detach() for t in leaves), kv_lengths=on_gpu(lengths)), *want["o"], "o")
        for name, g in zip(("q", "k", "v", "lam"), torch.autograd.grad(o, leaves, dout.cuda())):
            R.assert_within(g, *want[name], f"d{name}")


def test_attention_takes_tensors_as_they_lie(T):
    """slices of a packed projection, tokens 2^23 elements apart, heads before tokens, odd starts and strides, repeated key heads; gradients that arrive strided"""
    b, n, h, hk, d = 2, 70, 4, 2, 32
    packed = normal(1, b, n, 2 * (h + hk) * d + 2 * hk * d + 8).cuda()
    split = lambda off: [t.unflatten(-1, s) for t, s in zip(packed[..., off : off + 2 * (h + 2 * hk) * d].split([2 * h * d, 2 * hk * d, 2 * hk * d], -1),
                                                           ((2 * h, d), (2 * hk, d), (hk, 2 * d)))]
    lam = torch.rand(h, generator=torch.Generator().manual_seed(4)).to(F16).cuda()
    base = split(0)
    far = torch.zeros(2, n, (1 << 23) + 8, dtype=F16, device="cuda")[:, :, : 2 * h * d].unflatten(-1, (2 * h, d)).copy_(base[0])
    cases = [base, split(3), [far, *base[1:]], [t.transpose(1, 2).contiguous().transpose(1, 2) for t in base],
             [base[0], base[1][:, :, :2].repeat(1, 1, 2, 1), base[2][:, :, :1].expand(b, n, hk, 2 * d)]]
    grad = normal(6, b, h, 2 * d, n).cuda().permute(0, 3, 1, 2)
    seen = R.visible(n, n, None, True, None, b)
    for tensors in cases:
        leaves = [t.detach().requires_grad_() for t in tensors]
        o = T.differential_attention(*leaves, lam, causal=True)
        want = R.attention(*(t.cpu() for t in tensors), lam.cpu(), seen, dout=grad.cpu())
        R.assert_within(o, *want["o"], "o")
        for name, g in zip("qkv", torch.autograd.grad(o, leaves, grad)):
            R.assert_within(g, *want[name], "d" + name)


def test_attention_scores_far_from_zero(T):
    """scores of several hundred, all of one sign or mixed, and sums that grow tile by tile"""
    q, k, v, lam, dout = attention_inputs(1, 64, 500, 2, 2, 64, 128, F16)
    seen = R.visible(64, 500, None, False, None, 1)
    for scale in (0.125, 0.5, 1e-4):
        for shift in (0.0, 2.0):
            ramp = torch.linspace(-1, 1, 500)[None, :, None, None]
            k2 = (k.float() * 0.5 + shift * ramp).to(F16)
            q2 = (q.float() * 0.25 + shift / 4).to(F16)
            o = T.differential_attention(*(t.cuda() for t in (q2, k2, v, lam)), scale=scale)
            R.assert_within(o, *R.attention(q2, k2, v, lam, seen, scale=scale)["o"], f"scale {scale}")


@pytest.mark.parametrize("b,nq,nk", [(2, 8, 8), (1, 1, 600), (3, 5, 513), (1, 130, 1300), (2, 1, 1)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_gradient_of_lam_in_32_bits(T, b, nq, nk, dtype):
    """dlam adds up whole rows' do . o2, which cancel: it comes from 32-bit sums, not from the rounded output.  Bound: dP and scores are sums
    of Dv and D products in 32 bits, a score's error times its weight is the weight's; 64 more roundings for exponentials and sums."""
    h, d, dv = 2, 16, 16
    q, k, v = normal(1, b, nq, 2 * h, d, dtype=dtype), normal(2, b, nk, 2 * h, d, dtype=dtype), normal(3, b, nk, h, dv, dtype=dtype)
    grad, lam = normal(4, b, nq, h, dv, dtype=dtype), torch.tensor([0.3, 0.8])
    leaf = lam.cuda().requires_grad_()
    o = T.differential_attention(q.cuda(), k.cuda(), v.cuda(), leaf)
    got, = torch.autograd.grad(o, leaf, grad.cuda())
    q2, k2 = (t.double().transpose(1, 2)[:, 1::2] for t in (q, k))
    v, grad = (t.double().transpose(1, 2) for t in (v, grad))
    p = (q2 @ k2.transpose(-1, -2) * d ** -0.5).softmax(-1)
    want = -(p * (grad @ v.transpose(-1, -2))).sum((0, 2, 3))
    size = (p * (grad.abs() @ v.abs().transpose(-1, -2))).sum((0, 2, 3))
    score = float((q2.abs() @ k2.abs().transpose(-1, -2)).max()) * d ** -0.5
    assert ((got.cpu().double() - want).abs() <= (dv + d * score + 64) * 2.0 ** -24 * size).all(), (got.cpu(), want, size)


def test_attention_gradients_against_differences(T):
    """a step along each gradient changes the loss by its squared length"""
    q, k, v, lam, dout = attention_inputs(2, 24, 40, 2, 1, 32, 64, BF16)
    seen = R.visible(24, 40, None, True, None, 2)
    leaves = [t.cuda().requires_grad_() for t in (q, k, v, lam)]
    grads = torch.autograd.grad(T.differential_attention(*leaves, causal=True), leaves, dout.cuda())

    def loss(values):
        return (R.attention(*values, seen)["o"][0] * dout.double()).sum()

    values = [t.double() for t in (q, k, v, lam)]
    for at, g in enumerate(grads):
        g = g.double().cpu()
        step = 1e-4 / float(g.norm())
        ahead, behind = list(values), list(values)
        ahead[at], behind[at] = values[at] + step * g, values[at] - step * g
        slope = float((loss(ahead) - loss(behind)) / (2 * step))
        # the two differ by the gradient's own error, relative to its length: at most a few roundings of bf16, 2^-9 each
        assert abs(slope / float(g.square().sum()) - 1) < 8 * 2.0 ** -9, at


# ---------------------------------------------------------------------------------------------- a layer, streams, graphs
def layer(T, x, p, positions, sections, heads, kv_heads, size, lengths=None):
    """x + proj(attention(rotary(project(x)))), then a wide layer with its activation, as a block over tokens goes"""
    b, n, _ = x.shape
    packed = T.linear(x, p["qkv"], p["qkv_bias"])
    q, k, v = packed.split([2 * heads * size, 2 * kv_heads * size, 2 * kv_heads * size], -1)
    q, k = T.rotary(q.unflatten(-1, (2 * heads, size)), k.unflatten(-1, (2 * kv_heads, size)), positions, sections)
    o = T.differential_attention(q, k, v.unflatten(-1, (kv_heads, 2 * size)), p["lam"], kv_lengths=lengths)
    x = T.linear(o.flatten(-2), p["out"], p["out_bias"], residual=x)
    return T.linear(T.linear(x, p["up"], activation="silu"), p["down"], residual=x)


def layer_in_64_bits(x, p, positions, sections, heads, kv_heads, size, lengths=None):
    b, n, _ = x.shape
    packed = x @ p["qkv"].t() + p["qkv_bias"]
    q, k, v = packed.split([2 * heads * size, 2 * kv_heads * size, 2 * kv_heads * size], -1)
    q, k = (R.rotary(t.unflatten(-1, (-1, size)), positions, sections, 10000.0, False)[0] for t in (q, k))
    seen = R.visible(n, n, lengths, False, None, b)
    o = R.attention(q, k, v.unflatten(-1, (kv_heads, 2 * size)), p["lam"], seen)["o"][0]
    x = o.flatten(-2) @ p["out"].t() + p["out_bias"] + x
    h = x @ p["up"].t()
    return (h * torch.sigmoid(h)) @ p["down"].t() + x


def layer_inputs(dtype):
    heads, kv_heads, size, width = 4, 2, 32, 128
    shapes = {"qkv": (2 * (heads + 2 * kv_heads) * size, width), "out": (width, 2 * heads * size), "up": (256, width), "down": (width, 256)}
    p = {name: normal(i, *s, dtype=dtype, std=s[1] ** -0.5) for i, (name, s) in enumerate(shapes.items())}
    p["qkv_bias"], p["out_bias"] = normal(7, shapes["qkv"][0], dtype=dtype, std=0.1), normal(8, width, dtype=dtype, std=0.1)
    p["lam"] = torch.tensor([0.2, 0.4, 0.5, 0.8]).to(dtype)
    ys, xs = torch.meshgrid(torch.arange(6), torch.arange(9), indexing="ij")
    positions = torch.stack((ys, xs), -1).reshape(-1, 2).to(torch.int32)
    return p, normal(9, 3, 54, width, dtype=dtype), positions, ((8, 8), heads, kv_heads, size)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_a_layer_and_its_gradients(T, dtype):
    p, x, positions, how = layer_inputs(dtype)
    lengths = [54, 20, 0]
    params = {name: t.cuda().requires_grad_() for name, t in p.items()}
    lx = x.cuda().requires_grad_()
    y = layer(T, lx, params, positions.cuda(), *how, lengths=on_gpu(lengths))
    g = normal(10, *y.shape, dtype=dtype)
    got = torch.autograd.grad(y, [lx, *params.values()], g.cuda())
    ref = {name: t.double().requires_grad_() for name, t in p.items()}
    rx = x.double().requires_grad_()
    want_y = layer_in_64_bits(rx, ref, positions, *how, lengths=lengths)
    want = torch.autograd.grad(want_y, [rx, *ref.values()], g.double())
    # seven stored results in a row, each off by u of its length at most; gradients pass as many again, and cancel in lam's sum
    u = R.unit(dtype)
    rel = lambda a, b: float((a.double().cpu() - b).norm() / b.norm())
    assert rel(y, want_y.detach()) < 7 * u
    for name, a, b in zip(["x", *params], got, want):
        assert rel(a, b) < 14 * u, name


def test_on_another_stream(T):
    p, x, positions, how = layer_inputs(F16)
    params = {name: t.cuda() for name, t in p.items()}
    want = layer(T, x.cuda(), params, positions.cuda(), *how)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(20):
            big = big @ big * 1e-2                           # the stream is busy when its inputs are made
        late = x.cuda().clone()
        got = layer(T, late, params, positions.cuda(), *how)
    side.synchronize()
    assert torch.equal(got, want)


def test_captured_and_replayed(T):
    """a step and its gradients recorded into a graph: every replay gives what the eager call gives on the inputs of that replay; a
    second graph beside it, replayed in turn, has scratch memory of its own"""
    p, x, positions, how = layer_inputs(BF16)
    positions = positions.cuda()

    def step(leaf, params):
        y = layer(T, leaf, params, positions, *how)
        return (y, *torch.autograd.grad(y, [leaf, *params.values()], torch.ones_like(y)))

    def one(seed):
        # split keys and single queries: scratch memory inside the graph
        q, k, v, lam, _ = attention_inputs(2, 1, 3000, 4, 1, 64, 128, BF16)
        q = normal(seed, *q.shape, dtype=BF16)
        return [t.cuda() for t in (q, k, v, lam)]

    graphs = []
    for seed in (1, 2):
        params = {name: t.cuda().requires_grad_() for name, t in p.items()}
        leaf = x.cuda().requires_grad_()
        single = one(seed)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                step(leaf, params)
                T.differential_attention(*single)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = (*step(leaf, params), T.differential_attention(*single))
        graphs.append((graph, leaf, params, single, out))
    for trial in range(3):
        for n, (graph, leaf, params, single, out) in enumerate(graphs):
            with torch.no_grad():
                leaf.copy_(normal(20 + 2 * trial + n, *x.shape, dtype=BF16))
                single[0].copy_(normal(40 + 2 * trial + n, *single[0].shape, dtype=BF16))
            graph.replay()
        torch.cuda.synchronize()
        for graph, leaf, params, single, out in graphs:
            fresh = {name: t.detach().clone().requires_grad_() for name, t in params.items()}
            want = (*step(leaf.detach().clone().requires_grad_(), fresh), T.differential_attention(*single))
            for a, b in zip(out, want):
                assert torch.equal(a, b)


def test_offsets_past_32_bits(T):
    """rows, tokens and stored keys whose last elements lie more than 2^32 bytes from the first: what a copy that does not gives"""
    w, rows = normal(1, 24, 1024).cuda(), (1 << 31) // 1024 + 100
    x = torch.zeros(rows, 1024, dtype=F16, device="cuda")
    x[-200:] = normal(2, 200, 1024)
    # other tiles add up in another order: half a step of f16 on either side, and sums of 1024 (200) products in 32 bits, 2^-24 of their size each
    assert torch.allclose(T.linear(x, w)[-200:], T.linear(x[-200:].clone(), w), rtol=2 ** -10, atol=2 * 1024 * 1024 * 2.0 ** -24)
    y = torch.zeros(rows, 24, dtype=F16, device="cuda")
    y[-200:] = normal(3, 200, 24)
    leaf, part, weight = x.requires_grad_(), x[-200:].detach().clone().requires_grad_(), w.requires_grad_()
    dx, dw = torch.autograd.grad(T.linear(leaf, weight), [leaf, weight], y)
    ex, ew = torch.autograd.grad(T.linear(part, weight), [part, weight], y[-200:].contiguous())
    assert torch.allclose(dx[-200:], ex, rtol=2 ** -10, atol=2 * 24 * 24 * 2.0 ** -24) and torch.allclose(dw, ew, rtol=2 ** -10, atol=2 * 200 * 200 * 2.0 ** -24)
    assert not dx[:-200].any()
    del x, leaf, dx

    positions = torch.arange(300, dtype=torch.int32, device="cuda")[:, None]
    store = torch.zeros(1, 300, 1 << 23, dtype=F16, device="cuda")            # 5 GB
    h, hk, d = 4, 2, 64
    store[..., : 2 * hk * d] = normal(4, 1, 300, 2 * hk * d)
    store[..., 4096 : 4096 + hk * 2 * d] = normal(5, 1, 300, hk * 2 * d)
    k, v = store[..., : 2 * hk * d].unflatten(-1, (2 * hk, d)), store[..., 4096 : 4096 + hk * 2 * d].unflatten(-1, (hk, 2 * d))
    assert torch.equal(T.rotary(k, None, positions, (d // 2,)), T.rotary(k.contiguous(), None, positions, (d // 2,)))
    lam = torch.tensor([0.2, 0.4, 0.6, 0.8], device="cuda")
    for nq in (1, 300):
        q = normal(6, 1, nq, 2 * h, d).cuda()
        got, want = ([t.detach().requires_grad_() for t in (q, kk, vv)] for kk, vv in ((k, v), (k.contiguous(), v.contiguous())))
        o, p = T.differential_attention(*got, lam, causal=True), T.differential_attention(*want, lam, causal=True)
        assert torch.equal(o, p)
        g = normal(7, *o.shape).cuda()
        for a, b in zip(torch.autograd.grad(o, got, g), torch.autograd.grad(p, want, g)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("d", [64, 128])
def test_large_kernels_captured_beside_eager_ones(T, d):
    """the kernels that take more LDS than a launch has by default: replayed while eager calls of the same sizes run on another stream"""
    sizes = dict(x=(2048, 1024), w=(2048, 1024), q=(2, 700, 8, d), k=(2, 700, 4, d), v=(2, 700, 2, 2 * d))

    def inputs(seed):
        return {name: normal(seed + i, *size, dtype=BF16, std=0.5).cuda().requires_grad_() for i, (name, size) in enumerate(sizes.items())}

    lam = torch.tensor([0.2, 0.4, 0.6, 0.8], device="cuda", requires_grad=True)

    def work(t):
        y = T.linear(t["x"], t["w"], activation="gelu")
        o = T.differential_attention(t["q"], t["k"], t["v"], lam, causal=True)
        return (y, *torch.autograd.grad(y, [t["x"], t["w"]], torch.ones_like(y)), o,
                *torch.autograd.grad(o, [t["q"], t["k"], t["v"], lam], torch.ones_like(o)))

    mine, side = inputs(1), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(mine)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work(mine)
    others = [inputs(100 * n) for n in range(1, 4)]
    alone = [[t.clone() for t in work(other)] for other in others]
    torch.cuda.synchronize()
    for n, other in enumerate(others):
        with torch.no_grad():
            for name, t in mine.items():
                t.copy_(other[name])
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            beside = work(others[n - 1])
        torch.cuda.synchronize()
        for a, b in zip(out, alone[n]):
            assert torch.equal(a, b)
        for a, b in zip(beside, alone[n - 1]):
            assert torch.equal(a, b)


def test_the_same_bits_every_time(T):
    q, k, v, lam, dout = attention_inputs(2, 150, 150, 4, 2, 64, 128, F16)
    x, w = normal(1, 300, 520), normal(2, 260, 520, std=0.05)

    def once():
        leaves = [t.cuda().requires_grad_() for t in (q, k, v, lam)]
        o = T.differential_attention(*leaves, causal=True)
        lin = [t.cuda().requires_grad_() for t in (x, w)]
        y = T.linear(*lin, activation="gelu")
        return (o, *torch.autograd.grad(o, leaves, dout.cuda()), y, *torch.autograd.grad(y, lin, torch.ones_like(y)))

    first = once()
    for _ in range(3):
        for a, b in zip(first, once()):
            assert torch.equal(a, b)


# ---------------------------------------------------------------------------------------------- refusals
def test_refusals(T):
    x, w = torch.zeros(4, 16, dtype=F16, device="cuda"), torch.zeros(8, 16, dtype=F16, device="cuda")
    for call, error in [
        (lambda: T.linear(x.cpu(), w), RuntimeError), (lambda: T.linear(x.float(), w.float()), TypeError), (lambda: T.linear(x, w.bfloat16()), ValueError),
        (lambda: T.linear(x, w.cpu()), ValueError), (lambda: T.linear(x, w[:, :8]), ValueError), (lambda: T.linear(x, w, w), ValueError),
        (lambda: T.linear(x, w, residual=x), ValueError), (lambda: T.linear(x, w, activation="relu"), NotImplementedError),
        (lambda: T.linear(x[:, :0], w[:, :0]), ValueError),
    ]:
        with pytest.raises(error):
            call()
    q, pos = torch.zeros(2, 5, 4, 16, dtype=F16, device="cuda"), torch.zeros(5, 2, dtype=torch.int32, device="cuda")
    for call, error in [
        (lambda: T.rotary(q.cpu(), None, pos, (4, 4)), RuntimeError), (lambda: T.rotary(q.double(), None, pos, (4, 4)), TypeError),
        (lambda: T.rotary(q, q.bfloat16(), pos, (4, 4)), ValueError), (lambda: T.rotary(q, q[:1], pos, (4, 4)), ValueError),
        (lambda: T.rotary(q, None, pos, (4, 3)), NotImplementedError), (lambda: T.rotary(q, None, pos, (9, -1)), NotImplementedError),
        (lambda: T.rotary(q, None, pos, (8,)), ValueError), (lambda: T.rotary(q, None, pos[:4], (4, 4)), ValueError),
        (lambda: T.rotary(q, None, pos.cpu(), (4, 4)), ValueError), (lambda: T.rotary(q, None, pos.half(), (4, 4)), ValueError),
        (lambda: T.rotary(q, None, pos, (4, 4), base=0.0), NotImplementedError), (lambda: T.rotary(q[..., :15], None, pos, (4, 3)), NotImplementedError),
        (lambda: T.rotary(q, None, pos.float().requires_grad_(), (4, 4)), NotImplementedError),
    ]:
        with pytest.raises(error):
            call()
    k, v, lam = q[:, :, :2], torch.zeros(2, 5, 1, 32, dtype=F16, device="cuda"), torch.zeros(2, dtype=F16, device="cuda")
    A = T.differential_attention
    lengths = torch.zeros(2, dtype=torch.int32, device="cuda")
    for call, error in [
        (lambda: A(q.cpu(), k, v, lam), RuntimeError), (lambda: A(q.float(), k.float(), v.float(), lam.float()), TypeError),
        (lambda: A(q, k.bfloat16(), v, lam), ValueError), (lambda: A(q[:, :, :3], k, v, lam), ValueError), (lambda: A(q, k[:, :4], v, lam), ValueError),
        (lambda: A(q, k, v, lam[:1]), ValueError), (lambda: A(q, k, v, lam.bfloat16()), ValueError), (lambda: A(q, k, v, lam.cpu()), ValueError),
        (lambda: A(q, k, v, lam, q_start=lengths), ValueError), (lambda: A(q, k, v, lam, kv_lengths=lengths[:1]), ValueError),
        (lambda: A(q, k, v, lam, kv_lengths=lengths.float()), ValueError), (lambda: A(q, k, v, lam, kv_lengths=lengths.cpu()), ValueError),
        (lambda: A(q, k, v, lam, scale=-1.0), NotImplementedError), (lambda: A(q, k, v, lam, scale=0.0), NotImplementedError),
        (lambda: A(q[..., :12], k[..., :12], v, lam), NotImplementedError), (lambda: A(q, k, v[..., :12], lam), NotImplementedError), (lambda: A(q[..., :0], k[..., :0], v, lam), ValueError),
    ]:
        with pytest.raises(error):
            call()
    y = T.linear(x.requires_grad_(), w, activation="silu")   # once, not twice
    g, = torch.autograd.grad(y, x, torch.ones_like(y).requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
