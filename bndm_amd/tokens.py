"""Operators over image and video tokens on the HIP path, next to the network's own linear and attention layers:

* ``linear``                  y = act(x W^T + b) + r, a product with bias, activation and residual in one launch
* ``rotary``                  rotary positions on several axes (time, height, width) for query and key heads
* ``differential_attention``  (softmax(q1 k1^T s) - lam softmax(q2 k2^T s)) v, from single tokens to whole clips

Tensors are laid out token by token, ``[batch, tokens, heads, size]``, as a projection leaves them; slices of a packed projection are
taken as they are.  All three have gradients (once, not twice) and run on the current stream of their tensors' device; what they need
beside their results is allocated through torch for the one call, so they can be captured into graphs.  Storage is f16 or bf16
(``rotary`` also f32), sums and statistics are 32 bits.  There is no CPU fallback.
"""
from __future__ import annotations

import ctypes as C

import torch
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
_ACTIVATIONS = {None: 0, "silu": 1, "gelu": 2}
_POSITIONS = {torch.int32: 0, torch.int64: 1, torch.float32: 2}
_Strides = C.c_int64 * 3


# the handle of a device's current stream: what torch.cuda.current_stream(index).cuda_stream is, without making the Stream (2.6 us, more
# than some of these kernels take)
_stream_of = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else \
    lambda index: torch.cuda.current_stream(index).cuda_stream


def _launch(fn, what, device, *args):
    """fn(*args, stream) on the current stream of ``device``."""
    index = device.index
    if index == torch.cuda.current_device():
        rc = fn(*args, _stream_of(index))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _stream_of(index))
    if rc:
        _lib.check_tokens(rc, what)


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _same(what, first, **others):
    """The tensors have the first one's type and device."""
    dtype, device = first.dtype, first.device
    for name, t in others.items():
        if t is not None and (t.dtype != dtype or t.device != device):
            raise ValueError(f"{what}: {name} is {t.dtype} on {t.device}, not {first.dtype} on {first.device}")


def _type_of(what, t, types):
    _lib.require_gpu(t, what)
    if t.dtype not in types:
        raise TypeError(f"{what}: {t.dtype} is not one of {', '.join(str(x) for x in types)}")
    return _DTYPES[t.dtype]


def _recording(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


# ---------------------------------------------------------------------------------------------- linear
def _rows(t, width):
    """``t`` as rows of ``width`` next to each other's elements, and the distance of two rows."""
    if t.dim() != 2:
        t = t.reshape(-1, width)
    if width > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t, t.stride(0) if t.shape[0] > 1 else width


def _linear_forward(x, weight, bias, residual, act, dtype, keep):
    n, k = weight.shape
    rows, ldx = _rows(x, k)
    m = rows.shape[0]
    y = x.new_empty(x.shape[:-1] + (n,))
    z = x.new_empty((m, n)) if keep and act else None
    res, ldr = _rows(residual, n) if residual is not None else (None, 0)
    if m:
        lib = _lib.load_tokens()
        need = lib.bndm_tokens_linear_workspace_bytes(m, n, k)
        work = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
        _launch(lib.bndm_tokens_linear, "linear", x.device, rows.data_ptr(), ldx, weight.data_ptr(), _ptr(bias), _ptr(res), ldr, y.data_ptr(),
                _ptr(z), m, n, k, act, dtype, _ptr(work), need)
    return y, z


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, dtype):
        y, z = _linear_forward(x, weight, bias, residual, act, dtype, any(ctx.needs_input_grad[:3]))
        ctx.act, ctx.dtype = act, dtype
        ctx.save_for_backward(x, weight, z)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, z = ctx.saved_tensors
        n, k = weight.shape
        want_x, want_w, want_b, want_r = ctx.needs_input_grad[:4]
        rows, ldx = _rows(x, k)
        m = rows.shape[0]
        make = torch.empty if m else torch.zeros
        dx = make(x.shape, dtype=x.dtype, device=x.device) if want_x else None
        dw = make(weight.shape, dtype=x.dtype, device=x.device) if want_w else None
        db = make((n,), dtype=x.dtype, device=x.device) if want_b else None
        if m and (want_x or want_w or want_b):
            grad, lddy = _rows(dy, n)
            lib = _lib.load_tokens()
            need = lib.bndm_tokens_linear_backward_workspace_bytes(m, n, k, ctx.act, want_b)
            work = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
            _launch(lib.bndm_tokens_linear_backward, "linear backward", x.device, grad.data_ptr(), lddy, _ptr(z), rows.data_ptr(), ldx,
                    weight.data_ptr(), _ptr(dx), _ptr(dw), _ptr(db), m, n, k, ctx.act, ctx.dtype, _ptr(work), need)
        return dx, dw, db, dy if want_r else None, None, None


def linear(x, weight, bias=None, activation=None, residual=None):
    """``act(x weight^T + bias) + residual``, summed in 32 bits and rounded once.

    x [..., K], weight [N, K], bias [N] or None, residual [..., N] or None, all f16 or all bf16; ``activation`` None, ``"silu"`` or
    ``"gelu"`` (z Phi(z)).  Returns [..., N].  With an activation, a pass that records gradients keeps x weight^T + bias in the
    tensors' type for the backward pass.
    """
    dtype = _type_of("linear(x)", x, (torch.float16, torch.bfloat16))
    if activation not in _ACTIVATIONS:
        raise NotImplementedError(f"linear: activation {activation!r}: None, 'silu' or 'gelu'")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1] or 0 in weight.shape:
        raise ValueError(f"linear: x {tuple(x.shape)} and weight {tuple(weight.shape)} do not go together")
    n = weight.shape[0]
    if bias is not None and bias.shape != (n,):
        raise ValueError(f"linear: bias {tuple(bias.shape)} is not ({n},)")
    if residual is not None and residual.shape != x.shape[:-1] + (n,):
        raise ValueError(f"linear: residual {tuple(residual.shape)} is not {tuple(x.shape[:-1] + (n,))}")
    _same("linear", x, weight=weight, bias=bias, residual=residual)
    weight = weight.contiguous()
    bias = bias.contiguous() if bias is not None else None
    act = _ACTIVATIONS[activation]
    if _recording(x, weight, bias, residual):
        return _Linear.apply(x, weight, bias, residual, act, dtype)
    return _linear_forward(x, weight, bias, residual, act, dtype, False)[0]


# ---------------------------------------------------------------------------------------------- rotary
def _heads_in(t):
    """``t`` [B, N, H, D] with the elements of a head next to each other."""
    return t if t.stride(3) == 1 or t.shape[3] == 1 else t.contiguous()


def _rotary_launch(q, k, positions, sections, base, interleaved, inverse, dtype):
    some = q if q is not None else k
    b, n, _, d = some.shape
    out = []
    args = []
    for t in (q, k):
        if t is None:
            out.append(None)
            args += [0, None, 0, 0]
            continue
        t = _heads_in(t)
        y = torch.empty(t.shape, dtype=t.dtype, device=t.device)
        out.append((y, t))
        args += [t.data_ptr(), _Strides(*t.stride()[:3]), y.data_ptr(), t.shape[2]]
    shared = positions.dim() == 2
    ps = _Strides(0 if shared else positions.stride(0), positions.stride(-2), positions.stride(-1))
    _launch(_lib.load_tokens().bndm_tokens_rotary, "rotary", some.device, *args, positions.data_ptr(), ps, _POSITIONS[positions.dtype], b, n, d,
            (C.c_int * len(sections))(*sections), len(sections), base, interleaved, inverse, dtype)
    return tuple(None if o is None else o[0] for o in out)


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, sections, base, interleaved, dtype):
        ctx.set_materialize_grads(False)
        ctx.how = (sections, base, interleaved, dtype)
        ctx.save_for_backward(positions)
        out = _rotary_launch(q, k, positions, sections, base, interleaved, 0, dtype)
        return out[0] if k is None else out

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk=None):
        sections, base, interleaved, dtype = ctx.how
        dq = dq if ctx.needs_input_grad[0] else None
        dk = dk if ctx.needs_input_grad[1] else None
        if dq is None and dk is None:
            return (None,) * 7
        dq, dk = _rotary_launch(dq, dk, ctx.saved_tensors[0], sections, base, interleaved, 1, dtype)
        return dq, dk, None, None, None, None, None


def rotary(q, k, positions, sections, base=10000.0, interleaved=False):
    """Rotary positions on several axes.

    q [B, N, H, D] and k [B, N, Hk, D] (or None), f16, bf16 or f32, D even up to 256.  ``positions`` [N, axes] or [B, N, axes], int32,
    int64 or float32, up to four axes.  ``sections``: how many of the D / 2 pairs of a head each axis turns, adding up to D / 2; pair i
    of an axis with s pairs turns by ``position * base ** (-i / s)``, an angle formed in 64 bits.  Pairs are elements (j, j + D / 2), or
    (2j, 2j + 1) with ``interleaved``.  Returns new tensors: (q', k'), or q' alone where k is None.
    """
    dtype = _type_of("rotary(q)", q, (torch.float16, torch.bfloat16, torch.float32))
    if q.dim() != 4 or (k is not None and (k.dim() != 4 or k.shape[:2] != q.shape[:2] or k.shape[3] != q.shape[3])):
        raise ValueError(f"rotary: q {tuple(q.shape)} and k {None if k is None else tuple(k.shape)}: [B, N, heads, D] of one B, N and D")
    _same("rotary", q, k=k)
    sections = tuple(int(s) for s in sections)
    if positions.device != q.device or positions.dtype not in _POSITIONS:
        raise ValueError(f"rotary: positions are {positions.dtype} on {positions.device}: int32, int64 or float32 on {q.device}")
    if positions.dim() not in (2, 3) or positions.shape[-2:] != (q.shape[1], len(sections)) or \
            (positions.dim() == 3 and positions.shape[0] != q.shape[0]):
        raise ValueError(f"rotary: positions {tuple(positions.shape)}: [N, axes] or [B, N, axes] for q {tuple(q.shape)} and {len(sections)} axes")
    if positions.requires_grad:
        raise NotImplementedError("rotary: positions have no gradient")
    base, interleaved = float(base), int(bool(interleaved))
    if _recording(q, k):
        return _Rotary.apply(q, k, positions, sections, base, interleaved, dtype)
    out = _rotary_launch(q, k, positions, sections, base, interleaved, 0, dtype)
    return out[0] if k is None else out


# ---------------------------------------------------------------------------------------------- differential attention
def _aligned(t):
    """``t`` [B, N, H, D] as the kernels read it -- heads' elements next to each other, all else in steps of 16 bytes -- and its strides."""
    b, n, h, d = t.shape
    sb, sn, sh, sd = t.stride()
    sb, sn, sh = 0 if b == 1 else sb, 0 if n == 1 else sn, 0 if h == 1 else sh
    if (sd == 1 or d == 1) and not (t.data_ptr() % 16 or sb % 8 or sn % 8 or sh % 8 or sn > 1 << 23):
        return t, (sb, sn, sh)
    t = t.contiguous()
    if t.data_ptr() % 16 or d % 8:                          # (a head size that the kernels refuse: any strides will do)
        t = t.clone(memory_format=torch.contiguous_format)
    return t, (n * h * d, h * d, d)


def _attention_forward(q, k, v, lam, q_start, kv_lengths, causal, scale, dtype, keep):
    b, nq, maps, d = q.shape
    (q, qs), (k, ks), (v, vs) = _aligned(q), _aligned(k), _aligned(v)
    shape = _lib.AttentionShape(b, nq, k.shape[1], maps // 2, v.shape[2], d, v.shape[3], *qs, *ks, *vs, causal, dtype, lam.dtype == torch.float32, scale)
    o = torch.empty((b, nq, maps // 2, v.shape[3]), dtype=q.dtype, device=q.device)
    o2 = torch.empty_like(o) if keep else None
    lse = torch.empty((b, maps, nq), dtype=torch.float32, device=q.device) if keep else None
    lib = _lib.load_tokens()
    need = lib.bndm_tokens_attention_workspace_bytes(shape)
    work = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    _launch(lib.bndm_tokens_attention, "differential_attention", q.device, shape, q.data_ptr(), k.data_ptr(), v.data_ptr(), lam.data_ptr(),
            _ptr(q_start), _ptr(kv_lengths), o.data_ptr(), _ptr(o2), _ptr(lse), _ptr(work), need)
    return o, o2, lse


class _DifferentialAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lam, q_start, kv_lengths, causal, scale, dtype):
        o, o2, lse = _attention_forward(q, k, v, lam, q_start, kv_lengths, causal, scale, dtype, True)
        ctx.how = (causal, scale, dtype)
        ctx.save_for_backward(q, k, v, lam, q_start, kv_lengths, o, o2, lse)
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, lam, q_start, kv_lengths, o, o2, lse = ctx.saved_tensors
        causal, scale, dtype = ctx.how
        new = lambda t: torch.empty(t.shape, dtype=t.dtype, device=t.device)
        dq, dk, dv, dlam = new(q), new(k), new(v), new(lam)
        if q.shape[0] == 0 or q.shape[1] == 0:
            for t in (dq, dk, dv, dlam):
                t.zero_()
        else:
            b, nq, maps, d = q.shape
            (q, qs), (k, ks), (v, vs), (dout, ds) = _aligned(q), _aligned(k), _aligned(v), _aligned(dout)
            shape = _lib.AttentionShape(b, nq, k.shape[1], maps // 2, v.shape[2], d, v.shape[3], *qs, *ks, *vs, causal, dtype,
                                        lam.dtype == torch.float32, scale)
            lib = _lib.load_tokens()
            need = lib.bndm_tokens_attention_backward_workspace_bytes(shape)
            work = torch.empty(need, dtype=torch.uint8, device=q.device)
            _launch(lib.bndm_tokens_attention_backward, "differential_attention backward", q.device, shape, q.data_ptr(), k.data_ptr(),
                    v.data_ptr(), lam.data_ptr(), _ptr(q_start), _ptr(kv_lengths), o.data_ptr(), o2.data_ptr(), lse.data_ptr(),
                    dout.data_ptr(), _Strides(*ds), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), dlam.data_ptr(), work.data_ptr(),
                    need)
        want = ctx.needs_input_grad
        return (dq if want[0] else None, dk if want[1] else None, dv if want[2] else None, dlam if want[3] else None) + (None,) * 5


def _per_sequence(what, t, q):
    if t is None:
        return None
    if t.shape != (q.shape[0],) or t.device != q.device or t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"differential_attention: {what} is {t.dtype} {tuple(t.shape)} on {t.device}: int32 ({q.shape[0]},) on {q.device}")
    return t.to(torch.int32).contiguous()


def differential_attention(q, k, v, lam, causal=False, q_start=None, kv_lengths=None, scale=None):
    """``(softmax(scale q1 k1^T) - lam softmax(scale q2 k2^T)) v`` for every head.

    q [B, Nq, 2 H, D]: heads 2h and 2h + 1 hold the first and second map of head h; k [B, Nk, 2 Hk, D] likewise; v [B, Nk, Hk, Dv]; H a
    multiple of Hk, head h reads key head h // (H // Hk).  f16 or bf16; D a multiple of 8 up to 128, Dv up to 256.  lam [H], of the same
    type or float32.  ``scale``: 1 / sqrt(D) unless given, positive.  Returns [B, Nq, H, Dv].

    ``kv_lengths`` int32 [B]: the keys of each sequence; what lies past them is not read, and its gradients are zero.  ``causal``:
    query i of a sequence sees keys up to ``q_start + i``; ``q_start`` int32 [B] is where its first query stands among the keys, Nk - Nq
    unless given (0 for whole sequences, the tokens before it for a step that appends to stored keys).  A query that sees no key
    gives zeros.  Within a sequence's length, values that only later queries see must be finite numbers.

    With gradients, the weights and their gradients are rounded to the tensors' type between products: f16 gradients below about
    1e-5 of a score's lose digits, so scale a loss as for any f16 training.
    """
    dtype = _type_of("differential_attention(q)", q, (torch.float16, torch.bfloat16))
    if any(t.dim() != 4 for t in (q, k, v)) or q.shape[2] % 2 or k.shape[2] != 2 * v.shape[2] or k.shape[:2] != v.shape[:2] or \
            q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3] or v.shape[2] < 1 or q.shape[2] < 2 or q.shape[3] < 1 or (q.shape[2] // 2) % v.shape[2]:
        raise ValueError(f"differential_attention: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}: "
                         "[B, Nq, 2 H, D], [B, Nk, 2 Hk, D], [B, Nk, Hk, Dv] with H a multiple of Hk")
    if lam.shape != (q.shape[2] // 2,) or lam.device != q.device or lam.dtype not in (q.dtype, torch.float32):
        raise ValueError(f"differential_attention: lam is {lam.dtype} {tuple(lam.shape)} on {lam.device}: {q.dtype} or float32 "
                         f"({q.shape[2] // 2},) on {q.device}")
    _same("differential_attention", q, k=k, v=v)
    if q_start is not None and not causal:
        raise ValueError("differential_attention: q_start says where a causal mask begins: causal is False")
    scale = float(q.shape[3]) ** -0.5 if scale is None else float(scale)
    lam = lam.contiguous()
    q_start, kv_lengths = _per_sequence("q_start", q_start, q), _per_sequence("kv_lengths", kv_lengths, q)
    if _recording(q, k, v, lam):
        return _DifferentialAttention.apply(q, k, v, lam, q_start, kv_lengths, int(bool(causal)), scale, dtype)
    return _attention_forward(q, k, v, lam, q_start, kv_lengths, int(bool(causal)), scale, dtype, False)[0]
