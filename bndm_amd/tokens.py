"""Operators over image and video tokens on the HIP path, next to the network's own linear and attention layers:

* ``linear``                  y = act(x W^T + b) + r, a product with bias, activation and residual in one launch
* ``rotary``                  rotary positions on several axes (time, height, width) for query and key heads
* ``differential_attention``  (softmax(q1 k1^T s) - lam softmax(q2 k2^T s)) v, from single tokens to whole clips

Tensors are laid out token by token, ``[batch, tokens, heads, size]``, as a projection leaves them; slices of a packed projection are
taken as they are.  All three have gradients (once, not twice) and run on the current stream of their tensors' device; what they need
beside their results is allocated through torch for the one call, so they can be captured into graphs.  Storage is f16 or bf16
(``rotary`` also f32), sums and statistics are 32 bits.  There is no CPU fallback.  Forward-mode derivatives, tracers (``torch.jit.trace``,
``make_fx``) and tensors without memory of their own are refused.
"""
from __future__ import annotations

import ctypes as C
import functools
import sys

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

_HALVES = {torch.float16: 0, torch.bfloat16: 1}
_FLOATS = {**_HALVES, torch.float32: 2}
_ACTIVATIONS = {None: 0, "silu": 1, "gelu": 2}
_POSITIONS = {torch.int32: 0, torch.int64: 1, torch.float32: 2}
_Strides = C.c_int64 * 3


# Small calls are bound by what happens here, so it is kept short.  A device's current stream and the current device are asked for
# without making a Stream (2.6 us) or checking that there is a device (the tensors are on one).
_stream_of = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else \
    lambda index: torch.cuda.current_stream(index).cuda_stream
_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device


def _launch(fn, what, index, *args):
    """fn(*args, stream) on the current stream of device ``index``."""
    if index == _current_device():
        rc = fn(*args, _stream_of(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _stream_of(index))
    if rc:
        _lib.check_tokens(rc, what)


def _ptr(t):
    """An optional tensor's address: 0 stands for none, which a tensor without memory (a wrapper) must not pass for."""
    if t is None:
        return 0
    at = t.data_ptr()
    if not at and t.numel():
        raise NotImplementedError(f"{type(t).__name__} has no memory of its own for a kernel to read")
    return at


def _refuse_onlookers(what, *tensors):
    """The kernels take addresses, so what follows torch's operators by watching them would miss these: a tangent would end here and count
    as zero, a recorded graph would hold the allocation of the result and nothing that fills it."""
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError(f"{what}: no forward-mode derivatives")
    tracing = torch._C._is_tracing()
    if torch._C._len_torch_dispatch_stack() or torch._C._len_torch_function_stack():    # (or no tracer of torch.fx is at work: 2 us saved)
        proxies = sys.modules.get("torch.fx.experimental.proxy_tensor")                 # (loaded by whoever traces)
        tracing = tracing or (proxies is not None and proxies.get_proxy_mode() is not None)
    if tracing:
        raise NotImplementedError(f"{what}: a tracer would record its allocations only")


def _same(what, first, others):
    """The tensors (pairs of name and tensor or None) have the first one's type and device."""
    dtype, index = first.dtype, first.get_device()
    for name, t in others:
        if t is not None and (t.dtype is not dtype or t.get_device() != index):
            raise ValueError(f"{what}: {name} is {t.dtype} on {t.device}, not {first.dtype} on {first.device}")


def _type_of(what, t, types):
    if not t.is_cuda:
        _lib.require_gpu(t, what)
    dtype = types.get(t.dtype)
    if dtype is None:
        raise TypeError(f"{what}: {t.dtype} is not one of {', '.join(str(x) for x in types)}")
    return dtype


def _recording(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


# ---------------------------------------------------------------------------------------------- linear
def _rows(t, width):
    """``t`` as rows of ``width`` next to each other's elements, their number, and the distance of two rows, which the kernels take up to 2^22."""
    if t.dim() != 2:
        t = t.reshape(-1, width)
    step, inner = t.stride()
    m = t.shape[0]
    if (inner != 1 and width > 1) or (step > 1 << 22 and m > 1):
        t = t.contiguous()
        step = width
    return t, m, step if m > 1 else width


@functools.lru_cache(maxsize=256)
def _linear_work(m, n, k):
    return _lib.load_tokens().bndm_tokens_linear_workspace_bytes(m, n, k)


def _linear_forward(x, weight, bias, residual, act, dtype, keep):
    n, k = weight.shape
    rows, m, ldx = _rows(x, k)
    y = x.new_empty((*x.shape[:-1], n) if x.dim() != 2 else (m, n))
    z = x.new_empty((m, n)) if keep and act else None
    res, _, ldr = _rows(residual, n) if residual is not None else (None, 0, 0)
    if m:
        need = _linear_work(m, n, k)
        work = x.new_empty(need, dtype=torch.uint8) if need else None
        _launch(_lib.load_tokens().bndm_tokens_linear, "linear", x.get_device(), rows.data_ptr(), ldx, weight.data_ptr(), _ptr(bias), _ptr(res), ldr,
                y.data_ptr(), _ptr(z), m, n, k, act, dtype, _ptr(work), need)
    return y, z


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, dtype):
        y, z = _linear_forward(x, weight, bias, residual, act, dtype, True in ctx.needs_input_grad[:3])
        ctx.act, ctx.dtype = act, dtype
        ctx.save_for_backward(x, weight, z)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _refuse_onlookers("linear backward", dy)
        x, weight, z = ctx.saved_tensors
        n, k = weight.shape
        want_x, want_w, want_b, want_r = ctx.needs_input_grad[:4]
        rows, m, ldx = _rows(x, k)
        make = x.new_empty if m else x.new_zeros
        dx = make(x.shape) if want_x else None
        dw = make((n, k)) if want_w else None
        db = make(n) if want_b else None
        if m and (want_x or want_w or want_b):
            grad, _, lddy = _rows(dy, n)
            lib = _lib.load_tokens()
            need = lib.bndm_tokens_linear_backward_workspace_bytes(m, n, k, ctx.act, want_b)
            work = x.new_empty(need, dtype=torch.uint8) if need else None
            _launch(lib.bndm_tokens_linear_backward, "linear backward", x.get_device(), grad.data_ptr(), lddy, _ptr(z), rows.data_ptr(), ldx,
                    weight.data_ptr(), _ptr(dx), _ptr(dw), _ptr(db), m, n, k, ctx.act, ctx.dtype, _ptr(work), need)
        return dx, dw, db, dy if want_r else None, None, None


def linear(x, weight, bias=None, activation=None, residual=None):
    """``act(x weight^T + bias) + residual``, summed in 32 bits and rounded once.

    x [..., K], weight [N, K], bias [N] or None, residual [..., N] or None, all f16 or all bf16; ``activation`` None, ``"silu"`` or
    ``"gelu"`` (z Phi(z)).  Returns [..., N].  With an activation, a pass that records gradients keeps x weight^T + bias in the
    tensors' type for the backward pass.
    """
    _refuse_onlookers("linear", x, weight, bias, residual)
    dtype = _type_of("linear(x)", x, _HALVES)
    act = _ACTIVATIONS.get(activation)
    if act is None:
        raise NotImplementedError(f"linear: activation {activation!r}: None, 'silu' or 'gelu'")
    shape, of = tuple(x.shape), tuple(weight.shape)
    if len(of) != 2 or not shape or shape[-1] != of[1] or 0 in of:
        raise ValueError(f"linear: x {shape} and weight {of} do not go together")
    if bias is not None and bias.shape != of[:1]:
        raise ValueError(f"linear: bias {tuple(bias.shape)} is not ({of[0]},)")
    if residual is not None and residual.shape != shape[:-1] + of[:1]:
        raise ValueError(f"linear: residual {tuple(residual.shape)} is not {shape[:-1] + of[:1]}")
    _same("linear", x, (("weight", weight), ("bias", bias), ("residual", residual)))
    weight = weight.contiguous()
    if bias is not None:
        bias = bias.contiguous()
    if _recording(x, weight, bias, residual):
        return _Linear.apply(x, weight, bias, residual, act, dtype)
    return _linear_forward(x, weight, bias, residual, act, dtype, False)[0]


# ---------------------------------------------------------------------------------------------- rotary
@functools.lru_cache(maxsize=64)
def _sections_of(sections):
    return (C.c_int * len(sections))(*sections)


def _rotary_launch(q, k, positions, sections, base, interleaved, inverse, dtype):
    some = q if q is not None else k
    b, n, _, d = some.shape
    strides, args, out = [], [], []
    for t in (q, k):
        if t is None:
            out.append(None)
            strides += (0, 0, 0)
            args.append((0, 0, 0))
            continue
        if t.stride(3) != 1 and d != 1:
            t = t.contiguous()
        y = t.new_empty(t.shape)
        out.append(y)
        strides += t.stride()[:3]
        args.append((t.data_ptr(), y.data_ptr(), t.shape[2], t))    # (t stays until the launch)
    at = positions.stride()
    strides = (C.c_int64 * 9)(*strides, 0 if len(at) == 2 else at[0], at[-2], at[-1])
    s = C.addressof(strides)
    _launch(_lib.load_tokens().bndm_tokens_rotary, "rotary", some.get_device(), args[0][0], s, args[0][1], args[0][2], args[1][0], s + 24,
            args[1][1], args[1][2], positions.data_ptr(), s + 48, _POSITIONS[positions.dtype], b, n, d, _sections_of(sections), len(sections),
            base, interleaved, inverse, dtype)
    return out


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, sections, base, interleaved, dtype):
        ctx.set_materialize_grads(False)
        ctx.how = (sections, base, interleaved, dtype)
        ctx.save_for_backward(positions)
        out = _rotary_launch(q, k, positions, sections, base, interleaved, 0, dtype)
        return out[0] if k is None else tuple(out)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk=None):
        _refuse_onlookers("rotary backward", dq, dk)
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
    _refuse_onlookers("rotary", q, k, positions)
    dtype = _type_of("rotary(q)", q, _FLOATS)
    shape, other, where = tuple(q.shape), None if k is None else tuple(k.shape), tuple(positions.shape)
    if len(shape) != 4 or (k is not None and (len(other) != 4 or other[:2] != shape[:2] or other[3] != shape[3])):
        raise ValueError(f"rotary: q {shape} and k {other}: [B, N, heads, D] of one B, N and D")
    _same("rotary", q, (("k", k),))
    sections = tuple(map(int, sections))
    if positions.get_device() != q.get_device() or positions.dtype not in _POSITIONS:
        raise ValueError(f"rotary: positions are {positions.dtype} on {positions.device}: int32, int64 or float32 on {q.device}")
    if where != (shape[1], len(sections)) and where != (shape[0], shape[1], len(sections)):
        raise ValueError(f"rotary: positions {where}: [N, axes] or [B, N, axes] for q {shape} and {len(sections)} axes")
    if positions.requires_grad:
        raise NotImplementedError("rotary: positions have no gradient")
    base, interleaved = float(base), int(bool(interleaved))
    if _recording(q, k):
        return _Rotary.apply(q, k, positions, sections, base, interleaved, dtype)
    out = _rotary_launch(q, k, positions, sections, base, interleaved, 0, dtype)
    return out[0] if k is None else tuple(out)


# ---------------------------------------------------------------------------------------------- differential attention
def _aligned(t):
    """``t`` [B, N, H, D] as the kernels read it -- heads' elements next to each other, all else in steps of 16 bytes -- and its strides."""
    b, n, h, d = t.shape
    sb, sn, sh, sd = t.stride()
    sb, sn, sh = sb * (b > 1), sn * (n > 1), sh * (h > 1)       # (of one there is no distance)
    if (sd == 1 or d == 1) and not (t.data_ptr() % 16 or sb % 8 or sn % 8 or sh % 8 or sn > 1 << 23):
        return t, (sb, sn, sh)
    t = t.contiguous()
    if t.data_ptr() % 16 or d % 8:                          # (a head size that the kernels refuse: any strides will do)
        t = t.clone(memory_format=torch.contiguous_format)
    return t, (n * h * d, h * d, d)


@functools.lru_cache(maxsize=256)
def _attention_work(backward, b, nq, nk, h, hk, d, dv):
    """Bytes of scratch (0 for sizes that the call itself refuses)."""
    lib = _lib.load_tokens()
    ask = lib.bndm_tokens_attention_backward_workspace_bytes if backward else lib.bndm_tokens_attention_workspace_bytes
    return ask(_lib.AttentionShape(b, nq, nk, h, hk, d, dv, *(0,) * 9, 0, 0, 0, 1.0))


def _attention_forward(q, k, v, lam, q_start, kv_lengths, causal, scale, dtype, keep):
    b, nq, maps, d = q.shape
    _, nk, hk, dv = v.shape
    (q, qs), (k, ks), (v, vs) = _aligned(q), _aligned(k), _aligned(v)
    shape = _lib.AttentionShape(b, nq, nk, maps // 2, hk, d, dv, *qs, *ks, *vs, causal, dtype, lam.dtype is torch.float32, scale)
    o = q.new_empty((b, nq, maps // 2, dv))
    o2 = q.new_empty((b, nq, maps // 2, dv)) if keep else None
    lse = q.new_empty((b, maps, nq), dtype=torch.float32) if keep else None
    need = _attention_work(False, b, nq, nk, maps // 2, hk, d, dv)
    work = q.new_empty(need, dtype=torch.uint8) if need else None
    _launch(_lib.load_tokens().bndm_tokens_attention, "differential_attention", q.get_device(), shape, q.data_ptr(), k.data_ptr(), v.data_ptr(), lam.data_ptr(),
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
        _refuse_onlookers("differential_attention backward", dout)
        q, k, v, lam, q_start, kv_lengths, o, o2, lse = ctx.saved_tensors
        causal, scale, dtype = ctx.how
        dq, dk, dv, dlam = (t.new_empty(t.shape) for t in (q, k, v, lam))
        if q.shape[0] == 0 or q.shape[1] == 0:
            for t in (dq, dk, dv, dlam):
                t.zero_()
        else:
            b, nq, maps, d = q.shape
            (q, qs), (k, ks), (v, vs), (dout, ds) = _aligned(q), _aligned(k), _aligned(v), _aligned(dout)
            shape = _lib.AttentionShape(b, nq, k.shape[1], maps // 2, v.shape[2], d, v.shape[3], *qs, *ks, *vs, causal, dtype,
                                        lam.dtype is torch.float32, scale)
            need = _attention_work(True, b, nq, k.shape[1], maps // 2, v.shape[2], d, v.shape[3])
            work = q.new_empty(need, dtype=torch.uint8)
            _launch(_lib.load_tokens().bndm_tokens_attention_backward, "differential_attention backward", q.get_device(), shape, q.data_ptr(), k.data_ptr(),
                    v.data_ptr(), lam.data_ptr(), _ptr(q_start), _ptr(kv_lengths), o.data_ptr(), o2.data_ptr(), lse.data_ptr(),
                    dout.data_ptr(), _Strides(*ds), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), dlam.data_ptr(), work.data_ptr(),
                    need)
        want = ctx.needs_input_grad
        return (dq if want[0] else None, dk if want[1] else None, dv if want[2] else None, dlam if want[3] else None) + (None,) * 5


def _per_sequence(what, t, q):
    if t is None:
        return None
    if t.shape != (q.shape[0],) or t.get_device() != q.get_device() or t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"differential_attention: {what} is {t.dtype} {tuple(t.shape)} on {t.device}: int32 ({q.shape[0]},) on {q.device}")
    if t.dtype is torch.int64:
        t = t.clamp(-(1 << 31), (1 << 31) - 1).to(torch.int32)      # (further out than any key either way: wrapped, it would be among them)
    return t.contiguous()


def differential_attention(q, k, v, lam, causal=False, q_start=None, kv_lengths=None, scale=None):
    """``(softmax(scale q1 k1^T) - lam softmax(scale q2 k2^T)) v`` for every head.

    q [B, Nq, 2 H, D]: heads 2h and 2h + 1 hold the first and second map of head h; k [B, Nk, 2 Hk, D] likewise; v [B, Nk, Hk, Dv]; H a
    multiple of Hk, head h reads key head h // (H // Hk).  f16 or bf16; D a multiple of 8 up to 128, Dv up to 256.  lam [H], of the same
    type or float32.  ``scale``: 1 / sqrt(D) unless given, positive.  Returns [B, Nq, H, Dv].

    ``kv_lengths`` int32 (or int64) [B]: the keys of each sequence; what lies past them is not read, and its gradients are zero.  ``causal``:
    query i of a sequence sees keys up to ``q_start + i``; ``q_start``, likewise, is where its first query stands among the keys, Nk - Nq
    unless given (0 for whole sequences, the tokens before it for a step that appends to stored keys).  A query that sees no key
    gives zeros.  What no query of a sequence sees may hold anything; keys and values that only its later queries see must be finite numbers.

    In the backward pass weights and their gradients are rounded to the tensors' type between products, the gradients as parts of the
    largest of their sequence and key head, so that f16 gradients lose nothing to a loss's factor but what q, k, v's own gradients do.
    """
    _refuse_onlookers("differential_attention", q, k, v, lam)
    dtype = _type_of("differential_attention(q)", q, _HALVES)
    qs, ks, vs = tuple(q.shape), tuple(k.shape), tuple(v.shape)
    if len(qs) != 4 or len(ks) != 4 or len(vs) != 4 or qs[0] != ks[0] or ks[:2] != vs[:2] or qs[3] != ks[3] or qs[3] < 1 or vs[2] < 1 or \
            ks[2] != 2 * vs[2] or qs[2] < 2 or qs[2] % ks[2]:
        raise ValueError(f"differential_attention: q {qs}, k {ks}, v {vs}: [B, Nq, 2 H, D], [B, Nk, 2 Hk, D], [B, Nk, Hk, Dv] with H a multiple of Hk")
    heads = qs[2] // 2
    if lam.shape != (heads,) or lam.get_device() != q.get_device() or lam.dtype not in (q.dtype, torch.float32):
        raise ValueError(f"differential_attention: lam is {lam.dtype} {tuple(lam.shape)} on {lam.device}: {q.dtype} or float32 ({heads},) on {q.device}")
    _same("differential_attention", q, (("k", k), ("v", v)))
    if q_start is not None and not causal:
        raise ValueError("differential_attention: q_start says where a causal mask begins: causal is False")
    scale = qs[3] ** -0.5 if scale is None else float(scale)
    lam = lam.contiguous()
    q_start, kv_lengths = _per_sequence("q_start", q_start, q), _per_sequence("kv_lengths", kv_lengths, q)
    if _recording(q, k, v, lam):
        return _DifferentialAttention.apply(q, k, v, lam, q_start, kv_lengths, int(bool(causal)), scale, dtype)
    return _attention_forward(q, k, v, lam, q_start, kv_lengths, int(bool(causal)), scale, dtype, False)[0]
