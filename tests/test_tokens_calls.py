"""CPU checks of bndm_amd.tokens' Python side: calls whose results would be wrong in silence are refused before anything is launched.  Where a call
has to get past the device check, the launch is replaced by one that only counts."""
import pytest
import torch
from torch.autograd import forward_ad

F16 = torch.float16


@pytest.fixture
def T(monkeypatch):
    """bndm_amd.tokens with CPU tensors let through and nothing launched; T.launches names the calls"""
    from bndm_amd import tokens
    monkeypatch.setattr(tokens, "_type_of", lambda what, t, types: types[t.dtype])
    monkeypatch.setattr(tokens, "launches", [], raising=False)
    monkeypatch.setattr(tokens, "_launch", lambda fn, what, index, *args: tokens.launches.append((what, *args)))
    return tokens


def calls(T):
    """name -> (call of one tensor, that tensor)"""
    zeros = lambda *shape: torch.zeros(*shape, dtype=F16)
    w, pos = zeros(24, 16), torch.zeros(5, 2, dtype=torch.int32)
    k, v, lam = zeros(2, 5, 2, 16), zeros(2, 5, 1, 32), zeros(2)
    return {"linear": (lambda t: T.linear(t, w, activation="silu"), zeros(3, 16)), "rotary": (lambda t: T.rotary(t, None, pos, (4, 4)), zeros(2, 5, 4, 16)),
            "differential_attention": (lambda t: T.differential_attention(t, k, v, lam), zeros(2, 5, 4, 16))}


OPERATORS = ["linear", "rotary", "differential_attention"]


# ---------------------------------------------------------------------------------------------- who follows torch's operators misses these
@pytest.mark.parametrize("name", OPERATORS)
@pytest.mark.parametrize("leaf", [False, True])
def test_forward_mode_is_refused(T, name, leaf):
    call, x = calls(T)[name]
    with forward_ad.dual_level():
        call(x)                                              # (a tensor without a tangent is one like any other)
        before = len(T.launches)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(forward_ad.make_dual(x.clone().requires_grad_(leaf), torch.ones_like(x)))
        assert len(T.launches) == before
        other = x.clone().requires_grad_()
        y = call(other)
        before = len(T.launches)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(y, other, forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y)))
        assert len(T.launches) == before
    call(x)


def test_forward_mode_of_any_input_is_refused(T):
    x, w, b, r = (torch.zeros(*s, dtype=F16) for s in ((3, 16), (24, 16), (24,), (3, 24)))
    q, k, v, lam = (torch.zeros(*s, dtype=F16) for s in ((2, 5, 4, 16), (2, 5, 2, 16), (2, 5, 1, 32), (2,)))
    pos = torch.zeros(5, 2, dtype=torch.int32)
    for call, tensors in ((lambda x, w, b, r: T.linear(x, w, b, residual=r), [x, w, b, r]), (lambda q, k: T.rotary(q, k, pos, (4, 4)), [q, k]),
                          (T.differential_attention, [q, k, v, lam])):
        for at, t in enumerate(tensors):
            with forward_ad.dual_level():
                some = list(tensors)
                some[at] = forward_ad.make_dual(t, torch.ones_like(t))
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call(*some)
    assert T.launches == []


@pytest.mark.parametrize("name", OPERATORS)
def test_tracers_are_refused(T, name):
    from torch.fx.experimental.proxy_tensor import make_fx
    call, x = calls(T)[name]
    for trace in (lambda: torch.jit.trace(call, (x,), check_trace=False), lambda: make_fx(call)(x), lambda: make_fx(call, pre_dispatch=True)(x),
                  lambda: make_fx(call, tracing_mode="fake")(x)):
        with pytest.raises(NotImplementedError, match="tracer"):
            trace()
    assert T.launches == []
    call(x)
    assert len(T.launches) == 1


def test_optional_tensors_without_memory_are_refused(T):
    """an address of 0 stands for none"""
    class Wrapper(torch.Tensor):
        @staticmethod
        def __new__(cls, shape, dtype):
            return torch.Tensor._make_wrapper_subclass(cls, shape, dtype=dtype)

        @classmethod
        def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
            if func is torch.ops.aten.detach.default:
                return args[0]
            raise AssertionError(func)

    x, w = torch.zeros(3, 16, dtype=F16), torch.zeros(24, 16, dtype=F16)
    with pytest.raises(NotImplementedError, match="no memory"):
        T.linear(x, w, Wrapper((24,), F16))
    q, k, v, lam = (torch.zeros(*s, dtype=F16) for s in ((2, 5, 4, 16), (2, 5, 2, 16), (2, 5, 1, 32), (2,)))
    for name in ("q_start", "kv_lengths"):
        with pytest.raises(NotImplementedError, match="no memory"):
            T.differential_attention(q, k, v, lam, causal=True, **{name: Wrapper((2,), torch.int32)})
    assert T.launches == []


# ---------------------------------------------------------------------------------------------- rows and numbers that the kernels do not take as they are
def test_linear_rows_further_apart_than_the_kernels_take(T):
    """the last token of each of some long sequences; a gradient that arrives so"""
    far = (1 << 22) + 1
    h = torch.empty(3, far, dtype=F16)
    h[:, -16:] = torch.arange(48, dtype=F16).reshape(3, 16)
    w = torch.zeros(24, 16, dtype=F16).requires_grad_()
    y = T.linear(h[:, -16:], w)
    grad = h[:, -24:]
    torch.autograd.grad(y, w, grad)
    T.linear(h[:, -16:].detach(), w.detach(), residual=h[:, -24:])
    (_, x, ldx, *_), (_, dy, lddy, _, x2, ldx2, *_), (_, *last) = T.launches
    assert (ldx, lddy, ldx2, last[1], last[5]) == (16, 24, 16, 16, 24)
    assert T._rows(h[:, -16:], 16)[0].equal(h[:, -16:]) and T._rows(h[:1, -16:], 16)[0].data_ptr() == h[:1, -16:].data_ptr()
    near = torch.empty(2, 1 << 22, dtype=F16)
    rows, m, step = T._rows(near[:, 8:24], 16)
    assert rows.data_ptr() == near[:, 8:24].data_ptr() and (m, step) == (2, 1 << 22)


def test_places_past_32_bits(T):
    """int64 lengths and starts beyond 32 bits ("all of them") stay on their side of every key"""
    q = torch.zeros(4, 1, 2, 16, dtype=F16)
    big = torch.tensor([2 ** 63 - 1, 2 ** 32 + 5, -2 ** 40, 7])
    assert T._per_sequence("kv_lengths", big, q).tolist() == [2 ** 31 - 1, 2 ** 31 - 1, -2 ** 31, 7]
    same = torch.tensor([1, 2, 3, 4], dtype=torch.int32)
    assert T._per_sequence("q_start", same, q) is same
    wide = torch.tensor([[1, 2, 3, 4], [5, 6, 7, 8]], dtype=torch.int32).t()[:, 0]
    assert T._per_sequence("q_start", wide, q).tolist() == [1, 2, 3, 4] and T._per_sequence("q_start", wide, q).is_contiguous()


def test_more_heads_than_a_launch_takes():
    """the backward pass has a workgroup for each head and for each sequence's key heads in one launch"""
    from bndm_amd import _lib
    lib, P = _lib.load_tokens(), 4096                        # (4096 stands for a tensor: refused before any is read)
    b = (1 << 20) - 1
    strides = (16 * 32, 16 * 32, 16)
    shape = _lib.AttentionShape(b, 1, 1, 16, 16, 16, 16, *strides, *strides, *strides, 0, 0, 0, 0.25)
    need = lib.bndm_tokens_attention_backward_workspace_bytes(shape)
    rc = lib.bndm_tokens_attention_backward(shape, P, P, P, P, 0, 0, P, P, P, P, strides_of(strides), P, P, P, P, P, need, None)
    assert rc == -1 and b"more heads" in lib.bndm_tokens_last_error()


def strides_of(values):
    import ctypes
    return (ctypes.c_int64 * 3)(*values)
