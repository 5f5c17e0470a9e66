"""CPU checks of libbndm_tokens.so's boundary: it exports what include/bndm_tokens.h declares, and refuses bad arguments before any launch."""
import ctypes as C
import os
import re
import struct
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 4096                                                     # stands for a tensor: nothing below gets as far as reading one


def declared():
    text = open(os.path.join(ROOT, "include", "bndm_tokens.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    return sorted(set(re.findall(r"\b(bndm_tokens_[a-z0-9_]+)\s*\(", text)))


@pytest.fixture(scope="module")
def lib():
    from bndm_amd import _lib
    return _lib.load_tokens()


def test_header_and_ctypes_table_agree(lib):
    from bndm_amd import _lib
    assert declared() == sorted(_lib.TOKENS_SIGNATURES)
    assert all(hasattr(lib, name) for name in declared())
    assert lib.bndm_tokens_abi_version() == 1


def test_fails_loudly_without_gpu():
    from bndm_amd import _lib, tokens
    x = torch.zeros(2, 4, 2, 16, dtype=torch.float16)
    with pytest.raises(_lib.BndmError):
        tokens.linear(x, x[0, 0])
    with pytest.raises(_lib.BndmError):
        tokens.rotary(x, None, torch.zeros(4, 1, dtype=torch.int32), (8,))
    with pytest.raises(_lib.BndmError):
        tokens.differential_attention(x, x, x[:, :, :1], torch.zeros(1))


def refused(lib, rc, word):
    assert rc == -1
    assert word in lib.bndm_tokens_last_error().decode(), lib.bndm_tokens_last_error()


def test_linear_refusals(lib):
    need = lib.bndm_tokens_linear_workspace_bytes(128, 128, 65536)
    assert need > 0 and lib.bndm_tokens_linear_workspace_bytes(4, 8, 16) == 0          # one tile, a long sum: split
    big = dict(x=P, ldx=65536, w=P, b=0, r=0, ldr=0, y=P, z=0, M=128, N=128, K=65536, act=0, dtype=0)
    for work, size in ((P, need - 1), (0, need), (P + 8, need)):
        refused(lib, lib.bndm_tokens_linear(*big.values(), work, size, None), "workspace")
    good = dict(x=P, ldx=16, w=P, b=0, r=0, ldr=0, y=P, z=0, M=4, N=8, K=16, act=0, dtype=0, work=0, size=0)
    for change, word in [(dict(M=-1), "negative"), (dict(act=3), "activation"), (dict(dtype=2), "dtype"), (dict(N=1 << 24), "2^22"),
                         (dict(x=0), "NULL"), (dict(w=0), "NULL"), (dict(y=0), "NULL"), (dict(ldx=-1), "stride"), (dict(r=P, ldr=-1), "stride")]:
        refused(lib, lib.bndm_tokens_linear(*{**good, **change}.values(), None), word)
    assert lib.bndm_tokens_linear(*{**good, "M": 0}.values(), None) == 0
    need = lib.bndm_tokens_linear_backward_workspace_bytes(100, 8, 16, 1, 1)
    assert need >= 100 * 8 * 2 + 8 * 4
    good = dict(dy=P, lddy=8, z=P, x=P, ldx=16, w=P, dx=P, dw=P, db=P, M=100, N=8, K=16, act=1, dtype=1, work=P, size=need)
    for change, word in [(dict(M=0), "empty"), (dict(z=0), "NULL"), (dict(dy=0), "NULL"), (dict(x=0), "NULL"), (dict(w=0), "NULL"),
                         (dict(size=need - 1), "workspace"), (dict(work=0), "workspace"), (dict(lddy=-8), "stride"), (dict(act=9), "activation")]:
        refused(lib, lib.bndm_tokens_linear_backward(*{**good, **change}.values(), None), word)


def test_rotary_refusals(lib):
    S = C.c_int64 * 3
    two = lambda *v: (C.c_int * len(v))(*v)
    good = dict(q=P, qs=S(0, 0, 0), qo=P, hq=2, k=0, ks=None, ko=0, hk=0, pos=P, ps=S(0, 0, 0), pt=0, B=1, N=1, D=16, sections=two(4, 4), axes=2,
                base=10000.0, il=0, inv=0, dtype=0)
    for change, word in [(dict(B=-1), "negative"), (dict(D=15), "head size"), (dict(D=258), "head size"), (dict(D=0), "head size"), (dict(dtype=3), "dtype"),
                         (dict(pt=3), "position type"), (dict(sections=None), "axes"), (dict(axes=0), "axes"), (dict(axes=5), "axes"),
                         (dict(base=0.0), "base"), (dict(base=float("nan")), "base"), (dict(sections=two(4, 5)), "add up"), (dict(sections=two(4, 3)), "add up"),
                         (dict(sections=two(-4, 12)), "add up"), (dict(q=0), "NULL"), (dict(qo=0), "NULL"), (dict(qs=None), "NULL"), (dict(pos=0), "NULL"),
                         (dict(hk=1), "NULL"), (dict(B=1 << 20, N=1 << 20), "more tokens")]:
        refused(lib, lib.bndm_tokens_rotary(*{**good, **change}.values(), None), word)
    assert lib.bndm_tokens_rotary(*{**good, "N": 0}.values(), None) == 0


def test_attention_refusals(lib):
    from bndm_amd._lib import AttentionShape
    S = C.c_int64 * 3

    def shape(**change):
        v = dict(B=2, Nq=1, Nk=4096, H=4, Hk=2, D=64, Dv=128, q=S(512, 512, 64), k=S(1024, 256, 64), v=S(1024, 256, 128), causal=0, dtype=0, lam_f32=0,
                 scale=0.125)
        v.update(change)
        flat = [x for key in v for x in (v[key] if key in "qkv" else [v[key]])]
        return AttentionShape(*flat)

    need = lib.bndm_tokens_attention_workspace_bytes(shape())
    assert need > 0                                          # few queries, many keys: split
    good = dict(q=P, k=P, v=P, lam=P, start=0, lengths=0, o=P, o2=0, lse=0, work=P, size=need)
    bad = [(dict(Nk=-1), "sizes"), (dict(H=3), "heads"), (dict(Hk=0), "heads"), (dict(D=60), "head size"), (dict(D=136), "head size"), (dict(Dv=4), "value size"),
           (dict(Dv=264), "value size"), (dict(dtype=2), "dtype"), (dict(scale=0.0), "scale"), (dict(scale=float("inf")), "scale"),
           (dict(scale=float("nan")), "scale"), (dict(q=S(512, 512, 60)), "stride"), (dict(k=S(-8, 256, 64)), "stride"), (dict(v=S(0, 1 << 24, 128)), "stride"),
           (dict(B=1 << 20, Nq=1 << 20), "tiles")]
    for change, word in bad:
        refused(lib, lib.bndm_tokens_attention(shape(**change), *good.values(), None), word)
        assert lib.bndm_tokens_attention_workspace_bytes(shape(**change)) == 0
    for change, word in [(dict(q=0), "NULL"), (dict(k=0), "NULL"), (dict(lam=0), "NULL"), (dict(o=0), "NULL"), (dict(q=P + 2), "16 bytes"), (dict(v=P + 8), "16 bytes"),
                         (dict(o2=P), "together"), (dict(lse=P), "together"), (dict(size=need - 1), "workspace"), (dict(work=0), "workspace")]:
        refused(lib, lib.bndm_tokens_attention(shape(), *{**good, **change}.values(), None), word)
    assert lib.bndm_tokens_attention(shape(B=0), *good.values(), None) == 0
    need = lib.bndm_tokens_attention_backward_workspace_bytes(shape())
    good = dict(q=P, k=P, v=P, lam=P, start=0, lengths=0, o=P, o2=P, lse=P, dout=P, ds=S(512, 512, 128), dq=P, dk=P, dv=P, dlam=P, work=P, size=need)
    for change, word in bad:
        refused(lib, lib.bndm_tokens_attention_backward(shape(**change), *good.values(), None), word)
    for change, word in [(dict(o2=0), "NULL"), (dict(lse=0), "NULL"), (dict(dout=0), "NULL"), (dict(dk=0), "NULL"), (dict(dlam=0), "NULL"), (dict(dq=P + 4), "16 bytes"),
                         (dict(ds=S(512, 512, 4)), "stride"), (dict(size=need - 1), "workspace")]:
        refused(lib, lib.bndm_tokens_attention_backward(shape(), *{**good, **change}.values(), None), word)
    refused(lib, lib.bndm_tokens_attention_backward(shape(Nq=0), *good.values(), None), "no queries")


READELF = "/opt/rocm/llvm/bin/llvm-readelf"


@pytest.mark.skipif(not os.path.exists(READELF), reason="needs the ROCm LLVM tools")
def test_no_kernel_spills(lib, tmp_path):
    """Every kernel keeps what it works on in registers: one that does not is many times slower, and nothing else would tell."""
    from bndm_amd import _lib
    data, magic = open(_lib.TOKENS_LIB_PATH, "rb").read(), b"__CLANG_OFFLOAD_BUNDLE__"
    kernels, at = 0, data.find(magic)
    while at >= 0:
        pos = at + len(magic)
        count, = struct.unpack_from("<Q", data, pos)
        pos += 8
        for _ in range(count):
            offset, size, length = struct.unpack_from("<QQQ", data, pos)
            name = data[pos + 24 : pos + 24 + length].decode()
            pos += 24 + length
            if not name.startswith("host"):
                assert name.endswith("gfx950"), name
                code = tmp_path / "code.o"
                code.write_bytes(data[at + offset : at + offset + size])
                notes = subprocess.run([READELF, "--notes", str(code)], capture_output=True, text=True, check=True).stdout
                fields = re.findall(r"\.(name|vgpr_spill_count|symbol):\s+(\S+)", notes)
                spills = [int(v) for k, v in fields if k == "vgpr_spill_count"]
                symbols = [v for k, v in fields if k == "symbol"]
                assert len(spills) == len(symbols)
                assert [s for s, n in zip(symbols, spills) if n] == []
                kernels += len(symbols)
        at = data.find(magic, pos)
    assert kernels > 50
