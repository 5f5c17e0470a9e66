"""TEST INFRASTRUCTURE: instruction semantics of the gfx950 simulator -- one builder per mnemonic turns a parsed instruction
(loader.Inst) into a closure run(wave).  Only what hipcc emits for this repository's kernels (plus the few extra opcodes the
parked candidates use) is implemented; an unknown mnemonic raises, it is never skipped.

Sources for the semantics: the CDNA3 / GCN3 ISA as the author knows it, the fragment layouts in
/opt/skills/guides/cdna_hip_programming.md section 3, and CALIBRATION: kernels whose results on real MI355X hardware are on
record (profiles/r03_gpu_tests.log: every family but conv_t32's round-4 build) must reproduce oracle/ here too -- see
tests/test_gfx950sim.py.  Transcendentals (v_exp / v_rcp / v_rsq / v_sqrt / v_log) are computed exactly and rounded once;
hardware is within 1 ulp of that."""
import re

import numpy as np

from .core import (BARRIER, ENDPGM, EXEC, F16, F32, F64, I16, I32, I64, LANE, M0, M32, M64, U8, U16, U32, U64, VCC, Opnd,
                   Pending, SimError, bool_to_mask, const_bits, full, full64, mask_to_bool, parse_reg, sx)

BUILDERS = {}


def op(*names):
    def deco(f):
        for n in names:
            BUILDERS[n] = f
        return f
    return deco


def strip_suffix(m):
    for suf in ("_e64_dpp", "_e32", "_e64", "_sdwa", "_dpp"):
        if m.endswith(suf):
            return m[:-len(suf)], suf[1:]
    return m, ""


def mod_val(ins, key, default=None):
    for m in ins.mods:
        if m.startswith(key + ":"):
            v = m[len(key) + 1:]
            if v.startswith("["):
                return [int(x, 0) for x in v[1:-1].split(",")]
            return int(v, 0)
    return default


def has_mod(ins, key):
    return key in ins.mods


# ---------------------------------------------------------------------------------------------------------------------
# source accessors
# ---------------------------------------------------------------------------------------------------------------------
def _signbits(kind):
    return {"f32": (0x80000000, 0x7FFFFFFF), "f16": (0x8000, 0xFFFF7FFF), "i32": (0x80000000, 0x7FFFFFFF)}.get(kind, (0x80000000, 0x7FFFFFFF))


def vsrc(o, kind="i32"):
    """-> f(w) -> uint32[64] (treat as read-only)"""
    if not isinstance(o, Opnd):
        o = Opnd(o)
    if o.reg:
        f, i, n = o.reg
        if f == "v":
            def g(w, i=i):
                if w.npend and w.vpend[i]:
                    w.hazard(f"read of v{i} while a load into it is in flight")
                return w.v[i]
        else:
            def g(w, i=i):
                if w.npend and w.spend[i]:
                    w.hazard(f"read of s{i} while a load into it is in flight")
                return full(w.s[i])
    elif o.const == "scc":
        def g(w):
            return full(w.scc)
    else:
        arr = full(const_bits(o.const, kind))
        arr.setflags(write=False)

        def g(w, arr=arr):
            return arr
    if o.abs or o.neg:
        sb, am = _signbits(kind)
        g0, ab, ng = g, o.abs, o.neg

        def g(w):
            a = g0(w)
            if ab:
                a = a & U32(am)
            if ng:
                a = a ^ U32(sb)
            return a
    return g


def vsrc64(o, kind="u64"):
    """-> f(w) -> uint64[64]"""
    if not isinstance(o, Opnd):
        o = Opnd(o)
    if o.reg:
        f, i, n = o.reg
        if f == "v":
            assert n >= 2, o.text

            def g(w, i=i):
                if w.npend and (w.vpend[i] or w.vpend[i + 1]):
                    w.hazard(f"read of v[{i}:{i + 1}] while a load into it is in flight")
                return w.v[i].astype(U64) | (w.v[i + 1].astype(U64) << U64(32))
        else:
            if n == 1:        # a 32-bit SGPR used as a 64-bit operand: zero-extended (sign for i64 does not occur)
                def g(w, i=i):
                    return full64(w.s[i])
            else:
                def g(w, i=i):
                    if w.npend and (w.spend[i] or w.spend[i + 1]):
                        w.hazard(f"read of s[{i}:{i + 1}] while a load into it is in flight")
                    return full64(w.s[i] | (w.s[i + 1] << 32))
    else:
        arr = full64(const_bits(o.const, kind))
        arr.setflags(write=False)

        def g(w, arr=arr):
            return arr
    if o.abs or o.neg:
        g0, ab, ng = g, o.abs, o.neg

        def g(w):
            a = g0(w)
            if ab:
                a = a & U64(0x7FFFFFFFFFFFFFFF)
            if ng:
                a = a ^ U64(0x8000000000000000)
            return a
    return g


def ssrc(o, kind="i32"):
    """-> f(w) -> python int (32 bit)"""
    if not isinstance(o, Opnd):
        o = Opnd(o)
    if o.reg:
        f, i, n = o.reg
        assert f == "s", o.text

        def g(w, i=i):
            if w.npend and w.spend[i]:
                w.hazard(f"read of s{i} while a load into it is in flight")
            return w.s[i]
        return g
    if o.const == "scc":
        return lambda w: w.scc
    c = const_bits(o.const, kind)
    return lambda w: c


def ssrc64(o, kind="i64"):
    if not isinstance(o, Opnd):
        o = Opnd(o)
    if o.reg:
        f, i, n = o.reg
        assert f == "s", o.text
        if n == 1:
            return lambda w, i=i: w.s[i]

        def g(w, i=i):
            if w.npend and (w.spend[i] or w.spend[i + 1]):
                w.hazard(f"read of s[{i}:{i + 1}] while a load into it is in flight")
            return w.s[i] | (w.s[i + 1] << 32)
        return g
    c = const_bits(o.const, kind)
    return lambda w: c


def dreg(tok):
    r = parse_reg(tok)
    if r is None:
        raise SimError(f"destination {tok!r}")
    return r


def f32(a):
    return a.view(F32)


def bits(x):
    return np.ascontiguousarray(x, F32).view(U32)


def fma32(a, b, c):
    return (a.astype(F64) * b.astype(F64) + c.astype(F64)).astype(F32)


def i32(a):
    return a.view(I32)


# ---------------------------------------------------------------------------------------------------------------------
# SALU
# ---------------------------------------------------------------------------------------------------------------------
def _sop2(fn, scc=None, wide=False):
    """fn(a, b) -> result; scc(res, a, b) -> 0/1 or None"""
    def build(ins):
        d = dreg(ins.ops[0])
        if wide:
            a, b = ssrc64(ins.ops[1]), ssrc64(ins.ops[2])
        else:
            a, b = ssrc(ins.ops[1]), ssrc(ins.ops[2])
        di = d[1]
        if wide:
            def run(w):
                x, y = a(w), b(w)
                r = fn(x, y) & M64
                if scc:
                    w.scc = scc(r, x, y)
                w.ws64(di, r)
        else:
            def run(w):
                x, y = a(w), b(w)
                r = fn(x, y)
                if scc:
                    w.scc = scc(r, x, y)
                w.ws(di, r)
        return run
    return build


def _nz(r, a, b):
    return int((r & M64) != 0)


def _nz32(r, a, b):
    return int((r & M32) != 0)


BUILDERS["s_add_u32"] = _sop2(lambda a, b: a + b, lambda r, a, b: int(r > M32))
BUILDERS["s_sub_u32"] = _sop2(lambda a, b: a - b, lambda r, a, b: int(b > a))
BUILDERS["s_add_i32"] = _sop2(lambda a, b: a + b, lambda r, a, b: int(not (-(1 << 31) <= sx(a, 32) + sx(b, 32) < (1 << 31))))
BUILDERS["s_sub_i32"] = _sop2(lambda a, b: a - b, lambda r, a, b: int(not (-(1 << 31) <= sx(a, 32) - sx(b, 32) < (1 << 31))))
BUILDERS["s_mul_i32"] = _sop2(lambda a, b: (sx(a, 32) * sx(b, 32)))
BUILDERS["s_mul_hi_u32"] = _sop2(lambda a, b: (a * b) >> 32)
BUILDERS["s_mul_hi_i32"] = _sop2(lambda a, b: (sx(a, 32) * sx(b, 32)) >> 32)
BUILDERS["s_and_b32"] = _sop2(lambda a, b: a & b, _nz32)
BUILDERS["s_or_b32"] = _sop2(lambda a, b: a | b, _nz32)
BUILDERS["s_xor_b32"] = _sop2(lambda a, b: a ^ b, _nz32)
BUILDERS["s_andn2_b32"] = _sop2(lambda a, b: a & ~b, _nz32)
BUILDERS["s_orn2_b32"] = _sop2(lambda a, b: a | (~b & M32), _nz32)
BUILDERS["s_nand_b32"] = _sop2(lambda a, b: ~(a & b), _nz32)
BUILDERS["s_nor_b32"] = _sop2(lambda a, b: ~(a | b), _nz32)
BUILDERS["s_xnor_b32"] = _sop2(lambda a, b: ~(a ^ b), _nz32)
BUILDERS["s_and_b64"] = _sop2(lambda a, b: a & b, _nz, True)
BUILDERS["s_or_b64"] = _sop2(lambda a, b: a | b, _nz, True)
BUILDERS["s_xor_b64"] = _sop2(lambda a, b: a ^ b, _nz, True)
BUILDERS["s_andn2_b64"] = _sop2(lambda a, b: a & ~b, _nz, True)
BUILDERS["s_orn2_b64"] = _sop2(lambda a, b: a | (~b & M64), _nz, True)
BUILDERS["s_nand_b64"] = _sop2(lambda a, b: ~(a & b), _nz, True)
BUILDERS["s_nor_b64"] = _sop2(lambda a, b: ~(a | b), _nz, True)
BUILDERS["s_xnor_b64"] = _sop2(lambda a, b: ~(a ^ b), _nz, True)
BUILDERS["s_lshl_b32"] = _sop2(lambda a, b: a << (b & 31), _nz32)
BUILDERS["s_lshr_b32"] = _sop2(lambda a, b: a >> (b & 31), _nz32)
BUILDERS["s_ashr_i32"] = _sop2(lambda a, b: sx(a, 32) >> (b & 31), _nz32)
BUILDERS["s_min_i32"] = _sop2(lambda a, b: a if sx(a, 32) <= sx(b, 32) else b, lambda r, a, b: int(sx(a, 32) < sx(b, 32)))
BUILDERS["s_max_i32"] = _sop2(lambda a, b: a if sx(a, 32) >= sx(b, 32) else b, lambda r, a, b: int(sx(a, 32) > sx(b, 32)))
BUILDERS["s_min_u32"] = _sop2(lambda a, b: min(a, b), lambda r, a, b: int(a < b))
BUILDERS["s_max_u32"] = _sop2(lambda a, b: max(a, b), lambda r, a, b: int(a > b))
BUILDERS["s_bfm_b32"] = _sop2(lambda a, b: ((1 << (a & 31)) - 1) << (b & 31))
BUILDERS["s_lshl1_add_u32"] = _sop2(lambda a, b: (a << 1) + b, lambda r, a, b: int(r > M32))
BUILDERS["s_lshl2_add_u32"] = _sop2(lambda a, b: (a << 2) + b, lambda r, a, b: int(r > M32))
BUILDERS["s_lshl3_add_u32"] = _sop2(lambda a, b: (a << 3) + b, lambda r, a, b: int(r > M32))
BUILDERS["s_lshl4_add_u32"] = _sop2(lambda a, b: (a << 4) + b, lambda r, a, b: int(r > M32))
BUILDERS["s_pack_ll_b32_b16"] = _sop2(lambda a, b: (a & 0xFFFF) | ((b & 0xFFFF) << 16))


def _bfe_u32(a, b):
    off, wid = b & 31, (b >> 16) & 0x7F
    return (a >> off) & ((1 << wid) - 1) if wid else 0


def _bfe_i32(a, b):
    off, wid = b & 31, (b >> 16) & 0x7F
    if wid == 0:
        return 0
    return sx((a >> off) & ((1 << wid) - 1), min(wid, 32)) if wid < 32 else sx(a >> off, 32 - off)


BUILDERS["s_bfe_u32"] = _sop2(_bfe_u32, _nz32)
BUILDERS["s_bfe_i32"] = _sop2(_bfe_i32, _nz32)


@op("s_addc_u32")
def _(ins):
    d, a, b = dreg(ins.ops[0])[1], ssrc(ins.ops[1]), ssrc(ins.ops[2])

    def run(w):
        r = a(w) + b(w) + w.scc
        w.scc = int(r > M32)
        w.ws(d, r)
    return run


@op("s_subb_u32")
def _(ins):
    d, a, b = dreg(ins.ops[0])[1], ssrc(ins.ops[1]), ssrc(ins.ops[2])

    def run(w):
        x, y = a(w), b(w) + w.scc
        w.scc = int(y > x)
        w.ws(d, x - y)
    return run


@op("s_lshl_b64", "s_lshr_b64", "s_ashr_i64")
def _(ins):
    d, a, b = dreg(ins.ops[0])[1], ssrc64(ins.ops[1]), ssrc(ins.ops[2])
    kind = ins.base

    def run(w):
        x, n = a(w), b(w) & 63
        r = (x << n) if kind == "s_lshl_b64" else (x >> n) if kind == "s_lshr_b64" else (sx(x, 64) >> n)
        r &= M64
        w.scc = int(r != 0)
        w.ws64(d, r)
    return run


@op("s_cselect_b32")
def _(ins):
    d, a, b = dreg(ins.ops[0])[1], ssrc(ins.ops[1]), ssrc(ins.ops[2])
    return lambda w: w.ws(d, a(w) if w.scc else b(w))


@op("s_cselect_b64")
def _(ins):
    d, a, b = dreg(ins.ops[0])[1], ssrc64(ins.ops[1]), ssrc64(ins.ops[2])
    return lambda w: w.ws64(d, a(w) if w.scc else b(w))


@op("s_mov_b32")
def _(ins):
    d, a = dreg(ins.ops[0])[1], ssrc(ins.ops[1])
    return lambda w: w.ws(d, a(w))


@op("s_mov_b64")
def _(ins):
    d, a = dreg(ins.ops[0])[1], ssrc64(ins.ops[1])
    return lambda w: w.ws64(d, a(w))


@op("s_movk_i32")
def _(ins):
    d, k = dreg(ins.ops[0])[1], sx(int(ins.ops[1], 0), 16)
    return lambda w: w.ws(d, k)


@op("s_addk_i32")
def _(ins):
    d, k = dreg(ins.ops[0])[1], sx(int(ins.ops[1], 0), 16)

    def run(w):
        a = sx(w.s[d], 32)
        r = a + k
        w.scc = int(not (-(1 << 31) <= r < (1 << 31)))
        w.ws(d, r)
    return run


@op("s_mulk_i32")
def _(ins):
    d, k = dreg(ins.ops[0])[1], sx(int(ins.ops[1], 0), 16)
    return lambda w: w.ws(d, sx(w.s[d], 32) * k)


def _sop1(fn, scc=None):
    def build(ins):
        d, a = dreg(ins.ops[0])[1], ssrc(ins.ops[1])

        def run(w):
            x = a(w)
            r = fn(x) & M32
            if scc:
                w.scc = scc(r)
            w.ws(d, r)
        return run
    return build


BUILDERS["s_not_b32"] = _sop1(lambda a: ~a, lambda r: int(r != 0))
BUILDERS["s_brev_b32"] = _sop1(lambda a: int(f"{a:032b}"[::-1], 2))
BUILDERS["s_abs_i32"] = _sop1(lambda a: abs(sx(a, 32)), lambda r: int(r != 0))
BUILDERS["s_sext_i32_i8"] = _sop1(lambda a: sx(a, 8))
BUILDERS["s_sext_i32_i16"] = _sop1(lambda a: sx(a, 16))
BUILDERS["s_bcnt1_i32_b32"] = _sop1(lambda a: bin(a).count("1"), lambda r: int(r != 0))
BUILDERS["s_ff1_i32_b32"] = _sop1(lambda a: (a & -a).bit_length() - 1 if a else -1)
BUILDERS["s_flbit_i32_b32"] = _sop1(lambda a: 32 - a.bit_length() if a else -1)


@op("s_not_b64")
def _(ins):
    d, a = dreg(ins.ops[0])[1], ssrc64(ins.ops[1])

    def run(w):
        r = ~a(w) & M64
        w.scc = int(r != 0)
        w.ws64(d, r)
    return run


@op("s_bcnt1_i32_b64")
def _(ins):
    d, a = dreg(ins.ops[0])[1], ssrc64(ins.ops[1])

    def run(w):
        r = bin(a(w)).count("1")
        w.scc = int(r != 0)
        w.ws(d, r)
    return run


@op("s_ff1_i32_b64")
def _(ins):
    d, a = dreg(ins.ops[0])[1], ssrc64(ins.ops[1])

    def run(w):
        x = a(w)
        w.ws(d, (x & -x).bit_length() - 1 if x else -1)
    return run


@op("s_and_saveexec_b64", "s_or_saveexec_b64", "s_andn2_saveexec_b64", "s_xor_saveexec_b64", "s_andn1_saveexec_b64",
    "s_orn2_saveexec_b64")
def _(ins):
    d, a = dreg(ins.ops[0])[1], ssrc64(ins.ops[1])
    kind = ins.base

    def run(w):
        x, e = a(w), w.get_exec()
        if kind == "s_and_saveexec_b64":
            n = x & e
        elif kind == "s_or_saveexec_b64":
            n = x | e
        elif kind == "s_andn2_saveexec_b64":
            n = x & ~e
        elif kind == "s_andn1_saveexec_b64":
            n = ~x & e
        elif kind == "s_orn2_saveexec_b64":
            n = x | (~e & M64)
        else:
            n = x ^ e
        n &= M64
        w.ws64(d, e)
        w.set_exec(n)
        w.scc = int(n != 0)
    return run


_CMPS = {"eq": lambda a, b: a == b, "lg": lambda a, b: a != b, "ne": lambda a, b: a != b, "gt": lambda a, b: a > b,
         "ge": lambda a, b: a >= b, "lt": lambda a, b: a < b, "le": lambda a, b: a <= b}


def _scmp(ins):
    m = re.match(r"s_cmpk?_(\w+)_([iu])(32|64)$", ins.base)
    c, sg, wd = _CMPS[m.group(1)], m.group(2) == "i", int(m.group(3))
    isk = ins.base.startswith("s_cmpk")
    if wd == 64:
        a, b = ssrc64(ins.ops[0]), ssrc64(ins.ops[1])
    else:
        a = ssrc(ins.ops[0])
        if isk:
            kv = int(ins.ops[1], 0)
            kv = sx(kv, 16) & M32 if sg else kv & 0xFFFF
            b = lambda w: kv
        else:
            b = ssrc(ins.ops[1])

    def run(w):
        x, y = a(w), b(w)
        if sg:
            x, y = sx(x, wd), sx(y, wd)
        w.scc = int(c(x, y))
    return run


for _c in ("eq", "lg", "gt", "ge", "lt", "le"):
    for _t in ("i32", "u32"):
        BUILDERS[f"s_cmp_{_c}_{_t}"] = _scmp
        BUILDERS[f"s_cmpk_{_c}_{_t}"] = _scmp
BUILDERS["s_cmp_eq_u64"] = _scmp
BUILDERS["s_cmp_lg_u64"] = _scmp


@op("s_bitcmp0_b32", "s_bitcmp1_b32")
def _(ins):
    a, b = ssrc(ins.ops[0]), ssrc(ins.ops[1])
    one = ins.base.endswith("1_b32")

    def run(w):
        bit = (a(w) >> (b(w) & 31)) & 1
        w.scc = int(bit == (1 if one else 0))
    return run


def _target(ins):
    off = sx(int(ins.ops[0], 0), 16)
    return ins.addr + 4 + 4 * off


@op("s_branch")
def _(ins):
    t = _target(ins)

    def run(w):
        return w.kernel.index[t]
    return run


def _cbr(cond):
    def build(ins):
        t = _target(ins)

        def run(w):
            if cond(w):
                return w.kernel.index[t]
        return run
    return build


BUILDERS["s_cbranch_scc0"] = _cbr(lambda w: not w.scc)
BUILDERS["s_cbranch_scc1"] = _cbr(lambda w: w.scc)
BUILDERS["s_cbranch_vccz"] = _cbr(lambda w: (w.s[VCC] | w.s[VCC + 1]) == 0)
BUILDERS["s_cbranch_vccnz"] = _cbr(lambda w: (w.s[VCC] | w.s[VCC + 1]) != 0)
BUILDERS["s_cbranch_execz"] = _cbr(lambda w: (w.s[EXEC] | w.s[EXEC + 1]) == 0)
BUILDERS["s_cbranch_execnz"] = _cbr(lambda w: (w.s[EXEC] | w.s[EXEC + 1]) != 0)


@op("s_nop", "s_setprio", "s_sleep", "s_sethalt", "s_setkill", "s_inst_prefetch", "s_clause", "s_code_end", "s_icache_inv",
    "s_dcache_inv", "buffer_wbl2", "buffer_inv", "s_ttracedata", "s_incperflevel", "s_decperflevel")
def _(ins):
    return lambda w: None


@op("s_endpgm")
def _(ins):
    return lambda w: ENDPGM


@op("s_barrier")
def _(ins):
    def run(w):
        w.pc += 1
        return BARRIER
    return run


@op("s_waitcnt")
def _(ins):
    vm = lg = None
    for m in ins.mods:
        mm = re.match(r"(vmcnt|lgkmcnt|expcnt)\((\d+)\)", m)
        if not mm:
            raise SimError(f"s_waitcnt operand {m!r}")
        if mm.group(1) == "vmcnt":
            vm = int(mm.group(2))
        elif mm.group(1) == "lgkmcnt":
            lg = int(mm.group(2))

    def run(w):
        if vm is not None:
            w.wait_vm(vm)
        if lg is not None:
            w.wait_lgkm(lg)
    return run


@op("s_memtime", "s_memrealtime")
def _(ins):
    d = dreg(ins.ops[0])[1]

    def run(w):
        w.clock += 40 + w.ninst
        t = w.clock

        def apply():
            w.s[d], w.s[d + 1] = t & M32, (t >> 32) & M32
        w.push_lgkm(Pending(apply, sregs=(d, d + 1), what="s_memtime"))
    return run


@op("s_load_dword", "s_load_dwordx2", "s_load_dwordx4", "s_load_dwordx8", "s_load_dwordx16")
def _(ins):
    n = {"s_load_dword": 1, "s_load_dwordx2": 2, "s_load_dwordx4": 4, "s_load_dwordx8": 8, "s_load_dwordx16": 16}[ins.base]
    d = dreg(ins.ops[0])[1]
    base = ssrc64(ins.ops[1])
    o = Opnd(ins.ops[2])
    off = ssrc(o) if o.is_reg() else (lambda w, c=int(ins.ops[2], 0): c)
    imm = mod_val(ins, "offset", 0)

    def run(w):
        addr = (base(w) + off(w) + imm) & ~3
        raw = w.mem.host_read(addr, 4 * n)
        vals = np.frombuffer(raw, U32).tolist()

        def apply():
            w.s[d:d + n] = vals
            if d + n > EXEC:
                w.sync_exec()
        w.push_lgkm(Pending(apply, sregs=tuple(range(d, d + n)), what=ins.text))
    return run


# ---------------------------------------------------------------------------------------------------------------------
# VALU: table-driven 32-bit operations
# ---------------------------------------------------------------------------------------------------------------------
def _sh(a):
    return a & U32(31)


def _u24(a):
    return a & U32(0xFFFFFF)


def _i24(a):
    return ((a & U32(0xFFFFFF)).astype(I32) << 8) >> 8


def _bfe_u(a, off, wid):
    off, wid = off & U32(31), wid & U32(31)
    m = ((U64(1) << wid.astype(U64)) - U64(1)).astype(U32)
    return (a >> off) & m


def _bfe_i(a, off, wid):
    off, wid = off & U32(31), wid & U32(31)
    r = _bfe_u(a, off, wid)
    sh = (U32(32) - wid) & U32(31)
    out = ((r << sh).view(I32) >> sh.view(I32)).view(U32)
    return np.where(wid == 0, U32(0), out)


def _perm(s0, s1, sel):
    """v_perm_b32: byte select from {s0, s1} (s1 = bytes 0-3, s0 = bytes 4-7)"""
    src = (s0.astype(U64) << U64(32)) | s1.astype(U64)
    out = np.zeros(64, U32)
    for k in range(4):
        sb = (sel >> U32(8 * k)) & U32(0xFF)
        byte = ((src >> (np.minimum(sb, 7).astype(U64) * U64(8))) & U64(0xFF)).astype(U32)
        sign = lambda idx: np.where(((src >> U64(8 * idx + 7)) & U64(1)) == 1, U32(0xFF), U32(0))
        byte = np.where(sb == 8, sign(1), byte)
        byte = np.where(sb == 9, sign(3), byte)
        byte = np.where(sb == 10, sign(5), byte)
        byte = np.where(sb == 11, sign(7), byte)
        byte = np.where(sb == 12, U32(0), byte)
        byte = np.where(sb >= 13, U32(0xFF), byte)
        out |= byte << U32(8 * k)
    return out


def _ffbh(a):
    """leading zeros of a 32-bit value (-1 for 0): frexp of the exact float64 gives the bit length"""
    _, e = np.frexp(a.astype(F64))
    return np.where(a != 0, (32 - e).astype(np.int64), -1).astype(np.int64).astype(U32)


def _popc(a):
    return np.unpackbits(np.ascontiguousarray(a).view(U8).reshape(64, 4), axis=1).sum(1).astype(U32)


def _brev(a):
    b = np.unpackbits(a.view(U8).reshape(64, 4), axis=1, bitorder="little")     # [64, 32] LSB first
    return np.packbits(b[:, ::-1], axis=1, bitorder="little").view(U32).reshape(64)


def _alignbit(s0, s1, s2):
    v = (s0.astype(U64) << U64(32)) | s1.astype(U64)
    return ((v >> (s2 & U32(31)).astype(U64)) & U64(M32)).astype(U32)


def _alignbyte(s0, s1, s2):
    v = (s0.astype(U64) << U64(32)) | s1.astype(U64)
    return ((v >> ((s2 & U32(3)).astype(U64) * U64(8))) & U64(M32)).astype(U32)


def _cvt_u32_f32(a):
    x = f32(a).astype(F64)
    x = np.where(np.isnan(x), 0.0, x)
    return np.clip(np.trunc(x), 0, 4294967295.0).astype(U64).astype(U32)


def _cvt_i32_f32(a):
    x = f32(a).astype(F64)
    x = np.where(np.isnan(x), 0.0, x)
    return np.clip(np.trunc(x), -2147483648.0, 2147483647.0).astype(I64).astype(I32).view(U32)


def _bf16_rne(x32):
    u = np.ascontiguousarray(x32, F32).view(U32)
    r = ((u.astype(U64) + U64(0x7FFF) + ((u >> U32(16)) & U32(1)).astype(U64)) >> U64(16)).astype(U32) & U32(0xFFFF)
    nan = np.isnan(x32)
    return np.where(nan, (u >> U32(16)) | U32(0x40), r).astype(U32) & U32(0xFFFF)


def _f16lo(a):
    return (a & U32(0xFFFF)).astype(U16).view(F16)


def _f16hi(a):
    return (a >> U32(16)).astype(U16).view(F16)


def _pk16(lo, hi):
    return lo.view(U16).astype(U32) | (hi.view(U16).astype(U32) << U32(16))


def _class_f32(a, m):
    x = f32(a)
    u = a
    exp = (u >> U32(23)) & U32(0xFF)
    man = u & U32(0x7FFFFF)
    neg = (u >> U32(31)) == 1
    isnan = (exp == 255) & (man != 0)
    snan = isnan & ((man >> U32(22)) == 0)
    qnan = isnan & ~snan
    inf = (exp == 255) & (man == 0)
    den = (exp == 0) & (man != 0)
    zero = (exp == 0) & (man == 0)
    nor = ~isnan & ~inf & ~den & ~zero
    cls = (snan * 1 | qnan * 2 | (inf & neg) * 4 | (nor & neg) * 8 | (den & neg) * 16 | (zero & neg) * 32 | (zero & ~neg) * 64
           | (den & ~neg) * 128 | (nor & ~neg) * 256 | (inf & ~neg) * 512).astype(U32)
    return (cls & m) != 0


def _class_f64(a64, m):
    exp = (a64 >> U64(52)) & U64(0x7FF)
    man = a64 & U64((1 << 52) - 1)
    neg = (a64 >> U64(63)) == 1
    isnan = (exp == 0x7FF) & (man != 0)
    snan = isnan & ((man >> U64(51)) == 0)
    qnan = isnan & ~snan
    inf = (exp == 0x7FF) & (man == 0)
    den = (exp == 0) & (man != 0)
    zero = (exp == 0) & (man == 0)
    nor = ~isnan & ~inf & ~den & ~zero
    cls = (snan * 1 | qnan * 2 | (inf & neg) * 4 | (nor & neg) * 8 | (den & neg) * 16 | (zero & neg) * 32 | (zero & ~neg) * 64
           | (den & ~neg) * 128 | (nor & ~neg) * 256 | (inf & ~neg) * 512).astype(U32)
    return (cls & m) != 0


# name -> (number of sources, kind, fn).  kind 'u': uint32 arrays in, uint32 out; 'f': float32 views in, float32 out
VALU = {
    "v_mov_b32": (1, "u", lambda a: a),
    "v_not_b32": (1, "u", lambda a: ~a),
    "v_bfrev_b32": (1, "u", _brev),
    "v_ffbh_u32": (1, "u", _ffbh),
    "v_bcnt_u32_b32": (2, "u", lambda a, b: _popc(a) + b),
    "v_add_u32": (2, "u", lambda a, b: a + b),
    "v_sub_u32": (2, "u", lambda a, b: a - b),
    "v_subrev_u32": (2, "u", lambda a, b: b - a),
    "v_and_b32": (2, "u", lambda a, b: a & b),
    "v_or_b32": (2, "u", lambda a, b: a | b),
    "v_xor_b32": (2, "u", lambda a, b: a ^ b),
    "v_xnor_b32": (2, "u", lambda a, b: ~(a ^ b)),
    "v_lshlrev_b32": (2, "u", lambda a, b: b << _sh(a)),
    "v_lshrrev_b32": (2, "u", lambda a, b: b >> _sh(a)),
    "v_ashrrev_i32": (2, "u", lambda a, b: (i32(b) >> _sh(a).view(I32)).view(U32)),
    "v_mul_lo_u32": (2, "u", lambda a, b: a * b),
    "v_mul_hi_u32": (2, "u", lambda a, b: ((a.astype(U64) * b.astype(U64)) >> U64(32)).astype(U32)),
    "v_mul_hi_i32": (2, "u", lambda a, b: ((i32(a).astype(I64) * i32(b).astype(I64)) >> 32).astype(I32).view(U32)),
    "v_mul_u32_u24": (2, "u", lambda a, b: _u24(a) * _u24(b)),
    "v_mul_i32_i24": (2, "u", lambda a, b: (_i24(a) * _i24(b)).view(U32)),
    "v_mul_hi_u32_u24": (2, "u", lambda a, b: ((_u24(a).astype(U64) * _u24(b).astype(U64)) >> U64(32)).astype(U32)),
    "v_min_i32": (2, "u", lambda a, b: np.minimum(i32(a), i32(b)).view(U32)),
    "v_max_i32": (2, "u", lambda a, b: np.maximum(i32(a), i32(b)).view(U32)),
    "v_min_u32": (2, "u", lambda a, b: np.minimum(a, b)),
    "v_max_u32": (2, "u", lambda a, b: np.maximum(a, b)),
    "v_add3_u32": (3, "u", lambda a, b, c: a + b + c),
    "v_lshl_add_u32": (3, "u", lambda a, b, c: (a << _sh(b)) + c),
    "v_add_lshl_u32": (3, "u", lambda a, b, c: (a + b) << _sh(c)),
    "v_lshl_or_b32": (3, "u", lambda a, b, c: (a << _sh(b)) | c),
    "v_and_or_b32": (3, "u", lambda a, b, c: (a & b) | c),
    "v_or3_b32": (3, "u", lambda a, b, c: a | b | c),
    "v_xad_u32": (3, "u", lambda a, b, c: (a ^ b) + c),
    "v_bfe_u32": (3, "u", _bfe_u),
    "v_bfe_i32": (3, "u", _bfe_i),
    "v_bfi_b32": (3, "u", lambda a, b, c: (a & b) | (~a & c)),
    "v_alignbit_b32": (3, "u", _alignbit),
    "v_alignbyte_b32": (3, "u", _alignbyte),
    "v_perm_b32": (3, "u", _perm),
    "v_mad_u32_u24": (3, "u", lambda a, b, c: _u24(a) * _u24(b) + c),
    "v_mad_i32_i24": (3, "u", lambda a, b, c: (_i24(a) * _i24(b)).view(U32) + c),
    "v_min3_i32": (3, "u", lambda a, b, c: np.minimum(np.minimum(i32(a), i32(b)), i32(c)).view(U32)),
    "v_max3_i32": (3, "u", lambda a, b, c: np.maximum(np.maximum(i32(a), i32(b)), i32(c)).view(U32)),
    "v_min3_u32": (3, "u", lambda a, b, c: np.minimum(np.minimum(a, b), c)),
    "v_max3_u32": (3, "u", lambda a, b, c: np.maximum(np.maximum(a, b), c)),
    "v_med3_i32": (3, "u", lambda a, b, c: np.sort(np.stack([i32(a), i32(b), i32(c)]), axis=0)[1].view(U32)),
    # 16-bit integer (results zero-extended into the low half, VOP2 semantics on gfx9: high half zeroed)
    "v_add_u16": (2, "u", lambda a, b: (a + b) & U32(0xFFFF)),
    "v_sub_u16": (2, "u", lambda a, b: (a - b) & U32(0xFFFF)),
    "v_mul_lo_u16": (2, "u", lambda a, b: (a * b) & U32(0xFFFF)),
    "v_lshlrev_b16": (2, "u", lambda a, b: (b << (a & U32(15))) & U32(0xFFFF)),
    "v_lshrrev_b16": (2, "u", lambda a, b: ((b & U32(0xFFFF)) >> (a & U32(15)))),
    "v_max_u16": (2, "u", lambda a, b: np.maximum(a & U32(0xFFFF), b & U32(0xFFFF))),
    "v_min_u16": (2, "u", lambda a, b: np.minimum(a & U32(0xFFFF), b & U32(0xFFFF))),
    # float32
    "v_add_f32": (2, "f", lambda a, b: a + b),
    "v_sub_f32": (2, "f", lambda a, b: a - b),
    "v_subrev_f32": (2, "f", lambda a, b: b - a),
    "v_mul_f32": (2, "f", lambda a, b: a * b),
    "v_mul_legacy_f32": (2, "f", lambda a, b: np.where((a == 0) | (b == 0), F32(0), a * b)),
    "v_max_f32": (2, "f", lambda a, b: np.fmax(a, b)),
    "v_min_f32": (2, "f", lambda a, b: np.fmin(a, b)),
    "v_fma_f32": (3, "f", fma32),
    "v_mad_f32": (3, "f", lambda a, b, c: (a * b) + c),
    "v_max3_f32": (3, "f", lambda a, b, c: np.fmax(np.fmax(a, b), c)),
    "v_min3_f32": (3, "f", lambda a, b, c: np.fmin(np.fmin(a, b), c)),
    "v_med3_f32": (3, "f", lambda a, b, c: np.sort(np.stack([a, b, c]), axis=0)[1]),
    "v_rcp_f32": (1, "f", lambda a: (1.0 / a.astype(F64)).astype(F32)),
    "v_rcp_iflag_f32": (1, "f", lambda a: (1.0 / a.astype(F64)).astype(F32)),
    "v_rsq_f32": (1, "f", lambda a: (1.0 / np.sqrt(a.astype(F64))).astype(F32)),
    "v_sqrt_f32": (1, "f", lambda a: np.sqrt(a.astype(F64)).astype(F32)),
    "v_exp_f32": (1, "f", lambda a: np.exp2(a.astype(F64)).astype(F32)),
    "v_log_f32": (1, "f", lambda a: np.log2(a.astype(F64)).astype(F32)),
    "v_sin_f32": (1, "f", lambda a: np.sin(2 * np.pi * a.astype(F64)).astype(F32)),
    "v_cos_f32": (1, "f", lambda a: np.cos(2 * np.pi * a.astype(F64)).astype(F32)),
    "v_trunc_f32": (1, "f", np.trunc),
    "v_rndne_f32": (1, "f", np.rint),
    "v_floor_f32": (1, "f", np.floor),
    "v_ceil_f32": (1, "f", np.ceil),
    "v_fract_f32": (1, "f", lambda a: a - np.floor(a)),
    "v_cvt_u32_f32": (1, "u", _cvt_u32_f32),
    "v_cvt_i32_f32": (1, "u", _cvt_i32_f32),
    "v_cvt_f32_u32": (1, "u", lambda a: bits(a.astype(F32))),
    "v_cvt_f32_i32": (1, "u", lambda a: bits(i32(a).astype(F32))),
    "v_cvt_f32_ubyte0": (1, "u", lambda a: bits((a & U32(0xFF)).astype(F32))),
    "v_cvt_f32_ubyte1": (1, "u", lambda a: bits(((a >> U32(8)) & U32(0xFF)).astype(F32))),
    "v_cvt_f32_ubyte2": (1, "u", lambda a: bits(((a >> U32(16)) & U32(0xFF)).astype(F32))),
    "v_cvt_f32_ubyte3": (1, "u", lambda a: bits(((a >> U32(24)) & U32(0xFF)).astype(F32))),
    "v_cvt_f32_f16": (1, "u", lambda a: bits(_f16lo(a).astype(F32))),
    "v_cvt_f16_f32": (1, "u", lambda a: f32(a).astype(F16).view(U16).astype(U32)),
    "v_cvt_pk_f16_f32": (2, "u", lambda a, b: _pk16(f32(a).astype(F16), f32(b).astype(F16))),
    "v_cvt_pkrtz_f16_f32": (2, "u", lambda a, b: _pk16(_rtz16(f32(a)), _rtz16(f32(b)))),
    "v_cvt_pk_bf16_f32": (2, "u", lambda a, b: _bf16_rne(f32(a)) | (_bf16_rne(f32(b)) << U32(16))),
    "v_pack_b32_f16": (2, "u", lambda a, b: (a & U32(0xFFFF)) | (b << U32(16))),
    "v_ldexp_f32": (2, "u", lambda a, b: bits(np.ldexp(f32(a).astype(F64), np.clip(i32(b), -400, 400)).astype(F32))),
    "v_fmamk_f32": (3, "f", lambda a, k, b: fma32(a, k, b)),
    "v_fmaak_f32": (3, "f", lambda a, b, k: fma32(a, b, k)),
    "v_madmk_f32": (3, "f", lambda a, k, b: a * k + b),
    "v_madak_f32": (3, "f", lambda a, b, k: a * b + k),
    "v_dot2_f32_f16": (3, "u", lambda a, b, c: bits((_f16lo(a).astype(F64) * _f16lo(b).astype(F64)
                                                      + _f16hi(a).astype(F64) * _f16hi(b).astype(F64) + f32(c).astype(F64)).astype(F32))),
    "v_dot2_f32_bf16": (3, "u", lambda a, b, c: bits((f32(a << U32(16)).astype(F64) * f32(b << U32(16)).astype(F64)
                                                       + f32(a & U32(0xFFFF0000)).astype(F64) * f32(b & U32(0xFFFF0000)).astype(F64)
                                                       + f32(c).astype(F64)).astype(F32))),
    # float16 (scalar forms: low half in, low half out, high half of the destination zeroed as on gfx9)
    "v_add_f16": (2, "h", lambda a, b: a + b),
    "v_sub_f16": (2, "h", lambda a, b: a - b),
    "v_mul_f16": (2, "h", lambda a, b: a * b),
    "v_max_f16": (2, "h", lambda a, b: np.fmax(a, b)),
    "v_min_f16": (2, "h", lambda a, b: np.fmin(a, b)),
    "v_fma_f16": (3, "h", lambda a, b, c: (a.astype(F64) * b.astype(F64) + c.astype(F64)).astype(F16)),
    "v_rcp_f16": (1, "h", lambda a: (1.0 / a.astype(F64)).astype(F16)),
    "v_exp_f16": (1, "h", lambda a: np.exp2(a.astype(F64)).astype(F16)),
}


def _rtz16(x):
    h = x.astype(F16)
    over = np.abs(h.astype(F32)) > np.abs(x)
    hu = h.view(U16).copy()
    hu[over] -= 1
    return hu.view(F16)


_DPP_KEYS = ("quad_perm", "row_shl", "row_shr", "row_ror", "wave_shl", "wave_shr", "wave_rol", "wave_ror", "row_bcast",
             "row_newbcast", "row_share", "row_xmask")


def dpp_control(ins):
    """-> (src_lane int64[64], valid bool[64], enable bool[64], bound_ctrl)"""
    l = LANE
    r, rb = l & 15, l & ~15
    src, valid = l.copy(), np.ones(64, bool)
    found = False
    for m in ins.mods:
        key = m.split(":")[0]
        if key == "quad_perm":
            p = np.array(mod_val(ins, "quad_perm"), np.int64)
            src, found = (l & ~3) + p[l & 3], True
        elif key == "row_shl":
            n = mod_val(ins, key)
            src, valid, found = l + n, (r + n) <= 15, True
        elif key == "row_shr":
            n = mod_val(ins, key)
            src, valid, found = l - n, r >= n, True
        elif key == "row_ror":
            n = mod_val(ins, key)
            src, found = rb + ((r - n) & 15), True
        elif key == "wave_shl":
            src, valid, found = l + 1, l < 63, True
        elif key == "wave_shr":
            src, valid, found = l - 1, l > 0, True
        elif key == "wave_rol":
            src, found = (l + 1) & 63, True
        elif key == "wave_ror":
            src, found = (l - 1) & 63, True
        elif key == "row_mirror":
            src, found = rb + (15 - r), True
        elif key == "row_half_mirror":
            src, found = (l & ~7) + (7 - (l & 7)), True
        elif key == "row_bcast":
            n = mod_val(ins, key)
            if n == 15:
                src, valid = rb - 1, l >= 16
            else:
                src, valid = np.full(64, 31, np.int64), l >= 32
            found = True
        elif key == "row_newbcast" or key == "row_share":
            src, found = rb + mod_val(ins, key), True
    if not found:
        raise SimError(f"dpp control of `{ins.text}`")
    rm, bm = mod_val(ins, "row_mask", 0xF), mod_val(ins, "bank_mask", 0xF)
    enable = (((rm >> (l >> 4)) & 1) == 1) & (((bm >> ((l >> 2) & 3)) & 1) == 1)
    bc = any(m.startswith("bound_ctrl") for m in ins.mods)
    src = np.clip(src, 0, 63)
    return src, valid, enable, bc


_SEL = {"BYTE_0": (0, 0xFF), "BYTE_1": (8, 0xFF), "BYTE_2": (16, 0xFF), "BYTE_3": (24, 0xFF), "WORD_0": (0, 0xFFFF), "WORD_1": (16, 0xFFFF),
        "DWORD": (0, M32)}


def sdwa_src(g, sel, sext, kind, neg, absf):
    sh, mk = _SEL[sel]
    bitsn = 8 if mk == 0xFF else 16 if mk == 0xFFFF else 32

    def h(w):
        a = (g(w) >> U32(sh)) & U32(mk)
        if sext and bitsn < 32:
            a = ((a << U32(32 - bitsn)).view(I32) >> (32 - bitsn)).view(U32)
        if absf or neg:
            sb = 0x8000 if (kind == "h" or (kind != "f" and bitsn == 16)) else 0x80000000
            if kind == "f":
                sb = 0x80000000
            if absf:
                a = a & U32(~sb & M32)
            if neg:
                a = a ^ U32(sb)
        return a
    return h


def build_valu(ins):
    nsrc, kind, fn = VALU[ins.base]
    d = dreg(ins.ops[0])[1]
    variant = ins.mnem[len(ins.base) + 1:]
    k = {"f": "f32", "h": "f16", "u": "i32"}[kind]
    opnds = [Opnd(t) for t in ins.ops[1:1 + nsrc]]
    if len(opnds) != nsrc:
        raise SimError(f"operand count of `{ins.text}`")
    clamp = has_mod(ins, "clamp")
    omod = {"mul:2": 2.0, "mul:4": 4.0, "div:2": 0.5}
    om = next((omod[m] for m in ins.mods if m in omod), None)
    if variant == "sdwa":
        srcs = []
        for i, o in enumerate(opnds):
            raw = Opnd(o.text)
            raw.neg = raw.abs = raw.sext = False           # the SDWA select comes first, then the modifiers
            g = vsrc(raw, k)
            sel = next((m.split(":")[1] for m in ins.mods if m.startswith(f"src{i}_sel:")), "DWORD")
            srcs.append(sdwa_src(g, sel, o.sext, kind, o.neg, o.abs))
        dsel = next((m.split(":")[1] for m in ins.mods if m.startswith("dst_sel:")), "DWORD")
        dun = next((m.split(":")[1] for m in ins.mods if m.startswith("dst_unused:")), "UNUSED_PAD")
    else:
        srcs = [vsrc(o, k) for o in opnds]
        dsel = "DWORD"
    dpp = dpp_control(ins) if "dpp" in variant else None

    def run(w):
        a = [g(w) for g in srcs]
        enable = None
        if dpp is not None:
            src, valid, en, bc = dpp
            valid = valid & w.execb[src]
            s0 = a[0][src]
            if bc:
                s0 = np.where(valid, s0, U32(0))
                enable = en
            else:
                enable = en & valid
            a[0] = s0
        if kind == "f":
            r = fn(*[x.view(F32) for x in a])
            if om is not None:
                r = r * F32(om)
            if clamp:
                r = np.clip(r, F32(0), F32(1))
            r = np.ascontiguousarray(r, F32).view(U32)
        elif kind == "h":
            r = fn(*[_f16lo(x) for x in a])
            if clamp:
                r = np.clip(r, F16(0), F16(1))
            r = np.ascontiguousarray(r, F16).view(U16).astype(U32)
        else:
            r = fn(*a)
            if r.dtype != U32:
                r = r.astype(U32)
        if dsel != "DWORD":
            sh, mk = _SEL[dsel]
            old = w.v[d]
            piece = (r & U32(mk)) << U32(sh)
            if dun == "UNUSED_PRESERVE":
                r = (old & U32(~(mk << sh) & M32)) | piece
            elif dun == "UNUSED_SEXT":
                bitsn = 8 if mk == 0xFF else 16
                r = (((r & U32(mk)) << U32(32 - bitsn)).view(I32) >> (32 - bitsn - sh)).view(U32) & U32(~((1 << sh) - 1) & M32)
            else:
                r = piece
        if enable is None:
            w.wv(d, r)
        else:
            if w.npend and w.vpend[d]:
                w.hazard(f"write of v{d} while a load into it is in flight")
            np.copyto(w.v[d], r, where=enable & w.execb)
    return run


for _n in VALU:
    BUILDERS[_n] = build_valu


@op("v_fmac_f32", "v_mac_f32")
def _(ins):
    d = dreg(ins.ops[0])[1]
    a, b = vsrc(ins.ops[1], "f32"), vsrc(ins.ops[2], "f32")
    dpp = dpp_control(ins) if "dpp" in ins.mnem else None
    fused = ins.base == "v_fmac_f32"

    def run(w):
        x, y = a(w), b(w)
        en = None
        if dpp is not None:
            src, valid, e, bc = dpp
            valid = valid & w.execb[src]
            x = np.where(valid, x[src], U32(0)) if bc else x[src]
            en = e if bc else e & valid
        if w.npend and w.vpend[d]:
            w.hazard(f"read of v{d} while a load into it is in flight")
        r = bits(fma32(f32(x), f32(y), f32(w.v[d])) if fused else f32(x) * f32(y) + f32(w.v[d]))
        if en is None:
            w.wv(d, r)
        else:
            np.copyto(w.v[d], r, where=en & w.execb)
    return run


@op("v_fmac_f64")
def _(ins):
    d = dreg(ins.ops[0])[1]
    a, b = vsrc64(ins.ops[1], "f64"), vsrc64(ins.ops[2], "f64")

    def run(w):
        c = w.v[d].astype(U64) | (w.v[d + 1].astype(U64) << U64(32))
        r = a(w).view(F64) * b(w).view(F64) + c.view(F64)
        w.wv64(d, np.ascontiguousarray(r, F64).view(U64))
    return run


@op("v_dot2c_f32_f16", "v_dot2c_f32_bf16")
def _(ins):
    d = dreg(ins.ops[0])[1]
    a, b = vsrc(ins.ops[1]), vsrc(ins.ops[2])
    fn = VALU["v_dot2_f32_f16" if ins.base.endswith("f16") and not ins.base.endswith("bf16") else "v_dot2_f32_bf16"][2]
    return lambda w: w.wv(d, fn(a(w), b(w), w.v[d]))


@op("v_mov_b64")
def _(ins):
    d = dreg(ins.ops[0])[1]
    a = vsrc64(ins.ops[1], "u64")
    return lambda w: w.wv64(d, a(w))


@op("v_cndmask_b32")
def _(ins):
    d = dreg(ins.ops[0])[1]
    if "dpp" in ins.mnem:
        raise SimError(f"unsupported form `{ins.text}`")
    m = ssrc64(ins.ops[3]) if len(ins.ops) > 3 else (lambda w: w.s[VCC] | (w.s[VCC + 1] << 32))
    if "sdwa" in ins.mnem:
        srcs = []
        for i in (0, 1):
            o = Opnd(ins.ops[1 + i])
            raw = Opnd(o.text)
            raw.neg = raw.abs = raw.sext = False
            sel = next((x.split(":")[1] for x in ins.mods if x.startswith(f"src{i}_sel:")), "DWORD")
            srcs.append(sdwa_src(vsrc(raw, "f32"), sel, o.sext, "u", o.neg, o.abs))
        dsel = next((x.split(":")[1] for x in ins.mods if x.startswith("dst_sel:")), "DWORD")
        dun = next((x.split(":")[1] for x in ins.mods if x.startswith("dst_unused:")), "UNUSED_PAD")
        a, b = srcs

        def run(w):
            r = np.where(mask_to_bool(m(w)), b(w), a(w))
            if dsel != "DWORD":
                sh, mk = _SEL[dsel]
                piece = (r & U32(mk)) << U32(sh)
                r = (w.v[d] & U32(~(mk << sh) & M32)) | piece if dun == "UNUSED_PRESERVE" else piece
            w.wv(d, r)
        return run
    a, b = vsrc(ins.ops[1], "f32"), vsrc(ins.ops[2], "f32")
    return lambda w: w.wv(d, np.where(mask_to_bool(m(w)), b(w), a(w)))


@op("v_readfirstlane_b32")
def _(ins):
    d, a = dreg(ins.ops[0])[1], vsrc(ins.ops[1])

    def run(w):
        e = w.get_exec()
        lane = (e & -e).bit_length() - 1 if e else 0
        w.ws(d, int(a(w)[lane]))
    return run


@op("v_readlane_b32")
def _(ins):
    d, a, l = dreg(ins.ops[0])[1], vsrc(ins.ops[1]), ssrc(ins.ops[2])
    return lambda w: w.ws(d, int(a(w)[l(w) & 63]))


@op("v_writelane_b32")
def _(ins):
    d, a, l = dreg(ins.ops[0])[1], ssrc(ins.ops[1]), ssrc(ins.ops[2])

    def run(w):
        w.v[d][l(w) & 63] = a(w)
    return run


@op("v_mbcnt_lo_u32_b32", "v_mbcnt_hi_u32_b32")
def _(ins):
    d, av, b = dreg(ins.ops[0])[1], vsrc(ins.ops[1]), vsrc(ins.ops[2])
    hi = ins.base == "v_mbcnt_hi_u32_b32"
    lane = LANE.astype(U64)
    if hi:      # bits of the mask's HIGH word below this lane
        below = np.where(LANE >= 32, (U64(1) << np.where(LANE >= 32, lane - U64(32), U64(0))) - U64(1), U64(0))
    else:       # bits of the LOW word below this lane (all of it for lanes 32..63)
        below = np.where(LANE >= 32, U64(M32), (U64(1) << np.minimum(lane, U64(31))) - U64(1))

    def run(w):
        x = av(w).astype(U64) & below
        cnt = np.zeros(64, U32)
        for k in range(32):
            cnt += ((x >> U64(k)) & U64(1)).astype(U32)
        w.wv(d, cnt + b(w))
    return run


@op("v_accvgpr_write_b32", "v_accvgpr_write")
def _(ins):
    d, a = dreg(ins.ops[0])[1], vsrc(ins.ops[1])
    return lambda w: w.wv(d, a(w))


@op("v_accvgpr_read_b32", "v_accvgpr_read", "v_accvgpr_mov_b32")
def _(ins):
    d, a = dreg(ins.ops[0])[1], vsrc(ins.ops[1])
    return lambda w: w.wv(d, a(w))


def _carry_build(ins):
    """v_add_co_u32 / v_sub_co_u32 / v_subrev_co_u32 / v_addc_co_u32 / v_subb_co_u32 / v_subbrev_co_u32"""
    base = ins.base
    d = dreg(ins.ops[0])[1]
    co = dreg(ins.ops[1])[1]
    a, b = vsrc(ins.ops[2]), vsrc(ins.ops[3])
    cin = ssrc64(ins.ops[4]) if len(ins.ops) > 4 else None

    def run(w):
        x, y = a(w).astype(I64), b(w).astype(I64)
        c = mask_to_bool(cin(w)).astype(I64) if cin else 0
        if base in ("v_add_co_u32", "v_addc_co_u32"):
            r = x + y + c
            carry = r > M32
        elif base in ("v_sub_co_u32", "v_subb_co_u32"):
            r = x - y - c
            carry = r < 0
        else:
            r = y - x - c
            carry = r < 0
        w.wv(d, (r & M32).astype(U32))
        w.ws64(co, bool_to_mask(carry & w.execb))
    return run


for _n in ("v_add_co_u32", "v_sub_co_u32", "v_subrev_co_u32", "v_addc_co_u32", "v_subb_co_u32", "v_subbrev_co_u32"):
    BUILDERS[_n] = _carry_build


@op("v_mad_u64_u32", "v_mad_i64_i32")
def _(ins):
    d, co = dreg(ins.ops[0])[1], dreg(ins.ops[1])[1]
    a, b, c = vsrc(ins.ops[2]), vsrc(ins.ops[3]), vsrc64(ins.ops[4], "u64")
    signed = ins.base == "v_mad_i64_i32"

    def run(w):
        if signed:
            r = (i32(a(w)).astype(I64) * i32(b(w)).astype(I64)).view(U64) + c(w)
        else:
            r = a(w).astype(U64) * b(w).astype(U64) + c(w)
        w.wv64(d, r)
        w.ws64(co, 0)          # (carry out of bit 63: never consumed by compiled code here)
    return run


@op("v_lshl_add_u64")
def _(ins):
    d = dreg(ins.ops[0])[1]
    a, b, c = vsrc64(ins.ops[1], "u64"), vsrc(ins.ops[2]), vsrc64(ins.ops[3], "u64")
    return lambda w: w.wv64(d, (a(w) << (b(w) & U32(7)).astype(U64)) + c(w))


@op("v_lshlrev_b64", "v_lshrrev_b64", "v_ashrrev_i64")
def _(ins):
    d = dreg(ins.ops[0])[1]
    a, b = vsrc(ins.ops[1]), vsrc64(ins.ops[2], "u64")
    kind = ins.base

    def run(w):
        n = (a(w) & U32(63)).astype(U64)
        x = b(w)
        if kind == "v_lshlrev_b64":
            r = x << n
        elif kind == "v_lshrrev_b64":
            r = x >> n
        else:
            r = (x.view(I64) >> n.astype(I64)).view(U64)
        w.wv64(d, r)
    return run


@op("v_bitop3_b32", "v_bitop3_b16")
def _(ins):
    d = dreg(ins.ops[0])[1]
    a, b, c = vsrc(ins.ops[1]), vsrc(ins.ops[2]), vsrc(ins.ops[3])
    tt = mod_val(ins, "bitop3", 0)
    b16 = ins.base.endswith("b16")

    def run(w):
        x, y, z = a(w), b(w), c(w)
        r = np.zeros(64, U32)
        for i in range(8):
            if (tt >> i) & 1:
                t = (x if i & 4 else ~x) & (y if i & 2 else ~y) & (z if i & 1 else ~z)
                r |= t
        if b16:
            r &= U32(0xFFFF)
        w.wv(d, r)
    return run


@op("v_permlane16_swap_b32", "v_permlane32_swap_b32")
def _(ins):
    d, s = dreg(ins.ops[0])[1], dreg(ins.ops[1])[1]
    p32 = ins.base.startswith("v_permlane32")

    def run(w):
        if w.npend and (w.vpend[d] or w.vpend[s]):
            w.hazard("permlane swap of a register with a load in flight")
        vd, vs = w.v[d].copy(), w.v[s].copy()
        if p32:            # vdst[32:63] <-> src0[0:31]
            w.v[d][32:], w.v[s][:32] = vs[:32], vd[32:]
        else:              # odd rows of vdst <-> even rows of src0
            w.v[d][16:32], w.v[s][0:16] = vs[0:16], vd[16:32]
            w.v[d][48:64], w.v[s][32:48] = vs[32:48], vd[48:64]
    return run


# ---------------------------------------------------------------------------------------------------------------------
# mixed-precision, packed and double-precision VALU
# ---------------------------------------------------------------------------------------------------------------------
def _mix_srcs(ins):
    sel = mod_val(ins, "op_sel", [0, 0, 0])
    sel_hi = mod_val(ins, "op_sel_hi", [0, 0, 0])
    neg_lo = mod_val(ins, "neg_lo", [0, 0, 0])
    neg_hi = mod_val(ins, "neg_hi", [0, 0, 0])          # = abs for the mix instructions
    gs = []
    for i in range(3):
        o = Opnd(ins.ops[1 + i])
        neg, ab = o.neg or bool(neg_lo[i]), o.abs or bool(neg_hi[i])
        raw = Opnd(o.text.lstrip("-").strip("|"))
        if sel_hi[i]:
            g0 = vsrc(raw, "f16")
            half = sel[i]

            def g(w, g0=g0, half=half, neg=neg, ab=ab):
                a = g0(w)
                x = (_f16hi(a) if half else _f16lo(a)).astype(F32)
                if ab:
                    x = np.abs(x)
                return -x if neg else x
        else:
            g0 = vsrc(raw, "f32")

            def g(w, g0=g0, neg=neg, ab=ab):
                x = f32(g0(w))
                if ab:
                    x = np.abs(x)
                return -x if neg else x
        gs.append(g)
    return gs


@op("v_fma_mix_f32", "v_fma_mixlo_f16", "v_fma_mixhi_f16", "v_mad_mix_f32", "v_mad_mixlo_f16", "v_mad_mixhi_f16")
def _(ins):
    d = dreg(ins.ops[0])[1]
    gs = _mix_srcs(ins)
    clamp = has_mod(ins, "clamp")
    kind = ins.base

    def run(w):
        r = fma32(gs[0](w), gs[1](w), gs[2](w))
        if clamp:
            r = np.clip(r, F32(0), F32(1))
        if kind.endswith("_f32"):
            w.wv(d, bits(r))
        else:
            h = r.astype(F16).view(U16).astype(U32)
            old = w.v[d]
            w.wv(d, (old & U32(0xFFFF0000)) | h if kind.endswith("lo_f16") else (old & U32(0xFFFF)) | (h << U32(16)))
    return run


def _pk_f32(fn3):
    def build(ins):
        d = dreg(ins.ops[0])[1]
        n = len(ins.ops) - 1
        sel = mod_val(ins, "op_sel", [0] * n)
        sel_hi = mod_val(ins, "op_sel_hi", [1] * n)
        neg_lo = mod_val(ins, "neg_lo", [0] * n)
        neg_hi = mod_val(ins, "neg_hi", [0] * n)
        srcs = [vsrc64(Opnd(t), "u64") for t in ins.ops[1:]]
        # a 32-bit literal / inline constant of a packed-f32 source supplies the LOW dword of both halves
        consts = [not Opnd(t).is_reg() for t in ins.ops[1:]]
        ck = [const_bits(t, "f32") if c else None for t, c in zip(ins.ops[1:], consts)]

        def run(w):
            lo, hi = [], []
            for i, g in enumerate(srcs):
                if consts[i]:
                    x0 = x1 = full(ck[i]).view(F32)
                else:
                    a = g(w)
                    x0, x1 = (a & U64(M32)).astype(U32).view(F32), (a >> U64(32)).astype(U32).view(F32)
                l_ = x1 if sel[i] else x0
                h_ = x1 if sel_hi[i] else x0
                lo.append(-l_ if neg_lo[i] else l_)
                hi.append(-h_ if neg_hi[i] else h_)
            w.wv(d, bits(fn3(*lo)))
            w.wv(d + 1, bits(fn3(*hi)))
        return run
    return build


BUILDERS["v_pk_add_f32"] = _pk_f32(lambda a, b: a + b)
BUILDERS["v_pk_mul_f32"] = _pk_f32(lambda a, b: a * b)
BUILDERS["v_pk_fma_f32"] = _pk_f32(fma32)


def _pk_f16(fn):
    def build(ins):
        d = dreg(ins.ops[0])[1]
        n = len(ins.ops) - 1
        sel = mod_val(ins, "op_sel", [0] * n)
        sel_hi = mod_val(ins, "op_sel_hi", [1] * n)
        neg_lo = mod_val(ins, "neg_lo", [0] * n)
        neg_hi = mod_val(ins, "neg_hi", [0] * n)
        srcs = [vsrc(Opnd(t), "f16") for t in ins.ops[1:]]

        def run(w):
            lo, hi = [], []
            for i, g in enumerate(srcs):
                a = g(w)
                l_ = _f16hi(a) if sel[i] else _f16lo(a)
                h_ = _f16hi(a) if sel_hi[i] else _f16lo(a)
                lo.append(-l_ if neg_lo[i] else l_)
                hi.append(-h_ if neg_hi[i] else h_)
            w.wv(d, _pk16(np.asarray(fn(*lo), F16), np.asarray(fn(*hi), F16)))
        return run
    return build


BUILDERS["v_pk_add_f16"] = _pk_f16(lambda a, b: a + b)
BUILDERS["v_pk_mul_f16"] = _pk_f16(lambda a, b: a * b)
BUILDERS["v_pk_max_f16"] = _pk_f16(lambda a, b: np.fmax(a, b))
BUILDERS["v_pk_min_f16"] = _pk_f16(lambda a, b: np.fmin(a, b))
BUILDERS["v_pk_fma_f16"] = _pk_f16(lambda a, b, c: (a.astype(F64) * b.astype(F64) + c.astype(F64)).astype(F16))


def _f64_op(nsrc, fn):
    def build(ins):
        d = dreg(ins.ops[0])[1]
        srcs = [vsrc64(Opnd(t), "f64") for t in ins.ops[1:1 + nsrc]]

        def run(w):
            r = fn(*[g(w).view(F64) for g in srcs])
            w.wv64(d, np.ascontiguousarray(r, F64).view(U64))
        return run
    return build


BUILDERS["v_add_f64"] = _f64_op(2, lambda a, b: a + b)
BUILDERS["v_mul_f64"] = _f64_op(2, lambda a, b: a * b)
BUILDERS["v_max_f64"] = _f64_op(2, lambda a, b: np.fmax(a, b))
BUILDERS["v_min_f64"] = _f64_op(2, lambda a, b: np.fmin(a, b))
BUILDERS["v_fma_f64"] = _f64_op(3, lambda a, b, c: a * b + c)
BUILDERS["v_rcp_f64"] = _f64_op(1, lambda a: 1.0 / a)
BUILDERS["v_rsq_f64"] = _f64_op(1, lambda a: 1.0 / np.sqrt(a))
BUILDERS["v_sqrt_f64"] = _f64_op(1, np.sqrt)
BUILDERS["v_trunc_f64"] = _f64_op(1, np.trunc)
BUILDERS["v_floor_f64"] = _f64_op(1, np.floor)
BUILDERS["v_rndne_f64"] = _f64_op(1, np.rint)


@op("v_ldexp_f64")
def _(ins):
    d = dreg(ins.ops[0])[1]
    a, b = vsrc64(ins.ops[1], "f64"), vsrc(ins.ops[2])
    return lambda w: w.wv64(d, np.ascontiguousarray(np.ldexp(a(w).view(F64), np.clip(i32(b(w)), -4000, 4000)), F64).view(U64))


@op("v_cvt_f64_f32")
def _(ins):
    d, a = dreg(ins.ops[0])[1], vsrc(ins.ops[1], "f32")
    return lambda w: w.wv64(d, np.ascontiguousarray(f32(a(w)).astype(F64)).view(U64))


@op("v_cvt_f64_i32")
def _(ins):
    d, a = dreg(ins.ops[0])[1], vsrc(ins.ops[1])
    return lambda w: w.wv64(d, np.ascontiguousarray(i32(a(w)).astype(F64)).view(U64))


@op("v_cvt_f64_u32")
def _(ins):
    d, a = dreg(ins.ops[0])[1], vsrc(ins.ops[1])
    return lambda w: w.wv64(d, np.ascontiguousarray(a(w).astype(F64)).view(U64))


@op("v_cvt_f32_f64")
def _(ins):
    d, a = dreg(ins.ops[0])[1], vsrc64(ins.ops[1], "f64")
    return lambda w: w.wv(d, bits(a(w).view(F64).astype(F32)))


@op("v_cvt_i32_f64", "v_cvt_u32_f64")
def _(ins):
    d, a = dreg(ins.ops[0])[1], vsrc64(ins.ops[1], "f64")
    u = ins.base == "v_cvt_u32_f64"

    def run(w):
        x = a(w).view(F64)
        x = np.where(np.isnan(x), 0.0, np.trunc(x))
        w.wv(d, np.clip(x, 0, 4294967295.0).astype(U64).astype(U32) if u else np.clip(x, -2147483648.0, 2147483647.0).astype(I64).astype(I32).view(U32))
    return run


@op("v_div_scale_f32")
def _(ins):
    # the scaling exists to keep the Newton iteration in range; v_div_fixup below recomputes the quotient from the
    # original operands, so the unscaled operand and VCC = 0 give the correctly rounded result
    d, co = dreg(ins.ops[0])[1], dreg(ins.ops[1])[1]
    a = vsrc(ins.ops[2], "f32")

    def run(w):
        w.wv(d, a(w))
        w.ws64(co, 0)
    return run


@op("v_div_scale_f64")
def _(ins):
    d, co = dreg(ins.ops[0])[1], dreg(ins.ops[1])[1]
    a = vsrc64(ins.ops[2], "f64")

    def run(w):
        w.wv64(d, a(w))
        w.ws64(co, 0)
    return run


BUILDERS["v_div_fmas_f32"] = lambda ins: build_valu_named(ins, "v_fma_f32")
BUILDERS["v_div_fmas_f64"] = _f64_op(3, lambda a, b, c: a * b + c)


def build_valu_named(ins, name):
    saved = ins.base
    ins.base = name
    try:
        return build_valu(ins)
    finally:
        ins.base = saved


@op("v_div_fixup_f32")
def _(ins):
    d = dreg(ins.ops[0])[1]
    den, num = vsrc(ins.ops[2], "f32"), vsrc(ins.ops[3], "f32")
    return lambda w: w.wv(d, bits((f32(num(w)).astype(F64) / f32(den(w)).astype(F64)).astype(F32)))


@op("v_div_fixup_f64")
def _(ins):
    d = dreg(ins.ops[0])[1]
    den, num = vsrc64(ins.ops[2], "f64"), vsrc64(ins.ops[3], "f64")
    return lambda w: w.wv64(d, np.ascontiguousarray(num(w).view(F64) / den(w).view(F64), F64).view(U64))


# ---------------------------------------------------------------------------------------------------------------------
# compares
# ---------------------------------------------------------------------------------------------------------------------
_FCMP = {"f": lambda a, b: np.zeros(64, bool), "lt": lambda a, b: a < b, "eq": lambda a, b: a == b, "le": lambda a, b: a <= b,
         "gt": lambda a, b: a > b, "lg": lambda a, b: (a < b) | (a > b), "ge": lambda a, b: a >= b,
         "o": lambda a, b: ~(np.isnan(a) | np.isnan(b)), "u": lambda a, b: np.isnan(a) | np.isnan(b),
         "nge": lambda a, b: ~(a >= b), "nlg": lambda a, b: ~((a < b) | (a > b)), "ngt": lambda a, b: ~(a > b),
         "nle": lambda a, b: ~(a <= b), "neq": lambda a, b: ~(a == b), "nlt": lambda a, b: ~(a < b), "tru": lambda a, b: np.ones(64, bool)}
_ICMP = {"f": lambda a, b: np.zeros(64, bool), "lt": lambda a, b: a < b, "eq": lambda a, b: a == b, "le": lambda a, b: a <= b,
         "gt": lambda a, b: a > b, "ne": lambda a, b: a != b, "lg": lambda a, b: a != b, "ge": lambda a, b: a >= b,
         "t": lambda a, b: np.ones(64, bool)}
_CMP_RE = re.compile(r"v_cmpx?_(\w+?)_(f16|f32|f64|i16|u16|i32|u32|i64|u64)$")


def build_vcmp(ins):
    m = _CMP_RE.match(ins.base)
    cname, ty = m.group(1), m.group(2)
    cmpx = ins.base.startswith("v_cmpx")
    d = dreg(ins.ops[0])[1]
    if "sdwa" in ins.mnem or "dpp" in ins.mnem:
        raise SimError(f"unsupported form `{ins.text}`")
    if cname == "class":
        if ty == "f64":
            a, b = vsrc64(ins.ops[1], "f64"), vsrc(ins.ops[2])
            fn = lambda w: _class_f64(a(w), b(w))
        else:
            a, b = vsrc(ins.ops[1], "f32"), vsrc(ins.ops[2])
            fn = lambda w: _class_f32(a(w), b(w))
    elif ty in ("f64", "i64", "u64"):
        k = "f64" if ty == "f64" else ("i64" if ty == "i64" else "u64")
        a, b = vsrc64(ins.ops[1], k), vsrc64(ins.ops[2], k)
        view = {"f64": F64, "i64": I64, "u64": U64}[ty]
        c = (_FCMP if ty == "f64" else _ICMP)[cname]
        fn = lambda w: c(a(w).view(view), b(w).view(view))
    elif ty == "f32":
        a, b = vsrc(ins.ops[1], "f32"), vsrc(ins.ops[2], "f32")
        c = _FCMP[cname]
        fn = lambda w: c(f32(a(w)), f32(b(w)))
    elif ty == "f16":
        a, b = vsrc(ins.ops[1], "f16"), vsrc(ins.ops[2], "f16")
        c = _FCMP[cname]
        fn = lambda w: c(_f16lo(a(w)), _f16lo(b(w)))
    elif ty in ("i32", "u32"):
        a, b = vsrc(ins.ops[1]), vsrc(ins.ops[2])
        c = _ICMP[cname]
        fn = (lambda w: c(i32(a(w)), i32(b(w)))) if ty == "i32" else (lambda w: c(a(w), b(w)))
    else:  # i16 / u16
        a, b = vsrc(ins.ops[1]), vsrc(ins.ops[2])
        c = _ICMP[cname]
        if ty == "u16":
            fn = lambda w: c(a(w) & U32(0xFFFF), b(w) & U32(0xFFFF))
        else:
            fn = lambda w: c((a(w) & U32(0xFFFF)).astype(U16).view(I16), (b(w) & U32(0xFFFF)).astype(U16).view(I16))

    def run(w):
        r = bool_to_mask(fn(w) & w.execb)
        w.ws64(d, r)
        if cmpx:
            w.set_exec(r)
    return run


# ---------------------------------------------------------------------------------------------------------------------
# MFMA
# ---------------------------------------------------------------------------------------------------------------------
def _frag16(w, r0, nreg, bf):
    """8 (or 4) 16-bit elements per lane -> float64 [64, 2*nreg]"""
    regs = w.v[r0:r0 + nreg]                                  # [nreg, 64]
    h = np.ascontiguousarray(regs.T).view(U16)                 # [64, 2*nreg]
    if bf:
        return (h.astype(U32) << U32(16)).view(F32).astype(F64)
    return h.view(F16).astype(F64)


def _check_regs(w, r0, n, what):
    if w.npend and w.vpend[r0:r0 + n].any():
        w.hazard(f"MFMA reads {what} v[{r0}:{r0 + n - 1}] while a load into it is in flight")


def _mfma_src_c(o):
    od = Opnd(o)
    if od.reg:
        return od.reg[1], None
    return None, const_bits(o, "f32")


@op("v_mfma_f32_32x32x16_f16", "v_mfma_f32_32x32x16_bf16", "v_mfma_f32_32x32x8_f16", "v_mfma_f32_32x32x8_bf16_1k",
    "v_mfma_f32_32x32x8f16", "v_mfma_f32_32x32x8bf16_1k")
def _(ins):
    d = dreg(ins.ops[0])[1]
    a, b = dreg(ins.ops[1]), dreg(ins.ops[2])
    c, cconst = _mfma_src_c(ins.ops[3])
    bf = "bf16" in ins.base
    nreg = a[2]
    kper = 2 * nreg                                           # k elements per lane (8: x16 form, 4: x8 form)
    for mm in ins.mods:
        if mm.split(":")[0] in ("cbsz", "abid", "blgp") and int(mm.split(":")[1], 0) != 0:
            raise SimError(f"MFMA modifier {mm}")

    def run(w):
        _check_regs(w, a[1], nreg, "A")
        _check_regs(w, b[1], nreg, "B")
        A = _frag16(w, a[1], nreg, bf).reshape(2, 32, kper).transpose(1, 0, 2).reshape(32, 2 * kper)      # [i, k]
        B = _frag16(w, b[1], nreg, bf).reshape(2, 32, kper).transpose(0, 2, 1).reshape(2 * kper, 32)      # [k, n]
        if c is not None:
            _check_regs(w, c, 16, "C")
            Cm = w.v[c:c + 16].view(F32).reshape(4, 4, 2, 32).transpose(0, 2, 1, 3).reshape(32, 32).astype(F64)
        else:
            Cm = np.full((32, 32), np.array([cconst], U32).view(F32)[0], F64)
        D = (A @ B + Cm).astype(F32)
        out = D.reshape(4, 2, 4, 32).transpose(0, 2, 1, 3).reshape(16, 64)
        if w.npend and w.vpend[d:d + 16].any():
            w.hazard("MFMA writes a register with a load in flight")
        w.v[d:d + 16] = out.view(U32)
    return run


@op("v_mfma_f32_16x16x32_f16", "v_mfma_f32_16x16x32_bf16", "v_mfma_f32_16x16x16_f16", "v_mfma_f32_16x16x16_bf16_1k",
    "v_mfma_f32_16x16x16f16", "v_mfma_f32_16x16x16bf16_1k")
def _(ins):
    d = dreg(ins.ops[0])[1]
    a, b = dreg(ins.ops[1]), dreg(ins.ops[2])
    c, cconst = _mfma_src_c(ins.ops[3])
    bf = "bf16" in ins.base
    nreg = a[2]
    kper = 2 * nreg

    def run(w):
        _check_regs(w, a[1], nreg, "A")
        _check_regs(w, b[1], nreg, "B")
        A = _frag16(w, a[1], nreg, bf).reshape(4, 16, kper).transpose(1, 0, 2).reshape(16, 4 * kper)
        B = _frag16(w, b[1], nreg, bf).reshape(4, 16, kper).transpose(0, 2, 1).reshape(4 * kper, 16)
        if c is not None:
            _check_regs(w, c, 4, "C")
            # C/D: col = lane & 15, row = 4 * (lane >> 4) + reg
            Cm = w.v[c:c + 4].view(F32).reshape(4, 4, 16).transpose(1, 0, 2).reshape(16, 16).astype(F64)
        else:
            Cm = np.full((16, 16), np.array([cconst], U32).view(F32)[0], F64)
        D = (A @ B + Cm).astype(F32)
        w.v[d:d + 4] = np.ascontiguousarray(D.reshape(4, 4, 16).transpose(1, 0, 2).reshape(4, 64)).view(U32)
    return run


@op("v_mfma_f32_32x32x2_f32", "v_mfma_f32_32x32x2f32")
def _(ins):
    d = dreg(ins.ops[0])[1]
    a, b = vsrc(ins.ops[1], "f32"), vsrc(ins.ops[2], "f32")
    c, cconst = _mfma_src_c(ins.ops[3])

    def run(w):
        A = f32(a(w)).reshape(2, 32).astype(F64)               # [k, i]
        B = f32(b(w)).reshape(2, 32).astype(F64)               # [k, j]
        if c is not None:
            _check_regs(w, c, 16, "C")
            acc = w.v[c:c + 16].view(F32).reshape(4, 4, 2, 32).transpose(0, 2, 1, 3).reshape(32, 32).astype(F32)
        else:
            acc = np.full((32, 32), np.array([cconst], U32).view(F32)[0], F32)
        for k in range(2):                                     # k-ordered fp32 fma chain (guide section 3)
            acc = (np.outer(A[k], B[k]) + acc.astype(F64)).astype(F32)
        w.v[d:d + 16] = np.ascontiguousarray(acc.reshape(4, 2, 4, 32).transpose(0, 2, 1, 3).reshape(16, 64)).view(U32)
    return run


@op("v_mfma_f32_16x16x4_f32", "v_mfma_f32_16x16x4f32")
def _(ins):
    d = dreg(ins.ops[0])[1]
    a, b = vsrc(ins.ops[1], "f32"), vsrc(ins.ops[2], "f32")
    c, cconst = _mfma_src_c(ins.ops[3])

    def run(w):
        A = f32(a(w)).reshape(4, 16).astype(F64)
        B = f32(b(w)).reshape(4, 16).astype(F64)
        if c is not None:
            _check_regs(w, c, 4, "C")
            acc = w.v[c:c + 4].view(F32).reshape(4, 4, 16).transpose(1, 0, 2).reshape(16, 16).astype(F32)
        else:
            acc = np.full((16, 16), np.array([cconst], U32).view(F32)[0], F32)
        for k in range(4):
            acc = (np.outer(A[k], B[k]) + acc.astype(F64)).astype(F32)
        w.v[d:d + 4] = np.ascontiguousarray(acc.reshape(4, 4, 16).transpose(1, 0, 2).reshape(4, 64)).view(U32)
    return run


# ---------------------------------------------------------------------------------------------------------------------
# LDS
# ---------------------------------------------------------------------------------------------------------------------
def _lds_check(w, addr, nbytes, active, what, write=False):
    wg = w.wg
    a = addr[active]
    if a.size == 0:
        return
    if (a % min(nbytes, 4)).any() and nbytes >= 4:
        raise SimError(f"{what}: LDS address not dword aligned")
    if (a + nbytes > wg.lds_size).any() or (a < 0).any():
        w.hazard(f"{what}: LDS access beyond the {wg.lds_size} bytes of the workgroup's allocation")
        raise SimError("LDS out of range")
    idx = (a[:, None] + np.arange(nbytes, dtype=np.int64)).reshape(-1)
    pend = wg.lds_pending[idx] > 0
    if write:
        # a store over bytes with an LDS-DMA in flight: whichever lands last wins -> undefined until rewritten cleanly
        wg.lds_taint[idx] = pend
        return
    if pend.any():
        hit = idx[pend]
        owners = sorted(set(int(o) for o in wg.lds_owner[hit]))
        w.hazard(f"{what}: reads LDS bytes {int(hit.min()):#x}..{int(hit.max()):#x} while an LDS-DMA of wave(s) {owners} into them is "
                 f"still in flight (this wave has {len(w.vmq)} VMEM operations outstanding)")
    elif wg.lds_taint[idx].any():
        hit = idx[wg.lds_taint[idx]]
        w.hazard(f"{what}: reads LDS bytes {int(hit.min()):#x}..{int(hit.max()):#x} whose content is undefined (a store raced an LDS-DMA)")


# LDS banking per instruction (MI355X_MICROARCH.md, section LDS): a wave64 access is serviced in fixed lane groups, one LDS cycle per group
# when conflict-free; only lanes of the same group conflict, identical addresses broadcast, and each extra distinct address on a busy bank
# adds one cycle.  (lane groups, banks) by access width in dwords:
_G32 = [np.arange(0, 32), np.arange(32, 64)]
_G16 = [np.arange(16 * i, 16 * i + 16) for i in range(4)]
_G8 = [np.arange(8 * i, 8 * i + 8) for i in range(8)]
_G128R = [np.array([0, 1, 2, 3, 12, 13, 14, 15, 20, 21, 22, 23, 24, 25, 26, 27]), np.array([4, 5, 6, 7, 8, 9, 10, 11, 16, 17, 18, 19, 28, 29, 30, 31]),
          np.array([32, 33, 34, 35, 44, 45, 46, 47, 52, 53, 54, 55, 56, 57, 58, 59]), np.array([36, 37, 38, 39, 40, 41, 42, 43, 48, 49, 50, 51, 60, 61, 62, 63])]
_G96R = [np.array(g) for g in ([0, 1, 2, 3, 20, 21, 22, 23], [4, 5, 6, 7, 16, 17, 18, 19], [8, 9, 10, 11, 28, 29, 30, 31], [12, 13, 14, 15, 24, 25, 26, 27])]
_G96R += [g + 32 for g in _G96R]
_LDS_READ_BANKING = {1: (_G32, 32), 2: (_G32, 64), 3: (_G96R, 32), 4: (_G128R, 64), "read2_b64": (_G16, 32)}
_LDS_WRITE_BANKING = {1: (_G32, 32), 2: (_G16, 32), 3: (_G8, 32), 4: (_G8, 32)}


def _lds_bank_cycles(w, addr, act, ndw, write, pc=None, two=False):
    """LDS-array cycles and conflict cycles of one access (GFX950SIM_STATS=1): -> counters 'lds_cycles', 'lds_conflict'.
    two: one of the two accesses of a ds_read2 / ds_write2 (ds_read2_b64 is banked differently from ds_read_b64)"""
    groups, nb = (_LDS_WRITE_BANKING if write else _LDS_READ_BANKING)["read2_b64" if two and not write and ndw == 2 else ndw]
    cyc = 0
    for g in groups:
        ga = addr[g][act[g]] >> 2
        if ga.size == 0:
            continue
        dw = np.unique((ga[:, None] + np.arange(ndw)).reshape(-1))          # distinct dword addresses (identical ones broadcast)
        cyc += int(np.bincount(dw % nb, minlength=nb).max())
    c = w.mem.counters
    n = sum(1 for g in groups if act[g].any())
    c["lds_cycles"] = c.get("lds_cycles", 0) + cyc
    c["lds_conflict"] = c.get("lds_conflict", 0) + (cyc - n)
    if pc is not None and cyc > n:
        c["ldsc@%x" % pc] = c.get("ldsc@%x" % pc, 0) + (cyc - n)          # attribution: conflict cycles by instruction address


def _lds_read_builder(ndw, naddr=1, stride=0):
    """ds_read_b32/b64/b96/b128 (naddr = 1) and ds_read2(_st64)_b32/b64 (naddr = 2, stride in bytes per offset unit)"""
    def build(ins):
        d = dreg(ins.ops[0])[1]
        va = vsrc(ins.ops[1])
        if naddr == 1:
            offs = [mod_val(ins, "offset", 0)]
        else:
            offs = [mod_val(ins, "offset0", 0) * stride, mod_val(ins, "offset1", 0) * stride]
        nreg = ndw * naddr

        def run(w):
            w.flush_own_lds_writes()
            base = va(w).astype(np.int64)
            act = w.execb.copy()
            data = np.zeros((nreg, 64), U32)
            for k, off in enumerate(offs):
                addr = (base + off) & M32          # the LDS address is a 32-bit sum
                _lds_check(w, addr, 4 * ndw, act, ins.text)
                if w.stats_on:
                    _lds_bank_cycles(w, addr, act, ndw, False, ins.addr, naddr == 2)
                a = addr[act] >> 2
                for j in range(ndw):
                    data[k * ndw + j, act] = w.wg.lds32[a + j]

            def apply():
                for j in range(nreg):
                    np.copyto(w.v[d + j], data[j], where=act)
            w.push_lgkm(Pending(apply, regs=tuple(range(d, d + nreg)), what=ins.text))
        return run
    return build


BUILDERS["ds_read_b32"] = _lds_read_builder(1)
BUILDERS["ds_read_b64"] = _lds_read_builder(2)
BUILDERS["ds_read_b96"] = _lds_read_builder(3)
BUILDERS["ds_read_b128"] = _lds_read_builder(4)
BUILDERS["ds_read2_b32"] = _lds_read_builder(1, 2, 4)
BUILDERS["ds_read2_b64"] = _lds_read_builder(2, 2, 8)
BUILDERS["ds_read2st64_b32"] = _lds_read_builder(1, 2, 256)
BUILDERS["ds_read2st64_b64"] = _lds_read_builder(2, 2, 512)


def _lds_read_small(nbytes, signed, d16=None):
    def build(ins):
        d = dreg(ins.ops[0])[1]
        va = vsrc(ins.ops[1])
        off = mod_val(ins, "offset", 0)

        def run(w):
            w.flush_own_lds_writes()
            addr = (va(w).astype(np.int64) + off) & M32
            act = w.execb.copy()
            a = addr[act]
            if (a + nbytes > w.wg.lds_size).any():
                raise SimError(f"{ins.text}: LDS out of range")
            if w.wg.lds_pending[a].any() or w.wg.lds_taint[a].any():
                w.hazard(f"{ins.text}: reads LDS bytes with an LDS-DMA in flight / undefined content")
            v = np.zeros(a.size, U32)
            for k in range(nbytes):
                v |= w.wg.lds[a + k].astype(U32) << U32(8 * k)
            if signed:
                sh = 32 - 8 * nbytes
                v = ((v << U32(sh)).view(I32) >> sh).view(U32)
            data = np.zeros(64, U32)
            data[act] = v

            def apply():
                if d16 == "lo":
                    np.copyto(w.v[d], (w.v[d] & U32(0xFFFF0000)) | (data & U32(0xFFFF)), where=act)
                elif d16 == "hi":
                    np.copyto(w.v[d], (w.v[d] & U32(0xFFFF)) | (data << U32(16)), where=act)
                else:
                    np.copyto(w.v[d], data, where=act)
            w.push_lgkm(Pending(apply, regs=(d,), what=ins.text))
        return run
    return build


BUILDERS["ds_read_u16"] = _lds_read_small(2, False)
BUILDERS["ds_read_i16"] = _lds_read_small(2, True)
BUILDERS["ds_read_u8"] = _lds_read_small(1, False)
BUILDERS["ds_read_i8"] = _lds_read_small(1, True)
BUILDERS["ds_read_u16_d16"] = _lds_read_small(2, False, "lo")
BUILDERS["ds_read_u16_d16_hi"] = _lds_read_small(2, False, "hi")


def _lds_write_builder(ndw, naddr=1, stride=0):
    def build(ins):
        va = vsrc(ins.ops[0])
        datas = [dreg(t) for t in ins.ops[1:1 + naddr]]
        if naddr == 1:
            offs = [mod_val(ins, "offset", 0)]
        else:
            offs = [mod_val(ins, "offset0", 0) * stride, mod_val(ins, "offset1", 0) * stride]

        def run(w):
            base = va(w).astype(np.int64)
            act = w.execb.copy()
            items = []
            for k, off in enumerate(offs):
                addr = (base + off) & M32          # the LDS address is a 32-bit sum
                _lds_check(w, addr, 4 * ndw, act, ins.text, write=True)
                if w.stats_on:
                    _lds_bank_cycles(w, addr, act, ndw, True, ins.addr, naddr == 2)
                f, r0, n = datas[k]
                if w.npend and w.vpend[r0:r0 + ndw].any():
                    w.hazard(f"LDS store of v[{r0}:{r0 + ndw - 1}] while a load into it is in flight")
                items.append((addr[act] >> 2, w.v[r0:r0 + ndw][:, act].copy()))
            lds32 = w.wg.lds32

            def apply():
                for a, dat in items:
                    for j in range(ndw):
                        lds32[a + j] = dat[j]
            w.own_lds_writes += 1
            w.push_lgkm(Pending(apply, lds=True, what=ins.text))
        return run
    return build


BUILDERS["ds_write_b32"] = _lds_write_builder(1)
BUILDERS["ds_write_b64"] = _lds_write_builder(2)
BUILDERS["ds_write_b96"] = _lds_write_builder(3)
BUILDERS["ds_write_b128"] = _lds_write_builder(4)
BUILDERS["ds_write2_b32"] = _lds_write_builder(1, 2, 4)
BUILDERS["ds_write2_b64"] = _lds_write_builder(2, 2, 8)
BUILDERS["ds_write2st64_b32"] = _lds_write_builder(1, 2, 256)
BUILDERS["ds_write2st64_b64"] = _lds_write_builder(2, 2, 512)


def _lds_write_small(nbytes, hi=False):
    def build(ins):
        va = vsrc(ins.ops[0])
        r0 = dreg(ins.ops[1])[1]
        off = mod_val(ins, "offset", 0)

        def run(w):
            addr = (va(w).astype(np.int64) + off) & M32
            act = w.execb.copy()
            a = addr[act]
            if (a + nbytes > w.wg.lds_size).any():
                raise SimError(f"{ins.text}: LDS out of range")
            v = w.v[r0][act] >> U32(16) if hi else w.v[r0][act].copy()
            lds = w.wg.lds

            def apply():
                for k in range(nbytes):
                    lds[a + k] = ((v >> U32(8 * k)) & U32(0xFF)).astype(U8)
            w.own_lds_writes += 1
            w.push_lgkm(Pending(apply, lds=True, what=ins.text))
        return run
    return build


BUILDERS["ds_write_b16"] = _lds_write_small(2)
BUILDERS["ds_write_b8"] = _lds_write_small(1)
BUILDERS["ds_write_b16_d16_hi"] = _lds_write_small(2, True)


@op("ds_bpermute_b32", "ds_permute_b32")
def _(ins):
    d = dreg(ins.ops[0])[1]
    va, vd = vsrc(ins.ops[1]), vsrc(ins.ops[2])
    off = mod_val(ins, "offset", 0)
    fwd = ins.base == "ds_permute_b32"

    def run(w):
        idx = (((va(w).astype(np.int64) + off) >> 2) & 63)
        dat = vd(w)
        act = w.execb.copy()
        if fwd:
            res = np.zeros(64, U32)
            for l in np.nonzero(act)[0]:
                res[idx[l]] = dat[l]
        else:
            res = np.where(act[idx], dat[idx], U32(0))

        def apply():
            np.copyto(w.v[d], res, where=act)
        w.push_lgkm(Pending(apply, regs=(d,), what=ins.text))
    return run


@op("ds_add_f32", "ds_add_u32")
def _(ins):
    va = vsrc(ins.ops[0])
    r0 = dreg(ins.ops[1])[1]
    off = mod_val(ins, "offset", 0)
    isf = ins.base == "ds_add_f32"

    def run(w):
        w.flush_own_lds_writes()
        addr = (va(w).astype(np.int64) + off) & M32
        lds32 = w.wg.lds32
        for l in np.nonzero(w.execb)[0]:
            a = int(addr[l]) >> 2
            if isf:
                lds32[a:a + 1].view(F32)[0] += w.v[r0].view(F32)[l]
            else:
                lds32[a] += w.v[r0][l]
        w.push_lgkm(Pending(lambda: None, what=ins.text))
    return run


# ---------------------------------------------------------------------------------------------------------------------
# global / buffer memory
# ---------------------------------------------------------------------------------------------------------------------
def _global_addr(ins, first):
    """address accessor of a global_* instruction whose address operands start at ins.ops[first]: `v[a:b], off` or `vN, s[a:b]`"""
    o = Opnd(ins.ops[first])
    sa = ins.ops[first + 1] if len(ins.ops) > first + 1 else "off"
    off = mod_val(ins, "offset", 0)
    if sa == "off":
        g = vsrc64(o, "u64")
        return lambda w: g(w).astype(np.int64) + off
    sb = ssrc64(sa)
    g = vsrc(o)
    return lambda w: g(w).astype(np.int64) + sb(w) + off


def _gload(ndw):
    def build(ins):
        d = dreg(ins.ops[0])[1]
        addr = _global_addr(ins, 1)

        def run(w):
            a = addr(w)
            act = w.execb.copy()
            w.mem.check(a, 4 * ndw, ins.text, act)
            data = w.mem.gather(a, ndw, act)

            def apply():
                for j in range(ndw):
                    np.copyto(w.v[d + j], data[j], where=act)
            w.push_vm(Pending(apply, regs=tuple(range(d, d + ndw)), what=ins.text))
        return run
    return build


BUILDERS["global_load_dword"] = _gload(1)
BUILDERS["global_load_dwordx2"] = _gload(2)
BUILDERS["global_load_dwordx3"] = _gload(3)
BUILDERS["global_load_dwordx4"] = _gload(4)


def _gload_small(nbytes, signed, d16=None):
    def build(ins):
        d = dreg(ins.ops[0])[1]
        addr = _global_addr(ins, 1)

        def run(w):
            a = addr(w)
            act = w.execb.copy()
            w.mem.check(a, nbytes, ins.text, act)
            data = w.mem.gather_small(a, nbytes, act)
            if signed:
                sh = 32 - 8 * nbytes
                data = ((data << U32(sh)).view(I32) >> sh).view(U32)

            def apply():
                if d16 == "lo":
                    np.copyto(w.v[d], (w.v[d] & U32(0xFFFF0000)) | (data & U32(0xFFFF)), where=act)
                elif d16 == "hi":
                    np.copyto(w.v[d], (w.v[d] & U32(0xFFFF)) | (data << U32(16)), where=act)
                else:
                    np.copyto(w.v[d], data, where=act)
            w.push_vm(Pending(apply, regs=(d,), what=ins.text))
        return run
    return build


BUILDERS["global_load_ushort"] = _gload_small(2, False)
BUILDERS["global_load_sshort"] = _gload_small(2, True)
BUILDERS["global_load_ubyte"] = _gload_small(1, False)
BUILDERS["global_load_sbyte"] = _gload_small(1, True)
BUILDERS["global_load_short_d16"] = _gload_small(2, False, "lo")
BUILDERS["global_load_short_d16_hi"] = _gload_small(2, False, "hi")


def _gstore(ndw):
    def build(ins):
        # global_store_dwordx4 v[addr], v[data], off | global_store_dword vOff, vData, s[base]
        o0 = Opnd(ins.ops[0])
        r0 = dreg(ins.ops[1])[1]
        sa = ins.ops[2] if len(ins.ops) > 2 else "off"
        off = mod_val(ins, "offset", 0)
        if sa == "off":
            g = vsrc64(o0, "u64")
            addr = lambda w: g(w).astype(np.int64) + off
        else:
            sb, g = ssrc64(sa), vsrc(o0)
            addr = lambda w: g(w).astype(np.int64) + sb(w) + off

        def run(w):
            a = addr(w)
            act = w.execb.copy()
            w.mem.check(a, 4 * ndw, ins.text, act)
            if w.npend and w.vpend[r0:r0 + ndw].any():
                w.hazard(f"store of v[{r0}:{r0 + ndw - 1}] while a load into it is in flight")
            w.mem.scatter(a, w.v[r0:r0 + ndw], act)
            w.push_vm(Pending(_nothing, what=ins.text))
        return run
    return build


def _nothing():
    pass


BUILDERS["global_store_dword"] = _gstore(1)
BUILDERS["global_store_dwordx2"] = _gstore(2)
BUILDERS["global_store_dwordx3"] = _gstore(3)
BUILDERS["global_store_dwordx4"] = _gstore(4)


def _gstore_small(nbytes, hi=False):
    def build(ins):
        o0 = Opnd(ins.ops[0])
        r0 = dreg(ins.ops[1])[1]
        sa = ins.ops[2] if len(ins.ops) > 2 else "off"
        off = mod_val(ins, "offset", 0)
        if sa == "off":
            g = vsrc64(o0, "u64")
            addr = lambda w: g(w).astype(np.int64) + off
        else:
            sb, g = ssrc64(sa), vsrc(o0)
            addr = lambda w: g(w).astype(np.int64) + sb(w) + off

        def run(w):
            a = addr(w)
            act = w.execb.copy()
            w.mem.check(a, nbytes, ins.text, act)
            v = w.v[r0] >> U32(16) if hi else w.v[r0]
            w.mem.scatter_small(a, v, nbytes, act)
            w.push_vm(Pending(_nothing, what=ins.text))
        return run
    return build


BUILDERS["global_store_short"] = _gstore_small(2)
BUILDERS["global_store_byte"] = _gstore_small(1)
BUILDERS["global_store_short_d16_hi"] = _gstore_small(2, True)


def _lds_dma_issue(w, ins, data, act, lds_base, nbytes_per_lane):
    """data uint32 [ndw, 64] fetched now; lands in LDS at lds_base + lane * nbytes when the wave's vmcnt says so"""
    wg = w.wg
    ndw = nbytes_per_lane // 4
    lanes = np.nonzero(act)[0]
    dst = lds_base + lanes * nbytes_per_lane
    if dst.size and (dst.max() + nbytes_per_lane > wg.lds_size or lds_base < 0):
        w.hazard(f"LDS-DMA destination {lds_base:#x} beyond the workgroup's {wg.lds_size} bytes")
        raise SimError("LDS-DMA out of range")
    if lds_base & 3:
        raise SimError("LDS-DMA destination not dword aligned")
    idx = (dst[:, None] + np.arange(nbytes_per_lane, dtype=np.int64)).reshape(-1)
    wg.lds_taint[idx] = wg.lds_pending[idx] > 0          # a second DMA (another wave's) into bytes already in flight: order undefined
    wg.lds_pending[idx] += 1
    wg.lds_owner[idx] = w.wid
    vals = np.ascontiguousarray(data[:, lanes].T)                 # [n, ndw]
    d32 = (dst >> 2)

    def apply():
        for j in range(ndw):
            wg.lds32[d32 + j] = vals[:, j]
        wg.lds_pending[idx] -= 1
    w.push_vm(Pending(apply, what=ins.text))


@op("global_load_lds_dwordx4", "global_load_lds_dword", "global_load_lds_dwordx3")
def _(ins):
    ndw = {"global_load_lds_dword": 1, "global_load_lds_dwordx3": 3, "global_load_lds_dwordx4": 4}[ins.base]
    addr = _global_addr(ins, 0)
    ioff = mod_val(ins, "offset", 0)

    def run(w):
        a = addr(w)
        act = w.execb.copy()
        w.mem.check(a, 4 * ndw, ins.text, act)
        data = w.mem.gather(a, ndw, act)
        _lds_dma_issue(w, ins, data, act, (w.s[M0] & 0x3FFFF) + ioff, 4 * ndw)
    return run


def _buffer_access(ins, first):
    """-> f(w) -> (addr int64[64], inrange bool[64]) for `voffset, srsrc, soffset [offen] [offset:n]` starting at ins.ops[first]"""
    offen, idxen = has_mod(ins, "offen"), has_mod(ins, "idxen")
    if idxen:
        raise SimError("buffer idxen addressing")
    vo = vsrc(ins.ops[first]) if offen else None
    rs = dreg(ins.ops[first + 1])[1]
    so = ssrc(ins.ops[first + 2])
    ioff = mod_val(ins, "offset", 0)

    def f(w, nbytes):
        base = (w.s[rs] | ((w.s[rs + 1] & 0xFFFF) << 32))
        stride = (w.s[rs + 1] >> 16) & 0x3FFF
        nrec = w.s[rs + 2]
        if stride:
            raise SimError("buffer descriptor with a stride")
        off = (vo(w).astype(np.int64) if vo else np.zeros(64, np.int64)) + ioff
        s = so(w)
        # raw buffer: range-checked PER DWORD (a dwordx4 access straddling num_records returns its in-range dwords and zeros
        # for the rest); dword j is in range when offset + soffset + 4 * j + 4 <= num_records
        inr = [((off + s + 4 * j + 4) <= nrec) & (off >= 0) for j in range(nbytes // 4)]
        return base + s + off, inr
    return f


def _buffer_gather(w, ins, a, inr, act, ndw):
    data = np.zeros((ndw, 64), U32)
    for j in range(ndw):
        ok = act & inr[j]
        if ok.any():
            w.mem.check(a + 4 * j, 4, ins.text, ok)
            data[j] = w.mem.gather(a + 4 * j, 1, ok)[0]
    return data


@op("buffer_load_dword", "buffer_load_dwordx2", "buffer_load_dwordx3", "buffer_load_dwordx4")
def _(ins):
    ndw = {"buffer_load_dword": 1, "buffer_load_dwordx2": 2, "buffer_load_dwordx3": 3, "buffer_load_dwordx4": 4}[ins.base]
    lds = has_mod(ins, "lds")
    if lds:
        acc = _buffer_access(ins, 0)

        def run(w):
            a, inr = acc(w, 4 * ndw)
            act = w.execb.copy()
            data = _buffer_gather(w, ins, a, inr, act, ndw)       # out-of-range dwords deliver zeros
            _lds_dma_issue(w, ins, data, act, w.s[M0] & 0x3FFFF, 4 * ndw)
        return run
    d = dreg(ins.ops[0])[1]
    acc = _buffer_access(ins, 1)

    def run(w):
        a, inr = acc(w, 4 * ndw)
        act = w.execb.copy()
        data = _buffer_gather(w, ins, a, inr, act, ndw)

        def apply():
            for j in range(ndw):
                np.copyto(w.v[d + j], data[j], where=act)
        w.push_vm(Pending(apply, regs=tuple(range(d, d + ndw)), what=ins.text))
    return run


@op("buffer_store_dword", "buffer_store_dwordx2", "buffer_store_dwordx4")
def _(ins):
    ndw = {"buffer_store_dword": 1, "buffer_store_dwordx2": 2, "buffer_store_dwordx4": 4}[ins.base]
    r0 = dreg(ins.ops[0])[1]
    acc = _buffer_access(ins, 1)

    def run(w):
        a, inr = acc(w, 4 * ndw)
        for j in range(ndw):
            ok = w.execb & inr[j]
            if ok.any():
                w.mem.check(a + 4 * j, 4, ins.text, ok)
                w.mem.scatter(a + 4 * j, w.v[r0 + j:r0 + j + 1], ok)
        w.push_vm(Pending(_nothing, what=ins.text))
    return run


@op("global_atomic_add", "global_atomic_add_f32", "global_atomic_umax", "global_atomic_smax", "global_atomic_or", "global_atomic_inc")
def _(ins):
    ret = has_mod(ins, "sc0") or has_mod(ins, "glc")
    k = 1 if ret else 0
    d = dreg(ins.ops[0])[1] if ret else None
    o0 = Opnd(ins.ops[k])
    r0 = dreg(ins.ops[k + 1])[1]
    sa = ins.ops[k + 2] if len(ins.ops) > k + 2 else "off"
    off = mod_val(ins, "offset", 0)
    if sa == "off":
        g = vsrc64(o0, "u64")
        addr = lambda w: g(w).astype(np.int64) + off
    else:
        sb, g = ssrc64(sa), vsrc(o0)
        addr = lambda w: g(w).astype(np.int64) + sb(w) + off
    kind = ins.base

    def run(w):
        a = addr(w)
        act = w.execb.copy()
        w.mem.check(a, 4, ins.text, act)
        old = np.zeros(64, U32)
        for l in np.nonzero(act)[0]:
            cell = w.mem.u8[int(a[l]) - w.mem.base:int(a[l]) - w.mem.base + 4].view(U32)
            old[l] = cell[0]
            x = w.v[r0][l]
            if kind == "global_atomic_add":
                cell[0] = cell[0] + x
            elif kind == "global_atomic_add_f32":
                cell.view(F32)[0] += np.array([x], U32).view(F32)[0]
            elif kind == "global_atomic_umax":
                cell[0] = max(cell[0], x)
            elif kind == "global_atomic_smax":
                cell[0] = U32(max(sx(int(cell[0]), 32), sx(int(x), 32)) & M32)
            elif kind == "global_atomic_or":
                cell[0] |= x
            elif kind == "global_atomic_inc":
                cell[0] = 0 if cell[0] >= x else cell[0] + 1
        if ret:
            def apply():
                np.copyto(w.v[d], old, where=act)
            w.push_vm(Pending(apply, regs=(d,), what=ins.text))
        else:
            w.push_vm(Pending(_nothing, what=ins.text))
    return run


# scratch (register spills only): `scratch_store_dword off, vdata, off offset:N` / `scratch_load_dword vdst, off, off offset:N` -- a per-lane
# private slot addressed by the immediate offset alone
def _scratch(ins, store, ndw):
    if store:
        assert ins.ops[0] == "off" and ins.ops[2] == "off", f"scratch addressing of `{ins.text}`"
        r0 = dreg(ins.ops[1])[1]
    else:
        assert ins.ops[1] == "off" and ins.ops[2] == "off", f"scratch addressing of `{ins.text}`"
        r0 = dreg(ins.ops[0])[1]
    slot = mod_val(ins, "offset", 0) // 4

    def run(w):
        if w.scratch is None or slot + ndw > w.scratch.shape[0]:
            raise SimError(f"{ins.text}: beyond the kernel's private segment")
        act = w.execb.copy()
        if store:
            for j in range(ndw):
                np.copyto(w.scratch[slot + j], w.v[r0 + j], where=act)
            w.push_vm(Pending(_nothing, what=ins.text))
        else:
            data = w.scratch[slot:slot + ndw].copy()

            def apply():
                for j in range(ndw):
                    np.copyto(w.v[r0 + j], data[j], where=act)
            w.push_vm(Pending(apply, regs=tuple(range(r0, r0 + ndw)), what=ins.text))
    return run


for _n, _k in (("dword", 1), ("dwordx2", 2), ("dwordx3", 3), ("dwordx4", 4)):
    BUILDERS[f"scratch_store_{_n}"] = (lambda k: lambda ins: _scratch(ins, True, k))(_k)
    BUILDERS[f"scratch_load_{_n}"] = (lambda k: lambda ins: _scratch(ins, False, k))(_k)


# ---------------------------------------------------------------------------------------------------------------------
def compile_inst(ins):
    base, _ = strip_suffix(ins.mnem)
    ins.base = base
    b = BUILDERS.get(base)
    if b is None and _CMP_RE.match(base):
        b = build_vcmp
    if b is None:
        raise SimError(f"instruction not implemented: `{ins.text}` at {ins.addr:#x}")
    ins.fn = b(ins)
    return ins.fn
