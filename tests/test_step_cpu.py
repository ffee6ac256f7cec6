"""The argument contract of the C entry points of 8-bit linears, rotary positions and pages: answers given before any
device work.  The pointers here are never followed: the valid calls among them are those that a missing workspace
refuses, on a machine with a GPU too."""
import ctypes
import os

import pytest

torch = pytest.importorskip("torch")

A = 1 << 20


def _lib_or_skip():
    from w4a8_b200 import _lib
    if not os.path.exists(_lib.lib_path()):
        pytest.skip("libw4a8_b200.so not built")
    return _lib, _lib.lib()


def test_int8_argument_contract():
    _lib, L = _lib_or_skip()
    inv, uns, ok = _lib.ERR_INVALID, _lib.ERR_UNSUPPORTED, _lib.OK
    late = (_lib.ERR_CUDA, _lib.ERR_DEVICE, _lib.ERR_WORKSPACE)

    def linear(x=A, M=4, K=64, ldx=64, act=0, w=2 * A, ldw=64, ws=3 * A, b=None, N=8, y=4 * A, ldy=8, wk=None, wkb=0):
        return L.w4a8_int8_linear(x, M, K, ldx, act, w, ldw, ws, b, N, y, ldy, wk, wkb, None)

    assert linear(M=0) == ok and linear(M=-1) == inv and linear(K=0) == inv and linear(N=0) == inv
    assert linear(K=_lib.INT8_MAX_K + 1) == uns and linear(M=(1 << 24) + 1) == uns and linear(N=(1 << 24) + 1) == uns
    assert linear(x=None) == inv and linear(x=A + 1) == inv and linear(ldx=63) == inv
    assert linear(act=2) == uns and linear(act=1) == inv and linear(act=1, ldx=128) in late
    assert linear(w=None) == inv and linear(w=2 * A + 8) == inv and linear(ldw=48) == inv and linear(ldw=72) == inv
    assert linear(ws=None) == inv and linear(ws=3 * A + 2) == inv and linear(b=5 * A + 1) == inv
    assert linear(y=None) == inv and linear(y=4 * A + 1) == inv and linear(ldy=7) == inv
    assert linear() in late

    def norm(r=None, ldr=0, ro=None, ldro=0, w=6 * A, wd=0, eps=1e-6, K=64, ldx=64, M=4):
        return L.w4a8_int8_linear_rms_norm(A, M, K, ldx, r, ldr, ro, ldro, w, wd, eps, 2 * A, max(K, 64), 3 * A, None, 8, 4 * A, 8,
                                           None, 0, None)

    assert norm(M=0) == ok and norm(K=_lib.NORM_MAX_K + 16, ldx=1 << 16) == uns and norm(w=None) == inv and norm(wd=2) == uns
    assert norm(wd=1, w=6 * A + 2) == inv and norm(eps=-1.0) == inv and norm(eps=float("nan")) == inv
    assert norm(r=7 * A, ldr=63) == inv and norm(ro=7 * A, ldro=63) == inv and norm(r=7 * A + 1, ldr=64) == inv
    assert norm(r=7 * A, ldr=64, ro=7 * A, ldro=64) in late

    def gemm(q=A, ldq=64, s=5 * A, M=4, K=64, wk=None, wkb=0):
        return L.w4a8_int8_gemm(q, ldq, s, M, K, 2 * A, 64, 3 * A, None, 8, 4 * A, 8, wk, wkb, None)

    assert gemm(M=0) == ok and gemm(q=None) == inv and gemm(q=A + 8) == inv and gemm(ldq=72) == inv and gemm(ldq=48) == inv
    assert gemm(s=None) == inv and gemm() in late

    def quant(x=A, M=4, K=64, ldx=64, act=0, q=2 * A, ldq=64, s=3 * A):
        return L.w4a8_int8_quant(x, M, K, ldx, act, q, ldq, s, None)

    assert quant(M=0) == ok and quant(q=None) == inv and quant(ldq=63) == inv and quant(s=None) == inv and quant(s=3 * A + 2) == inv
    assert quant(act=7) == uns and quant(x=None) == inv
    assert L.w4a8_int8_workspace_size(4, 64) >= 1024 + 16 + 4 * 64 and L.w4a8_int8_workspace_size(0, 64) >= 1024
    assert L.w4a8_int8_workspace_size(-1, 64) == 0 and L.w4a8_int8_workspace_size(4, 0) == 0


def test_the_wrappers_workspace_holds_every_call():
    from w4a8_b200 import ops
    _, L = _lib_or_skip()
    for M in (1, 2, 255, 256, 257, 4095, 100001):
        for K in (1, 15, 16, 17, 1057, 27648):
            asked = []
            real, ops.workspace = ops.workspace, lambda n, dev: asked.append(n)
            try:
                ops._int8_ws(M, K, None)
            finally:
                ops.workspace = real
            assert asked[0] >= L.w4a8_int8_workspace_size(M, K), (M, K)


def test_rotary_argument_contract():
    _lib, L = _lib_or_skip()
    inv, uns = _lib.ERR_INVALID, _lib.ERR_UNSUPPORTED
    two = (ctypes.c_uint8 * 32)(*([0] * 16 + [1] * 16))
    bad = (ctypes.c_uint8 * 32)(*([0] * 31 + [2]))

    def rot(q=A, ldq=256, hq=4, qo=2 * A, ldqo=256, k=3 * A, ldk=128, hk=2, ko=4 * A, ldko=128, T=6, D=64, cs=5 * A, rows=10, r=64,
            pos=6 * A, ldp=6, axes=2, m=two):
        return L.w4a8_rotary(q, ldq, hq, qo, ldqo, k, ldk, hk, ko, ldko, T, D, cs, rows, r, 0, pos, ldp, axes, m, None)

    assert rot(T=0) == _lib.OK and rot(T=-1) == inv and rot(D=60) == uns and rot(D=0) == uns and rot(D=264, r=64) == uns
    assert rot(r=24) == uns and rot(r=80) == uns and rot(cs=None) == inv and rot(cs=5 * A + 4) == inv and rot(rows=0) == inv
    assert rot(q=None) == inv and rot(q=A + 8) == inv and rot(ldq=250) == inv and rot(ldq=248) == inv and rot(hq=0) == inv
    assert rot(qo=None) == inv and rot(ko=None) == inv and rot(ldko=120) == inv and rot(hk=0) == inv
    assert rot(pos=None) == inv and rot(pos=6 * A + 2) == inv and rot(ldp=5) == inv and rot(axes=0) == inv and rot(axes=5) == inv
    assert rot(m=None) == inv and rot(m=bad) == inv

    d = ctypes.byref(_lib.KvCacheDesc(A, 2 * A, 3 * A, 4 * A, 8, 2, 16, 64, 0))

    def write(cs=12 * A, pos=6 * A, ldp=6, axes=2, m=two, T=6, B=2):
        return L.w4a8_kv_write_axes(d, 5 * A, 4, 4, 6 * A, 7 * A, B, T, 8 * A, 128, 9 * A, 128, 10 * A, 256, 4, 11 * A, 256, cs, 10, 64, 0,
                                    pos, ldp, axes, m, None)

    assert write(T=0) == _lib.OK and write(cs=None) == inv and write(pos=None) == inv and write(ldp=5) == inv and write(m=bad) == inv
    assert write(axes=0) == inv


def test_pages_argument_contract():
    _lib, L = _lib_or_skip()
    inv, uns = _lib.ERR_INVALID, _lib.ERR_UNSUPPORTED

    def state(free=A, count=2 * A, table=3 * A, lens=4 * A, control=5 * A, pages=8, columns=4, sequences=3, page=16):
        return ctypes.byref(_lib.PageStateDesc(free, count, table, lens, control, pages, columns, sequences, page))

    def plan(st=None, rows=6 * A, counts=7 * A, B=2, T=6, axes=1, sc=None, sg=None, n=0, table=8 * A, lens=9 * A, cu=10 * A,
             slots=None, pos=None):
        return L.w4a8_pages_plan(st or state(), rows, counts, B, T, axes, sc, sg, n, table, lens, cu, slots, pos, None)

    for bad in (state(free=None), state(count=2 * A + 2), state(table=None), state(lens=None), state(control=None), state(pages=0),
                state(pages=1 << 28), state(columns=0), state(columns=1 << 40), state(sequences=0), state(columns=-1)):
        assert plan(bad) == inv
        assert L.w4a8_pages_shrink(bad, 6 * A, None, 2, None) == inv
    assert plan(state(page=24)) == uns and plan(state(sequences=_lib.PLAN_MAX_SEQUENCES + 1)) == uns
    assert plan(B=_lib.PLAN_MAX_BATCH + 1) == uns and plan(B=-1) == inv and plan(T=-1) == inv and plan(axes=0) == inv and plan(axes=5) == inv
    assert plan(rows=None) == inv and plan(rows=6 * A + 1) == inv and plan(counts=None) == inv and plan(table=None) == inv
    assert plan(lens=None) == inv and plan(cu=None) == inv and plan(slots=2) == inv and plan(pos=1) == inv
    assert plan(n=1, axes=1, sc=A, sg=A) == inv and plan(n=1, axes=3, sc=None, sg=A) == inv and plan(n=1, axes=3, sc=A, sg=A + 4) == inv
    assert plan(n=-1) == inv
    assert L.w4a8_pages_shrink(state(), 6 * A, None, 0, None) == _lib.OK
    assert L.w4a8_pages_shrink(state(), None, None, 2, None) == inv and L.w4a8_pages_shrink(state(), 6 * A, 7 * A + 2, 2, None) == inv
    assert L.w4a8_pages_shrink(None, 6 * A, None, 2, None) == inv


def test_cpu_tensors_are_refused():
    from w4a8_b200 import kvcache, ops
    i = torch.zeros(2, dtype=torch.int32)
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    for f in (lambda: ops.prepare_int8(torch.zeros(8, 64, dtype=torch.int8), torch.ones(8)), lambda: ops.quant_token(x),
              lambda: kvcache.rotary(x.view(2, 1, 64), None, torch.zeros(4, 64), i),
              lambda: kvcache.PageState.empty(4, 2, 2, 16, "cpu")):
        with pytest.raises(RuntimeError):
            f()


def test_members_without_a_bias_take_the_others_type():
    """A fused linear of which one member has a bias: zeros for the other, in fp32 and where the scales are."""
    from w4a8_b200 import vendor
    ckpt = {"a.weight": torch.ones(4, 8, dtype=torch.int8), "a.weight_scale": torch.ones(4, 1), "a.bias": torch.arange(4.0),
            "b.weight": torch.ones(2, 8, dtype=torch.int8), "b.weight_scale": torch.ones(2, 1)}
    old = torch.get_default_dtype()
    torch.set_default_dtype(torch.float64)
    try:
        got = vendor.load_int8(ckpt.__getitem__, ["b", "a"])
    finally:
        torch.set_default_dtype(old)
    assert got["bias"].dtype == torch.float32 and got["bias"].tolist() == [0, 0, 0, 1, 2, 3]
    meta = {k: t.to("meta") for k, t in ckpt.items()}
    assert vendor.load_int8(meta.__getitem__, ["a", "b"])["bias"].device.type == "meta"
