"""What of the decoder operators needs no GPU: rotary tables, and the C entry
points' argument checks (they answer before any device work)."""
import ctypes
import math
import os

import numpy as np
import pytest

torch = pytest.importorskip("torch")


def _table(*a, **k):
    from w4a8_b200 import kvcache
    return kvcache.rotary_table(*a, device="cpu", **k).double().numpy()


def test_rotary_table_plain_and_linear():
    t = _table(64, 100, base=1e4)
    p, i = np.arange(100)[:, None], np.arange(32)[None]
    ang = p * 1e4 ** (-2.0 * i / 64)
    assert np.abs(t - np.concatenate([np.cos(ang), np.sin(ang)], 1)).max() < 1e-7
    s = _table(64, 100, base=1e4, scaling={"type": "linear", "factor": 4.0})
    assert np.abs(s[::4][:25] - t[:25]).max() < 1e-6      # position 4 p of the stretched table turns as position p


def test_rotary_table_ntk():
    f, rot = 8.0, 128
    t, s = _table(rot, 65, base=1e4), _table(rot, 65, base=1e4, scaling={"type": "ntk", "factor": f})
    assert np.abs(s[:, 0] - t[:, 0]).max() < 1e-7         # the fastest pair turns as before
    assert np.abs(np.arcsin(s[64, -1]) * f - np.arcsin(t[64, -1])) < 1e-5   # the slowest 1 / f as far


def test_rotary_table_yarn_and_llama3():
    rot, orig, f = 128, 4096, 16.0
    freq = 1e4 ** (-2.0 * np.arange(64) / rot)
    y = _table(rot, 2, base=1e4, scaling={"type": "yarn", "factor": f, "original_positions": orig})
    m = 0.1 * math.log(f) + 1
    got = np.arctan2(y[1, 64:], y[1, :64])
    assert np.abs(np.hypot(y[1, 64:], y[1, :64]) - m).max() < 1e-6
    turns = orig * freq / (2 * math.pi)
    assert np.abs(got - freq)[turns > 33].max() < 1e-6 and np.abs(got - freq / f)[turns < 0.95].max() < 1e-6
    assert ((got <= freq * (1 + 1e-6)) & (got >= freq / f * (1 - 1e-4) - 1e-9)).all()
    z = _table(rot, 2, base=1e4, scaling={"type": "llama3", "factor": f, "original_positions": orig,
                                          "low_freq_factor": 1.0, "high_freq_factor": 4.0})
    got = np.arctan2(z[1, 64:], z[1, :64])
    assert np.abs(got - freq)[turns > 4.01].max() < 1e-6 and np.abs(got - freq / f)[turns < 0.99].max() < 1e-6
    mid = (turns > 1.01) & (turns < 3.99)
    assert mid.any() and ((got < freq) & (got > freq / f))[mid].all()


def test_rotary_table_refusals():
    for a, k in [((24, 10), {}), ((0, 10), {}), ((64, 0), {}), ((64, 4), {"base": -1.0}),
                 ((64, 4), {"scaling": {"type": "other", "factor": 2.0}}),
                 ((64, 4), {"scaling": {"type": "linear", "factor": 0.5}}),
                 ((64, 4), {"scaling": {"type": "yarn", "factor": 2.0}}),
                 ((64, 4), {"scaling": {"type": "llama3", "factor": 2.0, "original_positions": 64, "low_freq_factor": 4.0,
                                        "high_freq_factor": 4.0}})]:
        with pytest.raises(RuntimeError):
            _table(*a, **k)


def _lib_or_skip():
    from w4a8_b200 import _lib
    if not os.path.exists(_lib.lib_path()):
        pytest.skip("libw4a8_b200.so not built")
    return _lib, _lib.lib()


A = 1 << 20       # 1024-byte aligned fake device addresses, never read: every call below is refused first


def test_norm_argument_contract():
    _lib, L = _lib_or_skip()
    inv, uns = _lib.ERR_INVALID, _lib.ERR_UNSUPPORTED

    def call(x=A, M=4, K=64, ldx=64, r=None, ldr=0, ro=None, ldro=0, w=2 * A, wd=0, eps=1e-6, y=3 * A, ldy=64):
        return L.w4a8_rms_norm(x, M, K, ldx, r, ldr, ro, ldro, w, wd, eps, y, ldy, None)

    assert call(M=0) == _lib.OK
    assert call(M=-1) == inv and call(K=0) == inv and call(K=_lib.NORM_MAX_K + 1) == uns
    assert call(x=None) == inv and call(ldx=63) == inv and call(x=A + 1) == inv
    assert call(w=None) == inv and call(wd=2) == uns and call(wd=1, w=2 * A + 2) == inv
    assert call(r=A, ldr=63) == inv and call(r=A, ldr=64, ro=A, ldro=5) == inv
    assert call(eps=-1.0) == inv and call(eps=float("nan")) == inv
    assert call(y=None) == inv and call(ldy=63) == inv

    def quant(gk=128, q=3 * A, s=4 * A, sd=0):
        return L.w4a8_rms_norm_quant(A, 4, 64, 64, None, 0, None, 0, 2 * A, 0, 1e-6, gk, q, s, sd, None)

    assert quant(gk=32) == uns and quant(q=None) == inv and quant(s=None) == inv and quant(sd=3) == uns

    def lin(N=64, gk=128, prepared=4 * A, ws=None, nws=0):
        return L.w4a8_linear_prepared_rms_norm(A, 4, 256, 256, None, 0, None, 0, 2 * A, 0, 1e-6, N, gk, prepared, 0, 0,
                                               5 * A, 64, ws, nws, None)

    assert lin(N=12) == inv and lin(gk=3) == uns and lin(prepared=4 * A + 16) == inv
    assert lin() in (_lib.ERR_CUDA, _lib.ERR_DEVICE, _lib.ERR_WORKSPACE)


def test_cache_argument_contract():
    _lib, L = _lib_or_skip()
    inv, uns = _lib.ERR_INVALID, _lib.ERR_UNSUPPORTED

    def desc(k=A, v=2 * A, ks=3 * A, vs=4 * A, pages=8, heads=2, page=16, d=64):
        return ctypes.byref(_lib.KvCacheDesc(k, v, ks, vs, pages, heads, page, d, 0))

    def write(c=None, table=5 * A, ld=4, cols=4, kl=6 * A, cu=7 * A, B=2, T=6, k=8 * A, ldk=128, v=9 * A, ldv=128,
              q=10 * A, ldq=256, hq=4, qo=11 * A, ldqo=256, cs=12 * A, rows=10, rot=64):
        return L.w4a8_kv_write(c or desc(), table, ld, cols, kl, cu, B, T, k, ldk, v, ldv, q, ldq, hq, qo, ldqo, cs,
                               rows, rot, 0, None)

    assert write(B=0) == _lib.OK and write(T=0) == _lib.OK
    assert write(desc(d=80)) == uns and write(desc(page=8)) == uns and write(desc(heads=0)) == inv
    assert write(desc(k=None)) == inv and write(desc(k=A + 8)) == inv and write(desc(pages=-1)) == inv
    assert write(desc(pages=0)) == inv
    assert write(B=-1) == inv and write(T=-1) == inv and write(ld=3) == inv and write(cols=1 << 30, ld=1 << 30) == inv
    assert write(table=None) == inv and write(kl=None) == inv and write(cu=7 * A + 2) == inv
    assert write(k=None) == inv and write(k=8 * A + 2) == inv and write(ldk=120) == inv and write(ldv=132) == inv
    assert write(ldq=248) == inv and write(qo=None) == inv and write(hq=0) == inv
    assert write(rot=24) == uns and write(rot=128) == uns and write(rows=0) == inv and write(cs=12 * A + 4) == inv

    def read(c=None, T=6, k=8 * A, v=9 * A):
        return L.w4a8_kv_read(c or desc(), 5 * A, 4, 4, 6 * A, 7 * A, 2, T, k, v, None)

    assert read(T=0) == _lib.OK and read(T=-1) == inv and read(k=None) == inv and read(v=9 * A + 2) == inv

    def attend(c=None, B=2, T=6, q=8 * A, ldq=256, hq=4, mq=3, scale=0.1, out=9 * A, ldo=256, ws=None, nws=0):
        return L.w4a8_attention(c or desc(), 5 * A, 4, 4, 6 * A, 7 * A, B, T, q, ldq, hq, mq, scale, out, ldo, ws, nws,
                                None)

    assert attend(T=0) == _lib.OK and attend(hq=3) == inv and attend(hq=0) == inv and attend(mq=0) == inv
    assert attend(scale=float("nan")) == inv and attend(scale=-0.1) == inv and attend(B=_lib.ATTENTION_MAX_BATCH + 1) == uns
    assert attend(q=None) == inv and attend(ldo=255) == inv and attend(out=9 * A + 2) == inv
    assert attend() in (_lib.ERR_CUDA, _lib.ERR_DEVICE, _lib.ERR_WORKSPACE)
    assert L.w4a8_attention_workspace_size(2, 6, 4, 2, 64, 3) > 0
    assert L.w4a8_attention_workspace_size(2, 6, 3, 2, 64, 3) == 0
    assert L.w4a8_attention_workspace_size(2, 6, 4, 2, 80, 3) == 0


def test_cpu_tensors_are_refused():
    from w4a8_b200 import kvcache, ops
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        ops.rms_norm(x, torch.ones(64, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError):
        kvcache.KVCache.empty(2, 1, 16, 64, "cpu")


def test_cache_table_past_64_bits_is_refused():
    """Columns whose tokens do not fit 32 bits, however many: their product with the page size must not wrap."""
    _lib, L = _lib_or_skip()
    c = ctypes.byref(_lib.KvCacheDesc(A, 2 * A, 3 * A, 4 * A, 8, 2, 16, 64, 0))
    for cols in (1 << 27, 1 << 30, 1 << 60, (1 << 60) + 4, (1 << 63) - 1):
        assert L.w4a8_kv_read(c, 5 * A, cols, cols, 6 * A, 7 * A, 2, 0, None, None, None) == _lib.ERR_INVALID, cols
        assert L.w4a8_attention(c, 5 * A, cols, cols, 6 * A, 7 * A, 2, 0, None, 256, 4, 3, 0.1, None, 256, None, 0,
                                None) == _lib.ERR_INVALID, cols
    assert L.w4a8_kv_read(c, 5 * A, 4, 4, 6 * A, 7 * A, 2, 0, None, None, None) == _lib.OK
