"""The short way into the small operators' C entry points: it answers the dense common
case, with the results of the long way, and hands everything else over to it."""
import pytest

torch = pytest.importorskip("torch")


def _N():
    from w4a8_b200 import _lib
    N = _lib.native()
    assert N is not None, "w4a8_b200/_native.so was not built"
    return N


def test_declines_what_it_does_not_know():
    N = _N()
    x, w = torch.zeros(4, 8, dtype=torch.bfloat16), torch.ones(8, dtype=torch.bfloat16)
    assert N.rms_norm(x, w, None, 1e-6) is NotImplemented          # no CUDA tensor
    assert N.rms_norm(x, w) is NotImplemented
    assert N.rms_norm(1, None, "r", []) is NotImplemented
    assert N.rms_norm_quant(x, w, None, 1e-6, 1024, torch.float16) is NotImplemented
    assert N.kv_write(*[None] * 10) is NotImplemented
    assert N.kv_read(0, 0, x, x, x, 4) is NotImplemented
    assert N.attention(0, 0, x, x, x, x, 1, 1.0, 0, 0) is NotImplemented
    with pytest.raises(TypeError):
        N.bind(1)
    with pytest.raises(ValueError):
        N.bind(0, 0, 0, 0, 0)


@pytest.fixture
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda", 0)


def _long(monkeypatch, call):
    from w4a8_b200 import _lib
    with monkeypatch.context() as m:
        m.setattr(_lib, "_N", None)
        return call()


def _same(a, b):
    a, b = (t if isinstance(t, tuple) else (t,) for t in (a, b))
    assert len(a) == len(b)
    for s, t in zip(a, b):
        assert (s is None) == (t is None)
        if s is not None:
            assert s.dtype == t.dtype and s.shape == t.shape and torch.equal(s, t)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 5120), (3, 7), (2, 3, 264), (0, 64)])
@pytest.mark.parametrize("wdtype", [torch.bfloat16, torch.float32])
def test_norms(dev, monkeypatch, shape, wdtype):
    from w4a8_b200 import ops
    N = _N()
    g = torch.Generator(device=dev).manual_seed(1)
    x, r = (torch.randn(shape, generator=g, device=dev).bfloat16() for _ in range(2))
    w = torch.randn(shape[-1], generator=g, device=dev).to(wdtype)
    for res in (None, r):
        got = N.rms_norm(x, w, res, 1e-6)
        assert got is not NotImplemented
        _same(got, _long(monkeypatch, lambda: ops.rms_norm(x, w, 1e-6, res)))
        if len(shape) == 2:
            for sd in (torch.bfloat16, torch.float32):
                got = N.rms_norm_quant(x, w, res, 1e-6, 64, sd)
                assert got is not NotImplemented
                _same(got, _long(monkeypatch, lambda: ops.rms_norm_quant(x, w, 64, 1e-6, res, scale_dtype=sd)))
    assert N.rms_norm(x[..., ::2], w[::2], None, 1e-6) is NotImplemented
    assert N.rms_norm(x, w[:-1], None, 1e-6) is NotImplemented
    assert N.rms_norm(x.float(), w, None, 1e-6) is NotImplemented
    assert N.rms_norm(x, w, r[..., :-1], 1e-6) is NotImplemented


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_cache_and_attention(dev, monkeypatch, interleaved):
    from w4a8_b200 import kvcache as kv, ops
    N = _N()
    hq, h, d, lens, qs = 10, 2, 64, [37, 1, 90], [5, 1, 33]
    g = torch.Generator(device=dev).manual_seed(2)
    T = sum(qs)
    x = torch.randn((T, (hq + 2 * h) * d), generator=g, device=dev).bfloat16()
    q, k, v = (t.unflatten(1, (-1, d)) for t in x.split([hq * d, h * d, h * d], 1))
    table = torch.arange(18, dtype=torch.int32, device=dev).flip(0).view(3, 6).contiguous()
    kl = torch.tensor(lens, dtype=torch.int32, device=dev)
    cu = torch.tensor([0, 5, 6, 39], dtype=torch.int32, device=dev)
    cs = kv.rotary_table(32, 128, device=dev)
    caches = []
    for _ in range(2):
        c = kv.KVCache.empty(20, h, 16, d, device=dev)
        for t in (c.k, c.v, c.k_scale, c.v_scale):
            t.zero_()
        caches.append(c)
    a, b = caches

    def short(c, **kw):
        return N.kv_write(c._ref, c._index, table, kl, cu, k, v, kw.get("q"), kw.get("cs"), interleaved)

    got = short(a, q=q, cs=cs)
    assert got is not NotImplemented
    _same(got, _long(monkeypatch, lambda: kv.kv_write(b, k, v, table, kl, cu, q, cs, interleaved)))
    assert short(a) is None
    assert _long(monkeypatch, lambda: kv.kv_write(b, k, v, table, kl, cu, None, None, interleaved)) is None
    for s, t in ((a.k, b.k), (a.v, b.v), (a.k_scale, b.k_scale), (a.v_scale, b.v_scale)):
        _same(s, t)
    _same(N.kv_read(a._ref, a._index, table, kl, cu, T), _long(monkeypatch, lambda: kv.kv_read(b, table, kl, cu, T)))
    want = _long(monkeypatch, lambda: kv.attention(got, b, table, kl, cu, 33, 0.2))
    ws = ops.workspace(0, dev)
    _same(N.attention(a._ref, a._index, table, kl, cu, got, 33, 0.2, *ws), want)
    assert N.attention(a._ref, a._index, table, kl, cu, got, 33, 0.2, ws[0], 0) is NotImplemented   # too small
    assert N.attention(a._ref, a._index, table.long(), kl, cu, got, 33, 0.2, *ws) is NotImplemented
    assert N.attention(a._ref, a._index, table, kl, cu[:-1], got, 33, 0.2, *ws) is NotImplemented
    assert N.attention(a._ref, a._index, table, kl, cu, got.float(), 33, 0.2, *ws) is NotImplemented
    assert N.attention(a._ref, a._index, table, kl, cu, got, 33, -1.0, *ws) is NotImplemented
