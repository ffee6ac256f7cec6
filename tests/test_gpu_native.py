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


def test_launches_run_on_the_tensors_device(monkeypatch):
    """A call whose tensors are not on the current GPU is made with theirs current, and the other is put back."""
    from w4a8_b200 import ops
    log = []

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            log.append(("in", self.index))

        def __exit__(self, *a):
            log.append(("out", self.index))

    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(ops, "_current_index", lambda: 0)
    assert ops._launch(1, lambda *a: log.append(a) or 5, 2, 3) == 5
    assert log == [("in", 1), (2, 3), ("out", 1)]
    log.clear()
    assert ops._launch(0, lambda: log.append("here") or 0) == 0 and log == ["here"]

    def fails():
        raise RuntimeError("fails")

    log.clear()
    with pytest.raises(RuntimeError, match="fails"):
        ops._launch(1, fails)
    assert log == [("in", 1), ("out", 1)]


@pytest.mark.gpu
def test_every_wrapper_switches_to_its_tensors_device(dev, monkeypatch):
    """With another GPU said to be the current one, each call enters its tensors' device before it reaches the
    library (whose launches are then made on the only GPU here, as always)."""
    from w4a8_b200 import _lib, kvcache as kv, ops
    seen, inside = [], []

    class Device:
        def __init__(self, index):
            assert index == 0

        def __enter__(self):
            inside.append(1)

        def __exit__(self, *a):
            inside.pop()

    L = _lib.lib()

    class Library:
        def __getattr__(self, name):
            fn = getattr(L, name)
            if name.endswith("_size") or name in ("w4a8_status_string", "w4a8_last_cuda_error"):
                return fn

            def call(*a):
                seen.append((name, bool(inside)))
                return fn(*a)
            return call

    x = torch.randn(4, 512, device=dev).bfloat16()
    codes = torch.randint(-8, 8, (64, 512), dtype=torch.int8, device=dev)
    packed, ws = ops.pack_int4_grouped(codes, 128), torch.ones(4, 64, device=dev)
    w = torch.ones(512, dtype=torch.bfloat16, device=dev)
    cache = kv.KVCache.empty(4, 2, 16, 64, dev)
    i = dict(dtype=torch.int32, device=dev)
    batch = torch.tensor([[0, 1]], **i), torch.tensor([4], **i), torch.tensor([0, 4], **i)
    k = x[:, :128].contiguous().view(4, 2, 64)
    ops.workspace(32 << 20, dev)
    monkeypatch.setattr(_lib, "_N", None)
    monkeypatch.setattr(_lib, "_L", Library())
    monkeypatch.setattr(ops, "_current_index", lambda: 1)
    monkeypatch.setattr(torch.cuda, "device", Device)
    ops.quant_act(x, 128)
    ops.midgroup_quant_a(x, 128)
    ops.linear(x, packed, ws, None, 128)
    pw = ops.prepare_weights(packed, ws, None, 512, 128)
    y = ops.linear_prepared(x, pw)
    ops.linear_quant(x, 64, 128)
    ops.linear_gemm(4, 512, packed, ws, None, 128, y)
    ops.linear_gemm_prepared(4, pw, y)
    ops.group_partials(x, packed, None, 128)
    ops.rms_norm(x, w)
    ops.rms_norm_quant(x, w, 128)
    ops.linear_prepared_rms_norm(x, w, pw)
    kv.kv_write(cache, k, k, *batch, q=k)
    kv.kv_read(cache, *batch, 4)
    kv.attention(k, cache, *batch, 4)
    assert ops.workspace_status(dev) == 0
    names = [n for n, _ in seen]
    assert len(set(names)) >= 14 and {"w4a8_rms_norm", "w4a8_kv_write", "w4a8_kv_read", "w4a8_attention"} <= set(names)
    assert [n for n, ok in seen if not ok] == []


@pytest.mark.gpu
def test_refused_both_ways(dev, monkeypatch):
    """A table without rows or columns, and tokens of no sequence: refused by the short way's call as by the long one."""
    from w4a8_b200 import kvcache as kv
    cache = kv.KVCache.empty(4, 2, 16, 64, dev)
    i = dict(dtype=torch.int32, device=dev)
    t, kl, cu = torch.tensor([[0, 1]], **i), torch.tensor([5], **i), torch.tensor([0, 5], **i)
    k = torch.zeros(5, 2, 64, dtype=torch.bfloat16, device=dev)
    calls = [lambda: kv.kv_write(cache, k, k, t, kl, cu, q=k, cos_sin=torch.empty(0, 64, device=dev)),
             lambda: kv.kv_write(cache, k, k, t, kl, cu, cos_sin=torch.empty(8, 0, device=dev)),
             lambda: kv.kv_write(cache, k, k, t[:0], kl[:0], cu[:1], q=k),
             lambda: kv.kv_write(cache, k, k, t[:0], kl[:0], cu[:1])]
    for f in calls:
        with pytest.raises(RuntimeError):
            f()
        with pytest.raises(RuntimeError):
            _long(monkeypatch, f)
    assert kv.kv_write(cache, k[:0], k[:0], t[:0], kl[:0], cu[:1], q=k[:0]).shape == (0, 2, 64)
