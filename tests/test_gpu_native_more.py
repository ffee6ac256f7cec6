"""The short way into the 8-bit linears, rotary positions and pages: the long way's results, and its refusals."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_native import _N, _long, _same  # noqa: E402

BF, I = torch.bfloat16, torch.int32


@pytest.fixture
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda", 0)


def test_declines_what_it_does_not_know():
    N = _N()
    x, i = torch.zeros(4, 8, dtype=BF), torch.zeros(4, dtype=I)
    assert N.linear_int8(0, 0, x, 0, 0, 0) is NotImplemented and N.linear_int8(*[None] * 6) is NotImplemented
    assert N.linear_int8_rms_norm(x, x[0], None, 1e-6, 0, 0, 0) is NotImplemented and N.linear_int8_rms_norm() is NotImplemented
    assert N.rotary(x, None, x, i, 1, 4, 0, False) is NotImplemented and N.rotary(*[None] * 8) is NotImplemented
    assert N.pages_plan(0, 0, i, i, 4, 1, None, None) is NotImplemented and N.pages_plan(*[None] * 8) is NotImplemented
    assert N.pages_shrink(0, 0, i, None) is NotImplemented and N.pages_shrink(*[None] * 4) is NotImplemented
    with pytest.raises(TypeError):
        N.bind_more(1)
    with pytest.raises(ValueError):
        N.bind_more(0, 0, 0, 0, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 512), (3, 40), (2, 3, 264), (0, 64), (64,)])
@pytest.mark.parametrize("act", [None, "swiglu"])
def test_linears(dev, monkeypatch, shape, act):
    from w4a8_b200 import ops
    N = _N()
    K = shape[-1] // (2 if act else 1)
    g = torch.Generator(device=dev).manual_seed(1)
    layer = ops.prepare_int8(torch.randint(-128, 128, (24, K), generator=g, device=dev, dtype=torch.int8),
                             torch.rand(24, generator=g, device=dev), torch.rand(24, generator=g, device=dev))
    x = torch.randn(shape, generator=g, device=dev).to(BF)
    ops.linear_int8(torch.zeros(300, shape[-1], dtype=BF, device=dev), layer, act=act)
    if x.numel():
        assert N.linear_int8(layer._ref, 0, x, 1 if act else 0, *ops.workspace(0, dev)) is not NotImplemented
    assert N.linear_int8(layer._ref, 0, x, 1 if act else 0, 0, 0) is NotImplemented           # no workspace
    assert N.linear_int8(layer._ref, 0, x[..., 1:], 0, *ops.workspace(0, dev)) is NotImplemented
    _same(ops.linear_int8(x, layer, act=act), _long(monkeypatch, lambda: ops.linear_int8(x, layer, act=act)))
    if act or len(shape) == 1:
        return
    w, r = torch.rand(K, device=dev).to(BF), torch.randn(shape, generator=g, device=dev).to(BF)
    for res in (None, r, r.transpose(0, -1).contiguous().transpose(0, -1)):
        f = lambda: ops.linear_int8_rms_norm(x, w, layer, 1e-6, residual=res)             # noqa: E731,B023
        _same(f(), _long(monkeypatch, f))
    with pytest.raises(RuntimeError):
        ops.linear_int8_rms_norm(x, w, layer, -1.0)


@pytest.mark.gpu
def test_rotary(dev, monkeypatch):
    from w4a8_b200 import kvcache
    _N()
    axes, table = kvcache.RotaryAxes([24, 20, 20], mixed=True), kvcache.rotary_table(128, 40)
    x = torch.randn(7, 8 * 128, device=dev).to(BF)
    q, k = x[:, :512].unflatten(1, (4, 128)), x[:, 512:768].unflatten(1, (2, 128))
    pos = torch.randint(0, 40, (3, 7), device=dev, dtype=I)
    for a in ((q, k, table, pos), (q, None, table, pos), (q.contiguous(), k, table, pos), (q, k, table, pos.T.contiguous().T),
              (q[:0], k[:0], table, pos[:, :0])):
        for inter in (False, True):
            f = lambda: kvcache.rotary(*a, axes, interleaved=inter)                       # noqa: E731,B023
            _same(f(), _long(monkeypatch, f))
    for bad in ((q, k[:6], table, pos), (q, k, table[:, :64].contiguous(), pos), (q, k, table, pos[:2]), (q.float(), k, table, pos)):
        with pytest.raises(RuntimeError):
            kvcache.rotary(*bad, axes)


@pytest.mark.gpu
def test_pages(dev, monkeypatch):
    from w4a8_b200 import kvcache
    _N()
    i = dict(dtype=I, device=dev)
    states = [kvcache.PageState.empty(40, 5, 9, 16, dev) for _ in range(2)]
    rows, counts = torch.tensor([4, 0, 2], **i), torch.tensor([20, 1, 0], **i)
    images = (torch.tensor([0, 1, 1, 2], **i), torch.tensor([[2, 1, 3, 4], [0, 2, 2, 2]], **i))
    for axes, im in ((1, None), (3, images), (2, None)):
        got = kvcache.pages_plan(states[0], rows, counts, 25, axes=axes, images=im)
        want = _long(monkeypatch, lambda: kvcache.pages_plan(states[1], rows, counts, 25, axes=axes, images=im))   # noqa: B023
        assert isinstance(got, kvcache.StepMaps)
        _same(tuple(got), tuple(want))
    for keep in (torch.tensor([3, 1, 0], **i), None):
        kvcache.pages_shrink(states[0], rows, keep)
        _long(monkeypatch, lambda: kvcache.pages_shrink(states[1], rows, keep))           # noqa: B023
    for a, b in zip((states[0].table, states[0].lens, states[0].free, states[0].free_pages),
                    (states[1].table, states[1].lens, states[1].free, states[1].free_pages)):
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError):
        kvcache.pages_plan(states[0], rows, counts, 25, axes=1, images=images)
    with pytest.raises(RuntimeError):
        kvcache.pages_shrink(states[0], rows, counts[:2])
    assert states[0].status() == 0


@pytest.mark.gpu
def test_another_gpu_current(dev, monkeypatch):
    """With another GPU current the short way declines and the wrappers make the tensors' one current."""
    from w4a8_b200 import kvcache, ops
    seen = []
    real = torch.cuda.device

    class Device(real):
        def __init__(self, index):
            seen.append(index)
            super().__init__(index)
    layer = ops.prepare_int8(torch.ones(8, 16, dtype=torch.int8, device=dev), torch.ones(8, device=dev))
    x = torch.ones(2, 16, dtype=BF, device=dev)
    st = kvcache.PageState.empty(4, 2, 2, 16, dev)
    r = torch.zeros(1, dtype=I, device=dev)
    table, axes = kvcache.rotary_table(16, 4), kvcache.RotaryAxes([8])
    want = ops.linear_int8(x, layer)
    from w4a8_b200 import _lib
    with monkeypatch.context() as m:
        m.setattr(_lib, "_N", None)
        m.setattr(ops, "_current_index", lambda: 1)
        m.setattr(torch.cuda, "device", Device)
        assert torch.equal(ops.linear_int8(x, layer), want)
        ops.linear_int8_rms_norm(x, x[0], layer)
        ops.gemm_int8(*ops.quant_token(x), layer)
        kvcache.rotary(x.view(2, 1, 16), None, table, torch.zeros(1, 2, dtype=I, device=dev), axes)
        kvcache.pages_plan(st, r, r + 1, 1)
        kvcache.pages_shrink(st, r)
    assert seen == [0] * 7 and st.status() == 0


@pytest.mark.gpu
def test_images_need_three_axes_even_without_a_grid(dev, monkeypatch):
    from w4a8_b200 import kvcache
    _N()
    st = kvcache.PageState.empty(8, 2, 4, 16, dev)
    rows, counts = torch.arange(2, dtype=I, device=dev), torch.ones(2, dtype=I, device=dev)
    none = (torch.zeros(3, dtype=I, device=dev), torch.zeros(0, 4, dtype=I, device=dev))
    f = lambda: kvcache.pages_plan(st, rows, counts, 2, axes=1, images=none)              # noqa: E731
    for call in (lambda: _long(monkeypatch, f), f):
        with pytest.raises(RuntimeError, match="3 axes"):
            call()
    assert not st.lens.any() and st.status() == 0
    assert kvcache.pages_plan(st, rows, counts, 2, axes=3, images=none).positions.tolist() == [[0, 0]] * 3
