"""Linears in 8-bit integers.

Codes, scales and the product are elementary IEEE fp32 around exact integer sums (amax / 127, x / s
rounded half-even, float(sum) * s * ws + b, one rounding to bf16), so they are held bit for bit against
the same arithmetic on 64-bit integer sums.

Behind SwiGLU or a norm the row h itself is only known up to fp32 rounding, 2^-20 of a value here (a sum of
squares of K <= 8192 in trees of at most 8 + 10 + 5 additions, division, root, two products; exp and
a division for SwiGLU, which then rounds to bf16: where 64 bits put silu(g) u within 2^-18 of a
tie between two bf16 values both are right).  A code may then differ by one where h / s is
within 127.5 * 2^-18 of a half-integer (scale and value each off by 2^-20, doubled).  Let D be the sum
of |w| s ws over the row's such elements: y may be off by D (1 + 2^-6), by the fp32 roundings, 2^-20 of the
sum of |q w| s ws + |b|, and by half a step of bf16, 2^-8 of y.
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda", 0)


def codes32(h):
    """(codes, scale) of fp32 rows by the definition, on their device."""
    amax = h.abs().amax(1, keepdim=True)
    s = amax / torch.full_like(amax, 127.0)
    q = torch.where(s > 0, (h / s).round(), torch.zeros((), device=h.device)).clamp(-127, 127)
    return q.nan_to_num(0).to(torch.int8), s[:, 0]


def sums64(q, w):
    """Exact integer sums, in 64-bit floating point (all of them below 2^53)."""
    return q.double() @ w.double().T


def product32(acc, s, ws, b):
    y = acc.float() * s[:, None] * ws[None]          # (acc is an integer below 2^31: rounded once)
    return (y if b is None else y + b[None]).to(BF)


def _layer(N, K, g, bias=True, dev=None):
    from w4a8_b200 import ops
    w = torch.randint(-128, 128, (N, K), generator=g, dtype=torch.int8).to(dev)
    ws = (torch.rand(N, generator=g) * 0.01 + 1e-4).to(dev)
    b = torch.randn(N, generator=g).to(dev) if bias else None
    return w, ws, b, ops.prepare_int8(w, ws, b)


@pytest.mark.parametrize("M,K", [(1, 1), (3, 7), (5, 1057), (2, 5120), (300, 256), (4, 8200), (3, 20000), (2, 40001),
                                 (300, 9000), (400, 27648), (1000, 8192), (300, 65536), (70, 70000), (297, 20001),
                                 (300, 1029), (310, 9004), (2, 8)])
def test_codes(M, K):
    from w4a8_b200 import ops
    dev = _dev()
    g = torch.Generator().manual_seed(M * K)
    x = torch.randn(M, K, generator=g)
    x[:, ::97] *= 50.0
    x = x.to(BF).to(dev)
    q, s = ops.quant_token(x)
    q2, s2 = codes32(x.float().cpu())
    assert torch.equal(s.cpu(), s2) and torch.equal(q.cpu(), q2)
    wide = torch.empty(M, K + 5, dtype=BF, device=dev)
    wide[:, 3:K + 3] = x                                        # rows that begin at odd addresses
    qw, sw = ops.quant_token(wide[:, 3:K + 3])
    assert torch.equal(q, qw) and torch.equal(s, sw)


def test_codes_at_ties_and_edges():
    """Half-integer quotients, zeros, subnormal scales, values that are not finite."""
    from w4a8_b200 import ops
    dev = _dev()
    rows = [torch.arange(256) / 2 - 64, torch.zeros(256), torch.full((256,), 2.0 ** -133), torch.arange(256) * 2.0 ** -133,
            torch.full((256,), 3.0e38), torch.randn(256) * 1e-38]
    rows[0][0] = 127.0                                          # scale 1: every other quotient a tie
    x = torch.stack(rows).to(BF)
    q, s = ops.quant_token(x.to(dev))
    q2, s2 = codes32(x.float())
    assert torch.equal(s.cpu(), s2) and torch.equal(q.cpu(), q2)
    for bad in (float("nan"), float("inf"), -float("inf")):
        y = x.clone()
        y[0, 77], y[5, 0] = bad, bad
        q, s = ops.quant_token(y.to(dev))
        assert torch.isnan(s[[0, 5]]).all() and (q[[0, 5]] == 0).all()
        assert torch.equal(s[1:5].cpu(), s2[1:5]) and torch.equal(q[1:5].cpu(), q2[1:5])


GEMMS = [(M, N, K) for M, N, K in [
    (1, 1, 1), (1, 7168, 5120), (2, 127, 100), (16, 128, 128), (17, 129, 1057), (5, 300, 16), (16, 5120, 2000),
    (33, 2056, 129), (64, 640, 4096), (65, 1000, 333), (100, 8, 5120), (128, 256, 640), (3, 40001, 256), (40, 39000, 130),
    (129, 128, 128), (256, 256, 256), (257, 300, 1057), (333, 2056, 1057), (130, 1, 17), (700, 4099, 257),
    (2500, 1030, 300), (5000, 2049, 130)]]


@pytest.mark.parametrize("M,N,K", GEMMS)
def test_product(M, N, K):
    from w4a8_b200 import ops
    dev = _dev()
    g = torch.Generator().manual_seed(M + N + K)
    w, ws, b, layer = _layer(N, K, g, bias=(M + N) % 2 == 0, dev=dev)
    q = torch.randint(-128, 128, (M, K), generator=g, dtype=torch.int8).to(dev)
    s = (torch.rand(M, generator=g) * 0.02).to(dev)
    y = ops.gemm_int8(q, s, layer)
    assert ops.workspace_status(dev) == 0
    want = product32(sums64(q, w), s, ws, b)
    assert torch.equal(y, want)
    assert torch.equal(ops.gemm_int8(q, s, layer), y)


def test_the_largest_sums():
    """Every product 2^14 over the longest row: the 32-bit sum holds it."""
    from w4a8_b200 import _lib, ops
    dev = _dev()
    K = _lib.INT8_MAX_K
    for M in (2, 130):
        w = torch.full((3, K), -128, dtype=torch.int8, device=dev)
        w[1] = 127
        q = torch.full((M, K), -128, dtype=torch.int8, device=dev)
        one = torch.ones(M, device=dev)
        y = ops.gemm_int8(q, one, ops.prepare_int8(w, torch.ones(3, device=dev)))
        assert torch.equal(y, product32(sums64(q, w), one, torch.ones(3, device=dev), None))
    x = torch.ones(2, K, dtype=BF, device=dev)
    y = ops.linear_int8(x, ops.prepare_int8(w, torch.ones(3, device=dev)))
    qq, s = codes32(x.float())
    assert torch.equal(y, product32(sums64(qq, w), s, torch.ones(3, device=dev), None))


@pytest.mark.parametrize("M,N,K", [(1, 7168, 5120), (19, 1000, 1057), (64, 640, 256), (300, 513, 2048), (2, 3, 1)])
def test_linear(M, N, K):
    from w4a8_b200 import ops
    dev = _dev()
    g = torch.Generator().manual_seed(7 * M + N)
    w, ws, b, layer = _layer(N, K, g, dev=dev)
    x = torch.randn(M, K, generator=g).to(BF).to(dev)
    x[M // 2] = 0
    y = ops.linear_int8(x, layer)
    q, s = codes32(x.float())
    want = product32(sums64(q, w), s, ws, b)
    assert torch.equal(y, want)
    # leading dimensions, strided rows, a caller's output with longer and odd rows
    wide = torch.randn(M, K + 9, device=dev).to(BF)
    wide[:, 2:K + 2] = x
    out = torch.full((M, N + 3), 7.0, dtype=BF, device=dev)
    got = ops.linear_int8(wide[:, 2:K + 2], layer, out=out[:, 1:N + 1])
    assert got.data_ptr() == out[:, 1:].data_ptr() and torch.equal(got, want)
    assert (out[:, 0] == 7).all() and (out[:, N + 1:] == 7).all()
    assert torch.equal(ops.linear_int8(x.view(1, M, K), layer), want.view(1, M, N))
    x[0, 0] = float("inf")
    y = ops.linear_int8(x, layer)
    assert torch.isnan(y[0]).all() and torch.equal(y[1:], want[1:])


def _near(y, h, w, ws, b, tied=None):
    """y against the 64-bit rows h, by the bound above; ``tied``: elements whose bf16 value may be its neighbour."""
    amax = h.abs().amax(1, keepdim=True)
    s = (amax / 127).float().double()
    safe = torch.where(s == 0, torch.ones_like(s), s)
    z = h / safe
    q = torch.where(s == 0, torch.zeros_like(z), z.round().clamp(-127, 127))
    flips = ((z - z.floor() - 0.5).abs() < 127.5 * 2.0 ** -18).double()
    if tied is not None:                                     # the neighbour is 2^-7 of the value away
        flips = torch.maximum(flips, tied.double() * (1 + (z.abs() * 2.0 ** -7).ceil()))
    wf, c = w.double(), (s * ws.double()[None])
    acc, mag, d = q @ wf.T, q.abs() @ wf.abs().T, flips @ wf.abs().T
    want = acc * c + (0 if b is None else b.double()[None])
    bound = d * c * (1 + 2.0 ** -6) + (mag * c + (0 if b is None else b.double().abs()[None])) * 2.0 ** -19 + want.abs() * 2.0 ** -8
    assert ((y.double() - want).abs() <= bound + 1e-30).all()


@pytest.mark.parametrize("M,N,K", [(1, 512, 5120), (33, 130, 1057), (200, 640, 768), (16, 300, 27648), (2, 64, 40000), (300, 40, 9600),
                                   (310, 24, 5120), (2, 8, 70000), (300, 16, 9001), (310, 8, 1029), (40, 8, 9004), (7, 8, 9)])
def test_swiglu(M, N, K):
    from w4a8_b200 import ops
    dev = _dev()
    g = torch.Generator().manual_seed(M * 3 + K)
    w, ws, b, layer = _layer(N, K, g, dev=dev)
    gu = (torch.randn(M, 2 * K, generator=g) * 2).to(BF).to(dev)
    y = ops.linear_int8(gu, layer, act="swiglu")
    gate, up = gu.double().chunk(2, 1)
    a = gate * torch.sigmoid(gate) * up
    r = a.to(BF).double()
    lo, hi = (a * (1 - 2.0 ** -18)).to(BF), (a * (1 + 2.0 ** -18)).to(BF)
    _near(y, r, w, ws, b, tied=lo != hi)
    q, s = ops.quant_token(gu, act="swiglu")
    assert torch.equal(ops.gemm_int8(q, s, layer), y)


@pytest.mark.parametrize("M,N,K,res,f32", [(1, 512, 5120, True, False), (64, 300, 1057, True, True), (200, 256, 8192, False, False),
                                           (5, 640, 64, True, False), (3, 16, 32768, True, False), (300, 24, 9600, True, True),
                                           (320, 16, 27648, False, False), (297, 8, 32768, True, False), (400, 40, 768, True, False),
                                           (300, 16, 9001, True, False), (40, 16, 9003, True, True), (300, 8, 1029, True, False),
                                           (5, 8, 20006, True, False), (700, 8, 13, True, False)])
def test_behind_a_norm(M, N, K, res, f32):
    from w4a8_b200 import ops
    dev = _dev()
    g = torch.Generator().manual_seed(M * 5 + K)
    w, ws, b, layer = _layer(N, K, g, dev=dev)
    x = torch.randn(M, K, generator=g).to(BF).to(dev)
    r = (torch.randn(M, K, generator=g) * 3).to(BF).to(dev) if res else None
    nw = (1 + 0.2 * torch.randn(K, generator=g)).to(torch.float32 if f32 else BF).to(dev)
    got = ops.linear_int8_rms_norm(x, nw, layer, 1e-6, residual=r)
    y, ro = got if res else (got, None)
    h = x.double() + (r.double() if res else 0)
    if res:
        assert torch.equal(ro, h.to(BF))                     # (x + r is exact in 64 bits)
    _near(y, h / (h.square().mean(1, keepdim=True) + 1e-6).sqrt() * nw.double(), w, ws, b)
    if res:                                                  # in place of the residual
        keep = r.clone()
        y2, r2 = ops.linear_int8_rms_norm(x, nw, layer, 1e-6, residual=keep, residual_out=keep)
        assert r2.data_ptr() == keep.data_ptr() and torch.equal(keep, ro) and torch.equal(y2, y)


def test_captured_and_on_another_stream():
    from w4a8_b200 import ops
    dev = _dev()
    g = torch.Generator().manual_seed(1)
    w1, s1, b1, up = _layer(768, 512, g, dev=dev)
    w2, s2, b2, down = _layer(512, 384, g, dev=dev)
    xs = [torch.randn(M, 512, generator=g).to(BF).to(dev) for M in (3, 3, 3)]
    ops.linear_int8(torch.zeros(300, 512, dtype=BF, device=dev), up)          # the workspace
    plain = [ops.linear_int8(ops.linear_int8(x, up), down, act="swiglu") for x in xs]
    hold = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.linear_int8(ops.linear_int8(hold, up), down, act="swiglu")
    for x, want in zip(xs, plain):
        hold.copy_(x)
        graph.replay()
        assert torch.equal(out, want)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        y = ops.linear_int8(ops.linear_int8(xs[1], up), down, act="swiglu")
    side.synchronize()
    assert torch.equal(y, plain[1]) and ops.workspace_status(dev) == 0


def test_a_chain_without_waits():
    """Calls one after another on one workspace, few and many tokens: each reads its own codes, and weights
    that the call before it has just written."""
    from w4a8_b200 import ops
    dev = _dev()
    g = torch.Generator().manual_seed(2)
    layers = [_layer(N, K, g, dev=dev) for N, K in ((1024, 640), (640, 1024), (4096, 640))]
    xs = {(M, i): torch.randn(M, layers[i][3].K, generator=g).to(BF).to(dev) for M in (1, 40, 300) for i in range(3)}
    alone = {}
    for key, x in xs.items():
        alone[key] = ops.linear_int8(x, layers[key[1]][3])
        torch.cuda.synchronize()
    for _ in range(20):
        got = {key: ops.linear_int8(x, layers[key[1]][3]) for key, x in xs.items()}
        for key, y in got.items():
            assert torch.equal(y, alone[key])
    w, ws, b, layer = layers[0]
    for i in range(10):
        layer.w.copy_(torch.roll(w, i, 0) if i else w)
        y = ops.linear_int8(xs[1, 0], layer)
        q, s = codes32(xs[1, 0].float())
        assert torch.equal(y, product32(sums64(q, layer.w), s, ws, b))


def test_refusals():
    from w4a8_b200 import ops
    dev = _dev()
    w, ws = torch.zeros(8, 32, dtype=torch.int8, device=dev), torch.ones(8, device=dev)
    layer = ops.prepare_int8(w, ws)
    x = torch.zeros(4, 32, dtype=BF, device=dev)
    q, s = ops.quant_token(x)
    norm = torch.ones(32, dtype=BF, device=dev)
    bad = [
        lambda: ops.prepare_int8(w.float(), ws), lambda: ops.prepare_int8(w[0], ws), lambda: ops.prepare_int8(w, ws[:7]),
        lambda: ops.prepare_int8(w, ws.double()), lambda: ops.prepare_int8(w, ws, ws[:1]), lambda: ops.prepare_int8(w[:0], ws[:0]),
        lambda: ops.prepare_int8(w, ws.cpu()), lambda: ops.prepare_int8(w.cpu(), ws.cpu()),
        lambda: ops.prepare_int8(torch.zeros(1, 131072, dtype=torch.int8, device=dev), ws[:1]),
        lambda: ops.linear_int8(x.float(), layer), lambda: ops.linear_int8(x[:, :31], layer), lambda: ops.linear_int8(x.cpu(), layer),
        lambda: ops.linear_int8(x, layer, act="gelu"), lambda: ops.linear_int8(x, layer, act="swiglu"),
        lambda: ops.linear_int8(x, layer, out=torch.zeros(4, 8, device=dev)),
        lambda: ops.linear_int8(x, layer, out=torch.zeros(3, 8, dtype=BF, device=dev)),
        lambda: ops.linear_int8_rms_norm(x, norm[:31], layer), lambda: ops.linear_int8_rms_norm(x, norm, layer, residual=x[:3]),
        lambda: ops.linear_int8_rms_norm(x, norm, layer, residual_out=x),
        lambda: ops.linear_int8_rms_norm(torch.zeros(4, 16, dtype=BF, device=dev), norm[:16], layer),
        lambda: ops.linear_int8_rms_norm(x, norm, layer, eps=-1.0),
        lambda: ops.gemm_int8(q.float(), s, layer), lambda: ops.gemm_int8(q[:, :16], s, layer), lambda: ops.gemm_int8(q, s[:3], layer),
        lambda: ops.gemm_int8(q, s.double(), layer), lambda: ops.quant_token(x.float()), lambda: ops.quant_token(x[0]),
        lambda: ops.quant_token(x[:, :0]), lambda: ops.quant_token(x[:, :31], act="swiglu"),
    ]
    for f in bad:
        with pytest.raises(RuntimeError):
            f()
    assert ops.linear_int8(x[:0], layer).shape == (0, 8) and ops.gemm_int8(q[:0], s[:0], layer).shape == (0, 8)
    assert [t.shape for t in ops.linear_int8_rms_norm(x[:0], norm, layer, residual=x[:0])] == [(0, 8), (0, 32)]
    assert ops.quant_token(x[:0])[0].shape == (0, 32)


_FIRST = """
import sys, torch
sys.path.insert(0, sys.argv[1])
from w4a8_b200 import ops
dev = torch.device("cuda", 0)
ops.workspace(32 << 20, dev)
g = torch.Generator().manual_seed(3)
for M, N, K in ((3, 640, 4096), (40, 1280, 5120), (300, 512, 2048), (20, 64, 20000)):
    layer = ops.prepare_int8(torch.randint(-128, 128, (N, K), generator=g, dtype=torch.int8).to(dev), torch.rand(N, generator=g).to(dev))
    x = torch.randn(M, K, generator=g).bfloat16().to(dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.linear_int8(x, layer)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, ops.linear_int8(x, layer)), (M, N, K)
assert ops.workspace_status(dev) == 0
print("same")
"""


def test_captured_before_any_other_call():
    """The first call of a process inside a capture: kernels are loaded and their residency asked for there."""
    import os
    import subprocess
    import sys
    _dev()
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vllm-ascend910_b200")
    r = subprocess.run([sys.executable, "-c", _FIRST, root], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]


def _threads(*works):
    """Each work in a thread of its own; what any of them raised is raised here."""
    import threading
    wrong = []

    def run(f):
        try:
            f()
        except BaseException as e:                           # noqa: BLE001
            wrong.append(e)
    ts = [threading.Thread(target=run, args=(f,)) for f in works]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    if wrong:
        raise wrong[0]


def test_threads():
    """Calls of two threads, each in stream order on one workspace under the other's lock, as the rule asks."""
    import threading
    from w4a8_b200 import ops
    dev = _dev()
    g = torch.Generator().manual_seed(4)
    layers = [_layer(N, 512, g, dev=dev)[3] for N in (300, 700)]
    xs = [torch.randn(M, 512, generator=g).to(BF).to(dev) for M in (5, 200)]
    want = [ops.linear_int8(x, L) for x, L in zip(xs, layers)]
    lock = threading.Lock()

    def work(i):
        for _ in range(50):
            with lock:
                y = ops.linear_int8(xs[i], layers[i])
            assert torch.equal(y, want[i])
    _threads(lambda: work(0), lambda: work(1))


@pytest.mark.parametrize("M", [5, 200])
def test_a_threads_first_call(M):
    """The product alone as the first CUDA call of a thread, which has no context yet."""
    from w4a8_b200 import ops
    dev = _dev()
    g = torch.Generator().manual_seed(5)
    w, ws, b, layer = _layer(300, 512, g, dev=dev)
    q = torch.randint(-127, 128, (M, 512), generator=g, dtype=torch.int8).to(dev)
    s = torch.rand(M, generator=g).to(dev)
    out = torch.empty(M, 300, dtype=BF, device=dev)
    torch.cuda.synchronize()
    _threads(lambda: ops.gemm_int8(q, s, layer, out=out))
    torch.cuda.synchronize()
    assert torch.equal(out, product32(sums64(q, w), s, ws, b))


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(70_000, 32_768, 40), (128, 96, 72), (300, 96, 72)])
def test_offsets_past_32_bits(M, N, K):
    """More than 2^31 output elements, and rows of x, the residual and the output whose offsets pass 2^31 elements: rows are
    those of a call on them alone."""
    from w4a8_b200 import ops
    dev = torch.device("cuda", 0)
    if torch.cuda.mem_get_info(dev)[0] < 48 << 30:
        pytest.skip("needs 48 GB")
    g = torch.Generator(device=dev).manual_seed(M)
    layer = ops.prepare_int8(torch.randint(-128, 128, (N, K), generator=g, device=dev, dtype=torch.int8),
                             torch.rand(N, generator=g, device=dev), torch.rand(N, generator=g, device=dev))
    x, r = (torch.randn(M, K, generator=g, device=dev).to(BF) for _ in range(2))
    w = torch.rand(K, generator=g, device=dev).to(BF)
    if M == 70_000:
        y = ops.linear_int8(x, layer)
        for at in (0, 35_000, M - 200):
            assert torch.equal(y[at:at + 200], ops.linear_int8(x[at:at + 200], layer))
        return
    far = 2 ** 31 // (M - 1) // 8 * 8 + 1024                    # elements from row to row
    assert (M - 1) * far > 2 ** 31
    wide = [torch.empty(M * far, dtype=BF, device=dev).as_strided((M, n), (far, 1)) for n in (K, K, N)]
    wide[0].copy_(x), wide[1].copy_(r)
    want, sums = ops.linear_int8_rms_norm(x, w, layer, 1e-6, residual=r)
    got, ro = ops.linear_int8_rms_norm(wide[0], w, layer, 1e-6, residual=wide[1], out=wide[2])
    assert torch.equal(got, want) and torch.equal(ro, sums)
    assert torch.equal(ops.linear_int8(wide[0], layer, out=wide[2]), ops.linear_int8(x, layer))
    for one, two in zip(ops.quant_token(wide[0]), ops.quant_token(x)):
        assert torch.equal(one, two)


@pytest.mark.parametrize("M", [1, 5, 200])
def test_layers_of_one_channel(M):
    """Weights [1, K] whose row stride is not K: torch calls them contiguous whatever it is."""
    from w4a8_b200 import ops
    dev = _dev()
    g = torch.Generator().manual_seed(M)
    big = torch.randint(-128, 128, (8, 40), generator=g, dtype=torch.int8).to(dev)
    col = torch.randint(-128, 128, (32, 1), generator=g, dtype=torch.int8).to(dev)
    ws, b = torch.rand(1, generator=g).to(dev), torch.rand(1, generator=g).to(dev)
    x = torch.randn(M, 32, generator=g).to(BF).to(dev)
    q, s = codes32(x.float())
    for w in (big[2:3, :32], big[1:2, :32], col.T, big[0].as_strided((1, 32), (1 << 41, 1))):
        layer = ops.prepare_int8(w, ws, b)
        want = product32(sums64(q, w), s, ws, b)
        assert torch.equal(ops.linear_int8(x, layer), want) and torch.equal(ops.gemm_int8(q, s, layer), want)


# gates of a row, about: from where sigma(g) leaves fp32's normal numbers (-87.3) and e^-g all of them (-88.7), to where no up
# brings the product back into bf16's range
FAR = [-60, -80, -86, -87, -88, -90, -100, -120, -150, -165, -170, -300]


@pytest.mark.parametrize("M,K", [(12, 64), (12, 1057), (12, 27648), (320, 2048), (300, 9000), (300, 5003), (12, 70000)])
def test_gates_far_below_zero(M, K):
    """silu(g) up where sigma(g) is tiny and up large: the element is the product's, not the sigmoid's, to lose.

    A row's scale is exact: its largest element is 2^e out of a gate of 64, whose sigmoid rounds to 1.  The others lie
    within [2^e / 8, 0.9 2^e].  fp32 gives them within 2^-18 (four equal factors of two units in the last place each,
    four products), so that their bf16 value is the 64-bit one except within 2^-18 of a tie, where it may be its neighbour,
    2^-7 of the value or at most one code away; the codes of equal values are equal."""
    from w4a8_b200 import ops
    dev = _dev()
    g = torch.Generator().manual_seed(M + K)
    base = torch.tensor(FAR, dtype=torch.float64).repeat(-(-M // len(FAR)))[:M, None]
    gate = (base + 6 * torch.rand(M, K, generator=g, dtype=torch.float64) - 3).to(BF).double()
    silu = gate * torch.sigmoid(gate)
    e = ((base * torch.sigmoid(base)).abs().log2().floor() + 118).clamp(max=0)
    e = torch.where(base < -200, torch.zeros_like(e), e)
    target = 2.0 ** e * (0.125 + 0.775 * torch.rand(M, K, generator=g, dtype=torch.float64)) * torch.sign(torch.randn(M, K, generator=g))
    up = torch.where(base < -200, torch.full_like(target, 3e38), target / torch.where(silu == 0, torch.ones_like(silu), silu)).to(BF)
    at = K // 3
    gate[:, at] = 64.0
    up[:, at] = (2.0 ** (e[:, 0] - 6)).to(BF)
    assert torch.isfinite(up).all()
    a = gate * torch.sigmoid(gate) * up.double()
    assert torch.equal(a[:, at].to(BF).double(), 2.0 ** e[:, 0])
    r = a.to(BF)
    lo, hi = (a * (1 - 2.0 ** -18)).to(BF), (a * (1 + 2.0 ** -18)).to(BF)
    x = torch.cat([gate.to(BF), up], 1).to(dev)
    q, s = ops.quant_token(x, act="swiglu")
    q2, s2 = codes32(r.float())
    assert torch.equal(s.cpu(), s2)
    far = (q.cpu().int() - q2.int()).abs()
    assert (far[lo == hi] == 0).all() and far.max() <= 1 and (q2[base[:, 0] > -200] != 0).all()
    layer = _layer(8, K, g, dev=dev)[3]
    assert torch.equal(ops.linear_int8(x, layer, act="swiglu"), ops.gemm_int8(q, s, layer))


@pytest.mark.parametrize("gate,up", [(float("nan"), 1.0), (-90.0, float("nan")), (-90.0, float("inf")), (-float("inf"), 1.0),
                                     (-float("inf"), 0.0), (float("inf"), 1.0), (-1e30, float("inf"))])
def test_gates_that_are_not_finite(gate, up):
    """A gate or up without a value leaves its row without one and the others as they are; -inf's is the formula's
    -inf / (1 + e^inf), 0 times infinity."""
    from w4a8_b200 import ops
    dev = _dev()
    x = torch.randn(3, 80, generator=torch.Generator().manual_seed(3)).to(BF)
    want = ops.quant_token(x.to(dev), act="swiglu")
    x[1, 7], x[1, 47] = gate, up
    q, s = ops.quant_token(x.to(dev), act="swiglu")
    assert torch.isnan(s[1]) and (q[1] == 0).all()
    assert torch.equal(q[[0, 2]], want[0][[0, 2]]) and torch.equal(s[[0, 2]], want[1][[0, 2]])
    x[1, 7], x[1, 47] = -1e30, 3e38                             # finite and nothing left: as a zero
    q, s = ops.quant_token(x.to(dev), act="swiglu")
    x[1, 7], x[1, 47] = 0.0, 0.0
    q2, s2 = ops.quant_token(x.to(dev), act="swiglu")
    assert torch.equal(q, q2) and torch.equal(s, s2)


# Shapes that take every form of the product on a GPU of 148 SMs, ragged in every direction: the kernel, its tile of
# tokens (few) or channels (many), and how many CTAs, or pairs of them, cut a tile's K.
FORMS = [(("few", tt, split), (M, N, K)) for M, tt in ((5, 16), (20, 32), (50, 64), (100, 128))
         for split, N, K in ((1, 301, 500), (2, 8001, 1100), (3, 6001, 1101), (4, 4002, 1100), (6, 2501, 1700), (8, 2003, 2100))] + [
    (("many", 128, 1), (131, 101, 201)), (("many", 128, 2), (140, 103, 1101)), (("many", 128, 3), (131, 2401, 3001)),
    (("many", 128, 4), (257, 102, 3001)), (("many", 256, 1), (300, 5001, 201)), (("many", 256, 2), (131, 6401, 10001)),
    (("many", 256, 3), (200, 4803, 6007)), (("many", 256, 4), (140, 3201, 27650))]


@pytest.mark.parametrize("form,shape", FORMS)
def test_every_form_of_the_product(form, shape):
    from w4a8_b200 import ops
    dev = _dev()
    M, N, K = shape
    g = torch.Generator().manual_seed(M + N + K)
    w, ws, b, layer = _layer(N, K, g, bias=M % 2 == 0, dev=dev)
    q = torch.randint(-128, 128, (M, K), generator=g, dtype=torch.int8).to(dev)
    s = (torch.rand(M, generator=g) * 0.02).to(dev)
    want = product32(sums64(q, w), s, ws, b)
    assert torch.equal(ops.gemm_int8(q, s, layer), want)
    # rows that suit the widest stores, and what lies beside the output
    wide = torch.full((M + 2, -(-N // 16) * 16 + 16), 7.0, dtype=BF, device=dev)
    ops.gemm_int8(q, s, layer, out=wide[1:M + 1, :N])
    assert torch.equal(wide[1:M + 1, :N], want) and (wide[[0, -1]] == 7).all() and (wide[:, N:] == 7).all()
    assert ops.workspace_status(dev) == 0


def test_the_shapes_take_every_form():
    """The plans of the list above, by the names of the kernels that ran."""
    import re
    from torch.profiler import ProfilerActivity, profile
    from w4a8_b200 import ops
    dev = _dev()
    if torch.cuda.get_device_properties(dev).multi_processor_count != 148:
        pytest.skip("the list is for 148 SMs")
    taken = []
    for _, (M, N, K) in FORMS:
        layer = ops.prepare_int8(torch.zeros(N, K, dtype=torch.int8, device=dev), torch.ones(N, device=dev))
        q, s = torch.zeros(M, K, dtype=torch.int8, device=dev), torch.ones(M, device=dev)
        torch.cuda.synchronize()
        with profile(activities=[ProfilerActivity.CUDA]) as p:
            ops.gemm_int8(q, s, layer)
            torch.cuda.synchronize()
        names = [re.search(r"int8_(few|many)_kernel<(\d+), (\d+)>", e.name) for e in p.events()]
        taken.append([(m[1], int(m[2]), int(m[3])) for m in names if m])
    if not any(taken):
        pytest.skip("no kernel names on this machine")
    # (the last needs 13 clusters of eight at a time, which not every set of 148 SMs may hold)
    assert taken[:-1] == [[form] for form, _ in FORMS[:-1]] and taken[-1] in ([("many", 256, 4)], [("many", 128, 2)])
