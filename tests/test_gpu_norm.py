"""Residual addition + RMS norm against 64 bits.

bf16 outputs: one rounding (2^-8 of the value at most), and 1e-5 of it for the
fp32 sum, root and products before.  8-bit outputs: the scale is bf16(amax / 127)
of the fp32 result and a code is off its definition only where x / s lies within
the fp32 error of a half-integer: |code * s - y| <= s / 2 + 127 * 2e-5 * s."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from decoder_ref import bf16_np, norm64  # noqa: E402

pytestmark = pytest.mark.gpu


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda", 0)


def _inputs(M, K, seed, residual=True, wdtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g)
    x[:, : max(1, K // 100)] *= 20
    r = (torch.randn(M, K, generator=g) * 3).to(torch.bfloat16) if residual else None
    return x.to(torch.bfloat16), r, (1 + 0.2 * torch.randn(K, generator=g)).to(wdtype)


def _close(got, want, name):
    got = bf16_np(got)
    over = np.abs(got - want) - (2.0 ** -8 + 1e-5) * np.abs(want)
    assert over.max() <= 1e-37, (name, over.max())


SHAPES = [(1, 5120), (3, 1), (2, 7), (5, 33), (17, 1057), (64, 5120), (9, 8200), (2, 27648), (1, 32768), (300, 256), (1000, 5120), (500, 1057)]


@pytest.mark.parametrize("M,K", SHAPES)
@pytest.mark.parametrize("residual,wdtype", [(True, torch.bfloat16), (False, torch.float32)])
def test_bf16_output(M, K, residual, wdtype):
    from w4a8_b200 import ops
    dev = _dev()
    x, r, w = _inputs(M, K, M + K, residual, wdtype)
    got = ops.rms_norm(x.to(dev), w.to(dev), 1e-5, residual=None if r is None else r.to(dev))
    y, h = norm64(x, r, w.double().numpy(), 1e-5)
    if residual:
        _close(got[1], h, "residual")
        assert torch.equal(got[1].cpu(), (x.float() + r.float()).to(torch.bfloat16))
        got = got[0]
    _close(got, y, "y")


@pytest.mark.parametrize("M,K,gk", [(1, 5120, 128), (4, 5120, 1024), (3, 1057, 1024), (65, 256, 64), (2, 33, 64),
                                    (7, 1000, 256), (2, 27648, 128), (5, 12288, 1024), (1, 20000, 1024),
                                    # blocks that stay for several rows; groups that end inside a warp's vectors
                                    (600, 1288, 1024), (900, 5120, 1024), (470, 1057, 1024), (700, 2120, 256),
                                    (1000, 640, 64), (460, 9000, 1024)])
@pytest.mark.parametrize("sdt", [torch.bfloat16, torch.float32])
def test_8_bit_output(M, K, gk, sdt):
    from w4a8_b200 import ops
    dev = _dev()
    x, r, w = _inputs(M, K, 3 * M + K)
    q, s, res = ops.rms_norm_quant(x.to(dev), w.to(dev), gk, 1e-6, residual=r.to(dev), scale_dtype=sdt)
    y, h = norm64(x, r, w.double().numpy(), 1e-6)
    _close(res, h, "residual")
    G = -(-K // gk)
    assert q.shape == (M, K) and s.shape == (G, M) and s.dtype == sdt
    q, s = q.cpu().numpy().astype(np.float64), s.double().cpu().numpy()
    for g in range(G):
        part = y[:, g * gk:(g + 1) * gk]
        amax = np.abs(part).max(1)
        assert (np.abs(s[g] - amax / 127) <= (2.0 ** -8 + 1e-5) * amax / 127).all()
        back = q[:, g * gk:(g + 1) * gk] * s[g][:, None]
        assert (np.abs(back - part) <= (0.5 + 127 * 2e-5) * s[g][:, None]).all()


def test_quantised_codes_are_the_quantisers():
    """Where the norm leaves its input alone exactly (unit weight, rows whose mean square is 1 and eps 0),
    codes and scales equal the activation quantiser's on the same values."""
    from w4a8_b200 import ops
    dev = _dev()
    g = torch.Generator().manual_seed(5)
    x = torch.where(torch.rand(6, 512, generator=g) < 0.5, 1.0, -1.0).to(torch.bfloat16)
    q, s, _ = ops.rms_norm_quant(x.to(dev), torch.ones(512, device=dev), 128, 0.0)
    q2, s2, _ = ops.quant_act(x.to(dev), 128)
    assert torch.equal(q, q2) and torch.equal(s, s2)


def test_special_rows():
    """A row of zeros (its scale is bf16 tiny), of huge values, with NaN and infinity."""
    from w4a8_b200 import ops
    dev = _dev()
    x, _, w = _inputs(5, 640, 9, False)
    x[0] = 0
    x[2, 3] = float("nan")
    x[3, 4] = float("inf")
    y = ops.rms_norm(x.to(dev), w.to(dev), 1e-6).float().cpu()
    assert (y[0] == 0).all() and torch.isfinite(y[1]).all() and torch.isnan(y[2]).all() and torch.isfinite(y[4]).all()
    assert torch.isnan(y[3, 4]) and (y[3, :4] == 0).all()
    q, s, _ = ops.rms_norm_quant(x.to(dev), w.to(dev), 128, 1e-6)
    assert (q[0] == 0).all() and (s[:, 0].float() == torch.finfo(torch.bfloat16).tiny).all()
    assert torch.isnan(s[:, 2].float()).all() and torch.isnan(s[0, 3].float())
    assert torch.isfinite(s[:, [1, 4]].float()).all()
    y0 = ops.rms_norm(x[:1].to(dev), w.to(dev), 0.0).float()
    assert torch.isnan(y0).all()                                  # 0 / 0, as the formula has it


def test_in_place_strides_and_leading_dimensions():
    from w4a8_b200 import ops
    dev = _dev()
    x, r, w = (t.to(dev) for t in _inputs(12, 640, 10))
    y, h = ops.rms_norm(x, w, residual=r)
    stream = r.clone()
    y2, h2 = ops.rms_norm(x, w, residual=stream, residual_out=stream)
    assert torch.equal(y, y2) and torch.equal(h, h2) and h2.data_ptr() == stream.data_ptr()
    wide = torch.zeros(12, 700, dtype=torch.bfloat16, device=dev)
    wide[:, 5:645] = x                                            # rows that are not 16-byte aligned
    assert torch.equal(ops.rms_norm(wide[:, 5:645], w, residual=r)[0], y)
    out = torch.full((12, 650), 7.0, dtype=torch.bfloat16, device=dev)
    ops.rms_norm(x, w, residual=r, out=out[:, 3:643])
    assert torch.equal(out[:, 3:643], y) and (out[:, :3] == 7).all() and (out[:, 643:] == 7).all()
    assert torch.equal(ops.rms_norm(x.t().contiguous().t(), w, residual=r)[0], y)   # transposed: copied
    y3, h3 = ops.rms_norm(x.view(3, 4, 640), w, residual=r.view(3, 4, 640))
    assert y3.shape == (3, 4, 640) and torch.equal(y3.view(12, 640), y) and torch.equal(h3.view(12, 640), h)
    assert ops.rms_norm(x[:0], w).shape == (0, 640)


@pytest.mark.parametrize("M,N,K,gk", [(1, 256, 1024, 128), (16, 512, 640, 64), (33, 256, 5120, 256), (100, 384, 1057, 1024),
                                      (200, 256, 512, 128), (600, 256, 1288, 1024)])
def test_linear_on_the_norm(M, N, K, gk):
    """The norm-fed linear equals the GEMM on rms_norm_quant's codes bit for bit (the int4-plane entry
    point takes codes as they are)."""
    from w4a8_b200 import ops
    from w4a8_b200 import synthetic as syn
    dev = _dev()
    x, r, w = (t.to(dev) for t in _inputs(M, K, 11))
    wt = syn.weight_np(N, K, gk, 12, scale_bf16=True)
    packed = ops.pack_int4_grouped(torch.from_numpy(wt.codes), gk).to(dev)
    ws = torch.from_numpy(wt.scale).to(dev)
    pw = ops.prepare_weights(packed, ws, None, K, gk)
    y, res = ops.linear_prepared_rms_norm(x, w, pw, 1e-6, residual=r)
    q, s, res2 = ops.rms_norm_quant(x, w, gk, 1e-6, residual=r)
    assert torch.equal(res, res2)
    G, kp = ops.num_groups(K, gk), ops.k_pad_elems(K, gk)
    qp = torch.zeros(M, kp, dtype=torch.int16, device=dev)
    qp[:, :K] = q.to(torch.int16)                                  # only the last group is padded
    hi, lo = qp >> 4, (qp & 0xF) ^ 0x8
    pack = lambda v: ((v[:, 0::2] & 0xF) | ((v[:, 1::2] & 0xF) << 4)).to(torch.uint8).view(torch.int8)  # noqa: E731
    want = ops.midgroup_w4a8_gemm(pack(hi), pack(lo), s, None, packed, ws.to(torch.bfloat16), None, None, K, gk)
    assert torch.equal(y, want)
    assert ops.workspace_status(dev) == 0


def test_refusals():
    from w4a8_b200 import ops
    dev = _dev()
    x, r, w = (t.to(dev) for t in _inputs(4, 64, 13))
    bad = [
        lambda: ops.rms_norm(x.float(), w),
        lambda: ops.rms_norm(x, w[:32]),
        lambda: ops.rms_norm(x, w.half()),
        lambda: ops.rms_norm(x, w, residual=r[:3]),
        lambda: ops.rms_norm(x, w, residual=r.float()),
        lambda: ops.rms_norm(x, w, residual_out=r),
        lambda: ops.rms_norm(x, w, -1.0),
        lambda: ops.rms_norm(x, w, out=torch.empty(4, 65, device=dev)),
        lambda: ops.rms_norm(torch.zeros(1, 32769, dtype=torch.bfloat16, device=dev),
                             torch.zeros(32769, dtype=torch.bfloat16, device=dev)),
        lambda: ops.rms_norm(x.cpu(), w.cpu()),
        lambda: ops.rms_norm_quant(x, w, 100),
        lambda: ops.rms_norm_quant(x, w, 128, scale_dtype=torch.float16),
    ]
    for f in bad:
        with pytest.raises(RuntimeError):
            f()


@pytest.mark.parametrize("M,K,gk", [(3, 640, 128), (3, 2120, 1024), (2, 5120, 64), (900, 5120, 1024), (700, 2120, 256),
                                    (2, 27648, 128), (3, 20000, 1024)])
def test_products_out_of_fp32_range(M, K, gk):
    """Large weights: x * weight is near or past fp32's range while the result is not.  The scale is the result's."""
    from w4a8_b200 import ops
    dev = _dev()
    x, r, _ = _inputs(M, K, 5 * M + K)
    x, r = (x.float() * 2.0 ** 40).to(torch.bfloat16), (r.float() * 2.0 ** 40).to(torch.bfloat16)
    w = 1 + 0.2 * torch.randn(K, generator=torch.Generator().manual_seed(1))
    w[7], w[K // 2], w[K - 1] = 2.0 ** 100, -2.0 ** 60, 2.0 ** 90
    q, s, _ = ops.rms_norm_quant(x.to(dev), w.to(dev), gk, 1e-6, residual=r.to(dev), scale_dtype=torch.float32)
    y, _ = norm64(x, r, w.double().numpy(), 1e-6)
    q, s = q.cpu().numpy().astype(np.float64), s.double().cpu().numpy()
    assert np.isfinite(s).all()
    for g in range(-(-K // gk)):
        part = y[:, g * gk:(g + 1) * gk]
        amax = np.abs(part).max(1)
        assert (np.abs(s[g] - amax / 127) <= (2.0 ** -8 + 1e-5) * amax / 127).all()
        back = q[:, g * gk:(g + 1) * gk] * s[g][:, None]
        assert (np.abs(back - part) <= (0.5 + 127 * 2e-5) * s[g][:, None]).all()


@pytest.mark.parametrize("K,gk", [(640, 128), (5120, 1024)])
def test_rows_whose_squares_overflow(K, gk):
    """Magnitudes past 2^64: the sum of squares is infinite and the row zero, with codes as without them."""
    from w4a8_b200 import ops
    dev = _dev()
    x, _, w = _inputs(4, K, 6, False)
    x[1] = (x[1].float() * 2.0 ** 70).to(torch.bfloat16)
    x[2] = (x[2].float() * 2.0 ** 100).to(torch.bfloat16)
    y = ops.rms_norm(x.to(dev), w.to(dev), 1e-6)
    assert (y[1:3] == 0).all() and torch.isfinite(y).all()
    q, s, _ = ops.rms_norm_quant(x.to(dev), w.to(dev), gk, 1e-6)
    assert (q[1:3] == 0).all() and (s[:, 1:3].float() == torch.finfo(torch.bfloat16).tiny).all()
    q0, s0, _ = ops.rms_norm_quant(x[[0, 3]].contiguous().to(dev), w.to(dev), gk, 1e-6)
    assert torch.equal(q[[0, 3]], q0) and torch.equal(s[:, [0, 3]], s0)


def test_linear_on_a_norm_out_of_fp32_range():
    """The operand tiles take the same codes and scales."""
    from w4a8_b200 import ops
    dev = _dev()
    M, N, K, gk = 20, 64, 1288, 1024
    x, r, w = (t.to(dev) for t in _inputs(M, K, 21, True, torch.float32))
    x, r = x * 2.0 ** 40, r * 2.0 ** 40
    w[3], w[1100] = 2.0 ** 50, -2.0 ** 52
    g = torch.Generator().manual_seed(2)
    packed = ops.pack_int4_grouped(torch.randint(-8, 8, (N, K), generator=g, dtype=torch.int8), gk).to(dev)
    ws = torch.ones(2, N, device=dev)
    y, _ = ops.linear_prepared_rms_norm(x, w, ops.prepare_weights(packed, ws, None, K, gk), 1e-6, residual=r)
    q, s, _ = ops.rms_norm_quant(x, w, gk, 1e-6, residual=r, scale_dtype=torch.float32)
    assert torch.isfinite(s).all() and torch.isfinite(y).all()
    codes = ops.unpack_int4_grouped(packed.cpu(), K, gk).double()
    q, s = q.cpu().double(), s.cpu().double()
    want = sum((q[:, a:a + gk] @ codes[:, a:a + gk].T) * s[i][:, None] for i, a in enumerate(range(0, K, gk)))
    assert ((y.cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -20 * want.abs().max()).all()
