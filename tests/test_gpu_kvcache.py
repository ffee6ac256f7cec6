"""Cache writes and reads against the definition in IEEE fp32: the same bits.

The write's arithmetic (products of the rotation rounded one by one, amax / 127,
x / scale, code * (old / new), all round-to-nearest-even) is elementary fp32, so
codes, scales, rotated queries and values read back must all be equal."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from decoder_ref import rotate32, write32  # noqa: E402

pytestmark = pytest.mark.gpu


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda", 0)


class Twin:
    """A cache on the GPU and its plain copy on the CPU, with one page table."""

    def __init__(self, hkv, d, page, caps, seed=0, spare=2):
        from w4a8_b200 import kvcache
        g = torch.Generator().manual_seed(seed)
        npages = [-(-n // page) for n in caps]
        P = sum(npages) + spare
        order, at, self.table = torch.randperm(P, generator=g).tolist(), 0, []
        for n in npages:
            self.table.append(order[at:at + n] + [-1] * (max(npages) - n))
            at += n
        self.codes = [torch.randint(-128, 128, (P, hkv, page, d), generator=g, dtype=torch.int8) for _ in range(2)]
        self.scales = [torch.full((P, hkv), float("nan")) for _ in range(2)]       # what a free page holds
        self.cache = kvcache.KVCache(*[x.to(_dev()) for x in self.codes + self.scales])
        self.g, self.hkv, self.d = g, hkv, d

    def rows(self, T, heads, big=1.0):
        return (torch.randn(T, heads, self.d, generator=self.g) * big).to(torch.bfloat16)

    def write(self, k, v, lens, qs, q=None, table=None, interleaved=False, view=None):
        from w4a8_b200 import kvcache
        dev = _dev()
        cu = np.concatenate([[0], np.cumsum(qs)]).tolist()
        i = dict(dtype=torch.int32, device=dev)
        dk, dv, dq = (None if x is None else x.to(dev) for x in (k, v, q))
        if view is not None:
            dq, dk, dv = view(dq, dk, dv)
        out = kvcache.kv_write(self.cache, dk, dv, torch.tensor(self.table, **i), torch.tensor(lens, **i),
                               torch.tensor(cu, **i), q=dq, cos_sin=None if table is None else table.to(dev),
                               interleaved=interleaved)
        pos = torch.tensor([max(L - n + j, 0) for L, n in zip(lens, qs) for j in range(n)], dtype=torch.int64)
        kf, qf = k.float(), None if q is None else q.float()
        if table is not None:
            pos = pos.clamp(max=table.shape[0] - 1)
            kf = rotate32(kf, pos, table, interleaved)
            qf = None if q is None else rotate32(qf, pos, table, interleaved)
        write32(self.codes[0], self.scales[0], kf, self.table, lens, cu)
        write32(self.codes[1], self.scales[1], v.float(), self.table, lens, cu)
        if q is not None:
            assert torch.equal(out.cpu(), qf.to(torch.bfloat16))
        self.same()

    def same(self):
        for name, mine, plain in zip(("k", "v"), (self.cache.k, self.cache.v), self.codes):
            assert torch.equal(mine.cpu(), plain), name
        for name, mine, plain in zip(("k", "v"), (self.cache.k_scale, self.cache.v_scale), self.scales):
            assert torch.equal(mine.cpu().nan_to_num(-7.0), plain.nan_to_num(-7.0)), name

    def read(self, lens, ns):
        from w4a8_b200 import kvcache
        i = dict(dtype=torch.int32, device=_dev())
        cu = np.concatenate([[0], np.cumsum(ns)]).tolist()
        got = kvcache.kv_read(self.cache, torch.tensor(self.table, **i), torch.tensor(lens, **i), torch.tensor(cu, **i),
                              cu[-1])
        page = self.codes[0].shape[2]
        for mine, codes, scales in zip(got, self.codes, self.scales):
            want = torch.zeros(cu[-1], self.hkv, self.d)
            for s, n in enumerate(ns):
                for j in range(n):
                    p = lens[s] - n + j
                    pid = self.table[s][p // page] if 0 <= p < page * len(self.table[s]) else -1
                    if 0 <= pid < codes.shape[0]:
                        want[cu[s] + j] = codes[pid, :, p % page].float() * scales[pid][:, None]
            assert torch.equal(mine.cpu(), want.to(torch.bfloat16))


def _table(rot, n):
    from w4a8_b200 import kvcache
    return kvcache.rotary_table(rot, n, base=1e4, device="cpu")


WRITES = [
    # hkv, hq, d, page, query tokens, lengths after, rot, interleaved
    (1, 5, 128, 16, [1], [1], 128, False),
    (8, 40, 128, 16, [1, 1, 1], [17, 32, 100], 128, False),
    (2, 4, 128, 32, [50, 3, 33], [50, 40, 65], 64, True),
    (3, 6, 64, 64, [200], [200], 64, False),
    (1, 1, 64, 16, [5, 0, 7], [20, 9, 7], 16, True),
    (2, 2, 128, 128, [129, 1], [300, 257], 96, False),
    (9, 9, 64, 16, [40], [47], 32, False),
]


@pytest.mark.parametrize("hkv,hq,d,page,qs,lens,rot,inter", WRITES)
def test_write_and_read(hkv, hq, d, page, qs, lens, rot, inter):
    t = Twin(hkv, d, page, lens, seed=hkv + d)
    before = [max(L - n, 0) for L, n in zip(lens, qs)]
    T0 = sum(before)
    if T0:
        t.write(t.rows(T0, hkv), t.rows(T0, hkv), before, before)
    T = sum(qs)
    t.write(t.rows(T, hkv, 1.5), t.rows(T, hkv, 0.7), lens, qs, q=t.rows(T, hq), table=_table(rot, 400),
            interleaved=inter)
    t.read(lens, lens)
    t.read(lens, [min(L, 3) for L in lens])


@pytest.mark.parametrize("page,d", [(16, 128), (32, 64)])
def test_token_by_token(page, d):
    """A page that fills one token at a time, each now and then much larger than before: scales only
    grow, earlier codes follow."""
    t = Twin(2, d, page, [45, 60], seed=1)
    t.write(t.rows(17, 2), t.rows(17, 2), [1, 16], [1, 16])
    for step in range(2, 46):
        big = 1.0 if step % 7 else 10.0 ** (step % 3)
        t.write(t.rows(2, 2, big), t.rows(2, 2, 1.0 / big), [step, step + 15], [1, 1])
    t.read([45, 60], [45, 60])


def test_special_values():
    """Zeros, one page of them in front of ordinary tokens; NaN and infinity make their page NaN and no other."""
    t = Twin(1, 64, 16, [64], seed=2)
    z = torch.zeros(8, 1, 64, dtype=torch.bfloat16)
    t.write(z, z, [8], [8])
    assert (t.scales[0][t.table[0][0]] == 0).all()
    t.write(t.rows(4, 1), t.rows(4, 1), [12], [4])
    k, v = t.rows(30, 1), t.rows(30, 1)
    k[10, 0, 5], v[12, 0, 7] = float("nan"), float("inf")        # tokens 22, 24: the second page
    t.write(k, v, [42], [30])
    assert torch.isnan(t.scales[0][t.table[0][1]]).all() and torch.isinf(t.scales[1][t.table[0][1]]).all()
    t.write(t.rows(12, 1), t.rows(12, 1), [54], [12])
    from w4a8_b200 import kvcache
    i = dict(dtype=torch.int32, device=_dev())
    kk, vv = kvcache.kv_read(t.cache, torch.tensor(t.table, **i), torch.tensor([54], **i), torch.tensor([0, 54], **i), 54)
    assert torch.isnan(kk[16:32]).all() and torch.isnan(vv[16:32]).all()
    assert torch.isfinite(kk[:16]).all() and torch.isfinite(kk[32:]).all() and torch.isfinite(vv[32:]).all()


def test_subnormal_values():
    t = Twin(1, 64, 16, [16], seed=3)
    tiny = (torch.randn(16, 1, 64) * 3e-39).to(torch.bfloat16)
    t.write(tiny, tiny, [16], [16])
    t.read([16], [16])


def test_tokens_that_are_not_written():
    """Page ids outside the cache, more tokens in the call than in the sequence."""
    t = Twin(2, 64, 16, [100, 40], seed=4)
    t.table[0][2], t.table[0][4], t.table[1][0] = -1, len(t.codes[0]), 1 << 30
    t.write(t.rows(140, 2), t.rows(140, 2), [100, 40], [100, 40])
    t.read([100, 40], [100, 40])
    t2 = Twin(1, 64, 16, [10], seed=5)
    t2.write(t2.rows(14, 1), t2.rows(14, 1), [10], [14], q=t2.rows(14, 1), table=_table(32, 64))


def test_positions_past_the_table_use_its_last_row():
    t = Twin(1, 64, 16, [40], seed=6)
    t.write(t.rows(40, 1), t.rows(40, 1), [40], [40], q=t.rows(40, 2), table=_table(64, 21))


def test_views_of_one_row_and_in_place_q():
    """q, k, v as views of one [q | k | v] tensor, as a linear returns them; q rotated in place."""
    from w4a8_b200 import kvcache
    t = Twin(2, 128, 16, [37, 20], seed=7)
    keep = {}

    def view(q, k, v):
        wide = torch.cat([q.flatten(1), k.flatten(1), v.flatten(1)], 1).contiguous()
        keep["wide"] = wide
        return wide[:, :768].unflatten(1, (6, 128)), wide[:, 768:1024].unflatten(1, (2, 128)), \
            wide[:, 1024:].unflatten(1, (2, 128))

    q = t.rows(57, 6)
    t.write(t.rows(57, 2), t.rows(57, 2), [37, 20], [37, 20], q=q, table=_table(128, 64), view=view)
    i = dict(dtype=torch.int32, device=_dev())
    wide = keep["wide"].clone()
    qv = wide[:, :768].unflatten(1, (6, 128))
    args = (torch.tensor(t.table, **i), torch.tensor([37, 20], **i), torch.tensor([0, 37, 57], **i))
    ret = kvcache.kv_write(t.cache, wide[:, 768:1024].unflatten(1, (2, 128)), wide[:, 1024:].unflatten(1, (2, 128)),
                           *args, q=qv, cos_sin=_table(128, 64).to(_dev()), q_out=qv)
    assert ret.data_ptr() == wide.data_ptr()
    pos = torch.tensor(list(range(37)) + list(range(20)))
    assert torch.equal(ret.cpu(), rotate32(q.float(), pos, _table(128, 64), False).to(torch.bfloat16))
    t.same()


def test_many_sequences():
    lens = (np.arange(700) % 37).tolist()
    qs = [min(1, L) for L in lens]
    t = Twin(1, 64, 16, [40] * 700, seed=8)
    t.write(t.rows(sum(qs), 1), t.rows(sum(qs), 1), qs, qs)


def test_cache_past_32_bits():
    from w4a8_b200 import kvcache
    dev = _dev()
    P = (1 << 31) // (8 * 16 * 128) + 8
    cache = kvcache.KVCache.empty(P, 8, 16, 128, dev)
    i = dict(dtype=torch.int32, device=dev)
    k, v = (torch.randn(20, 8, 128, device=dev).to(torch.bfloat16) for _ in range(2))
    args = (torch.tensor([[P - 1, P - 2]], **i), torch.tensor([20], **i), torch.tensor([0, 20], **i))
    kvcache.kv_write(cache, k, v, *args)
    kk, vv = kvcache.kv_read(cache, *args, 20)
    for x, y in ((k, kk), (v, vv)):
        # half a code step, amax / 254 per page and head, and one rounding to bf16
        a = torch.stack([x[:16].float().abs().amax((0, 2)), x[16:].float().abs().amax((0, 2))])
        step = torch.cat([a[:1].expand(16, 8), a[1:].expand(4, 8)])[..., None] / 254
        assert ((x.float() - y.float()).abs() <= step * 1.001 + x.float().abs() * 2.0 ** -7).all()


def test_refusals():
    from w4a8_b200 import kvcache
    dev = _dev()
    cache = kvcache.KVCache.empty(4, 2, 16, 64, dev)
    i = dict(dtype=torch.int32, device=dev)
    t, kl, cu = torch.tensor([[0, 1]], **i), torch.tensor([5], **i), torch.tensor([0, 5], **i)
    k = torch.zeros(5, 2, 64, dtype=torch.bfloat16, device=dev)
    cs = kvcache.rotary_table(64, 8)
    bad = [
        lambda: kvcache.kv_write(cache, k.float(), k, t, kl, cu),
        lambda: kvcache.kv_write(cache, k[:, :1], k[:, :1], t, kl, cu),
        lambda: kvcache.kv_write(cache, k, k[:4], t, kl, cu),
        lambda: kvcache.kv_write(cache, k, k, t, kl, cu, q=k[:4]),
        lambda: kvcache.kv_write(cache, k, k, t, kl, cu, cos_sin=cs[:, :24].contiguous()),
        lambda: kvcache.kv_write(cache, k, k, t, kl, cu, cos_sin=cs.double()),
        lambda: kvcache.kv_write(cache, k, k, t, kl, cu, cos_sin=kvcache.rotary_table(128, 8)),
        lambda: kvcache.kv_write(cache, k, k, t, kl, cu, q_out=k),
        lambda: kvcache.kv_write(cache, k, k, t[0], kl, cu),
        lambda: kvcache.kv_write(cache, k, k, t, kl, cu.cpu()),
        lambda: kvcache.kv_read(cache, t, kl, cu, -1),
        lambda: kvcache.KVCache.empty(4, 2, 24, 64, dev),
        lambda: kvcache.KVCache.empty(4, 2, 16, 80, dev),
        lambda: kvcache.KVCache(cache.k, cache.v, cache.k_scale, cache.v_scale[:3]),
        lambda: kvcache.KVCache(cache.k, cache.v.float(), cache.k_scale, cache.v_scale),
    ]
    for f in bad:
        with pytest.raises(RuntimeError):
            f()
    assert kvcache.kv_write(cache, k[:0], k[:0], t, kl, cu) is None
    assert kvcache.kv_read(cache, t, kl, cu, 0)[0].shape == (0, 2, 64)


@pytest.mark.parametrize("page,d", [(16, 64), (32, 128), (128, 128)])
def test_lengths_past_the_table(page, d):
    """Tokens past the table's last column have no page: they are not written (and what is there stays), their q is
    turned by their own position, and they read back as zeros."""
    cap = 2 * page
    t = Twin(2, d, page, [cap, cap], seed=9)
    t.write(t.rows(2 * cap - 3, 2), t.rows(2 * cap - 3, 2), [cap, cap - 3], [cap, cap - 3])
    t.write(t.rows(18, 2), t.rows(18, 2), [cap + 7, cap + 5], [10, 8], q=t.rows(18, 3), table=_table(64, cap + 20))
    t.write(t.rows(5, 2), t.rows(5, 2), [cap + 100, cap - 3], [4, 1], q=t.rows(5, 3), table=_table(64, cap + 200))
    t.read([cap + 7, cap + 5], [20, 5])
    big = 2 ** 31 - 1
    t.write(t.rows(3, 2), t.rows(3, 2), [big, cap], [3, 0], q=t.rows(3, 3), table=_table(64, cap))
    t.read([big, cap], [2, cap])
