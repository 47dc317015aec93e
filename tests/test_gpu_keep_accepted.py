"""GPU parity: the accepted nodes' cache rows after a verification, against the oracle's moves (16-bit caches: bit for bit;
fp8 caches: the bytes of torch's own conversion, one 32-bit product in front of it)."""
import random

import pytest
import torch

from oracle import speculative as osp

pytestmark = pytest.mark.gpu


class Case:
    def __init__(self, dev, nodes, ctx, *, L=2, H=2, d=64, chunk=16, dtype=torch.bfloat16, fp8=False, seed=0, paths=None):
        rng, gen = random.Random(seed), torch.Generator().manual_seed(seed)
        self.lens = [n + c for n, c in zip(nodes, ctx)]
        self.cu = [0]
        for n in nodes:
            self.cu.append(self.cu[-1] + n)
        need = [-(-n // chunk) for n in self.lens]
        self.N = sum(need) + 2
        ids = torch.randperm(self.N, generator=gen).tolist()
        self.table = torch.full((len(nodes), max(need + [1])), -1, dtype=torch.int32)
        for r, k in enumerate(need):
            self.table[r, :k] = torch.tensor([ids.pop() for _ in range(k)], dtype=torch.int32)
        if paths is None:
            paths = [[0] + sorted(rng.sample(range(1, n), rng.randint(0, n - 1))) if n else [] for n in nodes]
        most = max([len(p) for p in paths] + [1])
        self.rows = torch.full((len(nodes), most + 1), -1, dtype=torch.int32)
        for r, p in enumerate(paths):
            self.rows[r, :len(p)] = torch.tensor([self.cu[r] + i for i in p], dtype=torch.int32)
        self.counts = [len(p) for p in paths]
        shape = (L, self.N, chunk, H, d)
        self.scales = None
        if fp8:
            self.k, self.v = ((torch.randn(shape, generator=gen) * 100).clamp(-448, 448).to(torch.float8_e4m3fn) for _ in "kv")
            self.scales = [0.004 + 0.01 * torch.rand(L, self.N, H, generator=gen) for _ in "kv"]
        else:
            self.k, self.v = (torch.randn(shape, generator=gen).to(dtype) for _ in "kv")
        self.dev = dev

    def rest(self):
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=self.dev)  # noqa: E731
        return self.rows.to(self.dev), i32(self.counts), i32(self.cu), i32(self.lens), self.table.to(self.dev)

    def check(self, mi, k=None, v=None):
        raw = lambda x: x.view(torch.uint8) if self.scales else x  # noqa: E731
        k, v = raw(self.k).to(self.dev) if k is None else k, raw(self.v).to(self.dev) if v is None else v
        scales = dict(k_scales=self.scales[0].to(self.dev), v_scales=self.scales[1].to(self.dev)) if self.scales else {}
        new = mi.ops.kv_keep_accepted(k, v, *self.rest(), **scales)
        torch.cuda.synchronize()
        assert new.dtype == torch.int32
        assert new.tolist() == [n - (b - a) + c for n, a, b, c in zip(self.lens, self.cu, self.cu[1:], self.counts)]
        for got, cache, s in ((k, self.k, 0), (v, self.v, 1)):
            want = osp.keep_accepted(cache.float() if self.scales else cache, self.rows, self.counts, self.cu, self.lens, self.table,
                                     self.scales[s] if self.scales else None)
            got = got.cpu().view(torch.float8_e4m3fn).float() if self.scales else got.cpu()
            assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,d,chunk", [(2, 64, 16), (8, 128, 256), (1, 64, 1), (3, 96, 48), (1, 576, 64), (16, 256, 32), (1, 8, 5)])
def test_layouts(mi, dev, dtype, H, d, chunk):
    Case(dev, [9, 1, 30, 0, 5], [20, 0, 100, 7, 31], H=H, d=d, chunk=chunk, dtype=dtype, seed=d + chunk).check(mi)


@pytest.mark.parametrize("H,d,chunk", [(2, 64, 16), (8, 128, 256), (4, 128, 7), (1, 64, 64)])
def test_fp8_caches(mi, dev, H, d, chunk):
    Case(dev, [9, 1, 30, 0, 5], [20, 0, 100, 7, 31], H=H, d=d, chunk=chunk, fp8=True, seed=d + chunk).check(mi)


def test_long_paths_and_their_overlaps(mi, dev):
    """Places that lie on nodes moved before them, more of them than a thread holds and than lie in LDS at a time."""
    n = 200
    for shift in (1, 2, 7, 9):
        Case(dev, [n], [13], paths=[[0] + list(range(1 + shift, n))], seed=shift).check(mi)
    Case(dev, [n, n], [13, 0], paths=[[0] + list(range(2, n, 2)), list(range(n))], seed=30).check(mi)


def test_a_chain_moves_nothing(mi, dev):
    Case(dev, [6, 6], [20, 3], paths=[[0, 1, 2], [0, 1, 2, 3, 4, 5]], seed=31).check(mi)


def test_one_layer_and_strided_layers(mi, dev):
    c = Case(dev, [9, 12], [20, 40], L=1, seed=32)
    k, v = c.k[0].to(dev), c.v[0].to(dev)
    mi.ops.kv_keep_accepted(k, v, *c.rest())
    torch.cuda.synchronize()
    assert torch.equal(k.cpu(), osp.keep_accepted(c.k, c.rows, c.counts, c.cu, c.lens, c.table)[0])
    c = Case(dev, [9, 12], [20, 40], L=3, seed=33)
    pool = torch.stack([c.k, c.v]).to(dev)                    # [2, layers, ...]: the context's buffer
    c.check(mi, pool[0], pool[1])
    wide = torch.zeros(3, c.N, 16, 2, 2, 64, dtype=torch.bfloat16, device=dev)   # tokens with a gap between them
    wide[:, :, :, 0] = c.k.to(dev)
    wide[:, :, :, 1] = c.v.to(dev)
    c.check(mi, wide[:, :, :, 0], wide[:, :, :, 1])


def test_a_cache_with_one_tensor(mi, dev):
    c = Case(dev, [9, 12], [20, 40], H=1, d=576, chunk=64, seed=34)
    k = c.k.to(dev)
    mi.ops.kv_keep_accepted(k, None, *c.rest())
    torch.cuda.synchronize()
    assert torch.equal(k.cpu(), osp.keep_accepted(c.k, c.rows, c.counts, c.cu, c.lens, c.table))


def test_entries_that_are_none(mi, dev):
    """Rows of other requests, places outside the table, chunks outside the cache: nothing moves there."""
    c = Case(dev, [9, 9, 9], [20, 14, 40], seed=35, paths=[[0, 2, 4, 8], [0, 3, 5], [0, 4, 6, 7]])
    c.rows[0, 2], c.rows[1, 1], c.rows[2, 3] = 17, -5, 1 << 30
    c.table[2, 2] = c.N
    c.lens[1] = 400
    c.check(mi)


def test_replays(mi, dev):
    c = Case(dev, [9, 12], [20, 40], seed=36)
    k, v, rest = c.k.to(dev), c.v.to(dev), c.rest()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        new = mi.ops.kv_keep_accepted(k, v, *rest)
    a, b = c.k.to(dev), c.v.to(dev)
    for _ in range(3):
        graph.replay()
        again = mi.ops.kv_keep_accepted(a, b, *rest)
        torch.cuda.synchronize()
        assert torch.equal(k, a) and torch.equal(v, b) and torch.equal(new, again)


def test_refusals(mi, dev):
    c = Case(dev, [5], [20], seed=37)
    k, v = c.k.to(dev), c.v.to(dev)
    rows, counts, cu, lens, table = c.rest()
    call = lambda **x: mi.ops.kv_keep_accepted(*{**dict(k=k, v=v, rows=rows, counts=counts, cu=cu, lens=lens, t=table), **x}.values())  # noqa: E731
    for change, word in ((dict(v=v[:, :, :8]), "differ"), (dict(k=k.float(), v=v.float()), "16-bit"), (dict(rows=rows.long()), "rows"),
                         (dict(counts=counts.long()), "counts"), (dict(lens=lens.cpu()), "one device"), (dict(k=k.view(torch.uint8), v=v.view(torch.uint8)), "scales"),
                         (dict(k=k[0, 0], v=v[0, 0]), "caches must be"), (dict(k=k[..., :32], v=v[..., :32]), "contiguous")):
        with pytest.raises(ValueError, match=word):
            call(**change)


@pytest.mark.parametrize("code", [0x7f, 0xff])
def test_nan_stays_nan(mi, dev, code):
    """A NaN of an fp8 cache is one wherever its row goes; the values beside it are converted as ever."""
    c = Case(dev, [9, 1, 30, 0, 5], [20, 0, 100, 7, 31], H=2, d=64, chunk=16, fp8=True, seed=40)
    for x in (c.k, c.v):
        x.view(torch.uint8)[:, :, :, 0, ::5] = code
        x.view(torch.uint8)[:, :, ::3, 1, 7] = code
    k, v = c.k.view(torch.uint8).to(dev), c.v.view(torch.uint8).to(dev)
    mi.ops.kv_keep_accepted(k, v, *c.rest(), k_scales=c.scales[0].to(dev), v_scales=c.scales[1].to(dev))
    torch.cuda.synchronize()
    for got, cache, s in ((k, c.k, 0), (v, c.v, 1)):
        want = osp.keep_accepted(cache.float(), c.rows, c.counts, c.cu, c.lens, c.table, c.scales[s])
        got = got.cpu().view(torch.float8_e4m3fn).float()
        assert want.isnan().any() and torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.nan_to_num(0), want.nan_to_num(0))


def test_scales_that_make_no_number(mi, dev):
    """Scales of zero, infinity and NaN on either side: the quotient's rules, value by value (0 * inf and NaN are NaN)."""
    c = Case(dev, [9, 1, 30, 0, 5], [20, 0, 100, 7, 31], H=2, d=64, chunk=16, fp8=True, seed=41)
    for x in (c.k, c.v):
        x.view(torch.uint8)[..., ::9] = 0
    for s in c.scales:
        s[:, 0::5], s[:, 1::7], s[:, 2::9] = 0, float("inf"), float("nan")
    k, v = c.k.view(torch.uint8).to(dev), c.v.view(torch.uint8).to(dev)
    mi.ops.kv_keep_accepted(k, v, *c.rest(), k_scales=c.scales[0].to(dev), v_scales=c.scales[1].to(dev))
    torch.cuda.synchronize()
    for got, cache, s in ((k, c.k, 0), (v, c.v, 1)):
        want = osp.keep_accepted(cache.float(), c.rows, c.counts, c.cu, c.lens, c.table, c.scales[s])
        got = got.cpu().view(torch.float8_e4m3fn).float()
        assert want.isnan().any() and torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.nan_to_num(0), want.nan_to_num(0))
