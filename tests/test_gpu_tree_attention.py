"""GPU parity: attention of drafted tokens over the paged cache against the 64-bit oracle.

Tolerance, element by element, with u half a step of the 16-bit type and A = sum p |v|: the probabilities are rounded once
(each by at most u, in the numerator and in the row sum: 2 u A), the result once (u |o|), scores are 32-bit sums of exact
products and the exponentials of 32-bit hardware precision: 2^-24 times a score of at most some 30 and a few roundings, 2e-5 A.
"""
import math
import random

import pytest
import torch

from oracle import speculative as osp

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def _trees(nodes, shape, rng):
    if shape == "chain":
        return [list(range(-1, n - 1)) for n in nodes]
    return [([-1] + [rng.randint(max(0, i - 9), i - 1) for i in range(1, n)])[:n] for n in nodes]


class Case:
    def __init__(self, dev, nodes, ctx, *, Hq=8, Hkv=2, d=128, chunk=64, dtype=BF16, fp8=False, shape="tree", seed=0, bits=None,
                 spare=0, words=None, spread=1.0):
        rng, gen = random.Random(seed), torch.Generator().manual_seed(seed)
        self.lens = [n + c for n, c in zip(nodes, ctx)]
        self.cu = [0]
        for n in nodes:
            self.cu.append(self.cu[-1] + n)
        T = self.cu[-1]
        self.bits = sum((osp.ancestors(t) for t in _trees(nodes, shape, rng)), []) if bits is None else bits
        need = [-(-max(n, 0) // chunk) for n in self.lens]
        self.N = sum(need) + 2
        ids = torch.randperm(self.N, generator=gen).tolist()
        self.table = torch.zeros(len(nodes), max(max(need), 1) + 1, dtype=torch.int32)
        for r, k in enumerate(need):
            self.table[r, :k] = torch.tensor([ids.pop() for _ in range(k)], dtype=torch.int32)
        self.q = (torch.randn(T + spare, Hq, d, generator=gen) * spread).to(dtype)
        shape4 = (self.N, chunk, Hkv, d)
        self.scales = None
        if fp8:
            self.k, self.v = ((torch.randn(shape4, generator=gen) * 100).clamp(-448, 448).to(torch.float8_e4m3fn) for _ in "kv")
            self.scales = [0.004 + 0.01 * torch.rand(self.N, Hkv, generator=gen) for _ in "kv"]
        else:
            self.k, self.v = (torch.randn(shape4, generator=gen).to(dtype) for _ in "kv")
        self.words = words or max(1, -(-max(max(nodes), 1) // 64))
        self.mask = osp.mask_rows(self.bits + [0] * spare, self.words)
        self.dev, self.scale, self.dtype = dev, d ** -0.5, dtype

    def run(self, mi, q=None, out=None, mask=None, **more):
        dev = self.dev
        cache = [x.view(torch.uint8) if self.scales else x for x in (self.k, self.v)]
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
        scales = dict(k_scales=self.scales[0].to(dev), v_scales=self.scales[1].to(dev)) if self.scales else {}
        return mi.ops.paged_tree_attention(
            self.q.to(dev) if q is None else q, cache[0].to(dev), cache[1].to(dev), i32(self.cu), i32(self.lens), self.table.to(dev),
            self.mask.to(dev) if mask is None else mask, softmax_scale=self.scale, out=out, **scales, **more)

    def reference(self):
        k, v = (x.float() if self.scales else x for x in (self.k, self.v))
        return osp.tree_attention(self.q[:self.cu[-1]], k, v, self.cu, self.lens, self.table, self.bits, self.scale,
                                  *(self.scales or ()))

    def check(self, mi, got=None, **more):
        got = self.run(mi, **more) if got is None else got
        torch.cuda.synchronize()
        got, (ref, size) = got.cpu().double().view(-1, *self.q.shape[1:]), self.reference()
        u = torch.finfo(self.dtype).eps / 2
        assert (got[self.cu[-1]:] == 0).all(), "rows behind the last request"
        got = got[:self.cu[-1]]
        assert torch.equal(got.isnan(), ref.isnan()), "NaN"
        fine = torch.isfinite(ref)
        assert torch.equal(got[~fine & ~ref.isnan()], ref[~fine & ~ref.isnan()])
        err = (got - ref).abs()[fine]
        bound = ((2 * u + 2e-5) * size * (1 + u) + u * ref.abs() + 1e-7)[fine]
        assert (err <= bound).all(), f"max err / bound {(err / bound).max():.3f}"
        return got


@pytest.mark.parametrize("nodes,ctx", [
    ([1], [0]), ([1], [1]), ([2], [0]), ([5], [777]), ([5, 1, 8], [64, 63, 65]), ([16, 17, 3], [0, 15, 16]), ([13], [47]),
    ([64], [130]), ([40, 7, 22, 1], [300, 5, 0, 999]),
])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_sizes(mi, dev, nodes, ctx, dtype):
    Case(dev, nodes, ctx, dtype=dtype, seed=sum(nodes)).check(mi)


@pytest.mark.parametrize("Hq,Hkv,d", [(8, 8, 64), (32, 8, 128), (7, 1, 96), (12, 4, 192), (16, 2, 256), (64, 1, 64), (28, 4, 128),
                                      (5, 5, 128), (24, 3, 96), (11, 11, 64), (16, 16, 128)])
def test_head_layouts(mi, dev, Hq, Hkv, d):
    Case(dev, [9, 21, 1], [100, 33, 250], Hq=Hq, Hkv=Hkv, d=d, seed=d + Hq).check(mi)


@pytest.mark.parametrize("chunk", [16, 48, 32, 80, 64, 256])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_chunk_sizes(mi, dev, chunk, d):
    Case(dev, [11, 30], [chunk - 5, 3 * chunk + 1], d=d, chunk=chunk, seed=chunk).check(mi)


@pytest.mark.parametrize("d,chunk,dtype", [(64, 64, BF16), (64, 16, FP16), (64, 32, BF16), (128, 256, FP16), (128, 48, BF16), (128, 32, FP16)])
def test_fp8_caches(mi, dev, d, chunk, dtype):
    Case(dev, [12, 1, 33], [270, 64, 511], Hq=16, Hkv=4, d=d, chunk=chunk, dtype=dtype, fp8=True, seed=d + chunk).check(mi)


def test_fp8_scales_of_every_size_and_sign(mi, dev):
    """Small scales (a probability times one is subnormal in fp16), a large one, a negative one and zeros."""
    for dtype in (BF16, FP16):
        c = Case(dev, [6, 9], [500, 130], Hq=8, Hkv=2, chunk=64, dtype=dtype, fp8=True, seed=5)
        for s in c.scales:
            s[0::4] *= 1e-4
            s[1::4] *= -1
            s[2::8] = 0
        c.check(mi)


@pytest.mark.parametrize("nodes", [65, 128, 200, 256])
def test_masks_of_several_words(mi, dev, nodes):
    Case(dev, [nodes, 3], [70, 10], Hq=4, Hkv=2, d=64, seed=nodes).check(mi)


def test_any_bits(mi, dev):
    """Masks that are no trees: rows that see everything, themselves only, later nodes, nothing; more words than needed."""
    rng, nodes = random.Random(9), [20, 33, 4]
    bits = [rng.choice((0, rng.getrandbits(n), (1 << n) - 1, 1 << rng.randrange(n))) for n in nodes for _ in range(n)]
    for ctx in ([40, 100, 7], [0, 0, 0]):
        Case(dev, nodes, ctx, bits=bits, words=2, seed=10).check(mi)


def test_rows_that_see_nothing_are_zeros(mi, dev):
    got = Case(dev, [4], [0], bits=[0, 1, 0, 15], seed=11).check(mi)
    assert (got[0] == 0).all() and (got[2] == 0).all() and (got[1] != 0).any()


@pytest.mark.parametrize("dtype,fp8,d", [(BF16, False, 128), (FP16, False, 64), (FP16, False, 256), (BF16, True, 128), (FP16, True, 64)])
def test_what_a_row_does_not_see_does_not_reach_it(mi, dev, dtype, fp8, d):
    """NaN and infinities in nodes' keys and values meet the rows that see them and no others."""
    parents = [-1, 0, 0, 1, 2, 2, 4]
    c = Case(dev, [7, 7], [60, 133], d=d, dtype=dtype, fp8=fp8, bits=osp.ancestors(parents) * 2, seed=12)
    for r in range(2):
        for node, v in ((3, math.nan), (5, math.inf), (6, -math.inf)):
            chunk, at = osp.position(c.table[r].tolist(), 64, c.N, c.lens[r] - 7 + node)
            bad = torch.full((d // 2,), math.nan if fp8 else v).to(c.v.dtype)
            c.v[chunk, at, 0, ::2] = bad
            if node == 3:
                c.k[chunk, at, 1, :] = torch.full((d,), math.nan).to(c.k.dtype)
    got = c.check(mi)
    assert torch.isfinite(got[[0, 1, 2, 4, 7, 8, 9, 11]]).all() and not torch.isfinite(got[3]).all()


@pytest.mark.parametrize("nodes,Hq,d,dtype", [(33, 8, 128, BF16), (70, 8, 128, FP16), (90, 4, 64, BF16), (150, 4, 64, FP16), (40, 8, 96, BF16), (40, 8, 256, FP16)])
def test_what_a_row_does_not_see_does_not_reach_it_in_large_trees(mi, dev, nodes, Hq, d, dtype):
    c = Case(dev, [nodes, nodes - 5], [60, 133], Hq=Hq, Hkv=2, d=d, dtype=dtype, shape="tree", seed=nodes)
    for r in range(2):
        for node, v in ((3, math.nan), (nodes // 2, math.inf), (nodes // 2 + 1, -math.inf), (nodes - 6, math.nan)):
            chunk, at = osp.position(c.table[r].tolist(), 64, c.N, c.lens[r] - c.cu[r + 1] + c.cu[r] + node)
            c.v[chunk, at, 0, ::3] = v
            c.k[chunk, at, 1, 5] = v
    got = c.check(mi)
    assert torch.isfinite(got[0]).all() and not torch.isfinite(got[3]).all()


@pytest.mark.parametrize("nodes,Hq,Hkv,d,chunk", [
    ([64, 64], 16, 2, 128, 256), ([17, 61, 40, 0, 33], 32, 8, 128, 64), ([100, 20], 8, 8, 64, 32), ([256], 16, 2, 64, 64), ([90, 1, 1], 5, 1, 128, 96),
    ([64, 64], 16, 2, 256, 64), ([64, 30], 16, 2, 96, 64), ([64, 64], 16, 2, 128, 48), ([130], 6, 6, 192, 16),
])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_many_rows(mi, dev, nodes, Hq, Hkv, d, chunk, dtype):
    Case(dev, nodes, [700 + 37 * i for i in range(len(nodes))], Hq=Hq, Hkv=Hkv, d=d, chunk=chunk, dtype=dtype, spare=2, seed=d + chunk).check(mi)
    Case(dev, nodes, [3 * i for i in range(len(nodes))], Hq=Hq, Hkv=Hkv, d=d, chunk=chunk, dtype=dtype, seed=d + chunk).check(mi)


def test_many_rows_of_an_fp8_cache(mi, dev):
    for d, chunk in ((64, 64), (128, 64), (128, 16)):
        Case(dev, [64, 41], [300, 777], Hq=16, Hkv=2, d=d, chunk=chunk, fp8=True, seed=d).check(mi)


def test_many_rows_with_tables_and_lengths_that_do_not_fit(mi, dev):
    c = Case(dev, [40, 50, 60], [300, 200, 500], seed=24)
    c.table[0, 2], c.table[1, 0], c.table[1, 3], c.table[2, 8] = -1, c.N, 1 << 30, -7
    c.check(mi)
    c.lens = [4096, 30, -1]
    c.check(mi)


def test_what_lies_behind_a_request_is_not_read(mi, dev):
    c = Case(dev, [5, 3], [70, 20], seed=13)
    used = torch.zeros(c.N, 64, dtype=torch.bool)
    for r in range(2):
        for k in range(c.lens[r]):
            used[osp.position(c.table[r].tolist(), 64, c.N, k)] = True
    c.k[~used] = math.nan
    c.v[~used] = math.nan
    assert torch.isfinite(c.check(mi)).all()
    c = Case(dev, [45, 33], [70, 20], seed=13)
    used = torch.zeros(c.N, 64, dtype=torch.bool)
    for r in range(2):
        for k in range(c.lens[r]):
            used[osp.position(c.table[r].tolist(), 64, c.N, k)] = True
    c.k[~used] = math.nan
    c.v[~used] = math.nan
    assert torch.isfinite(c.check(mi)).all()


def test_table_entries_that_name_no_chunk(mi, dev):
    c = Case(dev, [5, 9], [300, 200], seed=14)
    c.table[0, 2], c.table[1, 0], c.table[1, 3] = -1, c.N, 1 << 30
    c.check(mi)


def test_lengths_and_rows_outside_their_arrays(mi, dev):
    """Lengths beyond the table are cut to it, negative ones are none, nodes without a position have no key."""
    c = Case(dev, [4, 3, 5, 2], [100, 50, 0, 20], seed=15)
    c.lens = [4096, -7, 2, 22]
    c.check(mi)


def test_empty_requests_and_padding_rows(mi, dev):
    c = Case(dev, [0, 5, 0, 0, 2, 0], [10, 40, 0, 33, 7, 1], spare=9, seed=16)
    out = torch.full_like(c.q, 7).to(dev)
    assert c.run(mi, out=out) is out
    c.check(mi, got=out)


def test_strides(mi, dev):
    """Queries inside a wider tensor, results into one, caches with gaps between heads, a mask inside a wider one."""
    c = Case(dev, [6, 11], [90, 45], Hq=8, Hkv=4, d=64, chunk=32, seed=17)
    T = c.cu[-1]
    wide = torch.zeros(T, 3, 8, 128, dtype=BF16, device=dev)
    q = wide[:, 1, :, :64]
    q.copy_(c.q)
    out = torch.full((T, 12, 72), 5.0, dtype=BF16, device=dev)
    masks = torch.full((T, 7), -1, dtype=torch.int64, device=dev)
    masks[:, 2:3] = c.mask.to(dev)
    pools = torch.full((c.N, 32, 4, 2, 80), math.nan, dtype=BF16, device=dev)
    pools[..., 0, :64], pools[..., 1, :64] = c.k.to(dev), c.v.to(dev)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    table = torch.full((2, 16), -5, dtype=torch.int32, device=dev)
    table[:, :c.table.size(1)] = c.table.to(dev)
    got = mi.ops.paged_tree_attention(q, pools[..., 0, :64], pools[..., 1, :64], i32(c.cu), i32(c.lens), table, masks[:, 2:3],
                                      softmax_scale=c.scale, out=out[:, 4:, :64])
    c.check(mi, got=got)
    assert (out[:, :4] == 5).all() and (out[:, 4:, 64:] == 5).all()
    c.check(mi, mask=masks[:, 2])                                     # one word a row, as a column
    assert c.run(mi, q=c.q.to(dev).unsqueeze(1)).shape == (T, 1, 8, 64)


@pytest.mark.parametrize("layout", ["heads first", "one token for all", "padded rows"])
@pytest.mark.parametrize("nodes,Hq,fp8", [([5, 9], 8, False), ([12, 3], 16, True), ([40, 61], 16, False), ([30, 50], 16, True)])
def test_cache_layouts(mi, dev, layout, nodes, Hq, fp8):
    """Token rows nearer together than a row is long, at the same place, and further apart; the last chunk of the pool is used."""
    case = Case(dev, nodes, [100, 37], Hq=Hq, Hkv=4, d=64, chunk=32, fp8=fp8, seed=Hq)
    case.table[0, 0] = case.N - 1
    if layout == "one token for all":
        case.k, case.v = (x[:, :1].expand_as(x).contiguous() for x in (case.k, case.v))
    gpu = []
    for x in (case.k, case.v):
        x = (x.view(torch.uint8) if fp8 else x).to(dev)
        if layout == "heads first":
            x = x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
        elif layout == "one token for all":
            x = x[:, :1].contiguous().expand_as(x)
        else:
            wide = torch.empty(*x.shape[:2], 5, x.size(3), dtype=x.dtype, device=dev)
            wide[:, :, :4] = x
            x = wide[:, :, :4]
        gpu.append(x)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    scales = dict(k_scales=case.scales[0].to(dev), v_scales=case.scales[1].to(dev)) if fp8 else {}
    case.check(mi, mi.ops.paged_tree_attention(case.q.to(dev), *gpu, i32(case.cu), i32(case.lens), case.table.to(dev), case.mask.to(dev),
                                               softmax_scale=case.scale, max_kv_len=max(case.lens), **scales))


def test_many_requests(mi, dev):
    """More than one launch takes (their prefix sums lie in LDS): every one is answered, ragged and empty ones among them."""
    rng = random.Random(18)
    nodes = [rng.randint(0, 3) for _ in range(4999)]
    Case(dev, nodes, [rng.randint(0, 40) for _ in nodes], Hq=2, Hkv=1, d=64, chunk=16, spare=3, seed=18).check(mi)


@pytest.mark.parametrize("dtype,fp8", [(BF16, False), (FP16, False), (BF16, True)])
def test_long_contexts(mi, dev, dtype, fp8):
    Case(dev, [13, 2], [20011, 4096], Hq=4, Hkv=1, d=64, chunk=256, dtype=dtype, fp8=fp8, seed=19).check(mi)


def test_growing_and_large_scores(mi, dev):
    """Keys whose scores keep growing move the running maximum in every tile; 16-bit queries ten times as large."""
    c = Case(dev, [9], [800], seed=20, spread=3.0)
    for k in range(c.lens[0]):
        chunk, at = osp.position(c.table[0].tolist(), 64, c.N, k)
        c.k[chunk, at] = (c.k[chunk, at].float() * (0.1 + k / 400)).to(BF16)
    c.check(mi)


def test_a_chain_is_the_causal_call(mi, dev):
    c = Case(dev, [6, 6, 1], [500, 31, 64], shape="chain", Hq=32, Hkv=8, seed=21)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    other = mi.ops.paged_prefill_attention(c.q.to(dev), c.k.to(dev), c.v.to(dev), i32(c.cu), i32(c.lens), c.table.to(dev))
    c.check(mi, got=other)
    c.check(mi)


@pytest.mark.parametrize("nodes", [[5, 12], [40, 64]])
def test_replays_and_streams(mi, dev, nodes):
    """A captured call replayed among eager work, with new values in place, and a call on a stream of its own."""
    c = Case(dev, nodes, [300, 64], seed=22)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    q, k, v = c.q.to(dev), c.k.to(dev), c.v.to(dev)
    args = (i32(c.cu), i32(c.lens), c.table.to(dev), c.mask.to(dev))
    eager = mi.ops.paged_tree_attention(q, k, v, *args, softmax_scale=c.scale)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        aside = mi.ops.paged_tree_attention(q, k, v, *args, softmax_scale=c.scale)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(aside, eager)
    work = torch.empty(mi._lib.load().mi_tree_workspace_bytes(c.cu[-1], 2, 8, 2, 128), dtype=torch.uint8, device=dev)
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(q)
    with mi.ops.use_workspace(work):
        with torch.cuda.graph(graph):
            mi.ops.paged_tree_attention(q, k, v, *args, softmax_scale=c.scale, out=out)
    for step in range(4):
        q.mul_(0.9)
        out.zero_()
        graph.replay()
        again = mi.ops.paged_tree_attention(q, k, v, *args, softmax_scale=c.scale)
        torch.cuda.synchronize()
        assert torch.equal(out, again), step


def test_refusals(mi, dev):
    c = Case(dev, [5], [20], seed=23)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    q, k, v, table, mask = c.q.to(dev), c.k.to(dev), c.v.to(dev), c.table.to(dev), c.mask.to(dev)
    call = lambda **x: mi.ops.paged_tree_attention(*{**dict(q=q, k=k, v=v, cu=i32([0, 5]), lens=i32([25]), t=table, m=mask), **x}.values())  # noqa: E731
    for change, word in ((dict(m=mask.int()), "int64"), (dict(m=mask[:4]), "row for every"), (dict(m=mask.expand(5, 5)), "words"),
                         (dict(cu=i32([0])), "two entries"), (dict(k=k.half()), "16-bit type"), (dict(k=k[..., :64]), "shape"),
                         (dict(lens=i32([])), "shorter"), (dict(t=table.long()), "block_table"), (dict(q=q.float()), "bf16 or fp16"),
                         (dict(m=mask.cpu()), "one device")):
        with pytest.raises(ValueError, match=word):
            call(**change)
    with pytest.raises(mi._lib.KernelError, match="multiple of 16"):
        call(k=k[:, :24], v=v[:, :24])
    with pytest.raises(ValueError, match="go together"):
        mi.ops.paged_tree_attention(q, k, v, i32([0, 5]), i32([25]), table, mask, k_scales=torch.ones(c.N, 2, device=dev))


def _sink(c, gap, seed):
    """One key of every request ``gap`` above all others, which score alike; its values are zero, the others' near one."""
    gen = torch.Generator().manual_seed(seed)
    c.q.zero_()
    c.q[..., 0] = 1
    c.k, c.v = torch.zeros_like(c.k), (0.5 + torch.rand(c.v.shape, generator=gen)).to(c.v.dtype)
    for r, length in enumerate(c.lens):
        chunk, at = osp.position(c.table[r].tolist(), c.k.size(1), c.N, 3 if r % 2 else length // 2)
        c.k[chunk, at, :, 0] = gap / c.scale
        c.v[chunk, at] = 0
    return c


@pytest.mark.parametrize("gap", [6.0, 12.0, 13.5, 15.0, 16.0])
@pytest.mark.parametrize("d,chunk,nodes", [(128, 64, [2, 1]), (128, 48, [2, 1]), (64, 64, [9, 7]), (64, 16, [2, 1]), (96, 64, [2, 1]), (256, 64, [2, 1]),
                                           (128, 64, [40, 3])])
def test_a_token_far_above_a_long_context(mi, dev, gap, d, chunk, nodes):
    """fp16 probabilities of a long context far below one token keep their eleven bits: the row's largest one is at 2^10 at
    least, so that e^-16 of it (2^-23.1) is above the type's smallest normal number, 2^-14.  The bound is the others'."""
    _sink(Case(dev, nodes, [30011, 9000], Hq=4, Hkv=2, d=d, chunk=chunk, dtype=FP16, seed=25), gap, 25).check(mi)


@pytest.mark.parametrize("d,chunk", [(64, 16), (128, 64)])
def test_a_token_far_above_others_of_its_span(mi, dev, d, chunk):
    """The same where one wavefront takes a request's whole context (many KV heads), so that no partial leaves the token out."""
    _sink(Case(dev, [1, 1, 1, 1], [1500, 1000, 700, 1400], Hq=256, Hkv=256, d=d, chunk=chunk, dtype=FP16, seed=27), 16.0, 27).check(mi)


def test_scores_that_grow_by_every_amount(mi, dev):
    """fp16: a row's largest score grows tile by tile, by less and by more than the window of its probabilities."""
    for growth in (0.4, 3.0, 7.5, 11.0, 30.0):
        for chunk, nodes in ((64, [4, 2]), (48, [4, 2]), (64, [40, 9])):
            c = Case(dev, nodes, [700, 333], Hq=8, Hkv=2, dtype=FP16, chunk=chunk, seed=26)
            c.q.zero_()
            c.q[..., 0] = 1
            for r in range(2):
                for k in range(c.lens[r]):
                    at = osp.position(c.table[r].tolist(), chunk, c.N, k)
                    c.k[at[0], at[1], :, 0] = growth * (k // 32) / c.scale if k % 5 else 0
            c.check(mi)


@pytest.mark.parametrize("requests", [9, 100])
@pytest.mark.parametrize("Hq,Hkv,d,chunk", [(8, 2, 128, 64), (64, 1, 128, 64), (4, 2, 64, 16), (16, 2, 96, 48)])
def test_rows_that_fall(mi, dev, requests, Hq, Hkv, d, chunk):
    """Where cu_seqlens_q falls its running maximum counts: no row belongs to two requests, and the workspace, which has a place for
    every group of rows, is written inside its own bytes."""
    c = Case(dev, [7, 120, 0, 1] + [0] * (requests - 4), [40, 200, 3, 5] + [60] * (requests - 4), Hq=Hq, Hkv=Hkv, d=d, chunk=chunk, seed=28)
    legit, rows = c.cu, c.cu[-1]
    falling = [0, 7, 127, -5, 128] + [(0, rows, 3, rows + 9, -1)[i % 5] for i in range(5, requests + 1)]
    need = mi._lib.load().mi_tree_workspace_bytes(rows, requests, Hq, Hkv, d)
    work = torch.full((need + 8192,), 0x5a, dtype=torch.uint8, device=dev)
    c.cu = falling
    with mi.ops.use_workspace(work[:need]):
        got = c.run(mi)
    c.cu = legit
    c.check(mi, got=got)
    assert (work[need:] == 0x5a).all()


@pytest.mark.parametrize("requests", [65, 300, 2100])
@pytest.mark.parametrize("Hq,Hkv,d,chunk,fp8", [
    (8, 2, 128, 64, False), (64, 1, 128, 64, False),      # tiles through LDS: four wavefronts, eight
    (8, 1, 64, 64, False), (64, 1, 64, 32, False),        # the same of width 64
    (64, 1, 128, 48, False), (24, 1, 128, 48, False),     # through registers, eight and two or four parts sharing tokens
    (32, 4, 256, 64, False), (64, 1, 64, 64, True), (16, 8, 128, 64, True),
])
def test_more_requests_than_lanes(mi, dev, requests, Hq, Hkv, d, chunk, fp8):
    """Ragged batches, empty requests among them, whose sums lie in LDS beside the tiles or what wavefronts join: every row against
    the causal call (two bounds apart at values of at most five), some requests against the oracle."""
    rng = random.Random(requests)
    nodes = [rng.choice((0, 1, 2, 3, 4, 5)) for _ in range(requests)]
    nodes[rng.randrange(requests)], nodes[-1] = 40, 3
    c = Case(dev, nodes, [rng.randint(0, 70) for _ in nodes], Hq=Hq, Hkv=Hkv, d=d, chunk=chunk, fp8=fp8, shape="chain", spare=3, seed=requests)
    got = c.run(mi)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    scales = dict(k_scales=c.scales[0].to(dev), v_scales=c.scales[1].to(dev)) if fp8 else {}
    k, v = ((x.view(torch.uint8) if fp8 else x).to(dev) for x in (c.k, c.v))
    if not fp8 or chunk % 64 == 0:
        other = mi.ops.paged_prefill_attention(c.q.to(dev), k, v, i32(c.cu), i32(c.lens), c.table.to(dev), **scales)
        assert (got.float() - other.float()).abs().max() < 2 * 3 * 2.0 ** -8 * 5.5
    torch.cuda.synchronize()
    assert (got[c.cu[-1]:] == 0).all()
    picks = sorted({0, 1, 63, 64, requests - 1, requests // 2, min(2047, requests - 1), min(2048, requests - 1), nodes.index(40)})
    some = Case.__new__(Case)
    some.__dict__.update(c.__dict__)
    some.cu, rows = [0], []
    for r in picks:
        rows += range(c.cu[r], c.cu[r + 1])
        some.cu.append(len(rows))
    some.q, some.bits, some.lens, some.table = c.q[rows], [c.bits[i] for i in rows], [c.lens[r] for r in picks], c.table[picks]
    some.check(mi, got=got[rows])


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_a_value_scale_of_zero_behind_large_sums(mi, dev, dtype):
    """Every token the same score, values at e4m3's end with scales of one, then chunks with a scale of zero (and one with a scale after
    them): the sums of a whole context in one wavefront change to that unit and back without leaving fp32."""
    c = Case(dev, [1, 1], [5000, 3333], Hq=256, Hkv=256, d=64, chunk=64, dtype=dtype, fp8=True, seed=29)
    c.k = torch.zeros(c.k.shape).to(torch.float8_e4m3fn)
    c.v = torch.full(c.v.shape, 448.0).to(torch.float8_e4m3fn)
    for s in c.scales:
        s.fill_(1.0)
    for r in range(2):
        n = c.lens[r] // 64
        c.scales[1][c.table[r, n - 3:n - 1].long()] = 0
    c.check(mi)


def test_value_scales_that_are_no_number(mi, dev):
    """A NaN among the scales reaches the rows that see its chunk, and no others; a key scale's the same."""
    for which in (0, 1):
        c = Case(dev, [6, 5], [200, 150], chunk=64, fp8=True, dtype=FP16, seed=30)
        c.scales[which][c.table[0, 1].long(), 1] = math.nan
        got = c.check(mi)
        assert got[:6, 4:].isnan().all() and torch.isfinite(got[:6, :4]).all() and torch.isfinite(got[6:]).all()


@pytest.mark.parametrize("chunk", [32, 64, 256])
@pytest.mark.parametrize("requests,Hq,Hkv,dtype", [(31, 8, 8, BF16), (70, 24, 8, FP16), (33, 16, 16, BF16), (9, 32, 32, FP16)])
def test_few_rows_of_many_heads(mi, dev, chunk, requests, Hq, Hkv, dtype):
    """Width 128 with so many heads and requests to a row that tiles come through registers."""
    rng = random.Random(chunk + requests)
    nodes = [rng.choice((0, 1, 1, 2)) for _ in range(requests)]
    assert 80 * max(3, sum(nodes) * (Hq // Hkv) // requests) <= requests * Hkv
    Case(dev, nodes, [rng.randint(0, 300) for _ in nodes], Hq=Hq, Hkv=Hkv, chunk=chunk, dtype=dtype, spare=1, seed=chunk).check(mi)
