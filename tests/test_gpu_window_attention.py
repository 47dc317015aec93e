"""GPU parity: attention with a window and sinks over the paged cache against the 64-bit oracle.

Tolerance, element by element, with u half a step of the 16-bit type, A = sum p |v| and S = sum |v| over the n tokens in
sight: the probabilities are rounded once (each by at most u, in the numerator and in the row sum: 2 u A), the result once
(u |o|), scores are 32-bit sums of exact products and the exponentials of 32-bit hardware precision: 2^-24 times a score of at
most some 30 and a few roundings, 2e-5 A.  fp16 probabilities below 2^-14 of what the row's largest is taken for are
subnormal: off by half a step of 2^-24 there, against a row sum of at least one half: 2^-24 (S + n |o|).  Prompts over an
fp8 cache of width 64 round every value times its scale, once more u A.
"""
import math
import random

import pytest
import torch

from oracle import windows as ow

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


class Case:
    """``new`` rows of ``lens`` tokens per request; ``new`` None: the decode form, one row each."""

    def __init__(self, dev, new, lens, window, sinks, *, Hq=8, Hkv=2, d=128, chunk=64, dtype=BF16, fp8=False, seed=0, spare=0,
                 spread=1.0, columns=1):
        rng, gen = random.Random(seed), torch.Generator().manual_seed(seed)
        del rng
        self.decode, self.window, self.sinks, self.lens = new is None, window, sinks, list(lens)
        new = [1] * len(lens) if new is None else new
        self.cu = [0]
        for n in new:
            self.cu.append(self.cu[-1] + n)
        need = [-(-max(n, 0) // chunk) for n in lens]
        self.N = sum(need) + 2
        ids = torch.randperm(self.N, generator=gen).tolist()
        self.table = torch.zeros(len(new), max(max(need), 1) + columns, dtype=torch.int32)
        for r, k in enumerate(need):
            self.table[r, :k] = torch.tensor([ids.pop() for _ in range(k)], dtype=torch.int32)
        self.q = (torch.randn(self.cu[-1] + spare, Hq, d, generator=gen) * spread).to(dtype)
        shape = (self.N, chunk, Hkv, d)
        self.scales = None
        if fp8:
            self.k, self.v = ((torch.randn(shape, generator=gen) * 100).clamp(-448, 448).to(torch.float8_e4m3fn) for _ in "kv")
            self.scales = [0.004 + 0.01 * torch.rand(self.N, Hkv, generator=gen) for _ in "kv"]
        else:
            self.k, self.v = (torch.randn(shape, generator=gen).to(dtype) for _ in "kv")
        self.dev, self.scale, self.dtype, self.chunk, self.d = dev, d ** -0.5, dtype, chunk, d

    def inputs(self):
        dev, cache = self.dev, [x.view(torch.uint8) if self.scales else x for x in (self.k, self.v)]
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
        more = dict(k_scales=self.scales[0].to(dev), v_scales=self.scales[1].to(dev)) if self.scales else {}
        more.update(softmax_scale=self.scale, window=self.window, sinks=self.sinks)
        rows = [self.q.to(dev), cache[0].to(dev), cache[1].to(dev)]
        if not self.decode:
            rows.append(i32(self.cu))
        return rows + [i32(self.lens), self.table.to(dev)], more

    def run(self, mi, **over):
        args, more = self.inputs()
        more.update(over)
        return (mi.ops.paged_decode_attention if self.decode else mi.ops.paged_prefill_attention)(*args, **more)

    def reference(self):
        k, v = (x.float() if self.scales else x for x in (self.k, self.v))
        return ow.window_attention(self.q[:self.cu[-1]], k, v, self.cu, self.lens, self.table, self.window, self.sinks, self.scale,
                                   *(self.scales or ()))

    def check(self, mi, got=None, **over):
        got = self.run(mi, **over) if got is None else got
        torch.cuda.synchronize()
        got, (ref, size, total) = got.cpu().double().view(-1, *self.q.shape[1:]), self.reference()
        u = torch.finfo(self.dtype).eps / 2
        assert (got[self.cu[-1]:] == 0).all(), "rows behind the last request"
        got = got[:self.cu[-1]]
        assert torch.equal(got.isnan(), ref.isnan()), "NaN"
        fine = torch.isfinite(ref)
        assert torch.equal(got[~fine & ~ref.isnan()], ref[~fine & ~ref.isnan()])
        rounds = 3 if self.scales and self.d == 64 and not self.decode else 2
        bound = (rounds * u + 2e-5) * size * (1 + u) + u * ref.abs() + 1e-7
        if self.dtype == FP16:
            seen = min(self.window + self.sinks, max(self.lens))
            bound = bound + 2.0 ** -24 * (total + seen * ref.abs())
        err, bound = (got - ref).abs()[fine], bound[fine]
        assert (err <= bound).all(), f"max err / bound {(err / bound).max():.3f}"
        return got


# lengths, window, sinks: windows of one token, inside a tile, on its borders, over everything; sinks of none, inside the
# window's first tile, over several tiles, more than there are tokens
SHAPES = [
    ([1], 1, 0), ([1], 5, 3), ([2, 1], 1, 0), ([300], 1, 0), ([300], 1, 1), ([300], 64, 0), ([257], 65, 4), ([777], 100, 4),
    ([64, 63, 65, 128], 63, 1), ([500, 31, 400], 128, 64), ([500], 100, 130), ([129], 1000, 4), ([640], 96, 200), ([333], 40, 1000),
    ([0, 200, 5, 0], 33, 2), ([1024], 31, 33), ([700, 90], 640, 16),
]


@pytest.mark.parametrize("lens,window,sinks", SHAPES)
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_decode_shapes(mi, dev, lens, window, sinks, dtype):
    Case(dev, None, lens, window, sinks, dtype=dtype, seed=sum(lens)).check(mi)


@pytest.mark.parametrize("lens,window,sinks", SHAPES)
def test_decode_shapes_by_the_stream(mi, dev, lens, window, sinks):
    """The kernel of long or many requests, over spans of one tile and of several, whose parts are merged."""
    c = Case(dev, None, lens, window, sinks, seed=sum(lens))
    for grid in (1, 3, 40):
        with mi.ops.tuning(decode_grid=grid):
            c.check(mi)


@pytest.mark.parametrize("Hq,Hkv,d", [(8, 8, 64), (32, 8, 128), (7, 1, 96), (12, 4, 192), (16, 2, 256), (64, 1, 64), (28, 4, 128),
                                      (20, 1, 128), (24, 3, 96), (11, 11, 64)])
def test_decode_head_layouts(mi, dev, Hq, Hkv, d):
    c = Case(dev, None, [100, 333, 1, 250], 90, 5, Hq=Hq, Hkv=Hkv, d=d, seed=d + Hq)
    c.check(mi)
    with mi.ops.tuning(decode_grid=5):
        c.check(mi)


@pytest.mark.parametrize("chunk", [16, 48, 32, 80, 64, 256])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_decode_chunk_sizes(mi, dev, chunk, d):
    for sinks in (3, chunk + 7):
        c = Case(dev, None, [chunk - 5, 3 * chunk + 1, 9 * chunk + 11], 2 * chunk + 3, sinks, d=d, chunk=chunk, seed=chunk)
        c.check(mi)
        with mi.ops.tuning(decode_grid=4):
            c.check(mi)


@pytest.mark.parametrize("d,chunk,dtype", [(64, 64, BF16), (64, 16, FP16), (64, 32, BF16), (128, 256, FP16), (128, 48, BF16), (128, 32, FP16)])
def test_decode_fp8_caches(mi, dev, d, chunk, dtype):
    c = Case(dev, None, [270, 64, 1, 511, 900], 200, 20, Hq=16, Hkv=4, d=d, chunk=chunk, dtype=dtype, fp8=True, seed=d + chunk)
    c.check(mi)
    with mi.ops.tuning(decode_grid=7):
        c.check(mi)


@pytest.mark.parametrize("tiles", [1, 2, 4])
@pytest.mark.parametrize("d,fp8,dtype", [(128, False, BF16), (64, False, FP16), (192, False, BF16), (128, True, BF16), (64, True, FP16)])
@pytest.mark.parametrize("lens,window,sinks", SHAPES[3::2] + [([0, 200, 5, 0], 33, 2)])
def test_decode_tiles_of_every_size(mi, dev, lens, window, sinks, d, fp8, dtype, tiles):
    c = Case(dev, None, lens, window, sinks, d=d, fp8=fp8, dtype=dtype, seed=sum(lens) + d)
    for grid in (3, 17):
        with mi.ops.tuning(decode_tile_subtiles=tiles, decode_grid=grid):
            c.check(mi)


@pytest.mark.parametrize("d", [64, 128])
def test_decode_of_long_walks(mi, dev, d):
    """Walks past the line between small tiles and large ones."""
    Case(dev, None, [2900, 4100, 60], 2600, 4, Hq=4, Hkv=2, d=d, seed=d).check(mi)


@pytest.mark.parametrize("R", [4, 8, 16, 24, 31, 70, 127])
@pytest.mark.parametrize("d,fp8,alike", [(128, False, True), (64, True, True), (64, False, False)])
def test_workgroups_dealt_out_by_requests(mi, dev, R, d, fp8, alike):
    """Half a request, one, two and more for each of the grid's eight workgroups, and (requests not alike, or not going into the grid)
    spans by tiles: every part of every request once."""
    lens = [1000 + 17 * (7 * i % 5) for i in range(R)]
    if not alike:
        lens[R // 2] = 100
    c = Case(dev, None, lens, 700, 3, d=d, fp8=fp8, seed=R)
    with mi.ops.tuning(decode_grid=8):
        c.check(mi)


def test_many_requests_in_the_lanes_and_in_shared_memory(mi, dev):
    rng = random.Random(3)
    for n in (64, 65, 200):
        c = Case(dev, None, [rng.choice((0, 1, 40, 200, 333)) for _ in range(n)], 70, 4, Hq=4, Hkv=2, d=64, seed=n)
        c.check(mi)
        with mi.ops.tuning(decode_grid=33):
            c.check(mi)


PROMPTS = [
    ([5], [5], 2, 0), ([64], [64], 1, 0), ([65, 3], [65, 200], 64, 4), ([130], [130], 33, 1), ([200], [200], 1000, 10),
    ([70], [500], 100, 4), ([33, 1, 90], [400, 300, 90], 65, 70), ([300], [300], 63, 0), ([257], [257], 128, 64), ([2, 2], [2, 900], 1, 1),
    ([100], [700], 64, 640), ([150], [151], 90, 300), ([40, 1, 0, 1, 7], [40, 513, 0, 1, 600], 129, 3), ([90], [60], 20, 2),
]


@pytest.mark.parametrize("new,lens,window,sinks", PROMPTS)
@pytest.mark.parametrize("d,dtype", [(128, BF16), (64, FP16), (128, FP16), (64, BF16)])
def test_prompt_shapes(mi, dev, new, lens, window, sinks, d, dtype):
    c = Case(dev, new, lens, window, sinks, d=d, dtype=dtype, seed=sum(lens) + d, spare=3)
    c.check(mi)
    c.check(mi, one_row_requests=False)


@pytest.mark.parametrize("new,lens,window,sinks", PROMPTS)
@pytest.mark.parametrize("d,dtype", [(96, BF16), (192, FP16), (256, BF16)])
def test_prompt_shapes_of_other_widths(mi, dev, new, lens, window, sinks, d, dtype):
    Case(dev, new, lens, window, sinks, d=d, dtype=dtype, seed=sum(lens) + d, spare=2).check(mi, one_row_requests=False)


@pytest.mark.parametrize("where", ["keys", "values", "queries"])
@pytest.mark.parametrize("d,fp8", [(64, False), (128, True), (96, False)])
@pytest.mark.parametrize("new,lens,parts", [([257, 3], [300, 3], 0), ([40], [5000], 5)])
def test_nothing_but_nan(mi, dev, new, lens, parts, d, fp8, where):
    """Every row is made again and ends at its first tile."""
    c = Case(dev, new, lens, 200, 3, d=d, fp8=fp8, seed=d)
    if where == "queries":
        c.q.fill_(math.nan)
    elif fp8:
        c.scales[where == "values"].fill_(math.nan)
    else:
        (c.v if where == "values" else c.k).fill_(math.nan)
    with mi.ops.tuning(prefill_kv_split=parts):
        assert c.run(mi, one_row_requests=False).isnan().all()


@pytest.mark.parametrize("new,lens", [([130, 3, 0, 257, 7], [1600, 90, 40, 2500, 2500]), ([300, 299], [3000, 299]), ([5] * 130, [1500] * 130)])
@pytest.mark.parametrize("d,fp8", [(64, False), (128, False), (96, False), (128, True)])
def test_windows_short_beside_the_requests(mi, dev, new, lens, d, fp8):
    """Query blocks in the batch's order: a walk of at most a quarter of the longest request, no requests of one row."""
    Case(dev, new, lens, 20, 3, d=d, fp8=fp8, seed=d + len(lens), spare=3).check(mi, one_row_requests=False, max_kv_len=max(lens))


@pytest.mark.parametrize("d,chunk", [(64, 64), (96, 64), (128, 64), (128, 16)])
@pytest.mark.parametrize("lens", [[-5, 90, -2000000000, 70], [90, 2147483647, -1, 90], [-1] * 4])
@pytest.mark.parametrize("form", ["decode", "prompts", "many prompts"])
def test_lengths_are_kept_in_the_table(mi, dev, form, lens, d, chunk):
    """Below zero as zero, above the table's tokens as those."""
    more = 33 if form == "many prompts" else 1   # (more requests than the blocks are ordered for)
    new = None if form == "decode" else [40, 3, 7, 33] * more
    c = Case(dev, new, [min(n, 90) for n in lens] * more, 20, 3, d=d, chunk=chunk, seed=d)
    c.lens = lens * more
    c.table = c.table[:, :-(-90 // chunk)].contiguous()
    c.check(mi, one_row_requests=False) if new else c.check(mi)


@pytest.mark.parametrize("d,fp8", [(64, False), (96, False), (128, False), (128, True)])
@pytest.mark.parametrize("window,sinks", [(20, 3), (1, 0), (1 << 62, 3), (1 << 29, 0)])
@pytest.mark.parametrize("form", ["decode", "one row", "stream", "stream of many"])
def test_lengths_far_below_zero_are_zero(mi, dev, form, window, sinks, d, fp8):
    """Such a length less the window does not wrap: nothing is walked, the row is zeros, in decode calls and for one-row requests of prompts."""
    more = 40 if form == "stream of many" else 1
    lens = [-(1 << 31), 90, -2000000000, -1, 70, -(1 << 31) + 1] * more
    c = Case(dev, [1, 1, 1, 1, 7, 1] * more if form == "one row" else None, [max(n, 0) for n in lens], window, sinks, d=d, fp8=fp8, seed=d)
    c.lens = lens
    if form.startswith("stream"):
        with mi.ops.tuning(decode_grid=7):
            c.check(mi)
    else:
        c.check(mi)


@pytest.mark.parametrize("chunk", [16, 48, 80])
@pytest.mark.parametrize("d", [64, 96, 128, 192, 256])
def test_prompts_over_chunks_of_other_sizes(mi, dev, chunk, d):
    for new, lens, window, sinks in (([70, 1, 30], [300, 90, 30], 50, 20), ([40], [900], 33, 0), ([130], [130], 17, 1)):
        Case(dev, new, lens, window, sinks, d=d, chunk=chunk, seed=chunk + d, spare=1).check(mi)


@pytest.mark.parametrize("Hq,Hkv,d", [(8, 8, 64), (32, 8, 128), (7, 1, 96), (64, 1, 64), (28, 4, 128), (20, 1, 128), (24, 3, 64)])
def test_prompt_head_layouts(mi, dev, Hq, Hkv, d):
    Case(dev, [75, 130], [75, 400], 66, 9, Hq=Hq, Hkv=Hkv, d=d, seed=d + Hq).check(mi)


@pytest.mark.parametrize("new,lens,window,sinks", PROMPTS[2:])
@pytest.mark.parametrize("d,dtype", [(64, BF16), (128, FP16), (128, BF16), (64, FP16)])
def test_prompts_over_fp8_caches(mi, dev, new, lens, window, sinks, d, dtype):
    c = Case(dev, new, lens, window, sinks, Hq=8, Hkv=2, d=d, dtype=dtype, fp8=True, seed=d + sum(lens), spare=1)
    c.check(mi)
    c.check(mi, one_row_requests=False)


@pytest.mark.parametrize("d,fp8", [(128, False), (64, False), (128, True), (64, True), (96, False), (256, False)])
@pytest.mark.parametrize("parts", [2, 3, 5, 11])
def test_prompts_whose_keys_are_split(mi, dev, d, fp8, parts):
    for window, sinks in ((300, 70), (65, 0), (2000, 4)):
        c = Case(dev, [40, 9], [1100, 400], window, sinks, d=d, fp8=fp8, seed=parts)
        with mi.ops.tuning(prefill_kv_split=parts):
            c.check(mi, one_row_requests=False)


def test_long_prompts(mi, dev):
    """Workgroups of four and of eight wavefronts, many query blocks."""
    Case(dev, [1500], [1500], 300, 4, Hq=4, Hkv=1, seed=1).check(mi, max_kv_len=1500)
    Case(dev, [600, 700], [2600, 700], 1100, 4, Hq=4, Hkv=1, seed=2).check(mi, max_kv_len=200000)


@pytest.mark.parametrize("fp8", [False, True])
def test_scales_of_every_size_and_sign(mi, dev, fp8):
    """Small scales (a probability times one is subnormal in fp16), a large one, negative ones, zeros and NaN."""
    if not fp8:
        return
    for dtype in (BF16, FP16):
        for d in (64, 128):
            for new, lens in ((None, [500, 130]), ([66, 9], [500, 130])):
                c = Case(dev, new, lens, 200, 70, d=d, dtype=dtype, fp8=True, seed=5)
                for s in c.scales:
                    s[0::4] *= 1e-2
                    s[1::4] *= -1
                    s[2::8] = 0
                c.check(mi)
                c.scales[0][c.table[0, 7], 0] = math.nan
                c.scales[1][c.table[0, 0], 1] = math.nan
                c.check(mi)


@pytest.mark.parametrize("scale", [255.0, 256.0, 300.0, 511.9, 512.0, 1000.0, 30000.0])
@pytest.mark.parametrize("d,dtype", [(64, FP16), (128, FP16), (128, BF16)])
@pytest.mark.parametrize("form", ["decode", "prompts"])
def test_large_value_scales(mi, dev, form, d, dtype, scale):
    """Values beyond what fp16 holds, whose weighted sums it holds: e4m3 numbers times a scale of 256 and more, beside chunks of small scales."""
    new, lens = (None, [500, 130]) if form == "decode" else ([66, 9], [500, 130])
    for every in (1, 3):
        c = Case(dev, new, lens, 400, 70, d=d, dtype=dtype, fp8=True, seed=15)
        if scale > 5000:   # (sums within fp16's range as well)
            c.v = (c.v.float() / 50).to(c.v.dtype)
        c.scales[1][::every] = scale
        for grid in (0, 5):
            with mi.ops.tuning(decode_grid=grid):
                got = c.run(mi)
            if dtype == FP16:   # (65 520 and more round to infinity there, and 64 bits hold them: infinities of the right sign are right)
                wide, far = got.cpu().double().view(c.q.shape), c.reference()[0]
                beyond = (far.abs() >= 65504) & torch.isinf(wide) & (wide.sign() == far.sign())
                got = torch.where(beyond, far, wide)
            c.check(mi, got=got)


def _spoil(c, r, pos, key, value):
    """Put something that is no number into a token's key or value, all heads."""
    chunk, at = int(c.table[r, pos // c.chunk]), pos % c.chunk
    if key is not None:
        c.k[chunk, at] = torch.full(c.k.shape[2:], key).to(c.k.dtype)
    if value is not None:
        c.v[chunk, at, :, ::2] = torch.full((c.v.shape[2], c.d // 2), value).to(c.v.dtype)


@pytest.mark.parametrize("d,dtype,fp8,chunk", [(128, BF16, False, 64), (64, FP16, False, 64), (128, FP16, True, 64), (64, BF16, True, 64),
                                               (96, BF16, False, 64), (256, FP16, False, 64), (128, BF16, False, 16), (192, BF16, False, 48)])
@pytest.mark.parametrize("form", ["decode", "prompts"])
def test_what_a_row_does_not_see_does_not_reach_it(mi, dev, d, dtype, fp8, chunk, form):
    """NaN and infinities before the window, between sinks and window and behind a row meet the rows that see them and no others."""
    new, lens = (None, [300, 260, 40]) if form == "decode" else ([100, 33, 40], [300, 260, 40])
    c = Case(dev, new, lens, 50, 5, d=d, dtype=dtype, fp8=fp8, chunk=chunk, seed=12)
    nan, inf = math.nan, math.nan if fp8 else math.inf
    for r, first in ((0, 250), (1, 210)):
        for pos, key, value in ((5, nan, nan), (7, inf, inf), (100, nan, inf), (first - 1, nan, nan), (first - 2, -inf, inf)):
            _spoil(c, r, pos, key, value)
    if form == "prompts":
        for r, n in ((0, 300), (1, 260)):
            _spoil(c, r, n - 1, nan, nan)
            _spoil(c, r, n - 3, None, -inf)
        _spoil(c, 2, 20, nan, None)
        _spoil(c, 2, 30, None, inf)
    got = c.check(mi)
    if form == "decode":
        assert torch.isfinite(got).all()
        with mi.ops.tuning(decode_grid=5):
            c.check(mi)
    else:
        assert torch.isfinite(got[:99 - 55]).any() and torch.isfinite(got[133:153]).all() and not torch.isfinite(got[153:]).any()
        with mi.ops.tuning(prefill_kv_split=3):
            c.check(mi, one_row_requests=False)


@pytest.mark.parametrize("form", ["decode", "prompts"])
def test_infinite_scores(mi, dev, form):
    """Keys of -inf are worth nothing, before and behind finite ones; one of +inf leaves no number."""
    c = Case(dev, None if form == "decode" else [70], [300], 150, 3, Hq=2, Hkv=1, seed=4)
    c.q = c.q.abs()
    for pos in list(range(150, 190)) + [0, 230, 299 if form == "decode" else 250]:
        _spoil(c, 0, pos, -math.inf, None)
    c.check(mi)
    _spoil(c, 0, 299, math.inf, None)
    c.check(mi)


@pytest.mark.parametrize("d,fp8", [(128, False), (64, True), (256, False)])
@pytest.mark.parametrize("grid", [7, 9, 17, 25, 40])
def test_a_part_of_nothing_but_nan_reaches_the_result(mi, dev, grid, d, fp8):
    """A key that is no number, in the first, a middle or the last of the parts that a request is cut into: its part's sum is NaN, and so
    is the row, also where the merge has that part in a group of its own."""
    for pos in (0, 7, 700, 1151, 1300, 1499):
        c = Case(dev, None, [1500], 1480, 20, Hq=4, Hkv=2, d=d, fp8=fp8, seed=pos)
        _spoil(c, 0, pos, math.nan, None)
        with mi.ops.tuning(decode_grid=grid):
            assert c.check(mi).isnan().all()


def test_chunks_out_of_sight_need_not_exist(mi, dev):
    """Table entries of chunks that no row sees: anything, ids outside the cache among it."""
    for form in ("decode", "prompts"):
        for fp8 in (False, True):
            c = Case(dev, None if form == "decode" else [30], [1000], 130, 70, fp8=fp8, seed=8)
            first = 1000 - (130 if form == "decode" else 159)
            for i in range(2, first // 64):
                c.table[0, i] = (-5, 1 << 30, -(1 << 31), (1 << 31) - 1)[i % 4]
            c.check(mi)
            with mi.ops.tuning(decode_grid=9, prefill_kv_split=4):
                c.check(mi)


def test_strides_and_outputs_given(mi, dev):
    """Rows of a wider tensor, a layer of the context's buffer, a result in place; the same as from contiguous ones."""
    for form in ("decode", "prompts"):
        c = Case(dev, None if form == "decode" else [40, 1], [200, 333], 100, 4, seed=6, dtype=FP16)
        args, more = c.inputs()
        run = mi.ops.paged_decode_attention if form == "decode" else mi.ops.paged_prefill_attention
        plain = run(*args, **more)
        wide = torch.zeros(args[0].size(0), 3, *args[0].shape[1:], dtype=FP16, device=dev)
        wide[:, 1] = args[0]
        pool = torch.full((2, 3, *args[1].shape), math.nan, dtype=FP16, device=dev)
        pool[0, 1], pool[1, 1] = args[1], args[2]
        out = torch.full((args[0].size(0), 1, args[0].size(1), args[0].size(2) * 2), 7.0, dtype=FP16, device=dev)
        got = run(wide[:, 1].unsqueeze(1), pool[0, 1], pool[1, 1], *args[3:], out=out[..., :128], **more)
        assert got.data_ptr() == out.data_ptr() and torch.equal(got.squeeze(1), plain) and (out[..., 128:] == 7).all()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("form", ["decode", "prompts"])
def test_one_row_of_the_table_for_every_request(mi, dev, form, fp8):
    """Requests over the same tokens: a table expanded over them (stride 0), with a window as without one."""
    c = Case(dev, None if form == "decode" else [40, 1, 70], [500, 300, 411], 130, 5, fp8=fp8, seed=13)
    c.table = c.table[:1].expand(3, -1)
    args, more = c.inputs()
    args[-1] = args[-1][0].expand(3, -1)
    assert args[-1].stride(0) == 0
    run = mi.ops.paged_decode_attention if form == "decode" else mi.ops.paged_prefill_attention
    c.check(mi, got=run(*args, **more))
    with mi.ops.tuning(decode_grid=5):
        c.check(mi, got=run(*args, **more))
    more.update(window=None, sinks=0)
    c.window, c.sinks = 1000, 0
    c.check(mi, got=run(*args, **more))


def test_a_cache_of_more_than_four_gibibytes(mi, dev):
    """Chunks on both sides of 2^32 bytes."""
    chunk, Hkv, d = 256, 8, 128
    n = (5 << 30) // (chunk * Hkv * d * 2)
    gen = torch.Generator(device=dev).manual_seed(1)
    k, v = (torch.zeros(n, chunk, Hkv, d, dtype=BF16, device=dev) for _ in "kv")
    ids = [n - 1, 3, n // 2 + 7, n - 2, 0, n - 9]
    for x in (k, v):
        for i in ids:
            x[i].normal_(generator=gen)
    table = torch.tensor([ids, ids[::-1]], dtype=torch.int32, device=dev)
    small = torch.tensor([list(range(6)), list(range(5, -1, -1))], dtype=torch.int32, device=dev)
    ks, vs = k[ids], v[ids]
    lens = torch.tensor([1400, 1536], dtype=torch.int32, device=dev)
    q = torch.empty(2, 32, d, dtype=BF16, device=dev).normal_(generator=gen)
    a = mi.ops.paged_decode_attention(q, k, v, lens, table, window=700, sinks=300)
    b = mi.ops.paged_decode_attention(q, ks, vs, lens, small, window=700, sinks=300)
    assert torch.equal(a, b)
    cu = torch.tensor([0, 90, 150], dtype=torch.int32, device=dev)
    q = torch.empty(150, 32, d, dtype=BF16, device=dev).normal_(generator=gen)
    a = mi.ops.paged_prefill_attention(q, k, v, cu, lens, table, window=700, sinks=300)
    b = mi.ops.paged_prefill_attention(q, ks, vs, cu, lens, small, window=700, sinks=300)
    assert torch.equal(a, b)


def test_captured_calls(mi, dev):
    """A graph of both forms replayed over changed lengths and inputs, eager work in between; two graphs in two buffers."""
    c = Case(dev, [50, 1, 20], [400, 300, 20], 90, 4, seed=9)
    e = Case(dev, None, [400, 300, 20], 90, 4, seed=10)
    (pa, pm), (da, dm) = c.inputs(), e.inputs()
    graphs = []
    for _ in range(2):
        buffer = torch.empty(64 << 20, dtype=torch.uint8, device=dev)
        outs = [torch.empty_like(pa[0]), torch.empty_like(da[0])]

        def step():
            with mi.ops.use_workspace(buffer):
                mi.ops.paged_prefill_attention(*pa, out=outs[0], **pm)
                mi.ops.paged_decode_attention(*da, out=outs[1], **dm)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step()
        graphs.append((g, outs, buffer))
    for turn in range(4):
        da[3].copy_(torch.tensor([400 - 90 * turn, 300 - turn, 20], dtype=torch.int32))
        pa[0].mul_(-0.9)
        torch.cuda.synchronize()
        for g, outs, _ in graphs:
            for o in outs:
                o.fill_(3.0)
            g.replay()
        torch.cuda.synchronize()
        want = [mi.ops.paged_prefill_attention(*pa, **pm), mi.ops.paged_decode_attention(*da, **dm)]
        torch.cuda.synchronize()
        for _, outs, _ in graphs:
            assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_two_streams_at_once(mi, dev):
    cases = [Case(dev, None, [3000, 2500], 2000, 4, seed=s) for s in (1, 2)]
    want = [c.run(mi) for c in cases]
    torch.cuda.synchronize()
    inputs, streams = [c.inputs() for c in cases], [torch.cuda.Stream() for _ in cases]
    got = []
    torch.cuda.synchronize()
    for _ in range(5):
        for (args, more), s in zip(inputs, streams):
            with torch.cuda.stream(s):
                got.append(mi.ops.paged_decode_attention(*args, **more))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i % 2]) for i, g in enumerate(got))


def test_the_same_bits_every_time(mi, dev):
    for c in (Case(dev, None, [900, 33, 512], 600, 4, seed=3), Case(dev, [100, 64], [900, 64], 300, 4, seed=3)):
        args, more = c.inputs()
        run = mi.ops.paged_decode_attention if c.decode else mi.ops.paged_prefill_attention
        first = run(*args, **more)
        assert all(torch.equal(run(*args, **more), first) for _ in range(5))


def test_a_window_over_everything_is_the_ordinary_call(mi, dev):
    for new, lens in ((None, [500, 77]), ([40, 80], [500, 80])):
        c = Case(dev, new, lens, 1 << 62, 0, seed=7)
        a, b = c.run(mi), c.run(mi, window=None)
        c.check(mi, got=a)
        c.check(mi, got=b)
        c.sinks = 9
        c.check(mi)


@pytest.mark.parametrize("seed", range(40))
def test_drawn_cases(mi, dev, seed):
    rng = random.Random(seed)
    Hq, Hkv = rng.choice(((8, 2), (4, 4), (7, 1), (6, 3), (20, 1)))
    fp8 = rng.random() < 0.3
    d = rng.choice((64, 128)) if fp8 else rng.choice((64, 96, 128, 192, 256))
    decode = rng.random() < 0.5
    chunk = rng.choice((64, 128, 256)) if fp8 and not decode else rng.choice((16, 32, 48, 64, 80, 128, 256))
    n = rng.randint(1, 5)
    new = [rng.choice((1, 2, 17, 40, 90)) for _ in range(n)]
    lens = [k + rng.choice((0, 1, 63, 200, 500)) for k in new]
    window, sinks = rng.choice((1, 2, 15, 16, 17, 63, 64, 65, 100, 128, 300)), rng.choice((0, 1, 4, 16, 63, 64, 65, 130))
    c = Case(dev, None if decode else new, lens, window, sinks, Hq=Hq, Hkv=Hkv, d=d, chunk=chunk, fp8=fp8,
             dtype=rng.choice((BF16, FP16)), seed=seed, spare=0 if decode else rng.choice((0, 3)))
    c.check(mi)
    knobs = dict(decode_grid=rng.choice((1, 2, 9, 50)), prefill_kv_split=rng.choice((-1, 2, 4)))
    with mi.ops.tuning(**knobs):
        c.check(mi)


@pytest.mark.parametrize("d", [64, 128])
def test_a_buffer_sized_for_the_window(mi, dev, d):
    """``prefill_workspace_bytes`` with the call's window is what the call takes, where that is more than without one as well."""
    c = Case(dev, [9, 7], [560, 570], 189, 4, Hq=32, Hkv=8, d=d, seed=d)
    need = mi.ops.prefill_workspace_bytes(16, 2, 32, 8, d, 576, window=189, sinks=4)
    assert need > mi.ops.prefill_workspace_bytes(16, 2, 32, 8, d, 576)
    with mi.ops.use_workspace(torch.empty(need, dtype=torch.uint8, device=dev)):
        c.check(mi, max_kv_len=576)
    with mi.ops.use_workspace(torch.empty(need - 1, dtype=torch.uint8, device=dev)), pytest.raises(ValueError, match="too small"):
        c.run(mi, max_kv_len=576)
