"""GPU parity: head norm, rotary embedding with several axes and append against the 64-bit oracle.

Tolerance, element by element, with u half a step of the 16-bit type: rounded once, u |o| and 2e-6 of the two terms for the
32-bit norm, angles and products; with faithful rounding each term carries the rounding of the normed value, of its cos or sin
and of their product (3 u, and second-order terms), and their sum one more.  1e-7 beside it for subnormal fp16.
"""
import math
import random

import pytest
import torch

from oracle import windows as ow

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def _sections(pairs, axes):
    cut = [pairs * i // axes for i in range(axes + 1)]
    return [b - a for a, b in zip(cut, cut[1:])]


class Case:
    def __init__(self, dev, T, *, Hq=8, Hkv=2, d=128, rot=None, sections=None, alternate=False, interleaved=False, norm="rms",
                 dtype=BF16, chunk=64, seed=0, most=300, mscale=1.0, twisted=False):
        gen = torch.Generator().manual_seed(seed)
        rot = d if rot is None else rot
        self.T, self.Hq, self.Hkv, self.d, self.rot, self.dtype, self.dev = T, Hq, Hkv, d, rot, dtype, dev
        self.interleaved, self.norm, self.mscale, self.chunk = interleaved, norm, mscale, chunk
        sections = _sections(rot // 2, 3) if sections is None else sections
        self.axes = ow.axes_of_pairs(sections, alternate)
        self.positions = torch.randint(0, most, (len(sections), T), generator=gen)
        inv = 10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64) / (rot // 2))
        angles = (torch.arange(most)[:, None] * inv).float()
        self.table = angles.repeat_interleave(2, 1) if interleaved else torch.cat([angles, angles], 1)
        if twisted:   # the two elements of a pair with columns of their own
            self.table = self.table + torch.rand(self.table.shape, generator=gen)
        group = Hq // Hkv if Hkv and Hq % Hkv == 0 else 0
        self.group = group
        self.q = torch.randn(T, Hq, d, generator=gen).to(dtype) if Hq else None
        self.k = torch.randn(T, Hkv, d, generator=gen).to(dtype) if Hkv else None
        self.v = torch.randn(T, Hkv, d, generator=gen).to(dtype) if Hkv else None
        self.weights = [(1 + 0.1 * torch.randn(d, generator=gen)).to(dtype) if norm == "rms" else None for _ in "qk"]
        n = T // chunk + 3
        slots = torch.randperm(n * chunk, generator=gen)[:T]
        self.n, self.slots = n, (slots // chunk, slots % chunk)

    def common(self, mi, **over):
        dev = self.dev
        more = dict(q_weight=None if self.weights[0] is None else self.weights[0].to(dev),
                    k_weight=None if self.weights[1] is None else self.weights[1].to(dev), eps=1e-5, norm=self.norm,
                    rotary_emb=self.table.to(dev), q_positions=self.positions.to(dev), rotary_axes=bytes(self.axes),
                    rotary_interleaved=self.interleaved, mscale=self.mscale)
        more.update(over)
        return more

    def caches(self):
        return [torch.full((self.n, self.chunk, self.Hkv, self.d), 9.0, dtype=self.dtype, device=self.dev) for _ in "kv"]

    def reference(self, x, weight):
        args = (self.positions.clamp(0, self.table.size(0) - 1), self.table, self.axes)
        out = ow.norm_rotate(x, *args, norm=self.norm, weight=weight, interleaved=self.interleaved, mscale=self.mscale)
        pairs = len(self.axes)   # what the two terms of an element come to at most, from the normed values
        y = x.double() / torch.sqrt(x.double().square().mean(-1, keepdim=True) + 1e-5) if self.norm in ("rms", "l2") else x.double()
        if weight is not None:
            y = y * weight.double()
        size = y.abs().clone()
        terms = y.abs().clone()
        for i, axis in enumerate(self.axes):
            a, b = (2 * i, 2 * i + 1) if self.interleaved else (i, i + pairs)
            for e, o in ((a, b), (b, a)):
                angle = self.table[self.positions.clamp(0, self.table.size(0) - 1)[axis], e].double()[:, None]
                terms[..., e] = (y[..., e] * angle.cos()).abs() * self.mscale + (y[..., o] * angle.sin()).abs() * self.mscale
                size[..., e] = (y[..., a].abs() + y[..., b].abs()) * max(1.0, self.mscale)
        return out, terms, size

    def close(self, got, x, weight, faithful):
        ref, terms, size = self.reference(x, weight)
        u, err = torch.finfo(self.dtype).eps / 2, (got.cpu().double().view(ref.shape) - ref).abs()
        bound = u * ref.abs() + 2e-6 * size + 1e-7
        if faithful:
            bound = bound + 3.1 * u * terms * (1 + u)
        assert (err <= bound).all(), f"max err / bound {(err / bound).max():.3f}"

    def check(self, mi, *, faithful=False, mixed=False, decode=False, key_out=False, to_cache=True, tuned=0):
        dev, kc_vc = self.dev, self.caches()
        kc, vc = kc_vc
        q_out = torch.full((self.T, 1, self.Hq, self.d), 5.0, dtype=self.dtype, device=dev) if self.Hq else None
        k_out = torch.full((self.T, self.Hkv, self.d), 5.0, dtype=self.dtype, device=dev) if key_out else None
        more = self.common(mi, faithful_rounding=faithful, query_out=q_out, key_out=k_out)
        rows = self.slots
        if to_cache:
            more.update(k_cache=kc, v_cache=vc)
            if decode:
                lens = torch.tensor([(7 * i) % (self.chunk + 1) for i in range(self.T)])
                more.update(block_table=torch.arange(self.T, dtype=torch.int32)[:, None].to(dev), kv_lens=lens.int().to(dev))
            else:
                more.update(token_to_chunk_idx=rows[0].to(dev), token_to_local_pos=rows[1].to(dev))
        with mi.ops.tuning(norm_rope_vectorised=tuned):
            if mixed:
                both = torch.cat([self.q.view(self.T, self.Hkv, self.group, self.d), self.k[:, :, None], self.v[:, :, None]], 2)
                mi.ops.qkv_norm_rope_append(both.reshape(self.T, 1, -1).to(dev), num_query_heads=self.Hq, num_kv_heads=self.Hkv, **more)
            else:
                on = lambda x: None if x is None else x.to(dev)  # noqa: E731
                mi.ops.norm_rope_append(on(self.q), on(self.k), value=on(self.v) if to_cache else None, **more)
        torch.cuda.synchronize()
        if self.Hq:
            self.close(q_out, self.q, self.weights[0], faithful)
        if key_out:
            self.close(k_out, self.k, self.weights[1], faithful)
        if to_cache:
            if decode:
                live = lens > 0
                rows = (torch.arange(self.T)[live], (lens - 1)[live])
                every = torch.arange(self.T)[live]
            else:
                every = torch.arange(self.T)
            kc, vc = kc.cpu(), vc.cpu()
            assert torch.equal(vc[rows], self.v[every])
            written = torch.zeros(kc.shape[:2], dtype=torch.bool)
            written[rows] = True
            assert (kc[~written] == 9).all() and (vc[~written] == 9).all()
            full = torch.zeros_like(self.k)
            full[every] = kc[rows]
            ref, terms, size = self.reference(self.k, self.weights[1])
            u, err = torch.finfo(self.dtype).eps / 2, (full.double() - ref).abs()[every]
            bound = (u * ref.abs() + 2e-6 * size + 1e-7 + (3.1 * u * terms * (1 + u) if faithful else 0))[every]
            assert (err <= bound).all(), f"max err / bound {(err / bound).max():.3f}"
            if key_out:
                assert torch.equal(k_out.cpu()[every], full[every])


@pytest.mark.parametrize("faithful", [False, True])
@pytest.mark.parametrize("T", [1, 2, 3, 64, 257, 1000])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_tokens(mi, dev, T, faithful, dtype):
    c = Case(dev, T, dtype=dtype, seed=T)
    c.check(mi, faithful=faithful)
    c.check(mi, faithful=faithful, mixed=True, key_out=True)


@pytest.mark.parametrize("Hq,Hkv,d", [(32, 8, 128), (8, 8, 64), (7, 1, 96), (12, 4, 192), (16, 2, 256), (5, 5, 128), (64, 1, 64), (24, 3, 96)])
@pytest.mark.parametrize("norm", ["rms", "l2", None])
def test_head_layouts(mi, dev, Hq, Hkv, d, norm):
    for faithful in (False, True):
        Case(dev, 33, Hq=Hq, Hkv=Hkv, d=d, norm=norm, seed=d).check(mi, mixed=True, faithful=faithful)


@pytest.mark.parametrize("d,rot", [(128, 64), (128, 32), (128, 96), (128, 48), (128, 16), (128, 10), (64, 2), (96, 96), (96, 64), (192, 24), (256, 128),
                                   (64, 40), (256, 250)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_widths(mi, dev, d, rot, interleaved):
    for faithful in (False, True):
        sections = _sections(rot // 2, min(3, rot // 2))
        c = Case(dev, 40, d=d, rot=rot, interleaved=interleaved, sections=sections, seed=rot)
        c.check(mi, faithful=faithful)
        c.check(mi, faithful=faithful, mixed=True, tuned=-1)


@pytest.mark.parametrize("sections,alternate", [((64,), False), ((16, 24, 24), False), ((24, 20, 20), True), ((20, 20, 24), False), ((1, 62, 1), False),
                                                ((30, 2, 30, 2), False), ((16, 16, 16, 16), True), ((0, 64), False), ((44, 10, 10), True)])
def test_sections(mi, dev, sections, alternate):
    assert mi.ops.rotary_axes(sections, alternate) == bytes(ow.axes_of_pairs(sections, alternate))
    for interleaved in (False, True):
        Case(dev, 70, sections=sections, alternate=alternate, interleaved=interleaved, seed=1, mscale=1.3).check(mi, mixed=True)
        Case(dev, 70, sections=sections, alternate=alternate, interleaved=interleaved, seed=1).check(mi, faithful=True, tuned=-1)


def test_slots_of_a_decode_step(mi, dev):
    """Table and lengths name the slot; a request without tokens appends nothing."""
    for tuned in (0, -1):
        c = Case(dev, 130, chunk=64, seed=2)
        c.n = 130
        c.check(mi, decode=True, mixed=True, tuned=tuned)
        c.check(mi, decode=True, faithful=True, tuned=tuned)


def test_queries_or_keys_alone(mi, dev):
    for tuned in (0, -1):
        Case(dev, 20, Hkv=0, seed=3).check(mi, to_cache=False, tuned=tuned)
        Case(dev, 20, Hq=0, seed=3).check(mi, tuned=tuned)
        Case(dev, 20, Hq=0, seed=3).check(mi, to_cache=False, key_out=True, tuned=tuned)
        Case(dev, 20, Hq=7, Hkv=3, seed=3).check(mi, tuned=tuned)


def test_elements_with_columns_of_their_own(mi, dev):
    for interleaved in (False, True):
        Case(dev, 50, interleaved=interleaved, twisted=True, seed=4).check(mi)
        Case(dev, 50, interleaved=interleaved, twisted=True, rot=64, seed=4).check(mi, faithful=True, mixed=True)


def test_far_positions(mi, dev):
    """Angles beyond the fast reduction's range, as the table holds them."""
    c = Case(dev, 60, seed=5, most=400)
    c.table = c.table * 1e4
    c.check(mi)


def test_positions_outside_the_table_stay_in_it(mi, dev):
    c = Case(dev, 60, seed=6)
    c.positions[0, ::3], c.positions[1, 1::3], c.positions[2, ::2] = -4, 10 ** 12, 300
    for tuned in (0, -1):
        c.check(mi, mixed=True, tuned=tuned)


def test_rows_off_sixteen_bytes_and_wider_tensors(mi, dev):
    """Heads of a wider tensor, positions of a wider one, rows that start anywhere."""
    c = Case(dev, 45, seed=7)
    for shift in (8, 1):
        wide = torch.zeros(45, 8 * 128 + 32, dtype=BF16, device=dev)
        q = wide.as_strided((45, 8, 128), (wide.stride(0), 128, 1), shift)
        q.copy_(c.q)
        pos = torch.full((3, 90), -1, device=dev)
        pos[:, :45] = c.positions.to(dev)
        mi.ops.norm_rope_append(q, None, **c.common(mi, q_positions=pos, faithful_rounding=False))
        c.close(q.contiguous(), c.q, c.weights[0], False)
        assert (wide[:, :shift] == 0).all() and (wide[:, shift + 1024:] == 0).all()


def test_what_passes_through_is_untouched(mi, dev):
    """Infinities and NaN in columns beyond the rotary width stay where they are."""
    c = Case(dev, 9, rot=64, norm=None, seed=8)
    for x in (c.q, c.k):
        x[:, :, 64::7] = math.inf
        x[:, :, 65::9] = math.nan
    for tuned in (0, -1):
        for faithful in (False, True):
            out = torch.empty_like(c.q, device=dev)
            with mi.ops.tuning(norm_rope_vectorised=tuned):
                mi.ops.norm_rope_append(c.q.to(dev), None, **c.common(mi, query_out=out, faithful_rounding=faithful))
            assert torch.equal(out.cpu()[:, :, 64:].view(torch.int16), c.q[:, :, 64:].view(torch.int16)) and torch.isfinite(out[:, :, :64]).all()


def test_text_counts_alike_on_all_axes(mi, dev):
    """Equal positions on every axis are the ordinary call's, up to the order of the norm's sum."""
    c = Case(dev, 300, seed=9)
    c.positions[:] = torch.arange(300) % 299
    axes, plain = torch.empty(300, 8, 128, dtype=BF16, device=dev), torch.empty(300, 8, 128, dtype=BF16, device=dev)
    mi.ops.norm_rope_append(c.q.to(dev), None, **c.common(mi, query_out=axes))
    more = c.common(mi, query_out=plain)
    more.pop("rotary_axes")
    more["q_positions"] = more["q_positions"][0].contiguous()
    mi.ops.norm_rope_append(c.q.to(dev), None, **more)
    for x in (axes, plain):
        c.close(x, c.q, c.weights[0], True)
    assert (axes != plain).float().mean() < 0.01


@pytest.mark.parametrize("T", [1, 64, 1000])
@pytest.mark.parametrize("axes", [2, 3, 4])
def test_one_row_of_positions_for_every_axis(mi, dev, T, axes):
    """Steps of text come as one row expanded over the axes (stride 0): the same as rows of their own, in every kernel and call."""
    class Text(Case):
        def common(self, mi, **over):
            more = super().common(mi, **over)
            more["q_positions"] = more["q_positions"][0].expand(axes, T)
            assert more["q_positions"].stride(0) == 0
            return more
    c = Text(dev, T, sections=_sections(64, axes), seed=T)
    c.positions[:] = c.positions[:1].clone()
    for tuned in (0, -1):
        c.check(mi, tuned=tuned)
        c.check(mi, mixed=True, faithful=True, tuned=tuned)


def test_many_tokens(mi, dev):
    Case(dev, 5001, Hq=4, Hkv=1, d=64, seed=10).check(mi, mixed=True)
    Case(dev, 4500, Hq=2, Hkv=2, d=128, seed=10).check(mi, faithful=True)


def test_a_captured_call(mi, dev):
    c = Case(dev, 64, seed=11)
    both = torch.cat([c.q.view(64, 2, 4, 128), c.k[:, :, None], c.v[:, :, None]], 2).reshape(64, -1).to(dev)
    (kc, vc), out = c.caches(), torch.empty(64, 8, 128, dtype=BF16, device=dev)
    more = c.common(mi, query_out=out, k_cache=kc, v_cache=vc, token_to_chunk_idx=c.slots[0].to(dev), token_to_local_pos=c.slots[1].to(dev))

    def step():
        mi.ops.qkv_norm_rope_append(both, num_query_heads=8, num_kv_heads=2, **more)
    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for turn in range(3):
        more["q_positions"].add_(turn)
        both.mul_(0.7)
        g.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in (out, kc, vc)]
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (out, kc, vc)))


@pytest.mark.parametrize("seed", range(30))
def test_drawn_cases(mi, dev, seed):
    rng = random.Random(seed)
    d = rng.choice((64, 96, 128, 192, 256))
    rot = rng.choice((d, d, d // 2, 2 * rng.randint(1, d // 2)))
    pairs = rot // 2
    a = rng.randint(0, pairs)
    sections = rng.choice(((pairs,), (a, pairs - a), (pairs - 2 * (pairs // 3), pairs // 3, pairs // 3)))
    Hq, Hkv = rng.choice(((8, 2), (4, 4), (7, 1), (6, 3), (20, 1)))
    c = Case(dev, rng.choice((1, 5, 63, 300, 1100)), Hq=Hq, Hkv=Hkv, d=d, rot=rot, sections=sections, interleaved=rng.random() < 0.5,
             norm=rng.choice(("rms", "l2", None)), dtype=rng.choice((BF16, FP16)), chunk=rng.choice((16, 48, 256)), seed=seed)
    c.check(mi, faithful=rng.random() < 0.5, mixed=rng.random() < 0.5, key_out=rng.random() < 0.3, tuned=rng.choice((0, 0, -1, 1)))
