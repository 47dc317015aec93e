"""What pins the oracle of windows and of positions with several axes."""
import math

import torch

from oracle import paged_attention as oa
from oracle import windows as ow


def _case(new, lens, Hq=4, Hkv=2, d=8, chunk=16, seed=0):
    gen = torch.Generator().manual_seed(seed)
    need = [-(-n // chunk) for n in lens]
    N = sum(need) + 1
    ids = torch.randperm(N, generator=gen).tolist()
    table = torch.zeros(len(lens), max(max(need), 1), dtype=torch.int32)
    for r, k in enumerate(need):
        table[r, :k] = torch.tensor([ids.pop() for _ in range(k)], dtype=torch.int32)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    q = torch.randn(cu[-1], Hq, d, generator=gen)
    kc, vc = torch.randn(N, chunk, Hkv, d, generator=gen), torch.randn(N, chunk, Hkv, d, generator=gen)
    return q, kc, vc, cu, lens, table


def test_masks_by_hand():
    assert ow.visible(9, 10, 3, 0) == [7, 8, 9]
    assert ow.visible(9, 10, 3, 2) == [0, 1, 7, 8, 9]
    assert ow.visible(9, 10, 1, 0) == [9]
    assert ow.visible(4, 10, 3, 4) == [0, 1, 2, 3, 4]
    assert ow.visible(0, 10, 1, 3) == [0]
    assert ow.visible(-1, 5, 3, 2) == []
    assert ow.visible(2, 10, 100, 100) == [0, 1, 2]


def test_a_window_over_everything_is_causal_attention():
    q, kc, vc, cu, lens, table = _case([3, 1, 5], [23, 1, 12])
    ref = oa.paged_varlen_attention(q, kc, vc, torch.tensor(cu), torch.tensor(lens), table)
    for window, sinks in ((23, 0), (1 << 40, 5), (1, 23)):
        got, _, _ = ow.window_attention(q, kc, vc, cu, lens, table, window, sinks, 8 ** -0.5)
        assert (got - ref).abs().max() < 1e-5


def test_a_window_is_a_masked_softmax_and_what_is_not_seen_does_not_matter():
    q, kc, vc, cu, lens, table = _case([6], [40], seed=1)
    kc[table[0, 1]] = math.nan   # tokens 16 .. 31
    vc[table[0, 1]] = math.inf
    got, size, _ = ow.window_attention(q, kc, vc, cu, lens, table, 3, 4, 8 ** -0.5)
    k = torch.cat([kc[c] for c in table[0]])[:40].nan_to_num().double().repeat_interleave(2, 1)
    v = torch.cat([vc[c] for c in table[0]])[:40].nan_to_num(posinf=0).double().repeat_interleave(2, 1)
    x = torch.einsum("qhd,khd->hqk", q.double(), k) * 8 ** -0.5
    p, t = torch.arange(34, 40)[:, None], torch.arange(40)
    x = x.masked_fill(~((t <= p) & ((t > p - 3) | (t < 4))), -math.inf)
    ref = torch.einsum("hqk,khd->qhd", torch.softmax(x, -1), v)
    assert (got - ref).abs().max() < 1e-12 and (size >= got.abs() - 1e-12).all()


def test_axes_of_pairs():
    assert ow.axes_of_pairs((2, 1, 1)) == [0, 0, 1, 2]
    assert ow.axes_of_pairs((4, 2, 2), True) == [0, 1, 2, 0, 1, 2, 0, 0]
    assert ow.axes_of_pairs((3,)) == [0, 0, 0]


def test_rotation_in_the_plane():
    gen = torch.Generator().manual_seed(2)
    x, table = torch.randn(5, 3, 12, generator=gen), torch.rand(40, 4, generator=gen) * 7
    positions = torch.randint(0, 40, (3, 5), generator=gen)
    axes = [0, 2, 1, 2]
    for interleaved in (False, True):
        full = table.repeat_interleave(2, 1) if interleaved else torch.cat([table, table], 1)
        got = ow.norm_rotate(x, positions, full, axes, interleaved=interleaved, mscale=1.5)
        for i, axis in enumerate(axes):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + 4)
            turn = 1.5 * torch.exp(1j * table[positions[axis], i].double())[:, None]
            z = torch.complex(x[..., a].double(), x[..., b].double()) * turn
            assert (got[..., a] - z.real).abs().max() < 1e-12 and (got[..., b] - z.imag).abs().max() < 1e-12
        assert torch.equal(got[..., 8:], x[..., 8:].double())
    normed = ow.norm_rotate(x, positions, torch.cat([table, table], 1), axes, norm="l2", eps=0.0)
    assert (normed.square().mean(-1) - 1).abs().max() < 1e-12
