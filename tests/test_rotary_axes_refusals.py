"""Calls with rotary axes that are refused before anything is enqueued, and the axes of pairs: no GPU is needed."""
import ctypes

import pytest
import torch

P = 1 << 20   # an aligned address that is never read: every call here is refused
PAIRS = (ctypes.c_uint8 * 64)(*([0] * 16 + [1] * 24 + [2] * 24))


def _error(mi, rc, word):
    assert rc < 0, rc
    assert word in mi._lib.load().mi_last_error().decode(), mi._lib.load().mi_last_error()


def _split(mi, **change):
    a = dict(q=P, qst=1024, qo=P, qost=1024, k=P, kst=1024, ko=None, kost=0, v=P, vst=1024, qw=None, kw=None, eps=1e-5, norm=0, emb=P, est=128,
             rows=100, rot=128, inter=0, ms=1.0, pos=P, pst=5, axes=3, pairs=PAIRS, kc=P, vc=P, sc=65536, st=1024, ci=P, lp=P, bt=None, bts=0,
             lens=None, chunk=64, T=5, Hq=8, Hkv=8, d=128, faith=1, dtype=0, tune=None, stream=None)
    assert not set(change) - set(a)
    a.update(change)
    return mi._lib.load().mi_norm_rope_append_axes(*a.values())


def _mixed(mi, **change):
    a = dict(m=P, mst=12 * 128, qo=P, qost=1024, ko=None, kost=0, qw=None, kw=None, eps=1e-5, norm=0, emb=P, est=128, rows=100,
             rot=128, inter=0, ms=1.0, pos=P, pst=5, axes=3, pairs=PAIRS, kc=P, vc=P, sc=65536, st=1024, ci=P, lp=P, bt=None, bts=0,
             lens=None, chunk=64, T=5, Hq=8, Hkv=2, d=128, faith=1, dtype=0, tune=None, stream=None)
    assert not set(change) - set(a)
    a.update(change)
    return mi._lib.load().mi_qkv_norm_rope_append_axes(*a.values())


BOTH = [
    (dict(emb=None), "missing"), (dict(pos=None), "missing"), (dict(pairs=None), "missing"), (dict(axes=0), "axes"), (dict(axes=5), "axes"),
    (dict(axes=2), "among"), (dict(pst=4), "overlap"), (dict(rows=0), "no row"), (dict(rot=127), "rot_dim"), (dict(rot=258), "rot_dim"),
    (dict(rot=0), "rot_dim"), (dict(est=64), "rot_dim"), (dict(T=-1), "sizes"), (dict(d=80, rot=80), "head_dim"), (dict(norm=7), "norm"),
    (dict(dtype=2), "dtype"), (dict(ci=None), "slots"), (dict(vc=None), "v_cache"), (dict(qo=None), "missing"),
]


@pytest.mark.parametrize("change,word", BOTH + [(dict(k=None), "missing"), (dict(Hq=0, Hkv=0), "sizes")])
def test_split(mi, change, word):
    _error(mi, _split(mi, **change), word)


@pytest.mark.parametrize("change,word", BOTH + [(dict(m=None), "missing"), (dict(Hq=9), "multiple"), (dict(mst=1024), "stride"),
                                                (dict(kc=None), "destination")])
def test_mixed(mi, change, word):
    _error(mi, _mixed(mi, **change), word)


def test_no_tokens_is_a_no_op(mi):
    assert _split(mi, T=0, q=None) == 0 and _mixed(mi, T=0, m=None) == 0


def test_axes_of_pairs(mi):
    axes = mi.ops.rotary_axes
    assert axes((2, 1, 1)) == bytes([0, 0, 1, 2]) and axes((3,)) == bytes(3)
    assert axes((4, 2, 2), alternate=True) == bytes([0, 1, 2, 0, 1, 2, 0, 0])
    assert axes((24, 20, 20), alternate=True)[:60] == bytes([0, 1, 2] * 20)
    for bad in ((), (0, 0), (1, 2, 3, 4, 5), (4, -1)):
        with pytest.raises(ValueError):
            axes(bad)
    with pytest.raises(ValueError, match="turns"):
        axes((1, 4, 1), alternate=True)


def test_arguments_are_checked(mi):
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    table, pos, pairs = torch.zeros(9, 64), torch.zeros(3, 4, dtype=torch.int64), mi.ops.rotary_axes((12, 10, 10))
    run = mi.ops.norm_rope_append
    with pytest.raises(ValueError, match="one set of positions"):
        run(x, None, rotary_emb=table, q_positions=pos, k_positions=pos[0], rotary_axes=pairs)
    with pytest.raises(ValueError, match="one per rotary pair"):
        run(x, None, rotary_emb=table, q_positions=pos, rotary_axes=pairs[1:])
    with pytest.raises(ValueError, match="one per rotary pair"):
        run(x, None, rotary_emb=table, q_positions=pos, rotary_axes=(0,) * 32)
    with pytest.raises(ValueError, match="axes, >= T"):
        run(x, None, rotary_emb=table, q_positions=pos[:, :3], rotary_axes=pairs)
    with pytest.raises(ValueError, match="axes, >= T"):
        run(x, None, rotary_emb=table, q_positions=pos[0], rotary_axes=pairs)
    with pytest.raises(ValueError, match="need rotary_emb"):
        run(x, None, q_positions=pos, rotary_axes=pairs)
    with pytest.raises(RuntimeError, match="no CPU path"):
        run(x, None, rotary_emb=table, q_positions=pos, rotary_axes=pairs)
