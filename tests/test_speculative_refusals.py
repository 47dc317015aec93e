"""Calls of the speculative operators that are refused before anything is enqueued: no GPU is needed."""
import ctypes

import pytest
import torch

P = 1 << 20   # an aligned address that is never read: every call here is refused


def _error(mi, rc, word):
    assert rc < 0, rc
    assert word in mi._lib.load().mi_last_error().decode(), mi._lib.load().mi_last_error()


def _tree(mi, **change):
    a = dict(q=P, qst=1024, qsh=128, k=P, v=P, sc=65536, st=1024, sh=128, n=4, kv=0, ks=None, vs=None, bt=P, bts=4, cols=4,
             cu=P, lens=P, mask=P, mst=1, words=1, out=P, ost=1024, osh=128, ws=P, wsb=1 << 40, T=5, R=1, Hq=8, Hkv=8, d=128,
             chunk=64, scale=0.1, dtype=0, stream=None)
    assert not set(change) - set(a)
    a.update(change)
    return mi._lib.load().mi_paged_tree_attention(*a.values())


@pytest.mark.parametrize("change,word", [
    (dict(q=None), "null"), (dict(mask=None), "null"), (dict(cu=None), "null"), (dict(T=-1), "T >= 0"), (dict(R=0), "R > 0"),
    (dict(Hq=12), "multiple"), (dict(Hq=65 * 8), "64 query heads"), (dict(d=80), "head_dim"), (dict(d=96, kv=1, ks=P, vs=P), "fp8"),
    (dict(kv=1), "scale"), (dict(kv=2), "kv_dtype"), (dict(chunk=24), "multiple of 16"), (dict(n=0), "cache"),
    (dict(cols=1 << 26), "2^31"), (dict(words=0), "words"), (dict(words=5, mst=5), "words"), (dict(words=2, mst=1), "words"),
    (dict(q=P + 8), "aligned"), (dict(qst=1028), "aligned"), (dict(st=1 << 25), "2 GiB"), (dict(scale=0.0), "positive"),
    (dict(scale=float("nan")), "positive"), (dict(ws=None), "workspace"), (dict(wsb=16), "workspace"), (dict(ws=P + 4), "aligned"),
    (dict(dtype=2), "dtype"),
])
def test_tree_attention(mi, change, word):
    _error(mi, _tree(mi, **change), word)


def test_tree_attention_of_no_rows_is_a_no_op(mi):
    assert _tree(mi, T=0, q=None) == 0
    assert mi._lib.load().mi_tree_workspace_bytes(0, 4, 8, 8, 128) == 0
    assert mi._lib.load().mi_tree_workspace_bytes(5, 1, 8, 8, 128) > 0


def _verify(mi, **change):
    a = dict(logits=P, st=1000, dt=1, T=5, V=1000, tok=P, par=P, cu=P, R=1, path=3, greedy=0, draft=None, dst=0, ddt=0, u=P, temp=1.0,
             cut=None, ot=P, orows=P, oc=P, ws=P, wsb=1 << 40, stream=None)
    assert not set(change) - set(a)
    a.update(change)
    return mi._lib.load().mi_verify_drafted_tokens(*a.values())


@pytest.mark.parametrize("change,word", [
    (dict(logits=None), "null"), (dict(tok=None), "null"), (dict(par=None), "null"), (dict(cu=None), "null"), (dict(oc=None), "null"),
    (dict(T=-1), "T >= 0"), (dict(path=0), "max_path"), (dict(V=0), "vocab"), (dict(st=999), "stride"), (dict(V=600000, st=600000), "vocab"),
    (dict(dt=3), "fp32"), (dict(ddt=3), "fp32"), (dict(greedy=1, cut=P), "greedy"), (dict(greedy=1, draft=P, dst=1000), "greedy"),
    (dict(u=None), "uniform"), (dict(temp=0.0), "temperature"), (dict(draft=P, dst=10), "stride"), (dict(logits=P + 1), "aligned"),
    (dict(ws=None), "workspace"), (dict(wsb=16), "workspace"), (dict(ws=P + 8), "aligned"),
])
def test_verification(mi, change, word):
    _error(mi, _verify(mi, **change), word)


def test_verification_of_no_requests_is_a_no_op(mi):
    assert _verify(mi, R=0, cu=None) == 0


def _keep(mi, **change):
    a = dict(k=P, v=P, sl=1 << 20, sc=65536, st=1024, L=2, n=4, chunk=64, H=8, d=128, esz=2, ks=None, vs=None, ssl=0, bt=P, bts=4, cols=4,
             rows=P, rst=4, columns=4, counts=P, cu=P, lens=P, new=P, R=1, stream=None)
    assert not set(change) - set(a)
    a.update(change)
    return mi._lib.load().mi_kv_keep_accepted(*a.values())


@pytest.mark.parametrize("change,word", [
    (dict(k=None), "null"), (dict(new=None), "null"), (dict(L=0), "sizes"), (dict(chunk=0), "sizes"), (dict(columns=-1), "sizes"),
    (dict(esz=4), "bytes"), (dict(esz=1), "scales"), (dict(ks=P), "scales"), (dict(esz=1, ks=P), "scales"),
    (dict(H=1, d=12), "16-byte"), (dict(esz=1, ks=P, vs=P, d=8), "16-byte"), (dict(k=P + 8), "aligned"), (dict(st=1028), "aligned"),
])
def test_keep_accepted(mi, change, word):
    _error(mi, _keep(mi, **change), word)


def test_keep_accepted_of_no_requests_is_a_no_op(mi):
    assert _keep(mi, R=0, k=None) == 0


def test_cpu_tensors_raise(mi):
    z = torch.zeros
    i32, i64 = dict(dtype=torch.int32), dict(dtype=torch.int64)
    cache = z(2, 16, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        mi.ops.paged_tree_attention(z(1, 1, 64, dtype=torch.bfloat16), cache, cache, z(2, **i32), z(1, **i32), z(1, 1, **i32), z(1, **i64))
    with pytest.raises(RuntimeError, match="no CPU path"):
        mi.ops.verify_drafted_tokens(z(1, 8), z(1, **i64), z(1, **i32), z(2, **i32), 1, greedy=True)
    with pytest.raises(RuntimeError, match="no CPU path"):
        mi.ops.kv_keep_accepted(cache, cache, z(1, 1, **i32), z(1, **i32), z(2, **i32), z(1, **i32), z(1, 1, **i32))


def test_trees_that_are_none(mi):
    with pytest.raises(ValueError, match="precedes"):
        mi.ops.tree_masks([-1, 1])
    with pytest.raises(ValueError, match="256"):
        mi.ops.tree_masks(range(-1, 256))
    assert mi.ops.tree_masks([]).shape == (0, 1)
    assert isinstance(ctypes.c_int64(int(mi.ops.tree_masks(range(-1, 255))[255, 3])).value, int)


@pytest.mark.parametrize("cols,chunk", [(1 << 25, 16), ((1 << 24) + 1, 64), ((1 << 24) + 5, 32)])
def test_tables_of_too_many_columns(mi, cols, chunk):
    """A token's chunk is its number times 2^40 / chunk in 64 bits, which hold fewer than 2^24 chunks: from there on it would be
    another one, and reads would go astray."""
    assert cols * chunk <= 0x7fffff00 and cols * chunk * chunk < 1 << 40
    assert (cols * chunk - 1) * -(-(1 << 40) // chunk) >= 1 << 64
    _error(mi, _tree(mi, cols=cols, chunk=chunk), "2^24")


@pytest.mark.parametrize("cols,chunk", [((1 << 23) - 1, 256), (8947847, 240)])
def test_tables_of_almost_two_to_the_31_tokens(mi, cols, chunk):
    """A wavefront's next tile lies up to 512 tokens on (every eighth of 64), and its number has 32 bits behind the last token too."""
    assert cols < 1 << 24 and cols * chunk < 1 << 31 <= cols * chunk + 512
    _error(mi, _tree(mi, cols=cols, chunk=chunk), "2^31")
