"""Calls with a window that are refused before anything is enqueued: no GPU is needed."""
import pytest
import torch

P = 1 << 20   # an aligned address that is never read: every call here is refused


def _error(mi, rc, word):
    assert rc < 0, rc
    assert word in mi._lib.load().mi_last_error().decode(), mi._lib.load().mi_last_error()


def _decode(mi, **change):
    a = dict(q=P, qst=1024, qsh=128, k=P, v=P, sc=65536, st=1024, sh=128, n=4, kv=0, ks=None, vs=None, bt=P, bts=4, cols=4, lens=P,
             window=100, sinks=4, out=P, ost=1024, osh=128, ws=P, wsb=1 << 40, R=2, Hq=8, Hkv=8, d=128, chunk=64, scale=0.1, dtype=0,
             tune=None, stream=None)
    assert not set(change) - set(a)
    a.update(change)
    return mi._lib.load().mi_paged_window_decode_attention(*a.values())


def _prompts(mi, **change):
    a = dict(q=P, qst=1024, qsh=128, k=P, v=P, sc=65536, st=1024, sh=128, n=4, kv=0, ks=None, vs=None, bt=P, bts=4, cols=4, cu=P, lens=P,
             window=100, sinks=4, out=P, ost=1024, osh=128, ws=P, wsb=1 << 40, T=5, R=2, Hq=8, Hkv=8, d=128, chunk=64, most=0, one=1,
             scale=0.1, dtype=0, tune=None, stream=None)
    assert not set(change) - set(a)
    a.update(change)
    return mi._lib.load().mi_paged_window_prefill_attention(*a.values())


BOTH = [
    (dict(window=0), "window"), (dict(window=-1), "window"), (dict(sinks=-1), "sinks"), (dict(n=0), "cache"), (dict(cols=0), "column"),
    (dict(bts=3), "overlap"), (dict(q=None), "null"), (dict(bt=None), "null"), (dict(lens=None), "null"), (dict(out=None), "null"),
    (dict(Hq=12), "multiple"), (dict(Hq=65 * 8), "64 query heads"), (dict(d=80), "head_dim"), (dict(d=96, kv=1, ks=P, vs=P), "fp8"),
    (dict(chunk=24), "multiple of 16"), (dict(chunk=0), "multiple of 16"), (dict(kv=2), "kv_dtype"), (dict(q=P + 8), "aligned"),
    (dict(st=1 << 25), "2 GiB"), (dict(scale=0.0), "positive"), (dict(scale=float("nan")), "positive"), (dict(dtype=2), "dtype"),
    (dict(wsb=16), "workspace"), (dict(ws=P + 4), "aligned"), (dict(cols=1 << 25, bts=1 << 25, chunk=16), "2^24"),
    (dict(cols=1 << 26, bts=1 << 26), "2^31"), (dict(cols=(1 << 23) - 1, bts=1 << 23, chunk=256), "2^31"),
    (dict(cols=(1 << 20) * 2, bts=1 << 22, chunk=1008), "power of two"),
]


@pytest.mark.parametrize("change,word", BOTH + [(dict(kv=1), "scale"), (dict(ws=None), "workspace")])
def test_decode(mi, change, word):
    _error(mi, _decode(mi, **change), word)


@pytest.mark.parametrize("change,word", BOTH + [
    (dict(cu=None), "null"), (dict(T=-1), "T, R >= 0"), (dict(kv=1), "scale"), (dict(kv=1, ks=P, vs=P, chunk=48), "multiple of 64"),
])
def test_prompts(mi, change, word):
    _error(mi, _prompts(mi, **change), word)


@pytest.mark.parametrize("call", [_decode, _prompts])
def test_more_tiles_than_32_bits_count(mi, call):
    """What all requests see, in tiles of 16 tokens, is counted in 32 bits: 2 048 requests of 2^24 tokens each are too many."""
    room = dict(cols=1 << 16, bts=1 << 16, chunk=256, sc=256 * 1024)
    _error(mi, call(mi, R=2048, window=1 << 30, **room), "2^31")
    _error(mi, call(mi, R=2048, window=1 << 23, sinks=1 << 23, **room), "2^31")
    _error(mi, call(mi, R=1 << 20, window=1 << 23, **room), "2^31")   # (slices of 7 680 requests, 2^19 tiles each)
    for fine in (dict(R=2048, window=1 << 23), dict(R=1024, window=1 << 30), dict(R=1 << 20, window=1 << 21)):
        _error(mi, call(mi, lens=None, **fine, **room), "null")   # (refused for what comes after)


def test_kernels_that_have_no_window(mi):
    import ctypes
    for knob in (1, 2):
        _error(mi, _prompts(mi, tune=ctypes.byref(mi._lib.MiTuning(prefill_two_phase=knob))), "no kernel with a window")


def test_nothing_to_do_is_a_no_op(mi):
    assert _decode(mi, R=0, q=None) == 0
    assert _prompts(mi, T=0, q=None) == 0 and _prompts(mi, R=0, q=None) == 0


def test_the_workspace_goes_by_what_is_in_sight(mi):
    lib = mi._lib.load()
    full = lib.mi_prefill_workspace_bytes(300, 1, 8, 8, 128, 100000, 0, None)
    windowed = lib.mi_window_prefill_workspace_bytes(300, 1, 8, 8, 128, 100000, 1000, 4, None)
    assert 0 < windowed < full
    assert lib.mi_window_prefill_workspace_bytes(300, 1, 8, 8, 128, 100000, 2000000000, 2000000000, None) == full
    assert lib.mi_window_prefill_workspace_bytes(300, 1, 8, 8, 128, 0, 1000, 4, None) == windowed
    for window, sinks in ((0, 4), (-5, 4), (1000, -1)):
        assert lib.mi_window_prefill_workspace_bytes(300, 1, 8, 8, 128, 100000, window, sinks, None) == -1


def _tensors():
    i32 = dict(dtype=torch.int32)
    cache = torch.zeros(2, 16, 1, 64, dtype=torch.bfloat16)
    return torch.zeros(1, 1, 64, dtype=torch.bfloat16), cache, torch.zeros(2, **i32), torch.zeros(1, **i32), torch.zeros(1, 1, **i32)


def test_cpu_tensors_raise(mi):
    q, cache, cu, lens, table = _tensors()
    with pytest.raises(RuntimeError, match="no CPU path"):
        mi.ops.paged_decode_attention(q, cache, cache, lens, table, window=4)
    with pytest.raises(RuntimeError, match="no CPU path"):
        mi.ops.paged_prefill_attention(q, cache, cache, cu, lens, table, window=4)
