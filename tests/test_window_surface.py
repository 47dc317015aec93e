"""Windows, sinks and positions with several axes: what the layers and the flash-attention forms refuse, before any GPU is asked."""
import pytest
import torch


@pytest.mark.parametrize("more,error", [
    (dict(window_size=(-2, 0)), NotImplementedError), (dict(window_size=(5, 1)), NotImplementedError),
    (dict(window_size=(-1, 3)), NotImplementedError), (dict(window_size=(5, -2)), NotImplementedError),
    (dict(window_size=(5, 0), sink_tokens=-1), ValueError), (dict(sink_tokens=4), ValueError),
    (dict(window_size=(-1, -1), sink_tokens=4), ValueError),
])
def test_windows_that_there_are_not(mi, more, error):
    q, cache = torch.zeros(4, 2, 64), torch.zeros(1, 16, 2, 64)
    i32 = dict(dtype=torch.int32)
    with pytest.raises(error):
        mi.flash_attn_varlen_func(q, cache, cache, torch.tensor([0, 4], **i32), None, 4, 4, causal=True,
                                  block_table=torch.zeros(1, 1, **i32), seqused_k=torch.tensor([4], **i32), **more)
    with pytest.raises(error):
        mi.flash_attn_with_kvcache(q[:1, None], cache, cache, cache_seqlens=torch.tensor([4], **i32),
                                   block_table=torch.zeros(1, 1, **i32), **more)
    with pytest.raises(error):
        mi.PagedSelfAttentionCore(1, 64, **more)
    with pytest.raises(error):
        mi.PagedSelfAttentionLayer(1, 64, 2, 2, 64, **more)


def test_no_window_over_latent_caches(mi):
    from importlib import import_module
    attention = import_module(mi.__name__ + ".attention")
    i32 = dict(dtype=torch.int32)
    lens, table = torch.tensor([4], **i32), torch.zeros(1, 1, **i32)
    with pytest.raises(NotImplementedError, match="window"):   # keys wider than values
        mi.flash_attn_varlen_func(torch.zeros(4, 2, 192), torch.zeros(1, 16, 2, 192), torch.zeros(1, 16, 2, 128),
                                  torch.tensor([0, 4], **i32), None, 4, 4, causal=True, block_table=table, seqused_k=lens,
                                  window_size=(3, 0))
    with pytest.raises(NotImplementedError, match="window"):
        attention.flash_decode_and_prefill(torch.zeros(1, 1, 2, 576), torch.zeros(1, 16, 576), None, 1, 4, None, None, lens, table,
                                           mla_head_dim_v=512, window_size=(3, 0))


def test_positions_go_with_axes(mi):
    positions, emb = torch.zeros(3, 4, dtype=torch.int64), torch.zeros(8, 64)
    plain, several = mi.PagedSelfAttentionCore(1, 64), mi.PagedSelfAttentionCore(1, 64, rotary_sections=(8, 12, 12))
    q, kv, mixed = torch.zeros(4, 1, 2, 64), torch.zeros(4, 1, 1, 64), torch.zeros(4, 1, 4 * 64)
    for call in (lambda c, *a: c(q, kv, kv, None, emb, *a), lambda c, *a: c.forward_mixed_qkv(mixed, 2, None, emb, *a)):
        with pytest.raises(ValueError, match="rotary_sections"):
            call(plain, positions)
        with pytest.raises(ValueError, match="axis_positions"):
            call(several)
    with pytest.raises(NotImplementedError, match="fused"):
        mi.PagedSelfAttentionCore(1, 64, rotary_sections=(8, 12, 12), fused=False)
    with pytest.raises(ValueError):
        mi.PagedSelfAttentionCore(1, 64, rotary_sections=())
    layer = mi.PagedSelfAttentionLayer(1, 64, 2, 1, 64)
    with pytest.raises(ValueError, match="rotary_sections"):
        layer.core.forward_mixed_qkv(mixed, 2, None, emb, positions)


def test_calls_without_a_window_are_what_they_were(mi, monkeypatch):
    """Functions in the places of the two attention calls, contexts and stored layers that know no windows."""
    from importlib import import_module
    attention = import_module(mi.__name__ + ".attention")
    calls = []
    for name in ("flash_attn_varlen_func", "flash_attn_with_kvcache"):
        monkeypatch.setattr(attention, name, lambda *a, name=name, **k: calls.append((name, set(k))) or torch.zeros(4, 2, 64))
    q = torch.zeros(4, 1, 2, 64)
    attention.flash_decode_and_prefill(q, None, None, 4, 4, None, None, None, None)
    attention.flash_decode_and_prefill(q, None, None, 1, 4, None, None, None, None)
    assert [c[0] for c in calls] == ["flash_attn_varlen_func", "flash_attn_with_kvcache"]
    assert all(not c[1] & {"window_size", "sink_tokens"} for c in calls)
    attention.flash_decode_and_prefill(q, None, None, 1, 4, None, None, None, None, window_size=(3, 0), sink_tokens=2)
    assert {"window_size", "sink_tokens"} <= calls[-1][1]
    core = mi.PagedSelfAttentionCore(1, 64, window_size=(5, 0))
    for name in ("window_size", "sink_tokens", "rotary_axes"):
        delattr(core, name)
    assert (core.window_size, core.sink_tokens, core.rotary_axes) == (None, 0, None)
    layer = mi.PagedSelfAttentionLayer(1, 64, 2, 1, 64)
    seen = []
    layer.linear_qkv.forward = lambda x: (x, None)
    layer.linear_proj.forward = lambda x: (x, None)
    layer.core.forward_mixed_qkv = lambda mixed, heads, context, emb=None: seen.append(emb) or mixed
    layer(torch.zeros(4, 1, 64), None, None)
    assert seen == [None]


def test_the_workspace_of_captured_windows(mi):
    """A walk of 449 keys of 576 is cut into more parts than the whole 576 are: the graphs' buffer has room for either."""
    cls = mi.DynamicInferenceContext
    saved = (cls.TOKEN_ROUNDER, cls.REQUEST_ROUNDER)
    cls.TOKEN_ROUNDER = cls.REQUEST_ROUNDER = 4
    try:
        ctx = cls(params_dtype=torch.bfloat16, num_layers=1, kv_channels=128, num_attention_heads=8, max_sequence_length=576,
                  buffer_size_gb=0.05, buffer_guaranteed_fraction=0.1, chunk_size_tokens=64, max_requests_override=16,
                  max_tokens_override=1024, num_cuda_graphs=2, device="cpu")
    finally:
        cls.TOKEN_ROUNDER, cls.REQUEST_ROUNDER = saved
    core = mi.PagedSelfAttentionCore(1, 128, window_size=(188, 0), sink_tokens=4)
    need, plain = mi.ops.prefill_workspace_bytes(16, 16, 32, 8, 128, 576, window=189, sinks=4), mi.ops.prefill_workspace_bytes(16, 16, 32, 8, 128, 576)
    assert need == mi._lib.load().mi_window_prefill_workspace_bytes(16, 16, 32, 8, 128, 576, 189, 4, None) > plain
    assert mi.DecodeLayerGraphs(ctx, [torch.nn.Identity(), core], num_query_heads=32).workspace.numel() >= need
    foreign = torch.nn.Identity()
    foreign.window_size = 7   # (another module's own: not read)
    assert mi.DecodeLayerGraphs(ctx, [foreign], num_query_heads=32).workspace.numel() < need
    assert mi.ops.prefill_workspace_bytes(16, 16, 32, 8, 128, 576, window=1 << 62, sinks=1 << 62) == plain
    for bad in (dict(window=0), dict(window=5, sinks=-1), dict(window=5, split_tokens=16)):
        with pytest.raises(ValueError):
            mi.ops.prefill_workspace_bytes(16, 16, 32, 8, 128, 576, **bad)


def test_positions_go_to_the_layers_that_have_axes(mi):
    """One list of captured layers may hold both kinds, and modules that are no core: those get the positions, as they always did."""
    class Graphs(mi.DecodeLayerGraphs):
        def __init__(self, positions):   # (no context: only what a layer is called with is looked at)
            self.context, self.rotary_pos_emb, self.workspace, self.axis_positions = None, None, torch.empty(1), positions

    class Plain(mi.PagedSelfAttentionCore):
        def forward(self, *args):
            return args

    class Other(torch.nn.Module):
        def forward(self, *args):
            return args
    positions = torch.zeros(3, 4, dtype=torch.int64)
    plain, several = Plain(1, 64), Plain(1, 64, rotary_sections=(8, 12, 12))
    for layer, given in ((plain, 5), (several, 6), (Other(), 6)):
        assert len(Graphs(positions)._run(layer, None, None, None)) == given
        assert len(Graphs(None)._run(layer, None, None, None)) == 5


def test_the_latent_decode_branch_reads_windows_as_the_others_do(mi, monkeypatch):
    from importlib import import_module
    attention = import_module(mi.__name__ + ".attention")
    i32 = dict(dtype=torch.int32)
    lens, table = torch.tensor([4], **i32), torch.zeros(1, 1, **i32)

    def run(**more):
        return attention.flash_decode_and_prefill(torch.zeros(1, 1, 2, 576), torch.zeros(1, 16, 576), None, 1, 4, None, None, lens, table,
                                                  mla_head_dim_v=512, **more)
    for more in (dict(sink_tokens=4), dict(window_size=(-1, -1), sink_tokens=4), dict(window_size=(3, 0), sink_tokens=-1)):
        with pytest.raises(ValueError, match="sink_tokens"):
            run(**more)
    with pytest.raises(NotImplementedError, match="window"):
        run(window_size=(3, 0), sink_tokens=2)
    monkeypatch.setattr(attention, "get_mla_metadata", lambda *a: (None, None))
    monkeypatch.setattr(attention, "flash_mla_with_kvcache", lambda *a, **k: ("ran", None))
    for none in (None, (-1, -1), (-1, 0), [-1, -1]):
        assert run(window_size=none) == "ran"


def test_window_sizes_that_are_no_pairs(mi):
    """0 and False are no window, as they were before there were any; whatever else is no pair of whole numbers is refused by name."""
    from importlib import import_module
    window = import_module(mi.__name__ + ".flash_attn_interface").window_argument
    for none in (None, 0, False, 0.0, (-1, -1), [-1, 0]):
        assert window(none, 0) == {}
        assert mi.PagedSelfAttentionCore(1, 64, window_size=none).window_size is None
        with pytest.raises(ValueError, match="sink_tokens"):
            window(none, 4)
    assert window([5, 0], 2) == window((5, -1), 2) == dict(window=6, sinks=2)
    q, cache = torch.zeros(4, 2, 64), torch.zeros(1, 16, 2, 64)
    i32 = dict(dtype=torch.int32)
    for other in (5, True, 1.5, "5", (5,), (5, 0, 0), (None, 0), (5.0, 0), torch.tensor([-1, -1]), object()):
        with pytest.raises(NotImplementedError, match="window_size"):
            window(other, 0)
        with pytest.raises(NotImplementedError, match="window_size"):
            mi.flash_attn_with_kvcache(q[:1, None], cache, cache, cache_seqlens=torch.tensor([4], **i32),
                                       block_table=torch.zeros(1, 1, **i32), window_size=other)
