"""Windows, sinks and positions with several axes as a model uses them: layers of a dynamic context over prompts, decode steps and
steps of both, 16-bit and fp8 caches, and captured graphs.

Each layer's call is checked in two halves.  The queries and keys that norm, rotation and append make of the step's tensors are
compared with the 64-bit oracle by the bounds of the rotary tests (the keys where the cache holds them); attention is compared
with the 64-bit oracle over those queries and the cache as it is, by the bounds of the attention tests.
"""
import pytest
import torch

from oracle import paged_attention as oa
from oracle import rope_norm as orn
from oracle import windows as ow

pytestmark = pytest.mark.gpu

HQ, HKV, C, MOST = 8, 2, 64, 400
BF16, FP16 = torch.bfloat16, torch.float16


def _context(mi, dev, d, dtype, fp8=False, layers=2, **more):
    return mi.DynamicInferenceContext(
        params_dtype=dtype, num_layers=layers, kv_channels=d, num_attention_heads=HKV, max_sequence_length=MOST,
        buffer_size_gb=70 * (2 * layers * C * HKV * d * 2) / 1024 ** 3, buffer_guaranteed_fraction=0.1, chunk_size_tokens=C,
        max_requests_override=8, max_tokens_override=1024, kv_cache_dtype="fp8_e4m3" if fp8 else None, device=dev, **more)


def _prompt_positions(n, image):
    """Positions of a prompt of ``n`` tokens with an image of ``image`` rows and columns behind its third token, and how far the
    next token's lies from its place in the sequence."""
    rows, columns = image
    out, at = torch.zeros(3, n, dtype=torch.int64), 0
    text = min(3, n)
    out[:, :text] = torch.arange(text)
    at = base = text
    for i in range(rows * columns):
        if at < n:
            out[:, at] = torch.tensor([base, base + i // columns, base + i % columns])
            at += 1
    after = int(out[:, :at].max()) + 1
    out[:, at:] = after + torch.arange(n - at)
    return out, int(out.max()) + 1 - n


def _rows(ctx):
    """Where the rows of every request of the step begin, and the requests' lengths."""
    count = ctx.total_request_count
    cu = list(range(count + 1)) if ctx.is_decode_only() else ctx.cu_query_seq_lengths.tolist()[:count + 1]
    return cu, ctx.kv_seq_lengths.tolist()[:count]


def _step_positions(ctx, shifts, images, fresh):
    """``[3, padded tokens]`` of the step: a fresh request's prompt, else one token that many places off its own."""
    n = ctx.padded_active_token_count
    out = torch.randint(0, MOST, (3, n))   # (padding: any value)
    ids = ctx.request_ids[:ctx.total_request_count].tolist()
    (cu, lens), at = _rows(ctx), 0
    for r, request in enumerate(ids):
        rows, length = cu[r + 1] - cu[r], lens[r]
        if request in fresh:
            out[:, at:at + rows], shifts[request] = _prompt_positions(rows, images[request])
        else:
            assert rows == 1
            out[:, at] = length - 1 + shifts[request]
        at += rows
    assert at == ctx.active_token_count
    return out


def _near(got, x, positions, table, axes, weight, dtype):
    """Rounded op by op: the bound of the rotary tests with faithful rounding."""
    ref = ow.norm_rotate(x, positions, table.view(MOST, -1), axes, norm="rms", weight=weight)
    y = x.double() / torch.sqrt(x.double().square().mean(-1, keepdim=True) + 1e-5) * weight.double()
    both = y.abs() + torch.cat([y[..., len(axes):2 * len(axes)], y[..., :len(axes)], y[..., 2 * len(axes):]], -1).abs()
    u = torch.finfo(dtype).eps / 2
    bound = u * ref.abs() + 2e-6 * both + 1e-7 + 3.1 * u * both * (1 + u)
    err = (got.double() - ref).abs()
    assert (err <= bound).all(), f"max err / bound {(err / bound).max():.3f}"


def _attention(ctx, layer, query, got, window, sinks, d, dtype, fp8):
    act = ctx.active_token_count
    k, v, table = ctx.key_value_cache(layer)
    scales = [s.cpu() for s in ctx.key_value_scales(layer)] if fp8 else []
    k, v = (x.cpu().view(torch.float8_e4m3fn).float() if fp8 else x.cpu() for x in (k, v))
    cu, lens = _rows(ctx)
    ref, size, total = ow.window_attention(query[:act], k, v, cu, lens, table.cpu()[:len(lens)], window, sinks, d ** -0.5, *scales)
    u = torch.finfo(dtype).eps / 2
    rounds = 3 if fp8 and d == 64 and not ctx.is_decode_only() else 2
    bound = (rounds * u + 2e-5) * size * (1 + u) + u * ref.abs() + 1e-7
    if dtype == FP16:
        bound = bound + 2.0 ** -24 * (total + min(window + sinks, max(lens)) * ref.abs())
    err = (got[:act].double() - ref).abs()
    assert (err <= bound).all(), f"max err / bound {(err / bound).max():.3f}"


@pytest.mark.parametrize("d,dtype,fp8", [(128, BF16, False), (64, FP16, False), (96, BF16, False), (128, BF16, True), (64, FP16, True)])
@pytest.mark.parametrize("entry", ["split", "mixed"])
@pytest.mark.parametrize("window,sinks,sections", [((89, 0), 5, True), ((0, -1), 0, True), ((63, 0), 64, False), (None, 0, True)])
def test_prompts_decode_and_both(mi, dev, d, dtype, fp8, entry, window, sinks, sections):
    gen = torch.Generator().manual_seed(d + sinks)
    ctx = _context(mi, dev, d, dtype, fp8)
    sections = [d // 2 - 2 * (d // 6), d // 6, d // 6] if sections else None
    axes = ow.axes_of_pairs(sections) if sections else [0] * (d // 2)
    table = orn.rotary_table(MOST, d, base=10000.0)
    emb = table.to(dev)
    cores = []
    for layer in (1, 2):
        core = mi.PagedSelfAttentionCore(layer, d, qk_norm="rms", window_size=window, sink_tokens=sinks, rotary_sections=sections,
                                         dtype=dtype, device=dev).requires_grad_(False)
        for p in core.parameters():
            p.copy_(1 + 0.1 * torch.randn(d, generator=gen))
        cores.append(core)
    images, shifts = {0: (2, 3), 1: (6, 8), 2: (10, 10), 3: (0, 0), 4: (5, 4)}, {}
    fresh = {}
    for i, n in enumerate([30, 70, 300, 1]):
        fresh[i] = n
        ctx.add_request(i, torch.arange(n, device=dev), num_tokens_to_generate=20)
    kinds = set()
    for step in range(5):
        if step == 3:   # a prompt beside the others' next tokens
            fresh = {4: 130}
            ctx.add_request(4, torch.arange(130, device=dev), num_tokens_to_generate=20)
        ctx.initialize_attention_state()
        n, act = ctx.padded_active_token_count, ctx.active_token_count
        kinds.add((ctx.is_decode_only(), act > 130))
        places = ctx.token_to_pos_ids[:n].cpu()
        positions = _step_positions(ctx, shifts, images, fresh) if sections else places.expand(3, n)
        more = dict(axis_positions=positions.to(dev)) if sections else {}
        names = dict(rotary_axes=bytes(axes), q_positions=more["axis_positions"]) if sections else \
            dict(q_positions=ctx.token_to_pos_ids, k_positions=ctx.token_to_position_in_request)
        fresh = {}
        at = ctx.token_to_chunk_idx[:act].cpu(), ctx.token_to_local_position_within_kv_chunk[:act].cpu()
        for layer, core in enumerate(cores, 1):
            mixed = torch.randn(n, 1, (HQ + 2 * HKV) * d, generator=gen).to(dtype)
            q, k, v = (t.contiguous() for t in orn.split_mixed_qkv(mixed, HQ, HKV))
            qw, kw = core.q_layernorm_weight, core.k_layernorm_weight
            queries = torch.empty(n, 1, HQ, d, dtype=dtype, device=dev)
            # (queries and keys of the step once more, from the mixed tensor and without the cache)
            keys = torch.empty(n, 1, HKV, d, dtype=dtype, device=dev)
            mi.ops.qkv_norm_rope_append(mixed.to(dev), num_query_heads=HQ, num_kv_heads=HKV, query_out=queries, key_out=keys,
                                        q_weight=qw, k_weight=kw, eps=1e-5, norm="rms", rotary_emb=emb, **names)
            if entry == "mixed":
                out = core.forward_mixed_qkv(mixed.to(dev), HQ, ctx, (emb, emb), **more)
            else:
                out = core(q.to(dev), k.to(dev), v.to(dev), ctx, (emb, emb), **more)
            torch.cuda.synchronize()
            queries, keys = queries.cpu().view(n, HQ, d), keys.cpu().view(n, HKV, d)
            _near(queries[:act], q.view(n, HQ, d)[:act], positions[:, :act], table, axes, qw.cpu(), dtype)
            _near(keys[:act], k.view(n, HKV, d)[:act], positions[:, :act], table, axes, kw.cpu(), dtype)
            kc, vc = (x.cpu() for x in ctx.key_value_cache(layer)[:2])
            if not fp8:
                assert torch.equal(kc[at], keys[:act]) and torch.equal(vc[at], v.view(n, HKV, d)[:act])
            else:   # half a step of e4m3 at the scale that the chunk's first token set, whose range later tokens may pass
                ks = ctx.key_value_scales(layer)[0].cpu()
                held, step_of = oa.dequantize_fp8(kc, ks)[at], ks[at[0]][..., None]
                want = torch.maximum(torch.minimum(keys[:act].float(), 448 * step_of), -448 * step_of)
                assert ((held - want).abs() <= (2.0 ** -4 * want.abs()).maximum(2.0 ** -10 * step_of) * (1 + 1e-5)).all()
            left = MOST if window is None else window[0]
            _attention(ctx, layer, queries, out.cpu().view(n, HQ, d), left + 1, sinks, d, dtype, fp8)
        live = ctx.total_request_count - ctx.paused_request_count
        mask = torch.ones(live, dtype=torch.int32, device=dev)
        if step == 1:
            mask[1] = 0   # (a request ends: the last one takes its row)
        ctx.update_requests(mask, torch.arange(live, device=dev))
    assert kinds == {(False, True), (True, False)}


def test_layer_from_hidden_states(mi, dev):
    """The layer's projections around the core: the parts one by one give the same, decode steps too."""
    gen = torch.Generator(device=dev).manual_seed(3)
    table = orn.rotary_table(MOST, 128).to(dev)
    layer = mi.PagedSelfAttentionLayer(1, 256, HQ, HKV, 128, qk_norm="rms", window_size=(31, 0), sink_tokens=4,
                                       rotary_sections=(16, 24, 24), rotary_alternate=False, device=dev).requires_grad_(False)
    for p in layer.parameters():
        p.normal_(0, 0.05, generator=gen)
    outs = []
    for parts in (False, True):
        ctx = _context(mi, dev, 128, BF16, layers=1)
        for i, n in enumerate((40, 100)):
            ctx.add_request(i, torch.arange(n, device=dev))
        gen.manual_seed(4)
        for step in range(3):
            ctx.initialize_attention_state()
            n = ctx.padded_active_token_count
            x = torch.empty(n, 1, 256, dtype=BF16, device=dev).normal_(generator=gen)
            positions = torch.randint(0, MOST, (3, n), generator=gen, device=dev)
            if parts:
                mixed, _ = layer.linear_qkv(x)
                y = layer.linear_proj(layer.core.forward_mixed_qkv(mixed, HQ, ctx, (table, table), positions))[0]
            else:
                y = layer(x, ctx, (table, table), positions)[0]
            outs.append(y[:ctx.active_token_count].clone())
            live = ctx.total_request_count - ctx.paused_request_count
            ctx.update_requests(torch.ones(live, dtype=torch.int32, device=dev), torch.arange(live, device=dev))
    for a, b in zip(outs[:3], outs[3:]):
        assert a.isfinite().all() and torch.equal(a, b)


def test_graphs(mi, dev):
    """Captured layers against eager ones, bit for bit, steps of prompts and decode steps; positions are read where they stand."""
    cls = mi.DynamicInferenceContext
    saved = (cls.TOKEN_ROUNDER, cls.REQUEST_ROUNDER)
    cls.TOKEN_ROUNDER = cls.REQUEST_ROUNDER = 4
    try:
        gen = torch.Generator().manual_seed(9)
        table = orn.rotary_table(MOST, 128).to(dev)
        core = mi.PagedSelfAttentionCore(1, 128, window_size=(20, 0), sink_tokens=3, rotary_sections=(16, 24, 24),
                                         device=dev).requires_grad_(False)
        captured, eager = _context(mi, dev, 128, BF16, layers=1, num_cuda_graphs=1), _context(mi, dev, 128, BF16, layers=1)
        held = torch.zeros(3, max(captured.cuda_graph_token_counts), dtype=torch.int64, device=dev)
        with pytest.raises(ValueError, match="shorter"):
            mi.DecodeLayerGraphs(captured, [core], num_query_heads=HQ, axis_positions=held[:, 1:])
        graphs = mi.DecodeLayerGraphs(captured, [core], num_query_heads=HQ, rotary_pos_emb=(table, table), axis_positions=held)
        graphs.capture()
        for i, n in enumerate((2, 1, 3)):
            for ctx in (captured, eager):
                ctx.add_request(i, torch.arange(n, device=dev), num_tokens_to_generate=60)
        replayed = 0
        for step in range(30):
            for ctx in (captured, eager):
                ctx.initialize_attention_state()
            act = eager.active_token_count
            n = max(ctx.padded_active_token_count for ctx in (captured, eager))
            q, k, v = (torch.randn(n, 1, h, 128, generator=gen).bfloat16().to(dev) for h in (HQ, HKV, HKV))
            positions = torch.randint(0, MOST, (3, n), generator=gen).to(dev)
            assert captured.using_cuda_graph_this_step()
            held[:, :n] = positions
            got = graphs.replay(0, q, k, v).clone()
            m = eager.padded_active_token_count
            want = core(q[:m].clone(), k[:m], v[:m], eager, (table, table), positions)
            assert torch.equal(got[:act], want[:act]), f"step {step}"
            replayed += captured.is_decode_only()
            live = eager.total_request_count
            for ctx in (captured, eager):
                ctx.update_requests(torch.ones(live, dtype=torch.int32, device=dev), torch.arange(live, device=dev))
        assert replayed > 20
    finally:
        cls.TOKEN_ROUNDER, cls.REQUEST_ROUNDER = saved


@pytest.mark.parametrize("order", [(True, False), (False, True)])
def test_graphs_of_layers_with_and_without_axes(mi, dev, order):
    """One set of graphs over a layer of each kind: the positions go to those that have axes."""
    cls = mi.DynamicInferenceContext
    saved = (cls.TOKEN_ROUNDER, cls.REQUEST_ROUNDER)
    cls.TOKEN_ROUNDER = cls.REQUEST_ROUNDER = 4
    try:
        gen = torch.Generator().manual_seed(11)
        table = orn.rotary_table(MOST, 128).to(dev)
        cores = [mi.PagedSelfAttentionCore(i + 1, 128, rotary_sections=(16, 24, 24) if several else None, device=dev).requires_grad_(False)
                 for i, several in enumerate(order)]
        captured, eager = _context(mi, dev, 128, BF16, num_cuda_graphs=1), _context(mi, dev, 128, BF16)
        held = torch.zeros(3, max(captured.cuda_graph_token_counts), dtype=torch.int64, device=dev)
        graphs = mi.DecodeLayerGraphs(captured, cores, num_query_heads=HQ, rotary_pos_emb=(table, table), axis_positions=held)
        graphs.capture()
        for i, n in enumerate((2, 1, 3)):
            for ctx in (captured, eager):
                ctx.add_request(i, torch.arange(n, device=dev), num_tokens_to_generate=60)
        for step in range(6):
            for ctx in (captured, eager):
                ctx.initialize_attention_state()
            act, m = eager.active_token_count, eager.padded_active_token_count
            n = max(m, captured.padded_active_token_count)
            positions = torch.randint(0, MOST, (3, n), generator=gen).to(dev)
            held[:, :n] = positions
            for i, (core, several) in enumerate(zip(cores, order)):
                q, k, v = (torch.randn(n, 1, h, 128, generator=gen).bfloat16().to(dev) for h in (HQ, HKV, HKV))
                got = graphs.replay(i, q, k, v).clone()
                want = core(q[:m].clone(), k[:m], v[:m], eager, (table, table), *((positions,) if several else ()))
                # (a decode step of the layer without axes is one launch here and there: the same kernels on both sides)
                assert torch.equal(got[:act], want[:act]), f"step {step}, layer {i}"
            live = eager.total_request_count
            for ctx in (captured, eager):
                ctx.update_requests(torch.ones(live, dtype=torch.int32, device=dev), torch.arange(live, device=dev))
    finally:
        cls.TOKEN_ROUNDER, cls.REQUEST_ROUNDER = saved


def test_flash_attention_forms(mi, dev):
    """``window_size`` and ``sink_tokens`` of the adapters are the window and the sinks of the calls below them."""
    gen = torch.Generator(device=dev).manual_seed(1)
    k, v = (torch.empty(8, 64, HKV, 64, dtype=BF16, device=dev).normal_(generator=gen) for _ in "kv")
    table = torch.arange(8, dtype=torch.int32, device=dev).view(2, 4)
    lens = torch.tensor([200, 131], dtype=torch.int32, device=dev)
    q = torch.empty(2, 1, HQ, 64, dtype=BF16, device=dev).normal_(generator=gen)
    cu = torch.tensor([0, 3, 50], dtype=torch.int32, device=dev)
    rows = torch.empty(50, HQ, 64, dtype=BF16, device=dev).normal_(generator=gen)
    for left, right, sinks in ((0, 0, 0), (40, -1, 2), (-1, -1, 0), (-1, 0, 0)):
        seen = {} if left < 0 else dict(window=left + 1, sinks=sinks)
        more = dict(window_size=(left, right), sink_tokens=sinks)
        got = mi.flash_attn_with_kvcache(q, k, v, cache_seqlens=lens, block_table=table, causal=True, **more)
        assert torch.equal(got, mi.ops.paged_decode_attention(q, k, v, lens, table, **seen))
        got = mi.flash_attn_varlen_func(rows, k, v, cu, None, 47, 256, causal=True, block_table=table, seqused_k=lens, **more)
        assert torch.equal(got, mi.ops.paged_prefill_attention(rows, k, v, cu, lens, table, max_kv_len=256,
                                                               one_row_requests=False, **seen))
