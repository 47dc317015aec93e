"""Long contexts and images over the paged cache, as measurable cases.

Three operators of a serving step, the writer of the cache and the two forms of the attention that reads it:

* ``decode``  -- one new token per request attends to the last ``window`` tokens of its request and to the first ``sinks``.
* ``prompts`` -- the same for many new tokens per request (prompts, chunks of prompts over a context, a mix with requests of
                 one token): a token at position P sees a token at k <= P where k > P - window or k < sinks.
* ``axes``    -- head norm and rotary embedding of queries and keys whose positions have several axes (time, height,
                 width: every pair of elements belongs to one of them), and the keys and values written to the cache.

Chunks that no token of the call sees need not exist: where a case says ``released`` a program has given them back, and the
block table holds 0 in their place.  Where ``own`` is false the operators are computed in their plain form.

Lengths are drawn from the case itself, so that ``work`` knows them; values, tables and slots from the seed.
"""
import importlib
import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------------------------ the cases
def _decode(name, batch, heads, kv_heads, d, lo, hi, window, sinks, cache="16bit", dtype="bf16", chunk=256, released=False):
    return dict(name=name, kind="decode", batch=batch, heads=heads, kv_heads=kv_heads, d=d, lo=lo, hi=hi, window=window,
                sinks=sinks, cache=cache, dtype=dtype, chunk=chunk, released=released)


def _prompts(name, batch, new_lo, new_hi, context, heads, kv_heads, d, window, sinks, single=0, cache="16bit", dtype="bf16",
             chunk=256, released=False):
    return dict(name=name, kind="prompts", batch=batch, new_lo=new_lo, new_hi=new_hi, context=context, heads=heads,
                kv_heads=kv_heads, d=d, window=window, sinks=sinks, single=single, cache=cache, dtype=dtype, chunk=chunk,
                released=released)


def _axes(name, batch, new_lo, new_hi, heads, kv_heads, d, sections, alternate=False, pairs="halves", norm="rms", mixed=True,
          dtype="bf16", chunk=256):
    return dict(name=name, kind="axes", batch=batch, new_lo=new_lo, new_hi=new_hi, heads=heads, kv_heads=kv_heads, d=d,
                sections="-".join(map(str, sections)), alternate=alternate, pairs=pairs, norm=norm, mixed=mixed, dtype=dtype,
                chunk=chunk)


def listed():
    return [
        # one user in front of a chat, some thousand tokens into it
        _decode("decode_chat", 1, 32, 8, 128, 5000, 5000, 1024, 4),
        # a small fp16 model without grouped heads: ragged requests, many shorter than the window
        _decode("decode_ragged_d64_fp16", 24, 8, 8, 64, 33, 1500, 255, 1, dtype="fp16"),
        # the ordinary serving batch: 64 requests of U[512, 8192] tokens
        _decode("decode_batch64", 64, 32, 8, 128, 512, 8192, 2048, 4),
        # a large batch over an fp8 cache
        _decode("decode_fp8_cache", 256, 32, 8, 128, 1024, 32768, 4096, 16, cache="fp8", released=True),
        # long documents, 70B-shaped heads, a window of 32 768 tokens of 131 072
        _decode("decode_long_context", 16, 64, 8, 128, 131072, 131072, 32768, 64, released=True),
        # ragged prompts of a small fp16 model
        _prompts("prompts_ragged_d64_fp16", 11, 164, 2911, 0, 32, 8, 64, 500, 4, dtype="fp16"),
        # four prompts of some thousand tokens
        _prompts("prompts_window_1024", 4, 3500, 4100, 0, 32, 8, 128, 1024, 4),
        # prompts over an fp8 cache
        _prompts("prompts_fp8_cache", 6, 129, 4097, 0, 32, 8, 128, 2048, 16, cache="fp8"),
        # a chunk of a long prompt: 509 new tokens behind some 61 000
        _prompts("prompts_chunk_over_long_context", 1, 509, 509, 61234, 64, 8, 128, 16384, 64, released=True),
        # new prompts beside requests that go on decoding
        _prompts("prompts_mixed_with_decode", 8, 2048, 2048, 0, 32, 8, 128, 4096, 4, single=120),
        # the serving batch's tokens: 64 of one token each, split tensors
        _axes("axes_batch64", 64, 1, 1, 32, 8, 128, (16, 24, 24), mixed=False),
        # prompts with images in them, straight from the projection
        _axes("axes_prompts_with_images", 4, 3000, 4000, 32, 8, 128, (16, 24, 24)),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = {kind: [work(c) for c in listed() if c["kind"] == kind] for kind in ("decode", "prompts", "axes")}
    while True:
        c = _draw_one(rng)
        w, of = work(c), most[c["kind"]]
        if all(w[x] <= max(y[x] for y in of) for x in w) and _plain_values(c) <= 1.5e9 and _pool_values(c) <= 4e9:
            c.pop("name", None)
            return c


def _draw_one(rng):
    kind = rng.choice(("decode", "decode", "prompts", "prompts", "axes"))
    heads, kv_heads = rng.choice(((32, 8), (32, 8), (64, 8), (32, 4), (16, 2), (8, 8), (24, 8), (28, 4), (7, 1), (20, 1)))
    dtype, cache = rng.choice(("bf16", "bf16", "fp16")), rng.choice(("16bit", "16bit", "fp8"))
    d = rng.choice((64, 128)) if cache == "fp8" else rng.choice((64, 96, 128, 128, 192, 256))
    chunk = rng.choice((256, 256, 128, 64) if cache == "fp8" and kind == "prompts" else (256, 256, 128, 64, 48, 16))
    window, sinks = _log_int(rng, 1, 40000), rng.choice((0, 1, 4, 16, 63, 130))
    if kind == "decode":
        hi = _log_int(rng, 1, 131072)
        return _decode("", _log_int(rng, 1, 256), heads, kv_heads, d, max(1, hi // rng.choice((1, 4, 16))), hi, window, sinks, cache,
                       dtype, chunk, rng.random() < 0.5)
    batch, hi = _log_int(rng, 1, 16), _log_int(rng, 1, 4200)
    new = (max(1, hi // rng.choice((1, 3, 16))), hi)
    if kind == "prompts":
        return _prompts("", batch, *new, rng.choice((0, _log_int(rng, 1, 60000))), heads, kv_heads, d, window, sinks,
                        rng.choice((0, 0, _log_int(rng, 1, 100))), cache, dtype, chunk, rng.random() < 0.5)
    d = rng.choice((64, 96, 128, 128, 192, 256))
    pairs = d // 2 // rng.choice((1, 1, 2))
    if rng.random() < 0.25:
        pairs = rng.randint(3, d // 2)
    a = rng.randint(1, pairs // 2)
    b = rng.randint(1, max(1, (pairs - a) // 2))
    sections = (pairs - a - b, a, b) if pairs - a - b > 0 else (pairs,)
    return _axes("", batch, *new, heads, kv_heads, d, sections, rng.random() < 0.3, rng.choice(("halves", "halves", "neighbours")),
                 rng.choice(("rms", "rms", "l2", "none")), rng.random() < 0.6, dtype, chunk)


# ------------------------------------------------------------------------------------------------ sizes of a case
def _random(c, salt):
    return random.Random("%s %s" % (salt, sorted((k, v) for k, v in c.items() if k != "name")))


def _requests(c):
    """(new tokens, cached tokens with them) of every request; those that go on decoding last."""
    r = _random(c, "requests")
    if c["kind"] == "decode":
        return [(1, r.randint(c["lo"], c["hi"])) for _ in range(c["batch"])]
    new = [r.randint(c["new_lo"], c["new_hi"]) for _ in range(c["batch"])]
    if c["kind"] == "axes":
        return [(n, n + (r.randint(0, 4000) if n == 1 else 0)) for n in new]
    out = [(n, n + (r.randint(c["context"] // 2, c["context"]) if c["batch"] > 1 else c["context"])) for n in new]
    return out + [(1, r.randint(1, 8192)) for _ in range(c["single"])]


def _ranges(c, new, length):
    """Positions that some token of the request sees: [0, a) and [b, length)."""
    if c["kind"] == "axes":
        return length - new, length - new
    b = max(0, length - new + 1 - c["window"])
    return min(c["sinks"], b), b


def _seen(c, new, length):
    """Sum over a request's new tokens of how many tokens each sees."""
    total = 0
    for p in range(length - new, length):
        b = max(0, p + 1 - c["window"])
        total += min(c["sinks"], b) + p + 1 - b
    return total


def _item(c):
    return 1 if c.get("cache") == "fp8" else 2


def _chunks(c, new, length):
    """Which of a request's chunks its program keeps."""
    n, size = -(-length // c["chunk"]), c["chunk"]
    if c["kind"] != "axes" and not c["released"]:
        return list(range(n))
    a, b = _ranges(c, new, length)
    first = 0 if c["kind"] == "axes" else -(-a // size)
    return list(range(first)) + list(range(max(first, b // size), n))


def _pool_chunks(c):
    return sum(len(_chunks(c, *r)) for r in _requests(c)) + 3


def _pool_values(c):
    return _pool_chunks(c) * c["chunk"] * c["kv_heads"] * c["d"]


def _plain_values(c):
    """How many values the largest tensor of the plain form has."""
    rs = _requests(c)
    if c["kind"] == "axes":
        return sum(n for n, _ in rs) * (c["heads"] + 2 * c["kv_heads"]) * c["d"]
    widths = [(n, a + k - b) for n, k in rs for a, b in [_ranges(c, n, k)]]
    if c["kind"] == "decode":
        return len(rs) * max(w for _, w in widths) * c["kv_heads"] * c["d"]
    return max(max(n * c["heads"], c["kv_heads"] * c["d"]) * w for n, w in widths)


def _sections(c):
    return [int(x) for x in c["sections"].split("-")]


def _axis_of_pairs(c):
    """The axis of every pair of elements: its sections one after the other, or in turn as far as they go (then the first)."""
    sections = _sections(c)
    if not c["alternate"]:
        return [axis for axis, n in enumerate(sections) for _ in range(n)]
    axes, n = [0] * sum(sections), len(sections)
    for axis in range(1, n):
        for i in range(axis, min(len(axes), n * sections[axis]), n):
            axes[i] = axis
    return axes


def _positions(c):
    """Positions of every token on three axes: text counts on all three, an image's rows and columns count from where the
    text stopped; the text behind it goes on after the largest of them."""
    r, out = _random(c, "positions"), []
    for new, length in _requests(c):
        at, left = length - new, new
        if new == 1:
            out.append((at, at, at))
            continue
        while left > 0:
            text = min(left, r.randint(5, 300))
            out += [(at + i,) * 3 for i in range(text)]
            at, left = at + text, left - text
            t, h, w = r.choice((1, 1, 4)), r.randint(4, 40), r.randint(4, 40)
            grid = [(at + i, at + j, at + k) for i in range(t) for j in range(h) for k in range(w)][:left]
            out += grid
            left -= len(grid)
            at += max(t, h, w)
    return out


def work(case):
    c, rs = case, _requests(case)
    rows = sum(n for n, _ in rs)
    if c["kind"] == "axes":
        # queries and keys in and out, values in and out, positions, slots; angles of as many positions as there are
        angles = min(rows, max(max(p) for p in _positions(c)) + 1) * sum(_sections(c)) * 4
        values = rows * (c["heads"] + 2 * c["kv_heads"]) * c["d"]
        return {"bytes": 4 * values + rows * (8 * len(_sections(c)) + 16) + angles, "flops": 8 * values}
    seen = sum(a + k - b for n, k in rs for a, b in [_ranges(c, n, k)])
    # (a request's visible range of chunks that no token sees in whole counts by its tokens)
    nbytes = seen * c["kv_heads"] * c["d"] * 2 * _item(c) + 2 * rows * c["heads"] * c["d"] * 2 + 8 * len(rs)
    chunks = -(-seen // c["chunk"])
    nbytes += 4 * chunks + (8 * chunks * c["kv_heads"] if c["cache"] == "fp8" else 0)
    return {"bytes": nbytes, "flops": 4 * c["heads"] * c["d"] * sum(_seen(c, n, k) for n, k in rs)}


# ------------------------------------------------------------------------------------------------ inputs
def _device():
    return torch.device("cuda", torch.cuda.current_device())


def _randn(shape, dtype, gen, scale=1.0):
    return torch.empty(shape, dtype=dtype, device=_device()).normal_(0, scale, generator=gen)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=_device())


def _cu(c):
    cu = [0]
    for n, _ in _requests(c):
        cu.append(cu[-1] + n)
    return cu


def _table(c, seed):
    """Block table of shuffled chunks (0 where a request has none) and the pool's size."""
    n, host = _pool_chunks(c), torch.Generator().manual_seed(seed)
    ids = iter(torch.randperm(n, generator=host).tolist())
    table = torch.zeros(len(_requests(c)), max(-(-k // c["chunk"]) for _, k in _requests(c)), dtype=torch.int32)
    for r, (new, length) in enumerate(_requests(c)):
        kept = _chunks(c, new, length)
        table[r, kept] = torch.tensor([next(ids) for _ in kept], dtype=torch.int32)
    return table.to(_device()), n


def _fp8_cache(shape, gen):
    """Bytes of e4m3 values ~ N(0, 100) and their scales, one per chunk and head."""
    cache = torch.empty(shape, dtype=torch.uint8, device=_device())
    for part in cache.split(512):
        part.copy_(_randn(part.shape, torch.float32, gen, 100.0).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8))
    return cache, 0.005 + 0.01 * torch.rand(shape[0], shape[2], generator=gen, device=_device())


def prepare(case, seed):
    c, gen = case, torch.Generator(device=_device()).manual_seed(seed)
    dtype, rs, cu = _DTYPES[c["dtype"]], _requests(c), _cu(c)
    table, chunks = _table(c, seed)
    rows, shape = cu[-1], (chunks, c["chunk"], c["kv_heads"], c["d"])
    s = dict(kind=c["kind"], requests=rs, table=table, lens=_int32([k for _, k in rs]))
    if c["kind"] != "axes":
        s.update(q=_randn((rows, c["heads"], c["d"]), dtype, gen), cu=_int32(cu), window=c["window"], sinks=c["sinks"],
                 scale=c["d"] ** -0.5, most=max(k for _, k in rs), singles=any(n == 1 for n, _ in rs), k_scales=None, v_scales=None)
        if c["cache"] == "fp8":
            s["k"], s["k_scales"] = _fp8_cache(shape, gen)
            s["v"], s["v_scales"] = _fp8_cache(shape, gen)
        else:
            s["k"], s["v"] = _randn(shape, dtype, gen), _randn(shape, dtype, gen)
        return s
    axes, group, d = _axis_of_pairs(c), c["heads"] // c["kv_heads"], c["d"]
    token = [(r, p) for r, (n, k) in enumerate(rs) for p in range(k - n, k)]
    at = _int32([r for r, _ in token]).long(), _int32([p for _, p in token]).long()
    positions = torch.tensor(_positions(c), device=_device()).t()[:len(_sections(c))].contiguous()
    inv = 500000.0 ** (-torch.arange(len(axes), dtype=torch.float64, device=_device()) / len(axes))
    angles = (torch.arange(int(positions.max()) + 1, device=_device())[:, None] * inv).float()
    if c["pairs"] == "halves":
        angles = torch.cat([angles, angles], 1)
    else:
        angles = angles.repeat_interleave(2, 1)
    mixed = _randn((rows, c["kv_heads"], group + 2, d), dtype, gen)
    s.update(neighbours=c["pairs"] != "halves", norm=c["norm"], axes=bytes(axes), positions=positions, angles=angles.contiguous(),
             mixed=mixed, heads=c["heads"], slot=at[1] % c["chunk"], chunk=table[at[0], at[1] // c["chunk"]].long(),
             q_out=torch.empty(rows, c["heads"], d, dtype=dtype, device=_device()),
             k=torch.zeros(shape, dtype=dtype, device=_device()), v=torch.zeros(shape, dtype=dtype, device=_device()),
             weights=[1 + _randn((d,), torch.float32, gen, 0.1).to(dtype) for _ in "qk"] if c["norm"] == "rms" else [None, None])
    if not c["mixed"]:
        s["split"] = [mixed[:, :, :group].reshape(rows, c["heads"], d), mixed[:, :, group].contiguous(), mixed[:, :, group + 1].contiguous()]
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    if own:
        return _own(state)
    return {"decode": _plain_decode, "prompts": _plain_prompts, "axes": _plain_axes}[state["kind"]](state)


def _own(s):
    ops = importlib.import_module("megatron-mixtera_amd").ops
    if s["kind"] == "axes":
        common = dict(q_weight=s["weights"][0], k_weight=s["weights"][1], eps=1e-5, norm=s["norm"], rotary_emb=s["angles"],
                      q_positions=s["positions"], rotary_axes=s["axes"], rotary_interleaved=s["neighbours"], query_out=s["q_out"],
                      k_cache=s["k"], v_cache=s["v"], token_to_chunk_idx=s["chunk"], token_to_local_pos=s["slot"],
                      faithful_rounding=False)
        if "split" in s:
            ops.norm_rope_append(s["split"][0], s["split"][1], value=s["split"][2], **common)
        else:
            ops.qkv_norm_rope_append(s["mixed"].flatten(1), num_query_heads=s["heads"], num_kv_heads=s["k"].size(2), **common)
        return {"q": s["q_out"], "k": s["k"], "v": s["v"]}
    common = dict(softmax_scale=s["scale"], max_kv_len=s["most"], window=s["window"], sinks=s["sinks"], k_scales=s["k_scales"],
                  v_scales=s["v_scales"])
    if s["kind"] == "decode":
        return {"out": ops.paged_decode_attention(s["q"], s["k"], s["v"], s["lens"], s["table"], **common)}
    return {"out": ops.paged_prefill_attention(s["q"], s["k"], s["v"], s["cu"], s["lens"], s["table"], one_row_requests=s["singles"],
                                               **common)}


# ---- plain forms: elementary operations in 32 bits ---------------------------------------------------------------------
def _values(s, which, chunk, at):
    """Rows ``at`` of the chunks, as numbers."""
    x = s[which][chunk, at]
    if s["k_scales"] is None:
        return x.float()
    return x.view(torch.float8_e4m3fn).float() * s[which + "_scales"][chunk].unsqueeze(-1)


def _plain_decode(s):
    q, lens, size = s["q"], s["lens"].long()[:, None], s["k"].size(1)
    R, heads, d = q.shape
    n = max(a + k - b for _, k in s["requests"] for b in [max(0, k - s["window"])] for a in [min(s["sinks"], b)])
    i, first = torch.arange(n, device=q.device), (lens - s["window"]).clamp(min=0)
    sinks = first.clamp(max=s["sinks"])
    at = torch.where(i < sinks, i, i - sinks + first)                                   # [R, n]
    seen = at < lens
    at = at.clamp(max=lens - 1)
    chunk = torch.gather(s["table"].long(), 1, at // size)
    k, v = (_values(s, x, chunk, at % size).transpose(1, 2).contiguous() for x in "kv")  # [R, Hkv, n, d]
    rows = q.float().view(R, k.size(1), -1, d)
    x = torch.matmul(rows, k.transpose(2, 3).contiguous()) * s["scale"]
    x = x.masked_fill_(~seen[:, None, None], -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    return {"out": torch.matmul(x / x.sum(-1, keepdim=True), v).view(R, heads, d).to(q.dtype)}


def _plain_prompts(s):
    out, size, begin, device = torch.zeros_like(s["q"]), s["k"].size(1), 0, s["q"].device
    heads, d = s["q"].shape[1:]
    for r, (new, length) in enumerate(s["requests"]):
        b = max(0, length - new + 1 - s["window"])
        at = torch.cat([torch.arange(min(s["sinks"], b), device=device), torch.arange(b, length, device=device)])
        chunk = s["table"][r].long()[at // size]
        k, v = (_values(s, x, chunk, at % size).transpose(0, 1).contiguous() for x in "kv")   # [Hkv, n, d]
        p = torch.arange(length - new, length, device=device)[:, None]
        seen = (at <= p) & ((at > p - s["window"]) | (at < s["sinks"]))
        rows = s["q"][begin:begin + new].float().view(new, k.size(0), -1, d).transpose(0, 1).reshape(k.size(0), -1, d)
        x = torch.matmul(rows, k.transpose(1, 2).contiguous()) * s["scale"]
        x = x.view(k.size(0), new, -1, at.numel()).masked_fill_(~seen[:, None], -math.inf)
        x = torch.exp(x - x.amax(-1, keepdim=True))
        x = (x / x.sum(-1, keepdim=True)).view(k.size(0), -1, at.numel())
        o = torch.matmul(x, v).view(k.size(0), new, -1, d).transpose(0, 1).reshape(new, heads, d)
        out[begin:begin + new] = o.to(out.dtype)
        begin += new
    return {"out": out}


def _plain_axes(s):
    if "split" in s:
        q, k, v = s["split"]
    else:
        q, k, v = s["mixed"][:, :, :-2].flatten(1, 2), s["mixed"][:, :, -2], s["mixed"][:, :, -1]
    axis = torch.tensor(list(s["axes"]), device=q.device)
    pair = torch.arange(axis.numel(), device=q.device)
    column = 2 * pair if s["neighbours"] else pair
    angle = s["angles"][s["positions"][axis], column[:, None]].t()[:, None]              # [rows, 1, pairs]
    cos, sin, n = torch.cos(angle), torch.sin(angle), 2 * axis.numel()

    def rotated(x, weight):
        x = x.float()
        if s["norm"] != "none":
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-5)
        if weight is not None:
            x = x * weight.float()
        y = x.clone()
        a, b = (slice(0, n, 2), slice(1, n, 2)) if s["neighbours"] else (slice(0, n // 2), slice(n // 2, n))
        y[..., a] = x[..., a] * cos - x[..., b] * sin
        y[..., b] = x[..., b] * cos + x[..., a] * sin
        return y.to(s["q_out"].dtype)

    s["q_out"].copy_(rotated(q, s["weights"][0]))
    s["k"][s["chunk"], s["slot"]] = rotated(k, s["weights"][1])
    s["v"][s["chunk"], s["slot"]] = v
    return {"q": s["q_out"], "k": s["k"], "v": s["v"]}


# ------------------------------------------------------------------------------------------------ in 64 bits, from the definitions
def exact(case, seed):
    s = prepare(case, seed)
    return _exact_axes(case, s) if case["kind"] == "axes" else _exact_attention(case, s)


def _exact_attention(c, s):
    """Request by request, a few hundred rows and one head at a time: softmax over the positions that a row sees."""
    if sum(_seen(c, n, k) for n, k in s["requests"]) * c["heads"] * c["d"] > 4e12:
        return None
    out, group, at = torch.zeros(s["q"].shape, dtype=torch.float64, device=_device()), c["heads"] // c["kv_heads"], 0
    for r, (new, length) in enumerate(s["requests"]):
        kept, rows = _chunks(c, new, length), s["table"][r].tolist()
        where = torch.tensor([i * c["chunk"] + j for i in kept for j in range(c["chunk"])], device=_device())
        numbers = []
        for x, scales in ((s["k"], s["k_scales"]), (s["v"], s["v_scales"])):
            pages = [x[rows[i]] for i in kept]
            if scales is None:
                pages = [p.double() for p in pages]
            else:
                pages = [p.view(torch.float8_e4m3fn).double() * scales[rows[i]].double()[:, None] for i, p in zip(kept, pages)]
            numbers.append(torch.cat(pages).permute(1, 0, 2).contiguous())
        for lo in range(0, new, 512):
            hi = min(new, lo + 512)
            p = torch.arange(length - new + lo, length - new + hi, device=_device())[:, None]
            near = torch.nonzero((where < c["sinks"]) | (where > int(p[0]) - c["window"]) & (where <= int(p[-1])))[:, 0]
            w = where[near]
            hidden = (w > p) | (w <= p - c["window"]) & (w >= c["sinks"])
            for h in range(c["kv_heads"]):
                k, v = numbers[0][h, near], numbers[1][h, near]
                for u in range(h * group, (h + 1) * group):
                    x = (s["q"][at + lo:at + hi, u].double() @ k.t().contiguous()).mul_(s["scale"])
                    out[at + lo:at + hi, u] = torch.softmax(x.masked_fill_(hidden, -math.inf), 1) @ v
        at += new
    return {"out": out}


def _exact_axes(c, s):
    """Pair by pair: a rotation in the plane of its two elements by the angle of the position on its axis."""
    group, d, pairs = c["heads"] // c["kv_heads"], c["d"], len(s["axes"])
    x = s["mixed"].double()
    for part, weight in ((slice(0, group), s["weights"][0]), (slice(group, group + 1), s["weights"][1])):
        if c["norm"] != "none":
            x[:, :, part] /= torch.sqrt(x[:, :, part].square().sum(-1, keepdim=True) / d + 1e-5)
        if weight is not None:
            x[:, :, part] *= weight.double()
    for i, axis in enumerate(s["axes"]):
        a, b = (2 * i, 2 * i + 1) if s["neighbours"] else (i, i + pairs)
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=_device()), s["angles"][s["positions"][axis], a].double())
        plane = torch.complex(x[:, :, :-1, a], x[:, :, :-1, b]) * turn[:, None, None]
        x[:, :, :-1, a], x[:, :, :-1, b] = plane.real, plane.imag
    k, v = torch.zeros(s["k"].shape, dtype=torch.float64, device=_device()), torch.zeros(s["v"].shape, dtype=torch.float64, device=_device())
    k[s["chunk"], s["slot"]], v[s["chunk"], s["slot"]] = x[:, :, -2], x[:, :, -1]
    return {"q": x[:, :, :-2].flatten(1, 2), "k": k, "v": v}
