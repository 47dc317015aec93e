"""GPU parity: verification of drafted tokens against the 64-bit oracle.  Tokens, rows and counts are whole numbers: equal."""
import math
import random

import pytest
import torch

from oracle import speculative as osp

pytestmark = pytest.mark.gpu

MODES = ("draft", "target", "greedy")


def _tree(n, shape, rng):
    if shape == "chain":
        return list(range(-1, n - 1))
    if shape == "flat":
        return ([-1] + [0] * (n - 1))[:n]
    return ([-1] + [min(rng.randint(0, i - 1), rng.randint(0, i - 1)) for i in range(1, n)])[:n]


class Case:
    def __init__(self, dev, nodes, V, mode, *, dtype=torch.float32, shape="tree", temperature=1.0, top_k=0, seed=0, max_path=None,
                 near=0.6, draft_dtype=torch.float32, peaked=True):
        rng, gen = random.Random(seed), torch.Generator().manual_seed(seed)
        trees = [_tree(n, shape, rng) for n in nodes]
        self.cu = [0]
        for n in nodes:
            self.cu.append(self.cu[-1] + n)
        T = self.cu[-1]
        logits = torch.randn(T, V, generator=gen) * 2
        if peaked:
            logits.scatter_add_(1, torch.randint(0, V, (T, 8), generator=gen), 4 + 4 * torch.rand(T, 8, generator=gen))
        draft = torch.softmax(logits / temperature + near * torch.randn(T, V, generator=gen), 1)
        self.logits = logits.to(dtype)
        self.parents, self.tokens = sum(trees, []), []
        for r, tree in enumerate(trees):
            seen = {}
            for i, p in enumerate(tree):
                row = draft[self.cu[r] + max(p, 0)]
                rank = seen[p] = seen.get(p, -1) + 1
                self.tokens.append(int(torch.multinomial(row, 1, generator=gen)) if mode == "draft" else int(row.topk(min(rank + 1, V))[1][-1]))
        self.draft = draft.to(draft_dtype) if mode == "draft" else None
        self.uniform = None if mode == "greedy" else torch.rand(T, generator=gen)
        self.cut = None
        if top_k:
            self.cut = osp.scaled_logits(self.logits, temperature).topk(top_k, 1)[0][:, -1].contiguous()
        depth, self.max_path = [], max_path
        for tree in trees:
            d = []
            for p in tree:
                d.append(1 if p < 0 else d[p] + 1)
            depth += d
        self.max_path = max_path or max(depth + [1])
        self.mode, self.temperature, self.dev = mode, temperature, dev

    def run(self, mi, **change):
        def on(name, x, dtype=None):   # (what a call replaces is not copied from the host)
            if name in change:
                return change[name]
            return x if x is None else (x if dtype is None else torch.tensor(x, dtype=dtype)).to(self.dev)
        return mi.ops.verify_drafted_tokens(
            on("logits", self.logits), on("tokens", self.tokens, torch.int64), on("parents", self.parents, torch.int32),
            on("cu", self.cu, torch.int32), change.get("max_path", self.max_path), greedy=change.get("greedy", self.mode == "greedy"),
            draft_probs=on("draft_probs", self.draft), uniform=on("uniform", self.uniform),
            temperature=change.get("temperature", self.temperature), cut=on("cut", self.cut))

    def reference(self):
        return osp.verify(self.logits, self.tokens, self.parents, self.cu, self.max_path, greedy=self.mode == "greedy", draft_probs=self.draft,
                          uniform=None if self.uniform is None else self.uniform.double().tolist(), temperature=self.temperature,
                          cut=None if self.cut is None else self.cut.tolist())

    def check(self, mi, got=None, **change):
        got = self.run(mi, **change) if got is None else got
        torch.cuda.synchronize()
        for name, x, y in zip(("tokens", "rows", "counts"), got, self.reference()):
            assert x.dtype == y.dtype and torch.equal(x.cpu(), y), (name, x.cpu(), y)
        return got


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [1, 2, 7, 8, 513, 4099, 32003])
def test_vocabularies(mi, dev, mode, dtype, V):
    Case(dev, [5, 1, 9], V, mode, dtype=dtype, seed=V).check(mi)


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("shape", ["chain", "flat", "tree"])
@pytest.mark.parametrize("nodes", [[1], [2], [64, 3, 0, 17], [130, 1]])
def test_shapes(mi, dev, mode, shape, nodes):
    for seed in range(6):
        Case(dev, nodes, 300, mode, shape=shape, seed=seed).check(mi)


@pytest.mark.parametrize("mode,top_k", [("draft", 0), ("target", 0), ("draft", 5), ("target", 5), ("target", 1)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_temperatures_and_cuts(mi, dev, mode, top_k, dtype):
    for i, temperature in enumerate((0.05, 0.7, 1.3, 30.0)):
        Case(dev, [12, 7, 20], 2000, mode, dtype=dtype, temperature=temperature, top_k=top_k, seed=i).check(mi)


@pytest.mark.parametrize("mode", MODES)
def test_large_vocabulary_many_requests(mi, dev, mode):
    Case(dev, [4] * 24 + [0, 30], 128256, mode, dtype=torch.bfloat16, seed=1).check(mi)


def test_draws_of_flat_distributions(mi, dev):
    """A flat distribution over a large vocabulary: every token has a share of 1e-5, and the place of the draw is the sum's."""
    for seed in range(4):
        Case(dev, [2] * 16, 100003, "draft", dtype=torch.float32, seed=seed, peaked=False, temperature=50.0, near=0.3, shape="chain").check(mi)
        Case(dev, [3] * 16, 100003, "target", dtype=torch.float32, seed=seed, peaked=False, temperature=50.0).check(mi)


@pytest.mark.parametrize("mode", MODES)
def test_paths_are_cut(mi, dev, mode):
    for path in (1, 2, 3, 11):
        Case(dev, [8, 8, 8], 40, mode, shape="chain", seed=path, max_path=path, near=0.05).check(mi)


def test_draft_of_16_bits(mi, dev):
    for dtype in (torch.bfloat16, torch.float16):
        Case(dev, [6, 11], 1003, "draft", draft_dtype=dtype, seed=3).check(mi)


def test_siblings_with_one_token(mi, dev):
    """The same token drafted twice after a node: drawn twice it is tried twice, chosen twice it has left already."""
    for mode in ("draft", "target"):
        for seed in range(8):
            c = Case(dev, [6, 6], 12, mode, shape="flat", seed=seed)
            c.tokens = [0, 3, 3, 5, 3, 5] * 2
            c.check(mi)


def test_extreme_numbers(mi, dev):
    """Uniform numbers of zero and just under one; logits of -inf (masked vocabulary) and of the type's lowest value."""
    for mode in ("draft", "target"):
        for u in (0.0, 1 - 2.0 ** -24):
            c = Case(dev, [5, 9], 500, mode, seed=4)
            c.uniform.fill_(u)
            c.check(mi)
        c = Case(dev, [5, 9], 500, mode, seed=5)
        c.logits[:, 100:] = -math.inf
        c.logits[:, 3] = torch.finfo(torch.float32).min
        c.check(mi)
    c = Case(dev, [5, 9], 500, "greedy", seed=5)
    c.logits[:, :100] = -math.inf
    c.logits[:, 200:210] = 50.0     # ties: the first
    c.check(mi)


def test_an_equal_draft_is_accepted(mi, dev):
    """p = q: every draw of the draft is accepted (u < 1), up to the rounding of q's 32 bits at p's 64."""
    c = Case(dev, [6] * 8, 3000, "draft", shape="chain", near=0.0, seed=6)
    c.uniform.mul_(0.999)
    tokens, rows, counts = c.check(mi)
    assert (counts == 6).all()


def test_tokens_and_parents_outside(mi, dev):
    """Tokens that are none are rejected, parents that do not precede are never reached."""
    for mode in MODES:
        c = Case(dev, [6, 8], 200, mode, seed=7)
        c.tokens[1], c.tokens[8], c.tokens[9] = -1, 200, 1 << 40
        c.parents[3], c.parents[4], c.parents[10] = 3, 5, -7
        c.check(mi)


def test_strides(mi, dev):
    """Rows inside a wider tensor, from an odd column on (no row starts at a 16-byte line), poisoned all around."""
    for mode in MODES:
        for dtype in (torch.float32, torch.bfloat16):
            c = Case(dev, [7, 4], 1021, mode, dtype=dtype, seed=8)
            wide = torch.full((11, 1100), math.nan, dtype=dtype, device=dev)
            wide[:, 3:1024] = c.logits.to(dev)
            change = dict(logits=wide[:, 3:1024])
            if mode == "draft":
                more = torch.full((11, 1050), math.nan, device=dev)
                more[:, 5:1026] = c.draft.to(dev)
                change["draft_probs"] = more[:, 5:1026]
            c.check(mi, **change)


def test_the_first_thousand_nodes(mi, dev):
    """A request of more nodes than the walk holds: the first 1 024 are looked at."""
    c = Case(dev, [1300, 5], 50, "target", shape="flat", seed=9)
    cut = Case(dev, [1024, 5], 50, "target", shape="flat", seed=9)
    got = c.run(mi)
    rows = [i for i in range(c.cu[-1]) if not 1024 <= i < 1300]
    cut.logits, cut.uniform = c.logits[rows], c.uniform[rows]
    cut.tokens, cut.parents = [c.tokens[i] for i in rows], [c.parents[i] for i in rows]
    want = cut.reference()
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[2].cpu(), want[2])


def test_no_nodes_at_all(mi, dev):
    c = Case(dev, [0, 0], 100, "target", seed=10, max_path=3)
    c.check(mi)


def test_the_samplers_cut(mi, dev):
    """``cut`` as the sampler returns it: top-k and top-p targets, and tokens that all lie in what it keeps."""
    c = Case(dev, [5, 14, 3], 5000, "target", dtype=torch.bfloat16, temperature=0.8, seed=11)
    for top_k, top_p in ((20, 0.0), (0, 0.7)):
        cut = mi.ops.sample_from_logits(c.logits.to(dev), top_k=top_k, top_p=top_p, temperature=0.8, uniform=c.uniform.to(dev), return_cut=True)[2]
        c.cut = cut.cpu()
        tokens, rows, counts = c.check(mi)
        x = osp.scaled_logits(c.logits, 0.8)
        for r in range(3):
            for i in range(int(counts[r])):
                row = int(rows[r, i])
                assert x[row, int(tokens[r, i])] >= c.cut[row]


def test_replays_and_streams(mi, dev):
    for mode in MODES:
        c = Case(dev, [5, 12, 1], 20000, mode, dtype=torch.bfloat16, seed=12)
        on = lambda x: None if x is None else x.to(dev)  # noqa: E731
        logits, uniform, draft = on(c.logits), on(c.uniform), on(c.draft)
        change = dict(logits=logits, uniform=uniform, draft_probs=draft, tokens=torch.tensor(c.tokens, device=dev),
                      parents=torch.tensor(c.parents, dtype=torch.int32, device=dev), cu=torch.tensor(c.cu, dtype=torch.int32, device=dev))
        eager = c.check(mi, **change)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            aside = c.run(mi, **change)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(x, y) for x, y in zip(aside, eager))
        work = torch.empty(1 << 22, dtype=torch.uint8, device=dev)
        graph = torch.cuda.CUDAGraph()
        with mi.ops.use_workspace(work), torch.cuda.graph(graph):
            kept = c.run(mi, **change)
        for step in range(4):
            logits.copy_(logits.roll(1, 0))
            if uniform is not None:
                uniform.copy_(uniform.roll(1, 0))
            graph.replay()
            again = c.run(mi, **change)
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(kept, again)), (mode, step)


def test_refusals(mi, dev):
    c = Case(dev, [5], 100, "draft", seed=13)
    for change, word in ((dict(uniform=None), "uniform"), (dict(uniform=torch.zeros(4, device=dev)), "uniform"), (dict(tokens=torch.zeros(5, dtype=torch.int32, device=dev)), "tokens"),
                         (dict(parents=torch.zeros(5, dtype=torch.int64, device=dev)), "parents"), (dict(cu=torch.zeros(1, dtype=torch.int32, device=dev)), "two entries"),
                         (dict(max_path=0), "max_path"), (dict(draft_probs=torch.zeros(5, 99, device=dev)), "draft_probs"), (dict(greedy=True), "greedy"),
                         (dict(cut=torch.zeros(3, device=dev)), "cut"), (dict(logits=torch.zeros(5, 100, dtype=torch.float64, device=dev)), "fp32, bf16 or fp16"),
                         (dict(uniform=torch.zeros(5)), "one device")):
        with pytest.raises(ValueError, match=word):
            c.run(mi, **change)
    with pytest.raises(mi._lib.KernelError, match="temperature"):
        c.run(mi, temperature=0.0)


JUST_UNDER_ONE = 1 - 2.0 ** -24


def _kept_tokens(dev, V, kept, drafted, dtype, mode, mask, uniform, root):
    """Requests of a root and children, ``kept[r]`` a request's {token: logit}, everything else left out of its rows by a cut (or
    logits of -inf), ``drafted[r]`` its children's tokens."""
    most = max(len(d) for d in drafted)
    c = Case(dev, [1 + most] * len(kept), V, mode, dtype=dtype, shape="flat", seed=len(kept))
    low = -math.inf if mask == "-inf" else -3.0
    c.logits = torch.full(c.logits.shape, low, dtype=dtype)
    c.tokens, c.cut = [], None if mask == "-inf" else torch.full((c.cu[-1],), -2.0)
    for r, (tokens, children) in enumerate(zip(kept, drafted)):
        for t, x in tokens.items():
            c.logits[c.cu[r]:c.cu[r + 1], t] = x
        c.tokens += [0] + children + [-1] * (most - len(children))
    c.uniform = torch.full((c.cu[-1],), uniform)
    c.uniform[c.cu[:-1]] = root
    if mode == "draft":   # drawn by a draft that knows one of the tokens only
        c.draft = torch.zeros(c.cu[-1], V)
        for r, children in enumerate(drafted):
            c.draft[c.cu[r]:c.cu[r + 1], children[0]] = 1.0
    return c


@pytest.mark.parametrize("mask", ["cut", "-inf"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_the_last_token_of_a_cut_is_accepted(mi, dev, dtype, mask):
    """Two tokens are left, both drafted: the second has all that the first left, and every uniform number accepts it."""
    rng = random.Random(1)
    kept = [{700: 17.625, 9000: 10.375}] + [dict(zip(rng.sample(range(20000), 2), (10 + rng.uniform(0, 9), 10 + rng.uniform(0, 1)))) for _ in range(199)]
    drafted = [sorted(k, key=k.get, reverse=True) for k in kept]
    c = _kept_tokens(dev, 20000, kept, drafted, dtype, "target", mask, JUST_UNDER_ONE, JUST_UNDER_ONE)
    tokens, rows, counts = c.check(mi)
    assert (counts == 2).all()


@pytest.mark.parametrize("mode", ["target", "draft"])
@pytest.mark.parametrize("mask", ["cut", "-inf"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_a_part_without_a_token_is_not_drawn_from(mi, dev, dtype, mask, mode):
    """A rejected token takes its part's whole mass with it, wherever the part lies: what rounding leaves of it is nothing, also
    where the draw looks for the first token of all (a uniform number of zero), for the last one, or where little is left."""
    rng = random.Random(2)
    for root in (0.0, 2.0 ** -24, 1e-30, JUST_UNDER_ONE):
        kept, drafted = [], []
        for r in range(120):
            a, b, c = rng.choice(((100, 17000, 19999), (19000, 10, 11), (9000, 3, 19500), (12000, 12001, 12002)))
            kept.append({a: 15 + rng.uniform(0, 5), b: 10 + rng.uniform(0, 2), **({c: 10 + rng.uniform(0, 2)} if r % 2 else {})})
            drafted.append([a])
        c = _kept_tokens(dev, 20000, kept, drafted, dtype, mode, mask, JUST_UNDER_ONE, root)
        tokens, rows, counts = c.check(mi)
        assert all(int(t) in k for t, k in zip(tokens[:, 0], kept))


@pytest.mark.parametrize("mode", ["target", "draft"])
def test_rows_without_any_token(mi, dev, mode):
    """A cut above every logit leaves nothing to accept and nothing to draw: token 0, whatever the uniform numbers."""
    for root in (0.0, 0.5, JUST_UNDER_ONE):
        c = _kept_tokens(dev, 20000, [{5: 3.0, 17000: 2.0}] * 3, [[5, 17000]] * 3, torch.bfloat16, mode, "cut", 0.3, root)
        c.cut = torch.full((c.cu[-1],), 4.0)
        tokens, rows, counts = c.run(mi)
        assert counts.tolist() == [1, 1, 1] and tokens[:, 0].tolist() == [0, 0, 0]


def test_nothing_left_twice_over(mi, dev):
    """Tokens of probability zero after siblings that took everything: never accepted, and the draw stays among the kept ones."""
    rng = random.Random(3)
    kept = [dict(zip(rng.sample(range(500), 3), (10 + rng.uniform(0, 8) for _ in "abc"))) for _ in range(200)]
    drafted = [sorted(k, key=k.get, reverse=True) + [next(t for t in range(500) if t not in k), -1, sorted(k)[0]] for k in kept]
    for dtype in (torch.float32, torch.bfloat16):
        c = _kept_tokens(dev, 500, kept, drafted, dtype, "target", "cut", JUST_UNDER_ONE, 0.5)
        tokens, rows, counts = c.run(mi)
        for r, k in enumerate(kept):
            for i in range(int(counts[r])):
                assert int(tokens[r, i]) in k, (r, tokens[r], k)


def test_greedy_rows_of_nan(mi, dev):
    """A row without a number has no largest logit: no token is accepted after it, whichever is drafted, and token 0 follows."""
    c = Case(dev, [4, 3], 300, "greedy", shape="flat", seed=14)
    c.logits[:4] = math.nan
    c.tokens[1:4] = [0, (1 << 31) - 1, 299]
    tokens, rows, counts = c.run(mi)
    assert counts[0] == 1 and tokens[0].tolist() == [0, -1] and rows[0].tolist() == [0, -1]
    assert tokens[1, 0] == c.logits[4].argmax()


@pytest.mark.parametrize("draft_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,near", [("chain", 0.1), ("tree", 0.6), ("flat", 3.0)])
def test_draft_rows_of_nodes_without_children_are_not_read(mi, dev, shape, near, draft_dtype):
    """What the children of a node were drawn from exists where it has some: the other rows, the ends of accepted paths among them,
    may hold anything."""
    ends = 0
    for seed in range(6):
        c = Case(dev, [5, 9, 1, 3], 20011, "draft", shape=shape, near=near, seed=seed, draft_dtype=draft_dtype)
        leaves = [i for r in range(4) for i in range(c.cu[r], c.cu[r + 1]) if not any(p == i - c.cu[r] for p in c.parents[c.cu[r]:c.cu[r + 1]])]
        want = c.reference()
        for value in (math.nan, math.inf, 1e30):
            draft = c.draft.clone()
            draft[leaves, ::2] = value
            got = c.run(mi, draft_probs=draft.to(dev))
            assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want)), value
        ends += sum(int(want[1][r, int(want[2][r]) - 1]) in leaves for r in range(4))
    assert ends >= 6


@pytest.mark.parametrize("temperature", [0.3, 0.6, 0.48, 1.2])
@pytest.mark.parametrize("mode", ["draft", "target"])
def test_fp16_logits_over_a_temperature(mi, dev, mode, temperature):
    """Temperatures whose reciprocal brings many fp16 numbers next to the middle between two others: logits are multiplied in 32 bits,
    then rounded, by the sampler that makes the cut as by what is held against it."""
    for seed in range(8):
        for top_k in (1, 2, 5):
            Case(dev, [12, 7, 20, 1, 1, 1], 700, mode, dtype=torch.float16, temperature=temperature, top_k=top_k, seed=seed).check(mi)
    c = Case(dev, [12, 7, 20, 1, 1, 1], 700, mode, dtype=torch.float16, temperature=temperature, seed=9)
    for top_k in (2, 3, 9):
        cut = mi.ops.sample_from_logits(c.logits.to(dev), top_k=top_k, temperature=temperature, uniform=c.uniform.to(dev), return_cut=True)[2]
        c.cut = osp.scaled_logits(c.logits, temperature).topk(top_k, 1)[0][:, -1].contiguous()
        assert torch.equal(cut.cpu(), c.cut)
        c.check(mi)


@pytest.mark.parametrize("children", [0, 2])
@pytest.mark.parametrize("mode", ["draft", "target"])
def test_draws_next_to_a_border(mi, dev, mode, children):
    """Two tokens whose border lies within 1e-10 of the uniform number, but not within 5e-12: the sums that a draw walks along are
    64-bit wherever they come from, also where nothing was rejected, or nothing tried (paths of one node)."""
    gen, rng, found = torch.Generator().manual_seed(15), random.Random(15), []
    while len(found) < 200:
        a, b = (3 * torch.rand(2, 4096, generator=gen)).float()
        p = torch.sigmoid(a.double() - b.double())
        grid = (p * 2 ** 24).round()
        gap = (p - grid / 2 ** 24).abs()
        for i in ((gap > 5e-12) & (gap < 1e-10)).nonzero()[:, 0].tolist():
            found.append((float(a[i]), float(b[i]), float(grid[i] / 2 ** 24)))
    found = found[:200]
    c = Case(dev, [1 + children] * 200, 20000, mode, shape="flat", seed=15, max_path=1)
    c.logits.fill_(-math.inf)
    for r, (a, b, u) in enumerate(found):
        i, j = rng.choice(((3, 9), (3, 15000), (9000, 19999)))
        c.logits[c.cu[r]:c.cu[r + 1], i], c.logits[c.cu[r]:c.cu[r + 1], j] = a, b
        c.uniform[c.cu[r]] = u
    c.check(mi)
