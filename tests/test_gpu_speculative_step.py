"""Steps of speculative decoding as a program runs them: the drafted nodes' keys and values behind the context, attention
over the tree in every layer, the verification, the accepted rows moved together -- until the sequences are long enough.

The model is small enough to be written down: two attention layers whose queries, keys and values are rows of tables,
picked by a token and (keys and values) its position, and logits that are linear in the attention's outputs.  So the
cache after a step must hold, bit for bit, the rows of the sequence so far, and what a greedy step produces must be the
largest logit of the 64-bit model, up to the attention's own rounding:

* a probability is rounded to fp16 once (2^-11 of itself) in numerator and denominator alike: a row is off by 2 * 2^-11
  of the largest value; the output's own rounding is another 2^-11;
* the logits, sums of products with the weights, are off by that much times the sum of the weights' sizes (and the
  32-bit product's own rounding, which the factor 1.1 covers);
* the largest of them can lie behind another by twice that.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

LAYERS, HQ, HKV, D, VOCAB, SCALE = 2, 4, 2, 64, 211, 0.3


class Model:
    def __init__(self, dev, seed):
        g = torch.Generator().manual_seed(seed)
        self.dev = dev
        table = lambda h: torch.randn(LAYERS, VOCAB, h, D, generator=g).half().to(dev)
        self.q, self.k, self.v = table(HQ), table(HKV), table(HKV)
        self.w = torch.randn(LAYERS * HQ * D, VOCAB, generator=g).to(dev)
        self.q64, self.k64, self.v64 = (x.double().cpu() for x in (self.q, self.k, self.v))
        self.w64 = self.w.double().cpu()
        self.slack = 2 * 1.1 * 3 * 2.0 ** -11 * float(self.v64.abs().max()) * float(self.w64.abs().sum(0).max())

    @staticmethod
    def row(token, position):
        return (token + 31 * position) % VOCAB

    def logits64(self, tokens):
        """What follows ``tokens``, in 64 bits."""
        rows = torch.tensor([self.row(t, i) for i, t in enumerate(tokens)])
        out = []
        for l in range(LAYERS):
            q = self.q64[l, tokens[-1]].view(HKV, HQ // HKV, D)
            s = torch.einsum("hgd,nhd->hgn", q, self.k64[l, rows]) * SCALE
            out.append(torch.einsum("hgn,nhd->hgd", s.softmax(-1), self.v64[l, rows]).reshape(-1))
        return torch.cat(out) @ self.w64

    def logits(self, outs):
        return torch.cat([o.reshape(o.size(0), -1).float() for o in outs], 1) @ self.w


def draft(model, tokens, g, most):
    """A tree below the last token: mostly the model's own continuation, one node of it replaced, and random siblings."""
    nodes, parents = [tokens[-1]], [-1]
    at, path, wrong = 0, list(tokens), int(torch.randint(1, most + 1, (1,), generator=g))
    for depth in range(1, most + 1):
        for _ in range(int(torch.randint(0, 3, (1,), generator=g))):
            nodes.append(int(torch.randint(0, VOCAB, (1,), generator=g)))
            parents.append(at)
        token = int(model.logits64(path).argmax())
        nodes.append((token + 1) % VOCAB if depth == wrong else token)
        parents.append(at)
        at = len(nodes) - 1
        path.append(nodes[-1])
    return nodes, parents


class Cache:
    def __init__(self, model, requests, chunk, positions):
        dev = model.dev
        per = -(-positions // chunk)
        order = torch.randperm(requests * per, generator=torch.Generator().manual_seed(9))
        self.table = order.view(requests, per).int().to(dev)
        self.k = torch.full((LAYERS, requests * per, chunk, HKV, D), float("nan"), dtype=torch.half, device=dev)
        self.v = torch.full_like(self.k, float("nan"))
        self.chunk = chunk

    def write(self, model, r, first, rows):
        """Rows of the tables at the positions from ``first`` on."""
        for j, row in enumerate(rows):
            c, o = int(self.table[r, (first + j) // self.chunk]), (first + j) % self.chunk
            self.k[:, c, o], self.v[:, c, o] = model.k[:, row], model.v[:, row]

    def check(self, model, r, tokens):
        at = torch.arange(len(tokens), device=model.dev)
        c, o = self.table[r].long()[at // self.chunk], at % self.chunk
        rows = torch.tensor([model.row(t, i) for i, t in enumerate(tokens)], device=model.dev)
        assert torch.equal(self.k[:, c, o], model.k[:, rows])
        assert torch.equal(self.v[:, c, o], model.v[:, rows])


def prepare(mi, model, cache, seqs, trees):
    """The step's device inputs; ``seqs`` without their last token lie in the cache, which is the trees' root."""
    dev, cu, lens, tokens, parents, masks = model.dev, [0], [], [], [], []
    for r, (seq, (nodes, par)) in enumerate(zip(seqs, trees)):
        depth = []
        for p in par:
            depth.append(0 if p < 0 else depth[p] + 1)
        ctx = len(seq) - 1
        cache.write(model, r, ctx, [model.row(t, ctx + x) for t, x in zip(nodes, depth)])
        cu.append(cu[-1] + len(nodes))
        lens.append(ctx + len(nodes))
        tokens += nodes
        parents += par
        masks.append(mi.ops.tree_masks(par))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    tokens = torch.tensor(tokens, device=dev)
    return dict(cu=i32(cu), lens=i32(lens), tokens=tokens, parents=i32(parents), mask=torch.cat(masks).to(dev),
                q=model.q[:, tokens].contiguous())


def step(mi, model, cache, s, most_path, **verify):
    outs = [mi.ops.paged_tree_attention(s["q"][l], cache.k[l], cache.v[l], s["cu"], s["lens"], cache.table, s["mask"],
                                        softmax_scale=SCALE) for l in range(LAYERS)]
    tokens, rows, counts = mi.ops.verify_drafted_tokens(model.logits(outs), s["tokens"], s["parents"], s["cu"], most_path, **verify)
    lens = mi.ops.kv_keep_accepted(cache.k, cache.v, rows, counts, s["cu"], s["lens"], cache.table)
    return tokens, counts, lens


@pytest.mark.parametrize("chunk", [16, 64])
@pytest.mark.parametrize("mode", ["greedy", "sampled"])
def test_sequences_grow(mi, dev, mode, chunk):
    model, g = Model(dev, 3), torch.Generator().manual_seed(chunk)
    seqs = [[int(x) for x in torch.randint(0, VOCAB, (n,), generator=g)] for n in (1, 2, 40)]
    prompts, cache = [len(s) for s in seqs], Cache(model, len(seqs), chunk, 160)
    for r, seq in enumerate(seqs):
        cache.write(model, r, 0, [model.row(t, i) for i, t in enumerate(seq[:-1])])
    accepted = 0
    for turn in range(5):
        trees = [draft(model, seq, g, 1 + (turn + r) % 5) for r, seq in enumerate(seqs)]
        s = prepare(mi, model, cache, seqs, trees)
        verify = dict(greedy=True) if mode == "greedy" else dict(uniform=torch.rand(len(s["tokens"]), generator=g).to(dev), temperature=4.0)
        tokens, counts, lens = step(mi, model, cache, s, 6, **verify)
        for r, seq in enumerate(seqs):
            n = int(counts[r])
            accepted += n - 1
            seq += tokens[r, :n].tolist()
            assert int(lens[r]) == len(seq) - 1
            cache.check(model, r, seq[:-1])
    if mode == "greedy":
        assert accepted > 0
        for seq, n in zip(seqs, prompts):
            for i in range(n, len(seq)):
                logits = model.logits64(seq[:i])
                assert float(logits[seq[i]]) >= float(logits.max()) - model.slack


def test_a_captured_step(mi, dev):
    """The whole step in one graph, with room for more nodes than a step brings; every replay against an eager step."""
    model, g, most = Model(dev, 5), torch.Generator().manual_seed(1), 48
    seqs = [[int(x) for x in torch.randint(0, VOCAB, (n,), generator=g)] for n in (30, 3)]
    cache, check = Cache(model, 2, 16, 160), Cache(model, 2, 16, 160)
    for r, seq in enumerate(seqs):
        for c in (cache, check):
            c.write(model, r, 0, [model.row(t, i) for i, t in enumerate(seq[:-1])])
    fixed = dict(cu=torch.zeros(3, dtype=torch.int32, device=dev), lens=torch.zeros(2, dtype=torch.int32, device=dev),
                 tokens=torch.zeros(most, dtype=torch.int64, device=dev), parents=torch.full((most,), -1, dtype=torch.int32, device=dev),
                 mask=torch.zeros(most, 1, dtype=torch.int64, device=dev), q=torch.zeros(LAYERS, most, HQ, D, dtype=torch.half, device=dev))

    def fill(s):
        for name, x in s.items():
            if name == "q":
                fixed[name][:, :x.size(1)] = x
            else:
                fixed[name][:x.size(0)] = x

    run = lambda c, s: step(mi, model, c, s, 6, greedy=True)
    graph = None
    for turn in range(6):
        trees = [draft(model, seq, g, 1 + turn % 4) for seq in seqs]
        s = prepare(mi, model, cache, seqs, trees)
        prepare(mi, model, check, seqs, trees)
        fill(s)
        want = run(check, {name: x.clone() for name, x in fixed.items()})
        if graph is None:
            before = cache.k.clone(), cache.v.clone()
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                run(cache, fixed)
            torch.cuda.current_stream().wait_stream(side)
            cache.k.copy_(before[0])
            cache.v.copy_(before[1])
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                got = run(cache, fixed)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        for r, seq in enumerate(seqs):
            seq += got[0][r, :int(got[1][r])].tolist()
            cache.check(model, r, seq[:-1])
