"""What pins the oracle of speculative decoding."""
import math
import random

import torch

from oracle import paged_attention as oa
from oracle import speculative as osp


def _case(nodes, ctx, Hq=4, Hkv=2, d=8, chunk=16, seed=0):
    gen = torch.Generator().manual_seed(seed)
    lens = [n + c for n, c in zip(nodes, ctx)]
    need = [-(-n // chunk) for n in lens]
    N = sum(need) + 1
    ids = torch.randperm(N, generator=gen).tolist()
    table = torch.zeros(len(lens), max(max(need), 1), dtype=torch.int32)
    for r, k in enumerate(need):
        table[r, :k] = torch.tensor([ids.pop() for _ in range(k)], dtype=torch.int32)
    cu = [0]
    for n in nodes:
        cu.append(cu[-1] + n)
    q = torch.randn(cu[-1], Hq, d, generator=gen)
    kc, vc = torch.randn(N, chunk, Hkv, d, generator=gen), torch.randn(N, chunk, Hkv, d, generator=gen)
    return q, kc, vc, cu, lens, table


def test_a_chain_is_causal_attention():
    q, kc, vc, cu, lens, table = _case([3, 1, 5], [20, 0, 7])
    bits = sum((osp.ancestors(range(-1, n - 1)) for n in (3, 1, 5)), [])
    got, _ = osp.tree_attention(q, kc, vc, cu, lens, table, bits, 8 ** -0.5)
    ref = oa.paged_varlen_attention(q, kc, vc, torch.tensor(cu), torch.tensor(lens), table)
    assert (got - ref).abs().max() < 1e-5


def test_a_tree_is_masked_softmax_and_what_is_not_seen_does_not_matter():
    parents = [-1, 0, 0, 1, 1, 2]
    q, kc, vc, cu, lens, table = _case([6], [10], seed=1)
    bits = osp.ancestors(parents)
    assert bits == [1, 3, 5, 11, 19, 37]
    got, size = osp.tree_attention(q, kc, vc, cu, lens, table, bits, 0.3)
    K, V = kc[0 * 0 + table[0, 0].long()], vc[table[0, 0].long()]
    seen = torch.ones(6, 16, dtype=torch.bool)
    for i in range(6):
        for j in range(6):
            seen[i, 10 + j] = bool(bits[i] >> j & 1)
    for h in range(4):
        x = (q[:, h].double() @ K[:, h // 2].double().t() * 0.3).masked_fill(~seen, -math.inf)
        assert (got[:, h] - torch.softmax(x, 1) @ V[:, h // 2].double()).abs().max() < 1e-12
    assert (size >= got.abs() - 1e-12).all()
    V[10 + 4] = math.nan   # seen by node 4 alone
    K[10 + 4] = math.inf
    again, _ = osp.tree_attention(q, kc, vc, cu, lens, table, bits, 0.3)
    assert torch.equal(again[[0, 1, 2, 3, 5]], got[[0, 1, 2, 3, 5]]) and again[4].isnan().all()


def test_rows_without_keys_are_zeros():
    q, kc, vc, cu, lens, table = _case([2], [0], seed=2)
    got, _ = osp.tree_attention(q, kc, vc, cu, lens, table, [0, 1], 1.0)
    assert (got[0] == 0).all() and (got[1] != 0).any()


def test_masks_of_more_than_one_word(mi):
    parents = list(range(-1, 129))
    rows = osp.mask_rows(osp.ancestors(parents), 3)
    assert rows[0].tolist() == [1, 0, 0] and rows[63].tolist() == [-1, 0, 0] and rows[129].tolist() == [-1, -1, 3]
    assert torch.equal(mi.ops.tree_masks(parents), rows)
    tree = [-1, 0, 0, 1, 1, 2]
    assert mi.ops.tree_masks(tree, words=2).tolist() == [[b, 0] for b in osp.ancestors(tree)]


def _frequencies(run, V, n):
    count = torch.zeros(V, dtype=torch.float64)
    for _ in range(n):
        count[run()] += 1
    return count / n


def _first_token(rng, logits, draft, children, mode):
    """The first new token of one verification, drafted tokens drawn afresh."""
    if mode == "draft":
        tokens = [0] + rng.choices(range(draft.size(1)), weights=draft[0].tolist(), k=children)
    else:
        tokens = [0] + torch.topk(draft[0], children)[1].tolist()
    parents = [-1] + [0] * children
    uniform = [rng.random() for _ in tokens]
    got, _, _ = osp.verify(logits.expand(len(tokens), -1), tokens, parents, [0, len(tokens)], 2,
                           draft_probs=draft.expand(len(tokens), -1) if mode == "draft" else None, uniform=uniform)
    return int(got[0, 0])


def test_first_tokens_are_distributed_as_the_target():
    """Whatever is drafted, the first new token has the target's distribution: 20 000 draws, five standard deviations."""
    gen, rng, n = torch.Generator().manual_seed(3), random.Random(4), 20000
    logits, draft = torch.randn(1, 6, generator=gen), torch.softmax(torch.randn(1, 6, generator=gen), 1)
    p = torch.softmax(logits[0].double(), 0)
    for mode, children in (("draft", 1), ("draft", 3), ("target", 3)):
        f = _frequencies(lambda: _first_token(rng, logits, draft, children, mode), 6, n)  # noqa: B023
        assert ((f - p).abs() <= 5 * (p * (1 - p) / n).sqrt()).all(), (mode, children, f, p)


def test_greedy_paths():
    logits = torch.full((5, 7), -1.0)
    for i, best in enumerate((3, 4, 2, 6, 5)):
        logits[i, best] = 1.0
    tokens, parents = [9, 2, 3, 4, 6], [-1, 0, 0, 2, 3]   # root -> node 2 (token 3) says 2, its child's 4 is not it
    got = osp.verify(logits, tokens, parents, [0, 5], 4, greedy=True)
    assert got[0].tolist() == [[3, 2, -1, -1]] and got[1].tolist() == [[0, 2, -1, -1]] and got[2].tolist() == [2]
    assert osp.verify(logits, tokens, parents, [0, 5], 1, greedy=True)[0].tolist() == [[3]]


def test_moves():
    cache = torch.arange(2 * 3 * 4, dtype=torch.float32).view(2, 3, 4, 1, 1)
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32)
    rows = torch.tensor([[0, 2, 4]], dtype=torch.int32)
    got = osp.keep_accepted(cache, rows, [3], [0, 5], [8], table)          # nodes at positions 3 .. 7
    want = cache.clone()
    want[:, 0, 0], want[:, 0, 1] = cache[:, 0, 1], cache[:, 0, 3]          # node 2 (position 5) -> 4, node 4 (7) -> 5
    assert torch.equal(got, want)
