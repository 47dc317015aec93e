"""Steps of speculative decoding that append their nodes the way a program does: norm, rotary embedding and append of the QKV
projection's output in one call (rotary positions are depths, slots follow the node order), or the quantising append of an fp8
cache, whose chunk scales the append sets and the move of the accepted rows converts between.

Every step's nodes, appended in the midst of what earlier steps left, must leave the cache as a linear sequence would have it;
the attention is held against the 64-bit oracle on the cache as it is, within test_gpu_tree_attention's bound: probabilities
rounded once, in numerator and row sum (2 u A, A = sum p |v|), the result once (u |o|), 2e-5 A for exponentials and sums.
"""
import pytest
import torch

from oracle import paged_attention as oa
from oracle import speculative as osp

pytestmark = pytest.mark.gpu

LAYERS, HQ, HKV, VOCAB, MOST = 2, 8, 2, 97, 240


class Steps:
    """Sequences, their trees and their places; a greedy target whose logits follow a drafted child more often than not."""

    def __init__(self, dev, lengths, chunk, d, dtype, seed):
        self.gen, self.dev, self.chunk, self.d, self.dtype = torch.Generator().manual_seed(seed), dev, chunk, d, dtype
        self.seqs = [self.ints(0, VOCAB, n) for n in lengths]
        per = -(-MOST // chunk)
        self.N = len(lengths) * per
        self.table = torch.randperm(self.N, generator=self.gen).view(len(lengths), per).int()

    def ints(self, lo, hi, n):
        return torch.randint(lo, hi, (n,), generator=self.gen).tolist()

    def slots(self, r, positions):
        return [int(self.table[r, p // self.chunk]) for p in positions], [p % self.chunk for p in positions]

    def prompt(self, upto=-1):
        """Tokens, positions and slots of every sequence without its last token."""
        tokens, pos, ci, lo = [], [], [], []
        for r, seq in enumerate(self.seqs):
            n = len(seq) + upto
            c, o = self.slots(r, range(n))
            tokens, pos, ci, lo = tokens + seq[:n], pos + list(range(n)), ci + c, lo + o
        return [torch.tensor(x, dtype=torch.int64) for x in (tokens, pos, ci, lo)]

    def draft(self):
        cu, lens, tokens, parents, pos, ci, lo, bits = [0], [], [], [], [], [], [], []
        for r, seq in enumerate(self.seqs):
            n, ctx, tree, depth = self.ints(1, 14, 1)[0], len(seq) - 1, [-1], [0]
            for i in range(1, n):
                p = max(self.ints(0, i, 1)[0], self.ints(0, i, 1)[0])
                tree.append(p)
                depth.append(depth[p] + 1)
            c, o = self.slots(r, range(ctx, ctx + n))
            cu.append(cu[-1] + n)
            lens.append(ctx + n)
            tokens += [seq[-1]] + self.ints(0, VOCAB, n - 1)
            parents, pos, ci, lo = parents + tree, pos + [ctx + x for x in depth], ci + c, lo + o
            bits += osp.ancestors(tree)
        logits = torch.rand(len(tokens), VOCAB, generator=self.gen)
        for r in range(len(self.seqs)):
            for i in range(cu[r], cu[r + 1]):
                children = [j for j in range(cu[r], cu[r + 1]) if parents[j] == i - cu[r]]
                if children and self.ints(0, 5, 1)[0]:
                    logits[i, tokens[children[self.ints(0, len(children), 1)[0]]]] = 2.0
        return cu, lens, tokens, parents, [torch.tensor(x, dtype=torch.int64) for x in (pos, ci, lo)], bits, logits

    def device(self, *lists):
        return [torch.tensor(x, dtype=torch.int32, device=self.dev) for x in lists]

    def verify(self, mi, cu, tokens, parents, logits):
        """The step's path, which has to be the oracle's."""
        cu_d, parents_d = self.device(cu, parents)
        got = mi.ops.verify_drafted_tokens(logits.to(self.dev), torch.tensor(tokens, device=self.dev), parents_d, cu_d, 9, greedy=True)
        want = osp.verify(logits, tokens, parents, cu, 9, greedy=True)
        assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))
        return got

    def extend(self, tokens, counts, lens):
        for r, seq in enumerate(self.seqs):
            seq += tokens[r, :int(counts[r])].tolist()
            assert int(lens[r]) == len(seq) - 1


def _close(got, q, k, v, cu, lens, table, bits, scale, scales=(None, None)):
    ref, size = osp.tree_attention(q, k, v, cu, lens, table, bits, scale, *scales)
    u = torch.finfo(q.dtype).eps / 2
    err, bound = (got.cpu().double() - ref).abs(), (2 * u + 2e-5) * size * (1 + u) + u * ref.abs() + 1e-7
    assert (err <= bound).all(), float((err / bound).max())


@pytest.mark.parametrize("d,dtype,chunk,norm", [(128, torch.bfloat16, 64, "rms"), (64, torch.float16, 16, None), (128, torch.float16, 256, "l2"),
                                                (64, torch.bfloat16, 64, "rms")])
def test_steps_append_through_the_projections_output(mi, dev, d, dtype, chunk, norm):
    s = Steps(dev, (1, 30, 63, 5), chunk, d, dtype, seed=d + chunk)
    mixed = torch.randn(LAYERS, VOCAB, 1, (HQ + 2 * HKV) * d, generator=s.gen).to(dtype).to(dev)
    weight = (1 + 0.1 * torch.randn(d, generator=s.gen)).to(dtype).to(dev) if norm == "rms" else None
    rotary = mi.synthetic.rotary_angle_table(MOST, d, base=10000.0).to(dev)
    k, v = (torch.full((LAYERS, s.N, chunk, HKV, d), float("nan"), dtype=dtype, device=dev) for _ in "kv")
    table = s.table.to(dev)

    def append(k, v, tokens, pos, ci, lo):
        pos, ci, lo = pos.to(dev), ci.to(dev), lo.to(dev)
        outs = []
        for l in range(LAYERS):
            outs.append(torch.empty(len(tokens), 1, HQ, d, dtype=dtype, device=dev))
            if len(tokens):
                mi.ops.qkv_norm_rope_append(mixed[l, tokens.to(dev)], num_query_heads=HQ, num_kv_heads=HKV, query_out=outs[l], q_weight=weight,
                                            k_weight=weight, norm=norm, rotary_emb=rotary, q_positions=pos, k_positions=pos, k_cache=k[l],
                                            v_cache=v[l], token_to_chunk_idx=ci, token_to_local_pos=lo)
        return outs

    append(k, v, *s.prompt())
    accepted = 0
    for _ in range(6):
        cu, lens, tokens, parents, (pos, ci, lo), bits, logits = s.draft()
        q = append(k, v, torch.tensor(tokens), pos, ci, lo)
        cu_d, lens_d = s.device(cu, lens)
        mask = osp.mask_rows(bits, 1).to(dev)
        for l in range(LAYERS):
            out = mi.ops.paged_tree_attention(q[l], k[l], v[l], cu_d, lens_d, table, mask)
            assert out.shape == q[l].shape
            _close(out.squeeze(1), q[l].squeeze(1).cpu(), k[l].cpu(), v[l].cpu(), cu, lens, s.table, bits, d ** -0.5)
        new, rows, counts = s.verify(mi, cu, tokens, parents, logits)
        accepted += int(counts.sum()) - len(s.seqs)
        s.extend(new, counts, mi.ops.kv_keep_accepted(k, v, rows, counts, cu_d, lens_d, table))
        ref_k, ref_v = torch.zeros_like(k), torch.zeros_like(v)
        prompt = s.prompt()
        append(ref_k, ref_v, *prompt)
        at = (slice(None), prompt[2].to(dev), prompt[3].to(dev))
        assert torch.equal(v[at], ref_v[at]) and torch.equal(k[at], ref_k[at])
    assert accepted > 8


@pytest.mark.parametrize("d,dtype,chunk", [(128, torch.bfloat16, 16), (64, torch.float16, 64), (128, torch.float16, 64), (64, torch.bfloat16, 16)])
def test_steps_append_into_an_fp8_cache(mi, dev, d, dtype, chunk):
    """The append opens a chunk with a scale of its own, steps later overwrite what they did not keep, accepted rows cross chunks:
    bytes and scales are those of the CPU's append and move, step by step."""
    s = Steps(dev, (1, 12, 15, 60), chunk, d, dtype, seed=d + chunk)
    rows16 = [(torch.randn(VOCAB + MOST, HKV, d, generator=s.gen) * torch.linspace(0.3, 3, VOCAB + MOST)[:, None, None]).to(dtype) for _ in range(2 * LAYERS)]
    queries = torch.randn(VOCAB, HQ, d, generator=s.gen).to(dtype)
    table, shape = s.table.to(dev), (LAYERS, s.N, chunk, HKV, d)
    cache = [torch.zeros(shape, dtype=torch.uint8) for _ in "kv"]
    scales = [torch.full((LAYERS, s.N, HKV), 0.01) for _ in "kv"]
    cache_d, scales_d = [x.to(dev) for x in cache], [x.to(dev) for x in scales]

    def append(tokens, pos, ci, lo):
        if not len(tokens):
            return
        for l in range(LAYERS):
            key, value = (rows16[2 * l + i][tokens + (pos if i else 0)] for i in (0, 1))
            mi.ops.kv_append_fp8(key.to(dev), value.to(dev), cache_d[0][l], cache_d[1][l], scales_d[0][l], scales_d[1][l], ci.to(dev), lo.to(dev))
            for i, x in enumerate((key, value)):
                oa.kv_append_fp8(cache[i][l], scales[i][l], x, ci, lo)

    append(*s.prompt())
    crossed = 0
    for _ in range(6):
        cu, lens, tokens, parents, (pos, ci, lo), bits, logits = s.draft()
        append(torch.tensor(tokens), pos, ci, lo)
        cu_d, lens_d = s.device(cu, lens)
        q, mask = queries[tokens], osp.mask_rows(bits, 1).to(dev)
        for l in range(LAYERS):
            out = mi.ops.paged_tree_attention(q.to(dev), cache_d[0][l], cache_d[1][l], cu_d, lens_d, table, mask, softmax_scale=0.1 * d ** -0.5,
                                              k_scales=scales_d[0][l], v_scales=scales_d[1][l])
            _close(out, q, *(x[l].view(torch.float8_e4m3fn).float() for x in cache), cu, lens, s.table, bits, 0.1 * d ** -0.5, (scales[0][l], scales[1][l]))
        new, rows, counts = s.verify(mi, cu, tokens, parents, logits)
        for r in range(len(s.seqs)):
            for i in range(int(counts[r])):
                first = lens[r] - cu[r + 1] + cu[r]
                crossed += (first + i) // chunk != (first + int(rows[r, i]) - cu[r]) // chunk
        lens_new = mi.ops.kv_keep_accepted(*cache_d, rows, counts, cu_d, lens_d, table, k_scales=scales_d[0], v_scales=scales_d[1])
        for i in (0, 1):
            kept = osp.keep_accepted(cache[i].view(torch.float8_e4m3fn).float(), rows.cpu(), counts.tolist(), cu, lens, s.table, scales[i])
            cache[i] = kept.to(torch.float8_e4m3fn).view(torch.uint8)
            assert torch.equal(scales_d[i].cpu(), scales[i])
            assert torch.equal(cache_d[i].cpu().view(torch.float8_e4m3fn).float(), kept)
        s.extend(new, counts, lens_new)
    assert crossed or chunk == 64
