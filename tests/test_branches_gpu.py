"""Several continuations of a sequence: attention by a mask per row, selection over beams, the walk through a checked tree and moves of cached rows, operator by operator
and together, against branches_util's plain forms in 64 bits."""
import importlib.util
import os

import pytest
import torch

import branches_util as U
from conftest import pkg

pytestmark = pytest.mark.gpu
DEV, BF, I32 = "cuda", torch.bfloat16, torch.int32
NAN, INF = float("nan"), float("inf")


def _lib():
    abi = pkg("_abi")
    return abi.lib(), abi.check


def _ptr(t):
    return None if t is None else t.data_ptr()


def _dev(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


# ---- attention -------------------------------------------------------------------------------------------------------------------

class Step:
    """Rows of a step: of each sequence (tokens in front of the rows' contexts, rows' lists of tail tokens); contexts may differ from row to row."""

    def __init__(self, seqs, heads, hkv, block, seed, words=None, pad=0, spread=1.0):
        g = torch.Generator().manual_seed(seed)
        self.heads, self.scale = heads, 128 ** -0.5
        self.seq = torch.tensor([s for s, (_, rows) in enumerate(seqs) for _ in rows], dtype=I32)
        self.ctx = torch.tensor([c if isinstance(c, int) else c[i] for c, rows in seqs for i in range(len(rows))], dtype=I32)
        self.lines = [line for _, rows in seqs for line in rows]
        ends = [0] * len(seqs)
        for s, c, line in zip(self.seq.tolist(), self.ctx.tolist(), self.lines):
            ends[s] = max(ends[s], max(c, 0) + (max(line) + 1 if line else 0))
        self.cache = U.Cache(ends, hkv, block, g, spread=spread)
        self.words = max([1] + [max(line) // 32 + 1 for line in self.lines if line]) if words is None else words
        self.masks = U.masks(self.lines, self.words) if self.words else None
        self.T = len(self.lines)
        self.q = torch.full((self.T, heads * 128 + pad), NAN, dtype=BF)
        self.q[:, :heads * 128] = (torch.randn(self.T, heads * 128, generator=g) * 1.5).to(BF)

    def run(self, ws=None, stream=None, out=None, ldo_pad=0, dev=None):
        lib, check = _lib()
        c = self.cache
        if dev is None:
            dev = _dev(self.q, c.k, c.v, c.bt, self.seq, self.ctx, self.masks)
        q, k, v, bt, seq, ctx, masks = dev
        self.dev = dev
        size = int(lib.b200_paged_attn_tree_workspace_bytes(self.T, self.heads, c.hkv))
        ws = torch.full((size,), 0xff, dtype=torch.uint8, device=DEV) if ws is None else ws
        out = torch.full((self.T, self.heads * 128 + ldo_pad), 7.0, dtype=BF, device=DEV) if out is None else out
        check(lib.b200_paged_attn_tree(q.data_ptr(), q.stride(0), k.data_ptr(), v.data_ptr(), c.n_blocks, bt.data_ptr(), bt.shape[1], _ptr(seq), ctx.data_ptr(), _ptr(masks),
                                       self.words, out.data_ptr(), out.stride(0), self.T, self.heads, c.hkv, c.block, self.scale, ws.data_ptr(), ws.numel(), stream))
        self.ws = ws
        return out

    def seen(self, t):
        c, most = max(int(self.ctx[t]), 0), self.cache.bt.shape[1] * self.cache.block
        return [j for j in list(range(min(c, most))) + [c + i for i in sorted(set(self.lines[t]))] if j < most]

    def check(self, out, rows=None):
        """The result rounded to bf16 (2^-8 of itself); weights of 16 bits, scores and exponentials in fp32: scores off by at most 128 products' 2^-24 of a sum of magnitudes
        below 200, and by 2^-24 of themselves as exponents (below 2^-12 of each weight's share in all)."""
        out, kv, at = out.double().cpu()[:, :self.heads * 128].view(self.T, self.heads, 128), None, -1
        ends = {}
        for t in range(self.T):
            s = int(self.seq[t])
            ends[s] = max([ends.get(s, 0)] + [j + 1 for j in self.seen(t)[-1:]])
        for t in range(self.T) if rows is None else rows:
            s = int(self.seq[t])
            if s != at:
                kv, at = self.cache.rows(s, ends[s]), s
            q = self.q[t, :self.heads * 128].view(self.heads, 128)
            want, share = U.attention(q, *kv, self.seen(t), self.scale)
            off = (out[t] - want).abs() - (2.0 ** -8 * want.abs() + 2.0 ** -12 * share)
            assert (off <= 0).all(), (t, len(self.seen(t)), float(off.max()), int(off.argmax()), out[t].flatten()[off.argmax()], want.flatten()[off.argmax()])


def _random_tree(n, g, back=None):
    """Parents of n nodes, each any node in front of it (no further than `back`)."""
    return [-1] + [int(torch.randint(max(0, i - (back or i)), i, (1,), generator=g)) for i in range(1, n)]


@pytest.mark.parametrize("heads,hkv", [(1, 1), (4, 1), (8, 1), (16, 1), (32, 8), (40, 8), (6, 2), (28, 4), (22, 2), (64, 8), (8, 8)])
def test_trees_for_all_head_layouts(heads, hkv):
    g = torch.Generator().manual_seed(heads)
    seqs = [(c, U.lines(_random_tree(n, g))) for c, n in ((0, 1), (70, 9), (333, 40), (1000, 33), (64, 64), (127, 130))]
    step = Step(seqs, heads, hkv, 128, heads + hkv)
    step.check(step.run())


@pytest.mark.parametrize("block", [16, 32, 64, 128, 256, 384])
def test_blocks_that_end_inside_a_tile(block):
    g = torch.Generator().manual_seed(block)
    seqs = [(c, U.lines(_random_tree(n, g))) for c, n in ((block - 1, 3), (block, 17), (2 * block + 5, 70), (15, 2), (0, block + 3))]
    step = Step(seqs, 8, 2, block, block)
    step.check(step.run())


@pytest.mark.parametrize("ctx", [0, 1, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 640])
def test_edges_of_tiles(ctx):
    seqs = [(ctx, [[0]]), (ctx, [[]]), (ctx, [[0, 1], [0], [1], []]), (ctx, [[63], [64], [65], [31], [32]]), (ctx, [[0, 127, 128]] * 3)]
    step = Step(seqs, 8, 2, 64, ctx)
    step.check(step.run())


def test_rows_that_see_nothing_give_zeros():
    seqs = [(0, [[]]), (0, [[], [], []]), (-5, [[], [0]]), (0, [[], [0, 1], []]), (200, [[3], []]), (0, [[]] * 70)]
    step = Step(seqs, 8, 2, 128, 3)
    out = step.run(ldo_pad=8)
    step.check(out)
    assert (out[0, :1024] == 0).all() and (out[1:4, :1024] == 0).all() and (out[4, :1024] == 0).all() and (out[-70:, :1024] == 0).all()
    assert (out[:, 1024:] == 7).all()   # between the rows


def test_beams_that_share_a_prompt_see_their_own_tokens():
    g = torch.Generator().manual_seed(9)
    seqs = []
    for ctx, W, steps in ((300, 6, 40), (0, 3, 100), (1025, 1, 1), (64, 12, 79)):
        lines = [[b] for b in range(W)]
        for s in range(1, steps):
            lines = [lines[int(torch.randint(0, W, (1,), generator=g))] + [s * W + b] for b in range(W)]
        seqs.append((ctx, lines))
    step = Step(seqs, 32, 8, 32, 5)
    assert step.words == 30
    step.check(step.run())


def test_contexts_that_differ_from_row_to_row():
    g = torch.Generator().manual_seed(2)
    seqs = []
    for n in (5, 40, 90):
        ctx = torch.randint(0, 500, (n,), generator=g).tolist()
        seqs.append((ctx, [sorted(set(torch.randint(0, 200, (int(torch.randint(0, 9, (1,), generator=g)),), generator=g).tolist())) for _ in range(n)]))
    step = Step(seqs, 8, 1, 128, 4)
    step.check(step.run())


def test_no_masks_is_attention_over_contexts():
    step = Step([(list(range(1, 80)), [[]] * 79), (700, [[]] * 5)], 16, 4, 128, 6, words=0)
    step.check(step.run())


def test_masks_wider_than_the_table():
    """Bits that point behind a block table's end are tokens that do not exist."""
    step = Step([(100, [[0, 3], [5]]), (20, [[1], [2, 3]])], 8, 2, 64, 7)
    step.lines = [line + [28, 60, 90, 900] for line in step.lines]
    step.words = 32
    step.masks = U.masks(step.lines, 32)
    step.cache.bt = step.cache.bt[:, :2].contiguous()   # tokens 0..127
    step.cache.k[:], step.cache.v[:] = torch.randn_like(step.cache.k.float()).to(BF), torch.randn_like(step.cache.v.float()).to(BF)
    step.cache.bt[step.cache.bt < 0] = 0
    step.check(step.run())


@pytest.mark.parametrize("what", [NAN, INF, -INF, 3e38])
def test_what_stands_in_unseen_tokens_does_not_matter(what):
    """Keys and values that are no numbers in tokens that some rows see and others do not, and behind the contexts."""
    g = torch.Generator().manual_seed(8)
    seqs = [(70, U.lines(_random_tree(40, g, 3))), (200, [[2 * i] for i in range(64)]), (5, [[0], [1], [0, 2]])]
    step = Step(seqs, 8, 2, 64, 8)
    bad = [(0, 70 + 7), (1, 200 + 6), (1, 200 + 7), (1, 200 + 101), (2, 6)]
    for s, j in bad:
        b, o = step.cache.token(s, j)
        step.cache.k[b, :, o], step.cache.v[b, 0, o, 5], step.cache.v[b, 1, o] = what, what, what
    out = step.run()
    clean = [t for t in range(step.T) if not any(s == int(step.seq[t]) and j in step.seen(t) for s, j in bad)]
    assert 20 < len(clean) < step.T
    step.check(out, clean)
    if what != what:
        assert all(torch.isnan(out[t]).all() for t in range(step.T) if t not in clean)


@pytest.mark.parametrize("what", [NAN, INF, -INF])
def test_values_that_are_no_numbers_reach_the_rows_that_see_them(what):
    step = Step([(130, [[0, 1], [1], [0, 2], [2, 3], [3]]), (300, [[0], [1]])], 8, 2, 64, 9)
    b, o = step.cache.token(0, 131)
    step.cache.v[b, 0, o, 5] = what
    b, o = step.cache.token(1, 17)
    step.cache.v[b, 1, o, 100] = what
    out = step.run().view(step.T, 8, 128).double().cpu()
    for t, h, d in [(t, h, 5) for t in (0, 1) for h in range(4)] + [(t, h, 100) for t in (5, 6) for h in range(4, 8)]:
        assert torch.isnan(out[t, h, d]) if what != what else out[t, h, d] == what
        out[t, h, d] = 0
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("what", [NAN, INF, -INF])
@pytest.mark.parametrize("contexts,idle", [((0,), 0), ((0, 40, 64), 0), ((0, 64), 2), ((10, 70, 130, 5), 1)])
def test_values_that_are_no_numbers_in_walks_over_many_short_sequences(what, contexts, idle):
    """A CTA walks many items of two tiles of pairs and one to four key tiles: every third sequence has values that are no numbers in tokens that only the second tile's rows see,
    the others have none, and some sequences have rows that see nothing."""
    g = torch.Generator().manual_seed(idle + len(contexts))
    heads, hkv, n, seqs = 64, 16, 48, []   # 32 rows to a tile of pairs
    kinds = [k for _ in range(85) for k in ["bad", "clean", "clean"] + ["idle"] * idle][:85]
    for i, kind in enumerate(kinds):
        seqs.append((0, [[]] * n) if kind == "idle" else (contexts[i % len(contexts)], U.lines(_random_tree(n, g, 6))))
    step = Step(seqs, heads, hkv, 64, 40 + idle)
    first, marked = 0, []
    for s, (kind, (ctx, lines)) in enumerate(zip(kinds, seqs)):
        if kind == "bad":
            for j in range(32, n):
                b, o = step.cache.token(s, ctx + j)
                step.cache.v[b, :, o] = what
            marked += range(first + 32, first + n)   # (each sees itself)
        first += n
    clean = sorted(set(range(step.T)) - set(marked))
    out = step.run()
    for _ in range(5):
        got = out.view(step.T, heads * 128)
        assert (torch.isnan(got[marked]) if what != what else got[marked] == what).all()
        assert torch.isfinite(got[clean]).all()
        again = step.run(ws=step.ws, dev=step.dev)
        assert torch.equal(again[clean], out[clean])
        out = again
    step.check(out, [t for t in (*range(0, 2 * n, 7), *range(3 * n, 4 * n, 5)) if t in clean])


@pytest.mark.parametrize("what", [NAN, INF, -INF])
@pytest.mark.parametrize("heads,hkv,nodes,ctx", [(8, 2, 3, 70), (8, 2, 3, 5000), (4, 1, 30, 9000), (32, 8, 40, 9000), (4, 1, 200, 3000)])
def test_values_that_are_no_numbers_under_weights_of_next_to_nothing(what, heads, hkv, nodes, ctx):
    """One of the last tokens has nearly all of the weight, by more than fp32 can tell; what is no number far in front of it is seen all the same, whatever the CTAs' shares."""
    step = Step([(ctx, U.lines(_random_tree(nodes, torch.Generator().manual_seed(3))))], heads, hkv, 128, 50 + nodes)
    b, o = step.cache.token(0, ctx - 1)
    step.q[:] = step.q.abs()
    step.cache.k[b, :, o] = 30.0   # scores of some hundreds, next to some units
    b, o = step.cache.token(0, 5)
    step.cache.v[b, hkv - 1, o, 7] = what
    out = step.run().view(step.T, heads, 128)[:, heads - heads // hkv:, 7]
    assert (torch.isnan(out) if what != what else out == what).all()


def test_blocks_that_are_none_stand_for_zeros():
    step = Step([(300, [[0], [0, 1]]), (100, [[], [2]])], 8, 2, 64, 10)
    step.cache.bt[0, 1], step.cache.bt[0, 3], step.cache.bt[1, 0] = -1, step.cache.n_blocks, 2 ** 30
    step.check(step.run())


def test_rows_of_one_sequence_apart_and_strides():
    """Rows that share a sequence but do not follow one another; padded rows of q and out; sequences in any order."""
    step = Step([(150, U.lines([-1, 0, 0, 1])), (90, U.lines([-1, 0])), (40, [[0]])], 8, 2, 128, 11, pad=24)
    order = torch.tensor([4, 0, 6, 2, 5, 1, 3])
    step.seq, step.ctx, step.q, step.masks, step.lines = step.seq[order], step.ctx[order], step.q[order].contiguous(), step.masks[order].contiguous(), [step.lines[i] for i in order]
    out = step.run(ldo_pad=40)
    step.check(out)
    assert (out[:, 1024:] == 7).all()


def test_rows_without_a_map_are_sequences():
    step = Step([(c, [[0]]) for c in (5, 100, 300)], 8, 2, 128, 12)
    want = step.run()
    dev = list(step.dev)
    dev[4] = None
    assert torch.equal(step.run(dev=dev), want)


def test_long_contexts_and_many_tiles():
    g = torch.Generator().manual_seed(13)
    step = Step([(20000, U.lines(_random_tree(70, g, 6))), (9, U.lines(_random_tree(3, g))), (5003, U.lines(_random_tree(20, g)))], 4, 1, 128, 13)
    step.check(step.run(), [0, 1, 35, 69, 70, 72, 73, 92])


@pytest.mark.parametrize("heads,hkv,nodes,ctx", [(4, 1, 30, 9000), (16, 1, 1, 12000), (4, 1, 51, 2600), (1, 1, 3, 9000), (32, 8, 8, 600), (32, 8, 40, 9000), (64, 8, 2, 5000)])
def test_items_of_many_parts(heads, hkv, nodes, ctx):
    """One sequence over all CTAs: parts of 2 to 140 CTAs are joined by one to eight warps a job."""
    step = Step([(ctx, U.lines(_random_tree(nodes, torch.Generator().manual_seed(nodes))))], heads, hkv, 128, nodes + ctx)
    out = step.run()
    step.check(out, rows=sorted({0, nodes // 2, nodes - 1}))
    assert torch.equal(out, step.run())


def test_thousands_of_short_sequences_beside_a_long_one():
    """More walks of a CTA than its table holds; contexts of nothing among them."""
    g = torch.Generator().manual_seed(16)
    ctx = torch.randint(0, 90, (2000,), generator=g).tolist()
    ctx[1234], ctx[0], ctx[1999] = 9000, 0, 65
    step = Step([(c, [[] if c % 7 == 0 else [0]]) for c in ctx], 16, 8, 16, 16)
    first = step.run()
    step.check(first, [0, 1, 2, 500, 1000, 1233, 1234, 1235, 1998, 1999, *range(40, 1900, 97)])
    assert torch.equal(step.run(ws=step.ws, dev=step.dev), first)


@pytest.mark.parametrize("sizes", [(4096,), (1, 4000, 95), tuple(list(range(1, 90)) + [91])])
def test_steps_of_the_most_rows(sizes):
    g = torch.Generator().manual_seed(len(sizes))
    assert sum(sizes) == 4096
    seqs = [(int(torch.randint(0, 300, (1,), generator=g)), [torch.randperm(90, generator=g)[:int(torch.randint(0, 9, (1,), generator=g))].tolist() for _ in range(n)]) for n in sizes]
    step = Step(seqs, 4, 2, 64, 17)
    step.check(step.run(), [0, 1, 63, 64, 65, 127, 128, 1000, 2047, 4000, 4001, 4095, *range(300, 4000, 171)])


def test_scores_far_apart():
    """Maxima that rise along the context, and fall: rescaling, and weights of nothing."""
    step = Step([(700, [[0, 1], [1], [0]]), (640, [[]] * 3)], 8, 2, 64, 14)
    for s, n in ((0, 702), (1, 640)):
        for j in range(0, n, 50):
            b, o = step.cache.token(s, j)
            step.cache.k[b, :, o] = (step.cache.k[b, :, o].float() * (8 if s == 0 else 16)).to(BF)
    step.q = (step.q.float() * 2).to(BF)
    out = step.run().double().cpu().view(step.T, 8, 128)
    for t in range(step.T):   # scores up to some hundreds: off by 2^-23 of them and of their products' magnitudes
        kv = step.cache.rows(int(step.seq[t]), 702)
        want, share = U.attention(step.q[t].view(8, 128), *(x[:int(step.ctx[t]) + 2] for x in kv), step.seen(t), step.scale)
        off = (out[t] - want).abs() - (2.0 ** -8 * want.abs() + 2.0 ** -9 * share)
        assert (off <= 0).all(), (t, float(off.max()))


def test_values_far_apart_in_one_tile():
    step = Step([(200, [[0], [1], [0, 2]])], 8, 2, 64, 15, spread=12.0)
    step.check(step.run())


@pytest.mark.parametrize("T,ctx", [(1, 600), (3, 9000), (200, 300)])
def test_the_same_bits_every_time_and_whatever_the_workspace_holds(T, ctx):
    g = torch.Generator().manual_seed(T)
    step = Step([(ctx, U.lines(_random_tree(T, g)))], 8, 2, 128, T)
    first = step.run()
    for fill in (0, 0x7f, 0xff):
        step.ws.fill_(fill)
        assert torch.equal(step.run(ws=step.ws, dev=step.dev), first)


def test_captured_graphs_and_two_streams():
    g = torch.Generator().manual_seed(21)
    steps = [Step([(400 + 300 * i, U.lines(_random_tree(30, g))), (50, U.lines(_random_tree(5, g)))], 8, 2, 128, 21 + i) for i in range(2)]
    want = [s.run() for s in steps]
    torch.cuda.synchronize()
    outs, graphs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for s, stream in zip(steps, streams):
        out, graph = torch.zeros_like(want[0]), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            s.run(ws=s.ws, out=out, dev=s.dev, stream=torch.cuda.current_stream().cuda_stream)
        outs.append(out)
        graphs.append(graph)
    for _ in range(3):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
    # other inputs at the same addresses
    q2 = (steps[0].q.float() * -0.5).to(BF)
    steps[0].dev[0].copy_(q2)
    graphs[0].replay()
    torch.cuda.synchronize()
    steps[0].q = q2
    steps[0].check(outs[0])


# ---- selection over beams ---------------------------------------------------------------------------------------------------------

def select(logits, scores, starts, take, ws=None, stream=None, ld=None, vocab=None, at=None):
    lib, check = _lib()
    S, n = starts.shape[0] - 1, logits.shape[0]
    V, ld = vocab or logits.shape[1], ld or logits.stride(0)
    size = int(lib.b200_beam_select_workspace_bytes(n, V, take))
    ws = torch.full((size + 16,), 0xff, dtype=torch.uint8, device=DEV) if ws is None else ws
    rows, tokens = (torch.full((S, take), -9, dtype=I32, device=DEV) for _ in range(2))
    out = torch.full((S, take), 9.0, device=DEV)
    check(lib.b200_beam_select((logits if at is None else at).data_ptr(), ld, _ptr(scores), starts.data_ptr(), S, n, V, take, rows.data_ptr(), tokens.data_ptr(), out.data_ptr(), ws.data_ptr(), size, stream))
    return rows, tokens, out


def check_select(logits, scores, starts, take, **kw):
    l, sc, st = _dev(logits, scores, starts)
    got = [x.cpu() for x in select(l, sc, st, take, **kw)]
    want = U.select(logits, scores, starts, take)
    assert torch.equal(got[0].long(), want[0]) and torch.equal(got[1].long(), want[1]), (got, want)
    fine = torch.isfinite(want[2])
    assert torch.equal(torch.isfinite(got[2]), fine)
    # rounded once to fp32; a log-sum of fp32 exponentials is good to 2e-6
    assert ((got[2].double() - want[2])[fine].abs() <= 2.0 ** -24 * want[2][fine].abs() + 2e-6).all()


def _starts(*sizes):
    return torch.tensor([0, *sizes], dtype=torch.int64).cumsum(0).to(I32)


@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 9, 255, 2048, 2049, 4097, 16384, 16385, 32000, 50001])
@pytest.mark.parametrize("take", [1, 8, 37])
def test_select_at_many_vocabularies(vocab, take):
    g = torch.Generator().manual_seed(vocab + take)
    logits = (torch.randn(9, vocab, generator=g) * 3).to(BF)
    check_select(logits, -6 * torch.rand(9, generator=g), _starts(1, 4, 0, 3, 1), take)


@pytest.mark.parametrize("seqs,beams,vocab,take", [(1, 1, 128256, 1), (1, 4, 128256, 8), (3, 16, 128256, 32), (40, 8, 128256, 16), (300, 2, 32000, 4), (2, 64, 5000, 128), (1, 3, 393216, 128)])
def test_select_at_many_sizes(seqs, beams, vocab, take):
    g = torch.Generator().manual_seed(seqs)
    logits = (torch.randn(seqs * beams, vocab, generator=g) * 2 + torch.randn(vocab, generator=g)).to(BF)
    check_select(logits, -9 * torch.rand(seqs * beams, generator=g), _starts(*[beams] * seqs), take)


@pytest.mark.parametrize("seqs,beams,vocab,take", [(5, 3, 26316, 20), (3, 3, 128256, 64), (2, 8, 32000, 128), (4, 1, 1024, 64), (3, 2, 300, 128), (2, 40, 2100, 128), (1, 2, 26316, 100)])
@pytest.mark.parametrize("far", [0.0, 6.0, 40.0])
def test_select_from_few_blocks(seqs, beams, vocab, take, far):
    """Little more than as many blocks of logits as are to be taken, of rows that are far apart: the best row has thousands of entries in front of the other rows' best."""
    g = torch.Generator().manual_seed(vocab + take)
    logits = (torch.randn(seqs * beams, vocab, generator=g) * 2.5).to(BF)
    check_select(logits, -far * torch.rand(seqs * beams, generator=g), _starts(*[beams] * seqs), take)


@pytest.mark.parametrize("take", [1, 5, 16, 128])
def test_select_among_ties(take):
    """Entries alike within a row and between rows: the lower row, then the lower entry; more of them than any list holds."""
    g = torch.Generator().manual_seed(take)
    few = torch.randint(0, 3, (6, 30000), generator=g).to(BF)
    check_select(few, torch.tensor([-1.0, -1.0, -2.0, -1.0, -1.0, -1.0]), _starts(2, 4), take)
    same = few[:1].expand(6, -1).contiguous()
    check_select(same, None, _starts(6), take)
    check_select(torch.zeros(6, 30000, dtype=BF), None, _starts(3, 3), take)
    signs = torch.where(torch.rand(4, 9000, generator=g) < 0.5, 0.0, -0.0).to(BF)
    check_select(signs, None, _starts(4), take)
    climbing = (torch.arange(40000).float() / 40000).to(BF)[None].expand(5, -1).contiguous()   # a thread's entries are all larger than the next one's
    check_select(climbing, -torch.arange(5).float() * 1e-7, _starts(5), take)
    check_select(climbing.flip(1).contiguous(), torch.zeros(5), _starts(1, 4), take)


def test_select_between_rows_that_are_nearer_than_fp32_sums_tell():
    """Rows whose largest candidates differ by some 1e-8: the order is that of 64 bits."""
    g = torch.Generator().manual_seed(77)
    V = 20000
    base = (torch.randn(1, V, generator=g) * 2).to(BF)
    logits = base.repeat(12, 1)
    for r in range(12):
        logits[r, int(torch.randint(0, V, (1,), generator=g))] = -7.0 - r   # moves a log-sum a little
    x = logits.double()
    lse = x.logsumexp(1)
    assert float((lse.max() - lse.min())) < 1e-3
    check_select(logits, None, _starts(12), 24)
    check_select(logits[:4].contiguous(), (lse - lse[0]).float()[:4], _starts(4), 24)   # nearer still: fp32's rounding of the scores apart


@pytest.mark.parametrize("order", ["last", "first", "middle"])
def test_select_among_more_alike_than_any_list_holds(order):
    """Rows alike in every entry, whose scores differ by less than fp32 sums tell."""
    logits = torch.zeros(64, 50000, dtype=BF)
    scores = -1e-9 * torch.arange(64.0)
    scores = {"first": scores, "last": scores.flip(0), "middle": scores[torch.randperm(64, generator=torch.Generator().manual_seed(3))]}[order]
    check_select(logits, scores, _starts(64), 128)


def test_select_among_alike_rows_beside_rows_that_are_none():
    """The sums in 64 bits are asked for, and rows with a NaN, an infinity or nothing stay out of it."""
    logits = torch.zeros(7, 30000, dtype=BF)
    logits[0, 29999], logits[2, 77], logits[3], logits[5, :] = NAN, INF, -INF, 1e-39
    check_select(logits, None, _starts(7), 100)
    check_select(logits, torch.tensor([0.0, -1.0, 0.0, 0.0, -1.0, -1.0, NAN]), _starts(7), 100)


@pytest.mark.parametrize("rows,blocks,take,second,first", [(4, 16, 16, 40000, 600), (4, 16, 16, 40000, 700), (4, 16, 16, 20000, 400), (8, 8, 16, 20000, 400), (8, 8, 16, 40000, 700),
                                                           (4, 32, 8, 40000, 300), (4, 32, 8, 20000, 1000), (16, 8, 16, 20000, 200), (16, 8, 16, 40000, 1000)])
def test_select_among_more_than_a_list_holds_has_the_same_bits_every_time(rows, blocks, take, second, first):
    """One entry far in front, some hundreds a step behind it in few blocks, tens of thousands another step behind in all: a limit near the end depends on which of them are looked at, and
    with it whether sums are wanted in 64 bits.  Scores next to zero, where fp32 shows the difference."""
    g = torch.Generator().manual_seed(first + second)
    V = blocks * 2048
    x = (torch.randn(rows, V, generator=g) * 0.5 - 6).clamp(max=-3.0)
    few = torch.randperm(rows * blocks, generator=g)[:take - 4]
    x.view(-1)[torch.randperm(rows * V, generator=g)[:second]] = 2.0
    places = (few[:, None] * 2048 + torch.arange(2048)).reshape(-1)
    x.view(-1)[places[torch.randperm(len(places), generator=g)[:first]]] = 3.0
    x[0, 5] = 11.0
    logits = x.to(BF)
    scores = (logits.double().logsumexp(1) - 3.0 + 0.01 * torch.arange(1, rows + 1)).float()
    check_select(logits, scores, _starts(rows), take)
    dev = _dev(logits, scores, _starts(rows))
    want = select(*dev, take)
    for _ in range(40):
        assert all(torch.equal(a, b) for a, b in zip(select(*dev, take), want))


def test_select_between_many_rows_that_are_near():
    """More rows than are kept at hand, all of them in need of 64 bits; in two sequences."""
    g = torch.Generator().manual_seed(78)
    base = (torch.randn(1, 3000, generator=g) * 2).to(BF)
    logits = base.repeat(1300, 1)
    logits[torch.arange(1300), torch.randint(0, 3000, (1300,), generator=g)] = -9.0
    check_select(logits, None, _starts(100, 1200), 128)


def test_select_adds_up_a_row_once_wherever_it_stands():
    """A row's only candidate, and another row's 800 next to it: two rows are wanted in 64 bits, at the front of 1 200 rows and behind the first 1 024 (as often as they were
    compared, 6.0 ms against 0.27)."""
    g = torch.Generator().manual_seed(79)
    rest = (torch.randn(1200, 4096, generator=g) - 6).to(BF)
    times = []
    for at in (0, 1100):
        logits = rest.clone()
        logits[at], logits[at + 1] = -9.0, -9.0
        logits[at, 7] = logits[at + 1, 100:900] = 2.0
        scores = torch.full((1200,), -30.0)
        scores[at] = 5e-7   # (ahead of the others by some of it)
        scores[at + 1] = float(logits[at + 1].double().logsumexp(0) - logits[at].double().logsumexp(0))   # (fp32: nearer than sums tell)
        check_select(logits, scores, _starts(1200), 1)
        dev = _dev(logits, scores, _starts(1200))
        each = []
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            select(*dev, 1)
            b.record()
            torch.cuda.synchronize()
            each.append(a.elapsed_time(b))
        times.append(min(each))
    assert times[1] < 10 * times[0], times


def test_select_without_rows():
    starts = torch.zeros(4, dtype=I32, device=DEV)
    for rows, tokens, out in (select(torch.zeros(0, 50, dtype=BF, device=DEV), None, starts, 5, ld=50, vocab=50, at=starts), select(torch.zeros(3, 50, dtype=BF, device=DEV), None, starts, 5)):
        assert (rows == -1).all() and (tokens == -1).all() and (out == -INF).all()


def test_select_without_candidates():
    g = torch.Generator().manual_seed(5)
    logits = torch.randn(9, 500, generator=g).to(BF)
    logits[1], logits[2, 7], logits[3, 9] = -INF, NAN, INF
    logits[4, 3:], logits[5] = -INF, NAN
    scores = torch.tensor([-1.0, -1, -1, -1, -1, -1, -INF, NAN, INF])
    check_select(logits, scores, _starts(9), 16)
    check_select(logits, scores, _starts(1, 1, 1, 1, 1, 1, 1, 1, 1), 8)     # sequences with nothing, and with three
    check_select(logits, None, _starts(0, 2, 0, 7, 0), 4)
    check_select(logits[4:5].contiguous(), None, _starts(1), 8)


def test_select_of_logits_at_any_scale():
    g = torch.Generator().manual_seed(6)
    x = torch.randn(8, 3000, generator=g)
    for f in (1e-30, 1e-3, 1e3, 1e30, 1e38):
        logits = (x * f).clamp(-3e38, 3e38).to(BF)
        if f > 1e4:   # (as 64-bit numbers, scores of that size leave nothing of the beams' own)
            check_select(logits[:1].contiguous(), None, _starts(1), 4)
        else:
            check_select(logits, torch.rand(8, generator=g) * -4, _starts(4, 4), 12)
    below = -x.abs() - 0.5
    check_select(below.to(BF), torch.full((8,), -1e30), _starts(4, 4), 100)   # (sums of which nothing but the beams' own is left)
    low = torch.full((4, 3000), -3.3895e38).to(BF)   # masked by the type's lowest value
    low[:, 5:9] = x[:4, 5:9].to(BF)
    check_select(low, None, _starts(2, 2), 3)


def test_select_of_rows_at_any_address():
    g = torch.Generator().manual_seed(7)
    wide = torch.full((6 * 5003 + 9,), INF, dtype=BF)
    for shift in (0, 1, 3, 8):
        rows = torch.as_strided(wide, (6, 4999), (5003, 1), shift)
        rows.copy_((torch.randn(6, 4999, generator=g) * 3).to(BF))
        dev = wide.to(DEV)
        got = select(torch.as_strided(dev, (6, 4999), (5003, 1), shift), None, _starts(4, 2).to(DEV), 9)
        want = U.select(rows, None, _starts(4, 2), 9)
        assert torch.equal(got[0].cpu().long(), want[0]) and torch.equal(got[1].cpu().long(), want[1])
        wide.fill_(INF)


def test_select_leaves_rows_of_no_sequence_alone():
    g = torch.Generator().manual_seed(8)
    logits = torch.randn(7, 3000, generator=g).to(BF)
    starts = torch.tensor([2, 4, 6], dtype=I32)
    check_select(logits, None, starts, 5)


def test_select_captured_with_another_on_its_own_workspace():
    g = torch.Generator().manual_seed(9)
    cases = [((torch.randn(8, 9000, generator=g) * 3).to(BF).to(DEV), _starts(4, 4).to(DEV)) for _ in range(2)]
    cases[1] = (cases[1][0][:1].expand(8, -1).contiguous(), cases[1][1])   # (this one adds up in fp64)
    want = [select(l, None, st, 6) for l, st in cases]
    graphs, outs, keep = [], [], []
    for l, st in cases:
        ws, graph, stream = torch.full((1 << 20,), 0xff, dtype=torch.uint8, device=DEV), torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=stream):
            outs.append(select(l, None, st, 6, ws=ws, stream=torch.cuda.current_stream().cuda_stream))
        graphs.append((graph, stream))
        keep.append(ws)
    for _ in range(3):
        for graph, stream in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for got, ref in zip(outs, want) for a, b in zip(got, ref))


# ---- the walk through a checked tree, and moves -------------------------------------------------------------------------------------

def accept(target, drafts, parents, starts, slots):
    lib, check = _lib()
    n = target.shape[0]
    out, path, src, dst = (torch.full((n,), -9, dtype=I32, device=DEV) for _ in range(4))
    accepted = torch.full((len(starts) - 1,), -9, dtype=I32, device=DEV)
    t, d, p, st, sl = _dev(target, drafts, parents, starts, slots)
    check(lib.b200_accept_tree(t.data_ptr(), d.data_ptr(), p.data_ptr(), st.data_ptr(), _ptr(sl), len(starts) - 1, n, out.data_ptr(), path.data_ptr(), accepted.data_ptr(),
                               src.data_ptr() if slots is not None else None, dst.data_ptr() if slots is not None else None, None))
    return out, path, accepted, src, dst


@pytest.mark.parametrize("sizes", [(1,), (2,), (31, 32, 33), (0, 5, 0), (127, 128, 129), (300, 1, 64), tuple([9] * 200), (1000, 1025)])
@pytest.mark.parametrize("alphabet", [1, 2, 5])
def test_accept_walks_the_tree(sizes, alphabet):
    g = torch.Generator().manual_seed(sum(sizes) * 7 + alphabet)
    starts = _starts(*sizes)
    n = int(starts[-1])
    parents = torch.tensor([p for s in sizes for p in (_random_tree(s, g, 4) if s else [])], dtype=I32)
    drafts, target = (torch.randint(0, alphabet, (n,), generator=g).to(I32) for _ in range(2))
    slots = torch.randperm(3 * n + 1, generator=g)[:n].to(I32)
    got = accept(target, drafts, parents, starts, slots)
    for x, y in zip(got, U.accept(target, drafts, parents, starts, slots)):
        assert torch.equal(x.cpu().long(), y)


def test_accept_of_rows_of_no_sequence_and_of_parents_that_are_none():
    starts = torch.tensor([2, 6, 9], dtype=I32)
    parents = torch.tensor([9, 9, -1, 0, 7, -3, -1, 2, 1], dtype=I32)   # 7, -3: no rows in front; the last sequence's second row names the third
    drafts, target = torch.zeros(12, dtype=I32), torch.zeros(12, dtype=I32)
    parents = torch.cat([parents, torch.zeros(3, dtype=I32)])
    out, path, accepted, src, dst = (x.cpu().tolist() for x in accept(target, drafts, parents, starts, torch.arange(12, dtype=I32)))
    assert accepted == [1, 0]
    assert out == [-9, -9, 0, 0, -1, -1, 0, -1, -1, -9, -9, -9] and path == [-9, -9, 2, 3, -1, -1, 6, -1, -1, -9, -9, -9]
    got = accept(target, drafts, parents, starts, None)
    assert got[0].cpu().tolist() == out and (got[3] == -9).all()


def move(a, b, src, dst, starts, most):
    lib, check = _lib()
    L, N, H, B = a.shape[:4]
    row = a[0, 0, 0, 0].numel() * a.element_size()
    check(lib.b200_cache_move(a.data_ptr(), _ptr(b), L, a.stride(0) * a.element_size(), N, H, B, row, src.data_ptr(), dst.data_ptr(), starts.data_ptr(), starts.shape[0] - 1, most, None))


def _moves(slots, sizes, g, share):
    """Per group random sources and distinct destinations among its own slots, and some entries that are no moves."""
    src, dst, at = [], [], 0
    for n in sizes:
        own = slots[at:at + n]
        s = own[torch.randint(0, max(n, 1), (n,), generator=g)] if n else own
        d = own[torch.randperm(n, generator=g)]
        none = torch.rand(n, generator=g) < share
        src.append(torch.where(none, -1, s))
        dst.append(d)
        at += n
    return torch.cat(src).to(I32), torch.cat(dst).to(I32)


@pytest.mark.parametrize("layers,blocks,heads,block,width,dtype", [
    (3, 9, 4, 16, 128, BF), (1, 40, 1, 1, 4096, torch.float32), (2, 12, 3, 32, 1, torch.uint8), (2, 12, 2, 32, 129, torch.uint8), (1, 700, 1, 1, 6, BF), (2, 8, 2, 64, 100, torch.float32),
    (1, 24, 1, 1, 300001, torch.uint8), (1, 24, 1, 1, 70000, torch.float32), (5, 30, 8, 128, 128, BF)])
@pytest.mark.parametrize("sizes", [(8,), (1, 2, 0, 5), (3, 3, 3, 3)])
def test_moves_happen_at_once(layers, blocks, heads, block, width, dtype, sizes):
    g = torch.Generator().manual_seed(width + len(sizes))
    a, b = (torch.randint(0, 200, (layers, blocks, heads, block, width), generator=g).to(dtype) for _ in range(2))
    slots = torch.randperm(blocks * block, generator=g)[:sum(sizes)]
    src, dst = _moves(slots, sizes, g, 0.2)
    starts = _starts(*sizes)
    da, db, ds, dd, dst_ = _dev(a, b, src, dst, starts)
    move(da, db, ds, dd, dst_, max(sizes))
    assert torch.equal(da.cpu(), U.moved(a, src, dst, starts, max(sizes))) and torch.equal(db.cpu(), U.moved(b, src, dst, starts, max(sizes)))
    da = a.to(DEV)
    move(da, None, ds, dd, dst_, max(sizes))
    assert torch.equal(da.cpu(), U.moved(a, src, dst, starts, max(sizes)))


@pytest.mark.parametrize("n", [64, 257, 1000, 1024])
def test_moves_of_large_groups(n):
    g = torch.Generator().manual_seed(n)
    a = torch.randint(0, 99, (2, 40, 2, 32, 128), generator=g).to(BF)
    slots = torch.randperm(1280, generator=g)[:n]
    src, dst = _moves(slots, (n,), g, 0.1)
    starts = _starts(n)
    da, ds, dd, st = _dev(a, src, dst, starts)
    move(da, None, ds, dd, st, n)
    assert torch.equal(da.cpu(), U.moved(a, src, dst, starts, n))


@pytest.mark.parametrize("sizes,width", [((6, 3, 1, 6), 1 << 20), ((1,) * 9, 700000), ((40,), 300016)])
def test_moves_of_large_states(sizes, width):
    """Many batches to a CTA."""
    g = torch.Generator().manual_seed(width)
    n = sum(sizes) + 3
    a, b = (torch.randint(0, 256, (2, n, 1, 1, width), generator=g).to(torch.uint8) for _ in range(2))
    starts = _starts(*sizes)
    da, db, ds = _dev(a, b, starts)
    for _ in range(4):
        src, dst = _moves(torch.randperm(n, generator=g)[:sum(sizes)], sizes, g, 0.1)
        a, b = (U.moved(x, src, dst, starts, max(sizes)) for x in (a, b))
        move(da, db, src.to(DEV), dst.to(DEV), ds, max(sizes))
    assert torch.equal(da.cpu(), a) and torch.equal(db.cpu(), b)


def test_moves_of_keys_that_are_their_values():
    """The same cache given twice: rows that change places do so once."""
    g = torch.Generator().manual_seed(8)
    a = torch.randint(0, 99, (4, 64, 1, 64, 576), generator=g).to(BF)
    slots = torch.randperm(64 * 64, generator=g)[:2000]
    src, dst, starts = slots.to(I32), slots.view(-1, 2).flip(1).reshape(-1).to(I32), _starts(*[40] * 50)   # pairs change places
    da, ds, dd, st = _dev(a, src, dst, starts)
    want = U.moved(a, src, dst, starts, 40)
    for i in range(4):
        move(da, da, ds, dd, st, 40)
        assert torch.equal(da.cpu(), want if i % 2 == 0 else a)


def test_walk_and_moves_captured_with_another_pair():
    """Two graphs on streams of their own, replayed with other choices of the target at the same addresses."""
    lib, check = _lib()
    g = torch.Generator().manual_seed(6)
    starts, n, B = _starts(9, 20, 1), 30, 32
    parents = torch.tensor([p for s in (9, 20, 1) for p in _random_tree(s, g, 4)], dtype=I32)
    slots = torch.arange(n, dtype=I32) * 3 + 1
    runs = []
    for _ in range(2):
        cache = torch.randint(0, 99, (2, 3, 2, B, 64), generator=g).to(BF)
        dev = _dev(torch.zeros(n, dtype=I32), torch.randint(0, 2, (n,), generator=g).to(I32), parents, starts, slots, cache)
        out = [torch.full((n,), -9, dtype=I32, device=DEV) for _ in range(4)] + [torch.full((3,), -9, dtype=I32, device=DEV)]
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            st, (t, d, p, f, sl, c) = torch.cuda.current_stream().cuda_stream, dev
            check(lib.b200_accept_tree(t.data_ptr(), d.data_ptr(), p.data_ptr(), f.data_ptr(), sl.data_ptr(), 3, n, out[0].data_ptr(), out[1].data_ptr(), out[4].data_ptr(),
                                       out[2].data_ptr(), out[3].data_ptr(), st))
            check(lib.b200_cache_move(c.data_ptr(), None, 2, c.stride(0) * 2, 3, 2, B, 128, out[2].data_ptr(), out[3].data_ptr(), f.data_ptr(), 3, 20, st))
        runs.append((graph, stream, dev, out, [cache]))
    for _ in range(4):
        for graph, stream, dev, out, cache in runs:
            dev[0].copy_(torch.randint(0, 2, (n,), generator=g).to(I32))
        torch.cuda.synchronize()
        for graph, stream, *_ in runs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for graph, stream, dev, out, cache in runs:
            want = U.accept(dev[0].cpu(), dev[1].cpu(), parents, starts, slots)
            assert all(torch.equal(out[i].cpu().long(), y) for i, y in zip((0, 1, 4, 2, 3), want))
            cache[0] = U.moved(cache[0], want[3], want[4], starts, 20)
            assert torch.equal(dev[5].cpu(), cache[0])


def test_moves_outside_the_cache_and_behind_the_bound_are_not_made():
    g = torch.Generator().manual_seed(4)
    a = torch.randint(0, 99, (1, 10, 2, 16, 64), generator=g).to(BF)
    src = torch.tensor([3, -1, 160, 5, 2 ** 31 - 1, 9, 20, 21], dtype=I32)
    dst = torch.tensor([100, 101, 102, -2, 103, 160, 104, 105], dtype=I32)
    starts = _starts(8)
    for most in (8, 7, 1, 0):
        da, ds, dd, st = _dev(a, src, dst, starts)
        move(da, None, ds, dd, st, most)
        assert torch.equal(da.cpu(), U.moved(a, src, dst, starts, most))


# ---- together ----------------------------------------------------------------------------------------------------------------------

def test_a_drafted_tree_from_attention_to_the_cache():
    """Trees are attended, checked, and what is kept moves to the front: the next step's contexts hold the way that was kept."""
    g = torch.Generator().manual_seed(31)
    heads, hkv, block, V = 8, 2, 32, 1000
    shapes = [(100, _random_tree(20, g, 5)), (37, _random_tree(9, g, 3)), (64, [-1])]
    step = Step([(c, U.lines(p)) for c, p in shapes], heads, hkv, block, 31)
    out = step.run()
    step.check(out)
    starts = _starts(*[len(p) for _, p in shapes])
    proj = (torch.randn(heads * 128, V, generator=g) / 30).to(DEV)
    logits = (out.float() @ proj).to(BF).contiguous()
    lib, check = _lib()
    target = torch.empty(step.T, dtype=I32, device=DEV)
    check(lib.b200_argmax(logits.data_ptr(), V, step.T, V, 0, target.data_ptr(), None, None))
    parents = torch.tensor([p for _, ps in shapes for p in ps], dtype=I32)
    first = starts[step.seq.long()]
    drafts = target.cpu()[(first + parents.clamp(min=0)).long()].clone()
    drafts[torch.rand(step.T, generator=g) < 0.3] = 5
    slots = torch.tensor([int(b) * block + o for t in range(step.T) for b, o in [step.cache.token(int(step.seq[t]), int(step.ctx[t]) + t - int(first[t]))]], dtype=I32)
    got = accept(target.cpu(), drafts, parents, starts, slots)
    want = U.accept(target.cpu(), drafts, parents, starts, slots)
    assert all(torch.equal(x.cpu().long(), y) for x, y in zip(got, want)) and int(want[2].sum()) > 1
    k, v = (c.to(DEV)[None].contiguous() for c in (step.cache.k, step.cache.v))
    move(k, v, got[3], got[4], starts.to(DEV), 20)
    before = [step.cache.rows(s, c + len(p)) for s, (c, p) in enumerate(shapes)]
    step.cache.k, step.cache.v = k[0].cpu(), v[0].cpu()
    for s, (c, p) in enumerate(shapes):
        kept = int(want[2][s]) + 1
        at = [c + int(r) - int(starts[s]) for r in want[1][int(starts[s]):int(starts[s]) + kept]]
        for new, old in zip(step.cache.rows(s, c + kept), before[s]):
            assert torch.equal(new[:c], old[:c]) and torch.equal(new[c:], old[at])
    nxt = Step([(c + int(k_) + 1, [[]]) for (c, _), k_ in zip(shapes, want[2])], heads, hkv, block, 32, words=0)
    nxt.cache = step.cache
    nxt.check(nxt.run())


def test_a_beam_search_over_states():
    """Select, then the states follow their beams, three times over; against the same search in plain torch."""
    g = torch.Generator().manual_seed(33)
    S, W, V, size = 3, 4, 5000, 1024
    states = torch.randn(1, S * W, 1, 1, size, generator=g)
    proj = torch.randn(size, V, generator=g) / 16
    scores = torch.zeros(S * W)
    starts = _starts(*[W] * S)
    dev, d_proj, d_scores, d_starts = _dev(states, proj, scores, starts)
    for _ in range(3):
        logits = (dev[0, :, 0, 0] @ d_proj).to(BF).contiguous()
        rows, tokens, out = select(logits, d_scores, d_starts, W)
        want = U.select(logits.cpu(), scores, starts, W)
        assert torch.equal(rows.cpu().long(), want[0]) and torch.equal(tokens.cpu().long(), want[1])
        src, dst = rows.flatten(), torch.arange(S * W, dtype=I32, device=DEV)
        move(dev, None, src, dst, d_starts, W)
        states = U.moved(states, src.cpu(), dst.cpu(), starts, W)
        assert torch.equal(dev.cpu(), states)
        d_scores, scores = out.flatten(), out.flatten().cpu()


def test_captured_passes_over_the_cases_keep_their_workspaces():
    """A pass that a graph has captured writes to memory that is its own, whatever passes over larger cases come behind it."""
    spec = importlib.util.spec_from_file_location("more_operators", os.path.join(os.path.dirname(__file__), "..", "perf", "more_operators.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m.own = True
    cases = [{"kind": "tree", "seqs": 1, "nodes": 4, "even": True, "ctx": 300, "heads": 8, "kv": 2, "block": 16},
             {"kind": "select", "seqs": 2, "rows": 3, "even": True, "vocab": 5000, "take": 4}]
    states = [m.prepare(c, 1) for c in cases]
    want = [[t.clone() for t in (r if isinstance(r, tuple) else (r,))] for r in map(m.run, states)]
    graphs = []
    for st in states:
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=torch.cuda.Stream()):
            m.run(st)
    for c in ({"kind": "tree", "seqs": 8, "nodes": 64, "even": True, "ctx": 600, "heads": 32, "kv": 8, "block": 128}, {"kind": "select", "seqs": 20, "rows": 8, "even": True, "vocab": 128256, "take": 16}):
        m.run(m.prepare(c, 2))
    held = [torch.full((n,), 7, dtype=torch.uint8, device=DEV) for n in (1 << 10, 1 << 14, 1 << 18, 1 << 20, 3 << 20, 9 << 20, 30 << 20, 50 << 20) for _ in range(4)]
    for st, graph, outs in zip(states, graphs, want):
        for t in (st.out, *(st[k] for k in ("rows", "tokens") if k in st)):
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = (st.rows, st.tokens, st.out) if "rows" in st else (st.out,)
        assert all(torch.equal(a, b) for a, b in zip(got, outs))
    assert all((t == 7).all() for t in held)
