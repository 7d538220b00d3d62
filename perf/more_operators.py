"""The operators of decoding along several continuations of a sequence, as cases that can be timed and compared: attention of rows that see a cached prefix
and, by a mask of their own, some of the tokens behind it (trees of drafted tokens, beams over a shared prompt); a beam search's selection over beams and
vocabulary; the walk through a checked tree; and the cached rows or states that follow a selection to their new places.

listed() names the cases, draw() gives others of the same ranges, prepare() makes inputs, run() is one pass (own: through the C ABI; else in elementary torch
operations), exact() the same result in 64 bits."""
import importlib
import math
import random

import torch

own = False
BF16, F32, F64, I32, I64 = torch.bfloat16, torch.float32, torch.float64, torch.int32, torch.int64
DIM = 128
_kept = {}   # the library that a program keeps


def listed():
    return [
        # one sequence with a small tree of drafts behind a short prompt (latency)
        {"name": "tree_1x8", "kind": "tree", "seqs": 1, "nodes": 8, "even": True, "ctx": 600, "heads": 32, "kv": 8, "block": 128},
        # one sequence with a tree of 64 nodes behind a long context
        {"name": "tree_1x64_32k", "kind": "tree", "seqs": 1, "nodes": 64, "even": True, "ctx": 32000, "heads": 32, "kv": 8, "block": 128},
        # 32 running sequences with trees of different sizes, contexts of different lengths
        {"name": "tree_32x25", "kind": "tree", "seqs": 32, "nodes": 25, "even": False, "ctx": 4000, "heads": 32, "kv": 8, "block": 128},
        # large trees, five query heads to a kv head
        {"name": "tree_4x256", "kind": "tree", "seqs": 4, "nodes": 256, "even": True, "ctx": 6000, "heads": 40, "kv": 8, "block": 64},
        # a beam search of 16 requests, six beams each, 57 tokens behind their prompts; small blocks
        {"name": "beams_16x6", "kind": "beams", "seqs": 16, "nodes": 6, "steps": 57, "ctx": 2500, "heads": 64, "kv": 8, "block": 16},
        # one request, four beams, twice as many candidates
        {"name": "select_1x4", "kind": "select", "seqs": 1, "rows": 4, "even": True, "vocab": 128256, "take": 8},
        # a level of the drafted trees of 32 sequences: different widths, ten new nodes each
        {"name": "select_32x5", "kind": "select", "seqs": 32, "rows": 5, "even": False, "vocab": 32000, "take": 10},
        # 64 requests, eight beams each
        {"name": "select_64x8", "kind": "select", "seqs": 64, "rows": 8, "even": True, "vocab": 128256, "take": 16},
        # one small tree, checked
        {"name": "accept_1x8", "kind": "accept", "seqs": 1, "nodes": 8, "even": True},
        # 64 trees of up to 100 nodes
        {"name": "accept_64x50", "kind": "accept", "seqs": 64, "nodes": 50, "even": False},
        # the accepted rows of 48 trees in all layers' caches move to the end of their contexts
        {"name": "move_rows_48x32", "kind": "move_rows", "seqs": 48, "nodes": 32, "even": False, "layers": 32, "kv": 4, "block": 32},
        # recurrent states of 16 requests follow the selection among eight beams
        {"name": "move_states_16x8", "kind": "move_states", "seqs": 16, "nodes": 8, "values": 524288},
    ]


HEADS = [(4, 1), (8, 1), (32, 8), (40, 8), (64, 8), (8, 8), (16, 8), (28, 4), (32, 2)]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "tree", "beams", "select", "select", "accept", "move_rows", "move_states"])
    if kind in ("tree", "beams"):
        heads, kv = rng.choice(HEADS)
        seqs, case = _log(rng, 1, 64), {"kind": kind, "heads": heads, "kv": kv, "block": rng.choice([16, 32, 64, 128, 128, 256])}
        if kind == "beams":
            case.update(seqs=seqs, nodes=rng.randint(1, 12), steps=rng.randint(0, 80))
        else:
            case.update(seqs=seqs, nodes=_log(rng, 1, 256 if seqs <= 4 else 64), even=rng.random() < 0.5)
        case["ctx"] = rng.choice([0, _log(rng, 1, max(1, min(32000, 250000 // (seqs * kv), 200000000 // (seqs * case["nodes"] * heads))))])
        return case
    if kind == "select":
        seqs, rows = _log(rng, 1, 64), _log(rng, 1, 8)
        return {"kind": kind, "seqs": seqs, "rows": rows, "even": rng.random() < 0.5, "vocab": rng.choice([1024, 4096, 32000, 128256, 128256, _log(rng, 300, 128256)]),
                "take": rng.choice([1, 2 * rows, rng.randint(1, 64)])}
    if kind == "accept":
        return {"kind": kind, "seqs": _log(rng, 1, 64), "nodes": _log(rng, 1, 256), "even": rng.random() < 0.5}
    if kind == "move_rows":
        return {"kind": kind, "seqs": _log(rng, 1, 48), "nodes": _log(rng, 2, 64), "even": rng.random() < 0.5, "layers": rng.randint(1, 32), "kv": rng.choice([1, 2, 4]),
                "block": rng.choice([16, 32, 64])}
    seqs, beams = _log(rng, 1, 32), rng.randint(2, 8)
    return {"kind": kind, "seqs": seqs, "nodes": beams, "values": 4 * _log(rng, 64, min(131072, 16000000 // (seqs * beams)))}


# ---- shapes, from the case alone -----------------------------------------------------------------------------------------------

def _dice(case):
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _sizes(case, r):
    """Rows of each sequence: all alike, or between half and one and a half times as many."""
    n = case.get("rows") or case["nodes"]
    return [n if case.get("even", True) else r.randint(max(1, n // 2), n + n // 2) for _ in range(case["seqs"])]


def _tree(n, r):
    """Parents of n nodes, level by level, a node's before itself (the first one's: -1)."""
    width, levels, parents = max(1, round(n / 6)), [[0]], [-1]
    while len(parents) < n:
        level = range(len(parents), min(n, len(parents) + width))
        parents += [r.choice(levels[-1][:max(1, len(levels[-1]) // 2)]) for _ in level]
        levels.append(list(level))
    return parents


def _lines(parents):
    """The nodes on the way to each node, itself among them."""
    out = []
    for i, p in enumerate(parents):
        out.append((out[p] if p >= 0 else []) + [i])
    return out


def _attention_shape(case):
    """Of each sequence the tokens before its tail, the tail's length, and for each row the tail's tokens that it sees."""
    r, out = _dice(case), []
    for n in _sizes(case, r):
        ctx = case["ctx"] if case["seqs"] == 1 else r.randint(case["ctx"] // 2, case["ctx"])
        if case["kind"] == "tree":
            out.append((ctx, n, _lines(_tree(n, r))))
            continue
        seen = [[b] for b in range(n)]   # beams: the token of step s and beam b is token s * n + b of the tail
        for step in range(1, case["steps"] + 1):
            seen = [seen[r.randrange(n)] + [step * n + b] for b in range(n)]
        out.append((ctx, n * (case["steps"] + 1), seen))
    return out


def _moves(case):
    """Pairs (from, to) of each sequence, by place within it."""
    r = _dice(case)
    if case["kind"] == "move_states":
        picks = [[r.randrange(case["nodes"]) for _ in range(case["nodes"])] for _ in range(case["seqs"])]
        return [case["nodes"]] * case["seqs"], [[(p, i) for i, p in enumerate(ps) if p != i] for ps in picks]
    sizes = _sizes(case, r)
    lines = [r.choice(_lines(_tree(n, r))) for n in sizes]
    return sizes, [[(p, i) for i, p in enumerate(line) if p != i] for line in lines]


class State(dict):
    __getattr__ = dict.__getitem__


def _starts(sizes):
    return torch.tensor([0] + sizes, device="cuda").cumsum(0).to(I32)


def _by_row(st, sizes):
    """Each row's sequence and its place there."""
    st["starts"], st["most"] = _starts(sizes), max(sizes)
    st["seq"] = torch.repeat_interleave(torch.arange(len(sizes), device="cuda"), torch.tensor(sizes, device="cuda"))
    st["place"] = torch.arange(sum(sizes), device="cuda") - st.starts.long()[st.seq]


def _masks(lines, words):
    m = torch.zeros(len(lines), words, dtype=I64)
    rows = torch.tensor([i for i, line in enumerate(lines) for _ in line])
    bits = torch.tensor([j for line in lines for j in line])
    m.view(-1).index_add_(0, rows * words + bits // 32, torch.ones(len(bits), dtype=I64) << (bits % 32))
    return torch.where(m >= 2 ** 31, m - 2 ** 32, m).to(I32).cuda()


def _prepare_attention(st, case, g):
    shape = _attention_shape(case)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")   # noqa: E731
    B, hq, hkv = case["block"], case["heads"], case["kv"]
    _by_row(st, [len(lines) for _, _, lines in shape])
    need = [(ctx + tail + B - 1) // B for ctx, tail, _ in shape]
    st["n_blocks"] = sum(need) + 2
    order = torch.randperm(st.n_blocks, generator=g, device="cuda").to(I32)
    used = torch.arange(max(need), device="cuda")[None] < torch.tensor(need, device="cuda")[:, None]
    st["bt"] = torch.zeros(len(shape), max(need), dtype=I32, device="cuda")
    st.bt[used] = order[:sum(need)]
    st["longest"] = max(ctx + tail for ctx, tail, _ in shape)
    st["ctx"] = torch.tensor([ctx for ctx, _, _ in shape], device="cuda")[st.seq].to(I32)
    st["words"] = (max(tail for _, tail, _ in shape) + 31) // 32
    st["masks"] = _masks([line for _, _, lines in shape for line in lines], st.words)
    st["row_seq"] = st.seq.to(I32)
    spread = torch.exp2(rn(hkv, 1, DIM) * 0.7)   # some channels of keys are larger than others, some tokens' values too
    st["k"] = (rn(st.n_blocks, hkv, B, DIM) * spread).to(BF16)
    st["v"] = (rn(st.n_blocks, hkv, B, DIM) * torch.exp2(rn(st.n_blocks, hkv, B, 1))).to(BF16)
    T = len(st.seq)
    st["q"] = (rn(T, hq * DIM) * 1.5).to(BF16)
    st["out"] = torch.empty(T, hq * DIM, dtype=BF16, device="cuda")
    st["scale"] = DIM ** -0.5


def _prepare_select(st, case, g):
    sizes = _sizes(case, _dice(case))
    _by_row(st, sizes)
    n, V = sum(sizes), case["vocab"]
    # the continuations of one request look alike; their sums of log-probabilities are a few units apart
    like = torch.randn(case["seqs"], V, generator=g, device="cuda") * 2.5
    st["logits"] = (like[st.seq] + torch.randn(n, V, generator=g, device="cuda")).to(BF16)
    st["scores"] = -6 - 5 * torch.rand(n, generator=g, device="cuda")
    st["rows"], st["tokens"] = (torch.empty(case["seqs"], case["take"], dtype=I32, device="cuda") for _ in range(2))
    st["out"] = torch.empty(case["seqs"], case["take"], dtype=F32, device="cuda")


def _prepare_accept(st, case, g):
    r = _dice(case)
    trees = [_tree(n, r) for n in _sizes(case, r)]
    _by_row(st, [len(t) for t in trees])
    n = len(st.seq)
    st["parents"] = torch.tensor([p for t in trees for p in t], dtype=I32, device="cuda")
    st["words"] = (st.most + 31) // 32
    st["masks"] = _masks([line for t in trees for line in _lines(t)], st.words)   # (the attention's)
    st["drafts"] = torch.randint(0, 6, (n,), generator=g, device="cuda").to(I32) * 7001   # (siblings may be alike)
    # the target agrees with a child of a node about three times in four
    parent = (st.starts.long()[st.seq] + st.parents.clamp(min=0)).long()
    child = torch.zeros(n, dtype=I64, device="cuda").scatter_reduce_(0, parent, torch.arange(n, device="cuda"), "amax")
    agrees = (torch.rand(n, generator=g, device="cuda") < 0.75) & (child > 0)
    st["target"] = torch.where(agrees, st.drafts[child], 5 + torch.randint(0, 128000, (n,), generator=g, device="cuda").to(I32))
    st["slots"] = torch.randperm(4 * n, generator=g, device="cuda")[:n].to(I32)
    st["out"], st["path"], st["src"], st["dst"] = (torch.empty(n, dtype=I32, device="cuda") for _ in range(4))
    st["accepted"] = torch.empty(case["seqs"], dtype=I32, device="cuda")


def _prepare_move(st, case, g):
    sizes, moves = _moves(case)
    _by_row(st, sizes)
    n = len(st.seq)
    # a place for each row: the new end of a context in blocks anywhere, or a state's slot anywhere
    if case["kind"] == "move_states":
        st["units"] = n + 3
        st["slots"] = torch.randperm(st.units, generator=g, device="cuda")[:n]
        st["a"], st["b"] = torch.randn(st.units, case["values"], generator=g, device="cuda"), None
    else:
        B = case["block"]
        first = torch.randint(0, B, (case["seqs"],), generator=g, device="cuda")
        each = (B + max(sizes) - 1) // B + 1
        st["units"] = case["seqs"] * each + 1
        blocks = torch.randperm(st.units, generator=g, device="cuda")[:case["seqs"] * each].view(-1, each)
        at = first[st.seq] + st.place
        st["slots"] = blocks[st.seq, at // B] * B + at % B
        st["a"], st["b"] = (torch.randn(case["layers"], st.units, case["kv"], B, DIM, generator=g, device="cuda").to(BF16) for _ in range(2))
    # a sequence's moves are its first entries, behind them none
    at = [(f + k, f + a, f + b) for f, m in zip(st.starts.tolist(), moves) for k, (a, b) in enumerate(m)]
    at = torch.tensor(at, dtype=I64, device="cuda").reshape(-1, 3)
    st["src"], st["dst"] = (torch.full((n,), -1, dtype=I32, device="cuda") for _ in range(2))
    st.src[at[:, 0]] = st.slots[at[:, 1]].to(I32)
    st.dst[at[:, 0]] = st.slots[at[:, 2]].to(I32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    st = State(case=case)
    kind = case["kind"]
    (_prepare_attention if kind in ("tree", "beams") else _prepare_select if kind == "select" else _prepare_accept if kind == "accept" else _prepare_move)(st, case, g)
    return st


# ---- the plain forms -----------------------------------------------------------------------------------------------------------

def _bits(masks, n):
    j = torch.arange(n, device="cuda")
    return (masks[:, j // 32] >> (j % 32)) & 1 > 0


def _plain_attention(st):
    case = st.case
    hq, hkv, n_keys, most = case["heads"], case["kv"], st.longest, st.most
    S, G, T = st.bt.shape[0], hq // hkv, len(st.seq)
    k, v = (c[st.bt.long()].transpose(1, 2).reshape(S, hkv, -1, DIM)[:, :, :n_keys].float() for c in (st.k, st.v))
    # what each row sees, by sequence and place
    tail = torch.arange(n_keys, device="cuda")[None] - st.ctx[:, None]
    bits = _bits(st.masks, st.words * 32).gather(1, tail.clamp(0, st.words * 32 - 1).long())
    seen = torch.zeros(S, most, n_keys, dtype=torch.bool, device="cuda")
    seen[st.seq, st.place] = (tail < 0) | (bits & (tail < st.words * 32))
    q = torch.zeros(S, most, hq, DIM, device="cuda")
    q[st.seq, st.place] = st.q.view(T, hq, DIM).float()
    q = q.view(S, most, hkv, G, DIM).permute(0, 2, 3, 1, 4).reshape(S, hkv, -1, DIM)
    s = (q @ k.transpose(2, 3) * st.scale).view(S, hkv, G, most, n_keys)
    s = s.masked_fill(~seen[:, None, None], float("-inf"))
    p = (s - s.amax(-1, keepdim=True).clamp(min=-1e30)).exp()
    o = (p.view(S, hkv, -1, n_keys) @ v).view(S, hkv, G, most, DIM) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    st.out.copy_(o.permute(0, 3, 1, 2, 4)[st.seq, st.place].reshape(T, -1).to(BF16))
    return st.out


def _plain_select(st):
    # in 64 bits: candidates next to one another
    S, V, K = st.case["seqs"], st.case["vocab"], st.case["take"]
    x = st.logits.double()
    x = x - x.amax(1, keepdim=True)
    x = st.scores.double()[:, None] + (x - x.exp().sum(1, keepdim=True).log())
    if st.most * S == len(st.seq):
        x = x.view(S, -1)
    else:
        full = torch.full((S, st.most, V), float("-inf"), dtype=F64, device="cuda")
        full[st.seq, st.place] = x
        x = full.view(S, -1)
    least = x.topk(min(K, x.shape[1]), 1).values[:, -1:]
    seq, at = torch.nonzero((x >= least) & (x > float("-inf")), as_tuple=True)   # in order of places
    value = x[seq, at]
    order = torch.sort(value, descending=True, stable=True).indices
    order = order[torch.sort(seq[order], stable=True).indices]
    seq, at, value = seq[order], at[order], value[order]
    rank = torch.arange(len(seq), device="cuda") - torch.searchsorted(seq, seq)
    keep = rank < K
    seq, at, value, rank = seq[keep], at[keep], value[keep], rank[keep]
    st.rows.fill_(-1)
    st.tokens.fill_(-1)
    st.out.fill_(float("-inf"))
    st.rows[seq, rank] = (st.starts[seq] + at // V).to(I32)
    st.tokens[seq, rank] = (at % V).to(I32)
    st.out[seq, rank] = value.float()
    return st.rows, st.tokens, st.out


def _plain_accept(st):
    S, n, most = st.case["seqs"], len(st.seq), st.most
    parent = st.starts[st.seq] + st.parents.clamp(min=0)
    good = (st.drafts == st.target[parent]) | (st.place == 0)
    pad = torch.full((S, most), -2, dtype=I64, device="cuda")
    pad[st.seq, st.place] = st.parents.long()
    token = torch.zeros(S, most, dtype=I32, device="cuda")
    token[st.seq, st.place] = st.drafts
    # of siblings that are alike the first counts
    alike = (pad[:, :, None] == pad[:, None, :]) & (token[:, :, None] == token[:, None, :])
    first = ~alike.tril(-1).any(2)
    good &= first[st.seq, st.place]
    bad = torch.zeros(S, most, device="cuda")
    bad[st.seq, st.place] = (~good).float()
    above = _bits(st.masks, most)   # the nodes on the way to each row
    taken = ((above * bad[st.seq]).sum(1) == 0)
    count = torch.zeros(S, dtype=I64, device="cuda").scatter_add_(0, st.seq, taken.long())
    on = torch.zeros(S, most, dtype=I64, device="cuda")
    on[st.seq, st.place] = taken.long()
    depth = (on.cumsum(1) - 1)[st.seq, st.place]
    row = torch.nonzero(taken)[:, 0]
    to = (st.starts[st.seq[row]] + depth[row]).long()
    st.path.fill_(-1)
    st.path[to] = row.to(I32)
    st.out.fill_(-1)
    st.out[to] = st.target[row]   # (a kept draft is what its parent's target says)
    moved = row != to
    st.src.fill_(-1)
    st.dst.fill_(-1)
    st.src[to] = torch.where(moved, st.slots[row], -1)
    st.dst[to] = torch.where(moved, st.slots[to], -1)
    st.accepted.copy_(count - 1)
    return st.out, st.path, st.accepted, st.src, st.dst


def _plain_move(st):
    real = st.src >= 0
    src, dst = st.src[real].long(), st.dst[real].long()
    if st.case["kind"] == "move_states":
        st.a[dst] = st.a[src]
        return st.a
    B = st.case["block"]
    st.a[:, dst // B, :, dst % B] = st.a[:, src // B, :, src % B]
    st.b[:, dst // B, :, dst % B] = st.b[:, src // B, :, src % B]
    return st.a, st.b


# ---- the framework's operators -------------------------------------------------------------------------------------------------

def _library():
    if "lib" not in _kept:
        abi = importlib.import_module("enterprise-inference_b200._abi")
        _kept.update(lib=abi.lib(), check=abi.check, ptr=abi.ptr)
    return _kept["lib"], _kept["check"], _kept["ptr"]


def _workspace(st, stream, size):
    """One for each state and stream: passes that may run at the same time do not share one, and one that a captured pass writes to is there as long as its state."""
    kept = st.setdefault("workspaces", {})
    if stream not in kept:
        kept[stream] = torch.empty(size, dtype=torch.uint8, device="cuda")
    return kept[stream].data_ptr(), size


def _own(st):
    lib, check, ptr = _library()
    case, stream, n = st.case, torch.cuda.current_stream().cuda_stream, len(st.seq)
    kind = case["kind"]
    if kind in ("tree", "beams"):
        hq, hkv = case["heads"], case["kv"]
        ws = _workspace(st, stream, lib.b200_paged_attn_tree_workspace_bytes(n, hq, hkv))
        check(lib.b200_paged_attn_tree(ptr(st.q), hq * DIM, ptr(st.k), ptr(st.v), st.n_blocks, ptr(st.bt), st.bt.shape[1], ptr(st.row_seq), ptr(st.ctx), ptr(st.masks),
                                       st.words, ptr(st.out), hq * DIM, n, hq, hkv, case["block"], st.scale, *ws, stream))
        return st.out
    if kind == "select":
        ws = _workspace(st, stream, lib.b200_beam_select_workspace_bytes(n, case["vocab"], case["take"]))
        check(lib.b200_beam_select(ptr(st.logits), case["vocab"], ptr(st.scores), ptr(st.starts), case["seqs"], n, case["vocab"], case["take"], ptr(st.rows),
                                   ptr(st.tokens), ptr(st.out), *ws, stream))
        return st.rows, st.tokens, st.out
    if kind == "accept":
        check(lib.b200_accept_tree(ptr(st.target), ptr(st.drafts), ptr(st.parents), ptr(st.starts), ptr(st.slots), case["seqs"], n, ptr(st.out), ptr(st.path),
                                   ptr(st.accepted), ptr(st.src), ptr(st.dst), stream))
        return st.out, st.path, st.accepted, st.src, st.dst
    if kind == "move_states":
        size = 4 * case["values"]
        check(lib.b200_cache_move(ptr(st.a), None, 1, 0, st.units, 1, 1, size, ptr(st.src), ptr(st.dst), ptr(st.starts), case["seqs"], st.most, stream))
        return st.a
    check(lib.b200_cache_move(ptr(st.a), ptr(st.b), case["layers"], st.a.stride(0) * 2, st.units, case["kv"], case["block"], 2 * DIM, ptr(st.src), ptr(st.dst),
                              ptr(st.starts), case["seqs"], st.most, stream))
    return st.a, st.b


def run(state):
    if own:
        return _own(state)
    kind = state.case["kind"]
    if kind in ("tree", "beams"):
        return _plain_attention(state)
    return _plain_select(state) if kind == "select" else _plain_accept(state) if kind == "accept" else _plain_move(state)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind in ("tree", "beams"):
        shape = _attention_shape(case)
        rows = sum(len(lines) for _, _, lines in shape)
        seen = sum(ctx * len(lines) + sum(len(line) for line in lines) for ctx, _, lines in shape)
        words = (max(tail for _, tail, _ in shape) + 31) // 32
        keys = sum(ctx + len({j for line in lines for j in line}) for ctx, _, lines in shape)
        return {"bytes": keys * case["kv"] * 4 * DIM + 4 * rows * case["heads"] * DIM + rows * (8 + 4 * words), "flops": 4 * DIM * case["heads"] * seen}
    if kind == "select":
        n = sum(_sizes(case, _dice(case)))
        return {"bytes": 2 * n * case["vocab"] + 4 * n + 12 * case["seqs"] * case["take"], "flops": 4 * n * case["vocab"]}
    if kind == "accept":
        n = sum(_sizes(case, _dice(case)))
        return {"bytes": 32 * n + 8 * case["seqs"], "flops": 4 * n}
    _, moves = _moves(case)
    each = 4 * case["values"] if kind == "move_states" else 2 * case["layers"] * case["kv"] * 2 * DIM
    return {"bytes": each * sum(len({a for a, _ in m}) + len(m) for m in moves) + 8 * case["seqs"] * case["nodes"], "flops": 0}


# ---- the definitions, in 64 bits -----------------------------------------------------------------------------------------------

def _exact_attention(st):
    case = st.case
    hq, hkv = case["heads"], case["kv"]
    G, out, row = hq // hkv, torch.zeros(len(st.seq), hq, DIM, dtype=F64, device="cuda"), 0
    for s, (ctx, tail, lines) in enumerate(_attention_shape(case)):
        seen = torch.zeros(len(lines), ctx + tail, dtype=torch.bool)
        seen[:, :ctx] = True
        for i, line in enumerate(lines):
            seen[i, [ctx + j for j in line]] = True
        pages, n = st.bt[s, :(ctx + tail + case["block"] - 1) // case["block"]].long(), len(lines)
        for h in range(hkv):
            k, v = (c[pages, h].double().reshape(-1, DIM)[:ctx + tail] for c in (st.k, st.v))
            z = torch.einsum("rgd,td->rgt", st.q[row:row + n].view(n, hq, DIM)[:, h * G:(h + 1) * G].double(), k) * st.scale
            z = z.masked_fill(~seen.cuda()[:, None], float("-inf"))
            out[row:row + n, h * G:(h + 1) * G] = torch.einsum("rgt,td->rgd", torch.softmax(z, -1), v)
        row += n
    return out.reshape(len(st.seq), -1)


def _exact_select(st):
    case = st.case
    S, V, K = case["seqs"], case["vocab"], case["take"]
    rows, tokens = (torch.full((S, K), -1, dtype=I64) for _ in range(2))
    out = torch.full((S, K), float("-inf"), dtype=F64)
    for s in range(S):
        a, b = int(st.starts[s]), int(st.starts[s + 1])
        z = st.logits[a:b].double()
        z = (z - torch.logsumexp(z, 1, keepdim=True) + st.scores[a:b].double()[:, None]).reshape(-1)
        value, at = torch.sort(z, descending=True, stable=True)
        k = min(K, len(at))
        rows[s, :k], tokens[s, :k], out[s, :k] = (a + at[:k] // V).cpu(), (at[:k] % V).cpu(), value[:k].cpu()
    return rows, tokens, out


def _exact_accept(st):
    """A sequence at a time, from its root down."""
    target, drafts, parents, slots, starts = (x.tolist() for x in (st.target, st.drafts, st.parents, st.slots, st.starts))
    n = len(target)
    out, path, src, dst = ([-1] * n for _ in range(4))
    accepted = []
    for a, b in zip(starts, starts[1:]):
        line = [a]
        while True:
            nxt = [r for r in range(a + 1, b) if a + parents[r] == line[-1] and drafts[r] == target[line[-1]]]
            if not nxt:
                break
            line.append(nxt[0])
        for i, r in enumerate(line):
            out[a + i], path[a + i] = target[r], r
            if r != a + i:
                src[a + i], dst[a + i] = slots[r], slots[a + i]
        accepted.append(len(line) - 1)
    return tuple(torch.tensor(x) for x in (out, path, accepted, src, dst))


def _exact_move(st):
    case = st.case
    pairs = [(a, b) for a, b in zip(st.src.tolist(), st.dst.tolist()) if a >= 0]
    if case["kind"] == "move_states":
        new = st.a.clone()
        for a, b in pairs:
            new[b] = st.a[a]
        return new
    B, caches = case["block"], []
    for old in (st.a, st.b):
        new = old.clone()
        for a, b in pairs:
            new[:, b // B, :, b % B] = old[:, a // B, :, a % B]
        caches.append(new.float())
    return tuple(caches)


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind in ("tree", "beams"):
        return _exact_attention(st)
    return _exact_select(st) if kind == "select" else _exact_accept(st) if kind == "accept" else _exact_move(st)
