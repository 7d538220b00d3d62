"""The operators of drafted decoding over an 8-bit cache, as cases that can be timed and compared: keys and values quantised as they are
appended to a paged cache, attention of single rows and of runs of rows over that cache, and the check of drafted tokens against the
target's probabilities.

The cache holds, per token and kv head, 128 e4m3 codes and one exponent byte: value = code * 2^(byte - 127).  listed() names the cases,
draw() gives others of the same ranges, prepare() makes inputs, run() is one pass (own: through the C ABI; else in elementary torch
operations), exact() the same result in 64 bits."""
import importlib
import math
import random

import torch

own = False
BF16, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
E4M3 = torch.float8_e4m3fn
DIM = 128
_kept = {}   # the library and the workspace that a program keeps


def listed():
    return [
        # one sequence of an 8B model decodes: its new key and value row of a layer (the smallest call)
        {"name": "append_1", "kind": "append", "rows": 1, "seqs": 1, "ctx": 600, "heads": 32, "kv": 8, "block": 128},
        # 64 sequences with four drafts each
        {"name": "append_320", "kind": "append", "rows": 320, "seqs": 64, "ctx": 1000, "heads": 32, "kv": 8, "block": 128},
        # a prefill chunk of a 70B model, not a multiple of anything
        {"name": "append_2047", "kind": "append", "rows": 2047, "seqs": 1, "ctx": 5000, "heads": 64, "kv": 8, "block": 128},
        # one sequence decodes
        {"name": "decode_1", "kind": "decode", "rows": 1, "ctx": 601, "heads": 32, "kv": 8, "block": 128},
        # 64 running sequences of different lengths
        {"name": "decode_64", "kind": "decode", "rows": 64, "ctx": 1000, "heads": 32, "kv": 8, "block": 128},
        # small blocks, five query heads to a kv head
        {"name": "decode_33_small_blocks", "kind": "decode", "rows": 33, "ctx": 5000, "heads": 40, "kv": 8, "block": 16},
        # long contexts of a 70B model
        {"name": "decode_8_32k", "kind": "decode", "rows": 8, "ctx": 32768, "heads": 64, "kv": 8, "block": 128},
        # 48 sequences with four drafts each
        {"name": "drafts_48x5", "kind": "prefill", "rows": 240, "seqs": 48, "ctx": 2500, "heads": 32, "kv": 8, "block": 128, "even": True},
        # chunks of three sequences behind long contexts
        {"name": "chunk_300", "kind": "prefill", "rows": 300, "seqs": 3, "ctx": 6000, "heads": 40, "kv": 8, "block": 128, "even": False},
        # a 2048-row prefill chunk behind 1000 cached tokens
        {"name": "chunk_2048", "kind": "prefill", "rows": 2048, "seqs": 1, "ctx": 1000, "heads": 32, "kv": 8, "block": 128, "even": False},
        # one sequence, four drafts of a drafter without probabilities
        {"name": "verify_1x5", "kind": "verify", "rows": 5, "seqs": 1, "vocab": 128256, "probs": False, "greedy": 0.0},
        # 64 sequences, four drafts each, the drafter's logits there, every eighth sequence greedy
        {"name": "verify_64x5", "kind": "verify", "rows": 320, "seqs": 64, "vocab": 128256, "probs": True, "greedy": 0.125},
    ]


HEADS = [(4, 1), (8, 1), (32, 8), (40, 8), (64, 8), (8, 8), (16, 8), (28, 4), (32, 2)]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["append", "decode", "prefill", "prefill", "verify"])
    heads, kv = rng.choice(HEADS)
    block = rng.choice([16, 32, 64, 128, 128, 256])
    if kind == "append":
        rows = _log(rng, 1, 2047)
        return {"kind": kind, "rows": rows, "seqs": rng.choice([1, rng.randint(1, min(rows, 64))]), "ctx": rng.choice([0, _log(rng, 1, 30000)]), "heads": heads,
                "kv": kv, "block": block}
    if kind == "decode":
        rows = _log(rng, 1, 200)
        return {"kind": kind, "rows": rows, "ctx": _log(rng, 1, min(32768, 1500000 // (rows * kv))), "heads": heads, "kv": kv, "block": block}
    if kind == "prefill":
        if rng.random() < 0.4:   # drafts: a few rows a sequence
            seqs, each = _log(rng, 1, 64), rng.randint(2, 9)
            return {"kind": kind, "rows": seqs * each, "seqs": seqs, "ctx": _log(rng, 1, min(16384, 900000 // (seqs * kv))), "heads": heads, "kv": kv,
                    "block": block, "even": True}
        rows = _log(rng, 2, 2048)
        return {"kind": kind, "rows": rows, "seqs": rng.randint(1, min(rows, 4)), "ctx": rng.choice([0, _log(rng, 1, max(1, min(8000, 2000000 // rows)))]),
                "heads": min(heads, 32), "kv": kv, "block": block, "even": False}
    seqs = _log(rng, 1, 64)
    return {"kind": kind, "rows": seqs * rng.randint(1, 5), "seqs": seqs, "vocab": rng.choice([1024, 4096, 16032, 128256, 128256, _log(rng, 300, 120000)]),
            "probs": rng.random() < 0.6, "greedy": rng.choice([0.0, 0.25, 1.0])}


# ---- shapes of a step ------------------------------------------------------------------------------------------------------

def _shape(case):
    """Rows of each sequence and the tokens cached before them, from the case alone."""
    r = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    rows, seqs = case["rows"], case.get("seqs", case["rows"])
    if case.get("even", True):
        parts = [rows // seqs + (i < rows % seqs) for i in range(seqs)]
    else:
        cuts = sorted(r.sample(range(1, rows), seqs - 1))
        parts = [b - a for a, b in zip([0] + cuts, cuts + [rows])]
    ctx, last = case.get("ctx", 0), case["kind"] == "decode"   # a decoding row is the last of its context
    before = [max((ctx if seqs == 1 else r.randint(ctx // 2, ctx)) - last, 0) for _ in parts]
    return parts, before


class State(dict):
    __getattr__ = dict.__getitem__


def _paged(case, g, st):
    """Block tables in random order, the arrays of one step by row and, for the plain form, by (sequence, place)."""
    parts, before = _shape(case)
    B, dev = case["block"], "cuda"
    behind = [b // B if case["kind"] == "append" else 0 for b in before]   # blocks that the pass has nothing to do with
    need = [(n + b + B - 1) // B - o for n, b, o in zip(parts, before, behind)]
    st["n_blocks"] = sum(need) + 2
    order = torch.randperm(st.n_blocks, generator=g, device=dev).to(I32)
    used = torch.arange(max(need), device=dev)[None, :] < torch.tensor(need, device=dev)[:, None]
    st["bt"] = torch.zeros(len(parts), max(need), dtype=I32, device=dev)
    st.bt[used] = order[:sum(need)]
    seq = torch.repeat_interleave(torch.arange(len(parts), device=dev), torch.tensor(parts, device=dev))
    first = torch.tensor([0] + parts, device=dev).cumsum(0)
    place = torch.arange(len(seq), device=dev) - first[seq]
    st["positions"] = (torch.tensor(before, device=dev)[seq] + place).to(I32)
    st["ctx"], st["seq"], st["place"] = st.positions + 1, seq.to(I32), place
    st["longest"], st["most"] = max(n + b for n, b in zip(parts, before)), max(parts)
    st["slots"] = (st.bt[seq, (st.positions // B).long() - torch.tensor(behind, device=dev)[seq]] * B + st.positions % B).to(I32)


def _quantise(x):
    """fp32 [..., 128] -> (e4m3 codes, exponent bytes): the smallest e >= -100 with amax <= 448 * 2^e."""
    m, ex = torch.frexp(x.abs().amax(-1))
    e = torch.where(m > 0, ex - torch.where(m <= 0.875, 9, 8), -100).clamp(min=-100)
    return torch.ldexp(x, -e[..., None]).to(E4M3), (e + 127).to(torch.uint8)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")   # noqa: E731
    st = State(case=case)
    if case["kind"] == "verify":
        parts = [case["rows"] // case["seqs"]] * case["seqs"]
        n, V = case["rows"], case["vocab"]
        st["starts"] = torch.tensor([0] + parts, device="cuda").cumsum(0).to(I32)
        st["target"] = (rn(n, V) * 2.5 + (rn(V) * 1.5)[None]).to(BF16)
        drafter = (st.target.float() + rn(n, V) * 0.5).to(BF16)
        temp = 0.5 + torch.rand(case["seqs"], generator=g, device="cuda")
        st["temperature"] = torch.where(torch.arange(case["seqs"], device="cuda") < round(case["greedy"] * case["seqs"]), 0.0, temp)
        row_t = st.temperature.repeat_interleave(n // case["seqs"])[:, None]
        noise = -torch.log(-torch.log(torch.rand(n, V, generator=g, device="cuda").clamp(1e-9, 1 - 1e-7)))
        st["tokens"] = (drafter.float() + noise * row_t).argmax(1).to(I32)
        st["drafter"] = drafter if case["probs"] else None
        st["uniforms"] = torch.rand(n, 2, generator=g, device="cuda")
        st["out"] = torch.empty(n, dtype=I32, device="cuda")
        st["accepted"] = torch.empty(case["seqs"], dtype=I32, device="cuda")
        return st
    _paged(case, g, st)
    T, hq, hkv, B = case["rows"], case["heads"], case["kv"], case["block"]
    cells = (st.n_blocks, hkv, B)
    spread = torch.exp2(rn(hkv, 1, DIM) * 0.7)   # some channels of keys are larger than others, some tokens' values too
    if case["kind"] == "append":
        st["k"], st["v"] = (torch.zeros(*cells, DIM, dtype=torch.uint8, device="cuda") for _ in range(2))
        st["ke"], st["ve"] = (torch.zeros(*cells, dtype=torch.uint8, device="cuda") for _ in range(2))
        qkv = rn(T, hq + 2 * hkv, DIM)
        qkv[:, hq:hq + hkv] *= spread[:, 0]
        qkv[:, hq + hkv:] *= torch.exp2(rn(T, hkv, 1))
        st["qkv"] = qkv.to(BF16).reshape(T, -1)
        inv = 500000.0 ** (-torch.arange(0, DIM, 2, device="cuda", dtype=F64) / DIM)
        ang = torch.arange(st.longest, device="cuda", dtype=F64)[:, None] * inv[None]
        st["cos_sin"] = torch.cat([ang.cos(), ang.sin()], 1).to(BF16)
        st["q"] = torch.empty(T, hq * DIM, dtype=BF16, device="cuda")
        return st
    k, st["ke"] = _quantise(rn(*cells, DIM) * spread)
    v, st["ve"] = _quantise(rn(*cells, DIM) * torch.exp2(rn(*cells, 1)))
    st["k"], st["v"] = k.view(torch.uint8), v.view(torch.uint8)
    st["q"] = (rn(T, hq * DIM) * 1.5).to(BF16)
    st["out"] = torch.empty(T, hq * DIM, dtype=BF16, device="cuda")
    st["scale"] = DIM ** -0.5
    return st


# ---- the plain forms -------------------------------------------------------------------------------------------------------

def _values(codes, exps):
    return torch.ldexp(codes.view(E4M3).float(), exps.to(I32)[..., None] - 127)


def _plain_append(st):
    case = st.case
    T, hq, hkv, B = case["rows"], case["heads"], case["kv"], case["block"]
    x = st.qkv.view(T, -1, DIM).float()
    cs = st.cos_sin[st.positions.long()].float()[:, None]
    c, s, a, b = cs[..., :64], cs[..., 64:], x[:, :hq + hkv, :64], x[:, :hq + hkv, 64:]
    turned = torch.cat([a * c - b * s, b * c + a * s], -1)
    st.q.copy_(turned[:, :hq].reshape(T, -1).to(BF16))
    codes, exps = _quantise(torch.cat([turned[:, hq:], x[:, hq + hkv:]], 1))
    blk, off = (st.slots // B).long(), (st.slots % B).long()
    for cache, e, rows in ((st.k, st.ke, slice(0, hkv)), (st.v, st.ve, slice(hkv, None))):
        cache[blk, :, off] = codes[:, rows].view(torch.uint8)
        e[blk, :, off] = exps[:, rows]
    return st.q, st.k.view(E4M3), st.v.view(E4M3), st.ke, st.ve


def _plain_attention(st):
    case = st.case
    T, hq, hkv, B = case["rows"], case["heads"], case["kv"], case["block"]
    S, n_keys = st.bt.shape[0], st.longest
    # keys and values of each sequence in order, in 32 bits
    k, v = (_values(c[st.bt.long()], e[st.bt.long()]).transpose(1, 2).reshape(S, hkv, -1, DIM)[:, :, :n_keys] for c, e in ((st.k, st.ke), (st.v, st.ve)))
    seq = st.seq.long()
    q = torch.zeros(S, st.most, hq, DIM, device="cuda")
    q[seq, st.place] = st.q.view(T, hq, DIM).float()
    ctx = torch.zeros(S, st.most, dtype=I32, device="cuda")
    ctx[seq, st.place] = st.ctx
    q = q.view(S, st.most, hkv, hq // hkv, DIM).permute(0, 2, 3, 1, 4).reshape(S, hkv, -1, DIM)
    s = (q @ k.transpose(2, 3) * st.scale).view(S, hkv, hq // hkv, st.most, n_keys)
    s = s.masked_fill(torch.arange(n_keys, device="cuda") >= ctx[:, None, None, :, None], float("-inf"))
    p = (s - s.amax(-1, keepdim=True).clamp(min=-1e30)).exp()
    o = (p.view(S, hkv, -1, n_keys) @ v).view(S, hkv, hq // hkv, st.most, DIM) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    st.out.copy_(o.permute(0, 3, 1, 2, 4)[seq, st.place].reshape(T, -1).to(BF16))
    return st.out


def _plain_verify(st):
    # in 64 bits: a draw next to a border of the sums, a draft next to its limit
    n, S, V = st.case["rows"], st.case["seqs"], st.case["vocab"]
    per = n // S
    seq = torch.arange(S, device="cuda").repeat_interleave(per)
    temp = st.temperature[seq].double()[:, None]
    greedy, at = temp[:, 0] <= 0, torch.arange(n, device="cuda")
    by = torch.where(temp > 0, temp, 1.0)

    def weights(logits, rows):
        x = logits[rows].float()
        return ((x - x.amax(-1, keepdim=True)).double() / by[rows]).exp()

    x = st.tokens.long()
    best = torch.where(st.target == st.target.amax(-1, keepdim=True), torch.arange(V, device="cuda"), V).amin(-1)
    e = weights(st.target, at)
    p = e[at, x] / e.sum(-1)
    if st.drafter is None:
        q = torch.ones_like(p)
    else:
        d = weights(st.drafter, at)
        q = d[at, x] / d.sum(-1)
    ok = torch.where(greedy, best == x, st.uniforms[:, 0].double() * q < p).view(S, per)
    ok[:, -1] = False   # the row behind the last draft has none
    taken = ok.long().cumprod(1).sum(1)
    row = torch.arange(S, device="cuda") * per + taken
    e = weights(st.target, row)
    p = e / e.sum(-1, keepdim=True)
    if st.drafter is None:
        left = p.clone()
        left[torch.arange(S, device="cuda"), x[row]] = 0
    else:
        d = weights(st.drafter, row)
        left = (p - d / d.sum(-1, keepdim=True)).clamp(min=0)
    w = torch.where(((taken == per - 1) | (left.sum(-1) == 0))[:, None], p, left)
    c = w.cumsum(-1)
    drawn = (c <= st.uniforms[row, 1].double()[:, None] * c[:, -1:]).sum(-1)
    drawn = torch.where(st.temperature <= 0, best[row], drawn)
    place = torch.arange(per, device="cuda")[None]
    out = torch.where(place < taken[:, None], x.view(S, per), torch.where(place == taken[:, None], drawn[:, None], -1))
    st.out.copy_(out.reshape(-1))
    st.accepted.copy_(taken)
    return st.out, st.accepted


# ---- the framework's operators ---------------------------------------------------------------------------------------------

def _library():
    if "lib" not in _kept:
        abi = importlib.import_module("enterprise-inference_b200._abi")
        _kept.update(lib=abi.lib(), check=abi.check, ptr=abi.ptr)
    return _kept["lib"], _kept["check"], _kept["ptr"]


def _workspace(size):
    if size > _kept.get("size", 0):
        _kept.update(ws=torch.zeros(size, dtype=torch.uint8, device="cuda"), size=size)
    return _kept["ws"].data_ptr(), _kept["size"]


def _own(st):
    lib, check, ptr = _library()
    case, stream = st.case, torch.cuda.current_stream().cuda_stream
    if case["kind"] == "verify":
        ws = _workspace(lib.b200_verify_drafts_workspace_bytes(case["rows"], case["vocab"]))
        check(lib.b200_verify_drafts(ptr(st.target), case["vocab"], ptr(st.drafter), case["vocab"], ptr(st.tokens), ptr(st.starts), ptr(st.temperature),
                                     ptr(st.uniforms), case["seqs"], case["rows"], case["vocab"], ptr(st.out), ptr(st.accepted), *ws, stream))
        return st.out, st.accepted
    T, hq, hkv, B = case["rows"], case["heads"], case["kv"], case["block"]
    cache = (ptr(st.k), ptr(st.v), ptr(st.ke), ptr(st.ve), st.n_blocks)
    if case["kind"] == "append":
        check(lib.b200_rope_kv_append_fp8(ptr(st.qkv), (hq + 2 * hkv) * DIM, ptr(st.positions), ptr(st.slots), ptr(st.cos_sin), ptr(st.q), hq * DIM, *cache,
                                          T, hq, hkv, B, stream))
        return st.q, st.k.view(E4M3), st.v.view(E4M3), st.ke, st.ve
    ws = _workspace(lib.b200_paged_attn_fp8_workspace_bytes(T, hq, hkv))
    lead = (ptr(st.q), hq * DIM, *cache, ptr(st.bt), st.bt.shape[1], ptr(st.seq), ptr(st.ctx), ptr(st.out), hq * DIM, T, hq, hkv, B)
    if case["kind"] == "decode":
        check(lib.b200_paged_attn_decode_fp8(*lead, st.scale, *ws, stream))
    else:
        check(lib.b200_paged_attn_prefill_fp8(*lead, st.most, st.scale, *ws, stream))
    return st.out


def run(state):
    if own:
        return _own(state)
    kind = state.case["kind"]
    return _plain_append(state) if kind == "append" else _plain_verify(state) if kind == "verify" else _plain_attention(state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------

def work(case):
    n = case["rows"]
    if case["kind"] == "verify":
        V, S = case["vocab"], case["seqs"]
        greedy = round(case["greedy"] * S)
        drafted = (n // S - 1) * (S - greedy) if case["probs"] else 0   # rows whose drafter's probabilities matter
        return {"bytes": 2 * V * (n + drafted) + 16 * n + 12 * S, "flops": 4 * V * (n + drafted)}
    hq, hkv = case["heads"], case["kv"]
    if case["kind"] == "append":
        return {"bytes": n * (2 * DIM * (hq + 2 * hkv) + 2 * DIM + 8 + 2 * DIM * hq + 2 * hkv * (DIM + 1)), "flops": n * DIM * (3 * (hq + hkv) + 4 * hkv)}
    parts, before = _shape(case)
    keys = sum(a + b for a, b in zip(parts, before))
    pairs = sum(b * a + a * (a + 1) // 2 for a, b in zip(parts, before))
    return {"bytes": keys * hkv * 2 * (DIM + 1) + 2 * n * hq * DIM * 2 + 8 * n, "flops": 4 * DIM * hq * pairs}


# ---- the definitions, in 64 bits -------------------------------------------------------------------------------------------

def _exact_append(st):
    """Row by row of the step, all heads at once; a code is the nearest of the 253 finite e4m3 values, ties to the even code."""
    case = st.case
    T, hq, hkv, B = case["rows"], case["heads"], case["kv"], case["block"]
    x = st.qkv.double().view(T, hq + 2 * hkv, DIM)
    table = st.cos_sin.double()[st.positions.long()]
    z = torch.complex(x[:, :hq + hkv, :64], x[:, :hq + hkv, 64:]) * torch.complex(table[:, :64], table[:, 64:])[:, None]
    rot = torch.cat([z.real, z.imag], -1)
    rows = torch.cat([rot[:, hq:], x[:, hq + hkv:]], 1)
    e = torch.ceil(torch.log2(rows.abs().amax(-1).clamp(min=2.0 ** -90) / 448) - 1e-9).clamp(min=-100)   # (448 * 2^k takes k)
    y = rows * torch.exp2(-e)[..., None]
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)   # distance of neighbouring codes
    codes = torch.round(y / step) * step
    caches = [torch.zeros(st.n_blocks, hkv, B, DIM, dtype=F64, device="cuda") for _ in range(2)]
    exps = [torch.zeros(st.n_blocks, hkv, B, dtype=torch.int64, device="cuda") for _ in range(2)]
    at = (st.slots.long() // B, slice(None), st.slots.long() % B)
    for i, part in enumerate((slice(0, hkv), slice(hkv, 2 * hkv))):
        caches[i][at] = codes[:, part]
        exps[i][at] = (e[:, part] + 127).long()
    return (rot[:, :hq].reshape(T, -1), *caches, *exps)


def _exact_attention(st):
    case = st.case
    hq, hkv, B = case["heads"], case["kv"], case["block"]
    G, out = hq // hkv, torch.zeros(case["rows"], hq, DIM, dtype=F64, device="cuda")
    parts, before = _shape(case)
    row = 0
    for s, (n, b) in enumerate(zip(parts, before)):
        pages = st.bt[s, :(n + b + B - 1) // B].long()
        for h in range(hkv):
            k, v = ((c[pages, h].view(E4M3).double() * torch.exp2(e[pages, h].double() - 127)[..., None]).reshape(-1, DIM)[:n + b]
                    for c, e in ((st.k, st.ke), (st.v, st.ve)))
            q = st.q[row:row + n].view(n, hq, DIM)[:, h * G:(h + 1) * G].double()
            z = torch.einsum("rgd,td->rgt", q, k) * st.scale
            seen = torch.arange(n + b, device="cuda")[None, :] <= b + torch.arange(n, device="cuda")[:, None]
            z = z.masked_fill(~seen[:, None], float("-inf"))
            out[row:row + n, h * G:(h + 1) * G] = torch.einsum("rgt,td->rgd", torch.softmax(z, -1), v)
        row += n
    return out.reshape(case["rows"], -1)


def _exact_verify(st):
    """A sequence at a time, its drafts in order."""
    n, S, V = st.case["rows"], st.case["seqs"], st.case["vocab"]
    per, u, x, temp = n // S, st.uniforms.double().cpu(), st.tokens.cpu(), st.temperature.double().cpu()
    out, accepted = torch.full((n,), -1, dtype=torch.int64), torch.zeros(S, dtype=torch.int64)
    for s in range(S):
        for j in range(per):
            r = s * per + j
            logits, last, token = st.target[r].double(), j == per - 1, int(x[r])
            if temp[s] <= 0:
                best = int((logits == logits.max()).nonzero()[0])
                out[r] = best
                if last or best != token:
                    break
                accepted[s] += 1
                continue
            p = torch.softmax(logits / temp[s], 0)
            q = torch.zeros_like(p)
            if not last:
                if st.drafter is None:
                    q[token] = 1
                else:
                    q = torch.softmax(st.drafter[r].double() / temp[s], 0)
                if float(u[r, 0] * q[token]) < float(p[token]):
                    out[r] = token
                    accepted[s] += 1
                    continue
            w = (p - q).clamp(min=0)
            w = p if float(w.sum()) == 0 else w
            c = torch.cumsum(w, 0)
            out[r] = int((c > u[r, 1] * c[-1]).nonzero()[0])
            break
    return out, accepted


def exact(case, seed):
    st = prepare(case, seed)
    return _exact_append(st) if case["kind"] == "append" else _exact_verify(st) if case["kind"] == "verify" else _exact_attention(st)
