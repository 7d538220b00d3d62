"""Several continuations of a sequence in plain torch, 64 bits where values are computed: what the kernels are held to."""
import torch

I32, I64, F64 = torch.int32, torch.int64, torch.float64


def masks(lines, words):
    """Rows of bits, as int32 words, from each row's list of tail tokens."""
    m = torch.zeros(len(lines), words, dtype=I64)
    for i, line in enumerate(lines):
        for j in set(line):
            m[i, j // 32] |= 1 << (j % 32)
    return torch.where(m >= 2 ** 31, m - 2 ** 32, m).to(I32)


def lines(parents):
    """The way to each node of a tree, itself included (parents[0] is not looked at)."""
    out = []
    for i, p in enumerate(parents):
        out.append((out[p] if i else []) + [i])
    return out


class Cache:
    """A paged bf16 cache of several sequences: blocks in random order, NaN wherever nobody may look."""

    def __init__(self, lengths, hkv, block, g, spare=3, spread=1.0):
        need = [(n + block - 1) // block for n in lengths]
        self.block, self.hkv, self.n_blocks = block, hkv, sum(need) + spare
        order = torch.randperm(self.n_blocks, generator=g).to(I32)
        self.bt = torch.full((len(lengths), max(need + [1])), -7, dtype=I32)
        self.k, self.v = (torch.full((self.n_blocks, hkv, block, 128), float("nan"), dtype=torch.bfloat16) for _ in range(2))
        at = 0
        for s, n in enumerate(lengths):
            self.bt[s, :need[s]] = order[at:at + need[s]]
            at += need[s]
            for j in range(0, n, block):
                size = min(block, n - j)
                b = self.bt[s, j // block]
                for c in (self.k, self.v):
                    c[b, :, :size] = (torch.randn(hkv, size, 128, generator=g) * torch.exp2(torch.randn(hkv, size, 1, generator=g) * spread)).to(torch.bfloat16)

    def token(self, s, j):
        """(block, place) of a sequence's token."""
        return int(self.bt[s, j // self.block]), j % self.block

    def rows(self, s, n):
        """Keys and values of a sequence's first n tokens [n][hkv][128]; a block that is none: zeros."""
        out = []
        for c in (self.k, self.v):
            x = torch.zeros((n + self.block - 1) // self.block, self.hkv, self.block, 128, dtype=F64)
            for i in range(x.shape[0]):
                b = int(self.bt[s, i])
                if 0 <= b < self.n_blocks:
                    x[i] = c[b].double()
            out.append(x.transpose(1, 2).reshape(-1, self.hkv, 128)[:n])
        return out


def attention(q, k, v, seen, scale):
    """One row's heads over the tokens it sees: (result, sum of weighted magnitudes)."""
    heads, hkv = q.shape[0], k.shape[1]
    if len(seen) == 0:
        z = torch.zeros(heads, 128, dtype=F64)
        return z, z
    k, v = (x[seen].repeat_interleave(heads // hkv, 1) for x in (k, v))
    p = torch.softmax(torch.einsum("hd,chd->hc", q.double(), k) * scale, -1)
    return torch.einsum("hc,chd->hd", p, v), torch.einsum("hc,chd->hd", p, v.abs())


def select(logits, scores, starts, take):
    """(rows, tokens, scores) of each sequence's best candidates."""
    S, V = len(starts) - 1, logits.shape[1]
    rows, tokens = (torch.full((S, take), -1, dtype=I64) for _ in range(2))
    out = torch.full((S, take), float("-inf"), dtype=F64)
    for s in range(S):
        a, b = int(starts[s]), int(starts[s + 1])
        if b <= a:
            continue
        x = logits[a:b].double()
        m = x.amax(1, keepdim=True)
        base = (torch.zeros(b - a, dtype=F64) if scores is None else scores[a:b].double())[:, None] - (m + (x - m).exp().sum(1, keepdim=True).log())
        # within a row by the logits themselves: next to a large log-sum 64 bits may not tell two of them apart
        by = torch.sort(torch.where(torch.isnan(x), float("-inf"), x), dim=1, descending=True, stable=True).indices
        x, by = x.gather(1, by), (by + V * torch.arange(b - a)[:, None]).reshape(-1)
        x = torch.where(torch.isfinite(base) & torch.isfinite(x), base + x, float("-inf")).reshape(-1)   # (of a row that is none: nothing)
        value, at = torch.sort(x, descending=True, stable=True)
        n = min(take, int((value > float("-inf")).sum()))
        rows[s, :n], tokens[s, :n], out[s, :n] = a + by[at[:n]] // V, by[at[:n]] % V, value[:n]
    return rows, tokens, out


def accept(target, drafts, parents, starts, slots):
    n = len(target)
    out, path, src, dst = (torch.full((n,), -9, dtype=I64) for _ in range(4))
    accepted = []
    for a, b in zip(starts.tolist(), starts.tolist()[1:]):
        line = [a] if b > a else []
        while line:
            nxt = [r for r in range(line[-1] + 1, b) if a + int(parents[r]) == line[-1] and drafts[r] == target[line[-1]]]
            if not nxt:
                break
            line.append(nxt[0])
        for t in (out, path, src, dst):
            t[a:b] = -1
        for i, r in enumerate(line):
            out[a + i], path[a + i] = target[r], r
            if r != a + i:
                src[a + i], dst[a + i] = slots[r], slots[a + i]
        accepted.append(max(0, len(line) - 1))
    return out, path, torch.tensor(accepted, dtype=I64), src, dst


def moved(cache, src, dst, starts, most):
    """[layers][blocks][heads][block][...] after the moves."""
    new, B, n = cache.clone(), cache.shape[3], cache.shape[1] * cache.shape[3]
    for a, b in zip(starts.tolist(), starts.tolist()[1:]):
        for i in range(a, min(b, a + most)):
            x, y = int(src[i]), int(dst[i])
            if 0 <= x < n and 0 <= y < n:
                new[:, y // B, :, y % B] = cache[:, x // B, :, x % B]
    return new
