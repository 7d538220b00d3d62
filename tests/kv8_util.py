"""The 8-bit cache and the check of drafts in plain torch, 64 bits where values are computed: what the kernels are held to."""
import torch

E4M3 = torch.float8_e4m3fn


def exp_bytes(x):
    """Exponent byte of rows [..., 128]: the smallest e >= -100 with amax <= 448 * 2^e, + 127; 255 for inf and NaN."""
    m = x.double().abs().amax(-1)
    e = torch.full(m.shape, -100, dtype=torch.int32)
    for k in range(-100, 121):   # (by its definition: the bound of each exponent in turn)
        e = torch.where(m > 448.0 * 2.0 ** k, k + 1, e)
    return torch.where(torch.isfinite(m), e + 127, 255).to(torch.uint8)


def quantise(x):
    """fp32 rows -> (codes as bytes, exponent bytes)."""
    b = exp_bytes(x)
    f = torch.ldexp(torch.ones(b.shape), 127 - b.to(torch.int32))
    codes = (torch.where((b == 255)[..., None], torch.nan, x.float()) * torch.where(b == 255, 1.0, f)[..., None]).to(E4M3)
    return codes.view(torch.uint8) & torch.where((b == 255)[..., None], 0x7f, 0xff).to(torch.uint8), b


def values(codes, exps):
    e = exps.to(torch.int32)
    return codes.view(E4M3).double() * torch.where(e == 255, torch.nan, torch.exp2(e.double() - 127))[..., None]


def rope(x, pos, cos_sin):
    """fp32 rows [T][heads][128]: every output rounded once from exact products."""
    cs = cos_sin[pos.long()].double()[:, None]
    c, s, a, b = cs[..., :64], cs[..., 64:], x.double()[..., :64], x.double()[..., 64:]
    return torch.cat([(a * c - b * s).float(), (b * c + a * s).float()], -1)


class Cache:
    """A paged cache of several sequences: blocks in random order, NaN codes wherever nobody may look."""

    def __init__(self, lengths, hkv, block, g, spread=1.0, spare=3):
        need = [(n + block - 1) // block for n in lengths]
        self.block, self.hkv, self.n_blocks = block, hkv, sum(need) + spare
        order = torch.randperm(self.n_blocks, generator=g).to(torch.int32)
        self.bt = torch.full((len(lengths), max(need + [1]) + 1), -7, dtype=torch.int32)
        shape = (self.n_blocks, hkv, block)
        self.k, self.v = (torch.full((*shape, 128), 0x7f, dtype=torch.uint8) for _ in range(2))
        self.ke, self.ve = (torch.full(shape, 255, dtype=torch.uint8) for _ in range(2))
        self.rows, at = [], 0
        for s, n in enumerate(lengths):
            self.bt[s, :need[s]] = order[at:at + need[s]]
            at += need[s]
            kv = [quantise(torch.randn(n, hkv, 128, generator=g) * torch.exp2(torch.randn(n, hkv, 1, generator=g) * spread)) for _ in range(2)]
            for (codes, exps), c, e in ((kv[0], self.k, self.ke), (kv[1], self.v, self.ve)):
                for b in range(need[s]):
                    part = slice(b * block, min((b + 1) * block, n))
                    size = part.stop - part.start
                    c[self.bt[s, b], :, :size] = codes[part].transpose(0, 1)
                    e[self.bt[s, b], :, :size] = exps[part].transpose(0, 1)
            self.rows.append([values(*x) for x in kv])

    def to(self, dev):
        for n in ("k", "v", "ke", "ve", "bt"):
            setattr(self, n, getattr(self, n).to(dev))
        return self


def attention(q, rows, ctx, scale):
    """One row's heads over keys and values in 64 bits: (result, sum of weighted magnitudes, the largest magnitude)."""
    k, v = (x[:ctx] for x in rows)
    hkv, heads = k.shape[1], q.shape[0]
    if ctx <= 0:
        z = torch.zeros(heads, 128, dtype=torch.float64)
        return z, z, 0.0
    k, v = (x.repeat_interleave(heads // hkv, 1) for x in (k, v))
    p = torch.softmax(torch.einsum("hd,chd->hc", q.double(), k) * scale, -1)
    return torch.einsum("hc,chd->hd", p, v), torch.einsum("hc,chd->hd", p, v.abs()), float(v.abs().max())


def verify(target, draft, tokens, starts, temperature, uniforms):
    """(tokens, kept drafts, how near each decision came to its limit)."""
    n, V = target.shape
    out, kept, margins = torch.full((n,), -9, dtype=torch.int64), [], []
    for s in range(len(starts) - 1):
        r0, r1 = int(starts[s]), int(starts[s + 1])
        temp, took, token = (0.0 if temperature is None else float(temperature[s])), 0, -1
        for r in range(r0, r1):
            last, x, row = r == r1 - 1, int(tokens[r]), target[r].double()
            top = row.max()
            if temp <= 0 or top == float("-inf"):
                token = int((row == top).nonzero()[0])
                if not last and x == token and top > float("-inf"):
                    took += 1
                    continue
                break
            p = torch.softmax(row / temp, 0)
            q = torch.zeros(V, dtype=torch.float64)
            if not last and draft is None and 0 <= x < V:
                q[x] = 1
            elif not last and draft is not None and draft[r].max() > float("-inf"):
                q = torch.softmax(draft[r].double() / temp, 0)
            if not last and 0 <= x < V:
                a, b = float(uniforms[r, 0].double() * q[x]), float(p[x])
                margins.append(abs(a - b) / max(a, b, 1e-300))
                if a < b:
                    took += 1
                    continue
            w = (p - q).clamp(min=0)
            w = w if float(w.sum()) > 0 else p
            c = torch.cumsum(w, 0)
            limit = uniforms[r, 1].double() * c[-1]
            token = int((c > limit).nonzero()[0])
            margins.append(float((c - limit).abs().min() / c[-1]) * 1e6)   # (sums in 64 bits: 1e-12 is far)
            break
        if r1 > r0:
            for i in range(took):
                out[r0 + i] = tokens[r0 + i]
            out[r0 + took] = token
            out[r0 + took + 1:r1] = -1
        kept.append(took)
    return out, torch.tensor(kept, dtype=torch.int64), margins
