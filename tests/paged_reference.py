"""The operators over a paged cache in 64 bits, a token at a time, and batches to try them on."""

import torch


def places(lens, starts, tokens):
    """(row, sequence, position) of every token that belongs to a sequence."""
    lens = lens.tolist()
    bounds = list(range(len(lens) + 1)) if starts is None else starts.tolist()
    return [(t, b, lens[b] - (bounds[b + 1] - bounds[b]) + t - bounds[b])
            for b in range(len(lens)) for t in range(bounds[b], bounds[b + 1])]


def rotated(x, cos, sin, interleaved):
    """(x rotated, sum of the magnitudes of its terms) for one row of features in 64 bits."""
    out, size = x.clone(), x.abs().clone()
    if cos is None:
        return out, size
    R = 2 * cos.numel()
    i = torch.arange(R // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
    out[..., a], out[..., b] = x[..., a] * cos - x[..., b] * sin, x[..., b] * cos + x[..., a] * sin
    size[..., a] = (x[..., a] * cos).abs() + (x[..., b] * sin).abs()
    size[..., b] = (x[..., b] * cos).abs() + (x[..., a] * sin).abs()
    return out, size


def chosen_pages(query, bounds, page_size, table, lens, starts, k, first, last, width=None):
    """(T, H_kv, k); rows of no sequence are -1.  CPU tensors."""
    T, heads, D = query.shape
    H = bounds.shape[1]
    out = torch.full((T, H, k), -1, dtype=torch.int32)
    q, bd = query.double(), bounds.double()
    for t, b, pos in places(lens, starts, T):
        seen = pos // page_size + 1 if pos >= 0 else 0
        pages = min(seen, table.shape[1])
        for h in range(H):
            x = q[t, h * (heads // H):(h + 1) * (heads // H)]
            p, n = x.clamp(min=0).sum(0), (-x).clamp(min=0).sum(0)
            p, n = p + torch.where(x.isnan().any(0), torch.nan, 0.0), n
            must = {i for i in range(pages) if i < first or i >= seen - last}
            score = {}
            for i in range(pages):
                page = int(table[b, i])
                if not 0 <= page < bounds.shape[0]:
                    score[i] = -torch.inf
                    continue
                s = float((p * bd[page, h, 1]).sum() - (n * bd[page, h, 0]).sum())
                score[i] = torch.inf if s != s else s
            rest = sorted((i for i in range(pages) if i not in must), key=lambda i: (-score[i], i))
            got = sorted(sorted(must) + rest[:max(0, k - len(must))])[:k] if pages > k else list(range(pages))
            out[t, h, :len(got)] = torch.tensor(got, dtype=torch.int32)
    return out


def attention(query, key_pages, value_pages, table, lens, starts, pages, scale):
    """(out, lse, spread, reach): spread = sum of weight x |value|, reach = the largest sum of |scale q k| of a query."""
    T, heads, D = query.shape
    N, H, P, _ = key_pages.shape
    G = heads // H
    out = torch.zeros(T, heads, D, dtype=torch.float64)
    lse = torch.full((T, heads), -torch.inf, dtype=torch.float64)
    spread = torch.zeros(T, heads, D, dtype=torch.float64)
    reach = torch.zeros(T, heads, dtype=torch.float64)
    for t, b, pos in places(lens, starts, T):
        for h in range(H):
            keys, values = [], []
            for i in pages[t, h].tolist():
                n = min(P, pos + 1 - i * P)
                if i < 0 or n <= 0 or i >= table.shape[1] or not 0 <= int(table[b, i]) < N:
                    continue
                keys.append(key_pages[int(table[b, i]), h, :n])
                values.append(value_pages[int(table[b, i]), h, :n])
            if not keys:
                continue
            k, v = torch.cat(keys).double(), torch.cat(values).double()
            q = query[t, h * G:(h + 1) * G].double()
            s = scale * (q @ k.T)
            at = slice(h * G, (h + 1) * G)
            lse[t, at] = torch.logsumexp(s, 1)
            w = torch.softmax(s, 1)
            out[t, at], spread[t, at] = w @ v, w @ v.abs()
            reach[t, at] = (abs(scale) * (q.abs() @ k.abs().T)).amax(1)
    return out, lse, spread, reach


class Batch:
    """Sequences with pages anywhere in the pools, the tokens of the last call at their ends."""

    def __init__(self, seed, new, lens, page_size, kv_heads, heads, dim, dtype, tail=0, packed=True, spare_pages=3, width=None):
        g = self.g = torch.Generator().manual_seed(seed)
        self.P, self.H, self.heads, self.dim, self.dtype = page_size, kv_heads, heads, dim, dtype
        B = len(lens)
        held = [-(-n // page_size) for n in lens]
        self.N = sum(held) + spare_pages
        order = torch.randperm(self.N, generator=g).int()
        self.table = torch.full((B, width or max(max(held), 1)), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(held):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.lens = torch.tensor(lens, dtype=torch.int32)
        self.starts = torch.tensor([sum(new[:b]) for b in range(B + 1)], dtype=torch.int32) if packed else None
        self.T = sum(new) + tail

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.g).to(self.dtype)

    def rows(self, heads):
        return self.normal(self.T, heads, self.dim)

    def pool(self):
        return self.normal(self.N, self.H, self.P, self.dim)
