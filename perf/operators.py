"""The operators of a paged cache that is read in part: cases, inputs and plain forms.

`append_paged` writes a step's keys and values into the pages, rotated by their positions, and keeps the bounds of every page;
`select_pages` chooses, for each query and key/value head, the pages whose bounds promise the largest scores; `attend_pages` attends
over the chosen pages alone.  `run` computes them in elementary torch operations, or with `own` through the package's entry points.
"""

import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    a = dict(op="append", dtype="bf16", batch=1, new=1, ragged=0, context=4096, heads=32, kv_heads=8, dim=128, page=64, rotary=128,
             interleaved=False)
    s = dict(op="select", dtype="bf16", batch=1, new=1, ragged=0, context=131072, heads=32, kv_heads=8, dim=128, page=64, keep=32,
             first=1, last=2)
    t = dict(op="attend", dtype="bf16", batch=1, new=1, ragged=0, context=32768, heads=32, kv_heads=8, dim=128, page=64, keep=32,
             lse=False)
    return [
        # one token of one conversation: all latency
        dict(a, name="append one token"),
        # a decoding step of a full server
        dict(a, name="append a batch", batch=64, context=2048, ragged=3),
        # a few prompts of odd lengths in one call: every head its own keys, small pages, pairs side by side, a part of the head rotated
        dict(a, name="append ragged prompts", dtype="fp16", batch=7, new=219, ragged=5, context=1500, heads=16, kv_heads=16, dim=80,
             page=16, rotary=64, interleaved=True),
        # a long prompt at once
        dict(a, name="append a long prompt", new=16384, context=16384),
        # one query against a long context
        dict(s, name="select for one query"),
        # a decoding step of a full server, contexts of different lengths
        dict(s, name="select for a batch", batch=32, context=32768, ragged=7),
        # a chunk of a prompt: every query chooses for itself
        dict(s, name="select for a chunk", dtype="fp16", new=1021, context=32768, keep=48),
        # one query, the pages chosen out of a long context
        dict(t, name="attend one query"),
        # a decoding step of a full server
        dict(t, name="attend a batch", batch=32, context=8192, ragged=11),
        # a few tokens of each sequence at once (drafted ones to be verified): every head its own keys, small pages
        dict(t, name="attend drafted tokens", dtype="fp16", batch=24, new=3, ragged=13, context=4096, heads=16, kv_heads=16, dim=64, page=16,
             keep=64, lse=True),
        # few sequences that keep much of a long context
        dict(t, name="attend much of a context", batch=4, context=65536, keep=256, lse=True),
        # a chunk of a prompt: every query reads the pages it chose
        dict(t, name="attend a chunk", new=512, context=32768),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(("append", "select", "attend"))
    group = rng.choice((1, 2, 4, 4, 8))
    kv = rng.choice((2, 4, 8, 16) if group < 8 else (2, 4, 8))
    c = dict(op=op, dtype=rng.choice(("bf16", "fp16")), heads=group * kv, kv_heads=kv, dim=rng.choice((64, 64, 80, 96, 128, 128)),
             page=rng.choice((16, 32, 64, 64, 128)), ragged=rng.randrange(0, 100), batch=spread(1, 64), new=1)
    if rng.random() < 0.4:   # several tokens a sequence
        c["batch"] = spread(1, 8)
        c["new"] = spread(2, 16384 if op == "append" else 1024)
    c["context"] = 2 * c["new"] + spread(4096 if op == "select" else 16, 4096 if op == "append" else 131072)
    if op == "append":
        c["rotary"] = rng.choice((c["dim"], c["dim"], 32, 0))
        c["interleaved"] = rng.random() < 0.3
    else:
        c["keep"] = spread(4, 256)
        if op == "select":
            c["first"], c["last"] = rng.randrange(0, 2), rng.randrange(1, 3)
        else:
            c["lse"] = rng.random() < 0.5
    most = [work(d) for d in listed() if d["op"] == op]
    # (the plain form of `select` lays the pages' bounds out for each token)
    while (any(work(c)[what] > max(w[what] for w in most) for what in ("bytes", "flops"))
           or c["batch"] * c["new"] * -(-c["context"] // c["page"]) * c["kv_heads"] * c["dim"] * (op == "select") > 6e8
           or c["batch"] * c["new"] * c.get("keep", 0) * c["page"] * c["heads"] * c["dim"] > 2.2e9 * c["heads"] / c["kv_heads"]
           or c["batch"] * c["context"] * c["kv_heads"] * c["dim"] > 6e8 * (1 + 8 * (op == "select"))):
        if c["batch"] > 1 and (c["new"] == 1 or rng.random() < 0.5):
            c["batch"] = (c["batch"] + 1) // 2
        elif c["new"] > 1:
            c["context"] -= 2 * (c["new"] - (c["new"] + 1) // 2)
            c["new"] = (c["new"] + 1) // 2
        elif op == "attend" and c["keep"] > 4:
            c["keep"] //= 2
        else:
            c["context"] = (c["context"] + 1) // 2
    if op == "select":   # (there is something to choose)
        c["keep"] = max(4, min(c["keep"], c["context"] // (4 * c["page"])))
    return c


def _lengths(case):
    """New tokens and cached tokens (the new ones included) of every sequence."""
    r = random.Random(case["ragged"])
    odd = case["ragged"] > 0
    new = [r.randint(max(1, case["new"] // 2), case["new"] + case["new"] // 2) if odd else case["new"] for _ in range(case["batch"])]
    return new, [max(n, r.randint(case["context"] // 2, case["context"]) if odd else case["context"]) for n in new]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, B, P, H, D = TYPES[case["dtype"]], case["batch"], case["page"], case["kv_heads"], case["dim"]
    new, lens = _lengths(case)
    T, held = sum(new), [-(-n // P) for n in lens]
    width, pages = max(held), sum(held)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)

    # the pages of the sequences lie anywhere in the pools; entries of the table past a sequence's end are -1
    order = torch.randperm(pages, generator=g, device="cuda").int()
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b in range(B):
        table[b, :held[b]] = order[at:at + held[b]]
        at += held[b]
    starts = None
    if max(new) > 1:
        starts = torch.tensor([sum(new[:b]) for b in range(B + 1)], dtype=torch.int32, device="cuda")
    st = dict(case=case, query=normal(T, case["heads"], D), table=table, starts=starts,
              lens=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    if case["op"] == "append":
        st["key"], st["value"] = normal(T, H, D), normal(T, H, D)
        st["key_pages"], st["value_pages"] = normal(pages, H, P, D), normal(pages, H, P, D)
        st["bounds"] = torch.stack([st["key_pages"].amin(2), st["key_pages"].amax(2)], 2)
        st["cos"] = st["sin"] = None
        if case["rotary"]:
            rate = 500000.0 ** (-torch.arange(0, case["rotary"], 2, device="cuda", dtype=torch.float64) / case["rotary"])
            angle = torch.arange(max(lens), device="cuda", dtype=torch.float64)[:, None] * rate
            st["cos"], st["sin"] = angle.cos().float(), angle.sin().float()
    elif case["op"] == "select":
        # the extremes of P normal values around each page's own centre, drawn as such
        centre = 0.5 * torch.randn(pages, H, D, generator=g, device="cuda")
        u = torch.rand(2, pages, H, D, generator=g, device="cuda").clamp(1e-6, 1 - 1e-6).pow(1.0 / P).clamp(max=1 - 1e-6)
        reach = torch.special.ndtri(u)
        st["bounds"] = torch.stack([centre - reach[0].clamp(min=0), centre + reach[1].clamp(min=0)], 2).to(dtype)
    else:
        st["key_pages"], st["value_pages"] = normal(pages, H, P, D), normal(pages, H, P, D)
        # the first and the last page, and pages that matter to the sequence as a whole and to the query
        seq, pos = _places(st)
        last = (pos // P)[:, None, None]
        page = torch.arange(width, device="cuda")
        score = (torch.randn(B, H, width, generator=g, device="cuda")[seq]
                 + 0.5 * torch.randn(T, H, width, generator=g, device="cuda"))
        score = score.masked_fill((page == 0) | (page == last), 1e4).masked_fill(page > last, -1e4)
        keep = min(case["keep"], width)
        best = score.topk(keep, dim=2).indices
        best = best.masked_fill(best > last, width).sort(2).values
        st["pages"] = best.masked_fill(best == width, -1).int()
    return st


def _places(st):
    """Every new token's sequence and position."""
    lens = st["lens"].long()
    if st["starts"] is None:
        return torch.arange(lens.numel(), device=lens.device), lens - 1
    starts = st["starts"].long()
    t = torch.arange(st["query"].shape[0], device=lens.device)
    seq = (starts[1:] <= t[:, None]).sum(1)
    return seq, lens[seq] - starts[seq + 1] + t


def _rotated(x, st, pos):
    """x (T, heads, D) rotated by its tokens' positions: pairs half the rotated part apart, or side by side."""
    if st["cos"] is None:
        return x
    cos, sin = st["cos"][pos][:, None], st["sin"][pos][:, None]
    R = 2 * cos.shape[2]
    part, rest = x[..., :R].float(), x[..., R:]
    if st["case"]["interleaved"]:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], 3).flatten(2)
    else:
        a, b = part[..., :R // 2], part[..., R // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], 2)
    return torch.cat([turned.to(x.dtype), rest], 2)


def _plain_append(st):
    P = st["case"]["page"]
    seq, pos = _places(st)
    query, key = _rotated(st["query"], st, pos), _rotated(st["key"], st, pos)
    page, slot = st["table"].long()[seq, pos // P], pos % P
    st["key_pages"][page, :, slot] = key
    st["value_pages"][page, :, slot] = st["value"]
    # a page that is begun forgets what it held
    begun = torch.zeros(st["bounds"].shape[0], device=page.device).index_add_(0, page, (slot == 0).float()) > 0
    low, high = st["bounds"].float().unbind(2)
    low = low.masked_fill(begun[:, None, None], math.inf).index_reduce_(0, page, key.float(), "amin")
    high = high.masked_fill(begun[:, None, None], -math.inf).index_reduce_(0, page, key.float(), "amax")
    st["bounds"].copy_(torch.stack([low, high], 2))
    return query, st["key_pages"], st["value_pages"], st["bounds"]


def _plain_select(st):
    c = st["case"]
    T, B, width = st["query"].shape[0], c["batch"], st["table"].shape[1]
    seq, pos = _places(st)
    q = st["query"].double().view(T, c["kv_heads"], -1, c["dim"])       # (64 bits: scores next to the border)
    parts = torch.stack([-(-q).clamp(min=0).sum(2), q.clamp(min=0).sum(2)], 2).flatten(2)
    of_pages = st["bounds"][st["table"].long().clamp(min=0)].double().flatten(3)
    if B == 1:
        score = torch.einsum("thd,phd->thp", parts, of_pages[0])
    else:
        score = torch.einsum("thd,tphd->thp", parts, of_pages[seq])
    last = (pos // c["page"])[:, None, None]
    page = torch.arange(width, device=pos.device)
    score = score.masked_fill((page < c["first"]) | (page > last - c["last"]), math.inf).masked_fill(page > last, -math.inf)
    best = score.sort(dim=2, descending=True, stable=True).indices[..., :c["keep"]]
    best = best.masked_fill(best > last, width).sort(2).values
    best = torch.cat([best, best.new_full((T, c["kv_heads"], max(0, c["keep"] - width)), width)], 2)
    return best.masked_fill(best == width, -1).int()


def _plain_attend(st):
    c = st["case"]
    T, H, P, D = st["query"].shape[0], c["kv_heads"], c["page"], c["dim"]
    seq, pos = _places(st)
    chosen = st["pages"].long()
    page = st["table"].long()[seq[:, None, None], chosen.clamp(min=0)]
    head = torch.arange(H, device=pos.device)[None, :, None]
    at = chosen[..., None] * P + torch.arange(P, device=pos.device)
    seen = ((chosen[..., None] >= 0) & (at <= pos[:, None, None, None])).flatten(2)[:, :, None]
    q = st["query"].float().view(T, H, -1, D)
    score = q @ st["key_pages"][page, head].flatten(2, 3).float().transpose(2, 3) * D ** -0.5
    score = score.masked_fill(~seen, -math.inf)
    most = score.amax(3, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    weight = (score - most).exp()
    total = weight.sum(3, keepdim=True)
    out = weight @ st["value_pages"][page, head].flatten(2, 3).float() / total.clamp(min=1e-30)
    out = out.flatten(1, 2).to(st["query"].dtype)
    return (out, (most + total.log()).flatten(1)) if c["lse"] else out


def run(st):
    op = st["case"]["op"]
    if not own:
        return _plain_append(st) if op == "append" else _plain_select(st) if op == "select" else _plain_attend(st)
    import flash_colsum_b200 as fc
    c = st["case"]
    if op == "append":
        query = fc.append_paged(st["key"], st["value"], st["key_pages"], st["value_pages"], st["table"], st["lens"],
                                starts=st["starts"], query=st["query"], cos=st["cos"], sin=st["sin"],
                                interleaved=c["interleaved"], bounds=st["bounds"])
        return query, st["key_pages"], st["value_pages"], st["bounds"]
    if op == "select":
        return fc.select_pages(st["query"], st["bounds"], st["table"], st["lens"], c["keep"], page_size=c["page"],
                               starts=st["starts"], first=c["first"], last=c["last"])
    return fc.attend_pages(st["query"], st["key_pages"], st["value_pages"], st["table"], st["lens"], st["pages"],
                           starts=st["starts"], return_lse=c["lse"])


def exact(case, seed):
    """The same in 64 bits, a sequence at a time."""
    st = prepare(case, seed)
    P, H, D, G = case["page"], case["kv_heads"], case["dim"], case["heads"] // case["kv_heads"]
    new, lens = _lengths(case)
    query = st["query"].double()
    outs, sums, t = [], [], 0
    if case["op"] == "append":
        key_pages, value_pages, bounds = (st[n].double() for n in ("key_pages", "value_pages", "bounds"))
        half = case["rotary"] // 2
        pair = torch.arange(half, device="cuda")
        one, other = (2 * pair, 2 * pair + 1) if case["interleaved"] else (pair, pair + half)
        for b, (n, length) in enumerate(zip(new, lens)):
            rows, where = slice(t, t + n), torch.arange(length - n, length, device="cuda")
            turned = [query[rows].clone(), st["key"][rows].double()]
            if half:
                turn = torch.complex(st["cos"][length - n:length].double(), st["sin"][length - n:length].double())[:, None]
                for x in turned:
                    z = torch.complex(x[..., one], x[..., other]) * turn
                    x[..., one], x[..., other] = z.real, z.imag
            outs.append(turned[0])
            first = length - n
            while first < length:
                slot, end = first % P, min(length, first - first % P + P)
                page, part = int(st["table"][b, first // P]), turned[1][first - length + n:end - length + n]
                key_pages[page, :, slot:slot + end - first] = part.transpose(0, 1)
                value_pages[page, :, slot:slot + end - first] = st["value"][t + first - length + n:t + end - length + n].double().transpose(0, 1)
                low, high = part.min(0).values, part.max(0).values
                if slot:
                    low, high = torch.minimum(low, bounds[page, :, 0]), torch.maximum(high, bounds[page, :, 1])
                bounds[page, :, 0], bounds[page, :, 1] = low, high
                first = end
            t += n
        return torch.cat(outs), key_pages, value_pages, bounds
    if case["op"] == "select":
        for b, (n, length) in enumerate(zip(new, lens)):
            held = -(-length // P)
            low, high = st["bounds"][st["table"][b, :held].long()].double().unbind(2)
            chosen = torch.full((n, H, case["keep"]), -1, dtype=torch.int32)
            for h in range(H):
                score = 0.0
                for x in query[t:t + n, h * G:(h + 1) * G].unbind(1):
                    score = score + x.clamp(max=0) @ low[:, h].T + x.clamp(min=0) @ high[:, h].T
                score = score.cpu()
                for i in range(n):
                    see = (length - n + i) // P + 1
                    must = [p for p in range(see) if p < case["first"] or p >= see - case["last"]]
                    rest = [p for p in score[i, :see].sort(descending=True, stable=True).indices.tolist() if p not in set(must)]
                    got = sorted((must + rest)[:case["keep"]])
                    chosen[i, h, :len(got)] = torch.tensor(got, dtype=torch.int32)
            outs.append(chosen)
            t += n
        return torch.cat(outs)
    for b, (n, length) in enumerate(zip(new, lens)):
        held = -(-length // P)
        at = st["table"][b, :held].long()
        marks = torch.zeros(n, H, held + 1, dtype=torch.bool, device="cuda")
        chosen = st["pages"][t:t + n].long()
        marks.scatter_(2, torch.where(chosen < 0, held, chosen), True)
        seen = marks[..., :held].repeat_interleave(P, 2)
        seen &= torch.arange(held * P, device="cuda") <= torch.arange(length - n, length, device="cuda")[:, None, None]
        for h in range(H):
            k, v = (st[m][at, h].reshape(-1, D).double() for m in ("key_pages", "value_pages"))
            score = torch.where(seen[:, h, None], query[t:t + n, h * G:(h + 1) * G] @ k.T / math.sqrt(D), -math.inf)
            sums.append(torch.logsumexp(score, 2))
            outs.append(torch.softmax(score, 2) @ v)
        t += n
    out = torch.cat([torch.cat(outs[b * H:(b + 1) * H], 1) for b in range(len(new))])
    lse = torch.cat([torch.cat(sums[b * H:(b + 1) * H], 1) for b in range(len(new))])
    return (out, lse) if case["lse"] else out


def work(case):
    new, lens = _lengths(case)
    T, P, H, D = sum(new), case["page"], case["kv_heads"], case["dim"]
    if case["op"] == "append":
        touched = sum(-(-n // P) - (n - m) // P for m, n in zip(new, lens))
        return {"bytes": 2.0 * 2 * T * (case["heads"] + 2 * H) * D + 4.0 * T * case["rotary"] + 2.0 * 4 * touched * H * D,
                "flops": 3.0 * T * (case["heads"] + H) * case["rotary"]}
    if case["op"] == "select":
        # the bounds of every page that a query sees, once; the queries and the chosen pages
        held = sum(-(-n // P) for n in lens)
        return {"bytes": 4.0 * held * H * D + 2.0 * T * case["heads"] * D + 4.0 * T * H * case["keep"],
                "flops": sum(4.0 * m * -(-n // P) * H * D for m, n in zip(new, lens))}
    # the pages that are chosen, once for a sequence; a query's keys
    keep = [min(case["keep"], -(-n // P)) for n in lens]
    pages = sum(min(m * k, -(-n // P)) for m, n, k in zip(new, lens, keep))
    return {"bytes": 4.0 * pages * H * P * D + 4.0 * T * case["heads"] * D + 4.0 * T * H * case["keep"] + 4.0 * T * case["heads"] * case["lse"],
            "flops": sum(4.0 * m * k * P * case["heads"] * D for m, k in zip(new, keep))}
