"""Cases of the operators for a batch of users on one paged cache: attention that reads a prefix that all of them share once,
sampling of the next token and the truncation of logits to what may be sampled, and the hand-out of the cache's pages.

Each case names an operator and its sizes; `run` makes one pass, in plain torch operations or through the library."""
import ctypes
import math
import random

import torch

own = False

# (query heads, key/value heads, values per head): the heads of the served model (24/2/256), and generic ones.
HEADS = {"24/2/256": (24, 2, 256), "32/8/128": (32, 8, 128), "16/4/64": (16, 4, 64), "10/10/128": (10, 10, 128)}
# What users ask of the sampler: (temperature, top_k, top_p, min_p); 0, 0, 1 and 0 leave a setting out.
SETTINGS = [(0.8, 40, 0.95, 0.0), (1.0, 0, 0.9, 0.0), (0.7, 0, 1.0, 0.05), (0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.0), (0.6, 20, 0.95, 0.02),
            (1.3, 200, 1.0, 0.1), (0.9, 1000, 0.8, 0.0), (1.0, 0, 0.98, 0.0), (0.7, 5, 1.0, 0.0)]


def listed():
    return [
        # two users a few words after a system prompt of some lines: latency only
        {"name": "shared short", "op": "attention", "heads": "24/2/256", "seqs": 2, "tokens": 1, "shared": 208, "length": 9, "page": 16, "tree": False},
        # many users with a system prompt and tools, a token each
        {"name": "shared decode", "op": "attention", "heads": "32/8/128", "seqs": 64, "tokens": 1, "shared": 4112, "length": 700, "page": 16, "tree": False},
        # the verify batch of this framework (17 rows) for several users at once
        {"name": "shared verify", "op": "attention", "heads": "24/2/256", "seqs": 8, "tokens": 17, "shared": 8192, "length": 1000, "page": 64, "tree": True},
        # short chains of several users, small heads, an odd number of them
        {"name": "shared chains", "op": "attention", "heads": "16/4/64", "seqs": 33, "tokens": 5, "shared": 1504, "length": 300, "page": 32, "tree": False},
        # questions about one long document
        {"name": "shared document", "op": "attention", "heads": "24/2/256", "seqs": 48, "tokens": 5, "shared": 32768, "length": 2000, "page": 64, "tree": True},
        # the next token of one user
        {"name": "sample one", "op": "sample", "rows": 1, "vocab": 131072, "asked": 0, "rounded": False},
        # users who ask for different things, an odd vocabulary, logits of a head with 16-bit outputs
        {"name": "sample mixed", "op": "sample", "rows": 37, "vocab": 50001, "asked": -1, "rounded": True},
        # a large batch without any truncation but the nucleus
        {"name": "sample nucleus", "op": "sample", "rows": 256, "vocab": 131072, "asked": 1, "rounded": False},
        # what one user's verify batch may draw from
        {"name": "truncate verify", "op": "truncate", "rows": 17, "tokens": 17, "vocab": 131072, "asked": 0, "rounded": False},
        # the same for twelve users with settings of their own
        {"name": "truncate batch", "op": "truncate", "rows": 204, "tokens": 17, "vocab": 131072, "asked": -1, "rounded": True},
        # pages for the verify batches of a few users
        {"name": "pages few", "op": "pages", "seqs": 4, "tokens": 17, "length": 900, "page": 64, "ahead": 0, "scarce": False},
        # many users, prompts among them, more than the pool has room for
        {"name": "pages batch", "op": "pages", "seqs": 700, "tokens": 512, "length": 3000, "page": 16, "ahead": 8, "scarce": True},
    ]


def spread(rng, low, high):
    """A whole number between low and high, spread over the logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "sample", "sample", "truncate", "pages"])
    if op == "pages":
        seqs = spread(rng, 1, 1000)
        return {"op": op, "seqs": seqs, "tokens": spread(rng, 1, min(4096, 700 * 512 // seqs)), "length": spread(rng, 1, 3000),
                "page": rng.choice([16, 32, 64, 128, 256]), "ahead": rng.randrange(9), "scarce": rng.random() < 0.5}
    if op == "attention":
        heads = rng.choice(list(HEADS))
        hq, hkv, d = HEADS[heads]
        page = rng.choice([16, 32, 64, 128])
        seqs, tokens = spread(rng, 1, 64), spread(rng, 1, 24)
        most = min(32768 * 240 * 24 * 256 // (seqs * tokens * hq * d), 32768)
        shared = spread(rng, 1, max(1, most // page)) * page
        length = spread(rng, 1, max(1, min(3000, 48 * 2000 * 512 // (seqs * hkv * d))))
        return {"op": op, "heads": heads, "seqs": seqs, "tokens": tokens, "shared": shared, "length": length, "page": page, "tree": rng.random() < 0.5}
    vocab = spread(rng, 1000, 200000)
    case = {"op": op, "rows": 1, "vocab": vocab, "asked": rng.choice([-1, -1, *range(len(SETTINGS))]), "rounded": rng.random() < 0.4}
    if op == "sample":
        return dict(case, rows=spread(rng, 1, min(400, 256 * 131072 // vocab)))
    tokens = spread(rng, 1, 24)
    return dict(case, tokens=tokens, rows=tokens * spread(rng, 1, max(1, min(16, 204 * 131072 // (vocab * tokens)))))


def work(case):
    if case["op"] == "pages":
        touched = case["seqs"] * (case["tokens"] + 3.0 * (case["tokens"] / 2 / case["page"] + 1.0) + 5.0)
        return {"bytes": touched * 4.0, "flops": 0.0}
    if case["op"] == "attention":
        hq, hkv, d = HEADS[case["heads"]]
        rows, tails = case["seqs"] * case["tokens"], [n + case["tokens"] for n in case_lengths(case)]
        seen = case["tokens"] * sum(case["shared"] + n for n in tails)
        return {"bytes": (case["shared"] + sum(tails)) * hkv * d * 4.0 + rows * hq * d * 8.0, "flops": 4.0 * seen * hq * d}
    values = case["rows"] * case["vocab"]
    return {"bytes": values * (8.0 if case["op"] == "truncate" else 4.0), "flops": values * 4.0}


def case_lengths(case):
    """The committed tokens of each sequence, after what is shared: from short ones up to case["length"]."""
    return [case["length"] * (s + 1) // case["seqs"] for s in range(case["seqs"])]


def make_tree(rng, tokens, tree):
    """The parent of each node: a chain, or a tree of mostly small fan-out (node 0 is the root)."""
    return [-1] + [max(rng.randrange(i), rng.randrange(i)) if tree else i - 1 for i in range(1, tokens)]


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    rng = random.Random(seed)
    s = dict(case)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    floats = lambda v: torch.tensor(v, dtype=torch.float32, device=dev)  # noqa: E731
    if case["op"] == "attention":
        hq, hkv, d = HEADS[case["heads"]]
        seqs, tokens, page = case["seqs"], case["tokens"], case["page"]
        lengths = [case["shared"] + n for n in case_lengths(case)]
        table_pages, common = -(-(max(lengths) + tokens) // page), case["shared"] // page
        pages = common + seqs * (table_pages - common) + 3
        order = torch.randperm(pages, device=dev, generator=gen).int()
        table = order[common : common + seqs * (table_pages - common)].view(seqs, -1)
        table = torch.cat([order[:common].expand(seqs, common), table], dim=1).contiguous()
        s.update(hq=hq, hkv=hkv, d=d, table=table, table_pages=table_pages, pages=pages, longest=max(lengths) + tokens, scale=1.0 / math.sqrt(d))
        s.update(lengths=ints(lengths), shared_at=ints([case["shared"]]))
        s["k"] = torch.empty(pages, page, hkv, d, dtype=torch.float16, device=dev).normal_(generator=gen)
        s["v"] = torch.empty(pages, page, hkv, d, dtype=torch.float16, device=dev).normal_(generator=gen)
        s["q"] = 1.5 * torch.randn(seqs * tokens, hq, d, device=dev, generator=gen)
        s["out"] = torch.zeros_like(s["q"])
        s["tree_mask"] = None
        if case["tree"]:
            masks = []
            for _ in range(seqs):
                m = []
                for i, p in enumerate(make_tree(rng, tokens, True)):
                    m.append((m[p] if i else 0) | 1 << i)
                masks.append(m)
            s["tree_mask"] = torch.tensor(masks, dtype=torch.int64, device=dev)
        if own:
            from nebula_b200 import lib

            s["lib"] = lib
            s["cache"] = lib.KvCache(s["k"].data_ptr(), s["v"].data_ptr(), table.data_ptr(), s["lengths"].data_ptr(), s["k"].numel() * 2, 1,
                                     pages, page, table_pages, hkv, d)
            s["workspace"] = lib.shared_attention_workspace(seqs, tokens, hq, hkv, d)
        return s
    if case["op"] == "pages":
        seqs, tokens, page = case["seqs"], case["tokens"], case["page"]
        lengths = case_lengths(case)
        need = [-(-n // page) for n in lengths]
        most = sum(-(-(n + tokens) // page) for n in lengths) - sum(need)
        room = (most // 2 if case["scarce"] else most) + 5
        pages, left, held = sum(need) + room, room // 2, []
        for n in need:  # with what the step before did not commit
            more = min(left, rng.randrange(-(-tokens // page) + 1))
            held, left = held + [n + more], left - more
        counts = [rng.choice([tokens, rng.randrange(tokens + 1)]) for _ in range(seqs)]
        table_pages = max(need) + -(-tokens // page) + case["ahead"]
        order = torch.randperm(pages, device=dev, generator=gen).int()
        place = torch.arange(table_pages, device=dev)
        mine = place < ints(held)[:, None]
        table = torch.full((seqs, table_pages), -1, dtype=torch.int32, device=dev)
        table[mine] = order[: sum(held)]
        free = torch.full((pages,), -1, dtype=torch.int32, device=dev)
        free[: pages - sum(held)] = order[sum(held) :]
        s.update(table=table, table_pages=table_pages, pages=pages, held=ints(held), lengths=ints(lengths), counts=ints(counts), free=free)
        s.update(free_count=ints([pages - sum(held)]), slots=torch.zeros(seqs, tokens, dtype=torch.int32, device=dev))
        s.update(taken=ints([0] * seqs), freed=ints([0] * seqs))
        if own:
            from nebula_b200 import lib

            s["lib"] = lib
            s["pool"] = lib.PagePool(table.data_ptr(), s["held"].data_ptr(), free.data_ptr(), s["free_count"].data_ptr(), pages, page, table_pages)
        return s
    rows, vocab, per = case["rows"], case["vocab"], case.get("tokens", 1)
    logits = 2.0 * torch.randn(rows, vocab, device=dev, generator=gen)
    peak = torch.randint(vocab, (rows, 6), device=dev, generator=gen)
    logits.scatter_add_(1, peak, 6.0 + 6.0 * torch.rand(rows, 6, device=dev, generator=gen))
    logits.scatter_(1, torch.randint(vocab, (rows, 8), device=dev, generator=gen), -math.inf)  # tokens that a grammar forbids
    asked = [SETTINGS[case["asked"] if case["asked"] >= 0 else rng.randrange(len(SETTINGS))] for _ in range(rows // per)]
    s.update(per=per, logits=logits.bfloat16().float() if case["rounded"] else logits)
    s.update(temperature=floats([a[0] for a in asked]), top_k=ints([a[1] for a in asked]), top_p=floats([a[2] for a in asked]), min_p=floats([a[3] for a in asked]))
    if case["op"] == "sample":
        s.update(uniforms=torch.rand(rows, device=dev, generator=gen), token=ints([0] * rows))
    else:
        s["out"] = torch.zeros_like(logits)
    if own:
        from nebula_b200 import lib

        s["lib"] = lib
    return s


def run(s):
    return (run_own if own else run_plain)[s["op"]](s)


# ---- the library's operators ---------------------------------------------


def ptr(t):
    return None if t is None else t.data_ptr()


def own_attention(s):
    s["lib"].call("shared_attention", ptr(s["out"]), ptr(s["q"]), ctypes.byref(s["cache"]), 0, ptr(s["shared_at"]), ptr(s["tree_mask"]),
                  s["scale"], s["seqs"], s["tokens"], s["hq"], s["workspace"].p)
    return s["out"]


def own_sample(s):
    s["lib"].call("sample", ptr(s["token"]), ptr(s["logits"]), ptr(s["uniforms"]), ptr(s["temperature"]), ptr(s["top_k"]), ptr(s["top_p"]),
                  ptr(s["min_p"]), s["per"], s["rows"], s["vocab"])
    return s["token"]


def own_truncate(s):
    s["lib"].call("truncate_logits", ptr(s["out"]), ptr(s["logits"]), ptr(s["temperature"]), ptr(s["top_k"]), ptr(s["top_p"]), ptr(s["min_p"]),
                  s["per"], s["rows"], s["vocab"])
    return s["out"]


def own_pages(s):
    pool = ctypes.byref(s["pool"])
    s["lib"].call("pages_release", pool, ptr(s["freed"]), ptr(s["lengths"]), 0, s["seqs"])
    s["lib"].call("pages_reserve", pool, ptr(s["slots"]), ptr(s["taken"]), ptr(s["lengths"]), ptr(s["counts"]), s["seqs"], s["tokens"])
    return pages_state(s)


def pages_state(s):
    return {k: s[k] for k in ("table", "held", "free", "free_count", "slots", "taken", "freed")}


# ---- the plain forms -------------------------------------------------------


def plain_attention(s):
    """Scores of all rows against what is shared in one product, against their own sequence's positions in another."""
    seqs, tokens, hq, hkv, d, page, shared = s["seqs"], s["tokens"], s["hq"], s["hkv"], s["d"], s["page"], s["shared"]
    heads, common = hq // hkv, shared // page
    q = s["q"].view(seqs, tokens, hkv, heads, d)
    k1 = s["k"][s["table"][0, :common].long()].view(-1, hkv, d).float()  # [shared][hkv][d]
    v1 = s["v"][s["table"][0, :common].long()].view(-1, hkv, d).float()
    k2 = s["k"][s["table"][:, common:].long()].view(seqs, -1, hkv, d).permute(0, 2, 3, 1).float()  # [seqs][hkv][d][n]
    v2 = s["v"][s["table"][:, common:].long()].view(seqs, -1, hkv, d).permute(0, 2, 1, 3).float()
    far = q.permute(2, 0, 1, 3, 4).reshape(hkv, -1, d) @ k1.permute(1, 2, 0) * s["scale"]  # [hkv][seqs tokens heads][shared]
    near = (q.permute(0, 2, 1, 3, 4).reshape(seqs, hkv, -1, d) @ k2 * s["scale"]).view(seqs, hkv, tokens, heads, -1)
    near = near.masked_fill(~visible(s, near.shape[-1])[:, None, :, None, :], -math.inf)
    far = far.view(hkv, seqs, tokens, heads, shared)
    top = torch.maximum(far.amax(dim=-1), near.amax(dim=-1).permute(1, 0, 2, 3))[..., None]  # [hkv][seqs][tokens][heads][1]
    far = torch.exp(far - top)
    near = torch.exp(near - top.permute(1, 0, 2, 3, 4))
    total = far.sum(dim=-1) + near.sum(dim=-1).permute(1, 0, 2, 3)
    out = (far.view(hkv, -1, shared) @ v1.permute(1, 0, 2)).view(hkv, seqs, tokens, heads, d)
    out = out + (near.reshape(seqs, hkv, tokens * heads, -1) @ v2).view(seqs, hkv, tokens, heads, d).permute(1, 0, 2, 3, 4)
    return (out / total[..., None]).permute(1, 2, 0, 3, 4).reshape(-1, hq, d)


def visible(s, n):
    """[seqs][tokens][n]: which of its sequence's positions after the shared ones a row attends to."""
    pos = s["shared"] + torch.arange(n, device=s["q"].device)
    node = pos[None, :] - s["lengths"][:, None].long()  # [seqs][n]: which drafted token, or a committed one (< 0)
    i = torch.arange(s["tokens"], device=pos.device)
    if s["tree_mask"] is None:
        seen = node[:, None, :] <= i[None, :, None]
    else:
        seen = (s["tree_mask"][:, :, None] >> node.clamp(0, s["tokens"] - 1)[:, None, :]) & 1 == 1
    return (node < 0)[:, None, :] | (seen & (node < s["tokens"])[:, None, :])


def kept(s):
    """What may be sampled, and its weights relative to the largest. In 64 bits: sums of up to 200,000 weights are compared
    with borders that lie between two of them."""
    per = lambda v: v.repeat_interleave(s["per"])[:, None]  # noqa: E731
    t, k, p, least = per(s["temperature"]).double(), per(s["top_k"]), per(s["top_p"]).double(), per(s["min_p"]).double()
    x, order = torch.sort(s["logits"], dim=1, descending=True, stable=True)
    rank = torch.arange(x.shape[1], device=x.device)
    weight = torch.exp((x.double() - x[:, :1].double()) / torch.where(t > 0, t, torch.ones_like(t)))
    stay = (x > -math.inf) & ((k <= 0) | (rank < k)) & ((t > 0) | (rank == 0))
    weight = torch.where(stay, weight, torch.zeros_like(weight))
    run_sum = torch.cumsum(weight, dim=1)
    stay = stay & ((p >= 1) | (run_sum - weight < p * run_sum[:, -1:]) | (rank == 0)) & ((weight >= least) | (rank == 0))
    back = torch.zeros_like(stay).scatter_(1, order, stay)
    return back, torch.zeros_like(weight).scatter_(1, order, torch.where(stay, weight, torch.zeros_like(weight)))


def plain_sample(s):
    run_sum = torch.cumsum(kept(s)[1], dim=1)
    aim = s["uniforms"][:, None].double() * run_sum[:, -1:]
    return (run_sum <= aim).sum(dim=1).clamp(max=s["vocab"] - 1).int()


def plain_truncate(s):
    return torch.where(kept(s)[0], s["logits"], torch.full_like(s["logits"], -math.inf))


def plain_pages(s):
    seqs, tokens, page = s["seqs"], s["tokens"], s["page"]
    table, held, lengths, counts = s["table"], s["held"].long(), s["lengths"].long(), s["counts"].long()
    place = torch.arange(s["table_pages"], device=table.device)
    # pages past the committed positions go back, the first of them on top
    stay = torch.div(lengths + page - 1, page, rounding_mode="floor")
    gone = (place >= stay[:, None]) & (place < held[:, None])
    order = torch.cumsum(gone.view(-1), dim=0)
    top = s["free_count"].long() + order[-1]
    stack = torch.cat([s["free"], s["free"][:1]])  # the last place takes what is not given back
    stack[torch.where(gone.view(-1), top - order, torch.full_like(order, s["pages"]))] = table.view(-1)
    s["freed"].copy_(gone.sum(dim=1))
    held = torch.minimum(held, stay)
    # pages for the new positions, as long as there are enough for all sequences up to this one
    need = (torch.div(lengths + counts + page - 1, page, rounding_mode="floor") - held).clamp(min=0)
    upto = torch.cumsum(need, dim=0)
    given = (upto <= top) | (need == 0)
    need = torch.where(given, need, torch.zeros_like(need))
    new = (place >= held[:, None]) & (place < (held + need)[:, None])
    nth = (upto - need)[:, None] + place - held[:, None]
    table.copy_(torch.where(new, stack[(top - 1 - nth).clamp(0, s["pages"])], table))
    s["held"].copy_(held + need)
    s["free"].copy_(stack[:-1])
    s["free_count"].copy_(top - need.sum())
    s["taken"].copy_(torch.where(given, need, torch.full_like(need, -2)))
    i = torch.arange(tokens, device=table.device)
    at = lengths[:, None] + i
    row = torch.gather(table.long(), 1, torch.div(at, page, rounding_mode="floor").clamp(max=s["table_pages"] - 1)) * page + at % page
    s["slots"].copy_(torch.where((i < counts[:, None]) & given[:, None], row, torch.full_like(row, -1)))
    return pages_state(s)


run_own = {"attention": own_attention, "sample": own_sample, "truncate": own_truncate, "pages": own_pages}
run_plain = {"attention": plain_attention, "sample": plain_sample, "truncate": plain_truncate, "pages": plain_pages}


# ---- the definitions, in 64 bits -------------------------------------------


def exact(case, seed):
    if case["op"] == "pages":
        return exact_pages(prepare(case, seed))
    s = prepare(case, seed)
    if case["op"] == "attention":
        out = torch.zeros(s["seqs"], s["tokens"], s["hq"], s["d"], dtype=torch.float64, device="cuda")
        q, t = s["q"].double().view(out.shape), s["tokens"]
        for b, length in enumerate(s["lengths"].tolist()):
            n = length + t
            keys = s["k"][s["table"][b].long()].view(-1, s["hkv"], s["d"])[:n].double()
            vals = s["v"][s["table"][b].long()].view(-1, s["hkv"], s["d"])[:n].double()
            bias = torch.zeros(t, n, dtype=torch.float64, device="cuda")
            for i in range(t):
                m = (2 << i) - 1 if s["tree_mask"] is None else int(s["tree_mask"][b, i])
                hidden = [length + j for j in range(t) if not m >> j & 1]
                bias[i, hidden] = -math.inf
            for h in range(s["hq"]):
                g = h // (s["hq"] // s["hkv"])
                out[b, :, h] = torch.softmax(q[b, :, h] @ keys[:, g].T * s["scale"] + bias, dim=1) @ vals[:, g]
        return out.view(-1, s["hq"], s["d"])
    tokens, rows = [], []
    for r in range(case["rows"]):
        x = s["logits"][r].double()
        t, k, p, least = (float(s[n][r // s["per"]]) for n in ("temperature", "top_k", "top_p", "min_p"))
        # the tokens that may be sampled at all, best first and the lowest index of equals
        best = torch.nonzero(torch.isfinite(x))[:, 0]
        best = best[torch.argsort(-x[best], stable=True)]
        if t == 0:
            best, t = best[:1], 1.0
        elif k > 0:
            best = best[: int(k)]
        prob = torch.softmax(x[best] / t, dim=0)
        if p < 1:
            above = torch.cat([torch.zeros(1, dtype=torch.float64, device="cuda"), torch.cumsum(prob, dim=0)[:-1]])
            best = best[: max(1, int((above < p).sum()))]
            prob = prob[: len(best)]
        best = best[: max(1, int((prob >= least * prob[0]).sum()))]
        mine = torch.zeros_like(x)
        mine[best] = prob[: len(best)]
        if case["op"] == "sample":
            upto = torch.cumsum(mine, dim=0)
            tokens.append(min(case["vocab"] - 1, int((upto <= float(s["uniforms"][r]) * float(upto[-1])).sum())))
        else:
            row = torch.full_like(x, -math.inf)
            row[best] = x[best]
            rows.append(row.float())
    return torch.tensor(tokens, dtype=torch.int32) if case["op"] == "sample" else torch.stack(rows)


def exact_pages(s):
    """One sequence after the other, with a list as the stack."""
    table, held, free = s["table"].tolist(), s["held"].tolist(), s["free"].tolist()
    stack, lengths, counts, page = free[: int(s["free_count"])], s["lengths"].tolist(), s["counts"].tolist(), s["page"]
    freed, taken, slots, back = [], [], [], []
    for b in range(s["seqs"]):
        stay = min(held[b], -(-lengths[b] // page))
        back += table[b][stay : held[b]]
        freed.append(held[b] - stay)
        held[b] = stay
    stack += back[::-1]
    seen, short = len(stack), False
    free[:seen] = stack
    for b in range(s["seqs"]):
        need = max(0, -(-(lengths[b] + counts[b]) // page) - held[b])
        short = short or need > len(stack)
        if short and need:
            taken.append(-2)
            slots.append([-1] * s["tokens"])
            continue
        for _ in range(need):
            table[b][held[b]] = stack.pop()
            held[b] += 1
        taken.append(need)
        at = range(lengths[b], lengths[b] + counts[b])
        slots.append([table[b][a // page] * page + a % page for a in at] + [-1] * (s["tokens"] - counts[b]))
    ints = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return {"table": ints(table), "held": ints(held), "free": ints(free), "free_count": ints([len(stack)]), "slots": ints(slots),
            "taken": ints(taken), "freed": ints(freed)}
