"""Cases of the speculative-verify operators: the query/key preparation that writes the paged cache, tree attention over
that cache, the acceptance of drafted tokens, and the commit of the accepted ones.

Each case names an operator and its sizes; `run` makes one pass, in plain torch operations or through the library."""
import ctypes
import math
import random

import torch

own = False

# (query heads, key/value heads, values per head, rotated values): the heads of the served model (24/2/256, 64 of them
# rotated), and generic ones.
HEADS = {"24/2/256": (24, 2, 256, 64), "32/8/128": (32, 8, 128, 128), "16/4/64": (16, 4, 64, 64), "10/10/128": (10, 10, 128, 32)}
EPS = 1e-6


def listed():
    return [
        # one token of one user a few words into a conversation: latency only
        {"name": "attn decode short", "op": "attention", "heads": "24/2/256", "seqs": 1, "tokens": 1, "length": 33, "page": 16, "tree": False},
        # the verify batch of this framework (17 rows) as a tree, in an ordinary conversation
        {"name": "attn verify 4k", "op": "attention", "heads": "24/2/256", "seqs": 1, "tokens": 17, "length": 4097, "page": 64, "tree": True},
        # single tokens of several users with contexts of all lengths
        {"name": "attn decode batch", "op": "attention", "heads": "32/8/128", "seqs": 16, "tokens": 1, "length": 8191, "page": 16, "tree": False},
        # short chains of several users, small heads
        {"name": "attn chain batch", "op": "attention", "heads": "16/4/64", "seqs": 5, "tokens": 5, "length": 3000, "page": 32, "tree": False},
        # the longest context that the served model takes (98,304), full verify batch
        {"name": "attn verify 98k", "op": "attention", "heads": "24/2/256", "seqs": 1, "tokens": 17, "length": 98287, "page": 64, "tree": True},
        # query/key preparation of one verify batch
        {"name": "prep verify", "op": "prepare", "heads": "24/2/256", "seqs": 1, "tokens": 17, "length": 700, "page": 64, "tree": True},
        # the same for many users at once
        {"name": "prep batch", "op": "prepare", "heads": "24/2/256", "seqs": 96, "tokens": 17, "length": 45, "page": 16, "tree": True},
        # one verify batch, drafted tokens taken as they are (the draft's best)
        {"name": "verify tree", "op": "verify", "seqs": 1, "tokens": 17, "vocab": 131072, "temperature": 0.8, "sampled": False},
        # short sampled chains, an odd vocabulary
        {"name": "verify sampled", "op": "verify", "seqs": 7, "tokens": 6, "vocab": 50001, "temperature": 1.0, "sampled": True},
        # many users with full verify batches
        {"name": "verify batch", "op": "verify", "seqs": 12, "tokens": 17, "vocab": 131072, "temperature": 0.7, "sampled": True},
        # the accepted nodes of one user in the twelve attention layers of the served model
        {"name": "commit one", "op": "commit", "heads": "24/2/256", "seqs": 1, "tokens": 17, "length": 1000, "page": 64, "layers": 12},
        # many users
        {"name": "commit batch", "op": "commit", "heads": "32/8/128", "seqs": 48, "tokens": 32, "length": 150, "page": 16, "layers": 24},
    ]


def spread(rng, low, high):
    """A whole number between low and high, spread over the logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "prepare", "verify", "verify", "commit"])
    if op == "verify":
        sampled = rng.random() < 0.5
        seqs, tokens = spread(rng, 1, 16), spread(rng, 1, 24)
        vocab = spread(rng, 1000, min(200000, 12 * 17 * 131072 // (seqs * tokens)))
        return {"op": op, "seqs": seqs, "tokens": tokens, "vocab": vocab, "temperature": rng.choice([0.0, 0.6, 0.9, 1.0]), "sampled": sampled}
    heads = rng.choice(list(HEADS))
    hq, hkv, d, _ = HEADS[heads]
    page = rng.choice([16, 32, 64, 128])
    if op == "prepare":
        return {"op": op, "heads": heads, "seqs": spread(rng, 1, 64), "tokens": spread(rng, 1, 24), "length": spread(rng, 1, 64), "page": page, "tree": rng.random() < 0.5}
    if op == "commit":
        return {"op": op, "heads": heads, "seqs": spread(rng, 1, 32), "tokens": spread(rng, 4, 32), "length": spread(rng, 1, 300), "page": page, "layers": spread(rng, 1, 16)}
    seqs, tokens = spread(rng, 1, 32), spread(rng, 1, 33)
    most = min(98304 * 17 * 24 * 256 // (seqs * tokens * hq * d), 98304 * 2 * 256 // (seqs * hkv * d))
    length = spread(rng, 1, max(1, min(98304, most) - tokens))
    return {"op": op, "heads": heads, "seqs": seqs, "tokens": tokens, "length": length, "page": page, "tree": rng.random() < 0.6}


def work(case):
    if case["op"] == "verify":
        rows = case["seqs"] * case["tokens"] + (case["seqs"] if case["sampled"] else 0)
        return {"bytes": rows * case["vocab"] * 4.0, "flops": rows * case["vocab"] * 4.0}
    hq, hkv, d, _ = HEADS[case["heads"]]
    rows = case["seqs"] * case["tokens"]
    if case["op"] == "attention":
        n = sum(case_lengths(case)) + rows
        seen = sum(case["tokens"] * (x + case["tokens"]) for x in case_lengths(case))
        return {"bytes": n * hkv * d * 4.0 + rows * hq * d * 8.0, "flops": 4.0 * seen * hq * d}
    if case["op"] == "prepare":
        return {"bytes": rows * d * (8.0 * hq + 12.0 * hkv), "flops": rows * d * (hq + hkv) * 6.0}
    moved = case["seqs"] * (case["tokens"] // 2)
    return {"bytes": case["layers"] * moved * hkv * d * 8.0, "flops": 0.0}


def case_lengths(case):
    """The committed tokens of each sequence: from short ones up to case["length"]."""
    return [case["length"] * (s + 1) // case["seqs"] for s in range(case["seqs"])]


def make_tree(rng, tokens, tree):
    """The parent of each node: a chain, or a tree of mostly small fan-out (node 0 is the root)."""
    parents, fan = [-1], [0]
    for i in range(1, tokens):
        p = i - 1
        if tree:
            p = max(rng.randrange(i), rng.randrange(i))
            while fan[p] >= 6:
                p = (p + 1) % i
        parents.append(p)
        fan[p] += 1
        fan.append(0)
    return parents


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    rng = random.Random(seed)
    s = dict(case, rows=case["seqs"] * case["tokens"])
    seqs, tokens = case["seqs"], case["tokens"]
    randn = lambda *shape: torch.randn(*shape, device=dev, generator=gen)  # noqa: E731
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731

    parents = [make_tree(rng, tokens, case.get("tree", not case.get("sampled", False))) for _ in range(seqs)]
    if case["op"] == "verify":
        vocab = case["vocab"]
        logits = randn(seqs, tokens, vocab) * 2.0
        peak = torch.randint(vocab, (seqs, tokens, 6), device=dev, generator=gen)
        logits.scatter_add_(2, peak, 6.0 + 6.0 * torch.rand(seqs, tokens, 6, device=dev, generator=gen))
        banned = torch.randint(vocab, (seqs, tokens, 8), device=dev, generator=gen)  # tokens that a grammar forbids
        logits.scatter_(2, banned, -math.inf)
        above = ints([[max(p, 0) for p in ps] for ps in parents]).long()
        guess = torch.gather(logits, 1, above[:, :, None].expand(-1, -1, vocab)) + 0.7 * randn(seqs, tokens, vocab)
        s["probs"] = None
        if case["sampled"]:
            s["probs"] = torch.softmax(guess / max(case["temperature"], 0.5), dim=2)
            draft = torch.multinomial(s["probs"].view(-1, vocab), 1, generator=gen).view(seqs, tokens)
        else:  # siblings are the draft's best tokens, each another one
            rank = ints([[ps[:i].count(ps[i]) for i in range(tokens)] for ps in parents]).long()
            best = torch.topk(torch.gather(guess, 1, above[:, :, None].expand(-1, -1, vocab)), 8, dim=2).indices
            draft = torch.gather(best, 2, rank[:, :, None])[:, :, 0]
        s.update(logits=logits, draft=draft.int().contiguous(), parents=ints(parents),
                 uniforms=torch.rand(seqs, tokens, device=dev, generator=gen))
        s.update(path=ints([[0] * tokens] * seqs), accepted=ints([0] * seqs), next=ints([0] * seqs))
    else:
        hq, hkv, d, rotary = HEADS[case["heads"]]
        page, lengths, layers = case["page"], case_lengths(case), case.get("layers", 1)
        table_pages = -(-(max(lengths) + tokens) // page)
        pages = seqs * table_pages + 3
        order = torch.randperm(pages, device=dev, generator=gen)[: seqs * table_pages]
        s.update(hq=hq, hkv=hkv, d=d, rotary=rotary, table_pages=table_pages, pages=pages, layers=layers, longest=max(lengths) + tokens)
        s.update(table=order.int().view(seqs, table_pages).contiguous(), lengths=ints(lengths))
        shape = (layers, pages, page, hkv, d)
        s["k"] = torch.empty(shape, dtype=torch.float16, device=dev).normal_(generator=gen)
        s["v"] = torch.empty(shape, dtype=torch.float16, device=dev).normal_(generator=gen)
        if case["op"] == "attention":
            s["q"] = 1.5 * randn(s["rows"], hq, d)
            s["out"] = torch.zeros(s["rows"], hq, d, device=dev)
            s["scale"] = 1.0 / math.sqrt(d)
            s["tree_mask"] = None
            if case["tree"]:
                masks = []
                for ps in parents:
                    m = []
                    for i, p in enumerate(ps):
                        m.append((m[p] if i else 0) | 1 << i)
                    masks.append(m)
                s["tree_mask"] = torch.tensor(masks, dtype=torch.int64, device=dev)
        elif case["op"] == "prepare":
            s["qkv"] = randn(s["rows"], (hq + 2 * hkv) * d)  # one fused projection's rows
            s["q_weight"], s["k_weight"] = 1.0 + 0.1 * randn(d), 1.0 + 0.1 * randn(d)
            depth = []
            for ps in parents:
                dep = []
                for i, p in enumerate(ps):
                    dep.append(dep[p] + 1 if i else 0)
                depth.append(dep)
            s["depth"] = ints(depth) if case["tree"] else None
            s["positions"] = page * table_pages
            angle = torch.arange(s["positions"], device=dev, dtype=torch.float64)[:, None] * 1e6 ** (
                -torch.arange(rotary // 2, device=dev, dtype=torch.float64) * 2 / rotary)
            s["rope"] = torch.stack([angle.cos(), angle.sin()], dim=2).float().contiguous()
            s["q_out"] = torch.zeros(s["rows"], hq, d, device=dev)
        else:
            moved = tokens // 2  # accepted drafts, none of them in place
            path = [[0] + sorted(rng.sample(range(2, tokens), min(moved, tokens - 2))) for _ in range(seqs)]
            s["path"] = ints([p + [-1] * (tokens - len(p)) for p in path])
            s["accepted"] = ints([len(p) - 1 for p in path])
            s["new_lengths"] = ints([0] * seqs)
    if own:
        from nebula_b200 import lib

        s["lib"] = lib
        if case["op"] == "verify":
            s["workspace"] = lib.verify_workspace(seqs, tokens, case["vocab"])
        else:
            s["cache"] = lib.KvCache(s["k"].data_ptr(), s["v"].data_ptr(), s["table"].data_ptr(), s["lengths"].data_ptr(),
                                     s["k"][0].numel() * 2, s["layers"], s["pages"], case["page"], s["table_pages"], s["hkv"], s["d"])
        if case["op"] == "attention":
            s["workspace"] = lib.attention_workspace(seqs, tokens, s["hq"], s["hkv"], s["d"])
    return s


def run(s):
    return (run_own if own else run_plain)[s["op"]](s)


# ---- the library's operators ---------------------------------------------


def ptr(t):
    return None if t is None else t.data_ptr()


def own_attention(s):
    s["lib"].call("tree_attention", ptr(s["out"]), ptr(s["q"]), ctypes.byref(s["cache"]), 0, ptr(s["tree_mask"]), s["scale"],
                  s["seqs"], s["tokens"], s["hq"], s["workspace"].p)
    return s["out"]


def own_prepare(s):
    x, width, d = s["qkv"].data_ptr(), s["qkv"].shape[1], s["d"]
    s["lib"].call("qk_norm_rope", ptr(s["q_out"]), ctypes.byref(s["cache"]), 0, x, width, x + 4 * s["hq"] * d, width,
                  x + 4 * (s["hq"] + s["hkv"]) * d, width, ptr(s["q_weight"]), ptr(s["k_weight"]), EPS, ptr(s["rope"]),
                  s["positions"], s["rotary"], ptr(s["depth"]), s["seqs"], s["tokens"], s["hq"])
    return {"q": s["q_out"], "k": s["k"], "v": s["v"]}


def own_verify(s):
    s["lib"].call("verify_tree", ptr(s["path"]), ptr(s["accepted"]), ptr(s["next"]), ptr(s["logits"]), ptr(s["draft"]),
                  ptr(s["parents"]), ptr(s["probs"]), ptr(s["uniforms"]), s["temperature"], s["seqs"], s["tokens"], s["vocab"],
                  s["workspace"].p)
    return {"path": s["path"], "accepted": s["accepted"], "next": s["next"]}


def own_commit(s):
    s["lib"].call("cache_commit", ctypes.byref(s["cache"]), ptr(s["new_lengths"]), ptr(s["path"]), ptr(s["accepted"]),
                  s["seqs"], s["tokens"])
    return {"k": s["k"], "v": s["v"], "lengths": s["new_lengths"]}


# ---- the plain forms -------------------------------------------------------


def slots(s, positions):
    """Rows of the cache pool at `positions` [seqs][n] of each sequence."""
    page = torch.gather(s["table"].long(), 1, torch.div(positions, s["page"], rounding_mode="floor"))
    return page * s["page"] + positions % s["page"]


def visible(s):
    """[seqs][tokens][longest]: what each drafted token attends to."""
    pos = torch.arange(s["longest"], device=s["q"].device)
    node = pos[None, :] - s["lengths"][:, None].long()  # [seqs][n]: which drafted token, or a committed one (< 0)
    i = torch.arange(s["tokens"], device=pos.device)
    if s["tree_mask"] is None:
        seen = node[:, None, :] <= i[None, :, None]
    else:
        seen = (s["tree_mask"][:, :, None] >> node.clamp(0, s["tokens"] - 1)[:, None, :]) & 1 == 1
    return (node < 0)[:, None, :] | (seen & (node < s["tokens"])[:, None, :])


def plain_attention(s):
    seqs, tokens, hq, hkv, d, n = s["seqs"], s["tokens"], s["hq"], s["hkv"], s["d"], s["longest"]
    rows = slots(s, torch.arange(n, device=s["q"].device).expand(seqs, n))
    k = s["k"].view(-1, hkv, d)[rows].permute(0, 2, 3, 1).float()  # [seqs][hkv][d][n]
    v = s["v"].view(-1, hkv, d)[rows].permute(0, 2, 1, 3).float()
    q = s["q"].view(seqs, tokens, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(seqs, hkv, -1, d)
    score = (q @ k * s["scale"]).view(seqs, hkv, tokens, hq // hkv, n)
    score = score.masked_fill(~visible(s)[:, None, :, None, :], -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    total = p.sum(dim=-1, keepdim=True)
    out = (p.reshape(seqs, hkv, -1, n) @ v).view(seqs, hkv, tokens, hq // hkv, d)
    out = out / torch.where(total > 0, total, torch.ones_like(total))
    return out.permute(0, 2, 1, 3, 4).reshape(-1, hq, d)


def plain_prepare(s):
    seqs, tokens, hq, hkv, d, half = s["seqs"], s["tokens"], s["hq"], s["hkv"], s["d"], s["rotary"] // 2
    x = s["qkv"].view(s["rows"], hq + 2 * hkv, d)
    qk, v = x[:, : hq + hkv], x[:, hq + hkv:]
    i = torch.arange(tokens, device=x.device)
    y = qk * torch.rsqrt((qk * qk).mean(dim=2, keepdim=True) + EPS)
    y = torch.cat([y[:, :hq] * s["q_weight"], y[:, hq:] * s["k_weight"]], dim=1)
    depth = i.expand(seqs, tokens) if s["depth"] is None else s["depth"]
    turn = s["rope"][(s["lengths"][:, None] + depth).long().view(-1)][:, None]  # [rows][1][half][2]
    cos, sin, a, b = turn[..., 0], turn[..., 1], y[..., :half], y[..., half : 2 * half]
    y = torch.cat([a * cos - b * sin, b * cos + a * sin, y[..., 2 * half:]], dim=2)
    at = slots(s, s["lengths"][:, None].long() + i).view(-1)
    s["k"].view(-1, hkv, d)[at] = y[:, hq:].half()
    s["v"].view(-1, hkv, d)[at] = v.half()
    return {"q": y[:, :hq].contiguous(), "k": s["k"], "v": s["v"]}


def plain_verify(s):
    """Weights relative to the largest power of two of their row. Only sums over a row are held in 64 bits: the outputs are
    whole numbers, and they have to come out the same whatever the order of the sums."""
    seqs, tokens, vocab, logits = s["seqs"], s["tokens"], s["vocab"], s["logits"]
    if s["temperature"] > 0:
        t = logits * (1.0 / s["temperature"] * 1.4426950408889634)
        power = torch.floor(t)
        rel = torch.where(torch.isfinite(t), power - power.amax(dim=2, keepdim=True), torch.full_like(t, -999.0)).clamp(min=-127)
        weight = torch.exp2(torch.where(torch.isfinite(t), t - power, torch.zeros_like(t))) * ((rel.int() + 127) << 23).view(torch.float32)
    else:
        weight = torch.zeros_like(logits).scatter_(2, logits.argmax(dim=2, keepdim=True), 1.0)
    total = weight.double().sum(dim=2)  # [seqs][tokens]
    node = torch.arange(tokens, device=logits.device)
    parent = s["parents"].long()
    above = parent.clamp(min=0)
    draft = s["draft"].long()
    mine = torch.gather(weight.view(seqs, -1), 1, above * vocab + draft)  # the target's weight of each drafted token
    elder = (parent[:, :, None] == parent[:, None, :]) & (node[:, None] > node[None, :])  # [seqs][node][elder sibling]
    child = (node > 0)[None, :] & (parent >= 0)
    if s["probs"] is None:
        left = torch.gather(total, 1, above) - (elder * mine[:, None, :].double()).sum(dim=2)
        passed = child & (s["uniforms"].double() * left < mine.double())
    else:
        guess = torch.gather(s["probs"], 2, draft[:, :, None])[:, :, 0]
        passed = child & (s["uniforms"] * guess < mine / torch.gather(total, 1, above).float())
    chosen = passed & ~(elder & passed[:, None, :]).any(dim=2)
    up = (parent[:, :, None] == node) & child[:, :, None]
    lineage = torch.linalg.matrix_power(up.float() + torch.eye(tokens, device=node.device), tokens) > 0
    on = ~(lineage & ~(chosen | (node == 0))[:, None, :]).any(dim=2)  # the node and all above it are accepted
    last = (on * node).amax(dim=1)
    path = torch.sort(torch.where(on, node, node + tokens), dim=1).values
    accepted = on.sum(dim=1) - 1
    row = torch.gather(weight, 1, last[:, None, None].expand(-1, 1, vocab))[:, 0]
    under = (parent == last[:, None]) & child  # its children: all of them refused
    if s["probs"] is None:
        row = refused(row, under, draft).double()
    else:
        target = row / torch.gather(total, 1, last[:, None]).float()
        first = under.int().argmax(dim=1)
        rest = (target - torch.gather(s["probs"], 1, first[:, None, None].expand(-1, 1, vocab))[:, 0]).clamp(min=0).double()
        keep = under.any(dim=1) & (rest.sum(dim=1) > 0)
        row = torch.where(keep[:, None], rest, target.double())
    run_sum = torch.cumsum(row, dim=1)
    aim = s["uniforms"][:, :1].double() * run_sum[:, -1:]
    pick = (run_sum <= aim).sum(dim=1).clamp(max=vocab - 1)
    return {"path": torch.where(path < tokens, path, -torch.ones_like(path)).int(), "accepted": accepted.int(), "next": pick.int()}


def refused(row, under, draft):
    """`row` without the refused children's tokens."""
    gone = torch.zeros_like(row).scatter_add_(1, draft, under.float())
    return torch.where(gone > 0, torch.zeros_like(row), row)


def plain_commit(s):
    seqs, tokens, hkv, d = s["seqs"], s["tokens"], s["hkv"], s["d"]
    i = torch.arange(tokens, device=s["path"].device)
    live = i <= s["accepted"][:, None]
    base = s["lengths"][:, None].long()
    source = slots(s, base + torch.where(live, s["path"].long(), i))
    goal = slots(s, base + i)
    for pool in (s["k"], s["v"]):
        flat = pool.view(s["layers"], -1, hkv, d)
        flat[:, goal] = torch.where(live[None, :, :, None, None], flat[:, source], flat[:, goal])
    s["new_lengths"].copy_(s["lengths"] + s["accepted"] + 1)
    return {"k": s["k"], "v": s["v"], "lengths": s["new_lengths"]}


run_own = {"attention": own_attention, "prepare": own_prepare, "verify": own_verify, "commit": own_commit}
run_plain = {"attention": plain_attention, "prepare": plain_prepare, "verify": plain_verify, "commit": plain_commit}


# ---- the definitions, in 64 bits -------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        out = torch.zeros(s["seqs"], s["tokens"], s["hq"], s["d"], dtype=torch.float64, device="cuda")
        q = s["q"].double().view(s["seqs"], s["tokens"], s["hq"], s["d"])
        for b, length in enumerate(case_lengths(case)):
            n, t = length + s["tokens"], s["tokens"]
            keys = s["k"][0][s["table"][b].long()].view(-1, s["hkv"], s["d"])[:n].double()
            vals = s["v"][0][s["table"][b].long()].view(-1, s["hkv"], s["d"])[:n].double()
            bias = torch.zeros(t, n, dtype=torch.float64, device="cuda")
            for i in range(t):
                m = (2 << i) - 1 if s["tree_mask"] is None else int(s["tree_mask"][b, i])
                for j in range(t):
                    if not m >> j & 1:
                        bias[i, length + j] = -math.inf
            for h in range(s["hq"]):
                g = h // (s["hq"] // s["hkv"])
                w = torch.softmax(q[b, :, h] @ keys[:, g].T * s["scale"] + bias, dim=1)
                out[b, :, h] = w @ vals[:, g]
        return out.view(-1, s["hq"], s["d"])
    if case["op"] == "prepare":
        hq, hkv, d, half = s["hq"], s["hkv"], s["d"], s["rotary"] // 2
        x = s["qkv"].double().view(s["seqs"], s["tokens"], hq + 2 * hkv, d)
        k, v = s["k"].double(), s["v"].double()
        q = torch.empty(s["seqs"], s["tokens"], hq, d, dtype=torch.float64, device="cuda")
        table, depth = s["table"].tolist(), s["depth"].tolist() if s["depth"] is not None else None
        for b, length in enumerate(case_lengths(case)):
            for i in range(s["tokens"]):
                heads = x[b, i, : hq + hkv]
                heads = heads / torch.sqrt(heads.pow(2).mean(dim=1, keepdim=True) + EPS)
                heads[:hq] *= s["q_weight"].double()
                heads[hq:] *= s["k_weight"].double()
                turn = s["rope"][length + (i if depth is None else depth[b][i])].double()
                pair = torch.complex(heads[:, :half], heads[:, half : 2 * half]) * torch.complex(turn[:, 0], turn[:, 1])
                heads[:, :half], heads[:, half : 2 * half] = pair.real, pair.imag
                page, at = table[b][(length + i) // s["page"]], (length + i) % s["page"]
                q[b, i], k[0, page, at], v[0, page, at] = heads[:hq], heads[hq:], x[b, i, hq + hkv :]
        return {"q": q.view(-1, hq, d), "k": k, "v": v}
    if case["op"] == "commit":
        k, v = s["k"].double(), s["v"].double()
        new = s["lengths"].clone()
        table, path = s["table"].tolist(), s["path"].tolist()
        for b, length in enumerate(case_lengths(case)):
            at = lambda j: (table[b][(length + j) // s["page"]], (length + j) % s["page"])  # noqa: E731
            live = [j for j in path[b] if j >= 0]
            for pool in (k, v):
                held = [pool[:, at(j)[0], at(j)[1]].clone() for j in live]
                for i, row in enumerate(held):
                    pool[:, at(i)[0], at(i)[1]] = row
            new[b] = length + len(live)
        return {"k": k, "v": v, "lengths": new}
    # verify: the walk as it is defined, one node after the other
    path, accepted, nxt = [], [], []
    for b in range(s["seqs"]):
        parents, draft, u = s["parents"][b].tolist(), s["draft"][b].tolist(), s["uniforms"][b].double().tolist()
        at, trail = 0, [0]
        while True:
            row = s["logits"][b, at].double()
            if case["temperature"] > 0:
                p = torch.softmax(row / case["temperature"], dim=0)
            else:
                p = torch.zeros_like(row)
                p[int(row.argmax())] = 1.0
            to = None
            for c in [c for c in range(1, s["tokens"]) if parents[c] == at]:
                if s["probs"] is None:
                    if u[c] * float(p.sum()) < float(p[draft[c]]):
                        to = c
                        break
                    p[draft[c]] = 0.0
                else:
                    g = s["probs"][b, c].double()
                    if u[c] * float(g[draft[c]]) < float(p[draft[c]]):
                        to = c
                        break
                    rest = (p - g).clamp(min=0)
                    p = rest if float(rest.sum()) > 0 else p
            if to is None:
                break
            at = to
            trail.append(at)
        total = torch.cumsum(p, dim=0)
        path.append(trail + [-1] * (s["tokens"] - len(trail)))
        accepted.append(len(trail) - 1)
        nxt.append(min(s["vocab"] - 1, int((total <= u[0] * float(total[-1])).sum())))
    ints = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return {"path": ints(path), "accepted": ints(accepted), "next": ints(nxt)}
