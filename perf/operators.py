"""What is measured of the paged key-value cache's operators: attention of one new token over the
cache (with the attention weights that each position gathers), the cache's writes, and eviction by
gathered weight.

Sizes are those of the block-selection path next to them: 32 query heads over 2 kv heads of 128
(group 16), group 32, contexts up to 131072 tokens, and a decode batch of contexts between 4096 and
65536 tokens.  Head dim 64, fp16 and other groups are the operators' further types.
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # the first steps of a chat: one short sequence, where the launch is what counts
        dict(name="attend one short", op="attend", dtype="bf16", B=1, min_len=217, max_len=217, Hk=2, G=16, D=128,
             page=1, weights=False, empty=False),
        # a small server: a few ragged sequences, small heads, pages of 16, one slot of the batch unused
        dict(name="attend few ragged fp16", op="attend", dtype="fp16", B=7, min_len=1, max_len=2501, Hk=8, G=4, D=64,
             page=16, weights=False, empty=True),
        # one user at the longest context: all the work is along the length
        dict(name="attend one long", op="attend", dtype="bf16", B=1, min_len=131072, max_len=131072, Hk=2, G=16,
             D=128, page=1, weights=False, empty=False),
        # the decode batch's contexts, an eighth of its 512 sequences, slot by slot as the block table has them
        dict(name="attend decode batch", op="attend", dtype="bf16", B=64, min_len=4096, max_len=65536, Hk=2, G=16,
             D=128, page=1, weights=False, empty=False),
        # the same step while the weights for a later eviction are gathered, pages of one selection block
        dict(name="attend and weigh", op="attend", dtype="bf16", B=24, min_len=2048, max_len=32768, Hk=2, G=16,
             D=128, page=64, weights=True, empty=False),
        # 64 query heads on 2 kv heads: twice the arithmetic for each byte of the cache
        dict(name="attend group 32", op="attend", dtype="bf16", B=13, min_len=900, max_len=16384, Hk=2, G=32, D=128,
             page=16, weights=True, empty=True),
        # a decode step's writes: one token for each of 512 sequences
        dict(name="append decode step", op="append", dtype="bf16", B=512, tokens=512, context=40, Hk=2, D=128, page=1),
        # a chunk of prompts, ragged, into pages that end inside it
        dict(name="append prompts fp16", op="append", dtype="fp16", B=11, tokens=20011, context=333, Hk=8, D=64, page=16),
        # the longest prompt in one call
        dict(name="append long prompt", op="append", dtype="bf16", B=1, tokens=131072, context=0, Hk=2, D=128, page=1),
        # one sequence a little over its budget
        dict(name="evict one short", op="evict", B=1, min_len=1100, max_len=1100, Hk=2, page=1, budget=1024, init=4,
             local=64),
        # the longest context down to a quarter
        dict(name="evict one long", op="evict", B=1, min_len=131072, max_len=131072, Hk=2, page=1, budget=32768,
             init=64, local=4096),
        # a batch in pages of one selection block, some of it under its budget
        dict(name="evict batch of pages", op="evict", B=64, min_len=4096, max_len=65536, Hk=2, page=64, budget=256,
             init=1, local=2),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "evict"])
    page = rng.choice([1, 1, 2, 16, 64, 128])
    B = _log(rng, 1, 256)
    Hk = rng.choice([1, 2, 2, 4, 8])
    if op == "evict":
        most = min(131072, (1 << 23) // (B * Hk))
        max_len = _log(rng, 2, most)
        pages = -(-max_len // page)
        budget = rng.randint(1, pages + 1)
        local = rng.randint(1, max(1, budget // 2))
        init = rng.randint(0, min(8, budget - local))
        return dict(op=op, B=B, min_len=rng.randint(0, max_len), max_len=max_len, Hk=Hk, page=page, budget=budget,
                    init=init, local=local)
    dtype, D = rng.choice(["bf16", "bf16", "fp16"]), rng.choice([64, 128, 128])
    if op == "append":
        tokens = _log(rng, 1, 131072 * 256 // (Hk * D))
        return dict(op=op, dtype=dtype, B=min(B, tokens), tokens=tokens, context=rng.randint(0, 500), Hk=Hk, D=D,
                    page=page)
    G = rng.choice([1, 3, 4, 8, 16, 16, 32, 64])
    most = min(131072, (1 << 26) // (B * Hk * max(G, D // 8)))
    max_len = _log(rng, 1, most)
    return dict(op=op, dtype=dtype, B=B, min_len=rng.randint(1, max_len), max_len=max_len, Hk=Hk, G=G, D=D, page=page,
                weights=rng.random() < 0.4, empty=B > 1 and rng.random() < 0.4)


def _lengths(case):
    """The batch's lengths, before they are put in an order: evenly spaced, the longest among them."""
    n, lo, hi = case["B"], case["min_len"], case["max_len"]
    got = [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]
    if case.get("empty"):
        got[0] = 0
    return got


def _tokens(case):
    """New tokens of each sequence of an append, and the tokens that it has already."""
    n, t = case["B"], case["tokens"]
    if t == n:
        new = [1] * n
    else:
        cuts = [t * (i * (i + 1)) // (n * (n + 1)) for i in range(n + 1)]
        new = [b - a for a, b in zip(cuts, cuts[1:])]
    return new, [case["context"] * (i + 1) // n for i in range(n)]


def _table(lens, page, spare, g, dev):
    """Pages of a pool in any order, row by row, -1 past each row's own; and the pool's size in pages."""
    need = [-(-n // page) for n in lens]
    width, total = max(max(need), 1) + spare, sum(need) + 3
    own_ = torch.tensor(need, device=dev)
    used = torch.arange(width, device=dev)[None] < own_[:, None]
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device=dev)
    table[used] = torch.randperm(total, generator=g, device=dev)[:sum(need)].to(torch.int32)
    return table, total


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    page, Hk = case["page"], case["Hk"]

    def normal(dtype, *shape):
        x = torch.empty(shape, dtype=dtype, device=dev)
        return x.normal_(generator=g)

    s = {"case": dict(case)}
    if case["op"] == "append":
        new, had = _tokens(case)
        dt, D = _DT[case["dtype"]], case["D"]
        s["table"], pages = _table([a + b for a, b in zip(new, had)], page, 2, g, dev)
        s["bs"] = torch.repeat_interleave(torch.arange(len(new), device=dev), torch.tensor(new, device=dev)).to(torch.int32)
        start = torch.tensor([h - sum(new[:i]) for i, h in enumerate(had)], device=dev)
        # as get_block_table has it: token t sees token_pos_in_bs[t] positions, the last of them its own
        s["pos"] = (torch.arange(case["tokens"], device=dev) + start[s["bs"].long()] + 1).to(torch.int32)
        s["k"], s["v"] = normal(dt, case["tokens"], Hk, D), normal(dt, case["tokens"], Hk, D)
        s["k_cache"], s["v_cache"] = normal(dt, pages * page, Hk, D), normal(dt, pages * page, Hk, D)
        return s
    lens = _lengths(case)
    order = torch.randperm(len(lens), generator=g, device=dev)
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)[order]
    s["max_len"] = max(lens)
    table, pages = _table(lens, page, 0 if case["op"] == "evict" else 1, g, dev)
    s["table"] = table[order]
    width = table.shape[1] * page
    if case["op"] == "evict":
        # gathered weights: heavy-tailed, more at positions that have been read for longer, some never read at all
        w = torch.exp(2.0 * normal(torch.float32, len(lens), Hk, width))
        w *= torch.linspace(1.5, 0.05, width, device=dev)
        w *= torch.rand(w.shape, generator=g, device=dev) > 0.05
        s["weights"] = w * (torch.arange(width, device=dev)[None, None] < s["lens"][:, None, None])
        return s
    dt, D = _DT[case["dtype"]], case["D"]
    s["q"] = normal(dt, len(lens), Hk * case["G"], D)
    s["k_cache"], s["v_cache"] = normal(dt, pages * page, Hk, D), normal(dt, pages * page, Hk, D)
    if case["weights"]:
        s["weights"] = torch.rand((len(lens), Hk, width), generator=g, device=dev)
    return s


def run(state):
    return {"attend": _attend, "append": _append, "evict": _evict}[state["case"]["op"]](state)


def _attend(s):
    page = s["case"]["page"]
    if own:
        from unum_ops_b200 import paged_attention

        out, lse = paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], page_size=page,
                                   max_seqlen=s["max_len"], weights=s.get("weights"), return_lse=True)
        return {"out": out, "lse": lse, "weights": s["weights"]} if "weights" in s else {"out": out, "lse": lse}
    q, kc, vc, table, lens = s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"]
    (B, Hq, D), (n_tokens, Hk, _) = q.shape, kc.shape
    pos = torch.arange(s["max_len"], device=q.device)
    token = table[:, pos // page].long() * page + pos % page
    valid = (pos[None] < lens[:, None]) & (token >= 0) & (token < n_tokens)
    token = torch.where(valid, token, 0)
    qh = q.float().view(B, Hk, Hq // Hk, D)
    sc = torch.matmul(qh, kc[token].permute(0, 2, 3, 1).float()) * D ** -0.5
    sc = sc.masked_fill(~valid[:, None, None], -math.inf)
    m = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(m == -math.inf, 0.0, m))
    l = p.sum(-1, keepdim=True)
    lse = (m + torch.log(l)).view(B, Hq)
    p = torch.where(l > 0, p / l, 0.0)
    out = torch.matmul(p, vc[token].transpose(1, 2).float()).view(B, Hq, D).to(q.dtype)
    if "weights" not in s:
        return {"out": out, "lse": lse}
    s["weights"][:, :, :s["max_len"]] += p.sum(2)
    return {"out": out, "lse": lse, "weights": s["weights"]}


def _append(s):
    page = s["case"]["page"]
    if own:
        from unum_ops_b200 import append_cache

        append_cache(s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["bs"], s["pos"], page_size=page)
        return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    pos = s["pos"].long() - 1
    token = s["table"][s["bs"].long(), pos // page].long() * page + pos % page
    s["k_cache"][token] = s["k"]
    s["v_cache"][token] = s["v"]
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _evict(s):
    c = s["case"]
    page, budget, init, local = c["page"], c["budget"], c["init"], c["local"]
    table, lens, w = s["table"], s["lens"], s["weights"]
    if own:
        from unum_ops_b200 import evict_cache

        new, n, ww, gone = evict_cache(table, lens, w, budget=budget, init_pages=init, local_pages=local, page_size=page)
        return {"table": new, "lens": n, "weights": ww, "evicted": gone}
    (B, width), dev = table.shape, table.device
    Hk = w.shape[1]
    lens_ = lens.long()
    used = (lens_ + page - 1) // page
    e = torch.arange(width, device=dev)[None]
    held = torch.arange(width * page, device=dev)[None, None] < lens_[:, None, None]
    # a page's weight: the sum in 64 bits, rounded once
    score = torch.where(held, w, 0.0).double().view(B, Hk, width, page).sum((1, 3)).float()
    kept_anyway = (e < init) | (e >= (used - local)[:, None])
    score = torch.where(kept_anyway, math.inf, score)
    score = torch.where(e < used[:, None], score, -math.inf)
    order = torch.sort(score, dim=1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(1, order, e.expand(B, width))
    drop = (rank >= budget) & (e < used[:, None])
    # what stays closes up, in its order; -1 (0 for weights) fills the row's end
    first = torch.sort(drop.to(torch.int8), dim=1, stable=True).indices
    n_drop = drop.sum(1)
    new = torch.where(e < (width - n_drop)[:, None], table.gather(1, first), -1)
    gone = torch.where(e < n_drop[:, None], table.gather(1, torch.sort((~drop).to(torch.int8), dim=1, stable=True).indices), -1)
    n = lens_ - n_drop * page
    at = (first[:, :, None] * page + torch.arange(page, device=dev)).view(B, 1, width * page)
    ww = torch.where(torch.arange(width * page, device=dev)[None, None] < n[:, None, None],
                     w.gather(2, at.expand(B, Hk, width * page)), 0.0)
    return {"table": new, "lens": n.to(torch.int32), "weights": ww, "evicted": gone}


def work(case):
    Hk, page = case["Hk"], case["page"]
    if case["op"] == "append":
        t = case["tokens"]
        return {"bytes": t * (4 * Hk * case["D"] * 2 + 12), "flops": 0}
    lens = _lengths(case)
    total, B = sum(lens), len(lens)
    width = max(max(-(-n // page) for n in lens), 1)
    if case["op"] == "evict":
        return {"bytes": 4 * total * Hk + 4 * B * Hk * width * page + 4 * B * width * 3 + 8 * B, "flops": total * Hk}
    Hq, D = Hk * case["G"], case["D"]
    b = total * Hk * D * 4 + sum(-(-n // page) for n in lens) * 4 + B * Hq * (4 * D + 4) + 4 * B
    if case["weights"]:
        b += 8 * total * Hk
    return {"bytes": b, "flops": 4 * total * Hq * D}


def exact(case, seed):
    page, Hk = case["page"], case["Hk"]
    if case["op"] == "append":
        return None  # copies: nothing is computed
    s = prepare(case, seed)
    lens = s["lens"].tolist()
    if case["op"] == "evict":
        left = torch.zeros_like(s["weights"], dtype=torch.float64)
        for b, n in enumerate(lens):
            pages = -(-n // page)
            w = s["weights"][b, :, :n].double().cpu()
            weight = torch.nn.functional.pad(w, (0, pages * page - n)).view(Hk, pages, page).sum((0, 2)).float().tolist()
            must = {i for i in range(pages) if i < case["init"] or i >= pages - case["local"]}
            ranked = sorted(range(pages), key=lambda i: (i not in must, -weight[i], i))
            keep = sorted(ranked[:case["budget"]])
            at = torch.tensor([i * page + j for i in keep for j in range(min(page, n - i * page))], dtype=torch.long)
            left[b, :, :len(at)] = w[:, at].to(left.device)
        return {"weights": left}
    q, kc, vc = s["q"].double(), s["k_cache"], s["v_cache"]
    B, Hq, D = q.shape
    G = case["G"]
    out, lse = torch.zeros_like(q), torch.full((B, Hq), -math.inf, dtype=torch.float64, device=q.device)
    gathered = s["weights"].double() if "weights" in s else None
    for b, n in enumerate(lens):
        if n == 0:
            continue
        rows = (s["table"][b, :-(-n // page)].long()[:, None] * page + torch.arange(page, device=q.device)).reshape(-1)[:n]
        for h in range(Hk):
            k, v = kc[rows, h].double(), vc[rows, h].double()
            x = (q[b, h * G:(h + 1) * G] @ k.T) / math.sqrt(D)
            z = torch.logsumexp(x, 1)
            a = torch.exp(x - z[:, None])
            out[b, h * G:(h + 1) * G] = a @ v
            lse[b, h * G:(h + 1) * G] = z
            if gathered is not None:
                gathered[b, h, :n] += a.sum(0)
    return {"out": out, "lse": lse} if gathered is None else {"out": out, "lse": lse, "weights": gathered}
