"""The paged KV cache's operators as cases to measure: decode attention over pages, the decode step
(RoPE, append, attention) over pages, RoPE and append into pages, and the page operations (copy, fork,
truncate, extend, compact).

Where ``own`` is false ``run`` computes each operator in elementary torch operations; where it is true
it makes the calls of ``b200attn``. The sizes are the repository's: 16 query heads over 4 KV heads of
128 (and the 8 / 2 and 4 / 1 shares of a tensor-parallel rank, and 32 over 8), 36 layers, contexts up
to 64K tokens, ragged batches of 512 to 16K tokens.
"""
import math
import os
import random
import sys

import torch

own = False

D = 128          # head dim
THETA = 5.0e6    # RoPE base
LAYERS = 36      # a page holds the tokens of every layer: 2 * LAYERS planes (K and V of each)
MOST = 64 * 16384 * 512   # K elements of the largest padded batch


def _b200attn():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llm-inference_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import b200attn
    return b200attn


# ---- cases -------------------------------------------------------------------

def listed():
    return [
        # a chat's next token, early in the conversation: latency
        {"name": "decode, 1 short", "op": "decode", "seqs": 1, "heads": 16, "kv_heads": 4, "page": 16,
         "min_len": 300, "max_len": 300, "idle": 0},
        # continuous batching at a serving node's ordinary load: 64 conversations of 512 to 16K tokens
        {"name": "decode, 64 ragged", "op": "decode", "seqs": 64, "heads": 16, "kv_heads": 4, "page": 64,
         "min_len": 512, "max_len": 16384, "idle": 0},
        # one long document: the split over the cache's length and the join are what counts
        {"name": "decode, 1 of 64K", "op": "decode", "seqs": 1, "heads": 16, "kv_heads": 4, "page": 32,
         "min_len": 65537, "max_len": 65537, "idle": 0},
        # a captured batch of 256 slots on a tensor-parallel rank (4 / 1 heads), a fifth of them idle
        {"name": "decode, 256 slots, 1 KV head", "op": "decode", "seqs": 256, "heads": 4, "kv_heads": 1, "page": 16,
         "min_len": 1, "max_len": 4099, "idle": 51},
        # a layer of the decode step for a few users
        {"name": "step, 8 short", "op": "step", "seqs": 8, "heads": 16, "kv_heads": 4, "page": 16,
         "min_len": 30, "max_len": 700, "idle": 0, "rotate": True},
        # a layer of the decode step of a loaded node, 32 heads over 8 KV heads
        {"name": "step, 48 ragged, 8 KV heads", "op": "step", "seqs": 48, "heads": 32, "kv_heads": 8, "page": 32,
         "min_len": 200, "max_len": 8192, "idle": 3, "rotate": True},
        # the rows of one decode step into their pages
        {"name": "append, 64 tokens", "op": "append", "tokens": 64, "seqs": 64, "heads": 8, "kv_heads": 2, "page": 16,
         "rotate": True, "start": 3000},
        # four prompts of 4096 tokens at once, read from the projection's [Q | K | V] rows
        {"name": "append, 4 prompts of 4096", "op": "append", "tokens": 16384, "seqs": 4, "heads": 32, "kv_heads": 8,
         "page": 64, "rotate": True, "start": 0},
        # pages of a preempted conversation brought to other places, every layer
        {"name": "pages: copy 24", "op": "copy", "pairs": 24, "kv_heads": 4, "page": 16, "pages": 700,
         "planes": 2 * LAYERS},
        # parallel sampling: the losing beams dropped, the winner forked, a token's room for each
        {"name": "pages: 4 prompts, 8 beams", "op": "beam", "prompts": 4, "beams": 8, "kv_heads": 4, "page": 32,
         "len": 1805, "pages": 560, "planes": 2 * LAYERS},
        # speculative decoding: rejected drafts rolled back, room for the next ones
        {"name": "pages: 64 rolled back", "op": "rollback", "seqs": 64, "kv_heads": 4, "page": 16, "max_len": 500,
         "drop": 5, "take": 6, "planes": 2 * LAYERS},
        # a pool three fifths full after a busy hour, brought together at its low end
        {"name": "pages: compact 480", "op": "compact", "seqs": 40, "kv_heads": 4, "page": 32, "pages": 480,
         "fill": 0.6, "planes": 2 * LAYERS},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    heads, kvh = rng.choice([(16, 4), (16, 4), (8, 2), (4, 1), (32, 8), (8, 8), (24, 8)])
    op = rng.choice(["decode", "decode", "step", "step", "append", "copy", "beam", "rollback", "compact"])
    page = rng.choice([16, 16, 32, 48, 64, 128, 256, 5, 24])
    if op in ("decode", "step"):
        seqs = _log(rng, 1, 256)
        top = min(70000, MOST // (seqs * kvh * D))
        most = max(2, _log(rng, 2, top))
        case = {"op": op, "seqs": seqs, "heads": heads, "kv_heads": kvh, "page": page,
                "min_len": max(1, int(most * rng.choice([0.01, 0.2, 1.0]))), "max_len": most,
                "idle": rng.choice([0, 0, seqs // 5])}
        if op == "step":
            case["rotate"] = rng.random() < 0.75   # every fourth layer has no rotation
        return case
    if op == "append":
        tokens = _log(rng, 1, 20000)
        return {"op": op, "tokens": tokens, "seqs": rng.randint(1, min(tokens, 64)), "heads": heads, "kv_heads": kvh,
                "page": page, "rotate": rng.random() < 0.75, "start": rng.randint(0, 5000)}
    planes = 2 * rng.randint(1, LAYERS)
    kvh = min(kvh, 4)
    page = rng.choice([8, 16, 32, 5])
    if op == "copy":
        pairs = _log(rng, 1, 200)
        return {"op": op, "pairs": pairs, "kv_heads": kvh, "page": page, "pages": 2 * pairs + rng.randint(0, 60),
                "planes": planes}
    if op == "beam":
        prompts, beams, n = rng.randint(1, 4), rng.randint(2, 8), _log(rng, 1, 1800)
        return {"op": op, "prompts": prompts, "beams": beams, "kv_heads": kvh, "page": page, "len": n,
                "pages": prompts * (-(-n // page) + 4 * beams) + rng.randint(0, 40), "planes": planes}
    if op == "rollback":
        return {"op": op, "seqs": _log(rng, 1, 128), "kv_heads": kvh, "page": page, "max_len": _log(rng, 10, 250),
                "drop": rng.randint(0, 8), "take": rng.randint(1, 9), "planes": planes}
    pages = _log(rng, 20, 450)
    return {"op": op, "seqs": rng.randint(1, 40), "kv_heads": kvh, "page": page, "pages": pages,
            "fill": round(rng.uniform(0.2, 0.9), 2), "planes": planes}


# ---- inputs ------------------------------------------------------------------

def _up(a, b):
    return -(-a // b)


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(shape, g, std=1.0):
    x = torch.empty(shape, dtype=torch.float16, device="cuda")
    return x.normal_(0.0, std, generator=g)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _lens(case):
    """The batch's lengths, spread over their logarithm: the case's own, put in order by the seed."""
    lo, hi, live = case["min_len"], case["max_len"], case["seqs"] - case["idle"]
    rng = random.Random(hi * 4099 + live)
    return [hi] + [min(hi, max(lo, _log(rng, lo, hi))) for _ in range(live - 1)]


def _table(lens, page, width, g, spare):
    """A page table of shuffled pages for sequences of these lengths, and the number of pages."""
    held = torch.tensor([_up(n, page) for n in lens], device="cuda")
    total = sum(_up(n, page) for n in lens)
    perm = torch.randperm(total + spare, generator=g, device="cuda")
    j = torch.arange(width, device="cuda")[None]
    at = (held.cumsum(0) - held)[:, None] + j
    table = torch.where(j < held[:, None], perm[at.clamp(max=total + spare - 1)], -1)
    return table.to(torch.int32).contiguous(), total + spare


def _rope(rows):
    pos = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None]
    freq = THETA ** (-torch.arange(0, D, 2, device="cuda", dtype=torch.float64)[None] / D)
    return (pos * freq).cos().half(), (pos * freq).sin().half()


def prepare(case, seed):
    g = _gen(seed)
    op, page, kvh = case["op"], case["page"], case["kv_heads"]
    s = {"op": op, "page": page, "kv_heads": kvh}
    if op in ("decode", "step"):
        heads, n = case["heads"], case["seqs"]
        lens = _lens(case)
        random.Random(seed).shuffle(lens)
        lens += [0] * case["idle"]   # a captured batch's idle slots are its last
        width = _up(case["max_len"], page)
        table, pages = _table(lens, page, width, g, max(1, sum(lens) // page // 8))
        s.update(heads=heads, n=n, max_len=case["max_len"], table=table, width=width, pages=pages,
                 k=_normal((pages, page, kvh * D), g), v=_normal((pages, page, kvh * D), g),
                 q=_normal((n, heads * D), g, 2.0), out=torch.empty((n, heads * D), dtype=torch.float16, device="cuda"),
                 len=_ints(lens))
        if op == "step":
            s.update(k_new=_normal((n, kvh * D), g), v_new=_normal((n, kvh * D), g), rotate=case["rotate"],
                     pos=_ints([x - 1 for x in lens]))
            s["cos"], s["sin"] = _rope(case["max_len"])
        if own:
            s["ws"] = torch.zeros(_b200attn().decode_paged_workspace_bytes(n, heads, kvh, D), dtype=torch.uint8,
                                  device="cuda")
        return s
    if op == "append":
        heads, t, n, start = case["heads"], case["tokens"], case["seqs"], case["start"]
        each = _up(t, n)
        first = [start * i // n for i in range(n)]   # other places in each sequence
        random.Random(seed).shuffle(first)
        width = _up(start + each, page)
        table, pages = _table([f + each for f in first], page, width, g, 3)
        tok = torch.arange(t, device="cuda")
        seq = (tok // each).to(torch.int32)
        row = (heads + 2 * kvh) * D
        qkv = _normal((t, row), g)
        s.update(heads=heads, t=t, table=table, width=width, pages=pages, qkv=qkv,
                 k=_normal((pages, page, kvh * D), g), v=_normal((pages, page, kvh * D), g), seqs=seq,
                 pos=(_ints(first)[seq.long()] + (tok % each)).to(torch.int32), rotate=case["rotate"], row=row,
                 rows=start + each, n=n)
        s["cos"], s["sin"] = _rope(start + each)
        return s
    planes, elems = case["planes"], page * kvh * D
    s.update(planes=planes, elems=elems)
    rng = random.Random(seed)
    if op == "copy":
        pages = case["pages"]
        perm = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        n = case["pairs"]
        s.update(pool=_normal((planes, pages, elems), g), pages=pages, src=perm[:n].contiguous(),
                 dst=perm[n:2 * n].contiguous(), n=n)
        return s
    if op == "beam":
        # slot p * beams holds prompt p's winner; its other beams have a few tokens of their own to lose
        p, b, ln, pages = case["prompts"], case["beams"], case["len"], case["pages"]
        lens = [ln + 1 if i % b == 0 else rng.randint(1, min(ln, 3 * page)) for i in range(p * b)]
        width = _up(ln + 1, page) + 1
        table, used = _table(lens, page, width, g, pages - sum(_up(x, page) for x in lens))
        win, lose = list(range(0, p * b, b)), [i for i in range(p * b) if i % b]
        s.update(drop_seqs=_ints(win + lose), drop_len=_ints([ln] * len(win) + [0] * len(lose)),
                 parents=_ints([i - i % b for i in lose]), children=_ints(lose), take_seqs=_ints(list(range(p * b))),
                 take=_ints([1] * (p * b)))
    elif op == "rollback":
        n, top = case["seqs"], case["max_len"]
        lens = [1 + (top - 1) * i // n for i in range(n)]
        rng.shuffle(lens)
        width = _up(top + case["drop"] + case["take"], page)
        held = [x + case["drop"] for x in lens]
        need = sum(_up(x + case["take"], page) - _up(x, page) for x in lens)
        table, used = _table(held, page, width, g, need + 5)
        order = list(range(n))
        rng.shuffle(order)
        s.update(drop_seqs=_ints(order), drop_len=_ints([lens[i] for i in order]), take_seqs=_ints(order),
                 take=_ints([rng.randint(1, case["take"]) for _ in order]))
        lens = held
    else:
        n, pages = case["seqs"], case["pages"]
        live = max(1, int(pages * case["fill"]))
        share = [1.0 + i / n for i in range(n)]
        rng.shuffle(share)
        lens = [int(live * page * x / sum(share)) // page * page + rng.randint(0, page - 1) * (i % 2)
                for i, x in enumerate(share)]
        while sum(_up(x, page) for x in lens) > pages:
            lens[lens.index(max(lens))] -= page
        width = max(1, max(_up(x, page) for x in lens))
        table, used = _table(lens, page, width, g, pages - sum(_up(x, page) for x in lens))
        s.update(table_out=torch.empty_like(table), ref_out=torch.empty(pages, dtype=torch.int32, device="cuda"))
    ref = torch.zeros(used, dtype=torch.int32, device="cuda")
    flat = table.flatten().long()
    ref.scatter_add_(0, flat.clamp(min=0), (flat >= 0).int())
    s.update(pool=_normal((planes, used, elems), g), pages=used, table=table, width=width, len=_ints(lens), ref=ref,
             slots=len(lens), status=torch.zeros(2, dtype=torch.int32, device="cuda"),
             first=torch.empty(len(lens), dtype=torch.int32, device="cuda"))
    if own:
        s["ws"] = torch.zeros(_b200attn().kv_pages_workspace_bytes(used), dtype=torch.uint8, device="cuda")
    return s


# ---- the plain form --------------------------------------------------------------

def _rotate(x, cos, sin):
    """Rotate-half RoPE of rows [n, heads, D] in 32 bits, rounded to the 16 bits that are stored."""
    x, c, s = x.float(), cos.float()[:, None], sin.float()[:, None]
    lo, hi = x[..., :D // 2], x[..., D // 2:]
    return torch.cat([lo * c - hi * s, hi * c + lo * s], -1).half()


def _attend(q, s, lens):
    """softmax(q k / sqrt(D)) v of one query row a sequence over its pages, rows past its length masked."""
    n, h, g = s["n"], s["kv_heads"], s["heads"] // s["kv_heads"]
    at = s["table"].long().clamp(min=0)
    keep = torch.arange(s["width"] * s["page"], device="cuda")[None] < lens[:, None]
    k = s["k"][at].view(n, -1, h, D).transpose(1, 2).float()
    q = q.view(n, h, g, D).float()
    w = (q @ k.transpose(2, 3)) / math.sqrt(D)
    del k
    w = torch.where(keep[:, None, None], w, -math.inf)
    top = w.amax(-1, keepdim=True)
    w = (w - torch.where(top > -math.inf, top, 0.0)).exp()
    total = w.sum(-1, keepdim=True)
    v = s["v"][at].view(n, -1, h, D).transpose(1, 2).float()
    v = torch.where(keep[:, None, :, None], v, 0.0)
    return ((w @ v) / torch.where(total > 0, total, 1.0)).view(n, -1).half()


def _store(s, k, v, seqs, pos, live):
    """Rows k, v [t, kv_dim] to position pos of the sequence in table row seqs."""
    page = s["table"][seqs, (pos // s["page"]).clamp(min=0)].long()
    row = (page * s["page"] + pos % s["page"])[live]
    s["k"].view(-1, k.shape[1])[row] = k[live]
    s["v"].view(-1, v.shape[1])[row] = v[live]


def _step(s):
    n, h, pos = s["n"], s["kv_heads"], s["pos"].long()
    q, k = s["q"].view(n, -1, D), s["k_new"].view(n, h, D)
    if s["rotate"]:
        c, sn = s["cos"][pos.clamp(min=0)], s["sin"][pos.clamp(min=0)]
        q, k = _rotate(q, c, sn), _rotate(k, c, sn)
    _store(s, k.reshape(n, -1), s["v_new"], torch.arange(n, device="cuda"), pos, pos >= 0)
    return _attend(q.reshape(n, -1), s, pos + 1)


def _append(s):
    t, h, kv = s["t"], s["heads"] * D, s["kv_heads"] * D
    pos = s["pos"].long()
    q, k, v = s["qkv"][:, :h], s["qkv"][:, h:h + kv], s["qkv"][:, h + kv:]
    if s["rotate"]:
        c, sn = s["cos"][pos], s["sin"][pos]
        q.copy_(_rotate(q.reshape(t, -1, D), c, sn).view(t, -1))
        k = _rotate(k.reshape(t, -1, D), c, sn).view(t, -1)
    _store(s, k, v, s["seqs"].long(), pos, slice(None))


def _truncate(s, seqs, new):
    seqs, j = seqs.long(), torch.arange(s["width"], device="cuda")[None]
    rows, page = s["table"][seqs], s["page"]
    drop = (j >= _up(new, page)[:, None]) & (j < _up(s["len"][seqs], page)[:, None])
    s["ref"].scatter_add_(0, rows.flatten().long().clamp(min=0), -drop.flatten().int())
    s["table"][seqs] = torch.where(drop, -1, rows)
    s["len"][seqs] = new


def _fork(s, parents, children):
    parents, children = parents.long(), children.long()
    rows, n = s["table"][parents], s["len"][parents]
    share = torch.arange(s["width"], device="cuda")[None] < _up(n, s["page"])[:, None]
    s["ref"].scatter_add_(0, rows.flatten().long().clamp(min=0), share.flatten().int())
    s["table"][children] = torch.where(share, rows, -1)
    s["len"][children] = n


def _extend(s, seqs, take):
    """Room for `take` more tokens of each sequence: its own copy of a shared page that they begin in, then the
    lowest free pages. Of the sequences that alone share such a page the first keeps it."""
    seqs, page, ref = seqs.long(), s["page"], s["ref"]
    old = s["len"][seqs]
    held, want = _up(old, page), _up(old + take, page)
    last = s["table"][seqs, (held - 1).clamp(min=0).long()].long()
    part = (old % page != 0) & (take > 0)
    same = (last[:, None] == last[None]) & part[:, None] & part[None]
    first = same.int().argmax(1) == torch.arange(len(seqs), device="cuda")
    alone = same.sum(1) == ref[last.clamp(min=0)]
    cow = part & (ref[last.clamp(min=0)] > 1) & ~(alone & first)
    need = want - held + cow
    base = need.cumsum(0) - need
    free = ref == 0
    page_of = torch.zeros(s["pages"] + 1, dtype=torch.long, device="cuda")
    ids = torch.arange(s["pages"], device="cuda")
    page_of.scatter_(0, torch.where(free, free.cumsum(0) - 1, s["pages"]), ids)
    j = torch.arange(s["width"], device="cuda")[None]
    copied = cow[:, None] & (j == held[:, None] - 1)
    fresh = (j >= held[:, None]) & (j < want[:, None])
    got = page_of[(base[:, None] + torch.where(copied, 0, cow[:, None] + j - held[:, None])).clamp(0, s["pages"])]
    new = copied | fresh
    s["table"][seqs] = torch.where(new, got.int(), s["table"][seqs])
    to = got.gather(1, (held - 1).clamp(min=0).long()[:, None])[:, 0][cow]
    s["pool"][:, to] = s["pool"][:, last[cow]]
    ref.scatter_add_(0, got.flatten(), new.flatten().int())
    ref.scatter_add_(0, last.clamp(min=0), -cow.int())
    s["len"][seqs] = old + take
    s["first"][:len(seqs)] = old


def _compact(s):
    live = s["ref"] > 0
    n = live.sum()
    ids = torch.arange(s["pages"], device="cuda")
    src, dst = ids[live & (ids >= n)], ids[~live & (ids < n)]
    s["pool"][:, dst] = s["pool"][:, src]
    to = ids.clone()
    to[src] = dst
    s["table_out"].copy_(torch.where(s["table"] >= 0, to[s["table"].long().clamp(min=0)].int(), -1))
    s["ref_out"].copy_(torch.where(ids < n, s["ref"], 0))
    s["ref_out"][dst] = s["ref"][src]
    s["status"].copy_(torch.stack([torch.zeros_like(n), n]))


# ---- one pass ----------------------------------------------------------------------

def _bits(pool):
    return pool.view(torch.int16)


def run(s):
    op, page, kvh = s["op"], s["page"], s["kv_heads"]
    if own:
        b = _b200attn()
    if op == "decode":
        if own:
            b.launch_causal_attention_decode_paged(
                s["q"], 0, s["k"], s["v"], 0, s["pages"], page, s["table"], s["width"], s["n"], None, s["len"], 0,
                s["out"], 0, s["n"], s["heads"], kvh, D, s["ws"], s["ws"].numel())
            return s["out"]
        return _attend(s["q"], s, s["len"])
    if op == "step":
        if own:
            b.launch_decode_step_paged_fused(
                s["q"], 0, s["k_new"], s["v_new"], 0, s["k"], s["v"], 0, s["pages"], page, s["table"], s["width"],
                s["n"], None, s["cos"], s["sin"], s["max_len"], s["rotate"], s["pos"], s["out"], 0, s["n"],
                s["heads"], kvh, D, s["ws"], s["ws"].numel())
            return s["out"], s["k"], s["v"]
        return _step(s), s["k"], s["v"]
    if op == "append":
        # Q is rotated in place: each pass turns it on by its positions' angles
        h = s["heads"] * D
        if own:
            b.launch_rope_and_store_kv_paged(
                s["qkv"], s["qkv"][:, h:], s["qkv"][:, h + kvh * D:], s["k"], s["v"], 0, s["pages"], page, s["table"],
                s["width"], s["n"], s["seqs"], s["cos"], s["sin"], s["rows"], s["t"], s["heads"], kvh, D, s["row"],
                s["row"], s["pos"], s["rotate"])
        else:
            _append(s)
        return s["qkv"][:, :h], s["k"], s["v"]
    pool = s["pool"]
    if own:
        where = (pool, s["planes"], s["pages"] * s["elems"], s["pages"], s["elems"], s["elems"])
    if op == "copy":
        if own:
            b.launch_kv_pages_copy(*where, s["src"], s["dst"], s["n"])
        else:
            pool[:, s["dst"].long()] = pool[:, s["src"].long()]
        return _bits(pool)
    if op == "compact":
        if own:
            b.launch_kv_pages_compact(*where, s["table"], s["table_out"], s["width"], s["slots"], page, s["len"],
                                      s["ref"], s["ref_out"], s["status"], s["ws"], s["ws"].numel())
        else:
            _compact(s)
        # behind the live pages the pool holds what was moved away: it belongs to nobody
        return _bits(pool), s["table_out"], s["ref_out"], s["status"]
    if own:
        seqs = (s["table"], s["width"], s["slots"], page, s["pages"], s["len"], s["ref"])
        work = (s["status"], s["ws"], s["ws"].numel())
        b.launch_kv_pages_truncate(*seqs, s["drop_seqs"], s["drop_len"], len(s["drop_seqs"]), *work)
        if op == "beam":
            b.launch_kv_pages_fork(*seqs, s["parents"], s["children"], None, len(s["parents"]), *work)
        b.launch_kv_pages_extend(*where, *seqs[:4], *seqs[5:], s["take_seqs"], s["take"], len(s["take"]), s["first"],
                                 *work)
    else:
        _truncate(s, s["drop_seqs"], s["drop_len"])
        if op == "beam":
            _fork(s, s["parents"], s["children"])
        _extend(s, s["take_seqs"], s["take"])
    return _bits(pool), s["table"], s["len"], s["ref"], s["first"]


# ---- what a pass cannot do without -----------------------------------------------------

def work(case):
    op, page, kvh = case["op"], case["page"], case["kv_heads"]
    row = kvh * D * 2
    if op in ("decode", "step"):
        heads, n, live = case["heads"], case["seqs"], case["seqs"] - case["idle"]
        tokens = sum(_lens(case))
        table = 4 * tokens / page
        nbytes = tokens * 2 * row + table + 4 * n + 2 * n * heads * D * 2
        if op == "step":
            nbytes += live * (2 * row + (2 * D if case["rotate"] else 0))
        return {"bytes": nbytes, "flops": tokens * heads * D * 4}
    if op == "append":
        t, heads = case["tokens"], case["heads"]
        q = 2 * heads * D * 2 if case["rotate"] else 0
        # Q rotated in place, K and V read and written
        return {"bytes": t * (q + 4 * row + 8 + (2 * D if case["rotate"] else 0)),
                "flops": t * (heads + kvh) * D * 3 if case["rotate"] else 0}
    one = 2 * case["planes"] * page * row   # a page of every plane, read and written
    if op == "copy":
        return {"bytes": case["pairs"] * (one + 8), "flops": 0}
    if op == "compact":
        live = case["pages"] * case["fill"]
        return {"bytes": live * (1 - case["fill"]) * one + 8 * case["pages"] + 8 * live, "flops": 0}
    if op == "beam":
        n, held = case["prompts"] * case["beams"], _up(case["len"], page)
        copies = case["prompts"] * (case["beams"] - 1) if case["len"] % page else 0
        return {"bytes": copies * one + n * (held * 16 + 40) + 4 * case["pages"], "flops": 0}
    pages = case["seqs"] * _up(case["max_len"] // 2 + case["drop"] + 5, page)
    return {"bytes": case["seqs"] * 64 + 4 * pages, "flops": 0}


# ---- in 64 bits, from the definition ------------------------------------------------------

def _turned(x, pos, s):
    """Rows [n, heads * D] turned by their positions' angles (the tables are the operator's input), in 64 bits."""
    n = x.shape[0]
    z = torch.complex(*x.double().view(n, -1, 2, D // 2).unbind(2))
    z = z * torch.complex(s["cos"][pos].double(), s["sin"][pos].double())[:, None]
    return torch.stack([z.real, z.imag], 2).view(n, -1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] not in ("decode", "step", "append"):
        return None
    h, page = case["kv_heads"], case["page"]
    if case["op"] == "append":
        wide = case["heads"] * D
        q, k, v = s["qkv"][:, :wide].double(), s["qkv"][:, wide:wide + h * D].double(), s["qkv"][:, wide + h * D:]
        pos = s["pos"].long()
        if s["rotate"]:
            q, k = _turned(q, pos, s), _turned(k, pos, s)
        kp, vp = s["k"].double(), s["v"].double()
        at = s["table"].long()[s["seqs"].long(), pos // page]
        kp[at, pos % page] = k
        vp[at, pos % page] = v.double()
        return q, kp, vp
    lens, q = s["len"].tolist(), s["q"].double()
    kp, vp = s["k"], s["v"]
    if case["op"] == "step":
        on = [i for i, n in enumerate(lens) if n]
        pos = s["pos"].long()[on]
        k = s["k_new"][on].double()
        if s["rotate"]:
            # the turned query row and the cached row are 16-bit values by definition
            q[on], k = _turned(q[on], pos, s).float().half().double(), _turned(k, pos, s)
        kp, vp = kp.double(), vp.double()
        at = s["table"].long()[on, pos // page]
        kp[at, pos % page] = k
        vp[at, pos % page] = s["v_new"][on].double()
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for i, n in enumerate(lens):
        if not n:
            continue
        own_pages = s["table"][i, :_up(n, page)].long()
        k = kp[own_pages].reshape(-1, h, D)[:n].half().double()
        v = vp[own_pages].reshape(-1, h, D)[:n].double()
        w = torch.einsum("hgd,lhd->hgl", q[i].view(h, -1, D), k) * D ** -0.5
        out[i] = torch.einsum("hgl,lhd->hgd", torch.softmax(w, -1), v).reshape(-1)
    return out if case["op"] == "decode" else (out, kp, vp)
