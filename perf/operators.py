"""The paged key-value cache's operators as measured cases.

  map     block tables, free pages and slot maps of a step from the requests' lengths
  append  rotary positions on a step's queries and keys, keys and values into their slots
  attend  attention of single new tokens over the paged cache
  step    the three of them in a row, as one layer of a decode step runs them

Where `own` is false, run() computes them with elementary torch operations; where it is true, it makes the calls of
include/kv_paged.h through pk_b200.KvPaged.
"""
import math
import os
import sys

import torch

own = False

LEFT = -7.0  # what an output row that no call writes holds


def _shape(heads, kv_heads, head_size):
    return {"heads": heads, "kv_heads": kv_heads, "head_size": head_size}


TINYLLAMA = _shape(32, 4, 64)      # the model shapes that the benchmark quotes
LLAMA2_7B = _shape(32, 32, 128)
LLAMA3_8B = _shape(32, 8, 128)


def listed():
    return [
        # one decode step of a full batch: one token for each of 64 requests
        {"name": "map_decode", "op": "map", "n": 64, "page": 16, "most_len": 2048, "most_new": 1, "churn": 0},
        # a server's mixed step: decoding, rejected drafts taken back, requests that end, short prompts
        {"name": "map_churn", "op": "map", "n": 1000, "page": 16, "most_len": 2048, "most_new": 48, "churn": 1},
        # prompts of 256 requests admitted at once, a million rows
        {"name": "map_prompts", "op": "map", "n": 256, "page": 32, "most_len": 0, "most_new": 8192, "churn": 0},
        # one decode step of 64 requests, half cache
        {"name": "append_decode", "op": "append", "n": 64, "cache": "f16", "page": 16, "layout": "token", "rope": 128, **LLAMA3_8B},
        # a prompt chunk with an odd number of rows, float cache
        {"name": "append_chunk", "op": "append", "n": 1001, "cache": "f32", "page": 32, "layout": "token", "rope": 64, **TINYLLAMA},
        # the prompts of a whole batch, half cache with each head's tokens together
        {"name": "append_prompts", "op": "append", "n": 16384, "cache": "f16", "page": 64, "layout": "head", "rope": 128, **LLAMA3_8B},
        # the first tokens of one answer: latency alone
        {"name": "attend_short", "op": "attend", "n": 1, "cache": "f32", "page": 16, "layout": "token", "least": 40, "most": 40, **TINYLLAMA},
        # one sequence with a long context
        {"name": "attend_long", "op": "attend", "n": 1, "cache": "f16", "page": 16, "layout": "token", "least": 65536, "most": 65536, **LLAMA3_8B},
        # a batch of conversations of every age, float cache
        {"name": "attend_ragged", "op": "attend", "n": 64, "cache": "f32", "page": 16, "layout": "token", "least": 1, "most": 2048, **TINYLLAMA},
        # a key-value head for each query head, float cache
        {"name": "attend_mha", "op": "attend", "n": 16, "cache": "f32", "page": 32, "layout": "head", "least": 1000, "most": 1060, **LLAMA2_7B},
        # a full batch at up to the model's whole context, half cache: the most work
        {"name": "attend_batch", "op": "attend", "n": 64, "cache": "f16", "page": 64, "layout": "token", "least": 1, "most": 8192, **LLAMA3_8B},
        # a layer of a mixed step with odd sizes: 12 query heads to a key-value head, odd pages, padded rows
        {"name": "step_odd", "op": "step", "n": 33, "cache": "f16", "page": 24, "layout": "token", "most_len": 777, "most_new": 2, "rope": 40,
         **_shape(24, 2, 80)},
    ]


def _log(rng, lo, hi):
    """A whole number in lo .. hi, spread evenly over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["map", "append", "attend", "attend", "step"])
    page = rng.choice([8, 16, 16, 32, 64, _log(rng, 1, 128)])
    if op == "map":
        n = _log(rng, 1, 2048)
        new = _log(rng, 1, min(8192, max(1, 2097152 // n)))
        return {"op": op, "n": n, "page": page, "most_len": rng.choice([0, _log(rng, 1, 8192)]), "most_new": new, "churn": rng.randrange(2)}
    hs = rng.choice([64, 128, 128, 8 * rng.randrange(2, 33)])
    kv_heads = _log(rng, 1, 32)
    group = rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 8, 12, 16])
    while kv_heads * group > 64:
        kv_heads = max(1, kv_heads // 2)
    case = {"op": op, "cache": rng.choice(["f16", "f32"]), "page": page, "layout": rng.choice(["token", "head"])}
    case.update(_shape(kv_heads * group, kv_heads, hs))
    wide = (2 * group + 3) * kv_heads * hs  # values that a row reads and writes in append, about
    if op == "append":
        case.update(n=_log(rng, 1, max(1, min(16384, 150000000 // wide))), rope=rng.choice([0, hs, 2 * rng.randrange(1, hs // 2 + 1)]))
    elif op == "attend":
        n = _log(rng, 1, 128)
        most = _log(rng, 1, max(1, min(131072, 500000000 // (n * kv_heads * hs * (4 if case["cache"] == "f32" else 2)))))
        case.update(n=n, most=most, least=rng.choice([0, 1, most, max(1, most // 2)]))
    else:
        n = _log(rng, 1, 96)
        most = _log(rng, 1, max(1, min(16384, 200000000 // (n * kv_heads * hs))))
        case.update(n=n, most_len=most, most_new=_log(rng, 1, 3), rope=rng.choice([0, hs, 2 * rng.randrange(1, hs // 2 + 1)]))
    return case


def _ints(g, lo, hi, n):
    """n whole numbers in lo .. hi."""
    return torch.randint(lo, hi + 1, (n,), generator=g, device="cuda", dtype=torch.int32)


def _tables(g, lens, page, blocks, pages, extra):
    """A block table whose rows hold the pages of `lens` tokens (other entries -1), and the free pages under `extra` more entries."""
    held = (lens + page - 1) // page
    ids = torch.randperm(pages, generator=g, device="cuda", dtype=torch.int32)
    first = torch.cumsum(held, 0) - held
    at = torch.arange(blocks, device="cuda")
    table = torch.where(at[None] < held[:, None], ids[(first[:, None] + at[None]).clamp(max=pages - 1)], -1).to(torch.int32)
    used = held.sum()
    left = torch.arange(pages + extra, device="cuda") + used
    free = torch.where(left < pages, ids[left.clamp(max=pages - 1)], -1).to(torch.int32)[:pages].contiguous()
    return table.contiguous(), free, (pages - used).to(torch.int32).reshape(1)


def _lengths(case, g):
    """len, start and end of a step's requests."""
    n, new = case["n"], case["most_new"]
    lens = _ints(g, min(1, case["most_len"]), case["most_len"], n)
    start = lens.clone()
    end = start + (_ints(g, 1, new, n) if case["most_len"] == 0 or case.get("churn") or case["op"] == "step" else new)
    if case.get("churn"):
        kind = _ints(g, 0, 9, n)
        back = torch.minimum(lens, _ints(g, 0, 7, n))
        start = torch.where(kind < 3, lens - back, start)             # rejected drafts are taken back, and more tokens come
        end = torch.where(kind < 3, start + _ints(g, 0, min(8, new), n), end)
        end = torch.where((kind >= 3) & (kind < 7), start + 1, end)   # plain decoding
        gone = kind == 7                                              # the request ends
        start, end = torch.where(gone, 0, start), torch.where(gone, 0, end)
        end = torch.where(kind == 8, start, end)                      # nothing this step
    return lens.to(torch.int32), start.to(torch.int32), end.to(torch.int32)


def _values(g, shape, dtype, spread):
    """Normal values whose last axis has channels of unlike sizes, as keys and queries have them."""
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float16 if dtype == torch.float16 else torch.float32)
    by = torch.exp(spread * torch.randn(shape[-1], generator=g, device="cuda"))
    return x.mul_(by.to(x.dtype)) if spread else x


def _dtype(case):
    return torch.float16 if case["cache"] == "f16" else torch.float32


def _pool(case, g, pages, spread):
    """A pool of pages as the kernels get it: [page][token][head] or, by head, [page][head][token]."""
    order = (case["page"], case["kv_heads"]) if case["layout"] == "token" else (case["kv_heads"], case["page"])
    return _values(g, (pages, *order, case["head_size"]), _dtype(case), spread)


def _rope_table(length, dim):
    """(cos, sin) pairs of each position, from angles in 64 bits."""
    i = torch.arange(dim // 2, device="cuda", dtype=torch.float64)
    a = torch.arange(length, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-2.0 * i / dim)[None]
    return torch.stack([a.cos(), a.sin()], 2).to(torch.float32).reshape(length, dim).contiguous()


def _handle(case, pages, blocks, device=0):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    at = os.path.join(root, "llm-inference-c_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import pk_b200
    heads, kv, hs, page = case.get("heads", 1), case.get("kv_heads", 1), case.get("head_size", 64), case["page"]
    strides = (page * kv * hs, kv * hs, hs) if case.get("layout") != "head" else (page * kv * hs, hs, page * hs)
    return pk_b200.KvPaged(heads, kv, hs, pk_b200.F16 if case.get("cache") == "f16" else pk_b200.F32, page, pages,
                           case["n"] if case["op"] != "append" else 1, blocks, strides=strides, device=device)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    n, page, op = case["n"], case["page"], case["op"]
    s = {"case": case}
    if op in ("map", "step"):
        longest = case["most_len"] + case["most_new"]
        blocks = -(-longest // page)
        pages = n * blocks
        s["len"], s["start"], s["end"] = _lengths(case, g)
        s["table"], s["free"], s["n_free"] = _tables(g, s["len"], page, blocks, pages, 0)
        s["n_free_out"] = torch.zeros(1, device="cuda", dtype=torch.int32)
        rows = n * case["most_new"] if op == "map" else n * case["most_new"] + 3  # a step's last rows are padding
        s["rows"] = [torch.full((rows,), -1, device="cuda", dtype=torch.int32) for _ in range(3)]
        s["row0"] = torch.zeros(n + 1, device="cuda", dtype=torch.int32)
    if op == "append":
        rows, longest = n, 8192
        pages = -(-n * 5 // 4 // page) + 1
        blocks = 1
        at = torch.arange(n, device="cuda", dtype=torch.int32)
        if n > 256:  # prompts: the rows lie side by side in their pages, the pages anywhere
            slot = torch.randperm(pages, generator=g, device="cuda", dtype=torch.int32)[at // page] * page + at % page
        else:        # a decode step: each row in a page of another request
            slot = torch.randperm(pages * page, generator=g, device="cuda", dtype=torch.int32)[:n]
        s["rows"] = [at, (_ints(g, 0, longest - 1, 1) + at) % longest, slot.to(torch.int32).contiguous()]
    if op == "attend":
        rows = n
        blocks = max(1, -(-case["most"] // page))
        pages = n * blocks
        lens = _ints(g, case["least"], case["most"], n)
        lens[seed % n] = case["most"]
        s["table"], _, _ = _tables(g, lens, page, blocks, pages, 0)
        s["rows"] = [torch.arange(n, device="cuda", dtype=torch.int32), (lens - 1).to(torch.int32)]
    if op != "map":
        h, kv, hs = case["heads"], case["kv_heads"], case["head_size"]
        s["q"] = _values(g, (rows, h, hs), torch.float32, 0.3).mul_(1.5)
        s["kp"] = _pool(case, g, pages, 0.3 if op == "attend" else 0.0)
        s["vp"] = _pool(case, g, pages, 0.0)
        s["out"] = torch.full((rows, h, hs), LEFT, device="cuda")
        s["scale"] = 1.0 / math.sqrt(hs)
    if op in ("append", "step"):
        s["k"] = _values(g, (rows, kv, hs), torch.float32, 0.3)
        s["v"] = _values(g, (rows, kv, hs), torch.float32, 0.0)
        s["rope"] = _rope_table(longest, case["rope"]) if case["rope"] else None
        s["q_out"] = torch.full_like(s["q"], LEFT)
    if own:
        s["kv"] = _handle(case, pages, blocks)
    return s


# ---- plain forms -----------------------------------------------------


def _plain_map(s):
    page, (row_req, row_pos, row_slot) = s["case"]["page"], s["rows"]
    table, free = s["table"], s["free"]
    n, blocks, pages = table.shape[0], table.shape[1], free.shape[0]
    lens, start, end = s["len"].long(), s["start"].long(), s["end"].long()
    held, need = (lens + page - 1) // page, (end + page - 1) // page
    back, take = (held - need).clamp(min=0), (need - held).clamp(min=0)
    back0, take0 = torch.cumsum(back, 0) - back, torch.cumsum(take, 0) - take
    had = s["n_free"].long()
    at = torch.arange(blocks, device=table.device)[None]
    # pages behind a request's new end go on the free pages' top, in request and block order
    gone = (at >= need[:, None]) & (at < held[:, None])
    place = torch.where(gone, had + back0[:, None] + at - need[:, None], pages)
    stack = torch.cat([free, free.new_full((pages + 1 - free.shape[0],), -1)])
    stack.scatter_(0, place.clamp(max=pages).reshape(-1), torch.where(gone, table, -1).reshape(-1))
    top = had + back.sum()
    # and new ones come from the top, in request and block order
    fresh = (at >= held[:, None]) & (at < need[:, None])
    pop = top - 1 - (take0[:, None] + at - held[:, None])
    table.copy_(torch.where(fresh, stack[torch.where(fresh, pop, 0).clamp(min=0)], table))
    left = top - take.sum()
    kept = torch.arange(pages, device=table.device)
    free.copy_(torch.where((kept >= had) & (kept < left), stack[:pages], free))
    s["n_free_out"].copy_(left)
    # the rows of the step, request after request
    row0 = torch.cat([start.new_zeros(1), torch.cumsum(end - start, 0)])
    s["row0"].copy_(row0)
    r = torch.arange(row_req.shape[0], device=table.device)
    req = torch.searchsorted(row0[1:], r, right=True)
    live = req < n
    req = req.clamp(max=n - 1)
    pos = start[req] + r - row0[req]
    slot = table[req, (pos // page).clamp(max=blocks - 1)].long() * page + pos % page
    row_req.copy_(torch.where(live, req, -1))
    row_pos.copy_(torch.where(live, pos, -1))
    row_slot.copy_(torch.where(live, slot, -1))


def _plain_rope(x, rope, pos):
    if rope is None:
        return x
    dim = rope.shape[1]
    c, sn = rope[pos][:, None, 0::2], rope[pos][:, None, 1::2]
    a, b = x[..., 0:dim:2], x[..., 1:dim:2]
    turned = torch.stack([a * c - b * sn, a * sn + b * c], -1).flatten(-2)
    return torch.cat([turned, x[..., dim:]], -1)


def _by_token(case, pool):
    """The pool as [page][token][head][channel], whichever way it lies."""
    return pool if case["layout"] == "token" else pool.transpose(1, 2)


def _plain_append(s):
    case, (_, pos, slot) = s["case"], s["rows"]
    live = slot >= 0
    at = pos.clamp(min=0).long()
    s["q_out"].copy_(torch.where(live[:, None, None], _plain_rope(s["q"], s["rope"], at), s["q_out"]))
    k = _plain_rope(s["k"], s["rope"], at)
    to = slot[live].long()
    for pool, x in ((s["kp"], k), (s["vp"], s["v"])):
        _by_token(case, pool)[to // case["page"], to % case["page"]] = x[live].to(pool.dtype)


def _plain_attend(s, q):
    case, (req, pos) = s["case"], s["rows"][:2]
    n, h, hs = q.shape
    kv, page, longest = case["kv_heads"], case["page"], s["table"].shape[1] * case["page"]
    t = torch.arange(longest, device=q.device)
    live = req >= 0
    entry = s["table"][req.clamp(min=0).long()][:, t // page].clamp(min=0).long()
    keys = _by_token(case, s["kp"])[entry, t % page].float()
    score = torch.matmul(q.view(n, kv, h // kv, hs), keys.permute(0, 2, 3, 1)) * s["scale"]
    del keys
    seen = (t[None] <= pos[:, None])[:, None, None]
    score = torch.where(seen, score, -math.inf)
    top = score.amax(3, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    del score
    total = p.sum(3, keepdim=True)
    values = torch.where(seen.view(n, longest, 1, 1), _by_token(case, s["vp"])[entry, t % page], 0).float()
    out = torch.matmul(p, values.transpose(1, 2)) / torch.where(total == 0, 1.0, total)
    s["out"].copy_(torch.where(live[:, None, None], out.reshape(n, h, hs), s["out"]))


# ---- the framework's calls -------------------------------------------


def _own_map(s):
    kv, rows = s["kv"], s["rows"]
    kv.map(s["len"].data_ptr(), s["start"].data_ptr(), s["end"].data_ptr(), s["len"].shape[0], s["table"].data_ptr(),
           s["free"].data_ptr(), s["n_free"].data_ptr(), s["n_free_out"].data_ptr(), rows[0].shape[0],
           rows[0].data_ptr(), rows[1].data_ptr(), rows[2].data_ptr(), s["row0"].data_ptr())


def _own_append(s):
    rope, rows = s["rope"], s["rows"]
    s["kv"].append(s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), rows[1].data_ptr(), rows[2].data_ptr(),
                   rows[1].shape[0], s["q_out"].data_ptr(), s["kp"].data_ptr(), s["vp"].data_ptr(),
                   rope.data_ptr() if rope is not None else 0, rope.shape[1] if rope is not None else 0,
                   rope.shape[0] if rope is not None else 0)


def _own_attend(s, q):
    rows = s["rows"]
    s["kv"].attend(q.data_ptr(), s["kp"].data_ptr(), s["vp"].data_ptr(), s["table"].data_ptr(), s["table"].shape[0],
                   rows[0].data_ptr(), rows[1].data_ptr(), rows[0].shape[0], s["scale"], s["out"].data_ptr())


def run(s):
    op = s["case"]["op"]
    if op in ("map", "step"):
        _own_map(s) if own else _plain_map(s)
    if op in ("append", "step"):
        _own_append(s) if own else _plain_append(s)
    if op in ("attend", "step"):
        q = s["q"] if op == "attend" else s["q_out"]
        _own_attend(s, q) if own else _plain_attend(s, q)
    mapped = [s["table"], s["free"], s["n_free_out"], s["row0"], *s["rows"]] if op in ("map", "step") else []
    stored = [s["q_out"], s["kp"], s["vp"]] if op in ("append", "step") else []
    return {"map": mapped, "append": stored, "attend": [s["out"]] if op in ("attend", "step") else []}


def work(case):
    op, n = case["op"], case["n"]
    total = {"bytes": 0.0, "flops": 0.0}
    if op in ("map", "step"):
        rows = n * case["most_new"]  # every row of the three lists is written, -1 behind the last one
        total["bytes"] += 4 * (3 * n + n + 1) + 12 * rows + 8 * n * case["most_new"] / case["page"]
    if op == "map":
        return total
    h, kv, hs = case["heads"], case["kv_heads"], case["head_size"]
    size = 2 if case["cache"] == "f16" else 4
    if op == "step":
        n = n * (1 + case["most_new"]) / 2
    if op in ("append", "step"):
        total["bytes"] += n * (2 * h * hs * 4 + 2 * kv * hs * (4 + size) + 8 + 4 * case["rope"])
        total["flops"] += 3 * n * (h + kv) * case["rope"]
    if op in ("attend", "step"):
        least, most = (case["least"], case["most"]) if op == "attend" else (0, case["most_len"] + case["most_new"])
        seen = n * (least + most) / 2 if op == "attend" else case["n"] * (least + most) / 2
        total["bytes"] += 2 * seen * kv * hs * size + 2 * n * h * hs * 4
        total["flops"] += 4 * seen * h * hs * (1 if op == "attend" else n / case["n"])
    return total


# ---- the definition in 64 bits ---------------------------------------


def exact(case, seed):
    """The definitions, row by row in 64 bits. The map's outputs are whole numbers: nothing to say about them."""
    op = case["op"]
    if op == "map":
        return None
    global own
    was, own = own, False
    s = prepare(case, seed)
    own = was
    page = case["page"]
    if op == "step":  # where the step's rows go, found one page at a time on the host
        lens, start, end = (s[k].tolist() for k in ("len", "start", "end"))
        table, stack = s["table"].tolist(), s["free"].tolist()[:int(s["n_free"])]
        rows = []
        for i, row in enumerate(table):
            for b in range(-(-lens[i] // page), -(-end[i] // page)):
                row[b] = stack.pop()
            rows += [(i, p, row[p // page] * page + p % page) for p in range(start[i], end[i])]
        rows += [(-1, -1, -1)] * (s["q"].shape[0] - len(rows))
        s["table"] = torch.tensor(table, device="cuda")
        s["rows"] = [torch.tensor(c, device="cuda") for c in zip(*rows)]
    q, stored = s["q"].double(), []
    pools = [s["kp"].double(), s["vp"].double()]
    if op in ("append", "step"):
        where = [i for i, x in enumerate(s["rows"][2].tolist()) if x >= 0]
        to = s["rows"][2][where].long()
        q_out, k = s["q_out"].double(), s["k"].double()
        if case["rope"]:
            pair = torch.view_as_complex(s["rope"].double().view(-1, case["rope"] // 2, 2))[s["rows"][1][where].long()]
            for x in (q, k):
                part = torch.view_as_complex(x[where][..., :case["rope"]].unflatten(-1, (-1, 2)).contiguous())
                x[where, :, :case["rope"]] = torch.view_as_real(part * pair[:, None]).flatten(-2)
        q_out[where] = q[where]
        q = q_out
        for pool, x in zip(pools, (k, s["v"].double())):
            _by_token(case, pool)[to // page, to % page] = x[where]
        stored = [q_out, *pools]
    out = None
    if op in ("attend", "step"):
        out = s["out"].double()
        group = case["heads"] // case["kv_heads"]
        reqs, seen = s["rows"][0].tolist(), s["rows"][1].tolist()
        for r, (i, last) in enumerate(zip(reqs, seen)):
            if i < 0:
                continue
            entry = s["table"][i, :last // page + 1].long() if last >= 0 else s["table"][i, :0].long()
            k, v = (_by_token(case, p)[entry].flatten(0, 1)[:last + 1].repeat_interleave(group, 1) for p in pools)
            p = torch.softmax(torch.einsum("hd,thd->ht", q[r], k) * s["scale"], 1)
            out[r] = torch.einsum("ht,thd->hd", p, v)
    mapped = [None] * 7 if op == "step" else []
    return {"map": mapped, "append": stored, "attend": [out] if out is not None else []}
