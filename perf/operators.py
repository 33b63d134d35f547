"""The paged K/V cache operators and their plain forms: what each case computes,
on which inputs, and the bytes and operations that it cannot do without.

  tables     block tables, slot maps and positions of a step, built on the GPU
             from the requests' lengths
  append     the step's key and value rows into the cache at their slots
  attention  the step's query rows over the cached keys of their requests

With ``own`` false ``run`` is the plain form in elementary torch operations, with
``own`` true it calls the framework (``paged.py``).
"""
import importlib
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def _paged():
    return importlib.import_module("index-tts-25-metal_b200.paged")


# ---- cases ------------------------------------------------------------------


def listed():
    return [
        # one step of 16 requests in flight: one token each, one request finished
        {"name": "tables_step16", "op": "tables", "requests": 16, "cached": 420, "prompts": 0, "prompt": 1,
         "released": 1, "block": 64, "pad": 0},
        # a step of a busy server: mostly single tokens, some new prompts, some finished requests
        {"name": "tables_mixed256", "op": "tables", "requests": 256, "cached": 1500, "prompts": 32, "prompt": 451,
         "released": 24, "block": 16, "pad": 37},
        # admission of a large offline batch: a prompt for every request
        {"name": "tables_prompts2048", "op": "tables", "requests": 2048, "cached": 64, "prompts": 2040,
         "prompt": 400, "released": 3, "block": 16, "pad": 0},
        # one step of 16 requests: a row each into an fp32 cache with the Qwen3-0.6B heads
        {"name": "append_step16_f32", "op": "append", "rows": 16, "pad": 0, "heads": 8, "dim": 128, "block": 64,
         "blocks": 128, "source": "f32", "type": "f32", "layout": "token"},
        # fp32 rows of the GPT heads rounded into an fp16 cache, head-major pages
        {"name": "append_prefix_f32_f16", "op": "append", "rows": 3608, "pad": 41, "heads": 20, "dim": 64,
         "block": 32, "blocks": 160, "source": "f32", "type": "f16", "layout": "head"},
        # a full prompt pass of many requests
        {"name": "append_prompts_bf16", "op": "append", "rows": 32768, "pad": 0, "heads": 8, "dim": 128, "block": 16,
         "blocks": 2304, "source": "bf16", "type": "bf16", "layout": "token"},
        # a decode step of the emotion-text decoder: 16 short prompts, fp32
        {"name": "attend_step16_f32", "op": "attention", "requests": 16, "fresh_low": 1, "fresh": 1, "context_low": 23,
         "context": 420, "heads": 16, "kv_heads": 8, "dim": 128, "block": 64, "type": "f32", "layout": "token",
         "pad": 0},
        # a decode step of 64 requests of all lengths
        {"name": "attend_step64_bf16", "op": "attention", "requests": 64, "fresh_low": 1, "fresh": 1, "context_low": 0,
         "context": 16384, "heads": 16, "kv_heads": 8, "dim": 128, "block": 64, "type": "bf16", "layout": "token",
         "pad": 0},
        # one very long request: the work is split over the keys
        {"name": "attend_long1_f16", "op": "attention", "requests": 1, "fresh_low": 1, "fresh": 1,
         "context_low": 131089, "context": 131089, "heads": 16, "kv_heads": 8, "dim": 128, "block": 32, "type": "f16",
         "layout": "head", "pad": 0},
        # chunks of long prompts over what is cached already
        {"name": "attend_chunk_bf16", "op": "attention", "requests": 8, "fresh_low": 512, "fresh": 1024,
         "context_low": 1024, "context": 8192, "heads": 16, "kv_heads": 8, "dim": 128, "block": 64, "type": "bf16",
         "layout": "token", "pad": 0},
        # GPT conditioning and text prefixes with nothing cached, 20 heads of 64
        {"name": "attend_prefix_f16", "op": "attention", "requests": 16, "fresh_low": 75, "fresh": 451,
         "context_low": 0, "context": 0, "heads": 20, "kv_heads": 20, "dim": 64, "block": 16, "type": "f16",
         "layout": "head", "pad": 13},
        # prompt chunks of the fp32 decoder beside single tokens
        {"name": "attend_prompt_f32", "op": "attention", "requests": 6, "fresh_low": 1, "fresh": 1500,
         "context_low": 0, "context": 1000, "heads": 16, "kv_heads": 8, "dim": 128, "block": 64, "type": "f32",
         "layout": "token", "pad": 0},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(["tables", "append", "attention", "attention"])
    block = rng.choice([16, 32, 64, 128])
    if op == "tables":
        n = _log_int(rng, 1, 2048)
        prompts = rng.randint(0, n)
        return {"op": op, "requests": n, "cached": _log_int(rng, 1, 4096), "prompts": prompts,
                "prompt": _log_int(rng, 1, 400), "released": rng.randint(0, n - prompts), "block": block,
                "pad": rng.choice([0, 0, 1, 29])}
    if op == "append":
        heads, dim = rng.choice([(8, 128), (20, 64), (1, 128), (5, 64)])
        rows = _log_int(rng, 1, 32768)
        kind = rng.choice(["f32", "f16", "bf16"])
        return {"op": op, "rows": rows, "pad": rng.choice([0, 0, 7]), "heads": heads, "dim": dim, "block": block,
                "blocks": rows // block + 2 + rng.randint(0, 64), "source": rng.choice(["f32", kind]), "type": kind,
                "layout": rng.choice(["token", "head"])}
    heads, kv_heads, dim = rng.choice([(16, 8, 128), (20, 20, 64), (16, 2, 128), (12, 4, 64), (8, 1, 128), (3, 1, 64)])
    kind = rng.choice(["f32", "f16", "bf16"])
    step = rng.random() < 0.5
    requests = _log_int(rng, 1, 64 if step else 12)
    fresh = rng.choice([1, 1, 2, 5]) if step else _log_int(rng, 6, 1024)
    # keys in all stay below those of the listed cases: 64 requests of up to 16384, fewer where rows and fp32 cost more
    most = 400_000 // requests if step else 16_000 // requests
    if kind == "f32":
        most //= 4
    context = _log_int(rng, 1, max(1, min(131072 if requests == 1 else 16384, most)))
    return {"op": op, "requests": requests, "fresh_low": 1 if rng.random() < 0.5 else fresh, "fresh": fresh,
            "context_low": 0 if rng.random() < 0.5 else context, "context": context, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "block": block, "type": kind, "layout": rng.choice(["token", "head"]),
            "pad": rng.choice([0, 0, 3])}


# ---- inputs -----------------------------------------------------------------


def _spread(low, high, count, g):
    """`count` whole numbers spread evenly from `high` down to `low`, in an order that `g` gives."""
    values = torch.tensor([high - (high - low) * i // max(1, count - 1) for i in range(count)], dtype=torch.int64)
    return values[torch.randperm(count, generator=g)]


def _lengths(case, seed):
    """Per request: fresh rows and cached tokens before them (host lists)."""
    g = torch.Generator().manual_seed(int(seed) * 7919 + 11)
    b = case["requests"]
    return (_spread(case["fresh_low"], case["fresh"], b, g).tolist(),
            _spread(case["context_low"], case["context"], b, g).tolist())


def _cache(case, blocks, kind, g):
    """K and V caches [blocks, block, heads, dim], their memory token-major or head-major within a block."""
    heads = case["kv_heads"] if case["op"] == "attention" else case["heads"]
    a, b = (case["block"], heads) if case["layout"] == "token" else (heads, case["block"])
    shape = (blocks, a, b, case["dim"])
    made = [torch.randn(shape, device="cuda", generator=g, dtype=_TYPES[kind]) for _ in range(2)]
    return made if case["layout"] == "token" else [c.transpose(1, 2) for c in made]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"op": case["op"], "case": case}
    if case["op"] == "tables":
        h = torch.Generator().manual_seed(int(seed) * 104729 + 5)
        b, bs = case["requests"], case["block"]
        order = torch.randperm(b, generator=h)
        fresh = torch.ones(b, dtype=torch.int64)
        cached = _spread(0, case["cached"], b, h)
        # room for all that these ranges can hold, the same for every seed
        blocks = int(((cached + bs - 1) // bs).sum()) + 17
        new = order[:case["prompts"]]
        fresh[new] = _spread(1, case["prompt"], len(new), h)
        cached[new[len(new) // 4:]] = 0  # most prompts are new requests, the others go on with a cached one
        fresh[order[case["prompts"]:case["prompts"] + case["released"]]] = -1
        blocks += int((fresh.clamp(min=0) // bs + 2).sum())
        width = (case["cached"] + max(1, case["prompt"])) // bs + 4
        have = (cached + bs - 1) // bs
        held = int(have.sum())
        ids = torch.randperm(blocks, generator=h)
        table = torch.full((b, width), -1, dtype=torch.int64)
        table[torch.arange(width)[None, :] < have[:, None]] = ids[:held]
        free = torch.full((blocks,), -1, dtype=torch.int64)
        free[:blocks - held] = ids[held:]
        rows = int(fresh.clamp(min=0).sum()) + case["pad"]

        def put(x):
            return x.to(torch.int32).cuda()

        def room(n):
            return torch.empty(n, dtype=torch.int32, device="cuda")

        s.update(block=bs, blocks=blocks, cached=put(cached), fresh=put(fresh), table=put(table), free_list=put(free),
                 free_count=put(torch.tensor([blocks - held])), lens=room(b), q_start=room(b + 1),
                 positions=room(rows), slots=room(rows), free_out=room(1), status=room(1))
        return s
    if case["op"] == "append":
        rows, total = case["rows"], case["rows"] + case["pad"]
        s["k_cache"], s["v_cache"] = _cache(case, case["blocks"], case["type"], g)
        # key and value rows as slices of the projection that makes both
        both = torch.randn((total, 2, case["heads"], case["dim"]), device="cuda", generator=g,
                           dtype=_TYPES[case["source"]])
        s["k"], s["v"] = both[:, 0], both[:, 1]
        slots = torch.full((total,), -1, dtype=torch.int32, device="cuda")
        slots[:rows] = torch.randperm(case["blocks"] * case["block"], device="cuda", generator=g)[:rows].int()
        s["slots"] = slots
        return s
    fresh, cached = _lengths(case, seed)
    b, bs, kind = case["requests"], case["block"], _TYPES[case["type"]]
    lens = [f + c for f, c in zip(fresh, cached)]
    used = [(n + bs - 1) // bs for n in lens]
    blocks = sum(used) + 3
    s["k_cache"], s["v_cache"] = _cache(case, blocks, case["type"], g)
    h = torch.Generator().manual_seed(int(seed) + 1)
    ids = torch.randperm(blocks, generator=h).int()
    table = torch.full((b, max(used) + 1), -1, dtype=torch.int32)
    table[torch.arange(max(used) + 1)[None, :] < torch.tensor(used)[:, None]] = ids[:sum(used)]
    rows = sum(fresh) + case["pad"]
    start = torch.zeros(b + 1, dtype=torch.int32)
    start[1:] = torch.cumsum(torch.tensor(fresh), 0)
    q = torch.randn((rows, case["heads"], case["dim"]), device="cuda", generator=g, dtype=torch.float32)
    s.update(q=(q * 1.5).to(kind), table=table.cuda(), lens=torch.tensor(lens, dtype=torch.int32).cuda(),
             q_start=start.cuda(), out=torch.zeros((rows, case["heads"], case["dim"]), device="cuda", dtype=kind),
             max_fresh=max(fresh), max_len=max(lens), scale=1.0 / math.sqrt(case["dim"]))
    return s


# ---- the plain forms --------------------------------------------------------


def _plain_tables(s):
    bs, table, free, blocks = s["block"], s["table"].long(), s["free_list"].long(), s["blocks"]
    cached, fresh, rows = s["cached"].long(), s["fresh"].long(), s["slots"].numel()
    gone, n = fresh < 0, fresh.clamp(min=0)
    have = (cached + bs - 1) // bs
    need = torch.where(gone, 0, (cached + n + bs - 1) // bs - have)
    give = torch.where(gone, have, 0)
    column = torch.arange(table.shape[1], device=table.device)[None, :]
    # released blocks go on top of the stack of free ones, in request and column order
    at = s["free_count"].long() + (torch.cumsum(give, 0) - give)[:, None] + column
    at = torch.where(column < give[:, None], at, blocks)
    free = torch.cat([free, free.new_zeros(1)]).scatter(0, at.reshape(-1), table.reshape(-1))[:blocks]
    top = s["free_count"].long() + give.sum()
    # new blocks come off it, request by request
    at = top - 1 - ((torch.cumsum(need, 0) - need)[:, None] + column - have[:, None])
    new = (column >= have[:, None]) & (column < (have + need)[:, None])
    table = torch.where(new, free[at.clamp(0, blocks - 1)], table)
    q_start = torch.cat([n.new_zeros(1), torch.cumsum(n, 0)])
    t = torch.arange(rows, device=table.device)
    b = torch.searchsorted(q_start[1:], t, right=True).clamp(max=cached.numel() - 1)
    pos = cached[b] + t - q_start[b]
    inside = t < q_start[-1]
    slot = table[b, (pos // bs).clamp(0, table.shape[1] - 1)] * bs + pos % bs
    out = {"table": table, "free_list": free, "free_count": top - need.sum(),
           "lens": torch.where(gone, 0, cached + n), "q_start": q_start,
           "positions": torch.where(inside, pos, 0), "slots": torch.where(inside, slot, -1),
           "status": torch.zeros_like(top)}
    return {k: v.int().reshape(-1) if k != "table" else v.int() for k, v in out.items()}


def _plain_append(s):
    bs = s["case"]["block"]
    keep = s["slots"] >= 0
    slots = s["slots"][keep].long()
    s["k_cache"][slots // bs, slots % bs] = s["k"][keep].to(s["k_cache"].dtype)
    s["v_cache"][slots // bs, slots % bs] = s["v"][keep].to(s["v_cache"].dtype)
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_attention(s):
    case, dev = s["case"], s["q"].device
    bs, hk, dim = case["block"], case["kv_heads"], case["dim"]
    group = case["heads"] // hk
    start, lens = s["q_start"].long(), s["lens"].long()
    n = start[1:] - start[:-1]
    requests, rows = lens.numel(), s["q"].shape[0]
    key = torch.arange(s["max_len"], device=dev)
    page = s["table"].long()[:, key // bs].clamp(min=0)
    k = s["k_cache"][page, key % bs].float().permute(0, 2, 3, 1)  # [requests, kv head, dim, key]
    v = s["v_cache"][page, key % bs].float().permute(0, 2, 1, 3)
    i = torch.arange(s["max_fresh"], device=dev)
    q = s["q"][(start[:-1, None] + i).clamp(max=rows - 1)].float()
    q = q.reshape(requests, s["max_fresh"], hk, group, dim).permute(0, 2, 1, 3, 4)
    scores = torch.matmul(q.reshape(requests, hk, -1, dim), k) * s["scale"]
    last = lens[:, None] - n[:, None] + i  # each row's own position
    seen = key[None, None, :] <= last[:, :, None]
    seen = seen[:, None, :, None, :].expand(-1, -1, -1, group, -1).reshape(requests, 1, -1, s["max_len"])
    scores = torch.where(seen, scores, -torch.inf)
    high = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(scores - high)
    out = torch.matmul(p, v) / p.sum(-1, keepdim=True).clamp(min=1e-38)
    out = out.reshape(requests, hk, s["max_fresh"], group, dim).permute(0, 2, 1, 3, 4)
    out = out.reshape(requests, s["max_fresh"], case["heads"], dim)
    t = torch.arange(rows, device=dev)
    b = torch.searchsorted(start[1:], t, right=True).clamp(max=requests - 1)
    row = out[b, (t - start[b]).clamp(0, s["max_fresh"] - 1)].to(s["q"].dtype)
    return torch.where((t < start[-1])[:, None, None], row, s["out"])


def run(state):
    s = state
    if s["op"] == "tables":
        if own:
            _paged().tables(s["cached"], s["fresh"], s["table"], s["free_list"], s["free_count"], s["block"],
                            lens=s["lens"], q_start=s["q_start"], positions=s["positions"], slots=s["slots"],
                            free_out=s["free_out"], status=s["status"])
            return {"table": s["table"], "free_list": s["free_list"], "free_count": s["free_out"], "lens": s["lens"],
                    "q_start": s["q_start"], "positions": s["positions"], "slots": s["slots"], "status": s["status"]}
        return _plain_tables(s)
    if s["op"] == "append":
        if own:
            _paged().append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"])
            return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}
        return _plain_append(s)
    if own:
        return _paged().attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], s["q_start"],
                                  s["max_fresh"], scale=s["scale"], out=s["out"])
    return _plain_attention(s)


# ---- what a pass cannot do without -------------------------------------------


def work(case):
    if case["op"] == "tables":
        rows = case["prompts"] * (case["prompt"] + 1) // 2 + case["requests"] - case["prompts"] - case["released"]
        blocks = rows // case["block"] + case["released"] * (case["cached"] // 2 // case["block"] + 1)
        return {"bytes": 16 * case["requests"] + 8 * (rows + case["pad"]) + 8 * blocks, "flops": 0}
    if case["op"] == "append":
        return {"bytes": case["rows"] * (2 * case["heads"] * case["dim"] *
                                         (_BYTES[case["source"]] + _BYTES[case["type"]]) + 4), "flops": 0}
    # means over the requests, as prepare() spreads their lengths
    one = case["requests"] == 1
    fresh = case["fresh"] if one else (case["fresh_low"] + case["fresh"]) / 2
    context = case["context"] if one else (case["context_low"] + case["context"]) / 2
    row = case["heads"] * case["dim"]
    keys = case["requests"] * (fresh + context)
    pairs = case["requests"] * fresh * (context + (fresh + 1) / 2)
    return {"bytes": _BYTES[case["type"]] * (2 * keys * case["kv_heads"] * case["dim"] +
                                             2 * case["requests"] * fresh * row), "flops": 4 * pairs * row}


# ---- the definitions in 64 bits ------------------------------------------------


def exact(case, seed):
    if case["op"] == "tables":
        return None  # whole numbers only: the plain form's are the definition
    s = prepare(case, seed)
    if case["op"] == "append":
        out = {}
        for name in ("k", "v"):
            cache = s[name + "_cache"].double()
            for row, slot in enumerate(s["slots"].tolist()):
                if slot >= 0:
                    cache[slot // case["block"], slot % case["block"]] = s[name][row].double()
            out[name + "_cache"] = cache
        return out
    out = s["out"].double()
    group = case["heads"] // case["kv_heads"]
    start, lens, bs = s["q_start"].tolist(), s["lens"].tolist(), case["block"]
    for b, length in enumerate(lens):
        pages = s["table"][b, :(length + bs - 1) // bs].long()
        k = s["k_cache"][pages].reshape(-1, case["kv_heads"], case["dim"])[:length].double()
        v = s["v_cache"][pages].reshape(-1, case["kv_heads"], case["dim"])[:length].double()
        q = s["q"][start[b]:start[b + 1]].double()
        first = length - q.shape[0]
        mask = torch.arange(length, device=q.device)[None, :] > first + torch.arange(q.shape[0], device=q.device)[:, None]
        for h in range(case["heads"]):
            w = (q[:, h] @ k[:, h // group].T * s["scale"]).masked_fill(mask, -torch.inf).softmax(-1)
            out[start[b]:start[b + 1], h] = w @ v[:, h // group]
    return out
