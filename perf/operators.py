"""The operators of the paged key/value cache, as a serving program calls them: block tables and slot
maps built from the requests' lengths, the append of new keys and values to their pages, and the
attention of every request's new tokens over its pages.

A pool holds pages of `page` rows, [pages, kv_heads, page, head_dim] for keys and the same for values.
Request r holds `held[r]` rows before a step and brings `fresh[r]` new tokens; row j of a request lies in
page tables[r, j // page]. The new tokens of all requests are packed one request after another.

  tables   pages ceil(held/page) .. ceil((held+fresh)/page) - 1 of every request, in the requests' order,
           are taken from the end of the list of free pages; starts[r] = sum of fresh before r,
           kv_len = held + fresh, and per token its position held + i and its slot
           tables[r, position // page] * page + position % page (padding rows: position 0, slot -1)
  append   pages[slot // page, :, slot % page, :] = new[token], keys and values
  attend   o[i, h] = sum_j p_j v[j], p = softmax over j <= position of token i of scale * q[i, h] . k[j],
           with key/value head h // (heads / kv_heads) and scale = 1 / sqrt(head_dim)
"""
import math
import random

import torch

own = False

SIZE = {"float32": 4, "float16": 2, "bfloat16": 2}
LOOSE = 7        # padding rows behind the last token, pages beyond the ones in use


def _case(name, kind, requests, past, new, page, dtype="bfloat16", heads=10, kv_heads=2, head_dim=128, chunks=1.0):
    """past, new: ranges of the requests' lengths; chunks: the share of requests that bring `new` tokens
    (the others bring one)."""
    return dict(name=name, kind=kind, dtype=dtype, requests=requests, past_lo=past[0], past_hi=past[1], new_lo=new[0], new_hi=new[1],
                chunks=chunks, page=page, heads=heads, kv_heads=kv_heads, head_dim=head_dim)


def listed():
    return [
        # One decoding step of a small server: 64 requests, one token each, a new page now and then.
        _case("tables_decode", "tables", 64, (16, 2047), (1, 1), 16),
        # A step of a large one: new requests and running ones, up to 64 tokens each.
        _case("tables_mixed", "tables", 1000, (0, 4096), (1, 64), 16, chunks=0.5),
        # One token of each of 32 requests joins one layer's cache; grouped-query heads.
        _case("append_decode_bf16", "append", 32, (300, 2000), (1, 1), 16),
        # The prompts of 16 requests join it, GPT-2's heads, larger pages.
        _case("append_prompts_fp16", "append", 16, (0, 0), (700, 1023), 64, dtype="float16", heads=12, kv_heads=12, head_dim=64),
        # One user's next token, GPT-2 in fp32 as generate() runs it: latency.
        _case("attend_one_fp32", "attend", 1, (143, 143), (1, 1), 16, dtype="float32", heads=12, kv_heads=12, head_dim=64),
        # Next tokens of a batch, grouped-query heads, lengths all over the model's context.
        _case("attend_decode_gqa_bf16", "attend", 32, (300, 2000), (1, 1), 16),
        # Next tokens of a full server, multi-head, larger pages: the most bytes.
        _case("attend_decode_fp16", "attend", 256, (128, 1000), (1, 1), 64, dtype="float16", heads=12, kv_heads=12, head_dim=64),
        # A few drafted tokens per request that are checked at once.
        _case("attend_draft_bf16", "attend", 16, (500, 2000), (4, 4), 32),
        # Whole prompts, multi-head, nothing cached before: products.
        _case("attend_prompts_fp16", "attend", 8, (0, 0), (1024, 2047), 16, dtype="float16", heads=10, kv_heads=10),
        # The next chunk of two very long prompts over what is cached of them: the most operations.
        _case("attend_chunk_bf16", "attend", 2, (8000, 14000), (1024, 1024), 128),
        # A step of a busy server: most requests bring a token, some a piece of a prompt; an odd page size.
        _case("attend_mixed_bf16", "attend", 24, (100, 2000), (200, 700), 24, heads=10, kv_heads=10, chunks=0.25),
        # Prompts in full precision.
        _case("attend_prompts_fp32", "attend", 3, (0, 0), (100, 500), 16, dtype="float32", heads=12, kv_heads=12, head_dim=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tables", "append", "attend", "attend", "attend", "attend"])
    half = rng.choice(["float16", "bfloat16"])
    page = rng.choice([8, 16, 16, 24, 32, 64, 128, 100])
    if kind == "tables":
        top = _log(rng, 1, 4096)
        return {k: v for k, v in _case("", kind, _log(rng, 1, 1000), (0, top), (1, _log(rng, 1, 64)), page,
                                       chunks=rng.choice([0.2, 0.5, 1.0])).items() if k != "name"}
    dtype = rng.choice([half, half, half, "float32"])
    head_dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 4, 10, 12])
    heads = kv_heads * rng.choice([1, 1, 2, 4, 5, 7])
    heads = heads if heads <= 32 else kv_heads
    shape = rng.choice(["decode", "decode", "draft", "prompts", "chunk", "mixed"])
    if shape == "decode":
        top = _log(rng, 4, 8000)
        c = _case("", kind, _log(rng, 1, 256), (top // 4, top), (1, 1), page, dtype, heads, kv_heads, head_dim)
    elif shape == "draft":
        c = _case("", kind, _log(rng, 1, 64), (10, _log(rng, 20, 4000)), (2, rng.randint(2, 9)), page, dtype, heads, kv_heads, head_dim)
    elif shape == "prompts":
        top = _log(rng, 8, 2047)
        c = _case("", kind, _log(rng, 1, 32), (0, 0), (1 + top // 3, top), page, dtype, heads, kv_heads, head_dim)
    elif shape == "chunk":
        top = _log(rng, 200, 14000)
        c = _case("", kind, rng.randint(1, 4), (top // 2, top), (20, _log(rng, 30, 1024)), page, dtype, heads, kv_heads, head_dim)
    else:
        c = _case("", kind, _log(rng, 4, 48), (1, _log(rng, 30, 2000)), (16, _log(rng, 20, 700)), page, dtype, heads, kv_heads, head_dim,
                  chunks=rng.choice([0.1, 0.25, 0.5]))
    c.pop("name")
    most = {"bytes": 2.5e8, "flops": 2e9 if dtype == "float32" else 6e10}
    while c["requests"] > 1 and any(work(c)[k] > v for k, v in most.items()):
        c["requests"] = max(1, c["requests"] * 2 // 3)
    while any(work(c)[k] > v for k, v in most.items()):
        c["past_hi"], c["new_hi"] = max(c["past_lo"], c["past_hi"] * 2 // 3), max(c["new_lo"], c["new_hi"] * 2 // 3)
        c["past_lo"], c["new_lo"] = c["past_lo"] * 2 // 3, max(1, c["new_lo"] * 2 // 3)
    return c


# ----------------------------------------------------------------- prepare ----
def _lengths(case):
    """held and fresh of every request: the case's, not the seed's, so that a case is always the same work."""
    rng = random.Random("%(requests)d %(past_lo)d %(past_hi)d %(new_lo)d %(new_hi)d %(page)d" % case)
    held, fresh = [], []
    for _ in range(case["requests"]):
        held.append(rng.randint(case["past_lo"], case["past_hi"]))
        fresh.append(rng.randint(case["new_lo"], case["new_hi"]) if rng.random() < case["chunks"] else 1)
    return held, fresh


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    page, R = case["page"], case["requests"]
    held, fresh = _lengths(case)
    pages_of = lambda n: -(-n // page)
    before, after = [pages_of(h) for h in held], [pages_of(h + f) for h, f in zip(held, fresh)]
    n_pages, width = sum(after) + LOOSE, max(after) + 1
    order = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)     # pages in the order in which they came to be used
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")
    column = torch.arange(width, device="cuda")
    s = dict(kind=case["kind"], page=page, dtype=case["dtype"], held=i32(held), fresh=i32(fresh), max_new=max(fresh))
    tokens = sum(fresh)
    if case["kind"] == "tables":
        # the pages that the requests hold already; the rest of the pool is free
        have = column < i32(before)[:, None]
        tables = torch.full((R, width), -1, dtype=torch.int32, device="cuda")
        tables[have] = order[:sum(before)]
        free = torch.cat([order[sum(before):], i32([-1] * sum(before))])
        rows = tokens + LOOSE
        s.update(tables=tables, free=free, n_free=i32([n_pages - sum(before)]), starts=i32([0] * (R + 1)), kv_len=i32([0] * R),
                 position=i32([0] * rows), slot=i32([0] * rows), left=i32([0]))
        return s
    tables = torch.full((R, width), -1, dtype=torch.int32, device="cuda")
    tables[column < i32(after)[:, None]] = order[:sum(after)]
    H, Hk, D = case["heads"], case["kv_heads"], case["head_dim"]
    kind = getattr(torch, case["dtype"])
    normal = lambda *shape: torch.randn(shape, generator=gen, device="cuda", dtype=kind)
    s.update(tables=tables, k_pages=normal(n_pages, Hk, page, D), v_pages=normal(n_pages, Hk, page, D))
    starts = torch.cat([i32([0]), torch.cumsum(s["fresh"], 0).to(torch.int32)])
    if case["kind"] == "append":
        request = torch.repeat_interleave(torch.arange(R, device="cuda"), s["fresh"].long())
        position = s["held"][request] + torch.arange(tokens, device="cuda") - starts[request]
        s.update(k=normal(tokens, Hk, D), v=normal(tokens, Hk, D),
                 slot=(tables[request, position // page] * page + position % page).to(torch.int32))
        return s
    s.update(q=normal(tokens, H, D), starts=starts, kv_len=s["held"] + s["fresh"], max_kv=max(h + f for h, f in zip(held, fresh)),
             o=torch.zeros((tokens, H, D), dtype=kind, device="cuda"))
    return s


# --------------------------------------------------------------------- run ----
def run(state):
    call = {"tables": (_plain_tables, _own_tables), "append": (_plain_append, _own_append), "attend": (_plain_attend, _own_attend)}
    return call[state["kind"]][own](state)


def _plain_tables(s):
    held, fresh, page = s["held"].long(), s["fresh"].long(), s["page"]
    R, width = s["tables"].shape
    rows = s["position"].numel()
    kv_len = held + fresh
    first, last = (held + page - 1) // page, (kv_len + page - 1) // page
    taken = torch.cumsum(last - first, 0)
    column = torch.arange(width, device=held.device)
    rank = (taken - (last - first))[:, None] + column - first[:, None]                # which of the step's new pages
    new = (column >= first[:, None]) & (column < last[:, None])
    tables = torch.where(new, s["free"][(s["n_free"] - 1 - torch.where(new, rank, 0)).long()], s["tables"])
    ends = torch.cumsum(fresh, 0)
    starts = torch.cat([torch.zeros_like(ends[:1]), ends])
    token = torch.arange(rows, device=held.device)
    real = token < ends[-1]
    request = torch.searchsorted(ends, token, right=True).clamp(max=R - 1)
    position = torch.where(real, held[request] + token - starts[request], 0)
    slot = torch.where(real, tables[request, position // page] * page + position % page, -1)
    i32 = lambda a: a.to(torch.int32)
    return dict(tables=tables, starts=i32(starts), kv_len=i32(kv_len), position=i32(position), slot=i32(slot),
                left=i32(s["n_free"] - taken[-1:]))


def _plain_append(s):
    slot = s["slot"].long()
    for_page, row = slot // s["page"], slot % s["page"]
    s["k_pages"][for_page, :, row] = s["k"]
    s["v_pages"][for_page, :, row] = s["v"]
    return dict(k_pages=s["k_pages"], v_pages=s["v_pages"])


def _plain_attend(s):
    """All requests at once, padded to the longest: queries [R, Hk, group * new, D] against keys [R, Hk, kv, D]."""
    q, page, n, new = s["q"], s["page"], s["max_kv"], s["max_new"]
    _, H, D = q.shape
    R, Hk = s["tables"].shape[0], s["k_pages"].shape[1]
    g = H // Hk
    key = torch.arange(n, device=q.device)
    held = key < s["kv_len"][:, None]                                                  # [R, n]
    at = torch.where(held, s["tables"][:, key // page], 0).long()
    k = s["k_pages"][at, :, key % page].float().permute(0, 2, 1, 3)                    # [R, Hk, n, D]
    v = torch.where(held[:, None, :, None], s["v_pages"][at, :, key % page].float().permute(0, 2, 1, 3), 0.0)
    i = torch.arange(new, device=q.device)
    fresh = s["starts"][1:] - s["starts"][:-1]
    real = i < fresh[:, None]                                                          # [R, new]
    token = torch.where(real, s["starts"][:-1, None] + i, 0).long()
    rows = q[token].float().view(R, new, Hk, g, D).permute(0, 2, 1, 3, 4).reshape(R, Hk, new * g, D)
    score = torch.matmul(rows, k.transpose(-1, -2)) * D ** -0.5                        # [R, Hk, new * g, n]
    position = (s["kv_len"] - fresh)[:, None] + i
    seen = (held[:, None] & (key <= position[:, :, None])).repeat_interleave(g, 1)[:, None]
    score = score.masked_fill_(~seen, float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score.sub_(torch.where(top == float("-inf"), 0.0, top)))
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    o = o.view(R, Hk, new, g, D).permute(0, 2, 1, 3, 4).reshape(R, new, H, D)
    return o[real].to(q.dtype)


def _array(t):
    """A torch tensor's memory as a framework array."""
    from mytorch_b200.array import DeviceArray
    return DeviceArray(t.data_ptr(), t.shape, str(t.dtype)[6:], base=t)


def _own_tables(s):
    from mytorch_b200 import fused_ops as K
    a = {n: _array(s[n]) for n in ("held", "fresh", "tables", "free", "n_free", "starts", "kv_len", "position", "slot", "left")}
    K.fused_paged_tables(a["held"], a["fresh"], a["tables"], a["free"], a["n_free"], s["page"],
                         out=(a["starts"], a["kv_len"], a["position"], a["slot"], a["left"]))
    return {n: s[n] for n in ("tables", "starts", "kv_len", "position", "slot", "left")}


def _own_append(s):
    from mytorch_b200 import fused_ops as K
    K.fused_paged_append(_array(s["k"]), _array(s["v"]), _array(s["k_pages"]), _array(s["v_pages"]), _array(s["slot"]))
    return dict(k_pages=s["k_pages"], v_pages=s["v_pages"])


def _own_attend(s):
    from mytorch_b200 import fused_ops as K
    K.fused_paged_attention(_array(s["q"]), _array(s["k_pages"]), _array(s["v_pages"]), _array(s["tables"]), _array(s["starts"]),
                            _array(s["kv_len"]), max_new=s["max_new"], out=_array(s["o"]))
    return s["o"]


# -------------------------------------------------------------------- work ----
def work(case):
    held, fresh = _lengths(case)
    page, R, tokens = case["page"], case["requests"], sum(fresh)
    pages_of = lambda n: -(-n // page)
    if case["kind"] == "tables":
        new = sum(pages_of(h + f) - pages_of(h) for h, f in zip(held, fresh))
        # lengths, the free pages and the entries of pages that are partly filled in; entries, starts, lengths, positions, slots out
        return {"bytes": float(4 * (2 * R + 2 * new + R + 2 * R + 2 * (tokens + LOOSE))), "flops": float(8 * tokens)}
    row = case["head_dim"] * SIZE[case["dtype"]]
    if case["kind"] == "append":
        return {"bytes": float(2 * 2 * tokens * case["kv_heads"] * row + 4 * tokens), "flops": 0.0}
    kv = sum(h + f for h, f in zip(held, fresh))
    pairs = sum(f * h + f * (f + 1) / 2 for h, f in zip(held, fresh))                   # (query, key) of one head
    table = sum(pages_of(h + f) for h, f in zip(held, fresh))
    return {"bytes": float(2 * kv * case["kv_heads"] * row + 2 * tokens * case["heads"] * row + 4 * (table + 2 * R)),
            "flops": 4.0 * pairs * case["heads"] * case["head_dim"]}


# ------------------------------------------------------------------- exact ----
def exact(case, seed):
    """Request by request in 64 bits. Tables and appends hold no computed numbers."""
    if case["kind"] != "attend":
        return None
    s = prepare(case, seed)
    page, out = s["page"], []
    g = case["heads"] // case["kv_heads"]
    first = s["starts"].tolist()
    for r, n in enumerate(s["kv_len"].tolist()):
        pages = s["tables"][r, :-(-n // page)].long()
        gather = lambda pool: pool[pages].transpose(1, 2).flatten(0, 1)[:n].double().repeat_interleave(g, 1).transpose(0, 1)
        k, v = gather(s["k_pages"]), gather(s["v_pages"])                               # [H, n, D]
        q = s["q"][first[r]:first[r + 1]].double().transpose(0, 1)                      # [H, m, D]
        m = q.shape[1]
        for a in range(0, m, 256):                                                      # some rows at a time
            b = min(m, a + 256)
            z = torch.bmm(q[:, a:b], k[:, :n - m + b].transpose(1, 2)) / math.sqrt(case["head_dim"])
            late = torch.arange(n - m + b, device=z.device) > torch.arange(n - m + a, n - m + b, device=z.device)[:, None]
            z = torch.softmax(z.masked_fill(late, float("-inf")), -1)
            out.append(torch.bmm(z, v[:, :n - m + b]).transpose(0, 1))
    return torch.cat(out)
