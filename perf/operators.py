"""The paged-cache operators as a serving loop calls them, with their plain forms.

Three operators share one paged key/value cache (pages of `page_size` tokens, a
layer's K or V pool is [num_pages, Hkv, page_size, D]):

  tables     block tables, slot map and positions of a step, built on the GPU from
             the requests' lengths, pages taken from and returned to a free list;
  append     RoPE of the new tokens' q and k, and k, v written to their slots;
  attention  the new tokens of every request (a chunk, a verify block or a single
             token) over that request's pages.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # a speculative round on 8 long videos: 10 tokens appended to each, then all rejected (pages go back)
        {"name": "tables_verify_8x10", "op": "tables", "B": 8, "past_lo": 32906, "past_hi": 32906, "new_lo": 10,
         "new_hi": 10, "chunks": 0, "chunk": 0, "page": 64, "spare": 64, "lens": 1},
        # a busy server: 256 requests, most decoding, 12 with a prompt chunk; small pages
        {"name": "tables_mixed_256", "op": "tables", "B": 256, "past_lo": 1, "past_hi": 8000, "new_lo": 1,
         "new_hi": 1, "chunks": 12, "chunk": 600, "page": 16, "spare": 900, "lens": 2},
        # the q/k/v rows of a verify block: 8 requests of 10 tokens
        {"name": "append_verify_8x10", "op": "append", "B": 8, "past_lo": 32906, "past_hi": 32906, "new_lo": 10,
         "new_hi": 10, "chunks": 0, "chunk": 0, "page": 64, "Hq": 28, "Hkv": 4, "D": 128, "dtype": "bf16", "lens": 3},
        # a prompt chunk of 8192 tokens
        {"name": "append_chunk_8192", "op": "append", "B": 1, "past_lo": 8192, "past_hi": 8192, "new_lo": 8192,
         "new_hi": 8192, "chunks": 0, "chunk": 0, "page": 128, "Hq": 28, "Hkv": 4, "D": 128, "dtype": "bf16",
         "lens": 4},
        # one user, one token, a short context: latency
        {"name": "attn_one_token", "op": "attention", "B": 1, "past_lo": 199, "past_hi": 199, "new_lo": 1,
         "new_hi": 1, "chunks": 0, "chunk": 0, "page": 16, "Hq": 28, "Hkv": 4, "D": 128, "dtype": "bf16",
         "causal": True, "lse": False, "lens": 5},
        # one user, one token, a very long context: the keys have to be split over the GPU
        {"name": "attn_one_token_131k", "op": "attention", "B": 1, "past_lo": 131072, "past_hi": 131072, "new_lo": 1,
         "new_hi": 1, "chunks": 0, "chunk": 0, "page": 64, "Hq": 28, "Hkv": 4, "D": 128, "dtype": "bf16",
         "causal": True, "lse": False, "lens": 6},
        # a batch of decoding requests of all lengths, small pages
        {"name": "attn_decode_ragged_64", "op": "attention", "B": 64, "past_lo": 100, "past_hi": 8000, "new_lo": 1,
         "new_hi": 1, "chunks": 0, "chunk": 0, "page": 16, "Hq": 28, "Hkv": 4, "D": 128, "dtype": "bf16",
         "causal": True, "lse": False, "lens": 7},
        # the verify block of a speculative round on 8 long videos
        {"name": "attn_verify_8x10_33k", "op": "attention", "B": 8, "past_lo": 32896, "past_hi": 32906, "new_lo": 10,
         "new_hi": 10, "chunks": 0, "chunk": 0, "page": 64, "Hq": 28, "Hkv": 4, "D": 128, "dtype": "bf16",
         "causal": True, "lse": False, "lens": 8},
        # a server's step with a prompt chunk beside 16 decoding requests
        {"name": "attn_mixed_17", "op": "attention", "B": 17, "past_lo": 64, "past_hi": 4000, "new_lo": 1,
         "new_hi": 1, "chunks": 1, "chunk": 509, "page": 32, "Hq": 28, "Hkv": 4, "D": 128, "dtype": "bf16",
         "causal": True, "lse": False, "lens": 9},
        # a 2048-token chunk of a long prompt over what is cached of it
        {"name": "attn_chunk_2048_31k", "op": "attention", "B": 1, "past_lo": 30848, "past_hi": 30848,
         "new_lo": 2048, "new_hi": 2048, "chunks": 0, "chunk": 0, "page": 128, "Hq": 28, "Hkv": 4, "D": 128,
         "dtype": "bf16", "causal": True, "lse": False, "lens": 10},
        # a whole prompt of 8192 tokens at once
        {"name": "attn_prompt_8192", "op": "attention", "B": 1, "past_lo": 0, "past_hi": 0, "new_lo": 8192,
         "new_hi": 8192, "chunks": 0, "chunk": 0, "page": 64, "Hq": 28, "Hkv": 4, "D": 128, "dtype": "bf16",
         "causal": True, "lse": False, "lens": 11},
        # as many key heads as query heads, small heads, half precision, odd lengths, the log-sum-exp wanted too
        {"name": "attn_mha_d64_fp16", "op": "attention", "B": 5, "past_lo": 3, "past_hi": 1500, "new_lo": 33,
         "new_hi": 301, "chunks": 0, "chunk": 0, "page": 32, "Hq": 16, "Hkv": 16, "D": 64, "dtype": "fp16",
         "causal": True, "lse": True, "lens": 12},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["tables", "append", "attention", "attention"])
    page = rng.choice([16, 32, 64, 128])
    lens = rng.randrange(1 << 30)
    if op == "tables":
        B = _spread(rng, 1, 512)
        chunks = rng.choice([0, 0, 1, min(B, 5)])
        hi = _spread(rng, 16, 40000)
        return {"op": op, "B": B, "past_lo": rng.randint(0, hi), "past_hi": hi, "new_lo": rng.choice([0, 1, 1]),
                "new_hi": _spread(rng, 1, 20), "chunks": chunks, "chunk": _spread(rng, 30, 2000), "page": page,
                "spare": _spread(rng, 1, 2000), "lens": lens}
    Hq, Hkv = rng.choice([(28, 4), (28, 4), (7, 1), (16, 16), (32, 8), (12, 2), (8, 1), (40, 8)])
    case = {"op": op, "page": page, "Hq": Hq, "Hkv": Hkv, "D": rng.choice([64, 128, 128]),
            "dtype": rng.choice(["bf16", "bf16", "fp16"]), "lens": lens}
    if op == "append":
        B = _spread(rng, 1, 64)
        n = _spread(rng, 1, max(1, 8192 // B))
        hi = _spread(rng, 1, 40000)
        return {**case, "B": B, "past_lo": rng.randint(0, hi), "past_hi": hi, "new_lo": rng.randint(0, n),
                "new_hi": n, "chunks": 0, "chunk": 0}
    kind = rng.choice(["decode", "verify", "chunk", "mixed"])
    B = _spread(rng, 1, 8 if kind == "chunk" else 64)
    n = {"decode": 1, "verify": rng.randint(2, 18), "chunk": _spread(rng, 20, 4096), "mixed": 1}[kind]
    hi = _spread(rng, 1, 60000)
    chunks, chunk = (1, _spread(rng, 20, 1024)) if kind == "mixed" else (0, 0)
    while B * max(n, chunk) * Hq * (hi + max(n, chunk)) > 1.5e9 or B * hi > 400000:
        B, hi = max(1, B // 2), max(1, hi // 2)
    return {**case, "B": B, "past_lo": rng.randint(0, hi), "past_hi": hi, "new_lo": 1 if kind == "decode" else rng.randint(0, n),
            "new_hi": n, "chunks": chunks, "chunk": chunk, "causal": rng.random() < 0.8, "lse": rng.random() < 0.3}


def _lengths(case):
    """(tokens in the cache, new tokens) of each request: the same multiset for every seed."""
    rng = random.Random(case["lens"])
    pairs = []
    for b in range(case["B"]):
        new = case["chunk"] if b < case["chunks"] else rng.randint(case["new_lo"], case["new_hi"])
        pairs.append([rng.randint(case["past_lo"], case["past_hi"]), new])
    if not any(n for _, n in pairs):
        pairs[0][1] = case["new_hi"]
    return pairs


def _pages(n, page):
    return -(-n // page)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    pairs = _lengths(case)
    rng = random.Random(seed * 1000003 + 17)
    rng.shuffle(pairs)
    past, new = [p for p, _ in pairs], [n for _, n in pairs]
    page, B, T = case["page"], len(pairs), sum(new)
    held = past if case["op"] == "tables" else [p + n for p, n in pairs]
    n_blocks = [_pages(n, page) for n in held]
    width = max(_pages(p + n, page) for p, n in pairs) + 2
    num_pages = sum(n_blocks) + case.get("spare", 7)
    ids = list(range(num_pages))
    rng.shuffle(ids)
    table, at = torch.full((B, width), -1, dtype=torch.int32), 0
    for b, n in enumerate(n_blocks):
        table[b, :n] = torch.tensor(ids[at:at + n], dtype=torch.int32)
        at += n
    state = {"op": case["op"], "page": page, "tokens": T, "most": max(p + n for p, n in pairs), "most_new": max(new),
             "block_table": table.cuda(), "past": _ints(past), "new": _ints(new)}
    if case["op"] == "tables":
        state.update(n_blocks=_ints(n_blocks), free_pages=_ints(ids[at:] + ids[:at]), n_free=_ints([num_pages - at]),
                     none=_ints([0] * B))
        return state
    g = torch.Generator(device="cuda").manual_seed(seed)
    Hq, Hkv, D, dtype = case["Hq"], case["Hkv"], case["D"], DTYPES[case["dtype"]]

    def normal(*shape, by=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * by).to(dtype)

    if case["op"] == "append":
        positions = torch.cat([torch.arange(p, p + n) for p, n in pairs])
        owner = torch.cat([torch.full((n,), b) for b, n in enumerate(new)])
        slots = table[owner, positions // page].long() * page + positions % page
        inv = 1e6 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
        angle = torch.arange(state["most"] + 1, dtype=torch.float64)[:, None] * inv[None, :]
        state.update(qkv=normal(T, (Hq + 2 * Hkv) * D), positions=positions.int().cuda(), slots=slots.int().cuda(),
                     cos=angle.cos().to(dtype).cuda(), sin=angle.sin().to(dtype).cuda(), Hq=Hq, Hkv=Hkv, D=D,
                     k_pages=torch.zeros(num_pages, Hkv, page, D, dtype=dtype, device="cuda"),
                     v_pages=torch.zeros(num_pages, Hkv, page, D, dtype=dtype, device="cuda"))
        return state
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    state.update(q=normal(T, Hq, D, by=1.5), k_pages=normal(num_pages, Hkv, page, D),
                 v_pages=normal(num_pages, Hkv, page, D), cu_q=_ints(starts),
                 kv_lens=_ints([p + n for p, n in pairs]), causal=case["causal"], lse=case["lse"])
    return state


def _plain_update(s, past, new, T):
    """Block tables of one step: each request ends up with the pages that past + new tokens need."""
    page, table, held, free, n_free = s["page"], s["block_table"], s["n_blocks"], s["free_pages"], s["n_free"]
    B, width = table.shape
    num_pages, dev = free.numel(), table.device
    past, new = past.long(), new.long()
    want = (past + new + page - 1) // page
    j = torch.arange(width, device=dev)
    # returned pages go on top of the list so that the first one returned is the first one taken again
    back = (j >= want[:, None]) & (j < held[:, None])
    r = back.flatten().cumsum(0).view(B, width) - 1
    total = back.sum()
    to = torch.where(back, n_free + total - 1 - r, num_pages)
    stack = torch.cat([free, free.new_zeros(1)]).scatter(0, to.flatten(), table.flatten())[:num_pages]
    count = n_free + total
    need = (want - held).clamp(min=0)
    ok = (need == 0) | (need.cumsum(0) <= count)
    take = (j >= held[:, None]) & (j < want[:, None]) & ok[:, None]
    a = take.flatten().cumsum(0).view(B, width) - 1
    taken = stack[(count - 1 - a).clamp(min=0)]
    table.copy_(torch.where(take, taken, torch.where(back, -1, table)))
    free.copy_(stack)
    n_free.copy_(count - take.sum())
    held.copy_(torch.where(ok, want, held))
    cu_q = torch.cat([new.new_zeros(1), new.cumsum(0)])
    t = torch.arange(T, device=dev)
    b = torch.searchsorted(cu_q[1:], t, right=True)
    pos = past[b] + t - cu_q[b]
    pos = torch.where(ok[b], pos, -1)
    at = pos.clamp(min=0)
    slots = torch.where(ok[b], table[b, at // page].long() * page + at % page, -1)
    kv_lens = torch.where(ok, past + new, 0)
    return [cu_q.int(), kv_lens.int(), slots.int(), pos.int(), ok.int()]


def _plain_append(s):
    Hq, Hkv, D, page, T = s["Hq"], s["Hkv"], s["D"], s["page"], s["tokens"]
    x = s["qkv"].view(T, Hq + 2 * Hkv, D).float()
    rot, v = x[:, :Hq + Hkv], s["qkv"].view(T, Hq + 2 * Hkv, D)[:, Hq + Hkv:]
    pos, slots = s["positions"].long(), s["slots"].long()
    cos, sin = s["cos"][pos].float()[:, None], s["sin"][pos].float()[:, None]
    lo, hi = rot[..., :D // 2], rot[..., D // 2:]
    y = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1).to(s["qkv"].dtype)
    s["k_pages"][slots // page, :, slots % page] = y[:, Hq:]
    s["v_pages"][slots // page, :, slots % page] = v
    return [y[:, :Hq].contiguous(), s["k_pages"], s["v_pages"]]


def _plain_attention(s):
    q, page, L, n_max = s["q"], s["page"], s["most"], s["most_new"]
    T, Hq, D = q.shape
    Hkv, dev = s["k_pages"].shape[1], q.device
    B, G = s["kv_lens"].numel(), Hq // Hkv
    cu_q, kv_lens = s["cu_q"].long(), s["kv_lens"].long()
    new = cu_q[1:] - cu_q[:-1]
    key = torch.arange(L, device=dev)
    there = key < kv_lens[:, None]                                              # [B, L]
    pages = torch.where(there, s["block_table"][:, key // page], 0).long()
    k = s["k_pages"][pages, :, (key % page)[None, :]].float().permute(0, 2, 3, 1)   # [B, Hkv, D, L]
    v = s["v_pages"][pages, :, (key % page)[None, :]].float().permute(0, 2, 1, 3)   # [B, Hkv, L, D]
    v = torch.where(there[:, None, :, None], v, 0.0)
    t = torch.arange(n_max, device=dev)
    rows = (cu_q[:-1, None] + t).clamp(max=T - 1)
    x = q.float()[rows].view(B, n_max, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, n_max * G, D)
    p = (x @ k) / math.sqrt(D)                                                  # [B, Hkv, n * G, L]
    last = (kv_lens - new)[:, None] + t if s["causal"] else (kv_lens - 1)[:, None].expand(B, n_max)
    hidden = (key > last[:, :, None]) | ~there[:, None, :]                      # [B, n, L]
    hidden = hidden[:, None, :, None, :].expand(B, 1, n_max, G, L).reshape(B, 1, n_max * G, L)
    p.masked_fill_(hidden, -math.inf)
    m = p.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p @ v) / torch.where(total > 0, total, 1.0)
    lse = m + total.log()
    owner = torch.searchsorted(cu_q[1:], torch.arange(T, device=dev), right=True)
    mine = torch.arange(T, device=dev) - cu_q[owner]
    out = out.view(B, Hkv, n_max, G, D).permute(0, 2, 1, 3, 4)[owner, mine].reshape(T, Hq, D).to(q.dtype)
    lse = lse.view(B, Hkv, n_max, G).permute(0, 2, 1, 3)[owner, mine].reshape(T, Hq)
    return [out, lse] if s["lse"] else [out]


def run(state):
    if own:
        from std_b200 import ops
    s = state
    if s["op"] == "tables":
        tables = (s["block_table"], s["n_blocks"], s["free_pages"], s["n_free"])
        # a step's tokens are appended, then given up again: the tables end as they began
        if own:
            step = ops.paged_update(s["past"], s["new"], *tables, s["page"], s["tokens"])
            undo = ops.paged_update(s["past"], s["none"], *tables, s["page"], 0)
        else:
            step = _plain_update(s, s["past"], s["new"], s["tokens"])
            undo = _plain_update(s, s["past"], s["none"], 0)
        return [*step, undo[1], *tables]
    if s["op"] == "append":
        if not own:
            return _plain_append(s)
        q = torch.empty(s["tokens"], s["Hq"], s["D"], dtype=s["qkv"].dtype, device=s["qkv"].device)
        ops.paged_rope_append(s["qkv"], s["positions"], s["slots"], s["cos"], s["sin"], q, s["k_pages"], s["v_pages"])
        return [q, s["k_pages"], s["v_pages"]]
    if not own:
        return _plain_attention(s)
    q = s["q"]
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device) if s["lse"] else None
    out = ops.paged_attention(q, s["k_pages"], s["v_pages"], s["block_table"], s["cu_q"], s["kv_lens"],
                              causal=s["causal"], lse=lse)
    return [out, lse] if s["lse"] else [out]


def work(case):
    pairs, page = _lengths(case), case["page"]
    B, T = len(pairs), sum(n for _, n in pairs)
    if case["op"] == "tables":
        moved = sum(_pages(p + n, page) - _pages(p, page) for p, n in pairs)
        # lengths and page counts in and out, a page id moved twice each way, a slot and a position per token
        return {"bytes": 4 * (2 * (2 * B + 2 * B + 2) + 4 * B + 1 + 4 * moved + 2 * T + B), "flops": 0}
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    if case["op"] == "append":
        return {"bytes": 2 * T * (2 * (Hq + 2 * Hkv) * D + D) + 8 * T, "flops": 3 * T * (Hq + Hkv) * D}
    kv = sum(p + n for p, n in pairs if n)
    seen = sum(n * p + n * (n + 1) // 2 if case["causal"] else n * (p + n) for p, n in pairs)
    return {"bytes": 2 * (2 * T * Hq * D + 2 * kv * Hkv * D) + 4 * (3 * B + sum(_pages(p + n, page) for p, n in pairs)),
            "flops": 4 * D * Hq * seen}


def exact(case, seed):
    if case["op"] == "tables":
        return None
    s = prepare(case, seed)
    past, new, page = s["past"].tolist(), s["new"].tolist(), case["page"]
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    if case["op"] == "append":
        x = s["qkv"].double().view(-1, Hq + 2 * Hkv, 2, D // 2)
        z = torch.complex(x[:, :, 0], x[:, :, 1])
        at = s["positions"].long()
        turn = torch.complex(s["cos"].double(), s["sin"].double())[at]
        z = z[:, :Hq + Hkv] * turn[:, None]
        y = torch.cat([z.real, z.imag], -1)
        k, v = s["k_pages"].double(), s["v_pages"].double()
        rows = (s["slots"].long()[:, None] // page * Hkv + torch.arange(Hkv, device="cuda")) * page
        rows = (rows + s["slots"].long()[:, None] % page).flatten()
        k.view(-1, D)[rows] = y[:, Hq:].reshape(-1, D)
        v.view(-1, D)[rows] = s["qkv"].double().view(-1, Hq + 2 * Hkv, D)[:, Hq + Hkv:].reshape(-1, D)
        return [y[:, :Hq], k, v]
    out = torch.zeros(s["tokens"], Hq, D, dtype=torch.float64, device="cuda")
    lse = torch.full((s["tokens"], Hq), -math.inf, dtype=torch.float64, device="cuda")
    at = 0
    for b, (p, n) in enumerate(zip(past, new)):
        L = p + n
        if n and L:
            pages = s["block_table"][b, :_pages(L, page)].long()
            for h in range(Hkv):
                k = s["k_pages"][pages, h].reshape(-1, D)[:L].double()
                v = s["v_pages"][pages, h].reshape(-1, D)[:L].double()
                for g in range(Hq // Hkv):
                    head = h * (Hq // Hkv) + g
                    scores = s["q"][at:at + n, head].double() @ k.t() / math.sqrt(D)
                    if case["causal"]:
                        see = torch.ones(n, L, dtype=torch.bool, device="cuda").tril(p)
                        scores = scores.masked_fill(~see, -math.inf)
                    lse[at:at + n, head] = torch.logsumexp(scores, -1)
                    out[at:at + n, head] = torch.softmax(scores, -1) @ v
        at += n
    return [out, lse] if case["lse"] else [out]
