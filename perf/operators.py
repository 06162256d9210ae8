"""The paged serving operators, case by case: what a serving loop of the target model runs next
to the tree verification when its K/V live in pages.

  tables     block tables, slot map and positions of a step, built from the requests' lengths
             before and after it (growth, rollback and release at once)
  write      q / k RMS norm and rotary embedding of the fused projection, K / V rows written to
             their slots of the paged cache
  attention  causal attention of every request's new tokens (one to a long chunk) over its
             pages
  sample     one token per row from temperature, top-k, top-p and min-p, with a given uniform

``run`` computes an operator in its plain form (elementary torch operations in 32 bits), or,
with ``own`` set, through the package's entry points on the same state.  Sizes: the Qwen3-8B
attention shape (32 query heads, 8 key/value heads, head_dim 128) and the Qwen3-0.6B one (16
and 8), the 151936-token vocabulary, and prefixes of 1k to 32k keys as in the request mix.
"""
import math
import random

import torch

own = False

HEAD_DIM = 128
VOCAB = 151936
EPS = 1e-6
ROPE_THETA = 1e6
# weights of the sampling distribution are whole numbers of this unit (the row's largest
# weight is 2^40), so that sums do not depend on their order
UNIT = 40


# ---- the cases -----------------------------------------------------------------------------
def listed():
    return [
        # one token more for each of 64 running requests
        dict(name="tables_decode_64", op="tables", requests=64, page=16, max_pages=2048,
             lens="mix", step="decode", sizes=1),
        # a busy server's step: prompts' chunks enter, drafts roll back, requests end
        dict(name="tables_busy_1000", op="tables", requests=1000, page=16, max_pages=2048,
             lens="mix", step="busy", sizes=2),
        # 64 decoding requests' new rows
        dict(name="write_decode_64", op="write", tokens=64, q_heads=32, page=16,
             layout="heads_first", sizes=3),
        # a long prompt's rows in one step
        dict(name="write_prompt_8191", op="write", tokens=8191, q_heads=32, page=16,
             layout="heads_first", sizes=4),
        # one request answering, the smallest call of a decode loop
        dict(name="attn_decode_1", op="attention", requests=1, new=1, q_heads=32, page=16,
             layout="heads_first", low=1000, high=1000, mixed=False, sizes=5),
        # 64 requests of the mix, one token each
        dict(name="attn_decode_64", op="attention", requests=64, new=1, q_heads=32, page=16,
             layout="heads_first", low=1024, high=32768, mixed=False, sizes=6),
        # a drafted block of 16 tokens for each of 16 requests
        dict(name="attn_block_16x16", op="attention", requests=16, new=16, q_heads=32, page=32,
             layout="tokens_first", low=700, high=16000, mixed=False, sizes=7),
        # prompt chunks of four requests
        dict(name="attn_prompt_4x2048", op="attention", requests=4, new=2048, q_heads=32, page=64,
             layout="heads_first", low=2500, high=10000, mixed=False, sizes=8),
        # one prompt chunk entering among decoding requests, the Qwen3-0.6B shape
        dict(name="attn_mixed_33", op="attention", requests=33, new=1000, q_heads=16, page=16,
             layout="heads_first", low=1024, high=8192, mixed=True, sizes=9),
        # one request's next token
        dict(name="sample_1_f32", op="sample", rows=1, vocab=VOCAB, dtype="float32",
             rules="nucleus", sizes=10),
        # a batch whose requests ask for different things
        dict(name="sample_64_bf16", op="sample", rows=64, vocab=VOCAB, dtype="bfloat16",
             rules="any", sizes=11),
        # many rows, temperature alone or with min-p
        dict(name="sample_257_f32", op="sample", rows=257, vocab=VOCAB, dtype="float32",
             rules="untruncated", sizes=12),
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["tables", "write", "attention", "attention", "attention", "sample", "sample"])
    sizes = rng.randrange(1 << 30)
    page = rng.choice([16, 32, 64, 128])
    heads = rng.choice([16, 32])
    layout = rng.choice(["heads_first", "tokens_first"])
    if op == "tables":
        return dict(op=op, requests=_log_uniform(rng, 1, 1000), page=page,
                    max_pages=32768 // page, lens="mix", step=rng.choice(["decode", "busy"]),
                    sizes=sizes)
    if op == "write":
        return dict(op=op, tokens=_log_uniform(rng, 1, 8191), q_heads=heads, page=page,
                    layout=layout, sizes=sizes)
    if op == "sample":
        return dict(op=op, rows=_log_uniform(rng, 1, 257),
                    vocab=rng.choice([VOCAB, _log_uniform(rng, 1000, VOCAB)]),
                    dtype=rng.choice(["float32", "bfloat16"]),
                    rules=rng.choice(["nucleus", "any", "untruncated"]), sizes=sizes)
    kind = rng.choice(["decode", "block", "prompt", "mixed"])
    if kind == "decode":
        r, new, high = _log_uniform(rng, 1, 64), 1, _log_uniform(rng, 64, 32768)
    elif kind == "block":
        r, new, high = _log_uniform(rng, 1, 32), rng.randint(2, 33), _log_uniform(rng, 64, 16384)
    elif kind == "prompt":
        r, new, high = rng.randint(1, 4), _log_uniform(rng, 34, 2048), _log_uniform(rng, 2100, 10000)
    else:
        new, high = _log_uniform(rng, 34, 1000), _log_uniform(rng, 1100, 8192)
        r = rng.randint(2, max(2, min(33, 33 * 1000 * 8192 * 16 // (heads * new * high))))
    low = max(new, _log_uniform(rng, 1, high))
    return dict(op="attention", requests=r, new=new, q_heads=heads, page=page, layout=layout,
                low=low, high=max(low, high), mixed=kind == "mixed", sizes=sizes)


def _lengths(case):
    """The requests' lengths, from the case alone: (before, after) the step."""
    rng = random.Random(case["sizes"])
    if case["op"] == "tables":
        top = case["max_pages"] * case["page"]
        before, after = [], []
        for _ in range(case["requests"]):
            length = _log_uniform(rng, 1024, top - 1)
            if case["step"] == "decode":
                before.append(length)
                after.append(length + 1)
                continue
            what = rng.random()
            if what < 0.03:  # a prompt's first chunk
                before.append(0)
                after.append(rng.randint(1, 2048))
            elif what < 0.06:  # a later chunk
                before.append(min(length, top - 2048))
                after.append(before[-1] + rng.randint(1, 2048))
            elif what < 0.10:  # a request ends
                before.append(length)
                after.append(0)
            elif what < 0.30:  # rejected drafts roll back
                before.append(length)
                after.append(length - rng.randint(1, 16))
            elif what < 0.35:  # an idle place
                before.append(0)
                after.append(0)
            else:
                before.append(length)
                after.append(length + 1)
        return before, after
    after = [_log_uniform(rng, case["low"], case["high"]) for _ in range(case["requests"])]
    new = [case["new"]] * case["requests"]
    if case["mixed"]:  # one chunk, the others decode
        at = rng.randrange(case["requests"])
        new = [case["new"] if i == at else 1 for i in range(case["requests"])]
    elif case["new"] > 2 and case["requests"] > 1:  # the last chunks of a prompt are ragged
        new = [case["new"]] + [rng.randint(max(1, case["new"] // 2), case["new"])
                               for _ in range(case["requests"] - 1)]
    return [a - n for a, n in zip(after, new)], after


def _pages(n, page):
    return -(-n // page)


# ---- inputs --------------------------------------------------------------------------------
def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _page_pool(n_pages, kv_heads, page, layout, g):
    shape = (n_pages, kv_heads, page, HEAD_DIM) if layout == "heads_first" else \
        (n_pages, page, kv_heads, HEAD_DIM)
    t = torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    return t if layout == "heads_first" else t.permute(0, 2, 1, 3)


def _block_table(lens, page, max_pages, pages):
    """Request by request, the next pages of the list `pages` (device i32)."""
    need = torch.tensor([_pages(n, page) for n in lens], dtype=torch.int64, device="cuda")
    first = torch.cumsum(need, 0) - need
    col = torch.arange(max_pages, device="cuda")
    at = (first[:, None] + col).clamp(max=pages.numel() - 1)
    return torch.where(col < need[:, None], pages[at], 0).to(torch.int32).contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"tables": _prepare_tables, "write": _prepare_write, "attention": _prepare_attention,
            "sample": _prepare_sample}[case["op"]](case, g)


def _prepare_tables(case, g):
    before, after = _lengths(case)
    page, max_pages = case["page"], case["max_pages"]
    used = sum(_pages(n, page) for n in before)
    grown = sum(max(_pages(b, page) - _pages(a, page), 0) for a, b in zip(before, after))
    spare = grown + 64
    order = torch.randperm(used + spare, generator=g, device="cuda").to(torch.int32)
    free = torch.zeros(used + spare, dtype=torch.int32, device="cuda")
    free[:spare] = order[used:]
    tokens = sum(max(a - b, 0) for a, b in zip(after, before))
    return dict(op="tables", old_lens=_i32(before), new_lens=_i32(after),
                block_table=_block_table(before, page, max_pages, order[:max(used, 1)]),
                free_pages=free, free_count=_i32([spare]), page=page,
                max_tokens=-(-max(tokens, 1) // 64) * 64)


def _prepare_write(case, g):
    t, hq, hkv, page = case["tokens"], case["q_heads"], 8, case["page"]
    n_pages = _pages(t, page) + 8
    order = torch.randperm(n_pages, generator=g, device="cuda")
    tok = torch.arange(t, device="cuda")
    slots = order[tok // page] * page + tok % page
    start = random.Random(case["sizes"]).randrange(0, 8192)
    inv = ROPE_THETA ** (-torch.arange(0, HEAD_DIM, 2, device="cuda", dtype=torch.float32) / HEAD_DIM)
    ang = (start + tok).float()[:, None] * inv
    cos, sin = (x.to(torch.bfloat16).view(torch.int16).to(torch.int32) & 0xffff
                for x in (ang.cos(), ang.sin()))
    norm = [1 + 0.1 * torch.randn(HEAD_DIM, generator=g, device="cuda") for _ in range(2)]
    return dict(op="write",
                qkv=torch.empty((t, (hq + 2 * hkv) * HEAD_DIM), dtype=torch.bfloat16,
                                device="cuda").normal_(0, 2, generator=g),
                q_norm=norm[0].to(torch.bfloat16), k_norm=norm[1].to(torch.bfloat16),
                rope=(cos | (sin << 16)).contiguous(), slots=slots,
                k_pages=_page_pool(n_pages, hkv, page, case["layout"], g),
                v_pages=_page_pool(n_pages, hkv, page, case["layout"], g))


def _prepare_attention(case, g):
    before, after = _lengths(case)
    page, hkv = case["page"], 8
    new = [a - b for a, b in zip(after, before)]
    n_pages = sum(_pages(n, page) for n in after) + 3
    max_pages = max(_pages(n, page) for n in after)
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    return dict(op="attention",
                q=torch.empty((cu[-1], case["q_heads"], HEAD_DIM), dtype=torch.bfloat16,
                              device="cuda").normal_(generator=g),
                k_pages=_page_pool(n_pages, hkv, page, case["layout"], g),
                v_pages=_page_pool(n_pages, hkv, page, case["layout"], g),
                block_table=_block_table(after, page, max_pages, order), cu_new=_i32(cu),
                kv_lens=_i32(after), max_new=max(new), max_len=max(after))


def _prepare_sample(case, g):
    rng = random.Random(case["sizes"])
    rows, vocab = case["rows"], case["vocab"]
    logits = torch.empty((rows, vocab), device="cuda").normal_(0, 3, generator=g)
    # a few tokens stand out, as in a trained model's answers
    top = torch.randint(0, vocab, (rows, 8), generator=g, device="cuda")
    logits.scatter_add_(1, top, torch.rand((rows, 8), generator=g, device="cuda") * 10)
    rules = case["rules"]
    temp, k, p, mp = [], [], [], []
    for _ in range(rows):
        what = rng.random()
        temp.append(0.0 if rules == "any" and what < 0.1 else rng.choice([0.6, 0.8, 1.0, 1.3]))
        k.append(rng.choice([0, 1, 20, 50, 1000]) if rules == "any" else
                 rng.choice([0, 50]) if rules == "nucleus" else 0)
        p.append(rng.choice([1.0, 0.5, 0.9, 0.95]) if rules == "any" else
                 0.95 if rules == "nucleus" else 1.0)
        mp.append(rng.choice([0.0, 0.05]) if rules != "nucleus" else 0.0)
    f32 = dict(dtype=torch.float32, device="cuda")
    return dict(op="sample", logits=logits.to(getattr(torch, case["dtype"])),
                u=torch.rand(rows, generator=g, device="cuda"), temperature=torch.tensor(temp, **f32),
                top_k=_i32(k), top_p=torch.tensor(p, **f32), min_p=torch.tensor(mp, **f32))


# ---- one pass ------------------------------------------------------------------------------
def run(s):
    if own:
        return _own(s)
    return {"tables": _plain_tables, "write": _plain_write, "attention": _plain_attention,
            "sample": _plain_sample}[s["op"]](s)


def _own(s):
    from mdflash_b200 import kernels as K
    if s["op"] == "tables":
        step = K.page_tables(s["old_lens"], s["new_lens"], s["block_table"], s["free_pages"],
                             s["free_count"], s["page"], s["max_tokens"])
        return dict(kv_lens=step.kv_lens, cu_new=step.cu_new, slot_map=step.slot_map,
                    positions=step.positions, free_count=step.free_count,
                    block_table=s["block_table"], free_pages=s["free_pages"])
    if s["op"] == "write":
        q = K.paged_qk_norm_rope(s["qkv"], s["q_norm"], s["k_norm"], s["rope"], s["slots"],
                                 s["k_pages"], s["v_pages"], EPS)
        return dict(q=q, k_pages=s["k_pages"], v_pages=s["v_pages"])
    if s["op"] == "attention":
        return K.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["block_table"], s["cu_new"],
                                 s["kv_lens"], s["max_new"])
    tokens, logprobs = K.sample(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"],
                                s["min_p"])
    return dict(tokens=tokens, logprobs=logprobs)


def _plain_tables(s):
    """Pages that a request gives back go on top of the free stack (requests in order, a
    request's pages in order); then the pages it needs are taken from the top."""
    page, table, free = s["page"], s["block_table"].long(), s["free_pages"].long()
    old, new, count = s["old_lens"].long(), s["new_lens"].long(), s["free_count"].long()
    dev = old.device
    had, needs = (old + page - 1) // page, (new + page - 1) // page
    back, more, toks = (x.clamp(min=0) for x in (had - needs, needs - had, new - old))
    back_c, more_c, toks_c = (torch.cumsum(x, 0) for x in (back, more, toks))
    ok = (old.amin() >= 0) & (new.amin() >= 0) & (needs.amax() <= table.shape[1]) & \
        (count[0] + back_c[-1] >= more_c[-1]) & (toks_c[-1] <= s["max_tokens"])
    # the stack after the pages given back
    j = torch.arange(free.numel(), device=dev) - count
    r = torch.searchsorted(back_c, j, right=True).clamp(max=old.numel() - 1)
    col = (needs[r] + j - (back_c - back)[r]).clamp(0, table.shape[1] - 1)
    free = torch.where((j >= 0) & (j < back_c[-1]) & ok, table[r, col], free)
    # the pages taken
    c = torch.arange(table.shape[1], device=dev)
    at = count + back_c[-1] - 1 - ((more_c - more)[:, None] + c - had[:, None])
    takes = (c >= had[:, None]) & (c < needs[:, None]) & ok
    table = torch.where(takes, free[at.clamp(0, free.numel() - 1)], table)
    # the new tokens
    t = torch.arange(s["max_tokens"], device=dev)
    r = torch.searchsorted(toks_c, t, right=True).clamp(max=old.numel() - 1)
    pos = old[r] + t - (toks_c - toks)[r]
    live = (t < toks_c[-1]) & ok
    slot = table[r, (pos // page).clamp(0, table.shape[1] - 1)] * page + pos % page
    zero = torch.zeros(1, dtype=torch.int64, device=dev)
    return dict(kv_lens=torch.where(ok, new, old).int(),
                cu_new=torch.where(ok, torch.cat([zero, toks_c]), 0).int(),
                slot_map=torch.where(live, slot, -1), positions=torch.where(live, pos, 0),
                free_count=torch.where(ok, count + back_c[-1] - more_c[-1], count).int(),
                block_table=table.int(), free_pages=free.int())


def _plain_write(s):
    k_pages, v_pages, page = s["k_pages"], s["v_pages"], s["k_pages"].shape[2]
    hkv = k_pages.shape[1]
    x = s["qkv"].view(s["qkv"].shape[0], -1, HEAD_DIM).float()
    hq = x.shape[1] - 2 * hkv
    half = HEAD_DIM // 2
    cos = (s["rope"] << 16).view(torch.float32)[:, None]
    sin = (s["rope"] & -65536).view(torch.float32)[:, None]
    w = torch.cat([s["q_norm"].float().expand(hq, HEAD_DIM), s["k_norm"].float().expand(hkv, HEAD_DIM)])
    qk = x[:, :hq + hkv]
    qk = qk / torch.sqrt((qk * qk).mean(-1, keepdim=True) + EPS) * w
    a, b = qk[..., :half], qk[..., half:]
    qk = torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(torch.bfloat16)
    pid, row = s["slots"] // page, s["slots"] % page
    k_pages[pid, :, row] = qk[:, hq:]
    v_pages[pid, :, row] = x[:, hq + hkv:].to(torch.bfloat16)
    return dict(q=qk[:, :hq].contiguous(), k_pages=k_pages, v_pages=v_pages)


def _plain_attention(s):
    k_pages, page, hkv = s["k_pages"], s["k_pages"].shape[2], s["k_pages"].shape[1]
    cu, lens = s["cu_new"].long(), s["kv_lens"].long()
    t, hq, d = s["q"].shape
    r, n, m = lens.numel(), s["max_new"], s["max_len"]
    dev = cu.device
    new = cu[1:] - cu[:-1]
    row = torch.arange(n, device=dev)
    q = s["q"][(cu[:-1, None] + row).clamp(max=t - 1)].float()             # [r, n, hq, d]
    q = q.view(r, n, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(r, hkv, -1, d)
    key = torch.arange(m, device=dev)
    there = key < lens[:, None]                                             # [r, m]
    pid = torch.where(there, s["block_table"].long()[:, key // page], 0)
    k = k_pages[pid, :, key % page].permute(0, 2, 3, 1).float()             # [r, hkv, d, m]
    p = torch.matmul(q, k).view(r, hkv, -1, n, m)
    del k
    sees = there[:, None] & (key <= (lens - new)[:, None, None] + row[:, None])  # [r, n, m]
    p = (p * d ** -0.5).masked_fill_(~sees[:, None, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    p = torch.exp(p.sub_(torch.where(top > -math.inf, top, 0)))
    total = p.sum(-1, keepdim=True)
    v = s["v_pages"][pid, :, key % page].permute(0, 2, 1, 3).float()        # [r, hkv, m, d]
    o = torch.matmul(p.view(r, hkv, -1, m), v.masked_fill_(~there[:, None, :, None], 0))
    o = o.view(r, hkv, -1, n, d) / torch.where(total > 0, total, 1)
    o = o.permute(0, 3, 1, 2, 4).reshape(r, n, hq, d)
    tok = torch.arange(t, device=dev)
    req = torch.searchsorted(cu[1:], tok, right=True).clamp(max=r - 1)
    return o[req, tok - cu[req]].to(torch.bfloat16)


def _plain_sample(s):
    """The kept tokens are the first ones by (logit descending, index ascending): top_k of
    them, of these the fewest that hold top_p of their weight, of these the ones with at
    least min_p of the largest weight.  The token is the first by index whose running weight
    exceeds floor(u * total).  Temperatures below 1e-5 keep the first token alone; NaN counts
    as -inf; a row without a finite or +inf logit gives token -1."""
    x = s["logits"].float()
    rows, vocab = x.shape
    x = torch.where(torch.isnan(x), -math.inf, x)
    top = x.amax(-1, keepdim=True)
    greedy = s["temperature"][:, None] < 1e-5
    z = torch.where(x == top, 0.0, (x - top) / torch.where(greedy, 1.0, s["temperature"][:, None]))
    w = torch.exp(z)
    weight = (w * 2.0 ** UNIT).long()
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    rank = torch.arange(vocab, device=x.device)
    k = torch.where(greedy, 1, torch.where(s["top_k"] > 0, s["top_k"], vocab)[:, None])
    by_rank = torch.where(rank < k, weight.gather(1, order), 0)
    before = torch.cumsum(by_rank, -1) - by_rank
    p = s["top_p"].double()[:, None]
    fits = (p >= 1) | (before.double() < p * by_rank.sum(-1, keepdim=True).double())
    keep = (rank < k) & (fits | (rank == 0))
    keep = torch.zeros_like(keep).scatter_(1, order, keep) & \
        (w >= s["min_p"].clamp(max=1.0)[:, None])
    weight = torch.where(keep, weight, 0)
    running = torch.cumsum(weight, -1)
    total = running[:, -1:]
    target = (s["u"].double()[:, None] * total.double()).floor().long()
    target = torch.minimum(target, total - 1).clamp(min=0)
    token = (running <= target).sum(-1, keepdim=True).clamp(max=vocab - 1)
    logp = z.gather(1, token).double() - (total.double().log() - UNIT * math.log(2.0))
    empty = top == -math.inf
    return dict(tokens=torch.where(empty, -1, token)[:, 0],
                logprobs=torch.where(empty, -math.inf, logp).float()[:, 0])


# ---- what a pass cannot do without -----------------------------------------------------------
def work(case):
    if case["op"] == "tables":
        before, after = _lengths(case)
        page = case["page"]
        had, needs = (sum(_pages(n, page) for n in v) for v in (before, after))
        back = sum(max(_pages(b, page) - _pages(a, page), 0) for a, b in zip(after, before))
        tokens = sum(max(a - b, 0) for a, b in zip(after, before))
        taken = needs - had + back
        # lengths in and out, offsets; a page id read and written per page moved; the pages of
        # the new tokens read once, a slot and a position written per token
        return dict(bytes=4 * (4 * len(before) + 3) + 8 * (back + taken) + 16 * tokens, flops=0)
    if case["op"] == "write":
        t, hq, hkv = case["tokens"], case["q_heads"], 8
        row = 2 * HEAD_DIM
        return dict(bytes=t * (2 * (hq + 2 * hkv) * row + 4 * (HEAD_DIM // 2) + 8) + 2 * row,
                    flops=t * (hq + hkv) * HEAD_DIM * 8)
    if case["op"] == "sample":
        size = 4 if case["dtype"] == "float32" else 2
        return dict(bytes=case["rows"] * (case["vocab"] * size + 32), flops=0)
    before, after = _lengths(case)
    hq, hkv = case["q_heads"], 8
    seen = sum((a - b) * b + (a - b) * (a - b + 1) // 2 for a, b in zip(after, before))
    tokens = sum(a - b for a, b in zip(after, before))
    return dict(bytes=sum(after) * 2 * hkv * HEAD_DIM * 2 + 2 * tokens * hq * HEAD_DIM * 2 +
                4 * sum(_pages(n, case["page"]) for n in after),
                flops=4 * hq * HEAD_DIM * seen)


# ---- the definitions in 64 bits -----------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "tables":
        return None
    return {"write": _exact_write, "attention": _exact_attention, "sample": _exact_sample}[case["op"]](s)


def _exact_write(s):
    k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
    hkv, page = k_pages.shape[1], k_pages.shape[2]
    x = s["qkv"].double().unflatten(1, (-1, HEAD_DIM))
    hq = x.shape[1] - 2 * hkv
    bits = s["rope"]
    words = torch.stack([bits & 0xffff, (bits >> 16) & 0xffff]).to(torch.int32)
    cos, sin = ((w << 16).view(torch.float32).double() for w in words)
    angle = torch.complex(cos, sin)[:, None]                                # [t, 1, 64]

    def turned(heads, weight):
        rms = heads.pow(2).mean(-1, keepdim=True).add(EPS).sqrt()
        y = heads / rms * weight.double()
        y = torch.complex(y[..., :HEAD_DIM // 2].contiguous(), y[..., HEAD_DIM // 2:].contiguous()) * angle
        return torch.cat([y.real, y.imag], -1)

    slots = s["slots"]
    pid, row = torch.div(slots, page, rounding_mode="floor"), torch.remainder(slots, page)
    k_pages[pid, :, row] = turned(x[:, hq:hq + hkv], s["k_norm"])
    v_pages[pid, :, row] = x[:, hq + hkv:]
    return dict(q=turned(x[:, :hq], s["q_norm"]), k_pages=k_pages, v_pages=v_pages)


def _exact_attention(s):
    q, cu, lens = s["q"].double(), s["cu_new"].tolist(), s["kv_lens"].tolist()
    page, hkv = s["k_pages"].shape[2], s["k_pages"].shape[1]
    group = q.shape[1] // hkv
    out = torch.zeros_like(q)
    for r, length in enumerate(lens):
        n = cu[r + 1] - cu[r]
        ids = s["block_table"][r, :_pages(length, page)].long()
        for h in range(hkv):
            k = s["k_pages"][ids, h].reshape(-1, HEAD_DIM)[:length].double()
            v = s["v_pages"][ids, h].reshape(-1, HEAD_DIM)[:length].double()
            qh = q[cu[r]:cu[r + 1], h * group:(h + 1) * group].transpose(0, 1)  # [group, n, d]
            a = qh @ k.T / math.sqrt(HEAD_DIM)
            hidden = torch.ones(n, length, dtype=torch.bool, device=q.device).triu(length - n + 1)
            out[cu[r]:cu[r + 1], h * group:(h + 1) * group] = \
                (a.masked_fill(hidden, -math.inf).softmax(-1) @ v).transpose(0, 1)
    return out


def _exact_sample(s):
    """Row by row, with real weights in the place of whole numbers of a unit."""
    logp = []
    x = s["logits"].double()
    rules = [s[k].tolist() for k in ("u", "temperature", "top_k", "top_p", "min_p")]
    for row, (u, temp, k, p, min_p) in zip(x, zip(*rules)):
        if temp < 1e-5:
            logp.append(0.0)
            continue
        value, index = row.sort(descending=True, stable=True)
        w = ((value - value[0]) / temp).exp()
        n = min(k, w.numel()) if k > 0 else w.numel()
        w = w[:n]
        if p < 1:
            n = max(int((w.cumsum(0) - w < p * w.sum()).sum()), 1)
        n = min(n, int((w >= min(min_p, 1.0)).sum()))
        w, index = w[:n], index[:n]
        at = index.argsort()
        running = w[at].cumsum(0)
        pick = min(int((running <= u * running[-1]).sum()), n - 1)
        logp.append(float((w[at][pick] / running[-1]).log()))
    return dict(tokens=None, logprobs=torch.tensor(logp, dtype=torch.float64))
