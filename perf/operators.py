"""Cases for the serving operators: block tables and slot maps built on the GPU from request lengths,
a paged KV cache held in 4 bits (append and read back), and sliding-window + global-token attention of
new tokens over that cache.

The cache.  A pool is a uint8 tensor [pages, kv_heads, page_size, head_dim + 8]; page_size is a multiple
of 16.  One (page, head) is page_size / 16 blocks of 16 tokens, each block 16 * (head_dim + 8) bytes:

    K codes [16][head_dim / 2] | V codes [16][head_dim / 2] | K words [16] | V words [16]

A code row is head_dim / 8 little-endian 32-bit words; bits 4j .. 4j+3 of word i hold element 8i + j.
A word is an fp32 scale whose low four bits hold the zero point z; an element is scale * (code - z).
A row is quantised over [min(row, 0), max(row, 0)]: scale = hi/15 - lo/15 (as products with fp32 1/15)
with its low four bits cleared, z = rint(-lo / scale), code = clamp(rint(x / scale) + z, 0, 15), with
x / scale the fp32 product x * (1 / scale).  A row whose scale is below the smallest normal number is
stored as zeros.
"""
import math
import random

import torch

own = False

BLOCK = 16


# ---------------------------------------------------------------------------------- cases


def listed():
    return [
        # one decoding step of 64 requests, each up to 128K tokens long: only latency counts
        {"name": "layout decode 64", "op": "layout", "batch": 64, "rows": 64, "page": 64, "table": 2048, "longest": 131000,
         "mix": "decode", "spare": 1.0, "lens_seed": 1},
        # a continuous-batching step: decoding, idle and prompt-chunk requests, padded to a captured capacity
        {"name": "layout mixed 256", "op": "layout", "batch": 256, "rows": 8192, "page": 32, "table": 1024,
         "longest": 16384, "mix": "mixed", "spare": 1.0, "lens_seed": 2},
        # prompts of 512 requests at once, with a pool too small for the last of them
        {"name": "layout prompts 512", "op": "layout", "batch": 512, "rows": 131072, "page": 16, "table": 512,
         "longest": 1000, "mix": "prompts", "spare": 0.9, "lens_seed": 3},
        # one new token of each of 64 decoding requests, grouped heads
        {"name": "append decode 64", "op": "append", "rows": 64, "tokens": 64, "kv_heads": 8, "dim": 128, "page": 64,
         "type": "bf16"},
        # a prompt of odd length into small pages, rows padded behind the last token
        {"name": "append prompt 16k", "op": "append", "rows": 16384, "tokens": 16127, "kv_heads": 16, "dim": 64, "page": 32,
         "type": "fp16"},
        # a 128K-token context in one call
        {"name": "append context 128k", "op": "append", "rows": 131072, "tokens": 131072, "kv_heads": 8, "dim": 128,
         "page": 128, "type": "bf16"},
        # the smallest: one request, one token, a band and three globals of a 16K context
        {"name": "decode one 16k", "op": "attention", "batch": 1, "new": 1, "longest": 16384, "shortest": 16384,
         "heads": 16, "kv_heads": 16, "dim": 64, "page": 64, "window": 256, "globals": "range:3", "type": "fp16",
         "out": "fp16", "lse": False, "lens_seed": 4},
        # a batch of 4K contexts with 12 heads each, fp32 output
        {"name": "decode batch 4k", "op": "attention", "batch": 64, "new": 1, "longest": 4096, "shortest": 700,
         "heads": 12, "kv_heads": 12, "dim": 64, "page": 16, "window": 256, "globals": "range:1", "type": "bf16",
         "out": "fp32", "lse": False, "lens_seed": 5},
        # 65 global tokens scattered over 64K contexts
        {"name": "decode many globals 64k", "op": "attention", "batch": 32, "new": 1, "longest": 65536,
         "shortest": 60000, "heads": 16, "kv_heads": 16, "dim": 64, "page": 64, "window": 256, "globals": "random:65",
         "type": "bf16", "out": "bf16", "lse": True, "lens_seed": 6},
        # ragged whole-context decoding (the window covers everything), four query heads to a KV head
        {"name": "decode whole ragged", "op": "attention", "batch": 16, "new": 1, "longest": 131072, "shortest": 1000,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "window": 131072, "globals": "range:0", "type": "bf16",
         "out": "bf16", "lse": False, "lens_seed": 7},
        # a few drafted tokens verified over one whole 128K context
        {"name": "verify whole 128k", "op": "attention", "batch": 1, "new": 4, "longest": 131072, "shortest": 131072,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 128, "window": 131072, "globals": "range:0", "type": "fp16",
         "out": "fp16", "lse": True, "lens_seed": 8},
        # chunks of four prompts over 128K contexts, window 512 and 16 globals
        {"name": "chunk 2k of 128k", "op": "attention", "batch": 4, "new": 2048, "longest": 131072, "shortest": 20000,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "window": 512, "globals": "range:16", "type": "bf16",
         "out": "bf16", "lse": False, "lens_seed": 9},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["layout", "append", "attention", "attention"])
    if op == "layout":
        mix = rng.choice(["decode", "mixed", "prompts"])
        batch, page = _log(rng, 1, 512), rng.choice([16, 32, 48, 64, 128])
        rows = batch if mix == "decode" else max(batch, _log(rng, 64, 131072))
        longest = _log(rng, 500, 131000) if mix == "decode" else _log(rng, 100, 16000)
        return {"op": op, "batch": batch, "rows": rows, "page": page, "table": -(-(longest + 1) // page) + rng.randint(0, 300),
                "longest": longest, "mix": mix, "spare": rng.choice([0.7, 1.0, 1.0]), "lens_seed": rng.randrange(1 << 30)}
    if op == "append":
        tokens = _log(rng, 1, 65536)
        return {"op": op, "rows": tokens + rng.choice([0, 0, rng.randint(1, 200)]), "tokens": tokens,
                "kv_heads": rng.choice([1, 2, 5, 8, 12, 16]), "dim": rng.choice([64, 128]),
                "page": rng.choice([16, 32, 48, 64, 128]), "type": rng.choice(["fp16", "bf16"])}
    kind = rng.choice(["band", "band", "whole", "chunk"])
    kv_heads = rng.choice([1, 2, 3, 8, 12, 16])
    group = rng.choice([1, 1, 2, 4, 5, 8])
    dim = rng.choice([64, 128])
    case = {"op": op, "kv_heads": kv_heads, "heads": kv_heads * group, "dim": dim, "page": rng.choice([16, 32, 48, 64, 128]),
            "type": rng.choice(["fp16", "bf16"]), "lse": rng.random() < 0.5, "lens_seed": rng.randrange(1 << 30)}
    case["out"] = rng.choice([case["type"], "fp32"])
    if kind == "whole":
        batch = _log(rng, 1, 32)
        longest = _log(rng, 300, min(131072, 10 ** 9 // (batch * kv_heads * dim)))
        window, glob, new = 131072, "range:0", rng.choice([1, 1, 2, 4])
    elif kind == "band":
        batch, new = _log(rng, 1, 128), rng.choice([1, 1, 1, 3, 8])
        longest = _log(rng, 400, min(65536, 2 * 10 ** 9 // (batch * kv_heads * dim)))
        window, glob = rng.choice([0, 64, 128, 256, 512]), rng.choice(["range:0", "range:1", "range:3", "random:17", "random:65"])
    else:
        batch, longest, new = rng.randint(1, 4), _log(rng, 1500, 65536), _log(rng, 16, 1000)
        window, glob = rng.choice([64, 128, 256, 512]), rng.choice(["range:0", "range:3", "range:16", "random:17"])
        new = max(16, min(new, 16 * 10 ** 9 // (batch * case["heads"] * (window + new) * dim)))
    case.update(batch=batch, longest=longest, shortest=max(new + 100, longest // rng.choice([1, 2, 10])), new=new,
                window=window, globals=glob)
    case["shortest"] = min(case["shortest"], longest)
    return case


TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _lens(case):
    """The lengths that a case stands for: cached tokens and new tokens of each request."""
    r = random.Random(case["lens_seed"])
    if case["op"] == "attention":
        lens = [r.randint(case["shortest"], case["longest"]) for _ in range(case["batch"])]
        return [n - case["new"] for n in lens], [case["new"]] * case["batch"]
    batch, left = case["batch"], case["rows"]
    cached, new = [], []
    for b in range(batch):
        if case["mix"] == "decode":
            cached.append(r.randint(1, case["longest"]))
            new.append(1)
            continue
        kind = r.random() if case["mix"] == "mixed" else 1.0
        if kind < 0.6:
            cached.append(r.randint(1, case["longest"]))
            n = 1
        elif kind < 0.7:
            cached.append(r.randint(1, case["longest"]))
            n = 0
        else:
            cached.append(0 if kind > 0.8 else r.randint(1, case["longest"]))
            n = r.randint(1, max(1, 2 * case["rows"] // batch))
        n = max(0, min(n, left, case["longest"] + 1 - cached[-1]))
        left -= n
        new.append(n)
    return cached, new


def _global_tokens(case):
    kind, count = case["globals"].split(":")
    count = int(count)
    below = case["shortest"] - case["new"]  # a new token is never a global one itself
    if kind == "range":
        return list(range(min(count, below)))
    return sorted(random.Random(case["lens_seed"] + 1).sample(range(below), min(count, below)))


# ---------------------------------------------------------------------------------- inputs


def _rows(shape, gen, kind):
    """Key or value rows: a few channels far larger than the others, as keys have, and rows of different sizes."""
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    channel = 0.6 + torch.rand((1, shape[-2], shape[-1]), generator=gen, device="cuda")
    if kind == "k":
        channel = channel + 3.0 * (torch.rand(channel.shape, generator=gen, device="cuda") < 0.03)
    return x * channel * (0.5 + torch.rand(shape[:-1] + (1,), generator=gen, device="cuda"))


def _quantised(x):
    """Codes [.., dim] int32 and words [..] int32 of fp32 rows."""
    hi, lo = x.amax(-1).clamp_min(0.0), x.amin(-1).clamp_max(0.0)
    scale = hi * (1.0 / 15.0) - lo * (1.0 / 15.0)
    scale = (scale.view(torch.int32) & ~15).view(torch.float32)
    scale = torch.where(scale >= torch.finfo(torch.float32).tiny, scale, torch.zeros_like(scale))
    inverse = torch.where(scale > 0, 1.0 / scale, torch.zeros_like(scale))
    zero = torch.round(-lo * inverse)
    codes = (torch.round(x * inverse[..., None]) + zero[..., None]).clamp(0, 15).to(torch.int32)
    return codes, scale.view(torch.int32) | zero.to(torch.int32)


def _values(codes, words):
    """fp32 values of codes [.., dim] under words [..]."""
    scale = (words & ~15).view(torch.float32)
    return (codes - (words & 15)[..., None]).to(torch.float32) * scale[..., None]


def _packed(codes):
    """Codes [.., dim] as words [.., dim / 8] int32."""
    shifts = torch.arange(0, 32, 4, device=codes.device, dtype=torch.int64)
    words = (codes.view(*codes.shape[:-1], -1, 8).to(torch.int64) << shifts).sum(-1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)


def _filled_pool(pages, kv_heads, page, dim, gen):
    """A pool of quantised random rows."""
    pool = torch.empty(pages, kv_heads, page, dim + 8, dtype=torch.uint8, device="cuda")
    words = pool.view(pages, -1).view(torch.int32).view(pages, kv_heads, page // BLOCK, BLOCK * (dim + 8) // 4)
    step = max(1, (1 << 25) // (kv_heads * page * dim))
    half = BLOCK * dim // 8
    for at in range(0, pages, step):
        part = words[at:at + step]
        for k, kind in enumerate("kv"):
            x = _rows((part.shape[0] * page, kv_heads, dim), gen, kind)
            codes, scales = _quantised(x.view(part.shape[0], page, kv_heads, dim).transpose(1, 2))
            shape = (part.shape[0], kv_heads, page // BLOCK)
            part[..., k * half:(k + 1) * half] = _packed(codes).reshape(*shape, half)
            part[..., 2 * half + k * BLOCK:2 * half + (k + 1) * BLOCK] = scales.reshape(*shape, BLOCK)
    return pool


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "layout":
        cached, new = _lens(case)
        page, table = case["page"], case["table"]
        held = [-(-c // page) for c in cached]
        need = sum(-(-(c + n) // page) - h for c, n, h in zip(cached, new, held))
        free = max(1, int(need * case["spare"]))
        order = torch.randperm(sum(held) + free, generator=gen, device="cuda").to(torch.int32)
        block_table = torch.full((case["batch"], table), -1, dtype=torch.int32, device="cuda")
        slot = torch.arange(table, device="cuda")[None, :] < _ints(held)[:, None]
        block_table[slot] = order[:sum(held)]
        return {"case": case, "block_table": block_table, "seq_lens": _ints(cached), "new_lens": _ints(new),
                "free_pages": torch.cat([order[sum(held):], order[:sum(held)]]), "free_count": _ints([free])}
    dim, kv_heads, page, dtype = case["dim"], case["kv_heads"], case["page"], TYPES[case["type"]]
    if case["op"] == "append":
        rows, tokens = case["rows"], case["tokens"]
        pages = -(-tokens // page) + 1
        order = torch.randperm(pages, generator=gen, device="cuda")
        at = torch.arange(rows, device="cuda")
        slots = torch.where(at < tokens, order[at.clamp_max(tokens - 1) // page] * page + at % page, -1).to(torch.int32)
        k, v = (_rows((rows, kv_heads, dim), gen, kind).to(dtype) for kind in "kv")
        return {"case": case, "pool": torch.zeros(pages, kv_heads, page, dim + 8, dtype=torch.uint8, device="cuda"),
                "k": k, "v": v, "slots": slots, "out": dtype}
    cached, new = _lens(case)
    lens = [c + n for c, n in zip(cached, new)]
    held = [-(-n // page) for n in lens]
    pages = sum(held)
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    block_table = torch.full((case["batch"], max(held)), -1, dtype=torch.int32, device="cuda")
    block_table[torch.arange(max(held), device="cuda")[None, :] < _ints(held)[:, None]] = order
    rows = sum(new)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    q = torch.randn(rows, case["heads"], dim, generator=gen, device="cuda").to(dtype)
    return {"case": case, "pool": _filled_pool(pages, kv_heads, page, dim, gen), "block_table": block_table,
            "kv_lens": _ints(lens), "cu_seqlens": _ints(cu), "q": q, "globals": _global_tokens(case),
            "scale": 1.0 / math.sqrt(dim), "out": TYPES[case["out"]]}


# ---------------------------------------------------------------------------------- one pass


def run(state):
    case = state["case"]
    if own:
        import os
        import sys
        package = os.path.join(os.getcwd(), "long-context-attention-kernels_b200", "python")
        if package not in sys.path:
            sys.path.insert(0, package)
        import long_context_attention as lca
        if case["op"] == "layout":
            step = lca.kv_cache_layout(state["block_table"], state["seq_lens"], state["new_lens"], state["free_pages"],
                                       state["free_count"], case["page"], case["rows"])
            return {"block_table": state["block_table"], "slots": step.slots, "positions": step.positions,
                    "cu_seqlens": step.cu_seqlens, "kv_lens": step.kv_lens, "placed": step.placed,
                    "seq_lens": step.seq_lens, "free_count": step.free_count}
        if case["op"] == "append":
            lca.kv_cache_append(state["pool"], state["k"], state["v"], state["slots"])
            k, v = lca.kv_cache_read(state["pool"], state["slots"], out_dtype=state["out"])
            return {"k": k, "v": v}
        got = lca.sliding_window_attention_cached(state["q"], state["pool"], state["block_table"], state["kv_lens"],
                                                  state["cu_seqlens"], case["window"], state["globals"], state["scale"],
                                                  out_dtype=state["out"], return_lse=case["lse"])
        return {"out": got[0], "lse": got[1]} if case["lse"] else {"out": got}
    if case["op"] == "layout":
        return _plain_layout(state, case)
    if case["op"] == "append":
        return _plain_append(state)
    return _plain_attention(state, case)


def _plain_layout(state, case):
    page, rows = case["page"], case["rows"]
    table, free_pages = state["block_table"], state["free_pages"]
    batch, width = table.shape
    cached, want = state["seq_lens"].long().clamp_min(0), state["new_lens"].long().clamp_min(0)
    end = want.cumsum(0)
    fits = (end <= rows) & (cached + want <= width * page)
    held = (cached + page - 1) // page
    need = torch.where(fits, (cached + want + page - 1) // page - held, 0)
    taken = need.cumsum(0)
    count = state["free_count"].long().clamp(0, free_pages.numel())
    fits = fits & ((need == 0) | (taken <= count))
    end = end.clamp_max(rows)
    start = torch.cat([end.new_zeros(1), end[:-1]])
    at = torch.arange(rows, device=table.device)
    owner = torch.searchsorted(end, at, right=True)
    inside = owner < batch
    owner = owner.clamp_max(batch - 1)
    inside = inside & fits[owner]
    pos = cached[owner] + at - start[owner]
    pi = torch.where(inside, pos // page, 0)
    fresh = (count - 1 - ((taken - need)[owner] + pi - held[owner])).clamp(0, free_pages.numel() - 1)
    pages = torch.where(pi < held[owner], table[owner, pi], free_pages[fresh]).long()
    flat = torch.cat([table.view(-1), table.new_zeros(1)])
    flat[torch.where(inside, owner * width + pi, batch * width)] = pages.int()
    table.copy_(flat[:-1].view_as(table))
    slots = torch.where(inside & (pages >= 0), pages * page + pos % page, -1)
    return {"block_table": table, "slots": slots.int(), "positions": torch.where(inside, pos, -1).int(),
            "cu_seqlens": torch.cat([start, end[-1:]]).int(), "kv_lens": torch.where(fits, cached + want, 0).int(),
            "placed": torch.where(fits, want, 0).int(), "seq_lens": torch.where(fits, cached + want, cached).int(),
            "free_count": (count - torch.where(fits, need, 0).sum()).int()}


def _plain_append(state):
    kept = (state["slots"] >= 0)[:, None, None]
    return {name: torch.where(kept, _values(*_quantised(state[name].float())), 0.0).to(state["out"]) for name in ("k", "v")}


def _unpacked(words):
    shifts = torch.arange(0, 32, 4, device=words.device, dtype=torch.int32)
    return ((words[..., None] >> shifts) & 15).flatten(-2)


def _plain_attention(state, case):
    pool, table, lens, q = state["pool"], state["block_table"], state["kv_lens"].long(), state["q"]
    pages, kv_heads, page, dim = pool.shape[0], pool.shape[1], pool.shape[2], pool.shape[3] - 8
    batch, new, window = case["batch"], case["new"], case["window"]
    group = case["heads"] // kv_heads
    device = q.device
    # the keys that some new token of a request sees: the globals before its band, then the band
    span = min(case["longest"], window + new)
    first = (lens - span).clamp_min(0)
    ahead = torch.tensor(state["globals"], dtype=torch.long, device=device)
    key = torch.cat([ahead[None, :].expand(batch, -1), first[:, None] + torch.arange(span, device=device)], 1)
    there = torch.cat([ahead[None, :] < first[:, None], key[:, len(state["globals"]):] < lens[:, None]], 1)
    is_global = torch.zeros(case["longest"] + span + 1, dtype=torch.bool, device=device)
    is_global[ahead] = True
    key = torch.where(there, key, 0)
    block = (table.gather(1, key // page).long() * kv_heads)[..., None] + torch.arange(kv_heads, device=device)
    block = block * (page // BLOCK) + (key % page // BLOCK)[..., None]
    row = (key % BLOCK)[..., None]
    blocks = pool.view(-1).view(torch.int32).view(-1, BLOCK * (dim + 8) // 4)
    half = BLOCK * dim // 8
    code_k, code_v = (blocks[:, k * half:(k + 1) * half].unflatten(1, (BLOCK, dim // 8)) for k in (0, 1))
    word_k, word_v = (blocks[:, 2 * half + k * BLOCK:2 * half + (k + 1) * BLOCK] for k in (0, 1))
    k = _values(_unpacked(code_k[block, row]), word_k[block, row]).transpose(1, 2)  # [batch, kv_heads, keys, dim]
    pos = lens[:, None] - new + torch.arange(new, device=device)
    seen = (key[:, None, :] <= pos[:, :, None]) & there[:, None, :]
    seen = seen & ((pos[:, :, None] - key[:, None, :] <= window) | is_global[key][:, None, :])
    seen = seen[:, None, :, None, :]
    rows = q.view(batch, new, kv_heads, group, dim).permute(0, 2, 1, 3, 4).reshape(batch, kv_heads, new * group, dim)
    scores = (rows.float() @ k.transpose(-1, -2)).view(batch, kv_heads, new, group, -1) * state["scale"]
    del k
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(top > -math.inf, top, 0.0))
    total = weights.sum(-1, keepdim=True)
    v = _values(_unpacked(code_v[block, row]), word_v[block, row]).transpose(1, 2)
    out = (weights.view(batch, kv_heads, new * group, -1) @ v).view(batch, kv_heads, new, group, dim)
    out = torch.where(total > 0, out / total, 0.0).permute(0, 2, 1, 3, 4).reshape(q.shape).to(state["out"])
    if not case["lse"]:
        return {"out": out}
    lse = (top + torch.log(total)).squeeze(-1).permute(1, 3, 0, 2).reshape(case["heads"], batch * new)
    return {"out": out, "lse": lse}


# ---------------------------------------------------------------------------------- work


def work(case):
    if case["op"] == "layout":
        cached, new = _lens(case)
        page, total = case["page"], sum(new)
        fresh = sum(-(-(c + n) // page) - -(-c // page) for c, n in zip(cached, new))
        # lengths in and out, page ids taken and entered, a slot and a position a row
        return {"bytes": 4 * (6 * case["batch"] + 2 * fresh + 2 * case["rows"] + min(total, case["batch"])), "flops": 0}
    dim, kv_heads = case["dim"], case["kv_heads"]
    if case["op"] == "append":
        rows, kept = case["rows"] * kv_heads, case["tokens"] * kv_heads
        # K and V read, codes and words written, read again, and K and V written
        return {"bytes": 2 * 2 * dim * kept + 2 * (dim + 8) * kept + 2 * 2 * dim * rows + 8 * case["rows"],
                "flops": 6 * dim * kept}
    cached, new = _lens(case)
    tokens, window = _global_tokens(case), case["window"]
    keys = pairs = 0
    for c, n in zip(cached, new):
        lo = max(0, c - window)
        keys += c + n - lo + sum(t < lo for t in tokens)
        if n == 1:
            pairs += c + 1 - lo + sum(t < lo for t in tokens)
        else:
            pairs += sum(p + 1 - max(0, p - window) + sum(t < p - window for t in tokens) for p in range(c, c + n))
    rows = sum(new) * case["heads"]
    size = {"fp32": 4, "fp16": 2, "bf16": 2}[case["out"]]
    return {"bytes": keys * kv_heads * (dim + 8) + rows * dim * (2 + size) + (4 * rows if case["lse"] else 0)
            + 4 * (keys // case["page"]), "flops": 4 * dim * pairs * case["heads"]}


# ---------------------------------------------------------------------------------- 64 bits


def exact(case, seed):
    if case["op"] == "layout":
        return None  # whole numbers
    state = prepare(case, seed)
    if case["op"] == "append":
        return {name: _exact_rows(state[name], state["slots"]) for name in ("k", "v")}
    return _exact_attention(state, case)


def _exact_rows(x, slots):
    out = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    for at in range(0, x.shape[0], 8192):
        rows = x[at:at + 8192].double()
        hi = torch.maximum(rows.max(-1).values, torch.zeros((), dtype=torch.float64, device=x.device))
        lo = torch.minimum(rows.min(-1).values, torch.zeros((), dtype=torch.float64, device=x.device))
        step = ((hi - lo) / 15).float().view(torch.int32)
        step = (torch.bitwise_right_shift(step, 4) * 16).view(torch.float32).double()[..., None]
        safe = torch.where(step > 0, step, 1.0)
        zero = torch.round(-lo[..., None] / safe)
        codes = torch.minimum(torch.maximum(torch.round(rows / safe) + zero, torch.zeros_like(zero)), torch.full_like(zero, 15))
        out[at:at + 8192] = (codes - zero) * step * (slots[at:at + 8192] >= 0)[:, None, None]
    return out


def _exact_attention(state, case):
    pool, page, dim = state["pool"], case["page"], case["dim"]
    kv_heads, heads, new = case["kv_heads"], case["heads"], case["new"]
    group, device = heads // kv_heads, pool.device
    bytes_ = pool.view(pool.shape[0], kv_heads, page // BLOCK, BLOCK * (dim + 8))
    out = torch.empty(state["q"].shape, dtype=torch.float64, device=device)
    lse = torch.empty((heads, out.shape[0]), dtype=torch.float64, device=device)
    cached, _ = _lens(case)
    for b, c in enumerate(cached):
        count, lo = c + new, max(0, c - case["window"])
        want = sorted(set(t for t in state["globals"] if t < lo) | set(range(lo, count)))
        want = torch.tensor(want, device=device)
        at = state["block_table"][b].long()[want // page]
        chosen = bytes_[at, :, want % page // BLOCK]  # [keys, kv_heads, block bytes]
        line = want % BLOCK
        pos = torch.arange(c, count, device=device)
        visible = (want[None, :] <= pos[:, None]) & ((want[None, :] >= pos[:, None] - case["window"])
                                                     | torch.isin(want, torch.tensor(state["globals"], device=device, dtype=torch.long))[None, :])
        index = torch.arange(len(want), device=device)
        for h in range(kv_heads):
            side = []
            for k in (0, 1):
                codes = chosen[:, h, k * BLOCK * dim // 2:(k + 1) * BLOCK * dim // 2].reshape(-1, BLOCK, dim // 2)[index, line]
                at_word = BLOCK * dim + k * 4 * BLOCK
                word = chosen[:, h, at_word:at_word + 4 * BLOCK].reshape(-1, BLOCK, 4)[index, line].contiguous()
                zero = (word[:, 0] % 16).double()
                word[:, 0] -= word[:, 0] % 16
                scale = word.view(torch.float32)[:, 0].double()
                pair = torch.stack([codes % 16, codes // 16], -1).reshape(-1, dim).double()
                side.append((pair - zero[:, None]) * scale[:, None])
            for g in range(group):
                q = state["q"][b * new:(b + 1) * new, h * group + g].double()
                logit = torch.where(visible, q @ side[0].T * state["scale"], -math.inf)
                norm = torch.logsumexp(logit, -1)
                out[b * new:(b + 1) * new, h * group + g] = torch.exp(logit - norm[:, None]) @ side[1]
                lse[h * group + g, b * new:(b + 1) * new] = norm
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}
