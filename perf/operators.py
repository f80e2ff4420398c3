"""Attention over packed and paged batches, and the page bookkeeping below it: what is timed, and on which sizes.

Four operators of a serving step.  A step plans its pages (``paged.plan_pages``), writes its tokens into the
pools (``paged.append_tokens``), and attends: every request to its own keys (``attention.attention_varlen``,
``attention.attention_paged``), or to a prefix that the whole batch shares and to its own keys
(``attention.shared_prefix_attention`` and its paged form).

``run`` computes an operator either in elementary torch operations in 32 bits (``own`` false) or by the
package's entry points (``own`` true).  ``exact`` is the definition in 64 bits.
"""

from __future__ import annotations

import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
NEVER = float("-inf")


# --------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # -- every request attends to its own keys
        # one request's single new token over the context of the framework's smallest workload: latency
        dict(name="decode one", op="attention", dtype="bf16", heads=32, kv_heads=8, dim=128, seqs=1, whole=False,
             q_min=1, q_max=1, k_min=8192, k_max=8192, mix=1, page=0, lse=False),
        # a packed batch of whole prompts of odd lengths, from one token on
        dict(name="prompts ragged", op="attention", dtype="fp16", heads=32, kv_heads=8, dim=128, seqs=9, whole=True,
             q_min=1, q_max=1, k_min=1, k_max=2111, mix=5, page=0, lse=True),
        # a serving batch: single tokens of 64 requests over paged contexts of very different lengths
        dict(name="decode batch paged", op="attention", dtype="bf16", heads=64, kv_heads=8, dim=128, seqs=64, whole=False,
             q_min=1, q_max=1, k_min=65, k_max=32768, mix=3, page=128, lse=False),
        # a chunk of 4096 rows at the end of a context of 16384 keys: the framework's flagship shape
        dict(name="chunk 4096 of 16384", op="attention", dtype="bf16", heads=64, kv_heads=8, dim=128, seqs=1, whole=False,
             q_min=4096, q_max=4096, k_min=16384, k_max=16384, mix=4, page=0, lse=False),
        # a long whole prompt with one key head for each query head and narrow heads
        dict(name="prompt 32768 narrow", op="attention", dtype="bf16", heads=16, kv_heads=16, dim=64, seqs=1, whole=True,
             q_min=1, q_max=1, k_min=32768, k_max=32768, mix=5, page=0, lse=True),
        # -- a batch that shares a long prefix
        # a handful of requests behind a short system text: latency
        dict(name="prefix 2048 few", op="prefix", dtype="bf16", heads=32, kv_heads=8, dim=128, seqs=4, prefix=2048,
             q_min=1, q_max=1, k_min=17, k_max=150, mix=6, page=0, lse=False),
        # a serving batch behind a long document, paged
        dict(name="prefix 16384 paged", op="prefix", dtype="bf16", heads=64, kv_heads=8, dim=128, seqs=64, prefix=16384,
             q_min=1, q_max=1, k_min=33, k_max=2048, mix=7, page=256, lse=False),
        # many requests with two or three tokens each (drafted tokens) behind a very long document
        dict(name="prefix 131072 drafts", op="prefix", dtype="fp16", heads=32, kv_heads=4, dim=128, seqs=200, prefix=131072,
             q_min=2, q_max=3, k_min=3, k_max=512, mix=8, page=0, lse=True),
        # -- block tables and slot maps
        # the step of a small serving batch: one new token each
        dict(name="tables 8 decode", op="tables", seqs=8, table_pages=128, page=128, new_max=1, rows=8),
        # a large batch that admits prompts next to running requests, in a buffer with room to spare
        dict(name="tables 1024 mixed", op="tables", seqs=1024, table_pages=256, page=256, new_max=511, rows=300000),
        # -- tokens into the pools
        # the step of a serving batch: 64 tokens, with their index keys
        dict(name="append 64", op="append", dtype="bf16", kv_heads=8, dim=128, tokens=64, page=128, pages=64, holes=0.05),
        # a chunk of a prompt, some of its rows padding
        dict(name="append 8191", op="append", dtype="bf16", kv_heads=8, dim=128, tokens=8191, page=256, pages=48, holes=0.01),
    ]


def _log_int(rng, low, high):
    """A whole number between low and high, even over the logarithm."""
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    op = rng.choice(["attention", "attention", "prefix", "tables", "append"])
    if op == "tables":
        seqs = _log_int(rng, 1, 2000)
        page = rng.choice([128, 256, 512])
        new_max = _log_int(rng, 1, 512)
        return dict(op=op, seqs=seqs, table_pages=rng.randint(16, 300), page=page, new_max=new_max,
                    rows=seqs * new_max // rng.choice([1, 2]) + rng.randint(1, 9))
    if op == "append":
        tokens = _log_int(rng, 1, 8191)
        page = rng.choice([128, 256, 512])
        return dict(op=op, dtype=rng.choice(["bf16", "fp16"]), kv_heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 128]),
                    tokens=tokens, page=page, pages=-(-tokens // page) + rng.randint(1, 8),
                    holes=rng.choice([0.0, 0.02, 0.3]))
    dim = rng.choice([64, 128, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 5, 7, 8, 12, 16])
    same = dict(op=op, dtype=rng.choice(["bf16", "fp16"]), heads=heads, kv_heads=kv_heads, dim=dim,
                mix=rng.randint(0, 1 << 20), page=rng.choice([0, 0, 128, 256]), lse=rng.random() < 0.5)
    if op == "prefix":
        q_max = rng.randint(1, 4)
        return dict(same, seqs=_log_int(rng, 1, 128), prefix=_log_int(rng, 1, 65536), q_min=rng.randint(1, q_max), q_max=q_max,
                    k_min=4, k_max=_log_int(rng, 8, 2048))
    kind = rng.choice(["decode", "decode", "prompt", "chunk"])
    if kind == "decode":
        return dict(same, seqs=_log_int(rng, 1, 64), whole=False, q_min=1, q_max=rng.randint(1, 4), k_min=rng.randint(1, 64),
                    k_max=_log_int(rng, 64, 24000))
    if kind == "prompt":
        seqs = _log_int(rng, 1, 12)
        return dict(same, seqs=seqs, whole=True, q_min=1, q_max=1, k_min=rng.randint(0, 5), k_max=_log_int(rng, 16, 10000 // seqs))
    k_max = _log_int(rng, 300, 12000)
    return dict(same, seqs=rng.randint(1, 3), whole=False, q_min=rng.randint(1, 100), q_max=_log_int(rng, 100, 2000),
                k_min=k_max // 2, k_max=k_max)


def _lengths(case):
    """Query rows and own keys of every request of a case; the longest one comes first."""
    rng = random.Random(case["mix"])
    low, high = case["k_min"], case["k_max"]
    keys = [high] + [max(low, _log_int(rng, max(1, low), high) - (low == 0)) for _ in range(case["seqs"] - 1)]
    if case.get("whole"):
        return list(keys), keys
    return [min(k, rng.randint(case["q_min"], case["q_max"])) for k in keys], keys


def _prefix_sums(values):
    sums = [0]
    for v in values:
        sums.append(sums[-1] + v)
    return sums


# --------------------------------------------------------------------------------------------- inputs

def _normal(generator, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=generator, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    host = torch.Generator().manual_seed(int(seed))
    if case["op"] == "tables":
        return _prepare_tables(case, host)
    if case["op"] == "append":
        return _prepare_append(case, g, host)
    dtype, dim, heads, kv_heads = DTYPES[case["dtype"]], case["dim"], case["heads"], case["kv_heads"]
    q_lens, k_lens = _lengths(case)
    prefix = case.get("prefix", 0)
    state = {"case": case, "q_lens": q_lens, "k_lens": k_lens, "cu_q": _ints(_prefix_sums(q_lens)),
             "cu_k": _ints(_prefix_sums(k_lens)), "lens_k": _ints(k_lens),
             "q": _normal(g, (sum(q_lens), heads, dim), dtype, 1.5)}
    if case["page"] == 0:
        state["k"], state["v"] = (_normal(g, (sum(k_lens), kv_heads, dim), dtype) for _ in range(2))
        if prefix:
            state["k_prefix"], state["v_prefix"] = (_normal(g, (prefix, kv_heads, dim), dtype) for _ in range(2))
        return state
    # pages in the order an allocator that has been running for a while hands them out
    page = case["page"]
    need = [-(-k // page) for k in k_lens]
    prefix_need = -(-prefix // page)
    pages = sum(need) + prefix_need + 5
    order = torch.randperm(pages, generator=host).to(torch.int32)
    table = torch.full((len(k_lens), max(max(need), 1)), -1, dtype=torch.int32)
    at = prefix_need
    for row, count in enumerate(need):
        table[row, :count] = order[at:at + count]
        at += count
    state["table"], state["prefix_table"] = table.cuda(), order[:prefix_need].cuda()
    state["k"], state["v"] = (_normal(g, (pages, page, kv_heads, dim), dtype) for _ in range(2))
    return state


def _prepare_tables(case, host):
    seqs, page, columns = case["seqs"], case["page"], case["table_pages"]
    new = torch.randint(0, case["new_max"] + 1, (seqs,), generator=host)
    new = torch.minimum(new, (case["rows"] - (new.cumsum(0) - new)).clamp(min=0))      # the batch fits its rows
    room = columns * page - case["new_max"]
    old = (torch.rand(seqs, generator=host) * max(room, 0)).long().clamp(max=max(room, 0))
    old[torch.rand(seqs, generator=host) < 0.2] = 0                                    # newly admitted requests
    before, after = -(-old // page), -(-(old + new) // page)
    order = torch.randperm(int(after.sum()) + 16, generator=host)
    starts = before.cumsum(0) - before
    column = torch.arange(columns)
    held = column.unsqueeze(0) < before.unsqueeze(1)
    table = torch.where(held, order[(starts.unsqueeze(1) + column).clamp(max=order.numel() - 1)], torch.tensor(-1))
    state = {"case": case, "table": table.to(torch.int32).cuda(), "old": old.to(torch.int32).cuda(),
             "new": new.to(torch.int32).cuda(), "free": order[int(before.sum()):].to(torch.int32).cuda()}
    if own:
        from fusedindextopk_b200 import paged
        state["plan"] = paged.make_page_plan(seqs, columns, case["rows"], page_size=page, device="cuda")
    return state


def _prepare_append(case, g, host):
    dtype, rows = DTYPES[case["dtype"]], case["pages"] * case["page"]
    slots = torch.randperm(rows, generator=host)[:case["tokens"]]
    slots[torch.rand(case["tokens"], generator=host) < case["holes"]] = -1             # padding rows
    token = (case["tokens"], case["kv_heads"], case["dim"])
    pool = (case["pages"], case["page"], case["kv_heads"], case["dim"])
    state = {"case": case, "slots": slots.cuda()}
    state["k"], state["v"] = (_normal(g, token, dtype) for _ in range(2))
    state["k_pool"], state["v_pool"] = (_normal(g, pool, dtype) for _ in range(2))
    state["index"] = _normal(g, (case["tokens"], 128), torch.bfloat16, 2.0)
    state["index_pool"] = _normal(g, (case["pages"], case["page"], 128), torch.float8_e4m3fn)
    state["index_scales"] = torch.rand((case["pages"], case["page"]), generator=g, device="cuda")
    return state


# --------------------------------------------------------------------------------------------- one pass

def run(state):
    return {"attention": _run_attention, "prefix": _run_attention, "tables": _run_tables, "append": _run_append}[state["case"]["op"]](state)


def _run_attention(state):
    case = state["case"]
    if own:
        from fusedindextopk_b200 import attention
        pair = (state["k"], state["v"])
        if case["op"] == "attention" and case["page"] == 0:
            got = attention.attention_varlen(state["q"], pair, state["cu_q"], state["cu_k"], return_lse=case["lse"])
        elif case["op"] == "attention":
            got = attention.attention_paged(state["q"], pair, state["table"], state["cu_q"], state["lens_k"], return_lse=case["lse"])
        elif case["page"] == 0:
            got = attention.shared_prefix_attention(state["q"], (state["k_prefix"], state["v_prefix"]), pair, state["cu_q"],
                                                    state["cu_k"], return_lse=case["lse"])
        else:
            got = attention.shared_prefix_attention_paged(state["q"], pair, state["prefix_table"], case["prefix"], state["table"],
                                                          state["cu_q"], state["lens_k"], return_lse=case["lse"])
        return {"out": got[0], "lse": got[1]} if case["lse"] else {"out": got}
    return _plain_attention(state)


def _padded(rows, lengths, longest):
    """[sum of lengths, ...] -> [requests, longest, ...]; rows past a request's end repeat some row."""
    starts = lengths.cumsum(0) - lengths
    at = (starts.unsqueeze(1) + torch.arange(longest, device=rows.device)).clamp(max=max(rows.shape[0] - 1, 0))
    return rows[at]


def _plain_attention(state):
    case = state["case"]
    dim, heads, kv_heads = case["dim"], case["heads"], case["kv_heads"]
    group, scale = heads // kv_heads, dim ** -0.5
    q_lens, k_lens = (state["cu_q"][1:] - state["cu_q"][:-1]).long(), state["lens_k"].long()
    q_top, k_top, seqs = max(state["q_lens"]), max(state["k_lens"]), case["seqs"]
    if case["page"]:
        flat = [state[n].reshape(-1, kv_heads, dim) for n in ("k", "v")]
        position = torch.arange(k_top, device="cuda")
        at = (state["table"].long()[:, position // case["page"]].clamp(min=0) * case["page"] + position % case["page"])
        k, v = (x[at].float() for x in flat)
        position = torch.arange(case.get("prefix", 0), device="cuda")
        at = state["prefix_table"].long()[position // case["page"]] * case["page"] + position % case["page"]
        k_prefix, v_prefix = (x[at].float() for x in flat)
    else:
        k, v = (_padded(state[n], k_lens, k_top).float() for n in ("k", "v"))
        k_prefix, v_prefix = ((state[n] if "k_prefix" in state else state["k"][:0]).float() for n in ("k_prefix", "v_prefix"))
    prefix = k_prefix.shape[0]
    k, v = k.permute(0, 2, 3, 1), v.permute(0, 2, 1, 3)                       # [B,H,D,N], [B,H,N,D]
    k_prefix, v_prefix = k_prefix.permute(1, 2, 0), v_prefix.permute(1, 0, 2)
    q = _padded(state["q"], q_lens, q_top).float().view(seqs, q_top, kv_heads, group, dim).permute(0, 2, 1, 3, 4)
    out = torch.zeros((seqs, q_top, heads, dim), device="cuda")
    lse = torch.full((seqs, q_top, heads), NEVER, device="cuda")
    # rows are taken in pieces so that the scores of a piece fit the memory
    piece = max(1, (1 << 30) // (seqs * heads * (k_top + prefix)))
    for lo in range(0, q_top, piece):
        hi = min(q_top, lo + piece)
        rows = q[:, :, lo:hi].reshape(seqs, kv_heads, (hi - lo) * group, dim)
        visible = k_lens.unsqueeze(1) - q_lens.unsqueeze(1) + torch.arange(lo, hi, device="cuda") + 1
        visible = torch.minimum(visible, k_lens.unsqueeze(1)).repeat_interleave(group, dim=1)
        scores = (rows @ k).mul_(scale)
        scores.masked_fill_(torch.arange(k_top, device="cuda") >= visible[:, None, :, None], NEVER)
        top = scores.amax(-1, keepdim=True)
        if prefix:
            # all requests' rows against the one prefix
            shared_rows = rows.transpose(0, 1).reshape(kv_heads, -1, dim)
            shared = (shared_rows @ k_prefix).mul_(scale)
            shared_top = shared.amax(-1, keepdim=True).view(kv_heads, seqs, -1, 1).transpose(0, 1)
            top = torch.maximum(top, shared_top)
        top = torch.where(top == NEVER, torch.zeros_like(top), top)
        scores = scores.sub_(top).exp_()
        total = scores.sum(-1, keepdim=True)
        value = scores @ v
        if prefix:
            shared = shared.sub_(top.transpose(0, 1).reshape(kv_heads, -1, 1)).exp_()
            total = total + shared.sum(-1, keepdim=True).view(kv_heads, seqs, -1, 1).transpose(0, 1)
            value = value + (shared @ v_prefix).view(kv_heads, seqs, -1, dim).transpose(0, 1)
        value = torch.where(total > 0, value / total, torch.zeros_like(value))
        total = (total.log() + torch.where(total > 0, top, torch.zeros_like(top)))
        out[:, lo:hi] = value.view(seqs, kv_heads, hi - lo, group, dim).permute(0, 2, 1, 3, 4).reshape(seqs, hi - lo, heads, dim)
        lse[:, lo:hi] = total.view(seqs, kv_heads, hi - lo, group).permute(0, 2, 1, 3).reshape(seqs, hi - lo, heads)
    there = torch.arange(q_top, device="cuda") < q_lens.unsqueeze(1)
    out = out[there].to(state["q"].dtype)
    return {"out": out, "lse": lse[there]} if case["lse"] else {"out": out}


def _run_tables(state):
    case = state["case"]
    page, rows = case["page"], case["rows"]
    if own:
        from fusedindextopk_b200 import paged
        plan = paged.plan_pages(state["plan"], state["table"], state["old"], state["new"], state["free"])
        return {"table": plan.block_table, "slots": plan.slots, "cu_seqlens_q": plan.cu_seqlens_q, "lengths": plan.lengths,
                "flat_table": plan.flat_table, "k_start": plan.k_start, "k_end": plan.k_end, "pages_needed": plan.pages_needed}
    table, old, new = state["table"], state["old"].long(), state["new"].long()
    lengths = old + new
    before, after = (old + page - 1) // page, (lengths + page - 1) // page
    taken = (after - before).cumsum(0)
    column = torch.arange(case["table_pages"], device="cuda")
    fresh = (taken - (after - before)).unsqueeze(1) + column - before.unsqueeze(1)
    fresh = state["free"][fresh.clamp(0, state["free"].numel() - 1)]
    table.copy_(torch.where(column >= after.unsqueeze(1), -1, torch.where(column < before.unsqueeze(1), table, fresh)))
    cu_q = torch.cat([new.new_zeros(1), new.cumsum(0)])
    row = torch.arange(rows, device="cuda")
    request = torch.searchsorted(cu_q, row, right=True) - 1
    real = row < cu_q[-1]
    request = request.clamp(max=case["seqs"] - 1)
    position = old[request] + row - cu_q[request]
    slot = table[request, (position // page).clamp(max=case["table_pages"] - 1)].long() * page + position % page
    first = after.cumsum(0) - after
    flat = torch.zeros(case["seqs"] * case["table_pages"], dtype=torch.int32, device="cuda")
    entry = torch.arange(flat.numel(), device="cuda")
    owner = (torch.searchsorted(after.cumsum(0), entry, right=True)).clamp(max=case["seqs"] - 1)
    flat = torch.where(entry < after.sum(), table[owner, (entry - first[owner]).clamp(0, case["table_pages"] - 1)], flat)
    nothing = torch.zeros_like(row)
    return {"table": table, "slots": torch.where(real, slot, torch.full_like(slot, -1)), "cu_seqlens_q": cu_q.to(torch.int32),
            "lengths": lengths.to(torch.int32), "flat_table": flat,
            "k_start": torch.where(real, first[request] * page, nothing).to(torch.int32),
            "k_end": torch.where(real, first[request] * page + position + 1, nothing).to(torch.int32),
            "pages_needed": taken[-1:].to(torch.int32)}


def _run_append(state):
    pools = {n: state[n] for n in ("k_pool", "v_pool", "index_pool", "index_scales")}
    if own:
        from fusedindextopk_b200 import paged
        paged.append_tokens(state["slots"], (state["k"], state["v"]), (state["k_pool"], state["v_pool"]),
                            index_keys=state["index"], index_pools=(state["index_pool"], state["index_scales"]))
        return pools
    kept = state["slots"] >= 0
    slots = state["slots"][kept]
    for name in ("k", "v"):
        pool = state[name + "_pool"]
        pool.view(-1, *pool.shape[2:])[slots] = state[name][kept]
    index = state["index"][kept].float()
    amax = index.abs().amax(-1).clamp(min=1e-4)
    scales = amax / torch.full_like(amax, 448.0)           # by a tensor: a division, not a product with 1/448
    state["index_pool"].view(torch.uint8).view(-1, 128)[slots] = (index / scales.unsqueeze(1)).to(torch.float8_e4m3fn).view(torch.uint8)
    state["index_scales"].view(-1)[slots] = scales
    return pools


# --------------------------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    if case["op"] == "tables":
        cells = case["seqs"] * case["table_pages"]
        # lengths in and out, the table, its flat copy, and for every row a slot and a range
        return {"bytes": 16 * case["seqs"] + 12 * cells + 16 * case["rows"], "flops": 0}
    if case["op"] == "append":
        kept = case["tokens"] * (1 - case["holes"])
        kv = 2 * 2 * case["kv_heads"] * case["dim"]
        return {"bytes": 8 * case["tokens"] + kept * (2 * kv + 256 + 128 + 4), "flops": 0}
    q_lens, k_lens = _lengths(case)
    prefix = case.get("prefix", 0)
    pairs = sum(sum(max(0, k - q + i + 1) for i in range(q)) for q, k in zip(q_lens, k_lens)) + sum(q_lens) * prefix
    rows = sum(q_lens) * case["heads"] * case["dim"]
    size = 2 * 2 * rows + 2 * 2 * (sum(k_lens) + prefix) * case["kv_heads"] * case["dim"]
    return {"bytes": size + (4 * sum(q_lens) * case["heads"] if case["lse"] else 0),
            "flops": 4 * pairs * case["heads"] * case["dim"]}


# --------------------------------------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    """Every request and key head by itself: log-sum-exp of its scores, then the weighted sum of its values."""
    if case["op"] == "tables":
        return None                                          # whole numbers: nothing is rounded
    state = prepare(case, seed)
    if case["op"] == "append":
        x = state["index"].double()
        kept = [i for i, s in enumerate(state["slots"].tolist()) if s >= 0]
        scales = state["index_scales"].double().view(-1)
        scales[state["slots"][kept]] = torch.maximum(x.abs().max(dim=-1).values, torch.tensor(1e-4, device="cuda", dtype=torch.float64))[kept] / 448.0
        return {"k_pool": None, "v_pool": None, "index_pool": None, "index_scales": scales.view(case["pages"], case["page"])}
    group, dim, page = case["heads"] // case["kv_heads"], case["dim"], case["page"]
    out, lse = [], []
    row = key = 0
    prefix = case.get("prefix", 0)
    for request, (q_len, k_len) in enumerate(zip(state["q_lens"], state["k_lens"])):
        if page:
            pages = state["table"][request, :-(-k_len // page)].long()
            keys, values = (state[n][pages].flatten(0, 1)[:k_len] for n in ("k", "v"))
            if prefix:
                shared = state["prefix_table"].long()
                keys, values = (torch.cat([state[n][shared].flatten(0, 1)[:prefix], x]) for n, x in (("k", keys), ("v", values)))
        else:
            keys, values = (state[n][key:key + k_len] for n in ("k", "v"))
            if prefix:
                keys, values = torch.cat([state["k_prefix"], keys]), torch.cat([state["v_prefix"], values])
        position = torch.arange(prefix + k_len, device="cuda")
        out_r = torch.zeros((q_len, case["heads"], dim), dtype=torch.float64, device="cuda")
        lse_r = torch.full((q_len, case["heads"]), NEVER, dtype=torch.float64, device="cuda")
        for h in range(case["kv_heads"] if prefix + k_len else 0):
            kh, vh = keys[:, h].double(), values[:, h].double()
            for lo in range(0, q_len, 1024):
                hi = min(q_len, lo + 1024)
                rows = state["q"][row + lo:row + hi, h * group:(h + 1) * group].double()
                scores = torch.einsum("qgd,nd->gqn", rows, kh) / dim ** 0.5
                last = prefix + k_len - q_len + torch.arange(lo, hi, device="cuda")
                scores = scores.masked_fill(position > last.unsqueeze(1), NEVER)
                sums = torch.logsumexp(scores, dim=-1)
                weights = torch.exp(scores - torch.where(sums == NEVER, torch.zeros_like(sums), sums).unsqueeze(-1))
                out_r[lo:hi, h * group:(h + 1) * group] = torch.einsum("gqn,nd->qgd", weights, vh)
                lse_r[lo:hi, h * group:(h + 1) * group] = sums.T
        out.append(out_r)
        lse.append(lse_r)
        row += q_len
        key += k_len
    out, lse = torch.cat(out), torch.cat(lse)
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}
