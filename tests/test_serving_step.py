"""A serving step as a user runs it: pages planned, tokens appended, keys selected and attended, on one cache."""

from __future__ import annotations

import math

import pytest
import torch

from fusedindextopk_b200 import attention, paged, quantize


@pytest.fixture(scope="module")
def device():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return torch.device("cuda:0")


REQUESTS, COLUMNS, PAGE, ROWS = 3, 24, 128, 3000
HEADS, KV_HEADS, DIM = 8, 2, 128
PAGES = 80


class Cache:
    """The pools, the table and the plan that a serving program keeps between steps."""

    def __init__(self, device):
        shape = (PAGES, PAGE, KV_HEADS, DIM)
        self.k = torch.full(shape, float("nan"), dtype=torch.bfloat16, device=device)
        self.v = torch.full_like(self.k, float("nan"))
        self.index = torch.full((PAGES, PAGE, 128), 0x3C, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
        self.scales = torch.full((PAGES, PAGE), float("nan"), device=device)
        self.table = torch.full((REQUESTS, COLUMNS), -1, dtype=torch.int32, device=device)
        self.plan = paged.make_page_plan(REQUESTS, COLUMNS, ROWS, page_size=PAGE, device=device)
        self.lengths = torch.zeros(REQUESTS, dtype=torch.int32, device=device)
        self.free = torch.randperm(PAGES, generator=torch.Generator().manual_seed(3)).to(torch.int32).to(device)


def step(cache, new_tokens, tokens):
    """Everything between a step's projections and its output projection; nothing is read back to the host."""

    plan = paged.plan_pages(cache.plan, cache.table, cache.lengths, new_tokens, cache.free)
    paged.append_tokens(plan.slots, (tokens["k"], tokens["v"]), (cache.k, cache.v), index_keys=tokens["index_k"],
                        index_pools=(cache.index, cache.scales))
    index_q, weights = quantize.quantize_queries(tokens["index_q"], tokens["weights"])
    keys = REQUESTS * COLUMNS * PAGE
    ids = paged.fused_index_topk_paged(index_q, (cache.index, cache.scales), plan.flat_table, keys, weights, plan.k_start, plan.k_end)
    out = attention.attention_paged(tokens["q"], (cache.k, cache.v), cache.table, plan.cu_seqlens_q, plan.lengths)
    return ids, out


def projections(device, seed):
    g = torch.Generator(device=device).manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=device)

    return {"q": normal(ROWS, HEADS, DIM).bfloat16(), "k": normal(ROWS, KV_HEADS, DIM).bfloat16(),
            "v": normal(ROWS, KV_HEADS, DIM).bfloat16(), "index_q": normal(ROWS, 64, 128).bfloat16(),
            "index_k": normal(ROWS, 128).bfloat16(), "weights": normal(ROWS, 64).abs()}


@pytest.mark.gpu
def test_prompts_then_single_tokens(device):
    from fusedindextopk_b200 import fused_index_topk

    cache = Cache(device)
    history = [{n: [] for n in ("k", "v", "index_k")} for _ in range(REQUESTS)]
    used = 0
    for number, counts in enumerate(([2200, 700, 0], [1, 1, 90], [1, 1, 1])):
        tokens = projections(device, number)
        new_tokens = torch.tensor(counts, dtype=torch.int32, device=device)
        ids, out = step(cache, new_tokens, tokens)
        ids, out = ids.clone(), out.clone()
        paged.check_serving_status(device)
        first = 0
        for b, count in enumerate(counts):
            rows = slice(first, first + count)
            for name in history[b]:
                history[b][name].append(tokens[name][rows])
            first += count
            if count == 0:
                continue
            held = {n: torch.cat(parts) for n, parts in history[b].items()}
            length = held["k"].shape[0]
            # the keys selected among all of the request's keys, in its own positions
            q8, weights = quantize.quantize_queries(tokens["index_q"][rows].contiguous(), tokens["weights"][rows].contiguous())
            kv8 = quantize.quantize_contiguous_index_kv(held["index_k"].contiguous())
            ends = (length - count + 1 + torch.arange(count, device=device)).to(torch.int32)
            want = fused_index_topk(q8, kv8, weights, torch.zeros_like(ends), ends).clone()
            offset = cache.plan.k_start[rows].unsqueeze(1)
            got = torch.where(ids[rows] >= 0, ids[rows] - offset, ids[rows])
            assert torch.equal(got.sort(dim=-1).values, want.sort(dim=-1).values)
            # and all of them attended, against the definition in 64 bits
            for h in range(HEADS):
                k, v = held["k"][:, h // (HEADS // KV_HEADS)].double(), held["v"][:, h // (HEADS // KV_HEADS)].double()
                scores = tokens["q"][rows, h].double() @ k.T / math.sqrt(DIM)
                scores = scores.masked_fill(torch.arange(length, device=device) >= ends.unsqueeze(1), -math.inf)
                weights64 = torch.softmax(scores, dim=-1)
                expect, magnitude = weights64 @ v, weights64 @ v.abs()
                # one rounding of the weights and one of the output, half a bf16 step each; 2^-12 for the fp32 arithmetic
                # of scores up to 2^4 (D products, exponentials, sums of 2^12 terms)
                bound = (2.0 ** -8 + 2.0 ** -12) * magnitude + 2.0 ** -8 * expect.abs()
                assert bool(((out[rows, h].double() - expect).abs() <= bound).all())
        assert bool((out[first:] == 0).all()) and bool((ids[first:] == -1).all())
        cache.lengths.copy_(cache.plan.lengths)
        used = int(cache.plan.pages_needed)
        cache.free = torch.cat([cache.free[used:], cache.free[:used]])


@pytest.mark.gpu
def test_a_step_in_a_graph_follows_the_batch(device):
    """Plan, append and attention captured once, replayed for steps of other lengths."""

    eager, captured = Cache(device), Cache(device)
    tokens = projections(device, 5)
    new_tokens = torch.zeros(REQUESTS, dtype=torch.int32, device=device)

    def serve(cache):
        plan = paged.plan_pages(cache.plan, cache.table, cache.lengths, new_tokens, cache.free)
        paged.append_tokens(plan.slots, (tokens["k"], tokens["v"]), (cache.k, cache.v))
        return attention.attention_paged(tokens["q"], (cache.k, cache.v), cache.table, plan.cu_seqlens_q, plan.lengths)

    serve(captured)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = serve(captured)
    for counts in ([300, 0, 129], [1, 1, 1], [0, 128, 1]):
        new_tokens.copy_(torch.tensor(counts, dtype=torch.int32))
        graph.replay()
        want = serve(eager)
        torch.cuda.synchronize()
        paged.check_serving_status(device)
        assert torch.equal(held, want)
        assert torch.equal(captured.table, eager.table) and torch.equal(captured.k.nan_to_num(), eager.k.nan_to_num())
        for cache in (eager, captured):
            used = int(cache.plan.pages_needed)
            cache.lengths.copy_(cache.plan.lengths)
            cache.free.copy_(torch.cat([cache.free[used:], cache.free[:used]]))


@pytest.mark.gpu
def test_the_whole_step_in_a_graph_follows_the_batch(device):
    """Plan, append, quantisation, selection and attention captured once, replayed for steps of other lengths."""

    eager, captured = Cache(device), Cache(device)
    tokens = projections(device, 6)
    new_tokens = torch.zeros(REQUESTS, dtype=torch.int32, device=device)
    step(captured, new_tokens, tokens)                      # workspaces and buffers are made outside of the graph
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held_ids, held = step(captured, new_tokens, tokens)
    for counts in ([2300, 0, 129], [1, 1, 1], [0, 700, 1], [1, 1, 1]):
        new_tokens.copy_(torch.tensor(counts, dtype=torch.int32))
        graph.replay()
        ids, out = held_ids.clone(), held.clone()
        want_ids, want = (x.clone() for x in step(eager, new_tokens, tokens))
        paged.check_serving_status(device)
        assert torch.equal(ids.sort(dim=-1).values, want_ids.sort(dim=-1).values) and torch.equal(out, want)
        assert bool((ids[:sum(counts), 0] >= 0).all())
        for cache in (eager, captured):
            used = int(cache.plan.pages_needed)
            cache.lengths.copy_(cache.plan.lengths)
            cache.free.copy_(torch.cat([cache.free[used:], cache.free[:used]]))
