"""Attention over packed, paged and shared-prefix batches against the definition in 64 bits.

Tolerance of an output, from the arithmetic (u = eps / 2 of the element type, e = 2^-24):
* the weights may be rounded to the element type once: u * A with A = sum_j p_j |v_j|; fp16 weights (at most 1 after the row
  maximum is taken off, so the sum is at least 1) may also lose 2^-25 each below the normal range: 2^-25 * sum_j |v_j|;
* the output is rounded once: u * |out|;
* a score is a sum of D products in fp32, scaled: ds = (D + 3) e * scale * max_j sum_i |q_i k_ji|, and the exponential of a
  difference of two scores is off by 2 ds + 2^-20 relatively (the exponential itself is good to 2^-21);
* sums over n keys add n e, joining partial results another 2^-20.
"""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from fusedindextopk_b200 import _lib, attention
from fusedindextopk_b200.build import build

E = 2.0 ** -24


@pytest.fixture(scope="module")
def device():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return torch.device("cuda:0")


def sums(lengths, device):
    return torch.tensor([0] + list(lengths), dtype=torch.int64).cumsum(0).to(torch.int32).to(device)


def definition(q, keys, values, visible, scale):
    """One request: rows [Q,Hq,D], keys [N,H,D]; row i sees the first visible[i] keys.  (out, lse, tol_out, tol_lse) in 64 bits."""

    rows, heads, dim = q.shape
    n, kv_heads = keys.shape[:2]
    group = heads // kv_heads
    u = torch.finfo(q.dtype).eps / 2
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full((rows, heads), -math.inf, dtype=torch.float64, device=q.device)
    tol, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
    if n == 0 or rows == 0:
        return out, lse, tol, tol_lse
    mask = torch.arange(n, device=q.device) >= visible.unsqueeze(1)
    some = ~mask.all(dim=1)
    for h in range(heads):
        k, v = keys[:, h // group].double(), values[:, h // group].double()
        x = q[:, h].double()
        scores = ((x @ k.T) * scale).masked_fill(mask, -math.inf)
        top = scores.amax(1, keepdim=True)
        top = torch.where(top == -math.inf, torch.zeros_like(top), top)
        weights = torch.exp(scores - top)
        total = weights.sum(1, keepdim=True)
        seen = (~mask).double()
        o = torch.where(some.unsqueeze(1), (weights / total.clamp(min=1e-300)) @ v, torch.zeros((), dtype=torch.float64, device=q.device))
        magnitude = torch.where(some.unsqueeze(1), (weights / total.clamp(min=1e-300)) @ v.abs(), torch.zeros_like(o))
        ds = (dim + 3) * E * abs(scale) * ((x.abs() @ k.abs().T) * seen).amax(1, keepdim=True)
        rel = 2 * ds + 2.0 ** -20 + n * E + 2.0 ** -20
        extra = 2.0 ** -25 * (seen @ v.abs()) if q.dtype == torch.float16 else 0.0
        tol[:, h] = (u + rel) * magnitude + u * o.abs() * 1.01 + extra + 1e-30
        out[:, h] = o
        lse[:, h] = torch.where(some, top.squeeze(1) + torch.log(total.squeeze(1)), torch.full_like(lse[:, h], -math.inf))
        tol_lse[:, h] = ds.squeeze(1) + (2.0 ** -20 + n * E) + 4 * E * (lse[:, h].abs().nan_to_num(posinf=0.0) + top.squeeze(1).abs())
    return out, lse, tol, tol_lse


def expected(q, q_lens, requests, causal=True, scale=None):
    """``requests``: (own keys [N,H,D], own values, prefix keys or None, prefix values) per request."""

    scale = 1 / math.sqrt(q.shape[2]) if scale is None else scale
    parts, row = [], 0
    for count, (k, v, kp, vp) in zip(q_lens, requests):
        prefix = 0
        n = k.shape[0]
        if kp is not None:
            prefix = kp.shape[0]
            k, v = torch.cat([kp, k]), torch.cat([vp, v])
        own = n - count + 1 + torch.arange(count, device=q.device) if causal else torch.full((count,), n, device=q.device)
        parts.append(definition(q[row:row + count], k, v, prefix + own.clamp(0, n), scale))
        row += count
    return tuple(torch.cat([p[i] for p in parts]) for i in range(4))


def assert_close(got, lse, want):
    out, want_lse, tol, tol_lse = want
    off = (got[:out.shape[0]].double() - out).abs()
    assert bool((off <= tol).all()), f"worst {float((off / tol).max()):.3f} of the tolerance at {int((off / tol).argmax())}"
    if lse is not None:
        lse = lse[:out.shape[0]].double()
        assert torch.equal(lse == -math.inf, want_lse == -math.inf)
        fine = want_lse > -math.inf
        off = (lse - want_lse)[fine].abs()
        assert bool((off <= tol_lse[fine]).all()), f"lse worst {float((off / tol_lse[fine]).max()):.3f} of the tolerance"


def make(device, q_lens, k_lens, heads, kv_heads, dim, dtype, seed=0, spread=1.5):
    g = torch.Generator(device=device).manual_seed(seed)
    q = (torch.randn((sum(q_lens), heads, dim), generator=g, device=device) * spread).to(dtype)
    k = torch.randn((sum(k_lens), kv_heads, dim), generator=g, device=device).to(dtype)
    v = torch.randn((sum(k_lens), kv_heads, dim), generator=g, device=device).to(dtype)
    return q, k, v


def split(k, v, k_lens, kp=None, vp=None):
    return [(a, b, kp, vp) for a, b in zip(k.split(k_lens), v.split(k_lens))]


SHAPES = [
    # q_lens, k_lens, heads, kv_heads, dim, dtype
    ([1], [1], 1, 1, 128, torch.bfloat16),
    ([1], [1], 8, 8, 64, torch.float16),
    ([1], [129], 8, 1, 128, torch.bfloat16),
    ([1], [8192], 32, 8, 128, torch.bfloat16),
    ([1, 1, 1], [127, 128, 2000], 16, 2, 64, torch.bfloat16),
    ([128], [128], 4, 4, 128, torch.bfloat16),
    ([129, 0, 1, 300], [129, 0, 1, 300], 8, 2, 128, torch.float16),
    ([257], [257], 2, 2, 64, torch.bfloat16),
    ([100, 5, 64], [700, 5, 64], 12, 4, 128, torch.bfloat16),         # groups of 3
    ([33, 70], [33, 1000], 10, 2, 64, torch.float16),                 # groups of 5
    ([17, 1], [140, 555], 7, 1, 128, torch.bfloat16),                 # groups of 7
    ([9, 2], [300, 77], 128, 1, 128, torch.bfloat16),                 # a group fills a tile
    ([40], [400], 96, 1, 64, torch.bfloat16),                         # groups of 96: a tile holds one token
    ([5, 3], [2, 0], 4, 2, 128, torch.bfloat16),                      # rows that see no key
    ([600], [1300], 4, 1, 128, torch.float16),
    ([1] * 40, list(range(1, 2400, 60)), 8, 2, 128, torch.bfloat16),
    ([0, 0, 2], [5, 0, 500], 8, 8, 128, torch.bfloat16),
]


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("q_lens,k_lens,heads,kv_heads,dim,dtype", SHAPES)
def test_packed_batches_match_the_definition(device, q_lens, k_lens, heads, kv_heads, dim, dtype, causal):
    q, k, v = make(device, q_lens, k_lens, heads, kv_heads, dim, dtype, seed=sum(k_lens))
    got, lse = attention.attention_varlen(q, (k, v), sums(q_lens, device), sums(k_lens, device), causal=causal, return_lse=True)
    attention.check_status(device)
    assert_close(got, lse, expected(q, q_lens, split(k, v, k_lens), causal))


def paged(k, v, k_lens, page_size, seed, layout="rows", fill=float("nan")):
    """Scatter packed keys to random pages of pools full of NaN; returns (pools, table)."""

    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page_size) for n in k_lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g)
    heads, dim = k.shape[1:]
    table = torch.full((len(k_lens), max(max(need), 1)), -1, dtype=torch.int32)
    pools = []
    for x in (k, v):
        pool = torch.full((pages, page_size, heads, dim), fill, dtype=k.dtype, device=k.device)
        if layout == "heads":
            pool = pool.transpose(1, 2).contiguous().transpose(1, 2)
        at = 0
        for b, part in enumerate(x.split(k_lens)):
            for c in range(need[b]):
                chunk = part[c * page_size:(c + 1) * page_size]
                pool[int(order[at]), :chunk.shape[0]] = chunk
                table[b, c] = order[at]
                at += 1
        pools.append(pool)
    return tuple(pools), table.to(k.device)


@pytest.mark.gpu
@pytest.mark.parametrize("page_size,layout", [(128, "rows"), (256, "heads"), (384, "rows")])
@pytest.mark.parametrize("q_lens,k_lens,heads,kv_heads,dim,dtype", SHAPES[2:8:2] + SHAPES[8:17:3] + SHAPES[15:])
def test_paged_batches_match_the_definition(device, q_lens, k_lens, heads, kv_heads, dim, dtype, page_size, layout):
    q, k, v = make(device, q_lens, k_lens, heads, kv_heads, dim, dtype, seed=page_size)
    pools, table = paged(k, v, k_lens, page_size, seed=sum(k_lens), layout=layout)
    lens = torch.tensor(k_lens, dtype=torch.int32, device=device)
    got, lse = attention.attention_paged(q, pools, table, sums(q_lens, device), lens, return_lse=True)
    attention.check_status(device)
    assert_close(got, lse, expected(q, q_lens, split(k, v, k_lens)))


PREFIXES = [
    # prefix, q_lens, k_lens, heads, kv_heads, dim, dtype
    (1, [1], [1], 4, 2, 128, torch.bfloat16),
    (300, [1, 1, 1], [5, 1, 140], 8, 2, 64, torch.float16),
    (2048, [1, 2, 0, 3], [17, 128, 0, 300], 32, 8, 128, torch.bfloat16),
    (129, [1] * 50, [3 + i for i in range(50)], 16, 2, 128, torch.bfloat16),
    (1000, [70, 3, 130], [70, 40, 500], 6, 2, 128, torch.float16),
    (5000, [1, 1], [0, 1], 8, 8, 64, torch.bfloat16),                 # a request without a key of its own
    (0, [1, 9], [44, 9], 8, 2, 128, torch.bfloat16),                  # no prefix at all
    (256, [4, 2], [2, 2], 16, 1, 128, torch.bfloat16),                # rows that see the prefix only
    (4096, [3] * 30, [40 + 9 * i for i in range(30)], 28, 4, 128, torch.float16),   # groups of 7
]


@pytest.mark.gpu
@pytest.mark.parametrize("page_size", [0, 128, 256])
@pytest.mark.parametrize("prefix,q_lens,k_lens,heads,kv_heads,dim,dtype", PREFIXES)
def test_shared_prefixes_match_the_definition(device, prefix, q_lens, k_lens, heads, kv_heads, dim, dtype, page_size):
    q, k, v = make(device, q_lens, [prefix] + k_lens, heads, kv_heads, dim, dtype, seed=prefix)
    kp, vp, k_own, v_own = k[:prefix], v[:prefix], k[prefix:], v[prefix:]
    if page_size == 0:
        got, lse = attention.shared_prefix_attention(q, (kp, vp), (k_own, v_own), sums(q_lens, device), sums(k_lens, device),
                                                     return_lse=True)
    else:
        pools, table = paged(k, v, [prefix] + k_lens, page_size, seed=prefix)
        lens = torch.tensor(k_lens, dtype=torch.int32, device=device)
        prefix_table = table[0, :-(-prefix // page_size)].contiguous()
        got, lse = attention.shared_prefix_attention_paged(q, pools, prefix_table, prefix, table[1:], sums(q_lens, device), lens,
                                                           return_lse=True)
    attention.check_status(device)
    assert_close(got, lse, expected(q, q_lens, split(k_own, v_own, k_lens, kp, vp)))


@pytest.mark.gpu
def test_slices_of_one_projection_and_a_strided_output(device):
    q_lens, k_lens, heads, kv_heads, dim = [100, 30], [100, 30], 8, 2, 128
    g = torch.Generator(device=device).manual_seed(3)
    fused = torch.randn((130, heads + 2 * kv_heads, dim), generator=g, device=device).to(torch.bfloat16)
    q, k, v = fused.split([heads, kv_heads, kv_heads], dim=1)
    wide = torch.full((130, heads, 2 * dim), 7.0, dtype=torch.bfloat16, device=device)
    out = wide[:, :, :dim]
    got = attention.attention_varlen(q, (k, v), sums(q_lens, device), sums(k_lens, device), out=out, scale=0.3)
    assert got is out
    assert_close(out, None, expected(q, q_lens, split(k, v, k_lens), scale=0.3))
    assert bool((wide[:, :, dim:] == 7.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("prefix,q_lens,k_lens,heads,kv_heads,dim", [
    (0, [1] * 20, [300 * i + 1 for i in range(20)], 16, 2, 128), (0, [5, 300, 2, 90], [5, 900, 3000, 90], 8, 4, 64),
    (700, [3] * 12, [9 * i + 3 for i in range(12)], 14, 2, 128)])
def test_an_output_in_the_place_of_the_queries(device, prefix, q_lens, k_lens, heads, kv_heads, dim):
    q, k, v = make(device, q_lens, [prefix] + k_lens, heads, kv_heads, dim, torch.bfloat16)
    kp, vp, k, v = k[:prefix], v[:prefix], k[prefix:], v[prefix:]
    want = expected(q, q_lens, split(k, v, k_lens, kp if prefix else None, vp if prefix else None))
    attention.shared_prefix_attention(q, (kp, vp), (k, v), sums(q_lens, device), sums(k_lens, device), out=q)
    attention.check_status(device)
    assert_close(q, None, want)


@pytest.mark.gpu
@pytest.mark.parametrize("q_lens,k_lens,heads,kv_heads,dim", [
    ([150, 3, 200], [400, 3, 900], 8, 2, 128), ([1] * 9, [70 * i for i in range(9)], 14, 2, 64), ([1], [5000], 32, 8, 128)])
def test_tensors_with_their_heads_first(device, q_lens, k_lens, heads, kv_heads, dim):
    q, k, v = make(device, q_lens, k_lens, heads, kv_heads, dim, torch.bfloat16)
    first = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    want = expected(q, q_lens, split(k, v, k_lens))
    for out in (None, torch.empty_like(first[0])):
        got = attention.attention_varlen(first[0], tuple(first[1:]), sums(q_lens, device), sums(k_lens, device), out=out)
        assert got.is_contiguous() if out is None else got is out
        assert_close(got, None, want)
    attention.check_status(device)


@pytest.mark.gpu
@pytest.mark.parametrize("q_len,k_len", [(1, 70), (40, 200), (300, 300)])
def test_rows_behind_the_last_request(device, q_len, k_len):
    q, k, v = make(device, [q_len + 37], [k_len + 50], 8, 2, 128, torch.bfloat16)
    k[k_len:], v[k_len:] = float("nan"), float("inf")
    q[q_len:] = float("nan")
    cu_q, cu_k = sums([q_len], device), sums([k_len], device)
    want = expected(q[:q_len], [q_len], [(k[:k_len], v[:k_len], None, None)])
    got, lse = attention.attention_varlen(q, (k, v), cu_q, cu_k, return_lse=True)
    assert_close(got, lse, want)
    assert bool((got[q_len:] == 0).all()) and bool((lse[q_len:] == -math.inf).all())
    out = torch.full_like(q, 5.0)
    attention.attention_varlen(q, (k, v), cu_q, cu_k, out=out)
    assert_close(out, None, want)
    assert bool((out[q_len:] == 5.0).all()), "rows behind the last request were written"
    torch.full_like(lse, 7.0)                                # (what the next call's log-sum-exps may find in their memory)
    _, lse = attention.attention_varlen(q, (k, v), cu_q, cu_k, out=out, return_lse=True)
    assert_close(out, lse, want)
    assert bool((out[q_len:] == 5.0).all()) and bool((lse[q_len:] == -math.inf).all())
    # and rows in front of the first one
    for given in (None, torch.full_like(q, 5.0)):
        shifted = attention.attention_varlen(torch.cat([q[q_len:q_len + 30], q[:q_len], q[q_len:q_len + 7]]), (k, v), cu_q + 30, cu_k,
                                             out=None if given is None else given[:q_len + 37])
        assert_close(shifted[30:], None, want)
        rest = torch.cat([shifted[:30], shifted[30 + q_len:]])
        assert bool((rest == (0.0 if given is None else 5.0)).all())
    attention.check_status(device)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 2, 128), (16, 2, 64)])
@pytest.mark.parametrize("at", [317, 271, 0, 499])
def test_what_a_row_does_not_see_does_not_reach_it(device, bad, heads, kv_heads, dim, at):
    """Keys and values behind a row's last visible key may hold anything; the rows that see them get it."""

    n = 500
    q, k, v = make(device, [n], [n], heads, kv_heads, dim, torch.bfloat16, seed=1)
    clean = expected(q, [n], [(k, v, None, None)])
    k_bad, v_bad = k.clone(), v.clone()
    v_bad[at, 0, 3] = bad
    got, lse = attention.attention_varlen(q, (k, v_bad), sums([n], device), sums([n], device), return_lse=True)
    group = heads // kv_heads
    touched = torch.zeros_like(q, dtype=torch.bool)
    touched[at:, :group, 3] = True
    assert_close(torch.where(touched, clean[0].to(q.dtype), got), lse, clean)
    assert not bool(got[touched].isfinite().any())
    if not math.isnan(bad):
        assert bool((got[touched] == bad).all())
    k_bad[at, 0, 3] = float("nan")
    got, lse = attention.attention_varlen(q, (k_bad, v), sums([n], device), sums([n], device), return_lse=True)
    touched = torch.zeros((n, heads), dtype=torch.bool, device=device)
    touched[at:, :group] = True
    assert bool(lse[touched].isnan().all()) and bool(got[touched].isnan().all())
    assert_close(torch.where(touched.unsqueeze(2), clean[0].to(q.dtype), got), torch.where(touched, clean[1].float(), lse), clean)


@pytest.mark.gpu
def test_scores_far_from_zero(device):
    """Row maxima that keep growing along the keys, up to scores of several hundred."""

    q, k, v = make(device, [64], [2000], 4, 2, 128, torch.bfloat16, seed=2)
    ramp = torch.linspace(0.0, 3.0, 2000, device=device)[:, None, None]
    q = q.abs()
    k = (ramp * k.abs()).to(torch.bfloat16)
    for sign in (1, -1):
        got, lse = attention.attention_varlen(q, (sign * k, v), sums([64], device), sums([2000], device), return_lse=True)
        assert_close(got, lse, expected(q, [64], [(sign * k, v, None, None)]))


@pytest.mark.gpu
def test_a_captured_call_follows_its_buffers(device):
    """Two graphs of the same tensors, replayed with other lengths in place, next to an eager call on another stream."""

    q, k, v = make(device, [300], [4000], 8, 2, 128, torch.bfloat16, seed=4)
    cu_q, cu_k = sums([100, 200], device), sums([1000, 3000], device)
    stream = torch.cuda.Stream(device)
    stream.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(stream):
        attention.attention_varlen(q, (k, v), cu_q, cu_k)
    torch.cuda.current_stream(device).wait_stream(stream)
    graphs = []
    for causal in (True, False):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = attention.attention_varlen(q, (k, v), cu_q, cu_k, causal=causal, return_lse=True)
        graphs.append((graph, held, causal))
    for q_lens, k_lens in (([100, 200], [1000, 3000]), ([1, 250], [2500, 700]), ([0, 1], [0, 4000])):
        cu_q.copy_(sums(q_lens, device))
        cu_k.copy_(sums(k_lens, device))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            eager = attention.attention_varlen(q, (k, v), cu_q, cu_k, return_lse=True)
        for graph, _, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        total_q, total_k = sum(q_lens), sum(k_lens)
        parts = split(k[:total_k], v[:total_k], k_lens)
        for _, held, causal in graphs:
            assert_close(held[0], held[1], expected(q[:total_q], q_lens, parts, causal))
        assert_close(eager[0], eager[1], expected(q[:total_q], q_lens, parts))
    attention.check_status(device)


@pytest.mark.gpu
def test_calls_repeat_to_the_bit(device):
    q_lens, k_lens = [1, 300, 2, 1], [5000, 300, 900, 1]
    q, k, v = make(device, q_lens, k_lens, 16, 2, 128, torch.bfloat16, seed=5)
    cu_q, cu_k = sums(q_lens, device), sums(k_lens, device)
    first = attention.attention_varlen(q, (k, v), cu_q, cu_k, return_lse=True)
    for _ in range(5):
        again = attention.attention_varlen(q, (k, v), cu_q, cu_k, return_lse=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.gpu
def test_more_requests_than_a_plan_block_has_threads(device):
    g = torch.Generator().manual_seed(8)
    k_lens = torch.randint(0, 200, (1500,), generator=g).tolist()
    q_lens = [min(k, int(n)) for k, n in zip(k_lens, torch.randint(0, 4, (1500,), generator=g))]
    q, k, v = make(device, q_lens, k_lens, 2, 1, 64, torch.bfloat16, seed=8)
    got, lse = attention.attention_varlen(q, (k, v), sums(q_lens, device), sums(k_lens, device), return_lse=True)
    attention.check_status(device)
    assert_close(got, lse, expected(q, q_lens, split(k, v, k_lens)))


@pytest.mark.gpu
@pytest.mark.parametrize("q_lens,k_lens,heads,kv_heads,dim", [
    ([1] * 40, [257 + 31 * i for i in range(40)], 16, 2, 128), ([0] * 90 + [60, 1, 29] + [0] * 7, [300] * 90 + [700, 5, 29] + [9] * 7, 14, 2, 64),
    ([2, 0, 1, 0, 3, 0] * 7, [900, 0, 1, 4, 130, 128] * 7, 7, 1, 128), ([100] + [0] * 100, [6000] + [70] * 100, 32, 4, 128)])
def test_batches_with_no_more_tokens_than_requests(device, q_lens, k_lens, heads, kv_heads, dim):
    q, k, v = make(device, q_lens, k_lens, heads, kv_heads, dim, torch.bfloat16)
    for causal in (True, False):
        got, lse = attention.attention_varlen(q, (k, v), sums(q_lens, device), sums(k_lens, device), causal=causal, return_lse=True)
        assert_close(got, lse, expected(q, q_lens, split(k, v, k_lens), causal))
    attention.check_status(device)


@pytest.mark.gpu
@pytest.mark.parametrize("prefix,q_lens,k_lens,heads,kv_heads,dim", [
    (30000, [3] * 70, [5 + 11 * i for i in range(70)], 32, 4, 128),        # the prefix in many chunks, several waves of items
    (0, [1] * 30 + [700], [200 * i + 1 for i in range(30)] + [9000], 16, 2, 128),
    (0, [3000], [3000], 16, 4, 64)])
def test_batches_of_many_waves(device, prefix, q_lens, k_lens, heads, kv_heads, dim):
    q, k, v = make(device, q_lens, [prefix] + k_lens, heads, kv_heads, dim, torch.float16, seed=prefix + 1)
    kp, vp, k, v = k[:prefix], v[:prefix], k[prefix:], v[prefix:]
    got, lse = attention.shared_prefix_attention(q, (kp, vp), (k, v), sums(q_lens, device), sums(k_lens, device), return_lse=True)
    attention.check_status(device)
    assert_close(got, lse, expected(q, q_lens, split(k, v, k_lens, kp if prefix else None, vp if prefix else None)))


@pytest.mark.gpu
def test_rows_of_a_cache_whose_offsets_pass_32_bits(device):
    """Pools of 2.2 billion elements: the last pages lie beyond 2^32 bytes and 2^31 elements."""

    pages, page, heads, dim = 8400, 256, 8, 128
    pool = torch.empty((pages, page, heads, dim), dtype=torch.bfloat16, device=device)
    assert pool.numel() > 1 << 31
    k_len = 700
    q, k, v = make(device, [5], [k_len], 16, heads, dim, torch.bfloat16, seed=9)
    table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32, device=device)
    from fusedindextopk_b200 import paged as pages_module

    position = torch.arange(k_len, device=device)
    slots = table[0].long()[position // page] * page + position % page
    values = pool.clone()
    pages_module.append_tokens(slots, (k, v), (pool, values))
    lens = torch.tensor([k_len], dtype=torch.int32, device=device)
    got, lse = attention.attention_paged(q, (pool, values), table, sums([5], device), lens, return_lse=True)
    attention.check_status(device)
    assert_close(got, lse, expected(q, [5], [(k, v, None, None)]))


@pytest.mark.gpu
def test_calls_on_two_streams_at_once(device):
    shapes = [([1] * 20, [300 * i + 7 for i in range(20)]), ([900, 30], [900, 4000])]
    made = [make(device, ql, kl, 16, 2, 128, torch.bfloat16, seed=i) for i, (ql, kl) in enumerate(shapes)]
    ends = [(sums(ql, device), sums(kl, device)) for ql, kl in shapes]
    streams = [torch.cuda.Stream(device) for _ in shapes]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(attention.attention_varlen(made[i][0], made[i][1:], *ends[i]))
    torch.cuda.synchronize()
    attention.check_status(device)
    for i, (ql, kl) in enumerate(shapes):
        q, k, v = made[i]
        assert_close(got[i][0], None, expected(q, ql, split(k, v, kl)))
        assert all(torch.equal(got[i][0], other) for other in got[i])


@pytest.mark.gpu
def test_a_wait_that_runs_out_is_reported_and_the_next_call_is_right(device):
    q, k, v = make(device, [40], [500], 8, 2, 128, torch.bfloat16)
    cu_q, cu_k = sums([40], device), sums([500], device)
    out = torch.empty_like(q)
    template = attention._check_call(torch, q, (k, v), None, 0, cu_q, cu_k, out, True, None)
    args = _lib.AttentionArgs.from_buffer_copy(template.bytes)
    args.withhold_loads, args.wait_limit_ns = 1, 1_000_000
    workspace = torch.empty(template.workspace_bytes, dtype=torch.uint8, device=device)
    args.q, args.out, args.cu_q, args.cu_k = q.data_ptr(), out.data_ptr(), cu_q.data_ptr(), cu_k.data_ptr()
    args.k, args.v, args.workspace, args.workspace_bytes = k.data_ptr(), v.data_ptr(), workspace.data_ptr(), workspace.numel()
    _lib.check(_lib.load_library().itk_attention(ctypes.byref(args), _lib.current_stream(torch, device)))
    with pytest.raises(_lib.ItkError, match="wait"):
        attention.check_status(device)
    got, lse = attention.attention_varlen(q, (k, v), cu_q, cu_k, return_lse=True)
    attention.check_status(device)
    assert_close(got, lse, expected(q, [40], [(k, v, None, None)]))


@pytest.mark.gpu
def test_bad_lengths_and_pages_are_clamped_and_reported(device):
    q, k, v = make(device, [4], [300], 4, 2, 128, torch.bfloat16)
    cu = torch.tensor([0, 9], dtype=torch.int32, device=device)             # more rows than q has
    attention.attention_varlen(q, (k, v), cu, sums([300], device))
    with pytest.raises(_lib.ItkError, match="lengths"):
        attention.check_status(device)
    attention.check_status(device)                                          # reported once
    pools, table = paged(k, v, [300], 128, seed=1, fill=0.0)
    lens = torch.tensor([300], dtype=torch.int32, device=device)
    for page in (-1, 1000):
        table[0, 1] = page
        attention.attention_paged(q, pools, table, sums([4], device), lens)
        with pytest.raises(_lib.ItkError, match="page"):
            attention.check_status(device)
    attention.attention_paged(q, pools, table[:, :1], sums([4], device), lens)   # 300 keys on one page of 128
    with pytest.raises(_lib.ItkError, match="lengths"):
        attention.check_status(device)


@pytest.mark.gpu
def test_refusals(device):
    q, k, v = make(device, [4], [30], 4, 2, 128, torch.bfloat16)
    cu_q, cu_k = sums([4], device), sums([30], device)

    def refused(match, *args, call=attention.attention_varlen, **kwargs):
        with pytest.raises(ValueError, match=match):
            call(*args, **kwargs)

    refused("CUDA", q.cpu(), (k, v), cu_q, cu_k)
    refused("bfloat16 or float16", q.float(), (k, v), cu_q, cu_k)
    refused("64 or 128", q[..., :96], (k[..., :96], v[..., :96]), cu_q, cu_k)
    refused("type of q", q, (k.half(), v.half()), cu_q, cu_k)
    refused("multiple of", q[:, :3], (k, v), cu_q, cu_k)
    refused("shape", q, (k, v[:20]), cu_q, cu_k)
    refused("int32", q, (k, v), cu_q.long(), cu_k)
    refused("entries", q, (k, v), cu_q, sums([10, 20], device))
    refused("B >= 1", q, (k, v), cu_q[:1], cu_k[:1])
    refused("aligned", torch.empty(4, 4, 132, dtype=q.dtype, device=device)[..., 4:], (k, v), cu_q, cu_k)
    refused("last dimension", q.transpose(1, 2).contiguous().transpose(1, 2), (k, v), cu_q, cu_k)
    refused("out must", q, (k, v), cu_q, cu_k, out=torch.empty(4, 4, 64, dtype=q.dtype, device=device))
    refused("overlap", q, (k, v), cu_q, cu_k, out=torch.empty(4, 4, 128, dtype=q.dtype, device=device)[:1].expand(4, 4, 128))
    refused("finite", q, (k, v), cu_q, cu_k, scale=float("inf"))
    refused("less than 2\\^31 own keys", q, (k[:1].expand(1 << 32, 2, 128), v[:1].expand(1 << 32, 2, 128)), cu_q, cu_k)
    refused("no backward", q.clone().requires_grad_(), (k, v), cu_q, cu_k)
    refused("no backward", q, (k, v.clone().requires_grad_()), cu_q, cu_k)
    refused("no backward", q, (k.clone().requires_grad_(), v), (k, v), cu_q, cu_k, call=attention.shared_prefix_attention)
    with torch.no_grad():
        attention.attention_varlen(q.clone().requires_grad_(), (k, v), cu_q, cu_k)
    pools, table = paged(k, v, [30], 128, seed=1)
    lens = torch.tensor([30], dtype=torch.int32, device=device)
    refused("multiple of 128", q, tuple(p[:, :64] for p in pools), table, cu_q, lens, call=attention.attention_paged)
    refused("one row per request", q, pools, table.repeat(2, 1), cu_q, lens, call=attention.attention_paged)
    refused("int32", q, pools, table.long(), cu_q, lens, call=attention.attention_paged)
    refused("cover", q, pools, table[0], 129, table, cu_q, lens, call=attention.shared_prefix_attention_paged)
    refused("same heads", q, (k[:, :1], v[:, :1]), (k, v), cu_q, cu_k, call=attention.shared_prefix_attention)
    empty = attention.attention_varlen(q[:0], (k, v), sums([0], device), cu_k)
    assert empty.shape == (0, 4, 128)


def test_c_entry_refuses_before_any_launch():
    build()
    library = _lib.load_library()
    args = _lib.AttentionArgs()
    assert library.itk_attention(None, None) == -1
    assert library.itk_attention(ctypes.byref(args), None) == -1
    args.heads, args.kv_heads, args.dim, args.tokens = 8, 3, 128, 5
    assert library.itk_attention(ctypes.byref(args), None) == -1
    assert b"multiple of kv_heads" in library.itk_last_error()
    args.kv_heads, args.dim = 2, 96
    assert library.itk_attention(ctypes.byref(args), None) == -1
    assert b"64 or 128" in library.itk_last_error()
    args.dim = 128
    assert library.itk_attention(ctypes.byref(args), None) == -1
    assert b"at least one request" in library.itk_last_error()
    args.requests = 1
    assert library.itk_attention(ctypes.byref(args), None) == -1
    assert b"must not be null" in library.itk_last_error()
    args.q = args.out = args.cu_q = args.lens_k = 1 << 20
    args.k = args.v = args.table = 1 << 20
    args.own.pages, args.own.page_size = 4, 96
    assert library.itk_attention(ctypes.byref(args), None) == -1
    assert b"multiple of 128" in library.itk_last_error()
    args.own.pages, args.own.page_size = 1 << 24, 128
    assert library.itk_attention(ctypes.byref(args), None) == -1
    assert b"2^31" in library.itk_last_error()
    args.own.pages, args.own.k_row_stride = 4, 12
    assert library.itk_attention(ctypes.byref(args), None) == -1
    assert b"multiples of 8" in library.itk_last_error()
    args.tokens = 0
    args.own.k_row_stride = 16
    assert library.itk_attention(ctypes.byref(args), None) == 0      # nothing to do


def test_argument_structs_match_the_header():
    import re
    from pathlib import Path

    text = (Path(__file__).resolve().parents[1] / "include" / "itk_b200.h").read_text()
    for name, mirror in (("itk_attention_args", _lib.AttentionArgs), ("itk_kv_segment", _lib.KvSegment),
                         ("itk_append_args", _lib.AppendArgs), ("itk_page_plan_args", _lib.PagePlanArgs)):
        body = text[text.index(f"typedef struct {name} {{"):text.index(f"}} {name};")]
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S).split("{", 1)[1]
        fields = [re.sub(r"[\s*]", " ", f).split()[-1] for line in body.split(";") for f in line.split(",") if f.strip()]
        assert fields == [field for field, _ in mirror._fields_]


@pytest.mark.gpu
@pytest.mark.parametrize("prefix", [0, 1000])
@pytest.mark.parametrize("empty", [0, 90, 1300])         # the plan in the attention kernel, the plan kernel, its uncached lengths
@pytest.mark.parametrize("ends", [[0, 30, 100, 40], [0, 100, 4], [0, 3, 90, 0], [70, 90, 100, 20]])
def test_row_ends_that_decrease_are_clamped_to_the_last_one(device, prefix, empty, ends):
    """Rows behind ``cu_seqlens_q[-1]`` belong to no request, whatever the ends before it say."""

    heads, kv_heads, dim = 16, 2, 128
    ends = ends + ends[-1:] * empty
    k_lens = ([200, 45, 33] * len(ends))[:len(ends) - 1]
    q, k, v = make(device, [120], [prefix] + k_lens, heads, kv_heads, dim, torch.bfloat16, seed=11)
    kp, vp, k, v = k[:prefix], v[:prefix], k[prefix:], v[prefix:]
    cu_q = torch.tensor(ends, dtype=torch.int32, device=device)
    got, lse = attention.shared_prefix_attention(q, (kp, vp), (k, v), cu_q, sums(k_lens, device), return_lse=True)
    with pytest.raises(_lib.ItkError, match="lengths"):
        attention.check_status(device)
    clamped = [min(end, ends[-1]) for end in ends]
    q_lens = [max(b - a, 0) for a, b in zip(clamped, clamped[1:])]
    first, last = clamped[0], clamped[0] + sum(q_lens)
    want = expected(q[first:last], q_lens, split(k, v, k_lens, kp if prefix else None, vp if prefix else None))
    assert_close(got[first:last], lse[first:last], want)
    for rest, rest_lse in ((got[:first], lse[:first]), (got[last:], lse[last:])):
        assert bool((rest == 0).all()) and bool((rest_lse == -math.inf).all())


@pytest.mark.gpu
def test_requests_whose_rows_overlap_are_reported_and_stay_in_their_buffers(device):
    """More entries in all than the buffers hold: every other request claims all rows and all keys."""

    heads, kv_heads, dim, tokens, keys, requests = 8, 1, 64, 600, 500, 4000
    q, k, v = make(device, [tokens], [keys], heads, kv_heads, dim, torch.bfloat16, seed=12)
    held = torch.full((tokens + 2, heads, dim), 9.0, dtype=q.dtype, device=device)
    cu_q, cu_k = (torch.tensor([0, n] * (requests // 2) + [n], dtype=torch.int32, device=device) for n in (tokens, keys))
    for kp, vp in ((k[:0], v[:0]), (k[:70], v[:70])):
        attention.shared_prefix_attention(q, (kp, vp), (k, v), cu_q, cu_k, out=held[1:-1])
        with pytest.raises(_lib.ItkError, match="lengths"):
            attention.check_status(device)
        assert bool((held[0] == 9).all()) and bool((held[-1] == 9).all())
        assert_close(held[1:-1], None, expected(q, [tokens], [(k, v, kp, vp)]))      # they all say the same of a row


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_what_lies_behind_the_ends_of_requests_changes_no_bit(device, dim):
    """Every value tile that ends inside a page is cleared by the guard before it is multiplied, in every call."""

    q_lens = [1, 130, 5, 64, 1, 257, 2] * 6
    k_lens = [n + 37 * i for i, n in enumerate(q_lens)]
    q, k, v = make(device, q_lens, k_lens, 16, 4, dim, torch.bfloat16, seed=13)
    cu_q, lens = sums(q_lens, device), torch.tensor(k_lens, dtype=torch.int32, device=device)
    held = [paged(k, v, k_lens, 256, seed=13, fill=fill) for fill in (0.0, float("nan"), float("inf"))]
    want = attention.attention_paged(q, *held[0], cu_q, lens, return_lse=True)
    for _ in range(10):
        for pools, table in held[1:]:
            got = attention.attention_paged(q, pools, table, cu_q, lens, return_lse=True)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    attention.check_status(device)


@pytest.mark.gpu
@pytest.mark.parametrize("tail", [12.3, 20.04, 25.01, 31.0])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_long_tail_behind_one_strong_key_keeps_its_weight(device, tail, dtype):
    """262144 keys of weight 2^-tail behind one of weight 1, uncut: 400 requests on the same pages.

    Weights as fp16 may lose 2^-32 of the largest each (a step of 2^-24 at 2^7 times their size, rounded to the nearest);
    everything else as in ``definition``.
    """

    requests, n, dim, page = 400, 1 << 18, 64, 256
    u = torch.finfo(dtype).eps / 2
    k = torch.zeros((n // page, page, 1, dim), dtype=dtype, device=device)
    k[..., 0] = -1.0
    k[0, 0] = 0.0
    v = torch.ones_like(k)
    v[0, 0, 0, 32:] = 0.0                       # half of the columns hold the tail alone
    q = torch.zeros((requests, 1, dim), dtype=dtype, device=device)
    q[..., 0] = 1.0
    scale = tail * math.log(2.0)
    weight = math.exp(-ctypes.c_float(scale).value)
    table = torch.arange(n // page, dtype=torch.int32, device=device).unsqueeze(0).expand(requests, -1)
    lens = torch.full((requests,), n, dtype=torch.int32, device=device)
    got, lse = attention.attention_paged(q, (k, v), table, sums([1] * requests, device), lens, scale=scale, return_lse=True)
    attention.check_status(device)
    total = 1.0 + (n - 1) * weight
    # scores are 0 and -scale exactly up to the scale's own product with log2(e): 4 e of the largest
    rel = 2 * 4 * E * scale + 2.0 ** -20 + n * E
    lost = 2.0 ** -32 * n if dtype == torch.float16 else 0.0
    for columns, want in ((slice(0, 32), 1.0), (slice(32, 64), (n - 1) * weight / total)):
        off = (got[:, 0, columns].double() - want).abs().max().item()
        assert off <= (2.01 * u + rel) * want + lost, (off / want, tail)
    assert (lse.double() - math.log(total)).abs().max().item() <= rel + 2.0 ** -20


@pytest.mark.gpu
@pytest.mark.parametrize("magnitude", [2.0 ** 10, 2.0 ** 20, 2.0 ** 24, 2.0 ** 25])
def test_weights_stay_finite_at_any_size_of_the_scores(device, magnitude):
    """Maxima that grow by about 2^8 from step to step, where fp16 weights come nearest to their largest value."""

    g = torch.Generator(device=device).manual_seed(14)
    n, dim = 6000, 64
    q = torch.zeros((8, 1, dim), dtype=torch.float16, device=device)
    k = torch.zeros((n, 1, dim), dtype=torch.float16, device=device)
    q[..., 0], q[..., 1] = 256.0, 1.0
    k[..., 0] = 256.0
    growth = 8 * math.log(2.0) * 65536.0 / magnitude               # a factor of 2^8 between the weights
    k[:, 0, 1] = (torch.arange(n, device=device) // 64 + 1.1 * torch.rand(n, generator=g, device=device)) * growth
    v = torch.rand((n, 1, dim), generator=g, device=device).to(torch.float16)
    got, lse = attention.attention_varlen(q, (k, v), sums([8], device), sums([n], device), causal=False,
                                          scale=magnitude / 65536.0, return_lse=True)
    attention.check_status(device)
    assert bool(got.isfinite().all()) and bool(lse.isfinite().all())
    # A mean of values in [0, 1]: the base is rounded up by two steps of a scaled score at most, 8 at 2^25 * log2(e), so the largest
    # weight is 2^-1 at least and its rounding off by 2^-11 of it; smaller ones by 2^-11 of theirs or 2^-25.
    assert bool((got >= 0).all()) and bool((got <= 1 + 2.0 ** -11 + 2.0 ** -11 + n * 2.0 ** -24).all())


@pytest.mark.gpu
def test_a_long_request_among_empty_ones_fills_its_tiles(device):
    """What a step's buffers leave room for does not change how its rows are packed: 8 entries of 32 tokens, not 128 of two."""

    slots, heads, kv_heads, dim, keys = 256, 64, 8, 128, 3000
    q, k, v = make(device, [slots], [keys], heads, kv_heads, dim, torch.bfloat16, seed=15)
    cu_q, cu_k = sums([0] * 9 + [slots] + [0] * (slots - 10), device), sums([0] * 9 + [keys] + [0] * (slots - 10), device)
    out = torch.empty_like(q)
    template = attention._check_call(torch, q, (k, v), None, 0, cu_q, cu_k, out, True, None)
    args = _lib.AttentionArgs.from_buffer_copy(template.bytes)
    workspace = torch.empty(template.workspace_bytes, dtype=torch.uint8, device=device)
    args.q, args.out, args.cu_q, args.cu_k = q.data_ptr(), out.data_ptr(), cu_q.data_ptr(), cu_k.data_ptr()
    args.k, args.v, args.workspace, args.workspace_bytes = k.data_ptr(), v.data_ptr(), workspace.data_ptr(), workspace.numel()
    _lib.check(_lib.load_library().itk_attention(ctypes.byref(args), _lib.current_stream(torch, device)))
    attention.check_status(device)
    assert_close(out, None, expected(q, [slots], [(k, v, None, None)]))
    items = int(workspace[:4].view(torch.int32))          # the plan's first counter: units of work for every key head
    sms = torch.cuda.get_device_properties(device).multi_processor_count
    assert 8 <= items and items * kv_heads <= sms         # 64 entries fit a wave, cut as far as that allows


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 2, 128), (14, 2, 64), (96, 1, 128)])
def test_a_replayed_step_changes_between_single_tokens_and_chunks(device, heads, kv_heads, dim):
    """One graph of a step with 64 slots and 64 rows: single tokens, one long request, both, some rows unused."""

    slots = 64
    q, k, v = make(device, [slots], [6000], heads, kv_heads, dim, torch.bfloat16, seed=16)
    cu_q, cu_k = sums([1] * slots, device), sums([5] * slots, device)
    attention.attention_varlen(q, (k, v), cu_q, cu_k)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held, lse = attention.attention_varlen(q, (k, v), cu_q, cu_k, return_lse=True)
    for q_lens, k_lens in (([1] * 64, [90] * 64), ([0] * 30 + [64] + [0] * 33, [7] * 30 + [5000] + [3] * 33),
                           ([1] * 20 + [40] + [0] * 43, [150] * 20 + [900] + [1] * 43), ([2, 0, 3, 1] * 10 + [0] * 24, [60] * 64)):
        cu_q.copy_(sums(q_lens, device))
        cu_k.copy_(sums(k_lens, device))
        graph.replay()
        rows = sum(q_lens)
        assert_close(held, lse, expected(q[:rows], q_lens, split(k[:sum(k_lens)], v[:sum(k_lens)], k_lens)))
        assert bool((held[rows:] == 0).all()) and bool((lse[rows:] == -math.inf).all())
    attention.check_status(device)


def planned_rows(q_lens, k_lens, prefix, heads, kv_heads, sms, causal=True):
    """Partial rows and items of a plan, in plain arithmetic: entries, chunk length, slots (as ``csrc/itk_attention.cuh`` plans)."""

    group = heads // kv_heads
    tile_tokens = 128 // group
    span = 2 * tile_tokens
    entries = []                                              # tokens, key tiles, of the prefix
    if prefix:
        total_q = sum(q_lens)
        entries += [(min(span, total_q - at), -(-prefix // 128), True) for at in range(0, total_q, span)]
    for count, keys in zip(q_lens, k_lens):
        for at in range(0, count, span):
            tokens = min(span, count - at)
            seen = max(0, min(keys, keys - count + at + tokens)) if causal else keys
            entries.append((tokens, -(-seen // 128), False))
    units = [4 if tokens > tile_tokens else 3 for tokens, _, _ in entries]
    share = min(math.ceil(sum(t * u for (_, t, _), u in zip(entries, units)) * kv_heads / sms) + 1, 1 << 29)

    def chunks(tiles, unit, cost, whole):
        if whole and tiles * unit <= whole:
            return min(tiles, 1)
        return -(-tiles // max(2, -(-cost // unit)))

    cost, whole = min(share, max(share // 6, 24 * 4)), share // 2
    for eighth in range(8):
        length = share + share // 8 * eighth
        if sum(max(1, chunks(t, u, length, 0)) for (_, t, _), u in zip(entries, units)) * kv_heads <= sms:
            cost, whole = length, 0
            break
    rows = items = 0
    for (tokens, tiles, _), unit in zip(entries, units):
        cut = chunks(tiles, unit, cost, whole)
        slots = cut * (2 if unit == 3 and cut and -(-tiles // cut) > 1 else 1)
        items += max(1, cut)
        if prefix or slots > 1:
            rows += slots * tokens * group * kv_heads
    return rows, items


def test_the_workspace_holds_every_plan():
    """Against plans of random batches, of one long request among short ones, and of many equal ones."""

    build()
    import random

    library, rng, fullest = _lib.load_library(), random.Random(17), 0.0
    for case in range(600):
        kv_heads = rng.choice([1, 2, 3, 8, 16])
        heads, dim, sms = kv_heads * rng.choice([1, 2, 5, 7, 8, 16, 96]), rng.choice([64, 128]), rng.choice([132, 148, 160])
        requests = int(100 ** rng.random())
        q_lens = [int(10 ** rng.uniform(0, 3.3)) - 1 if rng.random() < 0.5 else 1 for _ in range(requests)]
        k_lens = [int(10 ** rng.uniform(0, rng.choice([2, 4, 5.5]))) for _ in range(requests)]
        if case % 3 == 0:                                     # one entry has nearly all of the work
            q_lens, k_lens = [1] * requests, [1] * requests
            q_lens[0], k_lens[0] = min(2 * (128 // (heads // kv_heads)), 1 + rng.randrange(300)), 1 << rng.randint(10, 20)
        prefix = rng.choice([0, 0, 100, 5000, 200000])
        args = _lib.AttentionArgs()
        args.tokens, args.requests, args.heads, args.kv_heads, args.dim, args.prefix_keys = (
            max(1, sum(q_lens)), requests, heads, kv_heads, dim, prefix)
        needed = ctypes.c_size_t(0)
        assert library.itk_attention_workspace_bytes(ctypes.byref(args), ctypes.byref(needed)) == 0
        rows, items = planned_rows(q_lens, k_lens, prefix, heads, kv_heads, sms, causal=rng.random() < 0.5)
        used = rows * 4 * (dim + 1) + 48 * items
        assert used <= needed.value, (case, used, needed.value)
        fullest = max(fullest, used / needed.value)
    assert 0.5 < fullest          # and it is no more than twice what some plan needs


def test_key_counts_whose_tiles_do_not_fit_31_bits_are_refused():
    build()
    library, args = _lib.load_library(), _lib.AttentionArgs()
    args.tokens, args.requests, args.heads, args.kv_heads, args.dim, args.scale = 1, 1, 1, 1, 64, 1.0
    args.q = args.out = args.cu_q = args.cu_k = args.k = args.v = 1 << 20
    args.own.pages = 1
    args.own.k_row_stride = args.own.k_head_stride = args.own.v_row_stride = args.own.v_head_stride = 64
    for keys in (_lib.MAX_ATTENTION_KEYS + 1, (1 << 31) - 1):
        args.own.page_size = keys
        assert library.itk_attention(ctypes.byref(args), None) == -1
        assert b"own keys: need at most 2147482624 keys" in library.itk_last_error()
    args.own.page_size = 1000
    args.k_prefix = args.v_prefix = args.prefix_table = 1 << 20
    args.prefix.pages, args.prefix.page_size, args.prefix.table_pages = 1, 128, 1 << 24
    for keys in (_lib.MAX_ATTENTION_KEYS + 1, (1 << 31) - 1):
        args.prefix_keys = keys
        assert library.itk_attention(ctypes.byref(args), None) == -1
        assert b"at most 2147482624 prefix keys" in library.itk_last_error()


@pytest.mark.gpu
def test_the_most_keys_a_request_may_have(device):
    """A table that names one page over and over; more keys than are allowed are clamped and reported."""

    page, columns, dim = 1024, 1 << 21, 64
    q, k, v = make(device, [1], [page], 1, 1, dim, torch.bfloat16, seed=18)
    pools = tuple(x.view(1, page, 1, dim) for x in (k, v))
    table = torch.zeros((1, columns), dtype=torch.int32, device=device)
    cu_q = sums([1], device)
    once = expected(q, [1], [(k, v, None, None)])[1].item()
    for keys in (_lib.MAX_ATTENTION_KEYS, (1 << 31) - 1):
        lens = torch.tensor([keys], dtype=torch.int32, device=device)
        got, lse = attention.attention_paged(q, pools, table, cu_q, lens, return_lse=True)
        if keys > _lib.MAX_ATTENTION_KEYS:
            with pytest.raises(_lib.ItkError, match="lengths"):
                attention.check_status(device)
        attention.check_status(device)
        assert bool(got.isfinite().all())
        # sums of 32 weights are added one after another by every thread: of n / 32 / 2 lanes / 148 CTAs, e each
        assert abs(lse.item() - once - math.log(_lib.MAX_ATTENTION_KEYS / page)) <= 2 * (1 << 31) / 32 / 2 / 148 * E + 1e-3


def test_attention_drops_no_gradient_and_no_tangent(monkeypatch):
    monkeypatch.setattr(_lib, "launch", lambda *_: pytest.fail("a launch"))
    q, k, v, kp, vp = (torch.ones(4, 2, 64) for _ in range(5))
    ends, out = torch.zeros(2, dtype=torch.int32), torch.ones(4, 2, 64)
    forward = torch.autograd.forward_ad

    def call(tensors, out=None):
        attention.shared_prefix_attention(tensors[0], tensors[3:], tensors[1:3], ends, ends, out=out)

    plain = [q, k, v, kp, vp]
    for i in range(5):
        with pytest.raises(ValueError, match="no backward"):
            call(plain[:i] + [plain[i].clone().requires_grad_()] + plain[i + 1:])
        with forward.dual_level(), torch.no_grad(), pytest.raises(ValueError, match="no forward-mode"):
            call(plain[:i] + [forward.make_dual(plain[i], torch.ones(4, 2, 64))] + plain[i + 1:])
    with pytest.raises(ValueError, match="no backward"):
        call(plain, out=out.clone().requires_grad_())
    with forward.dual_level(), pytest.raises(ValueError, match="CUDA"):         # a level without tangents changes nothing
        call(plain, out=out)


@pytest.mark.gpu
def test_a_given_output_counts_as_changed(device):
    q, k, v = make(device, [4], [30], 4, 2, 128, torch.bfloat16)
    out = torch.zeros_like(q)
    attention.attention_varlen(q, (k, v), sums([4], device), sums([30], device), out=out)
    assert (out._version, q._version, k._version) == (1, 0, 0)
