"""Page plans and token appends: block tables, slots and ranges against a plain loop, pools against torch."""

from __future__ import annotations

import copy
import ctypes
import dataclasses

import pytest
import torch

from fusedindextopk_b200 import _lib, paged
from fusedindextopk_b200.build import build


@pytest.fixture(scope="module")
def device():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return torch.device("cuda:0")


def plain_plan(table, old, new, free, page, rows):
    """The definition, one token at a time."""

    table = [list(r) for r in table]
    columns = len(table[0])
    slots, starts, ends, cu, lengths, flat, taken = [], [], [], [0], [], [], 0
    for b, (o, n) in enumerate(zip(old, new)):
        before, after = -(-o // page), -(-(o + n) // page)
        for c in range(before, columns):
            if c < after:
                table[b][c] = free[taken]
                taken += 1
            else:
                table[b][c] = -1
        first = len(flat)
        flat += table[b][:after]
        for position in range(o, o + n):
            slots.append(table[b][position // page] * page + position % page)
            starts.append(first * page)
            ends.append(first * page + position + 1)
        cu.append(cu[-1] + n)
        lengths.append(o + n)
    padding = rows - len(slots)
    flat += [0] * (len(table) * columns - len(flat))
    return table, slots + [-1] * padding, cu, lengths, flat, starts + [0] * padding, ends + [0] * padding, taken


def make(seed, requests, columns, page, new_max, spare=2):
    g = torch.Generator().manual_seed(seed)
    new = torch.randint(0, new_max + 1, (requests,), generator=g)
    old = torch.randint(0, columns * page - new_max + 1, (requests,), generator=g)
    old[torch.rand(requests, generator=g) < 0.3] = 0
    before = -(-old // page)
    need = int((-(-(old + new) // page) - before).sum())
    order = torch.randperm(int(before.sum()) + need + spare, generator=g).tolist()
    table = [[-7] * columns for _ in range(requests)]
    for b in range(requests):
        for c in range(int(before[b])):
            table[b][c] = order.pop()
    return table, old.tolist(), new.tolist(), order


def gpu(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


CASES = [(1, 1, 128, 1, 0), (1, 40, 128, 300, 5), (8, 16, 128, 1, 0), (7, 5, 256, 400, 100), (600, 9, 128, 200, 3),
         (513, 3, 384, 2, 17), (3000, 4, 128, 1, 0), (2000, 1, 128, 2, 1), (4001, 1, 128, 1, 2)]


@pytest.mark.gpu
@pytest.mark.parametrize("requests,columns,page,new_max,spare_rows", CASES)
def test_page_plans_match_the_definition(device, requests, columns, page, new_max, spare_rows):
    table, old, new, free = make(requests, requests, columns, page, new_max)
    rows = sum(new) + spare_rows
    want = plain_plan(table, old, new, free, page, rows)
    plan = paged.make_page_plan(requests, columns, rows, page_size=page, device=device)
    wide = torch.full((requests, columns + 3), 99, dtype=torch.int32, device=device)
    block_table = wide[:, :columns]
    block_table.copy_(gpu(table, device))
    for _ in range(2):                                       # the same step twice gives the same plan
        got = paged.plan_pages(plan, block_table, gpu(old, device), gpu(new, device), gpu(free, device))
        assert got.block_table is block_table
        assert block_table.tolist() == want[0]
        assert got.slots.tolist() == want[1]
        assert got.cu_seqlens_q.tolist() == want[2]
        assert got.lengths.tolist() == want[3]
        assert got.flat_table.tolist() == want[4]
        assert got.k_start.tolist() == want[5]
        assert got.k_end.tolist() == want[6]
        assert got.pages_needed.tolist() == [want[7]]
    assert bool((wide[:, columns:] == 99).all())
    paged.check_serving_status(device)


@pytest.mark.gpu
def test_a_captured_plan_follows_its_lengths(device):
    requests, columns, page, rows = 5, 6, 128, 40
    plan = paged.make_page_plan(requests, columns, rows, page_size=page, device=device)
    block_table = torch.full((requests, columns), -1, dtype=torch.int32, device=device)
    old, new, free = gpu([0] * 5, device), gpu([0] * 5, device), gpu(list(range(30)), device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.plan_pages(plan, block_table, old, new, free)
    held, used = [0] * requests, 0
    for step in ([8, 0, 1, 30, 1], [1, 1, 1, 1, 1], [0, 0, 0, 0, 40], [7, 9, 0, 0, 0]):
        table = block_table.tolist()
        pool = list(range(used, 30))
        want = plain_plan(table, held, step, pool, page, rows)
        old.copy_(gpu(held, device))
        new.copy_(gpu(step, device))
        free[:len(pool)] = gpu(pool, device)
        graph.replay()
        assert block_table.tolist() == want[0] and plan.slots.tolist() == want[1] and plan.flat_table.tolist() == want[4]
        held, used = want[3], used + want[7]
    paged.check_serving_status(device)


@pytest.mark.gpu
def test_plans_that_do_not_fit_are_reported_and_stay_in_their_buffers(device):
    page = 128
    plan = paged.make_page_plan(2, 2, 300, page_size=page, device=device)
    table = torch.full((2, 2), -1, dtype=torch.int32, device=device)
    # three pages wanted, two there
    got = paged.plan_pages(plan, table, gpu([0, 0], device), gpu([200, 100], device), gpu([4, 9], device))
    assert table.tolist() == [[4, 9], [-1, -1]] and got.pages_needed.tolist() == [3]
    assert got.slots[:200].tolist() == [4 * page + i for i in range(128)] + [9 * page + i for i in range(72)]
    assert bool((got.slots[200:] == -1).all())
    with pytest.raises(_lib.ItkError, match="out of pages"):
        paged.check_serving_status(device)
    # a request that outgrows its table row
    got = paged.plan_pages(plan, table, gpu([200, 0], device), gpu([100, 0], device), gpu([5, 6], device))
    assert got.lengths.tolist() == [256, 0] and bool((got.slots[56:] == -1).all()) and bool((got.slots[:56] >= 0).all())
    with pytest.raises(_lib.ItkError, match="out of pages"):
        paged.check_serving_status(device)
    # more new tokens than rows, and a negative length
    got = paged.plan_pages(plan, table, gpu([-5, 0], device), gpu([200, 200], device), gpu([1, 2, 3, 4], device))
    assert got.cu_seqlens_q.tolist() == [0, 200, 300]
    with pytest.raises(_lib.ItkError, match="lengths"):
        paged.check_serving_status(device)
    huge = 2 ** 31 - 1
    paged.plan_pages(plan, table, gpu([huge, huge], device), gpu([huge, huge], device), gpu([1], device))
    with pytest.raises(_lib.ItkError):
        paged.check_serving_status(device)


def plain_append(slots, k, v, pools, index=None, index_pools=None):
    kept = slots >= 0
    at = slots[kept]
    for x, pool in ((k, pools[0]), (v, pools[1])):
        flat = pool.reshape(-1, *pool.shape[2:]).clone()
        flat[at] = x[kept]
        pool.copy_(flat.view(pool.shape))
    if index is not None:
        x = index[kept].float()
        amax = x.abs().amax(-1).clamp(min=1e-4)
        scales = amax / torch.full_like(amax, 448.0)       # by a tensor: a true division, not a product with 1/448
        index_pools[0].view(torch.uint8).view(-1, 128)[at] = (x / scales.unsqueeze(1)).to(torch.float8_e4m3fn).view(torch.uint8)
        index_pools[1].view(-1)[at] = scales


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,heads,dim,page,layout,index_dtype", [
    (1, 1, 64, 128, "rows", torch.bfloat16), (5, 3, 128, 128, "rows", None), (64, 8, 128, 256, "heads", torch.float32),
    (1000, 2, 64, 100, "rows", torch.bfloat16), (333, 40, 128, 128, "heads", torch.bfloat16), (0, 2, 64, 128, "rows", None)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_appends_match_torch(device, tokens, heads, dim, page, layout, index_dtype, dtype):
    g = torch.Generator(device=device).manual_seed(tokens)
    pages = tokens // page + 3
    fused = torch.randn((tokens, 3 * heads, dim), generator=g, device=device).to(dtype)
    k, v = fused[:, :heads], fused[:, 2 * heads:]
    pools = [torch.randn((pages, page, heads, dim), generator=g, device=device).to(dtype) for _ in range(2)]
    if layout == "heads":
        pools = [p.transpose(1, 2).contiguous().transpose(1, 2) for p in pools]
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(tokens))[:tokens].to(device)
    slots[::7] = -1
    index = index_pools = want_index = None
    if index_dtype is not None:
        index = torch.randn((tokens, 128), generator=g, device=device).to(index_dtype)
        index[: tokens // 3] *= 1e-6                                       # below the amax floor
        index_pools = (torch.randn((pages, page, 128), generator=g, device=device).to(torch.float8_e4m3fn),
                       torch.rand((pages, page), generator=g, device=device))
        want_index = tuple(p.clone() for p in index_pools)
    want = [p.clone() for p in pools]
    plain_append(slots, k, v, want, index, want_index)
    paged.append_tokens(slots, (k, v), tuple(pools), index_keys=index, index_pools=index_pools)
    assert torch.equal(pools[0], want[0]) and torch.equal(pools[1], want[1])
    if index is not None:
        assert torch.equal(index_pools[0].view(torch.uint8), want_index[0].view(torch.uint8))
        assert bool((index_pools[1] == want_index[1]).all())
    paged.check_serving_status(device)


@pytest.mark.gpu
def test_slots_behind_the_pool_are_skipped_and_reported(device):
    k = torch.ones((3, 2, 64), dtype=torch.bfloat16, device=device)
    pools = [torch.zeros((2, 128, 2, 64), dtype=torch.bfloat16, device=device) for _ in range(2)]
    slots = torch.tensor([256, 3, 1 << 40], dtype=torch.int64, device=device)
    paged.append_tokens(slots, (k, k), tuple(pools))
    assert int(pools[0].sum()) == 128 and bool((pools[0][0, 3] == 1).all())
    with pytest.raises(_lib.ItkError, match="page or slot"):
        paged.check_serving_status(device)


@pytest.mark.gpu
def test_more_tokens_than_a_32_bit_thread_number_counts(device):
    tokens = (1 << 27) + 5
    k = torch.randn((1, 1, 64), dtype=torch.bfloat16, device=device)
    pools = [torch.zeros((1, 128, 1, 64), dtype=torch.bfloat16, device=device) for _ in range(2)]
    slots = torch.full((tokens,), -1, dtype=torch.int64, device=device)
    slots[-1], slots[1 << 20] = 7, 9
    paged.append_tokens(slots, (k.expand(tokens, 1, 64), k.expand(tokens, 1, 64)), tuple(pools))
    for pool in pools:
        assert torch.equal(pool[0, 7], k[0]) and torch.equal(pool[0, 9], k[0]) and int((pool != 0).any(-1).sum()) == 2


@pytest.mark.gpu
def test_two_plans_take_turns_and_one_does_not_read_itself(device):
    plans = [paged.make_page_plan(3, 4, 8, page_size=128, device=device) for _ in range(2)]
    table = torch.full((3, 4), -1, dtype=torch.int32, device=device)
    free, new = gpu(list(range(12)), device), gpu([1, 0, 2], device)
    paged.plan_pages(plans[0], table, gpu([127, 0, 255], device), new, free)
    paged.plan_pages(plans[1], table, plans[0].lengths, new, free[6:])
    assert plans[1].lengths.tolist() == [129, 0, 259]
    with pytest.raises(_lib.ItkError, match="share memory"):
        paged.plan_pages(plans[1], table, plans[1].lengths, new, free)


@pytest.mark.gpu
def test_append_refusals(device):
    k = torch.ones((3, 2, 64), dtype=torch.bfloat16, device=device)
    pool = torch.zeros((2, 128, 2, 64), dtype=torch.bfloat16, device=device)
    slots = torch.arange(3, device=device)

    def refused(match, *args, **kwargs):
        with pytest.raises(ValueError, match=match):
            paged.append_tokens(*args, **kwargs)

    refused("CUDA", slots, (k.cpu(), k.cpu()), (pool, pool))
    refused("shape", slots, (k, k[:2]), (pool, pool))
    refused("type of k", slots, (k, k), (pool.half(), pool))
    refused("int64", slots.int(), (k, k), (pool, pool))
    refused("64 or 128", slots, (k[..., :32], k[..., :32]), (pool[..., :32], pool[..., :32]))
    refused("index_pools", slots, (k, k), (pool, pool), index_keys=torch.zeros((3, 128), device=device))
    refused("aligned", slots, (torch.ones((3, 2, 68), dtype=k.dtype, device=device)[..., 4:], k), (pool, pool))
    plan = paged.make_page_plan(2, 4, 10, page_size=128, device=device)
    table, ints = torch.zeros((2, 4), dtype=torch.int32, device=device), gpu([1, 2], device)
    for bad in ((table[:1], ints, ints, ints), (table.long(), ints, ints, ints), (table, ints[:1], ints, ints),
                (table, ints, ints.long(), ints), (table, ints, ints, ints.cpu()), (table[:1].expand(2, 4), ints, ints, ints)):
        with pytest.raises(ValueError):
            paged.plan_pages(plan, *bad)


def test_page_plan_sizes_are_refused_without_a_gpu():
    for kwargs in (dict(requests=0), dict(requests=20000), dict(table_pages=0), dict(page_size=100), dict(rows=-1), dict(rows=1 << 31),
                   dict(requests=16384, table_pages=1024), dict(device="cpu")):
        size = dict(requests=4, table_pages=4, rows=4, page_size=128, device="cuda") | kwargs
        with pytest.raises(ValueError):
            paged.make_page_plan(size.pop("requests"), size.pop("table_pages"), size.pop("rows"), **size)


def test_c_entries_refuse_before_any_launch():
    build()
    library = _lib.load_library()
    plan, append = _lib.PagePlanArgs(), _lib.AppendArgs()
    assert library.itk_plan_pages(None, None) == -1
    assert library.itk_plan_pages(ctypes.byref(plan), None) == -1
    plan.requests, plan.table_pages, plan.page_size, plan.table_stride = 16384, 1024, 128, 1024
    assert library.itk_plan_pages(ctypes.byref(plan), None) == -1
    assert b"2^31" in library.itk_last_error()
    plan.requests = 4
    assert library.itk_plan_pages(ctypes.byref(plan), None) == -1
    assert b"must not be null" in library.itk_last_error()
    apart = {name: (i + 1) << 20 for i, name in enumerate(
        ("table", "old", "fresh", "free_pages", "slots", "cu_q", "lengths", "flat", "k_start", "k_end", "pages_needed"))}
    plan.free_count, plan.rows = 5, 10
    for read in ("old", "fresh", "free_pages"):
        for written in ("table", "slots", "cu_q", "lengths", "flat", "k_start", "k_end", "pages_needed"):
            for name, address in apart.items():
                setattr(plan, name, address)
            setattr(plan, read, apart[written] - 12)                # its last words on the other's first
            assert library.itk_plan_pages(ctypes.byref(plan), None) == -1
            assert b"share memory" in library.itk_last_error()
    assert library.itk_append_tokens(None, None) == -1
    assert library.itk_append_tokens(ctypes.byref(append), None) == -1
    append.tokens, append.kv_heads, append.dim, append.pages, append.page_size = 3, 2, 128, 2, 128
    assert library.itk_append_tokens(ctypes.byref(append), None) == -1
    assert b"must not be null" in library.itk_last_error()
    append.slots = append.k = append.v = append.k_pool = append.v_pool = 1 << 20
    append.k_row_stride = 4
    assert library.itk_append_tokens(ctypes.byref(append), None) == -1
    assert b"multiples of 8" in library.itk_last_error()
    append.k_row_stride, append.v = 8, (1 << 20) + 8
    assert library.itk_append_tokens(ctypes.byref(append), None) == -1
    assert b"aligned" in library.itk_last_error()


def cpu_plan(requests=2, columns=3, rows=5):
    """A plan whose buffers live on the CPU: enough for what the host keeps of it."""

    def buffer(count, dtype=torch.int32):
        return torch.zeros(count, dtype=dtype)

    return paged.PagePlan(requests, columns, rows, 128, buffer(rows, torch.int64), buffer(requests + 1), buffer(requests),
                          buffer(requests * columns), buffer(rows), buffer(rows), buffer(1))


def test_a_changed_plan_keeps_no_argument_block():
    plan = cpu_plan()
    plan.templates["key"] = "block"
    assert dataclasses.replace(plan, slots=torch.zeros(5, dtype=torch.int64)).templates == {}
    other = copy.copy(plan)
    assert plan.templates == other.templates == {"key": "block"}
    other.rows = 4
    assert other.templates == {} and plan.templates == {"key": "block"}
    plan.slots = torch.zeros(5, dtype=torch.int64)
    assert plan.templates == {}


def test_no_address_is_kept_between_plans(monkeypatch):
    """The block of a call holds the addresses of the plan it was made for, also of one copied after a call."""

    seen = []
    monkeypatch.setattr(_lib, "launch", lambda torch, function, block, *rest: seen.append(_lib.PagePlanArgs.from_buffer_copy(block)))
    sizes = _lib.PagePlanArgs(*[None] * 11, 3, 2, 3, 128, 4, 5)
    monkeypatch.setattr(paged, "_check_plan", lambda torch, plan, *tensors: _lib.CallTemplate(sizes, device=None))
    table, ints = torch.zeros((2, 3), dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    first = cpu_plan()
    paged.plan_pages(first, table, ints, ints, ints)
    moved = dataclasses.replace(first, lengths=torch.zeros(2, dtype=torch.int32))
    for plan in (first, copy.deepcopy(first), copy.copy(first), moved):
        paged.plan_pages(plan, table, ints, ints, ints)
        for field, name in (("slots", "slots"), ("cu_q", "cu_seqlens_q"), ("lengths", "lengths"), ("flat", "flat_table"),
                            ("k_start", "k_start"), ("k_end", "k_end"), ("pages_needed", "pages_needed")):
            assert getattr(seen[-1], field) == getattr(plan, name).data_ptr()
        assert (seen[-1].table, seen[-1].old, seen[-1].rows, seen[-1].page_size) == (table.data_ptr(), ints.data_ptr(), 5, 128)


@pytest.mark.gpu
def test_copied_and_replaced_plans_fill_their_own_buffers(device):
    plan = paged.make_page_plan(3, 4, 8, page_size=128, device=device)
    table = torch.full((3, 4), -1, dtype=torch.int32, device=device)
    free, old = gpu(list(range(12)), device), gpu([127, 0, 255], device)
    paged.plan_pages(plan, table, old, gpu([1, 0, 2], device), free)
    before = plan.lengths.tolist()
    changed = copy.copy(plan)
    changed.lengths = torch.zeros_like(plan.lengths)
    for other in (copy.deepcopy(plan), dataclasses.replace(plan, lengths=torch.zeros_like(plan.lengths)), changed):
        got = paged.plan_pages(other, table, old, gpu([2, 1, 3], device), free)
        assert got is other and other.lengths.tolist() == [129, 1, 258]
        assert plan.lengths.tolist() == before
    plan.k_end = torch.zeros(7, dtype=torch.int32, device=device)
    with pytest.raises(ValueError, match="k_end"):
        paged.plan_pages(plan, table, old, gpu([1, 0, 2], device), free)
    paged.check_serving_status(device)


@pytest.mark.gpu
def test_as_many_tokens_as_an_append_takes(device):
    tokens = (1 << 31) - 1
    k = torch.randn((1, 1, 64), dtype=torch.bfloat16, device=device)
    pools = [torch.zeros((1, 128, 1, 64), dtype=torch.bfloat16, device=device) for _ in range(2)]
    slots = torch.full((tokens,), -1, dtype=torch.int64, device=device)
    slots[-1], slots[0] = 7, 9
    paged.append_tokens(slots, (k.expand(tokens, 1, 64), k.expand(tokens, 1, 64)), tuple(pools))
    for pool in pools:
        assert torch.equal(pool[0, 7], k[0]) and torch.equal(pool[0, 9], k[0]) and int((pool != 0).any(-1).sum()) == 2
    paged.check_serving_status(device)


@pytest.mark.gpu
def test_a_report_is_not_lost_while_another_one_is_read(device):
    """Calls on another stream, of another thread, while this one reads and clears the status again and again."""

    import random
    import threading
    import time

    k = torch.ones((1, 1, 64), dtype=torch.bfloat16, device=device)
    pools = tuple(torch.zeros((1, 128, 1, 64), dtype=torch.bfloat16, device=device) for _ in range(2))
    slots = torch.full((1,), 500, dtype=torch.int64, device=device)            # behind the pool
    paged.check_serving_status(device)
    stream, rng = torch.cuda.Stream(device), random.Random(19)

    def call(delay):
        until = time.perf_counter() + delay
        while time.perf_counter() < until:
            pass
        with torch.cuda.stream(stream):
            paged.append_tokens(slots, (k, k), pools)

    def reported():
        try:
            paged.check_serving_status(device)
        except _lib.ItkError:
            return True
        return False

    torch.cuda.synchronize()
    for number in range(400):
        thread = threading.Thread(target=call, args=(rng.random() * 2e-4,))
        thread.start()
        seen = False
        while thread.is_alive():
            seen |= reported()
        thread.join()
        assert reported() or seen, f"the report of call {number} was lost"


def cpu_append(**changes):
    """Arguments of an append whose checks and launch are left out."""

    given = dict(slots=torch.arange(3), k=torch.ones(3, 2, 64), v=torch.ones(3, 2, 64), k_pool=torch.zeros(2, 128, 2, 64),
                 v_pool=torch.zeros(2, 128, 2, 64), index_keys=torch.ones(3, 128), index_pool=torch.zeros(2, 128, 128),
                 index_scales=torch.zeros(2, 128)) | changes
    return ((given["slots"], (given["k"], given["v"]), (given["k_pool"], given["v_pool"])),
            dict(index_keys=given["index_keys"], index_pools=(given["index_pool"], given["index_scales"])), given)


@pytest.mark.parametrize("name", ["k", "v", "k_pool", "v_pool", "index_keys", "index_pool", "index_scales"])
def test_an_append_drops_no_gradient_and_no_tangent(monkeypatch, name):
    monkeypatch.setattr(_lib, "launch", lambda *_: pytest.fail("a launch"))
    plain = cpu_append()[2][name]
    args, kwargs, _ = cpu_append(**{name: plain.clone().requires_grad_()})
    with pytest.raises(ValueError, match="no backward"):
        paged.append_tokens(*args, **kwargs)
    forward = torch.autograd.forward_ad
    with forward.dual_level(), torch.no_grad():
        args, kwargs, _ = cpu_append(**{name: forward.make_dual(plain, torch.ones_like(plain))})
        with pytest.raises(ValueError, match="no forward-mode"):
            paged.append_tokens(*args, **kwargs)


def test_what_the_calls_write_counts_as_changed(monkeypatch):
    """Autograd refuses to use a saved tensor that was written meanwhile: that takes its version."""

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0, raising=False)
    monkeypatch.setattr(_lib, "load_library", lambda: type("Library", (), {
        "itk_append_tokens": staticmethod(lambda block, stream: 0), "itk_plan_pages": staticmethod(lambda block, stream: 0)}))
    template = _lib.CallTemplate(_lib.AppendArgs(), device=torch.device("cuda", 0))
    monkeypatch.setattr(paged, "_check_append", lambda *_: template)
    monkeypatch.setattr(paged, "_APPEND_TEMPLATES", {})
    args, kwargs, given = cpu_append()
    monkeypatch.setattr(paged, "_require", lambda condition, message: None)         # (the alignment of CPU tensors)
    paged.append_tokens(*args, **kwargs)
    assert {name: t._version for name, t in given.items()} == dict(
        slots=0, k=0, v=0, k_pool=1, v_pool=1, index_keys=0, index_pool=1, index_scales=1)
    saved = torch.ones(2, 128, 2, 64, requires_grad=True)
    product = saved * given["k_pool"]
    paged.append_tokens(*args, **kwargs)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.sum().backward()
    plan = cpu_plan()
    monkeypatch.setattr(paged, "_check_plan", lambda *_: _lib.CallTemplate(_lib.PagePlanArgs(), device=torch.device("cuda", 0)))
    table, ints = torch.zeros((2, 3), dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    paged.plan_pages(plan, table, ints, ints, ints)
    assert ints._version == 0 and table._version == plan.slots._version == plan.lengths._version == plan.k_end._version == 1


@pytest.mark.gpu
def test_an_append_raises_the_versions_of_its_pools(device):
    k = torch.ones((3, 2, 64), dtype=torch.bfloat16, device=device)
    pools = tuple(torch.zeros((2, 128, 2, 64), dtype=torch.bfloat16, device=device) for _ in range(2))
    paged.append_tokens(torch.arange(3, device=device), (k, k), pools)
    assert [t._version for t in (k, *pools)] == [0, 1, 1]
    with torch.inference_mode():
        held = tuple(p.clone() for p in pools)
    paged.append_tokens(torch.arange(3, device=device), (k, k), held)           # inference tensors have no versions
    paged.check_serving_status(device)


@pytest.mark.gpu
def test_padding_of_the_free_list_counts_as_no_page(device):
    plan = paged.make_page_plan(3, 2, 300, page_size=128, device=device)
    table = torch.full((3, 2), -1, dtype=torch.int32, device=device)
    old, padded = gpu([0, 0, 0], device), gpu([4, 9, -1, -1], device)
    paged.plan_pages(plan, table, old, gpu([100, 100, 0], device), padded)
    paged.check_serving_status(device)                                        # the padding is not needed
    got = paged.plan_pages(plan, table, old, gpu([100, 130, 0], device), padded)
    assert table.tolist() == [[4, -1], [9, -1], [-1, -1]] and got.pages_needed.tolist() == [3]
    assert bool((got.slots[:228] >= 0).all()) and bool((got.slots[228:] == -1).all())
    with pytest.raises(_lib.ItkError, match="out of pages"):
        paged.check_serving_status(device)


def test_buffers_that_share_memory_are_refused():
    build()
    library, plan = _lib.load_library(), _lib.PagePlanArgs()
    plan.requests, plan.table_pages, plan.page_size, plan.table_stride, plan.free_count, plan.rows = 4, 6, 128, 8, 5, 10
    names = ("table", "slots", "cu_q", "lengths", "flat", "k_start", "k_end", "pages_needed")
    for first in names:
        for second in names:
            if first == second:
                continue
            for i, name in enumerate(("old", "fresh", "free_pages", *names)):
                setattr(plan, name, (i + 1) << 20)
            setattr(plan, first, getattr(plan, second))        # a table that is the plan's flat one, for example
            assert library.itk_plan_pages(ctypes.byref(plan), None) == -1
            assert b"share memory with one another" in library.itk_last_error()


@pytest.mark.gpu
def test_a_plan_may_have_more_room_than_it_says(device):
    plan = dataclasses.replace(paged.make_page_plan(3, 4, 20, page_size=128, device=device), rows=5)
    table = torch.full((3, 4), -1, dtype=torch.int32, device=device)
    plan.slots.fill_(77)
    got = paged.plan_pages(plan, table, gpu([0, 0, 0], device), gpu([1, 2, 1], device), gpu([3, 1, 2], device))
    assert got.slots.tolist() == [384, 128, 129, 256, -1] + [77] * 15
    paged.check_serving_status(device)
