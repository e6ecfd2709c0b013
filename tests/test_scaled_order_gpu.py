"""Appending to a cache of 8 bits rows of one block that do not stand together: they are taken one after another, as their tokens are."""

import pytest
import torch

from plain_scaled import BLOCK, normed, turned
from test_scaled_cache_gpu import DEVICE, TYPES, held_by, kernels, nearly, pages_of, prepared, same

pytestmark = pytest.mark.gpu


def append_in_order(plane, rows, slots):
    """The rule: rows of a block that follow each other are a run; a block of several runs has its tokens appended by one, the lowest first."""
    limit = plane.codes.shape[0] * plane.page
    runs, at = [], 0
    while at < len(slots):
        end = at + 1
        while end < len(slots) and 0 <= slots[at] < limit and slots[end] == slots[end - 1] + 1 and slots[end] // BLOCK == slots[at] // BLOCK:
            end += 1
        if 0 <= slots[at] < limit:
            runs.append((at, end))
        at = end
    by_block = {}
    for a, e in runs:
        by_block.setdefault(slots[a] // BLOCK, []).append((a, e))
    for mine in by_block.values():
        if len(mine) == 1:
            a, e = mine[0]
            plane.append(rows[a:e], slots[a:e])
        else:
            for row in sorted((r for a, e in mine for r in range(a, e)), key=lambda r: slots[r]):
                plane.append(rows[row : row + 1], slots[row : row + 1])


def orders(name, n, seed):
    """A permutation of the rows (-1: a row that goes nowhere)."""
    g = torch.Generator().manual_seed(seed)
    if name == "padding-between":
        return [i for r in range(n) for i in ([r, -1] if r % 5 == 2 else [r])]
    if name == "interleaved":
        half = -(-n // 2)
        return [i for r in range(half) for i in (r, half + r) if i < n]
    if name == "backwards":
        return list(range(n))[::-1]
    if name == "halves-exchanged":
        return list(range(n // 2, n)) + list(range(n // 2))
    if name == "one-far-away":
        return list(range(1, n)) + [0]
    return torch.randperm(n, generator=g).tolist()


@pytest.mark.parametrize("order", ["padding-between", "interleaved", "backwards", "halves-exchanged", "one-far-away", "anyhow"])
@pytest.mark.parametrize("starts,counts", [([3], [7]), ([0, 9, 40], [20, 3, 30]), ([5, 0], [170, 200])], ids=["few", "some", "many"])
@pytest.mark.parametrize("dtype,dim,vdim,size,page", [("f32", 64, 64, 64, 64), ("bf16", 128, 80, 128, 32), ("bf16", 40, 48, 48, 16)])
def test_rows_of_a_block_in_any_order(dtype, dim, vdim, size, page, starts, counts, order):
    heads, n = 3, sum(counts)
    own, planes = prepared(starts, counts, page, heads, size, n + size)
    at = orders(order, n, n)
    slots = [own[r] if r >= 0 else (-1 if i % 2 else 2**31 - 1) for i, r in enumerate(at)]
    g = torch.Generator().manual_seed(n)
    rows = (torch.randn((len(at), heads * (dim + vdim)), generator=g) * torch.exp(2.0 * torch.randn((len(at), 1), generator=g))).to(TYPES[dtype])
    k_pages, v_pages = pages_of(planes)
    kernels().scaled_append(rows.to(DEVICE), None, 0, heads * dim, k_pages, v_pages, torch.tensor(slots, dtype=torch.int32, device=DEVICE),
                            torch.zeros(len(at), dtype=torch.int32, device=DEVICE), heads, heads, dim, vdim)
    append_in_order(planes[0], rows[:, : heads * dim].view(-1, heads, dim), slots)
    append_in_order(planes[1], rows[:, heads * dim :].reshape(-1, heads, vdim), slots)
    for got, plane in zip(held_by(k_pages, v_pages), planes):
        same(got, plane.held())


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("counts", [[30, 1, 9], [200, 90, 3]], ids=["few", "many"])
def test_turned_and_normed_rows_in_any_order(counts, norm):
    heads, kv_heads, dim, page, starts = 4, 2, 64, 32, [3, 15, 0]
    n = sum(counts)
    own, planes = prepared(starts, counts, page, kv_heads, dim, 5)
    at = torch.randperm(n, generator=torch.Generator().manual_seed(n)).tolist()
    slots = [own[r] for r in at]
    g = torch.Generator().manual_seed(6)
    rows = torch.randn((n, (heads + 2 * kv_heads) * dim), generator=g)
    positions = torch.randint(0, 100000, (n,), generator=g, dtype=torch.int32)
    f = 10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32)
    gains = torch.rand(dim, generator=g) + 0.5 if norm else None
    on = lambda t: None if t is None else t.to(DEVICE)
    k_pages, v_pages = pages_of(planes)
    q = kernels().scaled_append(on(rows), 0, heads * dim, (heads + kv_heads) * dim, k_pages, v_pages, torch.tensor(slots, dtype=torch.int32, device=DEVICE), on(positions), heads,
                                kv_heads, dim, dim, q_gain=on(gains), k_gain=on(gains), eps=1e-5, frequencies=on(f), rot_dims=dim, v_frequencies=on(f), v_rot_dims=32, short_rows=20)
    wide = rows.double()
    q_want, k_want = wide[:, : heads * dim].view(n, heads, dim), wide[:, heads * dim : (heads + kv_heads) * dim].reshape(n, kv_heads, dim)
    v_want = turned(wide[:, (heads + kv_heads) * dim :].reshape(n, kv_heads, dim), positions, f, 32, "half")
    if norm:
        q_want, k_want = normed(q_want, gains, 1e-5), normed(k_want, gains, 1e-5)
    q_want, k_want = turned(q_want, positions, f, dim, "half"), turned(k_want, positions, f, dim, "half")
    # a norm (below 2^-19 relative), two products and a sum of pair elements, and the rounding to the type
    assert bool(((q.cpu().double().view(n, heads, dim) - q_want).abs() <= 2.0**-24 * q_want.abs() + 2.0**-19 * q_want.abs().amax()).all())
    append_in_order(planes[0], k_want, slots)
    append_in_order(planes[1], v_want, slots)
    k_got, v_got = held_by(k_pages, v_pages)
    same(v_got, planes[1].held())
    if norm:
        # (a code that fell to the other side of a border may be rounded again as its block grows, once a doubling at most: counted as a row more each time)
        nearly(k_got, planes[0], 4 * n)
    else:
        same(k_got, planes[0].held())


@pytest.mark.parametrize("shift", [0, 1, 2, 3])
@pytest.mark.parametrize("counts", [[257, 2], [1000, 30], [2049, 4], [2600, 1]], ids=str)
def test_slots_anywhere_in_memory_and_many_of_them(counts, shift):
    """Slots that begin on any four bytes, and as many as are looked over in one, two and more goes: the first row's block is met again by the last row, or by one in the middle."""
    page, size = 64, 16
    n = sum(counts)
    own, planes = prepared([2, 30], counts, page, 1, size, n)
    slots = own[1:] + own[:1]
    slots[n // 2], slots[n - 2] = slots[n - 2], slots[n // 2]
    rows = torch.randn((n, 2 * size), generator=torch.Generator().manual_seed(n)) * torch.exp(torch.randn((n, 1), generator=torch.Generator().manual_seed(1)))
    k_pages, v_pages = pages_of(planes)
    memory = torch.zeros(n + 8, dtype=torch.int32, device=DEVICE)
    given = memory[shift : shift + n]
    given.copy_(torch.tensor(slots, dtype=torch.int32))
    kernels().scaled_append(rows.to(DEVICE), None, 0, size, k_pages, v_pages, given, torch.zeros(n, dtype=torch.int32, device=DEVICE), 1, 1, size, size)
    for plane, at in zip(planes, (0, size)):
        append_in_order(plane, rows[:, at : at + size].reshape(n, 1, size), slots)
    for got, plane in zip(held_by(k_pages, v_pages), planes):
        same(got, plane.held())


def test_a_row_apart_in_a_captured_call():
    """Replayed with other slots: together at capture, apart at replay, and the other way round."""
    K, page, size, n = kernels(), 32, 32, 40
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEVICE)
    together, apart = list(range(n)), list(range(0, n, 2)) + list(range(1, n, 2))
    rows = [torch.randn((n, 2 * size), generator=torch.Generator().manual_seed(i)).to(DEVICE) for i in range(4)]
    for first, second in ((together, apart), (apart, together)):
        pages = K.scaled_pages(2, 1, page, size, DEVICE)
        x, slots = rows[0].clone(), ints(first)
        call = lambda: K.scaled_append(x, None, 0, size, *pages, slots, slots, 1, 1, size, size)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        for i, order in enumerate((first, second, second, first)):
            x.copy_(rows[i])
            slots.copy_(ints(order))
            graph.replay()
            torch.cuda.synchronize()
            wanted = K.scaled_pages(2, 1, page, size, DEVICE)
            K.scaled_append(rows[i], None, 0, size, *wanted, ints(order), ints(order), 1, 1, size, size)
            for a, b in zip(pages, wanted):   # (every block is begun afresh)
                assert torch.equal(a.codes.view(torch.uint8)[0], b.codes.view(torch.uint8)[0]) and torch.equal(a.scales[0], b.scales[0])


@pytest.mark.parametrize("starts,counts", [([0, 9, 40, 31], [20, 1, 30, 2]), ([5, 0], [170, 200])], ids=["some", "many"])
def test_a_caller_that_says_so_gets_the_same(starts, counts):
    heads, size, n = 3, 64, sum(counts)
    own, planes = prepared(starts, counts, 32, heads, size, n)
    rows = torch.randn((n, 2 * heads * size), generator=torch.Generator().manual_seed(n)) * torch.exp(torch.randn((n, 1), generator=torch.Generator().manual_seed(2)))
    slots = torch.tensor(own, dtype=torch.int32, device=DEVICE)
    results = []
    for together in (False, True):
        pages = pages_of(planes)
        kernels().scaled_append(rows.to(DEVICE), None, 0, heads * size, *pages, slots, slots, heads, heads, size, size, together=together)
        results.append(pages)
    for a, b in zip(*results):
        assert torch.equal(a.codes.view(torch.uint8), b.codes.view(torch.uint8)) and torch.equal(a.scales, b.scales)
