"""Keys and values in 8 bits: the append kernel and what the pages hold behind it, against the plain implementation in 64 bits."""

import pytest
import torch

from plain_scaled import BLOCK, PlainPlane, laid, normed, turned

pytestmark = pytest.mark.gpu
DEVICE = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def kernels():
    from mini_llm_amd.ops import kernels as K

    return K


def slots_of(starts, counts, page, seed):
    """A request of counts[i] tokens from offset starts[i] on, each page anywhere: (slots, pages)."""
    order = torch.randperm(sum(-(-(s + c) // page) for s, c in zip(starts, counts)) + 2, generator=torch.Generator().manual_seed(seed)).tolist()
    slots, total = [], len(order)
    for s, c in zip(starts, counts):
        mine = [order.pop() for _ in range(-(-(s + c) // page))]
        slots += [mine[p // page] * page + p % page for p in range(s, s + c)]
    return slots, total


def prepared(starts, counts, page, heads, size, seed, spread=1.0):
    """Pages in use: everything before and behind the new rows holds numbers, at scales that differ by block."""
    slots, pages = slots_of(starts, counts, page, seed)
    g = torch.Generator().manual_seed(seed + 1)
    planes = []
    for _ in range(2):
        plane = PlainPlane(pages, heads, page, size)
        old = torch.randn((pages * page, heads, size), generator=g).double() * torch.exp(spread * torch.randn((pages * page, 1, 1), generator=g).double())
        plane.append(old, range(pages * page))
        planes.append(plane)
    return slots, planes


def pages_of(planes):
    K = kernels()
    return K.ScaledPages(*laid(planes[0], True, DEVICE)), K.ScaledPages(*laid(planes[1], False, DEVICE))


def held_by(pages_k, pages_v):
    """Everything the pages hold, through the framework's own reading: [num_pages, heads, page, size] each."""
    num, heads, page, size = pages_k.shape
    k, v = kernels().scaled_rows(pages_k, pages_v, torch.arange(num * page, dtype=torch.int32, device=DEVICE), out_dtype=torch.float32)
    return [t.view(num, page, heads, size).transpose(1, 2).double().cpu() for t in (k, v)]


def same(got, want):
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


def nearly(got, plane, rows_of_call):
    """What is held, where keys were computed in 32-bit on their way (a norm): a number next to a border may fall to either side of it, so a
    code differs by one step, 2^-3 of the number (or of 2^-6 scale, the smallest with three bits behind the leading one), in few places."""
    want = plane.held()
    step = torch.maximum(want.abs(), 2.0**-6 * (2.0 ** plane.e.double()).repeat_interleave(BLOCK, dim=-1)[..., None]) * 2.0**-3
    assert bool(((got - want).abs() <= step).all())
    # a relative error of the key of at most 2^-20 (norm: sum of up to 256 squares, root, two products) crosses a border of steps 2^-4 apart or
    # more for at most one number in 2^14 on average; ten times that and three more are allowed
    assert int((got != want).sum()) <= rows_of_call * want.shape[1] * want.shape[3] * 10 / 2**14 + 3


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,dim,vdim,size,page", [(1, 16, 16, 16, 16), (3, 64, 64, 64, 64), (2, 40, 48, 48, 32), (2, 128, 80, 128, 128), (1, 256, 200, 256, 16)])
@pytest.mark.parametrize("starts,counts", [([0], [1]), ([15, 16, 3, 47], [1, 1, 1, 1]), ([0, 5, 15], [16, 40, 2]), ([7], [300])], ids=["first", "tokens", "portions", "long"])
def test_what_is_held_is_the_plain_rule_to_the_bit(dtype, heads, dim, vdim, size, page, starts, counts):
    n = sum(counts)
    slots, planes = prepared(starts, counts, page, heads, size, n + size)
    g = torch.Generator().manual_seed(n)
    spread = torch.exp(2.0 * torch.randn((n, 1), generator=g))       # scales grow in some blocks and not in others
    rows = (torch.randn((n, heads * (dim + vdim) + 3), generator=g) * spread).to(TYPES[dtype])
    k_pages, v_pages = pages_of(planes)
    device_rows = rows.to(DEVICE)
    kernels().scaled_append(device_rows, None, 1, 2 + heads * dim, k_pages, v_pages, torch.tensor(slots, dtype=torch.int32, device=DEVICE),
                            torch.zeros(n, dtype=torch.int32, device=DEVICE), heads, heads, dim, vdim)
    planes[0].append(rows[:, 1 : 1 + heads * dim].view(n, heads, dim), slots)
    planes[1].append(rows[:, 2 + heads * dim : 2 + heads * (dim + vdim)].reshape(n, heads, vdim), slots)
    for got, plane in zip(held_by(k_pages, v_pages), planes):
        same(got, plane.held())
    assert torch.equal(k_pages.scales.cpu().double(), 2.0 ** planes[0].e.double()) and torch.equal(v_pages.scales.cpu().double(), 2.0 ** planes[1].e.double())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("pairing,rot,v_rot", [("half", 64, 0), ("neighbours", 64, 64), ("half", 16, 32), ("neighbours", 2, 0)])
@pytest.mark.parametrize("norm", [None, "gains", "unit"])
def test_queries_and_keys_turn_on_their_way(dtype, pairing, rot, v_rot, norm):
    heads, kv_heads, dim, vdim, size, page = 4, 2, 64, 48, 64, 32
    starts, counts = [3, 0, 31], [30, 1, 2]
    n = sum(counts)
    slots, planes = prepared(starts, counts, page, kv_heads, size, 5)
    g = torch.Generator().manual_seed(6)
    rows = torch.randn((n, heads * dim + kv_heads * (dim + vdim)), generator=g).to(TYPES[dtype])
    positions = torch.randint(0, 100000, (n,), generator=g, dtype=torch.int32)
    f, vf = 10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32), 5000.0 ** (-torch.arange(16, dtype=torch.float64) / 16)
    if v_rot == 64:
        v_rot = 48
        vf = 5000.0 ** (-torch.arange(24, dtype=torch.float64) / 24)
    gains = (torch.rand(dim, generator=g) + 0.5, torch.rand(dim, generator=g) + 0.5) if norm == "gains" else (None, None)
    k_pages, v_pages = pages_of(planes)
    on = lambda t: None if t is None else t.to(DEVICE)
    q = kernels().scaled_append(on(rows), 0, heads * dim, (heads + kv_heads) * dim, k_pages, v_pages, torch.tensor(slots, dtype=torch.int32, device=DEVICE), on(positions), heads,
                                kv_heads, dim, vdim, q_gain=on(gains[0]), k_gain=on(gains[1]), unit=norm == "unit", eps=1e-5, frequencies=on(f), rot_dims=rot, pairing=pairing,
                                v_frequencies=on(vf) if v_rot else None, v_rot_dims=v_rot, v_pairing="half")
    wide = rows.double()
    q_want, k_want = wide[:, : heads * dim].view(n, heads, dim), wide[:, heads * dim : (heads + kv_heads) * dim].reshape(n, kv_heads, dim)
    v_want = wide[:, (heads + kv_heads) * dim :].reshape(n, kv_heads, vdim)
    if norm:
        q_want, k_want = normed(q_want, gains[0], 1e-5), normed(k_want, gains[1], 1e-5)
    q_want, k_want = (turned(t, positions, f, rot, pairing) for t in (q_want, k_want))
    v_want = turned(v_want, positions, vf, v_rot, "half")
    # the query: a norm (the sum of 64 squares, a root, two products: below 2^-19 relative), two products and a sum of pair elements, and the
    # rounding to the type
    size_of_pair = q_want.abs().amax()
    eps = torch.finfo(TYPES[dtype]).eps / 2
    assert q.dtype == TYPES[dtype] and bool(((q.cpu().double().view(n, heads, size)[..., :dim] - q_want).abs() <= eps * q_want.abs() + 2.0**-19 * size_of_pair).all())
    planes[0].append(k_want, slots)
    planes[1].append(v_want, slots)
    k_got, v_got = held_by(k_pages, v_pages)
    if norm:
        nearly(k_got, planes[0], n)
    else:
        same(k_got, planes[0].held())
    same(v_got, planes[1].held())


def test_heads_narrower_than_the_pages_leave_zeros():
    heads, dim, vdim, size = 2, 24, 9, 32
    slots, planes = prepared([4], [6], 16, heads, size, 3)
    k_pages, v_pages = pages_of(planes)
    rows = torch.randn((6, heads * (2 * dim + vdim)), device=DEVICE)
    q = kernels().scaled_append(rows, 0, heads * dim, 2 * heads * dim, k_pages, v_pages, torch.tensor(slots, dtype=torch.int32, device=DEVICE),
                                torch.arange(6, dtype=torch.int32, device=DEVICE), heads, heads, dim, vdim)
    assert torch.equal(q.view(6, heads, size)[..., :dim], rows[:, : heads * dim].view(6, heads, dim)) and not bool(q.view(6, heads, size)[..., dim:].any())
    k, v = kernels().scaled_rows(k_pages, v_pages, torch.tensor(slots, dtype=torch.int32, device=DEVICE))
    assert not bool(k[..., dim:].any()) and not bool(v[..., vdim:].any()) and bool(k[..., :dim].any())


@pytest.mark.parametrize("special", ["nan", "inf", "huge", "tiny", "zero", "denormal"])
def test_numbers_at_the_ends(special):
    heads, size, page = 2, 32, 16
    slots, planes = prepared([0, 6], [20, 4], page, heads, size, 11)
    rows = torch.randn((24, 2 * heads * size), generator=torch.Generator().manual_seed(1))
    value = {"nan": float("nan"), "inf": float("-inf"), "huge": 3.0e38, "tiny": 1e-36, "zero": 0.0, "denormal": 1e-42}[special]
    if special in ("tiny", "zero", "denormal"):
        rows[:] = value
    rows[3, 5] = rows[17, 40] = rows[22, 70] = value
    k_pages, v_pages = pages_of(planes)
    kernels().scaled_append(rows.to(DEVICE), None, 0, heads * size, k_pages, v_pages, torch.tensor(slots, dtype=torch.int32, device=DEVICE),
                            torch.zeros(24, dtype=torch.int32, device=DEVICE), heads, heads, size, size)
    flushed = torch.where(rows.abs() < 2.0**-126, 0.0, rows) if special == "denormal" else rows   # (either way below half the smallest code)
    planes[0].append(flushed[:, : heads * size].view(24, heads, size), slots)
    planes[1].append(flushed[:, heads * size :].reshape(24, heads, size), slots)
    for got, plane in zip(held_by(k_pages, v_pages), planes):
        same(got, plane.held())


def test_slots_that_name_no_place_and_tokens_behind_stay():
    heads, size, page = 2, 64, 32
    slots, planes = prepared([9], [3], page, heads, size, 2)
    pages = planes[0].codes.shape[0]
    k_pages, v_pages = pages_of(planes)
    before = [t.clone() for t in held_by(k_pages, v_pages)]
    given = [-1, pages * page] + slots + [2**31 - 1, -5]   # (rows of one block are neighbours)
    rows = torch.randn((len(given), 2 * heads * size), generator=torch.Generator().manual_seed(3)) * 1e-3   # (scales stay as they are)
    kernels().scaled_append(rows.to(DEVICE), None, 0, heads * size, k_pages, v_pages, torch.tensor(given, dtype=torch.int32, device=DEVICE),
                            torch.zeros(len(given), dtype=torch.int32, device=DEVICE), heads, heads, size, size)
    for plane, at in ((planes[0], 0), (planes[1], heads * size)):
        plane.append(rows[:, at : at + heads * size].reshape(-1, heads, size), given)
    after = held_by(k_pages, v_pages)
    written = torch.zeros((pages * page,), dtype=torch.bool)
    written[slots] = True
    for plane, old, new in zip(planes, before, after):
        same(new, plane.held())
        untouched = ~written.view(pages, 1, page, 1).expand_as(new)
        assert torch.equal(new[untouched], old[untouched])
    k, v = kernels().scaled_rows(k_pages, v_pages, torch.tensor([-1, pages * page, slots[0]], dtype=torch.int32, device=DEVICE))
    assert not bool(k[:2].any()) and not bool(v[:2].any()) and bool(k[2].any())


def test_a_layer_that_reads_another_layers_pages_only_turns_its_queries():
    K = kernels()
    k_pages, v_pages = K.scaled_pages(2, 1, 16, 32, DEVICE)
    rows = torch.randn((5, 64), device=DEVICE)
    q = K.scaled_append(rows, 0, None, None, k_pages, v_pages, None, torch.arange(5, dtype=torch.int32, device=DEVICE), 2, 1, 32, 32,
                        frequencies=torch.ones(16, dtype=torch.float64, device=DEVICE), rot_dims=32)
    want = turned(rows.double().cpu().view(5, 2, 32), torch.arange(5), torch.ones(16), 32, "half")
    assert bool(((q.double().cpu().view(5, 2, 32) - want).abs() <= 2.0**-21 * 8).all())
    assert not bool(k_pages.codes.view(torch.uint8).any())


def test_no_rows():
    K = kernels()
    k_pages, v_pages = K.scaled_pages(1, 1, 16, 16, DEVICE)
    none = torch.empty(0, dtype=torch.int32, device=DEVICE)
    assert K.scaled_append(torch.empty((0, 48), device=DEVICE), 0, 16, 32, k_pages, v_pages, none, none, 1, 1, 16, 16).shape == (0, 16)
    assert K.scaled_rows(k_pages, v_pages, none)[0].shape == (0, 1, 16)


def test_token_by_token_and_at_once_hold_the_same_where_the_scale_does_not_grow():
    """A block's first token with the block's largest magnitude: its scale is final from the start, so the order of appending makes no difference."""
    K = kernels()
    heads, size, n = 2, 64, 16
    rows = torch.randn((n, 2 * heads * size), device=DEVICE)
    rows[0] = 8.0
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEVICE)
    once, by_one = K.scaled_pages(1, heads, 16, size, DEVICE), K.scaled_pages(1, heads, 16, size, DEVICE)
    K.scaled_append(rows, None, 0, heads * size, *once, ints(range(n)), ints([0] * n), heads, heads, size, size)
    for r in range(n):
        K.scaled_append(rows[r : r + 1], None, 0, heads * size, *by_one, ints([r]), ints([0]), heads, heads, size, size)
    for a, b in zip(once, by_one):
        assert torch.equal(a.codes.view(torch.uint8), b.codes.view(torch.uint8)) and torch.equal(a.scales, b.scales)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 40])
def test_many_queries_alone(dtype, dim):
    """Rows of queries alone are taken sixteen at a time, the last of them fewer."""
    K, heads, n = kernels(), 3, 16 * 16 + 5
    g = torch.Generator().manual_seed(4)
    rows = torch.randn((n, heads * dim), generator=g).to(TYPES[dtype])
    positions = torch.randint(0, 5000, (n,), generator=g, dtype=torch.int32)
    f = 10000.0 ** (-torch.arange(8, dtype=torch.float64) / 8)
    k_pages, v_pages = K.scaled_pages(1, 1, 16, 64, DEVICE)
    q = K.scaled_append(rows.to(DEVICE), 0, None, None, k_pages, v_pages, None, positions.to(DEVICE), heads, 1, dim, dim, frequencies=f.to(DEVICE), rot_dims=16)
    want = turned(rows.double().view(n, heads, dim), positions, f, 16, "half")
    got = q.cpu().double().view(n, heads, 64)
    # two products and a sum in 32-bit (cosine and sine rounded to it), and the rounding to the type
    assert bool(((got[..., :dim] - want).abs() <= torch.finfo(TYPES[dtype]).eps / 2 * want.abs() + 2.0**-22 * rows.double().abs().amax() * 2).all())
    assert not bool(got[..., dim:].any())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [256, 250])
def test_the_widest_heads_turned_whole(dtype, dim):
    """Tables of the cosines of 128 pairs, of keys and of values: more memory of a block than any other call takes."""
    K, n = kernels(), 40
    slots, planes = prepared([5], [n], 32, 2, 256, 8)
    g = torch.Generator().manual_seed(9)
    rows = torch.randn((n, 5 * dim), generator=g).to(TYPES[dtype])
    positions = torch.randint(0, 5000, (n,), generator=g, dtype=torch.int32)
    f = 10000.0 ** (-torch.arange(dim // 2, dtype=torch.float64) / (dim // 2))
    k_pages, v_pages = pages_of(planes)
    q = K.scaled_append(rows.to(DEVICE), 0, dim, 3 * dim, k_pages, v_pages, torch.tensor(slots, dtype=torch.int32, device=DEVICE), positions.to(DEVICE), 1, 2, dim, dim,
                        frequencies=f.to(DEVICE), rot_dims=dim, v_frequencies=f.to(DEVICE), v_rot_dims=dim, v_pairing="neighbours")
    wide = rows.double()
    want = turned(wide[:, :dim].view(n, 1, dim), positions, f, dim, "half")
    got = q.cpu().double().view(n, 1, 256)[..., :dim]
    assert bool(((got - want).abs() <= torch.finfo(TYPES[dtype]).eps / 2 * want.abs() + 2.0**-22 * rows.double().abs().amax() * 2).all())
    planes[0].append(turned(wide[:, dim : 3 * dim].reshape(n, 2, dim), positions, f, dim, "half"), slots)
    planes[1].append(turned(wide[:, 3 * dim :].reshape(n, 2, dim), positions, f, dim, "neighbours"), slots)
    for got, plane in zip(held_by(k_pages, v_pages), planes):
        same(got, plane.held())


@pytest.mark.parametrize("queries", [True, False])
@pytest.mark.parametrize("told", [0, 5, 17, 20, 31, 400, 10**6], ids=str)
def test_being_told_of_single_rows_changes_no_result(told, queries):
    """Single rows, a portion that begins inside a block, rows that go nowhere, another portion: cut anywhere."""
    heads, size, page = 2, 64, 32
    starts, counts = [7, 16, 0, 31] * 5 + [5, 40], [1, 1, 1, 1] * 5 + [150, 100]
    slots, planes = prepared(starts, counts, page, heads, size, 21)
    slots = slots[:20] + [-1] * 37 + slots[20:170] + [2**31 - 1] * 3 + slots[170:]
    n = len(slots)
    g = torch.Generator().manual_seed(told % 1000)
    rows = torch.randn((n, 4 * heads * size), generator=g) * torch.exp(torch.randn((n, 1), generator=g))
    positions = torch.arange(n, dtype=torch.int32)
    f = 10000.0 ** (-torch.arange(16, dtype=torch.float64) / 16)
    k_pages, v_pages = pages_of(planes)
    width = heads * size
    q = kernels().scaled_append(rows.to(DEVICE), 0 if queries else None, 2 * width, 3 * width, k_pages, v_pages, torch.tensor(slots, dtype=torch.int32, device=DEVICE),
                                positions.to(DEVICE), 2 * heads, heads, size, size, frequencies=f.to(DEVICE), rot_dims=32, short_rows=told)
    wide = rows.double()
    if queries:
        want = turned(wide[:, : 2 * width].reshape(n, 2 * heads, size), positions, f, 32, "half")
        assert bool(((q.cpu().double().view(n, 2 * heads, size) - want).abs() <= 2.0**-24 * want.abs() + 2.0**-21 * rows.abs().amax()).all())
    planes[0].append(turned(wide[:, 2 * width : 3 * width].reshape(n, heads, size), positions, f, 32, "half"), slots)
    planes[1].append(wide[:, 3 * width :].reshape(n, heads, size), slots)
    for got, plane in zip(held_by(k_pages, v_pages), planes):
        same(got, plane.held())


@pytest.mark.parametrize("n", [3, 40, 5000])
def test_rows_that_name_no_place_read_as_zeros(n):
    K = kernels()
    k_pages, v_pages = pages_of(prepared([0], [64], 32, 4, 64, 2)[1])
    total = k_pages.shape[0] * 32
    slots = torch.arange(n, dtype=torch.int32) % total
    nowhere = (torch.arange(n) // 3) % 2 == 1
    slots[nowhere] = torch.where(torch.arange(n)[nowhere] % 2 == 0, -1, total).int()
    k, v = K.scaled_rows(k_pages, v_pages, slots.to(DEVICE))
    everything = K.scaled_rows(k_pages, v_pages, torch.arange(total, dtype=torch.int32, device=DEVICE))
    for got, whole in zip((k, v), everything):
        assert not bool(got[nowhere].any())
        assert torch.equal(got[~nowhere], whole[slots[~nowhere].long()])
