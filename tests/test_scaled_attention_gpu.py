"""Attention over a cache of 8 bits against the plain implementation in 64 bits, over what the pages hold."""

import pytest
import torch

from plain_scaled import PlainPlane, attended, laid

pytestmark = pytest.mark.gpu
DEVICE = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def kernels():
    from mini_llm_amd.ops import kernels as K

    return K


class Batch:
    """Requests with ``contexts`` stored tokens and ``news`` tokens of the step, pages anywhere, all keys and values given."""

    def __init__(self, dtype, heads, kv_heads, size, page, contexts, news, seed=0, spare_columns=0):
        g = torch.Generator().manual_seed(seed)
        self.heads, self.kv_heads, self.size, self.page, self.dtype = heads, kv_heads, size, page, TYPES[dtype]
        counts = [-(-(c + n) // page) for c, n in zip(contexts, news)]
        pages = sum(counts) + 1
        order = torch.randperm(pages, generator=g).tolist()
        self.unused = order.pop()
        self.tables = torch.full((len(news), max(counts) + spare_columns), self.unused, dtype=torch.int32)
        for b, n in enumerate(counts):
            self.tables[b, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
        self.planes = []
        for plane_size in (1.0, 0.5):
            plane = PlainPlane(pages, kv_heads, page, size)
            held = torch.randn((pages * page, kv_heads, size), generator=g).double() * plane_size * torch.exp(torch.randn((1, kv_heads, size), generator=g).double() * 0.5)
            plane.append(held, range(pages * page))
            self.planes.append(plane)
        n = sum(news)
        self.contexts, self.news = contexts, news
        self.positions = torch.tensor([c + i for c, m in zip(contexts, news) for i in range(m)], dtype=torch.int32)
        self.requests = torch.tensor([b for b, m in enumerate(news) for _ in range(m)], dtype=torch.int32)
        self.starts = torch.tensor([sum(news[:i]) for i in range(len(news) + 1)], dtype=torch.int32)
        self.q = torch.randn((n, heads * size), generator=g).to(self.dtype)

    def pages(self):
        K = kernels()
        return K.ScaledPages(*laid(self.planes[0], True, DEVICE)), K.ScaledPages(*laid(self.planes[1], False, DEVICE))

    def run(self, pages=None, q=None, **options):
        K = kernels()
        k_pages, v_pages = pages or self.pages()
        on = lambda t: t.to(DEVICE)
        shape = dict(max_q_len=max(self.news), max_len=max(c + n for c, n in zip(self.contexts, self.news)), q_starts=on(self.starts),
                     context_lens=torch.tensor(self.contexts, dtype=torch.int32, device=DEVICE))
        shape.update(options)
        return K.paged_attention(on(self.q) if q is None else q, k_pages, v_pages, on(self.requests), on(self.positions), on(self.tables), self.heads, self.kv_heads, self.size,
                                 shape.pop("scale", self.size**-0.5), **shape)

    def want(self, scale=None, window=0, keep_first=0, chunk=0, softcap=0.0, sinks=None):
        return attended(self.q.double().view(-1, self.heads, self.size), self.planes[0].held(), self.planes[1].held(), self.requests, self.positions, self.tables,
                        self.size**-0.5 if scale is None else scale, window=window, keep=keep_first, chunk=chunk, softcap=softcap, sinks=sinks).reshape(len(self.q), -1)


def close(got, want, batch, scale=None):
    """What the arithmetic allows, per element. Results are weighted means of values of at most ``largest``.

    bfloat16: every weight is rounded (half a step, 2^-8 of it) and the result once more (2^-8 of it); the scores are 32-bit sums of exact
    products, off by far less.
    float32: a score's sum of exact products has at most 16 roundings in a row for every 64 elements, each at most 2^-24 of sum |q_i k_i| <= |q| |k|
    (times the scale); a weight and the sum of weights are each off by as much, relatively, as their scores are in size: twice that. The
    exponential, the sums over the keys (in lanes, pieces and waves) and the division: 32 roundings."""
    got = got.double().cpu()
    largest = float(torch.nan_to_num(batch.planes[1].held()).abs().max())
    if batch.dtype == torch.bfloat16:
        bound = 2.0**-8 * largest + 2.0**-8 * want.abs()
    else:
        norms = torch.nan_to_num(batch.q.double(), posinf=0.0, neginf=0.0).view(-1, batch.size).norm(dim=1).max() * torch.nan_to_num(batch.planes[0].held()).norm(dim=-1).max()
        score = float(norms) * abs(batch.size**-0.5 if scale is None else scale)
        bound = 2.0**-24 * (32 + 2 * 16 * max(1.0, batch.size / 64) * score) * largest
    off = (got - want).abs()
    assert bool(torch.isfinite(got).all())
    assert bool((off <= bound).all()), f"{float((off / bound).max()):.3g} times what is allowed"


def check(batch, got, **options):
    close(got, batch.want(**options), batch)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads,kv_heads,size,page", [(3, 3, 64, 64), (4, 2, 16, 16), (8, 1, 32, 32), (40, 2, 48, 64), (6, 3, 80, 32), (4, 4, 128, 128), (16, 1, 128, 64), (5, 5, 256, 16), (2, 1, 208, 64)])
def test_rows_that_decode(dtype, heads, kv_heads, size, page):
    batch = Batch(dtype, heads, kv_heads, size, page, [0, 1, 15, 16, 63, 64, 65, 200, 700], [1] * 9, seed=size)
    check(batch, batch.run())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads,kv_heads,size,page", [(2, 2, 64, 64), (4, 2, 16, 16), (4, 1, 48, 32), (2, 1, 128, 128), (3, 1, 80, 16), (2, 2, 256, 64)])
@pytest.mark.parametrize("contexts,news", [([0], [9]), ([0, 5, 64], [64, 65, 63]), ([130, 0], [17, 200])], ids=["nine", "edges", "ragged"])
def test_portions(dtype, heads, kv_heads, size, page, contexts, news):
    batch = Batch(dtype, heads, kv_heads, size, page, contexts, news, seed=size + len(news))
    check(batch, batch.run())


MASKS = [dict(window=1), dict(window=20), dict(window=100, keep_first=3), dict(window=16, keep_first=70), dict(chunk=1), dict(chunk=50), dict(softcap=2.0), dict(sinks=True),
         dict(window=33, keep_first=17, softcap=5.0, sinks=True)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("size", [64, 128])
@pytest.mark.parametrize("options", MASKS, ids=str)
def test_masks_caps_and_sinks(dtype, size, options):
    batch = Batch(dtype, 4, 2, size, 32, [0, 300, 64, 10, 129], [1, 1, 70, 140, 20], seed=7)
    options = dict(options)
    if options.get("sinks"):
        options["sinks"] = torch.tensor([0.5, -3.0, 4.0, 0.0])
    given = {k: v.to(DEVICE) if isinstance(v, torch.Tensor) else v for k, v in options.items()}
    check(batch, batch.run(short_rows=2, short_requests=2, **given), **options)   # rows alone beside portions
    check(batch, batch.run(max_q_len=None, **given), **options)                    # rows without the shape of portions
    check(batch, batch.run(**given), **options)                                    # single rows as portions


@pytest.mark.parametrize("dtype,heads,kv_heads,size,page", [("bf16", 40, 2, 64, 64), ("bf16", 48, 4, 64, 16), ("bf16", 40, 1, 128, 64), ("bf16", 48, 2, 112, 32),
                                                            ("f32", 40, 2, 64, 64), ("f32", 48, 4, 48, 16)])
@pytest.mark.parametrize("options", [{}, dict(window=70, keep_first=5, softcap=4.0)], ids=["whole", "window"])
def test_many_blocks_take_more_rows_each(dtype, heads, kv_heads, size, page, options):
    """Enough blocks (320 of the larger tiles of rows) for the form that launches of fewer do not take; with numbers that are none in masked places
    and in one that some rows of a tile see."""
    batch = Batch(dtype, heads, kv_heads, size, page, [0, 37], [520, 61], seed=size)
    for plane in batch.planes:
        plane.codes[batch.unused] = torch.nan
    batch.planes[1].codes[int(batch.tables[0, 300 // page]), 0, 300 % page, 3] = torch.nan
    got = batch.run(**options).double().cpu()
    want = batch.want(**options)
    lost = torch.isnan(want)
    assert bool(lost.any()) and torch.equal(torch.isnan(got), lost)
    close(torch.where(lost, 0.0, got), torch.where(lost, 0.0, want), batch)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_short_portions_go_row_by_row(dtype):
    batch = Batch(dtype, 4, 2, 64, 64, [0, 100, 63, 5], [8, 3, 2, 1], seed=3)
    check(batch, batch.run())


@pytest.mark.parametrize("cut", [(1, 1, 40), (2, 3, 14), (8, 5, 8), (4, 40, 1), (1, 7, 3)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_every_cut_of_a_rows_keys_gives_the_same(dtype, cut, monkeypatch):
    """Waves, runs and a last run that takes what is left: (1, 7, 3) reaches over 21 of up to 40 tiles."""
    K = kernels()
    batch = Batch(dtype, 6, 3, 64, 64, [2500, 0, 64 * 7 - 1, 64 * 7, 1000, 63], [1] * 6, seed=9)
    monkeypatch.setattr(K, "scaled_cut", lambda *_: cut)
    check(batch, batch.run())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_reach_that_is_named_too_short_leaves_no_key_out(dtype):
    batch = Batch(dtype, 2, 1, 64, 64, [1500, 40], [1, 1], seed=10)
    check(batch, batch.run(max_len=64))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("news", [[1, 1, 1], [30, 9, 12]])
def test_padding_rows(dtype, news):
    """Rows without a request are zeros where rows go by themselves; portions of nobody are left alone."""
    batch = Batch(dtype, 2, 2, 64, 64, [100, 20, 33], news, seed=4)
    want = batch.want()
    first = news[0]
    out = torch.full((sum(news), 2 * 64), 7.0, dtype=batch.dtype, device=DEVICE)
    batch.requests[:first] = -1
    if max(news) == 1:
        got = batch.run(out=out)
        assert not bool(got[:first].any())
    else:
        got = batch.run(out=out, context_lens=torch.tensor([-1, 20, 33], dtype=torch.int32, device=DEVICE))
        assert bool((got[:first] == 7.0).all())
    close(got[first:], want[first:], batch)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_position_before_the_first_sees_nothing(dtype):
    batch = Batch(dtype, 2, 2, 64, 64, [10, 5], [1, 1], seed=4)
    batch.positions[1] = -1
    got = batch.run(sinks=torch.zeros(2, device=DEVICE))
    assert not bool(got[1].any()) and bool(got[0].any())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("news,mask", [([1, 1], {}), ([40, 70], {}), ([1, 1], dict(window=30, keep_first=2)), ([40, 70], dict(window=30)), ([40, 70], dict(chunk=32))])
def test_no_number_in_a_masked_place(dtype, news, mask):
    """Codes that are no number, where a row does not look: behind the last token, in pages that other requests hold, before a window, behind a
    row of the same portion. Rows that do not see them are as ever; rows that do are no numbers."""
    batch = Batch(dtype, 2, 1, 64, 64, [90, 57], news, seed=5)
    want = batch.want(**mask)
    bad_position = {0: 90 + news[0], 1: 20}   # request 0: right behind its last row; request 1: a key that windows and chunks leave out
    for b, p in bad_position.items():
        for plane in batch.planes:
            plane.codes[int(batch.tables[b, p // 64]) if p < 64 * batch.tables.shape[1] else batch.unused, :, p % 64] = torch.nan
    for plane in batch.planes:
        plane.codes[batch.unused] = torch.nan
    got = batch.run(**mask).double().cpu()
    sees = attended(batch.q.double().view(-1, 2, 64), batch.planes[0].held(), batch.planes[1].held(), batch.requests, batch.positions, batch.tables, 0.125,
                    window=mask.get("window", 0), keep=mask.get("keep_first", 0), chunk=mask.get("chunk", 0)).reshape(len(batch.q), -1)
    lost = torch.isnan(sees)
    assert torch.equal(torch.isnan(got), lost)
    close(torch.where(lost, 0.0, got), torch.where(lost, 0.0, want), batch)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_value_that_is_no_number_reaches_the_rows_that_see_it_alone(dtype):
    batch = Batch(dtype, 2, 2, 64, 64, [0, 30], [100, 1], seed=6)
    want = batch.want()
    batch.planes[1].codes[int(batch.tables[0, 0]), 1, 50, 7] = torch.nan   # key 50 of request 0, head 1, element 7
    got = batch.run().double().cpu().view(-1, 2, 64)
    lost = torch.zeros_like(got, dtype=torch.bool)
    lost[50:100, 1, 7] = True
    assert torch.equal(torch.isnan(got), lost)
    close(torch.where(lost, 0.0, got), torch.where(lost, 0.0, want.view_as(got)), batch)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_query_that_is_no_number_spoils_its_own_row_and_head_alone(dtype, value):
    batch = Batch(dtype, 4, 2, 64, 64, [40, 10], [1, 20], seed=8)
    want = batch.want()
    batch.q[0, 5] = value
    batch.q[9, 64 + 5] = value
    for options in ({}, {"max_q_len": None}):
        got = batch.run(**options).double().cpu().view(-1, 4, 64)
        lost = torch.zeros_like(got, dtype=torch.bool)
        lost[0, 0] = lost[9, 1] = True
        assert bool(torch.isnan(got[lost]).all())
        close(torch.where(lost, 0.0, got), torch.where(lost, 0.0, want.view_as(got)), batch)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("scale", [0.0, -0.125, 3.0])
def test_scales_of_the_scores(dtype, scale):
    batch = Batch(dtype, 2, 1, 64, 64, [70, 0], [1, 90], seed=12)
    batch.q *= 0.25
    got = batch.run(scale=scale)
    close(got, batch.want(scale=scale), batch, scale)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("news", [[1, 1], [30, 9]])
def test_strides_and_orders(dtype, news):
    """Queries that are columns of a wider product (their rows on no 16 bytes), results in columns of a wider tensor, wide results."""
    batch = Batch(dtype, 2, 2, 64, 64, [33, 100], news, seed=13, spare_columns=3)
    n = sum(news)
    for shift in (0, 1):
        wide = torch.zeros((n, 3 * 128 + 3), dtype=batch.dtype, device=DEVICE)
        wide[:, shift : shift + 128] = batch.q.to(DEVICE)
        into = torch.full((n, 200), 5.0, dtype=batch.dtype, device=DEVICE)
        got = batch.run(q=wide[:, shift : shift + 128], out=into[:, 7:135])
        assert got.data_ptr() == into[:, 7:135].data_ptr() and bool((into[:, :7] == 5.0).all()) and bool((into[:, 135:] == 5.0).all())
        check(batch, got)
    whole = batch.run(wide_out=True)
    assert whole.dtype == torch.float32
    check(batch, whole)


def test_rows_in_the_packed_layout():
    K = kernels()
    batch = Batch("bf16", 4, 2, 64, 64, [30, 5, 70], [1, 1, 1], seed=14)
    packed = batch.run(packed_out=True)
    assert isinstance(packed, K.PackedRows)
    plain = batch.run()
    weight = K.pack_matrix(torch.eye(256, dtype=torch.bfloat16, device=DEVICE))
    assert torch.equal(K.linear(packed, weight, out_dtype=torch.float32), plain.float())


def test_tables_that_name_no_page_lead_nowhere():
    """Entries outside the pages, where a row looks: the results mean nothing, and nothing outside the pages is read."""
    batch = Batch("bf16", 2, 1, 64, 64, [200, 10], [1, 40], seed=15)
    batch.tables[0, 1], batch.tables[1, 0] = -7, 2**30
    assert batch.run().shape == (41, 128)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_the_same_call_twice_and_on_another_stream(dtype):
    batch = Batch(dtype, 12, 12, 64, 64, [900, 20, 500], [1, 1, 1], seed=16)
    pages = batch.pages()
    one = batch.run(pages)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        two = batch.run(pages)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(one, two)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_layer_step_captured_and_replayed(dtype):
    """Append and attention as a decode step has them, in a graph: every replay with new rows gives what the eager calls give."""
    K = kernels()
    heads, size, steps = 4, 64, 40
    f = 10000.0 ** (-torch.arange(32, dtype=torch.float64, device=DEVICE) / 32)
    rows = [torch.randn((2, 3 * heads * size), device=DEVICE).to(TYPES[dtype]) for _ in range(steps)]
    tables = torch.tensor([[3, 0], [1, 2]], dtype=torch.int32, device=DEVICE)
    requests = torch.arange(2, dtype=torch.int32, device=DEVICE)

    def layer(pages, x, slots, positions):
        q = K.scaled_append(x, 0, heads * size, 2 * heads * size, *pages, slots, positions, heads, heads, size, size, frequencies=f, rot_dims=size)
        return K.paged_attention(q, *pages, requests, positions, tables, heads, heads, size, size**-0.5, max_q_len=1, max_len=64)

    def at(step):
        p = torch.tensor([step, step], dtype=torch.int32, device=DEVICE)
        return tables[:, 0] * 32 + p if step < 32 else tables[:, 1] * 32 + p - 32, p

    eager, captured = K.scaled_pages(4, heads, 32, size, DEVICE), K.scaled_pages(4, heads, 32, size, DEVICE)
    x, slots, positions = rows[0].clone(), *(t.clone() for t in at(0))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(captured, x, slots, positions)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(captured, x, slots, positions)
    for step in range(steps):
        want = layer(eager, rows[step], *at(step))
        x.copy_(rows[step])
        for to, value in zip((slots, positions), at(step)):
            to.copy_(value)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), step
    for a, b in zip(eager, captured):
        assert torch.equal(a.codes.view(torch.uint8), b.codes.view(torch.uint8)) and torch.equal(a.scales, b.scales)


@pytest.mark.parametrize("news", [[1, 1], [40, 70]], ids=["rows", "portions"])
def test_pages_beyond_offsets_of_32_bits(news):
    """The same requests in the first pages and in the last of a cache whose planes are larger than 2^32 bytes."""
    K, page, heads, kv_heads, size, num_pages = kernels(), 64, 16, 8, 128, 68000
    k_pages, v_pages = K.scaled_pages(num_pages, kv_heads, page, size, DEVICE)
    assert k_pages.codes.numel() > 2**32
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEVICE)
    contexts, total = [200, 30], sum(news)
    g = torch.Generator().manual_seed(12)
    stored = [torch.randn((c + n, 2 * kv_heads * size), generator=g).to(DEVICE) for c, n in zip(contexts, news)]
    q = torch.randn((total, heads * size), generator=g).bfloat16().to(DEVICE)
    positions = ints([c + i for c, n in zip(contexts, news) for i in range(n)])
    owner = ints([r for r, n in enumerate(news) for _ in range(n)])
    results = []
    for first in (0, num_pages - 16):
        tables = torch.arange(first, first + 16, dtype=torch.int32, device=DEVICE).view(2, 8).flip(0).contiguous()
        for rows, table in zip(stored, tables):
            at = torch.arange(rows.shape[0], device=DEVICE)
            K.scaled_append(rows, None, 0, kv_heads * size, k_pages, v_pages, (table[at // page] * page + (at % page).int()).int(), at.int(), heads, kv_heads, size, size)
        results.append(K.paged_attention(q, k_pages, v_pages, owner, positions, tables, heads, kv_heads, size, size**-0.5, max_q_len=max(news), max_len=512,
                                         q_starts=ints([0, news[0], total]), context_lens=ints(contexts)))
        read = K.scaled_rows(k_pages, v_pages, (tables[0, :1] * page).contiguous())[1]
        assert bool(((read.double() - stored[0][0, kv_heads * size :].view(kv_heads, size).double()).abs() <= stored[0].abs().max() * 2.0**-4).all())
    assert bool(results[0].any()) and torch.equal(results[0], results[1])


def test_a_context_at_the_end_of_all_numbers_stays_in_its_table():
    """A length that no table reaches counts as the table's last position: nothing is read behind it (its rows' results are nobody's)."""
    K = kernels()
    k_pages, v_pages = K.scaled_pages(4, 2, 64, 64, DEVICE)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEVICE)
    n = 30
    q = torch.randn((n, 128), device=DEVICE)
    out = K.paged_attention(q, k_pages, v_pages, ints([0] * n), ints(list(range(n))), ints([[0, 1, 2, 3]]), 2, 2, 64, 0.125, max_q_len=n, max_len=256, q_starts=ints([0, n]),
                            context_lens=ints([2**31 - 3]))
    assert out.shape == (n, 128) and not bool(out.any())   # (the pages hold zeros)


@pytest.mark.parametrize("size,page", [(128, 64), (80, 16)])
@pytest.mark.parametrize("options", [{}, dict(window=70, keep_first=5, softcap=4.0), dict(chunk=48)], ids=["whole", "window", "chunk"])
def test_blocks_in_plenty_take_twice_the_rows(size, page, options):
    """Enough blocks (2,048) for the form whose waves share a block's rows between them; the last tile of the first portion has rows for half of
    them only."""
    batch = Batch("bf16", 104, 2, size, page, [0, 37], [520, 61], seed=size)
    for plane in batch.planes:
        plane.codes[batch.unused] = torch.nan
    batch.planes[1].codes[int(batch.tables[0, 300 // page]), 0, 300 % page, 3] = torch.nan
    got = batch.run(**options).double().cpu()
    want = batch.want(**options)
    lost = torch.isnan(want)
    assert bool(lost.any()) and torch.equal(torch.isnan(got), lost)
    close(torch.where(lost, 0.0, got), torch.where(lost, 0.0, want), batch)


@pytest.mark.parametrize("one", [True, False], ids=["one-launch", "two-launches"])
@pytest.mark.parametrize("dtype,heads,kv_heads,size,page", [("bf16", 4, 2, 64, 64), ("bf16", 20, 1, 48, 16), ("bf16", 3, 3, 128, 32), ("bf16", 4, 1, 80, 128), ("f32", 4, 2, 64, 16),
                                                            ("f32", 18, 1, 128, 64)])
@pytest.mark.parametrize("options", [{}, dict(window=70, keep_first=5, softcap=4.0), dict(chunk=48)], ids=["whole", "window", "chunk"])
def test_a_step_of_rows_and_portions(dtype, heads, kv_heads, size, page, options, one, monkeypatch):
    """Rows that are cut into runs and put together (the first is long) beside portions, in one launch and in two."""
    monkeypatch.setattr(kernels(), "scaled_mixes", lambda *a: one)
    batch = Batch(dtype, heads, kv_heads, size, page, [2600, 7, 0, 60, 0], [1, 3, 1, 40, 100], seed=size)
    before = kernels().launch_counts()
    got = batch.run(short_rows=5, short_requests=3, **options)
    ran = kernels().launches_since(before)
    assert ("scaled_attention_mixed" in ran) == one and ("scaled_attention_tiles" in ran) != one
    check(batch, got, **options)


def test_a_step_of_both_kinds_with_numbers_that_are_none():
    batch = Batch("bf16", 4, 2, 64, 64, [130, 7, 60, 0], [1, 1, 40, 100], seed=3)
    for plane in batch.planes:
        plane.codes[batch.unused] = torch.nan
    batch.planes[1].codes[int(batch.tables[2, 1]), 0, 10, 3] = torch.nan   # position 74 of the third request: seen by the later rows of its portion
    got, want = batch.run(short_rows=2, short_requests=2).double().cpu(), batch.want()
    lost = torch.isnan(want)
    assert bool(lost.any()) and torch.equal(torch.isnan(got), lost)
    close(torch.where(lost, 0.0, got), torch.where(lost, 0.0, want), batch)
