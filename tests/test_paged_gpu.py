"""Appending to a paged cache, choosing pages and attending over them, against 64-bit evaluations."""

import math

import pytest
import torch

from paged_reference import Batch, attention, chosen_pages, places, rotated

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def device_stays_sound():
    if not torch.cuda.is_available():
        pytest.fail("the gpu-marked tests need a CUDA device")
    yield
    torch.cuda.synchronize()


def status_is(code):
    """The device's status word, which is cleared."""
    import flash_colsum_b200 as fc
    from flash_colsum_b200 import ops
    got = fc.device_status()
    ops._status_word(torch.device("cuda", torch.cuda.current_device())).zero_()
    assert got == code


def on_gpu(*tensors):
    return [None if t is None else t.cuda() for t in tensors]


# --------------------------------------------------------------------------- append
APPENDS = [
    # new tokens, lens, page, kv heads, heads, dim, type, rotated features, interleaved
    ([1], [1], 64, 1, 1, 8, BF16, 0, False),
    ([1], [130], 64, 8, 32, 128, BF16, 128, False),
    ([1, 1, 1], [1, 65, 64], 64, 2, 6, 80, FP16, 80, False),
    ([5, 0, 33, 1, 70], [5, 17, 40, 16, 131], 16, 3, 3, 64, BF16, 32, True),
    ([5, 0, 33, 1, 70], [50, 17, 40, 128, 131], 32, 4, 8, 96, FP16, 96, True),
    ([200, 3], [200, 131], 128, 2, 2, 128, FP16, 64, False),
    ([129, 64, 1], [257, 64, 1], 64, 1, 7, 72, BF16, 16, False),
    ([17] * 19, [17 + 5 * i for i in range(19)], 16, 2, 4, 120, BF16, 112, False),
    ([1] * 300, [1 + i for i in range(300)], 16, 1, 2, 16, FP16, 16, True),
]


@pytest.mark.parametrize("case", range(len(APPENDS)))
@pytest.mark.parametrize("layout", ["plain", "strided"])
def test_append_writes_rotated_keys_values_and_bounds(case, layout):
    import flash_colsum_b200 as fc
    new, lens, P, H, heads, D, dtype, R, inter = APPENDS[case]
    packed = max(new) > 1 or min(new) < 1
    tail = 3 if packed and case % 2 else 0
    a = Batch(case, new, lens, P, H, heads, D, dtype, tail=tail, packed=packed)
    key, value, query = a.rows(H), a.rows(H), a.rows(heads)
    pools = [a.pool(), a.pool()]
    bounds = torch.stack([pools[0].amin(2), pools[0].amax(2)], 2)
    cos = sin = positions = None
    if R:
        turn = torch.arange(max(lens) + 7, dtype=torch.float64)[:, None] * 10.0 ** -torch.linspace(0, 3, R // 2, dtype=torch.float64)
        cos, sin = turn.cos().float(), turn.sin().float()
        if case % 3 == 1:
            positions = torch.randint(0, max(lens) + 7, (a.T,), generator=a.g, dtype=torch.int32)
    d_key, d_value, d_query, d_bounds, d_cos, d_sin, d_pos, table, d_lens, starts = on_gpu(
        key, value, query, bounds, cos, sin, positions, a.table, a.lens, a.starts)
    if layout == "strided":      # rows of one fused projection, pools with the slots outside the heads in one tensor, a wider table
        fused = torch.cat([d_query, d_key, d_value], 1)
        d_query, d_key, d_value = fused[:, :heads], fused[:, heads:heads + H], fused[:, heads + H:]
        both = torch.stack([p.transpose(1, 2) for p in pools], 1).contiguous().cuda()
        d_pools = [both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)]
        table = torch.cat([table, torch.full_like(table, -1)], 1)[:, :table.shape[1]]
    else:
        d_pools = on_gpu(*pools)
    got = fc.append_paged(d_key, d_value, d_pools[0], d_pools[1], table, d_lens, starts=starts, query=d_query, cos=d_cos, sin=d_sin,
                          positions=d_pos, interleaved=inter, bounds=d_bounds)
    status_is(0)

    half, eps32 = torch.finfo(dtype).eps / 2, 2.0 ** -24
    floor = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2      # half a step among the subnormals
    want_keys, want_values = pools[0].double(), pools[1].double()
    stored = d_pools[0].cpu()
    low, high = bounds[:, :, 0].clone(), bounds[:, :, 1].clone()
    slack = torch.zeros_like(want_keys)

    def held(x, pos):
        """Exact value, and how far its rounded one may be: three roundings to 32 bits, one to 16."""
        c, s = (None, None) if R == 0 else (cos[pos].double(), sin[pos].double())
        exact, size = rotated(x.double(), c, s, inter)
        error = 2 * eps32 * size * (1 if R else 0)
        return exact, error + half * (exact.abs() + error) + floor

    got_query = got.cpu().double()
    for t, b, pos in places(a.lens, a.starts, a.T):
        m = pos if positions is None else int(positions[t])
        exact, room = held(query[t], m)
        assert ((got_query[t] - exact).abs() <= room).all()
        page, slot = int(a.table[b, pos // P]), pos % P
        want_keys[page, :, slot], slack[page, :, slot] = held(key[t], m)
        want_values[page, :, slot] = value[t].double()
        row = stored[page, :, slot]
        low[page] = row if slot == 0 else torch.minimum(low[page], row)
        high[page] = row if slot == 0 else torch.maximum(high[page], row)
    assert ((stored.double() - want_keys).abs() <= slack).all()                 # (what was not written: exactly as it was)
    assert torch.equal(d_pools[1].cpu().double(), want_values)
    assert torch.equal(d_bounds.cpu(), torch.stack([low, high], 2))
    assert (got_query[a.T - tail:] == 0).all()

    # given memory: rows behind the last sequence stay; the query's own memory will do; nothing but the pools
    mine = torch.full_like(got, 7.0)
    again = fc.append_paged(d_key, d_value, d_pools[0], d_pools[1], table, d_lens, starts=starts, query=d_query, cos=d_cos, sin=d_sin,
                            positions=d_pos, interleaved=inter, query_out=mine)
    assert again.data_ptr() == mine.data_ptr() and torch.equal(mine[:a.T - tail], got[:a.T - tail]) and (mine[a.T - tail:] == 7).all()
    inside = d_query.clone()
    fc.append_paged(d_key, d_value, d_pools[0], d_pools[1], table, d_lens, starts=starts, query=inside, cos=d_cos, sin=d_sin,
                    positions=d_pos, interleaved=inter, query_out=inside)
    assert torch.equal(inside[:a.T - tail], got[:a.T - tail]) and torch.equal(inside[a.T - tail:], d_query[a.T - tail:])
    assert fc.append_paged(d_key, d_value, d_pools[0], d_pools[1], table, d_lens, starts=starts, cos=d_cos, sin=d_sin,
                           positions=d_pos, interleaved=inter) is None
    assert torch.equal(d_pools[0].cpu(), stored) and torch.equal(d_pools[1].cpu().double(), want_values)
    status_is(0)


def test_append_bounds_keep_nan_and_take_in_a_page_token_by_token():
    import flash_colsum_b200 as fc
    a = Batch(5, [1], [1], 16, 2, 2, 64, BF16, packed=False, spare_pages=0)
    keys = torch.randn(20, 2, 64, generator=a.g).to(BF16)
    keys[3, 1, 5] = math.nan
    keys[18, 0, 0] = math.inf
    pool, values, table = torch.zeros(2, 2, 16, 64, dtype=BF16).cuda(), torch.zeros(2, 2, 16, 64, dtype=BF16).cuda(), torch.tensor([[1, 0]], dtype=torch.int32).cuda()
    bounds = torch.full((2, 2, 2, 64), 3.0, dtype=BF16).cuda()
    for i in range(20):
        fc.append_paged(keys[i:i + 1].cuda(), keys[i:i + 1].cuda(), pool, values, table, torch.tensor([i + 1], dtype=torch.int32).cuda(),
                        bounds=bounds)
    want = torch.stack([torch.stack([keys[16:].amin(0), keys[16:].amax(0)], 1), torch.stack([keys[:16].amin(0), keys[:16].amax(0)], 1)])
    assert torch.equal(torch.nan_to_num(bounds.cpu(), nan=77.0), torch.nan_to_num(want, nan=77.0))
    status_is(0)


def test_append_leaves_out_what_it_has_no_place_for():
    """Pages that the table does not have, positions past the tables: said in the status word, nothing written."""
    import flash_colsum_b200 as fc
    a = Batch(6, [40, 9], [40, 9], 16, 2, 4, 64, FP16, spare_pages=2)
    key, value, query = a.rows(2).cuda(), a.rows(2).cuda(), a.rows(4).cuda()
    clean = [a.pool().cuda(), a.pool().cuda()]
    for entry in (-1, a.N, 2 ** 31 - 1, -2 ** 31):
        pools = [p.clone() for p in clean]
        table = a.table.clone()
        lost = int(table[0, 1])
        table[0, 1] = entry
        fc.append_paged(key, value, *pools, table.cuda(), a.lens.cuda(), starts=a.starts.cuda())
        status_is(5)
        assert torch.equal(pools[0][lost], clean[0][lost])
        assert torch.equal(pools[1][int(table[0, 2])][:, :8], value[32:40].transpose(0, 1))
        assert torch.equal(pools[1][int(table[1, 0])][:, :9], value[40:49].transpose(0, 1))
    # a table that is too narrow
    pools = [p.clone() for p in clean]
    fc.append_paged(key, value, *pools, a.table[:, :2].contiguous().cuda(), a.lens.cuda(), starts=a.starts.cuda())
    status_is(5)
    assert torch.equal(pools[0][int(a.table[0, 2])], clean[0][int(a.table[0, 2])])
    # lens that count fewer tokens than there are rows: the rows without a place are left out
    pools = [p.clone() for p in clean]
    fc.append_paged(key, value, *pools, a.table.cuda(), torch.tensor([30, 9], dtype=torch.int32).cuda(), starts=a.starts.cuda())
    status_is(5)
    assert torch.equal(pools[1][int(a.table[0, 0])], value[10:26].transpose(0, 1))
    # positions that the rotation does not have
    cos = torch.ones(30, 32).cuda()
    pools = [p.clone() for p in clean]
    out = fc.append_paged(key, value, *pools, a.table.cuda(), a.lens.cuda(), starts=a.starts.cuda(), query=query, cos=cos,
                          sin=torch.zeros_like(cos))
    status_is(6)
    assert (out[30:40] == 0).all() and torch.equal(out[:30], query[:30]) and torch.equal(out[40:], query[40:])
    assert torch.equal(pools[1][int(a.table[0, 1])][:, :14], value[16:30].transpose(0, 1))
    assert torch.equal(pools[1][int(a.table[0, 1])][:, 14:], clean[1][int(a.table[0, 1])][:, 14:])
    assert torch.equal(pools[0][int(a.table[0, 2])], clean[0][int(a.table[0, 2])])


# --------------------------------------------------------------------------- select
SELECTS = [
    # new tokens, lens, page, kv heads, heads, dim, type, k, first, last
    ([1], [1], 64, 1, 1, 8, BF16, 1, 0, 1),
    ([1], [64 * 40], 64, 8, 32, 128, BF16, 9, 1, 2),
    ([1, 1, 1], [700, 16, 333], 16, 2, 6, 80, FP16, 7, 1, 1),
    ([5, 0, 33, 1], [500, 17, 900, 1], 16, 3, 3, 64, BF16, 6, 0, 1),
    ([5, 0, 33, 1], [5, 17, 200, 160], 32, 4, 8, 24, FP16, 4, 2, 2),
    ([130], [3000], 128, 2, 2, 96, BF16, 12, 1, 3),
    ([70], [16 * 300], 16, 1, 8, 128, FP16, 40, 3, 4),
    ([1] * 270, [1 + 3 * i for i in range(270)], 16, 1, 2, 16, FP16, 5, 1, 1),
    ([2], [16 * 2100], 16, 1, 4, 32, BF16, 1500, 1, 1),
    ([1], [16 * 2100 - 5], 16, 2, 4, 128, FP16, 33, 1, 2),
    # many tokens a sequence: pages up to 512, up to 1024, more
    ([70, 3, 0, 129], [16 * 300, 90, 7, 16 * 140 + 3], 16, 2, 6, 104, BF16, 21, 1, 1),
    ([40], [16 * 1000], 16, 1, 2, 64, BF16, 64, 1, 1),
    ([40], [16 * 900 + 7], 16, 1, 2, 128, FP16, 300, 0, 2),
    ([24], [16 * 1500], 16, 1, 8, 96, BF16, 50, 1, 1),
    ([24, 8], [16 * 1300, 16 * 1400], 16, 1, 1, 8, FP16, 700, 1, 1),
]


def select(a, query, bounds, k, first, last, **more):
    import flash_colsum_b200 as fc
    query, bounds, table, lens, starts = on_gpu(query, bounds, a.table, a.lens, a.starts)
    return fc.select_pages(query, bounds, table, lens, k, page_size=a.P, starts=starts, first=first, last=last, **more)


@pytest.mark.parametrize("case", range(len(SELECTS)))
@pytest.mark.parametrize("ties", [False, True])
def test_select_takes_the_best_pages(case, ties):
    new, lens, P, H, heads, D, dtype, k, first, last = SELECTS[case]
    packed = max(new) > 1 or min(new) < 1
    tail = 2 if packed and case % 2 else 0
    a = Batch(case, new, lens, P, H, heads, D, dtype, tail=tail, packed=packed)
    query = a.rows(heads)
    centre = torch.randn(a.N, H, D, generator=a.g)
    if ties:       # pages alike, and values whose products are exact, so that sums are
        query, centre = query.sign(), centre.sign() * (torch.arange(a.N) % 3)[:, None, None]
        centre[:, :, 1:] *= 0.0
    bounds = torch.stack([centre - 1.0, centre + 1.0], 2).to(dtype)
    want = chosen_pages(query, bounds, P, a.table, a.lens, a.starts, k, first, last)
    assert torch.equal(select(a, query, bounds, k, first, last).cpu(), want)
    mine = torch.full(want.shape, 9, dtype=torch.int32).cuda()
    assert select(a, query, bounds, k, first, last, out=mine).data_ptr() == mine.data_ptr()
    assert torch.equal(mine[:a.T - tail].cpu(), want[:a.T - tail]) and (mine[a.T - tail:] == 9).all()
    status_is(0)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("tokens,pages", [(4, 90), (20, 90), (9, 700), (9, 1100)])
def test_select_orders_scores_that_differ_in_the_last_bits(dtype, tokens, pages):
    """Scores whose large terms cancel, so that sums in 32 bits could not tell the pages apart."""
    a = Batch(3, [tokens], [16 * pages], 16, 2, 4, 64, dtype)
    query = a.rows(4).abs() + 1
    bounds = torch.zeros(a.N, 2, 2, 64, dtype=dtype)
    bounds[:, :, 1] = torch.randn(a.N, 2, 64, generator=a.g).to(dtype)
    big = 3.0e4
    query[:, :, 0] = query[:, :, 1] = 1.0
    bounds[:, :, 1, 0], bounds[:, :, 1, 1] = big, -big
    bounds[:, :, 1, 2:] *= 2.0 ** -12 if dtype == BF16 else 2.0 ** -9
    want = chosen_pages(query, bounds, 16, a.table, a.lens, a.starts, 11, 1, 1)
    assert torch.equal(select(a, query, bounds, 11, 1, 1).cpu(), want)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("tokens", [3, 16])
def test_select_with_the_largest_values_of_the_type(dtype, tokens):
    """Sums that overflow 32 bits (bf16) or parts that overflow 16 (fp16) are sums in 64 bits like any other."""
    a = Batch(14, [tokens], [16 * 70], 16, 1, 8, 32, dtype)
    most = torch.finfo(dtype).max
    query = (torch.rand(a.T, 8, 32, generator=a.g) * most).to(dtype)
    centre = torch.rand(a.N, 1, 32, generator=a.g) * 0.5
    bounds = (torch.stack([centre, centre + 0.4], 2) * most).to(dtype)
    want = chosen_pages(query, bounds, 16, a.table, a.lens, a.starts, 9, 1, 1)
    assert torch.equal(select(a, query, bounds, 9, 1, 1).cpu(), want)
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    small_query, small_bounds = (query.double() / most * 64 * tiny).to(dtype), (bounds.double() / most * 64 * tiny).to(dtype)
    want = chosen_pages(small_query, small_bounds, 16, a.table, a.lens, a.starts, 9, 1, 1)
    assert torch.equal(select(a, small_query, small_bounds, 9, 1, 1).cpu(), want)


def test_select_in_several_launches_under_a_wide_table():
    """A table far wider than the sequences are long: the scores of all tokens at once would take a gigabyte."""
    a = Batch(15, [70, 0, 30], [16 * 40, 5, 16 * 30], 16, 16, 16, 64, BF16, tail=5, width=60000)
    query = a.rows(16)
    bounds = torch.stack([a.normal(a.N, 16, 64) - 1, a.normal(a.N, 16, 64) + 1], 2)
    want = chosen_pages(query, bounds, 16, a.table, a.lens, a.starts, 6, 1, 1)
    assert torch.equal(select(a, query, bounds, 6, 1, 1).cpu(), want)
    status_is(0)


def test_one_token_a_sequence_under_a_table_that_shared_memory_does_not_hold():
    a = Batch(16, [1] * 3, [16 * 70, 16 * 9, 5], 16, 2, 4, 64, FP16, packed=False, width=40000)
    query = a.rows(4)
    bounds = torch.stack([a.normal(a.N, 2, 64) - 1, a.normal(a.N, 2, 64) + 1], 2)
    want = chosen_pages(query, bounds, 16, a.table, a.lens, None, 5, 1, 1)
    assert torch.equal(select(a, query, bounds, 5, 1, 1).cpu(), want)
    status_is(0)


def test_many_short_sequences_and_a_long_rest():
    """Sequences of none, one and some tokens in their thousands, and more rows behind them: every row finds its own."""
    import flash_colsum_b200 as fc
    g = torch.Generator().manual_seed(17)
    new = [(7 * i) % 4 if i % 5 else 0 for i in range(2500)]
    lens = [n + (i * 13) % 40 for i, n in enumerate(new)]
    a = Batch(17, new, lens, 16, 1, 2, 16, BF16, tail=900)
    owner = torch.full((a.T,), -1)
    for t, b, pos in places(a.lens, a.starts, a.T):
        owner[t] = b * 64 + pos
    # values that say whose they are: value = (sequence, position), each exact in bf16 by its parts
    value = torch.zeros(a.T, 1, 16, dtype=BF16)
    part = torch.stack([(owner >> s) & 63 for s in (0, 6, 12)], 1).clamp(min=0)
    value[:, 0, :3] = part.to(BF16)
    key, query = a.rows(1) * 0, a.rows(2)
    kp, vp = torch.zeros(a.N, 1, 16, 16, dtype=BF16).cuda(), torch.full((a.N, 1, 16, 16), 99.0, dtype=BF16).cuda()
    bounds = torch.zeros(a.N, 1, 2, 16, dtype=BF16).cuda()
    d = on_gpu(query, key, value, a.table, a.lens, a.starts)
    out = fc.append_paged(d[1], d[2], kp, vp, d[3], d[4], starts=d[5], query=d[0], bounds=bounds)
    assert torch.equal(out.cpu()[:a.T - 900], query[:a.T - 900]) and (out[a.T - 900:] == 0).all()
    held = vp.cpu()
    for t, b, pos in places(a.lens, a.starts, a.T):
        assert torch.equal(held[int(a.table[b, pos // 16]), 0, pos % 16, :3], part[t].to(BF16))
    pages = fc.select_pages(d[0], bounds, d[3], d[4], 3, page_size=16, starts=d[5])
    last = torch.full((a.T,), -1)
    for t, b, pos in places(a.lens, a.starts, a.T):
        last[t] = pos // 16
    assert torch.equal(pages.cpu()[:, 0].amax(1).long(), last)
    own = torch.full((a.T, 1, 1), -1, dtype=torch.int32)
    own[:, 0, 0] = last.int()
    got = fc.attend_pages(d[0], kp, vp, d[3], d[4], own.cuda(), starts=d[5]).cpu().double()
    # keys are zeros, so a result is the mean of what the token sees of its page
    for t, b, pos in places(a.lens, a.starts, a.T):
        seen = held[int(a.table[b, pos // 16]), 0, :pos % 16 + 1].double()
        mean, spread = seen.mean(0), seen.abs().mean(0)
        assert ((got[t] - mean).abs() <= 2.0 ** -8 * mean.abs() + 2.0 ** -14 * spread).all()
    assert (got[a.T - 900:] == 0).all()
    status_is(0)


@pytest.mark.parametrize("more", [0, 20])
def test_select_with_infinities_nan_and_pages_that_the_table_lacks(more):
    a = Batch(4, [3 + more, 1 + more], [16 * 60, 16 * 30], 16, 2, 2, 64, BF16)
    query = a.rows(2)
    bounds = torch.stack([a.normal(a.N, 2, 64) - 1, a.normal(a.N, 2, 64) + 1], 2)
    bounds[int(a.table[0, 20]), 0, 1, 3] = math.nan
    bounds[int(a.table[0, 40]), 1, 1, :] = math.inf
    bounds[int(a.table[1, 7]), 1, 0, 5] = -math.inf
    bounds[int(a.table[1, 9]), :, 1, :] = -math.inf
    bounds[int(a.table[1, 9]), :, 0, :] = math.inf
    query[2, 1] = math.nan
    a.table[0, 50], a.table[1, 3] = -1, a.N
    want = chosen_pages(query, bounds, 16, a.table, a.lens, a.starts, 8, 1, 1)
    assert torch.equal(select(a, query, bounds, 8, 1, 1).cpu(), want)
    status_is(5)
    for k in (57, 60):      # down to the pages that nothing speaks for
        want = chosen_pages(query, bounds, 16, a.table, a.lens, a.starts, k, 1, 1)
        assert torch.equal(select(a, query, bounds, k, 1, 1).cpu(), want)
    # a table narrower than the sequences are long
    a.table = a.table[:, :25].contiguous()
    want = chosen_pages(query, bounds, 16, a.table, a.lens, a.starts, 8, 1, 2)
    assert torch.equal(select(a, query, bounds, 8, 1, 2).cpu(), want)
    status_is(5)


# --------------------------------------------------------------------------- attend
ATTENDS = [
    # new tokens, lens, page, kv heads, heads, dim, type, k
    ([1], [1], 64, 1, 1, 8, BF16, 1),
    ([1], [64 * 40 - 3], 64, 8, 32, 128, BF16, 32),
    ([1, 1, 1], [700, 16, 333], 16, 2, 6, 80, FP16, 7),
    ([5, 0, 33, 1], [500, 17, 900, 1], 16, 3, 3, 64, BF16, 6),
    ([5, 0, 33, 1], [5, 17, 200, 160], 32, 4, 32, 40, FP16, 4),
    ([7], [3000], 128, 2, 24, 96, BF16, 12),
    ([9], [16 * 100 + 5], 16, 1, 16, 128, FP16, 40),
    ([1, 1], [128 * 70, 128 * 9 + 1], 128, 1, 20, 64, FP16, 64),
    ([3], [32 * 200], 32, 2, 18, 72, FP16, 150),
    ([1], [64 * 300], 64, 1, 8, 128, FP16, 290),
    ([1] * 260, [1 + 2 * i for i in range(260)], 16, 1, 4, 16, BF16, 3),
    # blocks of tokens: groups of four, eight, five and heads of their own, the last over one CTA, eight and four
    ([70, 1, 0, 33], [1500, 40, 9, 128 * 5], 64, 8, 32, 128, BF16, 9),
    ([40], [128 * 12 + 64], 128, 8, 64, 128, FP16, 7),
    ([40, 3, 11], [900, 16 * 30 + 3, 77], 16, 10, 50, 88, BF16, 20),
    ([300], [16 * 40], 16, 16, 16, 48, FP16, 11),
    ([100], [16 * 40], 16, 1, 1, 48, FP16, 11),
    ([100], [32 * 40 + 3], 32, 8, 8, 120, BF16, 13),
    # tokens one by one
    ([70, 1, 0, 33], [1500, 40, 9, 128 * 5], 64, 2, 8, 128, BF16, 9),
    ([65], [128 * 12 + 64], 128, 1, 32, 128, FP16, 7),
    ([1], [64 * 130], 64, 1, 12, 96, BF16, 128),      # one row over sixteen CTAs, three tokens over eight
    ([3], [64 * 130 + 7], 64, 1, 4, 128, FP16, 100),
]


def attend_room(dtype, D, keys, out, spread, reach):
    """How far a result may be: its own rounding, and to the sum of weights times magnitudes the relative error of a weight --
    what two roundings to 16 bits leave of it, its score's sum over D products (tensor-core sums drop what is below the largest
    term's last bit: D steps of 2^-23) and the exponential's and the sums' 32 bits."""
    half = torch.finfo(dtype).eps / 2
    weight = half * half + 2 * (D + 8) * 2.0 ** -23 * reach + 2.0 ** -19 + keys * 2.0 ** -24
    floor = torch.finfo(dtype).smallest_normal * half
    return half * out.abs() + (1 + half) * weight[..., None] * spread + floor


def listed_pages(a, k, dup=True):
    """Random lists: pages of the past, of the future, twice, none."""
    pages = torch.full((a.T, a.H, k), -1, dtype=torch.int32)
    for t, b, pos in places(a.lens, a.starts, a.T):
        seen = pos // a.P + 1
        for h in range(a.H):
            order = torch.randperm(seen, generator=a.g)[:k].sort().values.int()
            pages[t, h, :len(order)] = order
            if h % 2 and dup:
                pages[t, h] = pages[t, h, torch.randperm(k, generator=a.g)]
                pages[t, h, 0] = (pos // a.P) + (t + h) % 2
                if k > 2:
                    pages[t, h, k // 2] = -3
    return pages


@pytest.mark.parametrize("case", range(len(ATTENDS)))
@pytest.mark.parametrize("layout", ["plain", "strided"])
def test_attend_is_attention_over_the_listed_pages(case, layout):
    import flash_colsum_b200 as fc
    new, lens, P, H, heads, D, dtype, k = ATTENDS[case]
    packed = max(new) > 1 or min(new) < 1
    tail = 2 if packed and case % 2 else 0
    a = Batch(case, new, lens, P, H, heads, D, dtype, tail=tail, packed=packed)
    query, pools = a.rows(heads), [a.pool(), a.pool()]
    query[:, ::2] *= 4                   # heads that attend to a few keys
    for b, n in enumerate(lens):         # behind the last token lies anything
        if n % P:
            pools[0][int(a.table[b, n // P]), :, n % P:] = math.nan
            pools[1][int(a.table[b, n // P]), :, n % P:] = math.inf if b % 2 else math.nan
    pages = listed_pages(a, k)
    scale = None if case % 2 else -0.11
    used = D ** -0.5 if scale is None else scale
    want, lse, spread, reach = attention(query, *pools, a.table, a.lens, a.starts, pages, used)
    d_query, d_pages, table, d_lens, starts = on_gpu(query, pages, a.table, a.lens, a.starts)
    if layout == "strided":
        both = torch.stack([p.transpose(1, 2) for p in pools], 1).contiguous().cuda()
        d_pools = [both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)]
        d_query = torch.cat([d_query, d_query], 1)[:, heads:]
        table = torch.cat([table, table], 1)[:, :table.shape[1]]
    else:
        d_pools = on_gpu(*pools)
    out, got_lse = fc.attend_pages(d_query, *d_pools, table, d_lens, d_pages, starts=starts, scale=scale, return_lse=True)
    status_is(0)
    room = attend_room(dtype, D, k * P, want, spread, reach)
    assert ((out.cpu().double() - want).abs() <= room).all()
    some = lse.isfinite()
    assert torch.equal(got_lse.cpu()[~some].double(), lse[~some])
    lse_room = (D + 8) * 2.0 ** -23 * reach + 2.0 ** -19 + k * P * 2.0 ** -24 + lse.abs() * 2.0 ** -22
    assert ((got_lse.cpu().double() - lse).abs() <= lse_room)[some].all()
    assert (out[a.T - tail:] == 0).all()
    mine = torch.full((a.T, 2 * heads, D), 5.0, dtype=dtype, device="cuda")
    again = fc.attend_pages(d_query, *d_pools, table, d_lens, d_pages, starts=starts, scale=scale, out=mine[:, heads:])
    assert again.data_ptr() == mine[:, heads:].data_ptr() and torch.equal(mine[:a.T - tail, heads:], out[:a.T - tail])
    assert (mine[:, :heads] == 5).all() and (mine[a.T - tail:] == 5).all()


def test_attend_with_scores_at_the_ends_of_the_range():
    """Keys that are taken out by a feature of -inf or of the type's lowest value, a row whose keys all are, NaN and +inf."""
    import flash_colsum_b200 as fc
    for dtype in (BF16, FP16):
        a = Batch(8, [2], [40], 16, 6, 6, 64, dtype)
        query, pools = a.rows(6), [a.pool(), a.pool()]
        query[:, :, 0] = 1.0
        pages = torch.arange(3, dtype=torch.int32).expand(a.T, 6, 3).contiguous()
        at = a.table[0].long()
        pools[0][at[0], 0, 3:, 0] = -math.inf
        pools[0][at[1], 1, :, 0] = torch.finfo(dtype).min
        pools[0][at, 2, :, 0] = -math.inf                # all of them
        pools[0][at[1], 3, 2, 5] = math.nan
        pools[0][at[0], 4, 9, 0] = math.inf
        want, lse, spread, reach = attention(query, *pools, a.table, a.lens, a.starts, pages, 0.125)
        args = on_gpu(query, *pools, a.table, a.lens, pages)
        out, got = fc.attend_pages(*args, starts=a.starts.cuda(), return_lse=True)
        out, got = out.cpu().double(), got.cpu().double()
        for h in (0, 1, 5):
            finite = reach[:, h].clamp(max=64.0)        # (of the keys that are left)
            room = attend_room(dtype, 64, 48, want[:, h], spread[:, h], finite)
            assert ((out[:, h] - want[:, h]).abs() <= room).all(), (dtype, h)
            assert ((got[:, h] - lse[:, h]).abs() <= 72 * 2.0 ** -23 * finite + 2.0 ** -18).all(), (dtype, h)
        assert (out[:, 2] == 0).all() and (got[:, 2] == -math.inf).all()
        assert out[:, 3].isnan().all() and got[:, 3].isnan().all()
        assert out[:, 4].isnan().all() and (got[:, 4] == math.inf).all()
        status_is(0)


# (one CTA a block, two and eight: blocks for all SMs, or of eight tokens and more)
@pytest.mark.parametrize("D,P,group,H,tokens", [(128, 64, 4, 8, 90), (64, 16, 1, 2, 23), (96, 128, 8, 8, 41), (40, 32, 2, 20, 125),
                                                (128, 16, 3, 16, 50)])
def test_attend_keeps_the_tokens_of_a_block_apart(D, P, group, H, tokens):
    """Neighbouring tokens whose lists share pages: values that are not finite reach those that listed their page, and no others;
    nor do the keys behind a token, or a page that another token listed twice."""
    import flash_colsum_b200 as fc
    held = -(-tokens // P) + 9
    a = Batch(21, [tokens], [P * held + 5], P, H, H * group, D, BF16)
    query, pools = a.rows(H * group), [a.pool(), a.pool()]
    pages = torch.full((a.T, H, 6), -1, dtype=torch.int32)
    for t in range(a.T):
        for h in range(H):
            order = torch.randperm(9, generator=a.g)[:5].int()
            pages[t, h, :5] = order
    for kind in ("nan in a page", "inf in keys and values", "nan in a later token", "twice"):
        k, v, lists = pools[0].clone(), pools[1].clone(), pages.clone()
        if kind == "nan in a page":
            v[int(a.table[0, 3]), :, P - 1, 2] = math.nan
        elif kind == "inf in keys and values":
            v[int(a.table[0, 4]), 1, 0, :] = math.inf
            k[int(a.table[0, 5]), 0, 3, 1] = math.inf
        elif kind == "nan in a later token":          # the block's own page, which all of it lists
            own = (torch.arange(a.T) + P * held + 5 - tokens) // P
            lists[:, :, 5] = own[:, None].int()
            at = a.lens[0] - 2
            v[int(a.table[0, at // P]), :, int(at) % P, 0] = math.nan
        else:
            lists[11, 0, 5] = lists[11, 0, 1]
            lists[4, 1, 0:3] = 2
        want, lse, spread, reach = attention(query, k, v, a.table, a.lens, a.starts, lists, D ** -0.5)
        out, got = fc.attend_pages(*on_gpu(query, k, v, a.table, a.lens, lists), starts=a.starts.cuda(), return_lse=True)
        out, got = out.cpu().double(), got.cpu().double()
        assert torch.equal(out.isfinite(), want.isfinite())
        fine = want.isfinite()
        room = attend_room(BF16, D, 6 * P, want, spread, reach)
        assert ((out - want).abs() <= room)[fine].all()
        some = lse.isfinite()
        assert torch.equal(got[~some].isnan(), lse[~some].isnan())
        assert torch.equal(got == math.inf, lse == math.inf)
        assert ((got - lse).abs() <= (D + 8) * 2.0 ** -23 * reach + 2.0 ** -18 + lse.abs() * 2.0 ** -22)[some].all()
    status_is(0)


@pytest.mark.parametrize("width", [8192, 8193])
def test_attend_of_blocks_under_a_wide_table(width):
    """On both sides of the widest table that tokens share their pages under."""
    import flash_colsum_b200 as fc
    a = Batch(22, [9, 30], [16 * 50, 16 * 70 + 1], 16, 2, 2, 64, FP16, width=width, tail=3)
    query, pools = a.rows(2), [a.pool(), a.pool()]
    pages = listed_pages(a, 8)
    pages[2, 0, 0], pages[2, 1, 1] = 8192, 2 ** 31 - 1            # behind the token
    want, lse, spread, reach = attention(query, *pools, a.table, a.lens, a.starts, pages, 0.125)
    out = fc.attend_pages(*on_gpu(query, *pools, a.table, a.lens, pages), starts=a.starts.cuda())
    assert ((out.cpu().double() - want).abs() <= attend_room(FP16, 64, 128, want, spread, reach)).all()
    assert (out[39:] == 0).all()
    status_is(0)


def test_attend_reads_nothing_from_pages_that_the_table_lacks():
    import flash_colsum_b200 as fc
    a = Batch(9, [2, 1], [64 * 9, 64 * 4], 64, 2, 8, 128, BF16)
    query, pools = a.rows(8), [a.pool(), a.pool()]
    pages = listed_pages(a, 5, dup=False)
    a.table[0, 2], a.table[0, 5], a.table[1, 0], a.table[1, 3] = -1, a.N, 2 ** 31 - 1, -2 ** 31
    want, lse, spread, reach = attention(query, *pools, a.table, a.lens, a.starts, pages, 128 ** -0.5)
    args = on_gpu(query, *pools, a.table, a.lens, pages)
    out, got = fc.attend_pages(*args, starts=a.starts.cuda(), return_lse=True)
    status_is(5)
    assert ((out.cpu().double() - want).abs() <= attend_room(BF16, 128, 320, want, spread, reach)).all()
    pages[0, 0, 0] = 2 ** 31 - 1       # (far behind the token: no page of its)
    again = fc.attend_pages(*args[:5], pages.cuda(), starts=a.starts.cuda())
    status_is(5)
    assert torch.equal(again[1:], out[1:])


def test_pools_of_more_than_two_to_the_32_elements():
    import flash_colsum_b200 as fc
    P, H, D = 64, 8, 128
    N = 2 ** 32 // (P * H * D) + 40
    pools = [torch.empty(N, H, P, D, dtype=BF16, device="cuda") for _ in range(2)]
    bounds = torch.empty(N, H, 2, D, dtype=BF16, device="cuda")
    a = Batch(10, [100], [100], P, H, 32, D, BF16, spare_pages=0)
    table = torch.tensor([[N - 1, N - 7]], dtype=torch.int32).cuda()
    key, value, query = (t.cuda() for t in (a.rows(H), a.rows(H), a.rows(32)))
    lens, starts = a.lens.cuda(), a.starts.cuda()
    rotated_query = fc.append_paged(key, value, *pools, table, lens, starts=starts, query=query, bounds=bounds)
    assert torch.equal(rotated_query, query)
    assert torch.equal(pools[0][N - 1], key[:64].transpose(0, 1)) and torch.equal(pools[1][N - 7, :, :36], value[64:].transpose(0, 1))
    pages = fc.select_pages(query, bounds, table, lens, 2, page_size=P, starts=starts)
    assert pages[99, 0].tolist() == [0, 1] and pages[0, 0].tolist() == [0, -1]
    out = fc.attend_pages(query, *pools, table, lens, pages, starts=starts)
    small = [torch.zeros(2, H, P, D, dtype=BF16) for _ in range(2)]
    for s, p in zip(small, pools):
        s[0], s[1, :, :36] = p[N - 1].cpu(), p[N - 7, :, :36].cpu()
    want, _, spread, reach = attention(query.cpu(), *small, torch.tensor([[0, 1]]), a.lens, a.starts, pages.cpu(), D ** -0.5)
    assert ((out.cpu().double() - want).abs() <= attend_room(BF16, D, 128, want, spread, reach)).all()
    status_is(0)


# --------------------------------------------------------------------------- together
def test_a_pruned_prompt_and_the_steps_that_follow_it():
    """Column means choose the prompt's tokens, those are cached under their own positions, and every following step appends,
    chooses pages and attends; with pages enough for all the result is attention over everything that was kept."""
    import flash_colsum_b200 as fc
    torch.manual_seed(11)
    H, D, S, P, kept = 4, 64, 300, 16, 150
    prompt_q, prompt_k, prompt_v = (torch.randn(1, H, S, D, dtype=FP16, device="cuda") for _ in range(3))
    turn = torch.arange(S + 40, dtype=torch.float64)[:, None] * 10.0 ** -torch.linspace(0, 3, D // 2, dtype=torch.float64)
    cos, sin = turn.cos().float().cuda(), turn.sin().float().cuda()
    _, index = fc.topk_columns(fc.flash_colsum(prompt_q[:, :, -64:], prompt_k, is_causal=True), kept)
    take = index[0].long()
    N = 16
    pools = [torch.zeros(N, H, P, D, dtype=FP16, device="cuda") for _ in range(2)]
    bounds = torch.zeros(N, H, 2, D, dtype=FP16, device="cuda")
    table = torch.randperm(N, device="cuda").int()[None]
    lens = torch.tensor([kept], dtype=torch.int32, device="cuda")
    fc.append_paged(prompt_k[0, :, take].transpose(0, 1), prompt_v[0, :, take].transpose(0, 1), *pools, table, lens,
                    starts=torch.tensor([0, kept], dtype=torch.int32, device="cuda"), cos=cos, sin=sin, positions=index[0], bounds=bounds)
    keys = torch.cat([rotated(prompt_k[0, :, i].double().cpu(), cos[i].double().cpu(), sin[i].double().cpu(), False)[0][None]
                      for i in index[0].tolist()])
    values = prompt_v[0, :, take].transpose(0, 1).double().cpu()
    for step in range(30):
        q, k, v = (torch.randn(1, H, D, dtype=FP16, device="cuda") for _ in range(3))
        lens += 1
        where = torch.tensor([S + step], dtype=torch.int32, device="cuda")
        turned = fc.append_paged(k, v, *pools, table, lens, query=q, cos=cos, sin=sin, positions=where, bounds=bounds)
        pages = fc.select_pages(turned, bounds, table, lens, N, page_size=P)
        some = fc.select_pages(turned, bounds, table, lens, 4, page_size=P)
        out = fc.attend_pages(turned, *pools, table, lens, pages)
        part, lse = fc.attend_pages(turned, *pools, table, lens, some, return_lse=True)
        c, s = cos[S + step].double().cpu(), sin[S + step].double().cpu()
        keys = torch.cat([keys, rotated(k[0].double().cpu(), c, s, False)[0][None]])
        values = torch.cat([values, v.double().cpu()])
        x = rotated(q[0].double().cpu(), c, s, False)[0]
        w = torch.softmax(torch.einsum("hd,nhd->hn", x, keys) / D ** 0.5, 1)
        want = torch.einsum("hn,nhd->hd", w, values)
        spread = torch.einsum("hn,nhd->hd", w, values.abs())
        reach = torch.einsum("hd,nhd->hn", x.abs(), keys.abs()).amax(1) / D ** 0.5
        # queries and keys are held in 16 bits: each score off by two half steps of its terms
        room = (2.0 ** -11 * want.abs() + (2 * 2 * 2.0 ** -11 * reach + 2.0 ** -15)[:, None] * spread + 2.0 ** -25)
        assert ((out[0].cpu().double() - want).abs() <= room).all()
        assert pages[0, 0].tolist() == list(range(-(-int(lens) // P))) + [-1] * (N - -(-int(lens) // P))
        want_part, want_lse, spread, reach = attention(turned.cpu(), pools[0].cpu(), pools[1].cpu(), table.cpu(), lens.cpu(), None,
                                                       some.cpu(), D ** -0.5)
        assert ((part.cpu().double() - want_part).abs() <= attend_room(FP16, D, 64, want_part, spread, reach)).all()
        assert torch.equal(some.cpu(), chosen_pages(turned.cpu(), bounds.cpu(), P, table.cpu(), lens.cpu(), None, 4, 1, 1))
    status_is(0)


def test_a_captured_step_follows_its_batch_and_two_graphs_keep_apart():
    import flash_colsum_b200 as fc
    H, heads, D, P, N = 2, 8, 128, 64, 40

    def program(seed):
        g = torch.Generator().manual_seed(seed)
        s = dict(q=torch.randn(3, heads, D, generator=g).to(BF16).cuda(), k=torch.randn(3, H, D, generator=g).to(BF16).cuda(),
                 v=torch.randn(3, H, D, generator=g).to(BF16).cuda(), kp=torch.randn(N, H, P, D, generator=g).to(BF16).cuda(),
                 vp=torch.randn(N, H, P, D, generator=g).to(BF16).cuda(), table=torch.randperm(N, generator=g).int()[:36].view(3, 12).cuda(),
                 lens=torch.tensor([700, 64, 13], dtype=torch.int32).cuda(), cos=torch.rand(800, 64, generator=g).cuda(),
                 sin=torch.rand(800, 64, generator=g).cuda())
        s["bounds"] = torch.stack([s["kp"].amin(2), s["kp"].amax(2)], 2)
        return s

    def step(s):
        s["lens"] += 1
        q = fc.append_paged(s["k"], s["v"], s["kp"], s["vp"], s["table"], s["lens"], query=s["q"], cos=s["cos"], sin=s["sin"],
                            bounds=s["bounds"])
        pages = fc.select_pages(q, s["bounds"], s["table"], s["lens"], 4, page_size=P)
        return pages, *fc.attend_pages(q, s["kp"], s["vp"], s["table"], s["lens"], pages, return_lse=True)

    step(program(0))
    torch.cuda.synchronize()
    eager, held = [program(1), program(2)], [program(1), program(2)]
    graphs, outs = [], []
    for s in held:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step(s))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        want = [step(s) for s in eager]
        for s in held + eager:
            torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for w, o, s, e in zip(want, outs, held, eager):
            assert all(torch.equal(x, y) for x, y in zip(w, o))
            assert torch.equal(s["kp"], e["kp"]) and torch.equal(s["bounds"], e["bounds"])
            q = torch.randn(3, heads, D, device="cuda").to(BF16)
            s["q"].copy_(q)
            e["q"].copy_(q)
    status_is(0)
    del graphs


def test_calls_on_a_side_stream_and_results_that_repeat():
    import flash_colsum_b200 as fc
    a = Batch(12, [1] * 40, [64 * 30 + i for i in range(40)], 64, 4, 16, 128, BF16, packed=False)
    query, kp, vp, table, lens = on_gpu(a.rows(16), a.pool(), a.pool(), a.table, a.lens)
    bounds = torch.stack([kp.amin(2), kp.amax(2)], 2)
    pages = fc.select_pages(query, bounds, table, lens, 12, page_size=64)
    out = fc.attend_pages(query, kp, vp, table, lens, pages)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        with torch.cuda.stream(side):
            p2 = fc.select_pages(query, bounds, table, lens, 12, page_size=64)
            o2 = fc.attend_pages(query, kp, vp, table, lens, p2)
        p3 = fc.select_pages(query, bounds, table, lens, 12, page_size=64)
        o3 = fc.attend_pages(query, kp, vp, table, lens, p3)
        torch.cuda.synchronize()
        assert torch.equal(p2, pages) and torch.equal(p3, pages) and torch.equal(o2, out) and torch.equal(o3, out)


def test_refusals_and_calls_without_tokens():
    import flash_colsum_b200 as fc
    a = Batch(13, [2, 3], [40, 3], 16, 2, 4, 64, BF16)
    q, k, kp, vp, table, lens, starts = on_gpu(a.rows(4), a.rows(2), a.pool(), a.pool(), a.table, a.lens, a.starts)
    bounds = torch.stack([kp.amin(2), kp.amax(2)], 2)
    cos = torch.ones(64, 32).cuda()

    def append(match, *args, **kw):
        with pytest.raises(ValueError, match=match):
            fc.append_paged(*args, **kw)

    base = (k, k, kp, vp, table, lens)

    def swapped(i, x):
        return base[:i] + (x,) + base[i + 1:]

    append("float16 or bfloat16", *swapped(0, k.float()), starts=starts)
    append("value must be", *swapped(1, k[:4]), starts=starts)
    append("one token a sequence", *base)
    append("head_dim", *(t[..., :60] for t in base[:4]), table, lens, starts=starts)
    append("page size", k, k, kp[:, :, :15], vp[:, :, :15], table, lens, starts=starts)
    append("pools hold 2 heads", q, q, *base[2:], starts=starts)
    append("rows apart", *swapped(2, kp[:1].expand(a.N, 2, 16, 64)), starts=starts)
    append("unit inner stride", *swapped(2, kp.transpose(2, 3).contiguous().transpose(2, 3)), starts=starts)
    append("int32", *swapped(4, table.long()), starts=starts)
    append("int32", *swapped(5, lens.cpu()), starts=starts)
    append("3 entries", *base, starts=starts[:2])
    append("go together", *base, starts=starts, cos=cos)
    append("cos and sin must be", *base, starts=starts, cos=cos[:, :4].contiguous(), sin=cos[:, :4].contiguous())
    append("positions", *base, starts=starts, positions=lens)
    append("positions must have", *base, starts=starts, cos=cos, sin=cos, positions=lens)
    append("multiple of the 2", *base, starts=starts, query=q[:, :3])
    append("query_out", *base, starts=starts, query_out=q)
    append("bounds must be", *base, starts=starts, bounds=bounds[1:])
    append("bounds must be contiguous", *base, starts=starts, bounds=bounds.transpose(2, 3).contiguous().transpose(2, 3))
    with pytest.raises(ValueError, match="k must hold"):
        fc.select_pages(q, bounds, table, lens, 2, page_size=16, starts=starts, first=1, last=2)
    with pytest.raises(ValueError, match="last be at least 1"):
        fc.select_pages(q, bounds, table, lens, 2, page_size=16, starts=starts, last=0)
    with pytest.raises(ValueError, match="page size"):
        fc.select_pages(q, bounds, table, lens, 2, page_size=48, starts=starts)
    with pytest.raises(TypeError):
        fc.select_pages(q, bounds, table, lens, 2.5, page_size=16, starts=starts)
    with pytest.raises(ValueError, match="bounds must be"):
        fc.select_pages(q, bounds[..., :32].contiguous(), table, lens, 2, page_size=16, starts=starts)
    pages = fc.select_pages(q, bounds, table, lens, 2, page_size=16, starts=starts)
    with pytest.raises(ValueError, match="out must be"):
        fc.select_pages(q, bounds, table, lens, 2, page_size=16, starts=starts, out=pages[:, :, :1])
    with pytest.raises(ValueError, match="pages must be"):
        fc.attend_pages(q, kp, vp, table, lens, pages[:4], starts=starts)
    with pytest.raises(ValueError, match="not a number"):
        fc.attend_pages(q, kp, vp, table, lens, pages, starts=starts, scale=math.nan)
    with pytest.raises(ValueError, match="out needs"):
        fc.attend_pages(q, kp, vp, table, lens, pages, starts=starts, out=torch.empty(5, 64, 4, dtype=BF16, device="cuda").transpose(1, 2))
    with pytest.raises(ValueError, match="row of at least one page"):
        fc.attend_pages(q, kp, vp, table[:, :0], lens, pages, starts=starts)
    # no tokens at all
    none = torch.zeros(3, dtype=torch.int32).cuda()
    assert fc.append_paged(k[:0], k[:0], kp, vp, table, lens, starts=none, query=q[:0]).shape == (0, 4, 64)
    assert fc.append_paged(k[:0], k[:0], kp, vp, table, lens, starts=none) is None
    assert fc.select_pages(q[:0], bounds, table, lens, 2, page_size=16, starts=none).shape == (0, 2, 2)
    out, lse = fc.attend_pages(q[:0], kp, vp, table, lens, pages[:0], starts=none, return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    # rows that all lie behind the last sequence
    assert (fc.append_paged(k, k, kp, vp, table, lens, starts=none, query=q) == 0).all()
    assert (fc.select_pages(q, bounds, table, lens, 2, page_size=16, starts=none) == -1).all()
    out, lse = fc.attend_pages(q, kp, vp, table, lens, pages, starts=none, return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    status_is(0)
