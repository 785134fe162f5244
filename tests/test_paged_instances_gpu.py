"""Every instance that the calls over a paged cache dispatch to: types, head dimensions, columns, CTAs of a cluster, steps of heads.

Each case says which instance it is for and asks the library's plan, so that a rule that is tuned anew cannot leave one untested."""

import math

import pytest
import torch

from paged_reference import Batch, attention, chosen_pages, places
from test_paged_gpu import BF16, FP16, attend_room, device_stays_sound, on_gpu, select, status_is  # noqa: F401  (a fixture of all)
from test_paged_limits_gpu import c_cache

pytestmark = pytest.mark.gpu


def plan_of(a, k):
    from flash_colsum_b200 import _cabi
    table, lens, starts = on_gpu(a.table, a.lens, a.starts)
    pool = torch.empty(0, device="cuda")
    c = c_cache(a, table, lens, starts if starts is not None else pool)
    if starts is None:
        c.starts = None
    return _cabi.paged_plan(c, a.heads, k)


# --------------------------------------------------------------------------- append
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("rotation", ["none", "halves", "neighbours"])
@pytest.mark.parametrize("tokens,H,heads,group_heads,steps", [(64, 3, 9, 2, 1), (1003, 11, 44, 2, 2), (4003, 11, 44, 2, 4), (4003, 5, 50, 2, 4)])
def test_append_at_every_number_of_steps(tokens, H, heads, group_heads, steps, rotation, dtype):
    """Heads that are no multiple of those that a CTA has, in every kind of rotation."""
    import flash_colsum_b200 as fc
    P, D, R = 16, 24, 16
    a = Batch(50, [tokens], [tokens + 21], P, H, heads, D, dtype)
    plan = plan_of(a, 1)
    assert (plan["append_heads"], plan["append_steps"]) == (group_heads, steps)
    key, value, query, pools = a.rows(H), a.rows(H), a.rows(heads), [a.pool(), a.pool()]
    bounds = torch.stack([pools[0].amin(2), pools[0].amax(2)], 2)
    cos = sin = None
    if rotation != "none":
        turn = torch.arange(tokens + 21, dtype=torch.float64)[:, None] * 10.0 ** -torch.linspace(0, 3, R // 2, dtype=torch.float64)
        cos, sin = turn.cos().float(), turn.sin().float()
    d = on_gpu(key, value, *pools, a.table, a.lens, a.starts, query, cos, sin, bounds)
    got = fc.append_paged(*d[:6], starts=d[6], query=d[7], cos=d[8], sin=d[9], interleaved=rotation == "neighbours", bounds=d[10])
    where = torch.tensor([pos for _, _, pos in places(a.lens, a.starts, a.T)])
    page, slot = a.table[0, where // P].long(), where % P
    half, floor = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2

    def close(x, rows):       # three roundings to 32 bits, one to 16
        c, s = (None, None) if cos is None else (cos[where].double()[:, None], sin[where].double()[:, None])
        if c is None:
            return torch.equal(x, rows)
        exact, size = x.double().clone(), rows.double().abs()
        i = torch.arange(R // 2)
        m, n = (2 * i, 2 * i + 1) if rotation == "neighbours" else (i, i + R // 2)
        u, v = rows.double()[..., m], rows.double()[..., n]
        exact[..., m], exact[..., n] = u * c - v * s, v * c + u * s
        size[..., m], size[..., n] = (u * c).abs() + (v * s).abs(), (v * c).abs() + (u * s).abs()
        error = 2 * 2.0 ** -24 * size
        return torch.equal(x[..., R:], rows[..., R:]) and bool(((x.double() - exact).abs() <= error + half * (exact.abs() + error) + floor).all())

    stored, values = d[2].cpu(), d[3].cpu()
    assert close(got.cpu(), query) and close(stored[page, :, slot], key) and torch.equal(values[page, :, slot], value)
    # the rest of the pools is as it was, and the bounds are those of the keys since slot 0 was written
    clean = [pools[0].clone(), pools[1].clone()]
    clean[0][page, :, slot], clean[1][page, :, slot] = stored[page, :, slot], value
    assert torch.equal(stored, clean[0]) and torch.equal(values, clean[1])
    want = bounds.clone()
    for i in range(21 // P, -(-(tokens + 21) // P)):
        at, n = int(a.table[0, i]), min(P, tokens + 21 - i * P)
        first = max(0, 21 - i * P)
        low, high = stored[at, :, first:n].amin(1), stored[at, :, first:n].amax(1)
        if first:
            low, high = torch.minimum(low, bounds[at, :, 0]), torch.maximum(high, bounds[at, :, 1])
        want[at] = torch.stack([low, high], 1)
    assert torch.equal(d[10].cpu(), want)
    status_is(0)


# --------------------------------------------------------------------------- select
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [56, 128])
# rows, pages of the longest, width, CTAs: by the table's width, and by the rows that there are
@pytest.mark.parametrize("rows,H,pages,width,ctas", [(3, 2, 120, 127, 1), (3, 2, 127, 130, 2), (3, 2, 240, 260, 4), (3, 2, 500, 520, 8), (3, 2, 900, 1030, 16),
                                                     (225, 2, 40, 1030, 1), (56, 4, 60, 1030, 2), (28, 4, 70, 1030, 4), (14, 4, 90, 1030, 8)])
def test_select_a_row_at_a_time_at_every_cluster_size(rows, H, pages, width, ctas, D, dtype):
    k = 9
    a = Batch(51, [1] * rows, [16 * pages - 37 * i % (8 * pages) for i in range(rows)], 16, H, 2 * H, D, dtype, packed=False, width=width)
    plan = plan_of(a, k)
    assert (plan["select_tiles"], plan["select_ctas"], plan["select_launches"]) == (0, ctas, 1)
    query = a.rows(2 * H)
    centre = torch.randn(a.N, H, D, generator=a.g)
    bounds = torch.stack([centre - 1.0, centre + 1.0], 2).to(dtype)
    assert torch.equal(select(a, query, bounds, k, 1, 2).cpu(), chosen_pages(query, bounds, 16, a.table, a.lens, None, k, 1, 2))
    status_is(0)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_select_a_row_at_a_time_in_several_launches(dtype):
    """More tokens than one launch's sums in 64 bits have room for, which in the second launch are needed: its pages are equal."""
    rows, H, D, k = 70, 16, 16, 7
    a = Batch(52, [1] * rows, [16 * 12 + i % 90 for i in range(rows)], 16, H, H, D, dtype, packed=False, width=32700)
    plan = plan_of(a, k)
    assert (plan["select_tiles"], plan["select_launches"]) == (0, 2)
    query = a.rows(H)
    bounds = torch.stack([a.normal(a.N, H, D) - 1, a.normal(a.N, H, D) + 1], 2)
    bounds[a.table[66:68, :12].long().flatten()] = 1.0
    assert torch.equal(select(a, query, bounds, k, 1, 1).cpu(), chosen_pages(query, bounds, 16, a.table, a.lens, None, k, 1, 1))
    query[69, 3, 2] = math.inf                                    # (no finite error: 64 bits decide)
    assert torch.equal(select(a, query, bounds, k, 1, 1).cpu(), chosen_pages(query, bounds, 16, a.table, a.lens, None, k, 1, 1))
    status_is(0)


def test_select_for_a_chunk_in_several_launches_under_a_wide_table():
    """A table of 8192 pages, and more tokens than one launch's scores have room for."""
    a = Batch(53, [5, 380], [16 * 9, 16 * 40], 16, 8, 8, 16, FP16, width=8192, tail=3)
    plan = plan_of(a, 6)
    assert (plan["select_tiles"], plan["select_launches"]) == (1, 2)
    query = a.rows(8)
    bounds = torch.stack([a.normal(a.N, 8, 16) - 1, a.normal(a.N, 8, 16) + 1], 2)
    assert torch.equal(select(a, query, bounds, 6, 1, 1).cpu(), chosen_pages(query, bounds, 16, a.table, a.lens, a.starts, 6, 1, 1))
    status_is(0)


# --------------------------------------------------------------------------- attend
def lists(a, k):
    """Pages of the past in any order, fewer than k for some; of the second head one of them twice for some."""
    pages = torch.full((a.T, a.H, k), -1, dtype=torch.int32)
    for t, _, pos in places(a.lens, a.starts, a.T):
        seen = pos // a.P + 1
        for h in range(a.H):
            order = torch.randperm(seen, generator=a.g)[:k - (t + h) % 3].int()
            pages[t, h, :len(order)] = order
            if h == 1 and t % 7 == 3:        # (which sends the whole block through its tokens' own lists)
                pages[t, h, len(order) - 1] = order[0]
    return pages


def attends(a, k):
    import flash_colsum_b200 as fc
    query, pools = a.rows(a.heads), [a.pool(), a.pool()]
    query[:, ::2] *= 4                       # heads that attend to a few keys
    for b, n in enumerate(a.lens.tolist()):  # behind the last token lies anything
        if n % a.P:
            pools[0][int(a.table[b, n // a.P]), :, n % a.P:] = math.nan
            pools[1][int(a.table[b, n // a.P]), :, n % a.P:] = math.inf
    pages = lists(a, k)
    want, lse, spread, reach = attention(query, *pools, a.table, a.lens, a.starts, pages, a.dim ** -0.5)
    d = on_gpu(query, *pools, a.table, a.lens, pages, a.starts)
    out, got = fc.attend_pages(*d[:6], starts=d[6], return_lse=True)
    assert ((out.cpu().double() - want).abs() <= attend_room(a.dtype, a.dim, k * a.P, want, spread, reach)).all()
    room = (a.dim + 8) * 2.0 ** -23 * reach + 2.0 ** -19 + k * a.P * 2.0 ** -24 + lse.abs() * 2.0 ** -22
    assert ((got.cpu().double() - lse).abs() <= room).all()
    status_is(0)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [48, 128])
@pytest.mark.parametrize("group", [4, 8, 12])                 # one and two sets of eight queries
@pytest.mark.parametrize("rows,H,ctas", [(2, 4, 16), (4, 7, 8), (6, 8, 4), (10, 10, 2), (20, 10, 1)])
def test_attend_a_row_at_a_time_at_every_cluster_size(rows, H, ctas, group, D, dtype):
    P, k = 128, 16
    a = Batch(54, [1] * rows, [P * 18 - 31 * i for i in range(rows)], P, H, H * group, D, dtype, packed=False)
    plan = plan_of(a, k)
    assert (plan["attend_tokens"], plan["attend_queries"], plan["attend_ctas"]) == (1, 8 if group <= 8 else 16, ctas)
    attends(a, k)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [40, 112])
@pytest.mark.parametrize("group,H,tokens,together,ctas", [(8, 16, 40, 2, 1), (4, 20, 43, 4, 2), (2, 10, 83, 8, 4), (1, 2, 40, 16, 8)])
def test_attend_in_blocks_of_tokens_at_every_cluster_size(group, H, tokens, together, ctas, D, dtype):
    P, k = 16, 9
    a = Batch(55, [tokens], [P * 20 + tokens + 5], P, H, H * group, D, dtype)
    plan = plan_of(a, k)
    assert (plan["attend_tokens"], plan["attend_queries"], plan["attend_ctas"]) == (together, 16, ctas)
    attends(a, k)


@pytest.mark.parametrize("group", [5, 6, 7, 8])
def test_attend_in_blocks_of_few_tokens(group):
    """Groups of which two or three tokens fill a block's columns, and one of whose columns belongs to nobody."""
    a = Batch(56, [31, 2], [64 * 9 + 3, 64 * 4], 64, 16, 16 * group, 64, BF16)
    assert plan_of(a, 6)["attend_tokens"] == 16 // group
    attends(a, 6)
