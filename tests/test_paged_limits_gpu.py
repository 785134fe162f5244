"""What the entry points over a paged cache do at their limits: pages that the table lacks, the largest lists, results in odd memory."""

import ctypes

import pytest
import torch

from paged_reference import Batch, attention, chosen_pages, places
from test_paged_gpu import BF16, FP16, attend_room, device_stays_sound, on_gpu, select, status_is  # noqa: F401  (a fixture of all)

pytestmark = pytest.mark.gpu


# --------------------------------------------------------------------------- pages that the table lacks
@pytest.mark.parametrize("tokens", [1, 3, 23, 90])     # a cluster a row, and tiles of 64 tokens
@pytest.mark.parametrize("fault", ["narrow", "first", "own", "last but one", "competing", "behind", "other sequence's end"])
@pytest.mark.parametrize("k", [8, 60])                # fewer than the pages that are seen, and all of them
def test_a_selection_says_which_pages_it_misses(tokens, fault, k):
    """Forced pages, and those of rows that take all they see, are looked up like those that compete."""
    a = Batch(31, [tokens, 1], [16 * 50, 16 * 9], 16, 2, 2, 64, BF16, width=60)
    query = a.rows(2)
    bounds = torch.stack([a.normal(a.N, 2, 64) - 1, a.normal(a.N, 2, 64) + 1], 2)
    if fault == "narrow":
        a.table = a.table[:, :49].contiguous()       # the last token's page is the 50th
    else:
        sequence, entry = {"first": (0, 0), "own": (0, 49), "last but one": (0, 48), "competing": (0, 20), "behind": (0, 50),
                           "other sequence's end": (1, 9)}[fault]
        a.table[sequence, entry] = -1 if tokens % 2 else a.N
    want = chosen_pages(query, bounds, 16, a.table, a.lens, a.starts, k, 1, 2)
    assert torch.equal(select(a, query, bounds, k, 1, 2).cpu(), want)
    status_is(0 if fault in ("behind", "other sequence's end") else 5)


# --------------------------------------------------------------------------- the largest lists
@pytest.mark.parametrize("width", [4, 40000])         # a cluster a row, and tiles
@pytest.mark.parametrize("k", [2 ** 31 - 1, 2 ** 31 - 128])
def test_the_longest_list_ends_where_its_memory_ends(width, k):
    """A list may be as long as its type counts: what steps through it leaves nothing in front of it or behind it."""
    import flash_colsum_b200 as fc
    a = Batch(32, [1], [16 * 3 + 1], 16, 1, 1, 16, BF16, packed=False, width=width)
    query, table, lens = on_gpu(a.rows(1), a.table, a.lens)
    bounds = torch.zeros(a.N, 1, 2, 16, dtype=BF16, device="cuda")
    around = torch.full((k + 512,), 7, dtype=torch.int32, device="cuda")
    out = around[256:256 + k].view(1, 1, k)
    assert fc.select_pages(query, bounds, table, lens, k, page_size=16, out=out).data_ptr() == out.data_ptr()
    assert out[0, 0, :4].tolist() == [0, 1, 2, 3]
    assert int(out[0, 0, 4:].amin()) == int(out[0, 0, 4:].amax()) == -1
    assert (around[:256] == 7).all() and (around[256 + k:] == 7).all()
    del out, around
    none = torch.zeros(2, dtype=torch.int32, device="cuda")       # a row behind the last sequence
    out = fc.select_pages(query, bounds, table, lens, k, page_size=16, starts=none)
    assert int(out.amin()) == int(out.amax()) == -1
    status_is(0)


@pytest.mark.parametrize("tokens", [1, 2, 9])         # sixteen CTAs a row, and a block of tokens
def test_attention_over_the_longest_list(tokens):
    """Entries from one end of the longest list to the other, nothing between them; one more entry is refused."""
    import flash_colsum_b200 as fc
    a = Batch(33, [tokens], [16 * 6], 16, 1, 1, 16, FP16)
    query, pools = a.rows(1), [a.pool(), a.pool()]
    pages = torch.full((a.T, 1, 2 ** 26), -1, dtype=torch.int32, device="cuda")
    short = torch.full((a.T, 1, 5), -1, dtype=torch.int32)
    for i, place in enumerate((0, 31, 2 ** 25 + 1, 2 ** 26 - 33, 2 ** 26 - 1)):
        short[:, 0, i] = i
        pages[:, :, place] = i
    want, lse, spread, reach = attention(query, *pools, a.table, a.lens, a.starts, short, 0.25)
    args = on_gpu(query, *pools, a.table, a.lens)
    out, got = fc.attend_pages(*args, pages, starts=a.starts.cuda(), return_lse=True)
    assert ((out.cpu().double() - want).abs() <= attend_room(FP16, 16, 80, want, spread, reach)).all()
    assert ((got.cpu().double() - lse).abs() <= 24 * 2.0 ** -23 * reach + 2.0 ** -18 + lse.abs() * 2.0 ** -22).all()
    status_is(0)
    with pytest.raises(ValueError, match="at most 67108864 entries"):
        fc.attend_pages(*args, pages[:, :, :1].expand(-1, -1, 2 ** 26 + 1), starts=a.starts.cuda())


# --------------------------------------------------------------------------- memory for results
def a_step(seed):
    a = Batch(seed, [3], [40], 16, 2, 4, 64, BF16)
    q, k, v, kp, vp, table, lens, starts = on_gpu(a.rows(4), a.rows(2), a.rows(2), a.pool(), a.pool(), a.table, a.lens, a.starts)
    return q, k, v, kp, vp, torch.stack([kp.amin(2), kp.amax(2)], 2), table, lens, starts


def test_results_in_memory_that_overlaps_are_refused():
    import flash_colsum_b200 as fc
    T, H, heads, D = 5, 2, 4, 64
    a = Batch(34, [T], [40], 16, H, heads, D, BF16)
    q, k, kp, vp, table, lens, starts = on_gpu(a.rows(heads), a.rows(H), a.pool(), a.pool(), a.table, a.lens, a.starts)
    pages = torch.zeros(T, H, 1, dtype=torch.int32, device="cuda")
    memory = torch.zeros(1 << 16, dtype=BF16, device="cuda")
    for stride in ((0, D), (heads * D, 0), (0, 0), (heads * D, D - 8), (heads * D - 8, D), (D, D), (D, T * D - 8), (8, 4 * D)):
        odd = memory.as_strided((T, heads, D), (*stride, 1))
        with pytest.raises(ValueError, match="query_out needs .* keep its rows apart"):
            fc.append_paged(k, k, kp, vp, table, lens, starts=starts, query=q, query_out=odd)
        with pytest.raises(ValueError, match="out needs .* keep its rows apart"):
            fc.attend_pages(q, kp, vp, table, lens, pages, starts=starts, out=odd)
    assert (memory == 0).all()
    status_is(0)


def test_pools_whose_rows_overlap_are_not_written():
    import flash_colsum_b200 as fc
    q, k, v, kp, vp, bounds, table, lens, starts = a_step(42)
    memory, (N, H, P, D) = torch.zeros(kp.numel(), dtype=BF16, device="cuda"), kp.shape
    for stride in ((D, D, D), (H * P * D, P * D, D - 8), (H * P * D, P * D - 8, D), (H * P * D - 8, P * D, D), (D, N * D, N * H * D - 8)):
        odd = memory.as_strided(kp.shape, (*stride, 1))
        for pools in ((odd, vp), (kp, odd)):
            with pytest.raises(ValueError, match="keep its rows apart"):
                fc.append_paged(k, v, *pools, table, lens, starts=starts)
    assert (memory == 0).all()
    want = fc.append_paged(k, v, kp, vp, table, lens, starts=starts, query=q, bounds=bounds)
    for order in ((0, 1, 2), (0, 2, 1), (2, 1, 0), (1, 0, 2), (2, 0, 1), (1, 2, 0)):      # the axes, outermost first
        some = [torch.zeros([kp.shape[i] + (n == 1) for n, i in enumerate(order)] + [D + 8], dtype=BF16, device="cuda")[:, :kp.shape[order[1]], :, :D]
                .permute(*(order.index(i) for i in range(3)), 3) for _ in range(2)]
        assert some[0].shape == kp.shape and some[0].stride() != kp.stride()
        assert torch.equal(fc.append_paged(k, v, *some, table, lens, starts=starts, query=q), want)
        for held, full in zip(some, (kp, vp)):
            for i in range(40 - 3, 40):
                page = int(table[0, i // P])
                assert torch.equal(held[page, :, i % P], full[page, :, i % P])
    status_is(0)


def test_results_in_any_memory_that_does_not():
    """Heads outside the tokens, gaps, one token or one head at any stride, and the queries' own memory."""
    import flash_colsum_b200 as fc
    for T, H, heads, D in ((5, 2, 4, 64), (1, 2, 4, 64), (40, 8, 8, 64), (5, 1, 1, 128), (1, 1, 1, 8)):
        a = Batch(35, [T], [T + 70], 16, H, heads, D, BF16)
        q, k, kp, vp, table, lens, starts = on_gpu(a.rows(heads), a.rows(H), a.pool(), a.pool(), a.table, a.lens, a.starts)
        pages = torch.arange(3, dtype=torch.int32, device="cuda").expand(T, H, 3)
        turn = torch.rand(T + 70, D // 2 // 8 * 8, device="cuda") if D >= 16 else None
        call = dict(starts=starts, query=q, cos=turn, sin=turn)
        turned = fc.append_paged(k, k, kp, vp, table, lens, **call)
        want = fc.attend_pages(turned, kp, vp, table, lens, pages, starts=starts)
        strides = [(D, T * D), (heads * D + 8, D), (heads * (D + 8), D + 8), (heads * D if T > 1 else 0, D if heads > 1 else 0)]
        for stride in strides:
            odd = torch.full((1 << 17,), 7.0, dtype=BF16, device="cuda").as_strided((T, heads, D), (*stride, 1))
            assert fc.append_paged(k, k, kp, vp, table, lens, **call, query_out=odd).data_ptr() == odd.data_ptr()
            assert torch.equal(odd, turned)
            assert torch.equal(fc.attend_pages(odd, kp, vp, table, lens, pages, starts=starts, out=odd), want)
    status_is(0)


def test_pools_that_share_their_memory_until_they_are_written():
    """A lazy copy of pools, bounds and results gets memory of its own when it is written, and only then."""
    import flash_colsum_b200 as fc
    q, k, v, kp, vp, bounds, table, lens, starts = a_step(36)
    first = [t.clone() for t in (kp, vp, bounds, q)]
    own = [t.clone() for t in (kp, vp, bounds)]
    want = fc.append_paged(k, v, own[0], own[1], table, lens, starts=starts, query=q, bounds=own[2])
    pages = fc.select_pages(want, own[2], table, lens, 2, page_size=16, starts=starts)
    out = fc.attend_pages(want, *own[:2], table, lens, pages, starts=starts)

    lazy = [torch._lazy_clone(t) for t in (kp, vp, bounds, q)]
    turned = fc.append_paged(k, v, lazy[0], lazy[1], table, lens, starts=starts, query=lazy[3], bounds=lazy[2], query_out=lazy[3])
    assert turned.data_ptr() == lazy[3].data_ptr() and torch.equal(turned, want)
    assert all(torch.equal(x, y) for x, y in zip(lazy, own))
    assert all(torch.equal(x, y) for x, y in zip((kp, vp, bounds, q), first))

    lazy = [torch._lazy_clone(t) for t in (*own, want, pages, out)]
    assert torch.equal(fc.select_pages(lazy[3], lazy[2], table, lens, 2, page_size=16, starts=starts), pages)
    assert torch.equal(fc.attend_pages(lazy[3], lazy[0], lazy[1], table, lens, lazy[4], starts=starts), out)
    assert all(torch._C._is_cow_tensor(t) for t in lazy)          # (they have been read)
    pages_out, attend_out = lazy[4], lazy[5]
    fc.select_pages(want, own[2], table, lens, 2, page_size=16, starts=torch.tensor([0, 1], dtype=torch.int32).cuda(), out=pages_out)
    fc.attend_pages(-want, *own[:2], table, lens, pages, starts=starts, out=attend_out)
    again = fc.select_pages(want, own[2], table, lens, 2, page_size=16, starts=starts)
    assert torch.equal(pages, again) and torch.equal(out, fc.attend_pages(want, *own[:2], table, lens, pages, starts=starts))
    assert not torch.equal(attend_out, out)
    # a call that is refused has not asked for memory
    lazy = [torch._lazy_clone(t) for t in (kp, vp, bounds)]
    with pytest.raises(ValueError):
        fc.append_paged(k, v[:2], lazy[0], lazy[1], table, lens, starts=starts, bounds=lazy[2])
    assert all(torch._C._is_cow_tensor(t) for t in lazy)
    status_is(0)


def test_autograd_sees_what_the_calls_write():
    import flash_colsum_b200 as fc
    q, k, v, kp, vp, bounds, table, lens, starts = a_step(37)
    pages = torch.zeros(3, 2, 2, dtype=torch.int32, device="cuda")
    out, turned = torch.zeros_like(q), torch.zeros_like(q)
    calls = [((kp, vp, bounds, turned), lambda: fc.append_paged(k, v, kp, vp, table, lens, starts=starts, query=q, bounds=bounds, query_out=turned)),
             ((pages,), lambda: fc.select_pages(q, bounds, table, lens, 2, page_size=16, starts=starts, out=pages)),
             ((out,), lambda: fc.attend_pages(q, kp, vp, table, lens, pages, starts=starts, out=out))]
    for changed, call in calls:
        before = [t._version for t in changed]
        others = [t for t in (q, k, v, kp, vp, bounds, pages, out, turned) if all(t is not c for c in changed)]
        kept = [t._version for t in others]
        call()
        assert all(t._version > n for t, n in zip(changed, before)) and [t._version for t in others] == kept
    weight = torch.ones_like(kp, requires_grad=True)
    loss = (weight * kp).sum()
    calls[0][1]()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        held = [t.clone() for t in (kp, vp, bounds)]
    fc.append_paged(k, v, held[0], held[1], table, lens, starts=starts, bounds=held[2])      # (tensors without a counter)
    assert torch.equal(held[0], kp) and torch.equal(held[2], bounds)
    status_is(0)


def c_cache(a, table, lens, starts, pools=()):
    """The batch (and contiguous pools) as the C entries take it; the tensors have to outlive it."""
    from flash_colsum_b200 import _cabi
    c = _cabi.PagedCache(page_table=table.data_ptr(), table_stride=table.stride(0), lens=lens.data_ptr(), starts=starts.data_ptr(),
                         pages=a.N, kv_heads=a.H, page_size=a.P, dim=a.dim, dtype=0 if a.dtype == FP16 else 1, sequences=lens.numel(),
                         table_width=table.shape[1], tokens=a.T)
    if pools:
        c.key_pages, c.value_pages = (p.data_ptr() for p in pools)
        c.key_stride = c.value_stride = pools[0].stride()[:3]
    return c


# --------------------------------------------------------------------------- sums in 64 bits
@pytest.mark.parametrize("tokens", [2, 20])           # a cluster a row, and tiles
@pytest.mark.parametrize("group,D,size", [(32, 128, 20.0), (8, 128, 80.0), (4, 64, 1500.0), (1, 64, 2.0 ** 15)])
def test_large_queries_of_half_precision_need_no_more_sums_than_others(tokens, group, D, size):
    """Parts whose magnitudes sum up to more than fp16 holds, each of them within its range: the 64-bit sums that the workspace has
    room for stay unwritten but for rows with many pages next to the border.  Parts past it: all are."""
    from flash_colsum_b200 import _cabi, ops
    pages, k = 500, 24
    a = Batch(38, [tokens], [16 * pages], 16, 1, group, D, FP16)
    query = a.rows(group)
    query = (query * (size / (1.0 if group > 1 else 4.0))).clamp(-60000, 60000)      # (one head: no part past 6e4)
    bounds = torch.stack([a.normal(a.N, 1, D) - 1, a.normal(a.N, 1, D) + 1], 2)
    assert query.float().abs().sum((1, 2)).amin() > 6e4 and query.float().abs().sum(1).amax() < 6e4
    lib = _cabi.load()
    for overflow in (False, True):
        if overflow:
            query[:, :, 0] = 60000.0 / min(group, 2) + 3000.0
        want = chosen_pages(query, bounds, 16, a.table, a.lens, a.starts, k, 1, 1)
        q, b, table, lens, starts = on_gpu(query, bounds, a.table, a.lens, a.starts)
        c = c_cache(a, table, lens, starts)
        room = torch.full((lib.fcs_select_pages_workspace_bytes(ctypes.byref(c)),), 0xab, dtype=torch.uint8, device="cuda")
        out = torch.empty(tokens, 1, k, dtype=torch.int32, device="cuda")
        stride = (ctypes.c_int64 * 2)(q.stride(0), q.stride(1))
        assert lib.fcs_select_pages(ctypes.byref(c), q.data_ptr(), stride, group, b.data_ptr(), k, 1, 1, out.data_ptr(), 1, room.data_ptr(),
                                    room.numel(), ops._status_word(out.device).data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(out.cpu(), want)
        sums = room[:8 * tokens * (pages + 4)].view(torch.int64)             # (a pitch of the next multiple of four)
        written = (sums != int.from_bytes(b"\xab" * 8, "little", signed=True)).sum().item()
        # (a token's competing pages: those it sees but the first and its own; 4 of 20 tokens lie in the last page but one)
        assert written == (sum(pos // 16 - 1 for _, _, pos in places(a.lens, a.starts, tokens)) if overflow else 0)
    status_is(0)


# --------------------------------------------------------------------------- lengths
@pytest.mark.parametrize("tokens", [1, 20])           # a row at a time, and blocks of tokens
@pytest.mark.parametrize("length", [-2 ** 31, -2 ** 31 + 4, -2 ** 31 + 19, -1, 0])
def test_tokens_in_front_of_a_sequence_see_nothing(tokens, length):
    """Lengths that count fewer tokens than there are rows, down to the lowest: no key is seen, no page chosen, nothing is written."""
    import flash_colsum_b200 as fc
    a = Batch(39, [tokens], [16 * 8], 16, 1, 1, 64, BF16)
    q, k, kp, vp, table, starts = on_gpu(a.rows(1), a.rows(1), a.pool(), a.pool(), a.table, a.starts)
    lens = torch.tensor([length], dtype=torch.int32, device="cuda")
    pages = torch.arange(8, dtype=torch.int32, device="cuda").expand(tokens, 1, 8)
    out, lse = fc.attend_pages(q, kp, vp, table, lens, pages, starts=starts, return_lse=True)
    assert (out == 0).all() and (lse == -torch.inf).all()
    bounds = torch.stack([kp.amin(2), kp.amax(2)], 2)
    assert (fc.select_pages(q, bounds, table, lens, 3, page_size=16, starts=starts) == -1).all()
    status_is(0)
    before = [t.clone() for t in (kp, vp, bounds)]
    fc.append_paged(k, k, kp, vp, table, lens, starts=starts, bounds=bounds)
    assert all(torch.equal(x, y) for x, y in zip(before, (kp, vp, bounds)))
    status_is(5)


# --------------------------------------------------------------------------- waits that run out
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rows,pages,H", [(1, 40, 2), (2, 1100, 1), (150, 70, 8)])     # one CTA a row, sixteen, and one with others beside it
def test_a_selection_whose_bounds_never_come_returns(rows, pages, H, D):
    """The barriers count an arrival that never comes and the limit is 50 ms: the waits run out, every CTA returns, the status word says so, what is written are
    pages of the sequences; and the same call chooses as before."""
    from flash_colsum_b200 import _cabi
    lib, k = _cabi.load(), 9
    a = Batch(40, [1] * rows, [16 * pages - i % 7 for i in range(rows)], 16, H, H, D, BF16)
    query = a.rows(H)
    bounds = torch.stack([a.normal(a.N, H, D) - 1, a.normal(a.N, H, D) + 1], 2)
    first = select(a, query, bounds, k, 1, 1)
    q, b, table, lens, starts = on_gpu(query, bounds, a.table, a.lens, a.starts)
    c = c_cache(a, table, lens, starts)
    room = torch.empty(lib.fcs_select_pages_workspace_bytes(ctypes.byref(c)), dtype=torch.uint8, device="cuda")
    around = torch.full((rows * H * k + 512,), 7, dtype=torch.int32, device="cuda")
    out, word = around[256:-256], torch.zeros(1, dtype=torch.int32, device="cuda")
    stride = (ctypes.c_int64 * 2)(q.stride(0), q.stride(1))
    assert lib.fcs_selftest_wait_expiry_select(ctypes.byref(c), q.data_ptr(), stride, H, b.data_ptr(), k, 1, 1, out.data_ptr(), room.data_ptr(),
                                               room.numel(), word.data_ptr(), 0.05, torch.cuda.current_stream().cuda_stream) == 0, _cabi.last_error()
    torch.cuda.synchronize()
    assert int(word) == 3                        # FCS_STATUS_WAIT_CONSUMER: a warp waits for what it asked for itself
    assert int(out.amin()) >= -1 and int(out.amax()) < pages
    assert (around[:256] == 7).all() and (around[-256:] == 7).all()
    assert torch.equal(select(a, query, bounds, k, 1, 1), first)
    status_is(0)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("tokens,H,k,twice", [(1, 1, 2, False), (1, 1, 300, False), (300, 1, 3, False), (40, 1, 7, False), (40, 1, 7, True),
                                              (40, 100, 7, True)])
def test_an_attention_whose_pages_never_come_returns(tokens, H, k, twice, D):
    """A row at a time over one CTA and sixteen, blocks of tokens over eight and two, also where a list names a page twice and every
    token has a pass of its own: zeros and -inf, and a status; and the same call attends as before."""
    import flash_colsum_b200 as fc
    from flash_colsum_b200 import _cabi
    lib = _cabi.load()
    many = tokens == 300                          # sequences of one token
    a = Batch(41, [1] * tokens if many else [tokens], [16 * 20 + tokens] * (tokens if many else 1), 16, H, H, D, BF16, width=400)
    query, kp, vp, table, lens, starts = on_gpu(a.rows(H), a.pool(), a.pool(), a.table, a.lens, a.starts)
    pages = torch.randperm(20, generator=a.g).int()[torch.arange(k) % 20].expand(a.T, H, k).contiguous().cuda()
    if twice:
        pages[:, :, 0] = pages[:, :, 1]
    first = fc.attend_pages(query, kp, vp, table, lens, pages, starts=starts, return_lse=True)
    c = c_cache(a, table, lens, starts, (kp, vp))
    out, lse = torch.full_like(query, 7.0), torch.full((a.T, H), 7.0, device="cuda")
    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    stride = (ctypes.c_int64 * 2)(query.stride(0), query.stride(1))
    assert lib.fcs_selftest_wait_expiry_attend(ctypes.byref(c), query.data_ptr(), stride, H, pages.data_ptr(), k, 0.1, out.data_ptr(), stride,
                                               lse.data_ptr(), word.data_ptr(), 0.05, torch.cuda.current_stream().cuda_stream) == 0, _cabi.last_error()
    torch.cuda.synchronize()
    assert int(word) in (1, 3)                   # (the producer waits for tiles to become free)
    assert (out == 0).all() and (lse == -torch.inf).all()
    again = fc.attend_pages(query, kp, vp, table, lens, pages, starts=starts, return_lse=True)
    assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])
    status_is(0)


# --------------------------------------------------------------------------- bounds
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,H", [(64, 2), (128, 9)])
def test_bounds_of_a_page_whose_slot_0_is_left_out(D, H, interleaved):
    """A token whose position the rotation lacks is not written: where it is the first of a page, the page keeps what it had."""
    import flash_colsum_b200 as fc
    T, P = 48, 16
    a = Batch(43, [T], [T], P, H, H, D, BF16)
    key, pools = a.rows(H), [a.pool(), a.pool()]
    bounds = torch.stack([pools[0].amin(2), pools[0].amax(2)], 2)
    cos, sin = torch.ones(100, D // 2), torch.zeros(100, D // 2)              # (rotated by nothing: keys are stored as they are)
    positions = torch.arange(T, dtype=torch.int32)
    positions[16], positions[32:], positions[3] = 100, -1, -7                 # a page's first token, a page's tokens, one further in
    d = on_gpu(key, key, *pools, a.table, a.lens, a.starts, cos, sin, positions, bounds)
    fc.append_paged(*d[:6], starts=d[6], cos=d[7], sin=d[8], positions=d[9], bounds=d[10], interleaved=interleaved)
    status_is(6)
    want = bounds.clone()
    written = key[[i for i in range(16) if i != 3]], key[17:32]
    at = a.table[0].tolist()
    want[at[0]] = torch.stack([written[0].amin(0), written[0].amax(0)], 1)
    want[at[1]] = torch.stack([torch.minimum(written[1].amin(0), bounds[at[1], :, 0]), torch.maximum(written[1].amax(0), bounds[at[1], :, 1])], 1)
    assert torch.equal(d[10].cpu(), want)
