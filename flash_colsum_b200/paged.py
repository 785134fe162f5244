"""A cache of keys and values in pages, and the attention that reads the part of it that matters.

    lens += 1                                                       # (B,) tokens cached, this step's included
    q = append_paged(k, v, key_pages, value_pages, table, lens, query=q, cos=cos, sin=sin, bounds=bounds)
    pages = select_pages(q, bounds, table, lens, 32, page_size=64)  # per token and key/value head
    out = attend_pages(q, key_pages, value_pages, table, lens, pages)

What :func:`flash_colsum` and :func:`topk_columns` do once for a prompt -- find the keys that draw the
attention and keep those -- this does for every query of a cache that keeps all.  The reference has no
counterpart.

The three calls share a batch: ``page_table`` (B, W) int32, whose row b lists the pages of sequence b;
``lens`` (B,) int32, the tokens of every sequence in the cache with this call's included; and ``starts``
(B + 1,) int32, ascending from 0: rows ``starts[b]`` to ``starts[b + 1]`` of the packed tokens are the last tokens of
sequence b.  Without ``starts`` there is one token a sequence.  Rows behind ``starts[B]`` belong to nobody:
nothing is read from them, and results that a call makes are 0 there (pages -1, log-sums -inf); where the
caller gives the result's memory they are left as they are.  All three are read on the device, in
stream order, so that a captured call follows them.

The pools are (N, H_kv, P, D) fp16 or bf16 tensors, P 16, 32, 64 or 128 and D a multiple of 8 up to 128,
with unit inner stride and any order of the others in multiples of 8 elements -- the two halves of one
(N, 2, H_kv, P, D) tensor, or a (N, P, H_kv, D) one seen through ``transpose(1, 2)``.  They are written and read in place, and count
as changed in place for autograd; there is no gradient.  A page that a token needs and the table does not have is neither written nor
read, and :func:`device_status` says so (5); a position that the rotation's tables do not have, likewise (6).

Calls run on the current stream of the tensors' device without synchronising.
"""

from __future__ import annotations

import operator
from typing import Optional, Tuple, Union

import torch

from . import ops

_TYPES = (torch.float16, torch.bfloat16)
_PAGE_SIZES = (16, 32, 64, 128)
_LIST_MAX = 1 << 26          # FCS_LIST_MAX


def _rows_ready(t: torch.Tensor) -> bool:
    """Unit inner stride, the others multiples of 16 bytes, 16-byte aligned base."""
    outer = [s for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1]
    return ((t.shape[-1] == 1 or t.stride(-1) == 1) and all(s >= 0 and s % 8 == 0 for s in outer)
            and t.data_ptr() % 16 == 0)


def _check_rows(name: str, t: torch.Tensor) -> None:
    if t.ndim != 3:
        raise ValueError(f"{name} must be (tokens, heads, head_dim), got {tuple(t.shape)}")
    if t.device.type != "cuda":
        raise ValueError(f"{name} must be a CUDA tensor, got {t.device}")
    if t.dtype not in _TYPES:
        raise ValueError(f"{name} must be float16 or bfloat16, got {t.dtype}")
    if t.shape[2] % 8 or not 8 <= t.shape[2] <= 128:
        raise ValueError(f"head_dim must be a multiple of 8 from 8 to 128, got {t.shape[2]}")


def _rows_apart(t: torch.Tensor) -> bool:
    """Whether no row has an element in common with another: every stride holds what the shorter ones span."""
    span = t.shape[-1]
    for s, n in sorted(zip(t.stride()[:-1], t.shape[:-1])):
        if n > 1:
            if s < span:
                return False
            span += s * (n - 1)
    return True


def _check_result(name: str, t: torch.Tensor) -> None:
    if not _rows_ready(t) or not _rows_apart(t):
        raise ValueError(f"{name} needs unit inner stride, other strides in multiples of 8 elements that keep its rows apart, and a "
                         f"16-byte aligned base, got strides {t.stride()}")


def _check_like(name: str, t: torch.Tensor, rows: torch.Tensor, shape) -> None:
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be {tuple(shape)}, got {tuple(t.shape)}")
    if t.dtype != rows.dtype or t.device != rows.device:
        raise ValueError(f"{name} must be {rows.dtype} on {rows.device}, got {t.dtype} on {t.device}")


def _check_indices(name: str, t: torch.Tensor, rows: torch.Tensor, ndim: int) -> None:
    if t.ndim != ndim or t.dtype != torch.int32 or t.device != rows.device:
        raise ValueError(f"{name} must be a {ndim}-D int32 tensor on {rows.device}, got {tuple(t.shape)} {t.dtype} on {t.device}")


def _check_batch(rows: torch.Tensor, page_table: torch.Tensor, lens: torch.Tensor, starts: Optional[torch.Tensor]) -> None:
    _check_indices("page_table", page_table, rows, 2)
    _check_indices("lens", lens, rows, 1)
    B = lens.shape[0]
    if page_table.shape[0] != B or page_table.shape[1] == 0:
        raise ValueError(f"page_table must have a row of at least one page for each of {B} sequences, got {tuple(page_table.shape)}")
    if starts is None:
        if rows.shape[0] != B:
            raise ValueError(f"without starts there is one token a sequence, got {rows.shape[0]} tokens and {B} sequences")
    else:
        _check_indices("starts", starts, rows, 1)
        if starts.shape[0] != B + 1:
            raise ValueError(f"starts must have {B + 1} entries for {B} sequences, got {starts.shape[0]}")
    if B == 0 and rows.shape[0] > 0:
        raise ValueError("there are tokens and no sequence")


def _check_pools(rows: torch.Tensor, key_pages: torch.Tensor, value_pages: torch.Tensor, written: bool) -> None:
    if key_pages.ndim != 4 or key_pages.shape != value_pages.shape:
        raise ValueError(f"key_pages and value_pages must be (pages, kv_heads, page_size, head_dim) of one shape, got "
                         f"{tuple(key_pages.shape)} and {tuple(value_pages.shape)}")
    N, H, P, D = key_pages.shape
    if N == 0 or H == 0:
        raise ValueError("the pools are empty")
    if P not in _PAGE_SIZES:
        raise ValueError(f"page size must be 16, 32, 64 or 128, got {P}")
    if D != rows.shape[2]:
        raise ValueError(f"the pools hold heads of {D} features, the tokens have {rows.shape[2]}")
    for name, t in (("key_pages", key_pages), ("value_pages", value_pages)):
        if t.dtype != rows.dtype or t.device != rows.device:
            raise ValueError(f"{name} must be {rows.dtype} on {rows.device}, got {t.dtype} on {t.device}")
        if not _rows_ready(t) or any(s < D for s, n in zip(t.stride()[:3], t.shape[:3]) if n > 1) or (written and not _rows_apart(t)):
            raise ValueError(f"{name} needs unit inner stride, other strides in multiples of 8 elements that keep its rows "
                             f"apart, and a 16-byte aligned base, got strides {t.stride()}")


def _check_heads(name: str, heads: int, kv_heads: int) -> None:
    if heads == 0 or heads % kv_heads:
        raise ValueError(f"the heads of {name} must be a multiple of the {kv_heads} key/value heads, got {heads}")


def _native(device: torch.device):
    return ops._native if ops._native is not None and ops._status.get(device.index) is not None else ops._load_native(device)


def _refused(name: str) -> ValueError:
    return ValueError(f"{name}: unsupported operands")


def append_paged(
    key: torch.Tensor,
    value: torch.Tensor,
    key_pages: torch.Tensor,
    value_pages: torch.Tensor,
    page_table: torch.Tensor,
    lens: torch.Tensor,
    *,
    starts: Optional[torch.Tensor] = None,
    query: Optional[torch.Tensor] = None,
    cos: Optional[torch.Tensor] = None,
    sin: Optional[torch.Tensor] = None,
    positions: Optional[torch.Tensor] = None,
    interleaved: bool = False,
    bounds: Optional[torch.Tensor] = None,
    query_out: Optional[torch.Tensor] = None,
) -> Optional[torch.Tensor]:
    """Write a step's keys and values into their pages, the keys rotated by their positions.

    Args:
        key, value: (T, H_kv, D), the packed new tokens.
        key_pages, value_pages: the pools, written in place.
        page_table, lens, starts: the batch (see the module).
        query: (T, H_q, D), rotated like the keys; H_q a multiple of H_kv.
        cos, sin: (M, R / 2) fp32, contiguous: the first R features (a multiple of 16) of keys and queries are
            rotated, feature i with feature i + R / 2, by row m of the tables for the token at position m.  Without them
            nothing is rotated.
        positions: (T,) int32, the rows of ``cos`` and ``sin`` where those are not the places in the cache -- tokens
            kept out of a pruned prompt, say.
        interleaved: rotate feature 2 i with feature 2 i + 1 instead.
        bounds: (N, H_kv, 2, D) of the pools' type, contiguous: per page and head the smallest and the largest value of every
            feature, over the (rotated) keys written since the page's slot 0 was; kept up to date in place.
        query_out: memory for the rotated queries, whose rows do not overlap; may be ``query``.

    Returns:
        The rotated queries (T, H_q, D), or None without ``query``.
    """
    if ops._native is not None:
        out = ops._native.append_paged(key, value, key_pages, value_pages, page_table, lens, starts, query, cos, sin, positions,
                                       interleaved, bounds, query_out)
        if out is not None:
            return None if out is True else out
    _check_rows("key", key)
    _check_like("value", value, key, key.shape)
    _check_batch(key, page_table, lens, starts)
    _check_pools(key, key_pages, value_pages, True)
    N, H, _, D = key_pages.shape
    if key.shape[1] != H:
        raise ValueError(f"the pools hold {H} heads, key has {key.shape[1]}")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin go together")
    if cos is None and positions is not None:
        raise ValueError("positions are of no use without cos and sin")
    if cos is not None:
        for name, t in (("cos", cos), ("sin", sin)):
            if t.ndim != 2 or t.dtype != torch.float32 or t.device != key.device or not t.is_contiguous() or t.data_ptr() % 16:
                raise ValueError(f"{name} must be a contiguous 2-D float32 tensor on {key.device} with a 16-byte aligned base")
        if cos.shape != sin.shape or cos.shape[0] == 0 or cos.shape[1] % 8 or not 8 <= cos.shape[1] <= D // 2:
            raise ValueError(f"cos and sin must be of one shape, with rows for half of 16, 32, ... up to {D} features, got "
                             f"{tuple(cos.shape)} and {tuple(sin.shape)}")
        if positions is not None:
            _check_indices("positions", positions, key, 1)
            if positions.shape[0] != key.shape[0]:
                raise ValueError(f"positions must have an entry for each of {key.shape[0]} tokens, got {positions.shape[0]}")
    if bounds is not None:
        _check_like("bounds", bounds, key, (N, H, 2, D))
        if not bounds.is_contiguous() or bounds.data_ptr() % 16:
            raise ValueError("bounds must be contiguous, with a 16-byte aligned base")
    if query is None:
        if query_out is not None:
            raise ValueError("query_out is of no use without query")
    else:
        _check_rows("query", query)
        _check_heads("query", query.shape[1], H)
        _check_like("query", query, key, (key.shape[0], query.shape[1], D))
        if query_out is not None:
            _check_like("query_out", query_out, query, query.shape)
            _check_result("query_out", query_out)
    if key.shape[0] == 0:
        return query_out if query is None or query_out is not None else torch.empty_like(query, memory_format=torch.contiguous_format)
    out = _native(key.device).append_paged(key, value, key_pages, value_pages, page_table, lens, starts, query, cos, sin, positions,
                                           bool(interleaved), bounds, query_out)
    if out is None:
        raise _refused("append_paged")
    return None if out is True else out


def select_pages(
    query: torch.Tensor,
    bounds: torch.Tensor,
    page_table: torch.Tensor,
    lens: torch.Tensor,
    k: int,
    *,
    page_size: int,
    starts: Optional[torch.Tensor] = None,
    first: int = 1,
    last: int = 1,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """The ``k`` pages that every query attends to, per key/value head.

    Args:
        query: (T, H_q, D), rotated; the H_q / H_kv queries of a group choose together.
        bounds: (N, H_kv, 2, D), as :func:`append_paged` keeps them.
        page_table, lens, starts: the batch (see the module).
        k: pages to choose.
        page_size: tokens of a page.
        first, last: this many pages from the beginning, and up to the token's own (which is counted, ``last`` >= 1), are
            always chosen; first + last <= k.
        out: (T, H_kv, k) int32, contiguous, for the result.

    Returns:
        (T, H_kv, k) int32: places in the sequence's row of the table, ascending, -1 behind the last where
        the token sees fewer than k pages.  Of the pages that are not forced the best are those with the largest sum
        over the group of ``sum_d max(q_d low_d, q_d high_d)`` -- no less than the sum of the group's scores with any key of the
        page; ties go to the lower page and NaN counts as infinity.
    """
    if ops._native is not None:
        res = ops._native.select_pages(query, bounds, page_table, lens, k, page_size, starts, first, last, out)
        if res is not None:
            return res
    _check_rows("query", query)
    _check_batch(query, page_table, lens, starts)
    k, page_size, first, last = (operator.index(n) for n in (k, page_size, first, last))
    if bounds.ndim != 4 or bounds.shape[0] == 0 or bounds.shape[1] == 0:
        raise ValueError(f"bounds must be (pages, kv_heads, 2, head_dim), got {tuple(bounds.shape)}")
    _check_like("bounds", bounds, query, (bounds.shape[0], bounds.shape[1], 2, query.shape[2]))
    if not bounds.is_contiguous() or bounds.data_ptr() % 16:
        raise ValueError("bounds must be contiguous, with a 16-byte aligned base")
    _check_heads("query", query.shape[1], bounds.shape[1])
    if page_size not in _PAGE_SIZES:
        raise ValueError(f"page size must be 16, 32, 64 or 128, got {page_size}")
    if first < 0 or last < 1:
        raise ValueError(f"first must not be negative and last be at least 1, got {first} and {last}")
    if k < first + last:
        raise ValueError(f"k must hold the {first} first and {last} last pages, got {k}")
    shape = (query.shape[0], bounds.shape[1], k)
    if out is not None:
        _check_indices("out", out, query, 3)
        if tuple(out.shape) != shape or not out.is_contiguous():
            raise ValueError(f"out must be a contiguous tensor of shape {shape}, got {tuple(out.shape)}")
    if query.shape[0] == 0:
        return out if out is not None else torch.empty(shape, dtype=torch.int32, device=query.device)
    res = _native(query.device).select_pages(query, bounds, page_table, lens, k, page_size, starts, first, last, out)
    if res is None:
        raise _refused("select_pages")
    return res


def attend_pages(
    query: torch.Tensor,
    key_pages: torch.Tensor,
    value_pages: torch.Tensor,
    page_table: torch.Tensor,
    lens: torch.Tensor,
    pages: torch.Tensor,
    *,
    starts: Optional[torch.Tensor] = None,
    scale: Optional[float] = None,
    return_lse: bool = False,
    out: Optional[torch.Tensor] = None,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Softmax attention of every query over the keys of its pages, up to its own position.

    Args:
        query: (T, H_q, D), rotated.
        key_pages, value_pages: the pools, H_q a multiple of their heads.
        page_table, lens, starts: the batch (see the module).
        pages: (T, H_kv, k) int32, places in the sequence's row of the table, as :func:`select_pages` gives them
            but in any order; negative entries and pages behind the token's own weigh nothing, a page that is
            listed twice weighs twice.  At most 2 ** 26 of them.
        scale: score scale, default 1/sqrt(D).
        return_lse: return the natural logarithms of the sums of exp(score) too, for joining the result with
            that of other keys.
        out: (T, H_q, D) of the pools' type, for the result; its rows do not overlap.  May be ``query``.

    Returns:
        (T, H_q, D), and with ``return_lse`` (T, H_q) fp32.  A query that sees no key gets zeros and -inf.
    """
    if ops._native is not None:
        res = ops._native.attend_pages(query, key_pages, value_pages, page_table, lens, pages, starts, scale, return_lse, out)
        if res is not None:
            return res
    _check_rows("query", query)
    _check_batch(query, page_table, lens, starts)
    _check_pools(query, key_pages, value_pages, False)
    _check_heads("query", query.shape[1], key_pages.shape[1])
    _check_indices("pages", pages, query, 3)
    if tuple(pages.shape[:2]) != (query.shape[0], key_pages.shape[1]) or pages.shape[2] == 0:
        raise ValueError(f"pages must be ({query.shape[0]}, {key_pages.shape[1]}, k) with k >= 1, got {tuple(pages.shape)}")
    if pages.shape[2] > _LIST_MAX:
        raise ValueError(f"pages must have at most {_LIST_MAX} entries a list, got {pages.shape[2]}")
    if scale is not None and scale != scale:
        raise ValueError("scale is not a number")
    if out is not None:
        _check_like("out", out, query, query.shape)
        _check_result("out", out)
    if query.shape[0] == 0:
        res = out if out is not None else torch.empty_like(query, memory_format=torch.contiguous_format)
        return (res, torch.empty(query.shape[:2], dtype=torch.float32, device=query.device)) if return_lse else res
    res = _native(query.device).attend_pages(query, key_pages, value_pages, page_table, lens, pages, starts, scale,
                                             bool(return_lse), out)
    if res is None:
        raise _refused("attend_pages")
    return res


__all__ = ["append_paged", "select_pages", "attend_pages"]
