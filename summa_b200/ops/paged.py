"""The paged key/value cache: what describes it, the checks of the calls that use it, and their PyTorch form.

A layer's cache is a pool of pages `[num_pages, Hkv, page, D]` for the keys and one for the values (`PagedKV`); a batch says which
pages hold which sequence (`PagedRows`). Sequences of one call differ in length and in the rows they bring, and a slot of the batch
may be out of use. Pages are of the model's type, or e4m3 with one scale per page and head.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch

E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
LEAST_EXPONENT, MOST_EXPONENT = -60, 120
PAGE_SIZES = (16, 32, 64, 128)


class PagedKV(NamedTuple):
    """One layer's pages `[num_pages, Hkv, page, D]`. e4m3 pages come with `[num_pages, Hkv]` fp32 scales: an element is its code
    times the scale of its page and head, a power of two between 2^-60 and 2^120. A page needs no initial value: what its first
    slot is written with begins its scale."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: Optional[torch.Tensor] = None
    v_scale: Optional[torch.Tensor] = None


class PagedRows(NamedTuple):
    """The sequences of a call. `table` `[B, P]` int32: the pages of each, in order (entries that no position of it needs may hold
    anything). `lengths` `[B]` int32: the tokens it had in the cache before the call, negative for a slot that is not in use.
    `starts` `[B + 1]` int32, ascending from 0: sequence b has the rows starts[b] .. starts[b + 1] of the call, and rows behind the last
    belong to nobody; None: one row each. `max_rows`: the most rows of one sequence, which the launch is shaped for (None: the rows of the
    call); rows beyond it may be left out, and what is left out is reported in the error word."""
    table: torch.Tensor
    lengths: torch.Tensor
    starts: Optional[torch.Tensor] = None
    max_rows: Optional[int] = None

    def most(self, total: int) -> int:
        return 1 if self.starts is None else total if self.max_rows is None else min(int(self.max_rows), total)


# (The checks run in front of every launch of a decoding step: a message is only put together where one fails, and what they look up
# is handed on.)

class Layout(NamedTuple):
    """What a launch needs to know of the tensors, in its order: sizes, then strides in elements."""
    sequences: int
    table_pages: int
    page: int
    num_pages: int
    table_ld: int
    k_page: int
    k_head: int
    v_page: int
    v_head: int
    k_scale_ld: int
    v_scale_ld: int


def check(x: torch.Tensor, Hkv: int, D: int, kv: PagedKV, rows: PagedRows) -> Layout:
    """The checks that both calls share; `x` is what has a row per token."""
    k, v, k_scale, v_scale = kv
    table, lengths, starts, max_rows = rows
    dtype, device, shape = k.dtype, x.device, k.shape
    if len(shape) != 4 or v.shape != shape or v.dtype != dtype:
        raise ValueError("the pages of keys and values differ in shape or type, or are not [num_pages, Hkv, page, D]")
    pages, heads, page, d = shape
    if heads != Hkv or d != D:
        raise ValueError(f"pages of {heads} heads of {d}, and rows of {Hkv} heads of {D}")
    if page not in PAGE_SIZES:
        raise ValueError(f"page size {page}: one of {PAGE_SIZES}")
    k_page, k_head, k_row, k_one = k.stride()
    v_page, v_head, v_row, v_one = v.stride()
    if k_one != 1 or v_one != 1 or k_row != D or v_row != D or k.device != device or v.device != device:
        raise ValueError("the rows of a page and head have to lie together, on the device of the rows of the call")
    ks_ld = vs_ld = 0
    if dtype == E4M3:
        unit = 16
        if (k_scale is None or v_scale is None or k_scale.dtype != torch.float32 or v_scale.dtype != torch.float32
                or k_scale.shape != (pages, heads) or v_scale.shape != (pages, heads) or k_scale.device != device or v_scale.device != device):
            raise ValueError(f"e4m3 pages need fp32 scales [{pages}, {heads}] on the device of the rows")
        ks_ld, one = k_scale.stride()
        vs_ld, two = v_scale.stride()
        if one != 1 or two != 1:
            raise ValueError("the scales of a page's heads have to lie together")
    else:
        unit = 8
        if dtype != x.dtype or k_scale is not None or v_scale is not None:
            raise ValueError(f"pages of {dtype} for rows of {x.dtype}: of the same type without scales, or e4m3 with them")
    if x.is_cuda and (k.data_ptr() % 16 or v.data_ptr() % 16 or (k_page | k_head | v_page | v_head) % unit):
        raise ValueError("pages and heads have to begin on 16 bytes")
    if table.dim() != 2 or table.dtype != torch.int32 or table.device != device:
        raise ValueError("table: int32 [B, P] on the device of the rows")
    B, P = table.shape
    table_ld, one = table.stride()
    if one != 1:
        raise ValueError("the pages of a sequence in the table have to lie together")
    if lengths.dtype != torch.int32 or lengths.shape != (B,) or not lengths.is_contiguous() or lengths.device != device:
        raise ValueError(f"lengths: int32 [{B}] on the device of the rows")
    if starts is None:
        if x.shape[0] != B:
            raise ValueError(f"{x.shape[0]} rows for {B} sequences without starts")
    elif starts.dtype != torch.int32 or starts.shape != (B + 1,) or not starts.is_contiguous() or starts.device != device:
        raise ValueError(f"starts: int32 [{B + 1}] on the device of the rows")
    if x.shape[0] > 0 and not (B and P and pages):
        raise ValueError(f"{x.shape[0]} rows, and a table [{B}, {P}] over {pages} pages")
    if max_rows is not None and max_rows < 1:
        raise ValueError(f"max_rows {max_rows}")
    return Layout(B, P, page, pages, table_ld, k_page, k_head, v_page, v_head, ks_ld, vs_ld)


def check_out(out, shape, x) -> None:
    if out is None:
        return
    if out.shape != shape or out.dtype != x.dtype or out.device != x.device:
        raise ValueError(f"out: {list(shape)} of the type and device of the rows")
    if any(step == 0 and n > 1 for step, n in zip(out.stride(), out.shape)):
        raise ValueError("several elements of out are one in memory")


def check_append(qkv, q_gamma, k_gamma, cos, sin, Hq, Hkv, D, kv, rows, out) -> Layout:
    device = qkv.device
    if qkv.dim() != 2 or Hq < 1 or Hkv < 1 or qkv.shape[1] != (Hq + 2 * Hkv) * D:
        raise ValueError(f"qkv: [T, ({Hq} + 2 * {Hkv}) * {D}], got {list(qkv.shape)}")
    if (q_gamma is None) != (k_gamma is None) or (cos is None) != (sin is None):
        raise ValueError("q_gamma and k_gamma, cos and sin come in pairs")
    if q_gamma is not None and not (q_gamma.shape == k_gamma.shape == (D,) and q_gamma.device == k_gamma.device == device):
        raise ValueError(f"gains of a head: [{D}], on the device of the rows")
    if cos is not None:
        shape = cos.shape
        if (len(shape) != 2 or shape[1] != D // 2 or sin.shape != shape or cos.dtype != torch.float32 or sin.dtype != torch.float32
                or not cos.is_contiguous() or not sin.is_contiguous() or cos.device != device or sin.device != device):
            raise ValueError(f"cos, sin: fp32 [positions, {D // 2}], contiguous and on the device of the rows")
        if cos.is_cuda and (cos.data_ptr() % 16 or sin.data_ptr() % 16):
            raise ValueError("cos and sin have to begin on 16 bytes")
        if cos.shape[0] < 1:
            raise ValueError("cos, sin: no position")
    check_out(out, (qkv.shape[0], Hq, D), qkv)
    return check(qkv, Hkv, D, kv, rows)


def check_attention(q, kv, rows, window, scale, out) -> Layout:
    if q.dim() != 3 or kv.k.dim() != 4:
        raise ValueError("q: [T, Hq, D]; pages: [num_pages, Hkv, page, D]")
    _, Hq, D = q.shape
    Hkv = kv.k.shape[1]
    if Hq < 1 or Hkv < 1 or Hq % Hkv:
        raise ValueError(f"{Hq} query heads over {Hkv} kv heads")
    if window is not None and window < 0:
        raise ValueError(f"window {window}")
    if scale is not None and not 0.0 < scale < math.inf:
        raise ValueError(f"scale {scale}: it has to be positive")
    check_out(out, q.shape, q)
    return check(q, Hkv, D, kv, rows)


# ------------------------------------------------------------------ PyTorch form (CPU tensors)

def _sequences(total: int, rows: PagedRows):
    """(b, first row, rows, length) of each sequence that brings rows."""
    at = list(range(rows.table.shape[0] + 1)) if rows.starts is None else rows.starts.tolist()
    for b, length in enumerate(rows.lengths.tolist()):
        first, last = min(max(at[b], 0), total), min(max(at[b + 1], 0), total)
        if last > first:
            yield b, first, last - first, length


def _pages(kv: PagedKV, rows: PagedRows, b: int, begin: int, end: int):
    """Page numbers of positions [begin, end) of sequence b."""
    page = kv.k.shape[2]
    ids = rows.table[b, begin // page:-(-end // page)].tolist()
    if len(ids) < -(-end // page) - begin // page or any(not 0 <= i < kv.k.shape[0] for i in ids):
        raise RuntimeError(f"sequence {b} has no page for its positions {begin} .. {end - 1}")
    return ids


def _scale_of(most: torch.Tensor) -> torch.Tensor:
    """The smallest power of two s in the range with most <= 448 s, elementwise."""
    m, e = torch.frexp(most.double() / E4M3_MAX)
    e = torch.where(most > 0, torch.where(m > 0.5, e, e - 1), LEAST_EXPONENT).clamp(LEAST_EXPONENT, MOST_EXPONENT)
    return torch.exp2(e.double()).float()


def to_e4m3(x: torch.Tensor) -> torch.Tensor:
    """fp32 -> e4m3; what is not finite becomes NaN."""
    return torch.where(torch.isfinite(x), x, float("nan")).to(E4M3)


def _store(pages, scale, x, at: int, slot: int) -> None:
    """x `[n, Hkv, D]` (fp32) into page `at` from `slot` on."""
    n = x.shape[0]
    x = x.transpose(0, 1)
    if scale is None:
        pages[at, :, slot:slot + n] = x.to(pages.dtype)
        return
    new = _scale_of(torch.where(torch.isfinite(x), x.abs(), 0).amax((1, 2)))
    if slot > 0:
        old = scale[at].clone()
        new = torch.maximum(new, old)
        pages[at, :, :slot] = (pages[at, :, :slot].float() * (old / new)[:, None, None]).to(E4M3)
    scale[at] = new
    pages[at, :, slot:slot + n] = to_e4m3(x / new[:, None, None])


def append_reference(qkv, q_gamma, k_gamma, eps, cos, sin, Hq, Hkv, D, kv, rows, out=None):
    q = torch.zeros(qkv.shape[0], Hq, D, dtype=qkv.dtype, device=qkv.device) if out is None else out
    page = kv.k.shape[2]
    x = qkv.unflatten(1, (-1, D)).float()

    def turn(y, gamma, pos):
        if gamma is not None:
            y = y * torch.rsqrt(y.pow(2).mean(-1, keepdim=True) + eps) * gamma.float()
        if cos is not None:
            c, s = cos[pos:pos + y.shape[0], None], sin[pos:pos + y.shape[0], None]
            a, b = y[..., 0::2], y[..., 1::2]
            y = torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)
        return y

    for b, first, n, length in _sequences(qkv.shape[0], rows):
        if length < 0:
            q[first:first + n] = 0
            continue
        if cos is not None and length + n > cos.shape[0]:
            raise RuntimeError(f"position {length + n - 1} of sequence {b} is beyond the rotation's table of {cos.shape[0]}")
        ids = _pages(kv, rows, b, length, length + n)
        mine = x[first:first + n]
        q[first:first + n] = turn(mine[:, :Hq], q_gamma, length).to(qkv.dtype)
        k, v = turn(mine[:, Hq:Hq + Hkv], k_gamma, length), mine[:, Hq + Hkv:]
        done = 0
        for at in ids:
            slot = (length + done) % page
            m = min(page - slot, n - done)
            _store(kv.k, kv.k_scale, k[done:done + m], at, slot)
            _store(kv.v, kv.v_scale, v[done:done + m], at, slot)
            done += m
    return q


def read(kv: PagedKV, ids, lo: int, hi: int):
    """Keys and values `[hi - lo, Hkv, D]` in fp32 of positions [lo, hi) behind the first of the pages `ids`."""
    out = []
    for pages, scale in ((kv.k, kv.k_scale), (kv.v, kv.v_scale)):
        x = pages[ids].float()
        if scale is not None:
            x = x * scale[ids][..., None, None]
        out.append(x.transpose(1, 2).flatten(0, 1)[lo:hi])
    return out


def attention_reference(q, kv, rows, causal=True, window=None, scale=None, out=None):
    from . import reference
    o = torch.zeros_like(q, memory_format=torch.contiguous_format) if out is None else out
    page = kv.k.shape[2]
    scale = scale if scale is not None else 1.0 / math.sqrt(q.shape[2])
    for b, first, n, length in _sequences(q.shape[0], rows):
        if length < 0:
            o[first:first + n] = 0
            continue
        lo = 0 if window is None else max(length - window, 0)
        ids = _pages(kv, rows, b, lo, length + n)
        base = lo // page * page
        k, v = read(kv, ids, lo - base, length + n - base)
        y = reference.attention(q[None, first:first + n].float(), k[None], v[None], causal, window, scale, length - lo)
        o[first:first + n] = y[0].to(q.dtype)
    return o
