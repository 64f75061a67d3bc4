"""A paged key/value cache on the GPU: storing new tokens, and attention.

What an interactive session holds between two bursts is its key/value
cache: it is what the interposer pages out while the client thinks and
back when it goes on.  This module has the two operators of a step over
such a cache, as gfx950 kernels (hip/kvcache.hip):

    cache = PagedCache.empty(pages, page_size, kv_heads, dim, device="cuda")
    rotation = rotation_table(per_seq * page_size, dim, device="cuda")
    ...
    lens += new                       # each sequence's tokens, new ones in
    q = append(cache, k, v, table, lens, q=q, rotation=rotation)
    out = attend(cache, q, table, lens)

Sequences.  `table` [batch, per_seq] (int32) names each sequence's pages in
order, `lens` [batch] (int32) the tokens that it has, those of this step
included.  The step's rows q, k, v [total, heads, dim] hold the sequences
one after the other: sequence b has rows starts[b] .. starts[b + 1] - 1
(`starts` [batch + 1], int32, rising from its first entry; none and many
rows alike), or, without `starts`, total / batch rows each.  Row i of its n
rows has position lens[b] - n + i.  All three are read on the device when
the kernels run, so a captured graph follows what they then hold.

Pages.  Position j of a sequence is in slot j % page_size of page
table[b, j // page_size].  An entry that is no page of the cache (-1, say)
is allowed: what would be stored there is dropped, and what would be read
there is not attended to.  The same holds for positions below zero, where
lens is less than the rows, and behind the table.  Sequences may share
pages that they only read; where two rows of a step have the same slot, one
of them is stored.

Types.  bfloat16 or float16 rows; the cache in the rows' type, or in
float8_e4m3fn with a float32 scale for each cached head (a value is stored
as value / scale, and values over 448 as 448).  Head dimensions: multiples
of 16 for `append`, 64, 128 or 256 for `attend`; a cached head serves
heads / kv_heads query heads.  Tensors may be strided as long as each
head's values are contiguous and begin at 16 bytes.

Launches go to the current stream of the tensors' device, and their
workspace comes from torch's allocator, so both may be captured.  Forward
only: a call that would have to be differentiated is refused.  Tensors on
the CPU are computed with plain torch operations.  A refused argument
raises ValueError before anything runs; a failed launch, RuntimeError.
"""

from __future__ import annotations

import functools
import math
from typing import NamedTuple

import torch

from nvshare_amd import hiputil

E4M3_MAX = 448.0
ATTEND_DIMS = (64, 128, 256)

_ROW_TYPES = (torch.bfloat16, torch.float16)
_TYPES = {torch.bfloat16: hiputil.KV_BF16, torch.float16: hiputil.KV_FP16,
          torch.float8_e4m3fn: hiputil.KV_E4M3}


class PagedCache(NamedTuple):
    """Keys and values, [pages, page_size, kv_heads, dim] each."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor | None = None
    v_scale: torch.Tensor | None = None

    @classmethod
    def empty(cls, pages: int, page_size: int, kv_heads: int, dim: int,
              dtype: torch.dtype = torch.bfloat16,
              device: torch.device | str = "cuda") -> "PagedCache":
        """A cache whose pages are not touched (nor resident) until used;
        for float8_e4m3fn the scales are ones."""
        shape = (pages, page_size, kv_heads, dim)
        scales = [None, None]
        if dtype == torch.float8_e4m3fn:
            scales = [torch.ones(kv_heads, device=device) for _ in range(2)]
        return cls(torch.empty(shape, dtype=dtype, device=device),
                   torch.empty(shape, dtype=dtype, device=device), *scales)


def rotation_table(positions: int, rotary: int, base: float = 10000.0,
                   device: torch.device | str = "cuda") -> torch.Tensor:
    """[positions, rotary] float32: rotary / 2 cosines, then the sines, of
    position * base ** (-2 i / rotary).  The angles are made in 64 bits:
    in 32, those of far positions would be off by whole degrees."""
    if rotary <= 0 or rotary % 16:
        raise ValueError(f"rotary {rotary} is no positive multiple of 16")
    i = torch.arange(rotary // 2, dtype=torch.float64)
    speed = (base ** (-2.0 * i / rotary)).to(device)
    pos = torch.arange(positions, dtype=torch.float64, device=device)
    angle = pos[:, None] * speed
    return torch.cat((angle.cos(), angle.sin()), dim=1).float()


def append(cache: PagedCache, k: torch.Tensor, v: torch.Tensor,
           table: torch.Tensor, lens: torch.Tensor, *,
           starts: torch.Tensor | None = None,
           q: torch.Tensor | None = None,
           rotation: torch.Tensor | None = None, interleaved: bool = False,
           q_out: torch.Tensor | None = None) -> torch.Tensor | None:
    """Store k and v [total, kv_heads, dim] in the cache, and return the
    queries that go with them, rotated.

    `rotation` [positions, rotary] (rotation_table) turns the first
    `rotary` dimensions of keys and queries: pairs (i, i + rotary / 2), or
    with `interleaved` (2i, 2i + 1).  Without it both stay as they are.  It
    has a row for each position that the table can name.

    `q` [total, heads, dim] gives a new tensor, or goes into `q_out`, which
    may be q itself.  Rows of no sequence are zero in a new tensor and left
    as they are in `q_out`; rows without a place in the table are zero."""
    total, _, dim = _rows("k", k)
    _like("v", v, k)
    heads = k.shape[1]
    if q is not None:
        _like("q", q, k, heads=True)
        heads = q.shape[1]
    elif q_out is not None:
        raise ValueError("q_out without q")
    batch, per_seq = _check(cache, k, heads, table, lens, starts)
    if dim % 16:
        raise ValueError(f"dim {dim} is no multiple of 16")
    if rotation is not None:
        _check_rotation(rotation, k, per_seq * cache.k.shape[1])
    fill = q_out is None
    if q is not None:
        if fill:
            q_out = q.new_empty(q.shape)
        else:
            _like("q_out", q_out, q)
    _forward_only(k, v, q)
    if total == 0:
        return q_out
    if not k.is_cuda:
        _append_plain(cache, k, v, table, lens, starts, q, rotation,
                      interleaved, q_out, fill)
        return q_out
    q_at = out_at = at = rotary = 0
    q_step = out_step = (0, 0)
    if q is not None:
        q_at, q_step = _place("q", q)
        out_at, out_step = _place("q_out", q_out)
    k_at, k_step = _place("k", k)
    v_at, v_step = _place("v", v)
    row = 0
    if rotation is not None:
        at, rotary = rotation.data_ptr(), rotation.shape[1]
        row, last = rotation.stride()
        if last != 1 or row % 4 or at % 16:
            raise ValueError("rotation: rows are not contiguous at 16 bytes")
    args = hiputil.KV_APPEND.pack(
        q_at, k_at, v_at, out_at, at, *q_step, *k_step, *v_step, *out_step,
        row, rotary, interleaved, fill)
    kv = _pack(cache, k, heads, table, lens, starts, batch, per_seq)
    device = k.get_device()
    with _on(device):
        _lib().kv_append(kv, args, _stream(device))
    return q_out


def attend(cache: PagedCache, q: torch.Tensor, table: torch.Tensor,
           lens: torch.Tensor, *, starts: torch.Tensor | None = None,
           scale: float | None = None, window: int | None = None,
           max_new: int | None = None, out: torch.Tensor | None = None,
           return_lse: bool = False):
    """Attention of the rows q [total, heads, dim] over the cache, in which
    the step's own keys and values are already stored.

    A row at position p sees the keys at positions up to p, with `window`
    the last `window` of them.  `scale` (default dim ** -0.5) multiplies
    the scores.  `max_new`, where given, says that no sequence has more new
    rows than that; results never depend on it.

    Returns [total, heads, dim], or goes into `out`, which may be q itself;
    with `return_lse` also the logarithm of each row's sum of exponentials,
    float32 [total, heads].  A row that sees no key gives zeros, and -inf.
    Rows of no sequence give the same in a new tensor and are left as they
    are in `out` (their logarithm is -inf in both)."""
    total, heads, dim = _rows("q", q)
    batch, per_seq = _check(cache, q, heads, table, lens, starts)
    if dim not in ATTEND_DIMS:
        raise ValueError(f"dim {dim} is not one of {ATTEND_DIMS}")
    if scale is None:
        scale = dim ** -0.5
    elif not math.isfinite(scale):
        raise ValueError(f"scale {scale} is not finite")
    if window is None:
        window = 0
    elif window < 1:
        raise ValueError(f"window {window} is less than 1")
    if max_new is None:
        max_new = total
    elif max_new < 0:
        raise ValueError(f"max_new {max_new} is negative")
    fill = out is None
    if fill:
        out = q.new_empty(q.shape)
    else:
        _like("out", out, q)
    _forward_only(q, out)
    result, lse, lse_at = out, None, 0
    if return_lse:
        lse = q.new_empty((total, heads), dtype=torch.float32)
        result, lse_at = (out, lse), lse.data_ptr()
    if total == 0:
        return result
    if not q.is_cuda:
        _attend_plain(cache, q, table, lens, starts, scale, window, out, lse,
                      fill)
        return result
    q_at, q_step = _place("q", q)
    out_at, out_step = _place("out", out)
    args = hiputil.KV_ATTEND.pack(
        q_at, out_at, lse_at, *q_step, *out_step, scale,
        min(window, 2**31 - 1), min(max_new, total), fill)
    kv = _pack(cache, q, heads, table, lens, starts, batch, per_seq)
    device = q.get_device()
    lib = _lib()
    size = lib.kv_attend_work(kv, args)
    work = q.new_empty(size, dtype=torch.uint8) if size else None
    with _on(device):
        lib.kv_attend(kv, args, work.data_ptr() if size else None,
                      _stream(device))
    return result


# -- arguments ---------------------------------------------------------
#
# A step of a few tokens takes the GPU less time than it takes Python to
# look its arguments over with care, so each check is one condition, and
# what exactly is wrong is found out once it has failed.


def _rows(name: str, t: torch.Tensor) -> torch.Size:
    shape = t.shape
    if len(shape) != 3:
        raise ValueError(f"{name}: [total, heads, dim] is wanted, got "
                         f"{tuple(shape)}")
    if t.dtype not in _ROW_TYPES:
        raise ValueError(f"{name}: bfloat16 or float16 is wanted, got "
                         f"{t.dtype}")
    if shape[0] * shape[1] >= 2**31 - 1:
        raise ValueError(f"{name}: {shape[0]} rows of {shape[1]} heads pass "
                         "31 bits")
    return shape


def _like(name: str, t: torch.Tensor, k: torch.Tensor,
          heads: bool = False) -> None:
    """`t` has the rows, type and device of `k`, and its heads or others."""
    a, b = t.shape, k.shape
    if (t.dtype != k.dtype or t.get_device() != k.get_device()
            or (a != b and not (heads and len(a) == 3 and a[0] == b[0]
                                and a[2] == b[2]))):
        raise ValueError(
            f"{name}: {t.dtype} {tuple(a)} on {t.device} does not go with "
            f"{k.dtype} {tuple(b)} on {k.device}")


def _place(name: str, t: torch.Tensor) -> tuple[int, tuple[int, int]]:
    """Address and strides of rows [total, heads, dim]."""
    at = t.data_ptr()
    row, head, last = t.stride()
    if last != 1 or (row | head) % 8 or at % 16:
        raise ValueError(_unaligned(name, t))
    return at, (row, head)


def _unaligned(name: str, t: torch.Tensor) -> str:
    return (f"{name}: values of a head are not contiguous at 16 bytes "
            f"(strides {t.stride()})")


def _check(cache: PagedCache, rows: torch.Tensor, heads: int,
           table: torch.Tensor, lens: torch.Tensor,
           starts: torch.Tensor | None) -> tuple[int, int]:
    """What both operators ask of their common arguments; the table's
    shape."""
    ck, cv, k_scale, v_scale = cache
    device, total = rows.get_device(), rows.shape[0]
    shape, dtype = ck.shape, ck.dtype
    if (len(shape) != 4 or shape != cv.shape or dtype != cv.dtype
            or shape[3] != rows.shape[2] or ck.get_device() != device
            or cv.get_device() != device):
        raise ValueError(
            f"cache: keys {dtype} {tuple(shape)} on {ck.device} and values "
            f"{cv.dtype} {tuple(cv.shape)} on {cv.device} are not both "
            f"[pages, page_size, kv_heads, {rows.shape[2]}] on "
            f"{rows.device}")
    pages, page_size, kv_heads, _ = shape
    if (heads == 0 or kv_heads == 0 or heads % kv_heads or pages == 0
            or page_size == 0 or max(pages, page_size) > 2**31 - 1):
        raise ValueError(f"cache: {pages} pages of {page_size} with "
                         f"{kv_heads} heads cannot serve {heads} heads")
    if dtype == torch.float8_e4m3fn:
        for name, s in (("k_scale", k_scale), ("v_scale", v_scale)):
            if (s is None or s.dtype != torch.float32
                    or s.shape != (kv_heads,) or s.get_device() != device
                    or not s.is_contiguous()):
                raise ValueError(
                    f"{name}: float8_e4m3fn wants a contiguous float32 "
                    f"[{kv_heads}] tensor on the cache's device")
    elif dtype != rows.dtype:
        raise ValueError(f"cache: {dtype} is neither {rows.dtype} nor "
                         "float8_e4m3fn")
    elif k_scale is not None or v_scale is not None:
        raise ValueError(f"{'k' if k_scale is not None else 'v'}_scale: "
                         f"{dtype} goes without")
    if (table.dtype != torch.int32 or table.dim() != 2
            or table.get_device() != device
            or (table.shape[1] > 1 and table.stride(1) != 1)):
        raise ValueError(
            "table: an int32 [batch, pages] tensor with contiguous rows on "
            f"the rows' device is wanted, got {table.dtype} "
            f"{tuple(table.shape)} on {table.device}")
    batch, per_seq = table.shape
    if per_seq * page_size > 2**31 - 1:
        raise ValueError(f"table: {per_seq} pages of {page_size} pass 31 "
                         "bits of positions")
    if (lens.dtype != torch.int32 or lens.shape != (batch,)
            or lens.get_device() != device or not lens.is_contiguous()):
        raise ValueError(_no_index("lens", lens, batch))
    if starts is not None:
        if (starts.dtype != torch.int32 or starts.shape != (batch + 1,)
                or starts.get_device() != device
                or not starts.is_contiguous()):
            raise ValueError(_no_index("starts", starts, batch + 1))
    elif total % batch if batch else total:
        raise ValueError(f"{total} rows are not the same number for each of "
                         f"{batch} sequences: give starts")
    if total and (batch == 0 or per_seq == 0):
        raise ValueError("table: rows, but no sequences or no pages")
    return batch, per_seq


def _no_index(name: str, t: torch.Tensor, n: int) -> str:
    return (f"{name}: a contiguous int32 [{n}] tensor on the rows' device "
            f"is wanted, got {t.dtype} {tuple(t.shape)} on {t.device}")


def _check_rotation(rotation: torch.Tensor, k: torch.Tensor,
                    positions: int) -> None:
    if (rotation.dim() != 2 or rotation.dtype != torch.float32
            or rotation.get_device() != k.get_device()):
        raise ValueError("rotation: a float32 [positions, rotary] tensor on "
                         "the device of k is wanted")
    have, rotary = rotation.shape
    if rotary == 0 or rotary % 16 or rotary > k.shape[2]:
        raise ValueError(f"rotation: {rotary} dimensions are no multiple of "
                         f"16 up to {k.shape[2]}")
    if have < positions:
        raise ValueError(f"rotation: {have} positions, the table names "
                         f"{positions}")


def _pack(cache: PagedCache, rows: torch.Tensor, heads: int,
          table: torch.Tensor, lens: torch.Tensor,
          starts: torch.Tensor | None, batch: int, per_seq: int) -> bytes:
    ck, cv, k_scale, v_scale = cache
    pages, page_size, kv_heads, dim = ck.shape
    *k_step, k_last = ck.stride()
    *v_step, v_last = cv.stride()
    k_at, v_at = ck.data_ptr(), cv.data_ptr()
    step = 8 if k_scale is None else 16
    if k_last != 1 or (k_step[0] | k_step[1] | k_step[2]) % step \
            or k_at % 16:
        raise ValueError(_unaligned("cache.k", ck))
    if v_last != 1 or (v_step[0] | v_step[1] | v_step[2]) % step \
            or v_at % 16:
        raise ValueError(_unaligned("cache.v", cv))
    return hiputil.KV_CACHE.pack(
        k_at, v_at, 0 if k_scale is None else k_scale.data_ptr(),
        0 if v_scale is None else v_scale.data_ptr(), table.data_ptr(),
        lens.data_ptr(), 0 if starts is None else starts.data_ptr(),
        table.stride(0), *k_step, *v_step, _TYPES[rows.dtype],
        _TYPES[ck.dtype], batch, rows.shape[0], heads, kv_heads, dim, pages,
        page_size, per_seq)


def _forward_only(*tensors: torch.Tensor | None) -> None:
    if not torch.is_grad_enabled():
        return
    for t in tensors:
        if t is not None and t.requires_grad:
            raise ValueError("forward only: call under torch.no_grad(), or "
                             "detach the arguments")


@functools.cache
def _lib() -> hiputil.HipUtil:
    return hiputil.load()


# torch.cuda.current_stream() takes as long as the rest of a launch.
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


class _on:
    """The device made current, where it is not."""

    __slots__ = ("device", "before")

    def __init__(self, device: int) -> None:
        self.device = device

    def __enter__(self) -> None:
        self.before = torch._C._cuda_getDevice()
        if self.before != self.device:
            torch.cuda.set_device(self.device)

    def __exit__(self, *exc) -> None:
        if self.before != self.device:
            torch.cuda.set_device(self.before)


# -- plain forms, for tensors on the CPU -------------------------------


def _sequences(total, lens, starts):
    """(b, its rows as a slice, their positions) of each sequence."""
    batch = lens.shape[0]
    if starts is None:
        bounds = [total // batch * b for b in range(batch + 1)]
    else:
        bounds = starts.tolist()
    for b, length in enumerate(lens.tolist()):
        lo, hi = bounds[b], bounds[b + 1]
        yield b, slice(lo, hi), torch.arange(length - (hi - lo), length)


def _slots(cache, table, b, pos):
    """(whether the positions have a place, its page, its slot)."""
    page_size, per_seq = cache.k.shape[1], table.shape[1]
    inside = (pos >= 0) & (pos < per_seq * page_size)
    at = torch.where(inside, pos, torch.zeros_like(pos))
    page = table[b].long()[at // page_size]
    mapped = inside & (page >= 0) & (page < cache.k.shape[0])
    return inside, mapped, page, at % page_size


def _rotate(x, cs, interleaved):
    """The first dimensions of x [rows, heads, dim] turned, in float32."""
    rotary = cs.shape[1]
    cos, sin = cs[:, None].chunk(2, dim=-1)
    part = x[..., :rotary]
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        part = torch.stack((a * cos - b * sin, b * cos + a * sin),
                           dim=-1).flatten(-2)
    else:
        a, b = part.chunk(2, dim=-1)
        part = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((part, x[..., rotary:]), dim=-1)


def _append_plain(cache, k, v, table, lens, starts, q, rotation, interleaved,
                  q_out, fill):
    q_in = q.clone() if q is not None else None
    if fill and q_out is not None:
        q_out.zero_()
    for b, rows, pos in _sequences(k.shape[0], lens, starts):
        inside, mapped, page, slot = _slots(cache, table, b, pos)
        new = {"k": k[rows].float(), "v": v[rows].float()}
        if rotation is not None:
            cs = rotation[torch.where(inside, pos, torch.zeros_like(pos))]
            new["k"] = _rotate(new["k"], cs, interleaved)
        for name, to, scale in (("k", cache.k, cache.k_scale),
                                ("v", cache.v, cache.v_scale)):
            x = new[name]
            if scale is not None:
                x = (x / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX)
            to[page[mapped], slot[mapped]] = x[mapped].to(to.dtype)
        if q is not None:
            x = q_in[rows].float()
            if rotation is not None:
                x = _rotate(x, cs, interleaved)
            q_out[rows] = torch.where(inside[:, None, None], x,
                                      torch.zeros_like(x)).to(q.dtype)


def _attend_plain(cache, q, table, lens, starts, scale, window, out, lse,
                  fill):
    q_in = q.clone()
    if fill:
        out.zero_()
    if lse is not None:
        lse.fill_(-math.inf)
    heads, kv_heads = q.shape[1], cache.k.shape[2]
    for b, rows, pos in _sequences(q.shape[0], lens, starts):
        if not pos.numel():
            continue
        keys = torch.arange(max(0, int(pos[-1]) + 1))
        _, mapped, page, slot = _slots(cache, table, b, keys)
        keys, page, slot = keys[mapped], page[mapped], slot[mapped]
        k, v = cache.k[page, slot].float(), cache.v[page, slot].float()
        if cache.k_scale is not None:
            k, v = k * cache.k_scale[:, None], v * cache.v_scale[:, None]
        k, v = (x.repeat_interleave(heads // kv_heads, dim=1).transpose(0, 1)
                for x in (k, v))
        s = q_in[rows].float().transpose(0, 1) @ k.transpose(1, 2) * scale
        seen = keys <= pos[:, None]
        if window:
            seen &= keys > pos[:, None] - window
        s = s.masked_fill(~seen, -math.inf)
        total = s.logsumexp(-1)
        weight = torch.exp(s - total.masked_fill(
            total == -math.inf, 0.0)[..., None])
        # 0 * inf is no number: a value that is not seen is left out.
        x = weight @ torch.where(v.isfinite(), v, torch.zeros_like(v))
        for j in (~v.isfinite()).any(-1).any(0).nonzero().flatten().tolist():
            add = v[:, j][:, None].masked_fill(v[:, j][:, None].isfinite(),
                                               0.0)
            x = torch.where(seen[:, j][:, None], x + add, x)
        out[rows] = x.transpose(0, 1).to(q.dtype)
        if lse is not None:
            lse[rows] = total.transpose(0, 1)
