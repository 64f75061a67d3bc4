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
included.  The step's rows q, k, v [total, heads, dim] hold the sequences one
after the other: sequence b has rows starts[b] .. starts[b + 1] - 1
(`starts` [batch + 1], int32, rising from its first entry; none and many
rows alike; a sequence whose rows would pass total has none, and the rows
are of no sequence), or, without `starts`, total / batch rows each.  Row i of
its n rows has position lens[b] - n + i.  All three are read on the device
when the kernels run, so a captured graph follows what they then hold;
nothing may change them meanwhile.

Pages.  Position j of a sequence is in slot j % page_size of page
table[b, j // page_size].  An entry that is no page of the cache (-1, say)
is allowed: what would be stored there is dropped, and what would be read
there is not attended to.  The same holds for positions below zero, where
lens is less than the rows, and behind the table.  Sequences may share
pages that they only read; where two rows of a step have the same slot, each
value that it then holds is of either.

Types.  bfloat16 or float16 rows; the cache in the rows' type, or in
float8_e4m3fn with a float32 scale for each cached head (a value is stored
as value / scale, and values over 448 as 448).  Head dimensions: multiples
of 16 for `append`, 64, 128 or 256 for `attend`; a cached head serves
heads / kv_heads query heads.  Tensors may be strided as long as each
head's values are contiguous and begin at 16 bytes.  What a call writes to
(the cache, q_out, out) shares no memory with its other arguments, but that
q_out and out may be q itself.

Launches go to the current stream of the tensors' device, and their
workspace comes from torch's allocator, so both may be captured.  Forward
only: a call that would have to be differentiated, backwards or forwards,
is refused.  Tensors on the CPU are computed with plain torch operations;
they need the compiled calls (hip/kvbind.cpp, a C++ compiler's work) and
not the kernels.  A refused argument raises ValueError before anything
runs; a failed launch, RuntimeError.
"""

from __future__ import annotations

import functools
import importlib.util
import math
from typing import NamedTuple

import torch

from nvshare_amd.paths import artifacts

E4M3_MAX = 448.0


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
    device = k.get_device()
    fill = q_out is None
    q_out = _run(load().append, device, *cache, k, v, table, lens, starts, q,
                 rotation, interleaved, q_out)
    if device < 0:
        _append_plain(cache, k, v, table, lens, starts, q, rotation,
                      interleaved, q_out, fill)
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
    rows than that; the work is divided by it, and where it does not hold
    only the time suffers.

    Scores, weights and sums are made in 32 bits.  A sequence of many rows
    (more than 32 for a cached head, 16 beside longer ones) has its weights
    rounded to the rows' type before they meet the values, one of few rows
    keeps twice the bits.

    Returns [total, heads, dim], or goes into `out`, which may be q itself;
    with `return_lse` also the logarithm of each row's sum of exponentials,
    float32 [total, heads].  A row that sees no key gives zeros, and -inf.
    Rows of no sequence give the same in a new tensor and are left as they
    are in `out` (their logarithm is -inf in both)."""
    if window is not None and window < 1:
        raise ValueError(f"window {window} is less than 1")
    if max_new is not None and max_new < 0:
        raise ValueError(f"max_new {max_new} is negative")
    device = q.get_device()
    fill = out is None
    out, lse = _run(load().attend, device, *cache, q, table, lens, starts,
                    scale, window or 0, max_new, out, return_lse)
    if device < 0:
        if scale is None:
            scale = q.shape[-1] ** -0.5
        _attend_plain(cache, q, table, lens, starts, scale, window, out, lse,
                      fill)
    return (out, lse) if return_lse else out


@functools.cache
def load():
    """The compiled calls (hip/kvbind.cpp), which check their arguments."""
    path = artifacts().kvbind
    if not path.exists():
        raise FileNotFoundError(
            f"{path} missing; build with `make -C hip` (hipcc, gfx950), or "
            "for tensors on the CPU `make -C hip build/_kvbind.so` (a C++ "
            "compiler)")
    spec = importlib.util.spec_from_file_location("_kvbind", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _run(call, device: int, *args):
    """The call on the device's current stream, with the device current."""
    if device < 0:
        return call(*args, 0)
    # torch.cuda's own functions for these take as long as the call.
    if device == torch._C._cuda_getDevice():
        return call(*args, torch._C._cuda_getCurrentRawStream(device))
    with torch.cuda.device(device):
        return call(*args, torch._C._cuda_getCurrentRawStream(device))


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
        if not 0 <= lo <= hi <= total:
            lo = hi = 0
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
        # From the first that some row sees to the last with a place.
        first = max(0, int(pos[0]) + 1 - window) if window else 0
        last = min(int(pos[-1]) + 1, table.shape[1] * cache.k.shape[1])
        keys = torch.arange(first, max(first, last))
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
