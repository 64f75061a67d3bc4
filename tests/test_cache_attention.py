"""The paged key/value cache: append and attend against 64 bits.

Each case runs on the CPU (plain torch form) and, with -m gpu, through the
gfx950 kernels.  The oracle below computes in float64 from the formulas,
one sequence, row and head at a time, and shares no code with either.

Tolerances count roundings.  With u half a step of the rows' type (2^-8
for bfloat16, 2^-11 for float16, relative):
  attend: each weight may be rounded once before it meets the values, which
    moves the result by up to u * A with A = sum w |v| / sum w, and the
    result is rounded once, u * |o|.  What is done in 32 bits adds an error
    of the scores, up to dim * 2^-24 * sum |q k| * scale, twice (in the
    weight and in their sum), and 2^-20 for exponentials and sums.
  append: one rounding of the result, and three of 2^-24 in the turn.
"""

from __future__ import annotations

import math
import random

import pytest
import torch
from torch.autograd import forward_ad

from nvshare_amd.kvcache import PagedCache, append, attend, rotation_table
from nvshare_amd.paths import ensure_kernels

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module", autouse=True)
def kernels():
    ensure_kernels()


@pytest.fixture(params=DEVICES)
def device(request):
    if request.param == "cuda" and not torch.cuda.is_available():
        pytest.skip("no GPU here")
    return request.param


@pytest.fixture
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU here")
    return "cuda"


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


class Step:
    """A step's rows over a cache that holds earlier tokens already."""

    def __init__(self, device, seqs, *, heads=4, kv_heads=2, dim=64, page=16,
                 dtype=torch.bfloat16, cache=None, uniform=False, pad=0,
                 pages=None, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.seqs, self.page = seqs, page
        total = sum(n for n, _ in seqs) + pad
        self.q = torch.randn(total, heads, dim, generator=g).to(dtype)
        self.k = torch.randn(total, kv_heads, dim, generator=g).to(dtype)
        self.v = torch.randn(total, kv_heads, dim, generator=g).to(dtype)
        need = [-(-max(t, 0) // page) for _, t in seqs]
        pages = pages or sum(need) + 2
        order = torch.randperm(pages, generator=g)
        per_seq = max(need + [1])
        self.table = torch.full((len(seqs), per_seq), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n].int()
            at += n
        self.lens = torch.tensor([t for _, t in seqs], dtype=torch.int32)
        starts = [0]
        for n, _ in seqs:
            starts.append(starts[-1] + n)
        self.bounds = starts
        self.starts = None if uniform else torch.tensor(starts,
                                                        dtype=torch.int32)
        shape = (pages, page, kv_heads, dim)
        kc, vc = (torch.randn(shape, generator=g) for _ in range(2))
        scales = (None, None)
        if cache == E4M3:
            scales = tuple(0.01 + 0.02 * torch.rand(kv_heads, generator=g)
                           for _ in range(2))
            kc, vc = (x / s[:, None] for x, s in zip((kc, vc), scales))
            kc, vc = (x.clamp(-448, 448).to(E4M3) for x in (kc, vc))
        else:
            kc, vc = kc.to(dtype), vc.to(dtype)
        self.cache = PagedCache(kc, vc, *scales)
        self.device = device

    def to(self, device=None):
        """The arguments on the device, as copies."""
        d = device or self.device
        cache = PagedCache(*(None if x is None else x.to(d, copy=True)
                             for x in self.cache))
        return cache, {n: None if x is None else x.to(d, copy=True)
                       for n, x in (("q", self.q), ("k", self.k),
                                    ("v", self.v), ("table", self.table),
                                    ("lens", self.lens),
                                    ("starts", self.starts))}

    def slot(self, b, j):
        """(page, slot) of position j, or None where it has no place."""
        if not 0 <= j < self.table.shape[1] * self.page:
            return None
        page = int(self.table[b, j // self.page])
        if not 0 <= page < self.cache.k.shape[0]:
            return None
        return page, j % self.page

    def rows(self):
        """(row, sequence, position) of each row that belongs to one."""
        for b, (n, length) in enumerate(self.seqs):
            for i in range(n):
                yield self.bounds[b] + i, b, length - n + i


def attend_oracle(s, scale=None, window=None):
    """(o, its bound, lse, its bound), float64."""
    total, heads, dim = s.q.shape
    scale = dim ** -0.5 if scale is None else scale
    group = heads // s.cache.k.shape[2]
    out = torch.zeros(total, heads, dim, dtype=torch.float64)
    tol = torch.zeros_like(out)
    lse = torch.full((total, heads), -math.inf, dtype=torch.float64)
    lse_tol = torch.zeros_like(lse)
    u = half_step(s.q.dtype)
    kc, vc = s.cache.k.double(), s.cache.v.double()
    if s.cache.k_scale is not None:
        kc = kc * s.cache.k_scale.double()[:, None]
        vc = vc * s.cache.v_scale.double()[:, None]
    for row, b, pos in s.rows():
        low = 0 if window is None else max(0, pos - window + 1)
        at = [s.slot(b, j) for j in range(low, pos + 1)]
        at = [x for x in at if x is not None]
        if not at:
            continue
        page, slot = (torch.tensor(x) for x in zip(*at))
        for h in range(heads):
            k, v = kc[page, slot, h // group], vc[page, slot, h // group]
            q = s.q[row, h].double()
            score = k @ q * scale
            w = torch.exp(score - score.max())
            out[row, h] = w @ v / w.sum()
            lse[row, h] = score.max() + w.sum().log()
            off = dim * 2.0**-24 * (k.abs() @ q.abs()).max() * abs(scale)
            size = w @ v.abs() / w.sum()
            tol[row, h] = (u * (size + out[row, h].abs())
                           + (2 * off + 2.0**-20) * size)
            lse_tol[row, h] = off + 2.0**-20 + 2.0**-22 * lse[row, h].abs()
    if s.q.dtype == torch.float16:
        tol += 2.0**-25  # half a step of its smallest numbers
    return out, tol * 1.01, lse, lse_tol


def near(got, want, tol, what):
    got = got.double().cpu()
    both_nan = got.isnan() & want.isnan()
    same = (got == want) | both_nan
    off = torch.where(same, torch.zeros_like(want), (got - want).abs())
    bad = ~(off <= tol) & ~same
    assert not bad.any(), (
        f"{what}: {int(bad.sum())} of {bad.numel()} values off, the worst by "
        f"{float(off[bad].max()):.3g} where {float(tol[bad].min()):.3g} is "
        f"allowed; the first at {bad.nonzero()[0].tolist()}: "
        f"{got[bad][0]} for {want[bad][0]}")


def check_attend(s, scale=None, window=None, max_new=None):
    cache, a = s.to()
    out, lse = attend(cache, a["q"], a["table"], a["lens"],
                      starts=a["starts"], scale=scale, window=window,
                      max_new=max_new, return_lse=True)
    want, tol, want_lse, lse_tol = attend_oracle(s, scale, window)
    assert out.dtype == s.q.dtype and out.shape == s.q.shape
    assert lse.dtype == torch.float32
    near(out, want, tol, "out")
    near(lse, want_lse, lse_tol, "lse")
    return out


# -- attend: lengths, heads, dims, types -------------------------------


@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 33, 63, 64, 65,
                                    127, 129, 255, 257, 600])
def test_one_token(device, length):
    check_attend(Step(device, [(1, length)], uniform=True, seed=length))


@pytest.mark.parametrize("new", [1, 2, 3, 8, 15, 17, 31, 32, 33, 63, 65,
                                 127, 128, 129])
@pytest.mark.parametrize("context", [0, 1, 70])
def test_chunk(device, new, context):
    check_attend(Step(device, [(new, context + new)], uniform=True,
                      seed=new))


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (7, 1), (8, 2),
                                            (10, 5), (16, 1), (33, 1),
                                            (40, 2)])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 5])
def test_heads(device, heads, kv_heads, dim, new):
    check_attend(Step(device, [(new, 90), (new, 41)], heads=heads, dim=dim,
                      kv_heads=kv_heads, uniform=True))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cache", [None, E4M3])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 6, 70])
def test_types(device, dtype, cache, dim, new):
    check_attend(Step(device, [(new, new + 77)], dtype=dtype, cache=cache,
                      dim=dim, uniform=True, seed=dim))


@pytest.mark.parametrize("page", [1, 2, 8, 24, 32, 64, 100, 128, 256])
@pytest.mark.parametrize("new", [1, 50])
def test_pages(device, page, new):
    check_attend(Step(device, [(new, 170), (new, 299)], page=page,
                      uniform=True, seed=page))


@pytest.mark.parametrize("window", [1, 2, 5, 16, 63, 64, 65, 100, 5000])
@pytest.mark.parametrize("new", [1, 4, 90])
def test_window(device, window, new):
    check_attend(Step(device, [(new, 200), (new, 91)], uniform=True),
                 window=window)


def test_scale(device):
    s = Step(device, [(3, 60)], uniform=True)
    check_attend(s, scale=0.5)
    check_attend(s, scale=0.0)
    check_attend(s, scale=-0.2)


RAGGED = [
    [(1, 1), (0, 0), (1, 50), (1, 7)],
    [(0, 0), (0, 30), (130, 130), (1, 300), (0, 0)],
    [(5, 5), (40, 200), (1, 129), (0, 3), (17, 64), (64, 64)],
    [(0, 0), (0, 0), (3, 3)],
    [(1, 40)] * 70 + [(20, 33)],
]


@pytest.mark.parametrize("seqs", RAGGED)
@pytest.mark.parametrize("known", [False, True])
def test_ragged(device, seqs, known):
    s = Step(device, seqs, heads=4, kv_heads=2, seed=3)
    check_attend(s, max_new=max(n for n, _ in seqs) if known else None)


def test_max_new_does_not_change_results(device):
    """Even one that does not hold."""
    s = Step(device, [(50, 90), (3, 9)])
    for most in (0, 1, 53, 10000):
        check_attend(s, max_new=most)


def test_ragged_window_wide(device):
    check_attend(Step(device, [(33, 300), (1, 290), (140, 140)], dim=256,
                      dtype=torch.float16), window=70)


@pytest.mark.gpu
def test_long_context_is_split(gpu):
    """Few rows over many keys: partial results are joined."""
    for new, cache in ((1, None), (9, None), (40, None), (1, E4M3)):
        check_attend(Step(gpu, [(new, 5003)], heads=4, kv_heads=1, dim=128,
                          page=64, cache=cache, uniform=True, seed=new))


@pytest.mark.gpu
@pytest.mark.parametrize("new,length,dim", [(20, 17403, 128),
                                            (20, 17403, 256),
                                            (33, 16500, 64)])
def test_chunk_in_many_parts(gpu, new, length, dim):
    """Sixteen parts and more, joined by four waves a row."""
    check_attend(Step(gpu, [(new, length)], heads=4, kv_heads=1, dim=dim,
                      page=64, uniform=True))


@pytest.mark.gpu
def test_unlike_lengths_in_one_batch(gpu):
    check_attend(Step(gpu, [(1, 4000), (1, 1), (1, 130), (0, 0), (1, 2900)],
                      heads=8, kv_heads=2, dim=128))


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(12))
def test_any_batch(gpu, seed):
    """Whatever mixture of sequences: their tiles are dealt out evenly, and
    long ones are divided anywhere."""
    rng = random.Random(seed)
    seqs = []
    for _ in range(rng.choice((1, 3, 9, 40))):
        new = rng.choice((0, 1, 1, 1, 2, 7, 30, 150))
        seqs.append((new, new + rng.choice((0, 5, 300, 1500))))
    dim = rng.choice((64, 128, 256))
    kv_heads = rng.choice((1, 2, 3))
    check_attend(
        Step(gpu, seqs, heads=kv_heads * rng.choice((1, 4, 5)),
             kv_heads=kv_heads, dim=dim, page=rng.choice((8, 16, 48, 64)),
             cache=rng.choice((None, E4M3)), pad=rng.choice((0, 3)),
             seed=seed),
        window=rng.choice((None, None, 100)),
        max_new=rng.choice((None, max(n for n, _ in seqs))))


@pytest.mark.gpu
def test_many_sequences(gpu):
    seqs = [(1, 1 + 7 * b % 60) for b in range(1000)]
    check_attend(Step(gpu, seqs, heads=2, kv_heads=1, uniform=True))
    check_attend(Step(gpu, seqs[:333] + [(9, 40), (0, 0)], heads=2,
                      kv_heads=1))


# -- attend: rows that see little or nothing, bad pages ----------------


def test_rows_before_the_first_position(device):
    """More rows than tokens: the first rows have no position."""
    s = Step(device, [(6, 4), (3, 0), (40, 35)], seed=5)
    out = check_attend(s)
    assert not out[:2].any() and not out[6:9].any()


def test_negative_length(device):
    s = Step(device, [(2, 5), (2, -7)])
    check_attend(s)


@pytest.mark.parametrize("bad", [-1, 10**6, -2**31, 2**31 - 1])
@pytest.mark.parametrize("new", [1, 40])
def test_bad_pages_are_not_attended(device, bad, new):
    s = Step(device, [(new, 300), (new, 90)], seed=1)
    s.table[0, 3] = bad
    s.table[0, 7:9] = bad
    s.table[1, :] = bad
    out = check_attend(s)
    assert not out[new:].any()


def test_length_behind_the_table(device):
    """Positions that the table does not name hold no keys."""
    s = Step(device, [(4, 60), (1, 50)])
    s.lens += 45
    s.seqs = [(n, t + 45) for n, t in s.seqs]
    check_attend(s)
    check_attend(s, window=30)
    check_attend(s, window=9)


@pytest.mark.parametrize("new", [1, 40])
def test_any_length_behind_the_table(device, new):
    """Takes no more time and memory than the table's positions."""
    s = Step(device, [(new, 60)])
    want = check_attend(s)
    cache, a = s.to()
    lens = torch.tensor([2**31 - 1], dtype=torch.int32, device=device)
    q = a["q"][-1:].expand(new, -1, -1)
    seen = torch.tensor([64], dtype=torch.int32, device=device)
    last = attend(cache, a["q"][-1:], a["table"], seen)
    out = attend(cache, q, a["table"], lens)
    tol = 2 * half_step(s.q.dtype) * (last.abs() + s.cache.v.abs().max().to(
        device)).double().cpu()  # rounded by other kernels
    near(out, last.double().cpu().expand(out.shape), tol, "out")
    assert not attend(cache, q, a["table"], lens, window=9).any()
    assert not attend(cache, q, a["table"], lens - 2**31).any()
    assert torch.equal(attend(cache, a["q"], a["table"], a["lens"]), want)


def spoil(s, value, where):
    """Put `value` in every cached key and value that `where` names."""
    for b, j in where:
        page, slot = s.slot(b, j)
        s.cache.k[page, slot] = torch.tensor(value).to(s.cache.k.dtype)
        s.cache.v[page, slot] = torch.tensor(value).to(s.cache.v.dtype)


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("new", [1, 37])
def test_unused_slots_hold_anything(device, value, new):
    s = Step(device, [(new, 70), (new, 129)], seed=2)
    used = torch.zeros(s.cache.k.shape[:2], dtype=torch.bool)
    for b, (_, length) in enumerate(s.seqs):
        for j in range(length):
            used[s.slot(b, j)] = True
    s.cache.k[~used] = value
    s.cache.v[~used] = value
    assert check_attend(s).isfinite().all()


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("new,heads", [(3, 4), (12, 4), (70, 4), (140, 2)])
def test_later_tokens_hold_anything(device, value, new, heads):
    """A row's result does not hang on tokens that come after it."""
    s = Step(device, [(new, 40 + new)], heads=heads, kv_heads=2, seed=2)
    clean = check_attend(s)
    spoil(s, value, [(0, 40 + new - 1)])
    cache, a = s.to()
    out = attend(cache, a["q"], a["table"], a["lens"], starts=a["starts"])
    assert torch.equal(out[:-1], clean[:-1])
    assert not out[-1].isfinite().all()


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("new", [1, 40])
def test_queries_that_are_no_numbers(device, value, dtype, new):
    """Nor is their result, whatever the scores are multiplied by: 0 too."""
    s = Step(device, [(new, 60)], dtype=dtype, uniform=True)
    s.q[0, 1, 3] = value
    for scale in (None, -0.5, 0.0):
        cache, a = s.to()
        out, lse = attend(cache, a["q"], a["table"], a["lens"], scale=scale,
                          return_lse=True)
        spoilt = torch.zeros(new, 4, dtype=torch.bool, device=device)
        spoilt[0, 1] = True
        # Of infinite scores the sum is infinite, if not NaN.
        assert torch.equal(~lse.isfinite(), spoilt)
        assert torch.equal(out.isnan(), spoilt[..., None].expand_as(out))
        assert out[~spoilt].isfinite().all()


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("new", [1, 5, 66])
def test_tokens_before_the_window_hold_anything(device, value, new):
    s = Step(device, [(new, 150 + new)], seed=2)
    clean = check_attend(s, window=20)
    spoil(s, value, [(0, j) for j in range(131)])
    cache, a = s.to()
    out = attend(cache, a["q"], a["table"], a["lens"], starts=a["starts"],
                 window=20)
    assert torch.equal(out, clean)


@pytest.mark.parametrize("new", [1, 5, 66])
def test_infinite_value_reaches_the_rows_that_see_it(device, new):
    """+inf, -inf and NaN in one dimension each of a token that all see,
    and in the last, which only the last row sees."""
    s = Step(device, [(new, 90 + new)], seed=4)
    for j in (30, 90 + new - 1):
        page, slot = s.slot(0, j)
        s.cache.v[page, slot, :, 3] = math.inf
        s.cache.v[page, slot, :, 9] = -math.inf
        s.cache.v[page, slot, :, 21] = math.nan
    cache, a = s.to()
    out = attend(cache, a["q"], a["table"], a["lens"], starts=a["starts"])
    assert (out[..., 3] == math.inf).all()
    assert (out[..., 9] == -math.inf).all()
    assert out[..., 21].isnan().all()
    rest = [d for d in range(64) if d not in (3, 9, 21)]
    assert out[..., rest].isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("new,length", [(1, 1301), (1, 5003), (8, 5003),
                                        (40, 5203), (40, 17403)])
def test_infinite_value_in_divided_keys(gpu, new, length):
    """The same where the keys are divided and the parts joined, in the
    first part and in the last: by a wave a row (1301 and 5203 keys) and by
    four, none of them with a number of parts that fills their turns."""
    s = Step(gpu, [(new, length)], heads=4, kv_heads=1, dim=128, page=64,
             uniform=True, seed=new)
    cache, a = s.to()
    clean = attend(cache, a["q"], a["table"], a["lens"])
    places = [s.slot(0, j) for j in (3, length - new)]
    for value in (math.inf, -math.inf, math.nan):
        for at in places:
            cache, a = s.to()
            cache.v[at][:, 5] = value
            out = attend(cache, a["q"], a["table"], a["lens"])
            want = torch.full_like(out[..., 5], value)
            assert torch.equal(out[..., 5].nan_to_num(), want.nan_to_num())
            assert torch.equal(out[..., 5].isnan(), want.isnan())
            out[..., 5] = clean[..., 5]
            assert torch.equal(out, clean)
            # A key that is no number: nor is any row's result.
            cache, a = s.to()
            cache.k[at][:, 5] = math.nan
            out, lse = attend(cache, a["q"], a["table"], a["lens"],
                              return_lse=True)
            assert out.isnan().all() and lse.isnan().all()


def test_large_scores(device):
    """Scores far apart: exponentials neither overflow nor all vanish."""
    s = Step(device, [(2, 130)], dtype=torch.float16, seed=6)
    s.q *= 60
    s.cache.k.mul_(60)
    check_attend(s)


@pytest.mark.parametrize("new", [1, 50])
def test_scores_rise_along_the_keys(device, new):
    """Each key outweighs all before it: the maximum moves in each tile."""
    s = Step(device, [(new, 260)], dtype=torch.float16, uniform=True, seed=7)
    s.q.fill_(0.5)
    for j in range(260):
        page, slot = s.slot(0, j)
        s.cache.k[page, slot] = j / 8
    check_attend(s)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cache", [None, E4M3])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 6, 14])
def test_weights_of_few_rows_keep_their_bits(device, dtype, cache, dim, new):
    """Up to 32 rows of a sequence: weights meet the values in two parts.
    With u half a step, the first part (cut off) leaves 2u, and that is
    rounded to u: 2u^2; two additions that keep parts from being zero are
    2^-20 each, or 2^-24 of 2^11 for each key in float16.  Small queries
    leave next to nothing to the scores' own errors."""
    s = Step(device, [(new, 20)], dtype=dtype, cache=cache, dim=dim,
             uniform=True, seed=dim + new)
    s.q /= 16
    u = half_step(dtype)
    cache, a = s.to("cpu")
    k, v = (torch.stack([x[s.slot(0, j)] for j in range(20)]).double()
            for x in cache[:2])
    if s.cache.k_scale is not None:
        k, v = (x * c.double()[:, None] for x, c in zip((k, v), cache[2:]))
    k, v = (x.repeat_interleave(2, 1).transpose(0, 1) for x in (k, v))
    q = s.q.double().transpose(0, 1)
    scale = dim**-0.5
    hidden = torch.arange(20) > torch.arange(20 - new, 20)[:, None]
    w = (q @ k.transpose(1, 2) * scale).masked_fill(hidden, -math.inf)
    w = w.softmax(-1)
    want, size = w @ v, w @ v.abs()
    off = dim * 2.0**-24 * scale * (q.abs() @ k.abs().transpose(1, 2)).max()
    tol = u * want.abs() + (2 * u * u + 2.0**-19 + 2 * off + 2.0**-20) * size
    if dtype == torch.float16:
        tol += 20 * 2.0**-35 * size.max() + 2.0**-25
    cache, a = s.to()
    got = attend(cache, a["q"], a["table"], a["lens"])
    near(got, want.transpose(0, 1), 1.01 * tol.transpose(0, 1), "out")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cache", [None, E4M3])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 3, 16, 70])
def test_what_is_no_number_in_each_type(device, dtype, cache, dim, new):
    """Keys and values that are infinite or NaN spoil the rows that see
    them, in the dimensions that they are in, and no others; e4m3 has NaN
    only."""
    s = Step(device, [(new, 90 + new)], dtype=dtype, cache=cache, dim=dim,
             uniform=True, seed=dim + new)
    cache0, a = s.to()

    def run(k_at=(), v_at=()):
        c = PagedCache(*(None if x is None else x.clone() for x in cache0))
        for x, places in ((c.k, k_at), (c.v, v_at)):
            for j, d, value in places:
                bits = torch.tensor(value).to(x.dtype).view(
                    torch.uint8 if cache else torch.int16)
                x.view(bits.dtype)[s.slot(0, j)][:, d] = bits.to(device)
        return attend(c, a["q"], a["table"], a["lens"])

    clean = run()
    last = 90 + new - 1  # seen by the last row only
    values = (math.nan,) if cache else (math.nan, math.inf, -math.inf)
    for value in values:
        out = run(k_at=[(last, d, value) for d in range(dim)],
                  v_at=[(last, d, value) for d in range(dim)])
        assert torch.equal(out[:-1], clean[:-1])
        assert not out[-1].isfinite().any()
    spoilt = {3: values[0], 17: values[-1], dim - 1: values[len(values) // 2]}
    out = run(v_at=[(j, d, x) for j in (30, last) for d, x in spoilt.items()])
    for d, x in spoilt.items():
        assert torch.equal(out[..., d].nan_to_num(),
                           torch.full_like(out[..., d], x).nan_to_num())
        assert out[..., d].isnan().all() or not math.isnan(x)
        out[..., d] = clean[..., d]
    assert torch.equal(out, clean)


@pytest.mark.parametrize("new", [1, 6])
@pytest.mark.parametrize("dtype,less", [(torch.bfloat16, 1e-3),
                                        (torch.bfloat16, 60.0),
                                        (torch.float16, 1e-3),
                                        (torch.float16, 15.0)])
def test_infinite_values_with_little_weight(device, new, dtype, less):
    """They reach the rows that see them whatever a weight leaves behind
    its first bits: nothing at all where it is a power of two."""
    s = Step(device, [(new, 100)], dtype=dtype, uniform=True)
    s.q.zero_()
    s.cache.k.zero_()
    s.q[..., 0] = 8.0
    for j in (11, 70):
        at = s.slot(0, j)
        s.cache.k[at][:, 0] = -less
        s.cache.v[at][:, 5] = math.inf
        s.cache.v[at][:, 6] = -math.inf
    at = s.slot(0, 40)  # as much weight as the others: a power of two
    s.cache.v[at][:, 7] = math.inf
    cache, a = s.to()
    out = attend(cache, a["q"], a["table"], a["lens"])
    assert (out[..., 5] == math.inf).all() and (
        out[..., 6] == -math.inf).all() and (out[..., 7] == math.inf).all()
    assert out[..., 8:].isfinite().all()


# -- attend: buffers ---------------------------------------------------


def test_padding_rows(device):
    s = Step(device, [(3, 40), (1, 70)], pad=5)
    out = check_attend(s)
    assert not out[4:].any()
    cache, a = s.to()
    mine = torch.full_like(a["q"], 7.0)
    got, lse = attend(cache, a["q"], a["table"], a["lens"],
                      starts=a["starts"], out=mine, return_lse=True)
    assert got is mine and (mine[4:] == 7.0).all()
    assert torch.equal(mine[:4], out[:4])
    assert (lse[4:] == -math.inf).all()


@pytest.mark.parametrize("new", [1, 40])
def test_strides(device, new):
    """Rows inside a fused projection, a cache stored heads first, results
    inside a wider buffer, and a table inside a wider one."""
    s = Step(device, [(new, 70), (new, 140)], heads=8, kv_heads=2, dim=128)
    want = check_attend(s)
    cache, a = s.to()
    total = a["q"].shape[0]
    fused = torch.zeros(total, 12, 128, dtype=s.q.dtype, device=device)
    fused[:, :8] = a["q"]
    k, v = (x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
            for x in cache[:2])
    v = torch.cat((v, v), dim=-1)[..., :128]
    table = torch.cat((a["table"], a["table"]), 1)[:, :a["table"].shape[1]]
    wide = torch.zeros(total, 2, 8, 128, dtype=s.q.dtype, device=device)
    got = attend(PagedCache(k, v), fused[:, :8], table, a["lens"],
                 starts=a["starts"], out=wide[:, 1])
    assert torch.equal(got, want)
    assert not wide[:, 0].any()


@pytest.mark.parametrize("new", [1, 40, 150])
def test_out_may_be_q(device, new):
    s = Step(device, [(new, 300)], uniform=True)
    want = check_attend(s)
    cache, a = s.to()
    got = attend(cache, a["q"], a["table"], a["lens"], out=a["q"])
    assert got is a["q"] and torch.equal(got, want)


def test_strides_of_one(device):
    """What a dimension of one is strided by does not matter."""
    s = Step(device, [(1, 30)], heads=1, kv_heads=1, page=1, uniform=True)
    want = check_attend(s)
    cache, a = s.to()
    q = torch.as_strided(a["q"], (1, 1, 64), (3, 5, 1))
    k, v = (torch.as_strided(x, x.shape, (64, 7, 9, 1)) for x in cache[:2])
    got = attend(PagedCache(k, v), q, a["table"], a["lens"])
    assert torch.equal(got, want)


def test_shared_pages(device):
    """Two sequences read the same pages of a common beginning."""
    s = Step(device, [(2, 70), (5, 70)])
    s.table[1, :4] = s.table[0, :4]
    check_attend(s)


def test_no_rows(device):
    s = Step(device, [(0, 5), (0, 0)])
    cache, a = s.to()
    out, lse = attend(cache, a["q"], a["table"], a["lens"],
                      starts=a["starts"], return_lse=True)
    assert out.shape == a["q"].shape and lse.shape == (0, 4)
    assert append(cache, a["k"], a["v"], a["table"], a["lens"],
                  starts=a["starts"], q=a["q"]).shape == a["q"].shape


# -- append ------------------------------------------------------------


def append_oracle(s, rotary, interleaved, base=10000.0):
    """Queries and cache after the step, with bounds, in float64."""
    u32 = 2.0**-24

    def turn(x, pos):
        x, size = x.double().clone(), x.double().abs()
        for i in range(rotary // 2):
            a, b = ((2 * i, 2 * i + 1) if interleaved
                    else (i, i + rotary // 2))
            angle = pos * base ** (-2.0 * i / rotary)
            c, d = math.cos(angle), math.sin(angle)
            p, r = x[:, a].clone(), x[:, b].clone()
            x[:, a], x[:, b] = p * c - r * d, r * c + p * d
            size[:, a] = size[:, b] = p.abs() + r.abs()
        return x, 4 * u32 * size

    def rounded(x, off, dtype, scale=None):
        if scale is not None:
            x, off = x / scale[:, None], off / scale[:, None]
            x = x.clamp(-448, 448)
        tol = half_step(dtype) * (x.abs() + off) + off + x.abs() * u32
        return x, tol * 1.01 + (2.0**-10 if dtype == E4M3 else
                                2.0**-25 if dtype == torch.float16 else 0)

    q, q_tol = s.q.double().clone(), torch.zeros_like(s.q.double())
    seen = torch.zeros(s.q.shape[0], dtype=torch.bool)
    kc, vc = s.cache.k.double().clone(), s.cache.v.double().clone()
    k_tol, v_tol = torch.zeros_like(kc), torch.zeros_like(vc)
    scale = [None if x is None else x.double() for x in s.cache[2:]]
    capacity = s.table.shape[1] * s.page
    for row, b, pos in s.rows():
        seen[row] = True
        if not 0 <= pos < capacity:
            q[row] = 0
            continue
        q[row], q_tol[row] = rounded(*turn(s.q[row], pos), s.q.dtype)
        at = s.slot(b, pos)
        if at is not None:
            kc[at], k_tol[at] = rounded(*turn(s.k[row], pos),
                                        s.cache.k.dtype, scale[0])
            vc[at], v_tol[at] = rounded(s.v[row].double(),
                                        torch.zeros_like(s.v[row].double()),
                                        s.cache.v.dtype, scale[1])
    q[~seen] = 0
    return q, q_tol, kc, k_tol, vc, v_tol


def check_append(s, rotary=None, interleaved=False):
    cache, a = s.to()
    rotary = s.q.shape[2] if rotary is None else rotary
    rotation = None
    if rotary:
        rotation = rotation_table(s.table.shape[1] * s.page, rotary,
                                  device=s.device)
    q = append(cache, a["k"], a["v"], a["table"], a["lens"],
               starts=a["starts"], q=a["q"], rotation=rotation,
               interleaved=interleaved)
    want = append_oracle(s, rotary, interleaved)
    near(q, want[0], want[1], "q")
    near(cache.k.float(), want[2], want[3], "k")
    near(cache.v.float(), want[4], want[5], "v")
    return q, cache


@pytest.mark.parametrize("seqs", [[(1, 1)], [(1, 90)], [(7, 7)], [(33, 90)],
                                  [(1, 17), (0, 0), (64, 200), (2, 40)]])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary", [(64, 64), (128, 128), (128, 48),
                                        (256, 16), (80, 0), (96, 96)])
def test_append(device, seqs, interleaved, dim, rotary):
    check_append(Step(device, seqs, heads=6, kv_heads=2, dim=dim), rotary,
                 interleaved)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cache", [None, E4M3])
@pytest.mark.parametrize("page", [1, 16, 24])
def test_append_types(device, dtype, cache, page):
    s = Step(device, [(20, 70), (1, 30)], dtype=dtype, cache=cache,
             page=page, dim=128)
    s.v[3] *= 100  # beyond what the scale lets e4m3 hold
    check_append(s)


@pytest.mark.gpu
def test_append_many_rows(gpu):
    check_append(Step(gpu, [(401, 500), (77, 90), (1, 1)], heads=8,
                      kv_heads=2, dim=128, page=64))


def test_append_e4m3_keeps_what_is_no_number(device):
    s = Step(device, [(2, 20)], cache=E4M3)
    s.v[0, :, 5] = math.nan
    s.v[1, :, 6] = math.inf
    s.v[1, :, 7] = -math.inf
    cache, a = s.to()
    append(cache, a["k"], a["v"], a["table"], a["lens"], starts=a["starts"])
    v = cache.v.float().cpu()
    assert v[s.slot(0, 18)][:, 5].isnan().all()
    assert (v[s.slot(0, 19)][:, 6] == 448).all()
    assert (v[s.slot(0, 19)][:, 7] == -448).all()


def test_append_drops_what_has_no_page(device):
    s = Step(device, [(30, 60), (4, 2), (3, 40)], seed=8)
    s.table[0, 2] = -1
    s.table[0, 3] = 10**6
    check_append(s)
    s.lens[2] += 26  # partly behind the table
    s.seqs[2] = (3, 64 + 2)
    check_append(s)


def test_append_padding_rows(device):
    s = Step(device, [(3, 40), (1, 70)], pad=3)
    q, _ = check_append(s)
    assert not q[4:].any()
    cache, a = s.to()
    mine = torch.full_like(a["q"], 7.0)
    rotation = rotation_table(80, 64, device=device)
    append(cache, a["k"], a["v"], a["table"], a["lens"], starts=a["starts"],
           q=a["q"], q_out=mine, rotation=rotation)
    assert (mine[4:] == 7.0).all() and torch.equal(mine[:4], q[:4])


@pytest.mark.parametrize("bounds", [[0, 3, 4, 99], [0, 3, 9, 99],
                                    [5, 90, 95, 99], [0, 3, 5, 2**31 - 1],
                                    [99, 99, 99, 99]])
@pytest.mark.parametrize("max_new", [None, 2])
def test_sequences_that_pass_the_rows_have_none(device, bounds, max_new):
    """Neither operator takes their rows for a token: they are padding."""
    s = Step(device, [(3, 40), (1, 70), (2, 30)], seed=9)
    total = s.q.shape[0]
    s.bounds, s.starts = bounds, torch.tensor(bounds, dtype=torch.int32)
    s.seqs = [(hi - lo if hi <= total else 0, t) for (lo, hi), (_, t) in zip(
        zip(bounds, bounds[1:]), s.seqs)]
    used = sorted(row for row, _, _ in s.rows())
    free = [row for row in range(total) if row not in used]
    assert free
    q, _ = check_append(s)
    out = check_attend(s, max_new=max_new)
    assert not q[free].any() and not out[free].any()
    cache, a = s.to()
    for call in (lambda mine: append(
            cache, a["k"], a["v"], a["table"], a["lens"],
            starts=a["starts"], q=a["q"], q_out=mine),
            lambda mine: attend(cache, a["q"], a["table"], a["lens"],
                                starts=a["starts"], out=mine)):
        mine = torch.full_like(a["q"], 7.0)
        call(mine)
        assert (mine[free] == 7.0).all()


def test_append_in_place_and_strided(device):
    s = Step(device, [(9, 40), (2, 70)], heads=6, kv_heads=2, dim=128)
    q, cache = check_append(s)
    base, a = s.to()
    fused = torch.cat((a["q"], a["k"], a["v"]), dim=1)
    fq, fk, fv = fused.split((6, 2, 2), dim=1)
    other = PagedCache(*(x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1,
                                                                    3)
                         for x in base[:2]))
    got = append(other, fk, fv, a["table"], a["lens"], starts=a["starts"],
                 q=fq, q_out=fq,
                 rotation=rotation_table(80, 128, device=device))
    assert got is fq and torch.equal(fq, q)
    assert torch.equal(other.k, cache.k) and torch.equal(other.v, cache.v)
    assert torch.equal(fk, a["k"]) and torch.equal(fv, a["v"])


def test_append_without_queries(device):
    s = Step(device, [(9, 40)])
    cache, a = s.to()
    rotation = rotation_table(48, 64, device=device)
    assert append(cache, a["k"], a["v"], a["table"], a["lens"],
                  rotation=rotation) is None
    _, want = check_append(s)
    assert torch.equal(cache.k, want.k) and torch.equal(cache.v, want.v)


def test_rotation_of_far_positions(device):
    """Angles of a million radians, to 32 bits."""
    table = rotation_table(1 << 20, 32, device=device)
    pos = (1 << 20) - 1
    for i in (0, 3, 15):
        angle = pos * 10000.0 ** (-2.0 * i / 32)
        # The speed's own half step of 2^-53 turns the angle by 2^-33.
        assert abs(float(table[pos, i]) - math.cos(angle)) < 2.0**-24
        assert abs(float(table[pos, 16 + i]) - math.sin(angle)) < 2.0**-24


# -- both, as a session uses them --------------------------------------


def dense_session(qs, ks, vs, dim):
    """Causal attention over the whole of one sequence, float64."""
    s = qs.transpose(0, 1) @ ks.transpose(0, 1).transpose(1, 2) * dim**-0.5
    n = qs.shape[0]
    hidden = torch.ones(n, n, dtype=torch.bool).triu(1)
    return (s.masked_fill(hidden, -math.inf).softmax(-1)
            @ vs.transpose(0, 1)).transpose(0, 1)


@pytest.mark.parametrize("cache_type", [None, E4M3])
def test_session(device, cache_type):
    """Turns of unlike size for three sequences, stored and attended to step
    by step, give what attention over the whole gives."""
    g = torch.Generator().manual_seed(11)
    dim, heads, page, per_seq = 64, 2, 16, 12
    dtype = torch.float16
    cache = PagedCache.empty(40, page, heads, dim, cache_type or dtype,
                             device)
    if cache_type:
        for scale in cache[2:]:
            scale.fill_(0.02)
    table = torch.randperm(40, generator=g)[:36].view(3, 12).int().to(device)
    rotation = rotation_table(per_seq * page, dim, device=device)
    lens = torch.zeros(3, dtype=torch.int32, device=device)
    rows, got = [[], [], []], [[], [], []]
    for counts in ((37, 5, 0), (1, 1, 1), (1, 0, 90), (1, 1, 1), (70, 33, 1)):
        total = sum(counts)
        q, k, v = (torch.randn(total, heads, dim, generator=g).to(dtype)
                   for _ in range(3))
        starts = [0]
        for n in counts:
            starts.append(starts[-1] + n)
        lens += torch.tensor(counts, dtype=torch.int32, device=device)
        at = torch.tensor(starts, dtype=torch.int32, device=device)
        turned = append(cache, k.to(device), v.to(device), table, lens,
                        starts=at, q=q.to(device), rotation=rotation)
        out = attend(cache, turned, table, lens, starts=at,
                     max_new=max(counts))
        for b in range(3):
            part = slice(starts[b], starts[b + 1])
            rows[b].append((q[part], k[part], v[part]))
            got[b].append(out[part].cpu())
    for b in range(3):
        q, k, v = (torch.cat(x).double() for x in zip(*rows[b]))
        n = q.shape[0]
        speed = 10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32)
        angle = torch.arange(n, dtype=torch.float64)[:, None, None] * speed

        def turn(x):
            z = torch.complex(x[..., :32], x[..., 32:])
            z = z * torch.polar(torch.ones_like(angle), angle)
            return torch.cat((z.real, z.imag), -1)

        q, k = turn(q).to(dtype).double(), turn(k)
        if cache_type:
            k, v = ((x / 0.02).to(torch.float32).clamp(-448, 448).to(E4M3)
                    .double() * 0.02 for x in (k, v))
        else:
            k = k.to(dtype).double()
        want = dense_session(q, k, v, dim)
        # Rotated rows may be rounded to the other neighbour: with one step
        # of the stored type in keys and queries, a score of up to
        # |q||k|/8 ~ 8 moves by at most 2 * 2^-10 * 8 (16-bit), and the
        # result, a mean of values under 5, by 5 times that.  In e4m3 (a
        # step is 2^-3) only keys within 2^-22 of a border do so: none
        # here move the result beyond the same bound.
        off = (torch.cat(got[b]).double() - want).abs().max()
        assert off < 5 * 2 * 2.0**-10 * 8, float(off)


# -- streams, graphs, large caches (GPU only) --------------------------


@pytest.mark.gpu
def test_same_call_same_bits(gpu):
    for seqs in ([(1, 3000)] * 3, [(40, 700), (1, 2000)], [(200, 300)]):
        s = Step(gpu, seqs, heads=8, kv_heads=2, dim=128)
        cache, a = s.to()
        first = attend(cache, a["q"], a["table"], a["lens"],
                       starts=a["starts"])
        for _ in range(5):
            assert torch.equal(first, attend(
                cache, a["q"], a["table"], a["lens"], starts=a["starts"]))


@pytest.mark.gpu
def test_another_stream(gpu):
    s = Step(gpu, [(1, 2000), (30, 400)], heads=8, kv_heads=2, dim=128)
    want = check_attend(s)
    cache, a = s.to()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        late = a["q"].clone()
        got = attend(cache, late, a["table"], a["lens"], starts=a["starts"])
    # Two calls at once, each with a workspace of its own.
    other = attend(cache, a["q"], a["table"], a["lens"], starts=a["starts"])
    stream.synchronize()
    assert torch.equal(got, want) and torch.equal(other, want)


@pytest.mark.gpu
def test_graphs(gpu):
    """Three captured steps, replayed in turn with eager work between, follow
    lens, table and rows as they then are."""
    steps = []
    for seqs in ([(1, 901)] * 3, [(20, 170)] * 3,
                 [(1, 700), (40, 90), (3, 333)]):
        s = Step(gpu, seqs, heads=8, kv_heads=2, dim=128,
                 uniform=len(set(seqs)) == 1, seed=len(seqs[0]))
        cache, a = s.to()
        rotation = rotation_table(a["table"].shape[1] * s.page, 128,
                                  device=gpu)

        def step(cache=cache, a=a, rotation=rotation):
            q = append(cache, a["k"], a["v"], a["table"], a["lens"],
                       starts=a["starts"], q=a["q"], rotation=rotation)
            return attend(cache, q, a["table"], a["lens"],
                          starts=a["starts"])

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        steps.append((step, a, graph, out))
    for k in range(4):
        for step, a, graph, out in steps:
            a["lens"].sub_(7 * k)
            a["q"].mul_(1.25)
            a["table"].copy_(a["table"].flip(0))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, step())


@pytest.mark.gpu
def test_offsets_beyond_32_bits(gpu):
    """Pages whose values lie more than 2^32 values into the cache."""
    pages, page, heads, dim = 66000, 64, 8, 128
    assert (pages - 100) * page * heads * dim > 2**32
    cache = PagedCache.empty(pages, page, heads, dim, torch.bfloat16, gpu)
    s = Step("cpu", [(3, 200), (50, 120)], heads=8, kv_heads=8, dim=128,
             page=64)
    far = s.table.clone()
    far[far >= 0] += pages - s.cache.k.shape[0]
    base = pages - s.cache.k.shape[0]
    cache.k[base:] = s.cache.k.to(gpu)
    cache.v[base:] = s.cache.v.to(gpu)
    a = {n: getattr(s, n).to(gpu) for n in ("q", "k", "v", "lens", "starts")}
    out = attend(cache, a["q"], far.to(gpu), a["lens"], starts=a["starts"])
    want, tol, _, _ = attend_oracle(s)
    near(out, want, tol, "out")
    q = append(cache, a["k"], a["v"], far.to(gpu), a["lens"],
               starts=a["starts"], q=a["q"],
               rotation=rotation_table(256, 128, device=gpu))
    w = append_oracle(s, 128, False)
    near(q, w[0], w[1], "q")
    near(cache.k[base:], w[2], w[3], "k")
    near(cache.v[base:], w[4], w[5], "v")


@pytest.mark.gpu
@pytest.mark.parametrize("length", [2147483600, 2147483599, 2147483580])
@pytest.mark.parametrize("new", [1, 50])
@pytest.mark.parametrize("dim", [64, 128])
def test_last_positions_of_31_bits(gpu, length, new, dim):
    """Tables name up to 2^31 - 1 positions; the last tile of these ends
    beyond that."""
    s = Step(gpu, [(new, 300)], page=100, pages=5, dim=dim)
    s.table = (torch.arange(21474836, dtype=torch.int32) % 5)[None]
    s.lens = torch.tensor([length], dtype=torch.int32)
    s.seqs = [(new, length)]
    check_attend(s, window=70)
    check_append(s, rotary=0)


# -- refusals ----------------------------------------------------------


def refused(match, call):
    with pytest.raises(ValueError, match=match):
        call()


def test_refusals(device):
    s = Step(device, [(2, 30), (2, 9)], uniform=True)
    cache, a = s.to()
    q, k, v, table, lens = (a[n] for n in ("q", "k", "v", "table", "lens"))
    starts = torch.tensor([0, 2, 4], dtype=torch.int32, device=device)
    rotation = rotation_table(64, 64, device=device)

    def att(c=cache, q=q, table=table, lens=lens, **more):
        return lambda: attend(c, q, table, lens, **more)

    def app(c=cache, k=k, v=v, table=table, lens=lens, **more):
        return lambda: append(c, k, v, table, lens, **more)

    for make in (att, app):
        refused("table", make(table=table.long()))
        refused("table", make(table=table[0]))
        refused("lens", make(lens=lens.long()))
        refused("lens", make(lens=lens[:1]))
        refused("starts", make(starts=starts[:2]))
        refused("starts", make(starts=starts.float()))
        refused("cache", make(c=PagedCache(cache.k, cache.v[:1])))
        refused("cache", make(c=PagedCache(cache.k.half(), cache.v.half())))
        refused("cache", make(c=PagedCache(cache.k[0], cache.v[0])))
        refused("cache", make(c=PagedCache(cache.k[:0], cache.v[:0])))
        refused("k_scale", make(c=PagedCache(
            cache.k, cache.v, torch.ones(2, device=device), None)))
        refused("k_scale", make(c=PagedCache(cache.k.to(E4M3),
                                             cache.v.to(E4M3))))
        refused("v_scale", make(c=PagedCache(
            cache.k.to(E4M3), cache.v.to(E4M3),
            torch.ones(2, device=device), torch.ones(3, device=device))))
    refused("q: ", att(q=q[0]))
    refused("q: ", att(q=q.float()))
    refused("serve", att(q=q[:, :3]))
    refused("starts", att(q=q[:3]))
    refused("dim", att(c=PagedCache(*(x[..., :48].contiguous()
                                      for x in cache[:2])),
                       q=q[..., :48].contiguous()))
    refused("window", att(window=0))
    refused("scale", att(scale=math.nan))
    refused("scale", att(scale=1e300))
    refused("max_new", att(max_new=-1, starts=starts))
    refused("out", att(out=q[:2]))
    refused("out", att(out=q.float()))
    refused("forward only", att(q=q.clone().requires_grad_()))
    refused("v: ", app(v=v[:2]))
    refused("v: ", app(v=v[:, :1]))
    refused("q: ", app(q=q[..., :32]))
    refused("q_out", app(q_out=q))
    refused("q_out", app(q=q, q_out=q[:, :2]))
    refused("rotation", app(rotation=rotation.double()))
    refused("rotation", app(rotation=rotation[:20]))
    refused("rotation", app(rotation=rotation[:, :24]))
    refused("rotation", app(rotation=torch.cat((rotation, rotation), 1)))
    refused("forward only", app(k=k.clone().requires_grad_()))
    refused("rotary", lambda: rotation_table(4, 20))
    refused("out", att(out=q[:1].expand(4, -1, -1)))
    refused("q_out", app(q=q, q_out=q[:, :1].expand(-1, 4, -1)))
    refused("cache", app(c=PagedCache(cache.k, cache.v[:1].expand(
        *cache.k.shape))))
    held = PagedCache(cache.k.clone().requires_grad_(), cache.v)
    refused("forward only", att(c=held))
    refused("forward only", app(c=held))
    with torch.no_grad():
        attend(cache, q.clone().requires_grad_(), table, lens)


def test_rows_of_no_shape_are_refused(device):
    """Before anything is made of their dimensions."""
    s = Step(device, [(2, 30)], uniform=True)
    cache, a = s.to()
    k, v, table, lens = (a[n] for n in ("k", "v", "table", "lens"))
    for q in (a["q"][0, 0, 0], a["q"][0], a["q"][..., :0]):
        refused("wanted|cache", lambda: attend(cache, q, table, lens))
        refused("q: ", lambda: append(cache, k, v, table, lens, q=q))
    # More heads than the kernels count (and the memory of one).
    heads = k[:, :1].expand(-1, 2**30, -1)
    refused("31 bits", lambda: append(cache, k, v, table, lens, q=heads))
    refused("31 bits", lambda: attend(cache, heads, table, lens))


def test_shared_memory_is_refused(device):
    """Rows that are written where others are still read."""
    s = Step(device, [(6, 30)], uniform=True)
    cache, a = s.to()
    k, v, table, lens = (a[n] for n in ("k", "v", "table", "lens"))
    rows = torch.randn(7, 4, 64, device=device).to(s.q.dtype)
    late, early = rows[1:], rows[:-1]
    refused("out", lambda: attend(cache, late, table, lens, out=early))
    refused("q_out", lambda: append(cache, k, v, table, lens, q=late,
                                    q_out=early))
    refused("cache", lambda: append(PagedCache(cache.k, cache.k), k, v,
                                    table, lens))
    held = cache.k.view(-1, 4, 64)[:6]
    refused("out", lambda: attend(cache, a["q"], table, lens, out=held))
    refused("q_out", lambda: append(cache, k, v, table, lens, q=a["q"],
                                    q_out=held))
    refused("cache", lambda: append(cache, cache.k.view(-1, 2, 64)[:6], v,
                                    table, lens))
    refused("q_out", lambda: append(cache, k, v, table, lens, q=k, q_out=v))
    # Keys that are values too may be read.
    attend(PagedCache(cache.k, cache.k), a["q"], table, lens)


def test_scales_and_rotation_that_learn_are_refused(device):
    s = Step(device, [(2, 30)], uniform=True, cache=E4M3)
    cache, a = s.to()
    q, k, v, table, lens = (a[n] for n in ("q", "k", "v", "table", "lens"))
    rotation = rotation_table(table.shape[1] * cache.k.shape[1], 16,
                              device=device)
    for name in ("k_scale", "v_scale"):
        held = cache._replace(
            **{name: getattr(cache, name).clone().requires_grad_()})
        with pytest.raises(ValueError, match="forward only"):
            append(held, k, v, table, lens)
        with pytest.raises(ValueError, match="forward only"):
            attend(held, q, table, lens)
        with torch.no_grad():
            attend(held, q, table, lens)
    with pytest.raises(ValueError, match="forward only"):
        append(cache, k, v, table, lens, q=q,
               rotation=rotation.requires_grad_())
    with torch.no_grad():
        append(cache, k, v, table, lens, q=q, rotation=rotation)


@pytest.mark.parametrize("where", ["q", "k", "v", "k_cache", "v_cache",
                                   "k_scale", "v_scale", "rotation", "out"])
def test_forward_derivatives_are_refused(device, where):
    """A tangent would be lost, and read as a derivative of zero."""
    s = Step(device, [(2, 30)], uniform=True, cache=E4M3)
    cache, a = s.to()
    given = dict(zip(("k_cache", "v_cache", "k_scale", "v_scale"), cache),
                 q=a["q"], k=a["k"], v=a["v"], out=torch.empty_like(a["q"]),
                 rotation=rotation_table(32, 64, device=device))

    def calls(g):
        c = PagedCache(*(g[n] for n in ("k_cache", "v_cache", "k_scale",
                                        "v_scale")))
        return (lambda: attend(c, g["q"], a["table"], a["lens"],
                               out=g["out"]),
                lambda: append(c, g["k"], g["v"], a["table"], a["lens"],
                               q=g["q"], q_out=g["out"],
                               rotation=g["rotation"]))

    tangent = torch.ones(given[where].shape, device=device).to(
        given[where].dtype)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(given[where], tangent)
        for n, call in enumerate(calls({**given, where: dual})):
            if n == 0 and where in ("k", "v", "rotation"):
                continue  # attend has none
            refused("forward only", call)
            with torch.no_grad():  # leaves forward derivatives on
                refused("forward only", call)
            with torch.inference_mode():
                call()
    if where == "q":
        refused("forward only", lambda: torch.func.jvp(
            lambda q: attend(cache, q, a["table"], a["lens"]), (a["q"],),
            (tangent,)))


@pytest.mark.parametrize("where", ["k_cache", "v_cache", "q_out", "out"])
def test_autograd_sees_what_is_written(device, where):
    """What a backward pass has saved and a call overwrites is refused
    there."""
    s = Step(device, [(2, 30)], uniform=True)
    cache, a = s.to()
    mine = torch.empty_like(a["q"])
    saved = {"k_cache": cache.k, "v_cache": cache.v}.get(where, mine)

    def run():
        factor = torch.ones((), dtype=s.q.dtype, device=device,
                            requires_grad=True)
        y = (factor * saved).sum()
        if where == "out":
            attend(cache, a["q"], a["table"], a["lens"], out=mine)
        else:
            append(cache, a["k"], a["v"], a["table"], a["lens"], q=a["q"],
                   q_out=mine)
        return y

    with pytest.raises(RuntimeError, match="modified by an inplace"):
        run().backward()
    with torch.inference_mode():  # where versions are not kept
        mine = mine.clone()
        cache = PagedCache(*(x.clone() for x in cache[:2]))
        append(cache, a["k"], a["v"], a["table"], a["lens"], q=a["q"],
               q_out=mine)
        attend(cache, a["q"], a["table"], a["lens"], out=mine)


@pytest.mark.gpu
def test_refusals_of_layouts(gpu):
    s = Step(gpu, [(2, 30)], uniform=True)
    cache, a = s.to()
    q, k, v, table, lens = (a[n] for n in ("q", "k", "v", "table", "lens"))
    odd = torch.zeros(2, 4, 68, dtype=q.dtype, device=gpu)
    refused("q: ", lambda: attend(cache, odd[..., 4:], table, lens))
    refused("q: ", lambda: attend(cache, odd[..., :64], table, lens))
    turned = q.transpose(1, 2).contiguous().transpose(1, 2)
    refused("q: ", lambda: attend(cache, turned, table, lens))
    refused("out", lambda: attend(cache, q, table, lens, out=turned))
    refused("k: ", lambda: append(cache, k.transpose(1, 2).contiguous()
                                  .transpose(1, 2), v, table, lens))
    flat = PagedCache(cache.k, torch.empty(
        *cache.v.shape[:3], 68, dtype=q.dtype, device=gpu)[..., :64])
    refused("cache.v", lambda: attend(flat, q, table, lens))
    refused("device", lambda: attend(cache, q, table.cpu(), lens))
    refused("device", lambda: attend(cache, q, table, lens.cpu()))
    refused("cache", lambda: attend(PagedCache(cache.k, cache.v.cpu()), q,
                                    table, lens))
    refused("v: ", lambda: append(cache, k, v.cpu(), table, lens))
    refused("rotation", lambda: append(cache, k, v, table, lens,
                                       rotation=rotation_table(
                                           64, 64, device="cpu")))


def test_entries_refuse_what_the_kernels_cannot_take():
    """The C entries check again: no GPU is needed to be refused."""
    import ctypes

    from nvshare_amd.paths import artifacts

    lib = ctypes.CDLL(str(artifacts().hiputil))
    lib.nvs_kv_attend_work.restype = ctypes.c_int64
    zeros = bytes(512)
    assert lib.nvs_kv_append(zeros, zeros, None) == 1
    assert lib.nvs_kv_attend(zeros, zeros, None, None) == 1
    assert lib.nvs_kv_attend_work(zeros, zeros) == -1
    assert lib.nvs_kv_append(None, None, None) == 1
