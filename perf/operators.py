"""The paged key/value cache's operators, as cases to measure.

Two operators of a serving step are measured here, each at the sizes that
an inference client meets between its first prompt and a long session:

  append   stores a step's new keys and values in the pages of the cache
           and rotates the new queries and keys by their positions on the
           way;
  attend   lets the step's new queries attend to everything that their
           sequence has in the cache, the new tokens included.

`own` chooses between the plain form of each, written with elementary torch
operations in 32 bits, and the calls of nvshare_amd.kvcache.
"""

from __future__ import annotations

import math
import random

import torch

own = False

E4M3_MAX = 448.0


def _case(name, op, **more):
    case = {"name": name, "op": op, "type": "bfloat16", "cache": "same",
            "batch": 1, "new": 1, "context": 0, "ragged": False,
            "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
            "window": 0, "rotary": 128, "interleaved": False}
    case.update(more)
    return case


def listed():
    return [
        # The next token of a lone interactive session: all latency.
        _case("append, one token", "append", context=203),
        # A full batch of sessions generating into an 8-bit cache.
        _case("append, batch of 64, e4m3", "append", cache="e4m3", batch=64,
              context=211, ragged=True, page=32),
        # Short drafts of a small model with pair-wise, partial rotation.
        _case("append, drafts, fp16", "append", type="float16", batch=16,
              new=33, context=150, heads=14, kv_heads=2, dim=64, page=8,
              rotary=32, interleaved=True),
        # Prompts of several sessions at once, of unlike lengths.
        _case("append, ragged prompts", "append", batch=9, new=4001,
              ragged=True, context=130, page=64),
        # The next token of a lone session that has just begun.
        _case("attend, one token, short", "attend", context=610),
        # The next token after a whole book: one sequence fills the card.
        _case("attend, one token, long", "attend", context=120000, page=64),
        # A full batch of sessions of every age, one token each.
        _case("attend, batch of 64", "attend", batch=64, context=16383,
              ragged=True),
        # The same from an 8-bit cache, with more heads to a cached one.
        _case("attend, batch of 32, e4m3", "attend", cache="e4m3", batch=32,
              context=32000, ragged=True, heads=64, page=32),
        # Drafted tokens that are checked in one step, small heads.
        _case("attend, drafts, fp16", "attend", type="float16", batch=8,
              new=6, context=5003, heads=16, kv_heads=4, dim=64, rotary=64),
        # A chunk of a long prompt over what earlier chunks have stored.
        _case("attend, chunk over long context", "attend", new=2048,
              context=30001, page=64),
        # Prompts from their first token, mixed with generating sessions.
        _case("attend, ragged prompts", "attend", batch=6, new=4096,
              context=300, ragged=True, page=32),
        # A sliding window, wide heads, a chunk that begins mid-page.
        _case("attend, window, dim 256", "attend", type="float16", batch=2,
              new=1500, context=7003, heads=8, kv_heads=4, dim=256,
              page=128, window=1024, rotary=256),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    most = {op: max(_cost(c) for c in listed() if c["op"] == op)
            for op in ("append", "attend")}
    while True:
        op = rng.choice(("append", "attend", "attend"))
        kv_heads = rng.choice((1, 2, 4, 5, 8))
        dim = rng.choice((64, 128, 128, 256))
        step = rng.choice(("token", "token", "draft", "chunk"))
        case = _case(
            "", op, type=rng.choice(("bfloat16", "float16")),
            cache=rng.choice(("same", "same", "e4m3")),
            batch=_log(rng, 1, 64 if step != "chunk" else 8),
            new={"token": 1, "draft": rng.randint(2, 40),
                 "chunk": _log(rng, 41, 4096)}[step],
            context=(rng.randint(0, 255) if op == "append"
                     else _log(rng, 1, 120000) - 1),
            ragged=rng.random() < 0.5,
            kv_heads=kv_heads, heads=kv_heads * rng.choice((1, 4, 7, 8)),
            dim=dim, page=rng.choice((8, 16, 32, 64, 128)),
            window=rng.choice((0, 0, 0, _log(rng, 16, 8192))),
            rotary=rng.choice((dim, dim // 2)),
            interleaved=rng.random() < 0.3)
        del case["name"]
        if _cost(case) <= most[op] and _room(case) <= 1 << 31:
            return case


def _sequences(case):
    """[(tokens that are new, tokens in all)] of the batch, by the case alone."""
    new, context = case["new"], case["context"]
    if not case["ragged"]:
        return [(new, context + new)] * case["batch"]
    rng = random.Random("%d %d %d" % (case["batch"], new, context))
    got = []
    for b in range(case["batch"]):
        # Every third sequence generates, and one in a large batch waits.
        n = 1 if b % 3 == 2 else rng.randint((new + 1) // 2, new)
        n = 0 if b == 4 else n
        got.append((n, n + rng.randint(0, context)))
    return got


def _seen(case):
    """(query-key pairs, cached tokens that some query sees) of the batch."""
    pairs = tokens = 0
    for new, length in _sequences(case):
        width = case["window"] or length
        first = length - new  # the position of the first new token
        # Token i sees min(first + i + 1, width) keys.
        short = min(new, max(0, width - first))  # tokens that see all so far
        pairs += short * first + short * (short + 1) // 2
        pairs += (new - short) * width
        tokens += length - max(0, first + 1 - width) if new else 0
    return pairs, tokens


def work(case):
    total = sum(n for n, _ in _sequences(case))
    size = 1 if case["cache"] == "e4m3" else 2
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "append":
        rotated = total * (heads + kv_heads) * case["rotary"]
        return {"bytes": total * dim * (4 * heads + 2 * kv_heads * (2 + size))
                + total * 4 * case["rotary"],
                "flops": 3 * rotated}
    pairs, tokens = _seen(case)
    return {"bytes": total * heads * dim * 4
            + 2 * tokens * kv_heads * dim * size,
            "flops": 4 * pairs * heads * dim}


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def _room(case):
    """Values in the largest tensor of the plain form."""
    if case["op"] == "append":
        return 0
    new = max(n for n, _ in _sequences(case))
    length = max(t for _, t in _sequences(case))
    return case["batch"] * length * max(new * case["heads"],
                                        case["kv_heads"] * case["dim"])


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype = getattr(torch, case["type"])
    dev = torch.device("cuda")
    seqs = _sequences(case)
    batch, page = case["batch"], case["page"]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    total = sum(n for n, _ in seqs)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=dtype)

    # One projection makes queries, keys and values side by side.
    qkv = normal(total, heads + 2 * kv_heads, dim)
    q, k, v = qkv.split((heads, kv_heads, kv_heads), dim=1)

    need = [-(-t // page) for _, t in seqs]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device=dev,
                           dtype=torch.int64).to(torch.int32)
    per_seq = max(max(need), 1)
    table = torch.full((batch, per_seq), -1, dtype=torch.int32)
    at, slots = 0, torch.arange(sum(need), dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = slots[at:at + n]
        at += n
    table = table.to(dev)
    table = torch.where(table < 0, table, order[table.clamp(min=0).long()])

    state = {"case": case, "q": q, "k": k, "v": v, "table": table,
             "most_new": max(n for n, _ in seqs),
             "most": max(t for _, t in seqs), "k_scale": None,
             "v_scale": None, "starts": None}
    state["lens"] = torch.tensor([t for _, t in seqs], dtype=torch.int32,
                                 device=dev)
    starts = [0]
    for n, _ in seqs:
        starts.append(starts[-1] + n)
    state["row_starts"] = torch.tensor(starts, dtype=torch.int32, device=dev)
    if case["ragged"]:
        state["starts"] = state["row_starts"]

    kc = normal(pages, page, kv_heads, dim)
    vc = normal(pages, page, kv_heads, dim)
    if case["cache"] == "e4m3":
        # Scales such as a calibration gives: the largest value is near 448.
        low = torch.rand(2, kv_heads, generator=g, device=dev)
        state["k_scale"], state["v_scale"] = (0.01 + 0.02 * low).unbind(0)
        kc = (kc.float() / state["k_scale"][:, None]).clamp(
            -E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
        vc = (vc.float() / state["v_scale"][:, None]).clamp(
            -E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    state["k_cache"], state["v_cache"] = kc, vc

    if case["op"] == "append":
        half = case["rotary"] // 2
        turn = 10000.0 ** (-torch.arange(half, dtype=torch.float64,
                                         device=dev) / half)
        angle = torch.arange(per_seq * page, dtype=torch.float64,
                             device=dev)[:, None] * turn
        state["rotation"] = torch.cat((angle.cos(), angle.sin()), 1).float()
    return state


def run(s):
    if s["case"]["op"] == "append":
        return _append(s)
    return _attend(s)


def _append(s):
    case = s["case"]
    if own:
        from nvshare_amd import kvcache

        cache = kvcache.PagedCache(s["k_cache"], s["v_cache"], s["k_scale"],
                                   s["v_scale"])
        q = kvcache.append(cache, s["k"], s["v"], s["table"], s["lens"],
                           starts=s["starts"], q=s["q"],
                           rotation=s["rotation"],
                           interleaved=case["interleaved"])
        return {"q": q, "k_cache": cache.k, "v_cache": cache.v}

    seq, pos = _places(s)
    cos, sin = s["rotation"][pos].chunk(2, dim=1)
    q = _rotate(s["q"].float(), cos, sin, case).to(s["q"].dtype)
    k = _rotate(s["k"].float(), cos, sin, case)
    page = s["table"][seq, pos // case["page"]].long()
    slot = pos % case["page"]
    _store(s["k_cache"], page, slot, k, s["k_scale"])
    _store(s["v_cache"], page, slot, s["v"].float(), s["v_scale"])
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _places(s):
    """The sequence and the position of each new token."""
    row = torch.arange(s["q"].shape[0], device=s["q"].device)
    starts = s["row_starts"].long()
    seq = torch.searchsorted(starts, row, right=True) - 1
    return seq, s["lens"].long()[seq] - starts[seq + 1] + row


def _rotate(x, cos, sin, case):
    rotary = case["rotary"]
    part = x[..., :rotary]
    cos, sin = cos[:, None], sin[:, None]
    if case["interleaved"]:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin),
                             dim=-1).flatten(-2)
    else:
        a, b = part.chunk(2, dim=-1)
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, x[..., rotary:]), dim=-1)


def _store(cache, page, slot, x, scale):
    if scale is None:
        cache[page, slot] = x.to(cache.dtype)
        return
    x = (x / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(cache.dtype)
    cache.view(torch.uint8)[page, slot] = x.view(torch.uint8)


def _attend(s):
    case = s["case"]
    window = case["window"] or None
    if own:
        from nvshare_amd import kvcache

        cache = kvcache.PagedCache(s["k_cache"], s["v_cache"], s["k_scale"],
                                   s["v_scale"])
        return kvcache.attend(cache, s["q"], s["table"], s["lens"],
                              starts=s["starts"], window=window,
                              max_new=s["most_new"])

    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    batch, new, most = case["batch"], s["most_new"], s["most"]
    group = heads // kv_heads
    dev = s["q"].device
    starts, lens = s["row_starts"].long(), s["lens"].long()

    # Queries, one padded row of `new` tokens to a sequence.
    seq, pos = _places(s)
    at = torch.arange(s["q"].shape[0], device=dev) - starts[seq]
    q = torch.zeros(batch, new, heads, dim, device=dev)
    q[seq, at] = s["q"].float() / math.sqrt(dim)
    q = q.view(batch, new, kv_heads, group, dim).permute(0, 2, 3, 1, 4)
    q = q.reshape(batch, kv_heads, group * new, dim)

    table = s["table"].clamp(min=0).long()
    k = _gather(s["k_cache"], table, most, s["k_scale"])
    scores = q @ k.transpose(2, 3)
    del k

    key = torch.arange(most, device=dev)
    count = starts[1:] - starts[:-1]
    query = (lens - count)[:, None] + torch.arange(new, device=dev)
    seen = (key <= query[:, :, None]) & (key < lens[:, None, None])
    if window is not None:
        seen &= key > query[:, :, None] - window
    scores = scores.view(batch, kv_heads, group, new, most)
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    weight = scores.sub_(top).exp_()
    total = weight.sum(-1, keepdim=True)

    v = _gather(s["v_cache"], table, most, s["v_scale"])
    out = weight.view(batch, kv_heads, group * new, most) @ v
    out = out.view(batch, kv_heads, group, new, dim)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    out = out.permute(0, 3, 1, 2, 4).reshape(batch, new, heads, dim)
    return out[seq, at].to(s["q"].dtype)


def _gather(cache, table, most, scale):
    """[batch, kv_heads, most, dim] in 32 bits."""
    if scale is None:
        x = cache[table].float()
    else:
        x = cache.view(torch.uint8)[table].view(cache.dtype).float()
        x = x * scale[:, None]
    return x.flatten(1, 2)[:, :most].transpose(1, 2).contiguous()


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(case, s)
    return _exact_attend(case, s)


def _exact_append(case, s):
    """Turns each pair as a complex number, one sequence after the other."""
    rotary, half, page = case["rotary"], case["rotary"] // 2, case["page"]
    dev = s["q"].device
    index = torch.arange(half, dtype=torch.float64, device=dev)
    speed = torch.exp(index * (-math.log(10000.0) / half))
    if case["interleaved"]:
        first = 2 * torch.arange(half, device=dev)
        second = first + 1
    else:
        first = torch.arange(half, device=dev)
        second = first + half

    def turned(x, pos):
        x = x.double()
        angle = pos.double()[:, None, None] * speed
        z = torch.complex(x[..., first], x[..., second])
        z = z * torch.polar(torch.ones_like(angle), angle)
        x[..., first], x[..., second] = z.real, z.imag
        return x

    q = s["q"].double()
    caches = {n: s[n + "_cache"].double() for n in ("k", "v")}
    row = 0
    for b, (new, length) in enumerate(_sequences(case)):
        pos = torch.arange(length - new, length, device=dev)
        rows = slice(row, row + new)
        q[rows] = turned(s["q"][rows], pos)
        for n, x in (("k", turned(s["k"][rows], pos)),
                     ("v", s["v"][rows].double())):
            scale = s[n + "_scale"]
            if scale is not None:
                x = (x / scale.double()[:, None]).clamp(-E4M3_MAX, E4M3_MAX)
            flat = caches[n].view(-1, *x.shape[1:])
            flat[s["table"][b].long()[pos // page] * page + pos % page] = x
        row += new
    return {"q": q, "k_cache": caches["k"], "v_cache": caches["v"]}


def _exact_attend(case, s):
    """One sequence, one cached head and 1024 tokens at a time."""
    pairs, _ = _seen(case)
    if pairs * case["heads"] * case["dim"] > 2e12:
        return None  # minutes in 64 bits
    group = case["heads"] // case["kv_heads"]
    dev, page = s["q"].device, case["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=dev)
    row = 0
    for b, (new, length) in enumerate(_sequences(case)):
        if not new:
            continue
        key = torch.arange(length, device=dev)
        where = s["table"][b].long()[key // page]
        for h in range(case["kv_heads"]):
            k = s["k_cache"][where, key % page, h].double()
            v = s["v_cache"][where, key % page, h].double()
            if s["k_scale"] is not None:
                k = k * s["k_scale"][h].double()
                v = v * s["v_scale"][h].double()
            for i in range(0, new, 1024):
                n = min(1024, new - i)
                pos = torch.arange(length - new + i, length - new + i + n,
                                   device=dev)
                hidden = key[None] > pos[:, None]
                if case["window"]:
                    hidden |= pos[:, None] - key[None] >= case["window"]
                for j in range(h * group, (h + 1) * group):
                    x = s["q"][row + i:row + i + n, j].double()
                    x = x @ k.t() * dim_scale(case)
                    x = x.masked_fill(hidden, -math.inf).softmax(-1)
                    out[row + i:row + i + n, j] = x @ v
        row += new
    return out


def dim_scale(case):
    return case["dim"] ** -0.5
