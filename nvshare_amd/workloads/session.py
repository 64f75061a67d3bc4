"""Chat-like sessions over a paged key/value cache, for infer_burst.

What such a client holds while its user thinks is its sessions' cache, so
that is what a preempted client has paged out and back.  The model is the
part of a decoder that touches the cache: layers of attention with their
projections, random-init weights, random tokens.  Each turn appends a chunk
of new tokens to every session and then generates one token at a time; the
cache is fingerprinted before a pause and after it, and at the end one
answer is checked against plain torch.
"""

from __future__ import annotations

import torch
from torch import nn

from nvshare_amd import kvcache
from nvshare_amd.workloads.common import die


class Attention(nn.Module):
    """Normalised rows through one layer's attention, added to the rows."""

    def __init__(self, heads: int, kv_heads: int, dim: int):
        super().__init__()
        width = heads * dim
        self.split = (heads, kv_heads, kv_heads)
        self.dim = dim
        self.norm = nn.LayerNorm(width)
        self.qkv = nn.Linear(width, (heads + 2 * kv_heads) * dim, bias=False)
        self.out = nn.Linear(width, width, bias=False)

    def forward(self, x, cache, table, lens, rotation):
        qkv = self.qkv(self.norm(x)).view(x.shape[0], -1, self.dim)
        q, k, v = qkv.split(self.split, dim=1)
        q = kvcache.append(cache, k, v, table, lens, q=q, rotation=rotation)
        y = kvcache.attend(cache, q, table, lens)
        return x + self.out(y.flatten(1)), q, y


class Sessions(nn.Module):
    """`batch` sessions of up to `tokens` tokens each."""

    def __init__(self, batch: int, tokens: int, layers: int = 4,
                 heads: int = 32, kv_heads: int = 8, dim: int = 128,
                 page: int = 64, cache: str = "same",
                 dtype: str = "bfloat16", device: str = "cuda"):
        super().__init__()
        self.dtype = getattr(torch, dtype)
        self.device = torch.device(device)
        self.layers = nn.ModuleList(
            Attention(heads, kv_heads, dim) for _ in range(layers))
        self.to(self.device, self.dtype)
        held = torch.float8_e4m3fn if cache == "e4m3" else self.dtype
        per_seq = -(-tokens // page)
        self.caches = [
            kvcache.PagedCache.empty(batch * per_seq, page, kv_heads, dim,
                                     held, self.device)
            for _ in range(layers)]
        self.table = torch.randperm(batch * per_seq, dtype=torch.int32).view(
            batch, per_seq).to(self.device)
        self.lens = torch.zeros(batch, dtype=torch.int32,
                                device=self.device)
        self.rotation = kvcache.rotation_table(per_seq * page, dim,
                                               device=self.device)
        self.width, self.batch, self.tokens = heads * dim, batch, 0
        self.answer = None
        # What a word of a row, and a row of a session, count for.
        g = torch.Generator().manual_seed(0)
        words = kv_heads * dim * held.itemsize // 4
        self.place, self.position = (
            torch.randint(-2**62, 2**62, n, generator=g).mul_(2).add_(1).to(
                self.device) for n in ((words,), (batch, per_seq * page)))

    @torch.no_grad()
    def step(self, new: int) -> torch.Tensor:
        """`new` more tokens of each session through all layers."""
        x = torch.randn(self.batch * new, self.width, dtype=self.dtype,
                        device=self.device)
        self.lens += new
        self.tokens += new
        for layer, cache in zip(self.layers, self.caches):
            x, q, y = layer(x, cache, self.table, self.lens, self.rotation)
        self.answer = (new, q, y)
        return x

    def fingerprint(self) -> list[int]:
        """A sum over all that the sessions have stored, for each cache, in
        which a word counts by the session, position and place in the row
        that it is at: odd random factors, so that a changed bit always
        shows, and exchanged rows or pages do."""
        page = self.caches[0].k.shape[1]
        got = []
        for cache in self.caches:
            for x in (cache.k, cache.v):
                total = torch.zeros((), dtype=torch.int64,
                                    device=self.device)
                for b in range(self.batch):
                    for at in range(0, self.tokens, 64 * page):
                        # The last page's unwritten slots hold anything.
                        end = min(at + 64 * page, self.tokens)
                        used = self.table[b, at // page:-(-end // page)]
                        bits = x.view(torch.uint8)[used.long()]
                        bits = bits.flatten(2).view(torch.int32).flatten(0, 1)
                        rows = (bits[:end - at] * self.place).sum(-1)
                        total += (rows * self.position[b, at:end]).sum()
                got.append(int(total))
        return got

    def check(self) -> float:
        """Die unless the last layer's answer for the first session is what
        plain torch gives; the largest difference."""
        new, q, y = self.answer
        cache = kvcache.PagedCache(*(
            None if t is None else t.cpu() for t in self.caches[-1]))
        want = kvcache.attend(cache, q[:new].cpu(), self.table[:1].cpu(),
                              self.lens[:1].cpu())
        off = float((y[:new].cpu().float() - want.float()).abs().max())
        # Weights and results are rounded once on either side.
        v = cache.v[self.table[0].long().cpu()].flatten(0, 1)[:self.tokens]
        most = float(want.float().abs().max() + v.float().abs().max())
        step = torch.finfo(self.dtype).eps / 2
        if not off <= 2 * step * most:
            die(f"session: answers are {off} off")
        return off
