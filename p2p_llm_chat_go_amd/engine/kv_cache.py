"""Paged KV cache sized from free HBM.

Layout (one tensor for K, one for V, all layers):
    [n_layers, num_pages, n_kv_heads_local, PAGE=64, head_dim=128] bf16
One page of one kv head is a contiguous 16 KiB tile (what a decode-attention
wave streams).  Page 0 is reserved as the *null page*: padding rows of a
graph batch bucket write and read there, so bucketed graphs never touch a
live sequence.

Sequences may share pages: :meth:`KVCache.fork` gives a new sequence the full pages of the tokens it begins with and a
copy of the page that both go on writing to; a page returns to the free list when its last owner frees it.
:meth:`KVCache.compact` moves the tokens that a sequence keeps together and frees the pages behind them.

On a 288 GB MI355X, llama3.1-8B leaves ~270 GB for KV = ~2.1 M tokens at
128 KiB/token; the default fraction below keeps headroom for workspaces.
"""
from __future__ import annotations

import collections

import torch

from ..models.config import ModelConfig
from ..ops import HEAD_DIM, PAGE, compact_pages, copy_pages


class PageAllocator:
    """Free-list page allocator (page 0 reserved).  The C++ runtime has the same
    allocator for the scheduler (``_native.BlockAllocator``); this Python one is
    used when the native module is not built (CPU tests)."""

    def __init__(self, num_pages: int):
        if num_pages < 2:
            raise ValueError("need at least 2 pages (page 0 is the null page)")
        self.num_pages = num_pages
        self._free = list(range(num_pages - 1, 0, -1))
        self._owners = [0] * num_pages      # of every page; 0: free

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def shared(self, page: int) -> bool:
        """Whether more than one sequence owns the page."""
        return self._owners[page] > 1

    def owners(self, page: int) -> int:
        """How many sequences own a page (0: it is free)."""
        return self._owners[page]

    def check(self, pages):
        """Raises where one of them is no page that a sequence can own, or free."""
        for p in pages:
            if p <= 0 or p >= self.num_pages:
                raise ValueError("bad page %d" % p)
            if not self._owners[p]:
                raise ValueError("page %d is free" % p)

    def share(self, pages):
        """One more owner for each of the pages (which are in use); each owner frees them once."""
        self.check(pages)
        for p in pages:
            self._owners[p] += 1

    def alloc(self, n: int) -> list:
        if n > len(self._free):
            raise MemoryError("KV cache exhausted: want %d pages, %d free" % (n, len(self._free)))
        out = [self._free.pop() for _ in range(n)]
        for p in out:
            self._owners[p] = 1
        return out

    def free(self, pages):
        """Each of the pages loses an owner; nothing has changed where one of them cannot."""
        self.check(pages)
        for p, n in collections.Counter(pages).items():
            if n > self._owners[p]:
                raise ValueError("page %d is freed more often than it is owned" % p)
        for p in pages:
            self._owners[p] -= 1
            if not self._owners[p]:
                self._free.append(p)


def pages_for(tokens: int) -> int:
    return (tokens + PAGE - 1) // PAGE


class KVCache:
    def __init__(self, cfg: ModelConfig, num_pages: int, device, tp_size: int = 1,
                 dtype=torch.bfloat16):
        assert cfg.head_dim == HEAD_DIM
        self.cfg = cfg
        self.num_pages = num_pages
        self.n_kv_local = cfg.n_kv_heads // tp_size
        shape = (cfg.n_layers, num_pages, self.n_kv_local, PAGE, HEAD_DIM)
        self.k = torch.zeros(shape, device=device, dtype=dtype)
        self.v = torch.zeros(shape, device=device, dtype=dtype)
        self.allocator = PageAllocator(num_pages)

    @staticmethod
    def bytes_per_page(cfg: ModelConfig, tp_size: int = 1) -> int:
        return 2 * cfg.n_layers * (cfg.n_kv_heads // tp_size) * PAGE * HEAD_DIM * 2

    @classmethod
    def from_free_memory(cls, cfg: ModelConfig, device, fraction: float = 0.85, tp_size: int = 1,
                         max_pages: int | None = None, reserve_bytes: int = 4 << 30):
        dev = torch.device(device)
        if dev.type == "cuda":
            free, _total = torch.cuda.mem_get_info(dev)
            budget = max(0, int((free - reserve_bytes) * fraction))
        else:
            budget = 256 << 20
        n = max(2, budget // cls.bytes_per_page(cfg, tp_size))
        if max_pages:
            n = min(n, max_pages)
        return cls(cfg, int(n), dev, tp_size)

    def layer(self, i: int):
        return self.k[i], self.v[i]

    def fork(self, pages: list, tokens: int, sizes: list) -> list:
        """Page lists of ``len(sizes)`` new sequences that begin with the first ``tokens`` tokens of ``pages``, of sizes[i]
        pages each.  Full pages of those tokens are shared; of a last page that is not full every new sequence gets a copy
        (``ops.copy_pages``, all layers in one launch).  Whoever goes on writing to ``pages`` does so behind ``tokens``."""
        if not 0 <= tokens <= len(pages) * PAGE:
            raise ValueError("fork: %d tokens of %d pages" % (tokens, len(pages)))
        full, need = tokens // PAGE, pages_for(tokens)
        if any(n < need for n in sizes):
            raise ValueError("fork: %d tokens take %d pages, asked for %d" % (tokens, need, min(sizes)))
        self.allocator.check(pages[:need])
        if len(set(pages[:need])) < need:
            raise ValueError("fork: a page is given twice")
        copy_pages(self.k, self.v, [], [])      # what the copies would refuse: nothing has changed yet
        fresh = self.allocator.alloc(sum(n - full for n in sizes))
        out, at = [], 0
        for n in sizes:
            self.allocator.share(pages[:full])
            out.append(list(pages[:full]) + fresh[at:at + n - full])
            at += n - full
        if need > full:
            copy_pages(self.k, self.v, [pages[full]] * len(out), [p[full] for p in out], [tokens % PAGE] * len(out))
        return out

    def compact(self, pages: list, lens: list, keep, cos_sin=None, room: int = 0) -> tuple:
        """Sequences (their page lists and lengths) reduced to the tokens that ``keep`` ([sequences, tokens], true or false)
        keeps: (page lists, lengths) of what is left, with pages for ``room`` more tokens each.

        A sequence whose pages are its own is compacted in place, one that shares pages with others (``fork``) into new
        ones; pages that nobody owns any more are free.

        cos_sin (``LlamaModel.rope``): keys are turned to their new positions, and the sequence goes on at its new length:
        ``Engine.prefill`` (starts) and decode steps, which take a token's rotation, slot and context from one position, need
        it so.  None: keys stay as they are; the next tokens' rotations count on from the old length while their slots and
        contexts count from the new one, which ``LlamaModel.forward`` takes apart (pos; slots, ctx_lens) and the engine's
        calls do not."""
        keep = torch.as_tensor(keep, dtype=torch.bool)
        if keep.dim() != 2 or keep.shape[0] != len(pages) or len(lens) != len(pages):
            raise ValueError("compact: %d sequences, %d lengths, keep %s" % (len(pages), len(lens), list(keep.shape)))
        for p, n in zip(pages, lens):
            if not 0 <= n <= min(len(p) * PAGE, keep.shape[1]):
                raise ValueError("compact: a length of %d with %d pages and %d places in keep" % (n, len(p), keep.shape[1]))
        if room < 0:
            raise ValueError("compact: room for %d tokens" % room)
        given = collections.Counter(p for q in pages for p in q)
        self.allocator.check(given)
        if any(len(set(q)) < len(q) for q in pages) or any(n > self.allocator.owners(p) for p, n in given.items()):
            raise ValueError("compact: a page is given twice, or by more sequences than own it")
        if not pages:
            return [], []
        lens_t = torch.tensor(lens, dtype=torch.int32)
        host = keep.cpu()
        left = (host & (torch.arange(host.shape[1]) < lens_t[:, None])).sum(1).tolist()
        size = [pages_for(n + room) for n in left]
        apart = [any(self.allocator.shared(p) for p in q) for q in pages]
        # what the moves would refuse, then the new pages: nothing has changed where either fails
        dev = self.k.device
        none = torch.zeros(0, max(map(len, pages)), dtype=torch.int32, device=dev)
        keep = keep.to(dev)
        compact_pages(self.k, self.v, none, none.new_zeros(0), keep[:0], cos_sin=cos_sin)
        fresh = self.allocator.alloc(sum(n if a else max(0, n - len(q)) for n, a, q in zip(size, apart, pages)))
        out, gone = [], []
        for n, a, q in zip(size, apart, pages):
            take = n if a else max(0, n - len(q))
            mine, fresh = fresh[:take], fresh[take:]
            out.append(mine if a else q[:n] + mine)
            gone += q if a else q[n:]
        for way in (False, True):
            at = [i for i, a in enumerate(apart) if a == way and lens[i]]
            if not at:
                continue
            width = max(len(pages[i]) for i in at)
            table = torch.zeros(2, len(at), width, dtype=torch.int32)
            for j, i in enumerate(at):
                table[0, j, :len(pages[i])] = torch.tensor(pages[i], dtype=torch.int32)
                here = out[i][:width]
                table[1, j, :len(here)] = torch.tensor(here, dtype=torch.int32)
            table = table.to(dev)
            compact_pages(self.k, self.v, table[0], lens_t[at].to(dev), keep[torch.tensor(at, device=dev)],
                          out_tables=table[1] if way else None, cos_sin=cos_sin)
        self.allocator.free(gone)
        return out, left
