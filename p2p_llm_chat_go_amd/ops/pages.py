"""Pages of the K/V cache that change their place (csrc/kernels/page_moves.hip): copies and compaction, all layers at once.

A cache is ``[layers, pages, kv heads, PAGE, HEAD_DIM]`` for K and the same for V (``engine/kv_cache.py``; a part of the
layers, pages or heads of one may be given).  ``KVCache.fork`` and ``KVCache.compact`` are these with the pages' owners kept.
"""
from __future__ import annotations

import array
import ctypes

import torch

from . import _lib
from .attention import HEAD_DIM, PAGE


def _caches(k: torch.Tensor, v: torch.Tensor, what: str):
    """What the calls take of two caches: addresses, strides in bytes between layers, pages and heads of k, then of v, layers,
    heads, pages, bytes of a token's row; and their device's index (-1: not a GPU's)."""
    shape, strides, dev, size = k.shape, k.stride() + v.stride(), k.get_device(), k.element_size()
    if len(shape) != 5 or len(strides) != 10 or shape[3] != PAGE or shape[4] != HEAD_DIM:
        raise ValueError("%s: k and v must be [layers, pages, kv heads, %d, %d], got %s and %s"
                         % (what, PAGE, HEAD_DIM, list(shape), list(v.shape)))
    if shape != v.shape or k.dtype != v.dtype or dev != v.get_device() or (dev < 0 and k.device != v.device):
        raise ValueError("%s: k and v differ in shape, type or device" % what)
    if size not in (1, 2, 4) or k.is_complex():
        raise ValueError("%s: k and v have numbers of type %s" % (what, k.dtype))
    kl, kp, kh, kt, k1, vl, vp, vh, vt, v1 = strides
    ka, va = k.data_ptr(), v.data_ptr()
    if k1 != 1 or v1 != 1 or kt != HEAD_DIM or vt != HEAD_DIM or (kl | kp | kh | vl | vp | vh) * size % 16 or (ka | va) % 16:
        raise ValueError("%s: the tokens of a page must be contiguous and start at multiples of 16 bytes" % what)
    layers, pages, heads = shape[:3]
    if not (kl and kp and kh and vl and vp and vh) and any(n > 1 and not (a and b)
                                                           for n, a, b in ((layers, kl, vl), (pages, kp, vp), (heads, kh, vh))):
        raise ValueError("%s: layers, pages and heads must have memory of their own" % what)
    return (ka, va, _SIX(kl * size, kp * size, kh * size, vl * size, vp * size, vh * size), layers, heads, pages,
            HEAD_DIM * size), dev


_SIX = ctypes.c_long * 6
FAR = 2 ** 31          # strides of tables are below


def _ints(x, what: str) -> array.array:
    if isinstance(x, torch.Tensor):
        if x.device.type != "cpu":
            raise ValueError("copy_pages: %s are host numbers (a list or a CPU tensor)" % what)
        x = x.tolist()
    try:
        return array.array("i", x)
    except (TypeError, OverflowError):
        raise ValueError("copy_pages: %s must be whole numbers" % what) from None


def copy_pages(k: torch.Tensor, v: torch.Tensor, src, dst, tokens=None) -> None:
    """Pages ``src[i]`` of k and v to pages ``dst[i]``, in every layer and head.

    src, dst, tokens: host numbers, as allocators give them.  tokens: how many of a page's tokens are copied (None: all); the
    others of the page stay.  A page is in dst once at most and then not in src (but ``src[i] == dst[i]`` is nothing to do)."""
    caches, dev = _caches(k, v, "copy_pages")
    src, dst = _ints(src, "src"), _ints(dst, "dst")
    tokens = array.array("i", [PAGE]) * len(src) if tokens is None else _ints(tokens, "tokens")
    if not len(src) == len(dst) == len(tokens):
        raise ValueError("copy_pages: %d pages to %d, %d numbers of tokens" % (len(src), len(dst), len(tokens)))
    if not src:
        return
    P = caches[5]
    if min(min(src), min(dst)) < 0 or max(max(src), max(dst)) >= P:
        raise ValueError("copy_pages: pages must be 0 .. %d" % (P - 1))
    if min(tokens) < 0 or max(tokens) > PAGE:
        raise ValueError("copy_pages: tokens must be 0 .. %d" % PAGE)
    to = set(dst)
    if len(to) != len(dst):
        raise ValueError("copy_pages: a page is in dst twice")
    if not to.isdisjoint(src) and not {d for s, d in zip(src, dst) if s != d}.isdisjoint(src):
        raise ValueError("copy_pages: a page is in src and in dst")
    if caches[3] == 0 or caches[4] == 0:
        return
    if dev < 0:
        for s, d, n in zip(src, dst, tokens):
            k[:, d, :, :n] = k[:, s, :, :n]
            v[:, d, :, :n] = v[:, s, :, :n]
        return
    with _lib.device_of(dev):
        _lib.check(_lib.lib().p2p_copy_pages(
            *caches, src.buffer_info()[0], dst.buffer_info()[0], tokens.buffer_info()[0], len(src),
            torch._C._cuda_getCurrentRawStream(dev)), "copy_pages")


def compact_pages_ref(k, v, block_tables, lens, keep, out_tables, cos_sin):
    new = torch.zeros(lens.shape[0], dtype=torch.int32, device=lens.device)
    most = min(keep.shape[1], block_tables.shape[1] * PAGE)
    for b in range(lens.shape[0]):
        old = keep[b, :max(0, min(int(lens[b]), most))].nonzero()[:, 0]
        n = torch.arange(len(old), device=old.device)
        new[b] = len(old)
        to = block_tables[b] if out_tables is None else out_tables[b]
        fp, tp = block_tables[b][old // PAGE].long(), to[n // PAGE].long()
        pages = (fp >= 0) & (fp < k.shape[1]) & (tp >= 0) & (tp < k.shape[1])
        old, n, fp, tp = old[pages], n[pages], fp[pages], tp[pages]
        x, y = k[:, fp, :, old % PAGE], v[:, fp, :, old % PAGE]       # token, layer, head, number
        if cos_sin is not None:
            a, c = cos_sin[old].double(), cos_sin[n].double()
            cos = (a * c).sum(-1)[:, None, None]
            sin = (c[..., 1] * a[..., 0] - c[..., 0] * a[..., 1])[:, None, None]
            x1, x2 = x.double().chunk(2, -1)
            turned = torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin], -1).to(x.dtype)
            x = torch.where((old == n)[:, None, None, None], x, turned)
        k[:, tp, :, n % PAGE] = x
        v[:, tp, :, n % PAGE] = y
    return new


def _refuse(k, block_tables, lens, keep, out_tables, cos_sin):
    """Says which of compact_pages' conditions does not hold."""
    def need(ok, why):
        if not ok:
            raise ValueError("compact_pages: " + why)
    need(block_tables.dim() == 2 and block_tables.dtype == torch.int32 and (block_tables.stride(1) == 1 or block_tables.shape[1] < 2),
         "block_tables must be int32 [sequences, pages]")
    B, W = block_tables.shape
    need(lens.dim() == 1 and lens.dtype == torch.int32 and lens.shape[0] == B and (B < 2 or lens.stride(0) == 1),
         "lens must be int32 [%d]" % B)
    need(keep.dim() == 2 and keep.dtype == torch.bool and keep.shape[0] == B and (keep.stride(1) == 1 or keep.shape[1] < 2),
         "keep must be bool [%d, tokens]" % B)
    need(B <= 65535, "more than 65535 sequences")
    if out_tables is not None:
        need(out_tables.dtype == torch.int32 and out_tables.shape == block_tables.shape
             and (out_tables.stride(1) == 1 or W < 2), "out_tables must be like block_tables")
    need(all(t is None or t.stride(0) < FAR for t in (block_tables, out_tables)), "tables with rows too far apart")
    most = min(keep.shape[1], W * PAGE)
    if cos_sin is not None:
        need(k.dtype == torch.bfloat16, "keys are turned in bf16 caches only, not in %s" % k.dtype)
        need(cos_sin.dtype == torch.float32 and cos_sin.dim() == 3 and cos_sin.shape[1:] == (HEAD_DIM // 2, 2)
             and cos_sin.is_contiguous() and cos_sin.shape[0] >= most and cos_sin.data_ptr() % 16 == 0,
             "cos_sin must be float32 [%d or more, %d, 2], contiguous" % (most, HEAD_DIM // 2))
    need(all(t is None or t.device == k.device for t in (block_tables, lens, keep, out_tables, cos_sin)),
         "tensors must be on one device")
    raise AssertionError("compact_pages: the two forms of its conditions differ")


def compact_pages(k: torch.Tensor, v: torch.Tensor, block_tables: torch.Tensor, lens: torch.Tensor, keep: torch.Tensor,
                  out_tables: torch.Tensor | None = None, cos_sin: torch.Tensor | None = None) -> torch.Tensor:
    """The kept tokens of every sequence, together and in their order: in every layer and head, token p of sequence b becomes
    its token n, where n tokens before p are kept.  Returns the new lengths, int32 [B].

    block_tables: int32 [B, pages]; lens: int32 [B], the sequences' tokens (at most the table's and keep's); keep: bool
    [B, tokens].  out_tables: int32 like block_tables, the pages that the tokens go to, none of them in block_tables; None: in
    place.  In place no page is in the tables twice.  Rows of pages behind the new lengths stay as they were.
    cos_sin: float32 [positions, 64, 2] (``models.config.rope_table``): keys that were rotated for position p are turned on to
    position n (bf16 caches); None: they stay as they are, as for sequences that go on counting positions.  Entries of the
    tables that are no pages are skipped."""
    caches, dev = _caches(k, v, "compact_pages")
    try:
        (B, W), (n,), (rows, places) = block_tables.shape, lens.shape, keep.shape
        (sb, b1), (l1,), (sk, k1) = block_tables.stride(), lens.stride(), keep.stride()
        most = min(places, W * PAGE)
        ok = (n == rows == B <= 65535 and block_tables.dtype == lens.dtype == torch.int32 and keep.dtype == torch.bool
              and (b1 == 1 or W < 2) and (l1 == 1 or B < 2) and (k1 == 1 or places < 2) and sb < FAR
              and dev == block_tables.get_device() == lens.get_device() == keep.get_device())
        st = 0
        if ok and out_tables is not None:
            st, t1 = out_tables.stride()
            ok = (out_tables.dtype == torch.int32 and out_tables.shape == (B, W) and (t1 == 1 or W < 2) and st < FAR
                  and dev == out_tables.get_device())
        if ok and cos_sin is not None:
            positions, half, two = cos_sin.shape
            ok = (k.dtype == torch.bfloat16 and cos_sin.dtype == torch.float32 and half == HEAD_DIM // 2 and two == 2
                  and positions >= most and cos_sin.is_contiguous() and cos_sin.data_ptr() % 16 == 0
                  and dev == cos_sin.get_device())
        if ok and dev < 0:
            ok = all(t is None or t.device == k.device for t in (block_tables, lens, keep, out_tables, cos_sin))
    except ValueError:       # another number of dimensions
        ok = False
    if not ok:
        _refuse(k, block_tables, lens, keep, out_tables, cos_sin)
    if dev < 0:
        return compact_pages_ref(k, v, block_tables, lens, keep, out_tables, cos_sin)
    new = torch.empty(B, dtype=torch.int32, device=k.device)
    if B == 0:
        return new
    if most == 0 or 0 in k.shape:
        return new.copy_((keep & (torch.arange(places, device=k.device) < lens[:, None].clamp(max=most))).sum(1))
    with _lib.device_of(dev):
        _lib.check(_lib.lib().p2p_compact_pages(
            *caches, block_tables.data_ptr(), sb, W, _lib.ptr(out_tables), st, lens.data_ptr(), keep.data_ptr(), sk, places, B,
            _lib.ptr(cos_sin), new.data_ptr(), torch._C._cuda_getCurrentRawStream(dev)), "compact_pages")
    return new
