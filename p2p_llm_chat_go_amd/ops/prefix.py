"""Attention of rows whose sequences begin with the same pages (csrc/kernels/prefix_attention.hip).

:func:`paged_attention` reads a row's keys once per row.  Where a batch's sequences share their first pages (a system
prompt, a thread that several replies are drawn from; ``KVCache.fork`` makes such sequences), :func:`prefix_attention` reads
those once for all rows of the group, and a sequence's own pages once for the rows of that sequence.  Rows are as there: one
token each, of a decode step (one row per sequence) or of prompts (consecutive rows per sequence), with a block-table row
and a context length.
"""
from __future__ import annotations

import ctypes
import dataclasses
import math
import operator

import torch

from . import _lib
from .attention import HEAD_DIM, PAGE, paged_attention_ref

SCALE = 1.0 / math.sqrt(HEAD_DIM)
SHARED_PARTS = (1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64, 96)
OWN_PARTS = (1, 2, 4, 8, 16, 32, 64)
FAR = 2 ** 31          # strides are below
LEAST_SCALE, MOST_SCALE = 2.0 ** -64, 2.0 ** 64    # (the kernel's scores and their scale are fp32)
FEW, MANY = 32, 128    # (row, head) pairs of a workgroup, in the kernel's two roles


class _Launch(ctypes.Structure):
    """What a plan hands to its calls (PrefixPlan in the kernels' source)."""
    _fields_ = ([(n, ctypes.c_void_p) for n in ("works", "base", "row_tables")]
                + [(n, ctypes.c_int) for n in ("n_works", "waves", "tiles", "rows", "parts", "even", "n_heads", "n_kv", "head_dim",
                                               "max_ctx")])


@dataclasses.dataclass(frozen=True)
class PrefixPlan:
    """How a batch's rows and pages are cut into works: host data of :func:`prefix_plan`, on the device once."""
    rows: int
    n_heads: int
    n_kv: int
    max_ctx: int
    tables: int            # block tables it reads
    waves: int             # wavefronts of a workgroup, 4 or 8
    tiles: bool            # some workgroup has more than FEW pairs
    even: int              # results of every row, where they are equally many (else 0)
    parts: int             # results of parts, over all rows
    works: torch.Tensor    # int32 [n, 8]
    base: torch.Tensor     # int32 [rows + 1]: parts of the rows before
    row_tables: torch.Tensor   # int32 [rows]
    launch: _Launch = dataclasses.field(init=False, repr=False, compare=False)
    at: int = dataclasses.field(init=False, repr=False, compare=False)     # its address

    def __post_init__(self):
        launch = _Launch(self.works.data_ptr(), self.base.data_ptr(), self.row_tables.data_ptr(), self.works.shape[0], self.waves,
                         self.tiles, self.rows, self.parts, self.even, self.n_heads, self.n_kv, HEAD_DIM, self.max_ctx)
        object.__setattr__(self, "launch", launch)
        object.__setattr__(self, "at", ctypes.addressof(launch))


def _int(x, what: str) -> int:
    try:
        return operator.index(x)
    except TypeError:
        raise ValueError("prefix_plan: %s must be whole numbers, got %r" % (what, x)) from None


class _Shape:
    """A batch as tiles of rows, and the ways to cut its pages into parts.

    Shared: a group's rows are cut into tiles that read the shared pages, and every sequence's rows into tiles that read its
    own.  Alone: every sequence's rows read all of its pages.  A tile is a workgroup per kv head and part: up to 32 pairs of
    rows and heads, whose wavefronts take 32 keys each, or up to 128, 32 for each wavefront.  More parts are more workgroups
    and more results to write and to bring together; where every row has one part the second launch falls away."""

    def __init__(self, groups, seqs, n_heads, n_kv, max_ctx):
        self.n_heads, self.n_kv, self.G, self.R = n_heads, n_kv, n_heads // n_kv, len(seqs)
        self.pages = -(-max_ctx // PAGE)
        self.groups, r0 = [], 0          # (pages, tiles of the group, tiles of its sequences): (first row, rows, table)
        for n, p in groups:
            r1, runs, a = r0 + n, [], r0
            while a < r1:
                b = a + 1
                while b < r1 and seqs[b] == seqs[a]:
                    b += 1
                runs += self._cut(a, b, seqs[a])
                a = b
            if len({t for _a, _n, t in runs}) == 1:
                p = 0                    # one sequence shares with nobody
            self.groups.append((p, self._cut(r0, r1, seqs[r0]), runs))
            r0 = r1
        self.sums = [(p, len(tiles), tiles[0][1] * self.G > FEW, len(runs), any(n * self.G > FEW for _a, n, _t in runs),
                      sum(n for _a, n, _t in runs)) for p, tiles, runs in self.groups]

    def _cut(self, a, b, table):
        tile = (FEW if (b - a) * self.G <= FEW else MANY) // self.G
        return [(i, min(tile, b - i), table) for i in range(a, b, tile)]

    def works(self, share: bool, shared_parts: int, own_parts: int):
        """(the works, parts of every row)."""
        works, count = [], [0] * self.R
        for p, tiles, _runs in self.groups:
            if share and p:
                C = min(shared_parts, -(-p // 2))
                works += [(a, n, t, p * c // C, p * (c + 1) // C, c, 0, 0) for c in range(C) for a, n, t in tiles]
                for a, n, _t in tiles:
                    count[a:a + n] = [C] * n
        for p, _tiles, runs in self.groups:
            p = p if share else 0
            C = min(own_parts, -(-(self.pages - p) // 2))
            works += [(a, n, t, p, self.pages, c, C, count[a]) for a, n, t in runs for c in range(C)]
            for a, n, _t in runs:
                count[a:a + n] = [count[a] + C] * n
        return works, count

    def _sizes(self, share: bool, shared_parts: int, own_parts: int):
        """Workgroups and the longest one's pages of tiles of up to 128 pairs, of up to 32 pairs (in units of two pages), parts of
        all rows, pages of the batch and pages that workgroups load."""
        many = few = many_pages = few_units = parts = read = loaded = 0
        for p, tiles, tiles_many, runs, runs_many, rows in self.sums:
            # contexts end somewhere up to the plan's longest: half of the pages on average, some tokens more in the longest
            rest = self.pages - p
            own = (rest + 1) // 2
            longest = own + 4 if own + 4 < rest else rest
            read += p + runs * own
            if share and p:
                C = (p + 1) // 2
                if shared_parts < C:
                    C = shared_parts
                parts += rows * C
                loaded += tiles * p
                if tiles_many:
                    many += tiles * C
                    many_pages = max(many_pages, -(-p // C))
                else:
                    few += tiles * C
                    few_units = max(few_units, -(-p // (2 * C)))
                C = (rest + 1) // 2
            else:
                own, longest, C = p + own, self.pages, (self.pages + 1) // 2
            if own_parts < C:
                C = own_parts
            if C:
                parts += rows * C
                loaded += runs * own
                if runs_many:
                    many += runs * C
                    many_pages = max(many_pages, -(-longest // C))
                else:
                    few += runs * C
                    few_units = max(few_units, -(-longest // (2 * C)))
        return many * self.n_kv, many_pages, few * self.n_kv, few_units, parts, read, loaded

    def micros(self, waves: int, share: bool, sizes) -> float:
        """About how long a call takes: constants fitted to timings of 78 batches, of 2 to 768 rows behind 128 to 32768 tokens, cut
        in all ways.  A launch and its first loads 4.1 us (of 8 wavefronts 5.2); a page of a tile of 128 pairs 1.25 us where CUs
        have one workgroup, 1.4 where they have two, two pages of 8 wavefronts 2.25; 32 keys of a wavefront 0.65 (0.8); what memory
        and L2 add, as if they were three sides of a box, at 17.5 and 25 TB/s (the caches held much of it); a second launch 2.1,
        0.84 per MB of the parts' results; rows alone in parts a twentieth more.  The cut that it puts first takes 2.4 % longer
        than the fastest one on average."""
        many, many_pages, few, few_units, parts, read, loaded = sizes
        if waves == 8:
            t, most, page, unit = 5.2, 256, 2.25, 0.8       # (most: workgroups at once)
            many_pages, few_units = (many_pages + 1) // 2, (few_units + 1) // 2
        else:
            t, most, page, unit = 4.1, 512, 1.25 if many <= 256 else 1.4, 0.65
        t_many, t_few = many_pages * page * -(-many // most), few_units * unit * -(-few // most)
        mb = self.n_kv * 32768e-6                      # of a page
        t += math.hypot(max(t_many, t_few) if many + few <= most else t_many + t_few, read * mb / 17.5, loaded * mb / 25)
        if parts > self.R:
            t += 2.1 + 0.84e-6 * parts * self.n_heads * 512
            if not share:
                t *= 1.05
        return t

    def choose(self):
        """The way (wavefronts of a workgroup, shared or alone, parts of shared pages, parts of a sequence's own) to cut it."""
        upto = lambda parts, pages: [c for c in parts if c == 1 or c <= -(-pages // 2)]
        most = max(p for p, _t, _r in self.groups)
        least = min(p for p, _t, _r in self.groups)
        cuts = [(False, 1, own) for own in upto(OWN_PARTS, self.pages)]
        if most:
            cuts += [(True, shared, own) for shared in upto(SHARED_PARTS, most) for own in upto(OWN_PARTS, self.pages - least)]
        best = math.inf
        for cut in cuts:
            sizes = self._sizes(*cut)
            for waves in (4, 8):
                t = self.micros(waves, cut[0], sizes)
                if t < best:
                    best, way = t, (waves, *cut)
        return way


def prefix_plan(groups, n_heads: int, n_kv: int, max_ctx: int, device, seqs=None) -> PrefixPlan:
    """A plan for batches of ``sum(rows)`` query rows.

    groups: (rows, pages) of every group, in the order of the rows: the next ``rows`` rows, whose block tables begin with the
    same ``pages`` pages (0: they share nothing).  seqs: every row's block-table row (rows of one sequence one after the
    other); None: row r has row r, as in a decode step.  max_ctx: the longest context that the plan is used for.  Context
    lengths are not part of it: a decode step's plan serves its batch until a sequence joins or leaves.  Its tensors are kept
    until the calls that read them have ended, as any tensor that another stream than its own reads."""
    n_heads, n_kv, max_ctx = _int(n_heads, "n_heads"), _int(n_kv, "n_kv"), _int(max_ctx, "max_ctx")
    if n_kv < 1 or n_heads < n_kv or n_heads % n_kv or n_heads // n_kv > FEW:
        raise ValueError("prefix_plan: %d query heads on %d kv heads (1 to %d each)" % (n_heads, n_kv, FEW))
    if max_ctx < 1:
        raise ValueError("prefix_plan: max_ctx must be positive, got %d" % max_ctx)
    groups = [(_int(r, "rows"), _int(p, "pages")) for r, p in groups]
    pages_max = -(-max_ctx // PAGE)
    for r, p in groups:
        if r < 1 or p < 0 or p > pages_max:
            raise ValueError("prefix_plan: a group of %d rows that share %d pages (contexts up to %d)" % (r, p, max_ctx))
    R = sum(r for r, _ in groups)
    if R < 1:
        raise ValueError("prefix_plan: no rows")
    seqs = list(range(R)) if seqs is None else [_int(s, "seqs") for s in (seqs.tolist() if isinstance(seqs, torch.Tensor) else seqs)]
    if len(seqs) != R or min(seqs) < 0:
        raise ValueError("prefix_plan: seqs must give a block table (0 ..) to each of the %d rows" % R)

    shape = _Shape(groups, seqs, n_heads, n_kv, max_ctx)
    waves, *way = shape.choose()
    works, count = shape.works(*way)
    base = [0]
    for n in count:
        base.append(base[-1] + n)
    dev = torch.device(device)
    flat = [x for w in works for x in w] + seqs + base
    flat = torch.tensor(flat, dtype=torch.int32).to(dev)
    n = 8 * len(works)
    tiles = any(w[1] * (n_heads // n_kv) > FEW for w in works)
    even = count[0] if min(count) == max(count) else 0
    return PrefixPlan(R, n_heads, n_kv, max_ctx, max(seqs) + 1, waves, tiles, even, base[-1], flat[:n].view(-1, 8), flat[n + R:],
                      flat[n:n + R])


def prefix_workspace(plan: PrefixPlan) -> torch.Tensor:
    """The parts' outputs, maxima and sums for :func:`prefix_attention`, fp32; a call uses them until it ends, so calls that may
    run at once (on several streams, in several graphs) take one each."""
    return torch.empty(plan.parts * plan.n_heads * (HEAD_DIM + 2), device=plan.works.device, dtype=torch.float32)


def _overlap(q, out, R, width) -> bool:
    """Whether the first R rows of q and out (bf16, ``width`` numbers each) have memory in common."""
    sq, so, row = q.stride(0) * 2, out.stride(0) * 2, width * 2
    ahead = out.data_ptr() - q.data_ptr()
    if ahead >= (R - 1) * sq + row or -ahead >= (R - 1) * so + row:
        return False
    return sq != so or sq < row or ahead % sq < row or ahead % sq > sq - row


def _refuse(q, k_cache, v_cache, block_tables, ctx_lens, plan, out, workspace, scale):
    """Says which of prefix_attention's conditions does not hold."""
    R, n_heads, n_kv, width = plan.rows, plan.n_heads, plan.n_kv, plan.n_heads * HEAD_DIM
    def need(ok, why):
        if not ok:
            raise ValueError("prefix_attention: " + why)
    need(q.dim() == 2 and q.dtype == torch.bfloat16 and q.shape[0] >= R and q.shape[1] == width and q.stride(1) == 1
         and q.stride(0) < FAR, "q must be bf16 [%d or more, %d], rows contiguous" % (R, width))
    for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
        need(c.dim() == 4 and c.shape[1:] == (n_kv, PAGE, HEAD_DIM) and c.dtype == torch.bfloat16 and c.is_contiguous()
             and c.shape[0] > 0 and c.data_ptr() % 16 == 0,
             "%s must be bf16 [pages, %d, %d, %d], contiguous from a multiple of 16 bytes" % (name, n_kv, PAGE, HEAD_DIM))
    need(k_cache.shape == v_cache.shape, "k_cache and v_cache differ in shape")
    need(block_tables.dim() == 2 and block_tables.dtype == torch.int32 and block_tables.stride(1) == 1
         and block_tables.stride(0) < FAR and block_tables.shape[0] >= plan.tables and block_tables.shape[1] * PAGE >= plan.max_ctx,
         "block_tables must be int32 [%d or more, pages of %d tokens]" % (plan.tables, plan.max_ctx))
    need(ctx_lens.dim() == 1 and ctx_lens.dtype == torch.int32 and ctx_lens.shape[0] >= R and ctx_lens.stride(0) == 1,
         "ctx_lens must be int32 [%d or more]" % R)
    need(LEAST_SCALE <= scale <= MOST_SCALE, "scale must be 2^-64 .. 2^64, got %r" % scale)
    need(out.dim() == 2 and out.dtype == torch.bfloat16 and out.shape[0] >= R and out.shape[1] == width and out.stride(1) == 1
         and (out.stride(0) >= width or R == 1) and out.stride(0) < FAR,
         "out must be bf16 [%d or more, %d], rows contiguous and apart" % (R, width))
    need(not _overlap(q, out, R, width), "out overlaps q")
    need(all(t.device == q.device for t in (k_cache, v_cache, block_tables, ctx_lens, plan.works, out)),
         "tensors and plan must be on one device")
    need(workspace is None or (workspace.device == q.device and workspace.dtype == torch.float32 and workspace.is_contiguous()
                               and workspace.numel() >= plan.parts * n_heads * (HEAD_DIM + 2)
                               and workspace.data_ptr() % 16 == 0), "workspace is not this plan's (prefix_workspace)")
    raise AssertionError("prefix_attention: the two forms of its conditions differ")


def prefix_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                     ctx_lens: torch.Tensor, plan: PrefixPlan, out: torch.Tensor | None = None,
                     workspace: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
    """q: [R, n_heads * 128] bf16 -> out [R, n_heads * 128] bf16, as :func:`paged_attention` with the plan's tables.

    Row r attends the first ``min(ctx_lens[r], plan.max_ctx)`` tokens of its block table; a row that sees none is 0.  Rows
    behind the plan's are not read or written; out is other memory than q.  A group's shared pages are read through its
    first row's table.  Block tables hold pages of the cache; others read page 0 or the last one.  scale: 2^-64 .. 2^64
    (None: 128^-0.5).  Scores, softmax statistics and sums are fp32; weights are rounded to bf16 (by 2^-8 at most) for the
    product with the values, and divided by the sum of the rounded ones."""
    R, n_heads, n_kv = plan.rows, plan.n_heads, plan.n_kv
    width = n_heads * HEAD_DIM
    if scale is None:
        scale = SCALE
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    dev = q.get_device()     # (-1: not a GPU's)
    if workspace is None and dev >= 0:
        workspace = prefix_workspace(plan)
    works = plan.works
    try:
        Rq, wq = q.shape
        Ro, wo = out.shape
        tables, pages = block_tables.shape
        rows, = ctx_lens.shape
        (sq, q1), (so, o1), (sb, b1), (c1,) = q.stride(), out.stride(), block_tables.stride(), ctx_lens.stride()
        P, h, t, d = shape = k_cache.shape
        ok = (Rq >= R and wq == wo == width and Ro >= R and tables >= plan.tables and pages * PAGE >= plan.max_ctx and rows >= R
              and shape == v_cache.shape and h == n_kv and t == PAGE and d == HEAD_DIM and P > 0
              and q.dtype == out.dtype == k_cache.dtype == v_cache.dtype == torch.bfloat16
              and block_tables.dtype == ctx_lens.dtype == torch.int32
              and q1 == o1 == b1 == c1 == 1 and sq < FAR > so and sb < FAR and (so >= width or R == 1)
              and k_cache.is_contiguous() and v_cache.is_contiguous() and LEAST_SCALE <= scale <= MOST_SCALE
              and dev == out.get_device() == k_cache.get_device() == v_cache.get_device() == block_tables.get_device()
              == ctx_lens.get_device() == works.get_device())
        kp, vp, qp, op = k_cache.data_ptr(), v_cache.data_ptr(), q.data_ptr(), out.data_ptr()
        if qp + 2 * (R * sq + width) > op and op + 2 * (R * so + width) > qp:
            ok = ok and not _overlap(q, out, R, width)
        if ok and dev >= 0:
            wp = workspace.data_ptr()
            ok = ((kp | vp | wp) % 16 == 0 and workspace.get_device() == dev and workspace.dtype == torch.float32
                  and workspace.is_contiguous() and workspace.numel() >= plan.parts * n_heads * (HEAD_DIM + 2))
        elif ok:
            ok = all(t.device.type == "cpu" for t in (q, k_cache, v_cache, block_tables, ctx_lens, works, out))
    except ValueError:       # another number of dimensions
        ok = False
    if not ok:
        _refuse(q, k_cache, v_cache, block_tables, ctx_lens, plan, out, workspace, scale)
    if dev < 0:
        ctx = ctx_lens[:R].clamp(0, plan.max_ctx)
        paged_attention_ref(q[:R], k_cache, v_cache, block_tables.clamp(0, P - 1), plan.row_tables, ctx.clamp(min=1), n_heads,
                            n_kv, scale, out[:R])
        out[:R] = torch.where((ctx > 0)[:, None], out[:R], 0)
        return out
    if dev != torch._C._cuda_getDevice():
        with torch.cuda.device(dev):
            return prefix_attention(q, k_cache, v_cache, block_tables, ctx_lens, plan, out, workspace, scale)
    _lib.check(_lib.lib().p2p_prefix_attention(
        plan.at, qp, sq, kp, vp, P, block_tables.data_ptr(), sb, ctx_lens.data_ptr(), scale, op, so, wp,
        torch._C._cuda_getCurrentRawStream(dev)), "prefix_attention")
    return out
