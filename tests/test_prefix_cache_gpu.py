"""Operators over shared pages (``ops.prefix_attention``, ``ops.copy_pages``, ``ops.compact_pages``) against their
definitions in 64 bits."""
import math

import pytest
import torch

from p2p_llm_chat_go_amd import ops
from p2p_llm_chat_go_amd.ops import prefix
from p2p_llm_chat_go_amd.models.config import LLAMA31_8B, rope_table
from tests import prefix_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
PAGE, D = 64, 128
NAN, INF = float("nan"), float("inf")


def _batch(groups, Hq, Hkv, own, seed, tokens=1, by=1.7):
    """Groups of (sequences, pages): q, caches whose rows past a context are nan, tables, seqs, ctx, max_ctx; a sequence has
    up to ``own`` tokens of its own, the last ``tokens`` of them are query rows."""
    g = torch.Generator().manual_seed(seed)
    n = sum(s for s, _ in groups)
    own_pages = -(-own // PAGE)
    width = max(p for _, p in groups) + own_pages
    total = 1 + sum(p for _, p in groups) + n * own_pages
    perm = (torch.randperm(total - 1, generator=g) + 1).tolist()
    k, v = (torch.randn(total, Hkv, PAGE, D, generator=g).bfloat16() for _ in range(2))
    k[0], v[0] = NAN, NAN
    table = torch.zeros(n, width, dtype=torch.int32)
    seqs, ctx, rows, s = [], [], [], 0
    for count, p in groups:
        shared = [perm.pop() for _ in range(p)]
        r0 = len(seqs)
        for _ in range(count):
            lo = min(tokens, own)
            mine = int(torch.randint(lo, own + 1, (1,), generator=g))
            pages = shared + [perm.pop() for _ in range(own_pages)]
            table[s, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
            at = p * PAGE + mine
            for j in range(at, (p + own_pages) * PAGE):
                k[pages[j // PAGE], :, j % PAGE] = NAN
                v[pages[j // PAGE], :, j % PAGE] = NAN
            seqs += [s] * min(tokens, mine)
            ctx += range(at - min(tokens, mine) + 1, at + 1)
            s += 1
        rows.append((len(seqs) - r0, p))
    q = (torch.randn(len(seqs), Hq * D, generator=g) * by).bfloat16()
    return q, k, v, table, seqs, torch.tensor(ctx, dtype=torch.int32), rows, max(p for _, p in groups) * PAGE + own


def _check(got, want, bound):
    got = got.double().cpu().view(want.shape)
    assert torch.equal(torch.isfinite(got), torch.isfinite(want))
    far = ((got - want).abs() - bound).nan_to_num()
    assert float(far.max()) <= 0, (float(far.max()), (far > 0).nonzero()[:5])


def _run(q, k, v, table, ctx, plan, **kw):
    return ops.prefix_attention(q.to(DEV), k.to(DEV), v.to(DEV), table.to(DEV), ctx.to(DEV), plan, **kw)


# cuts of a batch (wavefronts of a workgroup, shared pages or not, parts of them, parts of a sequence's own pages); None: the one that the plan chooses
WAYS = [None, (4, True, 1, 1), (8, True, 1, 1), (4, True, 5, 2), (8, True, 3, 1), (4, False, 1, 1), (8, False, 1, 1), (4, False, 1, 3)]


@pytest.fixture(params=WAYS, ids=str)
def way(request, monkeypatch):
    if request.param is not None:
        monkeypatch.setattr(prefix._Shape, "choose", lambda self: request.param)
    return request.param


HEADS = [(8, 1), (8, 2), (4, 4), (6, 2), (16, 1), (32, 1), (5, 1)]


@pytest.mark.parametrize("Hq,Hkv", HEADS)
@pytest.mark.parametrize("groups,own", [([(2, 1)], 1), ([(1, 2)], 70), ([(3, 0)], 65), ([(7, 3), (1, 0), (20, 5), (2, 1)], 130),
                                        ([(70, 9)], 33), ([(5, 40)], 300)])
def test_prefix_attention_of_decode_rows(way, Hq, Hkv, groups, own):
    q, k, v, table, seqs, ctx, rows, most = _batch(groups, Hq, Hkv, own, Hq + own)
    plan = ops.prefix_plan(rows, Hq, Hkv, most, DEV)
    want, bound = oracle.attention(q, k, v, table, seqs, ctx, Hq, Hkv, 1 / math.sqrt(D), most)
    _check(_run(q, k, v, table, ctx, plan), want, bound)


@pytest.mark.parametrize("groups,own", [([(2, 560)], 9), ([(40, 150)], 3), ([(1, 0), (2, 700)], 2)])
def test_prefix_attention_in_many_parts(groups, own, monkeypatch):
    """One kv head: up to some 300 parts of a row."""
    monkeypatch.setattr(prefix._Shape, "choose", lambda self: (4, True, 400, 100))
    q, k, v, table, seqs, ctx, rows, most = _batch(groups, 8, 1, own, own)
    plan = ops.prefix_plan(rows, 8, 1, most, DEV)
    want, bound = oracle.attention(q, k, v, table, seqs, ctx, 8, 1, 1 / math.sqrt(D), most)
    _check(_run(q, k, v, table, ctx, plan), want, bound)


def test_prefix_attention_of_many_rows_in_many_parts(monkeypatch):
    """More than 2048 pairs of a row and a head, some of one part, others of 21."""
    monkeypatch.setattr(prefix._Shape, "choose", lambda self: (4, True, 20, 1))
    q, k, v, table, seqs, ctx, rows, most = _batch([(250, 40), (11, 0)], 8, 1, 3, 1)
    plan = ops.prefix_plan(rows, 8, 1, most, DEV)
    assert plan.even == 0 and plan.parts == 250 * 21 + 11
    want, bound = oracle.attention(q, k, v, table, seqs, ctx, 8, 1, 1 / math.sqrt(D), most)
    _check(_run(q, k, v, table, ctx, plan), want, bound)


@pytest.mark.parametrize("Hq,Hkv", [(8, 2), (4, 4), (8, 1), (3, 1)])
@pytest.mark.parametrize("groups,own,tokens", [([(3, 2)], 44, 44), ([(2, 4), (3, 1)], 100, 17), ([(1, 5)], 200, 130),
                                               ([(9, 1)], 64, 2)])
def test_prefix_attention_of_prompt_rows(way, Hq, Hkv, groups, own, tokens):
    q, k, v, table, seqs, ctx, rows, most = _batch(groups, Hq, Hkv, own, tokens, tokens)
    plan = ops.prefix_plan(rows, Hq, Hkv, most, DEV, seqs=seqs)
    want, bound = oracle.attention(q, k, v, table, seqs, ctx, Hq, Hkv, 0.2, most)
    _check(_run(q, k, v, table, ctx, plan, scale=0.2), want, bound)


@pytest.mark.parametrize("Hq,Hkv", [(8, 2), (2, 2)])
def test_rows_that_see_nothing_part_of_the_prefix_or_more_than_the_plan(way, Hq, Hkv):
    """Contexts of 0 and less give zeros; a context may end inside the shared pages, at any key of a page; what lies past the
    plan's longest context is not read."""
    q, k, v, table, seqs, ctx, rows, most = _batch([(24, 3), (3, 0)], Hq, Hkv, 40, 5)
    ctx[:9] = torch.tensor([0, -5, 1, 63, 64, 65, 127, 128, 191])
    ctx[9], ctx[24] = 10 ** 6, 0
    last = table[9, 3]
    k[last, :, 40:], v[last, :, 40:] = NAN, NAN
    k[last, :, :40], v[last, :, :40] = k[last, :, :40].nan_to_num(0.5), v[last, :, :40].nan_to_num(0.25)
    plan = ops.prefix_plan(rows, Hq, Hkv, most, DEV)
    want, bound = oracle.attention(q, k, v, table, seqs, ctx, Hq, Hkv, 1 / math.sqrt(D), most)
    got = _run(q, k, v, table, ctx, plan)
    _check(got, want, bound)
    assert bool((got[[0, 1, 24]] == 0).all())


def test_rows_inside_their_shared_pages(way):
    """Contexts that end in the shared pages, or before them; what none of the rows sees is nan."""
    q, k, v, table, seqs, _ctx, rows, _most = _batch([(30, 4)], 8, 2, 1, 8)
    ctx = torch.randint(0, 150, (30,), generator=torch.Generator().manual_seed(1)).int()
    ctx[:4] = torch.tensor([0, 149, 64, 0])
    for c in (k, v):
        c[table[0, 3]] = NAN
        c[table[0, 2], :, 149 - 128:] = NAN
    plan = ops.prefix_plan(rows, 8, 2, 256, DEV)
    want, bound = oracle.attention(q, k, v, table, seqs, ctx, 8, 2, 1 / math.sqrt(D), 256)
    _check(_run(q, k, v, table, ctx, plan), want, bound)
    ctx.zero_()
    assert bool((_run(q, k, v, table, ctx, plan) == 0).all())


@pytest.mark.parametrize("tokens", [1, 20])
def test_values_that_are_not_finite_reach_the_rows_that_see_them_only(way, tokens):
    q, k, v, table, seqs, ctx, rows, most = _batch([(12, 2), (6, 1)], 8, 2, 90, 3, tokens)
    if tokens == 1:
        ctx[:12] = torch.arange(100, 124, 2, dtype=torch.int32)
    plan = ops.prefix_plan(rows, 8, 2, most, DEV, seqs=seqs)
    k[table[0, 1], 0, 45, 3] = INF          # token 109 of the first group's prefix
    k[table[0, 1], 1, 50, 3] = NAN
    v[table[0, 1], 0, 51, 7] = -INF
    v[table[12, 0], 1, 5, 9] = NAN
    last = int(ctx[-1]) - 1                  # the last row's own token
    v[table[seqs[-1], last // PAGE], :, last % PAGE, 11] = INF
    want, bound = oracle.attention(q, k, v, table, seqs, ctx, 8, 2, 1 / math.sqrt(D), most)
    got = _run(q, k, v, table, ctx, plan).double().cpu().view(want.shape)
    # a key that is infinite makes its rows nan or gives it all the weight, by the sign of its score: as torch does
    same = torch.isnan(want) == torch.isnan(got)
    assert bool(same.all()), same.logical_not().nonzero()[:5]
    far = torch.where(got == want, 0, (got - want).abs() - bound).nan_to_num()
    assert float(far.max()) <= 0


def _same_nan(got, want, bound):
    """Equal where they are not finite, else within the bound."""
    got = got.double().cpu().view(want.shape)
    assert torch.equal(torch.isnan(want), torch.isnan(got)), (torch.isnan(want) != torch.isnan(got)).nonzero()[:5]
    far = torch.where(got == want, 0, (got - want).abs() - bound).nan_to_num()
    assert float(far.max()) <= 0, (float(far.max()), (far > 0).nonzero()[:5])


def test_scores_that_are_nan_make_their_rows_nan(way):
    """A query with a nan; a row whose last key, alone in its part, its page or its 32 keys, is nan."""
    q, k, v, table, seqs, ctx, rows, most = _batch([(12, 2), (6, 1)], 8, 2, 90, 3)
    q[3, 5 * D + 7] = NAN
    for r, at in ((7, 128), (8, 160), (13, 64), (14, 96), (15, 127)):     # the last key that the row sees
        page, ctx[r] = table[r, at // PAGE], at + 1
        for c in (k, v):
            c[page, :, :at % PAGE] = c[page, :, :at % PAGE].nan_to_num(0.5)
            c[page, :, at % PAGE] = 0.25
        k[page, 1, at % PAGE] = NAN
    plan = ops.prefix_plan(rows, 8, 2, most, DEV)
    want, bound = oracle.attention(q, k, v, table, seqs, ctx, 8, 2, 1 / math.sqrt(D), most)
    nan = torch.isnan(want).all(-1)
    assert nan[3].nonzero()[:, 0].tolist() == [5] and nan[[7, 8, 13, 14, 15]].sum(0).tolist() == [0] * 4 + [5] * 4 and nan.sum() == 21
    _same_nan(_run(q, k, v, table, ctx, plan), want, bound)


def test_rows_whose_scores_are_all_minus_infinity_are_nan(way):
    """No key has a weight then, as the softmax of the formula has it; rows without a key are 0."""
    q, k, v, table, seqs, ctx, rows, most = _batch([(12, 2), (6, 1)], 8, 2, 90, 4)
    q[:, 3::D] = q[:, 3::D].abs() + 0.1
    k[table[0, 0], 0, 0, 3] = -INF             # the first group's first key
    k[table[12, 0], 1, :, 3] = -INF            # and all of the second group's shared ones
    ctx[2], ctx[5], ctx[12], ctx[13], ctx[14] = 1, 0, 64, 40, 65
    for c in (k, v):
        c[table[14, 1], :, 0] = 0.25
    plan = ops.prefix_plan(rows, 8, 2, most, DEV)
    want, bound = oracle.attention(q, k, v, table, seqs, ctx, 8, 2, 1 / math.sqrt(D), most)
    # The bound's part of the scores is infinite for rows that see an infinite key: theirs is a rounding of the result and one of
    # every weight, U16 of the largest value each, and fp32 scores of up to 60 (2 D U32 60 = 0.24 U16)
    bound = torch.where(torch.isfinite(bound), bound, 2.5 * oracle.U16 * float(v.float().nan_to_num(0).abs().max()))
    assert torch.isnan(want).all(-1).nonzero().tolist() == [[2, h] for h in range(4)] + [[r, h] for r in (12, 13) for h in range(4, 8)]
    got = _run(q, k, v, table, ctx, plan)
    _same_nan(got, want, bound)
    assert bool((got[5] == 0).all())


@pytest.mark.parametrize("Hq,Hkv", [(8, 2), (32, 1)])
def test_values_that_are_alike_are_the_result(way, Hq, Hkv):
    """Weights are divided by the sum of the weights as they were multiplied, rounded ones, however many rows share a tile: the
    mean of equal values is that value but for fp32 sums (300 U32, far below half a step of bf16).  Of every
    32 keys the others are like one another, so that their weights beside the first's are all rounded by the same."""
    q, k, v, table, seqs, ctx, rows, most = _batch([(3, 2), (1, 1), (40, 3)], Hq, Hkv, 90, 6)
    g = torch.Generator().manual_seed(1)
    alike, first, other = (torch.randn(Hkv, 1, D, generator=g).bfloat16() for _ in range(3))
    k = torch.where(torch.isnan(k), k, torch.where((torch.arange(PAGE) % 32 == 0)[:, None], first, other))
    v = torch.where(torch.isnan(v), v, alike)
    plan = ops.prefix_plan(rows, Hq, Hkv, most, DEV)
    got = _run(q, k, v, table, ctx, plan).cpu().view(-1, Hkv, Hq // Hkv, D)
    assert torch.equal(got, alike[None].expand_as(got))


def test_values_near_the_type_s_largest(way):
    """Weights sum to 1: a result is no larger than its values, whatever the sums before the division are."""
    q, k, v, table, seqs, ctx, rows, most = _batch([(12, 2), (6, 1)], 8, 2, 90, 5)
    v[..., 5] = torch.where(torch.isnan(v[..., 5]), v[..., 5], torch.tensor(3e38).bfloat16())
    v[..., 9] = v[..., 9] * 2.0 ** 124
    q = q * 0.1                                # weights that are near one another
    plan = ops.prefix_plan(rows, 8, 2, most, DEV)
    want, bound = oracle.attention(q, k, v, table, seqs, ctx, 8, 2, 1 / math.sqrt(D), most)
    assert bool(torch.isfinite(want).all())
    _check(_run(q, k, v, table, ctx, plan), want, bound)


def test_rows_and_tables_of_any_stride_and_rows_behind_the_plan(way):
    q, k, v, table, seqs, ctx, rows, most = _batch([(9, 2)], 8, 2, 50, 9)
    wide = torch.randn(12, 8 * D + 3).bfloat16()
    wide[:9, 1:1 + 8 * D] = q
    out = torch.full((12, 8 * D + 5), 3.0, dtype=torch.bfloat16, device=DEV)
    tables = torch.full((9, table.shape[1] + 3), 10 ** 8, dtype=torch.int32)
    tables[:, :table.shape[1]] = table
    plan = ops.prefix_plan(rows, 8, 2, most, DEV)
    want, bound = oracle.attention(q, k, v, table, seqs, ctx, 8, 2, 1 / math.sqrt(D), most)
    got = ops.prefix_attention(wide.to(DEV)[:, 1:1 + 8 * D], k.to(DEV), v.to(DEV), tables.to(DEV)[:, :table.shape[1]],
                               ctx.to(DEV), plan, out=out[:, 2:2 + 8 * D])
    _check(got[:9], want, bound)
    assert bool((out[9:] == 3).all()) and bool((out[:, :2] == 3).all()) and bool((out[:, 2 + 8 * D:] == 3).all())


def test_pages_outside_of_the_cache_are_read_inside_it():
    q, k, v, table, seqs, ctx, rows, most = _batch([(4, 2)], 8, 2, 50, 9)
    k, v = k.nan_to_num(0.5), v.nan_to_num(0.5)
    want = table.clone()
    table[:, 1], want[:, 1] = 10 ** 9, len(k) - 1
    table[2, 2], want[2, 2] = -7, 0
    plan = ops.prefix_plan(rows, 8, 2, most, DEV)
    ref, bound = oracle.attention(q, k, v, want, seqs, ctx, 8, 2, 1 / math.sqrt(D), most)
    _check(_run(q, k, v, table, ctx, plan), ref, bound)


def test_one_plan_serves_a_captured_step_while_contexts_grow(way):
    """Two graphs with a workspace each, replayed in turn with eager work between; every replay is as the eager call."""
    q, k, v, table, seqs, ctx, rows, most = _batch([(11, 3), (4, 1)], 8, 2, 150, 21)
    k, v = k.nan_to_num(0.5), v.nan_to_num(0.5)
    plan = ops.prefix_plan(rows, 8, 2, most, DEV)
    q, k, v, table = q.to(DEV), k.to(DEV), v.to(DEV), table.to(DEV)
    ctxs, outs, graphs = [], [], []
    for i in range(2):
        ctxs.append(torch.ones(15, dtype=torch.int32, device=DEV))
        outs.append(torch.zeros(15, 8 * D, dtype=torch.bfloat16, device=DEV))
        ws = ops.prefix_workspace(plan)
        call = lambda: ops.prefix_attention(q, k, v, table, ctxs[i], plan, out=outs[i], workspace=ws)
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        graphs.append((graph, ws))
    for step in range(4):
        for i in range(2):
            ctxs[i].copy_(ctx - 3 + step * (i + 1))
            eager = ops.prefix_attention(q, k, v, table, ctxs[i], plan)
            graphs[i][0].replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[i], eager)


def test_prefix_attention_on_another_stream():
    q, k, v, table, seqs, ctx, rows, most = _batch([(9, 2)], 8, 2, 50, 9)
    plan = ops.prefix_plan(rows, 8, 2, most, DEV)
    want, bound = oracle.attention(q, k, v, table, seqs, ctx, 8, 2, 1 / math.sqrt(D), most)
    args = [t.to(DEV) for t in (q, k, v, table, ctx)]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = ops.prefix_attention(*args, plan)
    s.synchronize()
    _check(got, want, bound)


def test_pages_beyond_four_gigabytes():
    """A cache of 5 GB: offsets pass 32 bits."""
    q, k, v, table, seqs, ctx, rows, most = _batch([(5, 2)], 8, 2, 50, 9)
    P = 170000
    far = torch.empty(P, 2, PAGE, D, dtype=torch.bfloat16, device=DEV), torch.empty(P, 2, PAGE, D, dtype=torch.bfloat16, device=DEV)
    moved = torch.where(table > 0, P - table, table)
    for c, small in zip(far, (k, v)):
        c[0] = 0
        for p in range(1, len(small)):
            c[P - p] = small[p].to(DEV)
    plan = ops.prefix_plan(rows, 8, 2, most, DEV)
    want, bound = oracle.attention(q, k, v, table, seqs, ctx, 8, 2, 1 / math.sqrt(D), most)
    _check(ops.prefix_attention(q.to(DEV), *far, moved.to(DEV), ctx.to(DEV), plan), want, bound)
    ops.copy_pages(far[0][None], far[1][None], [P - 1, P - 2], [3, 4])
    for c, small in zip(far, (k, v)):
        assert torch.equal(c[3].cpu().view(torch.int16), small[1].view(torch.int16))
        assert torch.equal(c[4].cpu().view(torch.int16), small[2].view(torch.int16))
    ops.copy_pages(far[0][None], far[1][None], [3], [P - 2], [7])
    lens = ops.compact_pages(far[0][None], far[1][None], torch.tensor([[P - 2]], dtype=torch.int32, device=DEV),
                             torch.tensor([9], dtype=torch.int32, device=DEV), torch.arange(9, device=DEV)[None] >= 4)
    assert lens.tolist() == [5]
    for c, small in zip(far, (k, v)):
        want = torch.cat([small[1, :, 4:7], small[2, :, 7:9], small[1, :, 5:6]], 1)   # row 5: as it was
        assert torch.equal(c[P - 2, :, :6].cpu().view(torch.int16), want.view(torch.int16))


# ---------------------------------------------------------------------------------------- copies
def _caches(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 256, shape[:-1] + (shape[-1] * dtype.itemsize,), generator=g, dtype=torch.uint8).view(dtype)
            for _ in range(2)]


def _same(a, b):
    return torch.equal(a.cpu().contiguous().view(torch.uint8), b.cpu().contiguous().view(torch.uint8))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32, torch.uint8, torch.float8_e4m3fn])
@pytest.mark.parametrize("pairs", [1, 7, 300])
def test_copies(dtype, pairs):
    layers, kv = (2, 3) if pairs < 300 else (1, 1)
    k, v = _caches((layers, 2 * pairs + 5, kv, PAGE, D), dtype, pairs)
    g = torch.Generator().manual_seed(pairs)
    pages = torch.randperm(2 * pairs + 5, generator=g).tolist()
    src, dst = pages[:pairs], pages[pairs:2 * pairs]
    src[-1] = src[0]                                 # a page may be copied twice
    tokens = torch.randint(0, PAGE + 1, (pairs,), generator=g).tolist()
    tokens[0] = PAGE
    for n in (tokens, None):
        want = k.clone(), v.clone()
        ops.copy_pages(*want, src, dst, n)           # the reference, on the CPU
        for i, (s, d) in enumerate(zip(src, dst)):
            m = PAGE if n is None else n[i]
            assert _same(want[0][:, d, :, :m], k[:, s, :, :m]) and _same(want[1][:, d, :, m:], v[:, d, :, m:])
        got = k.to(DEV), v.to(DEV)
        ops.copy_pages(*got, torch.tensor(src), dst, n)
        assert _same(got[0], want[0]) and _same(got[1], want[1])


def test_copies_in_some_layers_and_heads():
    k, v = _caches((4, 9, 5, PAGE, D), torch.bfloat16, 4)
    kd, vd = k.to(DEV), v.to(DEV)
    for c in (k, v, kd, vd):
        part = c[1:3, 2:, 1:4]
        assert not part.is_contiguous()
    ops.copy_pages(k[1:3, 2:, 1:4], v[1:3, 2:, 1:4], [0, 3], [5, 6], [64, 9])
    ops.copy_pages(kd[1:3, 2:, 1:4], vd[1:3, 2:, 1:4], [0, 3], [5, 6], [64, 9])
    assert _same(kd, k) and _same(vd, v)


# ---------------------------------------------------------------------------------------- compaction
def _sequences(lens, seed, share=0.5, width=None):
    g = torch.Generator().manual_seed(seed)
    B, most = len(lens), max(max(lens), 1)
    W = width or -(-most // PAGE)
    pages = (torch.randperm(2 * B * W, generator=g) + 1).to(torch.int32)
    table, to = pages[:B * W].view(B, W), pages[B * W:].view(B, W)
    keep = torch.rand(B, most, generator=g) < share
    return table, to, torch.tensor(lens, dtype=torch.int32), keep


ROT = rope_table(LLAMA31_8B, max_pos=2048)


@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("turn", [False, True])
@pytest.mark.parametrize("lens,share", [([1], 1.0), ([1, 0, 5], 0.5), ([64, 65, 63], 0.0), ([300, 7, 128, 129], 0.5),
                                        ([1500], 0.9), ([513, 512], 0.03), ([200, 90], 1.0)])
def test_compaction(apart, turn, lens, share):
    table, to, n, keep = _sequences(lens, sum(lens), share)
    keep[0, :min(4, keep.shape[1])] = True               # the first tokens stay where they are
    k, v = (torch.randn(2, 1 + table.numel() * 2, 2, PAGE, D, generator=torch.Generator().manual_seed(i)).bfloat16()
            for i in range(2))
    rot = ROT if turn else None
    want_k, want_v, want_n, bound = oracle.compacted(k, v, table, n, keep, to if apart else None, rot)
    kd, vd = k.to(DEV), v.to(DEV)
    got = ops.compact_pages(kd, vd, table.to(DEV), n.to(DEV), keep.to(DEV), out_tables=to.to(DEV) if apart else None,
                            cos_sin=rot.to(DEV) if turn else None)
    assert got.tolist() == want_n and got.dtype == torch.int32
    assert torch.equal(vd.cpu().double(), want_v)
    assert bool(((kd.cpu().double() - want_k).abs() <= bound).all())
    kc, vc = k.clone(), v.clone()                        # the CPU's own
    assert ops.compact_pages(kc, vc, table, n, keep, out_tables=to if apart else None, cos_sin=rot).tolist() == want_n
    assert torch.equal(vc.double(), want_v) and bool(((kc.double() - want_k).abs() <= bound).all())


def _filled(shape, dtype, seed):
    if dtype == torch.uint8:
        return _caches(shape, dtype, seed)
    return [torch.randn(shape, generator=torch.Generator().manual_seed(seed + i)).to(dtype) for i in range(2)]


def _compacted_as(k, v, part, table, n, keep, to, rot):
    """Compaction of ``part`` of two caches on the GPU against the oracle's; the rest of them stays."""
    kd, vd = k.to(DEV), v.to(DEV)
    a, b, want_n, bound = oracle.compacted(part(k), part(v), table, n, keep, to, rot)
    got = ops.compact_pages(part(kd), part(vd), table.to(DEV), n.to(DEV), keep.to(DEV), out_tables=None if to is None else to.to(DEV),
                            cos_sin=None if rot is None else rot.to(DEV))
    assert got.tolist() == want_n
    kc, vc = kd.cpu(), vd.cpu()
    assert torch.equal(part(vc).double(), b) and bool(((part(kc).double() - a).abs() <= bound).all())
    part(kc).copy_(part(k))
    part(vc).copy_(part(v))
    assert torch.equal(kc, k) and torch.equal(vc, v)


@pytest.mark.parametrize("heads", [8, 7])      # pairs of heads of a workgroup, one head
@pytest.mark.parametrize("dtype,turn", [(torch.bfloat16, True), (torch.bfloat16, False), (torch.uint8, False), (torch.float32, False)])
def test_compaction_in_place_of_many_layers_and_heads(heads, dtype, turn):
    """16 layers and 3 sequences: two heads for a workgroup where they are even; heads 1 .. of a wider cache."""
    table, _to, n, keep = _sequences([300, 7, 129], 17, 0.6)
    keep[0, :70] = True
    k, v = _filled((16, 17, heads + 2, PAGE, D), dtype, 3)
    assert 16 * 8 * 3 >= 384      # where pairs begin
    _compacted_as(k, v, lambda c: c[:, :, 1:1 + heads], table, n, keep, None, ROT if turn else None)


@pytest.mark.parametrize("lens", [[2000, 700, 1500, 900], [620, 610, 600]])
@pytest.mark.parametrize("dtype,turn", [(torch.bfloat16, True), (torch.bfloat16, False), (torch.uint8, False), (torch.float32, False)])
def test_compaction_into_other_pages_of_many_layers_and_heads(lens, dtype, turn):
    """15 pairs of a layer and a head in fewer shares: a workgroup moves its tokens in several pairs, not equally many in each."""
    table, to, n, keep = _sequences(lens, 19, 0.5)
    chunks = -(-min(keep.shape[1], table.shape[1] * PAGE) // {1: 64, 2: 32, 4: 16}[dtype.itemsize])
    shares = max(1, min(15, 256 // (chunks * len(lens))))
    assert shares < 15 and (shares == 1 or 15 % shares)
    k, v = _filled((5, 1 + 2 * table.numel(), 4, PAGE, D), dtype, 5)
    _compacted_as(k, v, lambda c: c[:, :, :3], table, n, keep, to, ROT if turn else None)


@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.uint8])
def test_compaction_of_other_types_strides_and_lengths_past_the_table(apart, dtype):
    table, to, n, keep = _sequences([200, 5000, -3], 7, 0.6, width=3)
    keep = keep[:, :400]
    k, v = _caches((3, 20, 3, PAGE, D), dtype, 1)
    rows = torch.zeros(3, 2 * 400 + 3, dtype=torch.bool)
    rows[:, 1:401] = keep
    if dtype != torch.uint8:
        k, v = k.nan_to_num(0.5), v.nan_to_num(0.5)
    want_k, want_v = k.clone(), v.clone()
    part = lambda c: c[1:, :, :2]
    a, b, want_n, _ = oracle.compacted(part(k), part(v), table, n, keep, to if apart else None, None)
    want_k[1:, :, :2], want_v[1:, :, :2] = a.to(dtype), b.to(dtype)
    kd, vd = k.to(DEV), v.to(DEV)
    got = ops.compact_pages(part(kd), part(vd), table.to(DEV), n.to(DEV), rows.to(DEV)[:, 1:401],
                            out_tables=to.to(DEV) if apart else None)
    assert got.tolist() == want_n and want_n[2] == 0
    assert _same(kd, want_k) and _same(vd, want_v)


@pytest.mark.parametrize("apart", [False, True])
def test_compaction_skips_entries_that_are_no_pages(apart):
    table, to, n, keep = _sequences([300, 200], 11, 0.7)
    table[0, 2], to[1, 0] = 10 ** 9, -1
    k, v = _caches((1, 30, 2, PAGE, D), torch.bfloat16, 1)
    k, v = k.nan_to_num(0.5), v.nan_to_num(0.5)
    want_k, want_v, want_n, _ = oracle.compacted(k, v, table, n, keep, to if apart else None, None)
    kd, vd = k.to(DEV), v.to(DEV)
    got = ops.compact_pages(kd, vd, table.to(DEV), n.to(DEV), keep.to(DEV), out_tables=to.to(DEV) if apart else None)
    assert got.tolist() == want_n
    assert torch.equal(kd.cpu().double(), want_k) and torch.equal(vd.cpu().double(), want_v)


def test_compaction_of_a_sequence_of_more_pages_than_a_workgroup_holds():
    """263000 tokens in place, of which three leave: behind them all move."""
    n, W = 263000, 4110
    k, v = (torch.randn(1, W + 1, 1, PAGE, D, device=DEV).bfloat16() for _ in range(2))
    table = (torch.randperm(W, device=DEV).int() + 1)[None]
    gone = torch.tensor([261990, 262200, 262999], device=DEV)
    keep = torch.ones(1, n, dtype=torch.bool, device=DEV)
    keep[0, gone] = False
    flat = lambda c: c[0, :, 0][table[0].long()].reshape(-1, D)
    want = [flat(c)[:n][keep[0]] for c in (k, v)]
    assert ops.compact_pages(k, v, table, torch.tensor([n], dtype=torch.int32, device=DEV), keep).tolist() == [n - 3]
    assert torch.equal(flat(k)[:n - 3], want[0]) and torch.equal(flat(v)[:n - 3], want[1])


def test_nothing_to_compact():
    k, v = (torch.randn(1, 4, 1, PAGE, D, device=DEV).bfloat16() for _ in range(2))
    i32 = dict(dtype=torch.int32, device=DEV)
    assert ops.compact_pages(k, v, torch.zeros(0, 2, **i32), torch.zeros(0, **i32),
                             torch.zeros(0, 5, dtype=torch.bool, device=DEV)).shape == (0,)
    assert ops.compact_pages(k, v, torch.ones(1, 1, **i32), torch.ones(1, **i32),
                             torch.zeros(1, 0, dtype=torch.bool, device=DEV)).tolist() == [0]


def test_moves_in_a_captured_graph():
    """Copies and compaction replayed on new masks: every replay as the eager calls."""
    table, to, n, keep = _sequences([300, 90], 3, 0.5)
    k, v = (torch.randn(2, 30, 2, PAGE, D, device=DEV).bfloat16() for _ in range(2))
    table, to, n, keep = (t.to(DEV) for t in (table, to, n, keep))
    src, dst = to[0, :2].tolist(), [28, 29]
    def step(k, v):
        new = ops.compact_pages(k, v, table, n, keep, out_tables=to)
        ops.copy_pages(k, v, src, dst, [64, 5])
        return new
    gk, gv = k.clone(), v.clone()
    step(gk, gv)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        new = step(gk, gv)
    for i in range(4):
        keep.copy_(torch.rand(keep.shape, device=DEV) < 0.2 * (i + 1))
        ek, ev = gk.clone(), gv.clone()
        want = step(ek, ev)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(new, want) and torch.equal(gk, ek) and torch.equal(gv, ev)
