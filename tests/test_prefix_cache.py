"""Operators over shared pages on the CPU: what they refuse, how a plan cuts a batch, and their references."""
import random

import pytest
import torch

from p2p_llm_chat_go_amd import ops
from p2p_llm_chat_go_amd.models.config import LLAMA31_8B, rope_table
from p2p_llm_chat_go_amd.ops import prefix
from tests import prefix_oracle as oracle

PAGE, D = 64, 128
BF = torch.bfloat16


def _plan(groups=((3, 1),), heads=4, kv=2, ctx=128, **kw):
    return ops.prefix_plan(list(groups), heads, kv, ctx, "cpu", **kw)


@pytest.mark.parametrize("why,call", [
    ("query heads", lambda: _plan(heads=5)), ("query heads", lambda: _plan(heads=0)), ("query heads", lambda: _plan(kv=0)),
    ("query heads", lambda: _plan(heads=66)), ("max_ctx", lambda: _plan(ctx=0)), ("share 3 pages", lambda: _plan([(2, 3)])),
    ("group of 0", lambda: _plan([(0, 1)])), ("share -1", lambda: _plan([(1, -1)])), ("no rows", lambda: _plan([])),
    ("whole numbers", lambda: _plan([(1.5, 1)])), ("whole numbers", lambda: _plan(seqs=[0, 1, "2"])),
    ("seqs", lambda: _plan(seqs=[0, 1])), ("seqs", lambda: _plan(seqs=[0, 1, -1])),
])
def test_plans_that_are_refused(why, call):
    with pytest.raises(ValueError, match=why):
        call()


@pytest.mark.parametrize("way", [None, (4, True, 1, 1), (8, True, 3, 1), (4, True, 48, 8), (8, False, 1, 1), (4, False, 1, 16)])
def test_whatever_the_cut_every_key_of_a_row_is_in_one_part(way, monkeypatch):
    """way: the cut (None: the one that the plan chooses)."""
    if way is not None:
        monkeypatch.setattr(prefix._Shape, "choose", lambda self: way)
    rng = random.Random(0)
    for _ in range(30):
        kv = rng.choice([1, 2, 8])
        heads = kv * rng.choice([1, 2, 3, 4, 8, 32])
        groups, seqs, s = [], [], 0
        for _g in range(rng.randint(1, 4)):
            n = 0
            for _s in range(rng.randint(1, 30)):
                t = rng.choice([1, 1, 2, 40, 300])
                seqs += [s] * t
                n, s = n + t, s + 1
            groups.append((n, rng.choice([0, 1, 2, 30])))
        most = rng.randint(30 * PAGE, 40 * PAGE)
        plan = _plan(groups, heads, kv, most, seqs=seqs)
        R = len(seqs)
        counts = (plan.base[1:] - plan.base[:-1]).tolist()
        assert min(counts) >= 1 and plan.even == (counts[0] if len(set(counts)) == 1 else 0)
        assert plan.rows == R and plan.base[-1] == plan.parts and plan.row_tables.tolist() == seqs
        first, parts = [0] * R, [[] for _ in range(R)]
        at = 0
        for n, _p in groups:
            first[at:at + n] = [seqs[at]] * n
            at += n
        ctx = [rng.choice([0, 1, 64, 100, 1900, most]) for _ in range(R)]
        for row0, n, table, p0, p1, part, of, slot in plan.works.tolist():
            assert 1 <= n * (heads // kv) and (0 <= part < of or of == 0)
            seen = max(0, -(-min(max(ctx[row0:row0 + n]), p1 * PAGE) // PAGE) - p0)     # pages that some row sees
            a, b = (p0 + seen * part // of, p0 + seen * (part + 1) // of) if of else (p0, p1)
            for r in range(row0, row0 + n):
                assert table == seqs[r] or (table == first[r] and of == 0)
                parts[r].append((slot + part, a, b))
        for r in range(R):
            got = sorted(parts[r])
            assert [c for c, _, _ in got] == list(range(int(plan.base[r + 1] - plan.base[r])))
            pages = [p for _, a, b in got for p in range(a, b)]
            assert len(pages) == len(set(pages)) and set(range(-(-ctx[r] // PAGE))) <= set(pages)


def _given(**kw):
    a = dict(q=torch.randn(3, 4 * D).to(BF), k_cache=torch.randn(9, 2, PAGE, D).to(BF), v_cache=torch.randn(9, 2, PAGE, D).to(BF),
             block_tables=torch.tensor([[1, 2], [1, 3], [1, 4]], dtype=torch.int32),
             ctx_lens=torch.tensor([70, 0, 128], dtype=torch.int32), plan=_plan())
    a.update(kw)
    return a


@pytest.mark.parametrize("why,kw", [
    ("q must", dict(q=torch.zeros(2, 4 * D, dtype=BF))), ("q must", dict(q=torch.zeros(3, 4 * D))),
    ("q must", dict(q=torch.zeros(3, 2 * D, dtype=BF))), ("q must", dict(q=torch.zeros(4 * D, 3, dtype=BF).t())),
    ("k_cache", dict(k_cache=torch.zeros(9, 1, PAGE, D, dtype=BF))), ("v_cache", dict(v_cache=torch.zeros(9, 2, PAGE, D))),
    ("k_cache", dict(k_cache=torch.zeros(9, 4, PAGE, D, dtype=BF)[:, ::2])), ("differ", dict(v_cache=torch.zeros(8, 2, PAGE, D, dtype=BF))),
    ("block_tables", dict(block_tables=torch.zeros(2, 2, dtype=torch.int32))),
    ("block_tables", dict(block_tables=torch.zeros(3, 1, dtype=torch.int32))),
    ("block_tables", dict(block_tables=torch.zeros(3, 2, dtype=torch.int64))),
    ("ctx_lens", dict(ctx_lens=torch.zeros(2, dtype=torch.int32))), ("ctx_lens", dict(ctx_lens=torch.zeros(3))),
    ("scale", dict(scale=0.0)), ("scale", dict(scale=-1.0)), ("scale", dict(scale=float("nan"))),
    ("out must", dict(out=torch.zeros(3, 4 * D))), ("out must", dict(out=torch.zeros(2, 4 * D, dtype=BF))),
    ("out must", dict(out=torch.zeros(4 * D, dtype=BF).expand(3, -1))),
    ("q must", dict(q=torch.zeros(1, 1, dtype=BF, device="meta").as_strided((3, 4 * D), (2 ** 31, 1)))),
    ("one device", dict(ctx_lens=torch.zeros(3, dtype=torch.int32, device="meta"))),
])
def test_attention_that_is_refused(why, kw):
    with pytest.raises(ValueError, match=why):
        ops.prefix_attention(**_given(**kw))


@pytest.mark.parametrize("qs,outs,ok", [
    ((0, 4 * D), (0, 4 * D), False), ((0, 4 * D), (4 * D, 4 * D), False), ((0, 4 * D), (12 * D, 4 * D), True),
    ((12 * D, 4 * D), (0, 4 * D), True), ((0, 8 * D), (4 * D, 8 * D), True), ((4 * D, 8 * D), (0, 8 * D), True),
    ((0, 8 * D), (4 * D - 1, 8 * D), False), ((4 * D - 1, 8 * D), (0, 8 * D), False), ((0, 8 * D), (5 * D, 8 * D), False),
    ((0, 4 * D), (8 * D, 6 * D), False), ((0, 4 * D), (12 * D, 6 * D), True),
    ((0, 0), (0, 4 * D), False), ((0, 0), (4 * D, 4 * D), True), ((5 * D, 0), (0, 4 * D), False),
])
def test_out_is_other_memory_than_q(qs, outs, ok):
    """(start, stride) of both in one buffer: rows that lie between one another are fine."""
    buffer = torch.randn(60 * D).to(BF)
    a = _given(q=buffer.as_strided((3, 4 * D), (qs[1], 1), qs[0]), out=buffer.as_strided((3, 4 * D), (outs[1], 1), outs[0]))
    if ok:
        want = ops.prefix_attention(**dict(a, out=None))
        assert torch.equal(ops.prefix_attention(**a), want)
    else:
        with pytest.raises(ValueError, match="out overlaps q"):
            ops.prefix_attention(**a)


@pytest.mark.parametrize("scale", [1e-46, 2.0 ** -65, 2.0 ** 65, 1e39, 1e300])
def test_scales_that_fp32_scores_do_not_take_are_refused(scale):
    """Scores are fp32 numbers times the scale in fp32: one that is 0 or infinite there would leave no softmax."""
    with pytest.raises(ValueError, match="scale"):
        ops.prefix_attention(**_given(scale=scale))
    for fine in (2.0 ** -64, 2.0 ** 64):
        assert bool(torch.isfinite(ops.prefix_attention(**_given(scale=fine))).all())


def test_attention_on_the_cpu():
    a = _given()
    out = ops.prefix_attention(**a)
    want, bound = oracle.attention(a["q"], a["k_cache"], a["v_cache"], a["block_tables"], [0, 1, 2], a["ctx_lens"], 4, 2,
                                   D ** -0.5, 128)
    assert bool(((out.double().view(3, 4, D) - want).abs() <= bound).all()) and bool((out[1] == 0).all())


def test_attention_on_the_cpu_reads_entries_that_are_no_pages_inside_the_cache():
    a = _given()
    a["block_tables"] = torch.tensor([[1, 10 ** 9], [-7, 3], [-1, 4]], dtype=torch.int32)
    inside = torch.tensor([[1, 8], [0, 3], [0, 4]], dtype=torch.int32)
    want, bound = oracle.attention(a["q"], a["k_cache"], a["v_cache"], inside, [0, 1, 2], a["ctx_lens"], 4, 2, D ** -0.5, 128)
    assert bool(((ops.prefix_attention(**a).double().view(3, 4, D) - want).abs() <= bound).all())


def _pages(pages=8, **kw):
    return torch.zeros(2, pages, 2, PAGE, D, **kw), torch.zeros(2, pages, 2, PAGE, D, **kw)


@pytest.mark.parametrize("why,args", [
    ("pages must", ([8], [1])), ("pages must", ([-1], [1])), ("pages must", ([1], [8])), ("1 pages to 2", ([1], [2, 3])),
    ("numbers of tokens", ([1], [2], [3, 4])), ("tokens must", ([1], [2], [65])), ("tokens must", ([1], [2], [-1])),
    ("in dst twice", ([1, 2], [3, 3])), ("in src and in dst", ([1, 2], [2, 3])), ("whole numbers", ([1.0], [2])),
    ("whole numbers", (["1"], [2])), ("whole numbers", ([2 ** 40], [2])), ("host numbers", (torch.zeros(1, device="meta"), [2])),
])
def test_copies_that_are_refused(why, args):
    with pytest.raises(ValueError, match=why):
        ops.copy_pages(*_pages(), *args)


@pytest.mark.parametrize("k,v", [(torch.zeros(2, 8, 2, PAGE, 64), None), (torch.zeros(8, 2, PAGE, D), None),
                                 (torch.zeros(2, 8, 2, PAGE, D, dtype=torch.float64), None),
                                 (torch.zeros(2, 8, 2, D, PAGE).transpose(3, 4), None),
                                 (torch.zeros(2, 8, 2, PAGE, D), torch.zeros(2, 8, 1, PAGE, D)),
                                 (torch.zeros(2, 8, 2, PAGE, D), torch.zeros(2, 8, 2, PAGE, D, dtype=BF))])
def test_caches_that_are_refused(k, v):
    with pytest.raises(ValueError):
        ops.copy_pages(k, k if v is None else v, [1], [2])
    i32 = dict(dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.compact_pages(k, k if v is None else v, torch.ones(1, 1, **i32), torch.ones(1, **i32), torch.ones(1, 3, dtype=torch.bool))


@pytest.mark.parametrize("dim", [0, 1, 2])
def test_caches_that_repeat_their_memory_are_refused(dim):
    """An expanded cache has one memory for several layers, pages or heads, which would be written at once."""
    k, v = _pages()
    again = k.select(dim, 0).unsqueeze(dim).expand_as(k)
    i32 = dict(dtype=torch.int32)
    for a, b in ((again, v), (v, again)):
        with pytest.raises(ValueError, match="memory of their own"):
            ops.copy_pages(a, b, [1], [2])
        with pytest.raises(ValueError, match="memory of their own"):
            ops.compact_pages(a, b, torch.ones(1, 1, **i32), torch.ones(1, **i32), torch.ones(1, 3, dtype=torch.bool))
    one = k[:1, :, :1]
    ops.copy_pages(one.expand(1, -1, 1, -1, -1), one.clone(), [1], [2])


def test_nothing_to_copy():
    k, v = _pages()
    k[:, 3] = 1
    ops.copy_pages(k, v, [], [])
    ops.copy_pages(k, v, [3, 3], [3, 4])
    assert bool((k[:, 3:5] == 1).all())


@pytest.mark.parametrize("why,kw", [
    ("block_tables", dict(block_tables=torch.zeros(2, 3, dtype=torch.int64))), ("lens", dict(lens=torch.zeros(3, dtype=torch.int32))),
    ("lens", dict(lens=torch.zeros(2))), ("keep", dict(keep=torch.zeros(2, 9, dtype=torch.uint8))),
    ("keep", dict(keep=torch.zeros(3, 9, dtype=torch.bool))), ("out_tables", dict(out_tables=torch.zeros(2, 2, dtype=torch.int32))),
    ("bf16 caches only", dict(cos_sin=torch.zeros(200, 64, 2))),
    ("cos_sin", dict(bf=True, cos_sin=torch.zeros(99, 64, 2))), ("cos_sin", dict(bf=True, cos_sin=torch.zeros(200, 64, 2, dtype=BF))),
    ("one device", dict(lens=torch.zeros(2, dtype=torch.int32, device="meta"))),
    ("block_tables", dict(block_tables=torch.zeros(3, 2, dtype=torch.int32).t())), ("block_tables", dict(block_tables=torch.zeros(2, dtype=torch.int32))),
    ("too far", dict(block_tables=torch.ones(1, dtype=torch.int32, device="meta").as_strided((2, 3), (2 ** 31, 1)))),
    ("out_tables", dict(out_tables=torch.zeros(2, dtype=torch.int32))), ("out_tables", dict(out_tables=torch.zeros(2, 3))),
    ("cos_sin", dict(bf=True, cos_sin=torch.zeros(200, 128))), ("cos_sin", dict(bf=True, cos_sin=torch.zeros(200, 64, 4)[..., ::2])),
])
def test_compaction_that_is_refused(why, kw):
    a = dict(block_tables=torch.ones(2, 3, dtype=torch.int32), lens=torch.ones(2, dtype=torch.int32),
             keep=torch.ones(2, 100, dtype=torch.bool))
    bf = kw.pop("bf", False) if isinstance(kw, dict) else False
    k, v = _pages(dtype=BF if bf else torch.float32)
    a.update(kw)
    with pytest.raises(ValueError, match=why):
        ops.compact_pages(k, v, **a)


@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("turn", [False, True])
def test_compaction_skips_entries_that_are_no_pages(apart, turn):
    gen = torch.Generator().manual_seed(5)
    k, v = (torch.randn(2, 12, 2, PAGE, D, generator=gen).bfloat16() for _ in range(2))
    table, to = torch.tensor([[1, 2, 10 ** 9], [4, -1, 5]], dtype=torch.int32), torch.tensor([[6, 12, 7], [-5, 8, 9]],
                                                                                             dtype=torch.int32)
    n, keep = torch.tensor([190, 150], dtype=torch.int32), torch.rand(2, 192, generator=gen) < 0.8
    to, rot = to if apart else None, rope_table(LLAMA31_8B, max_pos=192) if turn else None
    want_k, want_v, want_n, bound = oracle.compacted(k, v, table, n, keep, to, rot)
    assert ops.compact_pages(k, v, table, n, keep, out_tables=to, cos_sin=rot).tolist() == want_n
    assert torch.equal(v.double(), want_v) and bool(((k.double() - want_k).abs() <= bound).all())
