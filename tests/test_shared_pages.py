"""Sequences that share pages: the allocator's owners, ``KVCache.fork`` and ``compact``, and generation over a shared prefix."""
import pytest
import torch

from p2p_llm_chat_go_amd import ops
from p2p_llm_chat_go_amd.engine import Engine
from p2p_llm_chat_go_amd.engine.engine import common_prefix
from p2p_llm_chat_go_amd.engine.kv_cache import KVCache, PageAllocator, pages_for
from p2p_llm_chat_go_amd.models import LLAMA31_8B, TINY_LLAMA
from p2p_llm_chat_go_amd.models.config import TINY_LLAMA_GQA, rope_table
from p2p_llm_chat_go_amd.models.reference import random_state_dict
from p2p_llm_chat_go_amd.models.weights import EngineWeights
from tests import prefix_oracle as oracle
from tests.test_engine import _greedy_ok

PAGE = 64
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def test_a_page_is_free_when_its_last_owner_frees_it():
    a = PageAllocator(8)
    p = a.alloc(3)
    a.share(p[:2])
    a.share(p[:1])
    assert a.free_pages == 4 and a.shared(p[0]) and a.shared(p[1]) and not a.shared(p[2])
    a.free(p)
    assert a.free_pages == 5 and a.shared(p[0]) and not a.shared(p[1])
    a.free(p[:2])
    assert a.free_pages == 6
    a.free(p[:1])
    assert a.free_pages == 7 and not a.shared(p[0])
    with pytest.raises(ValueError, match="bad page"):
        a.share([0])
    with pytest.raises(ValueError, match="bad page"):
        a.share([8])
    assert sorted(a.alloc(7)) == list(range(1, 8))


def _cache(device, pages=24, seed=0):
    kv = KVCache(TINY_LLAMA, pages, device)
    g = torch.Generator().manual_seed(seed)
    for c in (kv.k, kv.v):
        c.copy_(torch.randn(c.shape, generator=g))
    return kv


def _tokens(cache, pages, n):
    """[layers, heads, n, 128] of a sequence."""
    t = torch.arange(n)
    return cache.cpu()[:, torch.tensor(pages)[t // PAGE], :, t % PAGE].permute(1, 2, 0, 3)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("tokens", [0, 1, 64, 100, 128])
def test_forks_hold_the_tokens_that_they_begin_with(device, tokens):
    kv = _cache(device)
    mine = kv.allocator.alloc(3)
    want = _tokens(kv.k, mine, tokens), _tokens(kv.v, mine, tokens)
    forks = kv.fork(mine, tokens, [3, pages_for(tokens), 4])
    full = tokens // PAGE
    assert [len(f) for f in forks] == [3, pages_for(tokens), 4]
    assert all(f[:full] == mine[:full] for f in forks)
    own = [p for f in forks for p in f[full:]] + mine
    assert len(own) == len(set(own))
    for f in forks:
        if tokens:
            assert torch.equal(_tokens(kv.k, f, tokens), want[0]) and torch.equal(_tokens(kv.v, f, tokens), want[1])
    kv.allocator.free(mine)
    for f in forks:
        kv.allocator.free(f)
    assert kv.allocator.free_pages == 23


def test_forks_that_are_refused():
    kv = _cache("cpu", 6)
    mine = kv.allocator.alloc(2)
    for tokens, sizes, why in ((129, [3], "129 tokens of 2"), (-1, [3], "-1 tokens"), (65, [2, 1], "asked for 1")):
        with pytest.raises(ValueError, match=why):
            kv.fork(mine, tokens, sizes)
    with pytest.raises(MemoryError):
        kv.fork(mine, 64, [3, 3])
    for bad in ([0, mine[1]], [mine[0], 6], [mine[0], -1]):
        with pytest.raises(ValueError, match="bad page"):
            kv.fork(bad, 70, [2])
    assert kv.allocator.free_pages == 3 and not kv.allocator.shared(mine[0])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("turn", [False, True])
def test_compaction_leaves_the_pages_of_others_alone(device, turn):
    """Three sequences: one of its own, two that share their first page (and one of those has nothing left)."""
    kv = _cache(device)
    a, b = kv.allocator.alloc(4), kv.allocator.alloc(2)
    c, = kv.fork(b, 70, [2])
    lens = [200, 70, 100]
    g = torch.Generator().manual_seed(1)
    keep = torch.rand(3, 210, generator=g) < 0.6
    keep[1] = False
    rot = rope_table(TINY_LLAMA, max_pos=256)
    k0, v0, b_tokens = kv.k.cpu().clone(), kv.v.cpu().clone(), _tokens(kv.k, b, 70)
    d, = kv.fork(b, 70, [2])       # another owner of b's first page, not compacted
    free = kv.allocator.free_pages
    pages, left = kv.compact([a, b, c], lens, keep if device == "cpu" else keep.to(device), rot.to(device) if turn else None,
                             room=3)
    at = torch.arange(210)
    assert left == [int((keep[i] & (at < lens[i])).sum()) for i in range(3)] and left[1] == 0
    assert [len(p) for p in pages] == [pages_for(n + 3) for n in left]
    assert pages[0] == a[:len(pages[0])]
    assert torch.equal(_tokens(kv.k, d, 70), b_tokens)
    for i, old in enumerate((a, b, c)):
        table = torch.zeros(1, 4, dtype=torch.int32)
        table[0, :len(old)] = torch.tensor(old)
        want_k, want_v, n, bound = oracle.compacted(k0, v0, table, [lens[i]], keep[i:i + 1], table, rot if turn else None)
        assert n == [left[i]]
        if n[0]:
            take = lambda x, p: x[:, torch.tensor(p)[at[:n[0]] // PAGE], :, at[:n[0]] % PAGE]
            assert bool(((take(kv.k.cpu().double(), pages[i]) - take(want_k, old)).abs() <= take(bound, old)).all())
            assert torch.equal(take(kv.v.cpu().double(), pages[i]), take(want_v, old))
    for p in pages + [d]:
        kv.allocator.free(p)
    assert kv.allocator.free_pages == 23 and free < 23


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("cfg", [TINY_LLAMA, LLAMA31_8B], ids=lambda c: c.name)
def test_turned_keys_are_the_keys_that_the_model_rotates_for_the_new_places(device, cfg):
    """``ops.rope_cache`` for the old positions and compaction, against ``ops.rope_cache`` for the new ones."""
    n, KV, rot = 300, 2, rope_table(cfg, max_pos=320)
    g = torch.Generator().manual_seed(9)
    qkv = torch.randn(n, (2 + 2 * KV) * 128, generator=g).bfloat16()
    keep = torch.rand(1, n, generator=g) < 0.5
    keep[0, :3] = True
    left = int(keep.sum())
    table = (torch.randperm(5, generator=g) + 1).to(torch.int32)
    slots = lambda m: (table[torch.arange(m) // PAGE] * PAGE + torch.arange(m) % PAGE).int()
    def rotated(rows):
        m = len(rows)
        k, v = (torch.zeros(6, KV, PAGE, 128, dtype=torch.bfloat16, device=device) for _ in range(2))
        ops.rope_cache(rows.to(device), torch.arange(m, dtype=torch.int32, device=device), slots(m).to(device), rot.to(device), 2, KV,
                       torch.empty(m, 256, dtype=torch.bfloat16, device=device), k, v)
        return k[None], v[None]
    k, v = rotated(qkv)
    before = _tokens(k, table.tolist(), n)[:, :, keep[0]].double()
    assert ops.compact_pages(k, v, table[None].to(device), torch.tensor([n], dtype=torch.int32, device=device), keep.to(device),
                             cos_sin=rot.to(device)).tolist() == [left]
    want_k, want_v = (_tokens(c, table.tolist(), left).double() for c in rotated(qkv[keep[0]]))
    got = _tokens(k, table.tolist(), left).double()
    # old keys rounded (half a step of both numbers of a pair), the turned and the wanted ones rounded; products in fp32
    x1, x2 = before.abs().chunk(2, -1)
    pair = (x1 + x2).repeat(1, 1, 1, 2)
    bound = oracle.U16 * (pair + got.abs() + want_k.abs()) + 24 * oracle.U32 * pair
    assert bool(((got - want_k).abs() <= bound).all())
    assert torch.equal(_tokens(v, table.tolist(), left).double(), want_v)


def test_compactions_that_are_refused():
    kv = _cache("cpu", 8)
    a = kv.allocator.alloc(2)
    keep = torch.ones(1, 128, dtype=torch.bool)
    for args, why in ((([a], [129], keep), "a length of 129"), (([a], [100], keep[:, :50]), "a length of 100"),
                      (([a], [100, 3], keep), "2 lengths"), (([a, a], [5, 5], keep.repeat(2, 1)), "given twice")):
        with pytest.raises(ValueError, match=why):
            kv.compact(*args)
    with pytest.raises(MemoryError):
        kv.compact([a], [100], keep, room=1000)
    b, = kv.fork(a, 128, [2])
    for args, kw, why in ((([a, b, a], [9] * 3, keep.repeat(3, 1)), {}, "more sequences than own it"),
                          (([a], [100], keep), dict(room=-1), "room for -1"), (([[a[0], 8]], [9], keep), {}, "bad page 8"),
                          (([[0]], [9], keep), {}, "bad page 0"), (([a], [9], keep), dict(cos_sin=torch.zeros(9, 64, 2)), "cos_sin")):
        with pytest.raises(ValueError, match=why):
            kv.compact(*args, **kw)
    assert kv.compact([], [], keep[:0]) == ([], [])
    kv.allocator.free(a)
    kv.allocator.free(b)
    assert kv.allocator.free_pages == 7


def test_a_fork_whose_copy_is_refused_takes_no_pages():
    kv = KVCache(TINY_LLAMA, 8, "cpu", dtype=torch.float64)      # a type that copies do not take
    mine = kv.allocator.alloc(2)
    with pytest.raises(ValueError, match="float64"):
        kv.fork(mine, 100, [2])
    assert kv.allocator.free_pages == 5 and not kv.allocator.shared(mine[0])


def test_pages_that_nobody_owns_are_refused():
    """A page that is free is not shared, forked, compacted or freed once more: it would be handed out while it is held."""
    kv = _cache("cpu", 8)
    a = kv.allocator
    one, = a.alloc(1)
    assert a.owners(one) == 1
    a.free([one])
    assert a.owners(one) == 0
    keep = torch.ones(1, 64, dtype=torch.bool)
    for call in (lambda: a.share([one]), lambda: kv.fork([one], 64, [2]), lambda: kv.compact([[one]], [64], keep),
                 lambda: a.free([one])):
        with pytest.raises(ValueError, match="page %d is free" % one):
            call()
        assert a.free_pages == 7 and not a.shared(one)
    two = a.alloc(2)
    with pytest.raises(ValueError, match="more often than"):      # nothing is freed where one of them cannot be
        a.free([two[1], two[0], two[0]])
    assert a.free_pages == 5
    a.share(two[:1])
    a.free([two[0], two[0], two[1]])
    assert sorted(a.alloc(7)) == list(range(1, 8))


def test_a_page_twice_in_one_sequence_is_refused():
    """Two owners of a page are two sequences: one that lists it twice would give up the other's, too."""
    kv = _cache("cpu", 8)
    a = kv.allocator.alloc(2)
    b, = kv.fork(a, 128, [2])
    keep = torch.ones(2, 128, dtype=torch.bool)
    for pages, lens in (([[a[0], a[0]]], [128]), ([a, [b[1], b[1]]], [128, 9])):
        with pytest.raises(ValueError, match="given twice"):
            kv.compact(pages, lens, keep[:len(pages)])
    with pytest.raises(ValueError, match="given twice"):
        kv.fork([a[0], a[0]], 128, [2])
    assert kv.allocator.free_pages == 5 and all(kv.allocator.owners(p) == 2 for p in a)
    kv.allocator.free(a)
    kv.allocator.free(b)
    assert sorted(kv.allocator.alloc(7)) == list(range(1, 8))


def test_common_prefixes():
    assert common_prefix([[1, 2, 3], (1, 2, 3, 4)]) == 2
    assert common_prefix([[1, 2, 3], [1, 2, 4, 5]]) == 2 and common_prefix([[1, 2, 3], [1, 2, 3]]) == 2
    assert common_prefix([[1], [1, 2]]) == 0 and common_prefix([[5, 6], [1, 6]]) == 0


def _prompts(shared, tails, seed=3):
    g = torch.Generator().manual_seed(seed)
    draw = lambda n: torch.randint(3, 250, (n,), generator=g).tolist()
    head = draw(shared)
    return [head + draw(n) for n in tails]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("shared,tails,chunk", [(100, [5, 1, 30], 1024), (128, [3, 3], 1024), (64, [40, 2], 16), (20, [4, 4], 1024),
                                                (70, [9], 1024)])
def test_generation_over_a_shared_prefix(device, shared, tails, chunk):
    """The shared tokens once, forks, prompt rows and decode steps behind them; pages all come back."""
    cfg = TINY_LLAMA
    sd = random_state_dict(cfg, seed=1)
    eng = Engine(cfg, weights=EngineWeights.from_state_dict(sd, cfg, device), device=device, kv_pages=64, max_prefill_tokens=chunk,
                 max_batch=4)
    prompts = _prompts(shared, tails)
    res = eng.generate(prompts, max_new_tokens=9, stop_on_eos=False, share_prefix=True)
    for p, r in zip(prompts, res):
        assert len(r.tokens) == 9 and r.prompt_eval_count == len(p)
        _greedy_ok(sd, cfg, p, r.tokens)
    assert eng.kv.allocator.free_pages == 63
    if device == "cpu":
        assert [r.tokens for r in res] == [r.tokens for r in eng.generate(prompts, 9, stop_on_eos=False)]
    else:
        again = eng.generate(prompts, max_new_tokens=9, stop_on_eos=False, share_prefix=True)   # the graph that is there
        assert [r.tokens for r in again] == [r.tokens for r in res]
        other = eng.generate(prompts[:1] + prompts, 9, stop_on_eos=False, share_prefix=True)     # another batch of its bucket
        assert [r.tokens for r in other[1:]] == [r.tokens for r in res]


@pytest.mark.parametrize("shared,tails,forked", [(600, [5, 1], True), (500, [5, 1], False), (130, [5, 1, 30, 8], False),
                                                 (260, [5, 1, 30], True), (500, [9], False)])
def test_prefixes_are_shared_where_that_saves_enough(shared, tails, forked, monkeypatch):
    cfg = TINY_LLAMA
    eng = Engine(cfg, weights=EngineWeights.from_state_dict(random_state_dict(cfg, seed=1), cfg, "cpu"), device="cpu", kv_pages=64,
                 max_batch=4)
    calls, fork = [], eng.kv.fork
    monkeypatch.setattr(eng.kv, "fork", lambda *a: calls.append(a) or fork(*a))
    prompts = _prompts(shared, tails)
    with_it = eng.generate(prompts, 3, stop_on_eos=False, share_prefix=True)
    assert bool(calls) == forked and eng.kv.allocator.free_pages == 63
    assert [r.tokens for r in with_it] == [r.tokens for r in eng.generate(prompts, 3, stop_on_eos=False)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("shared,tails,chunk", [(100, [5, 1, 30], 1024), (128, [3, 3], 1024), (64, [40, 2], 16), (300, [5, 1, 30], 1024),
                                                (640, [9, 70, 3], 200)])
def test_generation_over_every_prefix_of_a_page(device, shared, tails, chunk):
    """Shared, however little that saves."""
    cfg = TINY_LLAMA
    sd = random_state_dict(cfg, seed=1)
    eng = Engine(cfg, weights=EngineWeights.from_state_dict(sd, cfg, device), device=device, kv_pages=64, max_prefill_tokens=chunk,
                 max_batch=4)
    eng.share_prefix_min = eng.share_steps_min = 0
    prompts = _prompts(shared, tails)
    for _again in range(2):
        for p, r in zip(prompts, eng.generate(prompts, max_new_tokens=9, stop_on_eos=False, share_prefix=True)):
            assert len(r.tokens) == 9 and r.prompt_eval_count == len(p)
            _greedy_ok(sd, cfg, p, r.tokens)
    assert eng.kv.allocator.free_pages == 63


@pytest.mark.gpu
@pytest.mark.parametrize("shared,tails,fused", [(130, [5, 1, 30], True), (300, [5, 1, 30], False)])
def test_steps_of_short_contexts_keep_the_model_s_fused_attention(shared, tails, fused):
    cfg = TINY_LLAMA
    sd = random_state_dict(cfg, seed=1)
    eng = Engine(cfg, weights=EngineWeights.from_state_dict(sd, cfg, "cuda"), device="cuda", kv_pages=64, max_batch=4)
    eng.share_prefix_min = eng.share_steps_min = 0
    prompts = _prompts(shared, tails)
    for p, r in zip(prompts, eng.generate(prompts, max_new_tokens=9, stop_on_eos=False, share_prefix=True)):
        assert len(r.tokens) == 9
        _greedy_ok(sd, cfg, p, r.tokens)
    assert bool(eng._graphs) == fused and bool(eng._shared_graphs) != fused
    assert eng.kv.allocator.free_pages == 63


@pytest.mark.gpu
def test_a_graph_over_shared_pages_is_captured_where_its_steps_earn_it():
    cfg = TINY_LLAMA
    sd = random_state_dict(cfg, seed=1)
    eng = Engine(cfg, weights=EngineWeights.from_state_dict(sd, cfg, "cuda"), device="cuda", kv_pages=64, max_batch=4)
    # a page of a layer's K and V are 32 KB: 8 steps of 2 more sequences behind 10 pages do not read 5.2 MB again
    prompts = _prompts(650, [5, 1, 30])
    for least, captured in ((8 * 2 * 10 * 32768 + 1, False), (8 * 2 * 10 * 32768, True), (10 ** 9, True)):
        eng.share_steps_min = least
        for p, r in zip(prompts, eng.generate(prompts, max_new_tokens=9, stop_on_eos=False, share_prefix=True)):
            assert len(r.tokens) == 9
            _greedy_ok(sd, cfg, p, r.tokens)
        assert bool(eng._shared_graphs) == captured       # (and one that is there is taken, whatever the steps)
    assert not eng.shared_steps(3, 690, 9, 8) and eng.shared_steps(3, 690, 10, 1)
    assert eng.kv.allocator.free_pages == 63


@pytest.mark.parametrize("B,shared,own,parts", [(19, 2048, 301, 2), (5, 2048, 301, 2), (5, 32768, 300, 8), (3, 512, 70, 1)])
def test_decode_graphs_are_planned_for_the_batch_that_they_run(B, shared, own, parts):
    """Not for the bucket's longest context nor for its rows without a sequence: rows behind a long prefix read it together."""
    cfg = TINY_LLAMA_GQA.replace(max_pos=40000)
    sd = random_state_dict(cfg, seed=1)
    eng = Engine(cfg, weights=EngineWeights.from_state_dict(sd, cfg, "cpu"), device="cpu", kv_pages=16, max_batch=32)
    g = eng.shared_decode_graph(B, shared + own, shared // PAGE)
    plan, _ws = g.state.prefix["prefix"]
    assert plan.rows == B and shared + own <= plan.max_ctx <= g.state.max_ctx
    together = [w for w in plan.works.tolist() if w[6] == 0]       # (of 0: pages that a group shares)
    assert len(together) >= parts and {p for w in together for p in range(w[3], w[4])} == set(range(shared // PAGE))
    assert eng.shared_decode_graph(B, shared + own - 3, shared // PAGE) is g
    assert g.state.B > B and bool((g.state.ws.attn == 0).all())     # rows without a sequence attend to nothing
    plan, _ws = eng.shared_decode_graph(B, shared + own + g.state.max_ctx // 8, shared // PAGE).state.prefix["prefix"]
    assert plan.max_ctx >= shared + own + g.state.max_ctx // 8      # a longer batch of the same bucket has a plan of its own


@pytest.mark.parametrize("device", DEVICES)
def test_prompts_over_shared_pages_have_the_logits_of_prompts_of_their_own(device):
    cfg = TINY_LLAMA
    sd = random_state_dict(cfg, seed=2)
    eng = Engine(cfg, weights=EngineWeights.from_state_dict(sd, cfg, device), device=device, kv_pages=64, max_batch=4)
    prompts = _prompts(150, [7, 80, 1])
    a = [eng.kv.allocator.alloc(pages_for(len(p))) for p in prompts]
    _, want = eng.prefill(prompts, a, return_logits=True)
    b = [eng.kv.allocator.alloc(pages_for(len(prompts[0])))]
    eng.prefill([prompts[0][:150]], b)
    b += eng.kv.fork(b[0], 150, [pages_for(len(p)) for p in prompts[1:]])
    _, got = eng.prefill(prompts, b, return_logits=True, starts=[150] * 3, shared_pages=2)
    assert float((got - want).norm() / want.norm()) < 2e-2      # two runs of bf16 layers
    with pytest.raises(ValueError, match="shared pages"):
        eng.prefill(prompts, b, starts=[150, 100, 150], shared_pages=2)
    with pytest.raises(ValueError, match="shared pages"):
        eng.prefill(prompts, b, shared_pages=2)


def _forward_without(sd, cfg, tokens, gone, n):
    """fp32 logits of a causal forward, where tokens from n on do not see those of ``gone`` (the ones before n do)."""
    T, D, H, KV = len(tokens), cfg.head_dim, cfg.n_heads, cfg.n_kv_heads
    cs = rope_table(cfg, max_pos=T)
    cos, sin = cs[..., 0][:, None], cs[..., 1][:, None]
    unseen = torch.ones(T, T, dtype=torch.bool).triu(1)
    unseen[n:, gone] = True
    x = sd["model.embed_tokens.weight"].float()[torch.tensor(tokens)]
    norm = lambda x, w: x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + cfg.eps) * w.float()
    turn = lambda x: torch.cat([x[..., :D // 2] * cos - x[..., D // 2:] * sin, x[..., D // 2:] * cos + x[..., :D // 2] * sin], -1)
    for i in range(cfg.n_layers):
        w = lambda name: sd["model.layers.%d.%s.weight" % (i, name)].float()
        h = norm(x, w("input_layernorm"))
        q, k, v = ((h @ w("self_attn.%s_proj" % c).t()).view(T, m, D) for c, m in (("q", H), ("k", KV), ("v", KV)))
        k, v = (t.repeat_interleave(H // KV, 1).transpose(0, 1) for t in (turn(k), v))
        s = (turn(q).transpose(0, 1) @ k.transpose(1, 2).contiguous() / D ** 0.5).masked_fill(unseen, -float("inf"))
        x = x + (torch.softmax(s, -1) @ v).transpose(0, 1).reshape(T, -1) @ w("self_attn.o_proj").t()
        h = norm(x, w("post_attention_layernorm"))
        x = x + (torch.nn.functional.silu(h @ w("mlp.gate_proj").t()) * (h @ w("mlp.up_proj").t())) @ w("mlp.down_proj").t()
    x = norm(x, sd["model.norm.weight"])
    return x @ sd["model.embed_tokens.weight" if cfg.tie_embeddings else "lm_head.weight"].float().t()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("share", [False, True])
def test_a_sequence_goes_on_behind_a_compaction(device, share):
    """With its keys turned by the engine's calls, at its new length; with its keys as they are by ``LlamaModel.forward``, whose
    positions count on while slots and lengths are the compacted ones."""
    cfg = TINY_LLAMA
    sd = random_state_dict(cfg, seed=4)
    for name in sd:     # attention that tells places and tokens apart: keys that were not turned are 3e-2 off, those of gone tokens 6e-2
        sd[name] = sd[name] * (4 if "q_proj" in name else 8 if "v_proj" in name else 1)
    eng = Engine(cfg, weights=EngineWeights.from_state_dict(sd, cfg, device), device=device, kv_pages=64, max_batch=4)
    thread, = _prompts(0, [210], seed=8)
    n, more = 190, 20
    keep = torch.ones(1, n, dtype=torch.bool)
    keep[0, 4:90] = torch.rand(86, generator=torch.Generator().manual_seed(2)) < 0.3
    gone = (~keep[0]).nonzero()[:, 0]
    want = _forward_without({k: v.float().cpu() for k, v in sd.items()}, cfg, thread, gone, n)
    logits = {}
    for turned in (True, False):
        pages = [eng.kv.allocator.alloc(pages_for(n))]
        eng.prefill([thread[:n]], pages)
        if share:        # another sequence holds the pages: into new ones
            eng.kv.fork(pages[0], n, [pages_for(n)])
        pages, (left,) = eng.kv.compact(pages, [n], keep, eng.model.rope if turned else None, room=more + 4)
        assert left == int(keep.sum())
        rest = thread[n:]
        if turned:
            kept = [t for t, k in zip(thread, keep[0].tolist()) if k]
            first, out = eng.prefill([kept + rest], pages, return_logits=True, starts=[left])
            logits[turned] = out[0].float().cpu()
            steps = [int(first[0])]
            steps += eng.decode_steps(steps, [left + more], pages, left + more + 4, 3)[0]
        else:
            dev = eng.device
            ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
            table = ints(pages)
            at = list(range(left, left + more))
            ws = eng.model.new_workspace(more, 256)
            out = eng.model.forward(ws, ints(rest), ints(range(n, n + more)), ints([pages[0][a // PAGE] * PAGE + a % PAGE for a in at]),
                                    table, ints([0] * more), ints([a + 1 for a in at]), more, 256)
            logits[turned] = out[-1].float().cpu()
    for got in logits.values():
        assert float((got - want[-1]).norm() / want[-1].norm()) < 2e-2      # bf16 layers against fp32
    toks = list(thread)
    for t in steps:
        ref = _forward_without({k: v.float().cpu() for k, v in sd.items()}, cfg, toks, gone, n)[-1]
        assert float(ref.max() - ref[t]) < 2e-2 * float(ref.abs().max())
        toks.append(t)


def test_prompts_whose_tables_do_not_share_their_pages_are_refused():
    cfg = TINY_LLAMA
    eng = Engine(cfg, weights=EngineWeights.from_state_dict(random_state_dict(cfg, seed=2), cfg, "cpu"), device="cpu", kv_pages=64)
    prompts = _prompts(150, [7, 80])
    pages = [eng.kv.allocator.alloc(4)]
    eng.prefill([prompts[0][:150]], pages)
    pages += eng.kv.fork(pages[0], 150, [4])
    eng.prefill(prompts, pages, starts=[150] * 2, shared_pages=2)
    eng.prefill(prompts, [tuple(pages[0]), torch.tensor(pages[1])], starts=[150] * 2, shared_pages=2)    # whatever holds the numbers
    for tables, n in (([pages[0], [pages[1][0]] + pages[1][2:]], 2), (pages, 3), ([pages[0], pages[1][:1]], 2), (pages, -1)):
        with pytest.raises(ValueError, match="share"):
            eng.prefill(prompts, tables, starts=[200] * 2, shared_pages=n)


@pytest.mark.gpu
def test_forks_attention_and_compaction_one_after_the_other():
    """A thread forks, rows of both attend the shared pages, tokens leave both, and rows attend what is left."""
    cfg = TINY_LLAMA
    kv = _cache("cuda", 40, seed=5)
    H, KV = cfg.n_heads, cfg.n_kv_heads
    mine = kv.allocator.alloc(5)
    tables = [mine] + kv.fork(mine, 230, [5, 4])
    lens = [300, 310, 256]
    q = torch.randn(3, H * 128, generator=torch.Generator().manual_seed(6)).bfloat16()

    def attend(tables, lens, pages):
        width = max(len(t) for t in tables)
        bt = torch.tensor([t + [0] * (width - len(t)) for t in tables], dtype=torch.int32)
        plan = ops.prefix_plan([(3, pages)], H, KV, width * PAGE, "cuda")
        ctx = torch.tensor(lens, dtype=torch.int32)
        for layer in range(cfg.n_layers):
            got = ops.prefix_attention(q.cuda(), kv.k[layer], kv.v[layer], bt.cuda(), ctx.cuda(), plan)
            want, bound = oracle.attention(q, kv.k[layer].cpu(), kv.v[layer].cpu(), bt, range(3), ctx, H, KV, 128 ** -0.5,
                                           width * PAGE)
            assert bool(((got.cpu().double().view(want.shape) - want).abs() <= bound).all())

    attend(tables, lens, 3)
    keep = torch.rand(3, 320, generator=torch.Generator().manual_seed(7)) < 0.7
    tables, lens = kv.compact(tables, lens, keep, rope_table(cfg, max_pos=400).cuda())
    attend(tables, lens, 0)
    for t in tables:
        kv.allocator.free(t)
    assert kv.allocator.free_pages == 39
