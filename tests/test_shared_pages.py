"""Sequences that share pages: the allocator's owners, ``KVCache.fork`` and ``compact``, and generation over a shared prefix."""
import pytest
import torch

from p2p_llm_chat_go_amd import ops
from p2p_llm_chat_go_amd.engine import Engine
from p2p_llm_chat_go_amd.engine.engine import common_prefix
from p2p_llm_chat_go_amd.engine.kv_cache import KVCache, PageAllocator, pages_for
from p2p_llm_chat_go_amd.models import TINY_LLAMA
from p2p_llm_chat_go_amd.models.config import rope_table
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
