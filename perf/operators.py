"""Operators over the paged key / value cache that let sequences share it, as cases that can be timed and checked.

A cache is ``[layers, pages, kv heads, PAGE, HEAD]`` for the keys and the same for the values; a sequence's token t is row
``t % PAGE`` of page ``table[t // PAGE]``.  Three operators work on it:

  prefix   attention of query rows whose sequences begin with the same pages (a system prompt, a thread that several
           replies are drawn from): a row attends the first ``ctx`` tokens of its own table, whose first pages are its
           group's.  One layer, as a model's layer calls it.
  copy     pages copied to others in all layers: a sequence that forks gets its own copy of the page it goes on writing to
           (its tokens so far), a thread that moves gets all of its pages copied.
  compact  the tokens of a sequence that are kept move together, in all layers, in their order, to the front of a table; a
           key that moves from place p to place n can be turned back from position p to position n as it moves.

``exact`` is the same in 64 bits, row by row or token by token.
"""
from __future__ import annotations

import math
import random

import torch

own = False
DEV = "cuda"
PAGE, HEAD = 64, 128


def listed() -> list:
    return [
        # two replies drawn for one chat message of a thread: the smallest batch that shares anything
        dict(name="two replies", op="prefix", heads=32, kv=8, groups=1, seqs=2, rows=1, prefix=256, own=70),
        # nineteen peers behind one system prompt, each some way into its own message and reply
        dict(name="peers behind a prompt", op="prefix", heads=32, kv=8, groups=1, seqs=19, rows=1, prefix=2048, own=301),
        # three rooms of unequal threads, as one of eight ranks of the large dense model sees them
        dict(name="rooms on a rank", op="prefix", heads=8, kv=1, groups=3, seqs=41, rows=1, prefix=6400, own=517),
        # the messages of sixteen peers being read behind the shared prompt, all of their tokens at once
        dict(name="messages behind a prompt", op="prefix", heads=32, kv=8, groups=1, seqs=16, rows=44, prefix=1536, own=44),
        # a full batch of replies over one long document
        dict(name="replies over a document", op="prefix", heads=64, kv=8, groups=1, seqs=64, rows=1, prefix=32768, own=900),
        # a thread forks: the page that both go on writing to, up to where they part
        dict(name="one fork", op="copy", layers=32, kv=8, pages=1, partial=True),
        # as many copies of a long prompt's pages as two replicas exchange in a step, with one page that is not full each
        dict(name="threads move", op="copy", layers=8, kv=8, pages=203, partial=True),
        # a thread that outgrew its context loses its oldest turns but for the first tokens; later keys are turned back
        dict(name="context shift", op="compact", layers=32, kv=8, seqs=1, tokens=1000, keep="turns", turn=True),
        # the tokens with little weight leave the caches of a batch of threads, the others keep their positions
        dict(name="light tokens leave", op="compact", layers=8, kv=8, seqs=7, tokens=2301, keep="heavy", turn=False),
        # the same for long threads that go on from their new lengths
        dict(name="long threads shrink", op="compact", layers=8, kv=8, seqs=6, tokens=8150, keep="heavy", turn=True),
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random) -> dict:
    op = rng.choice(["prefix", "prefix", "copy", "compact"])
    if op == "prefix":
        heads, kv = rng.choice([(32, 8), (64, 8), (8, 1), (8, 8), (16, 8), (24, 8)])
        if rng.random() < 0.3:    # prompts behind a prefix
            return dict(op=op, heads=heads, kv=kv, groups=rng.randint(1, 2), seqs=rng.randint(2, 12), rows=_log(rng, 2, 64),
                        prefix=PAGE * _log(rng, 2, 40), own=_log(rng, 64, 300))
        seqs = _log(rng, 2, 64)
        return dict(op=op, heads=heads, kv=kv, groups=rng.randint(1, min(3, seqs)), seqs=seqs, rows=1,
                    prefix=PAGE * _log(rng, 2, 400), own=_log(rng, 1, 900))
    if op == "copy":
        return dict(op=op, layers=rng.choice([1, 2, 8, 32]), kv=rng.choice([1, 2, 8]), pages=_log(rng, 1, 50),
                    partial=rng.random() < 0.5)
    return dict(op=op, layers=rng.choice([1, 2, 8]), kv=rng.choice([1, 2, 8]), seqs=rng.randint(1, 8),
                tokens=_log(rng, 40, 6000), keep=rng.choice(["turns", "heavy"]), turn=rng.random() < 0.5)


# ---------------------------------------------------------------------------------------- what a case holds
def _spread(i: int, lo: int, hi: int) -> int:
    """A number of lo .. hi that looks drawn and is the same for every seed."""
    return lo + (i * 7919 + 4241) % (hi - lo + 1)


def _groups(case: dict) -> list:
    """(sequences, tokens of the prefix) of every group, the first ones with the longer prefixes."""
    n, G = case["seqs"], case["groups"]
    out = []
    for g in range(G):
        pages = max(1, case["prefix"] // PAGE * (G - g) // G)
        out.append((n // G + (g < n % G), pages * PAGE))
    return out


def _lengths(case: dict) -> list:
    """Every sequence's (group, prefix, tokens of its own), the query rows' tokens among them."""
    out, i = [], 0
    for g, (n, p) in enumerate(_groups(case)):
        for _ in range(n):
            out.append((g, p, _spread(i, min(case["rows"], case["own"]), case["own"])))
            i += 1
    return out


def _kept(case: dict) -> list:
    """Every sequence's (length, places that are kept)."""
    out = []
    for s in range(case["seqs"]):
        n = _spread(s, max(1, case["tokens"] * 3 // 4), case["tokens"])
        rng = random.Random(1000 * s + n)
        if case["keep"] == "turns":    # the first tokens stay, then a third of the thread leaves
            first = min(n, 4)
            out.append((n, [t for t in range(n) if t < first or t >= first + n // 3]))
        else:                          # the first and the last ones stay, and some three of five between them
            out.append((n, [t for t in range(n) if t < 4 or t >= n - n // 8 or rng.random() < 0.6]))
    return out


def _copies(case: dict) -> list:
    """Tokens that every copied page holds."""
    n = case["pages"]
    return [_spread(i, 1, PAGE - 1) if case["partial"] and i % 9 == 0 else PAGE for i in range(n)]


def work(case: dict) -> dict:
    if case["op"] == "prefix":
        H, KV, T = case["heads"], case["kv"], case["rows"]
        kv_bytes, flops, rows = 0, 0, 0
        for _n, p in _groups(case):
            kv_bytes += p
        for _g, p, o in _lengths(case):
            kv_bytes += o
            r = min(T, o)
            rows += r
            flops += sum(4 * HEAD * H * (p + o - k) for k in range(r))
        return {"bytes": kv_bytes * KV * HEAD * 4 + rows * H * HEAD * 4, "flops": flops}
    if case["op"] == "copy":
        return {"bytes": 2 * sum(_copies(case)) * case["layers"] * case["kv"] * HEAD * 4, "flops": 0}
    kept = sum(len(k) for _n, k in _kept(case))
    numbers = kept * case["layers"] * case["kv"] * HEAD
    return {"bytes": 2 * numbers * 4 + sum(n for n, _k in _kept(case)), "flops": 6 * numbers if case["turn"] else 0}


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV).manual_seed(seed)
    host = random.Random(seed)
    st = dict(case)
    def randn(*shape, by=1.0):
        return (torch.randn(*shape, device=DEV, generator=g) * by).to(torch.bfloat16)
    def cache(layers, pages, kv):
        x = torch.empty(layers, pages, kv, PAGE, HEAD, device=DEV, dtype=torch.bfloat16)
        for i in range(layers):
            x[i] = randn(pages, kv, PAGE, HEAD)
        return x
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    if case["op"] == "prefix":
        H, KV, T = case["heads"], case["kv"], case["rows"]
        lens = _lengths(case)
        need = [p // PAGE for _n, p in _groups(case)]
        width = max((p + o + PAGE - 1) // PAGE for _g, p, o in lens)
        total = 1 + sum(need) + sum((o + PAGE - 1) // PAGE for _g, _p, o in lens)
        free = list(range(1, total))
        host.shuffle(free)
        shared = [[free.pop() for _ in range(n)] for n in need]
        table, seq, ctx = [], [], []
        for s, (gr, p, o) in enumerate(lens):
            pages = shared[gr] + [free.pop() for _ in range((o + PAGE - 1) // PAGE)]
            table.append(pages + [0] * (width - len(pages)))
            r = min(T, o)
            seq += [s] * r
            ctx += [p + o - r + 1 + k for k in range(r)]
        st.update(k=cache(1, total, KV)[0], v=cache(1, total, KV)[0], q=randn(len(seq), H * HEAD, by=1.7), table=ints(table),
                  ctx=ints(ctx), lens=lens, scale=1 / math.sqrt(HEAD))
        counts = [0] * case["groups"]
        for s in seq:
            counts[lens[s][0]] += 1
        st["counts"] = counts
        st["seq"] = ints(seq)
        if own:
            from p2p_llm_chat_go_amd import ops

            st["plan"] = ops.prefix_plan(list(zip(counts, need)), H, KV, max(p + o for _g, p, o in lens), DEV,
                                         seqs=seq if T > 1 else None)
            st["ws"] = ops.prefix_workspace(st["plan"])
        return st
    if case["op"] == "copy":
        n = case["pages"]
        pages = list(range(1, 2 * n + 4))
        host.shuffle(pages)
        st.update(k=cache(case["layers"], 2 * n + 4, case["kv"]), v=cache(case["layers"], 2 * n + 4, case["kv"]),
                  src=pages[:n], dst=pages[n:2 * n], tokens=_copies(case))
        return st
    kept = _kept(case)
    width = max((n + PAGE - 1) // PAGE for n, _k in kept)
    pages = list(range(1, 2 * len(kept) * width + 1))
    host.shuffle(pages)
    table = torch.tensor([[pages.pop() for _ in range(width)] for _ in kept], dtype=torch.int32)
    to = torch.tensor([[pages.pop() for _ in range(width)] for _ in kept], dtype=torch.int32)
    keep = torch.zeros(len(kept), max(n for n, _k in kept), dtype=torch.bool)
    for s, (_n, k) in enumerate(kept):
        keep[s, torch.tensor(k, dtype=torch.long)] = True
    P = 1 + 2 * len(kept) * width
    st.update(k=cache(case["layers"], P, case["kv"]), v=cache(case["layers"], P, case["kv"]), table=table.to(DEV), to=to.to(DEV),
              keep=keep.to(DEV), lens=ints([n for n, _k in kept]), rot=None)
    if case["turn"]:
        st["rot"] = _rotations(max(n for n, _k in kept)).float().to(DEV)
    return st


def _rotations(n: int) -> torch.Tensor:
    """[n, HEAD / 2, 2]: cosine and sine of a position's angles."""
    inv = 500000.0 ** -(torch.arange(0, HEAD, 2, dtype=torch.float64) / HEAD)
    a = torch.arange(n, dtype=torch.float64)[:, None] * inv
    return torch.stack([a.cos(), a.sin()], -1)


# ---------------------------------------------------------------------------------------- one pass
def run(st: dict):
    if own:
        from p2p_llm_chat_go_amd import ops

        if st["op"] == "prefix":
            return ops.prefix_attention(st["q"], st["k"], st["v"], st["table"], st["ctx"], st["plan"], workspace=st["ws"])
        if st["op"] == "copy":
            ops.copy_pages(st["k"], st["v"], st["src"], st["dst"], st["tokens"])
            return st["k"], st["v"]
        lens = ops.compact_pages(st["k"], st["v"], st["table"], st["lens"], st["keep"], out_tables=st["to"], cos_sin=st["rot"])
        return st["k"], st["v"], lens
    return {"prefix": _prefix, "copy": _copy, "compact": _compact}[st["op"]](st)


def _prefix(st: dict) -> torch.Tensor:
    """A group's prefix is read once for all of its rows, every row's own tokens are gathered for it."""
    H, KV, T = st["heads"], st["kv"], st["rows"]
    G = H // KV
    out, r0, width = [], 0, st["table"].shape[1]
    prefixes = {g: p for g, p, _o in st["lens"]}
    for g, n in enumerate(st["counts"]):
        pages = prefixes[g] // PAGE
        seq, ctx = st["seq"][r0:r0 + n].long(), st["ctx"][r0:r0 + n]
        q = st["q"][r0:r0 + n].float().view(n, KV, G, HEAD).permute(1, 0, 2, 3)          # kv head, row, head, number
        first = st["table"][seq[0], :pages].long()
        kp = st["k"][first].float().permute(1, 0, 2, 3).reshape(KV, pages * PAGE, HEAD)
        vp = st["v"][first].float().permute(1, 0, 2, 3).reshape(KV, pages * PAGE, HEAD)
        sp = (q.reshape(KV, n * G, HEAD) @ kp.transpose(1, 2).contiguous()).view(KV, n, G, -1)
        # every sequence's own tokens once, however many of its rows there are
        first_row = seq[0]
        n_seq = n if T == 1 else int(len([1 for x in st["lens"] if x[0] == g]))
        mine = st["table"][first_row + torch.arange(n_seq, device=DEV), pages:].long()   # sequence, page
        L = (width - pages) * PAGE
        ko = st["k"][mine].float().permute(2, 0, 1, 3, 4).reshape(KV, n_seq, L, HEAD)
        vo = st["v"][mine].float().permute(2, 0, 1, 3, 4).reshape(KV, n_seq, L, HEAD)
        at = seq - first_row
        if T == 1:
            so = q @ ko.transpose(2, 3).contiguous()
        else:
            so = torch.cat([q[:, at == s].reshape(KV, -1, HEAD) @ ko[:, s].transpose(1, 2).contiguous() for s in range(n_seq)],
                           1).view(KV, n, G, L)
        s = torch.cat([sp, so], -1) * st["scale"]
        place = torch.arange(s.shape[-1], device=DEV)
        s = s.masked_fill(place >= ctx[None, :, None, None], -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        o = (p[..., :pages * PAGE].reshape(KV, n * G, -1) @ vp).view(KV, n, G, HEAD)
        if T == 1:
            o = o + p[..., pages * PAGE:] @ vo
        else:
            o = o + torch.cat([p[:, at == s][..., pages * PAGE:].reshape(KV, -1, L) @ vo[:, s] for s in range(n_seq)],
                              1).view(KV, n, G, HEAD)
        out.append(o.permute(1, 0, 2, 3).reshape(n, H * HEAD))
        r0 += n
    return torch.cat(out).to(torch.bfloat16)


def _copy(st: dict) -> tuple:
    src, dst = torch.tensor(st["src"], device=DEV), torch.tensor(st["dst"], device=DEV)
    valid = torch.arange(PAGE, device=DEV) < torch.tensor(st["tokens"], device=DEV)[:, None]
    for c in (st["k"], st["v"]):
        c[:, dst] = torch.where(valid[None, :, None, :, None], c[:, src], c[:, dst])
    return st["k"], st["v"]


def _compact(st: dict) -> tuple:
    k, v, keep = st["k"], st["v"], st["keep"]
    places = torch.arange(keep.shape[1], device=DEV)
    keep = keep & (places < st["lens"][:, None])
    to = keep.cumsum(1) - 1
    seq, old = keep.nonzero(as_tuple=True)
    new = to[seq, old]
    sp, so = st["table"][seq, old // PAGE].long(), old % PAGE
    dp, do = st["to"][seq, new // PAGE].long(), new % PAGE
    for layer in range(k.shape[0]):
        x = k[layer, sp, :, so].float()                      # token, kv head, number
        if st["rot"] is not None:
            a, b = st["rot"][old], st["rot"][new]
            c = (a * b).sum(-1)[:, None]                     # cosine and sine of the angle from old to new
            s = (b[..., 1] * a[..., 0] - b[..., 0] * a[..., 1])[:, None]
            x1, x2 = x[..., :HEAD // 2], x[..., HEAD // 2:]
            x = torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], -1)
            x = torch.where((old == new)[:, None, None], k[layer, sp, :, so].float(), x)
        k[layer, dp, :, do] = x.to(k.dtype)
        v[layer, dp, :, do] = v[layer, sp, :, so]
    return k, v, keep.sum(1).to(torch.int32)


# ---------------------------------------------------------------------------------------- the definitions in 64 bits
def exact(case: dict, seed: int):
    st = prepare(case, seed)
    if case["op"] == "prefix":
        if work(case)["flops"] > 3e12:
            return None
        H, KV = case["heads"], case["kv"]
        G = H // KV
        out = torch.empty(st["q"].shape[0], H, HEAD, dtype=torch.float64, device=DEV)
        seq, ctx, table = st["seq"].tolist(), st["ctx"].tolist(), st["table"].long()
        for r in range(len(seq)):
            t = torch.arange(ctx[r], device=DEV)
            page, at = table[seq[r]][t // PAGE], t % PAGE
            keys, values = st["k"][page, :, at].double(), st["v"][page, :, at].double()     # token, kv head, number
            q = st["q"][r].double().view(KV, G, HEAD)
            s = torch.stack([keys[:, h] @ q[h].t() for h in range(KV)], 1) * st["scale"]     # token, kv head, head
            p = torch.softmax(s, 0)
            out[r] = torch.stack([p[:, h].t() @ values[:, h] for h in range(KV)]).reshape(H, HEAD)
        return out.view(-1, H * HEAD)
    if case["op"] == "copy":
        k, v = st["k"].double(), st["v"].double()
        for s, d, n in zip(st["src"], st["dst"], st["tokens"]):
            for c in (k, v):
                c[:, d, :, :n] = c[:, s, :, :n]
        return k, v
    k, v = st["k"].double(), st["v"].double()
    kept = _kept(case)
    rot = None if st["rot"] is None else torch.view_as_complex(st["rot"].double())
    for s, (_n, places) in enumerate(kept):
        table, to = st["table"][s].long(), st["to"][s].long()
        old = torch.tensor(places, device=DEV)
        new = torch.arange(len(places), device=DEV)
        x = st["k"][:, table[old // PAGE], :, old % PAGE].double()       # token, layer, kv head, number
        if rot is not None:
            turn = rot[new] * rot[old].conj()
            moved = torch.complex(x[..., :HEAD // 2], x[..., HEAD // 2:]) * turn[:, None, None]
            x = torch.where((old == new)[:, None, None, None], x, torch.cat([moved.real, moved.imag], -1))
        k[:, to[new // PAGE], :, new % PAGE] = x
        v[:, to[new // PAGE], :, new % PAGE] = st["v"][:, table[old // PAGE], :, old % PAGE].double()
    return k, v, torch.tensor([len(p) for _n, p in kept], dtype=torch.int32, device=DEV)
