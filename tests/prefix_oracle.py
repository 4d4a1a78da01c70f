"""The operators over shared pages in 64 bits, row by row and token by token, with what a correct result may be off by."""
import torch

PAGE, D = 64, 128
U16, U32 = 2.0 ** -8, 2.0 ** -24     # half a step of bf16 and of fp32, relative


def attention(q, k, v, table, seqs, ctx, Hq, Hkv, scale, max_ctx):
    """(result, bound) of every row, float64 [R, Hq, D].

    The bound: the result is rounded once to bf16 (U16 of itself) and every weight once (U16 of its part of sum p |v|).
    Scores are fp32 sums of D products (D U32 of sum |q k|, twice: numerator and denominator), weights fp32 exponentials of
    arguments rounded to U32 of themselves, and sums of N weights are fp32 (N U32, twice)."""
    R, G = len(seqs), Hq // Hkv
    out, bound = torch.zeros(R, Hq, D, dtype=torch.float64), torch.zeros(R, Hq, D, dtype=torch.float64)
    for r in range(R):
        n = min(int(ctx[r]), max_ctx)
        if n <= 0:
            continue
        t = torch.arange(n)
        page = table[int(seqs[r])][t // PAGE].long()
        keys, values = k[page, :, t % PAGE].double(), v[page, :, t % PAGE].double()
        x = q[r].double().view(Hkv, G, D)
        s = torch.einsum("hgd,nhd->hgn", x, keys) * scale
        p = torch.softmax(s, -1)
        out[r] = torch.einsum("hgn,nhd->hgd", p, values).reshape(Hq, D)
        most = torch.einsum("hgd,nhd->hgn", x.abs(), keys.abs()).amax() * scale
        weight = U16 * (1 + U16) + U32 * (2 * D * most + 8 * most + 2 * n + 1024)
        bound[r] = U16 * out[r].abs() + weight * torch.einsum("hgn,nhd->hgd", p, values.abs()).reshape(Hq, D)
    return out, bound


def compacted(k, v, table, lens, keep, to, rot):
    """(k, v, lengths, bound of k): token by token."""
    k0, v0 = k.clone(), v.clone()
    k, v = k.clone().double(), v.clone().double()
    bound = torch.zeros_like(k)
    to = table if to is None else to
    new = []
    for b in range(len(lens)):
        n = 0
        for p in range(max(0, min(int(lens[b]), keep.shape[1], table.shape[1] * PAGE))):
            if not keep[b, p]:
                continue
            f, t = int(table[b, p // PAGE]), int(to[b, n // PAGE])
            if 0 <= f < k.shape[1] and 0 <= t < k.shape[1]:
                x = k0[:, f, :, p % PAGE].double()
                if rot is not None and n != p:
                    a, c = rot[p].double(), rot[n].double()
                    cos = a[:, 0] * c[:, 0] + a[:, 1] * c[:, 1]
                    sin = c[:, 1] * a[:, 0] - c[:, 0] * a[:, 1]
                    x1, x2 = x.chunk(2, -1)
                    x = torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin], -1)
                    # one rounding to bf16; cosine, sine and the two products in fp32: some 4 roundings of numbers up to |x1| + |x2|
                    bound[:, t, :, n % PAGE] = U16 * x.abs() + 8 * U32 * (x1.abs() + x2.abs()).repeat(1, 1, 2)
                k[:, t, :, n % PAGE] = x
                v[:, t, :, n % PAGE] = v0[:, f, :, p % PAGE].double()
            n += 1
        new.append(n)
    return k, v, new, bound
