"""Attention mass and the eviction by it, from their definitions in 64 bits over the logical cache [blocks, block, kv heads, head_dim] -
and the bounds that the tests hold the kernels to.

Bounds.  A score is a sum of D products of bfloat16 numbers: in 32 bits off by at most (D + 2) 2^-24 A, A the sum of the products'
magnitudes times the scale (the scale's and the base-2 logarithm's rounding among the 2).  A weight has the score's and the row sum's error,
twice that, and its sums' roundings, each at most 2^-24 a term: n terms of the row sum, R of the column sum, some 16 for exp2, the joins of
partial sums and the quotient.  So a mass is off by at most 2^-24 (2 (D + 2) A + n + R + 16) of it, and of what was there before by 2^-24.
An output adds the roundings of the weights to two bfloat16 (2^-16) and of the result to one (2^-8)."""
import torch

U = 2.0 ** -24


def rows_of(cache, table, ctx):
    """[ctx, kv heads, head_dim] in 64 bits, and which of the tokens are there"""
    block = cache.shape[1]
    t = torch.arange(ctx)
    page = table[t // block].long()
    there = (page >= 0) & (page < cache.shape[0])
    rows = cache[torch.where(there, page, 0), t % block].double()
    return torch.where(there.view(-1, 1, 1), rows, 0.0), there


def weights(q, k, there, first, scale):
    """q [rows, heads, D] at positions first.., k [ctx, kv heads, D] -> weights [heads, rows, ctx], magnitude A of the scores"""
    G = q.shape[1] // k.shape[1]
    kk = k.repeat_interleave(G, 1)
    s = torch.einsum("ihd,jhd->hij", q.double(), kk) * scale
    A = float((torch.einsum("ihd,jhd->hij", q.double().abs(), kk.abs()) * abs(scale)).max()) if k.shape[0] else 0.0
    seen = (torch.arange(k.shape[0]).view(1, -1) <= first + torch.arange(q.shape[0]).view(-1, 1)) & there.view(1, -1)
    s = s.masked_fill(~seen, float("-inf"))
    m = s.amax(-1, keepdim=True) if k.shape[0] else torch.zeros(*s.shape[:2], 1).double()
    e = torch.exp(s - torch.where(m.isinf(), torch.zeros_like(m), m))
    total = e.sum(-1, keepdim=True)
    return torch.where(total > 0, e / total, 0.0), A


def mass_of(w, n_kv):
    """[heads, rows, ctx] -> [kv heads, ctx]"""
    return w.reshape(n_kv, w.shape[0] // n_kv * w.shape[1], w.shape[2]).sum(1)


def mass_bound(D, A, n, R):
    return U * (2 * (D + 2) * A + n + R + 16)


def keys(mass, position, length, sinks, recent):
    """the order of the choice: larger first"""
    out = []
    for m, p in zip(mass.tolist(), position.tolist()):
        if p < sinks or p >= length - recent:
            out.append((2, 0.0))
        elif m != m:
            out.append((0, 0.0))
        else:
            out.append((1, m))
    return out


def choose(mass, position, length, keep, sinks, recent):
    """slots in their new places [keep]: what stays, with those kept from behind `keep` in the free places in order"""
    k = keys(mass, position, length, sinks, recent)
    order = sorted(range(len(k)), key=lambda j: (-k[j][0], -k[j][1], j))[:keep]
    stay = set(order)
    src = list(range(keep))
    movers = iter(sorted(j for j in order if j >= keep))
    for i in range(keep):
        if i not in stay:
            src[i] = next(movers)
    return src


def position_of(origin, evicted, ctx):
    """[kv heads, ctx] positions of a row's slots; origin [kv heads, len], evicted (slots written down, tokens dropped)"""
    kept, dropped = int(evicted[0]), int(evicted[1])
    j = torch.arange(ctx, dtype=torch.int32).expand(origin.shape[0], ctx)
    return torch.where(j < kept, origin[:, :ctx], j + dropped)
