"""Attention mass and eviction: which rows of the state a call reads and writes - padded batches, rows that are not there, rows shorter than the
contexts, and the rows of a prompt that are not observed."""
import pytest
import torch

import attn_mass_ref as ref
from kv_layout import to_logical
from test_attn_mass_gpu import device_caches, pool

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from nanovllm import ops as _ops

    return _ops


def dev(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device=DEV)


@pytest.mark.parametrize("first", [False, True])
def test_padded_rows_of_an_eviction_into_other_rows(ops, first):
    """sequences of no tokens, ahead of the others or behind them: whatever rows they name, the others' are as without them, and a row that more than
    one of them names is left as it was; alone in naming it, one hands its pair on"""
    gen = torch.Generator().manual_seed(21)
    hkv, d, block, keep = 3, 64, 16, 48
    ctxs = [130, 40, 97]  # the second is within the budget: its row is copied
    real = [(0, 1), (2, 3), (4, 5)]
    pads = [pair for pair in real for _ in range(20)]                          # a sequence's own pair of rows
    pads += [(6, out) for _, out in real] * 10                                 # the row that one writes, from another
    pads += [(6, row) for row, _ in real] * 10                                 # the row that one reads, to be written
    pads += [(out, out) for _, out in real] + [(row, row) for row, _ in real]  # in place
    pads += [(6, 7), (8, 7)] * 10                                              # a row that several of them name
    pads += [(6, -1), (-1, 9), (6, 12)]                                        # rows that are not there
    alone = [(8, 10), (6, 11)]
    pads += alone
    n_rows, room = 12, 144
    kc, vc, bt = pool(gen, hkv, d, block, ctxs)
    mass = torch.rand(n_rows, hkv, room, generator=gen)
    origin = torch.stack([torch.randperm(3 * room, generator=gen)[:room] for _ in range(n_rows * hkv)]).view(n_rows, hkv, room).to(torch.int32)
    evicted = torch.tensor([[r + 20, 3 * room + r] for r in range(n_rows)], dtype=torch.int32)
    results = []
    for padded in (False, True):
        k, v = device_caches(kc, vc)
        m, o, e = mass.to(DEV), origin.to(DEV), evicted.to(DEV)
        rows, lens, table = list(real), list(ctxs), bt
        if padded:
            empty = torch.full((len(pads), bt.shape[1]), -1, dtype=torch.int32)
            table = torch.cat([empty, bt] if first else [bt, empty])
            rows = pads + rows if first else rows + pads
            lens = [0] * len(pads) + lens if first else lens + [0] * len(pads)
        after = ops.kv_cache_evict(k, v, table.to(DEV), dev(lens), m, o, e, dev([r for r, _ in rows]), keep, 2, 10, block,
                                   slots_out=dev([r for _, r in rows]))
        assert after.tolist() == [min(n, keep) for n in lens]
        results.append((m.cpu(), o.cpu(), e.cpu(), *(to_logical(c.cpu(), block, i == 1).view(torch.int16) for i, c in enumerate((k, v)))))
    bare, filled = results
    assert bare[2][[1, 3, 5]].tolist() == [[48, 3 * room + 130 - 48], [22, 3 * room + 2], [48, 3 * room + 4 + 97 - 48]]
    want = bare[2].clone()
    for r, out in alone:
        want[out] = evicted[r]
    assert torch.equal(filled[2], want)
    for i in (0, 1, 3, 4):
        assert torch.equal(filled[i], bare[i])


def check_rows(got, start, rows, news, ctxs, fresh, bounds):
    """rows: (read, written) per sequence; news: the step's mass [kv heads, ctx] per sequence; everything that no token has a place in stays"""
    n_rows, _, room = start.shape
    touched = torch.zeros(start.shape, dtype=torch.bool)
    for (r, out), new, ctx, f, bound in zip(rows, news, ctxs, fresh, bounds):
        if not 0 <= out < n_rows or ctx == 0:
            continue
        n = min(ctx, room)
        old = start[r, :, :n].double() if 0 <= r < n_rows else torch.zeros(new.shape[0], n).double()
        old = torch.where(torch.arange(n) < f, old, 0.0)
        limit = bound * new[:, :n] + ref.U * (old + new[:, :n]) + 1e-30
        diff = (got[out, :, :n].double() - old - new[:, :n]).abs()
        assert bool((diff <= limit).all()), (r, out, float((diff / limit).max()))
        touched[out, :, :n] = True
    assert torch.equal(got[~touched], start[~touched])


# rows read and written by four sequences, of five: there, in place, none to read, none to write
ROWS = [[(0, 1), (2, 2), (-1, 3), (5, 4)], [(0, -1), (1, 5), (2, 3), (4, 4)], [(-9, 0), (2 ** 31 - 1, 1), (2, 2 ** 31 - 1), (3, -2 ** 31)]]


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("geometry,ctxs,room", [
    ((16, 8, 128), [200, 17, 1, 130], 205), ((16, 8, 128), [200, 17, 1, 130], 100), ((14, 2, 64), [200, 16, 201, 130], 200),   # not split
    ((16, 8, 128), [700, 17, 1, 400], 705), ((16, 8, 128), [700, 401, 1, 400], 400), ((14, 2, 64), [1500, 300, 255, 257], 256)])
def test_decode_rows_and_their_length(ops, rows, geometry, ctxs, room):
    hq, hkv, d = geometry
    gen = torch.Generator().manual_seed(room)
    kc, vc, bt = pool(gen, hkv, d, 16, ctxs)
    k, v = device_caches(kc, vc)
    q = torch.randn(4, hq, d, generator=gen).bfloat16()
    start = torch.rand(5, hkv, room, generator=gen)
    mass = start.to(DEV)
    ops.paged_attn_decode_mass(q.to(DEV), k, v, bt.to(DEV), dev(ctxs), mass, dev([r for r, _ in rows]), hq, hkv, 16, d ** -0.5,
                               slots_out=dev([r for _, r in rows]))
    news, bounds = [], []
    for b, ctx in enumerate(ctxs):
        w, A = ref.weights(q[b:b + 1], *ref.rows_of(kc, bt[b], ctx), ctx - 1, d ** -0.5)
        news.append(ref.mass_of(w, hkv))
        bounds.append(ref.mass_bound(d, A, ctx, hq // hkv))
    check_rows(mass.cpu(), start, rows, news, ctxs, [c - 1 for c in ctxs], bounds)


def run_prompt_rows(ops, geometry, news, pasts, rows, room, window, max_q, wider, seed):
    """wider: entries of the tables beyond the contexts (what the form of the column sums goes by, too)"""
    hq, hkv, d = geometry
    gen = torch.Generator().manual_seed(seed)
    ctxs = [n + p for n, p in zip(news, pasts)]
    kc, vc, bt = pool(gen, hkv, d, 16, ctxs, width_more=wider)
    k, _ = device_caches(kc, vc)
    cu = [sum(news[:i]) for i in range(len(news) + 1)]
    q = torch.randn(cu[-1], hq, d, generator=gen).bfloat16()
    start = torch.rand(max(5, 2 * len(news)), hkv, room, generator=gen)
    mass = start.to(DEV)
    ops.prompt_attn_mass(q.to(DEV), k, bt.to(DEV), dev(cu), dev(ctxs), max_q, mass, dev([r for r, _ in rows]), hq, hkv, 16, d ** -0.5, window=window,
                         slots_out=dev([r for _, r in rows]))
    given, bounds = [], []
    for b, ctx in enumerate(ctxs):
        seen = min(news[b], max_q, window or max_q)
        A, w = 0.0, torch.zeros(hq, 1, ctx).double()
        if seen:
            w, A = ref.weights(q[cu[b + 1] - seen:cu[b + 1]], *ref.rows_of(kc, bt[b], ctx), ctx - seen, d ** -0.5)
        given.append(ref.mass_of(w, hkv))
        bounds.append(ref.mass_bound(d, A, ctx, seen * hq // hkv))
    check_rows(mass.cpu(), start, rows, given, ctxs, pasts, bounds)


WIDER = [2, 200]  # 4 sequences on 8 kv heads: key blocks of one wave's keys, and with 256 blocks of four waves' and more, those


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("wider", WIDER)
@pytest.mark.parametrize("room", [205, 150])
def test_prompt_rows_and_their_length(ops, rows, wider, room):
    run_prompt_rows(ops, (16, 8, 128), [60, 17, 1, 130], [140, 0, 64, 70], rows, room, 0, 130, wider, 31)
    run_prompt_rows(ops, (32, 8, 64), [60, 17, 1, 130], [140, 0, 64, 70], rows, room, 19, 130, wider, 32)


@pytest.mark.parametrize("max_q", [0, 1, 33, 64])
@pytest.mark.parametrize("window", [0, 1, 40])
@pytest.mark.parametrize("wider", WIDER)
def test_prompt_rows_behind_the_first_max_seqlen_q_are_not_taken(ops, max_q, window, wider):
    """counted from a sequence's end; the tokens that the step stored have their mass set all the same"""
    rows = [(0, 1), (2, 2), (3, 4), (5, 6)]
    run_prompt_rows(ops, (16, 8, 128), [90, 33, 5, 200], [0, 100, 20, 7], rows, 210, window, max_q, wider, 33)
    run_prompt_rows(ops, (32, 8, 64), [90, 33, 5, 200], [0, 100, 20, 7], rows, 210, window, max_q, wider, 34)


@pytest.mark.parametrize("wider", [2, 600])
def test_the_last_rows_of_a_prompt_in_portions(ops, wider):
    """max_seqlen_q = 0 sets the mass of a portion's tokens and observes nothing: the prompt's last 32 rows, however it is cut - the portion
    before the last one observes what the last is too short for"""
    hq, hkv, d, ctx, window = 16, 8, 128, 300, 32
    gen = torch.Generator().manual_seed(35)
    kc, vc, bt = pool(gen, hkv, d, 16, [ctx], width_more=wider)
    k, _ = device_caches(kc, vc)
    q = torch.randn(ctx, hq, d, generator=gen).bfloat16()
    w, A = ref.weights(q[-window:], *ref.rows_of(kc, bt[0], ctx), ctx - window, d ** -0.5)
    want, bound = ref.mass_of(w, hkv), ref.mass_bound(d, A, ctx, window * hq // hkv)
    for cuts in ([0, 300], [0, 100, 220, 300], [0, 1, 290, 300]):
        mass = torch.full((1, hkv, 304), float("nan"), device=DEV)  # rows need no clearing
        for lo, hi in zip(cuts, cuts[1:]):
            seen = max(0, hi - max(lo, ctx - window))  # of the portion's rows those among the prompt's last
            ops.prompt_attn_mass(q[lo:hi].to(DEV), k, bt.to(DEV), dev([0, hi - lo]), dev([hi]), seen, mass, dev([0]), hq, hkv, 16, d ** -0.5)
        got = mass[0, :, :ctx].cpu().double()
        # (a portion more, a rounding of the sum more)
        assert bool(((got - want).abs() <= (bound + len(cuts) * ref.U) * want + 1e-30).all())
        assert bool(mass[0, :, ctx:].isnan().all())


@pytest.mark.parametrize("read,written", [(-1, 1), (3, 1), (0, -1), (0, 3), (-2 ** 31, 2 ** 31 - 1)])
@pytest.mark.parametrize("ctx", [100, 40])
def test_eviction_with_a_row_that_is_not_there(ops, read, written, ctx):
    """... of either kind leaves its sequence as it is, and the others are evicted"""
    gen = torch.Generator().manual_seed(36)
    kc, vc, bt = pool(gen, 2, 64, 16, [ctx, 90])
    mass = torch.rand(3, 2, 104, generator=gen)
    origin, evicted = torch.full((3, 2, 104), -5, dtype=torch.int32), torch.tensor([[9, 90], [8, 80], [0, 0]], dtype=torch.int32)
    results = []
    for b in (0, 1):  # with the sequence, and the other one alone
        k, v = device_caches(kc, vc)
        state = [t.to(DEV) for t in (mass, origin, evicted)]
        after = ops.kv_cache_evict(k, v, bt[b:].to(DEV), dev([ctx, 90][b:]), *state, dev([read, 2][b:]), 48, 2, 10, 16, slots_out=dev([written, 2][b:]))
        assert after.tolist() == [ctx, 48][b:]
        results.append([t.cpu() for t in state] + [t.view(torch.int16).cpu() for t in (k, v)])
    for a, b in zip(*results):
        assert torch.equal(a, b)
    assert results[0][2].tolist() == [[9, 90], [8, 80], [48, 42]]


def test_narrow_views_of_wide_tables(ops):
    """rows of a table further apart than what may be used of them: the same bits as from a table of that width"""
    gen = torch.Generator().manual_seed(37)
    hq, hkv, d, block, ctxs = 16, 8, 128, 16, [300, 41, 170]
    kc, vc, bt = pool(gen, hkv, d, block, ctxs, width_more=60)
    assert bt.shape[1] == 79
    q = torch.randn(60, hq, d, generator=gen).bfloat16().to(DEV)
    start = torch.rand(3, hkv, 304, generator=gen)
    results = []
    for copied in (False, True):
        table = bt.to(DEV)[:, :19]
        table = table.contiguous() if copied else table
        k, v = device_caches(kc, vc)
        mass, lens, slots = start.to(DEV), dev(ctxs), dev([2, 0, 1])
        origin, evicted = torch.zeros(3, hkv, 304, dtype=torch.int32, device=DEV), torch.zeros(3, 2, dtype=torch.int32, device=DEV)
        ops.prompt_attn_mass(q, k, table, dev([0, 30, 40, 60]), lens, 30, mass, slots, hq, hkv, block, 0.1)
        out = ops.paged_attn_decode_mass(q[:3], k, v, table, lens, mass, slots, hq, hkv, block, 0.1)
        after = ops.kv_cache_evict(k, v, table, lens, mass, origin, evicted, slots, 100, 2, 10, block)
        assert after.tolist() == [100, 41, 100]
        results.append([t.cpu() for t in (out.view(torch.int16), mass, origin, evicted, k.view(torch.int16), v.view(torch.int16))])
    for a, b in zip(*results):
        assert torch.equal(a, b)
