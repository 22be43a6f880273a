"""Attention mass of cached tokens (csrc/attn_mass.hip): the decode attention that keeps it and the mass a prompt's rows give, against
the definition in 64 bits (tests/attn_mass_ref.py, with the bounds)."""
import math

import pytest
import torch

import attn_mass_ref as ref
from kv_layout import to_fragment

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

# (query heads, kv heads, head_dim)
GEOMETRIES = [(16, 8, 128), (8, 8, 64), (28, 4, 128), (14, 2, 64), (16, 1, 64), (64, 4, 128), (5, 1, 128), (3, 1, 64)]


@pytest.fixture(scope="module")
def ops():
    from nanovllm import ops as _ops

    return _ops


def pool(gen, hkv, d, block, ctxs, extra=3, width_more=2):
    """caches of random pages in any order; whatever no token of a sequence is in holds NaN"""
    need = [-(-c // block) for c in ctxs]
    nblk = sum(need) + extra
    kc = torch.full((nblk, block, hkv, d), float("nan")).bfloat16()
    vc = torch.full((nblk, block, hkv, d), float("nan")).bfloat16()
    order = torch.randperm(nblk, generator=gen).tolist()
    width = max(1, max(need)) + width_more
    bt = torch.full((len(ctxs), width), -1, dtype=torch.int32)
    for b, c in enumerate(ctxs):
        for i in range(need[b]):
            bt[b, i] = order.pop()
            n = min(block, c - i * block)
            kc[bt[b, i], :n] = torch.randn(n, hkv, d, generator=gen).bfloat16()
            vc[bt[b, i], :n] = torch.randn(n, hkv, d, generator=gen).bfloat16()
    return kc, vc, bt


def device_caches(kc, vc):
    return to_fragment(kc, False).to(DEV), to_fragment(vc, True).to(DEV)


def check_mass(got, start, b, slot_in, slot_out, new, ctx, fresh, bound, room):
    """row slot_out of got: the tokens' masses within the bound, slots behind the context as they were"""
    old = start[slot_in, :, :ctx].double() if slot_in is not None else torch.zeros(new.shape)
    old = torch.where(torch.arange(ctx) < fresh, old, 0.0)
    want = old + new
    diff = (got[slot_out, :, :ctx].double() - want).abs()
    limit = bound * new + ref.U * (old + new) + 1e-30
    assert bool((diff <= limit).all()), (b, float((diff / limit).max()), int((diff / limit).argmax()))
    assert torch.equal(got[slot_out, :, ctx:], start[slot_out, :, ctx:])


def run_decode(ops, geometry, block, ctxs, seed, own_rows=False, bad_pages=(), scale=None, dead=(), n_tables=2):
    hq, hkv, d = geometry
    gen = torch.Generator().manual_seed(seed)
    kc, vc, bt = pool(gen, hkv, d, block, ctxs, width_more=n_tables)
    for b, i, value in bad_pages:
        bt[b, i] = kc.shape[0] if value is None else value
    B = len(ctxs)
    packed = torch.randn(B, (hq + 2 * hkv) * d, generator=gen).bfloat16()
    q = packed[:, :hq * d]
    scale = d ** -0.5 if scale is None else scale
    room = max(max(ctxs), 1) + 5
    start = torch.rand(2 * B + 1, hkv, room, generator=gen) * 3
    perm = torch.randperm(2 * B + 1, generator=gen)
    slots = perm[:B].to(torch.int32)
    slots_out = slots if own_rows else perm[B:2 * B].to(torch.int32).clone()
    for b in dead:
        slots_out[b] = -1 if b % 2 else 2 * B + 1
    mass = start.to(DEV)
    kd, vd = device_caches(kc, vc)
    pq = packed.to(DEV)
    args = (pq[:, :hq * d], kd, vd, bt.to(DEV), torch.tensor(ctxs, dtype=torch.int32).to(DEV), mass, slots.to(DEV), hq, hkv, block, scale)
    out = ops.paged_attn_decode_mass(*args, slots_out=None if own_rows else slots_out.to(DEV)).cpu().view(B, hq, d)
    got = mass.cpu()
    touched = set()
    for b, ctx in enumerate(ctxs):
        k, there = ref.rows_of(kc, bt[b], ctx)
        v, _ = ref.rows_of(vc, bt[b], ctx)
        w, A = ref.weights(q[b].view(1, hq, d), k, there, ctx - 1, scale)
        G = hq // hkv
        want = torch.einsum("hj,jhd->hd", w[:, 0], v.repeat_interleave(G, 1)) if ctx else torch.zeros(hq, d).double()
        size = torch.einsum("hj,jhd->hd", w[:, 0], v.abs().repeat_interleave(G, 1)) if ctx else torch.zeros(hq, d).double()
        bound = ref.mass_bound(d, A, ctx, G)
        diff = (out[b].double() - want).abs()
        assert bool((diff <= 2.0 ** -8 * want.abs() + (bound + 2.0 ** -16) * size * 1.01 + 1e-30).all()), (b, ctx, float(diff.max()))
        row = int(slots_out[b])
        if 0 <= row < start.shape[0] and ctx:
            touched.add(row)
            check_mass(got, start, b, int(slots[b]), row, ref.mass_of(w, hkv), ctx, ctx - 1, bound, room)
    for r in set(range(start.shape[0])) - touched:
        assert torch.equal(got[r], start[r])
    # the same call, the same bits
    mass2 = start.to(DEV)
    out2 = ops.paged_attn_decode_mass(*args[:5], mass2, *args[6:], slots_out=None if own_rows else slots_out.to(DEV))
    assert torch.equal(out2.cpu().view(torch.int16), out.view(B, -1).view(torch.int16)) and torch.equal(mass2.cpu(), got)


@pytest.mark.parametrize("geometry", GEOMETRIES)
@pytest.mark.parametrize("block", [16, 48, 256])
def test_decode_ragged(ops, geometry, block):
    run_decode(ops, geometry, block, [1, 16, 0, 33, 15, 200, 17, 513], hash((geometry, block)) % 1000)


@pytest.mark.parametrize("geometry", GEOMETRIES[:5])
def test_decode_many_sequences_one_split(ops, geometry):
    n = 40 if geometry[1] > 1 else 260
    run_decode(ops, geometry, 16, [1 + 37 * i % 300 for i in range(n)], 7, own_rows=True)


@pytest.mark.parametrize("geometry", [(16, 8, 128), (32, 8, 64), (7, 1, 128)])
@pytest.mark.parametrize("ctx", [2047, 4099, 9001])
def test_decode_long_context_of_one_sequence(ops, geometry, ctx):
    run_decode(ops, geometry, 64, [ctx], ctx)


def test_decode_short_contexts_in_a_wide_table(ops):
    run_decode(ops, (16, 8, 128), 16, [1, 20, 100], 3, n_tables=500)


def test_decode_pages_that_are_not_there(ops):
    run_decode(ops, (16, 8, 128), 16, [100, 16, 50, 200], 5, bad_pages=[(0, 2, -1), (1, 0, -7), (2, 3, None), (3, 0, -1), (3, 12, None)])
    run_decode(ops, (8, 8, 64), 32, [3000], 6, bad_pages=[(0, i, -1) for i in range(0, 93, 5)])


def test_decode_rows_that_are_not_there(ops):
    run_decode(ops, (16, 8, 128), 16, [100, 16, 50, 200], 8, dead=(1, 2))


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
def test_decode_scales(ops, scale):
    run_decode(ops, (16, 8, 128), 16, [100, 700], 9, scale=scale)


def run_prompt(ops, geometry, block, news, pasts, window, seed, bad_pages=(), max_q=None, scale=None):
    hq, hkv, d = geometry
    gen = torch.Generator().manual_seed(seed)
    ctxs = [n + p for n, p in zip(news, pasts)]
    kc, vc, bt = pool(gen, hkv, d, block, ctxs)
    for b, i, value in bad_pages:
        bt[b, i] = value
    B, T = len(ctxs), sum(news)
    packed = torch.randn(max(T, 1), (hq + 2 * hkv) * d, generator=gen).bfloat16()
    scale = d ** -0.5 if scale is None else scale
    cu = torch.tensor([0] + [sum(news[:i + 1]) for i in range(B)], dtype=torch.int32)
    room = max(max(ctxs), 1) + 5
    start = torch.rand(2 * B, hkv, room, generator=gen) * 3
    perm = torch.randperm(2 * B, generator=gen).to(torch.int32)
    slots, slots_out = perm[:B], perm[B:]
    kd, vd = device_caches(kc, vc)
    pq = packed.to(DEV)[:T, :hq * d]
    got = []
    for own in (False, True):
        mass = start.to(DEV)
        ops.prompt_attn_mass(pq, kd, bt.to(DEV), cu.to(DEV), torch.tensor(ctxs, dtype=torch.int32).to(DEV), max(news) if max_q is None else max_q, mass,
                             slots.to(DEV), hq, hkv, block, scale, window=window, slots_out=None if own else slots_out.to(DEV))
        got.append(mass.cpu())
    for b, ctx in enumerate(ctxs):
        seen = min(window, news[b]) if window else news[b]
        k, there = ref.rows_of(kc, bt[b], ctx)
        w, A = ref.weights(packed[cu[b + 1] - seen:cu[b + 1], :hq * d].view(seen, hq, d), k, there, ctx - seen, scale) if seen else \
            (torch.zeros(hq, 1, ctx).double(), 0.0)
        new = ref.mass_of(w, hkv)
        bound = ref.mass_bound(d, A, ctx, seen * hq // hkv)
        if ctx:
            check_mass(got[0], start, b, int(slots[b]), int(slots_out[b]), new, ctx, ctx - news[b], bound, room)
            # in place: the same bits
            assert torch.equal(got[1][slots[b], :, :ctx], got[0][slots_out[b], :, :ctx])
        assert torch.equal(got[0][slots[b]], start[slots[b]])


@pytest.mark.parametrize("geometry", GEOMETRIES)
@pytest.mark.parametrize("window", [0, 1, 19, 64])
def test_prompt_ragged(ops, geometry, window):
    run_prompt(ops, geometry, 16, [1, 137, 0, 64, 31, 3], [0, 0, 0, 0, 0, 0], window, 11 + window)


@pytest.mark.parametrize("geometry", GEOMETRIES[:4])
@pytest.mark.parametrize("window", [0, 32])
def test_prompt_portions_behind_cached_tokens(ops, geometry, window):
    run_prompt(ops, geometry, 48, [70, 1, 0, 33, 200], [130, 1000, 65, 0, 47], window, 5)


@pytest.mark.parametrize("geometry", [(16, 8, 128), (32, 8, 64), (7, 1, 128)])
def test_prompt_long(ops, geometry):
    run_prompt(ops, geometry, 256, [900], [3301], 0, 2)
    run_prompt(ops, geometry, 64, [2500], [0], 40, 3)


def test_prompt_pages_that_are_not_there(ops):
    run_prompt(ops, (16, 8, 128), 16, [137, 60], [0, 60], 0, 4, bad_pages=[(0, 0, -1), (0, 4, 1000000), (1, 2, -1), (1, 7, -3)])


def test_prompt_scale(ops):
    run_prompt(ops, (16, 8, 128), 16, [137, 60], [0, 60], 0, 4, scale=1.5)


def test_prompt_and_decode_agree_on_one_row(ops):
    """a prompt's last row alone gives what a decode step of that token gives"""
    gen = torch.Generator().manual_seed(1)
    hq, hkv, d, block, ctx = 16, 8, 128, 16, 301
    kc, vc, bt = pool(gen, hkv, d, block, [ctx])
    kd, vd = device_caches(kc, vc)
    q = torch.randn(1, hq, d, generator=gen).bfloat16().to(DEV)
    lens, slot = torch.tensor([ctx], dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    a = torch.zeros(1, hkv, 320, device=DEV)
    b = torch.zeros(1, hkv, 320, device=DEV)
    ops.paged_attn_decode_mass(q, kd, vd, bt.to(DEV), lens, a, slot, hq, hkv, block, d ** -0.5)
    ops.prompt_attn_mass(q, kd, bt.to(DEV), torch.tensor([0, 1], dtype=torch.int32, device=DEV), lens, 1, b, slot, hq, hkv, block, d ** -0.5)
    k, there = ref.rows_of(kc, bt[0], ctx)
    _, A = ref.weights(q.cpu(), k, there, ctx - 1, d ** -0.5)
    assert bool(((a - b).abs() <= 2 * ref.mass_bound(d, A, ctx, 2) * a + 1e-30).all())
    assert math.isclose(float(a.sum()), hq, rel_tol=1e-4)


def test_captured_and_on_a_stream_of_its_own(ops):
    """replays with eager work between them, on the inputs of the moment"""
    gen = torch.Generator().manual_seed(2)
    hq, hkv, d, block = 16, 8, 128, 16
    ctxs = [300, 2100]
    kc, vc, bt = pool(gen, hkv, d, block, ctxs)
    kd, vd = device_caches(kc, vc)
    bt, lens = bt.to(DEV), torch.tensor(ctxs, dtype=torch.int32, device=DEV)
    slots, cu = torch.tensor([1, 0], dtype=torch.int32, device=DEV), torch.tensor([0, 40, 100], dtype=torch.int32, device=DEV)
    q, qp = torch.zeros(2, hq, d, device=DEV, dtype=torch.bfloat16), torch.zeros(100, hq, d, device=DEV, dtype=torch.bfloat16)
    mass = torch.zeros(2, hkv, 2112, device=DEV)

    def step(to):
        out = ops.paged_attn_decode_mass(q, kd, vd, bt, lens, to, slots, hq, hkv, block, 0.1)
        ops.prompt_attn_mass(qp, kd, bt, cu, lens, 60, to, slots, hq, hkv, block, 0.1, window=32)
        return out

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(mass)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(mass)
    for i in range(4):
        q.copy_(torch.randn(2, hq, d, generator=gen).bfloat16())
        qp.copy_(torch.randn(100, hq, d, generator=gen).bfloat16())
        had = torch.rand(2, hkv, 2112, generator=gen).to(DEV)
        mass.copy_(had)
        graph.replay()
        torch.cuda.synchronize()
        want = step(had)
        assert torch.equal(out.view(torch.int16), want.view(torch.int16)) and torch.equal(mass, had)
