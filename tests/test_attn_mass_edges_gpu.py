"""Attention mass and eviction where a program goes beyond the plain call: caches of more than 2^31 elements, captured evictions, padded
batches, workspaces of the caller's own, queries that are not numbers."""
import pytest
import torch

import attn_mass_ref as ref
from kv_layout import to_fragment, to_logical
from test_attn_mass_gpu import check_mass, device_caches, pool

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from nanovllm import ops as _ops

    return _ops


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def test_caches_of_more_than_2_to_the_31_elements(ops):
    """pages at the cache's two ends: 131 100 blocks of 16 384 elements"""
    gen = torch.Generator().manual_seed(3)
    hq, hkv, d, block, ctx = 16, 8, 128, 16, 75
    kc, vc, bt = pool(gen, hkv, d, block, [ctx], extra=0, width_more=0)
    n = kc.shape[0]
    big = 131100
    kd = torch.empty(ops.kv_cache_shape(big, hkv, block), dtype=torch.bfloat16, device=DEV)
    vd = torch.empty_like(kd)
    where = torch.tensor([big - 1, 0, big - 3, 65537, big - 2], device=DEV)
    assert n == 5 and kd.numel() > 2 ** 31
    far = torch.empty_like(bt)
    ks, vs = device_caches(kc, vc)
    for i in range(5):
        kd[where[i]], vd[where[i]] = ks[bt[0, i]], vs[bt[0, i]]
        far[0, i] = where[i]
    q = torch.randn(ctx, hq, d, generator=gen).bfloat16().to(DEV)
    lens, slot = i32(ctx), i32(0)
    got = {}
    for name, k, v, t in (("near", ks, vs, bt.to(DEV)), ("far", kd, vd, far.to(DEV))):
        mass = torch.zeros(1, hkv, 96, device=DEV)
        origin, evicted = torch.zeros(1, hkv, 96, dtype=torch.int32, device=DEV), torch.zeros(1, 2, dtype=torch.int32, device=DEV)
        ops.prompt_attn_mass(q, k, t, i32(0, ctx), lens, ctx, mass, slot, hq, hkv, block, d ** -0.5)
        out = ops.paged_attn_decode_mass(q[:1], k, v, t, lens, mass, slot, hq, hkv, block, d ** -0.5)
        after = ops.kv_cache_evict(k, v, t, lens, mass, origin, evicted, slot, 40, 2, 8, block)
        flat = (t.long()[0, :, None] * block + torch.arange(block, device=DEV)).view(-1)[:40].to(torch.int32)
        rows = [] if name == "far" else [ops.kv_cache_gather(k, False, flat, hkv, block), ops.kv_cache_gather(v, True, flat, hkv, block)]
        if name == "far":  # (flat slots of a cache this large do not fit the helper's 32 bits times a block)
            small = torch.arange(5, dtype=torch.int32, device=DEV)
            kk, vv = k[where].contiguous(), v[where].contiguous()
            flat = (small.long()[:, None] * block + torch.arange(block, device=DEV)).view(-1)[:40].to(torch.int32)
            rows = [ops.kv_cache_gather(kk, False, flat, hkv, block), ops.kv_cache_gather(vv, True, flat, hkv, block)]
        got[name] = [out, mass, origin, evicted, after, *rows]
    for a, b in zip(got["near"], got["far"]):
        assert torch.equal(a.view(torch.int16) if a.dtype == torch.bfloat16 else a, b.view(torch.int16) if b.dtype == torch.bfloat16 else b)


def test_eviction_captured(ops):
    """replays on other masses, with eager work between them; the graph's own workspace"""
    gen = torch.Generator().manual_seed(5)
    hkv, d, block, keep = 2, 64, 16, 48
    ctxs = [100, 70]
    bt = torch.randperm(16, generator=gen)[:14].view(2, 7).to(torch.int32).to(DEV)
    shape = ops.kv_cache_shape(16, hkv, block, d)
    k, v = torch.zeros(shape, dtype=torch.bfloat16, device=DEV), torch.zeros(shape, dtype=torch.bfloat16, device=DEV)
    mass = torch.zeros(2, hkv, 112, device=DEV)
    origin, evicted = torch.zeros(2, hkv, 112, dtype=torch.int32, device=DEV), torch.zeros(2, 2, dtype=torch.int32, device=DEV)
    lens, slots = i32(*ctxs), i32(1, 0)

    def step(k, v, lens, mass, origin, evicted):
        return ops.kv_cache_evict(k, v, bt, lens, mass, origin, evicted, slots, keep, 2, 10, block, context_lens_out=lens)

    state = (k, v, lens, mass, origin, evicted)
    step(*[t.clone() for t in state])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(*state)
    for i in range(4):
        start = [torch.randn(shape, generator=gen).bfloat16(), torch.randn(shape, generator=gen).bfloat16(), torch.tensor(ctxs, dtype=torch.int32),
                 torch.rand(2, hkv, 112, generator=gen), torch.zeros(2, hkv, 112, dtype=torch.int32), torch.zeros(2, 2, dtype=torch.int32)]
        for t, s in zip(state, start):
            t.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        want = [s.to(DEV) for s in start]
        step(*want)
        assert lens.tolist() == [keep, keep] and evicted.tolist() == [[keep, 70 - keep], [keep, 100 - keep]]
        for a, b in zip(state, want):
            assert torch.equal(a.view(torch.int16) if a.dtype == torch.bfloat16 else a, b.view(torch.int16) if b.dtype == torch.bfloat16 else b)


def test_padded_rows_may_name_a_sequences_row(ops):
    """rows of no tokens that name the row of a sequence of the call leave it to that sequence"""
    gen = torch.Generator().manual_seed(6)
    hq, hkv, d, block, ctx, keep = 16, 8, 128, 16, 130, 64
    kc, vc, bt = pool(gen, hkv, d, block, [ctx])
    pads = 40
    table = torch.full((1 + pads, bt.shape[1]), -1, dtype=torch.int32)
    table[0] = bt[0]
    lens = torch.zeros(1 + pads, dtype=torch.int32)
    lens[0] = ctx
    slots = torch.zeros(1 + pads, dtype=torch.int32)
    q = torch.randn(1 + pads, hq, d, generator=gen).bfloat16().to(DEV)
    results = []
    for rows in (1, 1 + pads):
        k, v = device_caches(kc, vc)
        mass = torch.rand(2, hkv, 160, generator=torch.Generator().manual_seed(1)).to(DEV)
        origin, evicted = torch.zeros(2, hkv, 160, dtype=torch.int32, device=DEV), torch.zeros(2, 2, dtype=torch.int32, device=DEV)
        t, n, s = table[:rows].to(DEV), lens[:rows].to(DEV), slots[:rows].to(DEV)
        out = ops.paged_attn_decode_mass(q[:rows], k, v, t, n, mass, s, hq, hkv, block, d ** -0.5)
        cu = torch.zeros(rows + 1, dtype=torch.int32, device=DEV)
        cu[1:] = 1
        ops.prompt_attn_mass(q[:1], k, t, cu, n, 1, mass, s, hq, hkv, block, d ** -0.5)
        after = ops.kv_cache_evict(k, v, t, n, mass, origin, evicted, s, keep, 2, 10, block)
        assert after.tolist() == [keep] + [0] * (rows - 1) and evicted.tolist() == [[keep, ctx - keep], [0, 0]]
        assert not bool(out[1:].any())
        # (one split and many are summed in different orders)
        results.append((mass, origin, to_logical(k.cpu(), block, False).nan_to_num(), out[0].float()))
    a, b = results
    _, A = ref.weights(q[:1].cpu(), *ref.rows_of(kc, bt[0], ctx), ctx - 1, d ** -0.5)
    bound = 2 * ref.mass_bound(d, A, ctx, 2)
    assert bool(((a[0] - b[0]).abs() <= (bound + 4 * ref.U) * a[0].abs().clamp(min=1e-30)).all())
    assert torch.equal(a[1], b[1]) and torch.equal(a[2], b[2])


def test_workspaces_of_the_caller(ops):
    from nanovllm import _C

    gen = torch.Generator().manual_seed(8)
    hq, hkv, d, block, ctx = 16, 8, 128, 16, 700
    kc, vc, bt = pool(gen, hkv, d, block, [ctx], width_more=0)
    k, v = device_caches(kc, vc)
    t, lens, slot = bt.to(DEV), i32(ctx), i32(0)
    q = torch.randn(30, hq * d, generator=gen).bfloat16().to(DEV)
    need = [_C.lib.mi_paged_attn_decode_mass_workspace(1, hq, hkv, d, block, t.shape[1]),
            _C.lib.mi_prompt_attn_mass_workspace(1, 30, 30, 0, hq, hkv, d, block, t.shape[1]), _C.lib.mi_kv_cache_evict_workspace(1, hkv, 512, block, t.shape[1])]
    results = []
    for ws in (None, torch.full((max(need),), 255, dtype=torch.uint8, device=DEV)):  # what it holds does not matter
        mass = torch.zeros(1, hkv, 704, device=DEV)
        origin, evicted = torch.zeros(1, hkv, 704, dtype=torch.int32, device=DEV), torch.zeros(1, 2, dtype=torch.int32, device=DEV)
        ops.prompt_attn_mass(q, k, t, i32(0, 30), lens, 30, mass, slot, hq, hkv, block, 0.1, workspace=ws)
        out = torch.empty(1, hq, d, dtype=torch.bfloat16, device=DEV)
        assert ops.paged_attn_decode_mass(q[:1], k, v, t, lens, mass, slot, hq, hkv, block, 0.1, out=out, workspace=ws) is out
        kk, vv = k.clone(), v.clone()
        ops.kv_cache_evict(kk, vv, t, lens, mass, origin, evicted, slot, 512, 2, 10, block, workspace=ws)
        results.append((out.view(torch.int16), mass, origin, evicted, kk.view(torch.int16), vv.view(torch.int16)))
    for a, b in zip(*results):
        assert torch.equal(a, b)
    short = torch.empty(64, dtype=torch.uint8, device=DEV)
    for call in (lambda: ops.paged_attn_decode_mass(q[:1], k, v, t, lens, mass, slot, hq, hkv, block, 0.1, workspace=short),
                 lambda: ops.prompt_attn_mass(q, k, t, i32(0, 30), lens, 30, mass, slot, hq, hkv, block, 0.1, workspace=short),
                 lambda: ops.kv_cache_evict(k, v, t, lens, mass, origin, evicted, slot, 512, 2, 10, block, workspace=short),
                 lambda: ops.paged_attn_decode_mass(q[:1], k, v, t.cpu(), lens, mass, slot, hq, hkv, block, 0.1)):
        with pytest.raises(_C.MiError):
            call()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_query_that_is_no_number_spoils_its_own_heads_only(ops, bad):
    gen = torch.Generator().manual_seed(9)
    hq, hkv, d, block, ctx = 16, 8, 128, 16, 300
    kc, vc, bt = pool(gen, hkv, d, block, [ctx, ctx])
    k, v = device_caches(kc, vc)
    q = torch.randn(2, hq, d, generator=gen).bfloat16()
    q[1, 5, 7] = bad  # kv head 2 of the second sequence
    lens, slots = i32(ctx, ctx), i32(0, 1)
    start = torch.rand(2, hkv, 310, generator=gen)
    for prompt in (False, True):
        mass = start.to(DEV)
        if prompt:
            ops.prompt_attn_mass(q.to(DEV), k, bt.to(DEV), i32(0, 1, 2), lens, 1, mass, slots, hq, hkv, block, d ** -0.5)
        else:
            out = ops.paged_attn_decode_mass(q.to(DEV), k, v, bt.to(DEV), lens, mass, slots, hq, hkv, block, d ** -0.5).view(2, hq, d).cpu()
            assert bool(out[1, 5].isnan().all()) and not bool(out[0].isnan().any()) and not bool(out[1, :5].isnan().any() or out[1, 6:].isnan().any())
        got = mass.cpu()
        assert bool(got[1, 2, :ctx].isnan().all())
        for b in range(2):
            rows, there = ref.rows_of(kc, bt[b], ctx)
            w, A = ref.weights(q[b:b + 1].nan_to_num(0.0, 0.0, 0.0), rows, there, ctx - 1, d ** -0.5)
            new, bound = ref.mass_of(w, hkv), ref.mass_bound(d, A, ctx, 2)
            for h in range(hkv):
                if (b, h) != (1, 2):
                    check_mass(got[:, h:h + 1], start[:, h:h + 1], b, b, b, new[h:h + 1], ctx, ctx - 1, bound, 310)


def test_a_key_of_infinite_negative_score_gets_nothing(ops):
    """... and spoils nothing: neither the other keys nor, through rows that a tile is filled up with, its own mass"""
    gen = torch.Generator().manual_seed(10)
    hq, hkv, d, block, ctx = 16, 8, 128, 16, 137
    kc, vc, bt = pool(gen, hkv, d, block, [ctx])
    kc[bt[0, 1], 3, :, 0] = float("inf")  # token 19
    q = torch.randn(ctx, hq, d, generator=gen).bfloat16()
    q[..., 0] = -q[..., 0].abs() - 0.5
    k, v = device_caches(kc, vc)
    start = torch.rand(1, hkv, 140, generator=gen)
    finite = kc.clone()
    finite[bt[0, 1], 3, :, 0] = 0.0
    rows, there = ref.rows_of(finite, bt[0], ctx)
    there[19] = False
    for n in (1, ctx):
        mass = start.to(DEV)
        ops.prompt_attn_mass(q[ctx - n:].to(DEV), k, bt.to(DEV), i32(0, n), i32(ctx), n, mass, i32(0), hq, hkv, block, d ** -0.5)
        w, A = ref.weights(q[ctx - n:], rows, there, ctx - n, d ** -0.5)
        check_mass(mass.cpu(), start, 0, 0, 0, ref.mass_of(w, hkv), ctx, ctx - n, ref.mass_bound(d, A, ctx, 2 * n), 140)
    mass = start.to(DEV)
    out = ops.paged_attn_decode_mass(q[-1:].to(DEV), k, v, bt.to(DEV), i32(ctx), mass, i32(0), hq, hkv, block, d ** -0.5)
    w, A = ref.weights(q[-1:], rows, there, ctx - 1, d ** -0.5)
    check_mass(mass.cpu(), start, 0, 0, 0, ref.mass_of(w, hkv), ctx, ctx - 1, ref.mass_bound(d, A, ctx, 2), 140)
    assert not bool(out.isnan().any())
