"""Eviction from the paged cache by attention mass (csrc/kv_evict.hip): what is kept and where it goes exactly as the definition says
(tests/attn_mass_ref.py), and a sequence that lives on a budget, against 64 bits over the tokens it still has."""
import pytest
import torch

import attn_mass_ref as ref
from kv_layout import to_fragment, to_logical

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from nanovllm import ops as _ops

    return _ops


def bits(t):
    return t.contiguous().view(torch.int16) if t.dtype == torch.bfloat16 else t.contiguous().view(torch.int32)


def run_evict(ops, hkv, d, block, ctxs, keep, sinks, recent, seed, masses="spread", earlier=True, own_rows=False, other_pages=False, alias=False,
              bad_pages=(), dead=()):
    gen = torch.Generator().manual_seed(seed)
    B = len(ctxs)
    need = [-(-c // block) for c in ctxs]
    width = max(1, max(need))
    wide_out = max(1, -(-min(keep, width * block) // block))
    nblk = sum(need) + 3 + (B * wide_out if other_pages else 0)
    kc = torch.randn(nblk, block, hkv, d, generator=gen).bfloat16()
    vc = torch.randn(nblk, block, hkv, d, generator=gen).bfloat16()
    order = torch.randperm(nblk, generator=gen).tolist()
    bt = torch.full((B, width), -1, dtype=torch.int32)
    for b in range(B):
        for i in range(need[b]):
            bt[b, i] = order.pop()
    for b, i, value in bad_pages:
        bt[b, i] = value
    out_table = bt
    if other_pages:  # every other page is a new one (the kept ones are the sequence's own)
        out_table = torch.full((B, wide_out), -1, dtype=torch.int32)
        for b in range(B):
            for i in range(wide_out):
                out_table[b, i] = order.pop() if i % 2 == 0 or i >= width or bt[b, i] < 0 else bt[b, i]
    room = max(max(ctxs), 1) + 3
    rows = 2 * B + 1
    if masses == "spread":
        mass = torch.exp(torch.randn(rows, hkv, room, generator=gen) * 2)
    elif masses == "ties":
        mass = torch.randint(0, 3, (rows, hkv, room), generator=gen).float()
    elif masses == "equal":
        mass = torch.full((rows, hkv, room), 0.25)
    else:  # everything a float can be
        special = torch.tensor([0.0, -0.0, float("inf"), float("-inf"), float("nan"), -float("nan"), 1e-42, -1e-42, 3e38, -3e38, 1.0, -1.0])
        mass = special[torch.randint(0, len(special), (rows, hkv, room), generator=gen)]
    origin = torch.cumsum(torch.randint(1, 4, (rows, hkv, room), generator=gen), -1).to(torch.int32)
    for i in range(min(sinks, room)):
        origin[..., i] = i
    for r in range(rows):  # as earlier evictions left them: in no order
        for h in range(hkv):
            origin[r, h, sinks:] = origin[r, h, sinks:][torch.randperm(room - sinks, generator=gen)] if room > sinks else origin[r, h, sinks:]
    perm = torch.randperm(rows, generator=gen).to(torch.int32)
    slots = perm[:B]
    slots_out = slots.clone() if own_rows else perm[B:2 * B].clone()
    for b in dead:
        slots_out[b] = -1 if b % 2 else rows
    evicted = torch.zeros(rows, 2, dtype=torch.int32)
    for b in range(B):
        if earlier and b % 2 == 0:
            kept = min(ctxs[b], max(1, keep - 3))
            evicted[slots[b]] = torch.tensor([kept, 3 * room + 5], dtype=torch.int32)
    dev = [to_fragment(kc, False).to(DEV), to_fragment(vc, True).to(DEV)]
    dm, do, de = mass.to(DEV), origin.to(DEV), evicted.to(DEV)
    lens = torch.tensor(ctxs, dtype=torch.int32, device=DEV)
    got_lens = ops.kv_cache_evict(dev[0], dev[1], bt.to(DEV), lens, dm, do, de, slots.to(DEV), keep, sinks, recent, block,
                                  block_tables_out=out_table.to(DEV) if other_pages else None,
                                  slots_out=None if own_rows else slots_out.to(DEV), context_lens_out=lens if alias else None)
    assert (got_lens.data_ptr() == lens.data_ptr()) == alias
    want_k, want_v, want_m, want_o, want_e, want_l = kc.clone(), vc.clone(), mass.clone(), origin.clone(), evicted.clone(), list(ctxs)
    for b, ctx in enumerate(ctxs):
        r, ro = int(slots[b]), int(slots_out[b])
        if not 0 <= ro < rows:
            continue
        pos = ref.position_of(origin[r], evicted[r], ctx)
        n = min(ctx, keep)
        want_l[b] = n
        for h in range(hkv):
            src = ref.choose(mass[r, h, :ctx], pos[h], ctx + int(evicted[r, 1]), keep, sinks, recent) if ctx > keep else list(range(ctx))
            for i, j in enumerate(src):
                to, page = int(out_table[b, i // block]), int(bt[b, j // block])
                if 0 <= to < nblk and 0 <= page < nblk:
                    want_k[to, i % block, h] = kc[page, j % block, h]
                    want_v[to, i % block, h] = vc[page, j % block, h]
            want_m[ro, h, :n] = mass[r, h, src]
            upto = n if ctx > keep else min(int(evicted[r, 0]), ctx)
            want_o[ro, h, :upto] = pos[h][src][:upto]
        want_e[ro] = torch.tensor([n, int(evicted[r, 1]) + ctx - n]) if ctx > keep else evicted[r]
    assert got_lens.tolist() == want_l
    assert torch.equal(de.cpu(), want_e)
    assert torch.equal(bits(dm.cpu()), bits(want_m))
    assert torch.equal(do.cpu(), want_o)
    assert torch.equal(bits(to_logical(dev[0].cpu(), block, False)), bits(want_k))
    assert torch.equal(bits(to_logical(dev[1].cpu(), block, True)), bits(want_v))


SIZES = [  # contexts, keep, sinks, recent
    ([100, 40, 300, 65, 64, 0, 1], 64, 4, 16),
    ([100, 37, 300, 65, 64, 90], 37, 0, 0),
    ([20, 5, 1, 2], 1, 0, 1),
    ([20, 5, 1, 2], 1, 0, 0),
    ([1500, 1100, 1024, 1025], 1024, 4, 128),
    ([2500, 1300], 50, 50, 0),
    ([700, 90], 80, 10, 70),
    ([16, 17, 15, 33], 16, 1, 2),
    ([50, 60], 100, 4, 4),
]


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("hkv,d,block", [(2, 128, 16), (3, 64, 48)])
def test_what_is_kept_and_where(ops, size, hkv, d, block):
    ctxs, keep, sinks, recent = size
    run_evict(ops, hkv, d, block, ctxs, keep, sinks, recent, keep + d)
    run_evict(ops, hkv, d, block, ctxs, keep, sinks, recent, keep + d + 1, own_rows=True, alias=True)


@pytest.mark.parametrize("masses", ["ties", "equal", "any"])
@pytest.mark.parametrize("own_rows", [False, True])
def test_masses_of_every_kind(ops, masses, own_rows):
    run_evict(ops, 2, 128, 16, [400, 130, 129], 128, 4, 30, 3, masses=masses, own_rows=own_rows)
    run_evict(ops, 2, 64, 32, [1300, 77], 70, 0, 0, 4, masses=masses, own_rows=own_rows, earlier=False)


def test_into_other_pages(ops):
    run_evict(ops, 2, 128, 16, [100, 40, 300, 65, 64, 0, 1], 64, 4, 16, 5, other_pages=True)
    run_evict(ops, 2, 64, 48, [100, 40, 300, 65], 50, 4, 16, 6, other_pages=True, own_rows=True)
    run_evict(ops, 2, 128, 64, [100, 140], 500, 4, 16, 7, other_pages=True, own_rows=True)


def test_pages_and_rows_that_are_not_there(ops):
    run_evict(ops, 2, 128, 16, [100, 40, 300, 65], 64, 4, 16, 8, bad_pages=[(0, 1, -1), (0, 5, 100000), (2, 0, -9), (2, 18, -1)])
    run_evict(ops, 2, 128, 16, [100, 90, 300, 80], 64, 4, 16, 9, dead=(0, 1))


@pytest.mark.parametrize("ctx,keep", [(33000, 2048), (40000, 39000), (70001, 100)])
def test_long_contexts(ops, ctx, keep):
    run_evict(ops, 1, 64, 256, [ctx, ctx - 17], keep, 4, 60, ctx)


@pytest.mark.parametrize("room", [5000, 40000])
def test_a_row_named_twice_spoils_its_own_tokens_only(ops, room):
    """sequences of one call that share a row (which a call may not do): whatever they keep, nothing but their own places is written"""
    from nanovllm import _C

    gen = torch.Generator().manual_seed(12)
    hkv, d, block, keep, B = 2, 64, 16, 90, 3
    width, rows = room // block, 3
    nblk = B * width + 2
    table = torch.arange(B * width, dtype=torch.int32).view(B, width) + 1
    k, v = (torch.randn(nblk, hkv, 1, 16 * d, generator=gen).bfloat16().to(DEV) for _ in range(2))
    mass = torch.rand(rows, hkv, room, generator=gen).to(DEV)
    origin = torch.full((rows, hkv, room), -7, dtype=torch.int32, device=DEV)
    evicted = torch.zeros(rows, 2, dtype=torch.int32, device=DEV)
    before = [t.clone() for t in (k, v, mass, origin, evicted)]
    need = _C.lib.mi_kv_cache_evict_workspace(B, hkv, keep, block, width)
    space = torch.full((need + (1 << 20),), 255, dtype=torch.uint8, device=DEV)
    lens = torch.tensor([room - 5, room - 9, room], dtype=torch.int32, device=DEV)
    after = ops.kv_cache_evict(k, v, table.to(DEV), lens, mass, origin, evicted, torch.tensor([1, 1, 0], dtype=torch.int32, device=DEV), keep, 2, 10, block,
                               slots_out=torch.tensor([1, 1, 1], dtype=torch.int32, device=DEV), workspace=space[:need])
    # (tables of 5000 // 16 pages hold 4992 tokens: contexts of more are left as they are)
    assert after.tolist() == [keep if n <= width * block else n for n in lens.tolist()]
    assert bool((space[need:] == 255).all())
    first = torch.zeros(nblk, dtype=torch.bool)
    first[table[:, :-(-keep // block)].flatten().long()] = True
    for got, was in zip((k, v), before):
        assert torch.equal(bits(got[~first]), bits(was[~first]))
    for got, was in zip((mass, origin, evicted), before[2:]):
        assert torch.equal(got[[0, 2]], was[[0, 2]])
    assert torch.equal(mass[1, :, keep:], before[2][1, :, keep:]) and bool((origin[1, :, keep:] == -7).all())


def test_context_longer_than_its_row_stays(ops):
    k = torch.randn(8, 1, 1, 2048, device=DEV).bfloat16()
    v, was = k.clone(), k.clone()
    bt = torch.arange(8, dtype=torch.int32, device=DEV).view(1, 8)
    lens = torch.tensor([100], dtype=torch.int32, device=DEV)
    mass, origin = torch.rand(1, 1, 64, device=DEV), torch.zeros(1, 1, 64, dtype=torch.int32, device=DEV)
    evicted, slot = torch.zeros(1, 2, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    assert ops.kv_cache_evict(k, v, bt, lens, mass, origin, evicted, slot, 32, 1, 1, 16).tolist() == [100]
    assert torch.equal(k.view(torch.int16), was.view(torch.int16)) and evicted.tolist() == [[0, 0]]


def test_a_sequence_on_a_budget(ops):
    """prompt in two portions -> eviction -> decode steps, each with an eviction when the context is 24 over the budget: outputs, masses and
    positions against 64 bits over the tokens kept, captured steps among them"""
    hq, hkv, d, block, keep, sinks, recent = 8, 2, 128, 16, 96, 2, 20
    gen = torch.Generator().manual_seed(4)
    scale, G = d ** -0.5, hq // hkv
    prompts = [150, 90]
    steps = 60
    total = [p + steps for p in prompts]
    B, nblk = 2, 40
    ks = [torch.randn(t, hkv, d, generator=gen).bfloat16() for t in total]
    vs = [torch.randn(t, hkv, d, generator=gen).bfloat16() for t in total]
    qs = [(torch.randn(t, hq, d, generator=gen) * 2).bfloat16() for t in total]
    kc = torch.zeros(ops.kv_cache_shape(nblk, hkv, block), dtype=torch.bfloat16, device=DEV)
    vc = torch.zeros_like(kc)
    pages = torch.randperm(nblk, generator=gen)[:24].view(2, 12).to(torch.int32)
    bt = pages.to(DEV)
    room = 12 * block
    mass = torch.full((3, hkv, room), float("nan"), device=DEV)  # rows need no clearing
    origin = torch.full((3, hkv, room), -5, dtype=torch.int32, device=DEV)
    evicted = torch.zeros(3, 2, dtype=torch.int32, device=DEV)
    slots = torch.tensor([2, 0], dtype=torch.int32, device=DEV)
    slot_rows = [2, 0]
    # the model of it: per sequence and kv head, the tokens' positions in slot order, and their masses with an error bound
    at = [[[] for _ in range(hkv)] for _ in range(B)]
    m64 = [[[] for _ in range(hkv)] for _ in range(B)]
    err = 0.0

    def flat(b, j):
        return int(pages[b, j // block]) * block + j % block

    # two portions
    for lo, hi in ((0, 70), (70, None)):
        portion = [(lo, min(hi, p) if hi else p) for p in prompts]
        k = torch.cat([ks[b][a:z] for b, (a, z) in enumerate(portion)]).to(DEV)
        v = torch.cat([vs[b][a:z] for b, (a, z) in enumerate(portion)]).to(DEV)
        q = torch.cat([qs[b][a:z] for b, (a, z) in enumerate(portion)]).to(DEV)
        where = torch.tensor([flat(b, j) for b, (a, z) in enumerate(portion) for j in range(a, z)], dtype=torch.int32, device=DEV)
        ops.reshape_and_cache(k, v, kc, vc, where, hkv, block)
        cu = torch.tensor([0, portion[0][1] - lo, portion[0][1] - lo + portion[1][1] - lo], dtype=torch.int32, device=DEV)
        lens = torch.tensor([z for _, z in portion], dtype=torch.int32, device=DEV)
        ops.prompt_attn_mass(q, kc, bt, cu, lens, max(z - a for a, z in portion), mass, slots, hq, hkv, block, scale)
    for b, p in enumerate(prompts):
        w, A = ref.weights(qs[b][:p], ks[b][:p].double(), torch.ones(p, dtype=torch.bool), 0, scale)
        err = max(err, ref.mass_bound(d, A, p, p * G))
        for h in range(hkv):
            at[b][h] = list(range(p))
            m64[b][h] = ref.mass_of(w, hkv)[h].tolist()
    ctx = list(prompts)
    dropped = [0, 0]
    lens = torch.tensor(ctx, dtype=torch.int32, device=DEV)

    def check_state():
        got = mass.cpu()
        for b in range(B):
            pos = ref.position_of(origin.cpu()[slot_rows[b]], evicted.cpu()[slot_rows[b]], ctx[b])
            for h in range(hkv):
                assert pos[h].tolist() == at[b][h]
                want = torch.tensor(m64[b][h], dtype=torch.float64)
                have = got[slot_rows[b], h, :ctx[b]].double()
                assert bool(((have - want).abs() <= (err + steps * ref.U) * want + 1e-30).all())

    def evict():
        ops.kv_cache_evict(kc, vc, bt, lens, mass, origin, evicted, slots, keep, sinks, recent, block, context_lens_out=lens)
        had = mass_before
        for b in range(B):
            if ctx[b] <= keep:
                continue
            for h in range(hkv):
                # by the device's own masses: two that are equal within the bound may stand in either order
                src = ref.choose(had[slot_rows[b], h, :ctx[b]], torch.tensor(at[b][h]), ctx[b] + dropped[b], keep, sinks, recent)
                at[b][h] = [at[b][h][j] for j in src]
                m64[b][h] = [m64[b][h][j] for j in src]
            dropped[b] += ctx[b] - keep
            ctx[b] = keep
        assert lens.tolist() == ctx

    check_state()
    mass_before = mass.cpu()
    evict()
    check_state()
    graph = None
    q = torch.zeros(B, hq, d, dtype=torch.bfloat16, device=DEV)
    for s in range(steps):
        lens += 1
        pairs, knew, vnew = [], [], []
        for b in range(B):
            t = prompts[b] + s
            pairs.append([int(pages[b, ctx[b] // block]), ctx[b] % block])
            knew.append(ks[b][t])
            vnew.append(vs[b][t])
            q[b].copy_(qs[b][t])
            ctx[b] += 1
            for h in range(hkv):
                at[b][h].append(t)
        ops.scatter_update_kv(torch.stack(knew).to(DEV), torch.stack(vnew).to(DEV), kc, vc, torch.tensor(pairs, dtype=torch.int32, device=DEV), hkv, block)
        if s == 8:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = ops.paged_attn_decode_mass(q, kc, vc, bt, lens, mass, slots, hq, hkv, block, scale)
        if graph is not None:
            graph.replay()
        else:
            out = ops.paged_attn_decode_mass(q, kc, vc, bt, lens, mass, slots, hq, hkv, block, scale)
        for b in range(B):
            for h in range(hkv):
                k, v = ks[b][at[b][h], h].double(), vs[b][at[b][h], h].double()
                rows = qs[b][prompts[b] + s, h * G:(h + 1) * G]
                w, A = ref.weights(rows.view(1, G, d), k.unsqueeze(1), torch.ones(ctx[b], dtype=torch.bool), ctx[b] - 1, scale)
                bound = ref.mass_bound(d, A, ctx[b], G)
                err = max(err, bound)
                want, size = w[:, 0] @ v, w[:, 0] @ v.abs()
                have = out.view(B, hq, d)[b, h * G:(h + 1) * G].cpu().double()
                assert bool(((have - want).abs() <= 2.0 ** -8 * want.abs() + (bound + 2.0 ** -16) * size * 1.01).all()), (s, b, h)
                now = w.sum((0, 1)).tolist()
                m64[b][h] = [x + y for x, y in zip(m64[b][h] + [0.0], now)]
        if max(ctx) > keep + 24:
            check_state()
            mass_before = mass.cpu()
            evict()
            check_state()
    check_state()


@pytest.mark.parametrize("ctx,block", [(1500, 16), (3000, 64), (12000, 64), (32768, 256), (33000, 256)])
@pytest.mark.parametrize("keep", [36, 63, 100, 163, 700, 1000])
def test_equal_masses_around_a_budget_off_64_slots(ops, ctx, block, keep):
    """The last of the equal masses that stay is in the 64 slots that the budget cuts.  First sequence: all slots below the budget and those from
    the budget's own place in the next 64 on are equal, and two behind are larger; the others: masses of two kinds, of one, and zero or not"""
    gen = torch.Generator().manual_seed(ctx + keep)
    hkv, d = 2, 64
    mass = torch.zeros(4, hkv, ctx)
    mass[0, :, :keep] = 1.0
    mass[0, :, keep + keep % 64:keep + 64] = 1.0
    mass[0, :, [ctx - 20, ctx - 1]] = 2.0
    mass[1] = torch.randint(0, 2, (hkv, ctx), generator=gen)
    mass[2] = 0.5
    mass[3] = torch.rand(hkv, ctx, generator=gen) * (torch.rand(hkv, ctx, generator=gen) < keep / ctx / 2)
    per = -(-ctx // block)
    bt = torch.randperm(4 * per, generator=gen).view(4, per).to(torch.int32)
    kc = torch.randn(4 * per, block, hkv, d, generator=gen).bfloat16()
    k, v = to_fragment(kc, False).to(DEV), to_fragment(kc, True).to(DEV)
    m, origin = mass.to(DEV), torch.zeros(4, hkv, ctx, dtype=torch.int32, device=DEV)
    evicted, slots = torch.zeros(4, 2, dtype=torch.int32, device=DEV), torch.arange(4, dtype=torch.int32, device=DEV)
    ops.kv_cache_evict(k, v, bt.to(DEV), torch.full((4,), ctx, dtype=torch.int32, device=DEV), m, origin, evicted, slots, keep, 0, 0, block)
    got_k, got_v = to_logical(k.cpu(), block, False), to_logical(v.cpu(), block, True)
    i = torch.arange(keep)
    for b in range(4):
        for h in range(hkv):
            src = torch.tensor(ref.choose(mass[b, h], torch.arange(ctx), ctx, keep, 0, 0))
            assert torch.equal(origin[b, h, :keep].cpu().long(), src), (b, h)
            assert torch.equal(m[b, h, :keep].cpu(), mass[b, h][src])
            for got in (got_k, got_v):
                assert torch.equal(bits(got[bt[b, i // block].long(), i % block, h]), bits(kc[bt[b, src // block].long(), src % block, h]))
