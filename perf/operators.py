"""A paged cache that keeps what is attended to: the attention mass of every cached token, and the eviction by it.

Three operators over the fragment-native cache (one tile of 16 tokens per kv head), per layer:

  decode  one new token per sequence attends its cached context, and every cached token's mass - the softmax weights that it
          has been given, summed over the query heads of its kv head - grows by this step's
              o_h = sum_j p_hj v_j,   mass_j += sum_h p_hj,   p_h = softmax_j(scale q_h . k_j)
  prompt  the mass that the last `window` rows of a prompt (0: all of them) give to the tokens they see
              mass_j += sum_i sum_h p_hij,   p_hi = softmax over j <= position(i)
  evict   of a context longer than `keep` the first `sinks` tokens, the last `recent` ones and those of the largest mass stay
          (ties: the lower slot), each kv head its own; kept tokens from behind `keep` move into the places that become free
          below it, the n-th of them into the n-th free one

A mass that a step's own tokens begin with is set, older ones are added to.  State rows: `slots` are read, `slots_out` written
(other rows here, as for a step that may be taken back, so that a pass can be repeated).
"""
import math
import os
import sys

import torch

own = False

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nano-vllm-ascend_amd")


def _case(op, name, heads, dim, block, seqs, lo, hi, past=0, window=0, keep=0, sinks=4, recent=64):
    return dict(name=name, op=op, q_heads=heads[0], kv_heads=heads[1], dim=dim, block=block, seqs=seqs, lo=lo, hi=hi, past=past,
                window=window, keep=keep, sinks=sinks, recent=recent)


def listed():
    return [
        # one user's short conversation, the next token: latency
        _case("decode", "decode 1 x 200", (16, 8), 128, 16, 1, 200, 200),
        # the batch of the headline workload
        _case("decode", "decode 32 x 1024", (16, 8), 128, 16, 32, 1024, 1024),
        # a busy server: ragged contexts, seven query heads per kv head
        _case("decode", "decode 24 ragged", (28, 4), 128, 16, 24, 101, 8000),
        # long documents in a batch, eight query heads per kv head
        _case("decode", "decode 8 x 32768", (64, 8), 128, 64, 8, 32768, 32768),
        # one very long document, 64-wide heads: the cache's length is all there is to split
        _case("decode", "decode 1 x 131072", (32, 8), 64, 256, 1, 131072, 131072),
        # a short question arriving, all its rows observed
        _case("prompt", "prompt 1 x 137", (16, 8), 128, 16, 1, 137, 137),
        # ragged prompts, the last 32 rows observed
        _case("prompt", "prompt 8 ragged, last 32", (32, 8), 64, 16, 8, 333, 2100, window=32),
        # one long document, the last 64 rows observed: what decides what is kept of it
        _case("prompt", "prompt 32768, last 64", (64, 8), 128, 64, 1, 32768, 32768, window=64),
        # a portion of 4096 rows behind 4096 cached ones, all rows observed
        _case("prompt", "prompt 4096 behind 4096", (32, 8), 128, 16, 1, 4096, 4096, past=4096),
        # one conversation grown past its budget
        _case("evict", "evict 1 x 1100 to 1024", (16, 8), 128, 16, 1, 1100, 1100, keep=1024, recent=128),
        # a batch of decoding sequences, each back to its budget after up to 257 tokens (some are within it)
        _case("evict", "evict 32 ragged to 4096", (32, 8), 128, 16, 32, 4065, 4353, keep=4096, recent=256),
        # long documents cut to an eighth once they are read
        _case("evict", "evict 8 x 32768 to 4096", (64, 8), 128, 64, 8, 32768, 32768, keep=4096, recent=512),
    ]


_HEADS = [((16, 8), 128), ((32, 8), 128), ((64, 8), 128), ((28, 4), 128), ((7, 1), 128), ((16, 1), 64), ((8, 8), 128), ((32, 8), 64),
          ((14, 2), 64), ((20, 4), 128)]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    op = rng.choice(["decode", "prompt", "evict"])
    heads, dim = rng.choice(_HEADS)
    block = rng.choice([16, 32, 64, 256])
    name = ""
    if op == "decode":
        seqs = _log_int(rng, 1, 64)
        hi = _log_int(rng, 1, min(131072, 8 * 32768 * 8 * 128 // (seqs * heads[1] * dim), 8 * 32768 * 64 // (seqs * heads[0])))
        return _case(op, name, heads, dim, block, seqs, _log_int(rng, 1, hi), hi)
    if op == "prompt":
        seqs = _log_int(rng, 1, 16)
        window = rng.choice([0, 0, rng.randint(1, 128)])
        hi = _log_int(rng, 1, min(4096, 131072 // heads[0]) // seqs if window == 0 else 32768 // seqs)
        past = rng.choice([0, _log_int(rng, 1, max(1, (6000 if window == 0 else 32768) // seqs - hi))])
        return _case(op, name, heads, dim, block, seqs, _log_int(rng, 1, hi), hi, past=past, window=window)
    seqs = _log_int(rng, 1, 48)
    hi = _log_int(rng, 32, min(65536, 8 * 32768 * 8 // (seqs * heads[1]) // 2))
    keep = _log_int(rng, 16, max(16, hi - 1))
    return _case(op, name, heads, dim, block, seqs, _log_int(rng, max(1, hi // 2), hi), hi, keep=keep, sinks=rng.randint(0, 4),
                 recent=rng.randint(0, min(256, keep // 2)))


def _lengths(case):
    """the sequences' new rows (prompt) or contexts (decode, evict), spread over lo..hi"""
    n = case["seqs"]
    return [case["lo"] + int((case["hi"] - case["lo"]) * ((i * 0.6180339887 + 1.0) % 1.0 if i else 1.0)) for i in range(n)]


def _contexts(case):
    return [case["past"] + n for n in _lengths(case)]


def work(case):
    H, G, D = case["kv_heads"], case["q_heads"] // case["kv_heads"], case["dim"]
    if case["op"] == "decode":
        n = sum(_lengths(case))
        return {"bytes": n * H * D * 4 + n * H * 8 + 4 * case["seqs"] * H * G * D, "flops": 4 * n * H * G * D}
    if case["op"] == "prompt":
        pairs = rows = 0
        for new in _lengths(case):
            w = min(case["window"] or new, new)
            rows += w
            pairs += sum(range(case["past"] + new - w + 1, case["past"] + new + 1))
        n = sum(_contexts(case))
        return {"bytes": n * H * D * 2 + rows * H * G * D * 2 + n * H * 8, "flops": 2 * pairs * H * G * D}
    size = 0
    for n in _lengths(case):
        if n <= case["keep"]:
            continue
        # kept tokens from behind `keep`: the recent ones there, and of the others the share that lies there
        size += n * H * 4
        recent = min(case["recent"], n - case["keep"])
        free = case["keep"] - case["sinks"] - case["recent"]
        share = max(0, n - case["keep"] - case["recent"]) / max(1, n - case["sinks"] - case["recent"])
        size += int((recent + free * share) * H * (D * 8 + 16))
    return {"bytes": max(size, case["seqs"] * H * 4), "flops": sum(_lengths(case)) * H}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    H, G, D, block, n = case["kv_heads"], case["q_heads"] // case["kv_heads"], case["dim"], case["block"], case["seqs"]
    ctx = _contexts(case)
    need = [-(-c // block) for c in ctx]
    n_blocks = sum(need) + 2
    order = torch.randperm(n_blocks, generator=host).tolist()
    width = max(need)
    tables = []
    for k in need:  # pages in any order, rows filled up with -1
        tables.append([order.pop() for _ in range(k)] + [-1] * (width - k))
    shape = (n_blocks, H, block // 16, 16 * D)
    room = -(-max(ctx) // 64) * 64

    def normal(*size, dtype=torch.float32):
        return torch.randn(size, generator=gen, device="cuda", dtype=dtype)

    st = dict(case=case, ctx=ctx, new=_lengths(case), k_cache=normal(*shape, dtype=torch.bfloat16), v_cache=normal(*shape, dtype=torch.bfloat16),
              tables=torch.tensor(tables, dtype=torch.int32, device="cuda"), lens=torch.tensor(ctx, dtype=torch.int32, device="cuda"))
    # state rows of the sequences, in any order, and the rows that receive the result
    rows = torch.randperm(2 * n, generator=host).to(torch.int32)
    st["slots"], st["slots_out"] = rows[:n].cuda(), rows[n:].cuda()
    # masses as they come to be: most tokens have little, a few a great deal
    st["mass"] = torch.exp(normal(2 * n, H, room) * 2 - 4)
    if case["op"] == "evict":
        # what an earlier eviction left: some sequences have had one (kept tokens' positions ascend with gaps), others none
        origin = torch.cumsum(torch.randint(1, 4, (2 * n, H, room), generator=gen, device="cuda"), -1).to(torch.int32)
        origin[..., :case["sinks"]] = torch.arange(min(case["sinks"], room), dtype=torch.int32, device="cuda")
        evicted = torch.zeros(2 * n, 2, dtype=torch.int32)
        for i in range(n):
            if i % 2 == 1:
                kept = min(case["keep"], ctx[i])
                evicted[rows[i]] = torch.tensor([kept, 3 * kept + 8], dtype=torch.int32)
        st["origin"], st["evicted"] = origin, evicted.cuda()
        st["lens_out"] = torch.zeros(n, dtype=torch.int32, device="cuda")
    else:
        # scores of a deviation of about two: weights that differ by orders of magnitude
        st["q"] = (normal(n if case["op"] == "decode" else sum(st["new"]), H * G, D) * 2).to(torch.bfloat16)
        st["scale"] = D ** -0.5
        cu = [0]
        for k in st["new"]:
            cu.append(cu[-1] + k)
        st["cu"], st["cu_host"] = torch.tensor(cu, dtype=torch.int32, device="cuda"), cu
    return st


# ---- the framework's calls ----------------------------------------------------------------------------------------------
def _run_own(st):
    if PKG not in sys.path:
        sys.path.insert(0, PKG)
    from nanovllm import ops

    case = st["case"]
    hq, h, block = case["q_heads"], case["kv_heads"], case["block"]
    if case["op"] == "decode":
        out = ops.paged_attn_decode_mass(st["q"], st["k_cache"], st["v_cache"], st["tables"], st["lens"], st["mass"], st["slots"],
                                         hq, h, block, st["scale"], slots_out=st["slots_out"])
        return {"out": out, "mass": st["mass"]}
    if case["op"] == "prompt":
        ops.prompt_attn_mass(st["q"], st["k_cache"], st["tables"], st["cu"], st["lens"], max(st["new"]), st["mass"], st["slots"],
                             hq, h, block, st["scale"], window=case["window"], slots_out=st["slots_out"])
        return {"mass": st["mass"]}
    ops.kv_cache_evict(st["k_cache"], st["v_cache"], st["tables"], st["lens"], st["mass"], st["origin"], st["evicted"], st["slots"],
                       case["keep"], case["sinks"], case["recent"], block, slots_out=st["slots_out"], context_lens_out=st["lens_out"])
    return _evict_outputs(st)


def _evict_outputs(st):
    return {"lens": st["lens_out"], "k_cache": st["k_cache"], "v_cache": st["v_cache"], "mass": st["mass"], "origin": st["origin"],
            "evicted": st["evicted"]}


# ---- the plain forms ----------------------------------------------------------------------------------------------------
def _keys(cache, blocks, dim):
    """[..., blocks] -> [..., kv heads, tokens, dim], 32 bits"""
    x = cache.view(cache.shape[0], cache.shape[1], cache.shape[2], dim // 32, 4, 16, 8)[blocks.clamp(min=0).long()]
    # [B, block, head, tile, 32 dims, 8 dims, token, dim]
    x = x.permute(0, 2, 1, 3, 6, 4, 5, 7)
    return x.reshape(x.shape[0], x.shape[1], -1, dim).float()


def _values(cache, blocks, dim):
    x = cache.view(cache.shape[0], cache.shape[1], cache.shape[2], dim // 32, 4, 16, 2, 4)[blocks.clamp(min=0).long()]
    # [B, block, head, tile, 32 dims, 4 tokens, dim, 16 dims, token]
    x = x.permute(0, 2, 1, 3, 5, 8, 4, 7, 6)
    return x.reshape(x.shape[0], x.shape[1], -1, dim).float()


def _plain_decode(st):
    case, H, D = st["case"], st["case"]["kv_heads"], st["case"]["dim"]
    n = case["seqs"]
    G = case["q_heads"] // H
    k, v = _keys(st["k_cache"], st["tables"], D), _values(st["v_cache"], st["tables"], D)
    s = (st["q"].view(n, H, G, D).float() @ k.transpose(2, 3)) * st["scale"]
    j = torch.arange(s.shape[-1], device="cuda", dtype=torch.int32)
    seen = j < st["lens"].view(n, 1, 1, 1)
    s = torch.where(seen, s, -torch.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = (p @ v).to(torch.bfloat16)
    room = st["mass"].shape[-1]
    t = min(room, s.shape[-1])
    j = j[:t]
    had = st["mass"][st["slots"].long(), :, :t]
    last = st["lens"].view(n, 1, 1) - 1
    now = torch.where(j < last, had, 0.0) + p.sum(2)[..., :t]
    to = st["slots_out"].long()
    st["mass"][to, :, :t] = torch.where(j <= last, now, st["mass"][to, :, :t])
    return {"out": out.view(n, -1), "mass": st["mass"]}


def _plain_prompt(st):
    case, H, D = st["case"], st["case"]["kv_heads"], st["case"]["dim"]
    G = case["q_heads"] // H
    slots, to = st["slots"].long(), st["slots_out"].long()
    for b, (new, ctx) in enumerate(zip(st["new"], st["ctx"])):
        w = min(case["window"] or new, new)
        q = st["q"][st["cu_host"][b + 1] - w:st["cu_host"][b + 1]].view(w, H, G, D).permute(1, 2, 0, 3).float()
        k = _keys(st["k_cache"], st["tables"][b:b + 1, :-(-ctx // case["block"])], D)[0, :, :ctx]
        at = torch.arange(ctx - w, ctx, device="cuda").view(w, 1)
        seen = torch.arange(ctx, device="cuda") <= at
        mass = torch.empty(H, ctx, device="cuda")
        step = max(1, (1 << 28) // (w * G * ctx))
        for h in range(0, H, step):
            s = q[h:h + step].reshape(-1, G * w, D) @ k[h:h + step].transpose(1, 2) * st["scale"]
            s = torch.where(seen, s.view(-1, G, w, ctx), -torch.inf)
            p = torch.exp(s - s.amax(-1, keepdim=True))
            p = p / p.sum(-1, keepdim=True)
            mass[h:h + step] = p.sum((1, 2))
        mass[:, :ctx - new] += st["mass"][slots[b], :, :ctx - new]
        st["mass"][to[b], :, :ctx] = mass
    return {"mass": st["mass"]}


def _plain_evict(st):
    case, n = st["case"], st["case"]["seqs"]
    H, D, keep, block = case["kv_heads"], case["dim"], case["keep"], case["block"]
    slots, to = st["slots"].long(), st["slots_out"].long()
    T = max(max(st["ctx"]), keep)
    lens = st["lens"].view(n, 1, 1)
    j = torch.arange(T, device="cuda", dtype=torch.int32)
    jc = j.clamp(max=st["mass"].shape[-1] - 1).long()
    mass, origin = st["mass"][slots][..., jc], st["origin"][slots][..., jc]
    had = st["evicted"][slots].view(n, 1, 2)
    position = torch.where(j < had[..., :1], origin, j + had[..., 1:])
    full = lens > keep
    stays = (position < case["sinks"]) | (position >= lens + had[..., 1:] - case["recent"])
    key = torch.where(stays, torch.inf, mass.nan_to_num(-torch.inf))
    key = torch.where(j < lens, key, -torch.inf)
    rank = torch.sort(key, dim=-1, descending=True, stable=True).indices
    kept = torch.zeros(n, H, T, dtype=torch.bool, device="cuda").scatter_(2, rank[..., :keep], True)
    # the n-th kept token from behind `keep` goes to the n-th free place below it
    free = ~kept[..., :keep]
    holes = torch.sort(free.to(torch.int8), dim=-1, descending=True, stable=True).indices
    movers = torch.sort(kept[..., keep:].to(torch.int8), dim=-1, descending=True, stable=True).indices + keep
    m = min(holes.shape[-1], movers.shape[-1])
    moved = (torch.arange(m, device="cuda") < free.sum(-1, keepdim=True)) & full
    source = torch.arange(keep, device="cuda").expand(n, H, keep).clone()
    source.scatter_(2, holes[..., :m], torch.where(moved, movers[..., :m], holes[..., :m]))
    # keys and values
    b, h, r = torch.nonzero(moved, as_tuple=True)
    dst, src = holes[b, h, r], movers[b, h, r]
    tables = st["tables"].long()
    db, ds, sb, ss = tables[b, dst // block], dst % block, tables[b, src // block], src % block
    k = st["k_cache"].view(-1, H, block // 16, D // 32, 4, 16, 8)
    k[db, h, ds // 16, :, :, ds % 16] = k[sb, h, ss // 16, :, :, ss % 16]
    v = st["v_cache"].view(-1, H, block // 16, D // 32, 4, 16, 2, 4)
    v[db, h, ds // 16, :, ds % 16 // 4, :, :, ds % 4] = v[sb, h, ss // 16, :, ss % 16 // 4, :, :, ss % 4]
    # the state's rows
    now = lens.clamp(max=keep)
    top = torch.where(full, keep, had[..., :1])
    t = min(keep, st["mass"].shape[-1])
    i = torch.arange(t, device="cuda")
    st["mass"][to, :, :t] = torch.where(i < now, mass.gather(2, source[..., :t]), st["mass"][to, :, :t])
    st["origin"][to, :, :t] = torch.where(i < torch.minimum(top, now), position.gather(2, source[..., :t]), st["origin"][to, :, :t])
    st["evicted"][to] = torch.where(full.view(n, 1), torch.stack([now.view(n), (st["lens"] + had[:, 0, 1] - keep)], 1).to(torch.int32),
                                    had.view(n, 2))
    st["lens_out"].copy_(now.view(n))
    return _evict_outputs(st)


@torch.inference_mode()
def run(state):
    if own:
        return _run_own(state)
    return {"decode": _plain_decode, "prompt": _plain_prompt, "evict": _plain_evict}[state["case"]["op"]](state)


# ---- in 64 bits, from the definition ------------------------------------------------------------------------------------
def _rows(cache, table, length, head, dim, transposed):
    """one sequence's cached rows [length, dim] of one head: element (t, d) of a tile at its offset"""
    block = cache.shape[2] * 16
    t = torch.arange(length, device=cache.device)
    d = torch.arange(dim, device=cache.device)
    slot = (t % 16).unsqueeze(1)
    if transposed:
        off = d // 32 * 512 + (slot // 4 * 16 + d % 16) * 8 + d // 16 % 2 * 4 + slot % 4
    else:
        off = d // 32 * 512 + (d // 8 % 4 * 16 + slot) * 8 + d % 8
    page = table[t // block].long().unsqueeze(1)
    return page, (t % block // 16).unsqueeze(1), off


@torch.inference_mode()
def exact(case, seed):
    st = prepare(case, seed)
    H, D, block = case["kv_heads"], case["dim"], case["block"]
    G = case["q_heads"] // H
    slots, to = st["slots"].tolist(), st["slots_out"].tolist()
    if case["op"] == "evict":
        return _exact_evict(case, st, slots, to)
    mass = st["mass"].double()
    out = torch.zeros(case["seqs"], case["q_heads"], D, dtype=torch.float64, device="cuda")
    for b, ctx in enumerate(st["ctx"]):
        new = 1 if case["op"] == "decode" else st["new"][b]
        seen_rows = 1 if case["op"] == "decode" else min(case["window"] or new, new)
        end = b + 1 if case["op"] == "decode" else st["cu_host"][b + 1]
        for h in range(H):
            k = st["k_cache"][:, h][_rows(st["k_cache"], st["tables"][b], ctx, h, D, False)].double()
            total = torch.zeros(ctx, dtype=torch.float64, device="cuda")
            for g in range(h * G, h * G + G):
                q = st["q"][end - seen_rows:end, g].double()
                s = (k @ q.T).T * st["scale"]
                s = s.masked_fill(torch.arange(ctx, device="cuda").unsqueeze(0) > torch.arange(ctx - seen_rows, ctx, device="cuda").unsqueeze(1),
                                  float("-inf"))
                p = torch.softmax(s, -1)
                total += p.sum(0)
                if case["op"] == "decode":
                    v = st["v_cache"][:, h][_rows(st["v_cache"], st["tables"][b], ctx, h, D, True)].double()
                    out[b, g] = (p @ v)[0]
            total[:ctx - new] += st["mass"][slots[b], h, :ctx - new].double()
            mass[to[b], h, :ctx] = total
    return {"out": out.view(case["seqs"], -1), "mass": mass} if case["op"] == "decode" else {"mass": mass}


def _exact_evict(case, st, slots, to):
    H, D, block, keep = case["kv_heads"], case["dim"], case["block"], case["keep"]
    mass_in, origin_in, had_in = st["mass"].cpu(), st["origin"].cpu(), st["evicted"].cpu()
    mass, origin, evicted = mass_in.clone(), origin_in.clone(), had_in.clone()
    lens = [min(c, keep) for c in st["ctx"]]
    for b, ctx in enumerate(st["ctx"]):
        kept_before, dropped = had_in[slots[b]].tolist()
        for h in range(H):
            m, pos = mass_in[slots[b], h, :ctx], torch.arange(ctx, dtype=torch.int32) + dropped
            pos[:kept_before] = origin_in[slots[b], h, :min(kept_before, ctx)]
            if ctx <= keep:
                mass[to[b], h, :ctx] = m
                origin[to[b], h, :min(kept_before, ctx)] = pos[:kept_before]
                continue
            value = m.double().clone()
            value[(pos < case["sinks"]) | (pos >= ctx + dropped - case["recent"])] = float("inf")
            # by mass downwards, slots upwards among equals
            order = sorted(range(ctx), key=(-value).tolist().__getitem__)[:keep]
            stay = set(order)
            src = list(range(keep))
            movers = sorted(x for x in order if x >= keep)
            for place, x in zip((x for x in range(keep) if x not in stay), movers):
                src[place] = x
            s = torch.tensor(src)
            mass[to[b], h, :keep], origin[to[b], h, :keep] = m[s], pos[s]
            if movers:
                dst = torch.nonzero(s >= keep)[:, 0]
                got = s[dst].cuda()
                for cache, transposed in ((st["k_cache"], False), (st["v_cache"], True)):
                    where = _rows(cache, st["tables"][b], ctx, h, D, transposed)
                    at = [x.expand(ctx, D) for x in where]
                    rows = cache[:, h][at[0][got], at[1][got], at[2][got]]
                    cache[:, h][at[0][dst.cuda()], at[1][dst.cuda()], at[2][dst.cuda()]] = rows
        evicted[to[b]] = torch.tensor([keep, dropped + ctx - keep] if ctx > keep else [kept_before, dropped])
    return {"lens": torch.tensor(lens, dtype=torch.int32).cuda(), "k_cache": st["k_cache"], "v_cache": st["v_cache"], "mass": mass.cuda().double(),
            "origin": origin.cuda(), "evicted": evicted.cuda()}
