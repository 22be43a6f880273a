"""Attention mass and eviction, without a GPU: what the entry points refuse (before anything is launched), workspace sizes, and the
reference that the GPU tests hold the kernels to."""
import pytest
import torch

import attn_mass_ref as ref
from nanovllm import _C, ops

P = 1 << 20  # an address on 16 bytes that nothing reads: every call here is refused on the host


def decode_args(**kw):
    a = dict(q=P, q_stride=2048, k=P, v=P, blocks=8, table=P, table_stride=4, width=4, lens=P, mass=P, rows=2, len=64, slots=P, slots_out=P, out=P,
             ws=P, ws_bytes=1 << 30, batch=2, hq=16, hkv=8, d=128, block=16, scale=0.1, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), -1), (dict(k=None), -1), (dict(v=None), -1), (dict(table=None), -1), (dict(lens=None), -1), (dict(mass=None), -1),
    (dict(slots=None), -1), (dict(slots_out=None), -1), (dict(out=None), -1), (dict(ws=None), -1), (dict(q=P + 8), -1), (dict(k=P + 2), -1),
    (dict(out=P + 4), -1), (dict(ws=P + 4), -1), (dict(q_stride=2044), -1), (dict(batch=-1), -1), (dict(hq=15), -1), (dict(hkv=0), -1),
    (dict(blocks=0), -1), (dict(width=0), -1), (dict(table_stride=3), -1), (dict(rows=-1), -1), (dict(len=-1), -1), (dict(block=0), -1),
    (dict(d=96), -2), (dict(d=256), -2), (dict(hq=136), -2), (dict(block=24), -2), (dict(batch=70000), -2), (dict(width=1 << 27, table_stride=1 << 27), -2),
    (dict(ws_bytes=2 * 16 * 64 * 4 - 1), -3), (dict(batch=0), 0)])
def test_decode_refusals(kw, code):
    assert _C.lib.mi_paged_attn_decode_mass(*decode_args(**kw)) == code


def prompt_args(**kw):
    a = dict(q=P, q_stride=2048, tokens=20, k=P, blocks=8, table=P, table_stride=4, width=4, cu=P, lens=P, seqs=2, most=12, window=0, mass=P, rows=2,
             len=64, slots=P, slots_out=P, ws=P, ws_bytes=1 << 30, hq=16, hkv=8, d=128, block=16, scale=0.1, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), -1), (dict(k=None), -1), (dict(table=None), -1), (dict(cu=None), -1), (dict(lens=None), -1), (dict(mass=None), -1),
    (dict(slots=None), -1), (dict(slots_out=None), -1), (dict(ws=None), -1), (dict(q=P + 8), -1), (dict(k=P + 2), -1), (dict(ws=P + 8), -1),
    (dict(q_stride=4), -1), (dict(seqs=-1), -1), (dict(tokens=-1), -1), (dict(most=-1), -1), (dict(hq=15), -1), (dict(blocks=0), -1), (dict(width=0), -1),
    (dict(table_stride=3), -1), (dict(rows=-1), -1), (dict(block=-16), -1), (dict(window=-1), -1), (dict(d=96), -2), (dict(hq=136), -2),
    (dict(block=24), -2), (dict(seqs=70000), -2), (dict(tokens=1 << 30), -2), (dict(ws_bytes=1000), -3), (dict(seqs=0), 0)])
def test_prompt_refusals(kw, code):
    assert _C.lib.mi_prompt_attn_mass(*prompt_args(**kw)) == code


def evict_args(**kw):
    a = dict(k=P, v=P, blocks=8, table=P, table_stride=4, table_out=P, out_stride=4, width=4, lens=P, lens_out=P, mass=P, origin=P, evicted=P, rows=2,
             len=64, slots=P, slots_out=P, keep=32, sinks=4, recent=8, ws=P, ws_bytes=1 << 30, batch=2, hkv=8, d=128, block=16, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(k=None), -1), (dict(v=None), -1), (dict(table=None), -1), (dict(table_out=None), -1), (dict(lens=None), -1), (dict(lens_out=None), -1),
    (dict(mass=None), -1), (dict(origin=None), -1), (dict(evicted=None), -1), (dict(slots=None), -1), (dict(slots_out=None), -1), (dict(ws=None), -1),
    (dict(k=P + 4), -1), (dict(v=P + 8), -1), (dict(keep=0), -1), (dict(sinks=-1), -1), (dict(recent=-1), -1), (dict(sinks=30), -1),
    (dict(sinks=2 ** 31 - 1, recent=2 ** 31 - 1), -1), (dict(out_stride=1), -1), (dict(table_stride=3), -1), (dict(blocks=0), -1), (dict(rows=-1), -1),
    (dict(d=32), -2), (dict(block=8), -2), (dict(batch=70000), -2), (dict(ws_bytes=2 * 8 * (2 + 3 * 32) * 4 - 1), -3), (dict(batch=0), 0)])
def test_evict_refusals(kw, code):
    assert _C.lib.mi_kv_cache_evict(*evict_args(**kw)) == code


@pytest.mark.parametrize("off", [4, 1])
def test_evict_refuses_a_workspace_off_16_bytes(off):
    assert _C.lib.mi_kv_cache_evict(*evict_args(ws=P + off)) == -1


def test_workspace_sizes():
    lib = _C.lib
    # scores of every head and token that the table has room for; 300 sequences are not split
    assert lib.mi_paged_attn_decode_mass_workspace(300, 16, 8, 128, 16, 4) == 300 * 16 * 64 * 4
    assert lib.mi_paged_attn_decode_mass_workspace(1, 16, 8, 128, 16, 1000) > 16 * 16000 * 4
    assert lib.mi_paged_attn_decode_mass_workspace(0, 16, 8, 128, 16, 4) == 0
    assert lib.mi_prompt_attn_mass_workspace(0, 0, 1, 0, 16, 8, 128, 16, 4) == 0
    assert lib.mi_prompt_attn_mass_workspace(2, 20, 12, 0, 16, 8, 128, 16, 4) >= 8 * (20 * 2 // 32 + 2) * 32 * (256 + 4)
    # nothing can be evicted where the table has no more room than what is kept
    assert lib.mi_kv_cache_evict_workspace(2, 8, 64, 16, 4) == 2 * 8 * 2 * 4
    assert lib.mi_kv_cache_evict_workspace(2, 8, 63, 16, 4) == 2 * 8 * (2 + 3 * 63) * 4


def good():
    n, hq, hkv, d, block = 2, 16, 8, 128, 16
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)
    cache = lambda: torch.zeros(6, hkv, 1, 16 * d, dtype=torch.bfloat16)
    return dict(q=torch.zeros(n, hq, d, dtype=torch.bfloat16), k=cache(), v=cache(), bt=i32(n, 3), lens=i32(n), mass=torch.zeros(4, hkv, 48), slots=i32(n),
                origin=i32(4, hkv, 48), evicted=i32(4, 2), cu=i32(n + 1), hq=hq, hkv=hkv, block=block, keep=16, sinks=2, recent=4, window=0, out=None,
                slots_out=None, bt_out=None, lens_out=None, ws=None)


def call(which, a):
    if which == "decode":
        return ops.paged_attn_decode_mass(a["q"], a["k"], a["v"], a["bt"], a["lens"], a["mass"], a["slots"], a["hq"], a["hkv"], a["block"], 0.1,
                                          slots_out=a["slots_out"], out=a["out"], workspace=a["ws"])
    if which == "prompt":
        return ops.prompt_attn_mass(a["q"], a["k"], a["bt"], a["cu"], a["lens"], 1, a["mass"], a["slots"], a["hq"], a["hkv"], a["block"], 0.1,
                                    window=a["window"], slots_out=a["slots_out"], workspace=a["ws"])
    return ops.kv_cache_evict(a["k"], a["v"], a["bt"], a["lens"], a["mass"], a["origin"], a["evicted"], a["slots"], a["keep"], a["sinks"], a["recent"],
                              a["block"], block_tables_out=a["bt_out"], slots_out=a["slots_out"], context_lens_out=a["lens_out"], workspace=a["ws"])


WRONG = [
    ("decode prompt", "q", lambda t: t.float()), ("decode prompt", "q", lambda t: t[:, :15]), ("decode", "q", lambda t: t[:1]),
    ("decode prompt", "q", lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)), ("decode prompt", "q", lambda t: t.unsqueeze(0)),
    ("decode prompt", "q", lambda t: torch.zeros(2 * 2048 + 8, dtype=torch.bfloat16)[4:4 + 4096].view(2, 16, 128)),
    ("decode prompt", "q", lambda t: torch.zeros(2, 2052, dtype=torch.bfloat16)[:, :2048]),
    ("decode prompt evict", "k", lambda t: t.float()), ("decode prompt evict", "k", lambda t: t[:, :4]), ("decode prompt evict", "k", lambda t: t[:0]),
    ("decode prompt evict", "k", lambda t: t.view(6, 8, 2048)), ("decode evict", "v", lambda t: t[:5]), ("decode prompt", "block", lambda t: 32),
    ("decode prompt evict", "bt", lambda t: t.long()), ("decode prompt evict", "bt", lambda t: t[:1]), ("decode prompt evict", "bt", lambda t: t[:, :0]),
    ("decode prompt evict", "bt", lambda t: t[0]), ("decode prompt evict", "bt", lambda t: t.t().contiguous().t()),
    ("decode prompt evict", "lens", lambda t: t.long()), ("decode prompt evict", "lens", lambda t: torch.zeros(3, dtype=torch.int32)),
    ("decode prompt evict", "slots", lambda t: t.long()), ("decode prompt evict", "slots", lambda t: t[:1]),
    ("decode prompt evict", "slots_out", lambda t: torch.zeros(3, dtype=torch.int32)), ("decode prompt evict", "mass", lambda t: t.bfloat16()),
    ("decode prompt evict", "mass", lambda t: t[:, :4]), ("decode prompt evict", "mass", lambda t: t[..., :40]), ("decode prompt", "hq", lambda t: 12),
    ("decode prompt", "hkv", lambda t: 4), ("decode", "out", lambda t: torch.zeros(2, 2048)), ("decode", "out", lambda t: torch.zeros(2, 4096, dtype=torch.bfloat16)[:, ::2]),
    ("prompt", "cu", lambda t: t[:2]), ("prompt", "cu", lambda t: t.long()), ("prompt", "window", lambda t: -1),
    ("evict", "origin", lambda t: t.long()), ("evict", "origin", lambda t: t[:, :, :40].contiguous()), ("evict", "evicted", lambda t: t[:3]),
    ("evict", "evicted", lambda t: t.float()), ("evict", "keep", lambda t: 0), ("evict", "keep", lambda t: 5), ("evict", "sinks", lambda t: -1),
    ("evict", "recent", lambda t: -1), ("evict", "bt_out", lambda t: torch.zeros(1, 3, dtype=torch.int32)),
    ("evict", "lens_out", lambda t: torch.zeros(2, dtype=torch.int64)), ("evict", "lens_out", lambda t: torch.zeros(3, dtype=torch.int32)),
    ("decode prompt evict", "ws", lambda t: torch.zeros(8, dtype=torch.uint8)),
]


@pytest.mark.parametrize("case", range(len(WRONG)))
def test_wrappers_refuse(monkeypatch, case):
    """the wrappers' own checks (the device's aside), each alone wrong"""
    monkeypatch.setattr(ops, "_here", lambda *a: 0)
    which, key, change = WRONG[case]
    for w in which.split():
        a = good()
        a[key] = change(a[key])
        with pytest.raises(_C.MiError):
            call(w, a)


@pytest.mark.parametrize("which", ["decode", "prompt", "evict"])
def test_wrappers_refuse_caches_without_heads(monkeypatch, which):
    monkeypatch.setattr(ops, "_here", lambda *a: 0)
    a = good()
    a.update(k=a["k"][:, :0], v=a["v"][:, :0], mass=a["mass"][:, :0], origin=a["origin"][:, :0], hkv=0)
    with pytest.raises(_C.MiError):
        call(which, a)


def test_tensors_must_be_on_the_gpu():
    for w in ("decode", "prompt", "evict"):
        with pytest.raises(_C.MiError, match="only run on a HIP device"):
            call(w, good())


def test_reference_of_the_choice():
    mass = torch.tensor([5.0, 1.0, 1.0, float("nan"), 9.0, 1.0, 0.5, 7.0])
    pos = torch.arange(8, dtype=torch.int32)
    assert ref.choose(mass, pos, 8, 4, 0, 0) == [0, 1, 4, 7]
    assert ref.choose(mass, pos, 8, 4, 0, 1) == [0, 1, 4, 7]
    assert ref.choose(mass, pos, 8, 4, 2, 2) == [0, 1, 6, 7]
    assert ref.choose(mass, pos, 8, 8, 0, 0) == list(range(8))
    origin = torch.tensor([[0, 4, 2, 9, 9]], dtype=torch.int32)
    assert ref.position_of(origin, (3, 5), 5).tolist() == [[0, 4, 2, 8, 9]]
