"""Attention mass and eviction: which rows of the state a call reads and writes - padded batches, rows that are not there, rows shorter than the
contexts, and the rows of a prompt that are not observed."""
import pytest
import torch

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
