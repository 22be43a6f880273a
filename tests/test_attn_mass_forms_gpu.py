"""Attention mass and eviction in every form that a launch takes, against the definition in 64 bits (tests/attn_mass_ref.py): each test names its form,
says what leads to it and, where the workspace's size tells, makes sure of it."""
import pytest

from test_attn_mass_gpu import run_decode, run_prompt
from test_kv_evict_gpu import run_evict

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from nanovllm import ops as _ops

    return _ops


def decode_room(ctxs, block, n_tables=2):
    return max(1, -(-max(ctxs) // block)) + n_tables


def is_split(B, geometry, block, width):
    """sequences' contexts over several workgroups: the workspace has more than the scores"""
    from nanovllm import _C

    hq, hkv, d = geometry
    return _C.lib.mi_paged_attn_decode_mass_workspace(B, hq, hkv, d, block, width) > B * hq * block * width * 4


# ---- decode
@pytest.mark.parametrize("geometry", [(28, 4, 128), (14, 2, 64), (7, 1, 128)])
def test_decode_not_split_with_seven_query_heads_per_kv_head(ops, geometry):
    n = -(-256 // geometry[1])
    ctxs = [1 + 37 * i % 300 for i in range(n)]
    assert not is_split(n, geometry, 16, decode_room(ctxs, 16))
    run_decode(ops, geometry, 16, ctxs, 41)


@pytest.mark.parametrize("geometry", [(5, 1, 128), (16, 1, 64)])
def test_decode_not_split_with_many_chunks_of_a_wave(ops, geometry):
    """eight waves deal a context's 32-token chunks: from none to eleven for a wave, odd numbers and even ones"""
    long = [2600, 2304, 2049, 2048, 1800, 1793, 1537, 1536, 1281, 1025, 1024, 1023, 800, 769, 768, 767, 544, 513, 512, 257, 256, 255]
    ctxs = long + [3 * i % 64 for i in range(260 - len(long))]
    assert not is_split(len(ctxs), geometry, 32, decode_room(ctxs, 32))
    run_decode(ops, geometry, 32, ctxs, 42)


@pytest.mark.parametrize("geometry,n", [((3, 1, 64), 255), ((16, 8, 128), 31)])
def test_decode_split_with_many_chunks_of_a_wave_and_tokens_of_a_joining_thread(ops, geometry, n):
    """just below 256 units: four splits, and the join's workgroups have 8192 tokens (255 units) and 8448 (248) at a time"""
    ctxs = [20000, 9000, 8449, 8193, 8192] if geometry[1] == 1 else [17000, 8449]
    ctxs += [5 * i % 90 for i in range(n - len(ctxs))]
    assert is_split(n, geometry, 64, decode_room(ctxs, 64))
    run_decode(ops, geometry, 64, ctxs, 43)


# ---- prompt
def prompt_parts(geometry, block, news, pasts, window):
    """parts of the keys that the row sums are split into, from the workspace: rows, their log-sums, and a pair a part and row"""
    from nanovllm import _C

    hq, hkv, d = geometry
    G, B = hq // hkv, len(news)
    width = max(1, max(-(-(n + p) // block) for n, p in zip(news, pasts))) + 2
    rows = min(window, max(news)) if window else max(news)
    tiles = B * -(-rows * G // 32) if window else sum(news) * G // 32 + B
    a_row = _C.lib.mi_prompt_attn_mass_workspace(B, sum(news), max(news), window, hq, hkv, d, block, width) // (hkv * tiles * 32)
    return max(1, (a_row - 2 * d - 4) // 8)


def key_blocks(geometry, block, news, pasts):
    width = max(1, max(-(-(n + p) // block) for n, p in zip(news, pasts))) + 2
    return len(news) * geometry[1] * -(-width * block // 256)


COLUMNS = [  # rows and cached tokens of four sequences on 8 kv heads: 256 blocks of 256 keys and more
    ([333, 40, 2100, 1], [1700, 2000, 0, 2099]),
    ([2000, 3, 0, 700], [0, 1000, 40, 1]),
]


@pytest.mark.parametrize("geometry", [(32, 8, 64), (8, 8, 64), (64, 8, 128), (16, 8, 128)])
@pytest.mark.parametrize("window", [1, 19, 64])
@pytest.mark.parametrize("sizes", COLUMNS)
def test_prompt_column_sums_of_four_waves_keys(ops, geometry, window, sizes):
    """few rows (below 2048 of a kv head) and 256 blocks of 256 keys or more: each wave has 64 keys and all rows"""
    assert key_blocks(geometry, 16, *sizes) >= 256
    run_prompt(ops, geometry, 16, *sizes, window, 51 + window)


@pytest.mark.parametrize("geometry", [(32, 8, 64), (16, 8, 128)])
def test_prompt_column_sums_of_four_waves_keys_all_rows(ops, geometry):
    sizes = ([70, 40, 5, 1], [2000, 1400, 2095, 600])
    for block in (48, 256):
        assert key_blocks(geometry, block, *sizes) >= 256
        run_prompt(ops, geometry, block, *sizes, 0, 52)


@pytest.mark.parametrize("geometry", [(32, 8, 64), (16, 8, 128)])
def test_prompt_column_sums_of_four_waves_keys_and_pages_that_are_not_there(ops, geometry):
    sizes = ([333, 40, 2100, 1], [1700, 2000, 0, 2099])
    gone = [(0, 0, -1), (0, 17, 10 ** 6), (0, 126, -3), (1, 37, -1), (2, 130, -1), (2, 131, -1), (2, 64, 10 ** 6), (3, 131, -1)]
    run_prompt(ops, geometry, 16, *sizes, 64, 53, bad_pages=gone)


@pytest.mark.parametrize("window", [992, 993])
def test_prompt_column_sums_on_both_sides_of_the_rule_on_rows(ops, window):
    """16 heads on 8: 1984 rows of a kv head are 31 groups of 64, 1986 are 32"""
    sizes = ([2100, 3, 1, 40], [0, 100, 1, 0])
    assert key_blocks((16, 8, 128), 16, *sizes) >= 256
    run_prompt(ops, (16, 8, 128), 16, *sizes, window, 54)


@pytest.mark.parametrize("ctx", [1760, 1761, 2016])
def test_prompt_column_sums_on_both_sides_of_the_rule_on_keys(ops, ctx):
    sizes = ([40, 33, 200, 64], [ctx - 40, 0, 0, 1000])
    assert key_blocks((16, 8, 128), 16, *sizes) == (224 if ctx == 1760 else 256)
    run_prompt(ops, (16, 8, 128), 16, *sizes, 33, 55)


@pytest.mark.parametrize("geometry,news,pasts,window,parts", [
    ((7, 1, 128), [5], [9000], 0, 17), ((8, 8, 64), [3], [20000], 0, 39), ((3, 1, 64), [40], [33500], 33, 64), ((16, 8, 128), [20, 7], [5000, 60], 0, 10)])
def test_prompt_rows_joined_from_more_than_eight_parts(ops, geometry, news, pasts, window, parts):
    """few rows and many keys: the join takes eight parts at a time"""
    assert prompt_parts(geometry, 64, news, pasts, window) == parts
    run_prompt(ops, geometry, 64, news, pasts, window, 56)


# ---- eviction: keys in LDS for tables of up to 8192 tokens, in more of it for contexts of up to 32768, read again for longer ones
@pytest.mark.parametrize("masses", ["spread", "ties", "any"])
@pytest.mark.parametrize("own_rows", [False, True])
def test_eviction_from_8193_to_32768_tokens(ops, masses, own_rows):
    run_evict(ops, 2, 64, 16, [8193, 20001, 300, 8192], 1500, 4, 100, 61, masses=masses, own_rows=own_rows)
    run_evict(ops, 1, 128, 256, [32768, 32767, 16385, 24577], 700, 0, 64, 62, masses=masses, own_rows=own_rows)


@pytest.mark.parametrize("own_rows", [False, True])
def test_eviction_from_8193_to_32768_tokens_after_one_that_kept_more_than_8192(ops, own_rows):
    run_evict(ops, 1, 64, 64, [20001, 9000, 32768], 12000, 4, 5000, 63, own_rows=own_rows)


def test_eviction_from_8193_to_32768_tokens_of_equal_masses_and_into_other_pages(ops):
    run_evict(ops, 1, 64, 64, [9000, 17000], 8500, 0, 0, 64, masses="equal", earlier=False)
    run_evict(ops, 2, 128, 64, [9000, 17000, 20], 1000, 4, 64, 65, other_pages=True)


@pytest.mark.parametrize("masses", ["spread", "ties"])
def test_eviction_in_a_table_of_8192_tokens(ops, masses):
    run_evict(ops, 2, 64, 16, [8192, 8191, 4097], 1000, 4, 64, 66, masses=masses)


@pytest.mark.parametrize("ctx", [32768, 32769])
def test_eviction_on_both_sides_of_the_keys_in_lds(ops, ctx):
    run_evict(ops, 1, 64, 48, [ctx, 200], 600, 4, 64, 67, masses="ties")
