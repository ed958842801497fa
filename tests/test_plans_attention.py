"""Work items of the attention kernel for prompts, by the kernel's own search run on the CPU: every token of every sequence is
worked on exactly once for each key head, in whatever order blocks are handed to the CTAs."""
import ctypes as C

import numpy as np
import pytest


@pytest.fixture(scope="module")
def lib():
    import tacker_b200
    from tacker_b200 import _build

    _build.build_library()
    return tacker_b200.lib()


def _p(a):
    return a.ctypes.data_as(C.POINTER(C.c_int))


def blocks_of(q_len, kv_heads, tile_tokens):
    """What the launcher starts: enough for every packing of that many rows into that many sequences."""
    return (sum(q_len) // (2 * tile_tokens) + len(q_len)) * kv_heads


def cover(lib, q_len, kv_heads, tile_tokens, order, ctas):
    q = np.array(q_len, dtype=np.int32)
    order = np.array(order, dtype=np.int32)
    out = np.zeros((kv_heads, max(1, sum(q_len))), dtype=np.int32)
    assert lib.tk_plan_attention(_p(q), len(q), kv_heads, tile_tokens, _p(order), len(order), ctas, _p(out)) == 0
    return out[:, :sum(q_len)]


LENGTHS = {
    "one": [1],
    "mixed": [300, 1, 0, 127, 128, 129, 256, 257, 2500],
    "many short": [1 + i % 7 for i in range(200)],
    "empty windows": [0] * 40 + [700, 3] + [0] * 90 + [1, 260] + [0] * 33,
}


@pytest.mark.parametrize("name", LENGTHS)
@pytest.mark.parametrize("kv_heads,tile_tokens", [(1, 128), (2, 32), (3, 18), (8, 1)])
@pytest.mark.parametrize("ctas", [1, 2, 7, 148])
def test_each_token_once_in_any_order_of_blocks(lib, name, kv_heads, tile_tokens, ctas):
    q_len = LENGTHS[name]
    n = blocks_of(q_len, kv_heads, tile_tokens)
    rng = np.random.default_rng(n + ctas)
    up = np.arange(n)
    for order in (up, up[::-1], np.roll(up, n // 2), rng.permutation(n), rng.permutation(n)):
        assert bool((cover(lib, q_len, kv_heads, tile_tokens, order, ctas) == 1).all()), (name, list(order[:10]))


def test_a_block_behind_the_last_item_does_not_end_the_search(lib):
    """Two items and eight blocks: a CTA that is handed blocks without work first still does the work it is handed next."""
    q_len = [200] + [0] * 6
    assert blocks_of(q_len, 1, 64) == 8
    for order in ([7, 1, 0, 2, 3, 4, 5, 6], [7, 6, 5, 4, 3, 2, 1, 0], [2, 0, 7, 1, 3, 4, 5, 6]):
        assert bool((cover(lib, q_len, 1, 64, order, 1) == 1).all()), order


def test_refusals(lib):
    a = np.zeros(4, dtype=np.int32)
    for change in (dict(q=None), dict(n=0), dict(kv=0), dict(tile=0), dict(order=None), dict(blocks=0), dict(ctas=0), dict(cover=None)):
        g = {**dict(q=_p(a), n=1, kv=1, tile=1, order=_p(a), blocks=1, ctas=1, cover=_p(a)), **change}
        assert lib.tk_plan_attention(*g.values()) == -1, change
    a[0] = -1
    assert lib.tk_plan_attention(_p(a), 1, 1, 1, _p(a), 1, 1, _p(a)) == -1
