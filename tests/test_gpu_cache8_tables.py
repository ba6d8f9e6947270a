"""block_table_extend's free list after a shortage: how blocks are given back and
how sequences that went short go on. And calls of nothing."""

import pytest
import torch

import fusedtok_amd as ft
from tests.test_gpu_cache8 import DEV, i32

pytestmark = pytest.mark.gpu

PAGE, WIDTH, BLOCKS = 4, 5, 7


def give_back(free, n_free, ids):
    """As the documentation has it; the new n_free."""
    ids = ids[ids >= 0]
    at = n_free.clamp(min=0)
    free[at + torch.arange(len(ids), device=DEV)] = ids
    return at + len(ids)


def spent():
    """Three sequences of 9 tokens, three blocks each, of seven: the last one
    gets one."""
    table = torch.zeros(3, WIDTH, dtype=torch.int32, device=DEV)
    free = torch.arange(BLOCKS, dtype=torch.int32, device=DEV)
    slots, _, off, lens, n_free = ft.block_table_extend(
        table, i32([0, 0, 0]), i32([9, 9, 9]), free, i32([BLOCKS]), PAGE, 27)
    assert n_free.tolist() == [-2] and lens.tolist() == [9, 9, 9]
    assert table[:, :3].tolist() == [[6, 5, 4], [3, 2, 1], [0, -1, -1]]
    assert (slots >= 0).tolist() == [True] * 22 + [False] * 5
    return table, free, n_free, lens


def held(table, lens):
    """The blocks of each row in use."""
    return [table[i, : -(-n // PAGE)].tolist() for i, n in enumerate(lens.tolist())]


def whole(table, lens, free, n_free):
    """Every block is held once or free once."""
    left = free[: max(int(n_free), 0)].tolist()
    return sorted(sum(held(table, lens), left)) == list(range(BLOCKS))


def test_blocks_given_back_after_a_shortage():
    """The first sequence ends; the third starts over."""
    table, free, n_free, lens = spent()
    n_free = give_back(free, n_free, table[0, :3])
    n_free = give_back(free, n_free, table[2, :3])
    assert n_free.tolist() == [4]
    lens = i32([0, 9, 0])
    assert whole(table, lens, free, n_free)
    slots, _, _, lens, n_free = ft.block_table_extend(table, lens, i32([0, 1, 9]), free, n_free,
                                                      PAGE, 10)
    assert n_free.tolist() == [1] and (slots >= 0).all()
    assert whole(table, lens, free, n_free)


def test_a_short_call_again():
    """The second sequence ends; the third's call is taken back and made again."""
    table, free, n_free, _ = spent()
    n_free = give_back(free, n_free, table[2, :3])   # what it got in that call
    n_free = give_back(free, n_free, table[1, :3])
    lens = i32([9, 0, 0])
    assert whole(table, lens, free, n_free)
    slots, _, _, lens, n_free = ft.block_table_extend(table, lens, i32([3, 0, 9]), free, n_free,
                                                      PAGE, 12)
    assert n_free.tolist() == [1] and (slots >= 0).all()
    assert whole(table, lens, free, n_free)


def test_a_negative_count_is_no_debt():
    """With nothing given back a further call hands out nothing; a count put to
    what the list holds is all that the next one looks at."""
    table, free, n_free, lens = spent()
    slots, _, _, lens, n_free = ft.block_table_extend(table, lens, i32([4, 0, 0]), free, n_free,
                                                      PAGE, 4)
    assert n_free.tolist() == [-3] and (slots >= 0).tolist() == [True] * 3 + [False]
    assert table[0, 3] == -1
    n_free = give_back(free, n_free, table[1, :3])
    assert n_free.tolist() == [3]
    slots, _, _, lens, n_free = ft.block_table_extend(table, i32([12, 0, 9]), i32([1, 8, 0]),
                                                      free, n_free, PAGE, 9)
    assert n_free.tolist() == [0] and (slots >= 0).all()


@pytest.mark.parametrize("b,width,tokens", [(0, 4, 0), (0, 0, 0), (2, 0, 0), (2, 0, 5)])
def test_extend_of_nothing(b, width, tokens):
    """No sequence, no table column, no token: the outputs are written whole."""
    table = torch.zeros(b, width, dtype=torch.int32, device=DEV)
    slots, pos, off, lens, n_free = ft.block_table_extend(
        table, i32([0] * b), i32([2] * b), i32([]), i32([3]), 16, tokens)
    fresh = [0, 1, 0, 1][: 2 * b] + [0] * tokens
    assert slots.tolist() == [-1] * tokens and pos.tolist() == fresh[:tokens]
    assert off.tolist() == [0, 2, 4][: b + 1] and lens.tolist() == [0] * b
    assert n_free.tolist() == [3]
