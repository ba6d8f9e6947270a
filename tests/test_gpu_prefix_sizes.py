"""GPU test of attention_decode_paged_prefix's workspace: the size it asks for is
the one that the restated split (test_prefix_plan) needs, and a call leaves
what lies before and behind a workspace of that size alone, whatever it held."""

import numpy as np
import pytest
import torch

import fusedtok_amd as ft
from tests.test_gpu_prefix import Case, i32
from tests.test_prefix_plan import Plan

pytestmark = pytest.mark.gpu

CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def up256(x):
    return -(-x // 256) * 256


def asked(dtype, b, hq, hkv, groups, page, pwidth, twidth, d):
    return ft._fusedtok.attention_decode_paged_prefix_workspace(CODE[dtype], b, hq, hkv, groups,
                                                                page, pwidth, twidth, d)


@pytest.mark.parametrize("dtype", list(CODE))
@pytest.mark.parametrize("b,hq,hkv,groups,d", [(1, 1, 1, 0, 64), (64, 32, 8, 1, 128), (7, 20, 4, 2, 96),
                                               (3000, 2, 1, 1096, 8), (5, 130, 1, 9, 256),
                                               (40, 33, 3, 40, 20)])
def test_size(b, hq, hkv, groups, d, dtype):
    segs = 2 * torch.cuda.get_device_properties(0).multi_processor_count
    p = Plan([0] * (groups + 1), [0] * groups, [0] * b, hq // hkv, hkv, segs, "half")
    rows = 16 * p.granules
    # a row's maximum and sum, its D sums, 64 bytes a sequence for the second launch
    want = up256(rows * 8) + up256(rows * d * 4) + up256(64 * b) + 256
    assert asked(dtype, b, hq, hkv, groups, 16, 5, 7, d) == want
    assert asked(dtype, 0, hq, hkv, groups, 16, 5, 7, d) == 0


@pytest.mark.parametrize("dtype", list(CODE))
@pytest.mark.parametrize("hq,hkv,d,plens,sizes,lens", [
    (8, 2, 64, [130], [3], [0, 5, 70]),
    (16, 1, 128, [700, 0, 64], [1, 4, 3], [9, 0, 64, 65, 1, 300, 2, 0]),
    (33, 1, 20, [200], [5], [1, 2, 3, 4, 5]),
    (8, 8, 256, [90, 90], [1, 1], [64, 64]),
    (32, 8, 128, [4000], [40], [(7 * i) % 90 for i in range(40)]),
    (5, 1, 96, [3000] * 6, [3] * 6, [(11 * i) % 400 for i in range(18)])])
def test_nothing_beside_the_workspace(hq, hkv, d, plens, sizes, lens, dtype):
    c = Case(hq, hq, hkv, d, 16, plens, sizes, lens, dtype)
    b, groups, wide = len(lens), len(plens), 1 << 16
    table, own = i32(c.ptable), i32(c.table)
    size = asked(dtype, b, hq, hkv, groups, 16, table.shape[1], own.shape[1], d)
    ints = [i32(c.plens), i32(c.offsets), i32(c.lens)]
    for fill in (0xff, 0x7f):   # NaN, and 3.4e38 or so, in what the workspace held
        room = torch.full((size + 2 * wide,), fill, dtype=torch.uint8, device="cuda")
        out = torch.empty_like(c.q)
        ft._fusedtok.attention_decode_paged_prefix_launch(
            c.q.data_ptr(), CODE[dtype], c.kp.data_ptr(), c.vp.data_ptr(), table.data_ptr(),
            ints[0].data_ptr(), ints[1].data_ptr(), own.data_ptr(), ints[2].data_ptr(),
            out.data_ptr(), room.data_ptr() + wide, size, b, hq, hkv, groups, c.kp.shape[0], 16,
            table.shape[1], own.shape[1], d, torch.cuda.current_stream().cuda_stream)
        assert (room[:wide] == fill).all() and (room[wide + size:] == fill).all()
        c.check(out)
        assert torch.equal(out, c.run())
