"""The append's rows of 4 values a lane (head dims that are no multiple of 8,
tensors aligned to 4 values only) in calls of many rows: the listed runs and the
windows of a block, by waves and by workgroups, with rows out of order, slots
twice, and blocks whose scales grow."""

import numpy as np
import pytest
import torch

import fusedtok_amd as ft
from tests import cache8_refs as refs
from tests.test_gpu_cache8 import DEV, dev, i32, pools, seq_slots

pytestmark = pytest.mark.gpu

CUS = 256


def reached(rows, hkv, page, d):
    """(how runs are found, who has one) for 4 values a lane."""
    how = "rows" if 2 * rows * hkv <= 16 * CUS else "listed" if rows <= 1024 else "windows"
    return how, "wave" if page * (d // 4) <= 256 else "workgroup"


@pytest.mark.parametrize("off", [0, 4])
@pytest.mark.parametrize("rows,how", [(900, "listed"), (3000, "windows")])
@pytest.mark.parametrize("page,d,who,dtype", [
    (16, 36, "wave", torch.bfloat16), (5, 100, "wave", torch.float32),
    (16, 100, "workgroup", torch.float16), (64, 36, "workgroup", torch.float32),
    (16, 64, "wave", torch.float16), (16, 128, "workgroup", torch.bfloat16),
    (100, 12, "workgroup", torch.bfloat16)])
def test_append_4_values_a_lane(page, d, who, dtype, rows, how, off):
    if d % 8 == 0 and off == 0:
        off = 12   # 8 bytes' alignment: these dims have 8 values a lane otherwise
    hkv = 8
    assert reached(rows, hkv, page, d) == (how, who)
    assert torch.cuda.get_device_properties(0).multi_processor_count == CUS
    rng = np.random.default_rng(rows + page + d + off)
    fresh = [rows // 2, rows // 3, 1, 1]
    fresh.append(rows - sum(fresh))
    lens = [0, 3, page - 1, page, page // 2 + 1]
    nb = sum(-(-(n + a) // page) for n, a in zip(lens, fresh)) + 2
    cache = pools(rng, nb, hkv, page, d)
    slots = np.array(seq_slots(rng, nb, page, lens, fresh))
    for a in range(7, rows - 8, 61):   # runs out of order, and a slot twice
        run = slice(a, a + 1 + np.argmin(np.append(slots[a:] // page == slots[a] // page, False)[1:]))
        slots[run] = rng.permutation(slots[run])
        if run.stop - a > 2:
            slots[a + 1] = slots[a]
    start = 1 + next(i for i in range(rows // 5, rows) if slots[i + 1] // page != slots[i] // page)
    slots[start:start + 2] = -1   # the first rows of a run (of one block: still one run)
    size = rng.choice([1e-3, 1, 8], (rows, 1, 1))   # some blocks grow, some do not
    got = [dev(x) for x in cache]
    new = []
    for _ in range(2):
        x = torch.as_tensor((rng.standard_normal((rows, hkv, d)) * size).astype(np.float32))
        x = x.to(dtype)
        buf = torch.zeros(x.numel() + 16, dtype=dtype, device=DEV)
        new.append(buf[off:off + x.numel()].view(x.shape))
        new[-1].copy_(x)
    ft.kv_append_paged_int8(*got, *new, i32(slots))
    for i in range(2):
        codes, scales = refs.append(cache[i], cache[2 + i], new[i].float().cpu().numpy(), slots)
        np.testing.assert_array_equal(got[2 + i].cpu().numpy(), scales)
        np.testing.assert_array_equal(got[i].cpu().numpy(), codes)
        assert (scales > cache[2 + i]).any()


def test_append_of_more_rows_than_a_grid():
    """Blocks of one row: a wave for each of 2^25 rows of K and of V, 2^24
    workgroups, the last of which a second launch has. Every block starts over,
    so its scale is max |x| / 127 and its codes rint(x * (1 / scale)), in
    float32 with divisions rounded once (by way of 64 bits)."""
    rows, d = 2 ** 25, 4
    gen = torch.Generator(device=DEV).manual_seed(3)
    k, v = (torch.randn(rows, 1, d, generator=gen, device=DEV, dtype=torch.float16)
            for _ in range(2))
    kp, vp = (torch.full((rows, 1, 1, d), 99, dtype=torch.int8, device=DEV) for _ in range(2))
    ks, vs = (torch.full((rows, 1), 7.0, device=DEV) for _ in range(2))
    slots = torch.randperm(rows, generator=gen, device=DEV).int()
    ft.kv_append_paged_int8(kp, vp, ks, vs, k, v, slots)
    for pool, scales, new in ((kp, ks, k), (vp, vs, v)):
        x = new[:, 0].float()
        want = (x.abs().amax(1).double() / 127).float().clamp(min=2.0 ** -120)
        codes = torch.round(x * (1 / want.double()).float()[:, None]).clamp(-127, 127)
        assert torch.equal(scales[slots.long(), 0], want)
        assert torch.equal(pool[slots.long(), 0, 0], codes.to(torch.int8))
