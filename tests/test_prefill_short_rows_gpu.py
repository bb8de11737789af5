"""GPU: prefill of many prompts of one key tile each on pools whose work items are single heads.  A CTA then works through
several items with one key tile in a row, in each of which only one of its two issuers has anything to do."""

import pytest
import torch

import workloads as wl
from fpkv import _lib
from test_prefill_gpu import compare_live_rows, oracle_prefill, run_product

pytestmark = pytest.mark.gpu
T = wl.image_text_tokens


@pytest.mark.parametrize("Hq,Hkv,D,dtype", [(16, 16, 128, torch.bfloat16), (12, 4, 64, torch.float16)])
@pytest.mark.parametrize("seed", [1, 2])
def test_one_key_tile_items_one_after_the_other(Hq, Hkv, D, dtype, seed):
    lens = [1 + (37 * i + seed) % 128 for i in range(70)] + [200, 128, 129]
    case = wl.make_prefill_case(700 + seed, [T(0, 0, n) for n in lens], Hq=Hq, Hkv=Hkv, D=D, P=128, dtype=dtype)
    assert len(lens) * Hq > 4 * 148                       # several items a CTA
    c, slots, bidx, ipos, mask, out, lse = run_product(case, 80 + len(lens), len(lens) + 2, dtype=dtype, kernel=_lib.PREFILL_TC)
    c.check_status()
    compare_live_rows(case, out, lse, *oracle_prefill(case, slots, dtype), f"{Hq}/{Hkv} heads")
