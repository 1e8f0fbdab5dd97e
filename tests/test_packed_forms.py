"""The forms in which the dK / dV kernel of packed sequences is built, and the call at which its two rules meet."""

from __future__ import annotations

import re
import shutil
import subprocess

import pytest
import torch

from flash_attention_triton_b200 import _lib, flash_attention_packed
from packed_helpers import exact_packed


@pytest.mark.skipif("shutil.which('nm') is None")
def test_no_form_is_built_that_no_call_reaches():
    """Clusters are for launches of few CTAs, 64-row steps for those of many; head dims up to 64 have the latter at all."""
    names = subprocess.run(["nm", "-C", str(_lib.LIB_PATH)], capture_output=True, text=True, check=True).stdout
    forms = {tuple(map(int, m)) for m in re.findall(r"packed_dkdv_kernel<(\d+), \w+, \d+, (\d+), (\d+)>", names)}
    assert forms == {(d, 128, s) for d in (32, 64, 128) for s in (1, 2, 4)} | {(d, 64, 1) for d in (32, 64)}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [32, 64])
@pytest.mark.parametrize("more", [-128, 0, 128])
def test_as_many_key_tiles_as_multiprocessors(more, d, dtype):
    """One sequence of 4 key heads: the last that clusters of two take, and those beside it."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    rows = (sms // 4 - 1) * 128 + more  # rows / 128 + 1 tiles at most
    g = torch.Generator().manual_seed(1)
    q, k, v, do = (torch.randn(rows, h, d, generator=g).to(dtype).cuda() for h in (8, 4, 4, 8))
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    o = flash_attention_packed(*leaves, torch.tensor([0, rows], dtype=torch.int32, device="cuda"))
    got = dict(zip(("o", "dq", "dk", "dv"), (o.detach(), *torch.autograd.grad(o, leaves, do))))
    for name, (value, tolerance) in exact_packed(*(t.detach() for t in leaves), [rows], do).items():
        assert ((got[name].double() - value).abs() <= tolerance).all(), name
    assert _lib.device_status() == 0
