"""FA2_B200_CHECK_STATUS=1 in the backward pass of flash_attention_packed."""

from __future__ import annotations

import pytest
import torch

from flash_attention_triton_b200 import _lib, flash_attention_packed

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("call", ["grad", "backward"])
def test_a_backward_pass_raises_where_asked(monkeypatch, call):
    """As that of the dense operator does.  The status is left by a forward whose cu_seqlens leave the rows, with nobody asking then."""
    monkeypatch.delenv("FA2_B200_CHECK_STATUS", raising=False)
    q = torch.randn(20, 2, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    good, bad = (torch.tensor([0, n], dtype=torch.int32, device="cuda") for n in (20, 21))
    o = flash_attention_packed(q, q, q, good)
    with torch.no_grad():
        flash_attention_packed(q, q, q, bad)
    monkeypatch.setenv("FA2_B200_CHECK_STATUS", "1")
    with pytest.raises(_lib.Fa2Error, match="fa2_packed_bwd .*status 0x80000"):
        torch.autograd.grad(o, [q], torch.ones_like(o), retain_graph=True) if call == "grad" else o.sum().backward()
    assert _lib.device_status() == 0  # read and cleared
    o = flash_attention_packed(q, q, q, good)
    (g,) = torch.autograd.grad(o, [q], torch.ones_like(o))
    assert g.isfinite().all()
