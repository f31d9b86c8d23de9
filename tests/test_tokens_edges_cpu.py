"""Edges of the token operators that need no GPU: the terms of float weights, refusals, the counts of a cache."""
import math

import pytest
import torch

from vision_assist_amd import _lib
from vision_assist_amd.tokens import _terms


def test_terms_of_any_weight():
    big, top = torch.finfo(torch.float32).max, torch.finfo(torch.bfloat16).max
    edge = float.fromhex("0x1.ffp127")  # the first value whose nearest bf16 is an infinity
    under = torch.nextafter(torch.tensor(edge), torch.tensor(0.0)).item()
    w = torch.tensor([[0.0, 1.0, -1.7, 3e-20, big, -big, edge, under, top, -under, 1e38, math.pi, -2.0 ** -100, 7.0, 65535.0, -0.1]])
    t = _terms(w)
    assert t.dtype == torch.bfloat16 and t.isfinite().all()
    assert torch.equal(t.double().sum(0), w.double())
    w[0, :3] = torch.tensor([math.inf, -math.inf, math.nan])
    t = _terms(w).float()
    assert t[:, 0, 0].tolist() == [1, 0, math.inf] and t[:, 0, 1].tolist() == [-1, 0, -math.inf] and t[:, 0, 2].isnan().any()
    assert torch.equal(t[:, :, 3:].double().sum(0), w[:, 3:].double())


def test_attend_refuses_to_lose_a_gradient():
    from vision_assist_amd.tokens import attend
    for i in range(3):
        a = [torch.zeros(2, 3, 4, 64), torch.zeros(2, 10, 2, 64), torch.zeros(2, 10, 2, 64)]
        a[i].requires_grad_()
        with pytest.raises(_lib.VaError, match="gradient"):
            attend(*a)
        with torch.no_grad(), pytest.raises(_lib.VaError, match="on the GPU"):
            attend(*a)
