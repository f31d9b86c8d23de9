"""Edges of the token operators: what enters a product as it is, values that are not finite, far ends of a stream's
life, and each form that a product's size chooses.  Plain implementations in float64; tolerances as in test_gpu_tokens.py
(half a step of a rounding relative to the value: bf16 2^-8, float 2^-24), with what is added derived beside each test."""
import math

import pytest
import torch

from tests.test_gpu_tokens import DT, U, attend_ref, rnd

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ attend
@pytest.mark.parametrize("B,S,Hq,Hk,D,slots,kv", [(3, 1, 8, 2, 128, 2500, 2500), (2, 2, 4, 4, 64, 700, 1900), (1, 4, 8, 1, 80, 333, 333),
                                                  (5, 1, 32, 1, 32, 60, 60)])
def test_attend_few_rows_round_once(B, S, Hq, Hk, D, slots, kv):
    """bf16, up to 32 rows of a key head: the probabilities enter the second product as two bf16 terms, each within 2^-8 of
    what it stands for, so 2^-16 of a probability is left out; the rest is the float form's bound and the output's rounding."""
    from vision_assist_amd.tokens import attend
    g = torch.Generator().manual_seed(slots)
    t = torch.bfloat16
    q, k, v = rnd(g, B, S, Hq, D, dtype=t), rnd(g, B, slots, Hk, D, dtype=t), rnd(g, B, slots, Hk, D, dtype=t)
    kl = [kv - 7 * b for b in range(B)]
    got = attend(q.cuda(), k.cuda(), v.cuda(), kv_len=torch.tensor(kl, dtype=torch.int32, device="cuda")).double().cpu()
    args = (D ** -0.5, 1, 0, 0, [S] * B, kl)
    want, tol = attend_ref(q.float(), k, v, *args)
    size, _ = attend_ref(q.float(), k, v.abs(), *args)
    tol = tol + 2.0 ** -16 * size + U[t] * want.abs()
    assert float(((got - want).abs() / tol).max()) <= 1
