"""The balance loss over sequences long enough that a warp's sum of normalised scores passes through several stretches."""
import numpy as np
import pytest
import torch

import k3moe

pytestmark = pytest.mark.gpu


def test_sums_over_many_rows(dev):
    """64 million equal rows: every p is 1 / 13, a number whose f32 sum drifts one way.

    A score and the row's sum of them are exact here (0.5 and 6.5).  Relative error in halves of a step (2^-24): the
    reciprocal 2, at most 257 sums of a warp, 9 over the warps, 1 from double, and the join of the blocks' 297 partial rows,
    ten a warp of 32 and 32 warps: 42.  311 in all; the loss adds four roundings of its own and sums 13 terms: 328."""
    T, E = 64_000_000, 13
    S = torch.zeros((T, E), device=dev)
    idx = torch.zeros((T, 1), dtype=torch.int32, device=dev)
    st = k3moe.balance_loss(S, idx, 1.0)
    assert st.counts.tolist() == [[T] + [0] * (E - 1)] and st.rows.tolist() == [T]
    off = (st.prob.double() * E / T - 1).abs().max()
    assert float(off) <= 311 * 2 ** -24, float(off) * 2 ** 24
    assert abs(float(st.loss) - 1) <= 328 * 2 ** -24  # E c / (K n) * P / n = 13 * 1 / 13


@pytest.mark.parametrize("E,K", [(5, 2), (130, 3), (300, 4), (900, 8)])
def test_sequences_that_end_anywhere(dev, E, K):
    """Sequences from one row to more than a million, rows before and behind them, masked rows, against sums in double.

    Beside the sums (311 as above, 297 instead of 42 where one warp joins the partial rows) a score is within 32 halves of a
    step where |S| < 8, and so is the sum of them."""
    T = 3_000_000 if E <= 300 else 1_300_000
    g = torch.Generator(device=dev).manual_seed(E)
    S = torch.randn((T, E), generator=g, device=dev).clamp_(-8, 8)
    idx = torch.randint(0, E, (T, K), generator=g, device=dev, dtype=torch.int32)
    mask = (torch.rand(T, generator=g, device=dev) < 0.9).to(torch.uint8)
    cuts = [5, 6, 6, 4102, 40_000, 1_100_003, 1_100_004, 1_108_196, T - 3]
    seq = torch.tensor(cuts, dtype=torch.int32, device=dev)
    st = k3moe.balance_loss(S, idx, 1.0, seq, mask)
    loss = full = 0
    for b, (lo, hi) in enumerate(zip(cuts, cuts[1:])):
        prob, hits, n = torch.zeros(E, dtype=torch.float64, device=dev), torch.zeros(E, dtype=torch.int64, device=dev), 0
        for at in range(lo, hi, 100_000):
            to = min(hi, at + 100_000)
            on = mask[at:to] != 0
            s = torch.sigmoid(S[at:to][on].double())
            prob += (s / (s.sum(1, keepdim=True) + 1e-20)).sum(0)
            hits += torch.bincount(idx[at:to][on].reshape(-1).long(), minlength=E)
            n += int(on.sum())
        assert torch.equal(st.counts[b].long(), hits) and int(st.rows[b]) == n, b
        np.testing.assert_allclose(st.prob[b].double().cpu().numpy(), prob.cpu().numpy(), rtol=(311 + 255 + 64) * 2 ** -24)
        if n:
            full += 1
            loss += float((E * hits.double() / (K * n) * prob / n).sum())
    np.testing.assert_allclose(float(st.loss), loss / full, rtol=(311 + 255 + 64 + 50) * 2 ** -24)
    again = k3moe.balance_loss(S, idx, 1.0, seq, mask)
    assert torch.equal(st.prob, again.prob) and torch.equal(st.loss, again.loss)
