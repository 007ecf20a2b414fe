"""The router's scores far from zero, as the loss's sums and the gradient show them."""
import numpy as np
import pytest
import torch

import k3moe

pytestmark = pytest.mark.gpu


def ladder():
    """A row a logit from -44 to 40 in steps of 1/32 and uneven ones, beside an expert at 0."""
    x = torch.cat([torch.arange(-44, 40, 1 / 32), torch.linspace(-43.9, 39.7, 1999)]).float()
    return torch.stack([x, torch.zeros_like(x)], 1)


def test_scores_keep_their_bits(dev):
    """Each row is a sequence of its own, so prob is the row's p = s / (s + 1/2 + 1e-20).

    Relative error of s in halves of a step (2^-24): the exponential instruction 4 (two units), the correction of its
    argument 1, ln 2 as one f32 2 (2.8e-9 * 44), 1 + e 1, the reciprocal 2: 10; of the sum z 10 + 1; its reciprocal 2, p's
    own rounding 1: 24."""
    S = ladder()
    T = len(S)
    seq = torch.arange(T + 1, dtype=torch.int32, device=dev)
    st = k3moe.balance_loss(S.to(dev), torch.zeros((T, 1), dtype=torch.int32, device=dev), 1.0, seq)
    s = 1 / (1 + torch.exp(-S.double()))
    p = s / (s.sum(1, keepdim=True) + 1e-20)
    off = (st.prob.double().cpu() / p - 1).abs()
    assert float(off.max()) <= 24 * 2 ** -24 * 1.001, (float(off.max()) * 2 ** 24, S[off[:, 0].argmax()].tolist())


def test_slopes_keep_their_bits(dev):
    """The weight term of one row and two picks, dwts = (1, 0): rs / den (1 - s_0 / den) s_0 (1 - s_0) and its opposite
    in the other expert's slope.

    1 - s_0 / den loses bits where s_1 is small beside s_0; with s_1 = 1/2 the quotient is below 2/3 and the difference
    at least a third, so its relative error is below 3 times that of the product 1 * s_0 / den (10 for s, 11 for den, 2 for its
    reciprocal, 2 products, in halves of a step) and its own rounding: 76.  rs / den 14, the slope e s s 7 + 10 + 10 + 2, two
    products: 121."""
    S = ladder()
    T = len(S)
    idx = torch.tensor([[0, 1]], dtype=torch.int32).repeat(T, 1)
    dw = torch.tensor([[1.0, 0.0]]).repeat(T, 1)
    rs = torch.ones(1, dtype=torch.bfloat16)
    got = k3moe.route_backward(S.to(dev), idx.to(dev), dwts=dw.to(dev), rs=rs.to(dev)).double().cpu()
    s = 1 / (1 + torch.exp(-S.double()))
    den = s.sum(1) + 1e-20
    slope = s / (1 + torch.exp(S.double()))
    want = torch.stack([(1 - s[:, 0] / den) * slope[:, 0] / den, -s[:, 0] / den * slope[:, 1] / den], 1)
    off = (got / want - 1).abs()
    assert float(off.max()) <= 121 * 2 ** -24, (float(off.max()) * 2 ** 24, S[off.max(1).values.argmax()].tolist())


def test_logits_past_the_ends(dev):
    """Scores of 1 and of 0, at the type's largest and lowest values, infinities and just inside the clamp."""
    low, high = [-88.5, -100.0, -1e30, -3.4028235e38, -float("inf")], [88.5, 100.0, 1e30, 3.4028235e38, float("inf")]
    S = torch.tensor([low + high, high + low, [0.0] * 10, low + low, high + high])
    T, E = S.shape
    seq = torch.arange(T + 1, dtype=torch.int32, device=dev)
    idx = torch.tensor([[0, 9]] * T, dtype=torch.int32, device=dev)
    st = k3moe.balance_loss(S.to(dev), idx, 1.0, seq)
    s = torch.sigmoid(S.double()).float().double()
    s[s < 2 ** -126] = 0
    p = s / (s.sum(1, keepdim=True) + 1e-20)
    got = st.prob.double().cpu()
    assert bool((got[p == 0] == 0).all())
    np.testing.assert_allclose(got.numpy(), p.numpy(), rtol=24 * 2 ** -24)
    dS = k3moe.route_backward(S.to(dev), idx, 1.0, st.counts, st.rows, seq=seq,
                              dwts=torch.ones((T, 2), device=dev), rs=torch.ones(1, dtype=torch.bfloat16, device=dev))
    assert bool((dS[[0, 1, 3, 4]] == 0).all()) and bool(torch.isfinite(dS).all())


@pytest.mark.parametrize("at", [0, 5, 39])
def test_a_logit_that_is_not_a_number(dev, at):
    """A NaN in a counted row reaches the row's sequence and the row's gradient, and nothing else."""
    S = torch.zeros((4, 40), device=dev)
    S[1, at] = float("nan")
    idx = torch.tensor([[0, 7]] * 4, dtype=torch.int32, device=dev)
    seq = torch.tensor([0, 2, 4], dtype=torch.int32, device=dev)
    st = k3moe.balance_loss(S, idx, 1.0, seq)
    assert bool(torch.isnan(st.prob[0]).all()) and bool(torch.isfinite(st.prob[1]).all()) and bool(torch.isnan(st.loss))
    dS = k3moe.route_backward(S, idx, 1.0, st.counts, st.rows, seq=seq)
    assert bool(torch.isnan(dS[1]).all()) and bool(torch.isfinite(dS[[0, 2, 3]]).all())
