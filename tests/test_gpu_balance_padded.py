"""The balance loss over batches whose sequences differ much in length: offsets padded with empty sequences to a fixed
number, one long sequence among short ones."""
import numpy as np
import pytest
import torch

import k3moe

pytestmark = pytest.mark.gpu


def short(lo, hi, n):
    return [lo + (hi - lo) * i // n for i in range(1, n + 1)]


CASES = {
    "one of 256": (2048, 256, 4, [0] + [2048] * 256),
    "one of 64, behind the empty ones": (8192, 896, 8, [0] * 64 + [8192]),
    "half and 63 short": (8192, 896, 8, [0, 4096] + short(4096, 8192, 63)),
    "two long ones of 300": (3000, 61, 2, [3] + [3] * 100 + [1400] + short(1400, 1500, 98) + [2990] + [2990] * 99),
    "long ones side by side in 40": (6000, 40, 3, [0, 1500, 3000, 4500, 6000] + [6000] * 36),
    "more groups than a turn takes": (4096, 896, 8, short(-2, 1022, 500) + [1022] * 10 + [4090, 4096, 4096]),
}


@pytest.mark.parametrize("name", CASES)
@pytest.mark.parametrize("masked", [False, True])
def test_uneven_sequences(dev, name, masked):
    """Against sums in double.  Relative error of prob in halves of an f32 step (2^-24): p 24 (test_gpu_balance_scores.py),
    a warp's rows 5, the warps 9, at most 257 partial rows by eight warps 33 + 8: 80.  The loss: its terms' products 4, their
    sums over a warp, its turns, the warps and the blocks 36: 120."""
    T, E, K, cuts = CASES[name]
    cuts = [max(0, c) for c in cuts]
    assert cuts == sorted(cuts) and cuts[-1] <= T
    g = torch.Generator(device=dev).manual_seed(T + E)
    S = (torch.randn((T, E), generator=g, device=dev) * 1.5).clamp_(-8, 8)
    idx = torch.topk(torch.rand((T, E), generator=g, device=dev), K, dim=1).indices.to(torch.int32)
    mask = torch.rand(T, generator=g, device=dev) < 0.8 if masked else torch.ones(T, dtype=torch.bool, device=dev)
    seq = torch.tensor(cuts, dtype=torch.int32, device=dev)
    st = k3moe.balance_loss(S, idx, 1.0, seq, mask if masked else None)
    B = len(cuts) - 1
    at = torch.arange(T, device=dev)
    of = torch.searchsorted(seq.long(), at, right=True) - 1
    on = mask & (at >= cuts[0]) & (at < cuts[-1])
    s = torch.sigmoid(S.double())
    p = s / (s.sum(1, keepdim=True) + 1e-20)
    prob = torch.zeros((B, E), dtype=torch.float64, device=dev).index_add_(0, of[on], p[on])
    hits = torch.zeros((T, E), dtype=torch.float64, device=dev).scatter_(1, idx.long(), 1.0)
    counts = torch.zeros((B, E), dtype=torch.float64, device=dev).index_add_(0, of[on], hits[on])
    rows = torch.bincount(of[on], minlength=B)
    n = rows.clamp(min=1).double()[:, None]
    loss = float((E * counts / (K * n) * prob / n).sum() / (rows > 0).sum())
    assert torch.equal(st.counts.long(), counts.long()) and torch.equal(st.rows.long(), rows)
    np.testing.assert_allclose(st.prob.double().cpu().numpy(), prob.cpu().numpy(), rtol=80 * 2 ** -24)
    np.testing.assert_allclose(float(st.loss), loss, rtol=120 * 2 ** -24)
    again = k3moe.balance_loss(S, idx, 1.0, seq, mask if masked else None)
    assert torch.equal(st.prob, again.prob) and torch.equal(st.loss, again.loss)
