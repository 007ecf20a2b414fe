"""The router's training operators (k3moe_balance_loss, k3moe_route_backward) against their definitions in 64 bits.

Tolerances, from the kernels' arithmetic.  A score s is off by at most 16 * 2^-23 relative where |S| <= 10 (__expf
2 + 1.173 |S| units in the last place, the division 2, one product); a sum of up to 1024 of them, and one of a row's
normalised scores over at most 32 rows a lane and 300 partial rows, add at most 400 * 2^-24 in all; every term is
positive.  So prob, and the loss (a few more products), are within RTOL = 3e-5 relative, and a gradient within RTOL of
the sum of its terms' magnitudes, plus half a step of the output's type."""
import numpy as np
import pytest
import torch

import k3moe

pytestmark = pytest.mark.gpu
RTOL = 3e-5


def definition(S, idx, alpha, seq, mask, dloss=1.0, dwts=None, rs=None, balance=True):
    """(stats, dS, the sum of the gradient's terms' magnitudes), plain loops over sequences in float64 on the CPU."""
    S = S.double().cpu()
    idx = idx.cpu().long()
    T, E = S.shape
    K = idx.shape[1]
    seq = [0, T] if seq is None else seq.cpu().tolist()
    on = torch.ones(T, dtype=torch.bool) if mask is None else mask.cpu() != 0
    B = len(seq) - 1
    sig, down = torch.sigmoid(S), torch.sigmoid(-S)
    z = sig.sum(1, keepdim=True) + 1e-20
    counts, prob, rows = torch.zeros(B, E, dtype=torch.int64), torch.zeros(B, E, dtype=torch.float64), []
    groups = []
    for b in range(B):
        at = [t for t in range(seq[b], seq[b + 1]) if on[t]]
        groups.append(at)
        rows.append(len(at))
        for t in at:
            for e in idx[t].tolist():
                if 0 <= e < E:
                    counts[b, e] += 1
        if at:
            prob[b] = (sig[at] / z[at]).sum(0)
    full = max(1, sum(n > 0 for n in rows))
    loss = 0.0
    dS = torch.zeros(T, E, dtype=torch.float64)
    size = torch.zeros(T, E, dtype=torch.float64)
    for b, at in enumerate(groups):
        n = rows[b]
        if n == 0:
            continue
        f = E * counts[b].double() / (K * n)
        loss += float((f * prob[b] / n).sum()) * alpha / full
        if balance:
            p = sig[at] / z[at]
            g = f * alpha * dloss / (n * full)
            m = (p * g).sum(1, keepdim=True)
            dS[at] = (g - m) * p * down[at]
            size[at] = (g + m).abs() * p * down[at]
    if dwts is not None:
        dwts, r = dwts.double().cpu(), float(rs.float().item())
        for t in range(T):
            ks = [(k, e) for k, e in enumerate(idx[t].tolist()) if 0 <= e < E]
            den = sum(sig[t, e] for _, e in ks) + 1e-20
            mean = sum(dwts[t, k] * sig[t, e] for k, e in ks) / den
            mag = sum(abs(dwts[t, k]) * sig[t, e] for k, e in ks) / den
            for k, e in ks:
                slope = sig[t, e] * down[t, e] * r / den
                dS[t, e] += slope * (dwts[t, k] - mean)
                size[t, e] += abs(slope) * (abs(dwts[t, k]) + mag)
    return {"loss": loss, "counts": counts, "prob": prob, "rows": torch.tensor(rows)}, dS, size


def make(dev, T, E, K, B, masked, seed, pad=0, wide=0):
    """Inputs; `pad` rows before the first and behind the last sequence, `wide` more logits a row in memory."""
    g = torch.Generator().manual_seed(seed)
    S = (torch.randn(T, E + wide, generator=g) * 1.5).to(dev)[:, :E]
    idx = torch.stack([torch.randperm(E, generator=g)[:K] for _ in range(T)]).to(torch.int32) if T else \
        torch.zeros(0, K, dtype=torch.int32)
    lo, hi = min(pad, T), max(T - pad, min(pad, T))
    cuts = torch.sort(torch.randint(lo, hi + 1, (max(B - 1, 0),), generator=g)).values
    seq = torch.cat([torch.tensor([lo]), cuts, torch.tensor([hi])]).to(torch.int32).to(dev) if B else None
    mask = (torch.rand(T, generator=g) < 0.7).to(torch.uint8).to(dev) if masked else None
    return S, idx.to(dev), seq, mask


# (T, E, K, B (0: no offsets), masked, pad, wide)
CASES = [(1, 1, 1, 0, False, 0, 0), (1, 896, 8, 1, False, 0, 0), (7, 61, 4, 3, True, 0, 0), (64, 8, 8, 1, True, 0, 0),
         (300, 897, 8, 5, True, 3, 0), (257, 256, 16, 40, False, 0, 0), (513, 1024, 16, 2, False, 0, 0),
         (333, 129, 2, 9, True, 10, 3), (700, 128, 3, 300, False, 5, 4), (0, 16, 2, 0, False, 0, 0),
         (5, 16, 2, 4, False, 5, 0), (2500, 40, 5, 17, True, 1, 0), (3000, 60, 4, 1500, True, 0, 0),
         (256, 900, 8, 64, False, 0, 0),
         (100, 70, 4, 100, True, 2, 0), (257, 100, 2, 1, False, 0, 0), (9000, 20, 2, 3, True, 7, 0)]


@pytest.mark.parametrize("T,E,K,B,masked,pad,wide", CASES)
def test_loss_counts_and_sums(dev, T, E, K, B, masked, pad, wide):
    S, idx, seq, mask = make(dev, T, E, K, B, masked, T + E, pad, wide)
    got = k3moe.balance_loss(S, idx, 0.37, seq, mask)
    ref, _, _ = definition(S, idx, 0.37, seq, mask)
    assert torch.equal(got.counts.cpu().long(), ref["counts"])
    assert torch.equal(got.rows.cpu().long(), ref["rows"])
    np.testing.assert_allclose(got.prob.cpu().double().numpy(), ref["prob"].numpy(), rtol=RTOL, atol=0)
    np.testing.assert_allclose(float(got.loss), ref["loss"], rtol=RTOL, atol=0)
    again = k3moe.balance_loss(S, idx, 0.37, seq, mask)
    assert torch.equal(got.prob, again.prob) and torch.equal(got.loss, again.loss)


@pytest.mark.parametrize("T,E,K,B,masked,pad,wide", CASES)
@pytest.mark.parametrize("terms", ["balance", "weights", "both"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradient(dev, T, E, K, B, masked, pad, wide, terms, dtype):
    S, idx, seq, mask = make(dev, T, E, K, B, masked, T + E + 1, pad, wide)
    g = torch.Generator().manual_seed(3)
    dwts = torch.randn(T, K, generator=g).to(dev) if terms != "balance" else None
    rs = torch.tensor([2.5], dtype=torch.bfloat16, device=dev) if terms != "balance" else None
    dloss = torch.tensor([1.75], device=dev)
    st = k3moe.balance_loss(S, idx, 50.0, seq, mask)
    bal = terms != "weights"
    out = torch.full((T + 1, E + wide), 7.0, dtype=dtype, device=dev)
    k3moe.route_backward(S, idx, 50.0, st.counts if bal else None, st.rows if bal else None, dloss, dwts, rs, seq, mask,
                         out=out[:T, :E])
    _, ref, size = definition(S, idx, 50.0, seq, mask, 1.75, dwts, rs, bal)
    got = out[:T, :E].double().cpu()
    tol = RTOL * size + (torch.finfo(dtype).eps / 2 * ref.abs() if dtype == torch.bfloat16 else 0)
    tol = tol * (1 + 2 ** -7) + 1e-37
    bad = (got - ref).abs() > tol
    assert not bad.any(), (float(((got - ref).abs() / tol).max()), int(bad.sum()))
    assert bool((out[T] == 7).all()) and bool((out[:, E:] == 7).all())  # nothing beside the gradient is written


def test_gradient_against_differences(dev):
    """The definition's gradient against central differences of its loss and of the weights, in 64 bits; the kernel
    holds to the same numbers (test_gradient)."""
    T, E, K = 9, 12, 3
    S, idx, seq, mask = make("cpu", T, E, K, 2, True, 5)
    g = torch.Generator().manual_seed(11)
    dwts, rs = torch.randn(T, K, generator=g), torch.tensor([2.5], dtype=torch.bfloat16)
    _, grad, _ = definition(S, idx, 3.0, seq, mask, 0.7, dwts, rs)

    def value(X):
        st, _, _ = definition(X, idx, 3.0, seq, mask)
        s = torch.sigmoid(X).gather(1, idx.long())
        return 0.7 * st["loss"] + float((dwts.double() * 2.5 * s / (s.sum(1, keepdim=True) + 1e-20)).sum())

    h = 1e-5
    for t in range(T):
        for e in range(E):
            X = S.double().clone()
            X[t, e] += h
            up = value(X)
            X[t, e] -= 2 * h
            num = (up - value(X)) / (2 * h)
            # truncation h^2/6 times a third derivative of order 1, and cancellation 2^-53 * value / h
            assert abs(num - float(grad[t, e])) < 1e-8, (t, e)
    st = k3moe.balance_loss(S.to(dev), idx.to(dev), 3.0, seq.to(dev), mask.to(dev))
    got = k3moe.route_backward(S.to(dev), idx.to(dev), 3.0, st.counts, st.rows, torch.tensor([0.7], device=dev),
                               dwts.to(dev), rs.to(dev), seq.to(dev), mask.to(dev))
    np.testing.assert_allclose(got.cpu().double().numpy(), grad.numpy(), rtol=0, atol=RTOL * 10)


def test_rows_that_do_not_count_are_not_read(dev):
    """NaN and infinite logits in masked rows and outside the sequences leave everything else as it was."""
    S, idx, seq, mask = make(dev, 90, 70, 4, 3, True, 8, pad=6)
    clean = k3moe.balance_loss(S, idx, 1.0, seq, mask)
    grad = k3moe.route_backward(S, idx, 1.0, clean.counts, clean.rows, seq=seq, mask=mask)
    out = mask == 0
    out[:6] = True
    out[-6:] = True
    X = S.clone()
    X[out] = float("nan")
    X[out, 0] = float("inf")
    got = k3moe.balance_loss(X, idx, 1.0, seq, mask)
    for a, b in zip((got.loss, got.counts, got.prob, got.rows), (clean.loss, clean.counts, clean.prob, clean.rows)):
        assert torch.equal(a, b)
    dirty = k3moe.route_backward(X, idx, 1.0, got.counts, got.rows, seq=seq, mask=mask)
    assert torch.equal(dirty, grad) and bool((dirty[out] == 0).all())


def test_a_mask_that_leaves_nothing(dev):
    S, idx, seq, _ = make(dev, 40, 33, 2, 4, False, 9)
    mask = torch.zeros(40, dtype=torch.bool, device=dev)
    st = k3moe.balance_loss(S, idx, 1.0, seq, mask)
    assert float(st.loss) == 0 and int(st.counts.abs().sum()) == 0 and float(st.prob.abs().sum()) == 0
    assert bool((k3moe.route_backward(S, idx, 1.0, st.counts, st.rows, seq=seq, mask=mask) == 0).all())


def test_extreme_logits(dev):
    """Experts switched off by -inf, a row with none left, saturated and far logits: finite, and by the definition."""
    E = 40
    S = torch.zeros(6, E)
    S[0, 5:] = -float("inf")
    S[1] = -float("inf")
    S[2, 3] = float("inf")
    S[3] = torch.linspace(-9, 9, E)
    S[4] = 1e30
    S[5] = -1e30
    idx = torch.arange(6 * 3, dtype=torch.int32).reshape(6, 3) % E
    g = torch.Generator().manual_seed(1)
    dw, rs = torch.randn(6, 3, generator=g), torch.tensor([1.0], dtype=torch.bfloat16)
    ref, grad, size = definition(S, idx, 2.0, None, None, dwts=dw, rs=rs)
    st = k3moe.balance_loss(S.to(dev), idx.to(dev), 2.0)
    np.testing.assert_allclose(st.prob.cpu().double().numpy(), ref["prob"].numpy(), rtol=RTOL, atol=0)
    got = k3moe.route_backward(S.to(dev), idx.to(dev), 2.0, st.counts, st.rows, None, dw.to(dev), rs.to(dev))
    got = got.cpu().double()
    assert bool(torch.isfinite(got).all())
    assert bool(((got - grad).abs() <= RTOL * size + 1e-37).all())


def test_picks_outside_the_experts_and_named_twice(dev):
    S, idx, seq, mask = make(dev, 50, 30, 4, 2, False, 12)
    idx[3] = torch.tensor([-1, 5, 30, 1000], dtype=torch.int32)
    idx[4] = torch.tensor([-7, -1, -1, -2 ** 31], dtype=torch.int32)
    idx[5] = torch.tensor([9, 9, 2, 9], dtype=torch.int32)
    g = torch.Generator().manual_seed(2)
    dw, rs = torch.randn(50, 4, generator=g).to(dev), torch.tensor([2.0], dtype=torch.bfloat16, device=dev)
    ref, grad, size = definition(S, idx, 1.0, seq, mask, dwts=dw, rs=rs)
    st = k3moe.balance_loss(S, idx, 1.0, seq, mask)
    assert torch.equal(st.counts.cpu().long(), ref["counts"])
    got = k3moe.route_backward(S, idx, 1.0, st.counts, st.rows, None, dw, rs, seq, mask).cpu().double()
    assert bool(((got - grad).abs() <= RTOL * size + 1e-37).all())


def test_offsets_that_go_down_stay_in_bounds(dev):
    """Offsets outside their contract: whatever is counted, nothing outside the outputs is written."""
    S, idx, _, _ = make(dev, 100, 20, 2, 1, False, 4)
    for seq in ([0, 90, 10, 100], [50, 20, 5], [-40, 30, 700], [2 ** 31 - 1, -2 ** 31]):
        q = torch.tensor(seq, dtype=torch.int32, device=dev)
        st = k3moe.balance_loss(S, idx, 1.0, q)
        k3moe.route_backward(S, idx, 1.0, st.counts, st.rows, seq=q)
    torch.cuda.synchronize()


def test_offsets_past_32_bits(dev):
    """2.5e9 logits (20 GB with their gradient): a last sequence behind 2^31 elements as by itself."""
    T, E, n = 2_500_000, 1000, 300
    S = torch.zeros((T, E), device=dev)
    g = torch.Generator(device=dev).manual_seed(4)
    S[-n:] = torch.randn(n, E, generator=g, device=dev)
    idx = torch.randint(0, E, (T, 2), generator=g, device=dev, dtype=torch.int32)
    seq = torch.tensor([0, T - n, T], dtype=torch.int32, device=dev)
    st = k3moe.balance_loss(S, idx, 1.0, seq)
    tail, tail_idx = S[-n:].contiguous(), idx[-n:].contiguous()
    one = k3moe.balance_loss(tail, tail_idx, 1.0)
    assert torch.equal(st.counts[1:], one.counts) and st.rows.tolist() == [T - n, n]
    np.testing.assert_allclose(st.prob[1].cpu().numpy(), one.prob[0].cpu().numpy(), rtol=RTOL)
    np.testing.assert_allclose(st.prob[0].cpu().numpy(), (T - n) / E, rtol=RTOL)
    dS = k3moe.route_backward(S, idx, 1.0, st.counts, st.rows, seq=seq)
    half = k3moe.route_backward(tail, tail_idx, 0.5, one.counts, one.rows)  # the loss is a mean over two sequences
    assert torch.equal(dS[-n:], half)


def test_captured_and_on_another_stream(dev):
    S, idx, seq, mask = make(dev, 400, 96, 4, 6, True, 21)
    st = k3moe.balance_loss(S, idx, 1.0, seq, mask)
    dS = k3moe.route_backward(S, idx, 1.0, st.counts, st.rows, seq=seq, mask=mask)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    s2 = k3moe.balance_loss(S, idx, 1.0, seq, mask, stream=side)
    side.synchronize()
    assert torch.equal(s2.loss, st.loss) and torch.equal(s2.counts, st.counts)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s3 = k3moe.balance_loss(S, idx, 1.0, seq, mask)
        d3 = k3moe.route_backward(S, idx, 1.0, s3.counts, s3.rows, seq=seq, mask=mask)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(s3.loss, st.loss) and torch.equal(s3.prob, st.prob) and torch.equal(d3, dS)


def test_the_router_trains(dev):
    """Router product -> top-k -> loss and weights -> dS -> router weight: the gradient of the whole against torch's
    own differentiation of the definition in 64 bits (products and picks taken from the device)."""
    T, H, E, K = 200, 256, 64, 4
    g = torch.Generator(device=dev).manual_seed(6)
    x = torch.randn(T, H, generator=g, device=dev).to(torch.bfloat16)
    W = (torch.randn(E, H, generator=g, device=dev) / 16).to(torch.bfloat16)
    bias = torch.rand(E, generator=g, device=dev) * 0.1
    rs = torch.tensor([2.5], dtype=torch.bfloat16, device=dev)
    seq = torch.tensor([0, 60, 61, 200], dtype=torch.int32, device=dev)
    S = k3moe.router_gemm(x, W)
    idx, wts = k3moe.route_topk(S, bias, rs, K)
    st = k3moe.balance_loss(S, idx, 0.5, seq)
    dwts = torch.randn(T, K, generator=g, device=dev)
    dS = k3moe.route_backward(S, idx, 0.5, st.counts, st.rows, None, dwts, rs, seq)
    S64 = S.double().requires_grad_()
    sig = torch.sigmoid(S64)
    p = sig / (sig.sum(1, keepdim=True) + 1e-20)
    sk = sig.gather(1, idx.long())
    w64 = 2.5 * sk / (sk.sum(1, keepdim=True) + 1e-20)
    np.testing.assert_allclose(wts.double().cpu().numpy(), w64.detach().cpu().numpy(), rtol=1e-5)
    loss = 0
    for a, b in ((0, 60), (60, 61), (61, 200)):
        c = torch.bincount(idx[a:b].reshape(-1).long(), minlength=E).double()
        loss = loss + (E * c / (K * (b - a)) * p[a:b].mean(0)).sum() * 0.5 / 3
    np.testing.assert_allclose(float(st.loss), float(loss.detach()), rtol=RTOL)
    (loss + (dwts.double() * w64).sum()).backward()
    # terms of a row's gradient are at most rs (|g| + mean |g|) / 4 / den, here below 10
    np.testing.assert_allclose(dS.double().cpu().numpy(), S64.grad.cpu().numpy(), rtol=0, atol=10 * RTOL)
