"""Codes of act(gate) * up (k3moe_act_quant_int8) where a code's rounding or the gate's own accuracy decides."""
import numpy as np
import pytest
import torch

import k3moe

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,cols", [(2000, 512), (1300, 900), (700, 2048), (400, 4100), (150, 16000), (90, 20001)])
def test_gated_codes_round_the_exact_quotient(dev, rows, cols):
    """Gates from 32 on: exp(-g) is below 2^-46, so the sigmoid is 1 and the gate's value the product g u, exact in f32 (8
    mantissa bits each).  Quotients lie as near to a half as 2^-24 of themselves; the codes are those of exact integers, to
    the bit."""
    g = torch.Generator().manual_seed(rows)
    gate = torch.randint(32, 128, (rows, cols), generator=g)
    up = torch.randint(128, 256, (rows, cols), generator=g) * (torch.randint(0, 2, (rows, cols), generator=g) * 2 - 1)
    gu = torch.cat([gate.float(), up.float() / 128], 1).to(torch.bfloat16)
    assert torch.equal(gu[:, :cols].long(), gate) and torch.equal((gu[:, cols:].float() * 128).long(), up)
    h = (gate * up).numpy()                          # 128 times the gate's value
    amax = np.abs(h).max(1, keepdims=True)
    k, left = np.divmod(254 * np.abs(h) + amax, 2 * amax)  # floor(127 |h| / amax + 1/2)
    want = np.sign(h) * (k - ((left == 0) & (k % 2 == 1)))
    q, s = k3moe.act_quant_int8(gu.to(dev))
    wrong = q.cpu().numpy() != want
    assert not wrong.any(), f"{int(wrong.sum())} of {wrong.size} codes"
    assert np.array_equal(s.cpu().numpy(), (amax[:, 0] / 128).astype(np.float32) / np.float32(127))


@pytest.mark.parametrize("act,up,steps", [(k3moe.ACT_SWIGLU, 1.0, 10), (k3moe.ACT_SITU, 20.0, 22)])
@pytest.mark.parametrize("cols", [1, 8])
def test_gates_far_from_zero_keep_their_bits(dev, act, up, steps, cols):
    """Every bf16 gate of magnitude 2^-20 to 80, a row each: the row's scale is |act(gate) up| / 127.

    Relative error in halves of an f32 step (2^-24): the exponential instruction 4 (two units), the correction of its
    argument 1, 1 + e 1, the reciprocal 2, the products with gate and up 1 (up = 1 is exact), the scale's division 1: 10.
    SiTU: sigmoid 8, two tanh 4 each (two units), 0.04 and its product 2, three products 3, the division 1: 22."""
    bits = torch.arange(0x3580, 0x42A1, dtype=torch.int32)
    gate = torch.cat([bits, bits | 0x8000]).to(torch.int16).view(torch.bfloat16)
    gu = torch.cat([gate[:, None].repeat(1, cols), torch.full((len(gate), cols), up, dtype=torch.bfloat16)], 1)
    q, s = k3moe.act_quant_int8(gu.to(dev), act)
    g = gate.double()
    h = g * torch.sigmoid(g) * up if act == k3moe.ACT_SWIGLU else \
        4 * torch.tanh(g / 4) * torch.sigmoid(g) * 25 * torch.tanh(torch.tensor(up / 25).double())
    off = (s.double().cpu() * 127 / h.abs() - 1).abs()
    assert float(off.max()) <= steps * 2 ** -24 * 1.001, (float(off.max()) * 2 ** 24, float(g[off.argmax()]))
    assert torch.equal(q.cpu().long(), (127 * torch.sign(g)).long()[:, None].expand(-1, cols))


def test_gates_past_the_ends(dev):
    """Gates whose sigmoid is 1 or below every normal f32, and what is not a number."""
    gate = torch.tensor([88.0, 1e4, 3e38, -90.0, -1e4, -3e38, float("inf"), -float("inf"), float("nan")])
    for act in (k3moe.ACT_SWIGLU, k3moe.ACT_SITU):
        gu = torch.stack([gate, torch.full_like(gate, 0.5)], 1).to(torch.bfloat16)
        q, s = k3moe.act_quant_int8(gu.to(dev), act)
        s = s.cpu().double() * 127
        g = gu[:3, 0].double()
        want = g / 2 if act == k3moe.ACT_SWIGLU else 4 * 25 * torch.tanh(torch.full_like(g, 0.02))
        assert bool(((s[:3] / want - 1).abs() <= 22 * 2 ** -24).all()) and bool((s[3:6] == 0).all())
        assert q.cpu()[:, 0].tolist()[:6] == [127, 127, 127, 0, 0, 0]
        if act == k3moe.ACT_SWIGLU:
            assert bool(torch.isnan(s[6:]).all()) and q.cpu()[6:].abs().max() == 0
        else:  # tanh bounds both factors: only the NaN is one
            assert abs(float(s[6]) / float(want[0]) - 1) <= 22 * 2 ** -24 and float(s[7]) == 0 and bool(torch.isnan(s[8]))
