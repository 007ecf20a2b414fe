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
