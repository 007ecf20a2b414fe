"""Outputs that the entries allocate, where torch does more than allocate."""
import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

import k3moe

pytestmark = pytest.mark.gpu


@pytest.fixture
def routed(dev):
    idx = torch.randint(0, 4, (60, 2), generator=torch.Generator().manual_seed(3)).to(torch.int32).to(dev)
    t = k3moe.route_tables(idx, 4)
    real = torch.zeros(t.cap_rows, dtype=torch.bool, device=dev)
    real[t.exp2perm[t.exp2perm >= 0].long()] = True
    return t, real


@pytest.mark.parametrize("cols", [64, 50])
def test_deterministic_mode_fills_what_is_not_written(dev, routed, cols):
    """Padding rows hold what torch.empty gives in that mode: the type's largest integer, NaN."""
    t, real = routed
    x = torch.randn(60, cols, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).to(dev)
    w, sw = k3moe.quant_int8(torch.randn(4 * 32, cols, generator=torch.Generator().manual_seed(5)).to(dev))
    plain = k3moe.grouped_gemm_int8(*k3moe.quant_int8_permute(x, t), w, sw, t, 4)
    was = torch.are_deterministic_algorithms_enabled()
    torch.use_deterministic_algorithms(True)
    try:
        q, s = k3moe.quant_int8_permute(x, t)
        y = k3moe.grouped_gemm_int8(q, s, w, sw, t, 4)
    finally:
        torch.use_deterministic_algorithms(was)
    assert q.stride() == (-(-cols // 16) * 16, 1)
    assert bool((q[~real] == 127).all()) and bool(torch.isnan(s[~real]).all()) and bool(torch.isnan(y[~real]).all())
    assert torch.equal(y[real], plain[real])


class Seen(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, kinds, args=(), kwargs=None):
        self.names.append(str(func))
        return func(*args, **(kwargs or {}))


def test_dispatch_modes_see_the_outputs(dev):
    x = torch.randn(5, 50, device=dev)
    q, s = k3moe.quant_int8(x)
    w = torch.zeros((3, 64), dtype=torch.int8, device=dev)[:, :50]
    with Seen() as seen:
        q2, s2 = k3moe.quant_int8(x)
        k3moe.gemm_int8(q2, s2, w, torch.ones(3, device=dev)[:3])
        st = k3moe.balance_loss(x, torch.zeros((5, 1), dtype=torch.int32, device=dev), 1.0)
    made = [n for n in seen.names if n.startswith("aten.empty")]
    assert "aten.empty_strided.default" in made and made.count("aten.empty.memory_format") >= 1 + 1 + 5, made
    assert torch.equal(q, q2) and torch.equal(s, s2) and st.loss.numel() == 1
