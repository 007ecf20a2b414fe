"""Refusals of the router's training entries and of the 8-bit integer products that need more than one argument's own
check: each is raised before any device work."""
import dataclasses

import pytest
import torch

import k3moe


def test_tables_of_other_tiles():
    """Tables of 64-row tiles (route_tables takes any) would leave most real rows without codes: refused."""
    n = 3
    words = [torch.zeros(n, dtype=torch.int32) for _ in range(3)]
    t = k3moe.Tables(counts=words[0], cta_batch=words[1], cta_limit=words[2], meta=torch.zeros(4, dtype=torch.int32),
                     route_map=torch.zeros(64 * n, dtype=torch.int32), exp2perm=torch.zeros((5, 1), dtype=torch.int32),
                     max_ctas=n, cap_rows=64 * n)
    with pytest.raises(k3moe.K3MoeError, match="128-row tiles"):
        k3moe.act_quant_int8(torch.zeros((64 * n, 32), dtype=torch.bfloat16), tables=t)


def test_counts_without_alpha():
    """A balance term whose weight was left out is refused, not taken as zero."""
    S, idx = torch.zeros(4, 8), torch.zeros((4, 2), dtype=torch.int32)
    c, n = torch.zeros((1, 8), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(k3moe.K3MoeError, match="alpha"):
        k3moe.route_backward(S, idx, counts=c, rows=n)
    for alpha in (0.0, 0.5):  # given: the host tensor is what is refused
        with pytest.raises(k3moe.K3MoeError, match="CUDA tensor"):
            k3moe.route_backward(S, idx, alpha, c, n)


def test_logits_that_autograd_follows():
    """The loss carries no graph: added to another one it would drop out of the backward pass without a word."""
    S, idx = torch.zeros(4, 8, requires_grad=True), torch.zeros((4, 2), dtype=torch.int32)
    with pytest.raises(k3moe.K3MoeError, match="detach"):
        k3moe.balance_loss(S, idx, 1.0)
    with pytest.raises(k3moe.K3MoeError, match="CUDA tensor"):  # the host tensor is what is refused
        k3moe.balance_loss(S.detach(), idx, 1.0)
    with torch.no_grad(), pytest.raises(k3moe.K3MoeError, match="CUDA tensor"):
        k3moe.balance_loss(S, idx, 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("words", [0, 1, 3])
def test_tables_with_a_short_meta(dev, words):
    """The kernels read meta[0] and meta[2]: a shorter array is refused, as every other table of a wrong length is."""
    idx = torch.randint(0, 4, (30, 2), generator=torch.Generator().manual_seed(0)).to(torch.int32).to(dev)
    good = k3moe.route_tables(idx, 4)
    t = dataclasses.replace(good, meta=good.meta[:words].contiguous())
    x = torch.zeros((30, 64), dtype=torch.bfloat16, device=dev)
    gu = torch.zeros((t.cap_rows, 128), dtype=torch.bfloat16, device=dev)
    q = torch.zeros((t.cap_rows, 64), dtype=torch.int8, device=dev)
    s, w, sw = torch.zeros(t.cap_rows, device=dev), torch.zeros((4 * 8, 64), dtype=torch.int8, device=dev), torch.zeros(32, device=dev)
    for call in (lambda: k3moe.quant_int8_permute(x, t), lambda: k3moe.act_quant_int8(gu, tables=t),
                 lambda: k3moe.grouped_gemm_int8(q, s, w, sw, t, 4)):
        with pytest.raises(k3moe.K3MoeError, match="meta"):
            call()
    k3moe.quant_int8_permute(x, good)
    k3moe.act_quant_int8(gu, tables=good)
    k3moe.grouped_gemm_int8(q, s, w, sw, good, 4)
    torch.cuda.synchronize()
