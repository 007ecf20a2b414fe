"""Two captured runs of the router's training entries and the integer products, replayed at the same time."""
import pytest
import torch

import k3moe

pytestmark = pytest.mark.gpu


class Run:
    """Its inputs, which the captured graph reads at every replay, and the calls of a step."""

    def __init__(self, dev, seed, T, C):
        g = torch.Generator(device=dev).manual_seed(seed)
        self.x = torch.randn(T, C, generator=g, device=dev).to(torch.bfloat16)
        self.S = torch.randn(T, 200, generator=g, device=dev)
        self.idx = torch.rand(T, 200, generator=g, device=dev).topk(4, 1).indices.to(torch.int32)
        self.seq = torch.tensor([0, T // 3, T // 3] + [T] * 70, dtype=torch.int32, device=dev)
        self.w, self.sw = k3moe.quant_int8(torch.randn(600, C, generator=g, device=dev))
        self.t = k3moe.route_tables((self.idx[:, :1] % 6).contiguous(), 6)
        self.we, self.swe = k3moe.quant_int8(torch.randn(6 * 256, C, generator=g, device=dev))
        self.real = self.t.exp2perm.reshape(-1).long()
        self.want = [v.clone() for v in self.step()]
        torch.cuda.synchronize()
        self.stream = torch.cuda.Stream()
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            self.got = self.step()

    def step(self):
        b = k3moe.balance_loss(self.S, self.idx, 0.5, seq=self.seq)
        dS = k3moe.route_backward(self.S, self.idx, 0.5, b.counts, b.rows, seq=self.seq)
        y = k3moe.gemm_int8(*k3moe.quant_int8(self.x), self.w, self.sw)
        q, s = k3moe.act_quant_int8(y, k3moe.ACT_SITU)
        o = k3moe.grouped_gemm_int8(*k3moe.quant_int8_permute(self.x, self.t), self.we, self.swe, self.t, 6)
        return [b.loss, b.counts, b.prob, b.rows, dS, y, q, s, o[self.real]]


def test_two_graphs_at_once(dev):
    runs = [Run(dev, 0, 700, 1024), Run(dev, 1, 90, 2048)]
    for _ in range(3):
        for r in runs:
            for v in r.got:
                v.zero_()
        torch.cuda.synchronize()
        for _ in range(20):
            for r in runs:
                with torch.cuda.stream(r.stream):
                    r.graph.replay()
        torch.cuda.synchronize()
        for r in runs:
            for i, (a, b) in enumerate(zip(r.got, r.want)):
                assert torch.equal(a, b), i
