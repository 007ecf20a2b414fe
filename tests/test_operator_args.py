"""CPU tests of the refusals of the router's training entries and of the 8-bit integer products: the C ABI rejects bad
arguments before any device work, the Python mirror before the C ABI."""
import types

import pytest
import torch

import k3moe


@pytest.fixture(scope="module")
def lib():
    import __graft_entry__

    __graft_entry__.build()
    return k3moe.lib()


P = 256  # a plausible, never dereferenced address


def balance(lib, **kw):
    a = dict(S=P, lds=64, idx=P, T=8, E=64, K=4, seq=P, B=2, mask=None, alpha=1.0, scratch=P, counts=P, prob=P, rows=P,
             loss=P)
    a.update(kw)
    return lib.k3moe_balance_loss(*a.values(), None)


def test_balance_loss_refusals(lib):
    for kw in (dict(S=None), dict(idx=None), dict(scratch=None), dict(scratch=8), dict(counts=None), dict(prob=None),
               dict(rows=None), dict(loss=None), dict(T=-1), dict(E=0), dict(E=1025, lds=2000), dict(K=0), dict(K=17),
               dict(T=2 ** 30 + 1), dict(lds=63), dict(B=0), dict(seq=None, B=2), dict(B=2 ** 31 - 1)):
        assert balance(lib, **kw) == -1, kw
    assert lib.k3moe_balance_scratch_bytes(-1, 8, 1) == 0 and lib.k3moe_balance_scratch_bytes(8, 1025, 1) == 0
    assert lib.k3moe_balance_scratch_bytes(8, 8, 0) == 0


def test_balance_scratch_covers_every_block_and_sequence(lib):
    # (blocks + B) partial rows of E f32 and E int32
    for T, E, B in ((0, 1, 1), (1, 896, 3), (256, 100, 1), (257, 100, 1), (1, 896, 1), (8192, 896, 16),
                    (65536, 1024, 4096), (2 ** 30, 8, 3)):
        nv = -(-E // 128)
        chunk = max(8, -(-T // (148 * (2 if nv <= 2 else 1))))
        blocks = max(1, -(-T // chunk))
        need = (blocks + B) * E * 8 + (blocks + B) * 4 + 8 * 148 * 8 + 4
        got = lib.k3moe_balance_scratch_bytes(T, E, B)
        assert need <= got <= need + 5 * 256, (T, E, B)


def backward(lib, **kw):
    a = dict(S=P, lds=64, idx=P, T=8, E=64, K=4, seq=P, B=2, mask=None, alpha=1.0, counts=P, rows=P, dloss=None, dwts=P,
             rs=P, dS=P, ldd=64, dtype=1)
    a.update(kw)
    return lib.k3moe_route_backward(*a.values(), None)


def test_route_backward_refusals(lib):
    for kw in (dict(S=None), dict(dS=None), dict(idx=None), dict(counts=None, dwts=None), dict(rows=None), dict(rs=None),
               dict(ldd=63), dict(dtype=2), dict(T=-1), dict(E=0), dict(K=17), dict(lds=1), dict(B=0),
               dict(seq=None, B=3)):
        assert backward(lib, **kw) == -1, kw
    assert backward(lib, T=0, S=None, dS=None, idx=None) == 0  # nothing to do


def test_quantiser_refusals(lib):
    def quant(x=P, dtype=0, ldx=64, rows=4, cols=64, q=P, ldq=64, scale=P):
        return lib.k3moe_quant_int8(x, dtype, ldx, rows, cols, q, ldq, scale, None)

    for kw in (dict(x=None), dict(q=None), dict(scale=None), dict(dtype=2), dict(ldx=63), dict(rows=-1), dict(cols=0),
               dict(q=P + 8), dict(ldq=72), dict(ldq=48)):
        assert quant(**kw) == -1, kw
    assert quant(rows=0, x=None, q=None, scale=None) == 0

    def act(gu=P, ldg=128, rows=4, I=64, a=0, limit=None, meta=None, ctas=0, q=P, ldq=64, scale=P):
        return lib.k3moe_act_quant_int8(gu, ldg, rows, I, a, limit, meta, ctas, q, ldq, scale, None)

    for kw in (dict(gu=None), dict(ldg=127), dict(I=0), dict(a=2), dict(limit=P), dict(meta=P), dict(limit=P, meta=P),
               dict(q=P + 1), dict(ldq=16), dict(scale=None)):
        assert act(**kw) == -1, kw

    def perm(x=P, ldx=64, R=4, cols=64, K=2, e2p=P, meta=P, q=P, ldq=64, scale=P, cap=128):
        return lib.k3moe_quant_int8_permute(x, ldx, R, cols, K, e2p, meta, q, ldq, scale, cap, None)

    for kw in (dict(x=None), dict(e2p=None), dict(meta=None), dict(K=0), dict(K=17), dict(cap=0), dict(R=-1),
               dict(ldq=65), dict(scale=None), dict(ldx=1)):
        assert perm(**kw) == -1, kw


def test_product_refusals(lib):
    def gemm(q=P, ldq=64, sx=P, w=P, ldw=64, sw=P, T=4, N=8, C=64, out=P, ldo=8, dtype=0):
        return lib.k3moe_gemm_int8(q, ldq, sx, w, ldw, sw, T, N, C, out, ldo, dtype, None, None)

    for kw in (dict(q=None), dict(q=P + 8), dict(ldq=72), dict(ldq=48), dict(sx=None), dict(w=None), dict(w=P + 4),
               dict(ldw=65), dict(sw=None), dict(out=None), dict(out=P + 1), dict(out=P + 2, dtype=1), dict(ldo=7),
               dict(T=-1), dict(N=0), dict(C=0), dict(C=131072, ldq=131072, ldw=131072), dict(dtype=3),
               dict(T=2 ** 31 - 255), dict(N=2 ** 31 - 255, ldo=2 ** 31)):
        assert gemm(**kw) == -1, kw
    assert gemm(T=0, q=None, out=None) == 0

    def grouped(q=P, ldq=64, sx=P, w=P, ldw=64, sw=P, cb=P, cl=P, meta=P, N=8, C=64, E=2, cap=256, ctas=2, out=P, ldo=8,
                dtype=0):
        return lib.k3moe_grouped_gemm_int8(q, ldq, sx, w, ldw, sw, cb, cl, meta, N, C, E, cap, ctas, out, ldo, dtype,
                                           None, None)

    for kw in (dict(q=None), dict(ldq=1), dict(sx=None), dict(w=None), dict(sw=None), dict(cb=None), dict(cl=None),
               dict(meta=None), dict(N=0), dict(C=0), dict(E=0), dict(cap=255), dict(ctas=0), dict(out=None),
               dict(ldo=1), dict(dtype=-1), dict(E=2 ** 20, N=2 ** 12), dict(C=131072, ldq=131072, ldw=131072)):
        assert grouped(**kw) == -1, kw


def test_the_mirror_refuses_host_tensors():
    x = torch.zeros(4, 64)
    i8 = torch.zeros(4, 64, dtype=torch.int8)
    s = torch.zeros(4)
    for call in (lambda: k3moe.quant_int8(x), lambda: k3moe.act_quant_int8(x.to(torch.bfloat16)),
                 lambda: k3moe.gemm_int8(i8, s, i8, s),
                 lambda: k3moe.balance_loss(x, torch.zeros(4, 2, dtype=torch.int32), 1.0),
                 lambda: k3moe.route_backward(x, torch.zeros(4, 2, dtype=torch.int32))):
        with pytest.raises(k3moe.K3MoeError):
            call()


@pytest.mark.gpu
def test_the_mirror_refuses_what_the_kernels_do_not_take(dev):
    i8 = torch.zeros(4, 64, dtype=torch.int8, device=dev)
    s, sw = torch.zeros(4, device=dev), torch.zeros(4, device=dev)
    S = torch.zeros(4, 8, device=dev)
    idx = torch.zeros(4, 2, dtype=torch.int32, device=dev)
    bad = [
        lambda: k3moe.quant_int8(torch.zeros(4, 64, dtype=torch.float16, device=dev)),
        lambda: k3moe.quant_int8(torch.zeros(64, 4, device=dev).t()),
        lambda: k3moe.quant_int8(torch.zeros(1, 64, device=dev).expand(4, 64)),
        lambda: k3moe.quant_int8(torch.zeros(4, 64, device=dev), out=(i8[:, 1:], s)),
        lambda: k3moe.quant_int8(torch.zeros(4, 64, device=dev), out=(i8, s[:3])),
        lambda: k3moe.act_quant_int8(torch.zeros(4, 63, dtype=torch.bfloat16, device=dev)),
        lambda: k3moe.act_quant_int8(torch.zeros(4, 64, dtype=torch.bfloat16, device=dev), activation=5),
        lambda: k3moe.gemm_int8(i8, s, i8[:, :48], sw),
        lambda: k3moe.gemm_int8(i8, s[:2], i8, sw),
        lambda: k3moe.gemm_int8(i8, s, i8, sw.cpu()),
        lambda: k3moe.gemm_int8(i8, s, i8, sw, dtype=torch.float16),
        lambda: k3moe.gemm_int8(i8, s, i8, sw, out=torch.zeros(4, 5, device=dev)),
        lambda: k3moe.gemm_int8(i8[:, 1:33], s, i8[:, :32], sw),
        lambda: k3moe.balance_loss(S.double(), idx, 1.0),
        lambda: k3moe.balance_loss(S, idx.long(), 1.0),
        lambda: k3moe.balance_loss(S, idx[:3], 1.0),
        lambda: k3moe.balance_loss(S, idx, 1.0, mask=torch.ones(3, dtype=torch.bool, device=dev)),
        lambda: k3moe.balance_loss(S, idx, 1.0, seq=torch.zeros(1, dtype=torch.int32, device=dev)),
        lambda: k3moe.balance_loss(S, torch.zeros(4, 17, dtype=torch.int32, device=dev), 1.0),
        lambda: k3moe.route_backward(S, idx),
        lambda: k3moe.route_backward(S, idx, counts=torch.zeros(1, 8, dtype=torch.int32, device=dev)),
        lambda: k3moe.route_backward(S, idx, dwts=torch.zeros(4, 2, device=dev)),
        lambda: k3moe.route_backward(S, idx, dwts=torch.zeros(4, 2, device=dev),
                                     rs=torch.ones(1, dtype=torch.bfloat16, device=dev), dtype=torch.float16),
    ]
    other = types.SimpleNamespace(device=torch.device("cuda", 7))
    bad += [lambda: k3moe.quant_int8(S, stream=other), lambda: k3moe.balance_loss(S, idx, 1.0, stream=other)]
    for i, call in enumerate(bad):
        with pytest.raises(k3moe.K3MoeError):
            call()
            pytest.fail(f"call {i} was taken")
