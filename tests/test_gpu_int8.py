"""The 8-bit integer products (k3moe_quant_int8, k3moe_act_quant_int8, k3moe_quant_int8_permute, k3moe_gemm_int8,
k3moe_grouped_gemm_int8) against plain 64-bit computations.

Codes and scales of bf16 and f32 rows are compared bit for bit: q is the half-even rounding of the real quotient
127 x / amax (decided here in exact integer comparisons), the scale amax / 127 rounded once.  Products too: the int32
sum is exact, so the result is fl(fl(fl(sum) * sx) * sw) in f32, rounded once more where the output is bf16."""
import numpy as np
import pytest
import torch

import k3moe

pytestmark = pytest.mark.gpu


def codes(x):
    """(q int8, scale f32) of f32-valued rows (numpy float32)."""
    x = np.asarray(x, np.float32)
    bad = ~np.isfinite(x).all(1)
    amax = np.abs(np.where(bad[:, None], 0, x)).max(1).astype(np.float64)
    a = np.abs(np.where(bad[:, None], 0, x)).astype(np.float64)
    safe = np.where(amax > 0, amax, 1.0)[:, None]
    k = np.floor(127.0 * a / safe)
    # 254 a and (2k + 1) amax have at most 32 + 24 bits: exact in float64 up to the quotient's own floor, fixed here
    for _ in range(2):
        k = np.where(127.0 * a < k * safe, k - 1, k)
        k = np.where(127.0 * a >= (k + 1) * safe, k + 1, k)
    twice, half = 254.0 * a, (2 * k + 1) * safe
    q = np.where((twice > half) | ((twice == half) & (k % 2 == 1)), k + 1, k)
    q = np.where(amax[:, None] > 0, q, 0) * np.sign(np.where(bad[:, None], 0, x))
    scale = (amax.astype(np.float32) / np.float32(127)).astype(np.float32)
    scale[bad] = np.nan
    return q.astype(np.int8), scale


def product(q, sx, w, sw, dtype):
    """fl(fl(fl(q w^T) sx) sw), the sum exact in float64."""
    acc = (q.double() @ w.double().t()).float()
    return (acc * sx[:, None] * sw[None]).to(dtype)


def same_bits(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def rand_codes(g, rows, cols, dev, ld=None):
    buf = torch.randint(-128, 128, (rows, ld or -(-cols // 16) * 16), generator=g, device=dev, dtype=torch.int8)
    return buf[:, :cols]


# ------------------------------------------------------------------ the quantiser
@pytest.mark.parametrize("rows,cols,dtype", [
    (1, 1, "bf16"), (3, 15, "bf16"), (5, 16, "f32"), (130, 512, "bf16"), (33, 513, "f32"), (17, 1000, "bf16"),
    (9, 1024, "f32"), (4, 1025, "bf16"), (70, 4096, "bf16"), (7, 4100, "f32"), (300, 7168, "bf16"), (5, 8193, "bf16"),
    (3, 16384, "f32"), (3, 16385, "bf16"), (2, 40000, "f32"), (2500, 64, "bf16"), (20000, 48, "f32")])
def test_codes_are_exact(dev, rows, cols, dtype):
    g = torch.Generator(device=dev).manual_seed(rows + cols)
    x = torch.randn(rows, cols, generator=g, device=dev) * torch.exp(
        torch.rand(rows, 1, generator=g, device=dev) * 40 - 20)
    x = x.to(torch.bfloat16 if dtype == "bf16" else torch.float32)
    x[rows // 2, cols // 2:] = 0
    q, s = k3moe.quant_int8(x)
    rq, rs = codes(x.float().cpu().numpy())
    assert np.array_equal(q.cpu().numpy(), rq)
    assert np.array_equal(s.cpu().numpy(), rs)


def test_every_bf16_quotient_of_some_maxima(dev):
    """All bf16 magnitudes up to a row's maximum, maxima over a whole binade and at the ends of the range: every tie and
    near tie of the rounding."""
    bits = np.arange(0, 0x7F80, dtype=np.int64)
    mant = np.concatenate([0x3F80 + np.arange(128), [0x0001, 0x007F, 0x0080, 0x7F7F, 0x0200, 0x7E00]])
    rows = []
    for m in mant:
        row = bits[(bits <= m) & (bits >= max(0, m - 14 * 128))]
        rows.append(np.pad(row, (0, 14 * 128 + 1 - len(row)), constant_values=m))
    x = torch.from_numpy(np.array(rows).astype(np.int16)).view(torch.bfloat16)
    x[:, ::2] *= -1
    q, s = k3moe.quant_int8(x.to(dev))
    rq, rs = codes(x.float().numpy())
    assert np.array_equal(q.cpu().numpy(), rq)
    assert np.array_equal(s.cpu().numpy(), rs)


def test_rows_at_the_ends_of_the_range(dev):
    """f32 rows from subnormal to the largest magnitudes, in registers and read twice, and gated rows far from 1."""
    g = torch.Generator().manual_seed(6)
    top = torch.tensor([1e-44, 1e-42, 1e-38, 3e-30, 2.0 ** -60, 2.0 ** -61, 2.0 ** 60, 2.0 ** 61, 1e30, 3.4e38])
    for cols in (96, 20001):
        x = (torch.rand(10, cols, generator=g, dtype=torch.float64) * 2 - 1)
        x[:, 5] = 1
        x = (x * top[:, None].double()).float()
        q, s = k3moe.quant_int8(x.to(dev))
        rq, rs = codes(x.numpy())
        assert np.array_equal(q.cpu().numpy(), rq) and np.array_equal(s.cpu().numpy(), rs)
    scale = torch.tensor([1e-15, 1e-10, 1e10, 1e17])[:, None]
    gu = torch.cat([torch.rand(4, 64, generator=g) * scale, torch.randn(4, 64, generator=g) * scale], 1).to(torch.bfloat16)
    q, s = k3moe.act_quant_int8(gu.to(dev))
    h = gate64(gu, k3moe.ACT_SWIGLU)
    amax = h.abs().amax(1, keepdim=True)
    np.testing.assert_allclose(s.double().cpu().numpy(), (amax[:, 0] / 127).numpy(), rtol=2 ** -18)
    assert bool(((q.cpu().double() - 127 * h / amax).abs() <= 0.5 + 127 * 2 ** -17).all())


def test_zero_and_non_finite_rows(dev):
    x = torch.randn(6, 100, generator=torch.Generator().manual_seed(0))
    x[1] = 0
    x[2, 7] = float("inf")
    x[3, 99] = -float("inf")
    x[4, 50] = float("nan")
    for dtype in (torch.bfloat16, torch.float32):
        q, s = k3moe.quant_int8(x.to(dtype).to(dev))
        rq, rs = codes(x.to(dtype).float().numpy())
        assert np.array_equal(q.cpu().numpy(), rq) and np.array_equal(s.cpu().numpy(), rs, equal_nan=True)
        w = torch.ones((5, 112), dtype=torch.int8, device=dev)[:, :100]
        y = k3moe.gemm_int8(q, s, w, torch.ones(5, device=dev), torch.float32).cpu()
        assert bool((y[1] == 0).all()) and bool(torch.isnan(y[2:5]).all()) and bool(torch.isfinite(y[[0, 1, 5]]).all())


@pytest.mark.parametrize("offset,ld", [(0, 136), (1, 135), (8, 144), (3, 131)])
def test_strides_and_alignment(dev, offset, ld):
    """Rows that start off 16 bytes are read element by element; bytes beside q's rows are left as they were."""
    g = torch.Generator(device=dev).manual_seed(ld)
    base = torch.randn(60 * ld + 16, generator=g, device=dev).to(torch.bfloat16)
    x = base[offset:offset + 60 * ld].reshape(60, ld)[:, :130]
    buf = torch.full((60, 160), 77, dtype=torch.int8, device=dev)
    s = torch.empty(60, device=dev)
    k3moe.quant_int8(x, out=(buf[:, :130], s))
    rq, rs = codes(x.float().cpu().numpy())
    assert np.array_equal(buf[:, :130].cpu().numpy(), rq) and np.array_equal(s.cpu().numpy(), rs)
    assert bool((buf[:, 130:] == 77).all())


def gate64(gu, act):
    g, u = gu.double().chunk(2, 1)
    sg = torch.sigmoid(g)
    return g * sg * u if act == k3moe.ACT_SWIGLU else 4 * torch.tanh(g / 4) * sg * 25 * torch.tanh(u / 25)


@pytest.mark.parametrize("act", [k3moe.ACT_SWIGLU, k3moe.ACT_SITU])
@pytest.mark.parametrize("rows,I", [(1, 1), (5, 17), (200, 256), (33, 2048), (9, 2050), (3, 9000), (2, 20000)])
def test_gated_codes(dev, act, rows, I):
    """act(gate) * up in f32 is within 2^-18 of the value (the exponential, the quotient and tanh, a few units each at
    gates below 16), so a code is off by at most one, and only where the quotient is within 127 * 2^-17 of a half."""
    g = torch.Generator(device=dev).manual_seed(rows * I)
    gu = (torch.randn(rows, 2 * I, generator=g, device=dev) * 3).to(torch.bfloat16)
    q, s = k3moe.act_quant_int8(gu, act)
    h = gate64(gu, act)
    amax = h.abs().amax(1, keepdim=True)
    np.testing.assert_allclose(s.double().cpu().numpy(), (amax[:, 0] / 127).cpu().numpy(), rtol=2 ** -18)
    y = 127 * h / amax
    assert bool(((q.double() - y).abs() <= 0.5 + 127 * 2 ** -17).all())


def test_gated_rows_of_the_tables(dev):
    """With tables only the real rows are read (padding holds NaN) and written."""
    idx = torch.randint(0, 5, (300, 1), generator=torch.Generator().manual_seed(1)).to(torch.int32).to(dev)
    t = k3moe.route_tables(idx, 5)
    gu = torch.full((t.cap_rows, 64), float("nan"), dtype=torch.bfloat16, device=dev)
    real = t.exp2perm.reshape(-1).long()
    gu[real] = torch.randn(300, 64, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(dev)
    q = torch.full((t.cap_rows, 32), 99, dtype=torch.int8, device=dev)
    s = torch.full((t.cap_rows,), -1.0, device=dev)
    k3moe.act_quant_int8(gu, tables=t, out=(q, s))
    rq, rs = k3moe.act_quant_int8(gu[real].contiguous())
    assert torch.equal(q[real], rq) and torch.equal(s[real], rs)
    pad = torch.ones(t.cap_rows, dtype=torch.bool, device=dev)
    pad[real] = False
    assert bool((q[pad] == 99).all()) and bool((s[pad] == -1).all())


@pytest.mark.parametrize("R,K,E,first,shared,cols", [(1, 8, 16, 0, 0, 256), (300, 4, 16, 0, 1, 100),
                                                     (77, 2, 8, 8, 0, 7168), (50, 1, 3, 0, 1, 20000)])
def test_permuted_codes(dev, R, K, E, first, shared, cols):
    g = torch.Generator().manual_seed(R)
    idx = torch.stack([torch.randperm(first + E + 4, generator=g)[:K] for _ in range(R)]).to(torch.int32).to(dev)
    t = k3moe.route_tables(idx, E, first, shared)
    x = torch.randn(R, cols, generator=g).to(torch.bfloat16).to(dev)
    ld = -(-cols // 16) * 16
    q = torch.full((t.cap_rows, ld), 99, dtype=torch.int8, device=dev)[:, :cols]
    s = torch.full((t.cap_rows,), -1.0, device=dev)
    k3moe.quant_int8_permute(x, t, out=(q, s))
    rq, rs = k3moe.quant_int8(x)
    want, ws = torch.full_like(q, 99), torch.full_like(s, -1.0)
    for k in range(K):
        at = t.exp2perm[:, k].long()
        want[at[at >= 0]], ws[at[at >= 0]] = rq[at >= 0], rs[at >= 0]
    if shared:
        b = int(t.meta[2])
        want[b:b + R], ws[b:b + R] = rq, rs
    assert torch.equal(q, want) and torch.equal(s, ws)


# ------------------------------------------------------------------ products
@pytest.mark.parametrize("T,N,C", [
    (1, 1, 1), (1, 128, 128), (1, 4096, 7168), (2, 200, 16), (15, 129, 130), (16, 256, 300), (17, 300, 1000),
    (33, 64, 2047), (64, 7168, 2048), (65, 1003, 640), (100, 2048, 512), (129, 500, 1500), (255, 130, 128),
    (256, 4096, 256), (257, 4096, 129), (300, 4096, 7168), (1000, 896, 1024), (2049, 515, 333), (4096, 2048, 400),
    (2305, 1803, 300), (4100, 1000, 2100), (20000, 130, 64), (260, 14400, 96), (5, 40, 131071)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_product_is_exact(dev, T, N, C, dtype):
    g = torch.Generator(device=dev).manual_seed(T + N + C)
    q, w = rand_codes(g, T, C, dev), rand_codes(g, N, C, dev)
    sx = torch.rand(T, generator=g, device=dev) * 0.01
    sw = torch.rand(N, generator=g, device=dev) * 0.01
    err = torch.zeros(2, dtype=torch.int32, device=dev)
    out = torch.full((T + 1, N + 3), 5.0, dtype=dtype, device=dev)
    k3moe.gemm_int8(q, sx, w, sw, out=out[:T, :N], err=err)
    torch.cuda.synchronize()
    assert err.tolist() == [0, 0]
    assert same_bits(out[:T, :N], product(q, sx, w, sw, dtype))
    assert bool((out[T] == 5).all()) and bool((out[:, N:] == 5).all())
    if T <= 64:
        plain = k3moe.gemm_int8(q, sx, w, sw, dtype)
        assert same_bits(plain, out[:T, :N])


def test_largest_sums(dev):
    """-128 * -128 over the longest reduction: 2^14 * 131071 is the largest sum and fits int32."""
    q = torch.full((3, 131072), -128, dtype=torch.int8, device=dev)[:, :131071]
    w = torch.full((130, 131072), -128, dtype=torch.int8, device=dev)[:, :131071]
    w[1] = 127
    one = torch.ones(130, device=dev)
    y = k3moe.gemm_int8(q, one[:3].contiguous(), w, one, torch.float32)
    assert same_bits(y, product(q, one[:3], w, one, torch.float32))
    assert float(y[0, 0]) == float(np.float32(2 ** 14 * 131071))


def test_operands_with_row_strides(dev):
    g = torch.Generator(device=dev).manual_seed(4)
    q, w = rand_codes(g, 90, 200, dev, 256), rand_codes(g, 140, 200, dev, 224)
    sx, sw = torch.rand(90, generator=g, device=dev), torch.rand(140, generator=g, device=dev)
    assert same_bits(k3moe.gemm_int8(q, sx, w, sw), product(q, sx, w, sw, torch.bfloat16))


@pytest.mark.parametrize("R,K,E,first,shared,N,C", [
    (1, 1, 1, 0, 0, 128, 128), (5, 2, 16, 0, 0, 200, 256), (300, 4, 16, 0, 1, 256, 300), (128, 1, 1, 0, 0, 130, 144),
    (500, 2, 3, 0, 0, 384, 512), (64, 8, 112, 224, 0, 512, 1024), (1024, 8, 32, 0, 0, 300, 700),
    (40, 4, 8, 50, 0, 64, 64)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_grouped_product_is_exact(dev, R, K, E, first, shared, N, C, dtype):
    g = torch.Generator().manual_seed(R + E)
    total = max(first + E, K)
    # experts of uneven popularity, some without a row, some ids of other ranks
    idx = torch.stack([torch.multinomial(1.0 / (1 + torch.arange(total).float()), K, generator=g)
                       for _ in range(R)]).to(torch.int32).to(dev)
    t = k3moe.route_tables(idx, E, first, shared)
    gd = torch.Generator(device=dev).manual_seed(9)
    n_exp = E + shared
    q, w = rand_codes(gd, t.cap_rows, C, dev), rand_codes(gd, n_exp * N, C, dev)
    sx = torch.rand(t.cap_rows, generator=gd, device=dev)
    sw = torch.rand(n_exp * N, generator=gd, device=dev)
    err = torch.zeros(2, dtype=torch.int32, device=dev)
    out = torch.full((t.cap_rows, N), 3.0, dtype=dtype, device=dev)
    k3moe.grouped_gemm_int8(q, sx, w, sw, t, n_exp, out=out, err=err)
    want = torch.full_like(out, 3.0)
    for c in range(int(t.meta[0])):
        e, r0, r1 = int(t.cta_batch[c]), c * 128, int(t.cta_limit[c])
        want[r0:r1] = product(q[r0:r1], sx[r0:r1], w[e * N:(e + 1) * N], sw[e * N:(e + 1) * N], dtype)
    assert err.tolist() == [0, 0]
    assert same_bits(out, want)


def test_no_row_on_this_rank(dev):
    """Every pick foreign: no tile, nothing read or written."""
    idx = torch.full((20, 2), 9, dtype=torch.int32, device=dev)
    idx[:, 1] = 11
    t = k3moe.route_tables(idx, 4)
    x = torch.randn(20, 64, device=dev).to(torch.bfloat16)
    q = torch.full((t.cap_rows, 64), 99, dtype=torch.int8, device=dev)
    s = torch.full((t.cap_rows,), -1.0, device=dev)
    k3moe.quant_int8_permute(x, t, out=(q, s))
    k3moe.act_quant_int8(torch.zeros((t.cap_rows, 128), dtype=torch.bfloat16, device=dev), tables=t, out=(q, s))
    out = torch.full((t.cap_rows, 256), 3.0, device=dev)
    w = torch.zeros((4 * 256, 64), dtype=torch.int8, device=dev)
    err = torch.zeros(2, dtype=torch.int32, device=dev)
    k3moe.grouped_gemm_int8(q, s, w, torch.ones(1024, device=dev), t, 4, out=out, err=err)
    assert int(t.meta[0]) == 0 and err.tolist() == [0, 0]
    assert bool((q == 99).all()) and bool((s == -1).all()) and bool((out == 3).all())


@pytest.mark.parametrize("N", [128, 512])  # a block a tile, a pair of blocks
def test_bad_tiles_are_skipped_and_reported(dev, N):
    """Tiles whose expert or row limit is out of range: the kernel's own checks record and skip them."""
    g = torch.Generator(device=dev).manual_seed(1)
    idx = torch.arange(4, dtype=torch.int32, device=dev).repeat(100)[:, None].contiguous()
    t = k3moe.route_tables(idx, 4)
    q, w = rand_codes(g, t.cap_rows, 128, dev), rand_codes(g, 4 * N, 128, dev)
    sx, sw = torch.ones(t.cap_rows, device=dev), torch.ones(4 * N, device=dev)
    good = torch.zeros((t.cap_rows, N), device=dev)
    k3moe.grouped_gemm_int8(q, sx, w, sw, t, 4, out=good)
    t.cta_batch[1] = 4
    t.cta_batch[2] = -1
    t.cta_limit[3] = 3 * 128 + 129
    err = torch.zeros(2, dtype=torch.int32, device=dev)
    out = torch.zeros((t.cap_rows, N), device=dev)
    k3moe.grouped_gemm_int8(q, sx, w, sw, t, 4, out=out, err=err)
    rc, words = k3moe.read_error(err)
    assert rc == -6 and words == (2, 0xD00)
    assert same_bits(out[:100], good[:100]) and bool((out[128:] == 0).all())


def test_offsets_past_32_bits(dev):
    """2.4e9 elements in, as codes and out (about 17 GB): the last rows as the same rows by themselves."""
    rows, cols = 36000, 65536
    x = torch.zeros((rows, cols), dtype=torch.bfloat16, device=dev)
    g = torch.Generator(device=dev).manual_seed(2)
    x[-3:] = torch.randn(3, cols, generator=g, device=dev).to(torch.bfloat16)
    q, s = k3moe.quant_int8(x)
    rq, rs = k3moe.quant_int8(x[-3:].contiguous())
    assert torch.equal(q[-3:], rq) and torch.equal(s[-3:], rs) and float(s[:-3].abs().max()) == 0
    w, sw = rand_codes(g, cols, 16, dev), torch.rand(cols, generator=g, device=dev)
    y = k3moe.gemm_int8(q[:, :16], s, w, sw)
    assert same_bits(y[-3:], product(rq[:, :16], rs, w, sw, torch.bfloat16)) and bool((y[:-3] == 0).all())


def test_captured_and_on_another_stream(dev):
    g = torch.Generator(device=dev).manual_seed(8)
    x = torch.randn(70, 1500, generator=g, device=dev).to(torch.bfloat16)
    wf = torch.randn(900, 1500, generator=g, device=dev)
    w, sw = k3moe.quant_int8(wf)
    q, sx = k3moe.quant_int8(x)
    y = k3moe.gemm_int8(q, sx, w, sw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    q2, s2 = k3moe.quant_int8(x, stream=side)
    y2 = k3moe.gemm_int8(q2, s2, w, sw, stream=side)
    side.synchronize()
    assert same_bits(y, y2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q3, s3 = k3moe.quant_int8(x)
        y3 = k3moe.gemm_int8(q3, s3, w, sw)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert same_bits(y, y3)


def test_captured_behind_a_join(dev):
    """A captured call that follows work on two streams: rows from one, weights from the other."""
    g = torch.Generator(device=dev).manual_seed(18)
    xf = torch.randn(40, 512, generator=g, device=dev)
    wf = torch.randn(300, 512, generator=g, device=dev)
    idx = torch.randint(0, 64, (40, 2), generator=g, device=dev, dtype=torch.int32)
    q, sx = k3moe.quant_int8(xf * 2)
    w, sw = k3moe.quant_int8(wf * 3)
    want = k3moe.gemm_int8(q, sx, w, sw)
    loss = k3moe.balance_loss(xf[:, :64], idx, 1.0).loss
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            w2, sw2 = k3moe.quant_int8(wf * 3)
        q2, sx2 = k3moe.quant_int8(xf * 2)
        main.wait_stream(side)
        y = k3moe.gemm_int8(q2, sx2, w2, sw2)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            b = k3moe.balance_loss(xf[:, :64], idx, 1.0)
        z = y * 2
        main.wait_stream(side)
        dS = k3moe.route_backward(xf[:, :64], idx, 1.0, b.counts, b.rows)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert same_bits(y, want) and torch.equal(b.loss, loss) and same_bits(z, want * 2)
    assert same_bits(dS, k3moe.route_backward(xf[:, :64], idx, 1.0, b.counts, b.rows))


def test_weights_from_a_late_stream(dev):
    """An overlapped launch still waits for an event that stands between it and the kernel before it: weights written
    late on another stream, rows written right before on this one."""
    g = torch.Generator(device=dev).manual_seed(19)
    x = torch.randn(40, 512, generator=g, device=dev)
    wf = torch.randn(300, 512, generator=g, device=dev)
    q, sx = k3moe.quant_int8(x)
    w, sw = k3moe.quant_int8(wf)
    want = k3moe.gemm_int8(q, sx, w, sw)
    w2, sw2 = torch.zeros_like(w), torch.zeros_like(sw)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(3):
        w2.zero_()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.cuda._sleep(5_000_000)  # a few milliseconds
            k3moe.quant_int8(wf, out=(w2, sw2))
        q2, sx2 = k3moe.quant_int8(x)
        torch.cuda.current_stream().wait_stream(side)
        assert same_bits(k3moe.gemm_int8(q2, sx2, w2, sw2), want)


def test_two_products_at_once(dev):
    """Calls share no state: split reductions on two streams at the same time."""
    g = torch.Generator(device=dev).manual_seed(5)
    q, w = rand_codes(g, 8, 7168, dev), rand_codes(g, 2048, 7168, dev)
    sx, sw = torch.rand(8, generator=g, device=dev), torch.rand(2048, generator=g, device=dev)
    want = product(q, sx, w, sw, torch.bfloat16)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [k3moe.gemm_int8(q, sx, w, sw, stream=streams[i % 2]) for i in range(20)]
    torch.cuda.synchronize()
    assert all(same_bits(y, want) for y in got)


def test_layer_in_int8(dev):
    """A routed layer with int8 experts: top-k -> tables -> codes -> gate-up products -> gate -> down products ->
    combine, against the same steps in float64 on the device's own int8 weights.

    Tolerance: the products are exact; what rounds are the gate-up outputs to bf16 (2^-8 relative an element), the codes
    of hidden states and of the gate (half a step of a 127th of the row's maximum, on both sides the same rule), the
    down outputs and the combined row to bf16.  The reference makes the same roundings at the same places, so what is
    left are codes that an f32 gate puts on the other side of a half (one step each, fewer than one in a thousand:
    1 / 127 * sqrt(1e-3) of a row's maximum, about 5 row-rms) and bf16 neighbours (2^-8): 5e-3 of the output's norm."""
    T, H, I, E, K = 200, 512, 384, 12, 4
    g = torch.Generator(device=dev).manual_seed(3)
    x = torch.randn(T, H, generator=g, device=dev).to(torch.bfloat16)
    S = torch.randn(T, E, generator=g, device=dev)
    bias = torch.rand(E, generator=g, device=dev) * 0.1
    rs = torch.tensor([2.5], dtype=torch.bfloat16, device=dev)
    w13, s13 = k3moe.quant_int8(torch.randn((E + 1) * 2 * I, H, generator=g, device=dev) / H ** 0.5)
    w2, s2 = k3moe.quant_int8(torch.randn((E + 1) * H, I, generator=g, device=dev) / I ** 0.5)
    idx, wts = k3moe.route_topk(S, bias, rs, K)
    t = k3moe.route_tables(idx, E, 0, 1)
    gu = k3moe.grouped_gemm_int8(*k3moe.quant_int8_permute(x, t), w13, s13, t, E + 1)
    down = k3moe.grouped_gemm_int8(*k3moe.act_quant_int8(gu, tables=t), w2, s2, t, E + 1)
    out = k3moe.combine(down, t, wts, T)

    def expert(e, rows):
        qx, sx = codes(rows.float().cpu().numpy())
        qx, sx = torch.from_numpy(qx).to(dev).double(), torch.from_numpy(sx).to(dev).double()[:, None]
        a = (qx @ w13[e * 2 * I:(e + 1) * 2 * I].double().t()) * sx * s13[e * 2 * I:(e + 1) * 2 * I].double()
        h = gate64(a.to(torch.bfloat16), k3moe.ACT_SWIGLU)
        amax = h.abs().amax(1, keepdim=True)
        qh = torch.round(127 * h / amax)
        y = (qh @ w2[e * H:(e + 1) * H].double().t()) * amax / 127 * s2[e * H:(e + 1) * H].double()
        return y.to(torch.bfloat16).double()

    ref = expert(E, x)
    for e in range(E):
        row, k = torch.nonzero(idx == e, as_tuple=True)
        if row.numel():
            ref[row] += wts[row, k].double()[:, None] * expert(e, x[row])
    rel = float((out.double() - ref).norm() / ref.norm())
    assert rel <= 5e-3, rel
