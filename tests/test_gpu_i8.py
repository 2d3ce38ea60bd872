"""Rows in 8 bits and the products of 8-bit integers on the GPU against oracle/int8.py in 64 bits.

Codes and scales are equal. Products: the sum is exact; its conversion to fp32 and the two scales round once each (2^-24), so
y is within 3 * 2^-24 of itself (a little over, for the products of the roundings). SwiGLU: both factors are such y; the
sigmoid's exponential and reciprocal are off by a few 2^-24 and |gate| 2^-24 for the exponent's rounding, and the gate's own
error moves silu by at most (1 + |gate|) times itself.
"""
import pytest
import torch

from gpu_util import announce, device
from oracle import int8
from q35hip import Q35Error, ops

pytestmark = pytest.mark.gpu
H = 2.0 ** -24


def weights(N, K, seed=0, extremes=False):
    g = torch.Generator().manual_seed(seed)
    W = torch.randint(-127, 128, (N, K), generator=g).to(torch.int8)
    if extremes:
        W[:] = 127
        W[1::2] = -128
    return W, torch.rand(N, generator=g) * 1e-3 + 1e-5


def rows(M, K, seed=0):
    return torch.randn(M, K, generator=torch.Generator().manual_seed(seed)) * 3


def check(y, want, slack=3.2):
    y = y.double().cpu()
    assert y.shape == want.shape
    err = (y - want).abs() - slack * H * want.abs()
    assert bool((err <= 1e-37).all()), float(((y - want).abs() / want.abs().clamp_min(1e-30)).max())


@pytest.mark.parametrize("M,K", [(1, 4), (3, 64), (2, 1000), (17, 1024), (5, 1028), (4, 3584), (2, 5000), (3, 8192), (2, 16384),
                                 (700, 256)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_codes_and_scales(M, K, dtype):
    x = rows(M, K, seed=K).to(dtype)
    announce(f"quantize_rows {dtype} M{M} K{K}")
    q, s = ops.quantize_rows(x.to(device()))
    wq, ws = int8.quantize_rows(x)
    assert torch.equal(q.cpu(), wq) and torch.equal(s.cpu(), ws)
    wide = torch.full((M, K + 8), 9e9, dtype=dtype, device=device())
    wide[:, 4:K + 4] = x.to(device())
    q, s = ops.quantize_rows(wide[:, 4:K + 4])
    assert torch.equal(q.cpu(), wq) and torch.equal(s.cpu(), ws)


def test_codes_at_ties_and_odd_rows():
    """Quotients of n + 1/2 exactly and one step beside it, rows of zeros, of the smallest values, of one large value, and rows
    that hold a value that is not finite."""
    K = 256
    x = torch.zeros(12, K)
    n = torch.arange(K, dtype=torch.float32) - 128
    x[0] = (n + 0.5) * 0.25
    x[0, 0] = 31.75  # s = 1 / 4
    x[0] = x[0].clamp(-31.75, 31.75)
    x[1] = torch.nextafter(x[0], torch.tensor(100.0)).clamp(-31.75, 31.75)
    x[2] = torch.nextafter(x[0], torch.tensor(-100.0)).clamp(-31.75, 31.75)
    x[4] = 1e-45 * torch.sign(n)
    x[5] = 1e-42 * n
    x[6, 3] = 3e38
    x[7] = 1.0
    x[7, 5] = float("nan")
    x[8, 9] = float("inf")
    x[9, 11] = -float("inf")
    x[10] = torch.finfo(torch.float32).max * torch.sign(n)
    x[11] = 1e-38 * n
    announce("quantize_rows ties")
    q, s = ops.quantize_rows(x.to(device()))
    wq, ws = int8.quantize_rows(x)
    assert torch.equal(q.cpu(), wq)
    assert torch.equal(s.cpu().isnan(), ws.isnan()) and torch.equal(s.cpu().nan_to_num(), ws.nan_to_num())


@pytest.mark.parametrize("M,K", [(1, 64), (5, 256), (33, 1024), (6, 2048), (3, 4100), (2, 12288)])
@pytest.mark.parametrize("add", [False, True])
def test_norm_codes(M, K, add):
    x, y = rows(M, K, 1), rows(M, K, 2)
    x[:, 0] *= 30
    w = 0.2 * torch.randn(K, generator=torch.Generator().manual_seed(3))
    announce(f"add_rmsnorm_i8 M{M} K{K} add {add}")
    xd = x.to(device())
    q, s = ops.add_rmsnorm_i8_(xd, y.to(device()) if add else None, w.to(device()), 1e-6)
    total = x + y if add else x
    assert torch.equal(xd.cpu(), total)
    wq, ws = int8.quantize_rows(int8.norm_rows(total, w, torch.tensor(1e-6).item()))
    # (64 bits here and there in another order: a quotient within 2^-40 of a half may fall on the other side; none does)
    assert torch.equal(q.cpu(), wq) and torch.equal(s.cpu(), ws)


SHAPES = [(1, 1, 64), (1, 40, 128), (5, 33, 192), (16, 5120, 1024), (31, 129, 64), (32, 1024, 3584), (33, 100, 320),
          (64, 64, 64), (65, 257, 448), (100, 7168, 1024), (127, 130, 1024), (333, 1024, 3584), (700, 1000, 576), (1000, 3000, 256),
          (2100, 8224, 256), (3000, 2050, 1024)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product(M, N, K):
    W, ws = weights(N, K, seed=M)
    q, s = int8.quantize_rows(rows(M, K, seed=N))
    want = int8.product(q, s, W, ws)
    dev = device()
    x = ops.RowsI8(q.to(dev), s.to(dev))
    announce(f"gemm_i8 M{M} N{N} K{K}")
    y = ops.gemm_i8(x, W.to(dev), ws.to(dev))
    check(y, want)
    base = torch.randn(M, N, generator=torch.Generator().manual_seed(5))
    out = base.to(dev)
    assert ops.gemm_i8(x, W.to(dev), ws.to(dev), out=out, epilogue="add") is out
    assert torch.equal(out, base.to(dev) + y)


@pytest.mark.parametrize("M,N,K", [(3, 64, 65536), (70, 130, 65536), (300, 300, 32768)])
def test_largest_sums(M, N, K):
    """Codes of 127 throughout: sums of up to 2^30, which fp32 rounds once."""
    W, ws = weights(N, K, extremes=True)
    q, s = torch.full((M, K), 127, dtype=torch.int8), torch.rand(M, generator=torch.Generator().manual_seed(1)) + 0.5
    dev = device()
    announce(f"gemm_i8 largest sums M{M} N{N} K{K}")
    check(ops.gemm_i8((q.to(dev), s.to(dev)), W.to(dev), ws.to(dev)), int8.product(q, s, W, ws))


@pytest.mark.parametrize("M,T,I,K", [(1, 1, 64, 64), (3, 1, 130, 256), (12, 4, 66, 128), (40, 20, 3584, 1024), (300, 100, 501, 320),
                                     (2100, 700, 4099, 192)])
def test_swiglu_pushes_and_capture(M, T, I, K):
    W, ws = weights(2 * I, K, seed=I)
    q, s = int8.quantize_rows(rows(M, K, seed=K))
    y = int8.product(q, s, W, ws)
    want = int8.swiglu(y)
    slack = 16 + 6 * y[:, 0::2].abs()
    dev = device()
    x = ops.RowsI8(q.to(dev), s.to(dev))
    announce(f"gemm_i8 swiglu M{M} T{T} I{I} K{K}")
    a = ops.gemm_i8(x, W.to(dev), ws.to(dev), epilogue="swiglu")
    check(a, want, slack)
    n = I // 2
    pushes = ops.pack_pushes([(n, "add", [1.0, -2.0, 3.0, 4.0]), (n, "mul", [0.5, 2.0, 3.0, 0.0]), (None, "add", [0.25] * 4),
                              (I + 5, "mul", [0.0] * 4)], dev)
    cap = torch.full((M // T, T + 2, I), 7.0, device=dev)
    b = ops.gemm_i8(x, W.to(dev), ws.to(dev), epilogue="swiglu", pushes=pushes, T=T, capture=cap[:, 1:T + 1])
    r = torch.clamp(torch.arange(M, device=dev) // T, max=3)
    ref = a.clone()
    ref[:, n] = (ref[:, n] + torch.tensor([1.0, -2.0, 3.0, 4.0], device=dev)[r]) * torch.tensor([0.5, 2.0, 3.0, 0.0], device=dev)[r]
    ref += 0.25
    assert torch.allclose(b, ref, rtol=1e-6, atol=1e-12) and torch.equal(cap[:, 1:T + 1].reshape(M, I), b)
    assert bool((cap[:, 0] == 7).all()) and bool((cap[:, T + 1] == 7).all())


def test_strided_rows_and_outputs():
    """Codes as columns of a wider tensor, results into columns of a wider one (other columns left alone), three dims."""
    M, N, K = 70, 100, 128
    W, ws = weights(N, K)
    q, s = int8.quantize_rows(rows(M, K))
    want = int8.product(q, s, W, ws)
    dev = device()
    wide = torch.full((M, K + 48), 77, dtype=torch.int8, device=dev)
    wide[:, 16:16 + K] = q.to(dev)
    out = torch.full((M, N + 7), 5.0, device=dev)
    announce("gemm_i8 strides")
    ops.gemm_i8((wide[:, 16:16 + K], s.to(dev)), W.to(dev), ws.to(dev), out=out[:, 3:3 + N])
    check(out[:, 3:3 + N], want)
    assert bool((out[:, :3] == 5).all()) and bool((out[:, 3 + N:] == 5).all())
    x3 = rows(M, K).view(7, 10, K).to(dev)
    r = ops.quantize_rows(x3)
    y = ops.gemm_i8(r, W.to(dev), ws.to(dev))
    assert r.s.shape == (7, 10) and y.shape == (7, 10, N)
    check(y.view(M, N), want)


def test_rows_that_are_not_finite_stay_their_own():
    M, N, K = 40, 65, 64
    x = rows(M, K)
    x[3, 5], x[39, 0] = float("nan"), float("inf")
    x[7] = 0
    W, ws = weights(N, K)
    dev = device()
    announce("gemm_i8 NaN rows")
    y = ops.gemm_i8(ops.quantize_rows(x.to(dev)), W.to(dev), ws.to(dev)).cpu()
    bad = y.isnan().all(1)
    assert bad.nonzero()[:, 0].tolist() == [3, 39] and not bool(y[~bad].isnan().any()) and bool((y[7] == 0).all())


def test_empty_and_refusals():
    dev = device()
    W, ws = (t.to(dev) for t in weights(10, 64))
    r = ops.quantize_rows(torch.empty(0, 64, device=dev))
    assert r.q.shape == (0, 64) and ops.gemm_i8(r, W, ws).shape == (0, 10)
    x = ops.quantize_rows(rows(4, 64).to(dev))
    announce("gemm_i8 refusals")
    for bad in (lambda: ops.quantize_rows(torch.zeros(2, 6, device=dev)), lambda: ops.quantize_rows(torch.zeros(2, 16388, device=dev)),
                lambda: ops.quantize_rows(torch.zeros(4, 64, device=dev).half()), lambda: ops.quantize_rows(torch.zeros(64, 4, device=dev).T),
                lambda: ops.quantize_rows(torch.zeros(4, 64, device=dev).expand(2, 4, 64)[:, :, :62]),
                lambda: ops.quantize_rows(torch.zeros(4, 64)),
                lambda: ops.add_rmsnorm_i8_(torch.zeros(4, 64, device=dev), None, torch.zeros(63, device=dev)),
                lambda: ops.add_rmsnorm_i8_(torch.zeros(4, 64, device=dev), torch.zeros(4, 60, device=dev), torch.zeros(64, device=dev)),
                lambda: ops.gemm_i8(x, W[:, :32].contiguous(), ws), lambda: ops.gemm_i8((x.q[:, :32].contiguous(), x.s), W[:, :32].contiguous(), ws),
                lambda: ops.gemm_i8((x.q, x.s[:3]), W, ws), lambda: ops.gemm_i8(x, W, ws[:9]), lambda: ops.gemm_i8(x, W.float(), ws),
                lambda: ops.gemm_i8(x, W, ws, epilogue="add"), lambda: ops.gemm_i8(x, W, ws, epilogue="add_fixed"),
                lambda: ops.gemm_i8(x, W, ws, out=torch.zeros(4, 9, device=dev)), lambda: ops.gemm_i8(x, W, ws, out=torch.zeros(10, 4, device=dev).T),
                lambda: ops.gemm_i8(x, W[:9], ws[:9], epilogue="swiglu"), lambda: ops.gemm_i8(x, W, ws, T=0),
                lambda: ops.gemm_i8(x, W, ws, capture=torch.zeros(4, 10, device=dev)),
                lambda: ops.gemm_i8((x.q.cpu(), x.s), W, ws), lambda: ops.gemm_i8(x, W, ws.cpu())):
        with pytest.raises(Q35Error):
            bad()


def test_captured_and_replayed():
    """Norm, quantisation and both products of a block in a graph, replayed on new inputs with eager calls between."""
    dev = device()
    M, K, I = 48, 256, 384
    Wg, sg = (t.to(dev) for t in weights(2 * I, K))
    Wd, sd = (t.to(dev) for t in weights(K, I, 1))
    w = torch.zeros(K, device=dev)
    x = rows(M, K).to(dev)

    def block():
        a = ops.gemm_i8(ops.add_rmsnorm_i8_(x, None, w), Wg, sg, epilogue="swiglu")
        return ops.gemm_i8(ops.quantize_rows(a), Wd, sd)
    announce("gemm_i8 capture")
    block()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block()
    for step in range(3):
        x.copy_(rows(M, K, 10 + step).to(dev))
        graph.replay()
        want = block()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = block()
    a = block()
    torch.cuda.synchronize()
    assert torch.equal(a, b)


@pytest.mark.parametrize("M,N,K", [(700, 1000, 64), (700, 1002, 192), (1000, 3000, 64), (1001, 2998, 448), (2500, 5000, 64),
                                   (2600, 8222, 320), (4100, 8200, 128)])
@pytest.mark.parametrize("epilogue", ["store", "swiglu"])
def test_each_tile(M, N, K, epilogue):
    """Sizes at which tiles of 64, 128 and 256 are chosen, inputs of one stage or less and those that end inside one."""
    W, ws = weights(N, K, seed=N)
    q, s = int8.quantize_rows(rows(M, K, seed=M))
    dev = device()
    announce(f"gemm_i8 tiles M{M} N{N} K{K} {epilogue}")
    y = ops.gemm_i8((q.to(dev), s.to(dev)), W.to(dev), ws.to(dev), epilogue=epilogue).double().cpu()
    v = int8.product(q, s, W, ws)
    if epilogue == "store":
        check(y, v)
        return
    gate, up = v[:, 0::2], v[:, 1::2]
    want = gate * torch.sigmoid(gate) * up
    assert bool(((y - want).abs() <= (12 + 8 * gate.abs()) * H * want.abs() + 1e-37).all())


@pytest.mark.parametrize("M,N", [(600, 900), (1100, 2100), (2500, 5000)])
def test_largest_sums_of_each_tile(M, N):
    K = 4096
    W, ws = weights(N, K, extremes=True)
    q, s = torch.full((M, K), -127, dtype=torch.int8), torch.rand(M, generator=torch.Generator().manual_seed(1)) + 0.5
    dev = device()
    announce(f"gemm_i8 largest sums M{M} N{N} K{K}")
    check(ops.gemm_i8((q.to(dev), s.to(dev)), W.to(dev), ws.to(dev)), int8.product(q, s, W, ws))


@pytest.mark.parametrize("M,K", [(2100, 516), (2048, 1000), (2300, 1024), (40, 1024), (40, 300), (12, 4096), (5, 8196)])
def test_codes_far_from_one(M, K):
    """Rows and gains over the whole range: what fp32 alone would lose is formed in 64 bits. Many rows of up to 1024 values are a
    wave's each, others a block's."""
    g = torch.Generator().manual_seed(M + K)
    x = torch.randn(M, K, generator=g)
    x[0::7] *= 1e-30
    x[1::7] *= 1e30
    x[2::7] *= torch.logspace(-20, 20, K)
    x[3::7, ::3] = 0.0
    x[4::7] = (torch.randint(-254, 255, (x[4::7].shape[0], K), generator=g).float() * 0.5)  # codes and halves
    x[4::7, 0] = 127.0
    w = torch.randn(K, generator=g) * 0.1
    w[:6] = torch.tensor([-1.0, -1.0000001, -0.99999994, 1e30, 1e-30, -1e25])
    dev = device()
    announce(f"rows in 8 bits far from one M{M} K{K}")
    q, s = ops.quantize_rows(x.to(dev))
    wq, ws = int8.quantize_rows(x)
    assert torch.equal(q.cpu(), wq) and torch.equal(s.cpu(), ws)
    for gain in (w, torch.cat([w[:3], w[6:9], w[6:]])[:K]):
        xd = x.to(dev)
        q, s = ops.add_rmsnorm_i8_(xd, None, gain.to(dev))
        wq, ws = int8.quantize_rows(int8.norm_rows(x, gain, torch.tensor(1e-6).item()))  # (eps is an fp32 argument)
        assert torch.equal(xd.cpu(), x)
        assert torch.equal(s.cpu(), ws) and torch.equal(q.cpu(), wq)
