"""Per-token quantisation and the scaled int8 product against a plain 64-bit
implementation.  Codes and scales are bit-exact; the product's tolerance is
derived from its roundings."""
import ctypes
from concurrent.futures import ThreadPoolExecutor

import numpy as np
import pytest
import torch

from iconnx_b200 import IcxError, _lib, ops
from tests import decoder_reference as ref

DEV = "cuda:0"
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def f64(t):
    return t.detach().cpu().double().numpy()


def rows(shape, dtype, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp(spread * torch.randn(shape[0], 1, generator=g))
    return x.to(dtype)


# ---------------------------------------------------------------- refusals
def test_quantize_refusals_before_any_launch():
    L = _lib.load()
    p = ctypes.c_void_p(16)
    assert L.icx_quantize_per_token(None, p, 1, 4, 8, 8, p, p) == -1
    assert b"must be Float32, Float16 or BFloat16" in L.icx_last_error()
    assert L.icx_quantize_per_token(None, p, 3, 4, 8, 7, p, p) == -1
    assert b"row stride" in L.icx_last_error()
    assert L.icx_quantize_per_token(None, None, 3, 4, 8, 8, p, p) == -1
    assert b"null" in L.icx_last_error()
    assert L.icx_quantize_per_token(None, None, 3, 0, 8, 8, None, None) == 0
    with pytest.raises(IcxError, match="expected a CUDA tensor"):
        ops.gpu_quantize_per_token(torch.zeros(2, 3))


def test_product_refusals_before_any_launch():
    L = _lib.load()
    p = ctypes.c_void_p(16)

    def call(q=p, M=2, K=4, N=3, t=3, out=p):
        return L.icx_matmul_integer_scaled(None, q, p, p, M, K, N, p, None, None, t, out)

    assert call(t=2) == -1 and b"output must be" in L.icx_last_error()
    assert call(K=_lib.ICX_SCALED_MAX_K + 1) == -1 and b"could wrap" in L.icx_last_error()
    assert call(M=1 << 22) == -1 and b"too large" in L.icx_last_error()
    assert call(M=65535 * 64 + 1) == -1 and b"too large" in L.icx_last_error()
    assert call(q=None) == -1 and b"null" in L.icx_last_error()
    assert call(out=None) == -1 and b"null" in L.icx_last_error()
    assert call(M=0, q=None, out=None) == 0


@pytest.mark.gpu
def test_python_refusals():
    x = torch.zeros(4, 8, device=DEV)
    for bad in (x.int(), x.double(), x[0, 0]):
        with pytest.raises(IcxError):
            ops.gpu_quantize_per_token(bad)
    q = torch.zeros(4, 8, dtype=torch.int8, device=DEV)
    s, ws = torch.ones(4, device=DEV), torch.ones(6, device=DEV)
    w = ops.prepare_weight(torch.zeros(8, 6, dtype=torch.int8, device=DEV))
    wu = ops.prepare_weight(torch.zeros(8, 6, dtype=torch.uint8, device=DEV))
    good = dict(bias=None, residual=None)
    ops.gpu_matmul_integer_scaled(q, s, w, ws, **good)
    for args, kw in [((q.float(), s, w, ws), {}), ((q[:, :7], s, w, ws), {}), ((q, s[:3], w, ws), {}),
                     ((q, s, wu, ws), {}), ((q, s, w, ws[:1]), {}), ((q, s.half(), w, ws), {}),
                     ((q, s.cpu(), w, ws), {}), ((q, s, w, ws), dict(bias=ws[:5])),
                     ((q, s, w, ws), dict(residual=torch.zeros(4, 6, device=DEV), out_dtype=torch.float16)),
                     ((q, s, w, ws), dict(out_dtype=torch.int32))]:
        with pytest.raises(IcxError):
            ops.gpu_matmul_integer_scaled(*args, **kw)


# ------------------------------------------------------------ quantisation
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 768), (3, 7), (5, 33), (17, 257), (4, 1000), (300, 768),
                                   (2, 8192), (3, 8195), (2, 16384), (2, 40000), (1, 70001)])
def test_quantize_bit_exact(shape, dtype):
    x = rows(shape, dtype, shape[0] * 1000 + shape[1])
    q, s = ops.gpu_quantize_per_token(x.to(DEV))
    rq, rs = ref.quantize_per_token(f64(x))
    assert q.dtype == torch.int8 and s.dtype == torch.float32
    np.testing.assert_array_equal(s.cpu().numpy(), rs)
    np.testing.assert_array_equal(q.cpu().numpy(), rq)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_special_rows(dtype):
    x = rows((12, 96), torch.float32, 5)
    x[0] = 0
    x[1, 7] = float("nan")
    x[2, 95] = float("inf")
    x[3, 0] = float("-inf")
    x[4] = -0.0
    x[5] = torch.arange(96) - 47.5          # scale 48.5 / 127
    x[6] = (torch.arange(96) - 48) * 0.5    # every other quotient a tie
    x[6, 0] = 127.0
    x[7] = 6e-8
    x[8] *= 1e-40                           # subnormal f32, zero in f16
    x[9] = 2e-45
    x[10] *= 1000.0
    x = x.to(dtype)
    q, s = ops.gpu_quantize_per_token(x.to(DEV))
    rq, rs = ref.quantize_per_token(f64(x))
    np.testing.assert_array_equal(s.cpu().numpy(), rs)
    np.testing.assert_array_equal(q.cpu().numpy(), rq)


@pytest.mark.gpu
def test_quantize_ties_and_largest_values():
    top = torch.finfo(torch.float32).max
    k = torch.arange(-127, 127, dtype=torch.float64) + 0.5
    for s in (1.0, 2.0 ** -100, 2.0 ** -149 * 6, 0.1, 1.2345e30):
        s = float(np.float32(s))
        x = torch.cat([(k * s).float(), torch.tensor([127 * s], dtype=torch.float64).float()])[None]
        near = torch.nextafter(x, torch.full_like(x, float("inf")))
        both = torch.cat([x, near, torch.full_like(x, top)])
        q, sc = ops.gpu_quantize_per_token(both.to(DEV))
        rq, rs = ref.quantize_per_token(f64(both))
        np.testing.assert_array_equal(sc.cpu().numpy(), rs)
        np.testing.assert_array_equal(q.cpu().numpy(), rq)


@pytest.mark.gpu
def test_quantize_views_shapes_and_empties():
    base = rows((20, 120), torch.bfloat16, 3).to(DEV)
    for view in (base[:, 3:100], base[::2, :64], base[:, ::2], base.t(), base.reshape(4, 5, 120),
                 base[1:, 1:], base[3], base[:1].expand(6, 120)):
        q, s = ops.gpu_quantize_per_token(view)
        c = view.cpu()
        rq, rs = ref.quantize_per_token(f64(c.reshape(-1, c.shape[-1])))
        assert q.shape == view.shape and s.shape == view.shape[:-1]
        np.testing.assert_array_equal(q.cpu().numpy().reshape(rq.shape), rq)
        np.testing.assert_array_equal(s.cpu().numpy().reshape(-1), rs)
    q, s = ops.gpu_quantize_per_token(base[:0])
    assert q.shape == (0, 120) and s.shape == (0,)
    q, s = ops.gpu_quantize_per_token(base[:, :0])
    assert q.shape == (20, 0) and (s == 0).all()


# ----------------------------------------------------------------- product
def product_case(M, K, N, dtype, bias, residual, seed, peak=127):
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(-peak, peak + 1, (M, K), generator=g, dtype=torch.int8)
    w = torch.randint(-128, 128, (K, N), generator=g, dtype=torch.int8)
    sa, sw = torch.rand(M, generator=g) + 0.1, (torch.rand(N, generator=g) + 0.1) / (5000 * max(K, 1) ** 0.5)
    b = torch.randn(N, generator=g) if bias else None
    r = torch.randn(M, N, generator=g).to(dtype) if residual else None
    return q, sa, w, sw, b, r


def check_product(M, K, N, dtype, bias=False, residual=False, seed=0, lead=None):
    q, sa, w, sw, b, r = product_case(M, K, N, dtype, bias, residual, seed)
    cu = [None if t is None else t.to(DEV) for t in (q, sa, w, sw, b, r)]
    if lead:
        cu[0], cu[1] = cu[0].reshape(*lead, K), cu[1].reshape(lead)
        cu[5] = cu[5].reshape(*lead, N) if residual else None
    out = ops.gpu_matmul_integer_scaled(cu[0], cu[1], ops.prepare_weight(cu[2]), cu[3], cu[4], cu[5], dtype)
    assert out.shape == (*(lead or (M,)), N) and out.dtype == dtype
    acc, want = ref.scaled_product(q.numpy(), sa.numpy(), w.numpy(), sw.numpy(),
                                   None if b is None else b.numpy(), None if r is None else f64(r))
    # f32: the sum, two products and up to two additions each round once (2^-24 of
    # the largest of the terms); then one rounding to the output type
    terms = np.abs(acc * f64(sa)[:, None] * f64(sw)) + (np.abs(f64(b)) if bias else 0) + (np.abs(f64(r)) if residual else 0)
    tol = 5 * 2.0 ** -24 * terms
    tol = ref.rounding(want, tol, dtype)
    got = f64(out).reshape(want.shape)
    assert (np.abs(got - want) <= tol).all(), np.abs(got - want).max()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", [(1, 1, 1), (1, 16, 8), (1, 768, 768), (2, 4096, 1024), (3, 77, 33),
                                   (4, 1000, 513), (7, 2048, 130), (8, 64, 2311), (9, 512, 96), (16, 768, 2304),
                                   (17, 4096, 200), (33, 48, 250), (48, 1040, 384), (64, 2064, 257),
                                   (65, 768, 128), (100, 100, 100), (129, 33, 65), (200, 4112, 300),
                                   (257, 768, 777), (128, 128, 128), (300, 32, 1)])
def test_product_sizes(M, K, N, dtype):
    check_product(M, K, N, dtype, seed=M + K + N)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", [(1, 512, 100), (5, 77, 64), (20, 512, 250), (130, 768, 260), (700, 272, 1001)])
@pytest.mark.parametrize("bias,residual", [(True, False), (False, True), (True, True)])
def test_product_bias_residual(M, K, N, dtype, bias, residual):
    check_product(M, K, N, dtype, bias, residual, seed=M)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [2, 40, 300])
def test_product_largest_sum_is_exact(M):
    """Every product at its largest: the s32 sum neither wraps nor loses bits."""
    K, N = 131056, 24
    q = torch.full((M, K), -128, dtype=torch.int8, device=DEV)
    w = torch.full((K, N), -128, dtype=torch.int8, device=DEV)
    out = ops.gpu_matmul_integer_scaled(q, torch.full((M,), 2.0 ** -14, device=DEV), ops.prepare_weight(w),
                                        torch.ones(N, device=DEV))
    assert (out == float(K)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N", [(1, 127, 1), (2, 129, 63), (3, 1633, 130), (5, 2049, 64), (63, 4099, 65),
                                   (64, 255, 700), (130, 1031, 200), (1000, 515, 129), (8, 7425, 520)])
def test_product_any_k(M, K, N):
    """Rows that start at every byte, and K shared out between CTAs."""
    check_product(M, K, N, torch.float32, True, True, seed=M + K)


@pytest.mark.gpu
@pytest.mark.parametrize("at", [1, 2, 3, 8])
def test_product_operands_at_any_byte(at):
    """q and the weight inside larger buffers whose bytes around them must not count."""
    M, K, N = 6, 640, 70
    q, sa, w, sw, _, _ = product_case(M, K, N, torch.float32, False, False, seed=at)
    buf = torch.full((M * K + 32,), 99, dtype=torch.int8, device=DEV)
    view = buf[at:at + M * K].view(M, K)
    view.copy_(q)
    L, out = _lib.load(), torch.empty(M, N, device=DEV)
    wt = torch.full((N * K + 32,), 77, dtype=torch.int8, device=DEV)
    wt[at:at + N * K].view(N, K).copy_(w.t())
    ptr = lambda t, d=0: ctypes.c_void_p(t.data_ptr() + d)
    csa, csw = sa.to(DEV), sw.to(DEV)
    assert L.icx_matmul_integer_scaled(None, ptr(buf, at), ptr(csa), ptr(wt, at), M, K, N, ptr(csw), None, None,
                                       _lib.ICX_F32, ptr(out)) == 0
    torch.cuda.synchronize()
    acc, want = ref.scaled_product(q.numpy(), sa.numpy(), w.numpy(), sw.numpy(), None, None)
    tol = 5 * 2.0 ** -24 * np.abs(acc * f64(sa)[:, None] * f64(sw))
    assert (np.abs(f64(out) - want) <= ref.rounding(want, tol, torch.float32)).all()


@pytest.mark.gpu
def test_product_large_tiles_and_leading_axes():
    check_product(1500, 768, 2304, torch.bfloat16, True, True, seed=1)
    check_product(8320, 1600, 520, torch.float16, seed=2)
    check_product(8320, 272, 384, torch.float32, residual=True, seed=3)
    check_product(24, 96, 40, torch.float32, True, True, seed=4, lead=(2, 3, 4))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N", [(8320, 8192), (300, 14336), (1500, 6144)])
def test_product_residual_where_a_warp_has_no_rows(M, N, dtype):
    """More tiles than CTAs, and a last token tile that leaves some warps (8320: a
    whole CTA of a pair) without a token: what the tile before still has to
    store must not be touched.  Integers, so that f32 and bf16 hold every sum."""
    K, top = 64, 100
    g = torch.Generator(DEV).manual_seed(M)
    q = torch.randint(-1, 2, (M, K), generator=g, device=DEV, dtype=torch.int8)
    w = torch.randint(-1, 2, (K, N), generator=g, device=DEV, dtype=torch.int8)
    r = torch.randint(-top, top + 1, (M, N), generator=g, device=DEV).to(dtype)
    one, pw = torch.ones(M, device=DEV), ops.prepare_weight(w)
    # at most 64 + 100: exact in every type
    want = ((q.float() @ w.float()) + r.float()).to(dtype)
    for _ in range(20):
        out = ops.gpu_matmul_integer_scaled(q, one, pw, torch.ones(N, device=DEV), residual=r, out_dtype=dtype)
        assert torch.equal(out, want)


@pytest.mark.gpu
def test_product_empties_and_nan_rows():
    w = ops.prepare_weight(torch.ones(32, 5, dtype=torch.int8, device=DEV))
    ws, bias = torch.ones(5, device=DEV), torch.arange(5.0, device=DEV)
    out = ops.gpu_matmul_integer_scaled(torch.zeros(0, 32, dtype=torch.int8, device=DEV), torch.zeros(0, device=DEV), w, ws)
    assert out.shape == (0, 5)
    w0 = ops.PreparedWeight(torch.empty(5, 0, dtype=torch.int8, device=DEV),
                            torch.zeros(5, dtype=torch.int32, device=DEV), 0, 5, torch.int8)
    out = ops.gpu_matmul_integer_scaled(torch.zeros(3, 0, dtype=torch.int8, device=DEV), torch.ones(3, device=DEV),
                                        w0, ws, bias)
    assert torch.equal(out, bias.expand(3, 5))
    x = torch.randn(70, 32, device=DEV)
    x[3, 4] = float("nan")
    x[66, 0] = float("inf")
    q, s = ops.gpu_quantize_per_token(x)
    out = ops.gpu_matmul_integer_scaled(q, s, w, ws, bias)
    bad = torch.zeros(70, dtype=torch.bool, device=DEV)
    bad[[3, 66]] = True
    assert torch.equal(out.isnan().any(1), bad) and torch.equal(out.isnan().all(1), bad)


@pytest.mark.gpu
def test_unaligned_operands():
    """Operands that start off a 16-byte boundary take the kernels for any alignment."""
    K, N = 64, 48
    g = torch.Generator(DEV).manual_seed(1)
    flat = torch.randint(-127, 128, (9 * K + 5,), generator=g, device=DEV, dtype=torch.int8)
    q = flat[5:].view(9, K)
    sflat = torch.rand(10, generator=g, device=DEV)
    w = torch.randint(-127, 128, (K, N), generator=g, device=DEV, dtype=torch.int8)
    wp = ops.prepare_weight(w)
    wsflat = torch.rand(N + 1, generator=g, device=DEV)
    got = ops.gpu_matmul_integer_scaled(q, sflat[1:], wp, wsflat[1:], bias=wsflat[:N], out_dtype=torch.float32)
    want = ops.gpu_matmul_integer_scaled(q.clone(), sflat[1:].clone(), wp, wsflat[1:].clone(), bias=wsflat[:N].clone())
    assert torch.equal(got, want)
    x = torch.randn(3 * 70 + 1, generator=g, device=DEV)[1:].view(3, 70)
    for dt in TYPES:
        a, b = ops.gpu_quantize_per_token(x.to(dt)), ops.gpu_quantize_per_token(
            torch.cat([torch.zeros(1, device=DEV, dtype=dt), x.to(dt).flatten()])[1:].view(3, 70))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.gpu
def test_calls_from_several_threads():
    """The first calls that need a kernel's limits, from threads at once."""
    M, K, N = 2048, 64, 512
    g = torch.Generator(DEV).manual_seed(3)
    q = torch.randint(-9, 10, (M, K), generator=g, device=DEV, dtype=torch.int8)
    w = torch.randint(-9, 10, (K, N), generator=g, device=DEV, dtype=torch.int8)
    pw, one, ws = ops.prepare_weight(w), torch.ones(M, device=DEV), torch.ones(N, device=DEV)
    want = q.float() @ w.float()   # at most 64 * 81
    torch.cuda.synchronize()

    def call(i):
        with torch.cuda.stream(torch.cuda.Stream(DEV)):
            out = ops.gpu_matmul_integer_scaled(q, one, pw, ws, out_dtype=TYPES[i % 2])
            torch.cuda.current_stream(DEV).synchronize()
            return torch.equal(out.float(), want.to(TYPES[i % 2]).float())

    with ThreadPoolExecutor(8) as pool:
        assert all(pool.map(call, range(32)))


@pytest.mark.gpu
def test_other_stream_and_graph_replay():
    x = rows((37, 512), torch.bfloat16, 9).to(DEV)
    w = ops.prepare_weight(torch.randint(-127, 128, (512, 300), dtype=torch.int8, device=DEV))
    ws = torch.rand(300, device=DEV)

    def layer(x):
        q, s = ops.gpu_quantize_per_token(x)
        return ops.gpu_matmul_integer_scaled(q, s, w, ws, out_dtype=torch.bfloat16)

    want = layer(x)
    torch.cuda.synchronize()
    side = torch.cuda.Stream(DEV)
    with torch.cuda.stream(side):
        got = layer(x)
    side.synchronize()
    assert torch.equal(got, want)
    buf = torch.zeros_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(buf)
    buf.copy_(x)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
