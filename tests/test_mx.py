"""Microscaled 4-bit floats: quantisation, its inverse and the product.

The oracle is written from the format's definition in float64 (numpy, on the
CPU).  Quantisation and its inverse are compared bit for bit; a product is off
by at most half a step of its type plus the fp32 sum's own error.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

import nibblegemm_amd as ng
from nibblegemm_amd import mx

INVALID, WORKSPACE = 1, 3
P = 1 << 20  # aligned, never dereferenced
dev = "cuda"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
DTYPES = [F16, BF16, F32]
GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


# ---------------------------------------------------------------------------
# the oracle
# ---------------------------------------------------------------------------
def oracle_quantize(x: torch.Tensor):
    """Codes [rows, K] and biased exponents [rows, K / 32] by the definition."""
    v = x.detach().to("cpu", torch.float64).numpy().reshape(x.shape[0], -1, 32)
    top = np.abs(v).max(-1)
    good = np.isfinite(top)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.where(good & (top > 0), np.floor(np.log2(np.where(good & (top > 0), top, 1))) - 2,
                     -127)
    # log2 of a value next to a power of two may round up to it
    e = np.where(good & (top > 0) & (np.ldexp(1.0, (e + 2).astype(int)) > top), e - 1, e)
    e = np.maximum(e, -127).astype(int)
    u = np.where(good[..., None], v, 0.0) / np.ldexp(1.0, e)[..., None]
    dist = np.abs(np.abs(u)[..., None] - GRID)
    best = dist.min(-1, keepdims=True)
    near = dist == best  # two where u is halfway: the even code
    first = near.argmax(-1)
    last = 7 - near[..., ::-1].argmax(-1)
    code = np.where(first % 2 == 0, first, last)
    code = code + 8 * np.signbit(u)
    return (code.reshape(x.shape).astype(np.uint8),
            np.where(good, e + 127, 255).astype(np.uint8))


def oracle_values(code: np.ndarray, biased: np.ndarray) -> np.ndarray:
    v = np.where(code & 8, -1.0, 1.0) * GRID[code & 7]
    e = np.repeat(biased.astype(int), 32, axis=1)
    return np.where(e == 255, np.nan, np.ldexp(v, e - 127))


def unpack(m: ng.MXMatrix):
    c = m.codes.cpu().numpy()
    code = np.stack([c & 15, c >> 4], -1).reshape(m.rows, m.K)
    return code, m.block_scales().cpu().numpy()


def values64(m: ng.MXMatrix) -> np.ndarray:
    return oracle_values(*unpack(m))


def check_quantized(m: ng.MXMatrix, x: torch.Tensor):
    code, biased = unpack(m)
    want_code, want_biased = oracle_quantize(x)
    assert np.array_equal(biased, want_biased)
    assert np.array_equal(code, want_code)
    rest = m.scales.transpose(0, 1).reshape(m.rows, -1)[:, m.K // 32:]
    assert not rest.any(), "the words are zero behind the last block"


def sample(rows, K, dtype, seed=0, wide=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, K), generator=g)
    if wide:  # blocks of very different sizes, some of zeros
        x = x * torch.exp2(torch.randint(-18, 12, (rows, K // 32, 1), generator=g).float()).expand(
            rows, K // 32, 32).reshape(rows, K)
        x[torch.rand((rows, K), generator=g) < 0.1] = 0.0
        x.view(rows, -1, 32)[torch.rand((rows, K // 32), generator=g) < 0.1] = 0.0
    return x.to(dtype)


def ties(dtype):
    """Every eighth of a step from -8 to 8 of several powers of two, with the
    block's largest value fixed at 4 steps of it."""
    u = torch.arange(-62, 63) / 8.0
    rows = []
    for e in (-14, -3, 0, 5, 12):
        for lo in range(0, len(u), 31):
            b = torch.full((32,), 4.0)
            part = u[lo:lo + 31]
            b[:len(part)] = part
            rows.append(b * 2.0 ** e)
    return torch.stack(rows).to(dtype)


# ---------------------------------------------------------------------------
# format and refusals (CPU)
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,K", [(1, 32), (3, 96), (5, 160), (2, 512)])
def test_host_quantize_is_the_definition(rows, K, dtype):
    for wide in (False, True):
        x = sample(rows, K, dtype, seed=K, wide=wide)
        m = ng.quantize_mx(x)
        assert m.scales.shape == (-(-K // 128), rows, 4) and m.codes.shape == (rows, K // 2)
        check_quantized(m, x)
        got = ng.dequantize_mx(m, F32).double().numpy()
        assert np.array_equal(got, values64(m), equal_nan=True)


def special_rows():
    x = torch.zeros((9, 64))
    x[0, 3] = float("inf")
    x[1, 40] = float("nan")
    x[2, 0] = -float("inf")
    x[2, 1] = float("nan")
    x[3] = -0.0
    x[4, 5] = torch.finfo(F32).max
    x[5, 7] = 2.0 ** -149
    x[6, :8] = torch.tensor([1.0, 2, 3, 4, 5, 6, 7, 0.5]) * 2.0 ** -129  # subnormal values
    x[7, :4] = torch.tensor([2.0 ** -126, 2.0 ** -125, -2.0 ** -127, 2.0 ** -128])
    x[8, 32:34] = torch.tensor([7.999, -7.0001])  # beyond 6 in a block of exponent 0
    return x


def test_host_quantize_of_special_values():
    x = special_rows()
    check_quantized(ng.quantize_mx(x), x)
    for dtype in DTYPES:
        check_quantized(ng.quantize_mx(ties(dtype)), ties(dtype))
    v = ng.dequantize_mx(ng.quantize_mx(x), F32)
    assert v[0, :32].isnan().all() and not v[0, 32:].any()
    assert v[1, 32:].isnan().all() and v[2, :32].isnan().all()


def test_from_blocks_and_back():
    m = ng.quantize_mx(sample(5, 288, F32, seed=3))
    again = ng.mx_from_blocks(m.codes, m.block_scales())
    assert torch.equal(again.scales, m.scales) and again.K == 288 and again.rows == 5
    assert m.nbytes == 5 * 144 + 3 * 5 * 4
    with pytest.raises(ValueError, match="rows"):
        ng.mx_from_blocks(m.codes[:, :-1], m.block_scales())
    with pytest.raises(RuntimeError, match="uint8"):
        ng.mx_from_blocks(m.codes.int(), m.block_scales())


def test_refusals():
    with pytest.raises(ValueError, match="divisible by 32"):
        ng.quantize_mx(torch.zeros(2, 40))
    with pytest.raises(ValueError, match="2-D"):
        ng.quantize_mx(torch.zeros(64))
    with pytest.raises(RuntimeError, match="fp16, bf16 or fp32"):
        ng.quantize_mx(torch.zeros((2, 64), dtype=torch.float64))
    x = torch.zeros((2, 64), requires_grad=True)
    with pytest.raises(RuntimeError, match="no backward"):
        ng.quantize_mx(x)
    with torch.no_grad():
        ng.quantize_mx(x)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(torch.zeros(2, 64), torch.ones(2, 64))
        with pytest.raises(RuntimeError, match="no backward"):
            ng.quantize_mx(dual)
    m = ng.quantize_mx(torch.zeros(2, 64))
    with pytest.raises(RuntimeError, match="on the GPU"):
        ng.matmul_mx(torch.zeros(2, 64), m)
    with pytest.raises(RuntimeError, match="fp16, bf16 or fp32"):
        ng.dequantize_mx(m, torch.float64)
    for bad, error in [(mx.MXMatrix(m.codes.int(), m.scales, 2, 64), RuntimeError),
                       (mx.MXMatrix(m.codes, m.scales[:, :1], 2, 64), ValueError),
                       (mx.MXMatrix(m.codes, m.scales, 3, 64), ValueError),
                       (mx.MXMatrix(m.codes, m.scales, 2, 128), ValueError),
                       (mx.MXMatrix(m.codes.t().contiguous().t(), m.scales, 2, 64), RuntimeError)]:
        with pytest.raises(error):
            ng.dequantize_mx(bad)


def quant(ext, X=P, rows=4, K=128, rs=128, ks=1, dt=0, c=P, s=P):
    return ext.mx_quantize(X, rows, K, rs, ks, dt, c, s, None)


def prod(ext, xc=P, xs=P, M=4, wc=P, ws=P, N=64, K=128, dt=0, Y=P):
    return ext.mx_matmul(xc, xs, M, wc, ws, N, K, dt, Y, None)


@pytest.mark.parametrize("call,needle", [
    (lambda e: quant(e, K=48), "multiple of 32"),
    (lambda e: quant(e, rows=-1), "negative"),
    (lambda e: quant(e, dt=3), "dtype"),
    (lambda e: quant(e, rs=2, ks=2), "strides"),
    (lambda e: quant(e, rs=0), "strides"),
    (lambda e: quant(e, X=P + 1), "misaligned"),
    (lambda e: quant(e, c=P + 8), "misaligned"),
    (lambda e: quant(e, s=P + 2), "misaligned"),
    (lambda e: quant(e, X=0), "null"),
    (lambda e: quant(e, rows=1 << 28, K=1024, rs=1024), "2^31"),
    (lambda e: quant(e, K=1 << 25, rs=1 << 25), "K above"),
    (lambda e: e.mx_dequantize(P, P, 4, 128, 5, P, None), "dtype"),
    (lambda e: e.mx_dequantize(P, P, 4, 100, 0, P, None), "multiple of 32"),
    (lambda e: e.mx_dequantize(P, P, 4, 128, 0, P + 8, None), "misaligned"),
    (lambda e: e.mx_dequantize(P, 0, 4, 128, 0, P, None), "null"),
    (lambda e: prod(e, K=100), "multiple of 32"),
    (lambda e: prod(e, M=-1), "negative"),
    (lambda e: prod(e, N=-1), "negative"),
    (lambda e: prod(e, dt=-1), "dtype"),
    (lambda e: prod(e, xc=0), "null"),
    (lambda e: prod(e, Y=0), "null"),
    (lambda e: prod(e, wc=P + 8), "misaligned"),
    (lambda e: prod(e, xs=P + 2), "misaligned"),
    (lambda e: prod(e, Y=P + 8), "misaligned"),
    (lambda e: prod(e, N=1 << 28, K=1024), "2^31"),
])
def test_library_rejections(call, needle):
    ext = ng.extension()
    assert call(ext) == INVALID
    assert needle in ext.last_error()


def dense(ext, X=P, M=2, rs=128, xdt=0, wc=P, ws=P, N=64, K=128, dt=0, Y=P, work=0, size=0):
    return ext.mx_matmul_dense(X, M, rs, xdt, wc, ws, N, K, dt, Y, work, size, None)


@pytest.mark.parametrize("kwargs,needle,status", [
    (dict(K=100), "multiple of 32", INVALID),
    (dict(xdt=3), "dtype", INVALID),
    (dict(dt=3), "dtype", INVALID),
    (dict(M=-1), "negative", INVALID),
    (dict(X=0), "null", INVALID),
    (dict(ws=0), "null", INVALID),
    (dict(rs=-1), "row_stride", INVALID),
    (dict(rs=1 << 62), "row_stride", INVALID),
    (dict(wc=P + 8), "misaligned", INVALID),
    # quantised into a workspace first
    (dict(rs=132), "workspace, got 0", WORKSPACE),
    (dict(X=P + 8), "workspace, got 0", WORKSPACE),
    (dict(rs=1 << 30), "workspace, got 0", WORKSPACE),
    (dict(M=17), "workspace, got 0", WORKSPACE),
    (dict(M=17, size=1 << 20), "workspace, got 0", WORKSPACE),
    (dict(M=17, work=P, size=17 * 68 - 1), "needs 1156 bytes", WORKSPACE),
    (dict(N=1 << 20, work=P, size=100), "workspace, got 100", WORKSPACE),
    (dict(M=17, work=P + 8, size=1 << 20), "16-byte", WORKSPACE),
    (dict(M=17, work=P, size=1 << 20, X=0), "null", INVALID),
    (dict(M=17, work=P, size=1 << 20, X=P + 1), "misaligned", INVALID),
    (dict(M=17, work=P, size=1 << 20, Y=P + 8), "misaligned", INVALID),
    (dict(M=17, work=P, size=1 << 20, ws=0), "null", INVALID),
    (dict(M=17, work=P, size=1 << 20, rs=0), "strides", INVALID),
])
def test_dense_rejections(kwargs, needle, status):
    ext = ng.extension()
    assert dense(ext, **kwargs) == status
    assert needle in ext.last_error()


def test_dense_workspace():
    need = ng.extension().mx_matmul_dense_workspace_bytes
    for M, N, K in [(1, 1024, 4096), (16, 4096, 4096), (1, 12288, 32), (16, 12288, 1024), (5, 8192, 2048)]:
        assert need(M, N, K, True) == 0  # one launch
        assert need(M, N, K, False) == M * (K // 2 + -(-K // 128) * 4)
    for M, N, K in [(17, 1024, 4096), (1, 28672, 4096), (1, 4097, 4096), (1, 4096, 4128), (1, 12289, 1024)]:
        assert need(M, N, K, True) == need(M, N, K, False) == M * (K // 2 + -(-K // 128) * 4)
    assert need(0, 64, 128, True) == need(64, 0, 128, True) == need(64, 64, 0, False) == 0
    assert need(17, 64, 100, True) == 0  # a refused product


def test_library_takes_empty_sizes():
    ext = ng.extension()
    assert dense(ext, M=0, X=0) == 0 and dense(ext, N=0, wc=0) == 0
    assert quant(ext, rows=0, X=0) == 0 and quant(ext, K=0, X=0) == 0
    assert ext.mx_dequantize(0, 0, 0, 128, 0, 0, None) == 0
    assert prod(ext, M=0, xc=0) == 0 and prod(ext, N=0, wc=0) == 0


# ---------------------------------------------------------------------------
# quantisation and its inverse (GPU)
# ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,K", [(1, 32), (1, 4096), (3, 96), (31, 480), (33, 544), (130, 1056),
                                    (257, 2048), (1000, 128)])
def test_quantize_rows(rows, K, dtype):
    x = sample(rows, K, dtype, seed=rows, wide=True)
    check_quantized(ng.quantize_mx(x.to(dev)), x)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,K", [(2, 32), (3, 96), (127, 160), (128, 512), (301, 1056)])
def test_quantize_transposed_views(rows, K, dtype):
    x = sample(rows, K, dtype, seed=rows + 1, wide=True)
    kn = x.t().contiguous().to(dev)
    assert not kn.t().is_contiguous()
    check_quantized(ng.quantize_mx(kn.t()), x)
    # columns of a wider matrix, from an odd one on
    wide = torch.zeros((K, rows + 7), dtype=dtype, device=dev)
    wide[:, 3:3 + rows] = kn
    check_quantized(ng.quantize_mx(wide[:, 3:3 + rows].t()), x)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_other_strides(dtype):
    x = sample(37, 192, dtype, seed=5)
    buf = torch.zeros((37, 211), dtype=dtype, device=dev)
    for first in (0, 3, 8):  # rows of an odd pitch, from aligned and other columns on
        buf[:, first:first + 192] = x.to(dev)
        check_quantized(ng.quantize_mx(buf[:, first:first + 192]), x)
    both = torch.zeros((74, 384), dtype=dtype, device=dev)
    both[::2, ::2] = x.to(dev)
    check_quantized(ng.quantize_mx(both[::2, ::2]), x)
    one = x[:1].to(dev).expand(37, 192)  # a stride of zero
    check_quantized(ng.quantize_mx(one), x[:1].expand(37, 192))
    if dtype == F32:
        z = torch.complex(torch.zeros_like(x), x).to(dev)
        assert z.conj().imag.is_neg()
        check_quantized(ng.quantize_mx(z.conj().imag), -x)


@pytest.mark.gpu
def test_quantize_special_values():
    x = special_rows()
    for t in (x.to(dev), x.t().contiguous().to(dev).t()):
        m = ng.quantize_mx(t)
        check_quantized(m, x)
        for dtype in DTYPES:
            got = ng.dequantize_mx(m, dtype).cpu()
            want = torch.from_numpy(values64(m)).float().to(dtype)
            assert torch.equal(got.isnan(), want.isnan())
            assert torch.equal(got[~got.isnan()], want[~want.isnan()])
    for dtype in DTYPES:
        check_quantized(ng.quantize_mx(ties(dtype).to(dev)), ties(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_every_code_at_every_scale(dtype):
    """All 256 bytes of two codes, against every exponent."""
    codes = torch.arange(256, dtype=torch.uint8).repeat(256, 1)
    scales = torch.arange(256, dtype=torch.uint8)[:, None].expand(256, 16)
    m = ng.mx_from_blocks(codes, scales).to(dev)
    got = ng.dequantize_mx(m, dtype).cpu()
    want = torch.from_numpy(values64(m)).float().to(dtype)
    assert torch.equal(got.isnan(), want.isnan())
    keep = ~want.isnan()
    assert torch.equal(got[keep], want[keep])
    assert torch.equal(torch.signbit(got[keep]), torch.signbit(want[keep]))


@pytest.mark.gpu
def test_empty_matrices():
    m = ng.quantize_mx(torch.zeros((0, 64), device=dev))
    assert m.codes.shape == (0, 32) and ng.dequantize_mx(m).shape == (0, 64)
    none = ng.quantize_mx(torch.zeros((3, 0), device=dev))
    assert none.scales.shape == (0, 3, 4) and ng.dequantize_mx(none).shape == (3, 0)
    w = ng.quantize_mx(torch.ones((5, 64), device=dev))
    assert ng.matmul_mx(torch.zeros((0, 64), device=dev), w).shape == (0, 5)
    assert ng.matmul_mx(torch.ones((4, 64), device=dev), m).shape == (4, 0)
    zero = ng.matmul_mx(none, ng.quantize_mx(torch.zeros((7, 0), device=dev)), F32)
    assert zero.shape == (3, 7) and not zero.any()


# ---------------------------------------------------------------------------
# the product (GPU)
# ---------------------------------------------------------------------------
def check_product(y: torch.Tensor, x64: np.ndarray, w64: np.ndarray, dtype):
    """Half a step of the type, and the fp32 sum's error: the terms are exact,
    and each of the at most K / 32 + 64 additions along the way (a block's sum
    into a lane's, lanes' and waves' sums at the end) is off by at most a step,
    2^-23, of a partial sum, which the magnitudes' sum bounds."""
    x, w = torch.from_numpy(x64).to(y.device), torch.from_numpy(w64).to(y.device)
    ref = x @ w.t().contiguous()
    mag = x.abs() @ w.abs().t().contiguous()
    K = x.shape[1]
    info = torch.finfo(dtype)
    bound = ref.abs() * info.eps / 2 + info.smallest_normal * info.eps / 2 \
        + mag * (K / 32 + 64) * 2.0 ** -23
    assert y.dtype == dtype and y.shape == ref.shape
    off = (y.double() - ref).abs() - bound
    assert (off <= 0).all(), f"worst {off.max().item():.3g} beyond its bound"


def product_case(M, N, K, seed):
    x = ng.quantize_mx(sample(M, K, F32, seed=seed).to(dev))
    w = ng.quantize_mx((sample(N, K, F32, seed=seed + 1) * 0.02).to(dev))
    return x, w


SIZES = [(1, 64, 32), (1, 1024, 4096), (2, 17, 96), (5, 100, 512), (8, 48, 544), (15, 130, 1024),
         (16, 256, 1056), (17, 64, 4128), (27, 333, 2048), (32, 96, 5536), (33, 260, 640),
         (63, 1000, 992), (64, 64, 14336), (65, 129, 256), (100, 515, 1120), (128, 128, 512),
         (130, 257, 2080), (200, 1023, 128), (256, 256, 4096), (257, 300, 160), (333, 2050, 1024),
         (513, 770, 1056), (1000, 1000, 544), (1024, 512, 2048), (2048, 1030, 64),
         # larger tiles of every form, whole and not
         (70, 2113, 992), (1024, 4096, 256), (1000, 4090, 96), (132, 10937, 288), (2048, 4096, 128),
         (2000, 4090, 352), (1921, 4033, 32), (1000, 4102, 544), (1674, 2370, 32), (261, 13148, 96),
         (1500, 6144, 512), (2346, 3361, 32), (515, 13236, 288), (2048, 7168, 512), (1999, 7001, 288),
         (1800, 7100, 1056)]


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", SIZES)
def test_product(M, N, K):
    x, w = product_case(M, N, K, seed=M + N)
    x64, w64 = values64(x), values64(w)
    for dtype in DTYPES:
        check_product(ng.matmul_mx(x, w, dtype), x64, w64, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", [(1, 1024, 4096), (3, 100, 96), (7, 516, 2080), (16, 64, 544),
                                   (2, 4100, 2048), (9, 4100, 2080), (1, 70, 4128), (16, 12288, 96),
                                   (27, 515, 1024), (64, 130, 4096), (150, 200, 672)])
def test_product_of_dense_rows(M, N, K, dtype):
    """Quantising within the call gives the values of quantising before it."""
    w = ng.quantize_mx((sample(N, K, F32, seed=2) * 0.02).to(dev))
    x = sample(M, K, dtype, seed=M, wide=True).to(dev)
    y = ng.matmul_mx(x, w)
    assert y.dtype == dtype
    xq = ng.quantize_mx(x)
    check_product(y, values64(xq), values64(w), dtype)
    check_product(ng.matmul_mx(x, w, F32), values64(xq), values64(w), F32)
    buf = torch.zeros((M, K + 24), dtype=dtype, device=dev)
    buf[:, 8:8 + K] = x
    assert torch.equal(ng.matmul_mx(buf[:, 8:8 + K], w), y)
    odd = torch.zeros((M, K + 3), dtype=dtype, device=dev)
    odd[:, 1:1 + K] = x
    assert torch.equal(ng.matmul_mx(odd[:, 1:1 + K], w), y)
    assert torch.equal(ng.matmul_mx(x.t().contiguous().t(), w), y)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 20, 70, 300])
def test_scales_over_their_whole_range(M):
    """Products whose powers of two reach from 2^-254 to 2^254: what fp32 can
    hold comes out, and nothing else makes it wrong."""
    K, N = 256, 40
    g = torch.Generator().manual_seed(M)
    codes = lambda rows: torch.randint(0, 256, (rows, K // 2), generator=g).to(torch.uint8)  # noqa: E731
    for base in (0, 60, 127, 160):
        xs = torch.full((M, K // 32), base, dtype=torch.uint8)
        ws = torch.full((N, K // 32), 254 - base, dtype=torch.uint8)  # the product's is 2^0
        x, w = ng.mx_from_blocks(codes(M), xs).to(dev), ng.mx_from_blocks(codes(N), ws).to(dev)
        check_product(ng.matmul_mx(x, w, F32), values64(x), values64(w), F32)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N", [(1, 70), (20, 70), (70, 64), (300, 513)])
def test_nan_blocks_stay_in_their_rows(M, N):
    K = 416
    x, w = sample(M, K, F32, seed=1), sample(N, K, F32, seed=2)
    x[M // 2, K - 1] = float("nan")
    w[N - 1, 130] = float("inf")
    xq, wq = ng.quantize_mx(x.to(dev)), ng.quantize_mx(w.to(dev))
    y = ng.matmul_mx(xq, wq, F32).cpu()
    want = torch.zeros((M, N), dtype=torch.bool)
    want[M // 2] = True
    want[:, N - 1] = True
    assert torch.equal(y.isnan(), want)


@pytest.mark.gpu
def test_matrices_beyond_32_bits():
    """Weights of more than 2^31 bytes of codes, and values of more than 2^32
    bytes quantised."""
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("not enough memory")
    N, K = 600_000, 8192
    g = torch.Generator(device=dev).manual_seed(0)
    codes = torch.randint(0, 256, (N, K // 2), generator=g, device=dev, dtype=torch.uint8)
    scales = torch.randint(120, 130, (K // 128, N, 4), generator=g, device=dev, dtype=torch.uint8)
    w = mx.MXMatrix(codes, scales, N, K)
    some = torch.tensor([0, 5, 262144, 599_000, N - 1], device=dev)
    part = mx.MXMatrix(codes[some].contiguous(), scales[:, some].contiguous(), 5, K)
    for M in (3, 70):
        x = ng.quantize_mx(sample(M, K, F16, seed=M).to(dev))
        y = ng.matmul_mx(x, w, F32)
        check_product(y[:, some], values64(x), values64(part), F32)
        del y
    assert torch.equal(ng.dequantize_mx(w, F16)[some], ng.dequantize_mx(part, F16))
    del w, codes, scales
    v = torch.empty((300_000, K), dtype=F16, device=dev)  # 4.9 GB
    v.normal_(generator=g)
    rows = torch.tensor([0, 131072, 262143, 262144, 299_999], device=dev)
    q = ng.quantize_mx(v)
    want = ng.quantize_mx(v[rows].contiguous())
    assert torch.equal(q.codes[rows], want.codes) and torch.equal(q.scales[:, rows], want.scales)
    t = ng.quantize_mx(v[:, :4096].contiguous().t().contiguous().t())
    assert torch.equal(t.codes[rows], want.codes[:, :2048])


@pytest.mark.gpu
def test_product_refusals_on_the_gpu():
    x, w = product_case(3, 64, 128, seed=0)
    with pytest.raises(RuntimeError, match="K=64"):
        ng.matmul_mx(torch.zeros((2, 64), device=dev), w)
    with pytest.raises(RuntimeError, match="same device"):
        ng.matmul_mx(torch.zeros((2, 128)), w)
    with pytest.raises(RuntimeError, match="same device"):
        ng.matmul_mx(x.to("cpu"), w)
    with pytest.raises(RuntimeError, match="no backward"):
        ng.matmul_mx(torch.zeros((2, 128), device=dev, requires_grad=True), w)
    with pytest.raises(RuntimeError, match="out_dtype"):
        ng.matmul_mx(x, w, torch.float64)


@pytest.mark.gpu
def test_quantised_activations_are_not_mixed_up():
    """Calls of different sizes on one stream share a workspace; calls on two
    streams, two graphs and one beyond what is kept do not."""
    w = ng.quantize_mx((sample(256, 512, F32, seed=4) * 0.02).to(dev))
    big = torch.zeros((70_000, 512), dtype=F16, device=dev)  # 19 MB of codes and scales
    big[:300] = sample(300, 512, F16, seed=3).to(dev)
    xs = [big[:300].clone(), big[:40].clone(), big[:18] * 2]
    want = [ng.matmul_mx(ng.quantize_mx(x), w) for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        got = [ng.matmul_mx(x, w) for x in xs]
        with torch.cuda.stream(side):
            other = [ng.matmul_mx(x, w) for x in reversed(xs)]
    torch.cuda.synchronize()
    for g, o, y in zip(got, reversed(other), want):
        assert torch.equal(g, y) and torch.equal(o, y)
    assert torch.equal(ng.matmul_mx(big, w)[:300], want[0])
    graphs, ys = [], []
    for x in xs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            ys.append(ng.matmul_mx(x, w))
    for _ in range(3):
        for graph in graphs:
            graph.replay()
        assert torch.equal(ng.matmul_mx(xs[1], w), want[1])
        torch.cuda.synchronize()
        for y, z in zip(ys, want):
            assert torch.equal(y, z)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 27, 200])
def test_product_on_another_stream_and_in_a_graph(M):
    w = ng.quantize_mx((sample(512, 1024, F32, seed=4) * 0.02).to(dev))
    xs = [sample(M, 1024, F16, seed=10 + i).to(dev) for i in range(3)]
    want = [ng.matmul_mx(x, w) for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ng.matmul_mx(xs[0], w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want[0])
    x = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ng.matmul_mx(x, w)
    for i in (0, 1, 2, 1):
        x.copy_(xs[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[i])
        assert torch.equal(ng.matmul_mx(xs[2], w), want[2])


@pytest.mark.gpu
@pytest.mark.parametrize("rows,K", [((1 << 27) + 9, 32), ((1 << 26) + 3, 544)])
def test_quantize_more_than_a_grid_dimension_holds(rows, K):
    """Rows whose workgroups have 2^32 threads and more together."""
    if torch.cuda.mem_get_info()[0] < 4 * rows * K:
        pytest.skip("not enough memory")
    some = torch.tensor([0, 7, 8, 8388607, 8388608, (1 << 26) - 1, 1 << 26, rows - 2, rows - 1],
                        device=dev)
    x = torch.zeros((rows, K), dtype=BF16, device=dev)
    x[some] = sample(len(some), K, BF16, seed=8).to(dev)
    m = ng.quantize_mx(x)
    want = ng.quantize_mx(x[some].contiguous())
    assert torch.equal(m.codes[some], want.codes) and torch.equal(m.scales[:, some], want.scales)
    other = torch.tensor([1, 8388609, 67108800, rows - 5], device=dev)
    assert not m.codes[other].any() and not m.scales[:, other].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_one_row_of_any_stride(dtype):
    """The stride over a single row does not matter, whatever it is."""
    x = sample(5, 192, dtype, seed=6)
    xd = x.to(dev)
    w = ng.quantize_mx(sample(40, 192, F32, seed=7).to(dev))
    want = ng.matmul_mx(ng.quantize_mx(xd[:1].clone()), w, F32)
    for one in (xd[0].expand(5, 192)[:1], xd[0].expand(1, 192), xd[:1], xd.t().contiguous().t()[:1],
                xd.as_strided((1, 192), (3, 1)), xd.as_strided((1, 192), (0, 1)),
                xd.as_strided((1, 192), (1, 1))):
        check_quantized(ng.quantize_mx(one), x[:1])
        assert torch.equal(ng.matmul_mx(one, w, F32), want)
    both = torch.zeros((5, 384), dtype=dtype, device=dev)
    both[:, ::2] = xd
    check_quantized(ng.quantize_mx(both[:1, ::2]), x[:1])
