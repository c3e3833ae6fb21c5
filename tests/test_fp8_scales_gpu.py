"""Products whose two scales multiplied leave the range of fp32 where the term itself does not.

An fp32 sum of m terms is off by at most m 2^-23 of the sum of their magnitudes (2^-23: the tensor cores may cut instead of
round); a block's sum meets its two scales in two roundings, and below 2^-126 a rounding is off by half of 2^-149 instead."""
import pytest
import torch

from tilelang_moe_b200 import kernels, ops

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn
# wide tiles, narrow ones, clusters that share a tile's k-blocks, few rows, rows of no alignment
SHAPES = [(2500, 640, 256), (300, 136, 384), (100, 512, 2048), (20, 264, 1024), (1, 256, 128), (40, 129, 400)]


def _scales(rows, K, exponents, g, cuda):
    """1 to 2 times a power of two, the rows in turn from `exponents`."""
    at = torch.tensor([float(exponents[i % len(exponents)]) for i in range(rows)], dtype=torch.float64, device=cuda)
    m = 1 + torch.rand(rows, -(-K // 128), dtype=torch.float64, generator=g, device=cuda)
    return (m * 2.0 ** at.unsqueeze(1)).float()


def _product(a, sa, b, sb):
    """The 64-bit product and the sum of its terms' magnitudes, one block of 128 at a time."""
    (M, K), N = a.shape, b.shape[0]
    y, size = torch.zeros(2, M, N, dtype=torch.float64, device=a.device)
    column = torch.arange(N, device=a.device) // 128
    for i in range(sa.shape[1]):
        x, w = a[:, i * 128:(i + 1) * 128].double(), b[:, i * 128:(i + 1) * 128].double()
        s = sa[:, i:i + 1].double() * sb.double()[column, i]
        y += x @ w.T * s
        size += x.abs() @ w.abs().T * s
    return y, size


def _check(y, want, size, K):
    blocks = -(-K // 128)
    limit = (K + 4 * blocks) * 2.0 ** -23 * size + torch.finfo(y.dtype).eps / 2 * want.abs() * (1 + 2.0 ** -8) + (blocks + 1) * 2.0 ** -149
    if y.dtype == torch.bfloat16:
        limit += 2.0 ** -134                   # half of its smallest subnormal
    # no partial sum is larger than `size` by more than the 2^-11 that 2048 terms may be off by: below 2^128 less a 256th of it
    # nothing overflows, bfloat16's last rounding included; above as much more a sum of numbers of one sign has to
    inside = size < 2.0 ** 128 * (1 - 2.0 ** -8)
    assert torch.all((y.double() - want).abs()[inside] <= limit[inside])
    assert torch.all(y[want > 2.0 ** 128 * (1 + 2.0 ** -8)] == float("inf"))


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("ea,eb,small", [((-75,), (-72,), False), ((-100,), (-46,), False), ((-21,), (-125,), False), ((-138,), (-8,), False),
                                         ((80,), (48,), True), ((3,), (126,), True), ((126,), (3,), True), ((120,), (-120,), False),
                                         ((-100, -40, 0, 30, 100), (-46, 28, -100, 0), True), ((-75, -75, 0), (-72, 0), False)])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_scales_of_every_size(cuda, lib, M, N, K, ea, eb, small, out_dtype):
    """Operands 2^-9 to 2^-5 where scales are large, up to 448 where they are small; all of one sign, so that the largest terms
    are as large as they can be."""
    g = torch.Generator(device=cuda).manual_seed(M + N + K)
    a, b = (torch.randint(1, 15, shape, generator=g, device=cuda).float() * (2.0 ** -9 if small else 32.0) for shape in ((M, K), (N, K)))
    a, b = a.to(E4M3), b.to(E4M3)
    sa, sb = _scales(M, K, ea, g, cuda), _scales(-(-N // 128), K, eb, g, cuda)
    y = kernels.fp8_gemm(a, sa, b, sb, out_dtype=out_dtype)
    ops.check_status(cuda)
    _check(y, *_product(a, sa, b, sb), K)


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_a_block_of_zeros_under_large_scales_adds_nothing(cuda, lib, M, N, K):
    """Scales of 2^100 and 2^60 are finite numbers, and zero times either is zero."""
    g = torch.Generator(device=cuda).manual_seed(K)
    a, b = (torch.randint(-14, 15, shape, generator=g, device=cuda).float() for shape in ((M, K), (N, K)))
    sa, sb = torch.ones(M, -(-K // 128), device=cuda), torch.ones(-(-N // 128), -(-K // 128), device=cuda)
    want = a @ b.T                             # whole numbers below 2^24: exact
    want -= a[:, :128] @ b[:, :128].T
    b[:, :128] = 0
    sa[::2, 0], sb[:, 0] = 1.5 * 2.0 ** 100, 1.5 * 2.0 ** 60
    y = kernels.fp8_gemm(a.to(E4M3), sa, b.to(E4M3), sb, out_dtype=torch.float32)
    ops.check_status(cuda)
    assert torch.equal(y, want)


def test_groups_of_zeros_and_scales_of_zero(cuda, lib):
    """What the quantisers make of zeros (a scale of 2^-100 / 448) against weights of every size, and scales that are 0."""
    g = torch.Generator(device=cuda).manual_seed(1)
    x, w = torch.randn(70, 512, generator=g, device=cuda), torch.randn(300, 512, generator=g, device=cuda)
    x[::3], x[:, 128:256], w[128:256, 256:384] = 0, 0, 0
    w[:128] *= 1e-30
    x[1::3] *= 1e-9
    a, sa = kernels.fp8_quantize(x)
    b, sb = kernels.fp8_quantize_blocks(w)
    y = kernels.fp8_gemm(a, sa, b, sb, out_dtype=torch.float32)
    assert torch.all(y[::3] == 0)
    _check(y, *_product(a, sa, b, sb), 512)
    sa[1::2], sb[1] = 0, 0
    y = kernels.fp8_gemm(a, sa, b, sb, out_dtype=torch.float32)
    assert torch.all(y[1::2] == 0) and torch.all(y[:, 128:256] == 0)
    _check(y, *_product(a, sa, b, sb), 512)
    ops.check_status(cuda)
