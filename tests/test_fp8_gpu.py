"""8-bit operands and their products against plain forms in 64 bits.

The products are compared in two ways.  With small whole numbers and scales that are powers of two every product and partial
sum is a number that fp32 holds, so the result has to be the exact one, rounded once.  With ordinary values an fp32 sum of m
terms is off by at most m 2^-23 of the sum of their magnitudes (2^-23 and not 2^-24: the tensor cores may cut instead of
round), and the final rounding by eps / 2 of its value."""
import math

import pytest
import torch

from tilelang_moe_b200 import kernels, ops

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


# ------------------------------------------------------------------------------------------------------- quantisers
def _tops(x, rows):
    """Largest magnitude of each group of `rows` x 128, spread over its places."""
    M, K = x.shape
    top = torch.zeros(-(-M // rows), -(-K // 128), dtype=torch.float64)
    for i in range(top.shape[0]):
        for j in range(top.shape[1]):
            top[i, j] = x[i * rows:(i + 1) * rows, j * 128:(j + 1) * 128].abs().amax().clamp(min=2.0 ** -100)
    return top, top.repeat_interleave(rows, 0)[:M].repeat_interleave(128, 1)[:, :K]


def _check(q, scale, x, rows, slack):
    """x: the 64-bit values; slack: relative error of what was divided and of what was quantised."""
    top, wide = _tops(x, rows)
    assert q.dtype == E4M3 and scale.dtype == torch.float32 and scale.shape == top.shape
    assert torch.all((scale.double() - top / 448).abs() <= (slack + 2.0 ** -24) * top / 448)
    v = x * (448 / wide)
    got = q.float().double()
    big = torch.maximum(v.abs(), got.abs())
    step = 2.0 ** (torch.floor(torch.log2(big.clamp(min=2.0 ** -6))) - 3)       # e4m3: 3 bits behind the leading one, 2^-9 at least
    assert torch.all((got - v).abs() <= step / 2 + v.abs() * (2 * slack + 2.0 ** -22))


def _values(M, K, g, dtype):
    x = torch.randn(M, K, generator=g) * torch.exp(2 * torch.randn(M, 1, generator=g))
    x[torch.rand(M, K, generator=g) < 0.1] = 0
    if M > 2:
        x[1] = 0                                  # a group of zeros
        x[2] *= 1e-4
    return x.to(dtype)


SHAPES = [(1, 1), (1, 128), (3, 7), (5, 127), (4, 129), (33, 256), (130, 200), (7, 1030), (300, 144), (2, 7168), (1000, 8)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K", SHAPES)
def test_quantize_rows(cuda, lib, M, K, dtype):
    x = _values(M, K, torch.Generator().manual_seed(M + K), dtype)
    q, scale = kernels.fp8_quantize(x.to(cuda))
    _check(q.cpu(), scale.cpu(), x.double(), 1, 0.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("E,M,K", [(1, 1, 1), (2, 128, 128), (3, 130, 72), (1, 127, 129), (2, 300, 515), (5, 8, 16), (1, 257, 1024)])
def test_quantize_blocks(cuda, lib, E, M, K, dtype):
    g = torch.Generator().manual_seed(M + K)
    x = torch.stack([_values(M, K, g, dtype) for _ in range(E)])
    q, scale = kernels.fp8_quantize_blocks(x.to(cuda))
    for e in range(E):
        _check(q[e].cpu(), scale[e].cpu(), x[e].double(), 128, 0.0)
    one, s1 = kernels.fp8_quantize_blocks(x[-1].to(cuda))
    assert torch.equal(one.view(torch.uint8), q[-1].view(torch.uint8)) and torch.equal(s1, scale[-1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,I", SHAPES)
def test_silu_mul(cuda, lib, M, I, dtype):
    """exp by the hardware is off by 2 + 1.173 |gate| units of 2^-23 at most, which is 2^-18 up to |gate| = 20; division,
    products and the sum under the quotient add four roundings."""
    g = torch.Generator().manual_seed(M + 3 * I)
    gate, up = (3 * torch.randn(M, I, generator=g)).clamp(-20, 20).to(dtype), _values(M, I, g, dtype)
    want = gate.double() * torch.sigmoid(gate.double()) * up.double()
    q, scale = kernels.fp8_silu_mul(gate.to(cuda), up.to(cuda))
    _check(q.cpu(), scale.cpu(), want, 1, 2.0 ** -18 + 2.0 ** -22)
    both = torch.cat([gate, up], dim=1).to(cuda)
    q2, s2 = kernels.fp8_silu_mul(both[:, :I], both[:, I:])
    assert torch.equal(q2.view(torch.uint8), q.view(torch.uint8)) and torch.equal(s2, scale)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K", [256, 250])
def test_quantize_what_is_no_number(cuda, lib, K, dtype):
    nan, inf = float("nan"), float("inf")
    x = torch.ones(5, K)
    x[0, 3], x[1, 4], x[2, 5], x[3, 6], x[4, 0] = nan, inf, -inf, -nan, 0.0
    for form, rows in ((kernels.fp8_quantize, 1), (kernels.fp8_quantize_blocks, 5)):
        q, scale = form(x.to(dtype).to(cuda))
        back = q.float().cpu().reshape(5, K)[:, :128] * scale.cpu()[:, :1]
        if rows == 1:
            assert torch.isnan(back[[0, 3]]).all() and torch.isnan(back[1, 4]) and torch.isnan(back[2, 5])
            assert scale[1, 0] == inf and scale[2, 0] == inf and back[4, 0] == 0 and torch.all(back[4, 1:] == 1)
        else:
            assert torch.isnan(scale[0, 0]) and torch.isnan(back).all()
        assert torch.all(q.float().cpu().reshape(5, K)[:, 128:] == 448)       # the group beside them is as it should be
    q, scale = kernels.fp8_quantize(torch.full((1, K), torch.finfo(dtype).tiny * torch.finfo(dtype).eps, dtype=dtype, device=cuda))
    assert torch.isfinite(q.float()).all() and torch.isfinite(scale).all() and torch.all(scale > 0)
    q, scale = kernels.fp8_quantize(torch.full((2, K), torch.finfo(dtype).max, dtype=dtype, device=cuda))
    assert torch.all(q.float() == 448) and torch.isfinite(scale).all()


def test_quantize_strides_and_shapes(cuda, lib):
    g = torch.Generator().manual_seed(1)
    base = torch.randn(12, 600, generator=g).bfloat16().to(cuda)
    for x in (base[:, :256], base[:, 8:264], base[:, 1:257], base[:, 3:258], base[::2, :256], base[:, ::2], base[:1, :256].expand(9, 256),
              base.view(3, 4, 600)[:, :, :128], base.view(3, 4, 600)[:, 1], base[0], base[:0]):
        q, s = kernels.fp8_quantize(x)
        qc, sc = kernels.fp8_quantize(x.contiguous())
        assert q.shape == x.shape and s.shape == (*x.shape[:-1], -(-x.shape[-1] // 128))
        assert torch.equal(q.view(torch.uint8), qc.view(torch.uint8)) and torch.equal(s, sc)
    w = base[:, :512].reshape(2, 6, 512)
    q, s = kernels.fp8_quantize_blocks(w.transpose(1, 2))
    qc, sc = kernels.fp8_quantize_blocks(w.transpose(1, 2).contiguous())
    assert torch.equal(q.view(torch.uint8), qc.view(torch.uint8)) and torch.equal(s, sc)
    assert kernels.fp8_quantize_blocks(w[:0])[0].shape == (0, 6, 512)


# ------------------------------------------------------------------------------------------------------- products
def _whole(M, N, K, E, g, cuda):
    """Whole numbers up to 3 and scales 1/2, 1, 2: sums below 2^20 in steps of 1/4, exact in fp32 in any order."""
    def scales(*shape):
        return 2.0 ** torch.randint(-1, 2, shape, generator=g, device=cuda).float()

    a = torch.randint(-3, 4, (M, K), generator=g, device=cuda).float()
    b = torch.randint(-3, 4, (E, N, K), generator=g, device=cuda).float()
    kb = -(-K // 128)
    return a.to(E4M3), scales(M, kb), b.to(E4M3), scales(E, -(-N // 128), kb)


def _product(a, sa, b, sb):
    """64-bit product of one group."""
    (N, K), M = b.shape, a.shape[0]
    wide_a = a.double() * sa.double().repeat_interleave(128, 1)[:, :K]
    wide_b = b.double() * sb.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    return wide_a @ wide_b.T, wide_a.abs() @ wide_b.abs().T


GEMMS = [(1, 1, 16), (1, 256, 128), (3, 7, 32), (128, 128, 128), (129, 257, 144), (64, 8, 4096), (300, 515, 400), (1000, 320, 1168),
         (17, 4096, 512), (256, 256, 7168), (40, 130, 2064), (2500, 640, 256), (33, 100, 16), (160, 72, 1000 // 16 * 16)]


@pytest.mark.parametrize("out_dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", GEMMS)
def test_gemm_is_exact_on_whole_numbers(cuda, lib, M, N, K, out_dtype):
    g = torch.Generator(device=cuda).manual_seed(M + N + K)
    a, sa, b, sb = _whole(M, N, K, 1, g, cuda)
    y = kernels.fp8_gemm(a, sa, b[0], sb[0], out_dtype=out_dtype)
    ops.check_status(cuda)
    assert y.shape == (M, N) and y.dtype == out_dtype
    assert torch.equal(y, _product(a, sa, b[0], sb[0])[0].float().to(out_dtype))


def _group_sizes(kind, M, E, g):
    if kind == "one":
        sizes = [0] * E
        sizes[E // 2] = M
    elif kind == "even":
        sizes = [M // E] * E
    else:                                      # a third of the groups empty, the others of every size; rows left over
        sizes = torch.multinomial(torch.rand(E, generator=g) * (torch.rand(E, generator=g) > 0.33) + 1e-9, max(1, M * 9 // 10), replacement=True, generator=g)
        sizes = torch.bincount(sizes, minlength=E).tolist()
    return sizes


@pytest.mark.parametrize("out_dtype", DTYPES)
@pytest.mark.parametrize("kind", ["one", "even", "ragged"])
@pytest.mark.parametrize("M,N,K,E", [(1, 8, 16, 1), (5, 264, 128, 7), (300, 136, 272, 4), (1000, 129, 512, 33), (2000, 512, 256, 3),
                                     (64, 256, 2048, 40), (700, 384, 128, 1000), (4000, 256, 1040, 9)])
def test_grouped_gemm_is_exact_on_whole_numbers(cuda, lib, M, N, K, E, kind, out_dtype):
    g = torch.Generator(device=cuda).manual_seed(M + N + K + E)
    a, sa, b, sb = _whole(M, N, K, E, g, cuda)
    sizes = _group_sizes(kind, M, E, torch.Generator().manual_seed(M))
    at = [0]
    for n in sizes:
        at.append(at[-1] + n)
    offsets = torch.tensor(at, dtype=torch.int32, device=cuda)
    want = torch.zeros(M, N, dtype=torch.float64, device=cuda)
    for e in range(E):
        if sizes[e]:
            want[at[e]:at[e + 1]] = _product(a[at[e]:at[e + 1]], sa[at[e]:at[e + 1]], b[e], sb[e])[0]
    y = kernels.fp8_grouped_gemm(a, sa, b, sb, offsets, out_dtype=out_dtype)
    ops.check_status(cuda)
    assert torch.equal(y, want.float().to(out_dtype))
    # into a caller's tensor with room around every row: nothing but the groups' rows changes
    room = torch.full((M + 2, N + 16), 7.0, dtype=out_dtype, device=cuda)
    out = room[1:M + 1, 8:8 + N]
    assert kernels.fp8_grouped_gemm(a, sa, b, sb, offsets, out=out) is out
    assert torch.equal(out[:at[-1]], y[:at[-1]]) and torch.all(out[at[-1]:] == 7)
    room[1:M + 1, 8:8 + N] = 7
    assert torch.all(room == 7)


@pytest.mark.parametrize("out_dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", [(1, 512, 7168), (200, 300, 1040), (129, 256, 4096), (16, 1024, 2048)])
def test_gemm_of_ordinary_values(cuda, lib, M, N, K, out_dtype):
    g = torch.Generator(device=cuda).manual_seed(K)
    a, sa = kernels.fp8_quantize(torch.randn(M, K, generator=g, device=cuda))
    b, sb = kernels.fp8_quantize_blocks(torch.randn(N, K, generator=g, device=cuda) / math.sqrt(K))
    y = kernels.fp8_gemm(a, sa, b, sb, out_dtype=out_dtype)
    want, size = _product(a, sa, b, sb)
    # K products and their sums, the block's scale, its product with the sum and the sum of the blocks
    limit = (K + 3 * -(-K // 128)) * 2.0 ** -23 * size + torch.finfo(out_dtype).eps / 2 * want.abs() * (1 + 2.0 ** -8) + 2.0 ** -25
    assert torch.all((y.double() - want).abs() <= limit)
    if out_dtype == torch.float32:             # and as near as fp32 sums of that length are as a rule
        assert (y.double() - want).norm() <= 4 * 2.0 ** -24 * math.sqrt(K) * want.norm()


def test_gemm_takes_scales_and_rows_of_any_stride(cuda, lib):
    g = torch.Generator(device=cuda).manual_seed(2)
    a, sa, b, sb = _whole(150, 264, 400, 1, g, cuda)
    b, sb = b[0], sb[0]
    want = kernels.fp8_gemm(a, sa, b, sb)
    wide = torch.zeros(150, 1024, dtype=torch.uint8, device=cuda)
    for at in (0, 16, 5):
        wide[:, at:at + 400] = a.view(torch.uint8)
        assert torch.equal(kernels.fp8_gemm(wide[:, at:at + 400].view(E4M3), sa, b, sb), want)
    assert torch.equal(kernels.fp8_gemm(a, sa.T.contiguous().T, b, sb.T.contiguous().T), want)
    assert torch.equal(kernels.fp8_gemm(a.view(torch.uint8).T.contiguous().T.view(E4M3), sa, b, sb), want)
    one = kernels.fp8_gemm(a, torch.full((1, 1), 0.5, device=cuda).expand(150, 4), b, sb)
    assert torch.equal(one, kernels.fp8_gemm(a, torch.full((150, 4), 0.5, device=cuda), b, sb))
    bw = torch.zeros(264 * 400 + 8, dtype=torch.uint8, device=cuda)
    bw[3:3 + 264 * 400] = b.reshape(-1).view(torch.uint8)
    assert torch.equal(kernels.fp8_gemm(a, sa, bw[3:3 + 264 * 400].view(E4M3).view(264, 400), sb), want)


def test_gemm_of_nothing_and_of_what_is_no_number(cuda, lib):
    g = torch.Generator(device=cuda).manual_seed(3)
    a, sa, b, sb = _whole(130, 140, 256, 2, g, cuda)
    assert kernels.fp8_gemm(a[:0], sa[:0], b[0], sb[0]).shape == (0, 140)
    none = torch.zeros(3, dtype=torch.int32, device=cuda)
    assert kernels.fp8_grouped_gemm(a[:0], sa[:0], b, sb, none).shape == (0, 140)
    assert torch.all(kernels.fp8_grouped_gemm(a, sa, b, sb, none) == 0)
    # a NaN in one row of a, in one row of b, in a scale: they reach their row, column and rows, nothing else
    want = kernels.fp8_gemm(a, sa, b[0], sb[0])
    a2, b2, s2 = a.clone(), b[0].clone(), sa.clone()
    a2.view(torch.uint8)[5, 9] = 0x7F
    b2.view(torch.uint8)[7, 200] = 0xFF
    s2[100, 1] = float("nan")
    s2[101, 0] = float("inf")
    y = kernels.fp8_gemm(a2, s2, b2, sb[0])
    bad = torch.zeros(130, 140, dtype=torch.bool, device=cuda)
    bad[5], bad[:, 7], bad[100] = True, True, True
    assert torch.isnan(y[bad]).all()
    bad[101] = True
    assert torch.equal(y[~bad], want[~bad]) and not torch.isfinite(y[101]).any()


def test_offsets_that_are_no_prefix_sum_stay_inside(cuda, lib):
    """Rows behind the tensor or before it are never read or written: starts and ends are cut to its rows."""
    g = torch.Generator(device=cuda).manual_seed(4)
    a, sa, b, sb = _whole(200, 64, 128, 3, g, cuda)
    room = torch.full((400, 64), 7.0, device=cuda)
    out = room[100:300]
    kernels.fp8_grouped_gemm(a, sa, b, sb, torch.tensor([-50, 100, 90, 100000], dtype=torch.int32, device=cuda), out=out)
    ops.check_status(cuda)
    assert torch.all(room[:100] == 7) and torch.all(room[300:] == 7)
    assert torch.equal(out[:90], _product(a[:90], sa[:90], b[0], sb[0])[0].float())
    assert torch.equal(out[100:], _product(a[100:], sa[100:], b[2], sb[2])[0].float())


def test_rows_behind_two_to_the_31(cuda, lib):
    """Elements of a, of b and of the result whose offsets pass 2^31."""
    g = torch.Generator(device=cuda).manual_seed(5)
    M, K, N = 320_000, 7168, 8192
    a = torch.zeros(M, K, dtype=torch.uint8, device=cuda)
    sa = torch.ones(M, 56, device=cuda)
    rows = torch.tensor([0, 1, M // 2, M - 2, M - 1], device=cuda)
    small, _, b, sb = _whole(5, N, K, 1, g, cuda)
    a[rows] = small.view(torch.uint8)
    y = kernels.fp8_gemm(a.view(E4M3), sa, b[0], sb[0])
    assert torch.equal(y[rows], _product(small, sa[:5], b[0], sb[0])[0].float().bfloat16())
    assert torch.count_nonzero(y[2:1000]) == 0
    del a, sa, y, b
    E = 40
    q = torch.zeros(E, 8192, 7168, dtype=torch.uint8, device=cuda)
    few, s1, one, so = _whole(3, 8192, 7168, 1, g, cuda)
    q[E - 1] = one[0].view(torch.uint8)
    scales = torch.ones(E, 64, 56, device=cuda)
    scales[E - 1] = so[0]
    offsets = torch.zeros(E + 1, dtype=torch.int32, device=cuda)
    offsets[E] = 3
    y = kernels.fp8_grouped_gemm(few, s1, q.view(E4M3), scales, offsets)
    assert torch.equal(y, _product(few, s1, one[0], so[0])[0].float().bfloat16())
    ops.check_status(cuda)


# ------------------------------------------------------------------------------------------------------- together
def _expert_layer(x, ids, w, gate_up, down, E):
    """An expert layer in 8 bits: quantise once per token, sort, both products, weigh and bring back."""
    (gu, gus), (dn, dns) = gate_up, down
    I = dn.shape[2]
    sort = kernels.moe_sort(ids, E)
    q, s = kernels.fp8_quantize(x)
    h = kernels.fp8_grouped_gemm(kernels.moe_permute(q, sort), kernels.moe_permute(s, sort), gu, gus, sort.offsets)
    q, s = kernels.fp8_silu_mul(h[:, :I], h[:, I:])
    return kernels.moe_unpermute(kernels.fp8_grouped_gemm(q, s, dn, dns, sort.offsets), sort, w)


def _layer_inputs(T, H, I, E, k, cuda, seed):
    g = torch.Generator(device=cuda).manual_seed(seed)
    x = torch.randn(T, H, generator=g, device=cuda).bfloat16()
    ids = torch.rand(T, E, generator=g, device=cuda).topk(k, dim=1).indices
    ids[torch.rand(T, k, generator=g, device=cuda) < 0.1] = -1
    w = torch.softmax(torch.randn(T, k, generator=g, device=cuda), 1)
    gate_up = kernels.fp8_quantize_blocks(torch.randn(E, 2 * I, H, generator=g, device=cuda) / math.sqrt(H))
    down = kernels.fp8_quantize_blocks(torch.randn(E, H, I, generator=g, device=cuda) / math.sqrt(I))
    return x, ids, w, gate_up, down


@pytest.mark.parametrize("T,H,I,E,k", [(1, 256, 128, 4, 2), (37, 512, 256, 8, 2), (300, 1024, 384, 16, 4)])
def test_expert_layer(cuda, lib, T, H, I, E, k):
    """Against the layer in 64 bits on the dequantised weights.  What the 8-bit steps cost: x and SiLU(gate)*up are each off
    by half an e4m3 step, 2^-4 of a value at most and evenly spread (a third of that squared on average), on all H or I
    terms of a sum independently: the result is off by sqrt(3) / 3 * 2^-4 for each of gate, up and the product between, as
    long as they add like independent errors; twice their sum bounds it, with the three 16-bit roundings far below."""
    x, ids, w, (gu, gus), (dn, dns) = _layer_inputs(T, H, I, E, k, cuda, T)
    y = _expert_layer(x, ids, w, (gu, gus), (dn, dns), E)
    ops.check_status(cuda)
    want = torch.zeros(T, H, dtype=torch.float64, device=cuda)
    for t in range(T):
        for j in range(k):
            e = int(ids[t, j])
            if e < 0:
                continue
            one = torch.ones(1, -(-H // 128), device=cuda)
            h = _product(x[t:t + 1].double(), one, gu[e], gus[e])[0]
            h = h[:, :I] * torch.sigmoid(h[:, :I]) * h[:, I:]
            want[t] += float(w[t, j]) * _product(h, torch.ones(1, -(-I // 128), device=cuda), dn[e], dns[e])[0][0]
    assert (y.double() - want).norm() <= 2 * 3 * math.sqrt(3) / 3 * 2.0 ** -4 * want.norm()
    assert torch.all(y[(ids < 0).all(1)] == 0)


def test_expert_layer_in_graphs_and_on_streams(cuda, lib):
    """Two captured layers replayed in turn on new tokens, and one on a stream of its own, give what plain calls give."""
    T, H, I, E, k = 64, 512, 256, 8, 2
    layers = []
    for seed in (1, 2):
        static = list(_layer_inputs(T, H, I, E, k, cuda, seed))
        side = torch.cuda.Stream(cuda)
        side.wait_stream(torch.cuda.current_stream(cuda))
        with torch.cuda.stream(side):
            _expert_layer(*static, E)
        torch.cuda.current_stream(cuda).wait_stream(side)
        torch.cuda.synchronize(cuda)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _expert_layer(*static, E)
        layers.append((graph, static, out))
    for round_ in range(2):
        for i, (graph, static, out) in enumerate(layers):
            fresh = _layer_inputs(T, H, I, E, k, cuda, 10 + 2 * round_ + i)
            for a, b in zip(static[:3], fresh[:3]):
                a.copy_(b)
            graph.replay()
        for graph, static, out in layers:
            assert torch.equal(out, _expert_layer(*static, E))
    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(side):
        got = _expert_layer(*layers[0][1], E)
    want = _expert_layer(*layers[1][1], E)     # meanwhile, on the current stream
    side.synchronize()
    assert torch.equal(got, layers[0][2]) and torch.equal(want, layers[1][2])
    ops.check_status(cuda)


# ------------------------------------------------------------------------------------------------------- more shapes
@pytest.mark.parametrize("out_dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", [(5000, 1000, 272), (4100, 1001, 128), (2000, 4500, 256), (128, 2304, 1536), (33, 640, 3600), (32, 640, 2048),
                                   (31, 129, 1296), (97, 1024, 512), (1, 8192, 1024), (640, 2176, 160), (20000, 136, 16)])
def test_gemm_of_every_tiling_is_exact(cuda, lib, M, N, K, out_dtype):
    """Wide tiles in several rounds and bands, narrow ones, clusters of 2, 4 and 8, few rows, and widths without vectors."""
    g = torch.Generator(device=cuda).manual_seed(M + N)
    a, sa, b, sb = _whole(M, N, K, 1, g, cuda)
    y = kernels.fp8_gemm(a, sa, b[0], sb[0], out_dtype=out_dtype)
    ops.check_status(cuda)
    assert torch.equal(y, _product(a, sa, b[0], sb[0])[0].float().to(out_dtype))
    # into rows of a wider tensor: other alignments, nothing beside them changes
    for left in (0, 1, 4):
        room = torch.full((M, N + 8), 7.0, dtype=out_dtype, device=cuda)
        kernels.fp8_gemm(a, sa, b[0], sb[0], out=room[:, left:left + N])
        assert torch.equal(room[:, left:left + N], y)
        room[:, left:left + N] = 7
        assert torch.all(room == 7)


@pytest.mark.parametrize("M,N,K,E", [(3000, 1500, 400, 20), (9000, 2056, 144, 37), (32, 512, 1024, 12), (20, 2048, 768, 256), (2048, 1024, 256, 1024)])
def test_grouped_gemm_of_every_tiling_is_exact(cuda, lib, M, N, K, E):
    g = torch.Generator(device=cuda).manual_seed(M + N + E)
    a, sa, b, sb = _whole(M, N, K, E, g, cuda)
    sizes = _group_sizes("ragged", M, E, torch.Generator().manual_seed(M))
    at = torch.tensor([0] + sizes).cumsum(0)
    y = kernels.fp8_grouped_gemm(a, sa, b, sb, at.int().to(cuda))
    ops.check_status(cuda)
    want = torch.zeros(M, N, dtype=torch.float64, device=cuda)
    for e in range(E):
        if sizes[e]:
            part = slice(int(at[e]), int(at[e + 1]))
            want[part] = _product(a[part], sa[part], b[e], sb[e])[0]
    assert torch.equal(y, want.float().bfloat16())


def test_first_group_may_start_behind_the_first_row(cuda, lib):
    g = torch.Generator(device=cuda).manual_seed(8)
    a, sa, b, sb = _whole(300, 256, 256, 2, g, cuda)
    y = kernels.fp8_grouped_gemm(a, sa, b, sb, torch.tensor([40, 200, 260], dtype=torch.int32, device=cuda))
    assert torch.all(y[:40] == 0) and torch.all(y[260:] == 0)
    assert torch.equal(y[40:200], _product(a[40:200], sa[40:200], b[0], sb[0])[0].float().bfloat16())
    assert torch.equal(y[200:260], _product(a[200:260], sa[200:260], b[1], sb[1])[0].float().bfloat16())


def test_products_on_two_streams_at_once(cuda, lib):
    """Nothing is shared between calls: products that overlap on the device give what they give alone."""
    g = torch.Generator(device=cuda).manual_seed(9)
    jobs = []
    for M, N, K in ((1500, 2048, 2048), (16, 4096, 4096)):
        a, sa, b, sb = _whole(M, N, K, 1, g, cuda)
        jobs.append((a, sa, b[0], sb[0], kernels.fp8_gemm(a, sa, b[0], sb[0])))
    torch.cuda.synchronize(cuda)
    streams = [torch.cuda.Stream(cuda) for _ in jobs]
    got = [[], []]
    for _ in range(20):
        for (a, sa, b, sb, _), stream, out in zip(jobs, streams, got):
            with torch.cuda.stream(stream):
                out.append(kernels.fp8_gemm(a, sa, b, sb))
    torch.cuda.synchronize(cuda)
    for job, out in zip(jobs, got):
        assert all(torch.equal(y, job[4]) for y in out)
    ops.check_status(cuda)


def test_results_repeat_bit_by_bit(cuda, lib):
    g = torch.Generator(device=cuda).manual_seed(10)
    for M, N, K in ((3, 512, 7168), (700, 2048, 4096)):
        a, sa = kernels.fp8_quantize(torch.randn(M, K, generator=g, device=cuda))
        b, sb = kernels.fp8_quantize_blocks(torch.randn(N, K, generator=g, device=cuda))
        y = kernels.fp8_gemm(a, sa, b, sb, out_dtype=torch.float32)
        for _ in range(5):
            assert torch.equal(kernels.fp8_gemm(a, sa, b, sb, out_dtype=torch.float32), y)


def test_bytes_around_the_operands_do_not_matter(cuda, lib):
    """a and b are views whose surroundings are NaN in every byte: what lies behind K, behind the last row and in the next
    expert's place is not multiplied."""
    g = torch.Generator(device=cuda).manual_seed(11)
    M, N, K = 77, 130, 208
    a, sa, b, sb = _whole(M, N, K, 1, g, cuda)
    wide = torch.full((M + 60, K + 48), 0x7F, dtype=torch.uint8, device=cuda)
    wide[30:30 + M, 16:16 + K] = a.view(torch.uint8)
    more = torch.full((3, N, K), 0x7F, dtype=torch.uint8, device=cuda)
    more[1] = b[0].view(torch.uint8)
    scales = torch.full((3, 2, 2), float("nan"), device=cuda)
    scales[1] = sb[0]
    around = torch.full((M + 2, 4), float("nan"), device=cuda)
    around[1:M + 1, 1:3] = sa
    want = _product(a, sa, b[0], sb[0])[0].float().bfloat16()
    view = wide[30:30 + M, 16:16 + K].view(E4M3)
    assert torch.equal(kernels.fp8_gemm(view, around[1:M + 1, 1:3], more[1].view(E4M3), scales[1]), want)
    offsets = torch.tensor([0, 0, M, M], dtype=torch.int32, device=cuda)
    assert torch.equal(kernels.fp8_grouped_gemm(view, around[1:M + 1, 1:3], more.view(E4M3), scales, offsets), want)
    # one group's rows beside another's: the neighbours in a tile are not multiplied into them either
    two = torch.cat([a, torch.full((50, K), 0x7F, dtype=torch.uint8, device=cuda).view(E4M3)])
    both = kernels.fp8_grouped_gemm(two, torch.cat([sa, torch.ones(50, 2, device=cuda)]), torch.cat([b, b]), torch.cat([sb, sb]),
                                    torch.tensor([0, M, M + 50], dtype=torch.int32, device=cuda))
    assert torch.equal(both[:M], want) and torch.isnan(both[M:]).all()


def test_graph_of_a_product_over_every_kind_of_launch(cuda, lib):
    """Captured once, replayed on other inputs: clusters, narrow and wide tiles, few rows."""
    g = torch.Generator(device=cuda).manual_seed(12)
    for M, N, K in ((1, 1024, 1024), (100, 512, 2048), (700, 640, 256), (2000, 4500, 256)):
        a, sa, b, sb = _whole(M, N, K, 1, g, cuda)
        kernels.fp8_gemm(a, sa, b[0], sb[0])
        torch.cuda.synchronize(cuda)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = kernels.fp8_gemm(a, sa, b[0], sb[0], out_dtype=torch.float32)
        for _ in range(2):
            na, nsa, nb, nsb = _whole(M, N, K, 1, g, cuda)
            for old, new in ((a, na), (sa, nsa), (b, nb), (sb, nsb)):
                old.view(torch.uint8).copy_(new.view(torch.uint8)) if old.dtype == E4M3 else old.copy_(new)
            graph.replay()
            assert torch.equal(y, _product(na, nsa, nb[0], nsb[0])[0].float())
