"""Tokens sorted by expert and back, and their gradients, against a plain form in 64 bits.

A sum of m products in fp32 is off by at most m 2^-24 times the sum of their magnitudes (each of the m additions rounds a
partial sum that is not larger), a result rounded to its type by half a step: eps / 2 of the value, or half the smallest
subnormal."""
import pytest
import torch

from tilelang_moe_b200 import kernels, ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
STEP0 = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}


def _off_by(got, want, magnitudes, terms):
    """got within the error of `terms` fp32 operations and one rounding of the 64-bit `want`."""
    t = got.dtype
    limit = torch.finfo(t).eps / 2 * want.abs() + STEP0[t] + (terms + 1) * U * (1 + 2.0 ** -7) * magnitudes
    off = (got.double() - want).abs()
    assert torch.all(off <= limit), f"off by {(off - limit).max().item():g} more than it may be"


def _ids(T, k, E, g, drop=0.2, dtype=torch.int32):
    ids = torch.randint(0, E, (T, k), generator=g)
    ids[torch.rand(T, k, generator=g) < drop] = -1
    if T > 2:
        ids[-1] = -1                       # a token without any expert
    return ids.to(dtype)


def _tables(ids, E):
    flat = ids.reshape(-1).tolist()
    order = [i for e in range(E) for i, v in enumerate(flat) if v == e] + [i for i, v in enumerate(flat) if not 0 <= v < E]
    offsets = [0]
    for e in range(E):
        offsets.append(offsets[-1] + flat.count(e))
    row_of = [0] * len(flat)
    for p, i in enumerate(order):
        row_of[i] = p
    return offsets, order, row_of


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("T,k,E", [(1, 1, 1), (1, 8, 3), (7, 2, 5), (300, 8, 17), (5000, 2, 64), (1, 40, 2), (40000, 2, 1200), (500, 3, 5119), (70000, 1, 100)])
def test_sort(cuda, lib, T, k, E, dtype):
    g = torch.Generator().manual_seed(T + k)
    ids = _ids(T, k, E, g, dtype=dtype)
    ids[0, 0] = E                          # above the range: no expert either
    s = kernels.moe_sort(ids.to(cuda), E)
    flat = ids.reshape(-1).long()
    key = torch.where((flat < 0) | (flat >= E), E, flat)
    perm = torch.argsort(key, stable=True)
    assert s.perm.tolist() == perm.tolist()
    assert s.offsets.tolist() == [0] + torch.bincount(key, minlength=E + 1)[:E].cumsum(0).tolist()
    assert torch.equal(s.row_of.cpu()[perm], torch.arange(T * k, dtype=torch.int32))
    assert (s.n_experts, s.tokens, s.k) == (E, T, k)
    ops.check_status(cuda)                 # entries without an expert are not an error


def test_sort_of_none_and_of_vectors(cuda, lib):
    s = kernels.moe_sort(torch.empty(0, 4, dtype=torch.int64, device=cuda), 3)
    assert s.offsets.tolist() == [0, 0, 0, 0] and s.tokens == 0
    x = torch.empty(0, 8, device=cuda, requires_grad=True)
    rows = kernels.moe_permute(x, s)
    y = kernels.moe_unpermute(rows, s, torch.empty(0, 4, device=cuda))
    assert rows.shape == (0, 8) and y.shape == (0, 8)
    assert torch.autograd.grad(y.sum(), x)[0].shape == (0, 8)
    assert kernels.moe_sort(torch.tensor([2, 0, 2], device=cuda), 3).perm.tolist() == [1, 0, 2]


@pytest.mark.parametrize("dtype", DTYPES + [torch.float8_e4m3fn, torch.uint8, torch.float64])
@pytest.mark.parametrize("T,k,E,H", [(1, 1, 1, 1), (3, 2, 4, 7), (33, 8, 6, 64), (130, 3, 9, 515), (17, 40, 5, 96), (9, 8, 4, 7168), (64, 4, 8, 1030)])
def test_permute(cuda, lib, T, k, E, H, dtype):
    g = torch.Generator().manual_seed(H + T)
    ids = _ids(T, k, E, g)
    x = torch.randint(0, 256, (T, H * torch.empty(0, dtype=dtype).element_size()), generator=g, dtype=torch.uint8)   # any bits at all
    offsets, order, _ = _tables(ids, E)
    want = x[torch.tensor(order) // k].clone()
    want[offsets[-1]:] = 0
    got = kernels.moe_permute(x.to(cuda).view(dtype), kernels.moe_sort(ids.to(cuda), E))
    assert got.dtype == dtype and got.shape == (T * k, H)
    assert torch.equal(got.view(torch.uint8).cpu(), want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("weighted", [True, False])
@pytest.mark.parametrize("T,k,E,H", [(1, 1, 1, 1), (3, 2, 4, 7), (33, 8, 6, 64), (130, 3, 9, 515), (17, 20, 5, 96), (9, 8, 4, 7168),
                                     (64, 4, 8, 1030), (40, 9, 8, 4104)])
def test_both_ways_with_gradients(cuda, lib, T, k, E, H, weighted, dtype):
    g = torch.Generator().manual_seed(H + T + k)
    ids = _ids(T, k, E, g)
    x, gr, gy = (torch.randn(n, H, generator=g).to(dtype) for n in (T, T * k, T))
    w = torch.randn(T, k, generator=g)
    rows = torch.randn(T * k, H, generator=g).to(dtype)
    offsets, order, row_of = _tables(ids, E)
    live = offsets[-1]
    rows[live:] = float("nan")             # rows behind the last expert are read by nobody
    gr[live:] = float("inf")
    sort = kernels.moe_sort(ids.to(cuda), E)
    perm = torch.tensor(order)[:live]
    token = perm // k

    xd = x.to(cuda).requires_grad_()
    got = kernels.moe_permute(xd, sort)
    grad, = torch.autograd.grad(got, xd, gr.to(cuda))
    zero = torch.zeros(T, H, dtype=torch.float64)
    _off_by(grad.cpu(), zero.index_add(0, token, gr[:live].double()), zero.index_add(0, token, gr[:live].double().abs()), k)

    rd, wd = rows.to(cuda).requires_grad_(), w.to(cuda).requires_grad_()
    y = kernels.moe_unpermute(rd, sort, wd if weighted else None)
    wl = w.double().reshape(-1)[perm].unsqueeze(1) if weighted else torch.ones(live, 1, dtype=torch.float64)
    part = wl * rows[:live].double()
    _off_by(y.detach().cpu(), zero.index_add(0, token, part), zero.index_add(0, token, part.abs()), k)

    got = torch.autograd.grad(y, (rd, wd) if weighted else (rd,), gy.to(cuda))
    want = torch.zeros(T * k, H, dtype=torch.float64)
    want[:live] = wl * gy.double()[token]
    _off_by(got[0].cpu(), want, want.abs(), 1)
    if weighted:
        each = gy.double()[token] * rows[:live].double()
        want, size = torch.zeros(T * k, dtype=torch.float64), torch.zeros(T * k, dtype=torch.float64)
        want[perm], size[perm] = each.sum(1), each.abs().sum(1)
        # a thread adds at most H / 32 + 8 products, 32 lanes and 8 warps are added up by 5 + 8 additions
        _off_by(got[1].cpu(), want.view(T, k), size.view(T, k), H // 32 + 8 + 13)


def test_gradients_against_differences(cuda, lib):
    """A step: sort, permute, a product, weighted sum.  The result is bilinear in x and the weights: central differences
    have no error of their own, and every number here is a small multiple of 2^-6, so fp32 has none either."""
    g = torch.Generator().manual_seed(5)
    T, k, E, H = 12, 3, 4, 10

    def eighths(*shape):
        return torch.randint(-8, 9, shape, generator=g).to(cuda).float() / 8

    ids = _ids(T, k, E, g).to(cuda)
    x, w, scale, out = eighths(T, H), eighths(T, k), eighths(T * k, 1), eighths(T, H)
    sort = kernels.moe_sort(ids, E)

    def f(x, w):
        return (kernels.moe_unpermute(kernels.moe_permute(x, sort) * scale, sort, w) * out).sum()

    x.requires_grad_()
    w.requires_grad_()
    gx, gw = torch.autograd.grad(f(x, w), (x, w))
    with torch.no_grad():
        for _ in range(8):
            dx, dw = eighths(T, H), eighths(T, k)
            assert float((gx * dx).sum()) == float(f(x + dx, w) - f(x - dx, w)) / 2
            assert float((gw * dw).sum()) == float(f(x, w + dw) - f(x, w - dw)) / 2


def test_strided_and_expanded_inputs(cuda, lib):
    g = torch.Generator().manual_seed(6)
    T, k, E, H = 21, 4, 5, 64
    sort = kernels.moe_sort(_ids(T, k, E, g).to(cuda), E)
    base = torch.randn(T, 3 * H + 2, generator=g).bfloat16().to(cuda)
    for x in (base[:, :H], base[:, H:2 * H], base[:, 1:H + 1], base[:1, :H].expand(T, H), base[:, :2 * H:2], base[:, :H].T.contiguous().T):
        assert torch.equal(kernels.moe_permute(x, sort), kernels.moe_permute(x.contiguous(), sort))
    wide = torch.randn(T * k, 2 * H + 1, generator=g).bfloat16().to(cuda)
    w = torch.randn(k, T, generator=g).to(cuda).T
    for rows in (wide[:, :H], wide[:, H:2 * H], wide[:, 1:H + 1], wide[:, :2 * H:2]):
        assert torch.equal(kernels.moe_unpermute(rows, sort, w), kernels.moe_unpermute(rows.contiguous(), sort, w.contiguous()))
    rows = wide[:, 1:H + 1].requires_grad_()
    w = w.detach().requires_grad_()
    a = torch.autograd.grad(kernels.moe_unpermute(rows, sort, w).sum(), (rows, w))      # the incoming gradient has stride 0
    one = torch.ones(T, H, dtype=torch.bfloat16, device=cuda)
    r2 = rows.detach().contiguous().requires_grad_()
    b = torch.autograd.grad(kernels.moe_unpermute(r2, sort, w), (r2, w), one)
    assert torch.equal(a[0], b[0])
    assert (a[1] - b[1]).abs().max() <= 2 * (H // 32 + 21) * U * rows.detach().float().abs().sum(1).max()   # other vector widths: another order of the sum


def test_one_gradient_at_a_time(cuda, lib):
    g = torch.Generator().manual_seed(7)
    T, k, E, H = 19, 5, 4, 72
    sort = kernels.moe_sort(_ids(T, k, E, g).to(cuda), E)
    rows, gy = torch.randn(T * k, H, generator=g).half().to(cuda), torch.randn(T, H, generator=g).half().to(cuda)
    w = torch.rand(T, k, generator=g).to(cuda)
    r, v = rows.clone().requires_grad_(), w.clone().requires_grad_()
    both = torch.autograd.grad(kernels.moe_unpermute(r, sort, v), (r, v), gy)
    assert torch.equal(torch.autograd.grad(kernels.moe_unpermute(r, sort, w), r, gy)[0], both[0])
    assert torch.equal(torch.autograd.grad(kernels.moe_unpermute(rows, sort, v), v, gy)[0], both[1])
    assert not kernels.moe_unpermute(rows, sort, w).requires_grad
    with torch.no_grad():
        assert not kernels.moe_unpermute(r, sort, v).requires_grad and not kernels.moe_permute(gy.clone().requires_grad_(), sort).requires_grad


def test_rows_that_are_not_numbers(cuda, lib):
    """A NaN or infinity in one token's row reaches that token's results and no other's."""
    T, k, E, H = 6, 2, 3, 40
    ids = torch.tensor([[0, 1], [1, 2], [2, 0], [0, 0], [1, -1], [-1, -1]], device=cuda)
    sort = kernels.moe_sort(ids, E)
    x = torch.ones(T, H, device=cuda)
    x[1, 3], x[3, 0] = float("nan"), float("inf")
    y = kernels.moe_unpermute(kernels.moe_permute(x, sort), sort, torch.full((T, k), 0.5, device=cuda))
    want = torch.tensor([1.0, 1.0, 1.0, 1.0, 0.5, 0.0], device=cuda).unsqueeze(1).repeat(1, H)
    want[1, 3], want[3, 0] = float("nan"), float("inf")
    assert torch.equal(torch.nan_to_num(y, nan=-7.0), torch.nan_to_num(want, nan=-7.0))


def test_many_rows(cuda, lib):
    """Rows whose offsets pass 2^31 elements: 300 k rows of 7200."""
    T, k, E, H = 75_000, 4, 16, 7200
    g = torch.Generator(device=cuda).manual_seed(8)
    sort = kernels.moe_sort(torch.randint(0, E, (T, k), device=cuda, generator=g, dtype=torch.int32), E)
    x = torch.randint(0, 256, (T, H), device=cuda, generator=g, dtype=torch.uint8).to(torch.bfloat16)
    rows = kernels.moe_permute(x, sort)
    at = torch.tensor([0, 1, T * k // 2, T * k - 2, T * k - 1], device=cuda)
    assert torch.equal(rows[at], x[sort.perm[at].long() // k])
    y = kernels.moe_unpermute(rows, sort, torch.full((T, k), 0.25, device=cuda))
    assert torch.equal(y, x)               # a quarter of four equal numbers each: exact
    ops.check_status(cuda)


def test_training_step_in_a_graph(cuda, lib):
    """Captured with its gradients and replayed on other inputs; two graphs of the same operators do not disturb each other."""
    g = torch.Generator().manual_seed(9)
    T, k, E, H = 50, 3, 7, 136
    def inputs():
        return [_ids(T, k, E, g).to(cuda), torch.randn(T, H, generator=g).bfloat16().to(cuda),
                torch.rand(T, k, generator=g).to(cuda), torch.randn(T, H, generator=g).bfloat16().to(cuda)]

    def step(ids, x, w, gy):
        x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
        sort = kernels.moe_sort(ids, E)
        y = kernels.moe_unpermute(kernels.moe_permute(x, sort), sort, w)
        return (y.detach(), *torch.autograd.grad(y, (x, w), gy))

    graphs = []
    for _ in range(2):
        static = inputs()
        side = torch.cuda.Stream(cuda)
        side.wait_stream(torch.cuda.current_stream(cuda))
        with torch.cuda.stream(side):
            step(*static)
        torch.cuda.current_stream(cuda).wait_stream(side)
        torch.cuda.synchronize(cuda)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*static)
        graphs.append((graph, static, out))
    for _ in range(2):
        fresh = [inputs(), inputs()]
        for (graph, static, _), new in zip(graphs, fresh):
            for a, b in zip(static, new):
                a.copy_(b)
            graph.replay()
        for (_, _, out), new in zip(graphs, fresh):
            for a, b in zip(out, step(*new)):
                assert torch.equal(a, b)


def test_on_another_stream(cuda, lib):
    g = torch.Generator().manual_seed(10)
    T, k, E, H = 400, 4, 9, 512
    ids, x = _ids(T, k, E, g).to(cuda), torch.randn(T, H, generator=g).to(cuda)
    sort = kernels.moe_sort(ids, E)
    want = kernels.moe_unpermute(kernels.moe_permute(x, sort), sort)
    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(side):
        s = kernels.moe_sort(ids, E)
        got = kernels.moe_unpermute(kernels.moe_permute(x, s), s)
    side.synchronize()
    assert torch.equal(got, want)
