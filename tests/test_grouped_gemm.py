"""Products of ragged groups of rows against products in 64 bits, group by group, and their refusals.

Tolerances.  fp32 sums of n products of bf16 numbers (exact in fp32) have an error of at most n 2^-24 of the sum of their magnitudes,
and the result is rounded to bf16 once: half a step, 2^-8 of the value."""
import itertools

import pytest
import torch


def _gg(x, w, ends):
    from mccl_b200.ops.gemm import grouped_gemm
    return grouped_gemm(x, w, ends)


def _bf(*shape, std=1.0):
    return (torch.randn(*shape, device="cuda") * std).to(torch.bfloat16)


def _close(got, want, magnitudes, n, what):
    limit = 2.0 ** -8 * want.abs() + n * 2.0 ** -24 * magnitudes + 2.0 ** -133
    got = got.double()
    assert got.shape == want.shape and torch.isfinite(got).all(), what
    off = (got - want).abs() - limit
    assert (off <= 0).all(), f"{what}: largest excess {off.max().item():.3g} at {torch.nonzero(off == off.max())[0].tolist()}"


def _groups(sizes):
    ends = list(itertools.accumulate(sizes))
    return [(e - s, e) for s, e in zip(sizes, ends)], ends


def _check(x, w, dy, sizes, y, dx, dw):
    """Rows behind the last group are zero in y and dx."""
    spans, ends = _groups(sizes)
    x, w, dy = x.double(), w.double(), dy.double()
    K, N = x.shape[1], w.shape[1]
    for e, (lo, hi) in enumerate(spans):
        a, b, g = x[lo:hi], w[e], dy[lo:hi]
        _close(y[lo:hi], a @ b.t(), a.abs() @ b.abs().t(), K, f"y of group {e}")
        if dx is not None:
            _close(dx[lo:hi], g @ b, g.abs() @ b.abs(), N, f"dx of group {e}")
            _close(dw[e], g.t() @ a, g.abs().t() @ a.abs(), hi - lo, f"dw of group {e}")
    assert (y[ends[-1]:] == 0).all()
    assert dx is None or (dx[ends[-1]:] == 0).all()


def _run(x, w, ends, dy):
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    y = _gg(x, w, ends)
    return y.detach(), *torch.autograd.grad(y, [x, w], dy)


@pytest.fixture(autouse=True)
def _seed():
    torch.manual_seed(0)


CASES = [([1], 8, 8), ([1], 64, 64), ([2, 0, 1], 72, 136), ([0, 5, 0, 130, 1, 0], 64, 64), ([127, 128, 129, 256, 257], 136, 264), ([300], 1032, 264),
         ([63, 64, 65, 1, 0, 191], 520, 776), ([700, 20], 256, 1024), ([33] * 70, 128, 192), ([1024, 3, 2048], 512, 512), ([5, 9], 2048, 64),
         ([17], 8, 2048), ([1] * 9, 256, 2056), ([16, 0, 48, 33], 2064, 520), ([127, 128, 129, 256, 257], 136, 4104), ([1024, 3, 2048, 0, 700], 520, 1032),
         ([1, 0, 2, 140], 1000, 8200), ([300, 0, 1], 8192, 136), ([128] * 30, 64, 640), ([2051, 1100], 264, 5000), ([2051, 1100], 2600, 1032), ([0, 3000, 77], 1032, 4104),
         ([2100], 4096, 2056), ([1, 4200, 0, 63], 2048, 2312)]


@pytest.mark.gpu
@pytest.mark.parametrize("sizes,K,N", CASES)
def test_against_64_bits(sizes, K, N):
    T, E = sum(sizes), len(sizes)
    x, w, dy = _bf(T, K), _bf(E, N, K, std=K ** -0.5), _bf(T, N)
    ends = torch.tensor(sizes, device="cuda").cumsum(0)
    for e in (ends, ends.int()):
        _check(x, w, dy, sizes, *_run(x, w, e, dy))
    with torch.no_grad():
        _check(x, w, dy, sizes, _gg(x, w, ends), None, None)


@pytest.mark.gpu
def test_many_experts():
    sizes = [(i * 7) % 5 for i in range(1024)]
    T, K, N = sum(sizes), 64, 72
    x, w, dy = _bf(T, K), _bf(1024, N, K), _bf(T, N)
    _check(x, w, dy, sizes, *_run(x, w, torch.tensor(sizes, device="cuda").cumsum(0), dy))


@pytest.mark.gpu
@pytest.mark.parametrize("T,K,N", [(5, 200, 328), (200, 200, 328), (1500, 200, 328), (6000, 2600, 2312)])
def test_rows_behind_the_last_group(T, K, N):
    """They may hold anything, and so may the rows of other groups: no group sees them."""
    sizes = [T // 5, 0, T // 3]
    used = sum(sizes)
    x, w, dy = _bf(T, K), _bf(3, N, K), _bf(T, N)
    x[used:], dy[used:] = float("nan"), float("inf")
    y, dx, dw = _run(x, w, torch.tensor(sizes, device="cuda").cumsum(0), dy)
    _check(x[:used], w, dy[:used], sizes, y[:used], dx[:used], dw)
    assert (y[used:] == 0).all() and (dx[used:] == 0).all()
    # NaN in one group stays in it
    x[:sizes[0]] = float("nan")
    y, dx, dw = _run(x, w, torch.tensor(sizes, device="cuda").cumsum(0), dy)
    lo = sizes[0]
    _check(x[lo:used], w[2:], dy[lo:used], sizes[2:], y[lo:used], dx[lo:used], dw[2:])
    assert y[:lo].isnan().all() and dw[0].isnan().all() and (dw[1] == 0).all() and torch.isfinite(dx).all()
    # of weights, too: an expert without rows may hold anything
    x[:lo], w[1] = 1.0, float("nan")
    y, dx, dw = _run(x, w, torch.tensor(sizes, device="cuda").cumsum(0), dy)
    assert torch.isfinite(y).all() and torch.isfinite(dx).all() and (dw[1] == 0).all()


@pytest.mark.gpu
def test_ends_out_of_order_or_range_are_read_as_the_nearest():
    T, K, N = 300, 64, 64
    x, w, dy = _bf(T, K), _bf(5, N, K), _bf(T, N)
    for ends, sizes in (([100, 50, 150, 1000, -3], [100, 0, 50, 150, 0]), ([-5, 2 ** 40, 7, 8, 9], [0, 300, 0, 0, 0]), ([0] * 5, [0] * 5),
                        ([-2 ** 40] * 4 + [1], [0, 0, 0, 0, 1])):
        y, dx, dw = _run(x, w, torch.tensor(ends, device="cuda"), dy)
        _check(x, w, dy, sizes, y, dx, dw)


@pytest.mark.gpu
def test_no_rows():
    x, w = _bf(0, 64), _bf(3, 32, 64)
    y, dx, dw = _run(x, w, torch.zeros(3, dtype=torch.int32, device="cuda"), _bf(0, 32))
    assert y.shape == (0, 32) and dx.shape == (0, 64) and (dw == 0).all() and dw.shape == w.shape


@pytest.mark.gpu
def test_strided_and_unaligned_operands():
    sizes, K, N = [40, 0, 90], 72, 80
    T = sum(sizes)
    x, w, dy = _bf(T, K), _bf(3, N, K), _bf(T, N)
    ends = torch.tensor(sizes, device="cuda").cumsum(0).int()
    want = _run(x, w, ends, dy)
    wide = _bf(T, K + 24)
    for off in (8, 5):                                           # rows further apart, at a 16-byte boundary and not
        view = wide[:, off:off + K]
        view.copy_(x)
        assert all(torch.equal(a, b) for a, b in zip(want, _run(view, w, ends, dy)))
    turned = x.t().contiguous().t()
    store = torch.empty(3 * N * K + 3, device="cuda", dtype=torch.bfloat16)
    odd = store[3:].view(3, N, K)
    odd.copy_(w)
    turned_w = w.transpose(1, 2).contiguous().transpose(1, 2)
    one = _bf(1, N).expand(T, N)                                 # a gradient of one row for all of them, as of a sum
    assert all(torch.equal(a, b) for a, b in zip(want, _run(turned, odd, ends, dy.t().contiguous().t())))
    assert all(torch.equal(a, b) for a, b in zip(want, _run(x, turned_w, ends, dy)))
    assert all(torch.equal(a, b) for a, b in zip(_run(x, w, ends, one.contiguous()), _run(x, w, ends, one)))


@pytest.mark.gpu
def test_partial_gradients_and_second_derivative():
    sizes, K, N = [40, 7], 64, 48
    ends = torch.tensor(sizes, device="cuda").cumsum(0)
    x, w, dy = _bf(47, K), _bf(2, N, K), _bf(47, N)
    _, dx, dw = _run(x, w, ends, dy)
    xr, wr = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(_gg(xr, w, ends), xr, dy)[0], dx)
    assert torch.equal(torch.autograd.grad(_gg(x, wr, ends), wr, dy)[0], dw)
    (g,) = torch.autograd.grad(_gg(xr, wr, ends), xr, dy, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.float().sum(), wr)


@pytest.mark.gpu
def test_gradients_against_differences():
    """y is linear in x and in w: a step along d changes <y, g> by <gradient, d> times the step, up to the roundings of the two results
    (2^-8 of each value) and of the gradient (2^-8)."""
    sizes, K, N = [40, 0, 65], 64, 40
    ends = torch.tensor(sizes, device="cuda").cumsum(0)
    x, w, dy = _bf(105, K), _bf(3, N, K, std=0.125), _bf(105, N)
    _, dx, dw = _run(x, w, ends, dy)
    for grad, args in ((dx, lambda d: (x + d, w)), (dw, lambda d: (x, w + d))):
        d = (torch.randint(0, 2, grad.shape, device="cuda") * 2 - 1).to(torch.bfloat16) * 0
        d.view(-1)[:: 7] = 4.0
        up, down = (args(s * d) for s in (1, -1))
        exact = [(a.double(), b.double()) for a, b in (up, down)]       # the steps as bf16 took them
        hi, lo = (_gg(a.contiguous(), b.contiguous(), ends).double() for a, b in (up, down))
        got = ((hi - lo) * dy.double()).sum()
        moved = (exact[0][0] - exact[1][0]) if grad is dx else (exact[0][1] - exact[1][1])
        want = (grad.double() * moved).sum()
        limit = 2.0 ** -8 * ((hi.abs() + lo.abs()) * dy.double().abs()).sum() + 2.0 ** -8 * (grad.double() * moved).abs().sum() + 1e-3
        assert abs(got - want) <= limit


@pytest.mark.gpu
def test_same_bits_on_another_stream_and_from_a_graph():
    sizes, K, N = [400, 0, 333, 1], 256, 320
    T = sum(sizes)
    x, w, dy = _bf(T, K), _bf(4, N, K), _bf(T, N)
    ends = torch.tensor(sizes, device="cuda").cumsum(0)
    first = _run(x, w, ends, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    xs, ws = x.clone().requires_grad_(True), w.clone().requires_grad_(True)

    def step():
        y = _gg(xs, ws, ends)
        return y.detach(), *torch.autograd.grad(y, [xs, ws], dy)
    with torch.cuda.stream(side):
        second = step()
        step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(first, out))
    other = [0, 100, 600, 20]                                    # the replayed graph reads the ends that are there then
    ends.copy_(torch.tensor(other).cumsum(0))
    graph.replay()
    _check(x, w, dy, other, *out)
    from mccl_b200.ops.gemm import last_error
    assert last_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("sizes,K,N", [([9, 0, 30], 264, 200), ([700, 0, 1900], 520, 1032), ([2500, 2700], 1032, 2312)])
def test_gradients_right_behind_what_makes_them(sizes, K, N):
    """The second product of a backward pass runs beside the first one: operands written just before, results read just behind, over memory that
    is used again and again."""
    T, E = sum(sizes), len(sizes)
    xs, ws, dys = [_bf(T, K) for _ in range(3)], [_bf(E, N, K) for _ in range(3)], [_bf(T, N) for _ in range(3)]
    ends = torch.tensor(sizes, device="cuda").cumsum(0)
    want = [_run(x, w, ends, dy) for x, w, dy in zip(xs, ws, dys)]
    torch.cuda.synchronize()
    x, w, dy = torch.empty_like(xs[0]).requires_grad_(True), torch.empty_like(ws[0]).requires_grad_(True), torch.empty_like(dys[0])
    big, wrong = torch.randn(4096, 4096, device="cuda"), torch.zeros((), device="cuda")
    for turn in range(30):
        i = turn % 3
        big = big @ big * 1e-2                                       # what follows is queued while this runs
        with torch.no_grad():
            x.copy_(xs[i])
            w.copy_(ws[i])
            dy.copy_(dys[i])
        y = _gg(x, w, ends)
        dx, dw = torch.autograd.grad(y, [x, w], dy)
        wrong += (y != want[i][0]).sum() + (dx != want[i][1]).sum() + (dw != want[i][2]).sum()
        del y, dx, dw
    assert wrong.item() == 0


def test_refusals():
    x, w, ends = torch.zeros(4, 16, dtype=torch.bfloat16), torch.zeros(2, 8, 16, dtype=torch.bfloat16), torch.tensor([2, 4])
    with pytest.raises(RuntimeError, match="CUDA"):
        _gg(x, w, ends)
    for bad in ((x[0], w, ends), (x, w[0], ends), (x[:, :8], w, ends), (x, w, ends[:1]), (x, w, ends.float()), (x, w, ends[:, None]),
                (x.float(), w, ends), (x, w.half(), ends), (x[:, :12], w[:, :, :12], ends), (x, w[:, :7], ends), (x, w[:0], ends[:0]),
                (x[:, :0], w[:, :, :0], ends), (x, w, torch.zeros(4, dtype=torch.int64)[::2]),
                (x, torch.zeros(1025, 8, 16, dtype=torch.bfloat16), torch.zeros(1025, dtype=torch.int64))):
        with pytest.raises(ValueError):
            _gg(*bad)


@pytest.mark.gpu
@pytest.mark.parametrize("T,E,K,N", [(900, 33, 8192, 8192), (280000, 2, 8192, 136), (280000, 2, 136, 8192)])
def test_more_elements_than_32_bits_count(T, E, K, N):
    """Weights, rows and results of 2^31 elements and more: the first group's ends and the last one's."""
    x, w, dy = _bf(T, K), torch.empty(E, N, K, device="cuda", dtype=torch.bfloat16).normal_(std=K ** -0.5), torch.empty(T, N, device="cuda", dtype=torch.bfloat16).normal_()
    ends = torch.arange(1, E + 1, device="cuda") * (T - 50) // E
    y, dx, dw = _run(x, w, ends, dy)
    for e in (0, E - 1):
        lo, hi = 0 if e == 0 else int(ends[e - 1]), int(ends[e])
        rows, cols = torch.tensor([lo, hi - 1], device="cuda"), torch.tensor([0, N - 1], device="cuda")
        a, g, b, d = x[rows].double(), dy[rows].double(), w[e].double(), dy[lo:hi][:, cols].double()
        _close(y[rows], a @ b.t(), a.abs() @ b.abs().t(), K, f"y of group {e}")
        _close(dx[rows], g @ b, g.abs() @ b.abs(), N, f"dx of group {e}")
        a = x[lo:hi].double()
        _close(dw[e][cols], d.t() @ a, d.abs().t() @ a.abs(), hi - lo, f"dw of group {e}")
    assert (y[T - 50:] == 0).all() and (dx[T - 50:] == 0).all()
