"""8-bit products by blocks of 128: the quantisation bit for bit, the product against 64 bits on the quantised values, and refusals.

Tolerances.  Products of two e4m3 numbers and powers of two are exact.  Their fp32 sums over K have an error of at most 2 K 2^-24 of the sum
of their magnitudes (the tensor core may cut bits where an fp32 addition would round: a whole step, not half), and the result is
rounded to bf16 once: half a step, 2^-8 of the value."""
import itertools

import pytest
import torch


def _fp8():
    from mccl_b200.ops import fp8
    return fp8


def _bf(*shape, std=1.0):
    return (torch.randn(*shape, device="cuda") * std).to(torch.bfloat16)


def _scaled(*shape):
    """Values whose blocks differ much in size."""
    return (torch.randn(*shape, device="cuda") * torch.exp2(torch.randint(-9, 10, (*shape[:-1], 1), device="cuda").float())
            * torch.exp(torch.randn(shape[-1], device="cuda"))).to(torch.bfloat16)


def _pow2(e):
    """2^e exactly, for whole e from -1022 on."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _plain(x, rows):
    """e4m3 values (as fp64) and exponents from the definition, in 64 bits."""
    m, k = x.shape[-2:]
    b = torch.nn.functional.pad(x.double(), (0, -k % 128, 0, -m % rows)).unflatten(-1, (-1, 128)).unflatten(-3, (-1, rows))
    finite = torch.where(torch.isfinite(b), b.abs(), 0.0)
    amax = finite.amax(dim=(-3, -1))
    mantissa, e = torch.frexp(amax / 448)                        # in [0.5, 1): only the powers of two themselves stay below their exponent
    e = torch.where(amax > 0, torch.where(mantissa == 0.5, e - 1, e).clamp(-127, 127), 0).double()
    v = b * _pow2(-e)[..., :, None, :, None]
    step = _pow2(torch.frexp(torch.where(torch.isfinite(v), v.abs(), 1.0).clamp(min=2.0 ** -6))[1] - 4)
    q = torch.round(v / step) * step
    q = torch.where(torch.isfinite(b), q, float("nan"))
    return q.flatten(-2).flatten(-3, -2)[..., :m, :k], e


def _value(q):
    return q.float().double()


def _exponent(s):
    return s.view(torch.uint8).double() - 127


def _dequantized(b):
    m, k = b.data.shape[-2:]
    s = _pow2(_exponent(b.scale))
    if s.shape[-2] != m:
        s = s.repeat_interleave(128, -2)[..., :m, :]
    return _value(b.data) * s.repeat_interleave(128, -1)[..., :k]


def _same(got, q, e):
    assert (_exponent(got.scale) == e).all()
    off = torch.nonzero(_value(got.data) != q)
    assert not len(off), f"{len(off)} values differ, the first {_value(got.data)[tuple(off[0])].item()} for {q[tuple(off[0])].item()} at {off[0].tolist()}"


@pytest.fixture(autouse=True)
def _seed():
    torch.manual_seed(0)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("shape", [(1, 16), (3, 128), (5, 144), (130, 272), (257, 2048), (1, 8192)])
def test_quantised_bit_for_bit(shape, rows):
    f = _fp8()
    x = _scaled(*shape)
    x[0, :8] = 0
    x[-1] = 0                                                    # a block of zeros, where a row is a block
    got = f.fp8_quantize(x, rows)
    q, e = _plain(x, rows)
    _same(got, q, e)
    assert torch.equal(got.dequantize().double(), _dequantized(got))
    if rows == 128:
        x3 = torch.stack([x, x * 3, x * 0])
        got = f.fp8_quantize(x3, rows)
        q, e = _plain(x3, rows)
        _same(got, q, e)


@pytest.mark.gpu
def test_quantisation_of_every_bf16_number():
    """Each as the largest of a block: the exponent's steps, subnormal numbers, the largest ones."""
    f = _fp8()
    every = torch.arange(0, 0x7f80, device="cuda", dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    x = torch.zeros(len(every), 128, device="cuda", dtype=torch.bfloat16)
    x[:, 77] = -every
    x[:, 3] = every / 3
    got = f.fp8_quantize(x)
    q, e = _plain(x, 1)
    _same(got, q, e)
    # and against a fixed scale: 448 in the block makes it one
    x = torch.zeros_like(x)
    x[:, 77], x[:, 0] = 448.0, every.clamp(max=448)
    got = f.fp8_quantize(x)
    assert (got.scale.view(torch.uint8) == 127).all()
    assert torch.equal(_value(got.data), _plain(x, 1)[0])


@pytest.mark.gpu
def test_what_is_not_finite_becomes_nan():
    f = _fp8()
    x = _bf(4, 256)
    x[0, 5], x[1, 200], x[2, 0] = float("inf"), float("-inf"), float("nan")
    x[3] = float("inf")
    got = f.fp8_quantize(x)
    q, e = _plain(x, 1)
    assert torch.equal(_exponent(got.scale), e)
    assert torch.equal(got.data.float().isnan(), ~torch.isfinite(x)) and torch.equal(_value(got.data).nan_to_num(), q.nan_to_num())
    w = f.fp8_quantize(_bf(16, 256), 128)
    y = f.fp8_gemm(x, w)
    assert y.isnan().all()
    x[0] = 1.0
    assert torch.isfinite(f.fp8_gemm(x, w)[0]).all()


def _product(x, w, y):
    want, mag = x @ w.t(), x.abs() @ w.abs().t()
    limit = 2.0 ** -8 * want.abs() + 2 * x.shape[1] * 2.0 ** -24 * mag + 2.0 ** -133
    assert y.dtype == torch.bfloat16 and y.shape == want.shape and torch.isfinite(y).all()
    off = (y.double() - want).abs() - limit
    assert (off <= 0).all(), f"largest excess {off.max().item():.3g} at {torch.nonzero(off == off.max())[0].tolist()}"


SHAPES = [(1, 8, 16), (1, 128, 128), (2, 136, 144), (16, 256, 512), (17, 264, 528), (33, 512, 640), (64, 1032, 2064), (65, 128, 4096), (100, 11008, 256),
          (128, 520, 1024), (129, 776, 1040), (300, 1024, 2048), (1000, 200, 656), (2049, 2056, 528), (5, 8, 8192), (1, 5504, 4096), (640, 2048, 128), (1500, 2000, 1040), (4100, 1024, 272), (3, 2048, 400), (400, 136, 8192), (1, 11008, 4096)]


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product_against_64_bits(M, N, K):
    f = _fp8()
    x, w = f.fp8_quantize(_scaled(M, K)), f.fp8_quantize(_scaled(N, K), 128)
    y = f.fp8_gemm(x, w)
    _product(_dequantized(x), _dequantized(w), y)


@pytest.mark.gpu
def test_rows_in_bf16_are_quantised_within_the_call():
    f = _fp8()
    for M in (1, 40, 700):
        x, w = _scaled(M, 400), f.fp8_quantize(_scaled(264, 400), 128)
        assert torch.equal(f.fp8_gemm(x, w), f.fp8_gemm(f.fp8_quantize(x), w))


GROUPS = [([1], 64, 128), ([2, 0, 1], 136, 144), ([0, 5, 0, 130, 1, 0], 64, 272), ([127, 128, 129, 256, 257], 264, 400), ([33] * 70, 192, 128),
          ([1024, 3, 2048], 512, 512), ([1] * 9, 2056, 256), ([16, 0, 48, 33], 520, 2064), ([700, 20], 1024, 1296), ([127, 128, 129, 256, 257], 4104, 144),
          ([1024, 3, 2048, 0, 700], 1032, 528), ([1, 0, 2, 140], 8200, 1008), ([300, 0, 1], 136, 8192)]


@pytest.mark.gpu
@pytest.mark.parametrize("behind", [0, 77])
@pytest.mark.parametrize("sizes,N,K", GROUPS)
def test_ragged_groups(sizes, N, K, behind):
    f = _fp8()
    T, ends = sum(sizes), list(itertools.accumulate(sizes))
    x, w = _scaled(T + behind, K), _scaled(len(sizes), N, K)
    x[T:] = float("nan")
    x, w = f.fp8_quantize(x), f.fp8_quantize(w, 128)
    xd, wd = _dequantized(x), _dequantized(w)
    for dtype in (torch.int32, torch.int64):
        y = f.fp8_gemm(x, w, torch.tensor(ends, device="cuda", dtype=dtype))
        for e, (size, end) in enumerate(zip(sizes, ends)):
            _product(xd[end - size:end], wd[e], y[end - size:end])
        assert (y[T:] == 0).all()


@pytest.mark.gpu
def test_no_rows():
    f = _fp8()
    w = f.fp8_quantize(_bf(2, 24, 64), 128)
    assert f.fp8_gemm(_bf(0, 64), f.BlockScaled(w.data[0], w.scale[0])).shape == (0, 24)
    assert f.fp8_gemm(_bf(0, 64), w, torch.zeros(2, dtype=torch.int32, device="cuda")).shape == (0, 24)
    assert f.fp8_quantize(_bf(0, 64)).data.shape == (0, 64)


@pytest.mark.gpu
def test_strided_and_unaligned_operands():
    f = _fp8()
    M, N, K = 40, 136, 656                                       # six blocks: scales of another pitch are copied
    x, w = _scaled(M, K), _scaled(N, K)
    xq, wq = f.fp8_quantize(x), f.fp8_quantize(w, 128)
    want = f.fp8_gemm(xq, wq)
    wide = _bf(M, K + 40)
    for off in (16, 5):
        view = wide[:, off:off + K]
        view.copy_(x)
        assert torch.equal(f.fp8_gemm(view, wq), want)
        assert torch.equal(f.fp8_quantize(view).data.view(torch.uint8), xq.data.view(torch.uint8))
    raw = torch.empty(M, K + 40, device="cuda", dtype=torch.uint8)
    for off in (16, 3):
        view = raw[:, off:off + K]
        view.copy_(xq.data.view(torch.uint8))
        data = view.view(torch.float8_e4m3fn)
        assert torch.equal(f.fp8_gemm(f.BlockScaled(data, xq.scale), wq), want)
    tight = lambda s: s.view(torch.uint8).contiguous().view(torch.float8_e8m0fnu)  # noqa: E731
    assert torch.equal(f.fp8_gemm(f.BlockScaled(xq.data, tight(xq.scale)), f.BlockScaled(wq.data, tight(wq.scale))), want)
    # weights as they are quantised (rows a multiple of 128 apart), without gaps, and with rows no multiple of 16 apart
    assert wq.data.stride(0) == 768
    for pitch in (656, 661):
        store = torch.empty(N, pitch, device="cuda", dtype=torch.uint8)
        store[:, :K] = wq.data.view(torch.uint8)
        assert torch.equal(f.fp8_gemm(xq, f.BlockScaled(store[:, :K].view(torch.float8_e4m3fn), wq.scale)), want)
    turned = f.BlockScaled(xq.data.view(torch.uint8).t().contiguous().t().view(torch.float8_e4m3fn),
                           xq.scale.view(torch.uint8).t().contiguous().t().view(torch.float8_e8m0fnu))
    assert torch.equal(f.fp8_gemm(turned, wq), want)
    assert torch.equal(f.fp8_gemm(x.t().contiguous().t(), wq), want)


@pytest.mark.gpu
def test_same_bits_on_another_stream_and_from_a_graph():
    f = _fp8()
    w = f.fp8_quantize(_bf(3, 264, 400), 128)
    ends = torch.tensor([4, 4, 30], device="cuda")
    x = _scaled(33, 400)
    first = f.fp8_gemm(x, w, ends)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = f.fp8_gemm(x, w, ends)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, second)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = f.fp8_gemm(x, w, ends)
    graph.replay()
    assert torch.equal(first, out)
    x.copy_(_scaled(33, 400))
    ends.copy_(torch.tensor([0, 33, 33]))
    graph.replay()
    assert torch.equal(out, f.fp8_gemm(x, w, ends))
    from mccl_b200.ops.gemm import last_error
    assert last_error() == 0


@pytest.mark.gpu
def test_rows_that_ask_for_a_gradient_are_refused():
    f = _fp8()
    x, w = _bf(4, 64).requires_grad_(True), f.fp8_quantize(_bf(16, 64), 128)
    with pytest.raises(RuntimeError, match="gradient"):
        f.fp8_gemm(x, w)
    with torch.no_grad():
        assert torch.equal(f.fp8_gemm(x, w), f.fp8_gemm(x.detach(), w))


def _empty(*shape, dtype):
    return torch.zeros(*shape, dtype=torch.uint8).view(dtype)


def test_refusals():
    f = _fp8()
    e4, e8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
    x, w = torch.zeros(4, 256, dtype=torch.bfloat16), f.BlockScaled(_empty(24, 256, dtype=e4), _empty(1, 2, dtype=e8))
    x8, w3 = f.BlockScaled(_empty(4, 256, dtype=e4), _empty(4, 2, dtype=e8)), f.BlockScaled(_empty(2, 24, 256, dtype=e4), _empty(2, 1, 2, dtype=e8))
    ends = torch.tensor([1, 4])
    for args in ((x, w), (x8, w), (x, w3, ends)):
        with pytest.raises(RuntimeError, match="CUDA"):
            f.fp8_gemm(*args)
    for args in ((x.float(), w), (x[:, :128], w), (x[0], w), (x, w3), (x, w, ends), (x, w3, ends[:1]), (x, w3, ends.float()),
                 (x, f.BlockScaled(w.data, w.scale[:, :1])), (x, f.BlockScaled(w.data, w.scale.view(torch.uint8))), (x, f.BlockScaled(w.data.view(torch.uint8), w.scale)),
                 (x, f.BlockScaled(w.data[:20], w.scale)), (f.BlockScaled(x8.data, x8.scale[:1]), w), (f.BlockScaled(x, x8.scale), w),
                 (x[:, :40], f.BlockScaled(w.data[:, :40], w.scale[:, :1])), (x[:, :0], f.BlockScaled(w.data[:, :0], w.scale[:, :0]))):
        with pytest.raises(ValueError):
            f.fp8_gemm(*args)
    with pytest.raises(RuntimeError, match="CUDA"):
        f.fp8_quantize(x)
    for args in ((x, 2), (x.float(),), (x[0],), (x[None],), (x[:, :40],), (x[:, :0],), (x[None, None], 128), (x[:0], 128)):
        with pytest.raises(ValueError):
            f.fp8_quantize(*args)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [3, 40, 2500])
def test_calls_right_behind_what_makes_their_operands(M):
    """Kernels of a call start before those in front of them have ended: rows, weights and ends that are written just before, by a long
    kernel, and results that are read just behind, over memory that is used again and again."""
    f = _fp8()
    N, K = 264, 528
    rows, weights = [_scaled(M, K) for _ in range(4)], [f.fp8_quantize(_bf(2, N, K), 128) for _ in range(4)]
    ends = [torch.tensor([i, M], device="cuda") for i in range(4)]
    want = [[f.fp8_gemm(x, w, e).clone() for x, e in zip(rows, ends)] for w in weights]
    torch.cuda.synchronize()
    x, e = torch.empty_like(rows[0]), torch.empty_like(ends[0])
    w = f.BlockScaled(torch.empty_like(weights[0].data), torch.empty_like(weights[0].scale))
    big = torch.randn(4096, 4096, device="cuda")
    wrong = torch.zeros((), device="cuda")
    for turn in range(40):
        i, j = turn % 4, turn // 4 % 4
        big = big @ big * 1e-2                                       # what follows is queued while this runs
        x.copy_(rows[i])
        e.copy_(ends[i])
        w.data.view(torch.uint8).copy_(weights[j].data.view(torch.uint8))
        w.scale.view(torch.uint8).copy_(weights[j].scale.view(torch.uint8))
        y = f.fp8_gemm(x, w, e)
        wrong += (y != want[j][i]).sum()
        del y
    assert wrong.item() == 0


@pytest.mark.gpu
def test_large_product_from_a_graph():
    f = _fp8()
    x, w = _scaled(2500, 528), f.fp8_quantize(_bf(1032, 528), 128)
    want = f.fp8_gemm(x, w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = f.fp8_gemm(x, w)
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("before", ["nothing", "copy", "from_host", "memset", "join", "join_of_a_copy"])
def test_captured_behind_other_work(before):
    """The kernel that quantises starts early behind what is in front of it, whatever that is in a graph: nothing, a kernel, a copy from the
    host, a memset, another stream's work."""
    f = _fp8()
    source, w = _scaled(48, 528), f.fp8_quantize(_bf(264, 528), 128)
    host, x, big = source.cpu().pin_memory(), torch.empty_like(source), torch.randn(1 << 24, device="cuda")
    want = f.fp8_gemm(torch.zeros_like(source) if before == "memset" else source, w)

    def call():
        if before == "nothing":
            return f.fp8_gemm(source, w)
        if before == "copy":
            x.copy_(source)
        elif before == "from_host":
            x.copy_(host, non_blocking=True)
        elif before == "memset":
            x.zero_()
        else:
            here, side = torch.cuda.current_stream(), torch.cuda.Stream()
            side.wait_stream(here)
            with torch.cuda.stream(side):
                big.mul_(1.0)                                        # long beside what follows here
                x.copy_(host if before == "join_of_a_copy" else source, non_blocking=True)
            if before == "join":
                big.sum()
            here.wait_stream(side)
        return f.fp8_gemm(x, w)

    x.fill_(7)
    assert torch.equal(call(), want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for _ in range(3):
        x.fill_(7)
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("M,E,N,K", [(280000, 1, 136, 8192), (280000, 1, 8192, 272), (900, 33, 8192, 8192)])
def test_more_elements_than_32_bits_count(M, E, N, K):
    """Rows, results and weights of 2^31 elements and more: the first rows and the last ones."""
    f = _fp8()
    x, raw = _bf(M, K), torch.empty(E, N, K, device="cuda", dtype=torch.bfloat16).normal_()
    w, ends = f.fp8_quantize(raw, 128), torch.arange(1, E + 1, device="cuda") * M // E
    q, y = f.fp8_quantize(x), f.fp8_gemm(x, w, ends)
    for rows, e in ((slice(0, 20), 0), (slice(M - 20, M), E - 1)):
        last = f.BlockScaled(q.data[rows], q.scale[rows])
        _same(last, *_plain(x[rows], 1))
        expert = f.BlockScaled(w.data[e], w.scale[e])
        _same(expert, *_plain(raw[e], 128))
        _product(_dequantized(last), _dequantized(expert), y[rows])
