"""What the ragged and the 8-bit products do when a wait of theirs runs out: the limit is made so short that it does.

Contractions are long, so that the sums of a tile are not there when the epilogue looks for them, twice within two microseconds: 60 blocks and
more a CTA, at 0.1 us and more each."""
import contextlib

import pytest
import torch

pytestmark = pytest.mark.gpu


@contextlib.contextmanager
def _limit(ns, block_ns=0):
    """Waits of the products launched meanwhile may take so long, and so much longer for each block of the contractions they cover."""
    import ctypes as C
    from mccl_b200 import _lib
    set_ns = _lib.load().mcclDbgGemmWaitNs
    set_ns.argtypes, set_ns.restype = [C.c_uint64, C.c_uint64], None
    set_ns(ns, block_ns)
    try:
        yield
    finally:
        set_ns(2_000_000_000, 20_000)


def _bf(*shape, std=1.0):
    return (torch.randn(*shape, device="cuda") * std).to(torch.bfloat16)


def _ends(sizes):
    return torch.tensor(sizes, device="cuda").cumsum(0)


def _grouped(sizes, K, N, which):
    """A function that launches one product: y, or the gradient of x or w."""
    from mccl_b200.ops.gemm import grouped_gemm
    T, E, ends = sum(sizes), len(sizes), _ends(sizes)
    x, w, dy = _bf(T, K), _bf(E, N, K, std=K ** -0.5), _bf(T, N)
    if which == "y":
        return lambda: grouped_gemm(x, w, ends)
    leaf = (x if which == "dx" else w).requires_grad_(True)
    y = grouped_gemm(x, w, ends)
    return lambda: torch.autograd.grad(y, leaf, dy, retain_graph=True)[0]


def _fp8(M, K, N, sizes=None, quantised=True):
    from mccl_b200.ops import fp8
    x, w = _bf(M, K), fp8.fp8_quantize(_bf(*([len(sizes)] if sizes else []), N, K), rows=128)
    rows = fp8.fp8_quantize(x) if quantised else x
    ends = _ends(sizes) if sizes else None
    return lambda: fp8.fp8_gemm(rows, w, ends)


CASES = {
    "few rows": lambda: _grouped([2], 131072, 1024, "y"),
    "few rows of several experts": lambda: _grouped([2, 0, 3], 131072, 1024, "y"),
    "y, 256 columns": lambda: _grouped([375] * 8, 8192, 2048, "y"),
    "y, 128 columns": lambda: _grouped([625] * 32, 4096, 128, "y"),
    "dx, 256 columns": lambda: _grouped([375] * 8, 2048, 8192, "dx"),
    "dx, 128 columns": lambda: _grouped([625] * 32, 128, 4096, "dx"),
    "dw, 256 columns": lambda: _grouped([18100] + [100] * 19, 2048, 2048, "dw"),
    "dw, 128 columns": lambda: _grouped([20001], 512, 512, "dw"),
    "dw, few rows an expert": lambda: _grouped([3841] + [0] * 63, 520, 776, "dw"),
    "y, pairs": lambda: _grouped([5000, 3192], 8192, 2048, "y"),
    "dx, pairs": lambda: _grouped([5000, 3192], 2048, 8192, "dx"),
    "dw, pairs": lambda: _grouped([8192, 8200], 2048, 4096, "dw"),
    "8 bits, 256 columns": lambda: _fp8(2500, 16384, 4096),
    "8 bits, 128 columns": lambda: _fp8(20000, 16384, 128),
    "8 bits, ragged": lambda: _fp8(3000, 16384, 2048, [375] * 8, quantised=False),
    "8 bits, few rows": lambda: _fp8(3, 131072, 1024),
    "8 bits, few rows in bf16": lambda: _fp8(40, 131072, 1024, quantised=False),
}


@pytest.mark.parametrize("case", CASES)
def test_a_wait_that_runs_out_is_recorded_and_harms_nothing_else(case):
    from mccl_b200.ops.gemm import last_error
    torch.manual_seed(0)
    run = CASES[case]()
    want = run()
    torch.cuda.synchronize()
    assert last_error() == 0
    for _ in range(3):
        with _limit(1):
            run()
        torch.cuda.synchronize()
        assert last_error() != 0
        again = run()
        torch.cuda.synchronize()
        assert last_error() == 0 and torch.equal(again, want)


@pytest.mark.parametrize("case", ["few rows", "y, 256 columns", "dw, pairs", "8 bits, 256 columns", "8 bits, few rows in bf16"])
def test_no_product_follows_one_that_gave_up_unheard(case):
    from mccl_b200.ops.gemm import last_error
    torch.manual_seed(0)
    calls = {c: CASES[c]() for c in {case, "few rows", "y, 128 columns", "dx, 128 columns", "dw, 128 columns", "dx, pairs", "8 bits, 128 columns", "8 bits, few rows"}}
    want = {c: run() for c, run in calls.items()}
    torch.cuda.synchronize()
    with _limit(1):
        calls[case]()
    torch.cuda.synchronize()
    for run in calls.values():
        for _ in range(2):                                   # raising does not clear it
            with pytest.raises(RuntimeError, match="last_error"):
                run()
    assert last_error() != 0 and last_error() == 0
    for c, run in calls.items():
        assert torch.equal(run(), want[c])
    torch.cuda.synchronize()
    assert last_error() == 0


LONG = {
    "few rows": lambda: _grouped([20], 1 << 23, 8, "y"),
    "y, 128 columns": lambda: _grouped([1] * 300, 1 << 18, 8, "y"),
    "dx, 128 columns": lambda: _grouped([700], 8, 1 << 18, "dx"),
    "dw, 128 columns": lambda: _grouped([4000001], 8, 8, "dw"),
    "dw, few rows an expert": lambda: _grouped([65000] + [0] * 1023, 8, 8, "dw"),
    "dw, pairs": lambda: _grouped([131072, 65536, 90001], 2048, 4096, "dw"),
    "8 bits, 128 columns": lambda: _fp8(300, 1 << 19, 8, [1] * 300),
    "8 bits, few rows": lambda: _fp8(3, 1 << 26, 8),
}


@pytest.mark.parametrize("case", LONG)
def test_a_contraction_may_take_longer_than_a_wait(case):
    """The limit is for a kernel that stands still.  A tile's contraction takes 0.2 ms and more here, none of its blocks a hundredth of that."""
    from mccl_b200.ops.gemm import last_error
    torch.manual_seed(0)
    run = LONG[case]()
    want = run()
    torch.cuda.synchronize()
    assert last_error() == 0
    with _limit(100_000, 20_000):
        got = run()
    torch.cuda.synchronize()
    assert last_error() == 0 and torch.equal(got, want)
