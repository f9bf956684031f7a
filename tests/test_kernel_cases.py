"""The arguments and inputs of bench/kernel_cases.py."""
import importlib.util
import os

import pytest

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bench", "kernel_cases.py")


@pytest.fixture(scope="module")
def cases():
    spec = importlib.util.spec_from_file_location("kernel_cases", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("argv,n,k", [("gemm", 3584, 8192), ("fp8", 3584, 8192), ("grouped", 2048, 1024), ("policy", 50257, None),
                                      ("policy --n 3584", 3584, None), ("grouped --n 3584 --k 8192", 3584, 8192), ("gemm --n 50257", 50257, 8192)])
def test_a_size_that_is_given_is_the_one_measured(cases, argv, n, k):
    args = cases.arguments(argv.split())
    assert (args.n, args.k) == (n, k)


@pytest.mark.gpu
def test_every_row_of_the_policy_loss_is_read_and_written(cases):
    import torch
    from mccl_b200.ops.loss import fused_policy_loss
    torch.manual_seed(0)
    z, terms = cases.policy_inputs(3000, 257, torch.device("cuda"))
    (g,) = torch.autograd.grad(fused_policy_loss(z.requires_grad_(True), **terms)[0], z)
    assert (g != 0).any(1).all()
