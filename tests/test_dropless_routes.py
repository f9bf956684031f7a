"""The expert layer without capacity where the ragged products' kernels stand aside: under torch.func, traces and dispatch modes, autocast and
with more experts than they take."""
import pytest
import torch
import torch.nn.functional as F
from torch.utils.flop_counter import FlopCounterMode

U = 2.0 ** -8        # half a step of bf16, relative to the value


def _layer(device="cpu", dtype=torch.float64, hidden=16, ffn=24, experts=5, top_k=2, seed=0):
    from mccl_b200.parallel.layers import DroplessMoE
    torch.manual_seed(seed)
    return DroplessMoE(hidden, ffn, experts, top_k, device=device, dtype=dtype)


def _rel(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm()).item()


def _plain(layer, x):
    from mccl_b200.parallel.layers import dropless_moe_reference
    return dropless_moe_reference(x, layer.router.weight, layer.w_in, layer.w_out, layer.top_k)


# ---- the plain route itself, in 64 bits (the routing's softmax is in 32: its last bits may differ) ------------------------
def test_a_trace_routes_other_tokens_anew():
    layer = _layer().requires_grad_(False)
    traced = torch.jit.trace(layer, (torch.randn(20, 16, dtype=torch.float64),), check_trace=False)
    for tokens in (20, 1, 33, 20):
        x = torch.randn(tokens, 16, dtype=torch.float64)
        assert torch.allclose(traced(x), _plain(layer, x), atol=1e-5, rtol=1e-5)


def test_gradients_by_torch_func():
    layer = _layer()
    x, dy = torch.randn(20, 16, dtype=torch.float64), torch.randn(20, 16, dtype=torch.float64)
    params = {n: p.detach() for n, p in layer.named_parameters()}
    got = torch.func.grad(lambda ps: (torch.func.functional_call(layer, ps, (x,)) * dy).sum())(params)
    want = torch.autograd.grad(_plain(layer, x), list(layer.parameters()), dy)
    for (n, _), g in zip(layer.named_parameters(), want):
        assert torch.allclose(got[n], g, atol=1e-5, rtol=1e-5), n
    v = torch.randn_like(x)
    _, along = torch.func.jvp(lambda t: layer(t), (x,), (v,))
    xr = x.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(_plain(layer, xr), xr, dy)
    assert abs((along * dy).sum() - (g * v).sum()) <= 1e-4


# ---- bf16 on CUDA --------------------------------------------------------------------------------------------------------
# Either route is off the exact result by six roundings in y and fourteen in a gradient (tests/test_expert_tuning.py), in the two-norm: the two
# are apart by no more than both.
Y, G = 2 * 6 * U, 2 * 14 * U


def _gpu(tokens=300, **kw):
    layer = _layer("cuda", torch.bfloat16, 128, 272, 6, **kw)
    x = torch.randn(tokens, 128, device="cuda").to(torch.bfloat16)
    return layer, x, torch.randn(tokens, 128, device="cuda").to(torch.bfloat16)


def _launches():
    from mccl_b200.ops import gemm
    return gemm.launches()


@pytest.mark.gpu
def test_trace_on_cuda():
    layer, x, _ = _gpu()
    layer.requires_grad_(False)
    traced = torch.jit.trace(layer, (x,), check_trace=False)
    for tokens in (300, 1, 77):
        x = torch.randn(tokens, 128, device="cuda").to(torch.bfloat16)
        before = _launches()
        want = layer(x)
        assert _launches() == before + 2                      # outside a trace: the kernels
        assert _rel(traced(x), want) <= Y
        assert _launches() == before + 2


@pytest.mark.gpu
def test_torch_func_on_cuda():
    layer, x, dy = _gpu()
    params = {n: p.detach() for n, p in layer.named_parameters()}
    got = torch.func.grad(lambda ps: (torch.func.functional_call(layer, ps, (x,)) * dy).float().sum())(params)
    want = torch.autograd.grad(layer(x), list(layer.parameters()), dy)
    for (n, _), g in zip(layer.named_parameters(), want):
        assert _rel(got[n], g) <= G, n
    v = torch.randn_like(x)
    y, along = torch.func.jvp(lambda t: layer(t), (x,), (v,))
    assert _rel(y, layer(x)) <= Y
    xr = x.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(layer(xr), xr, dy)
    along, dy, g, v = (t.double() for t in (along, dy, g, v))
    # both are <dy, J v>; one side's error is in J v, the other's in dy J
    assert abs((along * dy).sum() - (g * v).sum()) <= 14 * U * (along.norm() * dy.norm() + g.norm() * v.norm())


@pytest.mark.gpu
def test_dispatch_modes_on_cuda():
    from torch.utils.checkpoint import CheckpointPolicy, checkpoint, create_selective_checkpoint_contexts
    layer, x, dy = _gpu()
    xr = x.clone().requires_grad_(True)
    leaves = [xr, layer.w_in, layer.w_out]
    want = layer(xr)
    grads = torch.autograd.grad(want, leaves, dy)
    with FlopCounterMode(display=False) as counter:
        y = layer(xr)
    # the experts' two products, and the router's, two operations for each multiplication
    assert counter.get_total_flops() == 2 * 2 * (300 * 2) * 128 * 272 + 2 * 300 * 128 * 6
    assert _rel(y, want) <= Y

    def policy(ctx, op, *args, **kwargs):
        return CheckpointPolicy.MUST_SAVE if op == torch.ops.aten.mm.default else CheckpointPolicy.PREFER_RECOMPUTE
    y = checkpoint(layer, xr, use_reentrant=False, context_fn=lambda: create_selective_checkpoint_contexts(policy))
    assert _rel(y, want) <= Y
    for a, b in zip(torch.autograd.grad(y, leaves, dy), grads):
        assert _rel(a, b) <= G


@pytest.mark.gpu
def test_autocast_with_parameters_in_32_bits():
    layer, x, _ = _gpu()
    full = _layer("cuda", torch.float32, 128, 272, 6)
    full.load_state_dict(layer.state_dict())
    want = layer(x)
    with torch.autocast("cuda", torch.bfloat16):
        got = full(x.float())
        same = layer(x)
    assert _rel(got, want) <= Y and _rel(same, want) <= Y


@pytest.mark.gpu
@pytest.mark.parametrize("experts,kernels", [(1024, 2), (1025, 0), (1500, 0)])
def test_more_experts_than_the_kernels_take(experts, kernels):
    layer = _layer("cuda", torch.bfloat16, 16, 24, experts, 3)
    x = torch.randn(40, 16, device="cuda").to(torch.bfloat16).requires_grad_(True)
    dy = torch.randn(40, 16, device="cuda").to(torch.bfloat16)
    before = _launches()
    y = layer(x)
    assert _launches() == before + kernels
    got = torch.autograd.grad(y, [x, layer.w_in, layer.w_out], dy)
    weight, expert = (t.detach() for t in layer.route(x))
    xr, wi, wo = (t.detach().double().requires_grad_(True) for t in (x, layer.w_in, layer.w_out))
    w = torch.zeros(40, experts, device="cuda", dtype=torch.float64).scatter(1, expert, weight.double())
    want = torch.einsum("tef,edf,te->td", F.silu(torch.einsum("td,efd->tef", xr, wi)), wo, w)
    ref = torch.autograd.grad(want, [xr, wi, wo], dy.double())
    assert _rel(y, want) <= 6 * U
    assert _rel(got[1], ref[1]) <= 12 * U and _rel(got[2], ref[2]) <= 12 * U


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 9, 300, 3000])
def test_quantised_layer_against_64_bits_on_its_own_operands(tokens):
    """The operands are the quantised ones, so what is left are the second product's fp32 sums (a step for each addition, as in tests/test_fp8.py) and
    three roundings to bf16: that product's, its product's with the weight, the sum's.  Their products with one another are below a hundredth."""
    from mccl_b200.ops import fp8
    layer, x, _ = _gpu(tokens)
    eight = layer.quantized()
    weight, expert = layer.route(x)
    by_expert, order = expert.reshape(-1).sort(stable=True)
    sizes = torch.bincount(by_expert, minlength=6)
    h = F.silu(fp8.fp8_gemm(x.repeat_interleave(2, 0)[order], eight.w_in, sizes.cumsum(0)))     # the same rows in the same kernel: the same bits
    h, w = fp8.fp8_quantize(h).dequantize().double(), eight.w_out.dequantize().double()

    def by_token(h, w):
        rows = torch.empty(2 * tokens, 128, device="cuda", dtype=torch.float64)
        rows[order] = torch.cat([a @ w[e].t() for e, a in enumerate(h.split(sizes.tolist()))])
        return rows.view(tokens, 2, 128) * weight.double()[..., None]
    parts, most = by_token(h, w), by_token(h.abs(), w.abs()).sum(1)
    want = parts.sum(1)
    limit = 1.01 * (U * (2 * parts.abs().sum(1) + want.abs()) + 2 * 272 * 2.0 ** -24 * most)
    assert ((eight(x).double() - want).abs() <= limit).all()
