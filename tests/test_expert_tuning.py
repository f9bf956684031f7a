"""The operators together, as a program uses them: an expert layer without capacity (ragged products), a head and the policy loss in
training, the same experts in 8 bits while sampling."""
import pytest
import torch
import torch.nn.functional as F


def _grads(y, leaves, dy):
    return torch.autograd.grad(y, leaves, dy)


@pytest.mark.parametrize("experts,top_k,tokens", [(4, 2, 37), (3, 3, 5), (8, 1, 64), (5, 2, 1), (4, 2, 0)])
def test_dropless_layer_against_every_expert_on_every_token(experts, top_k, tokens):
    """On the CPU in fp64: the sorting, the groups and the weights."""
    from mccl_b200.parallel.layers import DroplessMoE, dropless_moe_reference
    torch.manual_seed(0)
    layer = DroplessMoE(16, 24, experts, top_k, dtype=torch.float64)
    x = torch.randn(tokens, 16, dtype=torch.float64, requires_grad=True)
    dy = torch.randn(tokens, 16, dtype=torch.float64)
    y = layer(x)
    leaves = [x, layer.router.weight, layer.w_in, layer.w_out]
    want = dropless_moe_reference(x, layer.router.weight, layer.w_in, layer.w_out, top_k)
    # the routing's softmax is in fp32 in both: its last bits may differ between the two
    for a, b in zip([y, *_grads(y, leaves, dy)], [want, *_grads(want, leaves, dy)]):
        assert torch.allclose(a, b, atol=1e-5, rtol=1e-5)


def test_dropless_layer_refuses_more_choices_than_experts():
    from mccl_b200.parallel.layers import DroplessMoE
    for k in (0, 5):
        with pytest.raises(ValueError):
            DroplessMoE(16, 16, 4, k)


def _rel(a, b):
    a, b = a.double(), b.double()
    return ((a - b).norm() / b.norm()).item()


U = 2.0 ** -8        # half a step of bf16, relative to the value: no error of one rounding has a larger two-norm than U times the result's


def _model(seed=0, hidden=128, ffn=272, experts=6, vocab=1000):
    from mccl_b200.parallel.layers import DroplessMoE
    torch.manual_seed(seed)
    layer = DroplessMoE(hidden, ffn, experts, 2, device="cuda", dtype=torch.bfloat16)
    embed = torch.nn.Embedding(vocab, hidden, device="cuda", dtype=torch.bfloat16)
    head = torch.nn.Linear(hidden, vocab, bias=False, device="cuda", dtype=torch.bfloat16)
    return layer, embed, head


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 7, 300, 2000, 7000])
def test_dropless_layer_in_bf16(tokens):
    """Against the same layer in fp64 on the same routing.  Roundings between x and y: two products, SiLU, the weights and their product, a
    sum of two: six; the gradients pass as many again.  Independent roundings add up as squares; U for each is a bound."""
    layer, _, _ = _model()
    x = torch.randn(tokens, 128, device="cuda").to(torch.bfloat16).requires_grad_(True)
    dy = torch.randn(tokens, 128, device="cuda").to(torch.bfloat16)
    y = layer(x)
    got = _grads(y, [x, layer.w_in, layer.w_out], dy)
    weight, expert = layer.route(x)
    xr, wi, wo = (t.detach().double().requires_grad_(True) for t in (x, layer.w_in, layer.w_out))
    w = torch.zeros(tokens, 6, device="cuda", dtype=torch.float64).scatter(1, expert, weight.detach().double())
    want = torch.einsum("tef,edf,te->td", F.silu(torch.einsum("td,efd->tef", xr, wi)), wo, w)
    ref = _grads(want, [xr, wi, wo], dy.double())
    assert _rel(y, want) <= 6 * U
    # x's gradient through the experts alone: the router's share is taken off
    through_router = torch.autograd.grad(layer.route(x)[0], x, _weight_grad(x, layer, expert, dy))[0]
    assert _rel(got[0].double() - through_router.double(), ref[0]) <= 14 * U
    assert _rel(got[1], ref[1]) <= 12 * U and _rel(got[2], ref[2]) <= 12 * U


def _weight_grad(x, layer, expert, dy):
    """Gradient of the routing weights: the experts' rows times the gradient of the output."""
    h = F.silu(torch.einsum("td,efd->tef", x.detach().float(), layer.w_in.detach().float()))
    rows = torch.einsum("tef,edf->ted", h, layer.w_out.detach().float()).gather(1, expert[..., None].expand(-1, -1, x.shape[1]))
    return (rows * dy.float()[:, None]).sum(-1).to(x.dtype)


@pytest.mark.gpu
def test_tuning_step_and_sampling_in_8_bits():
    """One step by rewards: the gradients of loss, head and experts against the same step in fp64 on the same routing; then the tuned
    experts sample in 8 bits."""
    from mccl_b200.ops.loss import fused_policy_loss
    layer, embed, head = _model(seed=1)
    T, vocab = 400, 1000
    idx = torch.randint(0, vocab, (T,), device="cuda")
    with torch.no_grad():
        x0 = embed(idx)
        logits0 = head(x0 + layer(x0))
        tokens = torch.multinomial(logits0.float().softmax(-1), 1)[:, 0]
        old = torch.log_softmax(logits0.double(), -1).gather(1, tokens[:, None])[:, 0].float()
    adv, ref = torch.randn(T, device="cuda"), old + 0.1 * torch.randn(T, device="cuda")
    mask = torch.rand(T, device="cuda") < 0.9
    x = embed(idx)
    z = head(x + layer(x))
    loss, logp = fused_policy_loss(z, tokens, old, adv, ref_logp=ref, weights=mask, kl_coef=0.1)
    leaves = [head.weight, layer.w_in, layer.w_out, embed.weight, layer.router.weight]
    grads = torch.autograd.grad(loss, leaves)
    assert all(torch.isfinite(g).all() for g in grads) and torch.isfinite(logp).all()
    # in fp64, the routing weights as the layer rounded them (their own gradient goes to the router: not compared)
    weight, expert = (t.detach() for t in layer.route(x))
    hw, wi, wo = (p.detach().double().requires_grad_(True) for p in leaves[:3])
    xr = x.detach().double()
    w = torch.zeros(T, 6, device="cuda", dtype=torch.float64).scatter(1, expert, weight.double())
    moe = torch.einsum("tef,edf,te->td", F.silu(torch.einsum("td,efd->tef", xr, wi)), wo, w)
    zr = (xr + moe) @ hw.t()
    # The ratio is one up to the roundings of the logits on the way: no row is near an end of the clamp.
    lp = torch.log_softmax(zr, -1).gather(1, tokens[:, None])[:, 0]
    r = (lp - old.double()).exp()
    d = ref.double() - lp
    term = -torch.minimum(r * adv.double(), r.clamp(0.8, 1.2) * adv.double()) + 0.1 * (d.exp() - d - 1)
    want = (term * mask).sum() / mask.sum()
    refs = torch.autograd.grad(want, [hw, wi, wo])
    # A logit of the size of ten is off by ten roundings' 8 U in the worst case; its probability and the ratio by as much, relatively: the
    # gradients' two-norms by no more than that and their own ten roundings.
    for g, f in zip(grads[:3], refs):
        assert _rel(g, f) <= (8 + 10) * U
    with torch.no_grad():
        for p, g in zip(leaves, grads):
            p.add_(g, alpha=-0.5)
        eight = layer.quantized()
        x = embed(idx)
        full, got = layer(x), eight(x)
        # two products, each of operands rounded to four bits (half a step, 2^-4, of which random signs leave a third), and SiLU
        assert _rel(got, full) <= 2 * (2 * 2.0 ** -4)
        assert torch.isfinite(head(x + got)).all()
    assert not eight(x).requires_grad


@pytest.mark.gpu
def test_a_decoding_step_replays_from_a_graph():
    """One token at a time in 8 bits; the graph routes anew on every replay."""
    layer, _, _ = _model(seed=2)
    eight = layer.quantized()
    x = torch.randn(1, 128, device="cuda").to(torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            eight(x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = eight(x)
    for seed in range(4):
        torch.manual_seed(10 + seed)
        x.copy_(torch.randn(1, 128, device="cuda"))
        graph.replay()
        assert torch.equal(out, eight(x))


@pytest.mark.gpu
@pytest.mark.filterwarnings("ignore:The AccumulateGrad node's stream")
def test_calls_at_once_from_several_threads_and_streams():
    """Every operator in four threads, each on a stream of its own, forward and backward: the same bits as alone."""
    import threading
    from mccl_b200.ops import fp8
    from mccl_b200.ops.gemm import grouped_gemm, last_error
    from mccl_b200.ops.loss import fused_policy_loss
    torch.manual_seed(0)

    def bf(*shape, std=1.0):
        return (torch.randn(*shape, device="cuda") * std).to(torch.bfloat16)

    shapes = [(3, 4, 520, 776), (900, 8, 264, 520), (5000, 3, 1024, 2048), (40, 6, 2048, 264)]       # tokens, experts, K, N: every form of the products
    jobs = []
    for t, e, k, n in shapes:
        k8 = k // 16 * 16
        jobs.append(dict(x=bf(t, k).requires_grad_(True), w=bf(e, n, k, std=k ** -0.5).requires_grad_(True), dy=bf(t, n), ends=torch.arange(1, e + 1, device="cuda") * t // e,
                         x8=bf(t, k8), w8=fp8.fp8_quantize(bf(e, n, k8), 128), one=fp8.fp8_quantize(bf(n, k8), 128), z=bf(t, 5003).requires_grad_(True),
                         tokens=torch.randint(0, 5003, (t,), device="cuda"), old=torch.full((t,), -9.0, device="cuda"), adv=torch.randn(t, device="cuda")))

    def run(j):
        y = grouped_gemm(j["x"], j["w"], j["ends"])
        loss, logp = fused_policy_loss(j["z"], j["tokens"], j["old"], j["adv"])
        return [y.detach(), *torch.autograd.grad(y, [j["x"], j["w"]], j["dy"]), fp8.fp8_gemm(j["x8"], j["w8"], j["ends"]), fp8.fp8_gemm(j["x8"], j["one"]),
                loss.detach(), logp, *torch.autograd.grad(loss, j["z"])]

    want = [run(j) for j in jobs]
    torch.cuda.synchronize()
    wrong = []

    def work(me):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for turn in range(40):
                    i = (me + turn) % len(jobs)
                    for at, (a, b) in enumerate(zip(run(jobs[i]), want[i])):
                        if not torch.equal(a, b):
                            wrong.append((me, turn, i, at))
        except Exception as error:                                   # a thread's exception would go unseen
            wrong.append(error)

    threads = [threading.Thread(target=work, args=(me,)) for me in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not wrong, wrong[:5]
    assert last_error() == 0
