"""The clipped policy loss against its formulas in 64 bits, and its refusals.

Tolerances.  A row's sum of exponentials is worked out in fp32: two to the power of a product of fp32 numbers (the instruction: 2^-22;
the product: at most 2^-24 x 1.45 |d| e^-|d| <= 2^-24 of the sum), at most 1024 additions one after another in the tests' largest row
(2^-24 each, of the sum so far: 2^-14 in the worst case, but each thread's share of the row is at most 512 values: 2^-15, and roundings
that fall either way: below 2^-18) and twelve merges of partial sums (2^-21 each).  DELTA = 2^-17 bounds the error of a log-probability
before its own rounding.  A row's term changes by slope x DELTA.  A gradient c ([j = a] - p) has a relative error of 2^-17 in p
and c, an absolute one of c 2^-17 where the two cancel, and one rounding to its type (half a step)."""
import pytest
import torch

DELTA = 2.0 ** -17
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
LEAST = {torch.bfloat16: 2.0 ** -125, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -125}     # half a step next to zero; flushed fp32 subnormals


def _loss(*args, **kw):
    from mccl_b200.ops.loss import fused_policy_loss
    return fused_policy_loss(*args, **kw)


def _formula(z, tokens, old, adv, ref, w, clip, kl, mean):
    """loss, logp, d loss / d z, c per row, in 64 bits."""
    z, old, adv, w = z.double(), old.double(), adv.double(), w.double()
    z = z - z.amax(1, keepdim=True)              # logits near the type's lowest value hold no fraction of their logsumexp, in 64 bits neither
    n = torch.logsumexp(z, 1)
    t = tokens.clamp(0, z.shape[1] - 1)
    lp = z.gather(1, t[:, None])[:, 0] - n
    r = (lp - old).exp()
    plain, held = r * adv, r.clamp(1 - clip[0], 1 + clip[1]) * adv
    term, slope = -torch.minimum(plain, held), torch.where(plain > held, 0.0, -plain)
    if kl:
        d = ref.double() - lp
        term, slope = term + kl * (d.exp() - d - 1), slope + kl * (1 - d.exp())
    on = w != 0
    over = w.sum() if mean else torch.ones((), dtype=torch.float64, device=z.device)
    scale = torch.where(over == 0, 0.0, 1 / over)
    loss = torch.where(on, w * term, 0.0).sum() * scale
    c = torch.where(on, w * slope, 0.0) * scale
    g = -c[:, None] * (z - n[:, None]).exp()
    g.scatter_add_(1, t[:, None], c[:, None])
    g = torch.where(on[:, None], g, 0.0)
    return loss, lp, g, c


def _inputs(rows, vocab, dtype, width=None, seed=0):
    """Ratios at chosen places on either side of the clamp's ends (0.8 and 1.28), none within a hundredth of them."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    z = (torch.randn(rows, width or vocab, device="cuda", generator=gen) * 2).to(dtype)
    tokens = torch.randint(0, vocab, (rows,), device="cuda", generator=gen)
    lp = torch.log_softmax(z[:, :vocab].double(), 1).gather(1, tokens[:, None])[:, 0]
    at = torch.tensor([0.5, 0.75, 0.9, 1.0, 1.1, 1.35, 2.0], device="cuda", dtype=torch.float64)
    r = at[torch.randint(0, 7, (rows,), device="cuda", generator=gen)] * (1 + 0.01 * torch.rand(rows, device="cuda", generator=gen))
    old = (lp - r.log()).float()
    ref = (lp + 0.5 * torch.randn(rows, device="cuda", generator=gen)).float()
    adv = torch.randn(rows, device="cuda", generator=gen) + 0.25
    w = (torch.rand(rows, device="cuda", generator=gen) < 0.8).float()
    w[0] = 1.0
    return z, tokens, old, adv, ref, w


CLIP = (0.2, 0.28)


def _check(z, tokens, old, adv, ref, w, kl, mean, loss, logp, grad, vocab, scale=1.0):
    want, lp, g, c = _formula(z[:, :vocab], tokens, old, adv, ref, w, CLIP, kl, mean)
    d = DELTA + 2.0 ** -23 * lp.abs()
    assert ((logp.double() - lp).abs() <= d)[torch.isfinite(lp)].all()
    assert (loss.double() - want).abs() <= (c.abs() * d * 2).sum() + 2.0 ** -23 * want.abs()
    limit = scale * ((HALF_STEP[z.dtype] + 2.0 ** -16) * g.abs() + (c.abs() * 2.0 ** -16)[:, None]) + LEAST[z.dtype]
    assert grad.dtype == z.dtype and grad.shape == z.shape
    assert torch.isfinite(grad).all()
    assert ((grad[:, :vocab].double() - scale * g).abs() <= limit).all()
    assert (grad[:, vocab:] == 0).all() and (grad[w == 0] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,vocab,width", [(1, 1, 1), (1, 2, 8), (3, 7, 7), (5, 64, 64), (2, 2049, 2112), (7, 4097, 4097), (33, 8200, 8200), (2, 50257, 50304),
                                              (1, 131072, 131072), (700, 1000, 1000)])
def test_against_the_formula(rows, vocab, width, dtype):
    z, tokens, old, adv, ref, w = _inputs(rows, vocab, dtype, width)
    for kl, mean in ((0.04, True), (0.0, False)):
        leaf = z.clone().requires_grad_(True)
        loss, logp = _loss(leaf, tokens, old, adv, ref_logp=ref, weights=w, clip=CLIP, kl_coef=kl, vocab=vocab, reduction="mean" if mean else "sum")
        (grad,) = torch.autograd.grad(loss, leaf)
        _check(z, tokens, old, adv, ref, w, kl, mean, loss, logp, grad, vocab)
        assert torch.equal(leaf, z) and not logp.requires_grad


@pytest.mark.gpu
def test_gradient_against_differences():
    """Along a direction d of unit length the central difference over h = 2^-5 is off by h^2 / 6 of the third derivative (each factor of
    the term has derivatives of the order of one: below 8 for r <= 2 and the advantages drawn) and by two of the loss's errors over 2 h."""
    rows, vocab, h = 9, 300, 2.0 ** -5
    z, tokens, old, adv, ref, w = _inputs(rows, vocab, torch.float32, seed=3)
    call = lambda x: _loss(x, tokens, old, adv, ref_logp=ref, weights=w, clip=(0.45, 1.2), kl_coef=0.1, reduction="sum")[0]  # noqa: E731
    leaf = z.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(call(leaf), leaf)
    for k in range(rows):
        d = torch.zeros_like(z)
        d[k] = torch.randn(vocab, device="cuda")
        d[k, tokens[k]] += 3.0
        d /= d.norm()
        # none of the steps crosses an end of the clamp: the ratio moves by a factor of exp(2 h) at most
        r = (torch.log_softmax(z.double(), 1).gather(1, tokens[:, None])[:, 0] - old.double()).exp()[k]
        if min(abs(r / 0.55 - 1), abs(r / 2.2 - 1)) < 0.08:
            continue
        got = (call(z + h * d).double() - call(z - h * d).double()) / (2 * h)
        want = (g.double() * d.double()).sum()
        assert abs(got - want) <= h * h / 6 * 8 * (1 + adv[k].abs()) + 2 * (20 * DELTA) / (2 * h)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_masked_vocabulary_and_extreme_logits(dtype):
    rows, vocab = 6, 1003
    z, tokens, old, adv, ref, w = _inputs(rows, vocab, dtype)
    w[:] = 1
    keep = torch.zeros(rows, vocab, dtype=torch.bool, device="cuda").scatter_(1, tokens[:, None], True)
    z[0] = torch.where(keep[0] | (torch.arange(vocab, device="cuda") < 10), z[0], float("-inf"))
    z[1] = torch.where(keep[1] | (torch.arange(vocab, device="cuda") < 10), z[1], torch.finfo(dtype).min)
    z[2] = torch.finfo(dtype).min                                   # every logit the lowest value: a uniform row
    z[3] = torch.where(keep[3], z[3], float("-inf"))                # the token alone is left: probability one, no gradient
    z[4] += 300.0
    lp = torch.log_softmax(z.double(), 1).gather(1, tokens[:, None])[:, 0]
    old, ref = (lp - 0.05).float(), (lp + 0.3).float()
    leaf = z.clone().requires_grad_(True)
    loss, logp = _loss(leaf, tokens, old, adv, ref_logp=ref, weights=w, clip=CLIP, kl_coef=0.04)
    (grad,) = torch.autograd.grad(loss, leaf)
    _check(z, tokens, old, adv, ref, w, 0.04, True, loss, logp, grad, vocab)


@pytest.mark.gpu
def test_rows_of_no_weight_take_no_part_whatever_they_hold():
    rows, vocab = 8, 513
    z, tokens, old, adv, ref, w = _inputs(rows, vocab, torch.bfloat16)
    w[:] = 1
    w[[1, 4, 7]] = 0
    z[1], z[4] = float("nan"), float("inf")
    tokens[7], tokens[1] = -100, vocab
    old[4], adv[7], ref[1] = float("nan"), float("inf"), float("-inf")
    on = w != 0
    for weights in (w, on):
        leaf = z.clone().requires_grad_(True)
        loss, logp = _loss(leaf, tokens, old, adv, ref_logp=ref, weights=weights, clip=CLIP, kl_coef=0.04)
        (grad,) = torch.autograd.grad(loss, leaf)
        assert (grad[~on] == 0).all()
        _check(z[on], tokens[on], old[on], adv[on], ref[on], w[on], 0.04, True, loss, logp[on], grad[on], vocab)


@pytest.mark.gpu
def test_token_outside_the_vocabulary_makes_the_loss_nan():
    z, tokens, old, adv, ref, w = _inputs(4, 100, torch.bfloat16, 128)
    w[:] = 1
    tokens[2] = 100                                                 # a padding column
    leaf = z.clone().requires_grad_(True)
    loss, logp = _loss(leaf, tokens, old, adv, weights=w, vocab=100)
    (grad,) = torch.autograd.grad(loss, leaf)
    assert loss.isnan() and logp[2].isnan() and torch.isfinite(logp[[0, 1, 3]]).all()
    assert grad[2, :100].isnan().all() and torch.isfinite(grad[[0, 1, 3]]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [0, 5])
def test_nothing_to_average(rows):
    z, tokens, old, adv, ref, w = _inputs(max(rows, 1), 50, torch.bfloat16)
    z, tokens, old, adv, w = z[:rows], tokens[:rows], old[:rows], adv[:rows], torch.zeros(rows, device="cuda")
    leaf = z.clone().requires_grad_(True)
    loss, logp = _loss(leaf, tokens, old, adv, weights=w)
    (grad,) = torch.autograd.grad(loss, leaf)
    assert loss.item() == 0 and logp.shape == (rows,) and (grad == 0).all() and grad.shape == z.shape


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_views_of_logits(dtype):
    """Rows further apart than they are wide, at any offset, and a transposed matrix."""
    rows, vocab = 5, 4100
    z, tokens, old, adv, ref, w = _inputs(rows, vocab, dtype)
    for off, extra in ((0, 3), (1, 8), (3, 13)):
        wide = torch.full((rows, vocab + off + extra), float("nan"), device="cuda", dtype=dtype)
        wide[:, off:off + vocab] = z
        wide.requires_grad_(True)
        loss, logp = _loss(wide[:, off:off + vocab], tokens, old, adv, ref_logp=ref, weights=w, clip=CLIP, kl_coef=0.04)
        (grad,) = torch.autograd.grad(loss, wide)
        _check(z, tokens, old, adv, ref, w, 0.04, True, loss, logp, grad[:, off:off + vocab], vocab)
    t = z.t().contiguous().requires_grad_(True)
    loss, logp = _loss(t.t(), tokens, old, adv, ref_logp=ref, weights=w, clip=CLIP, kl_coef=0.04)
    (grad,) = torch.autograd.grad(loss, t)
    _check(z, tokens, old, adv, ref, w, 0.04, True, loss, logp, grad.t(), vocab)


@pytest.mark.gpu
def test_retained_graph_scaled_loss_and_second_derivative():
    z, tokens, old, adv, ref, w = _inputs(12, 777, torch.float32)
    leaf = z.clone().requires_grad_(True)
    loss, logp = _loss(leaf, tokens, old, adv, ref_logp=ref, weights=w, clip=CLIP, kl_coef=0.04)
    (a,) = torch.autograd.grad(loss, leaf, retain_graph=True)
    (b,) = torch.autograd.grad(loss * -3.0, leaf, retain_graph=True)
    _check(z, tokens, old, adv, ref, w, 0.04, True, loss, logp, a, 777)
    assert ((b.double() + 3 * a.double()).abs() <= 3 * (2.0 ** -22 * a.double().abs() + 2.0 ** -22 * a.double().abs().max())).all()
    (c,) = torch.autograd.grad(loss, leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(c.sum(), leaf)


@pytest.mark.gpu
def test_same_bits_again_on_another_stream_and_from_a_graph():
    rows, vocab = 40, 5000
    z, tokens, old, adv, ref, w = _inputs(rows, vocab, torch.bfloat16)

    def once(leaf):
        loss, logp = _loss(leaf, tokens, old, adv, ref_logp=ref, weights=w, clip=CLIP, kl_coef=0.04)
        return [loss.detach(), logp, torch.autograd.grad(loss, leaf)[0]]
    first = once(z.clone().requires_grad_(True))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once(z.clone().requires_grad_(True))
        held = z.clone().requires_grad_(True)
        for _ in range(3):
            once(held)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = once(held)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(first, out))
    with torch.no_grad():
        held.copy_(z.flip(1))
    graph.replay()
    want = once(z.flip(1).contiguous().requires_grad_(True))
    assert all(torch.equal(a, b) for a, b in zip(want, out))


def test_refusals():
    z, row = torch.zeros(4, 16), torch.zeros(4)
    tokens = torch.zeros(4, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA"):
        _loss(z, tokens, row, row)
    for bad in (dict(reduction="none"), dict(clip=(-0.1, 0.2)), dict(clip=(0.2, float("nan"))), dict(vocab=0), dict(vocab=17), dict(kl_coef=0.1),
                dict(weights=torch.zeros(3)), dict(weights=torch.zeros(4, dtype=torch.int64)), dict(ref_logp=torch.zeros(4, dtype=torch.float64)),
                dict(ref_logp=torch.zeros(4, 1))):
        with pytest.raises(ValueError):
            _loss(z, tokens, row, row, **bad)
    for args in ((z.double(), tokens, row, row), (z[0], tokens, row, row), (z[:, :0], tokens, row, row), (z, tokens.int(), row, row),
                 (z, tokens[:3], row, row), (z, tokens, row.half(), row), (z, tokens, row, row[:2]),
                 (z, tokens, row.clone().requires_grad_(True), row)):
        with pytest.raises(ValueError):
            _loss(*args)


@pytest.mark.gpu
def test_more_logits_than_32_bits_count():
    rows, vocab = 43000, 50257
    z = torch.empty(rows, vocab, device="cuda", dtype=torch.bfloat16).normal_().requires_grad_(True)
    tokens, adv = torch.randint(0, vocab, (rows,), device="cuda"), torch.randn(rows, device="cuda")
    old, w = torch.full((rows,), -40.0, device="cuda"), torch.ones(rows, device="cuda")          # ratios far above the clamp's end
    loss, logp = _loss(z, tokens, old, adv, clip=CLIP, reduction="sum")
    (grad,) = torch.autograd.grad(loss, z)
    at = torch.cat([torch.arange(40), torch.arange(rows - 40, rows)]).cuda()
    _, lp, g, c = _formula(z.detach()[at], tokens[at], old[at], adv[at], None, w[at], CLIP, 0.0, False)
    d = DELTA + 2.0 ** -23 * lp.abs()
    assert ((logp[at].double() - lp).abs() <= d).all()
    # c = -r A: its relative error is that of lp, rounded to fp32 twice, beside that of p
    limit = (HALF_STEP[z.dtype] + 2.0 ** -15 + d[:, None]) * g.abs() + (c.abs() * (2.0 ** -16 + d))[:, None] + LEAST[z.dtype]
    assert ((grad[at].double() - g).abs() <= limit).all() and (c != 0).any() and (c == 0).any()
