"""8-bit weights of more rows than 65535 blocks of 128."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _plain(x):
    """Values and exponents by blocks of 128 rows, of one block of columns, in 64 bits (as in tests/test_fp8.py)."""
    n, k = x.shape
    b = torch.nn.functional.pad(x.double(), (0, 0, 0, -n % 128)).view(-1, 128, k)
    mantissa, e = torch.frexp(b.abs().amax((1, 2)) / 448)
    e = torch.where(mantissa == 0.5, e - 1, e)
    v = torch.ldexp(b, -e[:, None, None])
    step = torch.ldexp(torch.ones_like(v), torch.frexp(v.abs().clamp(min=2.0 ** -6))[1] - 4)
    return (torch.round(v / step) * step).view(-1, k)[:n], e


@pytest.mark.parametrize("E,N", [(1, 65535 * 128), (1, 65535 * 128 + 8), (2, 65536 * 128 + 136)])
def test_weights_of_many_rows(E, N):
    from mccl_b200.ops import fp8
    torch.manual_seed(0)
    w = (torch.randn(E, N, 16, device="cuda") * torch.exp2(torch.arange(N, device="cuda") % 1999 // 100)[:, None]).to(torch.bfloat16)
    got = fp8.fp8_quantize(w if E > 1 else w[0], rows=128)
    data, scale = got.data.view(E, N, 16), got.scale.view(torch.uint8).view(E, -1)
    for e in range(E):
        for lo in range(0, N, 1 << 20):                      # a multiple of 128
            q, exponent = _plain(w[e, lo:lo + (1 << 20)])
            assert (data[e, lo:lo + (1 << 20)].float() == q).all(), (e, lo)
            assert (scale[e, lo // 128:lo // 128 + len(exponent)].int() - 127 == exponent).all(), (e, lo)
    x = torch.randn(3, 16, device="cuda").to(torch.bfloat16)
    y = fp8.fp8_gemm(x, got, torch.tensor([1, 3], device="cuda") if E > 1 else None)
    rows = fp8.fp8_quantize(x).dequantize().double()
    # fp32 sums of 16 exact products, a step each, and a rounding to bf16
    for t in range(3):
        at = got.dequantize().view(E, N, 16)[0 if E == 1 or t < 1 else 1].double()
        want, most = at @ rows[t], at.abs() @ rows[t].abs()
        assert ((y[t].double() - want).abs() <= 2.0 ** -8 * want.abs() + 32 * 2.0 ** -24 * most).all()
