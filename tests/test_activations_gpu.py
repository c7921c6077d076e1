"""lily_linear's activations by themselves, against the functions in 64 bits: products of zeroes, the bias is the value.

What may differ. The value itself is rounded a few times on its way into exp, tanh's exponent or the normal
integral's, 2^-22 of it, so that the function moves by its slope. F32 outs: the functions and quotients add 2^-20 of
the result (GELU: a fit 2^-23.9 off, its evaluation 2^-21, a reciprocal and an exponential of 2^-22 each). BF16 outs: GELU's
fit is 2^-20.1 off, relative to the result, and the rest the same: below 2^-18; then half a step, 2^-8. Below 2^-120 a
quotient's denominator passes 2^126 and the result becomes 0."""
import pytest

pytestmark = pytest.mark.gpu

ACTS = ["none", "relu", "silu", "gelu", "gelu_tanh"]


def _function(torch, v, act):
    if act == "relu":
        return v.clamp_min(0)
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "gelu":
        return 0.5 * v * torch.erfc(-v * 0.5 ** 0.5)
    if act == "gelu_tanh":
        return v * torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (v + 0.044715 * v ** 3))
    return v.clone()


def _call(torch, lily, values, tokens, act, out_type, pad):
    n = values.shape[0]
    scratch = lily.SamplerScratch(64, max_rows=1, max_history=0)
    a, w = (torch.zeros((r, 64), dtype=torch.bfloat16, device="cuda") for r in (tokens, n))
    out = torch.full((tokens, n + pad), 9.0, dtype=out_type, device="cuda")
    scratch.linear(a, w, out[:, :n], bias=values, activation=act)
    assert scratch.status() == lily.OK and (out[:, n:] == 9.0).all()
    return out[:, :n]


# By single blocks, alone and among shares, by pairs; outs through shared memory and straight from the registers.
@pytest.mark.parametrize("tokens", [1, 20, 40, 100, 600])
@pytest.mark.parametrize("act", ACTS)
def test_activations_to_their_last_digits(cuda, lily, tokens, act):
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(tokens)
    values = torch.cat([torch.linspace(-14, 14, 3000, device="cuda"), torch.linspace(-8, -3, 1000, device="cuda"),
                        torch.randn(64, generator=g, device="cuda"), torch.randn(24, generator=g, device="cuda") * 1e-3,
                        torch.tensor([0.0, -0.0, 2.0 ** -60, -2.0 ** -60, 40.0, -40.0, 80.0, 1e30], device="cuda")])
    v = values.double().requires_grad_()
    y = _function(torch, v, act)
    slope, = torch.autograd.grad(y.sum(), v)
    y, v = y.detach(), v.detach()
    for out_type, half in ((torch.float32, 2.0 ** -24), (torch.bfloat16, 2.0 ** -8)):
        tol = (2.0 ** -18 if act == "gelu" and out_type == torch.bfloat16 else 2.0 ** -20) * y.abs() + 2.0 ** -22 * (slope * v).abs() + 2.0 ** -120
        tol = (tol + half * (y.abs() + tol)) if act not in ("none", "relu") else half * y.abs()
        for pad in (0, 3):
            out = _call(torch, lily, values, tokens, act, out_type, pad)
            off = (out.double() - y).abs()
            bad = off > tol
            assert not bad.any(), (out_type, values[bad.any(0)][:8].tolist(), out[0, bad.any(0)][:8].tolist(), y[bad.any(0)][:8].tolist())


@pytest.mark.parametrize("tokens", [3, 40, 300])
@pytest.mark.parametrize("act", ACTS)
def test_infinities_and_nan(cuda, lily, tokens, act):
    """As the header's formulas make of them; neighbours stay."""
    torch = cuda
    inf, nan = float("inf"), float("nan")
    values = torch.randn(264, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    clean = values.clone()
    values[5], values[9], values[130], values[263] = inf, -inf, nan, inf
    want = {inf: inf, -inf: {"none": -inf, "relu": 0.0}.get(act, nan)}
    for out_type in (torch.float32, torch.bfloat16):
        out = _call(torch, lily, values, tokens, act, out_type, 0).float()
        assert (out[:, 5] == want[inf]).all() and (out[:, 263] == want[inf]).all() and torch.isnan(out[:, 130]).all()
        assert torch.isnan(out[:, 9]).all() if want[-inf] != want[-inf] else (out[:, 9] == want[-inf]).all()
        same = _call(torch, lily, clean, tokens, act, out_type, 0).float()
        keep = torch.isfinite(values)
        assert torch.equal(out[:, keep], same[:, keep])
