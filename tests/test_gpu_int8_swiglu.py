"""quantize_int8 of SwiGLU rows whose gates all lie far below zero."""
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
D = 2.0 ** -149  # f32's subnormal step


@pytest.mark.parametrize("low,high", [(-70, -60), (-88.6, -87.5), (-88.0, -88.0), (-97, -89), (-110, -95)])
@pytest.mark.parametrize("cols", [40, 513, 3000])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_rows_of_far_gates(ffn, cuda, low, high, cols, dtype):
    """silu(g) = g / (1 + exp(-g)) is about g exp(g) here, down to 1e-45: through
    the range in which exp(-g) comes near f32's end and passes it."""
    import torch
    dt = getattr(torch, dtype)
    g = torch.Generator(device=cuda).manual_seed(cols)
    x = torch.empty(6, 2 * cols, device=cuda)
    x[:, :cols] = low + (high - low) * torch.rand(6, cols, device=cuda, generator=g)
    x[:, cols:] = torch.randn(6, cols, device=cuda, generator=g) * 6
    x[5, 7] = 0.5  # one ordinary gate: the others' codes are 0
    x = x.to(dt)
    q, s = ffn.quantize_int8(x, ffn.ACT_SWIGLU)
    gate, up = x[:, :cols].double(), x[:, cols:].double().clamp(-10, 10)
    v = gate / (1 + torch.exp(-gate)) * up
    # expf within a step, of its value or of the subnormals; two products, each
    # rounded to half a step of either kind; elsewhere a sum and a quotient within
    # two steps
    err = 10 * U * v.abs() + ((1.0 * gate.abs() + 0.5) * up.abs() + 0.5) * D
    m = v.abs().amax(1)
    se = (err / 127).amax(1) + U * m / 127 + D / 2  # the scale, rounded
    assert ((s.double() - m / 127).abs() <= se).all()
    # a code stands for its value within half a scale, and the value may pass
    # 127 scales by what the scale was rounded
    sd = s.double()[:, None]
    assert ((q.double() * sd - v).abs() <= sd * (0.5 + 128 * 4 * U) + err + 127 * se[:, None]).all()
