"""Row operators in calls at the edge of what they take: more choices a token than
a warp has lanes, rows named twice, and products on several streams at once."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24  # half a step of f32


@pytest.mark.parametrize("top_k", [31, 32, 33, 70])
@pytest.mark.parametrize("dtype,cols", [("float32", 1000), ("bfloat16", 1023), ("bfloat16", 2304)])
def test_more_choices_than_a_warp_has_lanes(ffn, cuda, top_k, dtype, cols):
    import torch
    dt, T, E = getattr(torch, dtype), 37, 96
    g = torch.Generator(device=cuda).manual_seed(top_k + cols)
    idx = torch.stack([torch.randperm(E, device=cuda, generator=g)[:top_k] for _ in range(T)]).to(torch.int32)
    offsets, pos, src = ffn.moe_sort(idx, 8, 80)
    n = int(offsets[-1])
    x = torch.randn(T, cols, device=cuda, generator=g).to(dt)
    rows = ffn.moe_permute(x, pos)
    assert torch.equal(rows[:n], x[(src[:n] // top_k).long()])

    y = torch.randn(T * top_k, cols, device=cuda, generator=g).to(dt)
    w = torch.rand(T, top_k, device=cuda, generator=g)
    p = pos.long()
    terms = torch.where((p >= 0)[..., None], y[p.clamp(min=0)].double(), 0.0) * w[..., None].double()
    ref, mag = terms.sum(1), terms.abs().sum(1)
    out = ffn.moe_combine(y, pos, w)
    # top_k fused multiply-adds in f32, then one rounding to the type
    err, u = (top_k + 2) * U * mag, torch.finfo(dt).eps / 2
    assert ((out.double() - ref).abs() <= err + u * (ref.abs() + err)).all()

    dout = torch.randn(T, cols, device=cuda, generator=g).to(dt)
    dy, dw = ffn.moe_combine_backward(dout, y, pos, w)
    want = torch.zeros(T * top_k, cols, device=cuda, dtype=torch.float64)
    on = p >= 0
    want[p[on]] = (w[..., None].double() * dout[:, None].double())[on]
    # the product rounds to f32 and then to the type
    assert ((dy.double() - want).abs() <= (u + U) * (1 + U) * want.abs()).all()
    dots = torch.where(on[..., None], y[p.clamp(min=0)].double(), 0.0) * dout[:, None].double()
    # a sum of cols fused multiply-adds, in whatever order
    assert ((dw.double() - dots.sum(2)).abs() <= (cols + 2) * U * dots.abs().sum(2)).all()


def test_rows_named_twice(ffn, cuda):
    """combine adds a row as often as it is named; permute leaves one of the
    tokens that name a row."""
    import torch
    y = torch.arange(12, device=cuda, dtype=torch.float32).view(3, 4)
    pos = torch.tensor([[2, 2], [0, -1], [2, 3]], dtype=torch.int32, device=cuda)  # 3: behind y's rows
    out = ffn.moe_combine(y, pos)
    assert torch.equal(out, torch.stack([2 * y[2], y[0], y[2]]))
    x = torch.arange(24, device=cuda, dtype=torch.float32).view(3, 8)
    rows = ffn.moe_permute(x, pos, out=torch.full((3, 8), -1.0, device=cuda))
    assert torch.equal(rows[0], x[1]) and (rows[1] == -1).all()
    assert any(torch.equal(rows[2], x[t]) for t in (0, 2))


def test_the_same_expert_twice_in_a_token(ffn, cuda):
    import torch
    idx = torch.tensor([[5, 5, 1], [1, 5, 5]], dtype=torch.int32, device=cuda)
    offsets, pos, src = ffn.moe_sort(idx, 0, 8)
    assert offsets.tolist() == [0, 0, 2, 2, 2, 2, 6, 6, 6]
    assert pos.tolist() == [[2, 3, 0], [1, 4, 5]] and src.tolist() == [2, 3, 0, 1, 4, 5]


def test_calls_on_several_streams_at_once(ffn, cuda):
    """Products of every kind (one token, K split over a cluster, narrow and wide
    tiles, groups) and norms on four streams together: the bits of calls alone."""
    import torch
    g = torch.Generator(device=cuda).manual_seed(3)

    def r(*s):
        return torch.randn(*s, device=cuda, generator=g)
    wide, long = ffn.Int8Matrix.quantize(r(1024, 2048)), ffn.Int8Matrix.quantize(r(512, 8192))
    groups = ffn.Int8Matrix.quantize(r(8, 512, 1024))
    norm = ffn.BlockNorm(pre_w=1 + 0.1 * r(2048), post_w=1 + 0.1 * r(2048))
    off = torch.tensor(np.arange(9) * 20, dtype=torch.int32, device=cuda)
    xs = [r(1, 2048), r(2048, 2048), r(16, 8192), r(160, 1024), r(700, 2048)]

    def run():
        a, b = norm.forward(xs[4], xs[4])
        grad = norm.backward(xs[4], a, dh=b, dxn=b)
        return [wide.matmul(xs[0]), wide.matmul(xs[1]), long.matmul(xs[2]), groups.matmul(xs[3], offsets=off),
                wide.matmul(xs[4]), a, b, *[grad[k] for k in ("dy", "dres", "dpost_w", "dpre_w")]]
    want = run()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(4)], []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(run())
    torch.cuda.synchronize()
    for outs in got:
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("dtype,bits,low", [("float16", 10, 0), ("float16", 10, -14), ("bfloat16", 7, 0), ("bfloat16", 7, -80),
                                            ("bfloat16", 7, -100)])
def test_codes_of_every_significand(ffn, cuda, dtype, bits, low):
    """A row for every significand of the largest value, holding every value of
    its type below it down to 2^-10 of it, in both signs: codes next to every
    half, and on it.  f16 rows around 2^-14 reach its subnormals."""
    import torch
    dt = getattr(torch, dtype)
    sig = torch.arange(1 << bits, 2 << bits, dtype=torch.float64)
    m = sig * 2.0 ** (low - bits)
    x = (sig[None, :] * 2.0 ** (low - bits)) * 2.0 ** -torch.arange(10, dtype=torch.float64)[:, None]
    x = x.reshape(1, -1).expand(m.numel(), -1).clone()
    x[x > m[:, None]] = 0.0
    x[:, 1::2] *= -1
    for flip in (1.0, -1.0):
        rows = torch.cat([m[:, None], flip * x], 1).to(dt)
        for take in (rows, rows[:, :-(rows.shape[1] % 8)]):  # single elements, and 16 bytes at a time
            take = take.contiguous()
            q, s = ffn.quantize_int8(take.to(cuda))
            # tensor by tensor: IEEE division in f32, ties to even
            scale = take.float().abs().amax(1) / torch.full((len(take),), 127.0)
            want = torch.round(take.float() / scale[:, None])
            assert torch.equal(s.cpu(), scale) and torch.equal(q.cpu().float(), want)
