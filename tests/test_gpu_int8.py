"""int8 products (quantize_int8, Int8Matrix, Int8Experts) against 64-bit
restatements: codes and scales bit for bit, products to a few f32 roundings."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def half_step(torch, dt):
    return torch.finfo(dt).eps / 2


def reference_codes(torch, x):
    """scale = fl32(max / 127), code = rne(fl32(x / scale)); a 64-bit quotient
    of two f32 values rounded to f32 is their f32 quotient."""
    x = x.cpu().double()
    s = (x.abs().amax(1) / 127).float()
    q = torch.round((x / torch.where(s > 0, s, 1).double()[:, None]).float()).clamp(-127, 127)
    bad = ~torch.isfinite(x).all(1)
    q[bad | (s == 0)] = 0
    s[bad] = float("nan")
    return q.to(torch.int8), s


def same(torch, a, b):
    return torch.equal(torch.nan_to_num(a, nan=-1.0), torch.nan_to_num(b, nan=-1.0))


@pytest.mark.parametrize("rows,cols", [(1, 1), (2, 3), (3, 16), (9, 64), (5, 127), (2, 512), (17, 513), (3, 1000), (2, 1024),
                                       (33, 1040), (9, 4096), (3, 5120), (1, 7168), (2, 8200), (2, 16384), (2, 16383)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_codes_and_scales(ffn, cuda, rows, cols, dtype):
    import torch
    dt = getattr(torch, dtype)
    g = torch.Generator(device=cuda).manual_seed(rows + cols)
    x = (torch.randn(rows, cols, device=cuda, generator=g) * torch.rand(rows, 1, device=cuda, generator=g) * 8).to(dt)
    q, s = ffn.quantize_int8(x)
    rq, rs = reference_codes(torch, x)
    assert torch.equal(s.cpu(), rs) and torch.equal(q.cpu(), rq)
    assert q.stride(0) % 16 == 0
    # values halfway between codes, and next to it
    if cols > 16:
        k = torch.randint(-127, 127, (rows, cols), device=cuda, generator=g).float()
        x = ((k + 0.5) * 0.0625).to(dt)
        x[:, 0] = 127 * 0.0625
        if dt == torch.float32:
            x[:, 1::3] = torch.nextafter(x[:, 1::3], torch.tensor(9e9, device=cuda))
            x[:, 2::3] = torch.nextafter(x[:, 2::3], torch.tensor(-9e9, device=cuda))
        q, s = ffn.quantize_int8(x)
        rq, rs = reference_codes(torch, x)
        assert torch.equal(s.cpu(), rs) and torch.equal(q.cpu(), rq)


@pytest.mark.parametrize("cols", [33, 640, 2056])
def test_codes_of_extreme_rows(ffn, cuda, cols):
    """Zeros, f32 subnormals, the largest values, and rows with NaN or infinity."""
    import torch
    x = torch.randn(8, cols, device=cuda)
    x[0] = 0
    x[1] *= 1e-41
    x[2] *= 1e-38
    x[3] *= 1e37
    x[3, 5] = 3.4e38
    x[4, cols - 1] = float("nan")
    x[5, 0] = float("inf")
    x[6, 7] = -float("inf")
    q, s = ffn.quantize_int8(x)
    rq, rs = reference_codes(torch, x)
    assert same(torch, s.cpu(), rs) and torch.equal(q.cpu(), rq)
    w = ffn.Int8Matrix.quantize(torch.randn(20, cols, device=cuda))
    y = w.matmul((q, s))
    assert (y[0] == 0).all() and torch.isnan(y[4:7]).all() and torch.isfinite(y[[0, 1, 2, 7]]).all()


def test_codes_of_slices_and_rows_in_use(ffn, cuda):
    import torch
    wide = torch.randn(20, 333, device=cuda).to(torch.bfloat16)
    x = wide[:, 5:5 + 200]
    codes = torch.full((20, 256), 99, dtype=torch.int8, device=cuda)
    scales = torch.full((20,), -2.0, device=cuda)
    for n in (0, 7, 20, 1000):
        codes.fill_(99), scales.fill_(-2.0)
        ffn.quantize_int8(x, codes=codes[:, 3:203], scales=scales, n_rows=torch.tensor([n], dtype=torch.int32, device=cuda))
        rq, rs = reference_codes(torch, x)
        n = min(n, 20)
        assert torch.equal(codes[:n, 3:203].cpu(), rq[:n]) and torch.equal(scales[:n].cpu(), rs[:n])
        assert (codes[n:] == 99).all() and (codes[:, :3] == 99).all() and (codes[:, 203:] == 99).all()
        assert (scales[n:] == -2).all()


@pytest.mark.parametrize("rows,cols", [(1, 16), (9, 100), (40, 512), (3, 2304), (2, 2048)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_swiglu_codes(ffn, cuda, rows, cols, dtype):
    import torch
    dt = getattr(torch, dtype)
    g = torch.Generator(device=cuda).manual_seed(cols)
    x = (torch.randn(rows, 2 * cols, device=cuda, generator=g) * 5).to(dt)
    x[0, 0], x[0, cols] = 40.0, -40.0  # both clamps
    q, s = ffn.quantize_int8(x, ffn.ACT_SWIGLU)
    gate, up = x[:, :cols].double(), x[:, cols:].double()
    v = torch.clamp(gate / (1 + torch.exp(-gate)), max=10) * up.clamp(-10, 10)
    # expf within a step (2 U), a sum, a quotient within two (4 U), a product: 8 U
    assert ((s.double() - v.abs().amax(1) / 127).abs() <= s.double() * 10 * U).all()
    assert ((q.double() * s.double()[:, None] - v).abs() <= s.double()[:, None] * (0.5 + 127 * 20 * U) + 10 * U * v.abs()).all()
    x[0, 1] = float("nan")
    assert torch.isnan(ffn.quantize_int8(x, ffn.ACT_SWIGLU)[1][0])


def product_ok(torch, out, q, s, w, ws, bias):
    """out against acc * s * ws + bias in 64 bits: acc to f32, two products, one
    sum, one rounding to the type."""
    acc = q.double() @ w.double().t()
    ref = acc * s.double()[:, None] * ws.double()
    err = 3 * U * ref.abs() * (1 + 4 * U)
    if bias is not None:
        ref = ref + bias.double()
        err = err + U * (ref.abs() + err)
    u = half_step(torch, out.dtype) if out.dtype != torch.float32 else 0.0
    return ((out.double() - ref).abs() <= err + u * (ref.abs() + err) + (2.0 ** -25 if out.dtype == torch.float16 else 1e-44)).all()


SHAPES = [(1, 1, 1), (1, 128, 128), (2, 16, 5), (1, 4096, 4096), (3, 1000, 129), (16, 64, 130), (17, 200, 129), (33, 1000, 257),
          (64, 4096, 384), (65, 333, 640), (77, 5120, 2304), (128, 640, 1000), (129, 128, 4096), (257, 512, 300),
          (300, 1040, 1000), (600, 256, 4096), (1025, 129, 131), (4, 8192, 128), (16, 16384, 256), (64, 7168, 128), (5, 31, 40000)]


@pytest.mark.parametrize("rows,k,n", SHAPES)
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("with_bias", [False, True])
def test_product(ffn, cuda, rows, k, n, dtype, with_bias):
    import torch
    dt = getattr(torch, dtype)
    g = torch.Generator(device=cuda).manual_seed(rows + k + n)
    x = torch.randn(rows, k, device=cuda, generator=g).to(dt)
    w = torch.randint(-127, 128, (n, k), device=cuda, generator=g, dtype=torch.int8)
    ws = (0.5 + torch.rand(n, device=cuda, generator=g)) * 0.01
    bias = torch.randn(n, device=cuda, generator=g) if with_bias else None
    m = ffn.Int8Matrix(w, ws, bias)
    wide = torch.full((rows, n + 3), 7.0, dtype=dt, device=cuda)
    out = m.matmul(x, out=wide[:, :n])
    q, s = ffn.quantize_int8(x)
    assert product_ok(torch, out, q, s, w, ws, bias)
    assert (wide[:, n:] == 7).all()
    assert torch.equal(m.matmul(x), out) and torch.equal(m.matmul((q, s), dtype=dt), out)


def test_the_largest_sums(ffn, cuda):
    """131072 products of +-127: just inside int32."""
    import torch
    k = 131072
    q = torch.full((3, k), 127, dtype=torch.int8, device=cuda)
    w = torch.full((130, k), 127, dtype=torch.int8, device=cuda)
    w[1] = -127
    w[2, ::2] = -127
    out = ffn.Int8Matrix(w, torch.ones(130, device=cuda)).matmul((q, torch.ones(3, device=cuda)))
    assert (out[:, 0] == 127 * 127 * k).all() and (out[:, 1] == -127 * 127 * k).all() and (out[:, 2] == 0).all()
    assert (out[:, 3:] == 127 * 127 * k).all()


GROUPS = [(1, [5]), (2, [0, 3]), (5, [4, 0, 0, 17, 1]), (5, [0, 0, 0, 0, 0]), (3, [300, 0, 513]), (48, None), (384, None),
          (1000, None), (4096, [1] + [0] * 4094 + [2])]


@pytest.mark.parametrize("groups,counts", GROUPS)
@pytest.mark.parametrize("k,n", [(128, 128), (257, 200), (1000, 129)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_grouped_product(ffn, cuda, groups, counts, k, n, dtype):
    import torch
    dt = getattr(torch, dtype)
    rng = np.random.default_rng(groups + k + n)
    if counts is None:
        counts = rng.poisson(2.0, groups)
    off = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    rows = int(off[-1]) + 9  # rows in no group
    g = torch.Generator(device=cuda).manual_seed(rows)
    q = torch.randint(-127, 128, (rows, (k + 15) // 16 * 16), device=cuda, generator=g, dtype=torch.int8)[:, :k]
    s = torch.rand(rows, device=cuda, generator=g) * 0.01
    w = torch.randint(-127, 128, (groups, n, k), device=cuda, generator=g, dtype=torch.int8)
    ws = torch.rand(groups, n, device=cuda, generator=g)
    bias = torch.randn(groups, n, device=cuda, generator=g)
    m = ffn.Int8Matrix(w, ws, bias)
    out = torch.full((rows, n), 3.0, dtype=dt, device=cuda)
    m.matmul((q, s), out=out, offsets=torch.from_numpy(off).to(cuda))
    for e in np.nonzero(np.diff(off))[0]:
        a, b = int(off[e]), int(off[e + 1])
        assert product_ok(torch, out[a:b], q[a:b], s[a:b], w[e], ws[e], bias[e]), e
    assert (out[off[-1]:] == 3).all()  # as they were


def test_offsets_are_kept_inside_the_rows(ffn, cuda):
    import torch
    w = torch.randint(-127, 128, (3, 64, 64), device=cuda, dtype=torch.int8)
    m = ffn.Int8Matrix(w, torch.ones(3, 64, device=cuda))
    q, s = torch.randint(-127, 128, (12, 64), device=cuda, dtype=torch.int8), torch.ones(12, device=cuda)
    out = torch.full((12, 64), -1.0, device=cuda)
    m.matmul((q, s), out=out, offsets=torch.tensor([-5, 2, 5, 99999], dtype=torch.int32, device=cuda))
    for e, (a, b) in enumerate(((0, 2), (2, 5), (5, 12))):
        assert torch.equal(out[a:b].double(), q[a:b].double() @ w[e].double().t())


def test_layouts_of_weights(ffn, cuda):
    """Padded rows are read in place; others are laid out once."""
    import torch
    x = torch.randn(5, 100, device=cuda)
    wide = torch.randint(-127, 128, (2, 40, 112), device=cuda, dtype=torch.int8)
    sc = torch.rand(2, 40, device=cuda)
    off = torch.tensor([0, 2, 5], dtype=torch.int32, device=cuda)
    a = ffn.Int8Matrix(wide[:, :, :100], sc)
    assert a.w.data_ptr() == wide.data_ptr() and a.ld == 112
    want = a.matmul(x, offsets=off)
    for w in (wide[:, :, :100].contiguous(), wide[:, :, :100].transpose(1, 2).contiguous().transpose(1, 2)):
        assert torch.equal(ffn.Int8Matrix(w, sc).matmul(x, offsets=off), want)
    one = ffn.Int8Matrix(wide[0, :, 3:103], sc[0])  # starts off a 16-byte boundary
    assert product_ok(torch, one.matmul(x), *ffn.quantize_int8(x), wide[0, :, 3:103], sc[0], None)
    row = ffn.Int8Matrix(wide[0, :1, :100], sc[0, :1])
    assert product_ok(torch, row.matmul(x), *ffn.quantize_int8(x), wide[0, :1, :100], sc[0, :1], None)
    floats = torch.randn(2, 40, 100, device=cuda)
    m = ffn.Int8Matrix.quantize(floats)
    rq, rs = reference_codes(torch, floats.view(80, 100))
    assert torch.equal(m.w.cpu().reshape(80, 100), rq) and torch.equal(m.scale.cpu().view(-1), rs)
    assert (m.dequant() - floats).abs().max() <= rs.max() * 0.5001
    with pytest.raises(ffn.FfnError):
        m.matmul(x)  # two groups without offsets
    with pytest.raises(ffn.FfnError):
        m.matmul(x[:, :99], offsets=off)
    with pytest.raises(ffn.FfnError):
        m.matmul(x, offsets=off.long())
    with pytest.raises(ffn.FfnError):
        ffn.Int8Matrix(wide, torch.rand(2, 39, device=cuda))


@pytest.mark.parametrize("tokens", [0, 1, 7, 130])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_experts_are_their_steps(ffn, cuda, tokens, dtype):
    """Int8Experts behind the top-k step: the same bits as its steps one by one,
    each of which is tested above, and near the float experts."""
    import torch
    dt = getattr(torch, dtype)
    E, H, I, K = 24, 192, 80, 4
    g = torch.Generator(device=cuda).manual_seed(tokens)
    w1 = torch.randn(E, 2 * I, H, device=cuda, generator=g) * H ** -0.5
    w2 = torch.randn(E, H, I, device=cuda, generator=g) * I ** -0.5
    gu, dn = ffn.Int8Matrix.quantize(w1), ffn.Int8Matrix.quantize(w2)
    x = torch.randn(tokens, H, device=cuda, generator=g).to(dt)
    logits = torch.randn(max(tokens, 1), E, device=cuda, generator=g)
    idx, wt = ffn.topk(logits, K)
    idx, wt = idx[:tokens].contiguous(), wt[:tokens].contiguous()
    out = ffn.Int8Experts(gu, dn).forward(x, idx, wt, residual=x)
    assert out.shape == x.shape and out.dtype == dt
    if not tokens:
        return
    # two ranks: their sum, up to the rounding of each part
    halves = [ffn.Int8Experts(ffn.Int8Matrix(gu.w[e:e + 12], gu.scale.view(E, -1)[e:e + 12]),
                              ffn.Int8Matrix(dn.w[e:e + 12], dn.scale.view(E, -1)[e:e + 12]), e).forward(x, idx, wt)
              for e in (0, 12)]
    off, pos, src = ffn.moe_sort(idx, 0, E)
    q, s = ffn.quantize_int8(x)
    rows, rs = ffn.moe_permute(q, pos, scales=s)
    h = gu.matmul((rows, rs), offsets=off, dtype=dt)
    y = dn.matmul(ffn.quantize_int8(h, ffn.ACT_SWIGLU), offsets=off, dtype=dt)
    assert torch.equal(out, ffn.moe_combine(y, pos, wt, residual=x))
    tok = torch.div(src.long(), K, rounding_mode="floor")
    assert torch.equal(rows, q[tok]) and torch.equal(rs, s[tok])
    u = half_step(torch, dt)
    part = sum(t.double() for t in halves) + x.double()
    mag = sum(t.double().abs() for t in halves) + x.double().abs()
    assert ((out.double() - part).abs() <= (2 * u + (K + 4) * 4 * U) * mag + 1e-30).all()
    # the float experts: a code is off by a uniform part of a step of 1/127 of its
    # row's largest value, rms step / sqrt(12).  Normal rows (largest about 3.5
    # rms): 0.8 % each for x and both matrices; the gated products have longer
    # tails (largest about 8 rms): 1.8 %.  In quadrature 2.3 %, doubled
    ref = torch.zeros(tokens, H, dtype=torch.float64, device=cuda)
    for t in range(tokens):
        for k in range(K):
            e = int(idx[t, k])
            a = w1[e].double() @ x[t].double()
            v = torch.clamp(a[:I] / (1 + torch.exp(-a[:I])), max=10) * a[I:].clamp(-10, 10)
            ref[t] += float(wt[t, k]) * (w2[e].double() @ v)
    err = (out.double() - x.double() - ref).norm() / ref.norm()
    assert err < 0.05 + (2 * u * x.double().norm() / ref.norm())


def test_streams_graphs_and_a_block_from_norm_to_norm(ffn, cuda):
    """norm -> int8 codes -> router's experts -> gated residual and norm, eager,
    on a stream of its own, and in two captured graphs replayed in turn."""
    import torch
    T, H, I, E, K = 33, 256, 128, 16, 4
    g = torch.Generator(device=cuda).manual_seed(9)
    r = lambda *s: torch.randn(*s, device=cuda, generator=g)  # noqa: E731
    experts = ffn.Int8Experts(ffn.Int8Matrix.quantize(r(E, 2 * I, H) * 0.06), ffn.Int8Matrix.quantize(r(E, H, I) * 0.09))
    before, after = ffn.BlockNorm(pre_w=1 + 0.1 * r(H)), ffn.BlockNorm(pre_w=1 + 0.1 * r(H), post_w=1 + 0.1 * r(H), beta=0.5)
    gate = r(H)
    router = r(E, H) * 0.06
    x = r(T, H).to(torch.bfloat16)

    def run():
        h, xn, q, s = before.forward(None, x, xn=torch.empty_like(x), codes=True)
        idx, wt = ffn.topk((xn.float()[:, None, :] * router).sum(2), K)
        y = experts.forward((q, s), idx, wt, out=torch.empty_like(x))
        return after.forward(y, h, gate=gate)
    want = run()
    assert all(torch.isfinite(t.float()).all() for t in want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):
        c = torch.cuda.CUDAGraph()
        with torch.cuda.graph(c):
            out = run()
        graphs.append((c, out))
    for c, _ in graphs * 3:
        c.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    x.copy_(r(T, H).to(torch.bfloat16))  # new inputs, the same graphs
    want = run()
    for c, _ in graphs:
        c.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_calls_with_and_without_the_module(ffn, cuda, monkeypatch):
    """The CPython module and the ctypes path: the same bits, and refusals of
    the same calls."""
    import torch
    T, H, E, K = 21, 200, 12, 3
    g = torch.Generator(device=cuda).manual_seed(1)
    x = torch.randn(T, H, device=cuda, generator=g).to(torch.float16)
    w = ffn.Int8Matrix(torch.randint(-127, 128, (E, 40, H), device=cuda, generator=g, dtype=torch.int8),
                       torch.rand(E, 40, device=cuda, generator=g) * 0.01, torch.randn(E, 40, device=cuda, generator=g))
    idx = torch.randint(0, E + 3, (T, K), device=cuda, generator=g, dtype=torch.int32)
    wt, gate = torch.rand(T, K, device=cuda, generator=g), torch.rand(T, 1, device=cuda, generator=g)
    p = torch.rand(H, device=cuda, generator=g)
    ffn.quantize_int8(x)
    assert ffn._calls is not None

    def run():
        off, pos, src = ffn.moe_sort(idx, 2, E + 2)
        xs = ffn.moe_permute(x, pos, out=torch.zeros(T * K, H, dtype=x.dtype, device=cuda))
        y = ffn.Int8Matrix(w.w, w.scale, w.bias).matmul(xs, offsets=off)[:int(off[-1])]
        back = ffn.moe_combine(xs, pos, wt, residual=x)
        return [off, pos, src, xs, y, back, *ffn.BlockNorm(p, p, 0.5, 2.0).forward(back, x, gate=gate),
                *ffn.BlockNorm(None, p).forward(x)[:1], *ffn.BlockNorm(p).forward(x, gate=p)]
    refused = [lambda: ffn.moe_sort(idx, 5, 5), lambda: ffn.moe_sort(idx, -1, 5), lambda: ffn.moe_combine(x, idx.long()),
               lambda: ffn.moe_permute(x[:3], idx), lambda: w.matmul(x), lambda: w.matmul(x[:, :100]),
               lambda: ffn.BlockNorm(p[:9]).forward(x, x), lambda: ffn.BlockNorm(p).forward(x, x.float()),
               lambda: ffn.BlockNorm(p, eps=-1.0).forward(x, x), lambda: ffn.moe_combine(x, idx, wt.half())]
    fast = run()
    for call in refused:
        with pytest.raises(ffn.FfnError):
            call()
    monkeypatch.setattr(ffn, "_calls", None)
    assert all(torch.equal(a, b) for a, b in zip(fast, run()))
    for call in refused:
        with pytest.raises(ffn.FfnError):
            call()
