"""The norms after and before a block with gate and scaled residual (BlockNorm)
and their gradient, against 64-bit restatements.

Tolerances count f32 roundings: a row sum is a tree of at most 48 additions
(32 values in a thread, 5 + 5 shuffles, and the products), so mean(v^2) is off
by at most 50 U relative and its root by 25 U; rsqrtf is within 2 steps (4 U)
and the sum with eps adds U.  Every further product or sum adds U of its terms.  The last rounding adds half a step of
the type."""
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
EPS = 1e-6
RS = 30 * U  # relative error of 1 / sqrt(mean(v^2) + eps)

ROWS_COLS = [(1, 1), (3, 7), (1, 64), (9, 65), (5, 512), (17, 513), (2, 1000), (300, 1024), (4, 1031), (33, 4096),
             (650, 5120), (1, 7168), (3, 8191), (2, 16384), (2, 16383), (2400, 96)]


def half_step(torch, dt):
    return torch.finfo(dt).eps / 2


def tiny(torch, dt):
    return 2.0 ** -25 if dt == torch.float16 else 2.0 ** -134 if dt == torch.bfloat16 else 2.0 ** -150


def inputs(torch, cuda, rows, cols, dt, gate, seed=0):
    g = torch.Generator(device=cuda).manual_seed(rows * 131 + cols + seed)
    r = lambda *s: torch.randn(*s, device=cuda, generator=g)  # noqa: E731
    y, res = (0.3 * r(rows, cols)).to(dt), r(rows, cols).to(dt)
    gt = None if gate == "none" else r(cols) if gate == "channel" else torch.sigmoid(r(rows, 1))
    return y, res, gt, 1 + 0.2 * r(cols), 1 + 0.2 * r(cols)


def rho(v):
    return 1 / ((v * v).mean(1, keepdim=True) + EPS).sqrt()


@pytest.mark.parametrize("rows,cols", ROWS_COLS)
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("gate", ["none", "channel", "token"])
@pytest.mark.parametrize("post,pre", [(True, True), (False, True), (True, False)])
def test_forward(ffn, cuda, rows, cols, dtype, gate, post, pre):
    import torch
    dt = getattr(torch, dtype)
    y, res, gt, wp, wq = inputs(torch, cuda, rows, cols, dt, gate)
    bn = ffn.BlockNorm(pre_w=wq if pre else None, post_w=wp if post else None, alpha=0.75, beta=-0.5, eps=EPS)
    h, xn = bn.forward(y, res, gate=gt)
    yd, rd, g64 = y.double(), res.double(), 1.0 if gt is None else gt.double()
    b = -0.5 * g64 * (yd * rho(yd) * wp.double() if post else yd)
    want = 0.75 * rd + b
    err = (RS + 5 * U) * b.abs() + 2 * U * (0.75 * rd.abs() + b.abs())
    u = half_step(torch, dt)
    assert h.dtype == dt
    assert ((h.double() - want).abs() <= err + u * (want.abs() + err) + tiny(torch, dt)).all()
    if not pre:
        assert xn is None
        return
    r = rho(want)
    ref = want * r * wq.double()
    # the stream's own error, and that of its norm: |d rho| / rho <= rms(err) / rms(h)
    rel = RS + 3 * U + err.square().mean(1, keepdim=True).sqrt() * r
    e2 = err * r * wq.double().abs() + ref.abs() * rel
    assert ((xn.double() - ref).abs() <= e2 + u * (ref.abs() + e2) + tiny(torch, dt)).all()


def test_forward_without_residual_without_block_and_in_place(ffn, cuda):
    import torch
    y, res, gt, wp, wq = inputs(torch, cuda, 37, 640, torch.bfloat16, "channel")
    bn = ffn.BlockNorm(pre_w=wq, post_w=wp, alpha=2.0, beta=0.5, eps=EPS)
    zero = torch.zeros_like(y)
    h0, x0 = bn.forward(y, zero, gate=gt)
    h1, x1 = bn.forward(y, None, gate=gt)
    assert torch.equal(h0, h1) and torch.equal(x0, x1)
    h, xn = bn.forward(None, res)  # the norm before the first block
    assert torch.equal(h, 2 * res)
    want = 2 * res.double() * rho(2 * res.double()) * wq.double()
    assert ((xn.double() - want).abs() <= want.abs() * (RS + 4 * U + 2.0 ** -8)).all()
    hw, xw = bn.forward(y, res, gate=gt)
    stream = res.clone()
    h, xn = bn.forward(y, stream, gate=gt, h=stream)
    assert h is stream and torch.equal(stream, hw) and torch.equal(xn, xw)


@pytest.mark.parametrize("rows,cols", [(1, 16), (5, 100), (3, 513), (70, 4096), (2, 7168), (9, 1032)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_codes_are_those_of_the_f32_norm(ffn, cuda, rows, cols, dtype):
    """With f32 rows the codes are quantize_int8's of xn, bit for bit; with
    bf16 rows they stand for the norm before its rounding to bf16."""
    import torch
    dt = getattr(torch, dtype)
    y, res, gt, wp, wq = inputs(torch, cuda, rows, cols, dt, "token", 5)
    y[0], res[0] = 0, 0  # a row of zeros: scale 0
    bn = ffn.BlockNorm(pre_w=wq, post_w=wp, eps=EPS)
    xn = torch.empty_like(y)
    h, got, q, s = bn.forward(y, res, gate=gt, xn=xn, codes=True)
    h2, xn2 = bn.forward(y, res, gate=gt)
    assert got is xn and torch.equal(xn, xn2) and torch.equal(h, h2)
    assert s[0] == 0 and (q[0] == 0).all()
    if dt == torch.float32:
        q2, s2 = ffn.quantize_int8(xn)
        assert torch.equal(q, q2) and torch.equal(s, s2)
    else:  # half a code, and half a bf16 step of xn
        d = (q.double() * s.double()[:, None] - xn.double()).abs()
        assert (d <= s.double()[:, None] * 0.5 * (1 + 1e-5) + 2.0 ** -8 * xn.double().abs() + 1e-30).all()
    none = bn.forward(y, res, gate=gt, codes=True)
    assert none[1] is None and torch.equal(none[2], q) and torch.equal(none[3], s)


def reference_backward(torch, y, h, dh, dxn, gt, wp, wq, alpha, beta, gate, post):
    """The gradients in 64 bits, and for each the same sums of absolute terms."""
    y, h, dh, dxn, wq = (t.double() for t in (y, h, dh, dxn, wq))
    n = h.shape[1]
    r_h = rho(h)
    u = dxn * wq
    g = dh + r_h * (u - h * r_h ** 2 * (u * h).mean(1, keepdim=True))
    ga = dh.abs() + r_h * (u.abs() + h.abs() * r_h ** 2 * (u * h).abs().mean(1, keepdim=True))
    g64 = torch.ones(1, 1, dtype=torch.float64, device=y.device) if gt is None else gt.double()
    w = wp.double() if post else torch.ones(n, dtype=torch.float64, device=y.device)
    r_y = rho(y) if post else torch.ones(y.shape[0], 1, dtype=torch.float64, device=y.device)
    yn = y * r_y
    t, ta = beta * g * yn * w, (beta * ga * yn * w).abs()
    v, va = beta * g64 * g * w, (beta * g64 * ga * w).abs()
    out = {"dres": (alpha * g, abs(alpha) * ga), "dpre_w": ((dxn * h * r_h).sum(0), (dxn * h * r_h).abs().sum(0))}
    if gate == "channel":
        out["dgate"] = (t.sum(0), ta.sum(0))
    if gate == "token":
        out["dgate"] = (t.sum(1, keepdim=True), ta.sum(1, keepdim=True))
    if post:
        out["dpost_w"] = ((beta * g64 * g * yn).sum(0), (beta * g64 * ga * yn).abs().sum(0))
        out["dy"] = (r_y * (v - yn * (v * yn).mean(1, keepdim=True)),
                     r_y * (va + yn.abs() * (va * yn.abs()).mean(1, keepdim=True)))
    else:
        out["dy"] = (v, va)
    return out


@pytest.mark.parametrize("rows,cols", ROWS_COLS)
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("gate", ["none", "channel", "token"])
@pytest.mark.parametrize("post", [True, False])
def test_backward(ffn, cuda, rows, cols, dtype, gate, post):
    import torch
    dt = getattr(torch, dtype)
    y, h, gt, wp, wq = inputs(torch, cuda, rows, cols, dt, gate, 1)
    dh, dxn = inputs(torch, cuda, rows, cols, dt, gate, 2)[:2]
    bn = ffn.BlockNorm(pre_w=wq, post_w=wp if post else None, alpha=0.75, beta=-0.5, eps=EPS)
    got = bn.backward(y, h, dh=dh, dxn=dxn, gate=gt)
    want = reference_backward(torch, y, h, dh, dxn, gt, wp, wq, 0.75, -0.5, gate, post)
    for name, t in got.items():
        if name not in want:
            assert t is None, name
            continue
        ref, mag = want[name]
        # every term of the chain carries at most two reciprocal roots and two
        # row means (30 + 50 each) and a dozen products; sums over rows add at
        # most one rounding a row
        c = 2 * (30 + 50) + 16 + (rows if name in ("dpre_w", "dpost_w") or (name == "dgate" and gate == "channel") else 50)
        err = c * U * mag
        u = half_step(torch, dt) if t.dtype == dt and name in ("dy", "dres") else U
        assert t.shape == ref.shape, name
        assert ((t.double() - ref).abs() <= err + u * (ref.abs() + err) + tiny(torch, dt)).all(), name
    assert all(torch.equal(a, b) for a, b in zip(got.values(), bn.backward(y, h, dh=dh, dxn=dxn, gate=gt).values())
               if a is not None)  # no atomics: the same bits again


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_backward_of_one_gradient_alone(ffn, cuda, dtype):
    import torch
    dt = getattr(torch, dtype)
    y, h, gt, wp, wq = inputs(torch, cuda, 40, 264, dt, "channel", 1)
    dh, dxn = inputs(torch, cuda, 40, 264, dt, "channel", 2)[:2]
    bn = ffn.BlockNorm(pre_w=wq, post_w=wp, alpha=0.5, beta=2.0, eps=EPS)
    z = torch.zeros_like(dh)
    for a, b in ((dict(dh=dh), dict(dh=dh, dxn=z)), (dict(dxn=dxn), dict(dh=z, dxn=dxn))):
        one, both = bn.backward(y, h, gate=gt, **a), bn.backward(y, h, gate=gt, **b)
        for k in ("dy", "dres", "dpost_w", "dgate"):
            assert torch.equal(one[k], both[k]), k
    assert bn.backward(y, h, dh=dh, gate=gt)["dpre_w"] is None
    alone = bn.backward(None, h, dh=dh, dxn=dxn)  # the norm before the first block
    assert torch.equal(alone["dres"], bn.backward(y, h, dh=dh, dxn=dxn, gate=gt)["dres"]) and alone["dy"] is None


def test_backward_against_differences(ffn, cuda):
    """Central differences of L = <c, h> + <d, xn> in f32 rows."""
    import torch
    rows, cols = 4, 24
    y, res, gt, wp, wq = inputs(torch, cuda, rows, cols, torch.float32, "channel", 7)
    c, d = inputs(torch, cuda, rows, cols, torch.float32, "channel", 8)[:2]

    def loss(y, res, gt, wp, wq):
        h, xn = ffn.BlockNorm(wq, wp, 0.75, 1.5, EPS).forward(y, res, gate=gt)
        return float((h.double() * c.double()).sum() + (xn.double() * d.double()).sum())
    h, _ = ffn.BlockNorm(wq, wp, 0.75, 1.5, EPS).forward(y, res, gate=gt)
    got = ffn.BlockNorm(wq, wp, 0.75, 1.5, EPS).backward(y, h, dh=c, dxn=d, gate=gt)
    args = [y, res, gt, wp, wq]
    step = 2.0 ** -7
    for at, name in enumerate(("dy", "dres", "dgate", "dpost_w", "dpre_w")):
        for i in range(0, args[at].numel(), 5):
            vals = []
            for s in (step, -step):
                a = [t.clone() for t in args]
                a[at].view(-1)[i] += s
                vals.append(loss(*a))
            diff, g = (vals[0] - vals[1]) / (2 * step), float(got[name].view(-1)[i])
            # rounding: ~200 terms of size < 4 at a few U over 2 * step; truncation:
            # step^2 / 6 times a third derivative, below 100 for rows of these sizes
            assert abs(diff - g) < 200 * 4 * 8 * U / (2 * step) + step ** 2 / 6 * 100, (name, i, diff, g)


def test_rows_of_wider_tensors_streams_and_graphs(ffn, cuda):
    import torch
    rows, cols = 50, 320
    y, res, gt, wp, wq = inputs(torch, cuda, rows, cols, torch.float16, "token", 3)
    dh, dxn = inputs(torch, cuda, rows, cols, torch.float16, "token", 4)[:2]
    wide = torch.empty(rows, 3 * cols + 1, dtype=torch.float16, device=cuda)
    wide[:, 1:1 + cols], wide[:, 1 + cols:1 + 2 * cols] = y, res
    ys, rs = wide[:, 1:1 + cols], wide[:, 1 + cols:1 + 2 * cols]  # rows start on odd elements
    bn = ffn.BlockNorm(pre_w=wq, post_w=wp, alpha=0.5, beta=2.0, eps=EPS)

    def run(y, res):
        h, xn = bn.forward(y, res, gate=gt)
        return [h, xn] + [v for v in bn.backward(y, h, dh=dh, dxn=dxn, gate=gt).values()]
    want = run(y, res)
    # another split of a row over threads: equal up to f32 sums, so up to one step of f16 (2^-10 relative)
    for a, b in zip(run(ys, rs), want):
        assert torch.allclose(a.float(), b.float(), rtol=2.0 ** -10, atol=1e-4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = bn.forward(y, res, gate=gt, stream=side)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run(y, res)
        graphs.append((g, out))
    for g, _ in graphs * 2:
        g.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_no_rows_and_bad_workspaces(ffn, cuda):
    import ctypes as C

    import torch
    wp = torch.ones(64, device=cuda)
    bn = ffn.BlockNorm(pre_w=wp, post_w=wp)
    e = torch.empty(0, 64, device=cuda)
    h, xn = bn.forward(e, e)
    assert h.shape == xn.shape == (0, 64)
    got = bn.backward(e, e, dh=e, dxn=e, gate=wp)
    assert all((got[k] == 0).all() for k in ("dpost_w", "dpre_w", "dgate"))
    x = torch.randn(4, 64, device=cuda)
    d = ffn.BlockNormDesc(4, 64, 0, 0, wp.data_ptr(), None, wp.data_ptr(), 1.0, 1.0, EPS, 0)
    dw = torch.empty(64, device=cuda)
    p = x.data_ptr()
    L = ffn.lib()
    args = [C.byref(d), p, 64, p, 64, p, 64, p, 64, None, 0, None, 0, None, None, dw.data_ptr()]
    assert L.ffn_b200_block_norm_bwd(*args, None, 0, None) == -1
    assert L.ffn_b200_block_norm_bwd(*args, p, 64, None) == -3
    with pytest.raises(ffn.FfnError):
        bn.forward(x, x, gate=torch.ones(4, device=cuda))
    with pytest.raises(ffn.FfnError):
        bn.forward(x, x.half())
    with pytest.raises(ffn.FfnError):
        ffn.BlockNorm(pre_w=wp.half()).forward(x, x)
