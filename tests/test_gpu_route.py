"""Routed pairs sorted by expert and back (moe_sort, moe_permute, moe_combine and
its gradient) against plain 64-bit restatements of their definitions."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24  # half a step of f32
NONE = 0x7FFFFFFF


def half_step(torch, dt):
    return torch.finfo(dt).eps / 2


def sorted_pairs(idx, lo, hi):
    flat = idx.reshape(-1).astype(np.int64)
    local = (flat >= lo) & (flat < hi)
    order = np.argsort(np.where(local, flat, hi), kind="stable")[:local.sum()]
    pos = np.full(flat.size, -1, dtype=np.int64)
    pos[order] = np.arange(order.size)
    src = np.full(flat.size, -1, dtype=np.int64)
    src[:order.size] = order
    counts = np.bincount(flat[local] - lo, minlength=hi - lo)
    return np.concatenate([[0], np.cumsum(counts)]), pos.reshape(idx.shape), src


@pytest.mark.parametrize("n_exp,lo,hi", [(1, 0, 1), (8, 0, 8), (8, 3, 4), (60, 10, 50), (384, 0, 384), (384, 336, 384),
                                         (1024, 0, 1024), (1500, 7, 1500), (4096, 0, 4096)])
@pytest.mark.parametrize("n_tok,top_k", [(0, 6), (1, 1), (1, 6), (5, 7), (64, 6), (341, 6), (342, 6), (683, 3), (8192, 6),
                                         (9001, 8)])
def test_sort(ffn, cuda, n_exp, lo, hi, n_tok, top_k):
    import torch
    rng = np.random.default_rng(n_exp * 31 + lo + n_tok * 7 + top_k)
    idx = (rng.integers(0, n_exp, (n_tok, top_k)) * rng.random((n_tok, top_k))).astype(np.int32)  # skewed to low ids
    if n_tok > 2:  # ids that no expert has
        idx[0, 0], idx[1, -1], idx[2, 0] = NONE, -1, -2 ** 31
    offsets, pos, src = ffn.moe_sort(torch.from_numpy(idx).to(cuda), lo, hi)
    torch.cuda.synchronize()
    ro, rp, rs = sorted_pairs(idx, lo, hi)
    np.testing.assert_array_equal(offsets.cpu().numpy(), ro)
    np.testing.assert_array_equal(pos.cpu().numpy(), rp)
    np.testing.assert_array_equal(src.cpu().numpy(), rs)


def test_sort_all_pairs_of_one_expert_and_of_none(ffn, cuda):
    import torch
    idx = torch.full((3001, 4), 17, dtype=torch.int32, device=cuda)
    offsets, pos, src = ffn.moe_sort(idx, 0, 32)
    assert offsets.tolist() == [0] * 18 + [12004] * 15
    assert torch.equal(pos.view(-1), torch.arange(12004, device=cuda, dtype=torch.int32))
    offsets, pos, src = ffn.moe_sort(idx, 18, 32)
    assert offsets.tolist() == [0] * 15 and (pos == -1).all() and (src == -1).all()


def test_sort_through_the_c_entry_without_pos_and_src(ffn, cuda):
    import torch
    idx = torch.tensor([[3, 1], [1, 0]], dtype=torch.int32, device=cuda)
    off = torch.full((6,), -7, dtype=torch.int32, device=cuda)
    ffn.check(ffn.lib().ffn_b200_moe_sort(2, 2, idx.data_ptr(), 0, 4, off.data_ptr(), None, None,
                                          torch.cuda.current_stream().cuda_stream))
    assert off.tolist() == [0, 1, 3, 3, 4, -7]


def routed(torch, cuda, seed, n_tok, top_k, n_exp, lo, hi):
    rng = np.random.default_rng(seed)
    idx = rng.integers(0, n_exp, (n_tok, top_k)).astype(np.int32)
    if n_tok > 1:
        idx[1] = NONE  # a token without any expert
    _, pos, _ = sorted_pairs(idx, lo, hi)
    return idx, torch.from_numpy(pos.astype(np.int32)).to(cuda), int((pos >= 0).sum())


CASES = [(1, 1, 1, 0, 1), (1, 6, 384, 0, 384), (3, 2, 8, 2, 6), (65, 6, 384, 336, 384), (257, 8, 60, 0, 60), (33, 17, 40, 5, 40)]
COLS = [1, 7, 8, 64, 129, 1000, 1023, 1032, 4096, 5120]


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16", "int8"])
@pytest.mark.parametrize("cols", COLS)
def test_permute(ffn, cuda, case, dtype, cols):
    import torch
    dt = getattr(torch, dtype)
    n_tok, top_k = case[:2]
    idx, pos, n = routed(torch, cuda, sum(case) + cols, *case)
    x = torch.randint(-100, 100, (n_tok, cols), device=cuda).to(dt)
    scales = torch.rand(n_tok, device=cuda)
    out = torch.full((n_tok * top_k, cols), 77, dtype=dt, device=cuda)
    got, sc = ffn.moe_permute(x, pos, out=out, scales=scales, out_scales=torch.full((n_tok * top_k,), -1.0, device=cuda))
    assert got is out
    p, xc = pos.cpu().long(), x.cpu()
    want, wsc = torch.full_like(xc, 77)[:1].repeat(n_tok * top_k, 1), torch.full((n_tok * top_k,), -1.0)
    for t in range(n_tok):
        for k in range(top_k):
            if p[t, k] >= 0:
                want[p[t, k]] = xc[t]
                wsc[p[t, k]] = scales.cpu()[t]
    assert torch.equal(got.cpu(), want) and torch.equal(sc.cpu(), wsc)  # rows behind the last: as they were
    assert torch.equal(ffn.moe_permute(x, pos)[:n].cpu(), want[:n])


def combine_reference(torch, y, pos, w, res):
    """(sum, sum of absolute terms) in 64 bits."""
    y, pos = y.cpu().double(), pos.cpu().long()
    w = torch.ones(pos.shape, dtype=torch.float64) if w is None else w.cpu().double()
    t = torch.where((pos >= 0)[:, :, None], y[pos.clamp(min=0)], 0.0) * w[:, :, None]
    s, m = t.sum(1), t.abs().sum(1)
    return (s, m) if res is None else (s + res.cpu().double(), m + res.cpu().double().abs())


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("weighted,with_res", [(True, True), (True, False), (False, False)])
def test_combine(ffn, cuda, case, dtype, cols, weighted, with_res):
    import torch
    dt = getattr(torch, dtype)
    n_tok, top_k = case[:2]
    _, pos, n = routed(torch, cuda, sum(case) * 3 + cols, *case)
    g = torch.Generator(device=cuda).manual_seed(cols)
    y = torch.randn(n_tok * top_k, cols, device=cuda, generator=g).to(dt)
    y[n:] = float("nan")  # rows behind the last are not read
    w = torch.rand(n_tok, top_k, device=cuda, generator=g) if weighted else None
    res = torch.randn(n_tok, cols, device=cuda, generator=g).to(dt) if with_res else None
    out = ffn.moe_combine(y, pos, w, residual=res)
    ref, mag = combine_reference(torch, y, pos, w, res)
    # top_k fused multiply-adds and one addition in f32, then one rounding to
    # the type (the smallest f16 step is 2^-24: half of it is an absolute bound)
    err, u = (top_k + 2) * U * mag, half_step(torch, dt)
    tol = err + u * (ref.abs() + err) + (2.0 ** -25 if dt == torch.float16 else 0.0)
    assert out.dtype == dt
    assert ((out.cpu().double() - ref).abs() <= tol).all()
    if with_res:  # in place over the residual
        again = ffn.moe_combine(y, pos, w, residual=res, out=res)
        assert again is res and torch.equal(again, out)


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("cols", COLS)
def test_combine_backward(ffn, cuda, case, dtype, cols):
    import torch
    dt = getattr(torch, dtype)
    n_tok, top_k = case[:2]
    _, pos, n = routed(torch, cuda, sum(case) * 5 + cols, *case)
    g = torch.Generator(device=cuda).manual_seed(cols + 1)
    y = torch.randn(n_tok * top_k, cols, device=cuda, generator=g).to(dt)
    y[n:] = float("nan")
    dout = torch.randn(n_tok, cols, device=cuda, generator=g).to(dt)
    w = torch.rand(n_tok, top_k, device=cuda, generator=g)
    dy0 = torch.full((n_tok * top_k, cols), 5.0, dtype=dt, device=cuda)
    dy, dw = ffn.moe_combine_backward(dout, y, pos, w, dy=dy0)
    assert dy is dy0 and (dy[n:] == 5).all()  # as they were
    p, d, u = pos.cpu().long(), dout.cpu().double(), half_step(torch, dt)
    tiny = 2.0 ** -25 if dt == torch.float16 else 0.0
    terms = torch.where((p >= 0)[:, :, None], y.cpu().double()[p.clamp(min=0)], 0.0) * d[:, None, :]
    # at most `cols` fused multiply-adds and additions in f32
    assert ((dw.cpu().double() - terms.sum(2)).abs() <= (cols + 1) * U * terms.abs().sum(2)).all()
    assert (dw.cpu()[p < 0] == 0).all()
    want = w.cpu().double()[:, :, None] * d[:, None, :]
    got = dy.cpu().double()[p.clamp(min=0)]
    ok = (got - want).abs() <= want.abs() * (U + u + U * u) + tiny
    assert (ok | (p < 0)[:, :, None]).all()
    # the gradient of permute, and weights of one
    dx = ffn.moe_permute_backward(y, pos)
    ref, mag = combine_reference(torch, y, pos, None, None)
    err = (top_k + 2) * U * mag
    assert ((dx.cpu().double() - ref).abs() <= err + u * (ref.abs() + err) + tiny).all()
    ones, _ = ffn.moe_combine_backward(dout, y, pos)
    assert torch.equal(ones.cpu()[p[p >= 0]], dout.cpu()[(p >= 0).nonzero()[:, 0]])
    assert (ones[n:] == 0).all()


def test_gradients_against_differences(ffn, cuda):
    """Central differences of L = <c, combine(permute(x) * a, w)> in f32."""
    import torch
    g = torch.Generator(device=cuda).manual_seed(3)
    idx = torch.randint(0, 6, (5, 3), device=cuda, generator=g, dtype=torch.int32)
    offsets, pos, _ = ffn.moe_sort(idx, 1, 6)
    x, c = (torch.randn(5, 12, device=cuda, generator=g) for _ in range(2))
    a = torch.randn(15, 12, device=cuda, generator=g)
    w = torch.rand(5, 3, device=cuda, generator=g)

    def loss(x, w):
        xs = ffn.moe_permute(x, pos, out=torch.zeros(15, 12, device=cuda))
        return float((ffn.moe_combine(xs * a, pos, w).double() * c.double()).sum())
    xs = ffn.moe_permute(x, pos, out=torch.zeros(15, 12, device=cuda))
    dy, dw = ffn.moe_combine_backward(c, xs * a, pos, w)
    dx = ffn.moe_permute_backward(dy * a, pos)
    # L is linear in x and in w, so a difference over 2 eps has no truncation
    # error; its rounding: 60 sums of magnitude < 100 at 2^-24 each way over 0.5
    for t, got in ((x, dx), (w, dw)):
        flat = t.view(-1)
        for i in range(0, flat.numel(), 7):
            hi, lo = t.clone(), t.clone()
            hi.view(-1)[i] += 0.25
            lo.view(-1)[i] -= 0.25
            args = ((hi, w), (lo, w)) if t is x else ((x, hi), (x, lo))
            diff = (loss(*args[0]) - loss(*args[1])) / 0.5
            assert abs(diff - float(got.view(-1)[i])) < 60 * 100 * U * 4


def test_slices_streams_and_a_captured_graph(ffn, cuda):
    import torch
    n_tok, top_k, cols = 70, 4, 96
    idx = torch.randint(0, 16, (n_tok, top_k), device=cuda, dtype=torch.int32)
    wide = torch.randn(n_tok, 3 * cols + 5, device=cuda, dtype=torch.float32).to(torch.bfloat16)
    x = wide[:, 3:3 + cols]  # misaligned rows of a wider tensor
    w = torch.rand(n_tok, top_k, device=cuda)

    def run():
        _, pos, _ = ffn.moe_sort(idx, 0, 16)
        xs = ffn.moe_permute(x, pos)
        out = torch.empty(n_tok, 2 * cols, device=cuda, dtype=torch.bfloat16)[:, :cols]
        ffn.moe_combine(xs, pos, w, residual=x, out=out)
        return out, *ffn.moe_combine_backward(out, xs, pos, w)
    want = run()
    ref, mag = combine_reference(torch, ffn.moe_permute(x, ffn.moe_sort(idx, 0, 16)[1]), ffn.moe_sort(idx, 0, 16)[1], w, x)
    err = (top_k + 2) * U * mag
    assert ((want[0].cpu().double() - ref).abs() <= err + 2.0 ** -8 * (ref.abs() + err)).all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run()
        graphs.append((g, out))
    for g, _ in graphs + graphs:  # replayed in turn, and once more with new inputs below
        g.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    idx.copy_(torch.randint(0, 16, (n_tok, top_k), device=cuda, dtype=torch.int32))
    want = run()
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(graphs[0][1], want))


def test_offsets_past_32_bits(ffn, cuda):
    """Rows whose byte and element offsets pass 2^32."""
    import torch
    cols, rows = 65536, 70000  # 4.6e9 elements, 9.2 GB
    y = torch.empty(rows, cols, dtype=torch.bfloat16, device=cuda)
    y[-3:] = torch.arange(3, device=cuda, dtype=torch.bfloat16)[:, None] + 1
    pos = torch.tensor([[rows - 1, rows - 3]], dtype=torch.int32, device=cuda)
    out = ffn.moe_combine(y, pos, torch.tensor([[2.0, 0.5]], device=cuda))
    assert (out == 6.5).all()
    x = torch.full((1, cols), 9.0, dtype=torch.bfloat16, device=cuda)
    ffn.moe_permute(x, pos, out=y)
    assert (y[-1] == 9).all() and (y[-3] == 9).all() and (y[-2] == 2).all()


def test_pos_outside_the_rows_is_skipped(ffn, cuda):
    import torch
    y = torch.ones(4, 8, device=cuda)
    pos = torch.tensor([[0, 4], [3, -9]], dtype=torch.int32, device=cuda)
    assert ffn.moe_combine(y, pos).tolist() == [[1.0] * 8] * 2
    out = torch.zeros(4, 8, device=cuda)
    ffn.moe_permute(torch.ones(2, 8, device=cuda), pos, out=out)
    assert out[:, 0].tolist() == [1, 0, 0, 1]
    with pytest.raises(ffn.FfnError):
        ffn.moe_combine(y, pos.long())
    with pytest.raises(ffn.FfnError):
        ffn.moe_combine(y.double(), pos)
    with pytest.raises(ffn.FfnError):
        ffn.moe_combine(y, pos, residual=torch.ones(3, 8, device=cuda))
    with pytest.raises(ffn.FfnError):
        ffn.moe_permute(torch.ones(2, 8, device=cuda), pos, out=torch.zeros(8, 4, device=cuda).t())
