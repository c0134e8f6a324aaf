"""Outputs in place of inputs, where the header allows it."""
import ctypes as C

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,cols", [(1500, 4096), (700, 1000), (701, 1023), (500, 8192), (333, 16384)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_norm_in_place(ffn, cuda, rows, cols, dtype):
    """h in y or in the residual; dresidual in dh, dy in y or in dxn: the same bits."""
    import torch
    dt = getattr(torch, dtype)
    g = torch.Generator(device=cuda).manual_seed(rows)
    y, res, dh, dxn = (torch.randn(rows, cols, device=cuda, generator=g).to(dt) for _ in range(4))
    w, gate = 1 + 0.2 * torch.randn(cols, device=cuda, generator=g), torch.rand(rows, 1, device=cuda, generator=g)
    norm = ffn.BlockNorm(w, w, 0.75, 0.5)
    h, xn = norm.forward(y, res, gate=gate)
    for at in (0, 1):
        a = [y.clone(), res.clone()]
        h2, xn2 = norm.forward(*a, gate=gate, h=a[at])
        assert h2 is a[at] and torch.equal(h2, h) and torch.equal(xn2, xn)
    want = norm.backward(y, h, dh=dh, dxn=dxn, gate=gate)
    L = ffn.lib()
    d = ffn.BlockNormDesc(rows, cols, 1 if dt == torch.bfloat16 else 0, ffn.GATE_TOKEN, w.data_ptr(), gate.data_ptr(),
                          w.data_ptr(), 0.75, 0.5, 1e-6, 0)
    nb = L.ffn_b200_block_norm_bwd_ws_bytes(C.byref(d))
    for dy_in in ("y", "dxn"):
        t = {"y": y.clone(), "dh": dh.clone(), "dxn": dxn.clone()}
        f = [torch.empty(n, device=cuda) for n in (cols, rows, cols)]
        ws = torch.empty(nb, dtype=torch.uint8, device=cuda)
        p = {k: v.data_ptr() for k, v in t.items()}
        rc = L.ffn_b200_block_norm_bwd(C.byref(d), p["y"], cols, h.data_ptr(), cols, p["dh"], cols, p["dxn"], cols, p["dh"], cols,
                                       p[dy_in], cols, f[0].data_ptr(), f[1].data_ptr(), f[2].data_ptr(), ws.data_ptr(), nb,
                                       torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        assert torch.equal(t["dh"], want["dres"]) and torch.equal(t[dy_in], want["dy"])
        assert torch.equal(f[0], want["dpost_w"]) and torch.equal(f[1], want["dgate"].view(-1)) and torch.equal(f[2], want["dpre_w"])


@pytest.mark.parametrize("tokens,cols", [(1, 64), (900, 4096), (901, 1023)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_combine_into_the_residual(ffn, cuda, tokens, cols, dtype):
    import torch
    dt = getattr(torch, dtype)
    g = torch.Generator(device=cuda).manual_seed(tokens)
    res, y = (torch.randn(n, cols, device=cuda, generator=g).to(dt) for n in (tokens, tokens * 6))
    pos = torch.randperm(tokens * 6, device=cuda, generator=g).to(torch.int32).view(tokens, 6)
    wt = torch.rand(tokens, 6, device=cuda, generator=g)
    want = ffn.moe_combine(y, pos, wt, residual=res)
    assert ffn.moe_combine(y, pos, wt, residual=res, out=res) is res and torch.equal(res, want)
