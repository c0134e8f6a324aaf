"""Row operators over no rows, through the module and through ctypes."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("module", [True, False])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_calls_over_nothing(ffn, cuda, monkeypatch, module, dtype):
    import torch
    ffn._setup()
    if not module:
        monkeypatch.setattr(ffn, "_calls", None)
    dt = getattr(torch, dtype)
    none = torch.empty(0, 64, device=cuda, dtype=dt)
    w = torch.ones(64, device=cuda)
    norm = ffn.BlockNorm(w, w)
    for gate in (None, w, torch.empty(0, 1, device=cuda)):
        h, xn = norm.forward(none, none, gate=gate)
        assert h.shape == xn.shape == (0, 64) and h.dtype == dt
        got = norm.backward(none, h, dh=none, dxn=none, gate=gate)
        assert (got["dpost_w"] == 0).all() and (got["dpre_w"] == 0).all()
        assert gate is None or got["dgate"].shape == gate.shape and (got["dgate"] == 0).all()
    h, xn, q, s = norm.forward(none, none, gate=torch.empty(0, 1, device=cuda), codes=True)
    assert q.shape == (0, 64) and s.shape == (0,)
    q, s = ffn.quantize_int8(none)
    assert q.shape == (0, 64) and s.shape == (0,)
    for groups, off in ((1, None), (3, torch.zeros(4, dtype=torch.int32, device=cuda))):
        m = ffn.Int8Matrix(torch.ones(groups, 8, 64, dtype=torch.int8, device=cuda), torch.ones(groups, 8, device=cuda))
        assert m.matmul(none, offsets=off).shape == (0, 8) and m.matmul((q, s), offsets=off).shape == (0, 8)

    # no tokens, then tokens whose pairs are all elsewhere
    off, pos, src = ffn.moe_sort(torch.empty(0, 2, dtype=torch.int32, device=cuda), 0, 4)
    assert off.tolist() == [0] * 5 and pos.shape == (0, 2) and src.shape == (0,)
    assert ffn.moe_permute(none, pos).shape == (0, 64) and ffn.moe_combine(none, pos).shape == (0, 64)
    dy, dw = ffn.moe_combine_backward(none, none, pos)
    assert dy.shape == (0, 64) and dw.shape == (0, 2)
    x = torch.ones(5, 64, device=cuda, dtype=dt)
    off, pos, src = ffn.moe_sort(torch.full((5, 2), 9, dtype=torch.int32, device=cuda), 0, 4)
    assert off.tolist() == [0] * 5 and (pos == -1).all() and (src == -1).all()
    assert ffn.moe_permute(x, pos, out=none) is none
    rows, scales = ffn.moe_permute(torch.ones(5, 64, dtype=torch.int8, device=cuda), pos,
                                   out=torch.empty(0, 64, dtype=torch.int8, device=cuda), scales=torch.ones(5, device=cuda))
    assert rows.shape == (0, 64) and scales.shape == (0,)
    assert torch.equal(ffn.moe_combine(none, pos, residual=x), x) and (ffn.moe_combine(none, pos) == 0).all()
    dy, dw = ffn.moe_combine_backward(x, none, pos)
    assert dy.shape == (0, 64) and (dw == 0).all() and dw.shape == (5, 2)
    torch.cuda.synchronize()
