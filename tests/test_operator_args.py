"""CPU tests: what the row operators (int8 products, expert dispatch and
combine, block norms) refuse, before any CUDA call.  Pointers are fakes."""
import ctypes as C

import pytest

OK, EINVAL, ENOSPC, EUNSUP = 0, -1, -3, -5
P = 4096  # a fake, well-aligned device address


def refused(ffn, rc, code, text):
    msg = ffn.lib().ffn_b200_last_error()
    assert rc == code and text in msg, (rc, msg)


def quant(ffn, rows=4, cols=64, dtype=1, x=P, ld_x=64, act=0, codes=P, ld_c=64, scales=P):
    return ffn.lib().ffn_b200_quantize_int8(rows, cols, dtype, x, ld_x, act, None, codes, ld_c, scales, None)


def test_quantize_int8_refusals(ffn):
    assert quant(ffn, rows=0) == OK
    for kw, code, text in (
            (dict(dtype=3), EINVAL, b"dtype"), (dict(dtype=-1), EINVAL, b"dtype"), (dict(act=2), EINVAL, b"act"),
            (dict(cols=0), EUNSUP, b"cols"), (dict(cols=16385, ld_x=16385, ld_c=16400), EUNSUP, b"cols"),
            (dict(x=None), EINVAL, b"null"), (dict(codes=None), EINVAL, b"null"), (dict(scales=None), EINVAL, b"null"),
            (dict(ld_x=63), EINVAL, b"overlap"), (dict(ld_c=63), EINVAL, b"overlap"),
            (dict(act=1), EINVAL, b"overlap"),  # gate and up need 128 columns
            (dict(x=P + 1), EINVAL, b"aligned"), (dict(scales=P + 2), EINVAL, b"aligned"),
            (dict(rows=1 << 31), EINVAL, b"rows")):
        refused(ffn, quant(ffn, **kw), code, text)


def product(ffn, rows=4, n=8, k=64, groups=1, offsets=None, x=P, ld_x=64, xs=P, w=P, ld_w=64, ws=P, bias=None, dtype=0,
            out=P, ld_out=8):
    return ffn.lib().ffn_b200_int8_matmul(rows, n, k, groups, offsets, x, ld_x, xs, w, ld_w, ws, bias, dtype, out, ld_out,
                                          None)


def test_int8_matmul_refusals(ffn):
    assert product(ffn, rows=0) == OK
    for kw, code, text in (
            (dict(dtype=9), EINVAL, b"dtype"), (dict(n=0), EUNSUP, b"n must"), (dict(k=0), EUNSUP, b"k in"),
            (dict(k=131073, ld_x=131088, ld_w=131088), EUNSUP, b"k in"), (dict(groups=0), EINVAL, b"n_groups"),
            (dict(groups=4097, offsets=P), EINVAL, b"n_groups"), (dict(groups=2), EINVAL, b"offsets"),
            (dict(x=None), EINVAL, b"null"), (dict(w=None), EINVAL, b"null"), (dict(xs=None), EINVAL, b"null"),
            (dict(ws=None), EINVAL, b"null"), (dict(out=None), EINVAL, b"null"),
            (dict(x=P + 8), EINVAL, b"16 bytes"), (dict(w=P + 1), EINVAL, b"16 bytes"),
            (dict(ld_x=72), EINVAL, b"16 bytes"), (dict(ld_w=65), EINVAL, b"16 bytes"),
            (dict(ld_x=48), EINVAL, b"overlap"), (dict(ld_w=48), EINVAL, b"overlap"), (dict(ld_out=7), EINVAL, b"overlap"),
            (dict(out=P + 2), EINVAL, b"aligned"), (dict(bias=P + 1), EINVAL, b"aligned"),
            (dict(rows=(1 << 30) + 1), EINVAL, b"rows"), (dict(n=1 << 29, groups=4, offsets=P, ld_out=1 << 29), EINVAL, b"rows")):
        refused(ffn, product(ffn, **kw), code, text)


def test_moe_sort_refusals(ffn):
    L = ffn.lib()
    for args, text in (
            ((4, 0, P, 0, 8, P, P, P), b"top_k"), ((1 << 30, 2, P, 0, 8, P, P, P), b"too many"),
            ((4, 2, None, 0, 8, P, P, P), b"null"), ((4, 2, P, 0, 8, None, P, P), b"null"),
            ((4, 2, P, -1, 8, P, P, P), b"range"), ((4, 2, P, 8, 8, P, P, P), b"range"),
            ((4, 2, P, 0, 4097, P, P, P), b"range")):
        refused(ffn, L.ffn_b200_moe_sort(*args, None), EINVAL, text)


def test_moe_permute_refusals(ffn):
    L = ffn.lib()
    assert L.ffn_b200_moe_permute(0, 2, 64, None, 0, None, 0, None, 0, None, None, None) == OK
    for args, text in (
            ((4, 2, 64, None, 64, P, 8, P, 64, None, None), b"null"), ((4, 2, 64, P, 64, None, 8, P, 64, None, None), b"null"),
            ((4, 2, 0, P, 64, P, 8, P, 64, None, None), b"row size"), ((4, 2, 64, P, 63, P, 8, P, 64, None, None), b"overlap"),
            ((4, 2, 64, P, 64, P, 8, P, 63, None, None), b"overlap"), ((4, 2, 64, P, 64, P, 8, P, 64, P, None), b"together"),
            ((4, 0, 64, P, 64, P, 8, P, 64, None, None), b"top_k"), ((4, 2, 64, P, 64, P, 1 << 31, P, 64, None, None), b"rows")):
        refused(ffn, L.ffn_b200_moe_permute(*args, None), EINVAL, text)


def test_moe_combine_refusals(ffn):
    L = ffn.lib()
    ok = dict(n=4, k=2, cols=16, dt=0, y=P, ld_y=16, rows=8, pos=P, w=P, res=None, ld_r=0, out=P, ld_o=16)

    def go(**kw):
        a = {**ok, **kw}
        return L.ffn_b200_moe_combine(a["n"], a["k"], a["cols"], a["dt"], a["y"], a["ld_y"], a["rows"], a["pos"], a["w"],
                                      a["res"], a["ld_r"], a["out"], a["ld_o"], None)
    assert go(n=0) == OK
    for kw, text in ((dict(dt=5), b"dtype"), (dict(cols=0), b"cols"), (dict(k=0), b"top_k"), (dict(y=None), b"null"),
                     (dict(pos=None), b"null"), (dict(out=None), b"null"), (dict(ld_y=15), b"overlap"),
                     (dict(ld_o=15), b"overlap"), (dict(res=P, ld_r=8), b"overlap"), (dict(y=P + 2), b"aligned")):
        refused(ffn, go(**kw), EINVAL, text)

    def back(**kw):
        a = {**ok, "dout": P, "ld_d": 16, "dy": P, "ld_dy": 16, "dw": P, **kw}
        return L.ffn_b200_moe_combine_bwd(a["n"], a["k"], a["cols"], a["dt"], a["dout"], a["ld_d"], a["y"], a["ld_y"],
                                          a["rows"], a["pos"], a["w"], a["dy"], a["ld_dy"], a["dw"], None)
    assert back(n=0) == OK and back(dy=None, dw=None) == OK
    for kw, text in ((dict(dt=5), b"dtype"), (dict(dout=None), b"null"), (dict(y=None), b"null"), (dict(pos=None), b"null"),
                     (dict(ld_d=3), b"overlap"), (dict(ld_dy=3), b"overlap"), (dict(dout=P + 1), b"aligned")):
        refused(ffn, back(**kw), EINVAL, text)


def desc(ffn, **kw):
    a = {**dict(rows=4, cols=64, dtype=0, kind=0, post=P, gate=None, pre=P, alpha=1.0, beta=1.0, eps=1e-6), **kw}
    return ffn.BlockNormDesc(a["rows"], a["cols"], a["dtype"], a["kind"], a["post"], a["gate"], a["pre"], a["alpha"],
                             a["beta"], a["eps"], 0)


def test_block_norm_refusals(ffn):
    L = ffn.lib()
    assert C.sizeof(ffn.BlockNormDesc) == 64

    def go(d=None, y=P, ld_y=64, r=P, ld_r=64, h=P, ld_h=64, xn=P, ld_x=64, codes=None, ld_c=0, cs=None):
        return L.ffn_b200_block_norm(C.byref(d or desc(ffn)), y, ld_y, r, ld_r, h, ld_h, xn, ld_x, codes, ld_c, cs, None)
    assert L.ffn_b200_block_norm(None, P, 64, P, 64, P, 64, P, 64, None, 0, None, None) == EINVAL
    assert go(desc(ffn, rows=0)) == OK
    for kw, code, text in (
            (dict(d=desc(ffn, dtype=4)), EINVAL, b"dtype"), (dict(d=desc(ffn, cols=0)), EUNSUP, b"cols"),
            (dict(d=desc(ffn, cols=16385)), EUNSUP, b"cols"), (dict(d=desc(ffn, kind=3, gate=P)), EINVAL, b"gate_kind"),
            (dict(d=desc(ffn, kind=1)), EINVAL, b"gate"), (dict(d=desc(ffn, gate=P)), EINVAL, b"gate"),
            (dict(d=desc(ffn, eps=-1.0)), EINVAL, b"eps"), (dict(d=desc(ffn, eps=float("nan"))), EINVAL, b"eps"),
            (dict(d=desc(ffn, post=P + 2)), EINVAL, b"4-byte"), (dict(d=desc(ffn, pre=None)), EINVAL, b"pre_w"),
            (dict(y=None, r=None), EINVAL, b"neither"), (dict(h=None, xn=None), EINVAL, b"no output"),
            (dict(y=None), EINVAL, b"need y"), (dict(codes=P), EINVAL, b"together"), (dict(ld_y=63), EINVAL, b"overlap"),
            (dict(ld_x=1), EINVAL, b"overlap"), (dict(codes=P, cs=P, ld_c=63), EINVAL, b"overlap"),
            (dict(h=P + 2), EINVAL, b"aligned")):
        refused(ffn, go(**kw), code, text)


def test_block_norm_bwd_refusals(ffn):
    L = ffn.lib()
    nb = L.ffn_b200_block_norm_bwd_ws_bytes(C.byref(desc(ffn)))
    assert nb > 0 and L.ffn_b200_block_norm_bwd_ws_bytes(C.byref(desc(ffn, rows=4000))) > nb

    def go(d=None, y=P, h=P, dh=P, dxn=P, dres=P, dy=P, post=None, gate=None, pre=None, ws=None, nws=0, ld=64):
        return L.ffn_b200_block_norm_bwd(C.byref(d or desc(ffn)), y, ld, h, ld, dh, ld, dxn, ld, dres, ld, dy, ld, post, gate,
                                         pre, ws, nws, None)
    for kw, code, text in (
            (dict(dh=None, dxn=None), EINVAL, b"neither"), (dict(h=None), EINVAL, b"needs h"),
            (dict(d=desc(ffn, pre=None)), EINVAL, b"pre_w"), (dict(dxn=None, pre=P), EINVAL, b"needs dxn"),
            (dict(d=desc(ffn, post=None), post=P), EINVAL, b"not there"), (dict(gate=P), EINVAL, b"not there"),
            (dict(y=None), EINVAL, b"need y"), (dict(ld=63), EINVAL, b"overlap"), (dict(dy=P + 1), EINVAL, b"aligned")):
        refused(ffn, go(**kw), code, text)


def test_python_wrappers_refuse_before_the_library(ffn):
    """Shapes, types and devices: FfnError, without a GPU."""
    import torch
    x, i8 = torch.zeros(4, 64), torch.zeros(4, 64, dtype=torch.int8)
    for call in (lambda: ffn.quantize_int8(x), lambda: ffn.moe_sort(torch.zeros(4, 2, dtype=torch.int32), 0, 8),
                 lambda: ffn.moe_permute(x, torch.zeros(4, 2, dtype=torch.int32)),
                 lambda: ffn.moe_combine(x, torch.zeros(2, 2, dtype=torch.int32)),
                 lambda: ffn.BlockNorm().forward(x), lambda: ffn.BlockNorm().forward(None),
                 lambda: ffn.BlockNorm().backward(x, x), lambda: ffn.Int8Matrix(i8, torch.ones(4)),
                 lambda: ffn.Int8Matrix(x, torch.ones(4))):
        with pytest.raises(ffn.FfnError):
            call()


def test_the_module_of_calls_is_built_and_leaves_what_it_does_not_take(ffn):
    """CPU tensors, wrong types and wrong counts: None, so that the Python path
    refuses them; the module holds the five calls of small kernels."""
    import torch
    ffn._setup()
    m = ffn._calls
    assert m is not None
    x, i32 = torch.zeros(4, 64), torch.zeros(4, 2, dtype=torch.int32)
    assert m.block_norm(None, None, 1.0, 1.0, 0.0, x, None, None) is None
    assert m.block_norm(None, None, 1.0, 1.0, 0.0, None, None, None) is None
    assert m.block_norm(None, None, "a", 1.0, 0.0, 3, None, None) is None
    assert m.int8_linear(x, 64, x, None, 1, 4, 64, x, None) is None
    assert m.moe_sort(i32, 0, 8) is None and m.moe_permute(x, i32, None) is None
    assert m.moe_combine(x, i32, None, None) is None
    with pytest.raises(TypeError):
        m.moe_sort(i32, 0)


def test_misaligned_side_arrays_are_refused(ffn):
    """Indices, offsets, weights, scales and parameter gradients of 4 bytes: a
    misaligned one is an error of the call, not of the GPU."""
    L, M = ffn.lib(), P + 2
    for at in (2, 5, 6, 7):
        a = [4, 2, P, 0, 8, P, P, P]
        a[at] = M
        refused(ffn, L.ffn_b200_moe_sort(*a, None), EINVAL, b"4-byte")
    for at in (5, 9, 10):
        a = [4, 2, 64, P, 64, P, 8, P, 64, P, P]
        a[at] = M
        refused(ffn, L.ffn_b200_moe_permute(*a, None), EINVAL, b"4-byte")
    for at in (7, 8):
        a = [4, 2, 16, 0, P, 16, 8, P, P, None, 0, P, 16]
        a[at] = M
        refused(ffn, L.ffn_b200_moe_combine(*a, None), EINVAL, b"4-byte")
    for at in (9, 10, 13):
        a = [4, 2, 16, 0, P, 16, P, 16, 8, P, P, P, 16, P]
        a[at] = M
        refused(ffn, L.ffn_b200_moe_combine_bwd(*a, None), EINVAL, b"4-byte")
    refused(ffn, product(ffn, offsets=M), EINVAL, b"aligned")
    refused(ffn, L.ffn_b200_quantize_int8(4, 64, 1, P, 64, 0, M, P, 64, P, None), EINVAL, b"aligned")
    refused(ffn, L.ffn_b200_block_norm(C.byref(desc(ffn)), P, 64, P, 64, P, 64, P, 64, P, 64, M, None), EINVAL, b"4-byte")
    d = desc(ffn, kind=1, gate=P)
    for at in (13, 14, 15):
        a = [C.byref(d), P, 64, P, 64, P, 64, P, 64, P, 64, P, 64, None, None, None]
        a[at] = M
        refused(ffn, L.ffn_b200_block_norm_bwd(*a, P, 1 << 30, None), EINVAL, b"4-byte")
