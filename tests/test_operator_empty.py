"""CPU tests: calls over nothing.  An empty tensor's address is null, which is no
error where nothing is read or written there."""
import ctypes as C

OK, EINVAL = 0, -1
P = 4096  # a fake, well-aligned device address


def desc(ffn, rows, kind, gate):
    return ffn.BlockNormDesc(rows, 64, 0, kind, P, gate, P, 1.0, 1.0, 1e-6, 0)


def test_norms_of_no_rows_with_a_gate_for_each(ffn):
    L = ffn.lib()
    d = desc(ffn, 0, ffn.GATE_TOKEN, None)
    assert L.ffn_b200_block_norm(C.byref(d), None, 64, None, 64, None, 64, None, 64, None, 0, None, None) == OK
    assert L.ffn_b200_block_norm_bwd(C.byref(d), None, 64, None, 64, None, 64, None, 64, None, 64, None, 64, None, None, None,
                                     None, 0, None) == OK
    # with rows, or a gate for each channel, it has to be there
    for bad in (desc(ffn, 4, ffn.GATE_TOKEN, None), desc(ffn, 0, ffn.GATE_CHANNEL, None), desc(ffn, 0, ffn.GATE_NONE, P)):
        assert L.ffn_b200_block_norm(C.byref(bad), P, 64, P, 64, P, 64, P, 64, None, 0, None, None) == EINVAL


def test_rows_sent_to_no_rows(ffn):
    L = ffn.lib()
    assert L.ffn_b200_moe_permute(4, 2, 64, P, 64, P, 0, None, 64, None, None, None) == OK
    assert L.ffn_b200_moe_permute(4, 2, 64, P, 64, P, 0, None, 64, P, None, None) == OK
    assert L.ffn_b200_moe_permute(4, 2, 64, P, 64, P, 1, None, 64, None, None, None) == EINVAL
