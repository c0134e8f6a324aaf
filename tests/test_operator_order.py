"""CPU tests: the order of what kernels and calls do where another order could
wait for good or race, read from the source or seen through stand-ins."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flash1017-engine_b200", "csrc")


def kernels(path):
    """(name, body) of each __global__ function of a source, comments taken out."""
    src = re.sub(r"//[^\n]*", "", open(path).read())
    for m in re.finditer(r"__global__[^;{]*?(\w+)\s*\(([^;{]*)\)\s*\{", src):
        depth, at = 1, m.end()
        while depth:
            depth += {"{": 1, "}": -1}.get(src[at], 0)
            at += 1
        yield m.group(1), src[m.end():at]


@pytest.mark.parametrize("source", ["int8_matmul.cu", "fp4_gemm.cu", "grouped_gemm.cu"])
def test_tensor_memory_is_taken_behind_the_wait_for_the_previous_kernel(source):
    """A kernel started early (programmatic dependent launch) that held tensor
    memory while it waits for the previous kernel could hold what a CTA of that
    kernel still waits for: both would wait for good.  So every kernel allocates
    only after pdl_enter()."""
    found = 0
    for name, body in kernels(os.path.join(CSRC, source)):
        allocs = [m.start() for m in re.finditer(r"tc::alloc\(|tcgen05\.alloc", body)]
        if allocs:
            found += 1
            assert 0 <= body.find("pdl_enter()") < allocs[0], name
    assert found == 1


def test_quantised_weights_are_copied_on_the_stream_of_the_call(ffn, monkeypatch):
    """Weights that are not contiguous are copied first.  The copy, the kernel
    that reads it and the copy's memory have to belong to one stream, the call's."""
    import contextlib
    now, seen = ["current"], []

    @contextlib.contextmanager
    def on(t, stream):
        now.append(stream)
        yield
        now.pop()

    class Weights:
        shape = (2, 40, 64)

        def dim(self):
            return 3

        def reshape(self, *shape):
            seen.append(("copied", now[-1]))
            return self

        def as_strided(self, *layout):
            return self

    class Matrix(ffn.Int8Matrix):
        def __init__(self, w, scale, bias=None):
            pass

    def kernel(x, stream=None):
        seen.append(("read", now[-1] if stream is None else stream))
        return x, None
    monkeypatch.setattr(ffn, "_on", on)
    monkeypatch.setattr(ffn, "_dev", lambda t, stream: 0 if stream is None else -1)
    monkeypatch.setattr(ffn, "quantize_int8", kernel)
    Matrix.quantize(Weights(), stream="side")
    assert seen == [("copied", "side"), ("read", "side")]
