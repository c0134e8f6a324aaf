"""Row operators on several streams: products whose CTAs share an SM, and copies
that belong to the call's stream."""
import pytest

pytestmark = pytest.mark.gpu


def test_products_of_short_k_behind_each_other_on_several_streams(ffn, cuda):
    """Several matrices behind one another from the same codes, on four streams
    at once.  With a K of 256 two CTAs have room on an SM in shared memory, but
    one fills its tensor memory, so the CTAs of one stream's products wait for
    those of another's, and each product starts before the one in front of it is
    done.  Sums are whole numbers, so the 64-bit product is met exactly where the
    scales are powers of two."""
    import torch
    g = torch.Generator(device=cuda).manual_seed(11)

    def codes(*s):
        return torch.randint(-127, 128, s, device=cuda, generator=g, dtype=torch.int8)
    k = 256
    xs = [codes(rows, k) for rows in (2048, 8192, 512, 2048)]  # tiles of 240, 256 and 128 tokens
    ws = [codes(n, k) for n in (4096, 2048, 4096)]
    mats = [ffn.Int8Matrix(w, torch.full((w.shape[0],), 0.5, device=cuda)) for w in ws]
    ones = [torch.full((x.shape[0],), 2.0, device=cuda) for x in xs]
    want = [[x.double() @ w.double().t() for w in ws] for x in xs]
    outs = [[torch.full((x.shape[0], w.shape[0]), -1.0, device=cuda) for w in ws] for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                for m, out in zip(mats, outs[i]):
                    m.matmul((xs[i], ones[i]), out=out)
    torch.cuda.synchronize()
    for got, ref in zip(outs, want):
        for a, b in zip(got, ref):
            assert torch.equal(a.double(), b)


def test_weights_quantised_on_a_stream_of_their_own(ffn, cuda):
    """Transposed weights, which are copied first, on a side stream, while the
    current stream is busy and takes new memory at once: the bits of a call alone."""
    import torch
    g = torch.Generator(device=cuda).manual_seed(12)
    w = torch.randn(6, 1024, 520, device=cuda, generator=g).transpose(1, 2)
    bias = torch.randn(6, 520, device=cuda, generator=g)
    want = ffn.Int8Matrix.quantize(w.contiguous(), bias)
    busy = torch.randn(4096, 4096, device=cuda, generator=g)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(4):
        for _ in range(4):
            busy = busy @ busy * 1e-3
        got = ffn.Int8Matrix.quantize(w, bias, stream=side)
        spoil = torch.full((6, 520, 1024), float("nan"), device=cuda)
        side.synchronize()
        assert torch.equal(got.w, want.w) and torch.equal(got.scale, want.scale) and got.bias is bias
        del spoil
    torch.cuda.synchronize()
