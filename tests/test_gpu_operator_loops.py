"""Row operators in sizes that turn the loops of their kernels: more rows than are
resident at once, more channels than the grid's warps, a K in several pieces, tiles
of two blocks of channels, and K split over 2, 4 and 8 CTAs.  Formulas and
tolerances are those of the operators' own tests."""
import pytest
from test_gpu_block_norm import test_backward as check_backward
from test_gpu_block_norm import test_forward as check_forward
from test_gpu_int8 import U, product_ok

pytestmark = pytest.mark.gpu
TYPES = ["float32", "bfloat16", "float16"]


def codes64(torch, x):
    """scale = fl32(max / 127), code = rne(fl32(x / scale)): 64-bit quotients of f32
    values rounded to f32 are their f32 quotients."""
    x = x.double()
    s = (x.abs().amax(1) / 127).float()
    q = torch.round((x / torch.where(s > 0, s, 1).double()[:, None]).float()).clamp(-127, 127)
    q[s == 0] = 0
    return q.to(torch.int8), s


def rows_of(torch, cuda, g, rows, cols, dt):
    x = torch.randn(rows, cols, device=cuda, generator=g) * (0.01 + 8 * torch.rand(rows, 1, device=cuda, generator=g))
    if rows > 2:
        x[rows // 2] = 0
    return x.to(dt)


@pytest.mark.parametrize("rows,cols", [(2500, 1024), (2500, 4096), (2501, 4095), (2500, 8192), (1300, 8191), (700, 16384), (9000, 48)])
@pytest.mark.parametrize("dtype", TYPES)
def test_codes_of_many_rows(ffn, cuda, rows, cols, dtype):
    import torch
    g = torch.Generator(device=cuda).manual_seed(rows + cols)
    x = rows_of(torch, cuda, g, rows, cols, getattr(torch, dtype))
    q, s = ffn.quantize_int8(x)
    rq, rs = codes64(torch, x)
    assert torch.equal(s, rs) and torch.equal(q, rq)


@pytest.mark.parametrize("rows,cols", [(2500, 1024), (1500, 4096), (1000, 5000), (700, 8190), (1000, 16384), (400, 16383)])
@pytest.mark.parametrize("dtype", TYPES)
def test_swiglu_codes_of_many_rows(ffn, cuda, rows, cols, dtype):
    import torch
    g = torch.Generator(device=cuda).manual_seed(rows + cols)
    x = (torch.randn(rows, 2 * cols, device=cuda, generator=g) * 5).to(getattr(torch, dtype))
    q, s = ffn.quantize_int8(x, ffn.ACT_SWIGLU)
    for a in range(0, rows, 250):  # in parts, for the memory of the 64-bit values
        gate, up = x[a:a + 250, :cols].double(), x[a:a + 250, cols:].double()
        v = torch.clamp(gate / (1 + torch.exp(-gate)), max=10) * up.clamp(-10, 10)
        sd = s[a:a + 250].double()
        # expf within a step (2 U), a sum, a quotient within two (4 U), a product: 8 U
        assert ((sd - v.abs().amax(1) / 127).abs() <= sd * 10 * U).all()
        sd = sd[:, None]
        assert ((q[a:a + 250].double() * sd - v).abs() <= sd * (0.5 + 127 * 20 * U) + 10 * U * v.abs()).all()


def product_of(ffn, torch, cuda, rows, k, n, dtype, seed, floats=True):
    """A product of codes and, where `floats`, of the rows that they are made from."""
    dt = getattr(torch, dtype)
    g = torch.Generator(device=cuda).manual_seed(seed)
    w = torch.randint(-127, 128, (n, k), device=cuda, generator=g, dtype=torch.int8)
    ws = (0.5 + torch.rand(n, device=cuda, generator=g)) * 0.01
    bias = torch.randn(n, device=cuda, generator=g)
    m = ffn.Int8Matrix(w, ws, bias)
    if floats:
        x = rows_of(torch, cuda, g, rows, k, dt)
        q, s = codes64(torch, x)
    else:
        q = torch.randint(-127, 128, (rows, k), device=cuda, generator=g, dtype=torch.int8)
        s = 0.001 + 0.05 * torch.rand(rows, device=cuda, generator=g)
    wide = torch.full((rows + 1, n + 5), 7.0, dtype=dt, device=cuda)
    out = m.matmul((q, s), out=wide[:rows, :n])
    assert product_ok(torch, out, q, s, w, ws, bias)
    assert (wide[rows:] == 7).all() and (wide[:, n:] == 7).all()
    if floats:
        assert torch.equal(m.matmul(x), out)


# one and two rows: K in pieces of 4096, the last one ragged or not, and more
# channels than the grid has warps (9472 on 148 SMs)
@pytest.mark.parametrize("k,n", [(4099, 700), (5120, 300), (7168, 129), (8192, 64), (12289, 50), (16384, 33), (640, 12000),
                                 (5120, 12000), (4111, 20001)])
@pytest.mark.parametrize("rows", [1, 2])
@pytest.mark.parametrize("dtype", TYPES)
def test_products_of_one_and_two_rows(ffn, cuda, rows, k, n, dtype):
    import torch
    product_of(ffn, torch, cuda, rows, k, n, dtype, rows + k + n)


# K over 2, 4 and 8 CTAs (148 SMs), tiles of 16 to 128 tokens, whole and ragged K
SPLITS = [(96, 12000, 2048), (512, 8192, 640), (200, 40000, 2048), (96, 12011, 2048),
          (2, 5000, 2048), (17, 7168, 2048), (512, 7168, 129), (65, 12000, 2048), (256, 16384, 1000), (300, 12345, 1000), (511, 12000, 700),
          (256, 5000, 5), (300, 7168, 129), (300, 7169, 257), (512, 12000, 129), (200, 8192, 700), (512, 12000, 257), (3, 131072, 60)]


@pytest.mark.parametrize("rows,k,n", SPLITS)
@pytest.mark.parametrize("dtype", TYPES)
def test_products_with_k_over_a_cluster(ffn, cuda, rows, k, n, dtype):
    import torch
    product_of(ffn, torch, cuda, rows, k, n, dtype, rows + k + n, floats=k <= 16384)


# one matrix in tiles of two blocks of channels and 128 to 256 tokens, up to two waves
WIDE = [(1025, 512, 4096), (1000, 512, 5120), (1500, 512, 4096), (1500, 1000, 4999), (3000, 512, 2304), (1500, 512, 5120),
        (2048, 520, 4096), (4096, 512, 2304), (3000, 1040, 4096), (4099, 2048, 4096)]


@pytest.mark.parametrize("rows,k,n", WIDE)
@pytest.mark.parametrize("dtype", TYPES)
def test_products_in_wide_tiles(ffn, cuda, rows, k, n, dtype):
    import torch
    product_of(ffn, torch, cuda, rows, k, n, dtype, rows + k + n)


@pytest.mark.parametrize("rows,cols", [(1500, 4096), (900, 6000), (700, 8192), (500, 16384), (1501, 4095), (333, 16383), (4000, 512)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gate,post", [("token", True), ("channel", True), ("none", False)])
def test_norms_of_many_rows(ffn, cuda, rows, cols, dtype, gate, post):
    check_forward(ffn, cuda, rows, cols, dtype, gate, post, True)


@pytest.mark.parametrize("rows,cols", [(1500, 4096), (500, 8192), (400, 16384), (901, 4095), (333, 16383)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gate,post", [("token", True), ("channel", True), ("none", False)])
def test_norm_gradients_of_many_rows(ffn, cuda, rows, cols, dtype, gate, post):
    check_backward(ffn, cuda, rows, cols, dtype, gate, post)


@pytest.mark.parametrize("rows,cols", [(1500, 4096), (400, 16384)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_codes_of_many_norms(ffn, cuda, rows, cols, dtype):
    """The norm's own codes are quantize_int8's of its f32 values."""
    import torch
    g = torch.Generator(device=cuda).manual_seed(rows + cols)
    dt = getattr(torch, dtype)
    x, y = rows_of(torch, cuda, g, rows, cols, dt), rows_of(torch, cuda, g, rows, cols, dt)
    w = 1 + 0.2 * torch.randn(cols, device=cuda, generator=g)
    norm = ffn.BlockNorm(w, w)
    xn = torch.empty_like(x)
    _, _, q, s = norm.forward(y, x, xn=xn, codes=True)
    if dt == torch.float32:
        rq, rs = codes64(torch, xn)
        assert torch.equal(s, rs) and torch.equal(q, rq)
    else:  # half a code, and half a bf16 step of xn
        d = (q.double() * s.double()[:, None] - xn.double()).abs()
        assert (d <= s.double()[:, None] * 0.5 * (1 + 1e-5) + 2.0 ** -8 * xn.double().abs() + 1e-30).all()
