"""GPU: the 8-bit linear layer against its definition in 64 bits (oracle/fp8.py, numpy and torch float64).

Tolerances, all from arithmetic (u = 2^-24, half a step of fp32; h(t) = eps/2, half a step of the output's type):
  quantize   bit for bit: v * 2^-e is exact, so one rounding decides, the same one
  rstd       the sum of squares adds at most 100 terms one after the other on any path: relative error < 100 u
  norm       y carries rstd's error and two products': < 104 u; its 8-bit form may be half an e4m3 step off
             (2^-4 of the value, 2^-10 of the scale below e4m3's normal numbers), and a scale one power of two off
             only where the block's largest value is within 104 u of the border
  backward   sums as above: 104 u of the sum of magnitudes, and one rounding to the output's type; dweight adds
             rows/148 terms in one thread, and 37 + 5 partial sums
  products   fp32 accumulation in any order: k u of the sum of magnitudes, and one rounding
"""
import itertools

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from oracle import fp8  # noqa: E402

U = 2.0 ** -24
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
HALF = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: 2.0 ** -24}
TINY = {F16: 2.0 ** -25, BF16: 2.0 ** -134, F32: 2.0 ** -150}  # half a step below the smallest normal number


@pytest.fixture(scope="module")
def vk():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import vibekernel_b200 as vkm
    return vkm


@pytest.fixture(autouse=True)
def no_device_error(vk):
    yield
    torch.cuda.synchronize()
    assert vk.device_error(0) == 0


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _rand(shape, dtype, seed, std=1.0):
    return (torch.randn(*shape, generator=_gen(seed), device="cuda") * std).to(dtype)


def _bytes(t):
    return t.contiguous().view(torch.uint8).cpu().numpy()


def _inside(shape, dtype, lead, tail, fill=0x55):
    """A [rows, cols] view that starts `lead` elements into its rows, with `tail` more behind; all filled with `fill`."""
    size = torch.empty((), dtype=dtype).element_size()
    room = torch.full((shape[0] + 2, (lead + shape[1] + tail) * size), fill, dtype=torch.uint8, device="cuda").view(dtype)
    return room[1:-1, lead:lead + shape[1]], room


def _untouched(room, view_shape, lead, fill=0x55):
    b = room.view(torch.uint8).reshape(room.shape[0], room.shape[1], -1)
    rows, cols = view_shape
    assert (b[0] == fill).all() and (b[-1] == fill).all()
    assert (b[:, :lead] == fill).all() and (b[:, lead + cols:] == fill).all()


def _deq(q, s, tile=False):
    """Values in float64 on the GPU."""
    w = torch.from_numpy(fp8.E4M3).cuda()[q.contiguous().view(torch.uint8).long()]
    e = torch.from_numpy(fp8.E8M0).cuda()[s.contiguous().view(torch.uint8).long()]
    e = e.repeat_interleave(128, 0)[: q.shape[0]] if tile else e
    return w * e.repeat_interleave(128, 1)[:, : q.shape[1]]


def _quantized(shape, seed, tile=False, std=1.0, pad=True):
    """An 8-bit operand made by the oracle's own rounding (rows padded to 16 bytes, or dense)."""
    v = np.random.default_rng(seed).standard_normal(shape) * std
    v *= np.exp(np.random.default_rng(seed + 1).standard_normal((1, shape[1])))
    codes, s = fp8.quantize(v.astype(np.float32), tile)
    q, _ = _inside(shape, torch.float8_e4m3fn, 0, -shape[1] % 16 if pad else 0, 0x7f)  # NaN around it
    q.copy_(torch.from_numpy(codes).cuda().view(torch.float8_e4m3fn))
    return q, torch.from_numpy(s).cuda().view(torch.float8_e8m0fnu)


# ------------------------------------------------------------------------------------------ quantize
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("tile", [False, True])
@pytest.mark.parametrize("shape", [(1, 1), (1, 4096), (3, 127), (129, 128), (128, 129), (300, 1000), (7, 3000), (1000, 64), (0, 5)])
def test_quantize_bitwise(vk, shape, tile, dtype):
    x = _rand(shape, dtype, 1)
    if shape[0] > 1:
        x[1] *= 1e-4
        x[shape[0] // 2, ::3] = 0
    q, s = vk.quantize_fp8(x, tile=tile)
    codes, scale = fp8.quantize(x.double().cpu().numpy(), tile)
    assert q.dtype == torch.float8_e4m3fn and s.dtype == torch.float8_e8m0fnu
    np.testing.assert_array_equal(_bytes(s), scale)
    np.testing.assert_array_equal(_bytes(q), codes)


@pytest.mark.parametrize("tile", [False, True])
def test_quantize_special_values(vk, tile):
    """Zeros, subnormal and huge values, values on a scale's border, infinities and NaN, each in a block of its own."""
    x = torch.zeros(256, 128 * 9)
    x[0, 5] = 1e-44
    x[0, 128:256] = torch.finfo(F32).max
    x[0, 256] = 448.0
    x[0, 384] = float(np.nextafter(np.float32(448.0), np.float32(500)))
    x[0, 512] = float("inf")
    x[0, 640] = float("nan")
    x[0, 768:896] = torch.linspace(-2.0 ** -130, 2.0 ** -127, 128)
    x[0, 896:1024] = torch.linspace(-1, 1, 128) * 2.0 ** -9
    q, s = vk.quantize_fp8(x.cuda(), tile=tile)
    codes, scale = fp8.quantize(x.double().numpy(), tile)
    np.testing.assert_array_equal(_bytes(s), scale)
    np.testing.assert_array_equal(_bytes(q), codes)
    assert scale[0, 4] == 255 and scale[0, 5] == 255 and scale[0, 8] == 127


@pytest.mark.parametrize("tile", [False, True])
@pytest.mark.parametrize("lead,tail", [(0, 0), (1, 0), (8, 8), (3, 6)])
def test_quantize_strides_and_surroundings(vk, tile, lead, tail):
    shape = (150, 333)
    x, _ = _inside(shape, BF16, lead, tail, 0x7f)
    x.copy_(_rand(shape, BF16, 2))
    q, qroom = _inside(shape, torch.float8_e4m3fn, lead, tail)
    s_shape = (2 if tile else 150, 3)
    s, sroom = _inside(s_shape, torch.float8_e8m0fnu, lead, tail)
    vk.quantize_fp8(x, tile=tile, q=q, scale=s)
    codes, scale = fp8.quantize(x.double().cpu().numpy(), tile)
    np.testing.assert_array_equal(_bytes(q), codes)
    np.testing.assert_array_equal(_bytes(s), scale)
    _untouched(qroom, shape, lead)
    _untouched(sroom, s_shape, lead)


# ------------------------------------------------------------------------------------------ norm
def _check_norm(x, w, residual, eps, q, s, h, rstd):
    want_h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    assert torch.equal(h, want_h)
    h64 = want_h.double()
    r64 = (h64.square().mean(dim=1) + eps).rsqrt()
    assert ((rstd.double() - r64).abs() <= 100 * U * r64).all()
    y = h64 * r64[:, None] * w.double()
    yn = y.cpu().numpy()
    top = fp8.tops(yn, False)
    scale = fp8.E8M0[_bytes(s)]
    near = 104 * U
    some = top > 0
    assert (scale[~some] == 1).all()
    assert (top[some] * (1 - near) <= 448 * scale[some]).all()
    assert ((top[some] * (1 + near) > 224 * scale[some]) | (scale[some] == 2.0 ** -127)).all()
    deq = _deq(q, s).cpu().numpy()
    per = fp8.spread(scale, yn.shape, False)
    assert (np.abs(deq - yn) <= np.maximum(2.0 ** -4 * np.abs(yn), 2.0 ** -10 * per) * (1 + 2.0 ** -12) + near * np.abs(yn)).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("shape", [(1, 1), (1, 4096), (2, 127), (5, 128), (33, 1000), (9, 2048), (4, 2056), (3, 4100), (6, 8192),
                                   (3, 8200), (2, 20001), (1000, 64)])
def test_norm(vk, shape, with_residual, dtype):
    x, w = _rand(shape, dtype, 3, 2.0), _rand((shape[1],), dtype, 4)
    r = _rand(shape, dtype, 5, 3.0) if with_residual else None
    out = vk.rmsnorm_fp8(x, w, residual=r, eps=1e-5)
    _check_norm(x, w, r, 1e-5, *out)


@pytest.mark.parametrize("cols", [333, 4096, 9000])
@pytest.mark.parametrize("lead,tail", [(1, 2), (8, 8)])
def test_norm_strides_and_surroundings(vk, cols, lead, tail):
    shape = (5, cols)
    x, _ = _inside(shape, BF16, lead, tail, 0x7f)
    r, _ = _inside(shape, BF16, lead, tail, 0x7f)
    x.copy_(_rand(shape, BF16, 6))
    r.copy_(_rand(shape, BF16, 7))
    h, hroom = _inside(shape, BF16, lead, tail)
    q, qroom = _inside(shape, torch.float8_e4m3fn, lead, tail)
    s_shape = (5, (cols + 127) // 128)
    s, sroom = _inside(s_shape, torch.float8_e8m0fnu, lead, tail)
    w = _rand((cols + 1,), BF16, 8)[1:]
    out = vk.rmsnorm_fp8(x, w, residual=r, q=q, scale=s, h=h)
    _check_norm(x, w, r, 1e-6, *out)
    for room, sh in ((hroom, shape), (qroom, shape), (sroom, s_shape)):
        _untouched(room, sh, lead)


@pytest.mark.parametrize("cols", [1000, 1001, 4096, 8191, 9001])
def test_norm_in_place(vk, cols):
    x, r, w = _rand((7, cols), F16, 9), _rand((7, cols), F16, 10), _rand((cols,), F16, 11)
    want = vk.rmsnorm_fp8(x, w, residual=r)
    for which in (0, 1):
        a, b = x.clone(), r.clone()
        got = vk.rmsnorm_fp8(a, w, residual=b, h=(a, b)[which])
        assert got[2] is (a, b)[which]
        for g, e in zip(got, want):
            assert torch.equal(g.view(torch.uint8), e.view(torch.uint8))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("cols,pitch", [(8320, 8320), (16376, 16380), (16384, 16384), (16385, 16385), (16392, 16400), (16392, 16397), (24576, 24576)])
def test_norm_of_long_rows(vk, cols, pitch, dtype):
    """Where a row stops fitting its threads' registers; `h` in x's place."""
    w, r = _rand((cols,), dtype, 13), _rand((3, cols), dtype, 14)
    x = _rand((3, pitch), dtype, 15)[:, :cols]
    want = x.clone()
    q, s, h, rstd = vk.rmsnorm_fp8(x, w, residual=r, h=x)
    assert h is x
    _check_norm(want, w, r, 1e-6, q, s, h, rstd)
    _check_norm(want, w, None, 1e-6, *vk.rmsnorm_fp8(want, w))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_norm_adds_over_the_whole_range(vk, dtype):
    """h is the fp32 sum rounded once (the sum of two 16-bit numbers is exact in fp32, or too lopsided for the rounding to
    matter): subnormal numbers, signed zeros, cancellation, ties, sums that overflow."""
    gen = _gen(16)
    bits = torch.randint(0, 1 << 16, (2, 64, 1024), generator=gen, device="cuda", dtype=torch.int32).to(torch.int16).view(dtype)
    x, r = torch.where(bits.float().isfinite(), bits, torch.zeros_like(bits))
    r[32:] = -x[32:] * (1 + torch.randint(0, 3, (32, 1024), generator=gen, device="cuda") * torch.finfo(dtype).eps).to(dtype)
    r[~r.float().isfinite()] = 0
    x[0, :4] = torch.tensor([0.0, -0.0, 0.0, -0.0], dtype=dtype)
    r[0, :4] = torch.tensor([0.0, -0.0, -0.0, 0.0], dtype=dtype)
    h = vk.rmsnorm_fp8(x, torch.ones(1024, dtype=dtype, device="cuda"), residual=r)[2]
    assert torch.equal(h.view(torch.int16), (x.float() + r.float()).to(dtype).view(torch.int16))


def test_norm_rows_of_zeros_and_non_finite_rows(vk):
    x = _rand((4, 512), BF16, 12)
    x[1] = 0
    x[2, 300] = float("inf")
    x[3, 10] = float("nan")
    q, s, h, rstd = vk.rmsnorm_fp8(x, torch.ones(512, dtype=BF16, device="cuda"), eps=1e-6)
    assert (_bytes(q)[1] & 127 == 0).all() and (_bytes(s)[1] == 127).all() and abs(rstd[1].item() - 1e3) < 1e3 * 100 * U
    # an infinity: rstd is 0 and 0 * inf is NaN in its block, 0 in the others
    assert rstd[2].item() == 0 and _bytes(s)[2].tolist() == [127, 127, 255, 127]
    assert np.isnan(rstd[3].item()) and (_bytes(s)[3] == 255).all() and (_bytes(q)[3] & 127 == 127).all()
    clean = vk.rmsnorm_fp8(x[:1], torch.ones(512, dtype=BF16, device="cuda"), eps=1e-6)
    assert torch.equal(q[:1].view(torch.uint8), clean[0].view(torch.uint8))


def _check_norm_back(dy, h, w, rstd, dres, dx, dw):
    n, rows = dy.shape[1], dy.shape[0]
    a, b, g64, r = dy.double(), h.double(), w.double(), rstd.double()[:, None]
    g, xhat = a * g64, b * r
    mean = (g * xhat).mean(dim=1, keepdim=True)
    want = r * (g - xhat * mean)
    size = r * (g.abs() + xhat.abs() * (g * xhat).abs().mean(dim=1, keepdim=True))
    if dres is not None:
        want, size = want + dres.double(), size + dres.double().abs()
    tol = 104 * U * size + HALF[dy.dtype] * (1 + 2.0 ** -8) * want.abs() + TINY[dy.dtype]
    assert ((dx.double() - want).abs() <= tol).all()
    wsize = (a * xhat).abs().sum(dim=0)
    depth = -(-rows // 148) + 37 + 5 + 4
    assert ((dw.double() - (a * xhat).sum(dim=0)).abs() <= depth * U * wsize).all()
    assert dw.dtype == F32 and dx.dtype == dy.dtype and n == dw.shape[0]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("with_res", [False, True])
@pytest.mark.parametrize("shape", [(1, 1), (1, 4096), (2, 127), (300, 128), (777, 1000), (297, 2048), (5, 2056), (400, 4096),
                                   (6, 8192), (3, 8200), (600, 8193), (2, 20001)])
def test_norm_backward(vk, shape, with_res, dtype):
    dy, h, w = _rand(shape, dtype, 13, 0.1), _rand(shape, dtype, 14, 2.0), _rand((shape[1],), dtype, 15)
    rstd = (h.float().square().mean(dim=1) + 1e-6).rsqrt()
    dres = _rand(shape, dtype, 16, 0.1) if with_res else None
    dx, dw = vk.rmsnorm_fp8_backward(dy, h, w, rstd, dres=dres)
    _check_norm_back(dy, h, w, rstd, dres, dx, dw)


@pytest.mark.parametrize("cols", [333, 4096, 9000])
def test_norm_backward_strides_in_place_and_surroundings(vk, cols):
    shape = (310, cols)
    rstd = torch.rand(310, generator=_gen(17), device="cuda") + 0.5
    w = _rand((cols + 1,), F16, 18)[1:]
    mats = []
    for i in range(3):
        m, _ = _inside(shape, F16, 1, 2, 0x7f)
        m.copy_(_rand(shape, F16, 19 + i))
        mats.append(m)
    dy, h, dres = mats
    dx, room = _inside(shape, F16, 1, 2)
    dx, dw = vk.rmsnorm_fp8_backward(dy, h, w, rstd, dres=dres, dx=dx)
    _check_norm_back(dy, h, w, rstd, dres, dx, dw)
    _untouched(room, shape, 1)
    for which in (0, 2):
        copies = [m.clone() for m in mats]
        got, dw2 = vk.rmsnorm_fp8_backward(copies[0], copies[1], w, rstd, dres=copies[2], dx=copies[which])
        assert torch.equal(got, dx) and torch.equal(dw2, dw)


def test_norm_backward_of_no_rows(vk):
    e = torch.empty((0, 256), dtype=BF16, device="cuda")
    dw = torch.full((256,), 7.0, device="cuda")
    dx, dw = vk.rmsnorm_fp8_backward(e, e, torch.ones(256, dtype=BF16, device="cuda"), torch.empty(0, device="cuda"), dweight=dw)
    assert dx.shape == (0, 256) and (dw == 0).all()


def test_norm_backward_against_differences(vk):
    """dx and dweight against central differences of the norm in 64 bits."""
    shape = (3, 40)
    dy, h, w = _rand(shape, BF16, 23), _rand(shape, BF16, 24), _rand((40,), BF16, 25)
    rstd = (h.double().square().mean(dim=1) + 1e-6).rsqrt().float()
    dx, dw = vk.rmsnorm_fp8_backward(dy, h, w, rstd)

    def loss(hh, ww):
        return (dy.double() * hh * (hh.square().mean(dim=1, keepdim=True) + 1e-6).rsqrt() * ww).sum()

    step = 1e-5
    h64, w64 = h.double(), w.double()
    for r, c in itertools.product(range(3), (0, 17, 39)):
        d = torch.zeros_like(h64)
        d[r, c] = step
        diff = (loss(h64 + d, w64) - loss(h64 - d, w64)) / (2 * step)
        assert abs(diff - dx[r, c].double()) <= HALF[BF16] * abs(diff) + 1e-6
    for c in (0, 17, 39):
        d = torch.zeros_like(w64)
        d[c] = step
        diff = (loss(h64, w64 + d) - loss(h64, w64 - d)) / (2 * step)
        assert abs(diff - dw[c].double()) <= 1e-5


# ------------------------------------------------------------------------------------------ products
def _check_product(got, want, size, k, base=None):
    t = got.dtype
    if base is not None:
        want, size = want + base.double(), size + base.double().abs()
    tol = max(k, 1) * U * size + HALF[t] * (1 + 2.0 ** -8) * want.abs() + TINY[t]
    assert got.shape == want.shape
    assert ((got.double() - want).abs() <= tol).all()


SHAPES = [(1, 1, 1), (1, 128, 128), (1, 4096, 512), (3, 130, 129), (8, 1000, 4096), (16, 256, 3000), (17, 136, 200), (33, 520, 640),
          (64, 300, 1032), (65, 264, 130), (128, 128, 1), (129, 257, 384), (200, 136, 72), (256, 256, 512), (300, 520, 1000),
          (513, 1025, 2049), (1024, 768, 3000)]


@pytest.mark.parametrize("out", [F16, BF16, F32])
@pytest.mark.parametrize("layout", ["nt_tile", "nt_row", "nn"])
@pytest.mark.parametrize("shape", SHAPES)
def test_gemm(vk, shape, layout, out):
    m, n, k = shape
    tile, trans = layout != "nt_row", layout != "nn"
    a, sa = _quantized((m, k), 30)
    b, sb = _quantized((n, k) if trans else (k, n), 31, tile, 0.05)
    c = vk.gemm_fp8(a, sa, b, sb, trans_b=trans, out_dtype=out)
    av, bv = _deq(a, sa), _deq(b, sb, tile)
    bv = bv.t() if trans else bv
    _check_product(c, av @ bv, av.abs() @ bv.abs(), k)


# more tiles than the GPU has pairs of SMs: whole tiles only (6 x 13 = 78: halves of 4), a half-full wave (10 x 11: 36 halved),
# most of a wave (12 x 12), a second wave of one tile (15 x 5), each with ragged edges
@pytest.mark.parametrize("shape", [(1400, 3300, 300), (2500, 2700, 600), (3000, 2900, 1200), (3800, 1100, 2100)])
@pytest.mark.parametrize("layout", ["nt_tile", "nt_row", "nn"])
def test_gemm_waves(vk, shape, layout):
    test_gemm(vk, shape, layout, BF16)


# few rows of A: clusters of every size, more tiles than SMs, more k than fits in flight
@pytest.mark.parametrize("shape", [(1, 500, 4096), (16, 1500, 1600), (17, 2000, 5000), (40, 3000, 1000), (5, 4096, 4096), (64, 20000, 300), (100, 1000, 3000), (128, 700, 4096),
                                   (2, 300, 20000)])
@pytest.mark.parametrize("layout", ["nt_tile", "nt_row"])
def test_gemm_few_rows(vk, shape, layout):
    test_gemm(vk, shape, layout, F16)
    test_gemm(vk, shape, layout, F32)


# few tiles and a long sum: two, three and four pairs to a tile
@pytest.mark.parametrize("shape", [(300, 520, 6000), (1000, 1200, 7000), (1024, 1900, 9000), (257, 1001, 8192), (130, 100, 20000)])
@pytest.mark.parametrize("layout", ["nt_tile", "nt_row", "nn"])
@pytest.mark.parametrize("out", [F16, F32])
def test_gemm_shared_tiles(vk, shape, layout, out):
    test_gemm(vk, shape, layout, out)


@pytest.mark.parametrize("m", [5, 300])
@pytest.mark.parametrize("k", [100, 500, 700, 1100, 1700, 2100, 8000])
@pytest.mark.parametrize("lead,tail", [(0, 0), (0, 1), (1, 0), (2, 1), (3, 2), (1, 3), (4, 4)])
def test_gemm_scales_anywhere(vk, lead, tail, k, m):
    """Rows of scales at any byte of a larger matrix of NaN scales: the same bits as packed ones."""
    n = 200
    a, sa = _quantized((m, k), 46)
    b, sb = _quantized((n, k), 47)
    want = vk.gemm_fp8(a, sa, b, sb, trans_b=True, out_dtype=F32)
    for tile in (False, True):
        if tile:
            b, sb = _quantized((n, k), 47, True)
            want = vk.gemm_fp8(a, sa, b, sb, trans_b=True, out_dtype=F32)
        moved = []
        for sc in (sa, sb):
            view, _ = _inside(tuple(sc.shape), torch.float8_e8m0fnu, lead, tail, 0xff)
            view.view(torch.uint8).copy_(sc.view(torch.uint8))
            moved.append(view)
        got = vk.gemm_fp8(a, moved[0], b, moved[1], trans_b=True, out_dtype=F32)
        assert torch.equal(got, want)


@pytest.mark.parametrize("m", [4, 200])
def test_gemm_tile_scales_of_a(vk, m):
    a, sa = _quantized((m, 1000), 32, True)
    b, sb = _quantized((300, 1000), 33, True)
    c = vk.gemm_fp8(a, sa, b, sb, trans_b=True, out_dtype=F32)
    av, bv = _deq(a, sa, True), _deq(b, sb, True).t()
    _check_product(c, av @ bv, av.abs() @ bv.abs(), 1000)


@pytest.mark.parametrize("layout", ["nt", "nn"])
@pytest.mark.parametrize("m", [5, 150])
@pytest.mark.parametrize("lead,tail", [(1, 2), (16, 16), (0, 3)])
def test_gemm_strides_and_surroundings(vk, m, lead, tail, layout):
    """Views inside larger NaN-filled matrices: aligned ones and ones that the tensor-core loads cannot take."""
    n, k = 264, 333
    trans = layout == "nt"
    a0, sa0 = _quantized((m, k), 34)
    b0, sb0 = _quantized((n, k) if trans else (k, n), 35, True)

    def placed(t, dtype, fill):
        v, _ = _inside(tuple(t.shape), dtype, lead, tail + (-(lead + t.shape[1] + tail) % 16 if lead % 16 == 0 and tail != 3 else 0), fill)
        return v.copy_(t)

    a, b = placed(a0, torch.float8_e4m3fn, 0x7f), placed(b0, torch.float8_e4m3fn, 0x7f)
    sa, sb = placed(sa0, torch.float8_e8m0fnu, 0xff), placed(sb0, torch.float8_e8m0fnu, 0xff)
    c, room = _inside((m, n), BF16, lead, tail)
    vk.gemm_fp8(a, sa, b, sb, c, trans_b=trans)
    av, bv = _deq(a, sa), _deq(b, sb, True)
    bv = bv.t() if trans else bv
    _check_product(c, av @ bv, av.abs() @ bv.abs(), k)
    _untouched(room, (m, n), lead)


@pytest.mark.parametrize("m", [2, 300])
def test_gemm_of_nothing(vk, m):
    a = torch.empty((m, 0), dtype=torch.float8_e4m3fn, device="cuda")
    b = torch.empty((40, 0), dtype=torch.float8_e4m3fn, device="cuda")
    sa, sb = torch.empty((m, 0), dtype=torch.float8_e8m0fnu, device="cuda"), torch.empty((1, 0), dtype=torch.float8_e8m0fnu, device="cuda")
    c = torch.full((m, 40), 3.0, dtype=F16, device="cuda")
    assert (vk.gemm_fp8(a, sa, b, sb, c, trans_b=True) == 0).all()


@pytest.mark.parametrize("m", [2, 300])
def test_gemm_nan_block_stays_in_its_row(vk, m):
    """A NaN scale makes the whole row of C NaN and nothing else; scales at both ends of their range are exact."""
    a, sa = _quantized((m, 512), 36)
    b, sb = _quantized((256, 512), 37, True)
    raw = sa.view(torch.uint8)
    raw[1, 2] = 255
    raw[0, :] = 127 - 100
    sb.view(torch.uint8)[:] = 127 + 60
    c = vk.gemm_fp8(a, sa, b, sb, trans_b=True, out_dtype=F32)
    assert c[1].isnan().all() and not c[[0, *range(2, m)]].isnan().any()
    av, bv = _deq(a, sa), _deq(b, sb, True).t()
    keep = [0, *range(2, m)]
    _check_product(c[keep], av[keep] @ bv, av[keep].abs() @ bv.abs(), 512)


def test_gemm_refusals(vk):
    a, sa = _quantized((8, 256), 38)
    b, sb = _quantized((256, 256), 39)
    with pytest.raises(vk.VkError, match="tile scales"):
        vk.gemm_fp8(a, sa, b, sb)
    with pytest.raises(ValueError, match="b_scale"):
        vk.gemm_fp8(a, sa, b, sb[:5], trans_b=True)
    with pytest.raises(ValueError, match="trans_b"):
        vk.gemm_fp8(a, sa, b[:, :128], sb[:, :1], trans_b=True)
    with pytest.raises(TypeError):
        vk.gemm_fp8(a.view(torch.uint8), sa, b, sb, trans_b=True)
    with pytest.raises(ValueError, match="overlapping"):
        vk.gemm_fp8(a[:1].expand(8, 256), sa, b, sb, trans_b=True)
    with pytest.raises(ValueError, match="unit column stride"):
        vk.gemm_fp8(a, sa, b.t(), sb, trans_b=True)
    with pytest.raises(TypeError):
        vk.gemm_fp8(a, sa, b, sb, trans_b=True, out_dtype=torch.int8)


WG_SHAPES = [(1, 1, 1), (1, 128, 128), (5, 8, 40), (64, 128, 128), (100, 136, 129), (300, 264, 200), (128, 512, 640), (777, 256, 300),
             (2000, 128, 256), (5000, 200, 136), (1000, 520, 1032)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("out", [None, F32])
@pytest.mark.parametrize("shape", WG_SHAPES)
def test_wgrad(vk, shape, dtype, out):
    t, n, k = shape
    dy = _rand((t, n), dtype, 40, 0.1)
    x, sx = _quantized((t, k), 41)
    dw = vk.wgrad_fp8(dy, x, sx, out_dtype=out)
    assert dw.dtype == (out or dtype)
    d, xv = dy.double().t(), _deq(x, sx)
    _check_product(dw, d @ xv, d.abs() @ xv.abs(), t)
    base = _rand((n, k), out or dtype, 42)
    acc = vk.wgrad_fp8(dy, x, sx, base.clone(), accumulate=True)
    _check_product(acc, d @ xv, d.abs() @ xv.abs(), t, base)


@pytest.mark.parametrize("shape", [(300, 1400, 3300), (600, 2504, 2700), (1200, 3000, 2900), (1100, 3800, 1100)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_wgrad_waves(vk, shape, dtype):
    test_wgrad(vk, shape, dtype, None)


@pytest.mark.parametrize("shape", [(3000, 300, 520), (4001, 1000, 1000), (5000, 1024, 1900), (12000, 64, 100)])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("out", [None, F32])
def test_wgrad_shared_tiles(vk, shape, dtype, out):
    test_wgrad(vk, shape, dtype, out)


@pytest.mark.parametrize("lead,tail", [(1, 2), (16, 16)])
def test_wgrad_strides_and_surroundings(vk, lead, tail):
    t, n, k = 333, 264, 200
    dy, _ = _inside((t, n), BF16, lead, tail + (-(lead + n + tail) % 8 if lead == 16 else 0), 0x7f)
    dy.copy_(_rand((t, n), BF16, 43))
    x0, s0 = _quantized((t, k), 44)
    x, _ = _inside((t, k), torch.float8_e4m3fn, lead, tail + (-(lead + k + tail) % 16 if lead == 16 else 0), 0x7f)
    s, _ = _inside((t, 2), torch.float8_e8m0fnu, lead, tail, 0xff)
    x.copy_(x0)
    s.copy_(s0)
    dw, room = _inside((n, k), BF16, lead, tail)
    vk.wgrad_fp8(dy, x, s, dw)
    d, xv = dy.double().t(), _deq(x, s)
    _check_product(dw, d @ xv, d.abs() @ xv.abs(), t)
    _untouched(room, (n, k), lead)


def test_wgrad_of_no_tokens(vk):
    dy = torch.empty((0, 64), dtype=BF16, device="cuda")
    x = torch.empty((0, 40), dtype=torch.float8_e4m3fn, device="cuda")
    s = torch.empty((0, 1), dtype=torch.float8_e8m0fnu, device="cuda")
    assert (vk.wgrad_fp8(dy, x, s) == 0).all()
    base = _rand((64, 40), F32, 45)
    assert torch.equal(vk.wgrad_fp8(dy, x, s, base.clone(), accumulate=True), base)


def test_wgrad_values_outside_fp16(vk):
    """fp16 holds a checkpoint's values above its range at its largest number, and is exact for what it can hold."""
    x = torch.zeros((64, 128), dtype=BF16, device="cuda")
    x[:, 0], x[:, 1], x[:, 2] = 1e6, 65504.0, 2.0 ** -12
    q, s = vk.quantize_fp8(x)
    dy = torch.ones((64, 8), dtype=F16, device="cuda") / 64
    dw = vk.wgrad_fp8(dy, q, s, out_dtype=F32)
    want = _deq(q, s).clamp(-65504, 65504)[0]
    assert torch.equal(dw[0].double(), want)


# ------------------------------------------------------------------------------------------ together
def _layer(vk, x, res, wn, wq, ws, dy, dres):
    """A linear layer behind a norm, forward and backward, as a training step calls it."""
    q, s, h, rstd = vk.rmsnorm_fp8(x, wn, residual=res)
    y = vk.gemm_fp8(q, s, wq, ws, trans_b=True, out_dtype=BF16)
    dyq, dys = vk.quantize_fp8(dy)
    dn = vk.gemm_fp8(dyq, dys, wq, ws, out_dtype=BF16)
    dw = vk.wgrad_fp8(dy, q, s, out_dtype=F32)
    dx, dwn = vk.rmsnorm_fp8_backward(dn, h, wn, rstd, dres=dres)
    return {"q": q, "s": s, "h": h, "rstd": rstd, "y": y, "dyq": dyq, "dys": dys, "dn": dn, "dw": dw, "dx": dx, "dwn": dwn}


def _layer_inputs(seed, t=300, k=640, n=520):
    x, res, wn = _rand((t, k), BF16, seed), _rand((t, k), BF16, seed + 1, 3.0), _rand((k,), BF16, seed + 2)
    wq, ws = _quantized((n, k), seed + 3, True, 0.05)
    return [x, res, wn, wq, ws, _rand((t, n), BF16, seed + 4, 0.1), _rand((t, k), BF16, seed + 5, 0.1)]


def _check_layer(o, x, res, wn, wq, ws, dy, dres):
    _check_norm(x, wn, res, 1e-6, o["q"], o["s"], o["h"], o["rstd"])
    a, w, d = _deq(o["q"], o["s"]), _deq(wq, ws, True), _deq(o["dyq"], o["dys"])
    _check_product(o["y"], a @ w.t(), a.abs() @ w.t().abs(), a.shape[1])
    codes, scale = fp8.quantize(dy.double().cpu().numpy())
    np.testing.assert_array_equal(_bytes(o["dyq"]), codes)
    np.testing.assert_array_equal(_bytes(o["dys"]), scale)
    _check_product(o["dn"], d @ w, d.abs() @ w.abs(), w.shape[0])
    _check_product(o["dw"], dy.double().t() @ a, dy.double().abs().t() @ a.abs(), a.shape[0])
    _check_norm_back(o["dn"], o["h"], wn, o["rstd"], dres, o["dx"], o["dwn"])


@pytest.mark.parametrize("sizes", [(1, 4096, 512), (300, 640, 520), (520, 1000, 264)])
def test_layer_forward_and_backward(vk, sizes):
    t, k, n = sizes
    data = _layer_inputs(50, t, k, n)
    _check_layer(_layer(vk, *data), *data)


def test_layer_is_the_same_every_time(vk):
    data = _layer_inputs(60, 700, 1032, 1000)
    first = _layer(vk, *data)
    for _ in range(5):
        for name, v in _layer(vk, *data).items():
            assert torch.equal(v.view(torch.uint8), first[name].view(torch.uint8)), name


def test_layer_captured_and_replayed(vk):
    """Two graphs of the same calls, replayed on new inputs at the same time on two streams."""
    streams = [torch.cuda.Stream() for _ in range(2)]
    held = [_layer_inputs(70 + 10 * i) for i in range(2)]
    graphs, outs = [], []
    for st, data in zip(streams, held):
        with torch.cuda.stream(st):
            _layer(vk, *data)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            outs.append(_layer(vk, *data))
        graphs.append(g)
    for i, data in enumerate(held):
        for old, new in zip(data, _layer_inputs(90 + 10 * i)):
            old.copy_(new)
    torch.cuda.synchronize()
    for _ in range(3):
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for o, data in zip(outs, held):
        _check_layer(o, *data)


def test_calls_on_a_given_stream(vk):
    data = _layer_inputs(120)
    want = _layer(vk, *data)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    x, res, wn, wq, ws, dy, dres = data
    q, s, h, rstd = vk.rmsnorm_fp8(x, wn, residual=res, stream=st)
    y = vk.gemm_fp8(q, s, wq, ws, trans_b=True, out_dtype=BF16, stream=st.cuda_stream)
    dyq, dys = vk.quantize_fp8(dy, stream=st)
    dn = vk.gemm_fp8(dyq, dys, wq, ws, out_dtype=BF16, stream=st)
    dw = vk.wgrad_fp8(dy, q, s, out_dtype=F32, stream=st)
    dx, dwn = vk.rmsnorm_fp8_backward(dn, h, wn, rstd, dres=dres, stream=st)
    st.synchronize()
    for got, name in ((q, "q"), (y, "y"), (dn, "dn"), (dw, "dw"), (dx, "dx"), (dwn, "dwn")):
        assert torch.equal(got.view(torch.uint8), want[name].view(torch.uint8)), name


# ------------------------------------------------------------------------------------------ far and odd places
def test_single_rows_of_any_width(vk):
    """A single row's stride means nothing: whatever the width, it runs where wider matrices run."""
    for k, n in ((1, 1), (333, 129), (3001, 515)):
        x, w = _rand((1, k), BF16, 130), _rand((k,), BF16, 131)
        q, s, h, rstd = vk.rmsnorm_fp8(x, w, residual=x)
        _check_norm(x, w, x, 1e-6, q, s, h, rstd)
        b, sb = _quantized((n, k), 132, True)
        av, bv = _deq(q, s), _deq(b, sb, True).t()
        _check_product(vk.gemm_fp8(q, s, b, sb, trans_b=True, out_dtype=F32), av @ bv, av.abs() @ bv.abs(), k)
        dy = _rand((1, n), BF16, 133)
        d = dy.double().t()
        _check_product(vk.wgrad_fp8(dy, q, s, out_dtype=F32), d @ av, d.abs() @ av.abs(), 1)
        dx, dw = vk.rmsnorm_fp8_backward(x, h, w, rstd)
        _check_norm_back(x, h, w, rstd, None, dx, dw)


ROWS, COLS = 66000, 33000  # 2.18e9 elements: beyond 31 bits


@pytest.fixture(scope="module")
def far(vk):
    """A matrix of zeros whose last rows are not."""
    x = torch.zeros((ROWS, COLS), dtype=BF16, device="cuda")
    x[-3:] = _rand((3, COLS), BF16, 140)
    yield x
    del x
    torch.cuda.empty_cache()


@pytest.mark.parametrize("tile", [False, True])
def test_far_rows_quantized(vk, far, tile):
    q, s = vk.quantize_fp8(far, tile=tile)
    first = ROWS // 128 * 128 if tile else ROWS - 5
    codes, scale = fp8.quantize(far[first:].double().cpu().numpy(), tile)
    np.testing.assert_array_equal(_bytes(q[first:]), codes)
    np.testing.assert_array_equal(_bytes(s[-scale.shape[0]:]), scale)
    assert (q[:1000].view(torch.uint8) == 0).all()


def test_far_rows_normalised_and_back(vk, far):
    w = _rand((COLS,), BF16, 141)
    q, s, h, rstd = vk.rmsnorm_fp8(far, w, residual=far)
    _check_norm(far[-4:], w, far[-4:], 1e-6, q[-4:], s[-4:], h[-4:], rstd[-4:])
    del q, s
    dx, dw = vk.rmsnorm_fp8_backward(far, h, w, rstd)
    _check_norm_back(far[-4:], h[-4:], w, rstd[-4:], None, dx[-4:], dw)


def test_far_rows_multiplied(vk, far):
    """The 8-bit operands' and the result's last rows lie beyond 31 bits."""
    q, s = vk.quantize_fp8(far)
    b, sb = _quantized((16, COLS), 142, True)
    bv = _deq(b, sb, True).t()
    av = _deq(q[-4:], s[-4:])
    c = vk.gemm_fp8(q, s, b, sb, trans_b=True, out_dtype=F32)  # q is A
    _check_product(c[-4:], av @ bv, av.abs() @ bv.abs(), COLS)
    c = vk.gemm_fp8(b, sb, q, s, trans_b=True, out_dtype=F32)  # q is B
    _check_product(c[:, -4:], bv.t() @ av.t(), bv.t().abs() @ av.t().abs(), COLS)
    dy = torch.zeros((ROWS, 8), dtype=BF16, device="cuda")
    dy[-4:] = _rand((4, 8), BF16, 143)
    d = dy[-4:].double().t()
    _check_product(vk.wgrad_fp8(dy, q, s, out_dtype=F32), d @ av, d.abs() @ av.abs(), 4)
    del q
    a, sa = _quantized((ROWS, 128), 144)
    b, sb = _quantized((128, COLS), 145, True)
    out = torch.empty((ROWS, COLS), dtype=BF16, device="cuda")
    vk.gemm_fp8(a, sa, b, sb, out)
    av, bv = _deq(a[-3:], sa[-3:]), _deq(b, sb, True)
    _check_product(out[-3:], av @ bv, av.abs() @ bv.abs(), 128)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("byte", [127 - 40, 127 - 14, 127, 127 + 7, 127 + 20])
def test_wgrad_scale_range(vk, dtype, byte):
    """One token, dY = 1: dW is X's values in dY's type, for scales far beyond the usual ones."""
    codes = torch.arange(256, dtype=torch.uint8, device="cuda")
    codes = codes[(codes & 127) != 127]
    x = torch.zeros((1, 256), dtype=torch.uint8, device="cuda")
    x[0, :254] = codes
    s = torch.full((1, 2), byte, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
    x = x.view(torch.float8_e4m3fn)
    dw = vk.wgrad_fp8(torch.ones((1, 8), dtype=dtype, device="cuda"), x, s, out_dtype=F32)
    want = _deq(x, s).float()
    want = (want.clamp(-65504, 65504) if dtype is F16 else want).to(dtype).double()
    assert torch.equal(dw[3].double(), want[0])


def test_wgrad_nan_stays_in_its_columns(vk):
    dy = _rand((300, 264), BF16, 146)
    x, s = _quantized((300, 400), 147)
    clean = vk.wgrad_fp8(dy, x, s, out_dtype=F32)
    s.view(torch.uint8)[17, 1] = 255       # columns 128 .. 255
    x.view(torch.uint8)[40, 399] = 0x7f    # a NaN value under a finite scale
    dw = vk.wgrad_fp8(dy, x, s, out_dtype=F32)
    bad = torch.zeros(400, dtype=torch.bool, device="cuda")
    bad[128:256] = True
    bad[399] = True
    assert dw[:, bad].isnan().all() and torch.equal(dw[:, ~bad], clean[:, ~bad])


def test_calls_at_the_same_time_on_two_streams(vk):
    """Eager calls that overlap on the GPU share nothing."""
    data = [_layer_inputs(150 + 10 * i, 600, 1032, 776) for i in range(2)]
    want = [_layer(vk, *d) for d in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(_layer(vk, *data[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for o in got[i]:
            for name, v in o.items():
                assert torch.equal(v.view(torch.uint8), want[i][name].view(torch.uint8)), name


def test_first_calls_of_a_process_captured(vk):
    """Nothing has to run before a capture: the first calls of a process are recorded and replayed."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = """
import torch, vibekernel_b200 as vk
x = torch.randn(300, 640, device="cuda").bfloat16()
w = torch.ones(640, device="cuda").bfloat16()
wt = torch.randn(512, 640, device="cuda").bfloat16()
dy = torch.randn(300, 512, device="cuda").bfloat16()
torch.cuda.synchronize()
def layer():
    q, s, h, rstd = vk.rmsnorm_fp8(x, w, residual=x)
    wq, ws = vk.quantize_fp8(wt, tile=True)
    y = vk.gemm_fp8(q, s, wq, ws, trans_b=True)
    y1 = vk.gemm_fp8(q[:5], s[:5], wq, ws, trans_b=True)
    dyq, dys = vk.quantize_fp8(dy)
    dn = vk.gemm_fp8(dyq, dys, wq, ws, out_dtype=torch.bfloat16)
    return [y, y1, vk.wgrad_fp8(dy, q, s), *vk.rmsnorm_fp8_backward(dn, h, w, rstd)]
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = layer()
g.replay()
torch.cuda.synchronize()
for a, b in zip(out, layer()):
    assert torch.equal(a, b)
assert vk.device_error(0) == 0
print("captured")
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stdout + r.stderr


# ------------------------------------------------------------------------------------------ largest sizes
WIDEST = 2 ** 31 - 256  # the most columns a matrix may have
END = 384               # whole blocks; what lies between both ends is zero


def _widest(dtype, seed):
    x = torch.zeros((1, WIDEST), dtype=dtype, device="cuda")
    x[:, :END], x[:, -END:] = _rand((1, END), dtype, seed), _rand((1, END), dtype, seed + 1)
    return x


def _ends(t, n=END):
    return torch.cat([t[..., :n], t[..., -n:]], dim=-1)


@pytest.mark.parametrize("tile", [False, True])
def test_widest_rows_quantized(vk, tile):
    x = _widest(BF16, 160)
    q, s = vk.quantize_fp8(x, tile=tile)
    codes, scale = fp8.quantize(_ends(x).double().cpu().numpy(), tile)
    np.testing.assert_array_equal(_bytes(_ends(q)), codes)
    np.testing.assert_array_equal(_bytes(_ends(s, END // 128)), scale)
    assert torch.count_nonzero(q.view(torch.uint8)) == np.count_nonzero(codes)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_widest_rows_normalised_and_back(vk, dtype):
    x, w = _widest(dtype, 162), _widest(dtype, 164)[0]
    q, s, h, rstd = vk.rmsnorm_fp8(x, w, residual=x)
    he, we = _ends(h).double(), _ends(w).double()
    assert torch.equal(_ends(h), (2 * _ends(x).float()).to(dtype))
    r64 = (he.square().sum() / WIDEST + 1e-6).rsqrt()
    assert abs(rstd[0].double() - r64) <= 100 * U * r64
    y = he * r64 * we
    per = torch.from_numpy(fp8.E8M0).cuda()[_ends(s, END // 128).view(torch.uint8).long()].repeat_interleave(128, 1)
    off = (_deq(_ends(q), _ends(s, END // 128)) - y).abs()
    assert (off <= torch.maximum(2.0 ** -4 * y.abs(), 2.0 ** -10 * per) * (1 + 2.0 ** -12) + 104 * U * y.abs()).all()
    assert torch.count_nonzero(q.view(torch.uint8)[:, END:-END]) == 0
    del q, s, x
    dy = _widest(dtype, 166)
    dx, dw = vk.rmsnorm_fp8_backward(dy, h, w, rstd)
    d, r = _ends(dy).double(), rstd.double()
    g, xhat = d * we, he * r
    want = r * (g - xhat * (g * xhat).sum() / WIDEST)
    size = r * (g.abs() + xhat.abs() * (g * xhat).abs().sum() / WIDEST)
    assert ((_ends(dx).double() - want).abs() <= 104 * U * size + HALF[dtype] * (1 + 2.0 ** -8) * want.abs() + TINY[dtype]).all()
    assert ((_ends(dw).double() - (d * xhat)[0]).abs() <= 4 * U * (d * xhat).abs()[0]).all()
    assert torch.count_nonzero(dx[:, END:-END]) == 0 and torch.count_nonzero(dw[END:-END]) == 0
    del dx, dw, dy, h
    torch.cuda.empty_cache()


TALL = 2 * 64 * 65535 + 33  # rows of tiles of the CUDA-core kernel: two grids' height and one more


@pytest.mark.parametrize("k", [0, 3])
def test_gemm_of_many_unaligned_rows(vk, k):
    """More rows than a grid of the CUDA-core kernel has: every row is the product of its own operands."""
    codes = torch.randint(0, 0x70, (TALL, max(k, 1)), generator=_gen(170), device="cuda", dtype=torch.uint8)[:, :k]
    a = codes.contiguous().view(torch.float8_e4m3fn)
    sa = torch.full((TALL, 1 if k else 0), 127, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
    b, sb = _quantized((2, k), 171, pad=False) if k else (a[:2], sa[:2])
    c, room = _inside((TALL, 2), F32, 1, 1)
    vk.gemm_fp8(a, sa, b, sb, c, trans_b=True)
    if k:
        av, bv = _deq(a, sa), _deq(b, sb).t()
        _check_product(c, av @ bv, av.abs() @ bv.abs(), k)
    else:
        assert torch.count_nonzero(c) == 0
    _untouched(room, (TALL, 2), 1)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_wgrad_of_many_unaligned_columns(vk, dtype):
    dy = _rand((2, TALL), dtype, 172)
    x, s = _quantized((2, 1), 173, pad=False)
    base = _rand((TALL, 1), F32, 174)
    d, xv = dy.double().t(), _deq(x, s)
    _check_product(vk.wgrad_fp8(dy, x, s, out_dtype=F32), d @ xv, d.abs() @ xv.abs(), 2)
    _check_product(vk.wgrad_fp8(dy, x, s, base.clone(), accumulate=True), d @ xv, d.abs() @ xv.abs(), 2, base)


@pytest.mark.parametrize("m", [2, 300])
@pytest.mark.parametrize("n", [40, 300])
def test_gemm_of_nothing_not_transposed(vk, m, n):
    """An empty sum with B stored k x n: zeros, whatever C held."""
    a = torch.empty((m, 0), dtype=torch.float8_e4m3fn, device="cuda")
    b = torch.empty((0, n), dtype=torch.float8_e4m3fn, device="cuda")
    sa = torch.empty((m, 0), dtype=torch.float8_e8m0fnu, device="cuda")
    sb = torch.empty((0, (n + 127) // 128), dtype=torch.float8_e8m0fnu, device="cuda")
    c, room = _inside((m, n), BF16, 8, 8)
    assert torch.count_nonzero(vk.gemm_fp8(a, sa, b, sb, c)) == 0
    _untouched(room, (m, n), 8)


@pytest.fixture
def short_waits(vk):
    vk.set_option("wait_timeout_ns", 1000000)
    yield
    vk.set_option("wait_timeout_ns", 2000000000)


def _ones(rows, cols):
    q = torch.full((rows, cols), 0x38, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    return q, torch.full((rows, (cols + 127) // 128), 127, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)


@pytest.mark.parametrize("m,k", [(1, 2 ** 27), (130, 2 ** 25)])
def test_gemm_sums_longer_than_the_wait_limit(vk, short_waits, m, k):
    """A sum that takes many times the limit of a wait, each of its stages far less.  Every partial sum is exact."""
    a, sa = _ones(m, k)
    b, sb = _ones(8, k)
    c = vk.gemm_fp8(a, sa, b, sb, trans_b=True, out_dtype=F32)
    assert (c == k).all()
    assert vk.device_error(0) == 0


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_wgrad_sums_longer_than_the_wait_limit(vk, short_waits, dtype):
    tokens = 2 ** 23
    x, s = _ones(tokens, 16)
    dw = vk.wgrad_fp8(torch.ones((tokens, 8), dtype=dtype, device="cuda"), x, s, out_dtype=F32)
    assert (dw == tokens).all()
    assert vk.device_error(0) == 0


def test_longest_sums(vk):
    """As many terms as a sum may have, those in the middle zero: the last ones' indexes end just below 2^31."""
    x = _widest(BF16, 176)
    q, s = vk.quantize_fp8(x)
    b, sb = vk.quantize_fp8(_widest(BF16, 178))
    del x
    c = vk.gemm_fp8(q, s, b, sb, trans_b=True, out_dtype=F32)
    av = _deq(_ends(q), _ends(s, END // 128))
    bv = _deq(_ends(b), _ends(sb, END // 128)).t()
    _check_product(c, av @ bv, av.abs() @ bv.abs(), 2 * END)
    dy = _rand((1, 8), BF16, 180)
    dw = vk.wgrad_fp8(dy, q, s, out_dtype=BF16)  # as wide an output
    want = dy.double().t() @ av
    _check_product(_ends(dw), want, want.abs(), 1)
    del dw, b, sb, q, s
    torch.cuda.empty_cache()


# ------------------------------------------------------------------------------------------ the norm's backward pass over many rows
# A CTA has 2 rows until there are more than 2 * 148 to each that fits an SM (8 at most 1024 wide, 4 at most 2048, 2 at most 4096, else
# 1); these have 7 to 17, so that every stage of the ring of rows in shared memory is filled again, several times over.
RINGS = [(20001, 128), (9001, 1000), (9000, 1024), (5001, 2048), (3001, 4096), (1501, 4104), (1501, 8192)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("with_res", [False, True])
@pytest.mark.parametrize("shape", RINGS)
def test_norm_backward_of_many_rows(vk, shape, with_res, dtype):
    test_norm_backward(vk, shape, with_res, dtype)


@pytest.mark.parametrize("shape", [(9001, 1000), (3001, 4096), (1501, 8192)])
def test_norm_backward_of_many_rows_in_place(vk, shape):
    """dx in dy's or dres's place on the aligned path: the same bits, and the same every time."""
    mats = [_rand(shape, BF16, 190 + i) for i in range(3)]
    w = _rand((shape[1],), BF16, 193)
    rstd = torch.rand(shape[0], generator=_gen(194), device="cuda") + 0.5
    dx, dw = vk.rmsnorm_fp8_backward(mats[0], mats[1], w, rstd, dres=mats[2])
    _check_norm_back(mats[0], mats[1], w, rstd, mats[2], dx, dw)
    for which in (0, 2, 0, 2):
        copies = [m.clone() for m in mats]
        got, dw2 = vk.rmsnorm_fp8_backward(copies[0], copies[1], w, rstd, dres=copies[2], dx=copies[which])
        assert got is copies[which] and torch.equal(got, dx) and torch.equal(dw2, dw)


@pytest.mark.parametrize("shape", [(1, 8), (149, 1000), (3001, 4096), (1501, 8192), (300, 8200), (301, 333)])
def test_norm_backward_stays_in_its_workspace(vk, shape):
    """The C call with a workspace of exactly the size asked for, and what lies around it and around the outputs."""
    import ctypes
    rows, cols = shape
    need = ctypes.c_size_t(0)
    assert vk.lib.vk_rmsnorm_fp8_workspace(rows, cols, ctypes.byref(need)) == vk.VK_OK
    room = torch.full((need.value + 8192,), 0x55, dtype=torch.uint8, device="cuda")
    at = 4096 - room.data_ptr() % 16
    dy, h, w = _rand(shape, F16, 196), _rand(shape, F16, 197), _rand((cols,), F16, 198)
    rstd = torch.rand(rows, generator=_gen(199), device="cuda") + 0.5
    dx, dxroom = _inside(shape, F16, 8, 8)
    dw = torch.full((cols + 16,), 5.0, device="cuda")
    args = vk.RmsnormFp8BackwardArgs(dY=dy.data_ptr(), H=h.data_ptr(), weight=w.data_ptr(), rstd=rstd.data_ptr(), dX=dx.data_ptr(),
                                     dweight=dw[8:].data_ptr(), workspace=room.data_ptr() + at, workspace_bytes=need.value,
                                     rows=rows, cols=cols, lddx=dx.stride(0), dtype=vk.DTYPE_F16,
                                     stream=torch.cuda.current_stream().cuda_stream)
    assert vk.lib.vk_rmsnorm_fp8_backward(ctypes.byref(args)) == vk.VK_OK
    _check_norm_back(dy, h, w, rstd, None, dx, dw[8:-8])
    assert (room[:at] == 0x55).all() and (room[at + need.value:] == 0x55).all()
    assert (dw[:8] == 5).all() and (dw[-8:] == 5).all()
    _untouched(dxroom, shape, 8)


# ------------------------------------------------------------------------------------------ both ends of the scales
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("byte", [0, 1, 2, 3, 246, 247, 254, 255])
@pytest.mark.parametrize("tokens,n", [(1, 8), (2, 7)])
def test_wgrad_of_the_first_and_last_scales(vk, dtype, byte, tokens, n):
    """Every e4m3 value under the smallest and largest scales, on both kernels: rounded once to dY's type below its smallest step
    (bf16: 2^-133, met by bytes below 3), infinite in bf16 from 2^128 on (byte 247 and up), fp16's largest number in fp16."""
    codes = torch.arange(256, dtype=torch.uint8, device="cuda")
    x = torch.zeros((tokens, 256), dtype=torch.uint8, device="cuda")
    x[0, :254] = codes[(codes & 127) != 127]
    s = torch.full((tokens, 2), byte, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
    x = x.view(torch.float8_e4m3fn)
    dy = torch.zeros((tokens, n), dtype=dtype, device="cuda")
    dy[0] = 1
    dw = vk.wgrad_fp8(dy, x, s, out_dtype=F32)
    want = _deq(x, s)[0].float()  # exact, or infinite
    want = (want.clamp(-65504, 65504) if dtype is F16 else want).to(dtype).float()
    assert want.isnan().all() if byte == 255 else not want.isnan().any()
    assert torch.equal(dw.nan_to_num(nan=1.5, posinf=float("inf"), neginf=-float("inf")),
                       want.nan_to_num(nan=1.5, posinf=float("inf"), neginf=-float("inf")).expand(n, 256))
    if dtype is BF16:
        assert bool(want.isinf().any()) == (247 <= byte < 255)


def test_wgrad_of_a_block_at_the_top_of_bf16(vk):
    """The largest value that stays finite through the 8-bit form, and the smallest that does not."""
    x = torch.zeros((8, 256), dtype=BF16, device="cuda")
    x[0, 0], x[0, 128] = 247 * 2.0 ** 120, 248 * 2.0 ** 120
    q, s = vk.quantize_fp8(x)
    assert _bytes(s)[0].tolist() == [247, 247]
    dw = vk.wgrad_fp8(torch.ones((8, 8), dtype=BF16, device="cuda"), q, s, out_dtype=F32)
    assert (dw[:, 0] == 240 * 2.0 ** 120).all() and dw[:, 128].isposinf().all()
    dw[:, [0, 128]] = 0
    assert torch.count_nonzero(dw) == 0
