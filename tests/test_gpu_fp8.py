"""8-bit floating-point operators on the GPU against their definition in 64
bits: codes and scales exactly, products within the bound of 32-bit sums
(fp8_ref.product_bound), the layer's output and gradients by its formulas, by
differences, captured and replayed, and as a chain of layers."""
import pytest

torch = pytest.importorskip("torch")
import fp8_ref as R  # noqa: E402
import fp64_emu  # noqa: E402

pytestmark = pytest.mark.gpu

E4, E5, E8 = torch.float8_e4m3fn, torch.float8_e5m2, torch.float8_e8m0fnu
BF, HF, SF = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("CUDA required")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def data(rows, cols, dtype, seed=0, spread=6):
    """Values whose size differs by row, by column and by element."""
    g = gen(seed)
    p = lambda *s: torch.exp2(torch.randint(-spread, spread + 1, s, generator=g, device="cuda").float())  # noqa: E731
    return (torch.randn(rows, cols, generator=g, device="cuda") * p(rows, 1) * p(1, cols) * 0.05).to(dtype)


def same(a, b):
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


def check_codes(x, q, s, blocks, code):
    v, e = R.quantize(x, blocks, code)
    assert q.dtype == code and q.shape == x.shape and s.dtype == E8
    assert torch.equal(s.view(torch.uint8).long() - 127, e)
    ok = same(q.float().double(), v)
    assert ok


# --------------------------------------------------------------- quantise --
SHAPES = [(1, 1), (1, 7), (1, 128), (3, 129), (16, 256), (127, 128), (128, 127), (129, 513), (200, 1000), (513, 72)]


@pytest.mark.parametrize("blocks", ["row", "col", "tile"])
@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("code", [E4, E5])
def test_quantize(blocks, dtype, code):
    for i, (r, c) in enumerate(SHAPES):
        x = data(r, c, dtype, i)
        q, s = fp64_emu.quantize_fp8(x, blocks, code)
        assert q.stride(0) % 16 == 0 or r == 1
        assert q.data_ptr() % 16 == 0
        check_codes(x, q, s, blocks, code)


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("code", [E4, E5])
def test_quantize_both(dtype, code):
    for i, (r, c) in enumerate(SHAPES):
        x = data(r, c, dtype, 50 + i)
        q, s, qc, sc = fp64_emu.quantize_fp8_both(x, code)
        check_codes(x, q, s, "row", code)
        check_codes(x, qc, sc, "col", code)
        q2, s2, qt, st = fp64_emu.quantize_fp8_both(x, code, transposed=True)
        assert qt.t().is_contiguous() or qt.stride(0) == 1
        check_codes(x, qt, st, "col", code)
        assert same(q2.float(), q.float()) and torch.equal(s2.view(torch.uint8), s.view(torch.uint8))


@pytest.mark.parametrize("blocks", ["row", "col", "tile"])
def test_quantize_strided_inputs(blocks):
    big = data(300, 700, BF, 9)
    for x in (big[:, 1:400], big[3:200, 5:133], big.t(), big[::2], big[:, ::3], big[7:8, 9:10]):
        check_codes(x, *fp64_emu.quantize_fp8(x, blocks), blocks, E4)
    q, s, qc, sc = fp64_emu.quantize_fp8_both(big[1:, 3:])
    check_codes(big[1:, 3:], q, s, "row", E4)
    check_codes(big[1:, 3:], qc, sc, "col", E4)
    _, _, qc, sc = fp64_emu.quantize_fp8_both(big[1:, 3:], transposed=True)
    check_codes(big[1:, 3:], qc, sc, "col", E4)


@pytest.mark.parametrize("blocks", ["row", "col", "tile"])
@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("code", [E4, E5])
def test_quantize_special_values(blocks, dtype, code):
    x = data(260, 260, dtype, 4)
    x[:, 128:256] = 0                      # blocks of zeros
    x[130, 3] = float("inf")
    x[131, 4] = -float("inf")
    x[132, 5] = float("nan")
    x[5, :] = float("nan")                 # rows and columns with nothing finite
    x[:, 7] = float("inf")
    x[9, 200] = -0.0
    x[257, 258] = torch.finfo(dtype).max
    x[258, 259] = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps   # a subnormal
    check_codes(x, *fp64_emu.quantize_fp8(x, blocks, code), blocks, code)
    q, s, qc, sc = fp64_emu.quantize_fp8_both(x, code)
    check_codes(x, q, s, "row", code)
    check_codes(x, qc, sc, "col", code)
    check_codes(x, *fp64_emu.quantize_fp8_both(x, code, transposed=True)[2:], "col", code)
    odd = x[:, 1:258]
    check_codes(odd, *fp64_emu.quantize_fp8(odd, blocks, code), blocks, code)
    check_codes(odd, *fp64_emu.quantize_fp8_both(odd, code, transposed=True)[2:], "col", code)
    q, s = fp64_emu.quantize_fp8(x, blocks, code)
    assert torch.signbit(q.float()[9, 200])


def test_quantize_borders_and_ties():
    """Largest magnitudes at FMAX * 2^e and one step either side; every tie of the code."""
    base = torch.arange(0, 2 ** 15, device="cuda", dtype=torch.int32)
    x = (base << 16).view(SF).to(BF)       # every positive bfloat16, infinities and NaNs among them
    x = torch.cat([x, -x]).view(512, 128)
    for code in (E4, E5):
        for blocks in ("row", "col", "tile"):
            check_codes(x, *fp64_emu.quantize_fp8(x, blocks, code), blocks, code)
    # one exponent for all, so that every rounding border of the code is met
    for code in (E4, E5):
        fmax = R.FORMAT[code][0]
        x = (torch.arange(0, 2 ** 14, device="cuda").float() / 2 ** 14 * fmax).view(128, 128)
        x[:, 0] = fmax
        x[1] *= 2.0 ** -12
        check_codes(x, *fp64_emu.quantize_fp8(x, "row", code), "row", code)
    for m in (1.0, 1.75, 1.7500001, 1.9999999):
        for p in (-149, -140, -127, -126, -119, -1, 0, 8, 100, 127):
            x = torch.tensor([[m * 2.0 ** p, -(m * 2.0 ** p) / 3, 2.0 ** -149]], device="cuda", dtype=torch.float64).to(SF)
            for code in (E4, E5):
                check_codes(x, *fp64_emu.quantize_fp8(x, "row", code), "row", code)


def test_quantize_empty():
    for shape in ((0, 5), (5, 0), (0, 0)):
        for blocks in ("row", "col", "tile"):
            q, s = fp64_emu.quantize_fp8(torch.empty(shape, device="cuda"), blocks)
            assert q.shape == shape
            assert fp64_emu.dequantize_fp8(q, s, blocks).shape == shape
        fp64_emu.quantize_fp8_both(torch.empty(shape, device="cuda"))


def test_quantize_writes_nothing_beyond_its_columns():
    """Through the C ABI into a part of a wider buffer: up to the next 16 columns and no further."""
    import ctypes
    import os
    L = ctypes.CDLL(os.path.join(os.path.dirname(fp64_emu.__file__), "libf64e.so"))
    vp, i64, i32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32
    L.f64e_fp8_quantize.argtypes = [vp, i32, i64, i64, i64, i32, i32, vp, i64, vp, vp]
    x = data(130, 37, SF, 2)
    for blocks in (0, 1, 2):
        q = torch.full((131, 96), 0xAB, dtype=torch.uint8, device="cuda")
        n = (130 * 1, 2 * 37, 2 * 1)[blocks]
        s = torch.full((n + 1,), 0xCD, dtype=torch.uint8, device="cuda")
        rc = L.f64e_fp8_quantize(x.data_ptr(), 0, 130, 37, 37, blocks, 0, q.data_ptr() + 16, 96, s.data_ptr(),
                                 torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        assert (q[:, :16] == 0xAB).all() and (q[:, 64:] == 0xAB).all() and (q[130] == 0xAB).all()
        assert (q[:130, 53:64] == 0).all()
        assert int(s[n]) == 0xCD


@pytest.mark.parametrize("blocks", ["row", "col", "tile"])
@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("code", [E4, E5])
def test_dequantize(blocks, dtype, code):
    for i, (r, c) in enumerate(SHAPES):
        q, s = fp64_emu.quantize_fp8(data(r, c, SF, 70 + i), blocks, code)
        want = R.values(q, s, blocks).to(dtype)
        assert same(fp64_emu.dequantize_fp8(q, s, blocks, dtype), want)
        # rows that start anywhere, scales with strides of their own
        q1 = torch.empty(r, c + 3, dtype=torch.uint8, device="cuda").view(code)[:, 3:]
        q1.view(torch.uint8).copy_(q.view(torch.uint8))
        s1 = s.view(torch.uint8).t().contiguous().t().view(E8)
        assert same(fp64_emu.dequantize_fp8(q1, s1, blocks, dtype), want)


def test_dequantize_every_code_and_scale():
    q = torch.arange(256, dtype=torch.uint8, device="cuda").repeat(256, 1)
    s = torch.arange(256, dtype=torch.uint8, device="cuda")[:, None].repeat(1, 2)
    for code in (E4, E5):
        want = q.view(code).float().double() * s.view(E8).float().double().repeat_interleave(128, 1)
        got = fp64_emu.dequantize_fp8(q.view(code), s.view(E8), "row", SF)
        assert same(got, want.to(SF))


# --------------------------------------------------------------- products --
def operand(rows, cols, blocks, code, seed, spread=2):
    """Codes, scales and the values they stand for."""
    q, s = fp64_emu.quantize_fp8(data(rows, cols, BF, seed, spread), blocks, code)
    return q, s, R.values(q, s, blocks)


def columns_first(q):
    """The same codes with columns contiguous."""
    t = torch.empty(q.shape[1], q.shape[0] + (-q.shape[0] % 16), dtype=torch.uint8, device="cuda")[:, :q.shape[0]]
    t.copy_(q.view(torch.uint8).t())
    return t.view(q.dtype).t()


def product(layout, M, N, K, out, a_blocks, b_blocks, ac=E4, bc=E4, seed=0, stored=False):
    if layout == "tn":
        a, sa, av = operand(K, M, a_blocks, ac, seed)
        av = av.t()
    else:
        a, sa, av = operand(M, K, a_blocks, ac, seed)
    if layout == "nt":
        b, sb, bv = operand(N, K, b_blocks, bc, seed + 1)
        bv = bv.t()
    else:
        b, sb, bv = operand(K, N, b_blocks, bc, seed + 1)
    f = {"nt": fp64_emu.mm_fp8, "nn": fp64_emu.mm_nt_fp8, "tn": fp64_emu.mm_tn_fp8}[layout]
    got = f(a, b, sa, sb, out)
    assert got.shape == (M, N) and got.dtype == out and got.is_contiguous()
    R.check_product(got, av, bv)
    if stored:   # either operand, and both, stored the other way
        for qa, qb in ((columns_first(a), b), (a, columns_first(b)), (columns_first(a), columns_first(b))):
            R.check_product(f(qa, qb, sa, sb, out), av, bv)


MM_SHAPES = [(1, 1, 1), (1, 128, 128), (2, 3, 129), (17, 40, 512), (64, 256, 640), (128, 255, 1000), (130, 129, 127),
             (257, 300, 513), (255, 513, 2048), (300, 17, 4100), (700, 900, 260)]


@pytest.mark.parametrize("M,N,K", MM_SHAPES)
@pytest.mark.parametrize("layout", ["nt", "nn", "tn"])
def test_products(layout, M, N, K):
    a_vec = "col" if layout == "tn" else "row"
    b_vec = "row" if layout == "nt" else "col"
    product(layout, M, N, K, BF, a_vec, "tile", seed=M + N)
    product(layout, M, N, K, SF, a_vec, b_vec, seed=M + N + 1)
    product(layout, M, N, K, HF, "tile", b_vec, seed=M + N + 2)


@pytest.mark.parametrize("layout", ["nt", "nn", "tn"])
@pytest.mark.parametrize("ac,bc", [(E4, E5), (E5, E4), (E5, E5)])
def test_products_of_codes(layout, ac, bc):
    a_vec = "col" if layout == "tn" else "row"
    product(layout, 200, 264, 700, SF, a_vec, "tile", ac, bc)
    product(layout, 5, 264, 700, BF, a_vec, "tile", ac, bc)


@pytest.mark.parametrize("layout", ["nt", "nn", "tn"])
@pytest.mark.parametrize("out", [BF, SF])
def test_products_of_operands_stored_either_way(layout, out):
    a_vec = "col" if layout == "tn" else "row"
    b_vec = "row" if layout == "nt" else "col"
    for M, N, K in ((1, 3, 5), (130, 264, 700), (300, 520, 4100), (17, 600, 1000)):
        product(layout, M, N, K, out, a_vec, b_vec, seed=3, stored=True)


@pytest.mark.parametrize("M", [1, 2, 8, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 96, 127, 128, 129, 192, 256])
def test_products_with_few_rows(M):
    for N, K in ((256, 512), (1000, 1100), (4096, 256), (130, 8192)):
        product("nt", M, N, K, BF, "row", "tile", seed=M)
        product("nt", M, N, K, SF, "row", "row", seed=M + 1)


def test_products_many_tiles_and_long_k():
    product("nt", 2100, 2300, 384, BF, "row", "tile")
    product("nn", 2100, 2300, 384, BF, "row", "tile")
    product("tn", 2100, 2300, 384, SF, "col", "col")
    product("nt", 256, 256, 65536 + 40, SF, "row", "tile")
    product("tn", 128, 384, 65536 + 40, SF, "col", "col")
    product("nt", 3, 256, 65536 + 40, SF, "row", "tile")


def test_product_sums_are_exact_for_small_integers():
    """Integers whose products and sums fit 24 bits: every order and grouping of the sums gives the same number."""
    g = gen(5)
    for M, N, K in ((300, 400, 1000), (4, 512, 3000)):
        a = torch.randint(-8, 9, (M, K), generator=g, device="cuda").float()
        b = torch.randint(-8, 9, (N, K), generator=g, device="cuda").float()
        (qa, sa), (qb, sb) = fp64_emu.quantize_fp8(a), fp64_emu.quantize_fp8(b, "tile")
        want = (a.double() @ b.double().t()).float()
        assert torch.equal(fp64_emu.mm_fp8(qa, qb, sa, sb, SF), want)
        qa, sa = fp64_emu.quantize_fp8(a.t().contiguous(), "col")
        qb, sb = fp64_emu.quantize_fp8(b.t().contiguous(), "col")
        assert torch.equal(fp64_emu.mm_tn_fp8(qa, qb, sa, sb, SF), want)


def test_products_scales_of_every_block_and_row_are_used():
    """Ones times ones with another power of two in every scale: a scale taken from a neighbour shows."""
    M, N, K = 300, 270, 128 * 9 + 5
    one = lambda r, c: torch.full((r, c + (-c % 16)), 0x38, dtype=torch.uint8, device="cuda").view(E4)[:, :c]  # noqa: E731
    g = gen(1)
    rnd = lambda r, c: torch.randint(120, 135, (r, c), generator=g, device="cuda", dtype=torch.uint8).view(E8)  # noqa: E731
    nb = (K + 127) // 128
    n = torch.full((nb,), 128.0, dtype=torch.float64, device="cuda")
    n[-1] = K - 128 * (nb - 1)
    # All K terms are positive, so each of the K additions in 32 bits is off by at most 2^-23 of the final sum.
    lim = K * 2.0 ** -23
    for m in (M, 4):
        sa, sb = rnd(m, nb), rnd(N, nb)
        want = (sa.float().double() * n) @ sb.float().double().t()
        got = fp64_emu.mm_fp8(one(m, K), one(N, K), sa, sb, SF)
        assert ((got.double() - want).abs() <= lim * want).all()
        ta = sa.view(torch.uint8).t().contiguous().view(E8)
        tb = sb.view(torch.uint8).t().contiguous().view(E8)
        got = fp64_emu.mm_tn_fp8(one(K, m), one(K, N), ta, tb, SF)
        assert ((got.double() - want).abs() <= lim * want).all()


def test_products_extreme_scales():
    """Scales at both ends of their range, opposite in the two operands."""
    q = torch.full((160, 256), 0x38, dtype=torch.uint8, device="cuda").view(E4)   # ones
    hi = torch.full((160, 2), 254, dtype=torch.uint8, device="cuda").view(E8)     # 2^127
    lo = torch.full((160, 2), 1, dtype=torch.uint8, device="cuda").view(E8)       # 2^-126
    got = fp64_emu.mm_fp8(q, q, hi, lo, SF)
    assert torch.equal(got, torch.full_like(got, 512.0))
    assert torch.isinf(fp64_emu.mm_fp8(q, q, hi, hi, SF)).all()


@pytest.mark.parametrize("M", [4, 200])
def test_products_nan_and_infinity_stay_in_their_rows(M):
    a = data(M, 300, SF, 3)
    a[1, 7] = float("nan")
    b = data(256, 300, SF, 4)
    b[9, 299] = float("nan")
    (qa, sa), (qb, sb) = fp64_emu.quantize_fp8(a), fp64_emu.quantize_fp8(b, "tile")
    got = fp64_emu.mm_fp8(qa, qb, sa, sb, BF)
    nan = got.isnan()
    want = torch.zeros_like(nan)
    want[1] = True
    want[:, 9] = True
    assert torch.equal(nan, want)
    b[9, 299] = float("inf")
    qb, sb = fp64_emu.quantize_fp8(b, "row", E5)
    got = fp64_emu.mm_fp8(qa, qb, sa, sb, SF)
    other = torch.arange(M, device="cuda") != 1
    assert torch.isinf(got[other, 9]).logical_or(got[other, 9].isnan()).all()
    assert torch.isfinite(got[other][:, [i for i in range(256) if i != 9]]).all()


def test_products_take_any_strides():
    """Codes with unaligned rows, transposed codes and scales, parts of larger tensors."""
    a, sa, av = operand(100, 300, "row", E4, 1)
    b, sb, bv = operand(260, 300, "tile", E4, 2)
    odd = torch.empty(100, 301, dtype=torch.uint8, device="cuda").view(E4)[:, 1:]
    odd.view(torch.uint8).copy_(a.view(torch.uint8))
    flip = a.view(torch.uint8).t().contiguous().t().view(E4)
    st = sa.view(torch.uint8).t().contiguous().t().view(E8)
    wide = torch.zeros(100, 512, dtype=torch.uint8, device="cuda").view(E4)
    wide.view(torch.uint8)[:, 16:316].copy_(a.view(torch.uint8))
    sb2 = torch.full((3, 8), 255, dtype=torch.uint8, device="cuda")
    sb2[:, 1:7:2] = sb.view(torch.uint8)
    for q, s in ((odd, sa), (flip, st), (wide[:, 16:316], st)):
        R.check_product(fp64_emu.mm_fp8(q, b, s, sb2.view(E8)[:, 1:7:2], SF), av, bv.t())
    R.check_product(fp64_emu.mm_fp8(a[::2], b, sa[::2], sb, SF), av[::2], bv.t())


def test_products_empty():
    a, sa, _ = operand(1, 64, "row", E4, 1)
    b, sb, _ = operand(16, 64, "tile", E4, 2)
    assert fp64_emu.mm_fp8(a[:0], b, sa[:0], sb).shape == (0, 16)
    assert fp64_emu.mm_fp8(a, b[:0], sa, sb[:0]).shape == (1, 0)


def test_products_repeat_bit_for_bit():
    for M, N, K in ((5, 4096, 2048), (100, 512, 4096), (600, 700, 1500)):
        a, sa, _ = operand(M, K, "row", E4, 1)
        b, sb, _ = operand(N, K, "tile", E4, 2)
        first = fp64_emu.mm_fp8(a, b, sa, sb, SF)
        for _ in range(5):
            assert torch.equal(fp64_emu.mm_fp8(a, b, sa, sb, SF), first)


@pytest.mark.parametrize("M,N", [(513, 384), (384, 513), (300, 289), (257, 257)])
def test_products_whose_last_tile_is_nearly_empty(M, N):
    """Most of a warp's output blocks lie outside the matrix there; the few inside must not share a buffer with them."""
    a, sa, av = operand(M, 640, "row", E4, 1)
    b, sb, bv = operand(640, N, "tile", E4, 2)
    c, sc, cv = operand(N, 640, "tile", E4, 3)
    for out in (SF, BF):
        for _ in range(60):
            first = fp64_emu.mm_nt_fp8(a, b, sa, sb, out)
            second = fp64_emu.mm_fp8(a, c, sa, sc, out)
        R.check_product(first, av, bv)
        R.check_product(second, av, cv.t())
        for _ in range(200):
            assert torch.equal(fp64_emu.mm_nt_fp8(a, b, sa, sb, out), first)
            assert torch.equal(fp64_emu.mm_fp8(a, c, sa, sc, out), second)


def test_two_streams_at_once():
    a, sa, av = operand(300, 1024, "row", E4, 1)
    b, sb, bv = operand(512, 1024, "tile", E4, 2)
    c, sc, cv = operand(3, 1024, "row", E4, 3)
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    outs = []
    for i in range(40):
        with torch.cuda.stream(streams[i % 4]):
            outs.append(fp64_emu.mm_fp8(a, b, sa, sb, SF) if i & 1 else fp64_emu.mm_fp8(c, b, sc, sb, SF))
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        assert torch.equal(o, outs[i & 1])
    R.check_product(outs[1], av, bv.t())
    R.check_product(outs[0], cv, bv.t())


# ------------------------------------------------------------------ layer --
def layer_reference(x, w, dy=None):
    """Operands of y, dx and dw as float64 pairs."""
    xr, wt = R.round_trip(x, "row"), R.round_trip(w, "tile")
    if dy is None:
        return xr, wt.t()
    return (xr, wt.t()), (R.round_trip(dy, "row"), wt), (R.round_trip(dy, "col").t(), R.round_trip(x, "col"))


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 256, 512), (4, 130, 70), (33, 384, 1000), (130, 300, 257),
                                   (513, 640, 384)])
def test_layer_and_gradients(dtype, M, N, K):
    x = data(M, K, dtype, 1, 1).requires_grad_()
    w = data(N, K, dtype, 2, 1).requires_grad_()
    dy = data(M, N, dtype, 3, 1)
    y = fp64_emu.linear_fp8(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert y.dtype == dx.dtype == dw.dtype == dtype
    for got, (a, b) in zip((y, dx, dw), layer_reference(x.detach(), w.detach(), dy)):
        R.check_product(got, a, b)
    with torch.no_grad():
        assert torch.equal(fp64_emu.linear_fp8(x, w), y)


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("M", [1, 2, 7, 16, 17, 32, 50, 64, 65, 128, 200])
def test_layer_with_kept_weights(dtype, M):
    for N, K in ((256, 512), (1000, 1100), (2048, 260), (130, 4096), (1, 5)):
        w = data(N, K, dtype, 2, 1)
        q, s = fp64_emu.quantize_fp8(w, "tile")
        x = data(M, K, dtype, 1, 1)
        R.check_product(fp64_emu.linear_fp8(x, q, s), *layer_reference(x, w))
        if K > 300:
            xs = data(M, K + 3, dtype, 5, 1)[:, 3:]     # rows that start anywhere
            R.check_product(fp64_emu.linear_fp8(xs, q, s), *layer_reference(xs, w))


@pytest.mark.parametrize("M", [1, 5, 16, 17, 70])
def test_layer_with_kept_weights_stored_otherwise(M):
    for N, K in ((300, 520), (1000, 2100), (129, 257)):
        w, x = data(N, K, BF, 2, 1), data(M, K, BF, 1, 1)
        q, s = fp64_emu.quantize_fp8(w, "tile")
        nb, kb = s.shape
        by_columns = torch.empty(K, (N + 15) // 16 * 16, dtype=torch.uint8, device="cuda")[:, :N].t()
        odd = torch.empty(N, K + 3, dtype=torch.uint8, device="cuda")[:, 3:]
        for store in (by_columns, odd):
            store.copy_(q.view(torch.uint8))
        scales = torch.empty(kb, 2 * nb, dtype=torch.uint8, device="cuda")[:, ::2].t()
        scales.copy_(s.view(torch.uint8))
        assert scales.stride() == (2, 2 * nb)
        want = layer_reference(x, w)
        for codes in (by_columns, odd):
            for sc in (s, scales.view(s.dtype)):
                y = fp64_emu.linear_fp8(x, codes.view(q.dtype), sc)
                R.check_product(y, *want)


def test_layer_with_kept_weights_special_values():
    w = data(300, 520, BF, 2, 1)
    q, s = fp64_emu.quantize_fp8(w, "tile")
    for M in (3, 40, 200):
        x = data(M, 520, BF, 1, 1)
        x[1, 130] = float("inf")
        x[2, :] = 0
        x[0, 256:384] = 0
        y = fp64_emu.linear_fp8(x, q, s)
        assert y[1].isnan().all() and (y[2] == 0).all()
        rows = [i for i in range(M) if i != 1]
        R.check_product(y[rows], *layer_reference(x[rows], w))


def test_layer_kept_weights_gradient_of_input():
    w = data(300, 520, BF, 2, 1)
    q, s = fp64_emu.quantize_fp8(w, "tile")
    x = data(77, 520, BF, 1, 1).requires_grad_()
    dy = data(77, 300, BF, 3, 1)
    y = fp64_emu.linear_fp8(x, q, s)
    dx, = torch.autograd.grad(y, x, dy)
    R.check_product(y, *layer_reference(x.detach(), w)[:2])
    R.check_product(dx, R.round_trip(dy, "row"), R.round_trip(w, "tile"))


def test_layer_leading_dimensions_and_strides():
    x = data(6 * 5, 200, BF, 1, 1).view(6, 5, 200).transpose(0, 1).requires_grad_()
    w = data(200, 136, BF, 2, 1).t().requires_grad_()
    dy = data(5, 6 * 136, BF, 3, 1).view(5, 6, 136)
    y = fp64_emu.linear_fp8(x, w)
    assert y.shape == (5, 6, 136)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert dx.shape == x.shape and dw.shape == w.shape
    flat = x.detach().reshape(30, 200)
    for got, (a, b) in zip((y.reshape(30, 136), dx.reshape(30, 200), dw),
                           layer_reference(flat, w.detach(), dy.reshape(30, 136))):
        R.check_product(got, a, b)
    v = data(1, 200, BF, 5, 1)[0]
    assert torch.equal(fp64_emu.linear_fp8(v, w), fp64_emu.linear_fp8(v[None], w)[0])
    # the gradient of a broadcast output: one row for all
    dx1, = torch.autograd.grad(fp64_emu.linear_fp8(x, w).sum(), x)
    ones = torch.ones(30, 136, dtype=BF, device="cuda")
    R.check_product(dx1.reshape(30, 200), R.round_trip(ones, "row"), R.round_trip(w.detach(), "tile"))


def test_layer_gradients_only_where_wanted():
    x, w = data(40, 300, BF, 1, 1), data(64, 300, BF, 2, 1)
    dy = data(40, 64, BF, 3, 1)
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(fp64_emu.linear_fp8(xg, wg), (xg, wg), dy)
    a = x.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(fp64_emu.linear_fp8(a, w), a, dy)[0], dx)
    b = w.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(fp64_emu.linear_fp8(x, b), b, dy)[0], dw)
    assert not fp64_emu.linear_fp8(x, w).requires_grad
    # one tensor as both
    s = data(96, 96, BF, 6, 1).requires_grad_()
    g = data(96, 96, BF, 7, 1)
    ds, = torch.autograd.grad(fp64_emu.linear_fp8(s, s), s, g)
    p = layer_reference(s.detach(), s.detach(), g)
    lim = R.product_bound(*p[1], BF, 96) + R.product_bound(*p[2], BF, 96)
    want = p[1][0] @ p[1][1] + p[2][0] @ p[2][1]
    assert ((ds.double() - want).abs() <= lim + 2.0 ** -8 * want.abs() * (1 + 2.0 ** -6) + 2.0 ** -8 * lim).all()


def test_layer_empty_batch():
    x = torch.empty(0, 64, dtype=BF, device="cuda", requires_grad=True)
    w = data(48, 64, BF, 1).requires_grad_()
    y = fp64_emu.linear_fp8(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.empty(0, 48, dtype=BF, device="cuda"))
    assert y.shape == (0, 48) and dx.shape == (0, 64) and (dw == 0).all()
    q, s = fp64_emu.quantize_fp8(w.detach(), "tile")
    assert fp64_emu.linear_fp8(x.detach(), q, s).shape == (0, 48)


def test_layer_keeps_eight_bits_of_its_input():
    x, w = data(4096, 1024, BF, 1), data(256, 1024, BF, 2).requires_grad_()
    torch.cuda.synchronize()
    y = fp64_emu.linear_fp8(x, w)
    before = torch.cuda.memory_allocated()
    grad_fn = y.grad_fn
    del y
    kept = before - torch.cuda.memory_allocated()
    assert kept <= 4096 * 256 * 2 + 512
    held = torch.cuda.memory_allocated()
    del grad_fn
    assert 4096 * 1024 <= held - torch.cuda.memory_allocated() <= 4096 * 1024 * 1.02 + 4096


def test_layer_gradients_by_differences():
    """Inputs on the codes' grid, where the layer is linear: differences are exact."""
    g = gen(8)
    pick = lambda *s: torch.randint(-6, 7, s, generator=g, device="cuda").float()  # noqa: E731
    x, w, dy = pick(5, 140), pick(9, 140), pick(5, 9)
    x[:, 0], w[:, 0], dy[:, 0] = 8, 8, 8          # the scales stay where they are
    x[:, 128], w[:, 128] = 8, 8
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(fp64_emu.linear_fp8(xg, wg), (xg, wg), dy)
    loss = lambda x, w: float((fp64_emu.linear_fp8(x, w).double() * dy.double()).sum())  # noqa: E731
    for i, j in ((0, 1), (3, 127), (4, 129), (2, 139)):
        for t, d in ((x, dx), (w, dw)):
            hi, lo = t.clone(), t.clone()
            hi[i, j] += 1
            lo[i, j] -= 1
            diff = (loss(hi, w) - loss(lo, w)) / 2 if t is x else (loss(x, hi) - loss(x, lo)) / 2
            assert diff == float(d[i, j])


def test_layer_has_no_second_derivative():
    x, w = data(4, 32, SF, 1).requires_grad_(), data(8, 32, SF, 2).requires_grad_()
    y = fp64_emu.linear_fp8(x, w)
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(y, x, torch.ones_like(y).requires_grad_(), create_graph=True)


def test_a_chain_of_layers_trains():
    """Two layers and a loss as a program runs them; every operator is held to its formula on the tensors it met."""
    x = data(300, 256, BF, 1, 1).requires_grad_()
    w1, w2 = data(520, 256, BF, 2, 1).requires_grad_(), data(192, 520, BF, 3, 1).requires_grad_()
    h = fp64_emu.linear_fp8(x, w1)
    a = torch.nn.functional.gelu(h)
    y = fp64_emu.linear_fp8(a, w2)
    for t in (h, a, y):
        t.retain_grad()
    (y.float() ** 2).mean().backward()
    first = layer_reference(x.detach(), w1.detach(), h.grad)
    second = layer_reference(a.detach(), w2.detach(), y.grad)
    for got, pair in zip((h, x.grad, w1.grad, y, a.grad, w2.grad), first + second):
        R.check_product(got.detach(), *pair)


def test_served_layers_captured_and_replayed():
    """A captured chain of two served layers, replayed on new inputs, and a second graph of the same weights."""
    w1, s1 = fp64_emu.quantize_fp8(data(512, 256, BF, 2, 1), "tile")
    w2, s2 = fp64_emu.quantize_fp8(data(256, 512, BF, 3, 1), "tile")
    chain = lambda x: fp64_emu.linear_fp8(fp64_emu.linear_fp8(x, w1, s1), w2, s2)  # noqa: E731
    graphs = []
    for M in (2, 150):
        x = data(M, 256, BF, 4, 1)
        chain(x)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            y = chain(x)
        graphs.append((g, x, y, M))
    for seed in (5, 6, 7):
        fresh = [data(M, 256, BF, seed, 1) for _, _, _, M in graphs]
        for (g, x, y, _), f in zip(graphs, fresh):
            x.copy_(f)
            g.replay()
        torch.cuda.synchronize()
        for (g, x, y, _), f in zip(graphs, fresh):
            assert torch.equal(y, chain(f))


def test_training_step_captured_and_replayed():
    w = data(384, 256, BF, 2, 1).requires_grad_()
    x = data(200, 256, BF, 1, 1).requires_grad_()
    dy = data(200, 384, BF, 3, 1)

    def step():
        y = fp64_emu.linear_fp8(x, w)
        return (y,) + torch.autograd.grad(y, (x, w), dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = step()
    with torch.no_grad():
        x.copy_(data(200, 256, BF, 11, 1))
        w.copy_(data(384, 256, BF, 12, 1))
        dy.copy_(data(200, 384, BF, 13, 1))
    g.replay()
    torch.cuda.synchronize()
    for a, b in zip(captured, step()):
        assert torch.equal(a, b)


def test_traces_under_compile():
    w, s = fp64_emu.quantize_fp8(data(256, 256, BF, 2, 1), "tile")
    f = lambda x: torch.relu(fp64_emu.linear_fp8(x, w, s))  # noqa: E731
    x = data(20, 256, BF, 1, 1)
    assert torch.equal(torch.compile(f, backend="aot_eager", fullgraph=True)(x), f(x))


def test_training_step_traces_under_compile():
    w = data(256, 384, BF, 2, 1).requires_grad_()
    x = data(200, 384, BF, 1, 1).requires_grad_()
    dy = data(200, 256, BF, 3, 1)
    f = lambda x, w: torch.relu(fp64_emu.linear_fp8(x, w))  # noqa: E731
    want = torch.autograd.grad(f(x, w), (x, w), dy)
    got = torch.autograd.grad(torch.compile(f, backend="aot_eager", fullgraph=True)(x, w), (x, w), dy)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_two_host_threads_at_once():
    """Products, layers and backward passes from four threads, each on a stream of its own."""
    import threading
    w = data(512, 384, BF, 2, 1)
    q, s = fp64_emu.quantize_fp8(w, "tile")
    x = [data(m, 384, BF, 10 + m, 1) for m in (1, 17, 300, 700)]
    want = [fp64_emu.linear_fp8(t, q, s) for t in x]
    dy = [data(t.shape[0], 512, BF, 3, 1) for t in x]
    grads = []
    for t, d in zip(x, dy):
        a, b = t.clone().requires_grad_(), w.clone().requires_grad_()
        grads.append(torch.autograd.grad(fp64_emu.linear_fp8(a, b), (a, b), d))
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(30):
                    if not torch.equal(fp64_emu.linear_fp8(x[i], q, s), want[i]):
                        wrong.append(i)
                    a, b = x[i].clone().requires_grad_(), w.clone().requires_grad_()
                    for g, h in zip(torch.autograd.grad(fp64_emu.linear_fp8(a, b), (a, b), dy[i]), grads[i]):
                        if not torch.equal(g, h):
                            wrong.append((i, "grad"))
        except Exception as e:   # noqa: BLE001
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not wrong, wrong[:5]


def test_layer_through_the_c_abi():
    """Few rows (one launch) and many (with a workspace), into a wider output whose other columns stay as they were."""
    import ctypes
    import os
    from test_fp8_cpu import Operand, Problem
    L = ctypes.CDLL(os.path.join(os.path.dirname(fp64_emu.__file__), "libf64e.so"))
    vp, i64 = ctypes.c_void_p, ctypes.c_int64
    L.f64e_fp8_linear.argtypes = [ctypes.POINTER(Problem), vp, i64, vp, vp, vp, vp, ctypes.c_size_t, vp]
    L.f64e_fp8_linear_workspace_size.argtypes = [i64, i64]
    L.f64e_fp8_linear_workspace_size.restype = ctypes.c_size_t
    N, K = 300, 500
    w = data(N, K, BF, 2, 1)
    q, s = fp64_emu.quantize_fp8(w, "tile")
    for M in (1, 7, 16, 17, 300):
        for wide in (N, N + 1, N + 20):
            x = data(M, K, BF, 1, 1)
            out = torch.full((M + 1, wide), 77.0, dtype=BF, device="cuda")
            p = Problem(M, N, K, 2, wide, Operand(), Operand(q.stride(0), 0, 1, 1, s.stride(0), s.stride(1)))
            nb = L.f64e_fp8_linear_workspace_size(M, K)
            ws = torch.empty(max(nb, 1), dtype=torch.uint8, device="cuda")
            rc = L.f64e_fp8_linear(ctypes.byref(p), x.data_ptr(), K, q.data_ptr(), s.data_ptr(), out.data_ptr(),
                                   ws.data_ptr() if nb else None, nb, torch.cuda.current_stream().cuda_stream)
            assert rc == 0
            R.check_product(out[:M, :N].contiguous(), *layer_reference(x, w))
            assert (out[:, N:] == 77).all() and (out[M] == 77).all()


def test_status_is_clear():
    a, sa, _ = operand(300, 256, "row", E4, 1)
    b, sb, _ = operand(256, 256, "tile", E4, 2)
    fp64_emu.mm_fp8(a, b, sa, sb)
    fp64_emu.mm_fp8(a[:3], b, sa[:3], sb)
    assert fp64_emu.fp8_status() == 0
    assert fp64_emu.fp8_status("cuda:0") == 0


def test_offsets_beyond_32_bits():
    """More than 2^32 bytes of values, and of output: the last rows are right."""
    rows, cols = 70003, 32784
    x = torch.zeros(rows, cols, dtype=BF, device="cuda")
    x[-200:] = data(200, cols, BF, 1, 2)
    lo = rows // 128 * 128 - 128     # whole row blocks from here on
    for blocks in ("row", "col", "tile"):
        q, s = fp64_emu.quantize_fp8(x, blocks)
        at = lo if blocks == "row" else lo // 128
        check_codes(x[lo:], q[lo:], s[at:], blocks, E4)
        back = fp64_emu.dequantize_fp8(q, s, blocks, BF)
        assert torch.equal(back[lo:].double(), R.values(q[lo:], s[at:], blocks))
        del back
    q, s, qt, st = fp64_emu.quantize_fp8_both(x, transposed=True)
    check_codes(x[lo:], q[lo:], s[lo:], "row", E4)
    check_codes(x[lo:], qt[lo:], st[lo // 128:], "col", E4)
    del x, qt, st
    a, sa, av = operand(rows, 128, "row", E4, 3)
    b, sb, bv = operand(cols, 128, "row", E4, 4)
    out = fp64_emu.mm_fp8(a, b, sa, sb, SF)
    R.check_product(out[-150:], av[-150:], bv.t())
    del out
    out = fp64_emu.mm_fp8(b[:4], q[:, :128].contiguous(), sb[:4], s[:, :1].contiguous(), SF)
    R.check_product(out[:, -150:].contiguous(), bv[:4], R.values(q[-150:, :128], s[-150:, :1], "row").t())


def test_another_device_than_the_current_one():
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU")
    x = data(40, 300, BF, 1, 1).to("cuda:1")
    w = data(64, 300, BF, 2, 1).to("cuda:1")
    assert torch.cuda.current_device() == 0
    y = fp64_emu.linear_fp8(x, w)
    assert y.device.index == 1
    R.check_product(y, *layer_reference(x, w))
    with pytest.raises(RuntimeError, match="on one device"):
        fp64_emu.linear_fp8(x, w.to("cuda:0"))


@pytest.mark.parametrize("alive", [False, True])
def test_backward_captured_beside_an_eager_graph(alive):
    """A whole step with .backward() in a graph, in a process of its own, with and without an eager graph of the same
    leaves alive; torch refuses the second with an exception where it cannot do it, and nothing ends the process."""
    import subprocess
    import sys
    code = """
import sys
sys.path[:0] = %r
import torch, fp64_emu
x = torch.randn(64, 256, device="cuda").bfloat16().requires_grad_()
w = torch.randn(128, 256, device="cuda").bfloat16().requires_grad_()
dy = torch.randn(64, 128, device="cuda").bfloat16()
eager = fp64_emu.linear_fp8(x, w) if %r else None
side = torch.cuda.Stream()
side.wait_stream(torch.cuda.current_stream())
with torch.cuda.stream(side):
    fp64_emu.linear_fp8(x, w).backward(dy)
torch.cuda.synchronize()
want = x.grad.clone(), w.grad.clone()
x.grad = w.grad = None
g = torch.cuda.CUDAGraph()
try:
    with torch.cuda.graph(g, stream=side):
        fp64_emu.linear_fp8(x, w).backward(dy)
    x.grad.zero_(); w.grad.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(x.grad, want[0]) and torch.equal(w.grad, want[1])
    print("replayed")
except RuntimeError as e:
    print("refused")
""" % ([p for p in sys.path if p], alive)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-1500:]
    assert "replayed" in r.stdout or (alive and "refused" in r.stdout), r.stdout


def test_training_step_compiled_for_any_batch():
    """One traced program for all batch sizes: a dimension marked dynamic stays so, values and gradients are the eager ones."""
    w = data(256, 384, BF, 2, 1).requires_grad_()
    f = lambda x, w: torch.relu(fp64_emu.linear_fp8(x, w))  # noqa: E731
    traced = torch.compile(f, backend="aot_eager", fullgraph=True)
    for shape in ((200, 384), (33, 384), (1021, 384)):
        x = data(*shape, BF, 1, 1).requires_grad_()
        dy = data(shape[0], 256, BF, 3, 1)
        torch._dynamo.mark_dynamic(x, 0)
        y, want = traced(x, w), f(x, w)
        assert torch.equal(y, want)
        for got, right in zip(torch.autograd.grad(y, (x, w), dy), torch.autograd.grad(want, (x, w), dy)):
            assert torch.equal(got, right)


def test_layer_refuses_tangents_and_second_derivatives():
    import torch.autograd.forward_ad as fw
    x, w = data(20, 384, BF, 1, 1), data(256, 384, BF, 2, 1)
    with fw.dual_level(), pytest.raises(RuntimeError, match="no forward-mode derivative"):
        fp64_emu.linear_fp8(fw.make_dual(x, torch.ones_like(x)), w)
    x.requires_grad_()
    y = fp64_emu.linear_fp8(x, w)
    plain, = torch.autograd.grad(y, x, torch.ones_like(y), retain_graph=True)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y), create_graph=True)
    assert torch.equal(dx.detach(), plain)
    with pytest.raises(RuntimeError, match="no second derivative"):
        (y.float().sum() + (dx.float() ** 2).sum()).backward()


# ------------------------------------------------------------------ long K --
def whole_numbers(rows, cols, seed, per_row):
    """Integers of -2 .. 2 times a power of two for each block of 128 columns (and each row): exact as codes."""
    g = gen(seed)
    v = torch.randint(-2, 3, (rows, cols), generator=g, device="cuda").float()
    m = torch.randint(0, 4, (rows if per_row else 1, (cols + 127) // 128), generator=g, device="cuda").float()
    return v * torch.exp2(m).repeat_interleave(128, 1)[:, :cols]


def exact_product(a, b):
    """a @ b^T in 64 bits; every partial sum in whatever order is a whole number below 2^24, so 32-bit sums are exact."""
    want = sum(a[:, k:k + 16384].double() @ b[:, k:k + 16384].double().t() for k in range(0, a.shape[1], 16384))
    most = sum(a[:, k:k + 16384].abs().double() @ b[:, k:k + 16384].abs().double().t()
               for k in range(0, a.shape[1], 16384))
    assert float(most.max()) < 2 ** 24
    return want.float()


@pytest.mark.parametrize("M,N,K", [(3, 256, 65576), (128, 128, 65576), (128, 128, 131112), (256, 200, 65576),
                                   (1024, 1024, 131072), (16, 40, 300000), (2309, 2311, 4136)])
@pytest.mark.parametrize("layout", ["nt", "tn"])
def test_products_over_long_k_are_exact_for_whole_numbers(M, N, K, layout):
    """A block, a part of the sums or a scale that is left out, taken twice or taken from a neighbour shows."""
    a, b = whole_numbers(M, K, M, True), whole_numbers(N, K, N + 1, True)
    want = exact_product(a, b)
    if layout == "nt":
        (qa, sa), (qb, sb) = fp64_emu.quantize_fp8(a), fp64_emu.quantize_fp8(b)
        del a, b
        got = fp64_emu.mm_fp8(qa, qb, sa, sb, SF)
    else:
        qa, sa = fp64_emu.quantize_fp8(a.t().contiguous(), "col")
        qb, sb = fp64_emu.quantize_fp8(b.t().contiguous(), "col")
        del a, b
        got = fp64_emu.mm_tn_fp8(qa, qb, sa, sb, SF)
    assert torch.equal(got, want)


@pytest.mark.parametrize("M,N,K", [(1, 300, 70000), (4, 130, 442368), (4, 130, 442500), (16, 20000, 60000)])
def test_layer_over_long_k_is_exact_for_whole_numbers(M, N, K):
    """Few rows, quantised in the product up to K = 442368 and before it beyond."""
    x, w = whole_numbers(M, K, 1, True), whole_numbers(N, K, 2, False)
    want = exact_product(x, w)
    q, s = fp64_emu.quantize_fp8(w, "tile")
    del w
    assert torch.equal(fp64_emu.linear_fp8(x, q, s), want)


def one_large_many_small(K, large, small):
    """[1, K]: `large`, then `small` at every 32nd place; codes and scales of its row blocks."""
    v = torch.zeros(1, K, device="cuda")
    v[0, 1::32] = small
    v[0, 0] = large
    q, s = fp64_emu.quantize_fp8(v)
    assert torch.equal(fp64_emu.dequantize_fp8(q, s, "row", SF), v)
    return q.view(torch.uint8), s.view(torch.uint8)


def same_rows(layout, rows, q, s):
    """`rows` times that row: [rows, K] with row blocks, or [K, rows] with column blocks."""
    q, s = q.expand(rows, -1), s.expand(rows, -1)
    if layout == "tn":
        q, s = q.t(), s.t()
    return q.contiguous().view(E4), s.contiguous().view(E8)


@pytest.mark.parametrize("layout,M,N,K", [("nt", 128, 128, 262144), ("nt", 1024, 1024, 131072), ("tn", 256, 256, 131072),
                                          ("nt", 2304, 2304, 8192), ("nt", 16, 512, 131072)])
def test_sums_of_long_products_restart(layout, M, N, K):
    """2^25, then K / 32 ones.  Beside the large term a 32-bit sum holds multiples of 4, and a one added to it is cut
    off; so an accumulator that runs on loses all ones after it.  One that starts anew after 2048 values loses at most
    the 64 of its own part: other parts' sums are exact, and, 4 to a block of 128, multiples of 4, so adding them to
    the large one is exact too."""
    a, b = one_large_many_small(K, 2.0 ** 13, 1.0), one_large_many_small(K, 2.0 ** 12, 1.0)
    (qa, sa), (qb, sb) = same_rows(layout, M, *a), same_rows(layout, N, *b)
    got = (fp64_emu.mm_fp8 if layout == "nt" else fp64_emu.mm_tn_fp8)(qa, qb, sa, sb, SF).double()
    lost = 2.0 ** 25 + K // 32 - got
    assert float(lost.min()) >= 0 and float(lost.max()) <= 64


def test_sums_of_a_layer_over_long_k_restart():
    """The same in a layer on few rows, in 32 bits, within the product's own quantisation and beyond it."""
    for K in (131072, 442368, 524288):
        x = torch.zeros(3, K, device="cuda")
        x[:, 1::32], x[:, 0] = 1.0, 2.0 ** 13
        q, s = one_large_many_small(K, 2.0 ** 12, 1.0)
        lost = 2.0 ** 25 + K // 32 - fp64_emu.linear_fp8(x, q.expand(200, -1).contiguous().view(E4),
                                                         s.expand(2, -1).contiguous().view(E8)).double()
        assert float(lost.min()) >= 0 and float(lost.max()) <= 64


@pytest.mark.parametrize("layout,M,N,K", [("tn", 256, 256, 2 ** 20), ("tn", 300, 136, 2 ** 20), ("nt", 512, 512, 2 ** 21),
                                          ("nt", 1024, 1024, 2 ** 21), ("nt", 256, 256, 2 ** 22)])
def test_sums_of_very_long_products_in_16_bits_restart(layout, M, N, K):
    """2^14, then K / 32 times 2^-10, in float16, whose values are multiples of 16 there.  An accumulator holds
    multiples of 2^-9 beside the large term and would lose all of the small ones; after 131072 values it starts anew,
    and at most 4096 of them, 4 in all, are lost.  The sum, a multiple of 16, less 4 at most, rounds to itself."""
    a, b = one_large_many_small(K, 2.0 ** 7, 2.0 ** -5), one_large_many_small(K, 2.0 ** 7, 2.0 ** -5)
    (qa, sa), (qb, sb) = same_rows(layout, M, *a), same_rows(layout, N, *b)
    got = (fp64_emu.mm_fp8 if layout == "nt" else fp64_emu.mm_tn_fp8)(qa, qb, sa, sb, HF)
    assert torch.equal(got, torch.full_like(got, 2.0 ** 14 + K / 2 ** 15))


def test_status_reports_a_wait_that_ran_out_once():
    """Either kernel's word reaches the caller, the large products' first, and the read clears both; products after it
    are right and leave it clear."""
    run_out = lambda split: fp64_emu.ops.fp8_wait_selftest(0, split, 5_000_000)   # noqa: E731  5 ms
    assert fp64_emu.fp8_status() == 0
    for splits, site in (((False,), 9), ((True,), 10), ((True, False), 9), ((False, True), 9)):
        for split in splits:
            run_out(split)
        assert fp64_emu.fp8_status() == site
        assert fp64_emu.fp8_status() == 0
    a, sa, av = operand(300, 1024, "row", E4, 1)
    b, sb, bv = operand(2304, 1024, "tile", E4, 2)
    for m in (300, 3):
        R.check_product(fp64_emu.mm_fp8(a[:m], b, sa[:m], sb), av[:m], bv.t())
    assert fp64_emu.fp8_status() == 0
    for bad in (0, 10_000_000_001):
        with pytest.raises(RuntimeError, match="limit must be"):
            fp64_emu.ops.fp8_wait_selftest(0, False, bad)


@pytest.mark.parametrize("code,first", [(E4, 63488.0), (E5, 61440.0)])
def test_restored_float16_overflows_where_documented(code, first):
    x = torch.arange(57344, 65505, 1, device="cuda").to(HF).unique()[:, None]
    back = fp64_emu.dequantize_fp8(*fp64_emu.quantize_fp8(x, "row", code), "row", HF)
    assert torch.equal(torch.isinf(back), x >= first)
    for dtype in (BF, SF):
        assert torch.isfinite(fp64_emu.dequantize_fp8(*fp64_emu.quantize_fp8(x, "row", code), "row", dtype)).all()


def test_layer_under_vmap_and_saved_tensor_hooks():
    x, w, dy = data(4 * 30, 300, BF, 1, 1).view(4, 30, 300), data(64, 300, BF, 2, 1), data(30, 64, BF, 3, 1)
    each = torch.stack([fp64_emu.linear_fp8(t, w) for t in x])
    assert torch.equal(torch.vmap(lambda t: fp64_emu.linear_fp8(t, w))(x), each)
    a, b = x[0].clone().requires_grad_(), w.clone().requires_grad_()
    want = torch.autograd.grad(fp64_emu.linear_fp8(a, b), (a, b), dy)
    with torch.autograd.graph.save_on_cpu():
        y = fp64_emu.linear_fp8(a, b)
    for got, right in zip(torch.autograd.grad(y, (a, b), dy, retain_graph=True), want):
        assert torch.equal(got, right)
    # several gradients of the output at once
    many = torch.stack([dy, 2 * dy, data(30, 64, BF, 4, 1)])
    y = fp64_emu.linear_fp8(a, b)
    batched = torch.autograd.grad(y, (a, b), many, is_grads_batched=True, retain_graph=True)
    for i in range(3):
        for got, right in zip(batched, torch.autograd.grad(y, (a, b), many[i], retain_graph=True)):
            assert torch.equal(got[i], right)
