"""CPU checks of the 8-bit floating-point operators: refusals of the Python
surface, the torch ops and the C ABI (all before any device call), result
shapes of the fake kernels, and the reference definition against torch's own
8-bit types."""
import ctypes
import os

import pytest
import torch

import fp64_emu
import fp8_ref as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
E4, E5, E8 = torch.float8_e4m3fn, torch.float8_e5m2, torch.float8_e8m0fnu


def codes(r, c, dtype=E4):
    return torch.zeros(r, c, dtype=torch.uint8).view(dtype)


def scales(r, c):
    return torch.full((r, c), 127, dtype=torch.uint8).view(E8)


# ------------------------------------------------------------- definition --
@pytest.mark.parametrize("code", [E4, E5])
def test_reference_rounding_is_the_types_own(code):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(256, 256, generator=g) * torch.exp2(torch.randint(-20, 8, (256, 256), generator=g).float())
    v, e = R.quantize(x, "tile", code)
    t = torch.ldexp(x, -e.repeat_interleave(128, 0).repeat_interleave(128, 1).int())
    assert torch.equal(v.float(), t.to(code).float())
    fmax = R.FORMAT[code][0]
    assert (v.abs().view(2, 128, 2, 128).amax((1, 3)) <= fmax).all()
    assert (v.abs().view(2, 128, 2, 128).amax((1, 3)) > fmax / 2 * (1 - 2.0 ** -3)).all()


@pytest.mark.parametrize("amax,e", [(448.0, 0), (448.0 * (1 + 2.0 ** -23), 1), (224.0, -1), (1.0, -8), (1.75, -8),
                                    (1.7500001, -7), (2.0 ** -149, -127), (3.4e38, 120), (0.0, 0)])
def test_reference_exponent_at_borders(amax, e):
    x = torch.zeros(1, 5)
    x[0, 3] = -amax
    assert int(R.exponents(x, "row", E4)) == e


# --------------------------------------------------------------- refusals --
@pytest.mark.parametrize("call,msg", [
    (lambda f: f.quantize_fp8(torch.zeros(2, 3, 4)), "must be a matrix"),
    (lambda f: f.quantize_fp8(torch.zeros(3, 4, dtype=torch.float64)), "float32, float16 or bfloat16"),
    (lambda f: f.quantize_fp8(torch.zeros(3, 4, dtype=torch.int32)), "float32, float16 or bfloat16"),
    (lambda f: f.quantize_fp8(torch.zeros(3, 4), "row", torch.bfloat16), "the code must be"),
    (lambda f: f.quantize_fp8(torch.zeros(3, 4)), "must be a CUDA tensor"),
    (lambda f: f.quantize_fp8_both(torch.zeros(3)), "must be a matrix"),
    (lambda f: f.quantize_fp8_both(torch.zeros(3, 4)), "must be a CUDA tensor"),
    (lambda f: f.dequantize_fp8(torch.zeros(3, 4), scales(3, 1)), "codes must be"),
    (lambda f: f.dequantize_fp8(codes(3, 4), torch.ones(3, 1)), "scales must be float8_e8m0fnu"),
    (lambda f: f.dequantize_fp8(codes(3, 4), scales(1, 1)), "one entry per block"),
    (lambda f: f.dequantize_fp8(codes(3, 4), scales(3, 1), "col"), "one entry per block"),
    (lambda f: f.dequantize_fp8(codes(3, 4), scales(3, 1), dtype=torch.float64), "the result must be"),
    (lambda f: f.dequantize_fp8(codes(3, 4), scales(3, 1)), "must be a CUDA tensor"),
    (lambda f: f.mm_fp8(codes(3, 4), codes(5, 6), scales(3, 1), scales(5, 1)), "inner dimensions differ"),
    (lambda f: f.mm_fp8(codes(3, 4), codes(5, 4), scales(3, 2), scales(5, 1)), "do not fit codes"),
    (lambda f: f.mm_fp8(codes(300, 4), codes(5, 4), scales(2, 1), scales(5, 1)), "do not fit codes"),
    (lambda f: f.mm_fp8(codes(3, 4), codes(5, 4), scales(3, 1), torch.ones(5, 1)), "float8_e8m0fnu"),
    (lambda f: f.mm_fp8(codes(3, 4).view(torch.uint8), codes(5, 4), scales(3, 1), scales(5, 1)), "codes must be"),
    (lambda f: f.mm_fp8(codes(3, 4)[0], codes(5, 4), scales(3, 1), scales(5, 1)), "must be matrices"),
    (lambda f: f.mm_fp8(codes(3, 0), codes(5, 0), scales(3, 0), scales(5, 0)), "at least 1"),
    (lambda f: f.mm_fp8(codes(3, 4), codes(5, 4), scales(3, 1), scales(5, 1), torch.float64), "the result must be"),
    (lambda f: f.mm_fp8(codes(3, 4), codes(5, 4), scales(3, 1), scales(5, 1)), "must be a CUDA tensor"),
    (lambda f: f.mm_nt_fp8(codes(3, 4), codes(5, 4), scales(3, 1), scales(1, 4)), "inner dimensions differ"),
    (lambda f: f.mm_nt_fp8(codes(3, 4), codes(4, 5), scales(3, 1), scales(4, 1)), "do not fit codes"),
    (lambda f: f.mm_tn_fp8(codes(4, 3), codes(4, 5), scales(4, 1), scales(1, 5)), "do not fit codes"),
    (lambda f: f.mm_tn_fp8(codes(4, 3), codes(4, 5), scales(1, 3), scales(1, 5)), "must be a CUDA tensor"),
    (lambda f: f.linear_fp8(torch.zeros(2, 4), torch.zeros(3, 5)), "last dimension"),
    (lambda f: f.linear_fp8(torch.zeros(2, 4), torch.zeros(4)), "w two"),
    (lambda f: f.linear_fp8(torch.zeros(()), torch.zeros(3, 5)), "at least one dimension"),
    (lambda f: f.linear_fp8(torch.zeros(2, 4, dtype=torch.float64), torch.zeros(3, 4)), "float32, float16"),
    (lambda f: f.linear_fp8(torch.zeros(2, 4), torch.zeros(3, 4, dtype=torch.float64)), "float32, float16"),
    (lambda f: f.linear_fp8(torch.zeros(2, 4), torch.zeros(0, 4)), "must not be empty"),
    (lambda f: f.linear_fp8(torch.zeros(2, 4), torch.zeros(3, 4), scales(1, 1)), "codes must be"),
    (lambda f: f.linear_fp8(torch.zeros(2, 4), codes(3, 4)), "w must be float32"),
    (lambda f: f.linear_fp8(torch.zeros(2, 4), codes(300, 4), scales(300, 1)), "128 x 128 square"),
    (lambda f: f.linear_fp8(torch.zeros(2, 4), torch.zeros(3, 4)), "must be a CUDA tensor"),
    (lambda f: f.linear_fp8(torch.zeros(2, 4, requires_grad=True), torch.zeros(3, 5)), "last dimension"),
    (lambda f: f.linear_fp8(torch.zeros(2, 4, requires_grad=True), torch.zeros(3, 4)), "must be a CUDA tensor"),
])
def test_refusals(call, msg):
    with pytest.raises(RuntimeError, match=msg.replace("(", r"\(")):
        call(fp64_emu)


def test_unknown_blocks_are_refused():
    with pytest.raises(AssertionError, match="blocks must be"):
        fp64_emu.quantize_fp8(torch.zeros(3, 4), "square")
    with pytest.raises(AssertionError, match="blocks must be"):
        fp64_emu.dequantize_fp8(codes(3, 4), scales(3, 1), "square")


# ------------------------------------------------------------------- ABI --
class Operand(ctypes.Structure):
    _fields_ = [("ld", ctypes.c_int64), ("code", ctypes.c_int32), ("tile", ctypes.c_int32),
                ("k_major", ctypes.c_int32), ("scale_row", ctypes.c_int64), ("scale_block", ctypes.c_int64)]


class Problem(ctypes.Structure):
    _fields_ = [("M", ctypes.c_int64), ("N", ctypes.c_int64), ("K", ctypes.c_int64), ("out_type", ctypes.c_int32), ("ldo", ctypes.c_int64), ("a", Operand), ("b", Operand)]


@pytest.fixture(scope="module")
def lib():
    L = ctypes.CDLL(os.path.join(ROOT, "fp64-emu_b200", "fp64_emu", "libf64e.so"))
    vp, i64, i32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32
    L.f64e_fp8_quantize.argtypes = [vp, i32, i64, i64, i64, i32, i32, vp, i64, vp, vp]
    L.f64e_fp8_quantize_both.argtypes = [vp, i32, i64, i64, i64, i32, vp, vp, i64, vp, vp, i32, i64, vp]
    L.f64e_fp8_dequantize.argtypes = [vp, i32, i64, i64, i64, i32, vp, i64, i64, vp, i32, vp]
    L.f64e_fp8_gemm.argtypes = [ctypes.POINTER(Problem), vp, vp, vp, vp, vp, vp, ctypes.c_size_t, vp]
    L.f64e_fp8_workspace_size.argtypes = [ctypes.POINTER(Problem)]
    L.f64e_fp8_workspace_size.restype = ctypes.c_size_t
    L.f64e_fp8_linear.argtypes = [ctypes.POINTER(Problem), vp, i64, vp, vp, vp, vp, ctypes.c_size_t, vp]
    L.f64e_fp8_linear_workspace_size.argtypes = [i64, i64]
    L.f64e_fp8_linear_workspace_size.restype = ctypes.c_size_t
    L.f64e_last_error.restype = ctypes.c_char_p
    return L


P = 1 << 20   # a pointer value that no refused call may follow


@pytest.mark.parametrize("args,msg", [
    ((P, 7, 4, 16, 16, 0, 0, P, 16, P, None), "element type"),
    ((P, 0, 4, 16, 16, 0, 2, P, 16, P, None), "code must be"),
    ((P, 0, 4, 16, 16, 3, 0, P, 16, P, None), "blocks must be"),
    ((P, 0, -1, 16, 16, 0, 0, P, 16, P, None), "negative"),
    ((P, 0, 4, 1 << 31, 1 << 31, 0, 0, P, 1 << 31, P, None), "too large"),
    ((None, 0, 4, 16, 16, 0, 0, P, 16, P, None), "null"),
    ((P, 0, 4, 16, 15, 0, 0, P, 16, P, None), "pitch of x"),
    ((P, 0, 4, 17, 17, 0, 0, P, 16, P, None), "below their columns"),
    ((P, 0, 4, 17, 17, 0, 0, P, 24, P, None), "16-byte"),
    ((P, 0, 4, 16, 16, 0, 0, P + 8, 16, P, None), "16-byte"),
])
def test_quantize_abi_refusals(lib, args, msg):
    assert lib.f64e_fp8_quantize(*args) == 1
    assert msg in lib.f64e_last_error().decode()


@pytest.mark.parametrize("args,msg", [
    ((P, 0, 40, 20, 20, 0, P, P, 32, P, P, 2, 32, None), "transposed must be"),
    ((P, 0, 40, 20, 20, 0, P, P, 32, P, P, 0, 48, None), "same pitch"),
    ((P, 0, 40, 20, 20, 0, P, P, 32, P, P, 1, 32, None), "below their columns"),
    ((P, 0, 40, 20, 20, 0, P, P, 32, P + 1, P, 1, 48, None), "16-byte"),
    ((P, 0, 40, 20, 20, 0, P, P, 32, P, None, 1, 48, None), "null"),
])
def test_quantize_both_abi_refusals(lib, args, msg):
    assert lib.f64e_fp8_quantize_both(*args) == 1
    assert msg in lib.f64e_last_error().decode()


def test_quantize_abi_empty_is_done_without_a_device(lib):
    assert lib.f64e_fp8_quantize(None, 0, 0, 16, 16, 0, 0, None, 16, None, None) == 0
    assert lib.f64e_fp8_quantize_both(None, 0, 5, 0, 0, 0, None, None, 0, None, None, 0, 0, None) == 0
    assert lib.f64e_fp8_dequantize(None, 0, 0, 16, 16, 0, None, 1, 1, None, 0, None) == 0


def good():
    return Problem(64, 32, 256, 0, 32, Operand(256, 0, 0, 1, 2, 1), Operand(256, 0, 1, 1, 2, 1))


@pytest.mark.parametrize("change,msg", [
    (dict(out_type=3), "element type"), (dict(M=-1), "negative"),
    (dict(N=(1 << 30) + 1), "too large"), (dict(K=0), "at least 1"), (dict(ldo=31), "pitch of the output"),
    (dict(a=Operand(255, 0, 0, 1, 2, 1)), "below their columns"), (dict(a=Operand(264, 0, 0, 1, 2, 1)), "16-byte"),
    (dict(b=Operand(256, 2, 0, 1, 2, 1)), "code must be"), (dict(b=Operand(256, 0, 2, 1, 2, 1)), "tile must be"),
    (dict(b=Operand(256, 0, 0, 2, 2, 1)), "k_major must be"), (dict(b=Operand(16, 0, 0, 0, 2, 1)), "below their columns"),
])
def test_gemm_abi_refusals(lib, change, msg):
    p = good()
    for k, v in change.items():
        setattr(p, k, v)
    assert lib.f64e_fp8_gemm(ctypes.byref(p), P, P, P, P, P, None, 0, None) == 1
    assert msg in lib.f64e_last_error().decode()


def test_gemm_abi_null_and_empty(lib):
    p = good()
    assert lib.f64e_fp8_gemm(None, P, P, P, P, P, None, 0, None) == 1
    assert lib.f64e_fp8_gemm(ctypes.byref(p), P, None, P, P, P, None, 0, None) == 1
    assert lib.f64e_fp8_gemm(ctypes.byref(p), P + 4, P, P, P, P, None, 0, None) == 1
    assert "16-byte" in lib.f64e_last_error().decode()
    p.M = 0
    assert lib.f64e_fp8_gemm(ctypes.byref(p), None, None, None, None, None, None, 0, None) == 0


def test_gemm_abi_workspace(lib):
    p = good()
    assert lib.f64e_fp8_workspace_size(ctypes.byref(p)) == 0
    p = Problem(2048, 4096, 16380, 0, 4096, Operand(2048, 0, 0, 0, 1, 2048), Operand(4096, 0, 0, 0, 1, 4096))
    need = lib.f64e_fp8_workspace_size(ctypes.byref(p))
    assert need == 2048 * 16384
    for ws, nb in ((None, need), (P, need - 1), (P + 16, need)):
        assert lib.f64e_fp8_gemm(ctypes.byref(p), P, P, P, P, P, ws, nb, None) == 2
        assert "workspace" in lib.f64e_last_error().decode()
    p.b.k_major, p.b.ld = 1, 16384
    assert lib.f64e_fp8_workspace_size(ctypes.byref(p)) == 0


def test_linear_abi_refusals(lib):
    call = lambda p, x=P, ldx=256, w=P, out=P, ws=P, nb=1 << 30: lib.f64e_fp8_linear(  # noqa: E731
        p and ctypes.byref(p), x, ldx, w, P, out, ws, nb, None)
    p = good()
    assert call(None) == 1
    for kw, msg in ((dict(x=None), "null"), (dict(out=None), "null"), (dict(ldx=255), "pitch of x"),
                    (dict(w=P + 8), "16-byte")):
        assert call(p, **kw) == 1
        assert msg in lib.f64e_last_error().decode()
    for field, value, msg in (("K", 0, "at least 1"), ("ldo", 5, "pitch of the output"), ("out_type", 9, "element type"),
                              ("N", -1, "negative")):
        q = good()
        setattr(q, field, value)
        assert call(q) == 1
        assert msg in lib.f64e_last_error().decode()
    need = lib.f64e_fp8_linear_workspace_size(64, 250)
    assert need == 64 * 256 + 64 * 2
    assert lib.f64e_fp8_linear_workspace_size(16, 250) == 0
    for ws, nb in ((None, need), (P, lib.f64e_fp8_linear_workspace_size(64, 256) - 1), (P + 64, 1 << 20)):
        assert call(good(), ws=ws, nb=nb) == 2
        assert "workspace" in lib.f64e_last_error().decode()
    p.M = 0
    assert call(p, x=None, ldx=0, w=None, out=None, ws=None, nb=0) == 1   # its pitch is still wrong
    assert call(p, x=None, w=None, out=None, ws=None, nb=0) == 0


# ------------------------------------------------------------------ fakes --
def test_fake_kernels_give_shapes_and_types():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(200, 300, dtype=torch.bfloat16, device="cuda")
        q, s = fp64_emu.quantize_fp8(x)
        assert q.shape == (200, 300) and q.stride() == (304, 1) and q.dtype == E4
        assert s.shape == (200, 3) and s.dtype == E8
        assert fp64_emu.quantize_fp8(x, "col", E5)[1].shape == (2, 300)
        assert fp64_emu.quantize_fp8(x, "tile")[1].shape == (2, 3)
        q, s, qc, sc = fp64_emu.quantize_fp8_both(x)
        assert s.shape == (200, 3) and sc.shape == (2, 300)
        assert fp64_emu.quantize_fp8_both(x, transposed=True)[2].stride() == (1, 208)
        assert fp64_emu.dequantize_fp8(q, s, dtype=torch.float16).dtype == torch.float16
        assert fp64_emu.mm_fp8(q, q, s, s).shape == (200, 200)
        assert fp64_emu.mm_tn_fp8(qc, qc, sc, sc, torch.float32).shape == (300, 300)
        assert fp64_emu.linear_fp8(torch.empty(2, 7, 300, device="cuda"), x.float()).shape == (2, 7, 200)


@pytest.mark.parametrize("kind,off", [(0, 1), (0, 2), (1, 1), (2, 1)])
def test_c_abi_refuses_addresses_inside_an_element(lib, kind, off):
    """kind: F64E_F32, F64E_F16, F64E_BF16.  Refused on the host: no device is asked."""
    bad = P + off
    p = Problem(64, 64, 256, kind, 64, Operand(256, 0, 0, 1, 2, 1), Operand(256, 0, 1, 1, 2, 1))
    calls = (lambda: lib.f64e_fp8_quantize(bad, kind, 64, 256, 256, 0, 0, P, 256, P, None),
             lambda: lib.f64e_fp8_quantize_both(bad, kind, 64, 256, 256, 0, P, P, 256, P, P, 0, 256, None),
             lambda: lib.f64e_fp8_dequantize(P, 0, 64, 256, 256, 0, P, 2, 1, bad, kind, None),
             lambda: lib.f64e_fp8_gemm(ctypes.byref(p), P, P, P, P, bad, None, 0, None),
             lambda: lib.f64e_fp8_linear(ctypes.byref(p), bad, 256, P, P, P, P, 1 << 30, None),
             lambda: lib.f64e_fp8_linear(ctypes.byref(p), P, 256, P, P, bad, P, 1 << 30, None))
    for call in calls:
        assert call() == 1 and b"not aligned to their type" in lib.f64e_last_error()


# ---------------------------------------------------------------- sources --
def source(name):
    """A kernel source without its comments."""
    import re
    with open(os.path.join(ROOT, "fp64-emu_b200", "csrc", name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


@pytest.mark.parametrize("name", ["f64e_fp8_gemm.cu", "f64e_fp8_split.cu"])
def test_whole_warp_barriers_follow_a_warp_barrier(name):
    """cluster_sync and the TMEM allocation are .aligned: all lanes of a warp execute them together.  Loops, waits and
    branches before them may have parted the lanes, so nothing but a condition stands between __syncwarp and them."""
    import re
    text = source(name)
    calls = list(re.finditer(r"\b(cluster_sync|tmem_alloc|tmem_alloc_pair)\(", text))
    assert len(calls) >= 3
    for m in calls:
        assert re.search(r"__syncwarp\(\);\s*(if \((?:[^(){};]|\([^(){};]*\))*\)\s*\{?\s*)?$", text[:m.start()]), \
            text[max(0, m.start() - 200):m.end()]


def enclosing(text, at):
    """What stands before each of the blocks that hold position `at`, innermost first."""
    heads, depth = [], 0
    for i in range(at - 1, -1, -1):
        if text[i] == "}":
            depth += 1
        elif text[i] == "{":
            if depth:
                depth -= 1
            else:
                j, parens = i, 0
                while j > 0 and (parens or text[j - 1] not in ";{}"):
                    j -= 1
                    parens += {")": 1, "(": -1}.get(text[j], 0)
                heads.append(text[j:i])
    return heads


@pytest.mark.parametrize("name", ["f64e_fp8_gemm.cu", "f64e_fp8_split.cu"])
def test_a_warp_that_waits_decides_as_one(name):
    """A bounded wait either belongs to one elected thread or its outcome is agreed on by the warp: lanes that parted
    when it runs out would reach the aligned instructions behind it in parts."""
    import re
    text = source(name)
    waits = [m.start() for m in re.finditer(r"\bmbar_wait_poll\b", text)]
    assert len(waits) >= 6
    for at in waits:
        statement = text[max(text.rfind(c, 0, at) for c in ";{}"):at]
        heads = enclosing(text, at)
        one_thread = any(re.search(r"if \((producer\b|issuer\b|elect_one\(\))", h) for h in heads)
        assert one_thread or "warp_all(" in statement, text[max(0, at - 200):at + 80]
    # and so is the abort flag: read with a wait's outcome, by an elected thread, or behind the CTA's last barrier
    for m in re.finditer(r"[!|& (]\*abort_flag\b(?! =)", text):
        statement = text[max(text.rfind(c, 0, m.start()) for c in ";{}"):m.start()]
        one_thread = any(re.search(r"if \((producer\b|issuer\b|elect_one\(\))", h) for h in enclosing(text, m.start()))
        behind = text.rfind("cluster_sync", 0, m.start()) > text.rfind("mbar_wait_poll", 0, m.start())
        if "volatile int" not in statement:
            assert one_thread or behind or "warp_all(" in statement, \
                text[max(0, m.start() - 200):m.end()]


# ----------------------------------------------------------- derivatives --
@pytest.mark.parametrize("which", ["x", "w", "both"])
@pytest.mark.parametrize("requires_grad", [False, True])
def test_layer_refuses_forward_mode(which, requires_grad):
    """A tangent is refused, not dropped, whether or not the input requires grad too, and without reverse mode on."""
    import torch.autograd.forward_ad as fw
    x, w = torch.ones(2, 4, requires_grad=requires_grad), torch.ones(3, 4, requires_grad=requires_grad)
    with fw.dual_level():
        a = fw.make_dual(x, torch.ones(2, 4)) if which != "w" else x
        b = fw.make_dual(w, torch.ones(3, 4)) if which != "x" else w
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="no forward-mode derivative"):
                fp64_emu.linear_fp8(a, b)
    if not requires_grad and which != "both":
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            torch.func.jvp(lambda t: fp64_emu.linear_fp8(*((t, w) if which == "x" else (x, t))),
                           (x if which == "x" else w,), (torch.ones_like(x if which == "x" else w),))


def test_layer_refuses_forward_mode_beside_kept_weights():
    import torch.autograd.forward_ad as fw
    with fw.dual_level(), pytest.raises(RuntimeError, match="no forward-mode derivative"):
        fp64_emu.linear_fp8(fw.make_dual(torch.ones(2, 4), torch.ones(2, 4)), codes(3, 4), scales(1, 1))


@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("shape", [(40, 300), (5, 8, 300), (300,)])
def test_layer_and_gradients_on_meta_tensors(shape, kept):
    """Shapes and types of the output and the gradients without a device, as without gradients."""
    x = torch.empty(shape, dtype=torch.bfloat16, device="meta", requires_grad=True)
    if kept:
        w, s = torch.empty(200, 300, dtype=E4, device="meta"), torch.empty(2, 3, dtype=E8, device="meta")
    else:
        w, s = torch.empty(200, 300, device="meta", requires_grad=True), None
    with torch.no_grad():
        assert fp64_emu.linear_fp8(x, w, s).shape == (*shape[:-1], 200)
    y = fp64_emu.linear_fp8(x, w, s)
    assert y.shape == (*shape[:-1], 200) and y.dtype == torch.bfloat16 and y.requires_grad
    wanted = (x,) if kept else (x, w)
    for t, g in zip(wanted, torch.autograd.grad(y, wanted, torch.empty_like(y))):
        assert g.shape == t.shape and g.dtype == t.dtype and g.is_meta


def test_layer_on_two_devices_is_refused():
    for grad in (False, True):
        x = torch.zeros(2, 4, requires_grad=grad)
        with pytest.raises(RuntimeError, match="on one device"):
            fp64_emu.linear_fp8(x, torch.zeros(3, 4, device="meta"))


def meta_layer(kept=False):
    x = torch.empty(6, 40, device="meta", requires_grad=True)
    if kept:
        return x, torch.empty(20, 40, dtype=E4, device="meta"), torch.empty(1, 1, dtype=E8, device="meta")
    return x, torch.empty(20, 40, device="meta", requires_grad=True), None


@pytest.mark.parametrize("kept", [False, True])
def test_layer_second_derivative_is_refused_not_left_out(kept):
    """A gradient taken with create_graph depends on the inputs: differentiating it, alone or beside the loss, is
    refused, also where the output's gradient is a constant."""
    x, w, s = meta_layer(kept)
    y = fp64_emu.linear_fp8(x, w, s)
    grads = torch.autograd.grad(y, (x,) if kept else (x, w), torch.empty_like(y), create_graph=True)
    for g in grads:
        with pytest.raises(RuntimeError, match="no second derivative"):
            (g * g).sum().backward(retain_graph=True)
        with pytest.raises(RuntimeError, match="no second derivative"):
            (y.sum() + (g * g).sum()).backward(retain_graph=True)


def test_layer_first_derivative_under_create_graph():
    x, w, _ = meta_layer()
    fp64_emu.linear_fp8(x, w).sum().backward(create_graph=True)
    assert x.grad.shape == x.shape and w.grad.shape == w.shape
    dx, = torch.autograd.grad(fp64_emu.linear_fp8(x, w).sum(), x)
    assert not dx.requires_grad


def symbolic(shape, dynamic, dtype=torch.float32):
    """A fake tensor that requires grad, the dimensions in `dynamic` symbolic, and its shape environment."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.symbolic_shapes import DimDynamic, ShapeEnv, StatelessSymbolicContext
    env = ShapeEnv()
    mode = FakeTensorMode(shape_env=env)
    x = mode.from_tensor(torch.empty(shape, dtype=dtype), symbolic_context=StatelessSymbolicContext(
        dynamic_sizes=[DimDynamic.DYNAMIC if d in dynamic else DimDynamic.STATIC for d in range(len(shape))]))
    return x.requires_grad_(), mode, env


@pytest.mark.parametrize("shape,dynamic", [((20, 384), (0,)), ((4, 20, 384), (1,)), ((4, 20, 384), (0, 1))])
@pytest.mark.parametrize("kept", [False, True])
def test_layer_and_gradients_keep_dynamic_dimensions(shape, dynamic, kept):
    """Tracing with a batch size left open: no guard ties it to the size at hand, in either direction."""
    x, mode, env = symbolic(shape, dynamic)
    with mode:
        if kept:
            w, s = torch.empty(256, 384, dtype=E4), torch.empty(2, 3, dtype=E8)
        else:
            w, s = torch.empty(256, 384, requires_grad=True), None
        y = fp64_emu.linear_fp8(x, w, s)
        wanted = (x,) if kept else (x, w)
        grads = torch.autograd.grad(y, wanted, torch.empty_like(y))
    for d in dynamic:
        assert isinstance(y.shape[d], torch.SymInt) and isinstance(grads[0].shape[d], torch.SymInt)
        assert y.shape[d].node.expr == x.shape[d].node.expr == grads[0].shape[d].node.expr
    assert [g.shape for g in grads] == [t.shape for t in wanted]
    assert y.shape[-1] == 256
    assert not env.guards, env.guards


def test_linear_abi_workspace_over_long_k(lib):
    """Few rows of more than 442368 values are quantised before the product, into a workspace."""
    assert lib.f64e_fp8_linear_workspace_size(16, 442368) == 0
    need = lib.f64e_fp8_linear_workspace_size(4, 442369)
    assert need == (4 * 442384 + 255) // 256 * 256 + 4 * 3457
    p = Problem(4, 64, 442369, 0, 64, Operand(), Operand(442384, 0, 1, 1, 3457, 1))
    assert lib.f64e_fp8_linear(ctypes.byref(p), P, 442369, P, P, P, P, need - 1, None) == 2
    assert "workspace" in lib.f64e_last_error().decode()


def test_wait_selftest_abi_refusals(lib):
    lib.f64e_fp8_wait_selftest.argtypes = [ctypes.c_int32, ctypes.c_uint64, ctypes.c_void_p]
    for split, limit, msg in ((2, 1000, "split must be"), (0, 0, "limit must be"), (1, 10 ** 10 + 1, "limit must be")):
        assert lib.f64e_fp8_wait_selftest(split, limit, None) == 1
        assert msg in lib.f64e_last_error().decode()


def test_codes_and_products_are_detached():
    """As documented: constants to autograd in both modes, whatever the inputs require."""
    import torch.autograd.forward_ad as fw
    x = torch.empty(6, 40, device="meta", requires_grad=True)
    with fw.dual_level():
        for t in (x, fw.make_dual(x.detach(), torch.empty(6, 40, device="meta"))):
            q, s = fp64_emu.quantize_fp8(t)
            results = (q, s, *fp64_emu.quantize_fp8_both(t), fp64_emu.dequantize_fp8(q, s), fp64_emu.mm_fp8(q, q, s, s))
            for r in results:
                assert not r.requires_grad and fw.unpack_dual(r).tangent is None
    for f in (fp64_emu.quantize_fp8, fp64_emu.quantize_fp8_both, fp64_emu.dequantize_fp8):
        assert "detached" in f.__doc__ or "without a\n    gradient" in f.__doc__


@pytest.mark.parametrize("loss", [lambda y: y.sum(), lambda y: (y.float() ** 2).mean(), lambda y: torch.relu(y).sum()])
def test_chain_of_layers_under_create_graph(loss):
    """First derivatives of a chain come with create_graph too, whatever stands between and behind its layers; only
    differentiating them is refused."""
    x, w, _ = meta_layer()
    w2 = torch.empty(30, 20, device="meta", requires_grad=True)
    y = fp64_emu.linear_fp8(fp64_emu.linear_fp8(x, w), w2)
    grads = torch.autograd.grad(loss(y), (x, w, w2), create_graph=True)
    assert [g.shape for g in grads] == [x.shape, w.shape, w2.shape]
    for g in grads:
        with pytest.raises(RuntimeError, match="no second derivative"):
            g.sum().backward(retain_graph=True)
