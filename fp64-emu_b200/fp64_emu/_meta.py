"""Fake-tensor registrations so the product ops trace under torch.compile
(the ops write into caller-allocated `out` and return nothing)."""
import torch

from ._ops import ops


def _noop(*args, **kwargs):
    return None


for _name in ("fp64_emu_mm", "fp64_emu_bmm", "fp64_emu_mm_nt", "fp64_emu_bmm_nt",
              "fp64_emu_mm_timed", "fp64_emu_gemm_ws"):
    _packet = getattr(ops, _name, None)
    _qual = getattr(_packet, "_qualified_op_name", None) if _packet is not None else None
    if _qual is None:
        continue
    try:
        torch.library.register_fake(_qual)(_noop)
    except (AttributeError, RuntimeError):
        pass


# The 8-bit operators return new tensors.
def _codes(x, code):
    rows, cols = x.shape
    ld = (cols + 15) // 16 * 16
    return torch.empty_strided((rows, cols), (ld, 1), dtype=code, device=x.device)


def _scales(x, rows, cols):
    return torch.empty((rows, cols), dtype=torch.float8_e8m0fnu, device=x.device)


def _nb(n):
    return (n + 127) // 128


@torch.library.register_fake("fp64_emu_b200::fp8_quantize")
def _fake_quantize(x, blocks, code):
    rows, cols = x.shape
    return _codes(x, code), _scales(x, rows if blocks == 0 else _nb(rows), cols if blocks == 1 else _nb(cols))


@torch.library.register_fake("fp64_emu_b200::fp8_quantize_both")
def _fake_quantize_both(x, code, transposed):
    rows, cols = x.shape
    qc = _codes(x.t(), code).t() if transposed else _codes(x, code)
    return _codes(x, code), _scales(x, rows, _nb(cols)), qc, _scales(x, _nb(rows), cols)


@torch.library.register_fake("fp64_emu_b200::fp8_dequantize")
def _fake_dequantize(q, s, blocks, dtype):
    return torch.empty(q.shape, dtype=dtype, device=q.device)


@torch.library.register_fake("fp64_emu_b200::fp8_mm")
def _fake_fp8_mm(a, b, sa, sb, layout, dtype):
    m = a.shape[1] if layout == 2 else a.shape[0]
    n = b.shape[0] if layout == 0 else b.shape[1]
    return torch.empty((m, n), dtype=dtype, device=a.device)


@torch.library.register_fake("fp64_emu_b200::fp8_linear")
def _fake_linear(x, w, ws=None):
    torch._check(w.device == x.device and (ws is None or ws.device == x.device),
                 lambda: "x, w and its scales must be on one device")
    return torch.empty((*x.shape[:-1], w.shape[0]), dtype=x.dtype, device=x.device)
