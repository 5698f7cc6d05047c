"""Cases of the 8-bit floating-point operators: what a pass of each computes, in plain torch and by
the framework's own calls, and the bytes and operations it cannot do without.

Definition.  A block of up to 128 values with largest finite magnitude `amax` is held as 8-bit codes
and one power-of-two scale 2^e, e the smallest integer with amax <= FMAX * 2^e (FMAX = 448 for e4m3,
57344 for e5m2; e = 0 for a block of zeros, never below -127).  code = round-to-nearest-even(x / 2^e).
A block is 128 neighbours of a row ("row"), of a column ("col"), or a 128 x 128 square ("tile").
A product multiplies the values that codes and scales stand for and rounds its sums once.

Kinds of case:
  checkpoint  a tensor is saved in 8 bits and restored (an activation kept for the backward pass)
  mm          A[M, K] @ B[N, K]^T,  codes and scales in hand     (a layer's forward product)
  mm_nt       A[M, K] @ B[K, N]                                  (gradient of a layer's input)
  mm_tn       A[K, M]^T @ B[K, N]                                (gradient of a layer's weights)
  serve       x[M, K] @ w[N, K]^T, x in 16 bits, w kept in 8     (a layer in serving)
  train       one training step of a layer: its output, the gradient of its input, of its weights
"""
import functools
import math
import os
import sys

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_CT = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}


@functools.lru_cache(maxsize=None)
def _framework():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fp64-emu_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import fp64_emu
    return fp64_emu


# ------------------------------------------------------------------ cases --
def listed():
    return [
        # One decoding batch's activations saved and restored: latency.
        dict(name="checkpoint 16x4096 row", kind="checkpoint", rows=16, cols=4096, blocks="row", x="bf16", code="e4m3"),
        # A training step's activations, blocks along the tokens as the weight gradient contracts them.
        dict(name="checkpoint 16384x4096 col", kind="checkpoint", rows=16384, cols=4096, blocks="col", x="bf16",
             code="e4m3"),
        # Master weights in 32 bits, square blocks, odd sizes.
        dict(name="checkpoint 4099x2045 tile", kind="checkpoint", rows=4099, cols=2045, blocks="tile", x="fp32",
             code="e4m3"),
        # A small batch against a layer's weights, both in hand: bound by reading the weights.
        dict(name="mm 48x4096x4096", kind="mm", M=48, N=4096, K=4096, b="tile", a_code="e4m3", b_code="e4m3",
             out="bf16"),
        # The size of the repository's headline product.
        dict(name="mm 8192x8192x8192", kind="mm", M=8192, N=8192, K=8192, b="tile", a_code="e4m3", b_code="e4m3",
             out="bf16"),
        # Ragged in every dimension, 32-bit output, both operands with a scale per row block.
        dict(name="mm 777x2043x1234", kind="mm", M=777, N=2043, K=1234, b="row", a_code="e4m3", b_code="e4m3",
             out="fp32"),
        # Input gradient of a square layer; gradients in the wider-range code.
        dict(name="mm_nt 4096x4096x4096", kind="mm_nt", M=4096, N=4096, K=4096, b="tile", a_code="e5m2",
             b_code="e4m3", out="bf16"),
        # Weight gradient over many tokens, 32-bit output.
        dict(name="mm_tn 2048x4096x16384", kind="mm_tn", M=2048, N=4096, K=16384, b="col", a_code="e4m3",
             b_code="e4m3", out="fp32"),
        # One token through a served layer: latency.
        dict(name="serve 1x4096x4096", kind="serve", M=1, N=4096, K=4096, x="bf16"),
        # A decoding batch through a wide served layer: bound by reading the weights.
        dict(name="serve 32x8192x8192", kind="serve", M=32, N=8192, K=8192, x="bf16"),
        # A training step of a square layer on an ordinary batch of tokens.
        dict(name="train 8192x4096x4096", kind="train", M=8192, N=4096, K=4096, x="bf16"),
        # A training step with odd sizes in half precision.
        dict(name="train 1023x1500x2008", kind="train", M=1023, N=1500, K=2008, x="fp16"),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over the logarithm; every other one a multiple of 16."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5 and v >= 16:
        v = v // 16 * 16
    return max(lo, min(hi, v))


def draw(rng):
    kind = rng.choice(["checkpoint", "mm", "mm_nt", "mm_tn", "serve", "train"])
    if kind == "checkpoint":
        return dict(kind=kind, rows=_spread(rng, 1, 16384), cols=_spread(rng, 64, 8192),
                    blocks=rng.choice(["row", "col", "tile"]), x=rng.choice(["bf16", "fp16", "fp32"]),
                    code=rng.choice(["e4m3", "e4m3", "e5m2"]))
    if kind in ("mm", "mm_nt", "mm_tn"):
        return dict(kind=kind, M=_spread(rng, 1, 8192), N=_spread(rng, 64, 8192), K=_spread(rng, 64, 8192),
                    b=rng.choice(["tile", "row" if kind == "mm" else "col"]), a_code=rng.choice(["e4m3", "e5m2"]),
                    b_code="e4m3", out=rng.choice(["bf16", "fp16", "fp32"]))
    if kind == "serve":
        return dict(kind=kind, M=_spread(rng, 1, 256), N=_spread(rng, 256, 8192), K=_spread(rng, 256, 8192),
                    x=rng.choice(["bf16", "fp16"]))
    return dict(kind=kind, M=_spread(rng, 1, 8192), N=_spread(rng, 128, 4096), K=_spread(rng, 128, 4096),
                x=rng.choice(["bf16", "fp16", "fp32"]))


# ----------------------------------------------------------------- inputs --
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)


def _activations(g, rows, cols, dtype):
    """Unit-variance values whose columns differ in size, a few of them strongly, as activations' channels do."""
    size = torch.exp(0.5 * torch.randn(cols, generator=g, device="cuda"))
    size = torch.where(torch.rand(cols, generator=g, device="cuda") < 0.004, size * 30, size)
    return (torch.randn(rows, cols, generator=g, device="cuda") * size).to(dtype)


def _gradients(g, rows, cols, dtype):
    """Small values whose rows differ in size, as tokens' losses do.  Half precision is trained with a loss scale."""
    size = torch.exp(torch.randn(rows, 1, generator=g, device="cuda")) * (0.1 if dtype == torch.float16 else 1e-4)
    return (torch.randn(rows, cols, generator=g, device="cuda") * size).to(dtype)


def _weights(g, rows, cols, dtype):
    return (torch.randn(rows, cols, generator=g, device="cuda") / math.sqrt(cols)).to(dtype)


def _pitched(codes):
    """Codes with rows on 16-byte boundaries, as the framework's quantisation returns them."""
    rows, cols = codes.shape
    buf = torch.zeros(rows, (cols + 15) // 16 * 16, dtype=torch.uint8, device=codes.device).view(codes.dtype)
    buf[:, :cols] = codes
    return buf[:, :cols]


def _in_hand(x, blocks, code):
    q, s = _quantize(x, blocks, code)
    return _pitched(q), s


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    if kind == "checkpoint":
        return dict(case=case, x=_activations(g, case["rows"], case["cols"], _DT[case["x"]]))
    M, N, K = case["M"], case["N"], case["K"]
    if kind == "mm":
        a = _in_hand(_activations(g, M, K, torch.bfloat16), "row", case["a_code"])
        b = _in_hand(_weights(g, N, K, torch.bfloat16), case["b"], case["b_code"])
    elif kind == "mm_nt":
        a = _in_hand(_gradients(g, M, K, torch.bfloat16), "row", case["a_code"])
        b = _in_hand(_weights(g, K, N, torch.bfloat16), case["b"], case["b_code"])
    elif kind == "mm_tn":
        a = _in_hand(_gradients(g, K, M, torch.bfloat16), "col", case["a_code"])
        b = _in_hand(_activations(g, K, N, torch.bfloat16), case["b"], case["b_code"])
    elif kind == "serve":
        w, ws = _in_hand(_weights(g, N, K, torch.bfloat16), "tile", "e4m3")
        return dict(case=case, x=_activations(g, M, K, _DT[case["x"]]), w=w, ws=ws)
    else:
        dt = _DT[case["x"]]
        return dict(case=case, x=_activations(g, M, K, dt).requires_grad_(), w=_weights(g, N, K, dt).requires_grad_(),
                    dy=_gradients(g, M, N, dt))
    return dict(case=case, a=a[0], sa=a[1], b=b[0], sb=b[1])


# ------------------------------------------------------------ plain forms --
_FMAX = {"e4m3": 448.0, "e5m2": 57344.0}


def _exponents(amax, code):
    """Smallest e with amax <= FMAX * 2^e: amax = m * 2^p with m in [0.5, 1), FMAX = 0.875 * 2^9 (or 2^16)."""
    m, p = torch.frexp(amax)
    e = p - (9 if code == "e4m3" else 16) + (m > 0.875).to(torch.int32)
    return torch.where(amax > 0, e, torch.zeros_like(e)).clamp(min=-127)


def _grid(x, blocks):
    """x padded with zeros and seen as [row blocks, 128 or 1, column blocks, 128 or 1]."""
    br, bc = (1 if blocks == "row" else 128), (1 if blocks == "col" else 128)
    rows, cols = x.shape
    x = torch.nn.functional.pad(x, (0, -cols % bc, 0, -rows % br))
    return x.view(x.shape[0] // br, br, x.shape[1] // bc, bc)


def _quantize(x, blocks, code):
    """(codes [rows, cols] in 8 bits, scales [row blocks, column blocks] as powers of two in 8 bits)."""
    rows, cols = x.shape
    v = _grid(x.float(), blocks)
    e = _exponents(v.abs().amax(dim=(1, 3)), code)
    q = torch.ldexp(v, -e[:, None, :, None])
    q = q.to(_CT[code]).view(torch.uint8).reshape(q.shape[0] * q.shape[1], -1)[:rows, :cols].contiguous()
    return q.view(_CT[code]), (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _values(q, s, blocks):
    """The numbers that codes and scales stand for, in 32 bits (exact)."""
    rows, cols = q.shape
    s = s.float()
    if blocks != "row":
        s = s.repeat_interleave(128, 0)[:rows]
    if blocks != "col":
        s = s.repeat_interleave(128, 1)[:, :cols]
    return q.float() * s


def _round_trip(x, blocks, code="e4m3"):
    return _values(*_quantize(x, blocks, code), blocks)


def _plain(st):
    c = st["case"]
    kind = c["kind"]
    if kind == "checkpoint":
        return _round_trip(st["x"], c["blocks"], c["code"]).to(st["x"].dtype)
    if kind == "serve":
        return (_round_trip(st["x"], "row") @ _values(st["w"], st["ws"], "tile").t()).to(st["x"].dtype)
    if kind == "train":
        x, w, dy = st["x"].detach(), st["w"].detach(), st["dy"]
        wv = _round_trip(w, "tile")
        y = _round_trip(x, "row") @ wv.t()
        dx = _round_trip(dy, "row") @ wv
        dw = _round_trip(dy, "col").t() @ _round_trip(x, "col")
        return dict(y=y.to(x.dtype), dx=dx.to(x.dtype), dw=dw.to(w.dtype))
    if kind == "mm":
        r = _values(st["a"], st["sa"], "row") @ _values(st["b"], st["sb"], c["b"]).t()
    elif kind == "mm_nt":
        r = _values(st["a"], st["sa"], "row") @ _values(st["b"], st["sb"], c["b"])
    else:
        r = _values(st["a"], st["sa"], "col").t() @ _values(st["b"], st["sb"], c["b"])
    return r.to(_DT[c["out"]])


def run(state):
    if not own:
        return _plain(state)
    emu = _framework()
    c = state["case"]
    kind = c["kind"]
    if kind == "checkpoint":
        q, s = emu.quantize_fp8(state["x"], c["blocks"], _CT[c["code"]])
        return emu.dequantize_fp8(q, s, c["blocks"], state["x"].dtype)
    if kind == "serve":
        return emu.linear_fp8(state["x"], state["w"], state["ws"])
    if kind == "train":
        y = emu.linear_fp8(state["x"], state["w"])
        dx, dw = torch.autograd.grad(y, (state["x"], state["w"]), state["dy"])
        return dict(y=y, dx=dx, dw=dw)
    mm = {"mm": emu.mm_fp8, "mm_nt": emu.mm_nt_fp8, "mm_tn": emu.mm_tn_fp8}[kind]
    return mm(state["a"], state["b"], state["sa"], state["sb"], _DT[c["out"]])


# ------------------------------------------------------------------- work --
def _scales(rows, cols, blocks):
    return (rows if blocks == "row" else -(-rows // 128)) * (cols if blocks == "col" else -(-cols // 128))


def work(case):
    kind = case["kind"]
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    if kind == "checkpoint":
        # the tensor read, the restored tensor written; a few operations a value
        n = case["rows"] * case["cols"]
        return {"bytes": 2 * n * size[case["x"]], "flops": 4 * n}
    M, N, K = case["M"], case["N"], case["K"]
    mnk = 2.0 * M * N * K
    if kind == "serve":
        e = size[case["x"]]
        return {"bytes": e * M * K + N * K + _scales(N, K, "tile") + e * M * N, "flops": mnk}
    if kind == "train":
        e = size[case["x"]]
        return {"bytes": e * (2 * M * K + 2 * N * K + 2 * M * N), "flops": 3 * mnk}
    a = (K, M, "col") if kind == "mm_tn" else (M, K, "row")
    b = (N, K, case["b"]) if kind == "mm" else (K, N, case["b"])
    return {"bytes": M * K + N * K + _scales(*a) + _scales(*b) + size[case["out"]] * M * N, "flops": mnk}


# ------------------------------------------------ the definition in 64 bits --
def _exact_values(x, blocks, code="e4m3"):
    """Block scale and rounding written from the definition, in 64 bits: the spacing of an 8-bit float with `man`
    mantissa bits at magnitude t is 2^(max(floor(log2 t), emin) - man)."""
    man, emin, fmax = (3, -6, 448.0) if code == "e4m3" else (2, -14, 57344.0)
    rows, cols = x.shape
    x = x.detach().double()
    br, bc = (1 if blocks == "row" else 128), (1 if blocks == "col" else 128)
    nr, nc = -(-rows // br), -(-cols // bc)
    full = x.new_zeros(nr * br, nc * bc)
    full[:rows, :cols] = x
    v = full.reshape(nr, br, nc, bc).transpose(1, 2)
    top = v.abs().flatten(2).max(dim=2).values
    e = torch.ceil(torch.log2(torch.where(top > 0, top, torch.full_like(top, fmax)) / fmax)).clamp(min=-127.0)
    # log2 may miss a whole number by its rounding: settle by the inequality itself
    e = torch.where(top > fmax * torch.exp2(e), e + 1, e)
    e = torch.where((top <= fmax * torch.exp2(e - 1)) & (e > -127) & (top > 0), e - 1, e)
    s = torch.exp2(e)[:, :, None, None]
    t = v / s
    step = torch.exp2(torch.floor(torch.log2(t.abs().clamp(min=2.0 ** emin))).clamp(min=float(emin)) - man)
    r = torch.round(t / step) * step * s
    return r.transpose(1, 2).reshape(nr * br, nc * bc)[:rows, :cols]


def _exact_held(q, s, blocks):
    rows, cols = q.shape
    r = torch.arange(rows, device=q.device) // (1 if blocks == "row" else 128)
    c = torch.arange(cols, device=q.device) // (1 if blocks == "col" else 128)
    e = s.view(torch.uint8).long() - 127
    return q.double() * torch.exp2(e.double())[r][:, c]


def exact(case, seed):
    st, kind = prepare(case, seed), case["kind"]
    if kind == "checkpoint":
        return _exact_values(st["x"], case["blocks"], case["code"])
    if kind == "serve":
        return torch.einsum("mk,nk->mn", _exact_values(st["x"], "row"), _exact_held(st["w"], st["ws"], "tile"))
    if kind == "train":
        w = _exact_values(st["w"], "tile")
        return dict(y=torch.einsum("mk,nk->mn", _exact_values(st["x"], "row"), w),
                    dx=torch.einsum("mn,nk->mk", _exact_values(st["dy"], "row"), w),
                    dw=torch.einsum("mn,mk->nk", _exact_values(st["dy"], "col"), _exact_values(st["x"], "col")))
    a = _exact_held(st["a"], st["sa"], "col" if kind == "mm_tn" else "row")
    b = _exact_held(st["b"], st["sb"], case["b"])
    return torch.einsum({"mm": "mk,nk->mn", "mm_nt": "mk,kn->mn", "mm_tn": "km,kn->mn"}[kind], a, b)
