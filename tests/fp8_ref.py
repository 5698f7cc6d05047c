"""The 8-bit block format and its products in 64 bits, written from the
definition: scale 2^e with e the smallest integer >= -127 such that
amax <= FMAX * 2^e over a block's finite values, codes round-to-nearest-even.
Torch float64 on whatever device the input is on."""
import torch

E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2
FORMAT = {E4M3: (448.0, -6, 3), E5M2: (57344.0, -14, 2)}   # FMAX, smallest normal exponent, mantissa bits


def pow2(e):
    """2^e exactly, -1022 <= e <= 1023 (the library's pow rounds on the GPU)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def block_ids(n, per_value, device):
    i = torch.arange(n, device=device)
    return i if per_value else i // 128


def grids(shape, blocks, device):
    """Block row of every row and block column of every column."""
    return (block_ids(shape[0], blocks == "row", device), block_ids(shape[1], blocks == "col", device))


def exponents(x, blocks, code):
    fmax = FORMAT[code][0]
    r, c = grids(x.shape, blocks, x.device)
    nr, nc = int(r[-1]) + 1, int(c[-1]) + 1
    mag = torch.where(torch.isfinite(x), x.double().abs(), torch.zeros((), dtype=torch.float64, device=x.device))
    amax = torch.zeros(nr * nc, dtype=torch.float64, device=x.device)
    amax.scatter_reduce_(0, (r[:, None] * nc + c[None, :]).reshape(-1), mag.reshape(-1), "amax")
    e = torch.zeros(nr * nc, dtype=torch.int64, device=x.device)
    live = amax > 0
    # the smallest e among a window that holds it, by the inequality itself
    guess = torch.floor(torch.log2(amax[live] / fmax)).long() - 2
    best = guess + 5
    for k in range(4, -1, -1):
        ok = amax[live] <= fmax * pow2(guess + k)
        best = torch.where(ok, guess + k, best)
    e[live] = best.clamp(min=-127)
    return e.view(nr, nc)


def quantize(x, blocks, code):
    """(codes' values, exponents), float64 [R, C] and int64 [blocks]."""
    fmax, emin, man = FORMAT[code]
    e = exponents(x, blocks, code)
    r, c = grids(x.shape, blocks, x.device)
    t = x.double() * pow2(-e)[r][:, c]
    ex = torch.floor(torch.log2(t.abs().clamp(min=2.0 ** emin))).clamp(min=emin)
    step = pow2(ex - man)
    v = torch.round(t / step) * step
    return torch.where(torch.isinf(t), torch.full_like(v, float("nan")), v), e


def values(codes, scales, blocks):
    r, c = grids(codes.shape, blocks, codes.device)
    e = scales.view(torch.uint8).long() - 127
    return codes.float().double() * pow2(e)[r][:, c]


def round_trip(x, blocks, code=E4M3):
    v, e = quantize(x, blocks, code)
    r, c = grids(x.shape, blocks, x.device)
    return v * pow2(e)[r][:, c]


def product_bound(a, b, out, K):
    """How far a product may be off, element by element: its K sums are held
    in 32 bits, each addition off by at most one step of the running sum
    (2^-23 of it, a truncated addition), which never exceeds sum |a b|; then
    one rounding, at most eps / 2 of the value, or half the smallest step."""
    return K * 2.0 ** -23 * (a.abs() @ b.abs()) + torch.finfo(out).eps / 2 * (a @ b).abs() * (1 + 2.0 ** -10) \
        + torch.finfo(out).smallest_normal * torch.finfo(out).eps / 2


def check_product(got, a, b):
    """got against a @ b (float64)."""
    want = a @ b
    err = (got.double() - want).abs()
    lim = product_bound(a, b, got.dtype, a.shape[1])
    bad = ~(err <= lim)
    assert not bad.any(), "%d of %d outside, worst %.3g against %.3g" % (
        int(bad.sum()), bad.numel(), float(err[bad].max()), float(lim[bad].max()))
