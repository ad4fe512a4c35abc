"""GPU tests of the 4-bit microscaled operators (mx4_quantize, mx4_dequantize, mxmm) against 64-bit numpy.

Tolerances. Quantisation and its inverse are exact: codes, scales and values are compared bitwise. A
product whose dense factor holds small integers and whose scales are 2^0 .. 2^3 has sums below 2^24, so
every order of summation is exact: compared bitwise as well. Products of random numbers: a sum of k
products in 32 bits is within (k + 2) 2^-24 of the sum of magnitudes, whatever the order (k - 1 additions
and the product's own rounding, one each for alpha and for the final addition of beta C), and the result
is rounded once to its type, half a step (eps / 2).
"""
import os
import subprocess

import numpy as np
import pytest
import torch

import mx4_reference as R
import randblas_amd as rb

pytestmark = pytest.mark.gpu

TORCH = {"f64": torch.float64, "f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def stored(a, layout, op, pad, cuda, fill=float("nan")):
    """A buffer that holds A with op(A) = a (a tensor of the type under test), rows padded by `pad`, and lda."""
    t = a if (layout == "R") == (op == "N") else a.t()
    buf = torch.full((t.shape[0], t.shape[1] + pad), fill, dtype=a.dtype)
    buf[:, : t.shape[1]] = t
    return buf.to(cuda).view(-1), t.shape[1] + pad


def unstored(buf, ld, rows, cols, layout, op):
    """op(A) of a host copy of a buffer, and the padding."""
    straight = (layout == "R") == (op == "N")
    r, c = (rows, cols) if straight else (cols, rows)
    m = buf.cpu().view(r, ld)
    return (m[:, :c] if straight else m[:, :c].t()), m[:, c:]


def inputs(rows, cols, t, seed):
    g = torch.Generator().manual_seed(seed)
    a = torch.randn(rows, cols, generator=g, dtype=torch.float64)
    a = a * torch.exp2(torch.randint(-6, 7, (rows, 1), generator=g).double())
    # ties and exact values too
    pick = torch.rand(rows, cols, generator=g) < 0.3
    a = torch.where(pick, torch.round(4 * a) / 4, a)
    return a.to(TORCH[t])


def empty(rows, cols, cuda, pad_codes=0, pad_scales=0):
    nb = (cols + 31) // 32
    return rb.MX4Matrix(rows, cols, torch.full((rows, 16 * (nb + pad_codes)), 0xAA, dtype=torch.uint8, device=cuda),
                        torch.full((rows, nb + pad_scales), 0xAA, dtype=torch.uint8, device=cuda))


def check_quantized(Q, x, words=None):
    code, scale = R.quantize(x, words)
    nb = scale.shape[1]
    got_c, got_s = Q.codes.cpu().numpy(), Q.scales.cpu().numpy()
    assert np.array_equal(got_s[:, :nb], scale)
    assert np.array_equal(got_c[:, : 16 * nb], R.pack(code))
    assert np.all(got_c[:, 16 * nb:] == 0xAA) and np.all(got_s[:, nb:] == 0xAA)   # padding untouched


@pytest.mark.parametrize("rounding", ["nearest", "stochastic"])
@pytest.mark.parametrize("layout,op", [("R", "N"), ("R", "T"), ("C", "N"), ("C", "T")])
@pytest.mark.parametrize("t", ["f64", "f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols,pad", [(1, 1, 0), (3, 31, 0), (5, 64, 0), (70, 100, 3), (129, 257, 7), (64, 1024, 8)])
def test_quantize(cuda, rows, cols, pad, t, layout, op, rounding):
    a = inputs(rows, cols, t, rows + cols)
    buf, lda = stored(a, layout, op, pad, cuda)
    Q = empty(rows, cols, cuda, pad_codes=1 if pad else 0, pad_scales=pad)
    seed = rb.RNGState(11, counter=(2 ** 32 - 3, 0, 0, 0)) if rounding == "stochastic" else None
    nxt = rb.mx4_quantize(layout, op, rows, cols, buf, lda, Q, rounding=rounding, seed=seed)
    torch.cuda.synchronize()
    words = None
    if seed:
        words = R.philox_words(rows, cols, 11, 2 ** 32 - 3)
        at = 2 ** 32 - 3 + rows * ((cols + 3) // 4)
        assert nxt.counter == (at & 0xFFFFFFFF, at >> 32, 0, 0) and nxt.key == 11
    check_quantized(Q, a.double().numpy(), words)


@pytest.mark.parametrize("offset", [1, 3, 8])
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_quantize_unaligned(cuda, t, offset):
    a = inputs(9, 90, t, 5)
    buf = torch.zeros(9 * 90 + offset, dtype=TORCH[t], device=cuda)
    buf[offset:] = a.view(-1).to(cuda)
    Q = empty(9, 90, cuda)
    rb.mx4_quantize("R", "N", 9, 90, buf[offset:], 90, Q)
    check_quantized(Q, a.double().numpy())


@pytest.mark.parametrize("layout", ["R", "C"])
@pytest.mark.parametrize("rounding", ["nearest", "stochastic"])
@pytest.mark.parametrize("t", ["f64", "f32", "f16", "bf16"])
def test_quantize_special_values(cuda, t, rounding, layout):
    """Zero and subnormal blocks, the largest numbers, every tie, infinities and NaNs, signs of zeros."""
    big, tiny = torch.finfo(TORCH[t]).max, torch.finfo(TORCH[t]).smallest_normal
    x = torch.zeros(14, 64, dtype=torch.float64)
    x[1, :5] = torch.tensor([tiny, -tiny, tiny / 2, tiny / 4, tiny * 1.5])
    x[2, :3] = torch.tensor([big, -big, big / 2])
    x[3, 3] = float("inf")
    x[4, 40] = float("nan")
    x[4, :32] = 1.0
    x[5, 0], x[5, 33] = -float("inf"), 2.0
    x[6, :32] = torch.arange(32) / 4 - 4.0
    x[7] = -0.0
    x[8, :4] = torch.tensor([6.0, 6.03125, 7.96875, 5.96875])
    x[9, :4] = torch.tensor([1e-30, 1e-38, 1e-20, 1e-39])
    x[10, :4] = torch.tensor([4.0, 3.984375, 2.0, 1.0])
    x[11, :3] = torch.tensor([2.0 ** -126, 2.0 ** -127, 2.0 ** -128])
    x[12, :3] = torch.tensor([2.0 ** -149, 2.0 ** -140, -2.0 ** -149])
    if t == "f64":
        x[13, :5] = torch.tensor([1e300, 2.0 ** 200, 2.0 ** 127, 1.0, -1e300], dtype=torch.float64)
        x[6, 31] = 0.25 + 2.0 ** -50   # just above a tie: a rounding to 32 bits on the way would lose it
        x[6, 30] = 0.25 - 2.0 ** -50
        x[6, 29] = -1e-300
    a = x.to(TORCH[t])
    buf, lda = stored(a, layout, "N", 0, cuda)
    Q = empty(14, 64, cuda)
    seed = rb.RNGState(5) if rounding == "stochastic" else None
    rb.mx4_quantize(layout, "N", 14, 64, buf, lda, Q, rounding=rounding, seed=seed)
    check_quantized(Q, a.double().numpy(), R.philox_words(14, 64, 5) if seed else None)


def test_quantize_threefry_words(cuda):
    import oracle_lib as O

    a = inputs(6, 40, "f32", 8)
    Q = empty(6, 40, cuda)
    st = rb.RNGState(21, key_hi=4, rng="threefry", key_ext=(9, 8))
    rb.mx4_quantize("R", "N", 6, 40, a.to(cuda).view(-1), 40, Q, rounding="stochastic", seed=st)
    words = np.array([[O.threefry([r * 10 + c // 4, 0, 0, 0], [21, 4, 9, 8])[c % 4] for c in range(40)] for r in range(6)])
    check_quantized(Q, a.double().numpy(), words)


@pytest.mark.parametrize("layout,op", [("R", "N"), ("R", "T"), ("C", "N"), ("C", "T")])
@pytest.mark.parametrize("t", ["f64", "f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols,ro,co,pad", [(1, 1, 0, 0, 0), (40, 70, 0, 0, 0), (33, 129, 5, 32, 3), (64, 512, 1, 64, 8)])
def test_dequantize(cuda, rows, cols, ro, co, pad, t, layout, op):
    rng = np.random.default_rng(rows * cols + ro)
    low, high = (112, 140) if t == "f16" else (0, 252)
    codes, scales = R.random_mx4(rng, rows + ro, cols + co, low, high)
    scales[0, 0] = 255
    Q = rb.MX4Matrix(rows + ro, cols + co, torch.from_numpy(codes).to(cuda), torch.from_numpy(scales).to(cuda))
    exp = torch.from_numpy(R.values(codes, scales, cols + co)[ro:, co:])
    buf, lda = stored(torch.zeros(rows, cols, dtype=TORCH[t]), layout, op, pad, cuda, fill=7.0)
    buf.fill_(7.0)
    rb.mx4_dequantize(layout, op, rows, cols, Q, buf, lda, ro=ro, co=co)
    got, padding = unstored(buf, lda, rows, cols, layout, op)
    # exact in f64, f32 and bf16; f16 rounds to nearest even
    assert torch.equal(torch.nan_to_num(got.double(), nan=123.0), torch.nan_to_num(exp.to(TORCH[t]).double(), nan=123.0))
    assert torch.equal(torch.signbit(got), torch.signbit(exp.to(TORCH[t]))) or torch.isnan(exp).any()
    assert torch.all(padding == 7.0)


@pytest.mark.parametrize("layout,op", [("R", "N"), ("R", "T"), ("C", "N"), ("C", "T")])
@pytest.mark.parametrize("t", ["f64", "f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 16), (40, 70), (33, 129)])
def test_signs_of_dequantized_values(cuda, rows, cols, t, layout, op):
    """Every sign, of zeros too, those that a small scale rounds to 0 in f16 among them; a NaN block's have none."""
    rng = np.random.default_rng(rows + cols)
    codes, scales = R.random_mx4(rng, rows, cols, 90 if t == "f16" else 0, 140 if t == "f16" else 252)
    codes[0, 0] = 0x98 if cols > 1 else 0x08   # -0 first, then -0.5
    if cols > 32:
        scales[0, 1] = 255
    Q = rb.MX4Matrix(rows, cols, torch.from_numpy(codes).to(cuda), torch.from_numpy(scales).to(cuda))
    exp = torch.from_numpy(R.values(codes, scales, cols)).to(TORCH[t])
    buf, lda = stored(torch.zeros(rows, cols, dtype=TORCH[t]), layout, op, 0, cuda)
    rb.mx4_dequantize(layout, op, rows, cols, Q, buf, lda)
    got, _ = unstored(buf, lda, rows, cols, layout, op)
    nan = torch.isnan(exp)
    assert torch.equal(torch.isnan(got), nan) and torch.equal(got[~nan], exp[~nan])
    assert torch.equal(torch.signbit(got)[~nan], torch.signbit(exp)[~nan]) and bool(torch.signbit(got[0, 0])) and got[0, 0] == 0


@pytest.mark.parametrize("offset,pad", [(1, 0), (3, 5), (8, 8)])
@pytest.mark.parametrize("layout", ["R", "C"])
@pytest.mark.parametrize("t", ["f64", "f32", "f16", "bf16"])
def test_dequantize_unaligned(cuda, t, layout, offset, pad):
    """A result at any multiple of an element; what lies around it is left as it was."""
    rows, cols = 37, 93
    codes, scales = R.random_mx4(np.random.default_rng(offset), rows, cols)
    Q = rb.MX4Matrix(rows, cols, torch.from_numpy(codes).to(cuda), torch.from_numpy(scales).to(cuda))
    inner, outer = (cols, rows) if layout == "R" else (rows, cols)
    buf = torch.full((offset + outer * (inner + pad) + 16,), 7.0, dtype=TORCH[t], device=cuda)
    rb.mx4_dequantize(layout, "N", rows, cols, Q, buf[offset:], inner + pad)
    got = buf.cpu()
    body = got[offset: offset + outer * (inner + pad)].view(outer, inner + pad)
    exp = torch.from_numpy(R.values(codes, scales, cols)).to(TORCH[t])
    assert torch.equal(body[:, :inner], exp if layout == "R" else exp.t())
    assert torch.all(body[:, inner:] == 7.0) and torch.all(got[:offset] == 7.0) and torch.all(got[-16:] == 7.0)


def test_dequantize_extreme_scales(cuda):
    """2^-127 (a subnormal) to 2^127: 64-bit values are exact, 32-bit ones overflow to infinity."""
    codes = np.tile(np.arange(0, 256, 16, dtype=np.uint8), (3, 1))
    scales = np.array([[0], [254], [255]], np.uint8)
    Q = rb.MX4Matrix(3, 32, torch.from_numpy(codes).to(cuda), torch.from_numpy(scales).to(cuda))
    exp = torch.from_numpy(R.values(codes, scales, 32))
    for t in ("f64", "f32", "bf16"):
        out = torch.empty(96, dtype=TORCH[t], device=cuda)
        rb.mx4_dequantize("R", "N", 3, 32, Q, out, 32)
        assert torch.equal(torch.nan_to_num(out.cpu().double().view(3, 32), nan=5.0),
                           torch.nan_to_num(exp.to(TORCH[t]).double(), nan=5.0)), t


def test_large_offsets(cuda):
    """Elements beyond 2^31: the last rows of a matrix of 2.2e9 elements."""
    rows, cols = 140_000, 16_000
    a = torch.zeros(rows * cols, dtype=torch.bfloat16, device=cuda)
    tail = inputs(3, cols, "bf16", 1)
    a[-3 * cols:] = tail.to(cuda).view(-1)
    Q = rb.mx4_empty(rows, cols, device=cuda)
    rb.mx4_quantize("R", "N", rows, cols, a, cols, Q)
    code, scale = R.quantize(tail.double().numpy())
    assert np.array_equal(Q.codes[-3:].cpu().numpy(), R.pack(code))
    assert np.array_equal(Q.scales[-3:, : cols // 32].cpu().numpy(), scale)
    a.fill_(1.0)
    rb.mx4_dequantize("R", "N", rows, cols, Q, a, cols)
    assert np.array_equal(a[-3 * cols:].cpu().double().numpy().reshape(3, cols), R.values(R.pack(code), scale, cols))
    assert not a[: cols].any()


@pytest.mark.parametrize("t,rows,cols", [("f32", 8192, 8200), ("f64", 4096, 8193), ("bf16", 64, 40), ("f16", 128, 100)])
def test_across_memory_as_along_it(cuda, t, rows, cols):
    """Matrices above and below 256 MB, whole lines across memory: the same codes and values as along it."""
    g = torch.Generator(device=cuda).manual_seed(rows)
    a = torch.randn(rows, cols, generator=g, device=cuda, dtype=TORCH["f32"]).to(TORCH[t])
    across = a.t().contiguous()
    P, Q = rb.mx4_empty(rows, cols, device=cuda), rb.mx4_empty(rows, cols, device=cuda)
    rb.mx4_quantize("R", "N", rows, cols, a.view(-1), cols, P)
    rb.mx4_quantize("C", "N", rows, cols, across.view(-1), rows, Q)
    nb = (cols + 31) // 32
    assert torch.equal(P.codes, Q.codes) and torch.equal(P.scales[:, :nb], Q.scales[:, :nb])
    pick = torch.arange(0, rows, max(1, rows // 8), device=cuda)
    code, scale = R.quantize(a[pick].cpu().double().numpy())
    assert np.array_equal(Q.codes[pick].cpu().numpy(), R.pack(code)) and np.array_equal(Q.scales[pick, :nb].cpu().numpy(), scale)
    a.fill_(7.0)
    across.fill_(7.0)
    rb.mx4_dequantize("R", "N", rows, cols, P, a.view(-1), cols)
    rb.mx4_dequantize("C", "N", rows, cols, P, across.view(-1), rows)
    assert torch.equal(a, across.t())
    exp = torch.from_numpy(R.values(R.pack(code), scale, cols)).to(TORCH[t])
    assert torch.equal(a[pick].cpu(), exp)


# ---------------------------------------------------------------------------------------------
# products
# ---------------------------------------------------------------------------------------------
def mx4(rng, rows, cols, cuda, low=127, high=130, scale_pad=None):
    codes, scales = R.random_mx4(rng, rows, cols, low, high)
    nb = scales.shape[1]
    wide = np.full((rows, nb + (-nb % 4 if scale_pad is None else scale_pad)), 255, np.uint8)   # padding: NaN scales
    wide[:, :nb] = scales
    Q = rb.MX4Matrix(rows, cols, torch.from_numpy(codes).to(cuda), torch.from_numpy(wide).to(cuda))
    return Q, R.values(codes, scales, cols)


class Case:
    """One product: factors, the call and its expected value in 64 bits."""

    def __init__(self, cuda, side, m, n, k, t, layout, opA, opB, seed, integers, alpha=1.0, beta=0.0, pad=0, ro=0, co=0,
                 low=127, high=130, scale_pad=None):
        rng = np.random.default_rng(seed)
        self.m, self.n, self.k, self.t, self.layout = m, n, k, t, layout
        self.head = (layout, opA, opB, m, n, k, alpha)

        def dense(rows, cols, op):
            x = rng.integers(-4, 5, (rows, cols)).astype(np.float64) if integers else rng.standard_normal((rows, cols))
            x = torch.from_numpy(x).to(TORCH[t])
            buf, ld = stored(x, layout, op, pad, cuda)
            return buf, ld, x.double().numpy()

        def quantised(rows, cols, op):
            r, c = (rows, cols) if op == "N" else (cols, rows)
            Q, v = mx4(rng, r + ro, c + co, cuda, low, high, scale_pad)
            v = v[ro:, co:]
            return Q, (v if op == "N" else v.T)

        if side == "right":
            bufA, lda, a = dense(m, k, opA)
            Q, b = quantised(k, n, opB)
            self.factors = (bufA, lda, Q, ro, co)
        elif side == "left":
            Q, a = quantised(m, k, opA)
            bufB, ldb, b = dense(k, n, opB)
            self.factors = (Q, ro, co, bufB, ldb)
        else:
            QA, a = quantised(m, k, opA)
            QB, b = quantised(k, n, opB)
            self.factors = (QA, ro, co, QB, ro, co)
        c0 = rng.integers(-4, 5, (m, n)).astype(np.float64)
        self.beta, self.pad = beta, pad
        self.c0 = torch.from_numpy(c0).to(TORCH[t])
        self.exact = alpha * (a @ b) + (beta * c0 if beta else 0.0)
        self.size = abs(alpha) * (np.abs(a) @ np.abs(b)) + abs(beta) * np.abs(c0)
        self.new(cuda)

    def new(self, cuda):
        c = self.c0 if self.beta else torch.full_like(self.c0, float("nan"))   # beta = 0 reads nothing
        self.C, self.ldc = stored(c, self.layout, "N", self.pad, cuda, fill=9.0)

    def run(self, **kw):
        rb.mxmm(*self.head, *self.factors, self.beta, self.C, self.ldc, **kw)

    def result(self):
        torch.cuda.synchronize()
        got, padding = unstored(self.C, self.ldc, self.m, self.n, self.layout, "N")
        assert torch.all(padding == 9.0)
        return got

    def check_bitwise(self):
        got = self.result()
        exp = torch.from_numpy(np.ascontiguousarray(self.exact)).to(TORCH[self.t])
        bad = (got != exp).nonzero()
        assert len(bad) == 0, (len(bad), bad[:5].tolist(), got[tuple(bad[0])], exp[tuple(bad[0])])

    def check_close(self):
        got = self.result().double().numpy()
        bound = (self.k + 2) * 2.0 ** -24 * self.size
        bound = bound + torch.finfo(TORCH[self.t]).eps / 2 * (np.abs(self.exact) + bound) + torch.finfo(TORCH[self.t]).smallest_normal
        assert np.all(np.abs(got - self.exact) <= bound), np.max(np.abs(got - self.exact) / bound)


SIZES = [(1, 1, 1), (1, 16, 32), (1, 300, 100), (2, 33, 257), (7, 64, 512), (16, 130, 96), (17, 48, 1000), (33, 200, 64),
         (64, 64, 160), (100, 257, 130), (130, 70, 520), (257, 300, 288)]


@pytest.mark.parametrize("side", ["right", "left"])
@pytest.mark.parametrize("layout", ["R", "C"])
@pytest.mark.parametrize("opA,opB", [("N", "N"), ("T", "N"), ("N", "T"), ("T", "T")])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_mixed_products_exact(cuda, t, opA, opB, layout, side):
    """Integers: every sum is exact (|x y| <= 4 * 6 * 2^3, k <= 1000), so the results are bitwise."""
    for i, (m, n, k) in enumerate(SIZES):
        if side == "left":
            m, n = n, m
        pad, off = (0, 8, 3)[i % 3], i % 2
        c = Case(cuda, side, m, n, k, t, layout, opA, opB, i, True, pad=pad, ro=off, co=32 * off)
        c.run()
        c.check_bitwise()


@pytest.mark.parametrize("layout", ["R", "C"])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_both_products_exact(cuda, t, layout):
    """|x y| <= 36 * 2^6 in quarters, k <= 1000: sums are multiples of 1/4 below 2^22."""
    for i, (m, n, k) in enumerate(SIZES):
        for mm, nn in ((m, n), (n, m)):
            c = Case(cuda, "both", mm, nn, k, t, layout, "N", "T", i, True, pad=(0, 8, 3)[i % 3], ro=i % 2, co=32 * (i % 2))
            c.run()
            c.check_bitwise()


@pytest.mark.parametrize("side,opA,opB", [("right", "N", "T"), ("right", "T", "N"), ("left", "N", "T"), ("both", "N", "T")])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("alpha,beta", [(1.0, 0.0), (0.5, 1.0), (-1.25, 0.75)])
@pytest.mark.parametrize("m,n,k", [(1, 513, 2100), (13, 200, 4096), (40, 120, 333), (200, 190, 1500)])
def test_products_close(cuda, m, n, k, alpha, beta, t, side, opA, opB):
    """Random numbers, scales 2^-7 .. 2^3, alpha and beta, within the bound of 32-bit sums."""
    c = Case(cuda, side, m, n, k, t, "R", opA, opB, m + k, False, alpha=alpha, beta=beta, low=120, high=130)
    c.run()
    c.check_close()


@pytest.mark.parametrize("m,n,k", [(1, 16390, 70), (9, 8200, 300), (16, 16384, 544), (20, 16390, 96), (32, 8195, 520),
                                   (5, 700, 5000), (31, 300, 9000)])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("opB", ["T", "N"])
def test_few_rows_exact(cuda, opB, t, m, n, k):
    """Few rows against wide and against long 4-bit matrices; |x y| <= 4 * 6 in halves, k <= 9000."""
    for side, layout in (("right", "R"), ("left", "C")):
        a, b = (m, n) if side == "right" else (n, m)
        ops = ("N", opB) if side == "right" else ("N" if opB == "T" else "T", "N")
        c = Case(cuda, side, a, b, k, t, layout, *ops, m, True, low=126, high=127)
        c.run()
        c.check_bitwise()


@pytest.mark.parametrize("side,t,opB,layout,m,n,k,pad", [
    ("right", "bf16", "T", "R", 4100, 4099, 200, 1),    # 256 x 256, rows of C at odd multiples of an element
    ("right", "bf16", "N", "C", 4100, 4100, 264, 0),
    ("left", "bf16", "T", "C", 4099, 4100, 264, 3),
    ("left", "bf16", "N", "R", 4100, 4100, 200, 4),
    ("right", "bf16", "T", "C", 2100, 4100, 300, 1),    # 256 x 128
    ("right", "f32", "N", "R", 2100, 4098, 136, 2),
    ("left", "f16", "T", "R", 4098, 2100, 300, 0),
    ("left", "f32", "N", "C", 4100, 2100, 328, 0),
    ("right", "bf16", "T", "R", 700, 1030, 2500, 3),    # 128 x 128, the contraction cut
    ("right", "f16", "N", "C", 700, 1001, 2500, 0),
    ("left", "f32", "T", "C", 1030, 700, 2500, 1),
    ("right", "bf16", "N", "R", 130, 260, 9000, 0),
    ("right", "bf16", "T", "R", 50, 4100, 300, 1),      # several groups of few rows
    ("right", "f16", "T", "C", 75, 900, 5000, 0),
    ("left", "f32", "T", "R", 64, 100, 3000, 1),
    ("right", "f32", "N", "R", 100, 600, 3000, 2),
    ("right", "bf16", "N", "R", 100, 90, 3000, 1),
    ("left", "f16", "T", "C", 100, 75, 2000, 3),
    ("right", "f16", "N", "C", 300, 300, 1000, 0),      # few tiles
    ("both", "f32", "T", "R", 4100, 4099, 300, 1),      # 256 x 256
    ("both", "bf16", "T", "C", 4099, 4100, 520, 0),
    ("both", "f16", "T", "R", 1050, 1060, 4500, 2),     # 128 x 128, the contraction cut
    ("both", "f32", "T", "C", 2090, 700, 8200, 1),
    ("both", "bf16", "T", "R", 260, 130, 9000, 0),      # small, the contraction cut
])
def test_every_kernel_exact(cuda, side, t, opB, layout, m, n, k, pad):
    """Each tile, orientation and split with edges in every direction. Scales 2^-1 and 2^0: a dense factor's
    products are at most 24 in quarters, two 4-bit factors' at most 36 in 1/16: sums of 9000 are exact."""
    ops = ("N", "T") if side == "both" else ("N", opB) if side == "right" else (opB, "N")
    c = Case(cuda, side, m, n, k, t, layout, *ops, m + n, True, alpha=0.5, beta=2.0, pad=pad, ro=1, co=32, low=126, high=127)
    c.run()
    c.check_bitwise()


@pytest.mark.parametrize("scale_pad", [0, 1, 3])
@pytest.mark.parametrize("side,opB", [("right", "T"), ("right", "N"), ("both", "T")])
def test_scales_of_any_alignment(cuda, side, opB, scale_pad):
    c = Case(cuda, side, 70, 150, 300, "bf16", "R", "N", opB, 3, True, scale_pad=scale_pad)
    c.run()
    c.check_bitwise()


@pytest.mark.parametrize("opB", ["T", "N"])
@pytest.mark.parametrize("m", [1, 20, 150])
def test_all_bits_of_the_dense_factor(cuda, m, opB):
    """A 4-bit factor with one +-2^e a column copies the dense one: every bit of 32 has to arrive, from
    subnormals to the largest numbers, and an infinity or a NaN stays in its row."""
    k = n = 96
    rng = np.random.default_rng(m)
    code = np.zeros((k, n), np.uint8)
    perm = rng.permutation(k)
    sign = rng.integers(0, 2, n)
    code[perm, np.arange(n)] = 2 + 8 * sign   # +-1
    q = code if opB == "N" else code.T
    scales = np.full((q.shape[0], 3), 127, np.uint8)
    Q = rb.MX4Matrix(*q.shape, torch.from_numpy(R.pack(np.ascontiguousarray(q))).to(cuda), torch.from_numpy(scales).to(cuda))
    bits = rng.integers(0, 2 ** 32, (m, k), dtype=np.uint64).astype(np.uint32)
    x = bits.view(np.float32).copy()
    x[~np.isfinite(x)] = 1.0
    x[np.abs(x) < 2.0 ** -110] = 3.0   # the third part of a smaller one is below the smallest 16-bit number
    x[0, 0], x[0, 1] = np.finfo(np.float32).max, -np.finfo(np.float32).max
    C = torch.empty(m * n, dtype=torch.float32, device=cuda)
    rb.mxmm("R", "N", opB, m, n, k, 1.0, torch.from_numpy(x).to(cuda).view(-1), k, Q, 0, 0, 0.0, C, n)
    exp = x[:, perm] * np.where(sign, np.float32(-1), np.float32(1))
    assert np.array_equal(C.cpu().numpy().reshape(m, n), exp)
    # an infinite entry: its row is +-inf in its column and NaN elsewhere (inf * 0), other rows are as before
    if m > 1:
        x[1, perm[5]] = np.inf
        rb.mxmm("R", "N", opB, m, n, k, 1.0, torch.from_numpy(x).to(cuda).view(-1), k, Q, 0, 0, 0.0, C, n)
        got = C.cpu().numpy().reshape(m, n)
        assert np.array_equal(np.delete(got, 1, 0), np.delete(exp, 1, 0))
        assert np.isinf(got[1, 5]) and np.all(np.isnan(np.delete(got[1], 5)))


@pytest.mark.parametrize("opB", ["T", "N"])
@pytest.mark.parametrize("m", [1, 20, 150, 600])
def test_smallest_numbers_of_the_dense_factor(cuda, m, opB):
    """f32 from the smallest subnormal to 2^-100, each times one +-2^90: what a number has from 2^-133 on arrives, cut
    towards 0. So all its bits from 2^-110 on, and below that the sum is off by less than 2^-133 times the 4-bit value."""
    k = n = 96
    rng = np.random.default_rng(m)
    code = np.zeros((k, n), np.uint8)
    perm = rng.permutation(k)
    sign = rng.integers(0, 2, n)
    code[perm, np.arange(n)] = 2 + 8 * sign
    q = np.ascontiguousarray(code if opB == "N" else code.T)
    Q = rb.MX4Matrix(*q.shape, torch.from_numpy(R.pack(q)).to(cuda), torch.from_numpy(np.full((q.shape[0], 3), 127 + 90, np.uint8)).to(cuda))
    x = rng.integers(1, 27 << 23, (m, k)).astype(np.uint32).view(np.float32)   # exponents to 2^-101
    x[:, ::5] = rng.integers(1, 1 << 23, (m, len(range(0, k, 5)))).astype(np.uint32).view(np.float32)   # subnormals
    x[rng.random((m, k)) < 0.5] *= np.float32(-1)
    C = torch.empty(m * n, dtype=torch.float32, device=cuda)
    rb.mxmm("R", "N", opB, m, n, k, 1.0, torch.from_numpy(x).to(cuda).view(-1), k, Q, 0, 0, 0.0, C, n)
    got = C.cpu().double().numpy().reshape(m, n)
    value = np.where(sign, -1.0, 1.0) * 2.0 ** 90
    exact, kept = x.astype(np.float64)[:, perm] * value, np.trunc(x.astype(np.float64)[:, perm] * 2.0 ** 133) * 2.0 ** -133 * value
    assert np.array_equal(got, kept)
    assert np.array_equal(got[np.abs(x[:, perm]) >= 2.0 ** -110], exact[np.abs(x[:, perm]) >= 2.0 ** -110])
    assert np.all(np.abs(got - exact) < 2.0 ** -133 * 2.0 ** 90)


@pytest.mark.parametrize("side,opB", [("right", "T"), ("right", "N"), ("both", "T")])
@pytest.mark.parametrize("m", [3, 140])
def test_nan_scale_reaches_its_outputs_only(cuda, m, side, opB):
    c = Case(cuda, side, m, 90, 200, "f32", "R", "N", opB, 4, True)
    Q = c.factors[-3] if side == "both" else c.factors[2]
    Q.scales[7, 2] = 255   # row 7, columns 64 .. 95
    c.run()
    got, exp = c.result().numpy(), c.exact.copy()
    if opB == "T":
        exp[:, 7] = np.nan
    else:
        exp[:, 64:90] = np.nan
    assert np.array_equal(np.isnan(got), np.isnan(exp))
    assert np.array_equal(got[~np.isnan(exp)], exp[~np.isnan(exp)].astype(np.float32))


@pytest.mark.parametrize("side,opA,opB", [("right", "N", "T"), ("right", "N", "N"), ("left", "N", "T"), ("left", "T", "N"),
                                          ("both", "N", "T")])
@pytest.mark.parametrize("m,n,k", [(3, 5, 1), (1, 70, 40), (40, 33, 100), (260, 700, 333), (700, 1030, 300), (20, 20, 9000)])
def test_window_inside_a_block(cuda, m, n, k, side, opA, opB):
    """Windows that end inside a block of wider matrices, at rows and columns that end inside them too: the
    block's further codes are of 2^127 (as a product infinite, times 0 a NaN) and do not count. Scales 2^0."""
    rng = np.random.default_rng(k)
    ro, co, more = 2, 64, 45

    def factor(rows, cols, op):
        r, c = (rows, cols) if op == "N" else (cols, rows)
        codes, scales = R.random_mx4(rng, r + ro + 3, c + co + more, 127, 127)
        if c % 32:
            scales[:, (co + c) // 32] = 255 - 1
            inside = R.random_mx4(rng, r + ro + 3, c + co, 127, 127)[0] * 0   # in the window's last block zeros
            a, b = (co + c) // 32 * 16, (co + c) // 2
            codes[:, a:b] = inside[:, a:b]
            if c % 2:
                codes[:, b] &= 0xF0
            codes[:, b + c % 2: a + 16] = 0x77
        Q = rb.MX4Matrix(r + ro + 3, c + co + more, torch.from_numpy(codes).to(cuda), torch.from_numpy(scales).to(cuda))
        v = R.values(codes, scales, c + co + more)[ro: ro + r, co: co + c]
        return Q, v if op == "N" else v.T

    def dense(rows, cols, op):
        x = rng.integers(-4, 5, (rows, cols)).astype(np.float64)
        buf, ld = stored(torch.from_numpy(x).float(), "R", op, 1, cuda)
        return buf, ld, x

    if side == "right":
        buf, ld, a = dense(m, k, opA)
        Q, b = factor(k, n, opB)
        args = (buf, ld, Q, ro, co)
    elif side == "left":
        Q, a = factor(m, k, opA)
        buf, ld, b = dense(k, n, opB)
        args = (Q, ro, co, buf, ld)
    else:
        QA, a = factor(m, k, opA)
        QB, b = factor(k, n, opB)
        args = (QA, ro, co, QB, ro, co)
    C = torch.full((m * n,), float("nan"), device=cuda)
    rb.mxmm("R", opA, opB, m, n, k, 1.0, *args, 0.0, C, n)
    assert np.array_equal(C.cpu().double().numpy().reshape(m, n), a @ b)


@pytest.mark.parametrize("m,n", [(3, 5), (64, 300), (700, 1030)])
def test_both_windows_inside_a_block(cuda, m, n):
    """Ordinary codes behind both windows, and behind one of them only."""
    rng = np.random.default_rng(m)
    for k, past_a, past_b in ((40, 24, 24), (335, 9, 200), (335, 0, 200), (335, 200, 0)):
        (ca, sa), (cb, sb) = (R.random_mx4(rng, r, k + past, 126, 128) for r, past in ((m, past_a), (n, past_b)))
        A, B = (rb.MX4Matrix(c.shape[0], k + past, torch.from_numpy(c).to(cuda), torch.from_numpy(s).to(cuda))
                for c, s, past in ((ca, sa, past_a), (cb, sb, past_b)))
        C = torch.full((m * n,), float("nan"), device=cuda)
        rb.mxmm("C", "N", "T", m, n, k, 1.0, A, 0, 0, B, 0, 0, 0.0, C, m)
        exp = R.values(ca, sa, k + past_a)[:, :k] @ R.values(cb, sb, k + past_b)[:, :k].T
        assert np.array_equal(C.cpu().double().numpy().reshape(n, m).T, exp)


@pytest.mark.parametrize("side", ["right", "left", "both"])
def test_alpha_zero_and_empty_contraction(cuda, side):
    """alpha = 0 or k = 0: C = beta C, factors unread (NaN in them does not show), beta = 0 writes zeros."""
    for k, alpha in ((64, 0.0), (0, 1.0)):
        for beta in (0.0, 2.0):
            c = Case(cuda, side, 5, 9, k, "f32", "C", "N", "T", 1, True, alpha=alpha, beta=beta, pad=2)
            if side != "both" and k:
                (c.factors[0] if side == "right" else c.factors[3]).fill_(float("nan"))
            c.run()
            c.check_bitwise()


def test_large_products_agree_with_64_bits(cuda):
    """Several tiles in each direction and a long contraction, 64-bit sums on the device."""
    for side, m, n, k, t, opB in (("right", 500, 1000, 4128, "bf16", "T"), ("right", 700, 900, 2000, "f32", "N"),
                                  ("both", 900, 1100, 4128, "f32", "T"), ("right", 16, 2048, 8192, "f16", "T")):
        c = Case(cuda, side, m, n, k, t, "R", "N", opB, 2, False, low=120, high=130)
        c.run()
        c.check_close()


@pytest.mark.parametrize("m", [2, 150])
@pytest.mark.parametrize("side,opB", [("right", "T"), ("right", "N"), ("both", "T")])
def test_products_of_extreme_scales(cuda, m, side, opB):
    """One E2M1 value a column under 2^-127 .. 2^125, times 1: exact, subnormal results included."""
    k, n = 64, 9 * 16
    scale = np.repeat(np.array([0, 1, 2, 60, 127, 200, 250, 251, 252]), 16)   # of a column
    code = np.zeros((n, k), np.uint8)
    code[:, 33] = np.tile(np.arange(16), 9)
    if opB == "T":
        q, s = code, np.full((n, 2), 127)
        s[:, 1] = scale
    else:   # a row's blocks hold 32 columns: the even blocks' columns get the lower of two scales
        q = np.ascontiguousarray(code.T)
        s = np.full((k, (n + 31) // 32), 127)
        s[33] = scale[::32][: s.shape[1]]
    Q = rb.MX4Matrix(*q.shape, torch.from_numpy(R.pack(np.pad(q, ((0, 0), (0, -q.shape[1] % 32))))).to(cuda),
                     torch.from_numpy(s.astype(np.uint8)).to(cuda))
    v = R.values(Q.codes.cpu().numpy(), s, q.shape[1])
    v = v.T if opB == "T" else v
    C = torch.empty(m * n, dtype=torch.float32, device=cuda)
    if side == "both":
        one = rb.MX4Matrix(m, k, torch.full((m, k // 2), 0x22, dtype=torch.uint8, device=cuda),
                           torch.full((m, 2), 127, dtype=torch.uint8, device=cuda))
        rb.mxmm("R", "N", "T", m, n, k, 1.0, one, 0, 0, Q, 0, 0, 0.0, C, n)
    else:
        x = torch.ones(m * k, dtype=torch.float32, device=cuda)
        rb.mxmm("R", "N", opB, m, n, k, 1.0, x, k, Q, 0, 0, 0.0, C, n)
    exp = np.broadcast_to(v.sum(0), (m, n)).astype(np.float32)
    assert np.array_equal(C.cpu().numpy().reshape(m, n), exp)


def infinite_case(rng, m, n, k, t, opB):
    """A dense m x k, codes and scales of a 4-bit k x n (after op): one code that counts a column, under a scale of
    2^123 .. 2^127; the dense entry it meets has one plane, all planes, or is 0 or an infinity."""
    special = np.array([1.0, -1.0, 0.0, 3.0, -0.75, 1.0 + 2.0 ** -10, -1.5 - 2.0 ** -9, np.inf, -np.inf, np.nan, 2.0 ** -14])
    if t == "f32":
        special = np.concatenate((special, [1.0 + 2.0 ** -23, -3.14159274, 2.0 ** -100, -2.0 ** -120]))
    x = rng.integers(-2, 3, (m, k)).astype(np.float64)
    at = rng.integers(0, k, n)
    x[:, np.unique(at)] = rng.choice(special, (m, len(np.unique(at))))
    for r in range(m):   # an infinity or a NaN meets every column of its row: in some rows only
        if r % 3:
            x[r, ~np.isfinite(x[r])] = 2.0
    code = np.zeros((k, n), np.uint8)
    code[at, np.arange(n)] = rng.integers(0, 16, n)
    q = np.ascontiguousarray(code if opB == "N" else code.T)
    scales = rng.integers(250, 255, (q.shape[0], (q.shape[1] + 31) // 32)).astype(np.uint8)
    return torch.from_numpy(x).to(TORCH[t]), R.pack(np.pad(q, ((0, 0), (0, -q.shape[1] % 32)))), scales


@pytest.mark.parametrize("side", ["right", "left"])
@pytest.mark.parametrize("opB", ["T", "N"])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m,n,k", [(1, 40, 64), (2, 16390, 100), (3, 300, 500), (16, 70, 4100), (30, 600, 333), (40, 200, 9000), (150, 260, 1000),
                                   (300, 700, 5000), (2100, 4100, 264)])
def test_infinite_values_of_a_4_bit_factor(cuda, m, n, k, t, opB, side):
    """4-bit values of 2^128 or more enter as infinities whatever the dense factor's type: infinite sums where 32-bit
    arithmetic has them, NaN where it multiplies them with 0. One product a sum that is not 0, so sums are exact."""
    rng = np.random.default_rng(m + n + k)
    x, codes, scales = infinite_case(rng, m, n, k, t, opB)
    Q = rb.MX4Matrix(codes.shape[0], n if opB == "N" else k, torch.from_numpy(codes).to(cuda), torch.from_numpy(scales).to(cuda))
    v = torch.from_numpy(R.values(codes, scales, Q.n_cols)).float()   # 2^128 and more: infinite
    v = (v if opB == "N" else v.t()).double().to(cuda)
    xd = x.double().to(cuda)
    code_at = (v != 0).double()
    # the one product that counts; a code of 0 counts where the dense entry is not finite
    bad = ((~xd.isfinite()).double() @ (1 - code_at)) > 0
    pick, col = code_at.max(0).values > 0, code_at.argmax(0)
    one = xd[:, col] * v[col, torch.arange(n, device=cuda)]
    exp = torch.where(pick, one, torch.zeros_like(one))
    exp[bad] = float("nan")
    exp = exp.float().to(TORCH[t])
    C = torch.full((m * n,), 5.0, dtype=TORCH[t], device=cuda)
    if side == "right":
        rb.mxmm("R", "N", opB, m, n, k, 1.0, x.to(cuda).view(-1), k, Q, 0, 0, 0.0, C, n)
    else:   # C^T = op(B)^T A^T
        rb.mxmm("R", "T" if opB == "N" else "N", "T", n, m, k, 1.0, Q, 0, 0, x.to(cuda).view(-1), k, 0.0, C, m)
    got = C.view(m, n) if side == "right" else C.view(n, m).t()
    wrong = ~((got == exp) | (got.isnan() & exp.isnan()))
    at = wrong.nonzero()[:5].tolist()
    assert not at, (int(wrong.sum()), [(i, j, float(got[i, j]), float(exp[i, j]), float(xd[i, col[j]]), float(v[col[j], j])) for i, j in at])
    assert m == 1 or bool(exp.isinf().any())   # row 0 keeps its infinities and NaN


@pytest.mark.parametrize("m,n,k", [(3, 144, 64), (150, 300, 500), (700, 1030, 300), (1050, 1060, 4500)])
def test_two_factors_of_extreme_scales(cuda, m, n, k):
    """Two 4-bit factors up to 2^127: products are exact, those of 2^128 or more infinite as 32-bit results, and those
    of a value of 2^128 or more and a small one finite."""
    rng = np.random.default_rng(k)
    code = np.zeros((n, -(-k // 32) * 32), np.uint8)
    at = rng.integers(0, k, n)
    code[np.arange(n), at] = rng.integers(0, 16, n)
    scales = rng.integers(250, 255, (n, code.shape[1] // 32)).astype(np.uint8)
    Q = rb.MX4Matrix(n, k, torch.from_numpy(R.pack(code)).to(cuda), torch.from_numpy(scales).to(cuda))
    small = rng.choice(np.array([100, 126, 127], np.uint8), (m, code.shape[1] // 32))
    ones = np.zeros((m, code.shape[1]), np.uint8)
    ones[:, :k] = 2
    P = rb.MX4Matrix(m, k, torch.from_numpy(R.pack(ones)).to(cuda), torch.from_numpy(small).to(cuda))
    C = torch.full((m * n,), 5.0, device=cuda)
    rb.mxmm("R", "N", "T", m, n, k, 1.0, P, 0, 0, Q, 0, 0, 0.0, C, n)
    with np.errstate(over="ignore"):
        exp = (R.values(R.pack(ones), small, k) @ R.values(R.pack(code), scales, k).T).astype(np.float32)
    assert np.array_equal(C.cpu().numpy().reshape(m, n), exp) and np.isinf(exp).any()


def test_two_streams_at_once(cuda):
    """Calls that need workspaces, in flight on two streams together, keep apart."""
    cases = [Case(cuda, "right", 150, 700, 2100, "f32", "R", "N", "T", 1, True, low=126, high=127),
             Case(cuda, "right", 300, 500, 3000, "f32", "R", "N", "N", 2, True, low=126, high=127),
             Case(cuda, "both", 700, 700, 2100, "f32", "R", "N", "T", 3, True, low=126, high=127)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = []
    for i in range(12):
        c = cases[i % 3]
        out = torch.full_like(c.C, float("nan"))
        outs.append((c, out))
    torch.cuda.synchronize()
    for i, (c, out) in enumerate(outs):
        rb.mxmm(*c.head, *c.factors, 0.0, out, c.ldc, stream=streams[(i // 3) % 2].cuda_stream)
    torch.cuda.synchronize()
    for c, out in outs:
        c.C = out
        c.check_bitwise()


def test_workspace_of_the_callers(cuda):
    """The C ABI: a query, a block that is large enough, one that is too small, one that is not aligned."""
    import ctypes

    c = Case(cuda, "right", 150, 300, 1100, "f32", "R", "N", "T", 5, True)
    buf, lda, Q, ro, co = c.factors
    fn, w = rb.lib.rbh_mxmm_right_f32, rb.WorkC()
    call = lambda: fn(b"R", b"N", b"T", 150, 300, 1100, 1.0, buf.data_ptr(), lda, Q._c, ro, co, 0.0, c.C.data_ptr(), c.ldc,
                      ctypes.byref(w), torch.cuda.current_stream().cuda_stream)
    assert call() == 0 and w.bytes > 0
    need = w.bytes
    block = torch.zeros(need + 512, dtype=torch.uint8, device=cuda)
    guard = block[need:].clone()
    w.ptr = block.data_ptr()
    assert call() == 0
    c.check_bitwise()
    assert torch.equal(block[need:], guard)   # nothing behind what was asked for
    w.bytes = need - 1
    assert call() != 0 and "work->bytes" in rb.lib.rbh_last_error().decode()
    w.bytes, w.ptr = need, block.data_ptr() + 16
    assert call() != 0
    host = np.zeros(need + 256, np.uint8)
    w.ptr = host.ctypes.data + (-host.ctypes.data % 256)
    assert call() != 0 and "work_here" in rb.lib.rbh_last_error().decode()


def test_another_stream(cuda):
    c = Case(cuda, "right", 150, 260, 500, "f32", "R", "N", "T", 6, True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.run()
    torch.cuda.current_stream().wait_stream(side)
    c.check_bitwise()
    c.new(cuda)
    torch.cuda.synchronize()
    c.run(stream=side.cuda_stream)
    c.check_bitwise()


@pytest.mark.parametrize("side,t,opB,m", [("right", "bf16", "T", 1), ("right", "f32", "T", 150), ("right", "f16", "N", 150),
                                          ("right", "f32", "N", 9), ("left", "f32", "T", 150), ("both", "bf16", "T", 150),
                                          ("both", "f32", "T", 5)])
def test_captured_and_replayed(cuda, side, t, opB, m):
    """Two graphs of the same stream, replayed in turn with eager calls and new inputs between them, share
    no workspace: every replay gives the eager result."""
    cases = [Case(cuda, side, m, 260, 1056, t, "R", "N", opB, s, True) for s in (1, 2)]
    st, graphs = torch.cuda.Stream(), []
    torch.cuda.synchronize()
    for c in cases:
        with torch.cuda.stream(st):
            c.run()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            c.run()
        graphs.append(g)
    other = torch.cuda.Stream()
    for rep in range(4):
        for c in cases:
            c.C.view(-1, c.ldc).fill_(float("nan") if rep % 2 else 3.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            graphs[0].replay()
        with torch.cuda.stream(other):
            graphs[1].replay()
        torch.cuda.synchronize()
        for c in cases:
            c.check_bitwise()
            c.run()
            c.check_bitwise()


@pytest.mark.parametrize("side,t,opB,m", [("right", "f32", "T", 150), ("right", "f16", "N", 150), ("right", "f32", "N", 9),
                                          ("both", "bf16", "T", 150)])
def test_captured_on_a_stream_of_the_callers(cuda, side, t, opB, m):
    """A capture that forks to a stream passed as stream=: the product's workspace is that stream's, so what the
    capturing stream allocates and writes beside the product does not meet it."""
    st, fork = torch.cuda.Stream(), torch.cuda.Stream()
    cases = [Case(cuda, side, m, 260, 1056, t, "R", "N", opB, s, True) for s in (1, 2)]
    for c in cases:
        c.run(stream=fork.cuda_stream)
        c.run(stream=st.cuda_stream)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        ahead = torch.zeros(1 << 26, dtype=torch.uint8, device=cuda)   # so that the fork's calls start beside the fills
        fork.wait_stream(torch.cuda.current_stream())
        cases[0].run(stream=fork.cuda_stream)
        beside = [torch.empty(n, dtype=torch.uint8, device=cuda).fill_(0xFF)
                  for n in (1 << 12, 1 << 14, 1 << 16, 1 << 18, 1 << 20, 1 << 22) for _ in range(4)]
        cases[1].run()
        again = [torch.empty_like(b).fill_(0xFE) for b in beside]
        cases[0].run(stream=fork.cuda_stream)
        torch.cuda.current_stream().wait_stream(fork)
    for rep in range(4):
        for c in cases:
            c.C.view(-1, c.ldc).fill_(float("nan") if rep % 2 else 3.0)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for c in cases:
            c.check_bitwise()
            c.run()
            c.check_bitwise()
        assert all(bool((b == 0xFF).all()) for b in beside) and all(bool((b == 0xFE).all()) for b in again)
        assert not ahead.any()


def test_capturing_stream_is_the_calls(cuda):
    """stream= captures and the current stream does not: a workspace of the graph's. The other way round, an eager
    call during a capture: the arena of its own stream."""
    st, eager = torch.cuda.Stream(), torch.cuda.Stream()
    a, b = (Case(cuda, "right", 150, 260, 1056, "f32", "R", "N", "T", s, True) for s in (1, 2))
    for c in (a, b):
        for s in (st, eager):
            c.run(stream=s.cuda_stream)
    torch.cuda.synchronize()
    a.new(cuda)
    b.new(cuda)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        b.run(stream=eager.cuda_stream)
        with torch.cuda.stream(eager):
            a.run(stream=st.cuda_stream)
    torch.cuda.synchronize()
    b.check_bitwise()
    for rep in range(3):
        a.C.fill_(9.0)
        b.C.fill_(9.0)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        a.check_bitwise()
        assert bool((b.C == 9.0).all())   # no part of the graph
        b.run()
        b.check_bitwise()


def test_captured_call_without_a_workspace_is_refused(cuda):
    """The C ABI without a caller's workspace, where the call needs one: an error, and the capture ends well."""
    import ctypes

    c = Case(cuda, "right", 150, 260, 1056, "f32", "R", "N", "T", 1, True)
    A, lda, Q = c.factors[:3]
    fn = rb.lib.rbh_mxmm_right_f32
    head = (b"R", b"N", b"T", 150, 260, 1056, 1.0, A.data_ptr(), lda, ctypes.byref(Q._c), 0, 0, 0.0, c.C.data_ptr(), c.ldc)
    work = rb.WorkC()
    assert fn(*head, ctypes.byref(work), None) == rb.RBH_OK
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        rc = fn(*head, None, st.cuda_stream)
        c.C.zero_()
    if work.bytes:
        assert rc == rb.RBH_ERR_REQUIRE
        small = rb.WorkC(A.data_ptr() // 256 * 256, work.bytes - 1)
        assert fn(*head, ctypes.byref(small), None) == rb.RBH_ERR_REQUIRE
    else:
        assert rc == rb.RBH_OK
    c.run()
    c.check_bitwise()


def test_host_arrays(cuda):
    """Host arrays are staged: the call is synchronous, windows are copied back."""
    rng = np.random.default_rng(0)
    a = rng.standard_normal((40, 70)).astype(np.float32)
    Q = rb.MX4Matrix(40, 70, np.full((40, 64), 7, np.uint8), np.full((40, 5), 7, np.uint8))
    if Q._c.codes % 16:
        pytest.skip("numpy gave an unaligned block")
    rb.mx4_quantize("R", "N", 40, 70, a.ravel(), 70, Q)
    code, scale = R.quantize(a.astype(np.float64))
    assert np.array_equal(Q.codes[:, :48], R.pack(code)) and np.array_equal(Q.scales[:, :3], scale)
    assert np.all(Q.codes[:, 48:] == 7) and np.all(Q.scales[:, 3:] == 7)
    x = rng.integers(-3, 4, (5, 70)).astype(np.float32)
    C = np.full((5, 44), 9.0, np.float32)
    rb.mxmm("R", "N", "T", 5, 40, 70, 1.0, x.ravel(), 70, Q, 0, 0, 0.0, C, 44)
    v = R.values(R.pack(code), scale, 70)
    bound = 72 * 2.0 ** -24 * (np.abs(x) @ np.abs(v.T)) * 1.01
    assert np.all(np.abs(C[:, :40] - x @ v.T) <= bound) and np.all(C[:, 40:] == 9.0)
    out = np.zeros((70, 40), np.float64)
    rb.mx4_dequantize("C", "N", 40, 70, Q, out, 40)
    assert np.array_equal(out.T, v)


def test_host_and_device_arrays_in_order(cuda):
    """On a stream of its own, behind a queue of work: what a host array is made from, or goes into, is on the device,
    and the call takes its turn there."""
    rng = np.random.default_rng(1)
    n, cols = 600, 2080
    a = torch.from_numpy(rng.integers(-6, 7, (n, cols)).astype(np.float32))
    a[:, ::32] = 6.0   # every block's scale is 1, every integer but 5 a value of its own
    a[a.abs() == 5] = 4.0
    there = a.to(cuda)
    x = rng.integers(-3, 4, (5, cols)).astype(np.float32)
    work = torch.randn(4096, 4096, device=cuda)
    late = torch.zeros_like(there)
    Q, P = rb.mx4_empty(n, cols, device=cuda), rb.mx4_empty(n, cols, device=cuda)
    Q.codes.zero_()
    Q.scales.zero_()
    P.codes.zero_()
    P.scales.zero_()
    torch.cuda.synchronize()
    out, C = np.zeros(n * cols, np.float32), np.zeros(5 * n, np.float32)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(20):
            work = torch.tanh(work @ work)
        late.copy_(there)
        rb.mx4_quantize("R", "N", n, cols, late.view(-1), cols, Q)
        rb.mx4_dequantize("R", "N", n, cols, Q, out, cols)   # device to host
        for _ in range(20):
            work = torch.tanh(work @ work)
        P.codes.fill_(0x11)
        P.scales.fill_(1)
        rb.mx4_quantize("R", "N", n, cols, a.numpy().ravel(), cols, P)   # host to device, behind the fills
        for _ in range(20):
            work = torch.tanh(work @ work)
        Q.codes.copy_(P.codes ^ 0x88)   # the signs
        rb.mxmm("R", "N", "T", 5, n, cols, 1.0, x.ravel(), cols, Q, 0, 0, 0.0, C, n)
    torch.cuda.synchronize()
    assert np.array_equal(out.reshape(n, cols), a.numpy())
    code, scale = R.quantize(a.double().numpy())
    assert np.array_equal(P.codes.cpu().numpy(), R.pack(code)) and np.array_equal(P.scales[:, : cols // 32].cpu().numpy(), scale)
    assert np.array_equal(C.reshape(5, n), -(x @ a.numpy().T))


@pytest.mark.parametrize("opB", ["T", "N"])
def test_gradient_of_the_dense_factor(cuda, opB):
    """C = A op(B): with G the gradient of C, A's is G op(B)^T, the product with op flipped. C is linear in
    A, so the difference quotient along D is the product of D itself; both are integers, hence exact."""
    m, n, k = 50, 180, 140
    rng = np.random.default_rng(3)
    Q, v = mx4(rng, *((n, k) if opB == "T" else (k, n)), cuda)
    a, d, g = (rng.integers(-3, 4, s).astype(np.float64) for s in ((m, k), (m, k), (m, n)))

    def product(x, rows, cols, inner, op):
        c = torch.empty(rows * cols, dtype=torch.float32, device=cuda)
        rb.mxmm("R", "N", op, rows, cols, inner, 1.0, torch.from_numpy(x).float().to(cuda).view(-1), inner, Q, 0, 0, 0.0, c, cols)
        return c.cpu().double().numpy().reshape(rows, cols)

    grad = product(g, m, k, n, "N" if opB == "T" else "T")
    assert np.array_equal(grad, g @ (v if opB == "T" else v.T))
    difference = product(a + d, m, n, k, opB) - product(a, m, n, k, opB)
    assert (g * difference).sum() == (grad * d).sum()


def test_run_together(cuda):
    """Two data matrices sketched by one operator, the sketches made 4-bit without bias, multiplied in 4
    bits, and the same product with one sketch kept in 32 bits: (S A1)^T (S A2)."""
    d, m, n1, n2 = 256, 1000, 90, 120
    rng = np.random.default_rng(1)
    S = rb.DenseSkOp(rb.DenseDist(d, m), rb.RNGState(7))
    B, Q, state = [], [], S.next_state
    for n in (n1, n2):
        A = torch.from_numpy(rng.standard_normal(m * n).astype(np.float32)).to(cuda)
        b = torch.empty(d * n, dtype=torch.float32, device=cuda)
        rb.sketch_general("C", "N", "N", d, n, m, 1.0, S, A, m, 0.0, b, d)
        q = rb.mx4_empty(n, d, device=cuda)
        state = rb.mx4_quantize("C", "T", n, d, b, d, q, rounding="stochastic", seed=state)   # op T: a sketch's columns
        B.append(b)
        Q.append(q)
    C = torch.empty(n1 * n2, dtype=torch.float32, device=cuda)
    rb.mxmm("C", "N", "T", n1, n2, d, 1.0 / d, Q[0], 0, 0, Q[1], 0, 0, 0.0, C, n1)
    M = torch.empty(n1 * n2, dtype=torch.float32, device=cuda)
    rb.mxmm("C", "T", "T", n1, n2, d, 1.0 / d, B[0], d, Q[1], 0, 0, 0.0, M, n1)
    b1, b2 = (b.cpu().double().numpy().reshape(n, d) for b, n in zip(B, (n1, n2)))
    q1, q2 = (R.values(q.codes.cpu().numpy(), q.scales.cpu().numpy()[:, : d // 32], d) for q in Q)
    for got, x, y in ((C, q1, q2), (M, b1, q2)):
        got = got.cpu().double().numpy().reshape(n2, n1).T
        assert np.all(np.abs(got - x @ y.T / d) <= (d + 2) * 2.0 ** -24 * (np.abs(x) @ np.abs(y.T)) / d + 1e-30)
    # the words of the second matrix follow those of the first
    at = list(S.next_state.counter)
    first = (at[0] + (at[1] << 32)) + n1 * (d // 4)
    code, scale = R.quantize(b2, R.philox_words(n2, d, 7, first))
    assert np.array_equal(Q[1].codes.cpu().numpy(), R.pack(code))
    # unbiased rounding: an element is off by less than a gap of its block (at most 2 units)
    unit = np.repeat(2.0 ** (scale.astype(np.float64) - 127), 32, 1)
    assert np.all(np.abs(q2 - b2) < 2 * unit)


def test_cpp_client(tmp_path):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    exe, libdir = str(tmp_path / "test_mx4"), os.path.join(root, "randblas_amd")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-I", os.path.join(root, "include"), "-I", "/opt/rocm/include",
                    "-D__HIP_PLATFORM_AMD__", os.path.join(root, "tests", "cpp", "test_mx4.cc"), "-L", libdir, "-lrandblas_hip",
                    "-L/opt/rocm/lib", "-lamdhip64", f"-Wl,-rpath,{libdir}", "-o", exe], check=True)
    out = subprocess.run([exe], capture_output=True, text=True, timeout=100)
    assert out.returncode == 0 and "ALL PASSED" in out.stdout, out.stdout + out.stderr
