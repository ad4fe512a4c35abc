"""Cases of the microscaled 4-bit operators: quantisation of a matrix, its inverse, and products with
4-bit matrices, each in a plain torch form and as calls of the framework.

A 4-bit matrix has one row of codes (two elements a byte, the even column in the low half) and one
scale a block of 32 columns. An element is sign, 2 exponent bits, 1 mantissa bit (0, 0.5, 1, 1.5, 2, 3,
4, 6 and their negatives); a scale is a power of two, stored as its exponent + 127.
"""
import math

import numpy as np
import torch

own = False

BLOCK = 32
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DTYPES = {"f64": torch.float64, "f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f64": 8, "f32": 4, "f16": 2, "bf16": 2}

# The limits of the drawn sizes, in elements (quantisation) and multiplications (products): no drawn
# case costs more than the largest listed one.
MOST_ELEMENTS = 8192 * 16384
MOST_PRODUCT = 8192 ** 3


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def listed():
    def quantise(name, rows, cols, dtype, layout="R", op="N", rounding="nearest"):
        return dict(name=name, kind="quantise", rows=rows, cols=cols, dtype=dtype, layout=layout, op=op,
                    rounding=rounding)

    def both(name, m, n, k, dtype, layout="R", beta=0.0):
        return dict(name=name, kind="both", m=m, n=n, k=k, dtype=dtype, layout=layout, beta=beta)

    def mixed(name, m, n, k, dtype, side="right", layout="R", opd="N", opq="T", beta=0.0):
        return dict(name=name, kind="mixed", m=m, n=n, k=k, dtype=dtype, side=side, layout=layout, opd=opd, opq=opq,
                    beta=beta)

    return [
        # the rows of a few tokens, made 4-bit before a product: a call that is all latency
        quantise("quantise rows", 16, 4096, "bf16"),
        # a weight matrix or a data matrix, once
        quantise("quantise matrix", 8192, 16384, "f32"),
        # a sketch d = 1024 of 16384 columns as sketch_general leaves it (ColMajor), blocks along its
        # columns (the other direction than its storage), rounded without bias
        quantise("quantise sketch", 1024, 16384, "f32", layout="C", rounding="stochastic"),
        # the same from a 64-bit sketch of odd size, blocks along the stored direction
        quantise("quantise odd sketch", 2999, 1013, "f64", layout="C", op="T", rounding="stochastic"),
        # both factors in 4 bits: a prompt's rows against a layer
        both("both large", 8192, 8192, 8192, "bf16"),
        # the approximate product of two data matrices from their sketches: (S A1)^T (S A2), d = 1024
        both("both sketches", 4096, 4096, 1024, "f32", layout="C"),
        # a small product of ragged sizes, added to what is there
        both("both ragged", 77, 1000, 2080, "f16", beta=1.0),
        # one token through a 4-bit layer
        mixed("one row", 1, 16384, 4096, "bf16"),
        # a batch of tokens through a 4-bit layer
        mixed("sixteen rows", 16, 4096, 16384, "bf16"),
        # a prompt through a 4-bit layer
        mixed("prompt", 4096, 8192, 4096, "bf16"),
        # the gradient of that layer's input: contracted along the rows of the 4-bit matrix
        mixed("gradient", 2048, 4096, 8192, "bf16", opq="N"),
        # a 4-bit data matrix times a 32-bit test matrix of odd width, ColMajor as this library's users keep it
        mixed("data times test matrix", 4096, 1001, 8192, "f32", side="left", layout="C", opq="N"),
    ]


def draw(rng):
    def size(lo, hi):
        v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        # half of the sizes are round, as most are in use
        if rng.random() < 0.5:
            step = 32 if v >= 256 else 8 if v >= 64 else 1
            v = max(step, v // step * step)
        return min(max(v, lo), hi)

    kind = rng.choice(["quantise", "both", "mixed"])
    if kind == "quantise":
        rows, cols = size(1, 32768), size(1, 32768)
        while rows * cols > MOST_ELEMENTS // 4:
            rows, cols = (rows + 1) // 2, cols
        return dict(kind=kind, rows=rows, cols=cols, dtype=rng.choice(["f64", "f32", "f16", "bf16"]),
                    layout=rng.choice("RC"), op=rng.choice("NT"), rounding=rng.choice(["nearest", "stochastic"]))
    k = size(32, 16384)
    if kind == "both":
        m, n = size(1, 8192), size(16, 16384)
    else:
        # few rows (answers) as often as many (prompts)
        m, n = size(1, 32) if rng.random() < 0.5 else size(33, 8192), size(16, 16384)
    while m * n * k > MOST_PRODUCT // 4:
        m, n, k = m, (n + 1) // 2, (k + 1) // 2
    case = dict(kind=kind, m=m, n=n, k=k, dtype=rng.choice(["f32", "f16", "bf16"]), layout=rng.choice("RC"),
                beta=rng.choice([0.0, 0.0, 1.0]))
    if kind == "mixed":
        side = rng.choice(["left", "right"])
        if side == "left":  # the dense factor's rows are the columns of the result
            case["m"], case["n"] = n, m
        case.update(side=side, opd=rng.choice("NT"), opq=rng.choice("NT"))
    return case


def _blocks(cols):
    return (cols + BLOCK - 1) // BLOCK


def _packed_bytes(rows, cols):
    return rows * _blocks(cols) * (BLOCK // 2 + 1)


def work(case):
    if case["kind"] == "quantise":
        n = case["rows"] * case["cols"]
        return {"bytes": 2 * n * SIZE[case["dtype"]] + _packed_bytes(case["rows"], case["cols"]), "flops": 0}
    m, n, k, e = case["m"], case["n"], case["k"], SIZE[case["dtype"]]
    out = m * n * e * (2 if case["beta"] else 1)
    if case["kind"] == "both":
        moved = _packed_bytes(m, k) + _packed_bytes(n, k)
    else:
        rows, cols = _mx_shape(case)
        moved = _packed_bytes(rows, cols) + (m * k if case["side"] == "right" else k * n) * e
    return {"bytes": moved + out, "flops": 2 * m * n * k}


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _dense(gen, rows, cols, dtype):
    """Gaussian entries, rows of different sizes and a few large columns, as activations, weights and
    sketches of real data have them."""
    a = torch.randn(rows, cols, generator=gen, device="cuda", dtype=torch.float32)
    a *= torch.exp2(torch.randint(-3, 4, (rows, 1), generator=gen, device="cuda").float())
    a *= torch.where(torch.rand(1, cols, generator=gen, device="cuda") < 0.01, 8.0, 1.0)
    if dtype == "f64":  # bits below the 32-bit ones too
        a = a.double() * (1 + 2.0 ** -30 * torch.rand(rows, 1, generator=gen, device="cuda", dtype=torch.float64))
    return a.to(DTYPES[dtype])


def _stored(a, layout, op):
    """The buffer that holds op(A) = a in `layout`, and its leading dimension."""
    t = a if (layout == "R") == (op == "N") else a.t()
    return t.contiguous().view(-1), max(1, t.shape[1])


def _mx_input(gen, rows, cols):
    """A 4-bit matrix in hand: codes (rows x 16 bytes a block) and scales (rows padded to whole 32-bit words)."""
    codes, scales = _pack(*_quantise_plain(_dense(gen, rows, cols, "f32"), "nearest", 0))
    wide = torch.zeros(rows, (scales.shape[1] + 3) // 4 * 4, dtype=torch.uint8, device="cuda")
    wide[:, : scales.shape[1]] = scales
    return codes, wide


def _mx_shape(case):
    """Rows and columns of the 4-bit factor of a mixed product."""
    inner, outer = case["k"], case["n"] if case["side"] == "right" else case["m"]
    # right factor: op(Q) is k x n; left factor: op(Q) is m x k
    straight = (case["side"] == "right") == (case["opq"] == "N")
    return (inner, outer) if straight else (outer, inner)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = dict(case)
    if case["kind"] == "quantise":
        a = _dense(gen, case["rows"], case["cols"], case["dtype"])
        state["A"], state["lda"] = _stored(a, case["layout"], case["op"])
        state["key"] = seed & 0xFFFFFFFF
        return state
    m, n, k = case["m"], case["n"], case["k"]
    if case["kind"] == "both":  # A: m x k, B: n x k, both with blocks along the contraction
        state["A"], state["B"] = _mx_input(gen, m, k), _mx_input(gen, n, k)
    else:
        d = _dense(gen, m, k, case["dtype"]) if case["side"] == "right" else _dense(gen, n, k, case["dtype"]).t()
        state["D"], state["ldd"] = _stored(d, case["layout"], case["opd"])
        state["Q"] = _mx_input(gen, *_mx_shape(case))
    state["alpha"] = 1.0 / math.sqrt(k)
    c = torch.randn(m, n, generator=gen, device="cuda", dtype=torch.float32).to(DTYPES[case["dtype"]])
    state["C"] = (c if case["layout"] == "R" else c.t()).contiguous().view(-1)
    return state


# ---------------------------------------------------------------------------------------------
# the plain form, in 32 bits (64 for 64-bit inputs)
# ---------------------------------------------------------------------------------------------
def _words(rows, cols, key):
    """32 random bits an element: word c % 4 of Philox4x32-10 at counter r * ceil(cols / 4) + c // 4."""
    quads = (cols + 3) // 4
    mask = 0xFFFFFFFF
    c0 = torch.arange(rows * quads, device="cuda", dtype=torch.int64)
    c0, c1, c2, c3 = c0 & mask, c0 >> 32, torch.zeros_like(c0), torch.zeros_like(c0)
    k0, k1 = key, 0
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((p1 >> 32) & mask) ^ c1 ^ k0, p1 & mask, ((p0 >> 32) & mask) ^ c3 ^ k1, p0 & mask
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    return torch.stack((c0, c1, c2, c3), 1).view(rows, quads * 4)


def _quantise_plain(a, rounding, key):
    """Codes (rows x padded columns) and scale exponents + 127 (rows x blocks) of a."""
    rows, cols = a.shape
    nb = _blocks(cols)
    x = torch.zeros(rows, nb * BLOCK, dtype=torch.float64 if a.dtype == torch.float64 else torch.float32, device="cuda")
    x[:, :cols] = a
    x = x.view(rows, nb, BLOCK)
    size = x.abs()
    top = size.amax(2)
    e = torch.frexp(top)[1] - 3  # floor(log2(top)) - 2
    if rounding == "stochastic":
        e = e + (top > torch.ldexp(torch.full_like(top, 6.0), e))
    e = torch.where(top == 0, -127, e).clamp(-127, 125)
    v = torch.ldexp(size, -e[:, :, None]).clamp(max=6.0)
    if rounding == "nearest":  # ties go to the even code: below 0.25, 1.25, 2.5 and 5, above 0.75, 1.75 and 3.5
        code = ((v > 0.25).byte() + (v >= 0.75).byte() + (v > 1.25).byte() + (v >= 1.75).byte() + (v > 2.5).byte()
                + (v >= 3.5).byte() + (v > 5.0).byte())
    else:
        grid = torch.tensor(GRID + (8.0,), dtype=x.dtype, device="cuda")
        code = torch.bucketize(v, grid[1:8], right=True)
        low = grid[code]
        part = (v - low) / (grid[code + 1] - low)
        words = torch.zeros(rows, nb * BLOCK, dtype=torch.int64, device="cuda")
        words[:, :cols] = _words(rows, cols, key)[:, :cols]
        code = code + (words.view(v.shape) < (part * 2.0 ** 32).to(torch.int64))
    code = code.byte() + 8 * torch.signbit(x).byte()
    return code.view(rows, nb * BLOCK), (e + 127).byte()


def _pack(code, scales):
    return code[:, 0::2] + 16 * code[:, 1::2], scales


def _values_plain(codes, scales, cols, dtype=torch.float32):
    """The matrix (rows x cols) that codes and scales stand for."""
    both = torch.stack((codes & 15, codes >> 4), 2).view(codes.shape[0], -1, BLOCK)
    table = torch.tensor(GRID + tuple(-g for g in GRID), dtype=dtype, device="cuda")
    v = torch.ldexp(table[both.int()], scales[:, : both.shape[1], None].int() - 127)
    return v.view(codes.shape[0], -1)[:, :cols]


def _matrix(buf, ld, rows, cols, layout, op):
    """op(A), rows x cols, of a buffer that holds A in `layout`."""
    straight = (layout == "R") == (op == "N")
    return buf.view(rows, ld) if straight else buf.view(cols, ld).t()


def _plain(s):
    if s["kind"] == "quantise":
        a = _matrix(s["A"], s["lda"], s["rows"], s["cols"], s["layout"], s["op"])
        codes, scales = _pack(*_quantise_plain(a, s["rounding"], s["key"]))
        dtype = torch.float64 if s["dtype"] == "f64" else torch.float32
        v = _values_plain(codes, scales, s["cols"], dtype).to(DTYPES[s["dtype"]])
        return _stored(v, s["layout"], s["op"])[0]
    m, n, k = s["m"], s["n"], s["k"]
    if s["kind"] == "both":
        p = _values_plain(*s["A"], k) @ _values_plain(*s["B"], k).t()
    else:
        rows, cols = _mx_shape(s)
        q = _values_plain(*s["Q"], cols)
        q = q if s["opq"] == "N" else q.t()
        if s["side"] == "right":
            p = _matrix(s["D"], s["ldd"], m, k, s["layout"], s["opd"]).float() @ q
        else:
            p = q @ _matrix(s["D"], s["ldd"], k, n, s["layout"], s["opd"]).float()
    p = s["alpha"] * p
    if s["beta"]:
        p = p + s["beta"] * (s["C"].view(m, n) if s["layout"] == "R" else s["C"].view(n, m).t()).float()
    return (p if s["layout"] == "R" else p.t()).to(DTYPES[s["dtype"]]).contiguous().view(-1)


# ---------------------------------------------------------------------------------------------
# the framework's operators
# ---------------------------------------------------------------------------------------------
def _framework(s):
    import randblas_amd as rb

    layout = s["layout"]
    if s["kind"] == "quantise":
        q = rb.mx4_empty(s["rows"], s["cols"], device="cuda")
        seed = rb.RNGState(s["key"]) if s["rounding"] == "stochastic" else None
        rb.mx4_quantize(layout, s["op"], s["rows"], s["cols"], s["A"], s["lda"], q, rounding=s["rounding"], seed=seed)
        out = torch.empty_like(s["A"])
        rb.mx4_dequantize(layout, s["op"], s["rows"], s["cols"], q, out, s["lda"])
        return out
    m, n, k = s["m"], s["n"], s["k"]
    c = s["C"].clone() if s["beta"] else torch.empty_like(s["C"])
    ldc = n if layout == "R" else m
    if s["kind"] == "both":
        a, b = rb.MX4Matrix(m, k, *s["A"]), rb.MX4Matrix(n, k, *s["B"])
        rb.mxmm(layout, "N", "T", m, n, k, s["alpha"], a, 0, 0, b, 0, 0, s["beta"], c, ldc)
    elif s["side"] == "right":
        q = rb.MX4Matrix(*_mx_shape(s), *s["Q"])
        rb.mxmm(layout, s["opd"], s["opq"], m, n, k, s["alpha"], s["D"], s["ldd"], q, 0, 0, s["beta"], c, ldc)
    else:
        q = rb.MX4Matrix(*_mx_shape(s), *s["Q"])
        rb.mxmm(layout, s["opq"], s["opd"], m, n, k, s["alpha"], q, 0, 0, s["D"], s["ldd"], s["beta"], c, ldc)
    return c


def run(state):
    return _framework(state) if own else _plain(state)


# ---------------------------------------------------------------------------------------------
# 64 bits, from the definitions
# ---------------------------------------------------------------------------------------------
def _exact_words(rows, cols, key):
    """The same random bits from 64-bit unsigned integers."""
    u = np.uint64
    quads = (cols + 3) // 4
    index = np.arange(rows * quads, dtype=u)
    x = [index & u(0xFFFFFFFF), index >> u(32), np.zeros_like(index), np.zeros_like(index)]
    with np.errstate(over="ignore"):
        for r in range(10):
            k0 = u((key + r * 0x9E3779B9) % 2 ** 32)
            k1 = u((r * 0xBB67AE85) % 2 ** 32)
            a, b = u(0xD2511F53) * x[0], u(0xCD9E8D57) * x[2]
            x = [(b >> u(32)) ^ x[1] ^ k0, b & u(0xFFFFFFFF), (a >> u(32)) ^ x[3] ^ k1, a & u(0xFFFFFFFF)]
    w = np.stack(x, 1).reshape(rows, quads * 4)[:, :cols].astype(np.float64)
    return torch.from_numpy(w).cuda()


def _exact_round(a, rounding, key):
    """The values that a's entries are rounded to, by the spacing of the 4-bit numbers around each entry."""
    rows, cols = a.shape
    a = a.double()
    pad = torch.nn.functional.pad(a, (0, -cols % BLOCK)).view(rows, -1, BLOCK)
    top = pad.abs().amax(2, keepdim=True)
    e = torch.floor(torch.log2(top.clamp(min=2.0 ** -1000)))
    # log2 of a number just below a power of two may round up to it
    e = e - (torch.exp2(e) > top).double() - 2
    if rounding == "stochastic":
        e = e + (top * torch.exp2(-e) > 6).double()
    unit = torch.exp2(e.clamp(-127, 125)).expand_as(pad).reshape(rows, -1)[:, :cols]
    v = (a / unit).abs().clamp(max=6.0)
    step = torch.where(v < 2, 0.5, torch.where(v < 4, 1.0, 2.0)).double()
    if rounding == "nearest":
        r = torch.round(v / step) * step  # halves go to the even multiple
    else:
        low = torch.floor(v / step)
        r = (low + (_exact_words(rows, cols, key) < torch.floor((v / step - low) * 2.0 ** 32)).double()) * step
    return torch.copysign(r, a) * unit


def _exact_values(codes, scales, cols):
    """sign * (1 + m / 2) * 2^(e - 1), or sign * m / 2 where e = 0, times the block's scale."""
    b = codes.to(torch.int64)
    c = torch.empty(b.shape[0], 2 * b.shape[1], dtype=torch.int64, device="cuda")
    c[:, 0::2], c[:, 1::2] = b % 16, b // 16
    s, e, f = 1.0 - 2.0 * (c // 8), (c // 2) % 4, (c % 2).double()
    mag = torch.where(e == 0, f / 2, (1 + f / 2) * torch.exp2(e.double() - 1))
    scale = torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, 1)[:, : c.shape[1]]
    return (s * mag * scale)[:, :cols]


def exact(case, seed):
    s = prepare(case, seed)
    lay = case["layout"]
    if case["kind"] == "quantise":
        stored = s["A"].view(-1, s["lda"])
        a = stored if (lay == "R") == (case["op"] == "N") else stored.t()
        v = _exact_round(a, case["rounding"], s["key"])
        return (v if (lay == "R") == (case["op"] == "N") else v.t()).contiguous().view(-1)
    m, n, k = case["m"], case["n"], case["k"]
    if case["kind"] == "both":
        p = torch.matmul(_exact_values(*s["A"], k), _exact_values(*s["B"], k).t().contiguous())
    else:
        d = s["D"].view(-1, s["ldd"]).double()
        d = d if (lay == "R") == (case["opd"] == "N") else d.t().contiguous()
        q = _exact_values(*s["Q"], _mx_shape(case)[1])
        q = q if case["opq"] == "N" else q.t().contiguous()
        p = torch.matmul(d, q) if case["side"] == "right" else torch.matmul(q, d)
    p = s["alpha"] * p
    c = s["C"].double()
    if case["beta"]:
        p = p + case["beta"] * (c.view(m, n) if lay == "R" else c.view(n, m).t())
    return (p if lay == "R" else p.t()).contiguous().view(-1)
