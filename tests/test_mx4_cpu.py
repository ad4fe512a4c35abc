"""CPU tests of the 4-bit microscaled operators: the reference itself, the handle and every refusal of the
C ABI (all of them come before any GPU work)."""
import ctypes

import os
import subprocess

import numpy as np
import pytest

import mx4_reference as R
import oracle_lib as O
import randblas_amd as rb


def handle(rows, cols, ld_codes=None, ld_scales=None):
    nb = (cols + 31) // 32
    codes = np.zeros((rows, ld_codes or max(16, 16 * nb)) if rows else (0, 16), np.uint8)
    # numpy aligns large arrays only to 16 bytes; take an aligned start in a larger block
    block = np.zeros(codes.size + 64, np.uint8)
    start = -block.ctypes.data % 64
    codes = block[start:start + codes.size].reshape(codes.shape)
    return rb.MX4Matrix(rows, cols, codes, np.zeros((rows, ld_scales or max(1, nb)), np.uint8))


def refused(fragment, fn, *args, **kw):
    with pytest.raises(rb.RandBLASError) as ei:
        fn(*args, **kw)
    assert ei.value.code == rb.RBH_ERR_REQUIRE and fragment in str(ei.value), str(ei.value)


def test_reference_rounds_to_nearest_even():
    x = np.zeros((1, 32))
    x[0, :16] = [6, 0.25, 0.26, 0.75, 0.74, 1.25, 1.26, 1.75, 2.5, 2.51, 3.5, 3.49, 5, 5.01, -0.25, -5]
    code, scale = R.quantize(x)
    assert scale[0, 0] == 127
    got = R.values(R.pack(code), scale, 32)[0, :16]
    assert got.tolist() == [6, 0, 0.5, 1, 0.5, 1, 1.5, 2, 2, 3, 4, 3, 4, 6, 0, -4]
    assert np.signbit(got[14])


def test_reference_words_are_the_oracles_philox():
    w = R.philox_words(3, 10, 77)
    for r, c in ((0, 0), (1, 3), (2, 9)):
        assert w[r, c] == O.philox([r * 3 + c // 4, 0, 0, 0], [77, 0])[c % 4]


def test_reference_stochastic_rounding_has_the_right_mean():
    # 4096 rows of one row: the mean of a value between neighbours `gap` apart is off by at most
    # 6 standard deviations of gap / 2 / sqrt(4096)
    row = np.linspace(-7.3, 7.9, 32)
    x = np.tile(row, (4096, 1))
    code, scale = R.quantize(x, R.philox_words(4096, 32, 5))
    mean = R.values(R.pack(code), scale, 32).mean(0)
    unit = 2.0 ** (int(scale[0, 0]) - 127)
    assert np.abs(np.abs(row) / unit).max() <= 6
    gap = np.where(np.abs(row) / unit < 2, 0.5, np.where(np.abs(row) / unit < 4, 1.0, 2.0)) * unit
    assert np.all(np.abs(mean - row) <= 6 * gap / 2 / 64)


def test_two_stochastic_roundings_have_the_right_mean_of_squares():
    """The mean of q1 q2 is x^2 for two roundings with words of their own; q1 q1 has the variance besides. Means of 4096
    rows within 6 standard deviations of the differences from x^2, at most those of gap / 2 times twice the value and gap."""
    rows, row = 4096, np.random.default_rng(2).standard_normal(32)
    x = np.tile(row, (rows, 1))
    q1, q2 = (R.values(R.pack(c), s, 32) for c, s in (R.quantize(x, R.philox_words(rows, 32, 5, at)) for at in (0, rows * 8)))
    unit = 2.0 ** np.floor(np.log2(np.abs(row).max() / 6) + 1)
    gap = np.where(np.abs(row) / unit < 2, 0.5, np.where(np.abs(row) / unit < 4, 1.0, 2.0)) * unit
    low = np.floor(np.abs(row) / gap) * gap
    variance = (np.abs(row) - low) * (low + gap - np.abs(row))
    off = 6 * (np.abs(row) * gap + gap * gap) / np.sqrt(rows)
    assert np.all(np.abs((q1 * q2).mean(0) - row * row) <= off)
    assert np.all(np.abs((q1 * q1).mean(0) - row * row - variance) <= off)
    assert ((q1 * q1).mean(0) - row * row).sum() > 0.9 * variance.sum() > 0.01 * (row * row).sum()


@pytest.mark.parametrize("t", ["f64", "f32"])
def test_quantize_refusals(t):
    dt = np.float64 if t == "f64" else np.float32
    A = np.zeros(40 * 70, dt)
    q = rb.mx4_quantize
    refused("layout == 'C' || layout == 'R'", q, "X", "N", 40, 70, A, 70, handle(40, 70))
    refused("op == 'N' || op == 'T'", q, "R", "C", 40, 70, A, 70, handle(40, 70))
    refused("n_rows >= 0", q, "R", "N", -1, 70, A, 70, handle(40, 70))
    refused("lda >=", q, "R", "N", 40, 70, A, 69, handle(40, 70))
    refused("lda >=", q, "C", "N", 40, 70, A, 39, handle(40, 70))
    refused("lda >=", q, "R", "T", 40, 70, A, 39, handle(40, 70))
    refused("Q->n_rows == n_rows", q, "R", "N", 40, 70, A, 70, handle(41, 70))
    refused("n_cols >= (n_cols)", q, "R", "N", 40, 70, A, 70, handle(40, 69))
    refused("ld_codes % 16 == 0", q, "R", "N", 40, 70, A, 70, handle(40, 70, ld_codes=56))
    refused("A != nullptr", q, "R", "N", 40, 70, Null(dt), 70, handle(40, 70))
    with pytest.raises(ValueError):
        q("R", "N", 40, 70, A, 70, handle(40, 70), rounding="up")
    with pytest.raises(ValueError):
        q("R", "N", 40, 70, A, 70, handle(40, 70), rounding="stochastic")
    with pytest.raises(TypeError):
        q("R", "N", 40, 70, np.zeros(2800, np.int32), 70, handle(40, 70))


class Null:
    """An array of a type whose address is NULL."""

    def __init__(self, dtype):
        self.dtype = np.dtype(dtype)

    def data_ptr(self):
        return 0


def test_quantize_refusals_of_the_c_abi():
    A = np.zeros(64, np.float32)
    Q = handle(2, 32)
    fn = rb.lib.rbh_mx4_quantize_f32
    head = (b"R", b"N", 2, 32, A.ctypes.data, 32)
    assert fn(*head, None, 0, None, None, None) == rb.RBH_ERR_REQUIRE
    assert fn(*head, ctypes.byref(Q._c), 2, None, None, None) == rb.RBH_ERR_REQUIRE
    assert fn(*head, ctypes.byref(Q._c), 1, None, None, None) == rb.RBH_ERR_REQUIRE
    seed = rb.RNGState(1).c()
    seed.rng = 7
    assert fn(*head, ctypes.byref(Q._c), 1, ctypes.byref(seed), None, None) == rb.RBH_ERR_REQUIRE
    for change in (dict(codes=Q._c.codes + 8), dict(codes=None), dict(scales=None), dict(ld_codes=0),
                   dict(ld_codes=1 << 24), dict(ld_scales=0), dict(ld_scales=1 << 24), dict(n_rows=-1)):
        c = rb.MX4MatrixC(2, 32, Q._c.codes, 16, Q._c.scales, 1)
        for k, v in change.items():
            setattr(c, k, v)
        assert fn(*head, ctypes.byref(c), 0, None, None, None) == rb.RBH_ERR_REQUIRE, change


def test_dequantize_refusals():
    A = np.zeros(40 * 70, np.float32)
    d = rb.mx4_dequantize
    refused("layout == 'C'", d, "x", "N", 40, 70, handle(40, 70), A, 70)
    refused("lda >=", d, "R", "N", 40, 70, handle(40, 70), A, 69)
    refused("n_rows - (n_rows) >= (ro)", d, "R", "N", 40, 70, handle(40, 70), A, 70, ro=1)
    refused("n_cols - (n_cols) >= (co)", d, "R", "N", 40, 70, handle(40, 70), A, 70, co=32)
    refused("(co) % 32 == 0", d, "R", "N", 40, 8, handle(40, 70), A, 70, co=16)
    refused("(ro) >= 0", d, "R", "N", 40, 8, handle(40, 70), A, 70, ro=-1)
    refused("A != nullptr", d, "R", "N", 40, 70, handle(40, 70), Null(np.float32), 70)


def test_product_refusals():
    A, C = np.zeros(5 * 64, np.float32), np.zeros(5 * 9, np.float32)
    B = handle(9, 64)
    mm = rb.mxmm
    refused("layout == 'C'", mm, "x", "N", "T", 5, 9, 64, 1.0, A, 64, B, 0, 0, 0.0, C, 9)
    refused("opA == 'N'", mm, "R", "x", "T", 5, 9, 64, 1.0, A, 64, B, 0, 0, 0.0, C, 9)
    refused("opB == 'N'", mm, "R", "N", "x", 5, 9, 64, 1.0, A, 64, B, 0, 0, 0.0, C, 9)
    refused("m >= 0", mm, "R", "N", "T", -5, 9, 64, 1.0, A, 64, B, 0, 0, 0.0, C, 9)
    refused("ldc >=", mm, "R", "N", "T", 5, 9, 64, 1.0, A, 64, B, 0, 0, 0.0, C, 8)
    refused("ldd >=", mm, "R", "N", "T", 5, 9, 64, 1.0, A, 63, B, 0, 0, 0.0, C, 9)
    refused("n_cols - (cols_B) >= (co_b)", mm, "R", "N", "T", 5, 9, 64, 1.0, A, 64, B, 0, 32, 0.0, C, 9)
    refused("n_rows - (rows_B) >= (ro_b)", mm, "R", "N", "T", 5, 9, 64, 1.0, A, 64, B, 1, 0, 0.0, C, 9)
    refused("(co_b) % 32 == 0", mm, "R", "N", "T", 5, 9, 32, 1.0, A, 64, B, 0, 8, 0.0, C, 9)
    refused("n_rows - (rows_A) >= (ro_a)", mm, "R", "N", "N", 10, 5, 64, 1.0, B, 0, 0, A, 5, 0.0, np.zeros(50, np.float32), 5)
    refused("D != nullptr", mm, "R", "N", "T", 5, 9, 64, 1.0, Null(np.float32), 64, B, 0, 0, 0.0, C, 9)
    refused("opA == 'N' && opB == 'T'", mm, "R", "N", "N", 9, 64, 9, 1.0, handle(9, 9), 0, 0, B, 0, 0, 0.0,
            np.zeros(9 * 64, np.float32), 64)
    # sizes beyond what offsets of 32 bits and the grids reach; offsets whose sum with a size would wrap
    big = 2 ** 28 + 1
    refused("m <= (1 << 28)", mm, "R", "N", "T", big, 9, 64, 1.0, A, 64, B, 0, 0, 0.0, C, 9)
    refused("n <= (1 << 28)", mm, "R", "N", "T", 5, big, 64, 1.0, A, 64, B, 0, 0, 0.0, C, big)
    refused("k <= (1 << 21)", mm, "R", "N", "T", 5, 9, 2 ** 21 + 1, 1.0, A, 2 ** 21 + 1, B, 0, 0, 0.0, C, 9)
    refused("n_rows - (rows_B) >= (ro_b)", mm, "R", "N", "T", 5, 9, 64, 1.0, A, 64, B, 2 ** 63 - 1, 0, 0.0, C, 9)
    refused("n_cols - (cols_B) >= (co_b)", mm, "R", "N", "T", 5, 9, 64, 1.0, A, 64, B, 0, 2 ** 63 - 32, 0.0, C, 9)
    with pytest.raises(TypeError):   # no 64-bit products
        mm("R", "N", "T", 5, 9, 64, 1.0, A.astype(np.float64), 64, B, 0, 0, 0.0, C.astype(np.float64), 9)
    with pytest.raises(TypeError):   # one type
        mm("R", "N", "T", 5, 9, 64, 1.0, A.astype(np.float16), 64, B, 0, 0, 0.0, C, 9)
    with pytest.raises(TypeError):   # a 4-bit factor
        mm("R", "N", "T", 5, 9, 64, 1.0, A, 64, A, 0, 0, 0.0, C, 9)


class OnDevice:
    """What the calls ask of a tensor on device 3 (never read: the C entry is replaced)."""

    is_cuda = True
    device = type("device", (), {"index": 3})

    def __init__(self, dtype):
        self.dtype = dtype

    def data_ptr(self):
        return 1 << 40


@pytest.mark.parametrize("place", range(5))
def test_stream_is_that_of_any_device_array(monkeypatch, place):
    """Host and device arrays in one call: the current stream of the device array's device, whichever it is."""
    torch = pytest.importorskip("torch")
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 1000 + i, raising=False)
    seen = []
    entry = lambda *args: seen.append(args[-1]) or 0
    monkeypatch.setattr(rb, "_captures", lambda stream: False, raising=False)
    for table in (rb._MX4_QUANTIZE, rb._MX4_DEQUANTIZE, rb._MXMM):
        for key in table:
            monkeypatch.setitem(table, key, entry)

    def matrix(codes, scales):
        Q = handle(9, 64)
        object.__setattr__(Q, "codes", OnDevice(torch.uint8) if codes else Q.codes)
        object.__setattr__(Q, "scales", OnDevice(torch.uint8) if scales else Q.scales)
        return Q

    def dense(here):
        return OnDevice(torch.float32) if here else torch.zeros(9 * 64)

    at = [i == place for i in range(5)]
    if place < 3:
        rb.mx4_quantize("R", "N", 9, 64, dense(at[0]), 64, matrix(at[1], at[2]))
        rb.mx4_dequantize("R", "N", 9, 64, matrix(at[1], at[2]), dense(at[0]), 64)
    if place < 4:
        rb.mxmm("R", "N", "T", 5, 9, 64, 1.0, dense(at[1]), 64, matrix(at[2], at[3]), 0, 0, 0.0, dense(at[0]), 9)
        rb.mxmm("R", "N", "N", 9, 5, 64, 1.0, matrix(at[2], at[3]), 0, 0, dense(at[1]), 5, 0.0, dense(at[0]), 5)
    rb.mxmm("R", "N", "T", 9, 9, 64, 1.0, matrix(at[1], at[2]), 0, 0, matrix(at[3], at[4]), 0, 0, 0.0, dense(at[0]), 9)
    assert seen and seen == [1003] * len(seen)
    rb.mx4_dequantize("R", "N", 9, 64, matrix(True, True), dense(False), 64, stream=7)
    assert seen[-1] == 7
    rb.mx4_dequantize("R", "N", 9, 64, matrix(False, False), dense(False), 64)
    assert seen[-1] is None


def test_null_result_is_refused():
    A, B = np.zeros(5 * 64, np.float32), handle(9, 64)
    refused("C != nullptr", rb.mxmm, "R", "N", "T", 5, 9, 64, 1.0, A, 64, B, 0, 0, 0.0, Null(np.float32), 9)


def test_handle_checks_its_arrays():
    ok = np.zeros((4, 48), np.uint8)
    with pytest.raises(TypeError):
        rb.MX4Matrix(4, 70, ok.astype(np.int8), ok)
    with pytest.raises(TypeError):
        rb.MX4Matrix(4, 70, ok.ravel(), ok)
    with pytest.raises(ValueError):
        rb.MX4Matrix(4, 97, ok, ok)
    with pytest.raises(ValueError):
        rb.MX4Matrix(5, 70, ok, np.zeros((5, 3), np.uint8))
    with pytest.raises(ValueError):
        rb.MX4Matrix(4, 70, ok, np.zeros((4, 2), np.uint8))
    with pytest.raises(ValueError):
        rb.MX4Matrix(4, 20, np.zeros((4, 64), np.uint8)[:, ::2], ok)
    assert rb.MX4Matrix(4, 70, np.zeros((4, 64), np.uint8), ok)._c.ld_codes == 64
    one = np.zeros((1, 16), np.uint8)[:, :16]
    assert rb.MX4Matrix(1, 32, one, one)._c.ld_codes == 16


def test_next_state_of_stochastic_rounding_carries():
    # an empty matrix reads no words and needs no GPU
    st = rb.mx4_quantize("R", "N", 0, 70, np.zeros(0, np.float32), 70, handle(0, 70), rounding="stochastic",
                         seed=rb.RNGState(3, counter=(5, 0, 0, 0)))
    assert st.counter == (5, 0, 0, 0) and st.key == 3


@pytest.mark.parametrize("m,n,k", [(0, 9, 64), (5, 0, 64), (0, 0, 0)])
def test_empty_products(m, n, k):
    C = np.full(64, 7.0, np.float32)
    rb.mxmm("R", "N", "T", m, n, k, 1.0, np.zeros(512, np.float32), max(k, 1), handle(n, k), 0, 0, 0.0, C, max(n, 1))
    assert np.all(C == 7.0)


@pytest.mark.parametrize("std", ["c++17", "c++20"])
def test_cpp_client_compiles_and_links(tmp_path, std):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    libdir = os.path.join(root, "randblas_amd")
    r = subprocess.run(["g++", f"-std={std}", "-O1", "-Wall", "-Werror", "-I", os.path.join(root, "include"), "-I", "/opt/rocm/include",
                        "-D__HIP_PLATFORM_AMD__", os.path.join(root, "tests", "cpp", "test_mx4.cc"), "-L", libdir, "-lrandblas_hip",
                        "-L/opt/rocm/lib", "-lamdhip64", f"-Wl,-rpath,{libdir}", "-o", str(tmp_path / "t")],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
