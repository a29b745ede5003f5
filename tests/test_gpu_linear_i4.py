"""4-bit linears on gfx950 against the plain formula in 64 bits.

The bound on an output: a product carries 22 significant bits (2^-22), and its
sum passes at most 32 additions inside a matrix instruction, 8 of those into a
group, then the row's groups and 8 waves, each addition off by at most 2^-23 of
the terms' magnitudes (a matrix core may truncate); what of an input lies 2^-39
below the largest of its 128 may be lost; and the result is rounded once to its
type."""
import ctypes

import numpy as np
import pytest

import esm_gfx950 as eg
from conftest import rng
from esm_gfx950 import synthetic as syn

pytestmark = pytest.mark.gpu

TYPES = {"fp32": eg.F32, "fp16": eg.F16, "bf16": eg.BF16}
HALF_STEP = {"fp32": 2.0 ** -24, "fp16": 2.0 ** -11, "bf16": 2.0 ** -8}


def to_bits(x, kind):
    """fp32 values as the type's array (bf16: uint16 bits, nearest even)."""
    if kind == "fp32":
        return np.ascontiguousarray(x, np.float32)
    if kind == "fp16":
        return x.astype(np.float16)
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    nan = np.isnan(x)
    u = (u + 0x7FFF + ((u >> 16) & 1)) >> 16
    return np.where(nan, 0x7FC0, u).astype(np.uint16)


def to_f64(a, kind):
    if kind == "bf16":
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


def empty_as(kind, shape, fill):
    return np.full(shape, fill, np.uint16 if kind == "bf16" else np.float16 if kind == "fp16" else np.float32)


class At:
    """A device pointer some bytes into an array."""

    def __init__(self, array, offset):
        self.array, self.ptr = array, ctypes.c_void_p(array.ptr.value + offset)


def decode(packed, scales, K, group):
    codes = np.empty((packed.shape[0], packed.shape[1] * 2), np.float64)
    codes[:, 0::2] = (packed & 15).astype(np.float64) - 8
    codes[:, 1::2] = (packed >> 4).astype(np.float64) - 8
    return codes[:, :K] * np.repeat(scales.astype(np.float64), group, axis=1)[:, :K]


def tolerance(x, w, y, kind):
    K = x.shape[1]
    tiles = (K + 127) // 128
    padded = np.zeros((x.shape[0], tiles * 128))
    padded[:, :K] = np.abs(x)
    amax = np.repeat(padded.reshape(-1, tiles, 128).max(axis=2), 128, axis=1)[:, :K]
    depth = 32 + 8 + 4 * tiles + 8
    fixed = 2.0 ** -22 + depth * 2.0 ** -23
    tiny = 2.0 ** -25 if kind == "fp16" else 2.0 ** -39  # fp16 inputs are taken as they are
    lost = amax * tiny if kind != "fp16" else np.zeros_like(amax)
    return (fixed * np.abs(x) + lost) @ np.abs(w).T + 2 * HALF_STEP[kind] * np.abs(y) + 1e-30


def check(dev, kind, M, N, K, group, seed, bias=True, x=None):
    r = rng(seed)
    packed = r.integers(0, 256, size=(N, (K + 1) // 2)).astype(np.uint8)  # every code, -8 too
    scales = (r.standard_normal((N, (K + group - 1) // group)) * 0.01).astype(np.float32)
    b = r.standard_normal(N).astype(np.float32) * np.float32(0.02) if bias else None
    xb = to_bits(r.standard_normal((M, K)).astype(np.float32) if x is None else x, kind)
    W = dev.weight_i4(packed, scales, K, group)
    C = dev.array(empty_as(kind, (M, N), 7))
    dev.linear_i4(dev.array(xb), W, dev.array(b) if bias else None, C, M, N, K, TYPES[kind])
    got = to_f64(C.numpy(), kind)
    xf, w = to_f64(xb, kind), decode(packed, scales, K, group)
    want = xf @ w.T + (b.astype(np.float64) if bias else 0.0)
    assert np.all(np.isfinite(got))
    off = np.abs(got - want) / tolerance(xf, w, want, kind)
    assert off.max() <= 1.0, (off.max(), np.unravel_index(off.argmax(), off.shape))
    W.free()
    return got


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("M,N,K,group", [
    (1, 1, 1, 32), (1, 16, 128, 128), (1, 1280, 1280, 128), (2, 33, 77, 32), (3, 17, 129, 64), (7, 320, 320, 64),
    (16, 960, 320, 32), (17, 48, 257, 128), (31, 100, 640, 256), (33, 64, 1280, 1280), (64, 81, 95, 32),
    (65, 130, 384, 128), (129, 257, 515, 64), (200, 640, 1280, 128), (301, 96, 2560, 32)])
def test_against_the_formula(dev, kind, M, N, K, group):
    check(dev, kind, M, N, K, group, seed=M * 7 + N + K)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("M,N,K,group", [(700, 5130, 200, 32), (700, 5130, 200, 64), (700, 5130, 256, 128),
                                         (1030, 2570, 1400, 256)])
def test_many_rows_and_columns(dev, kind, M, N, K, group):
    """Sizes at which the products run as a GEMM, with tiles that M, N and K end inside."""
    check(dev, kind, M, N, K, group, seed=M + N + K + group)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("M,N,K,group", [(301, 1290, 5120, 128), (301, 1290, 5000, 128), (291, 1300, 5120, 64),
                                         (291, 1300, 4999, 64), (100, 3850, 1270, 32)])
def test_some_rows_of_long_sums(dev, kind, M, N, K, group):
    """Sizes at which small tiles share the CUs, and 16-bit types take wider ones."""
    check(dev, kind, M, N, K, group, seed=M + N + K + group)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("offset,pad", [(0, 8), (1, 3)])
def test_strides_of_many_rows_and_columns(dev, kind, offset, pad):
    M, N, K, group = 650, 5130, 256, 64
    r = rng(pad)
    size = 4 if kind == "fp32" else 2
    packed = r.integers(0, 256, size=(N, K // 2)).astype(np.uint8)
    scales = r.standard_normal((N, K // group)).astype(np.float32)
    lda, ldc = K + pad, N + pad
    x = to_bits(r.standard_normal((M * lda + offset,)).astype(np.float32), kind)
    x[offset + 3 * lda + 7] = to_bits(np.array([np.inf], np.float32), kind)[0]
    X, W = dev.array(x), dev.weight_i4(packed, scales, K, group)
    C = dev.array(empty_as(kind, (M * ldc,), 99))
    dev.linear_i4(At(X, offset * size), W, None, C, M, N, K, TYPES[kind], lda=lda, ldc=ldc)
    rows = C.numpy().reshape(M, ldc)
    xr = to_f64(x[offset:], kind).reshape(M, lda)[:, :K]
    w = decode(packed, scales, K, group)
    sane = np.arange(M) != 3
    want = xr[sane] @ w.T
    assert np.all(np.abs(to_f64(rows[sane, :N], kind) - want) <= tolerance(xr[sane], w, want, kind))
    assert not np.any(np.isfinite(to_f64(rows[3, :N], kind)))
    assert np.all(rows[:, N:] == empty_as(kind, (1,), 99)[0])
    W.free()


@pytest.mark.parametrize("M", [1, 40, 300])
def test_without_bias(dev, M):
    check(dev, "fp32", M, 70, 200, 64, seed=M, bias=False)


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("M", [2, 50, 200])
@pytest.mark.parametrize("scale", [1e-36, 1e-20, 1e-4, 1e20, 1e34])
def test_magnitudes(dev, kind, M, scale):
    """fp16 parts of the activations hold at any magnitude of fp32 and bf16."""
    x = rng(5).standard_normal((M, 300)).astype(np.float32) * np.float32(scale)
    x[:, ::7] *= np.float32(1e-3)
    check(dev, kind, M, 40, 300, 32, seed=8, bias=False, x=x)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("M", [3, 70, 260])
def test_infinities_and_nans_stay_in_their_rows(dev, kind, M):
    N, K, group = 40, 256, 64
    r = rng(3)
    packed = r.integers(0, 256, size=(N, K // 2)).astype(np.uint8)
    packed[packed % 16 == 8] += 1  # no zero codes: infinity times one is NaN
    packed[packed // 16 == 8] += 16
    scales = np.abs(r.standard_normal((N, K // group))).astype(np.float32) + np.float32(0.1)
    x = r.standard_normal((M, K)).astype(np.float32)
    clean = x.copy()
    x[1, 9], x[2, 200] = np.inf, np.nan
    W = dev.weight_i4(packed, scales, K, group)
    outs = []
    for a in (x, clean):
        C = dev.array(empty_as(kind, (M, N), 0))
        dev.linear_i4(dev.array(to_bits(a, kind)), W, None, C, M, N, K, TYPES[kind])
        outs.append(to_f64(C.numpy(), kind))
    with np.errstate(invalid="ignore"):
        want = x.astype(np.float64) @ decode(packed, scales, K, group).T
    rows = [i for i in range(M) if i not in (1, 2)]
    np.testing.assert_array_equal(outs[0][rows], outs[1][rows])
    np.testing.assert_array_equal(outs[0][1], want[1])
    assert np.all(np.isnan(outs[0][2]))
    W.free()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("M,offset,pad", [(1, 1, 3), (9, 0, 8), (40, 1, 1), (150, 0, 8), (150, 1, 5)])
def test_strides_and_alignment(dev, kind, M, offset, pad):
    """Rows of any stride from any element on; what lies between and behind the
    output's rows stays as it was."""
    N, K, group = 50, 200, 32
    r = rng(M + pad)
    size = 4 if kind == "fp32" else 2
    packed = r.integers(0, 256, size=(N, K // 2)).astype(np.uint8)
    scales = r.standard_normal((N, (K + group - 1) // group)).astype(np.float32)
    lda, ldc = K + pad, N + pad
    x = to_bits(r.standard_normal((M * lda + offset,)).astype(np.float32), kind)
    c = empty_as(kind, (M * ldc + offset + 16,), 99)
    X, Cd, W = dev.array(x), dev.array(c), dev.weight_i4(packed, scales, K, group)
    dev.linear_i4(At(X, offset * size), W, None, At(Cd, offset * size), M, N, K, TYPES[kind], lda=lda, ldc=ldc)
    got = Cd.numpy()
    xr = to_f64(x[offset:], kind).reshape(M, lda)[:, :K]
    w = decode(packed, scales, K, group)
    want = xr @ w.T
    rows = got[offset:offset + M * ldc].reshape(M, ldc)
    assert np.all(np.abs(to_f64(rows[:, :N], kind) - want) <= tolerance(xr, w, want, kind))
    assert np.all(rows[:, N:] == c[0]) and np.all(got[:offset] == c[0]) and np.all(got[offset + M * ldc:] == c[0])
    W.free()


@pytest.mark.parametrize("M", [1, 20, 100])
def test_zero_scales_and_one_channel_groups(dev, M):
    N, K = 24, 512
    r = rng(1)
    packed = r.integers(0, 256, size=(N, K // 2)).astype(np.uint8)
    x = r.standard_normal((M, K)).astype(np.float32)
    for group in (512, 1024):
        scales = np.zeros((N, 1), np.float32)
        scales[::2] = 0.5
        W = dev.weight_i4(packed, scales, K, group)
        C = dev.empty((M, N), np.float32)
        dev.linear_i4(dev.array(x), W, None, C, M, N, K)
        got = C.numpy()
        assert np.all(got[:, 1::2] == 0)
        w = decode(packed, np.repeat(scales, 1, axis=1), K, group)
        want = x.astype(np.float64) @ w.T
        assert np.all(np.abs(got - want) <= tolerance(x.astype(np.float64), w, want, "fp32"))
        W.free()


def test_rows_of_a_larger_call_and_repeats_agree(dev):
    """The same call gives the same bits, also where two calls of other sizes
    ran in between (nothing is kept from call to call)."""
    N, K = 1280, 1280
    r = rng(2)
    q, s = syn.quantize_weight_i4(r.standard_normal((N, K)).astype(np.float32), 128)
    W = dev.weight_i4(q, s, K, 128)
    x = r.standard_normal((333, K)).astype(np.float32)
    X = dev.array(x)
    a, b, c = (dev.empty((333, N), np.float32) for _ in range(3))
    dev.linear_i4(X, W, None, a, 333, N, K)
    dev.linear_i4(X, W, None, c, 5, N, K)
    dev.linear_i4(X, W, None, c, 70, N, K)
    dev.linear_i4(X, W, None, b, 333, N, K)
    np.testing.assert_array_equal(a.numpy(), b.numpy())
    W.free()


def test_many_rows(dev):
    """More rows than one dimension of a grid of 16-row tiles holds."""
    check(dev, "bf16", 65536 * 16 + 5, 1, 8, 32, seed=1)


def test_two_contexts_at_once(dev):
    """Calls of two contexts (two streams) in flight together."""
    other = eg.Device(0)
    N, K = 640, 1280
    r = rng(4)
    q, s = syn.quantize_weight_i4(r.standard_normal((N, K)).astype(np.float32), 64)
    x = r.standard_normal((600, K)).astype(np.float32)
    w = decode(q, s, K, 64)
    want = x.astype(np.float64) @ w.T
    state = []
    for d in (dev, other):
        state.append((d, d.weight_i4(q, s, K, 64), d.array(x), d.empty((600, N), np.float32)))
    for _ in range(20):
        for d, W, X, Y in state:
            d.linear_i4(X, W, None, Y, 600, N, K)
    for d, W, X, Y in state:
        d.sync()
        assert np.all(np.abs(Y.numpy() - want) <= tolerance(x.astype(np.float64), w, want, "fp32"))
        W.free()
        X.free()
        Y.free()
    other.close()


def test_refusals(dev):
    packed, scales = np.zeros((4, 8), np.uint8), np.zeros((4, 1), np.float32)
    for group in (0, -32, 16, 48, 96, 160):
        with pytest.raises((eg.Gfx950Error, ValueError)):
            dev.weight_i4(packed, scales, 16, group)
    with pytest.raises(ValueError):
        dev.weight_i4(packed, scales, 18, 32)
    W = dev.weight_i4(packed, scales, 16, 32)
    A, C = dev.empty((4, 16), np.float32), dev.empty((4, 16), np.float32)

    def refused(code, *args, **kw):
        with pytest.raises(eg.Gfx950Error) as e:
            dev.linear_i4(*args, **kw)
        assert e.value.code == code

    refused(eg.SHAPE_MISMATCH, A, W, None, C, 4, 4, 15)
    refused(eg.SHAPE_MISMATCH, A, W, None, C, 4, 5, 16)
    refused(eg.INVALID_ARGUMENT, A, W, None, C, -1, 4, 16)
    refused(eg.INVALID_ARGUMENT, A, W, None, C, 4, 4, 16, 3)
    refused(eg.INVALID_ARGUMENT, A, W, None, C, 4, 4, 16, lda=15)
    refused(eg.INVALID_ARGUMENT, A, W, None, C, 4, 4, 16, ldc=3)
    refused(eg.INVALID_ARGUMENT, A, W, None, A, 4, 4, 16)
    refused(eg.INVALID_ARGUMENT, At(A, 2), W, None, C, 3, 4, 16)
    dev.linear_i4(A, W, None, C, 0, 4, 16)  # no rows: nothing to do
    W.free()


def test_outputs_over_the_bias_are_refused(dev):
    """The bias is read while other outputs are written."""
    W = dev.weight_i4(np.zeros((4, 8), np.uint8), np.zeros((4, 1), np.float32), 16, 32)
    A, C = dev.array(np.zeros((4, 16), np.float32)), dev.array(np.zeros(64, np.float32))
    with pytest.raises(eg.Gfx950Error) as e:
        dev.linear_i4(A, W, At(C, 15 * 4), C, 4, 4, 16)
    assert e.value.code == eg.INVALID_ARGUMENT
    dev.linear_i4(A, W, At(C, 16 * 4), C, 4, 4, 16)
    assert (C.numpy() == 0).all()
    W.free()
