"""Block-sparse attention on gfx950 against the plain formulas in 64 bits.

Block means: one rounding to fp32 of a 64-bit sum. Selection: equal to the
64-bit scores' order. Attention: with es the error of a score (operands of 22
bits, dim additions), an output is off by at most (2 es + the additions of its
sum and of l + 4 exponentials' 2^-22) times the largest |v|, and is rounded once
to its type. An addition is taken as off by 2^-23 (a matrix core may
truncate)."""
import numpy as np
import pytest

import esm_gfx950 as eg
from conftest import cu_from_lengths, rng
from esm_gfx950 import synthetic as syn
from test_gpu_linear_i4 import HALF_STEP, TYPES, At, decode, empty_as, to_bits, to_f64

pytestmark = pytest.mark.gpu


def means64(k, cu_k, block):
    out = []
    for a, b in zip(cu_k[:-1], cu_k[1:]):
        for t in range(a, b, block):
            out.append(k[t:min(b, t + block)].mean(axis=0))
    return np.array(out).reshape(-1, *k.shape[1:])


def select64(q, means, cu_q, cb, top):
    """[rows, H, top] by the definition."""
    rows, H, _ = q.shape
    group = H // means.shape[1]
    out = np.full((rows, H, top), -1, np.int32)
    for b in range(len(cu_q) - 1):
        m = means[cb[b]:cb[b + 1]].astype(np.float64)
        n = min(top, len(m))
        for t in range(cu_q[b], cu_q[b + 1]):
            for h in range(H):
                with np.errstate(invalid="ignore"):
                    s = m[:, h // group] @ q[t, h]
                s = np.where(np.isnan(s), -np.inf, s)
                out[t, h, :n] = np.sort(np.argsort(-s, kind="stable")[:n])
    return out


def attend64(q, k, v, blocks, cu_q, cu_k, block):
    """(out, tolerance without the final rounding), [rows, H, dim] each."""
    rows, H, dim = q.shape
    group = H // k.shape[1]
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    top = blocks.shape[2]
    for b in range(len(cu_q) - 1):
        k0, k1 = cu_k[b], cu_k[b + 1]
        nb = -(-(k1 - k0) // block)
        for t in range(cu_q[b], cu_q[b + 1]):
            for h in range(H):
                js = sorted({int(j) for j in blocks[t, h] if 0 <= j < nb})
                if not js:
                    continue
                at = np.concatenate([np.arange(k0 + j * block, min(k1, k0 + (j + 1) * block)) for j in js])
                kk, vv = k[at, h // group], v[at, h // group]
                s = kk @ q[t, h]
                p = np.exp(s - s.max())
                out[t, h] = p @ vv / p.sum()
                es = (2.0 ** -21 + (dim + 8) * 2.0 ** -23) * (np.abs(kk) @ np.abs(q[t, h])).max() + 2.0 ** -30
                tol[t, h] = (2 * es + (128 + top + 64) * 2.0 ** -23 + 2.0 ** -20) * np.abs(vv).max()
    return out, tol


class Batch:
    def __init__(self, dev, kind, q_lens, k_lens, H, Hkv, dim, block, seed, scale=1.0):
        r = rng(seed)
        self.dev, self.kind, self.block, self.H, self.Hkv, self.dim = dev, kind, block, H, Hkv, dim
        self.cu_q, self.cu_k = cu_from_lengths(q_lens), cu_from_lengths(k_lens)
        self.cb = eg.key_blocks(self.cu_k, block)
        self.rows, self.keys = int(self.cu_q[-1]), int(self.cu_k[-1])
        make = lambda n, h, s: to_bits((r.standard_normal((n, h, dim)) * s).astype(np.float32), kind)
        self.q, self.k, self.v = make(self.rows, H, scale * dim ** -0.5 * 2), make(self.keys, Hkv, 1.0), make(
            self.keys, Hkv, 1.0)

    def f64(self):
        return (to_f64(a, self.kind) for a in (self.q, self.k, self.v))

    def shape(self):
        return self.H, self.Hkv, self.dim, self.block

    def attend(self, blocks, top):
        dev = self.dev
        out = dev.array(empty_as(self.kind, (self.rows, self.H * self.dim), 3))
        dev.attention_blocks(dev.array(self.q), dev.array(self.k), dev.array(self.v), dev.array(blocks), self.cu_q,
                             self.cu_k, *self.shape(), top, out, TYPES[self.kind])
        return out.numpy()

    def check(self, blocks):
        got = to_f64(self.attend(blocks, blocks.shape[2]), self.kind).reshape(self.rows, self.H, self.dim)
        q, k, v = self.f64()
        want, tol = attend64(q, k, v, blocks, self.cu_q, self.cu_k, self.block)
        if self.kind == "bf16":  # probabilities and partial sums of 16-bit types may be fp16
            tol = tol + 2.0 ** -9 * np.abs(v).max()
        if self.kind == "fp16":
            tol = tol + 2.0 ** -9 * np.abs(v).max()
        assert np.all(np.isfinite(got))
        off = np.abs(got - want) - (tol + 2 * HALF_STEP[self.kind] * np.abs(want))
        assert off.max(initial=-1) <= 0, (off.max(), np.unravel_index(off.argmax(), off.shape))


SHAPES = [  # queries, keys, heads, key heads, dim, block, top
    ([1], [1], 1, 1, 8, 16, 1), ([1], [17], 2, 2, 16, 16, 3), ([3], [70], 4, 2, 24, 16, 2),
    ([5, 0, 2], [0, 40, 33], 4, 4, 32, 32, 4), ([33], [33], 3, 3, 64, 16, 2), ([1, 1], [500, 129], 4, 1, 64, 64, 5),
    ([130], [130], 2, 2, 64, 32, 3), ([70, 1, 90], [70, 1, 90], 2, 1, 128, 64, 2), ([40], [1030], 2, 2, 40, 128, 3),
    ([260], [700], 2, 2, 64, 64, 4), ([65], [3000], 1, 1, 64, 16, 20), ([300], [300], 4, 2, 16, 48, 7),
    ([150], [900], 2, 2, 64, 256, 2), ([90], [2100], 1, 1, 96, 1024, 2)]


LARGE = [  # as SHAPES; enough work that blocks are taken in turn
    ([600], [600], 20, 20, 64, 64, 4), ([260, 0, 300], [260, 5, 333], 16, 4, 128, 32, 9),
    ([700], [700], 20, 20, 24, 48, 7), ([400], [1500], 10, 5, 64, 256, 3), ([350, 1], [2100, 1], 8, 8, 96, 1024, 2),
    ([800], [801], 20, 20, 32, 16, 20)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("shape", LARGE, ids=[str(i) for i in range(len(LARGE))])
def test_many_rows(dev, kind, shape):
    """A sample of the rows against the formula, lists of every sort."""
    q_lens, k_lens, H, Hkv, dim, block, top = shape
    b = Batch(dev, kind, q_lens, k_lens, H, Hkv, dim, block, seed=sum(k_lens))
    r = rng(dim)
    most = int(np.max(np.diff(b.cb)))
    blocks = r.integers(-1, most + 1, size=(b.rows, H, top)).astype(np.int32)
    blocks[::3] = np.sort(blocks[::3], axis=2)
    blocks[7] = -1
    blocks[:, 1, 0] = 0
    got = to_f64(b.attend(blocks, top), kind).reshape(b.rows, H, dim)
    assert np.all(np.isfinite(got)) and np.all(got[7, [0] + list(range(2, H))] == 0)
    q, k, v = b.f64()
    for t in [0, 7, b.rows - 1] + list(r.integers(0, b.rows, size=25)):
        s = int(np.searchsorted(b.cu_q, t, side="right")) - 1
        k0, k1 = b.cu_k[s], b.cu_k[s + 1]
        one = np.array([0, 1]), np.array([0, k1 - k0])
        want, tol = attend64(q[t:t + 1], k[k0:k1], v[k0:k1], blocks[t:t + 1], *one, block)
        if kind != "fp32":
            tol = tol + 2.0 ** -9 * np.abs(v).max()
        assert np.all(np.abs(got[t] - want[0]) <= tol[0] + 2 * HALF_STEP[kind] * np.abs(want[0])), t
    np.testing.assert_array_equal(b.attend(blocks, top), b.attend(blocks, top))


def selected(b, top):
    q, k, _ = b.f64()
    return select64(q, means64(k, b.cu_k, b.block).astype(np.float32), b.cu_q, b.cb, top)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=[str(i) for i in range(len(SHAPES))])
def test_the_three_ops(dev, kind, shape):
    q_lens, k_lens, H, Hkv, dim, block, top = shape
    b = Batch(dev, kind, q_lens, k_lens, H, Hkv, dim, block, seed=sum(k_lens) + dim)
    _, k, _ = b.f64()
    n = int(b.cb[-1])
    means = dev.array(np.full((n, Hkv, dim), 5, np.float32))
    dev.key_block_means(dev.array(b.k), b.cu_k, Hkv, dim, block, means, TYPES[kind])
    want = means64(k, b.cu_k, block)
    assert np.all(np.abs(means.numpy() - want) <= 2.0 ** -23 * np.abs(want) + 1e-15)
    blocks = dev.array(np.full((b.rows, H, top), 77, np.int32))
    dev.attention_select_blocks(dev.array(b.q), means, b.cu_q, b.cu_k, H, Hkv, dim, block, top, blocks, TYPES[kind])
    q, _, _ = b.f64()
    np.testing.assert_array_equal(blocks.numpy(), select64(q, means.numpy(), b.cu_q, b.cb, top))
    b.check(blocks.numpy())


@pytest.mark.parametrize("nb,top", [(1, 1), (63, 64), (64, 5), (65, 64), (129, 256), (1023, 16), (1025, 16),
                                    (2500, 200), (4100, 1)])
def test_selection_among_many_blocks(dev, nb, top):
    """Fewer blocks than a wave to more than LDS holds at once; the row's order
    is that of 64-bit scores."""
    r = rng(nb)
    H, dim, rows, block = 2, 16, 5, 16
    cu_q, cu_k = cu_from_lengths([rows]), cu_from_lengths([nb * block - 3])
    q = r.standard_normal((rows, H, dim)).astype(np.float32)
    m = r.standard_normal((nb, H, dim)).astype(np.float32)
    out = dev.empty((rows, H, top), np.int32)
    dev.attention_select_blocks(dev.array(q), dev.array(m), cu_q, cu_k, H, H, dim, block, top, out)
    np.testing.assert_array_equal(out.numpy(), select64(q.astype(np.float64), m, cu_q, eg.key_blocks(cu_k, block), top))


@pytest.mark.parametrize("nb,top", [(40, 7), (300, 16), (1500, 30)])
def test_selection_near_and_equal_scores(dev, nb, top):
    """Scores that differ in the last bits of fp32 or not at all, infinities,
    NaN and zeros of both signs."""
    r = rng(top)
    H, dim, rows, block = 1, 64, 9, 32
    cu_q, cu_k = cu_from_lengths([rows]), cu_from_lengths([nb * block])
    base = r.standard_normal(dim).astype(np.float32)
    m = np.repeat(base[None, None, :], nb, axis=0)
    m[r.integers(0, nb, size=nb // 2), 0, 5] *= np.float32(1 + 2.0 ** -23)  # one last bit
    q = r.standard_normal((rows, H, dim)).astype(np.float32)
    q[3] = 0  # every score is a zero: the first blocks
    q[4, 0, 0] = np.nan
    q[5] = np.abs(q[5])
    m2 = m.copy()
    m2[3], m2[nb // 2], m2[nb - 1] = np.inf, -np.inf, np.nan
    for means in (m, m2):
        out = dev.empty((rows, H, top), np.int32)
        dev.attention_select_blocks(dev.array(q), dev.array(means), cu_q, cu_k, H, H, dim, block, top, out)
        got = out.numpy()
        want = select64(q.astype(np.float64), means, cu_q, eg.key_blocks(cu_k, block), top)
        # Equal blocks have equal scores here and there; those that differ do by
        # 2^-24 of a term, far above 64-bit rounding.
        np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("kind", list(TYPES))
def test_lists_that_a_caller_makes(dev, kind):
    """Any order, repeats, negative entries, entries past the sequence, empty
    rows; short last blocks; a block that every row lists."""
    b = Batch(dev, kind, [40, 150], [100, 300], 4, 2, 64, 32, seed=3)
    r = rng(9)
    blocks = r.integers(-2, 12, size=(190, 4, 9)).astype(np.int32)
    blocks[5] = -1
    blocks[:, 1, 0] = 3
    blocks[50:90, 2] = 9
    blocks[7, 3] = [2 ** 31 - 1, -2 ** 31, 3, 3, 3, 3, 0, 10, 11]
    b.check(blocks)
    assert np.all(to_f64(b.attend(blocks, 9), kind).reshape(190, 4, 64)[5, [0, 2, 3]] == 0)  # head 1 lists block 3


@pytest.mark.parametrize("rows", [2, 200])
def test_large_scores_and_far_apart_values(dev, rows):
    """Scores in the hundreds (exponentials that underflow in all but one
    block), keys and values from 1e-6 to 1e6."""
    b = Batch(dev, "fp32", [rows], [520], 2, 2, 64, 64, seed=6, scale=40.0)
    b.v = (b.v * np.exp(rng(1).uniform(-13, 13, size=(520, 2, 1)))).astype(np.float32)
    b.check(selected(b, 4))
    b.q, b.k = b.q * np.float32(1e-5), b.k * np.float32(1e5)
    b.check(selected(b, 4))


@pytest.mark.parametrize("rows", [2, 900])
def test_repeats_behind_negative_entries(dev, rows):
    """A repeat is one whatever stands between: the most negative number too."""
    b = Batch(dev, "fp32", [rows], [300], 4, 4, 64, 32, seed=7)
    for middle in (-1, -2 ** 31):
        for j in (0, 3):
            blocks = np.full((rows, 4, 4), -1, np.int32)
            blocks[:, :, 0], blocks[:, :, 1], blocks[:, :, 2], blocks[:, :, 3] = j, middle, j, 7
            once = blocks.copy()
            once[:, :, 2] = -1
            np.testing.assert_array_equal(b.attend(blocks, 4), b.attend(once, 4))


@pytest.mark.parametrize("rows", [3, 700])
@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e25])
def test_values_of_any_magnitude(dev, rows, scale):
    """The output is linear in V: scaling it by a power of two scales the result."""
    b = Batch(dev, "fp32", [rows], [400], 4, 4, 64, 64, seed=15)
    blocks = rng(3).integers(0, 7, size=(rows, 4, 3)).astype(np.int32)
    want = b.attend(blocks, 3)
    by = np.float32(2.0 ** round(np.log2(scale)))
    b.v = b.v * by
    np.testing.assert_allclose(b.attend(blocks, 3), want * by, rtol=2e-6, atol=2e-6 * float(by))


@pytest.mark.parametrize("scale", [1e-36, 1e-30, 1e-20, 1e15, 1e18])
def test_selection_of_any_magnitude(dev, scale):
    """Scores from below fp32's smallest to near its largest numbers."""
    r = rng(5)
    rows, H, dim, nb, top, block = 40, 2, 32, 70, 9, 16
    cu_q, cu_k = cu_from_lengths([rows]), cu_from_lengths([nb * block])
    q = (r.standard_normal((rows, H, dim)) * scale).astype(np.float32)
    m = (r.standard_normal((nb, H, dim)) * min(scale, 1e4)).astype(np.float32)
    out = dev.empty((rows, H, top), np.int32)
    dev.attention_select_blocks(dev.array(q), dev.array(m), cu_q, cu_k, H, H, dim, block, top, out)
    np.testing.assert_array_equal(out.numpy(), select64(q.astype(np.float64), m, cu_q, eg.key_blocks(cu_k, block), top))


@pytest.mark.parametrize("rows", [2, 130])
@pytest.mark.parametrize("kind", list(TYPES))
def test_what_is_not_listed_is_not_read(dev, kind, rows):
    """NaN in unlisted blocks, and behind a short last block (the next
    sequence's keys), reaches no output."""
    b = Batch(dev, kind, [rows, 3], [90, 64], 2, 2, 32, 32, seed=4)
    blocks = np.full((rows + 3, 2, 3), -1, np.int32)
    blocks[:rows, :, 0], blocks[:rows, :, 1] = 2, 0  # keys 64..89 and 0..31
    want = b.attend(blocks, 3)
    nan = 0x7FC0 if kind == "bf16" else np.nan
    b.k[32:64], b.v[32:64], b.k[90:], b.v[90:] = nan, nan, nan, nan
    np.testing.assert_array_equal(b.attend(blocks, 3), want)


@pytest.mark.parametrize("rows", [2, 130])
def test_nan_stays_in_the_rows_that_read_it(dev, rows):
    b = Batch(dev, "fp32", [rows], [128], 2, 2, 64, 64, seed=5)
    blocks = np.zeros((rows, 2, 1), np.int32)
    blocks[0] = 1
    want = b.attend(blocks, 1)
    b.k[100] = np.nan
    got = b.attend(blocks, 1)
    assert np.all(np.isnan(got[0]))
    np.testing.assert_array_equal(got[1:], want[1:])


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows,offset,pad", [(4, 0, 8), (4, 1, 3), (150, 0, 16), (150, 1, 3)])
def test_fused_rows(dev, kind, rows, offset, pad):
    """Q, K and V as parts of one row, at any element offset and stride."""
    H, dim, block, top = 2, 64, 32, 3
    keys = max(rows, 150)
    size = 4 if kind == "fp32" else 2
    ld = 3 * H * dim + pad
    fused = to_bits(rng(8).standard_normal(keys * ld + offset).astype(np.float32), kind)
    f = fused[offset:].reshape(keys, ld)
    b = Batch(dev, kind, [rows], [keys], H, H, dim, block, seed=1)
    b.q, b.k, b.v = (np.ascontiguousarray(f[:n, i * H * dim:(i + 1) * H * dim]).reshape(n, H, dim)
                     for i, n in enumerate((rows, keys, keys)))
    F = dev.array(fused)
    q, k, v = (At(F, (offset + i * H * dim) * size) for i in range(3))
    means = dev.empty((int(b.cb[-1]), H, dim), np.float32)
    dev.key_block_means(k, b.cu_k, H, dim, block, means, TYPES[kind], ldk=ld)
    blocks = dev.empty((rows, H, top), np.int32)
    dev.attention_select_blocks(q, means, b.cu_q, b.cu_k, H, H, dim, block, top, blocks, TYPES[kind], ldq=ld)
    q64, k64, _ = b.f64()
    np.testing.assert_array_equal(
        blocks.numpy(), select64(q64, means64(k64, b.cu_k, block).astype(np.float32), b.cu_q, b.cb, top))
    out = dev.array(empty_as(kind, (rows, H * dim), 1))
    dev.attention_blocks(q, k, v, blocks, b.cu_q, b.cu_k, H, H, dim, block, top, out, TYPES[kind], ldq=ld, ldkv=ld)
    np.testing.assert_array_equal(out.numpy(), b.attend(blocks.numpy(), top))


@pytest.mark.parametrize("n", [64, 65, 200])
def test_many_sequences(dev, n):
    """Batches up to and past what the kernels' arguments hold, with empty sequences."""
    r = rng(n)
    lens = r.integers(0, 40, size=n)
    b = Batch(dev, "fp32", lens, lens[::-1], 2, 2, 16, 16, seed=n)
    b.check(selected(b, 2))


def test_every_block_equals_dense_attention(dev):
    """With every block listed this is attention_varlen."""
    lens = [200, 65, 1, 333]
    b = Batch(dev, "fp32", lens, lens, 4, 4, 64, 64, seed=11)
    blocks = np.tile(np.arange(6, dtype=np.int32), (b.rows, 4, 1))
    out = dev.empty((b.rows, 256), np.float32)
    dev.attention_varlen(dev.array(b.q), dev.array(b.k), dev.array(b.v), b.cu_q, 4, 64, out, eg.ATTN_FP32)
    np.testing.assert_allclose(b.attend(blocks, 6), out.numpy(), rtol=1e-5, atol=1e-5)


def test_repeats_agree(dev):
    """The same call gives the same bits, also after calls of other sizes."""
    b = Batch(dev, "fp32", [900], [900], 4, 4, 64, 64, seed=12)
    blocks = rng(1).integers(0, 15, size=(900, 4, 6)).astype(np.int32)
    first = b.attend(blocks, 6)
    Batch(dev, "bf16", [40], [300], 2, 2, 128, 32, seed=1).attend(np.zeros((40, 2, 3), np.int32), 3)
    for _ in range(3):
        np.testing.assert_array_equal(b.attend(blocks, 6), first)


def test_two_contexts_at_once(dev):
    other = eg.Device(0)
    b = Batch(dev, "fp32", [700], [700], 2, 2, 64, 32, seed=13)
    blocks = rng(2).integers(-1, 22, size=(700, 2, 5)).astype(np.int32)
    want = b.attend(blocks, 5)
    state = []
    for d in (dev, other):
        state.append((d, [d.array(a) for a in (b.q, b.k, b.v, blocks)], d.empty((700, 128), np.float32)))
    for _ in range(10):
        for d, (q, k, v, bl), out in state:
            d.attention_blocks(q, k, v, bl, b.cu_q, b.cu_k, 2, 2, 64, 32, 5, out)
    for d, arrays, out in state:
        d.sync()
        np.testing.assert_array_equal(out.numpy(), want)
        for a in arrays + [out]:
            a.free()
    other.close()


def test_one_layer_of_a_long_protein(dev):
    """Together, as they are used: QKV by a 4-bit linear, its fused rows read by
    the block means, the selection and the attention, then the output linear."""
    T, d, H, dim, block, top = 700, 320, 20, 16, 64, 4
    r = rng(21)
    x = r.standard_normal((T, d)).astype(np.float32)
    wq, sq = syn.quantize_weight_i4(r.standard_normal((3 * d, d)).astype(np.float32) * 0.05, 64)
    wo, so = syn.quantize_weight_i4(r.standard_normal((d, d)).astype(np.float32) * 0.05, 64)
    Wq, Wo = dev.weight_i4(wq, sq, d, 64), dev.weight_i4(wo, so, d, 64)
    cu = cu_from_lengths([T])
    qkv, y, out = dev.empty((T, 3 * d), np.float32), dev.empty((T, d), np.float32), dev.empty((T, d), np.float32)
    means, blocks = dev.empty((11, H, dim), np.float32), dev.empty((T, H, top), np.int32)
    dev.linear_i4(dev.array(x), Wq, None, qkv, T, 3 * d, d)
    q, k, v = At(qkv, 0), At(qkv, 4 * d), At(qkv, 8 * d)
    dev.key_block_means(k, cu, H, dim, block, means, ldk=3 * d)
    dev.attention_select_blocks(q, means, cu, cu, H, H, dim, block, top, blocks, ldq=3 * d)
    dev.attention_blocks(q, k, v, blocks, cu, cu, H, H, dim, block, top, y, ldq=3 * d, ldkv=3 * d)
    dev.linear_i4(y, Wo, None, out, T, d, d)
    qkv64 = x.astype(np.float64) @ decode(wq, sq, d, 64).T
    got = qkv.numpy()
    np.testing.assert_allclose(got, qkv64, rtol=1e-5, atol=2e-5 * np.abs(qkv64).max())
    q64, k64, v64 = (got[:, i * d:(i + 1) * d].astype(np.float64).reshape(T, H, dim) for i in range(3))
    listed = blocks.numpy()
    np.testing.assert_array_equal(listed, select64(q64, means.numpy(), cu, np.array([0, 11]), top))
    want, tol = attend64(q64, k64, v64, listed, cu, cu, block)
    assert np.all(np.abs(y.numpy() - want.reshape(T, d)) <= tol.reshape(T, d) + 2.0 ** -23 * np.abs(want).reshape(T, d))
    final = y.numpy().astype(np.float64) @ decode(wo, so, d, 64).T
    np.testing.assert_allclose(out.numpy(), final, rtol=1e-5, atol=2e-5 * np.abs(final).max())
    Wq.free()
    Wo.free()


def test_refusals(dev):
    a = dev.empty((64, 2, 64), np.float32)
    o, m, ids = dev.empty((64, 128), np.float32), dev.empty((64, 2, 64), np.float32), dev.empty((64, 2, 4), np.int32)
    cu = cu_from_lengths([64])

    def refused(fn, *args, **kw):
        with pytest.raises((eg.Gfx950Error, ValueError)) as e:
            fn(*args, **kw)
        if isinstance(e.value, eg.Gfx950Error):
            assert e.value.code == eg.INVALID_ARGUMENT

    for H, Hkv, dim, block, top in [(2, 0, 64, 64, 4), (3, 2, 64, 64, 4), (2, 2, 60, 64, 4), (2, 2, 136, 64, 4),
                                    (2, 2, 64, 0, 4), (2, 2, 64, 8, 4), (2, 2, 64, 72, 4), (2, 2, 64, 2048, 4),
                                    (2, 2, 64, 64, 0), (2, 2, 64, 64, 257), (0, 0, 64, 64, 4), (2, 2, 0, 64, 4)]:
        refused(dev.attention_blocks, a, a, a, ids, cu, cu, H, Hkv, dim, block, top, o)
        refused(dev.attention_select_blocks, a, m, cu, cu, H, Hkv, dim, block, top, ids)
        if top == 4 and H != 3:
            refused(dev.key_block_means, a, cu, Hkv, dim, block, m)
    refused(dev.attention_blocks, a, a, a, ids, cu, cu, 2, 2, 64, 64, 4, o, 3)
    refused(dev.attention_blocks, a, a, a, ids, cu, cu, 2, 2, 64, 64, 4, o, ldq=127)
    refused(dev.attention_blocks, a, a, a, ids, cu, cu, 2, 2, 64, 64, 4, o, ldkv=127)
    refused(dev.attention_blocks, a, a, a, ids, cu, cu, 2, 2, 64, 64, 4, a)
    refused(dev.attention_blocks, a, a, a, ids, cu, cu_from_lengths([32, 32]), 2, 2, 64, 64, 4, o)
    refused(dev.attention_blocks, a, a, a, ids, np.array([0, 70, 64], np.int32), cu_from_lengths([32, 32]), 2, 2, 64, 64,
            4, o)
    refused(dev.key_block_means, a, cu, 2, 64, 64, a)
    refused(dev.key_block_means, At(a, 2), cu, 2, 64, 64, m)
    refused(dev.attention_select_blocks, a, m, cu, cu, 2, 2, 64, 64, 4, m)
    for bad in ([1, 5], [0, 5, 4]):
        with pytest.raises(eg.Gfx950Error):
            eg.key_blocks(np.array(bad, np.int32), 64)
    with pytest.raises(eg.Gfx950Error):
        eg.key_blocks(cu, 40)
    # No rows, no keys: nothing to do, and zeros.
    dev.attention_blocks(a, a, a, ids, np.array([0, 0], np.int32), cu, 2, 2, 64, 64, 4, o)
    dev.attention_blocks(a, a, a, ids, cu, np.array([0, 0], np.int32), 2, 2, 64, 64, 4, o)
    assert np.all(o.numpy() == 0)
    dev.attention_select_blocks(a, m, cu, np.array([0, 0], np.int32), 2, 2, 64, 64, 4, ids)
    assert np.all(ids.numpy() == -1)
