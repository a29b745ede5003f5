"""The framework's newest operators as cases that can be timed: 4-bit linears
and block-sparse attention.

  linear   Device.linear_i4: y = x W^T + bias, W held as 4-bit codes with one
           scale per group of inputs, from one row to a packed batch
  means    Device.key_block_means: the mean key of every block of a packed
           batch's keys
  select   Device.attention_select_blocks: for each query and head the blocks
           whose mean key scores highest
  attend   Device.attention_blocks: attention over those blocks alone

own: whether run() makes the framework's calls, or computes the same from
elementary torch operations in 32 bits (64 for sums and scores that decide
which block is taken). The package is only imported for the former.

Shapes are those of the repository's ESM-2 configurations (linears of 320,
1280 and 2560 channels; 20 or 40 heads of 16 or 64), and generic ones beside
them (odd sizes, grouped key heads, heads of 32 and 128).
"""
from __future__ import annotations

import ctypes
import functools
import math
import os
import sys

import numpy as np
import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_WHERE = "cuda" if torch.cuda.is_available() else "cpu"
_TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_WEIGHT_SEED = 20261206


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # One masked position through one projection of the 650M model: the
        # smallest call, all launch and latency.
        {"name": "linear one row", "kind": "linear", "type": "fp32", "rows": 1, "n": 1280, "k": 1280, "group": 128},
        # One row through the largest linear of the 3B model: weight bytes.
        {"name": "linear one row 3b up", "kind": "linear", "type": "fp32", "rows": 1, "n": 10240, "k": 2560,
         "group": 128},
        # A few masked positions, half-precision activations, finer groups.
        {"name": "linear few rows", "kind": "linear", "type": "bf16", "rows": 7, "n": 5120, "k": 1280, "group": 64},
        # A short protein's QKV, the finest groups.
        {"name": "linear short protein", "kind": "linear", "type": "fp32", "rows": 67, "n": 3840, "k": 1280,
         "group": 32},
        # A protein of ordinary length, FFN down.
        {"name": "linear one protein", "kind": "linear", "type": "fp16", "rows": 301, "n": 1280, "k": 5120,
         "group": 128},
        # A packed batch's FFN up, an odd number of rows: matrix-core work.
        {"name": "linear batch", "kind": "linear", "type": "fp32", "rows": 4099, "n": 5120, "k": 1280, "group": 128},
        # One ordinary protein's keys.
        {"name": "means one protein", "kind": "means", "type": "fp32", "keys": "1021", "heads": 20, "kv_heads": 20,
         "dim": 64, "block": 64},
        # A long batch's keys, ragged, half precision: bandwidth.
        {"name": "means long batch", "kind": "means", "type": "bf16", "keys": "32771,20000,0,9001,1", "heads": 20,
         "kv_heads": 20, "dim": 64, "block": 64},
        # Three masked positions scored against one very long assembly.
        {"name": "select few queries", "kind": "select", "type": "fp32", "queries": "3", "keys": "32771", "heads": 20,
         "kv_heads": 20, "dim": 64, "block": 64, "top": 16},
        # Every position of a batch of long proteins.
        {"name": "select long batch", "kind": "select", "type": "fp32", "queries": "4097,2500,1333",
         "keys": "4097,2500,1333", "heads": 20, "kv_heads": 20, "dim": 64, "block": 64, "top": 16},
        # The attention of those three positions in half precision: latency.
        {"name": "attend few queries", "kind": "attend", "type": "bf16", "queries": "3", "keys": "32771", "heads": 20,
         "kv_heads": 20, "dim": 64, "block": 64, "top": 16},
        # Every position of one very long protein.
        {"name": "attend long protein", "kind": "attend", "type": "fp32", "queries": "8195", "keys": "8195",
         "heads": 20, "kv_heads": 20, "dim": 64, "block": 64, "top": 16},
    ]


def draw(rng):
    """One more case of the listed ones' ranges."""
    def log(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    kind = rng.choice(["linear", "linear", "means", "select", "attend", "attend"])
    kind_type = rng.choice(["fp32", "fp32", "bf16", "fp16"])
    if kind == "linear":
        n, k = rng.choice([(1280, 1280), (3840, 1280), (5120, 1280), (1280, 5120), (2560, 2560), (10240, 2560),
                           (2560, 10240), (960, 320), (320, 1280), (log(17, 4000), log(33, 4000))])
        rows = log(1, max(1, min(4096, 4099 * 5120 * 1280 // (n * k))))
        return {"kind": kind, "type": kind_type, "rows": rows, "n": n, "k": k,
                "group": rng.choice([32, 64, 128, 128, 256])}
    heads, kv_heads, dim = rng.choice([(20, 20, 64), (20, 20, 64), (40, 40, 64), (20, 20, 16), (20, 20, 32),
                                       (16, 4, 128), (8, 8, 128), (12, 4, 64)])
    block = rng.choice([32, 64, 64, 128])
    seqs = rng.choice([1, 1, 2, 4])
    if kind == "means":
        keys = [log(1, 60000 * 1280 // (kv_heads * dim * seqs)) for _ in range(seqs)]
        return {"kind": kind, "type": kind_type, "keys": ",".join(map(str, keys)), "heads": heads,
                "kv_heads": kv_heads, "dim": dim, "block": block}
    most = 8000 * 20 // heads
    if rng.random() < 0.4:  # a few queries, each sequence's own number
        keys = [log(1, 32000 // seqs) for _ in range(seqs)]
        queries = [log(1, 40) for _ in range(seqs)]
    else:
        keys = [log(1, most // seqs) for _ in range(seqs)]
        queries = keys
    return {"kind": kind, "type": kind_type, "queries": ",".join(map(str, queries)),
            "keys": ",".join(map(str, keys)), "heads": heads, "kv_heads": kv_heads, "dim": dim, "block": block,
            "top": min(rng.choice([1, 4, 8, 16, 24]), 1024 // block)}


def _offsets(text):
    cu = [0]
    for n in text.split(","):
        cu.append(cu[-1] + int(n))
    return cu


def _block_offsets(cu, block):
    cb = [0]
    for a, b in zip(cu[:-1], cu[1:]):
        cb.append(cb[-1] + (b - a + block - 1) // block)
    return cb


# ------------------------------------------------------------------ inputs
def _randn(seed, what, shape):
    g = torch.Generator(device=_WHERE)
    g.manual_seed(seed * 16 + what)
    return torch.randn(shape, generator=g, device=_WHERE)


@functools.lru_cache(None)
def _weight(n, k, group):
    """(packed codes [n, ceil(k / 2)], scales [n, ceil(k / group)], bias) of a
    linear, made once as a program's weights are: codes of the nearest multiple
    of max|w| / 7 of the group, stored as code + 8, the even input low."""
    w = _randn(_WEIGHT_SEED + n, k, (n, k)) * 0.02
    groups = (k + group - 1) // group
    w = torch.nn.functional.pad(w, (0, groups * group - k)).reshape(n, groups, group)
    scale = w.abs().amax(dim=2) / 7.0
    codes = torch.clamp(torch.round(w / scale[:, :, None]), -8, 7).reshape(n, groups * group)[:, :k]
    codes = torch.nn.functional.pad((codes + 8).to(torch.uint8), (0, k % 2), value=8)
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).contiguous(), scale, _randn(_WEIGHT_SEED, 7, (n,)) * 0.02


def _activations(seed, rows, k):
    """Rows as a LayerNorm leaves them: normal, each channel with a gain of
    its own, a few channels ten times the rest."""
    gain = torch.exp(0.3 * _randn(seed, 1, (k,)))
    gain[::97] *= 10.0
    return _randn(seed, 2, (rows, k)) * gain


def _place(cu, device):
    """Each row's sequence, and its place in it."""
    t = torch.arange(cu[-1], device=device)
    starts = torch.tensor(cu[:-1], device=device)
    ends = torch.tensor(cu[1:], device=device)
    seq = torch.searchsorted(ends, t, right=True)
    return seq, t - starts[seq]


def _keys(seed, what, cu, heads, dim):
    """Keys and values whose mean drifts along the sequence, so that some
    blocks are nearer to a query than others."""
    drift = _randn(seed, what, (cu[-1] // 48 + 1, heads, dim))
    at = torch.arange(cu[-1], device=_WHERE) // 48
    return _randn(seed, what + 1, (cu[-1], heads, dim)) + drift[at]


# ------------------------------------------------- the framework's side
@functools.lru_cache(None)
def _package():
    sys.path.insert(0, os.path.join(_ROOT, "esm-cpp_amd"))
    import esm_gfx950
    return esm_gfx950


@functools.lru_cache(None)
def _device():
    return _package().Device(0)


@functools.lru_cache(None)
def _weight_i4(n, k, group):
    packed, scale, _ = _weight(n, k, group)
    return _device().weight_i4(packed.cpu().numpy(), scale.cpu().numpy(), k, group)


class _Dev:
    """A torch tensor as the entry points take it: a device pointer."""

    def __init__(self, t):
        self.t, self.ptr = t, ctypes.c_void_p(t.data_ptr())


def _dtype(s):
    eg = _package()
    return {"fp32": eg.F32, "fp16": eg.F16, "bf16": eg.BF16}[s["type"]]


# ------------------------------------------------------------ prepare
def prepare(case, seed):
    s = dict(case)
    s.pop("name", None)
    kind, dtype = case["kind"], _TYPES[case["type"]]
    if kind == "linear":
        n, k, group = case["n"], case["k"], case["group"]
        s["packed"], s["scale"], bias = _weight(n, k, group)
        s["x"] = _Dev(_activations(seed, case["rows"], k).to(dtype))
        s["bias"] = _Dev(bias)
        s["y"] = _Dev(torch.empty((case["rows"], n), dtype=dtype, device=_WHERE))
        if own:
            s["w"] = _weight_i4(n, k, group)
        return s
    heads, kv, dim, block = case["heads"], case["kv_heads"], case["dim"], case["block"]
    s["cu_k"] = _offsets(case["keys"])
    s["cb"] = _block_offsets(s["cu_k"], block)
    s["host_cu_k"] = np.array(s["cu_k"], np.int32)
    keys = _keys(seed, 1, s["cu_k"], kv, dim).to(dtype)
    if kind == "means":
        s["keys"] = _Dev(keys)
        s["means"] = _Dev(torch.empty((s["cb"][-1], kv, dim), device=_WHERE))
    else:
        top = case["top"]
        s["cu_q"] = _offsets(case["queries"])
        s["host_cu_q"] = np.array(s["cu_q"], np.int32)
        rows = s["cu_q"][-1]
        drift = _randn(seed, 5, (rows // 48 + 1, heads, dim))[torch.arange(rows, device=_WHERE) // 48]
        q = (drift + _randn(seed, 6, (rows, heads, dim))) * (dim ** -0.5)
        s["q"] = _Dev(q.to(dtype))
        means = _means(keys, s["cu_k"], s["cb"], block)
        if kind == "select":
            s["means"] = _Dev(means)
            s["blocks"] = _Dev(torch.empty((rows, heads, top), dtype=torch.int32, device=_WHERE))
        else:
            s["keys"] = _Dev(keys)
            s["values"] = _Dev(_keys(seed, 3, s["cu_k"], kv, dim).to(dtype))
            s["blocks"] = _Dev(_select(s["q"].t, means, s["cu_q"], s["cb"], top))
            s["y"] = _Dev(torch.empty((rows, heads * dim), dtype=dtype, device=_WHERE))
    if own:
        _device()
    return s


# ------------------------------------------------------------ the plain forms
def _linear(x, packed, scale, bias, k, group):
    codes = torch.stack((packed & 15, packed >> 4), dim=2).reshape(packed.shape[0], -1)[:, :k].float() - 8.0
    w = codes * scale.repeat_interleave(group, dim=1)[:, :k]
    return (torch.matmul(x.float(), w.t()) + bias).to(x.dtype)


def _means(keys, cu_k, cb, block):
    seq, pos = _place(cu_k, keys.device)
    at = torch.tensor(cb[:-1], device=keys.device)[seq] + pos // block
    sums = torch.zeros((cb[-1],) + tuple(keys.shape[1:]), dtype=torch.float64, device=keys.device)
    sums.index_add_(0, at, keys.double())
    count = torch.bincount(at, minlength=cb[-1]).reshape(-1, 1, 1)
    return (sums / count).float()


def _select(q, means, cu_q, cb, top):
    """[rows, heads, top]: the blocks of the `top` largest scores, ascending,
    then -1."""
    rows, heads, dim = q.shape
    kv, total = means.shape[1], means.shape[0]
    out = torch.full((rows, heads, top), -1, dtype=torch.int32, device=q.device)
    if rows == 0 or total == 0:
        return out
    seq, _ = _place(cu_q, q.device)
    first = torch.tensor(cb[:-1], device=q.device)[seq]
    last = torch.tensor(cb[1:], device=q.device)[seq]
    qh = q.double().reshape(rows, kv, heads // kv * dim).transpose(0, 1).reshape(kv, rows * (heads // kv), dim)
    score = torch.matmul(qh, means.double().permute(1, 2, 0).contiguous()).reshape(kv, rows, heads // kv, total)
    at = torch.arange(total, device=q.device)
    inside = (at >= first[:, None]) & (at < last[:, None])
    score = score.masked_fill(torch.isnan(score), -math.inf).masked_fill_(~inside[None, :, None, :], -math.inf)
    # Blocks of other sequences come behind every one of the query's own.
    order = torch.sort(score, dim=3, descending=True, stable=True).indices
    own_first = torch.sort((~inside[None, :, None, :].expand(score.shape).gather(3, order)).to(torch.uint8), dim=3,
                           stable=True).indices
    picked = order.gather(3, own_first[..., :top])
    n = min(top, total)
    valid = torch.arange(n, device=q.device) < (last - first)[None, :, None, None]
    picked = torch.where(valid, picked - first[None, :, None, None], total).sort(dim=3).values
    picked = torch.where(picked < total, picked, -1)
    out[:, :, :n] = picked.permute(1, 0, 2, 3).reshape(rows, heads, n).to(torch.int32)
    return out


def _softmax_times(score, allowed, values):
    """softmax over the allowed keys (rows with none: 0), times the values."""
    score = score.masked_fill_(~allowed, -math.inf)
    most = score.amax(dim=-1, keepdim=True)
    p = torch.exp(score.sub_(torch.where(torch.isinf(most), 0.0, most)))
    total = p.sum(dim=-1, keepdim=True)
    return torch.matmul(p, values) / torch.where(total > 0, total, 1.0)


def _attend(q, keys, values, blocks, cu_q, cu_k, cb, block):
    rows, heads, dim = q.shape
    kv, top, n_keys = keys.shape[1], blocks.shape[2], keys.shape[0]
    each = heads // kv
    seq, _ = _place(cu_q, q.device)
    first = torch.tensor(cb[:-1], device=q.device)[seq]
    lengths = torch.tensor(cu_k, device=q.device)
    if rows * heads * top * block < kv * n_keys:  # few rows: gather what they list
        starts = lengths[:-1][seq][:, None, None, None]
        ends = lengths[1:][seq][:, None, None, None]
        at = starts + blocks[..., None].long() * block + torch.arange(block, device=q.device)
        allowed = ((blocks[..., None] >= 0) & (at < ends)).reshape(rows, heads, 1, top * block)
        at = torch.where(at < ends, at, 0).clamp_(min=0).reshape(rows, heads, top * block)
        head = (torch.arange(heads, device=q.device) // each)[None, :, None]
        score = torch.matmul(q.float()[:, :, None, :], keys[at, head].float().transpose(2, 3).contiguous())
        return _softmax_times(score, allowed, values[at, head].float()).reshape(rows, heads * dim).to(q.dtype)
    qh, kh, vh = (x.float().transpose(0, 1).contiguous() for x in (q, keys, values))
    score = torch.matmul(qh.reshape(kv, each * rows, dim), kh.transpose(1, 2).contiguous())
    listed_blocks = torch.zeros((heads, rows, cb[-1] + 1), dtype=torch.bool, device=q.device)
    at = torch.where(blocks >= 0, blocks + first[:, None, None], cb[-1]).permute(1, 0, 2).long()
    listed_blocks.scatter_(2, at, True)
    kseq, kpos = _place(cu_k, q.device)
    block_of = torch.tensor(cb[:-1], device=q.device)[kseq] + kpos // block
    allowed = listed_blocks[:, :, block_of].reshape(kv, each * rows, n_keys)
    y = _softmax_times(score, allowed, vh).reshape(heads, rows, dim)
    return y.transpose(0, 1).reshape(rows, heads * dim).to(q.dtype)


# ------------------------------------------------------------ run
def run(s):
    kind = s["kind"]
    if own:
        dev, dtype = _device(), _dtype(s)
        if kind == "linear":
            dev.linear_i4(s["x"], s["w"], s["bias"], s["y"], s["rows"], s["n"], s["k"], dtype)
            return s["y"].t
        shape = (s["heads"], s["kv_heads"], s["dim"], s["block"])
        if kind == "means":
            dev.key_block_means(s["keys"], s["host_cu_k"], s["kv_heads"], s["dim"], s["block"], s["means"], dtype)
            return s["means"].t
        if kind == "select":
            dev.attention_select_blocks(s["q"], s["means"], s["host_cu_q"], s["host_cu_k"], *shape, s["top"],
                                        s["blocks"], dtype)
            return s["blocks"].t
        dev.attention_blocks(s["q"], s["keys"], s["values"], s["blocks"], s["host_cu_q"], s["host_cu_k"], *shape,
                             s["top"], s["y"], dtype)
        return s["y"].t
    if kind == "linear":
        return _linear(s["x"].t, s["packed"], s["scale"], s["bias"].t, s["k"], s["group"])
    if kind == "means":
        return _means(s["keys"].t, s["cu_k"], s["cb"], s["block"])
    if kind == "select":
        return _select(s["q"].t, s["means"].t, s["cu_q"], s["cb"], s["top"])
    return _attend(s["q"].t, s["keys"].t, s["values"].t, s["blocks"].t, s["cu_q"], s["cu_k"], s["cb"], s["block"])


# ------------------------------------------------------------ work
def work(case):
    size = 4 if case["type"] == "fp32" else 2
    if case["kind"] == "linear":
        m, n, k = case["rows"], case["n"], case["k"]
        groups = (k + case["group"] - 1) // case["group"]
        return {"bytes": size * m * (k + n) + n * ((k + 1) // 2) + 4 * n * groups + 4 * n, "flops": 2.0 * m * n * k}
    heads, kv, dim, block = case["heads"], case["kv_heads"], case["dim"], case["block"]
    cu_k = _offsets(case["keys"])
    cb = _block_offsets(cu_k, block)
    if case["kind"] == "means":
        return {"bytes": cu_k[-1] * kv * dim * size + cb[-1] * kv * dim * 4, "flops": 1.0 * cu_k[-1] * kv * dim}
    cu_q = _offsets(case["queries"])
    rows, top = cu_q[-1], case["top"]
    pairs = [(b - a, n, d - c) for a, b, c, d, n in zip(cu_q[:-1], cu_q[1:], cu_k[:-1], cu_k[1:],
                                                         (y - x for x, y in zip(cb[:-1], cb[1:])))]
    if case["kind"] == "select":
        return {"bytes": rows * heads * (dim * size + 4 * top) + cb[-1] * kv * dim * 4,
                "flops": 2.0 * sum(q * n for q, n, _ in pairs) * heads * dim}
    # Keys that a row attends to, and keys that some row may need at all.
    taken = sum(q * min(k, top * block) for q, _, k in pairs) * heads
    needed = sum(min(k * kv, q * heads * min(k, top * block)) for q, _, k in pairs)
    return {"bytes": rows * heads * (2 * dim * size + 4 * top) + 2 * needed * dim * size, "flops": 4.0 * taken * dim}


# ------------------------------------------------------------ 64 bits
def exact(case, seed):
    if case["kind"] == "select":
        return None  # whole numbers
    s = prepare(case, seed)
    if case["kind"] == "linear":
        k, group = case["k"], case["group"]
        codes = torch.empty((case["n"], s["packed"].shape[1] * 2), dtype=torch.float64, device=_WHERE)
        codes[:, 0::2] = (s["packed"] % 16).double() - 8
        codes[:, 1::2] = (s["packed"] // 16).double() - 8
        x = s["x"].t.double()
        y = s["bias"].t.double().expand(case["rows"], case["n"]).clone()
        for g in range(s["scale"].shape[1]):
            a, b = g * group, min(k, (g + 1) * group)
            y += torch.matmul(x[:, a:b], codes[:, a:b].t()) * s["scale"][:, g].double()
        return y
    keys = s["keys"].t.double()
    if case["kind"] == "means":
        rows = []
        for a, b in zip(s["cu_k"][:-1], s["cu_k"][1:]):
            for at in range(a, b, case["block"]):
                rows.append(keys[at:min(b, at + case["block"])].mean(dim=0))
        return torch.stack(rows) if rows else torch.empty_like(s["means"].t).double()
    q, values = s["q"].t.double(), s["values"].t.double()
    blocks, block = s["blocks"].t.long(), case["block"]
    y = torch.zeros_like(q)
    for b in range(len(s["cu_q"]) - 1):
        q0, q1, k0, k1 = s["cu_q"][b], s["cu_q"][b + 1], s["cu_k"][b], s["cu_k"][b + 1]
        if q0 == q1 or k0 == k1:
            continue
        n = (k1 - k0 + block - 1) // block
        key_block = torch.arange(k1 - k0, device=_WHERE) // block
        for h in range(case["heads"]):
            hk = h // (case["heads"] // case["kv_heads"])
            chosen = torch.zeros((q1 - q0, n + 1), dtype=torch.float64, device=_WHERE)
            mine = blocks[q0:q1, h]
            chosen.scatter_(1, torch.where(mine < 0, n, mine), 1.0)
            score = torch.matmul(q[q0:q1, h], keys[k0:k1, hk].t().contiguous())
            bias = torch.log(chosen[:, :n])[:, key_block]
            y[q0:q1, h] = torch.matmul(torch.softmax(score + bias, dim=1), values[k0:k1, hk].contiguous())
    return y.reshape(q.shape[0], -1)
