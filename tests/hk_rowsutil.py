"""Shared by the row-product tests: organs with their exact weights, rows in
every type, and the error bounds the products are held to.

Bounds (elementwise, of |y - exact|), counting every rounding:
  sums      cols additions in f32, each at most 2^-23 of the sum S = sum |w x|
            (half a step when rounded to nearest, a whole one when cut off)
  weights   y bf16: code * scale rounded to f16, 2^-11 of each; y f32 or f16:
            exact (two f16)
  x         bf16, f16: exact.  f32: y bf16: f16, 2^-11 of each; else two f16,
            2^-22 of each, and the left-out product of the two remainders, 2^-22
  f16 range values below 2^-28 of their row's largest lose up to 2^-39 of it
            (the f16 subnormals): cols 2^-39 max |x| max |w|
  y         half a step of its type: f32 2^-24, f16 2^-11, bf16 2^-8 of |y|
            (f16 below 2^-14: 2^-25)
"""
from __future__ import annotations

import numpy as np

from tests import hk_testutil as U

KINDS = {"q4": 0, "bin": 1, "mixed": 2, "q8": 4, "u3": 5}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def key(oracle, *tag):
    k = 0
    for t in tag:
        k = k * 1009 + int(t)
    return oracle.stream_key(U.SEED, (0x206 << 48) ^ (k & ((1 << 44) - 1)))


def make_organ(ctx, oracle, kind, rows, cols, tag, group=32, sigma=0.02):
    """(organ, exact f64 weights): N(0, sigma) packed by the oracle."""
    from hawking_amd import organs as O
    w = oracle.normal(key(oracle, 1, tag), rows * cols, sigma).reshape(rows, cols)
    if kind == "q4":
        s, c = oracle.q4_pack(w, group)
        return O.Qwen80Q4PackedTensor(ctx, s, c, rows, cols, group), oracle.q4_decode(s, c, rows, cols, group).astype(np.float64).reshape(rows, cols)
    if kind == "bin":
        s, g = oracle.bin_pack(w)
        return O.BinaryGroupPacked(ctx, s, g, rows, cols), oracle.bin_decode(s, g, rows, cols).astype(np.float64).reshape(rows, cols)
    if kind in ("q8", "u3"):
        bits = 8 if kind == "q8" else 3
        s, c = oracle.uniform_pack(w, rows, cols, bits, 64)
        cls = O.UniformFactorPacked if kind == "q8" else O.UniformFactor3
        return cls(ctx, s, c, rows, cols), oracle.uniform_decode(s, c, rows, cols, bits, 64).astype(np.float64).reshape(rows, cols)
    m = oracle.mixed_pack(w, oracle.mixed_coins(key(oracle, 2, tag), rows * cols // 128))
    return (O.MixedPackedTensor(ctx, rows, cols, m.tags, m.bin_scales, m.bin_signs, m.q2_scales, m.q2_codes),
            oracle.mixed_decode(m).astype(np.float64).reshape(rows, cols))


def to_type(a, dtype):
    """f32 values -> (the array as stored, its exact f64 values)."""
    a = np.ascontiguousarray(a, np.float32)
    if dtype == "f32":
        return a, a.astype(np.float64)
    if dtype == "f16":
        h = a.astype(np.float16)
        return h, h.astype(np.float64)
    b = U.to_bf16_bits(a)
    return b, U.bf16_to_f32(b).astype(np.float64).reshape(a.shape)


def from_type(a, dtype):
    return U.bf16_to_f32(a).astype(np.float64).reshape(a.shape) if dtype == "bf16" else a.astype(np.float64)


def np_type(dtype):
    return {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}[dtype]


def rows_on(ctx, values, dtype, stride=None, lead=0, fill=0.0):
    """Device rows of `values` [n, cols] with `stride` elements a row, `lead`
    elements into an allocation whose other elements hold `fill`; returns
    (Rows, buffer, exact f64 values)."""
    from hawking_amd.rows import Rows
    n, cols = values.shape
    stride = cols if stride is None else stride
    full = np.full(lead + max(n, 1) * stride + 8, fill, np.float32)
    body = full[lead:lead + max(n, 1) * stride].reshape(max(n, 1), stride)
    body[:n, :cols] = values
    stored, exact = to_type(full, dtype)
    buf = ctx.to_device(stored)
    exact = exact[lead:lead + max(n, 1) * stride].reshape(max(n, 1), stride)[:n, :cols]
    rows = Rows(buf.offset(lead), n, cols, dtype, stride)
    rows.owner = buf  # the allocation lives as long as the rows
    return rows, buf, exact


def read_rows(buf, rows):
    """(the rows' values, every other element of the allocation) in f64."""
    a = from_type(buf.download(), rows.dtype)
    lead = (rows.src.data - buf.addr) // buf.dtype.itemsize
    body = a[lead:lead + max(rows.n, 1) * rows.stride].reshape(max(rows.n, 1), rows.stride)
    out = body[:rows.n, :rows.cols].copy()
    rest = a.copy()
    rest[lead:lead + max(rows.n, 1) * rows.stride].reshape(max(rows.n, 1), rows.stride)[:rows.n, :rows.cols] = np.nan
    return out, rest[~np.isnan(rest)]


def product_bound(x, w, x_type, y_type):
    """Bound on the error of x w^T before the rounding to y's type (x, w exact f64)."""
    cols = x.shape[1]
    s = np.abs(x) @ np.abs(w).T
    eps = cols * 2.0 ** -23
    if y_type == "bf16":
        eps += 2.0 ** -11 + (2.0 ** -11 if x_type == "f32" else 0.0)
    elif x_type == "f32":
        eps += 2.0 ** -21
    tiny = cols * 2.0 ** -39 * np.abs(x).max(1, initial=0.0)[:, None] * np.abs(w).max(initial=0.0)
    return eps * s + tiny


def rounded(bound, exact, y_type):
    b = bound + HALF_STEP[y_type] * (np.abs(exact) + bound)
    return b + 2.0 ** -25 if y_type == "f16" else b


def silu(v):
    return v / (1.0 + np.exp(-v))


def swiglu_bound(g, bg, u, bu):
    """|silu'| <= 1.1; e^v, the division and two products in f32: 8 steps of the value."""
    sg = np.abs(silu(g))
    return 1.1 * bg * (np.abs(u) + bu) + sg * bu + 2.0 ** -20 * (sg * np.abs(u))


def group_oracle(ids, groups):
    ids = np.asarray(ids, np.int64)
    k = np.where((ids >= 0) & (ids < groups), ids, groups)
    order = np.argsort(k, kind="stable").astype(np.int32)
    offsets = np.searchsorted(k[order], np.arange(groups + 1)).astype(np.int32)
    pos = np.empty(ids.size, np.int32)
    pos[order] = np.arange(ids.size, dtype=np.int32)
    pos[k == groups] = -1
    return offsets, order, pos
