"""hk_gemm_lora against 64 bits: y_i = W x_i + s_a B_a (A_a x_i), adapters of
different ranks, rows without one, tiles shared by several adapters."""
import sys

import numpy as np
import pytest

from tests import hk_rowsutil as R
from tests import hk_testutil as U

pytestmark = pytest.mark.gpu
TYPES = [("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32"), ("f16", "f16"), ("f32", "bf16")]


def say(*a):
    print("[gpu-case]", *a, flush=True)
    sys.stdout.flush()


@pytest.fixture(scope="module")
def ctx():
    from hawking_amd.runtime import Context
    return Context(0)


def _adapter(ctx, rng, rank, rows, cols, dtype, a_scale=1.0, b_scale=1.0):
    a, ae = R.to_type(rng.standard_normal((rank, cols)) * a_scale / np.sqrt(cols), dtype)
    b, be = R.to_type(rng.standard_normal((rows, rank)) * 0.1 * b_scale, dtype)
    return ctx.to_device(a), ctx.to_device(b), ae, be


def _exact(xe, we, ids, adapters, x_type, y_type):
    """y and the bound before its rounding.  The adapter's part adds: A x (as a
    product of exact weights), mid rounded to f16 (y bf16: 2^-11; else two f16:
    2^-22) and below 2^-28 of its row's largest to 2^-39 of it, B mid summed in
    f32 over the rank, and the scale (half a step)."""
    y, bound = xe @ we.T, R.product_bound(xe, we, x_type, y_type)
    for s, (ae, be, scale) in adapters.items():
        at = np.flatnonzero(ids == s)
        if not at.size or ae is None:
            continue
        x = xe[at]
        mid = x @ ae.T
        mb = R.product_bound(x, ae, x_type, "f32" if y_type != "bf16" else "bf16")
        mb = mb + (2.0 ** -11 if y_type == "bf16" else 2.0 ** -22) * (np.abs(mid) + mb) + 2.0 ** -24 * np.abs(mid)
        mb = mb + 2.0 ** -39 * (np.abs(mid) + mb).max(1, keepdims=True)
        y[at] += scale * (mid @ be.T)
        sb = abs(scale) * (mb @ np.abs(be).T + (be.shape[1] * 2.0 ** -23 + 2.0 ** -22) * ((np.abs(mid) + mb) @ np.abs(be).T))
        bound[at] += sb + xe.shape[1] * 2.0 ** -23 * sb
    # the additions of the adapter's part go on in the projection's sums
    return y, bound + 256 * 2.0 ** -23 * (np.abs(xe) @ np.abs(we).T)


def _run(ctx, oracle, kind, rows, cols, ids, ranks, max_rank, x_type, y_type, a_type="bf16", tag=0, in_order=False, scales=(1.0, 1.0),
         stride=0, lead=0):
    from hawking_amd.rows import LoraBank, LoraGemm, RowGroups
    rng = np.random.default_rng(rows + cols + len(ids))
    w, we = R.make_organ(ctx, oracle, kind, rows, cols, 8000 + tag)
    bank = LoraBank(ctx, w, len(ranks), max_rank)
    adapters, keep = {}, []
    for s, r in enumerate(ranks):
        if r == 0:
            continue
        a, b, ae, be = _adapter(ctx, rng, r, rows, cols, a_type, *scales)
        scale = float(np.float32(0.25 * (s + 1)))
        bank.set(s, r, a, b, a_type, scale)
        adapters[s] = (ae, be, scale)
        keep += [a, b]
    n = len(ids)
    ids = np.asarray(ids, np.int32)
    plan = RowGroups(ctx, n, len(ranks)).build(ctx.to_device(ids))
    x, _, xe = R.rows_on(ctx, rng.standard_normal((n, cols)), x_type, stride=cols + stride, lead=lead, fill=np.nan)
    y, yb, _ = R.rows_on(ctx, np.full((n, rows), 5.0), y_type, stride=rows + stride, lead=lead, fill=5.0)
    ctx.device_status()
    LoraGemm(ctx, w, bank, n, x_type, y_type)(x, plan, y, in_order=in_order)
    got, rest = R.read_rows(yb, y)
    assert np.all(rest == 5.0) and ctx.device_status() == 0
    exact, bound = _exact(xe, we, ids, adapters, x_type, y_type)
    over = np.abs(got - exact) - R.rounded(bound, exact, y_type)
    assert over.max() <= 0.0, (float(over.max()), np.unravel_index(np.argmax(over), over.shape))
    if y_type == "f32":
        assert np.linalg.norm(got - exact) <= 2e-5 * np.linalg.norm(exact)
    return got, exact


def _mix(rng, n, slots):
    return rng.integers(-1, slots, n)


@pytest.mark.parametrize("x_type,y_type", TYPES)
@pytest.mark.parametrize("n", [1, 2, 17, 64, 65, 129, 300])
@pytest.mark.parametrize("kind,rows,cols", [("q4", 60, 160), ("q8", 272, 320), ("mixed", 100, 640), ("bin", 33, 128), ("u3", 48, 96)])
def test_lora(ctx, oracle, kind, rows, cols, n, x_type, y_type):
    say("lora", kind, rows, cols, n, x_type, y_type)
    ranks = [16, 1, 0, 33, 64, 7]
    _run(ctx, oracle, kind, rows, cols, _mix(np.random.default_rng(n), n, len(ranks)), ranks, 64, x_type, y_type)


@pytest.mark.parametrize("max_rank,ranks", [(8, [8, 3]), (16, [16]), (32, [32, 5, 17]), (100, [100, 97, 1]), (128, [128, 64]), (256, [256, 129, 31])])
@pytest.mark.parametrize("x_type,y_type", [("bf16", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("a_type", ["bf16", "f16"])
def test_ranks(ctx, oracle, max_rank, ranks, x_type, y_type, a_type):
    say("lora ranks", max_rank, ranks, x_type, y_type, a_type)
    for n in (3, 90):
        _run(ctx, oracle, "q4", 80, 256, _mix(np.random.default_rng(n), n, len(ranks)), ranks, max_rank, x_type, y_type, a_type)


@pytest.mark.parametrize("x_type,y_type", TYPES)
@pytest.mark.parametrize("n", [645, 6605])
@pytest.mark.parametrize("kind,cols", [("q4", 288), ("q8", 192), ("mixed", 640), ("bin", 512), ("u3", 160)])
def test_many_rows(ctx, oracle, kind, cols, n, x_type, y_type):
    """Rows and outputs enough for the kernel that tiles through LDS, with two and with four row tiles a wave."""
    say("lora many rows of all", kind, n, x_type, y_type)
    ranks = [16, 0, 33, 64, 7]
    ids = _mix(np.random.default_rng(cols), n, len(ranks))
    ids[100:400] = 2
    _run(ctx, oracle, kind, 1100, cols, ids, ranks, 64, x_type, y_type, stride=5)


@pytest.mark.parametrize("x_type,y_type", TYPES)
@pytest.mark.parametrize("ranks,max_rank", [([16, 9], 16), ([64, 33, 5, 0], 64), ([128, 40], 128)])
def test_many_rows_a_slot(ctx, oracle, ranks, max_rank, x_type, y_type):
    """Slots of hundreds and thousands of rows, and one of a single row among them."""
    say("lora many rows", ranks, x_type, y_type)
    rng = np.random.default_rng(len(ranks))
    for n in (531, 4200):
        ids = _mix(rng, n, len(ranks))
        ids[ids == len(ranks) - 1] = 0
        ids[n // 2] = len(ranks) - 1
        _run(ctx, oracle, "q4", 52, 288, ids, ranks, max_rank, x_type, y_type)


@pytest.mark.parametrize("ids", [[-1] * 20, [0] * 150, [2] * 5 + [-1] * 5, list(range(70)), [9999, -7, 1]])
def test_who_has_an_adapter(ctx, oracle, ids):
    """No row, every row, one slot of many, a slot a row (one tile, many adapters)."""
    say("lora ids", len(ids))
    for t in (("bf16", "bf16"), ("bf16", "f32")):
        _run(ctx, oracle, "q8", 64, 192, ids, [16] * 70, 16, *t)


@pytest.mark.parametrize("scales", [(1e-6, 1.0), (1e6, 1.0), (1.0, 1e-6), (1e4, 1e4), (1e-15, 1e-15), (1e15, 1e-15)])
def test_magnitudes(ctx, oracle, scales):
    """Adapters far below and far above the projection's part."""
    say("lora magnitudes", scales)
    _run(ctx, oracle, "q4", 48, 256, _mix(np.random.default_rng(0), 40, 3), [8, 16, 24], 32, "bf16", "f32", scales=scales)


@pytest.mark.parametrize("n", [5, 140])
def test_in_order_and_strided(ctx, oracle, n):
    say("lora in order", n)
    ids = np.sort(_mix(np.random.default_rng(n), n, 4)) % 5  # -1 -> 4 (outside), sorted apart
    ids = np.sort(ids)
    _run(ctx, oracle, "q4", 70, 160, ids, [4, 8, 16, 32], 32, "bf16", "f32", in_order=True)
    _run(ctx, oracle, "q4", 70, 160, _mix(np.random.default_rng(n), n, 4), [4, 8, 16, 32], 32, "f32", "bf16", stride=3, lead=1)


@pytest.mark.parametrize("n", [6, 40, 400])
def test_rows_before_the_first_slot(ctx, oracle, n):
    """offsets[0] > 0: the rows before it have no adapter, whatever the workspace holds."""
    from hawking_amd.rows import LoraBank, LoraGemm, RowGroups
    say("lora first rows", n)
    rng = np.random.default_rng(n)
    rows, cols, k = 48, 128, n // 3
    w, we = R.make_organ(ctx, oracle, "q4", rows, cols, 8400)
    bank = LoraBank(ctx, w, 2, 16)
    a, b, ae, be = _adapter(ctx, rng, 16, rows, cols, "bf16")
    bank.set(1, 16, a, b)
    plan = RowGroups(ctx, n, 2, offsets=ctx.to_device(np.array([k, k, n - 1], np.int32)))
    x, _, xe = R.rows_on(ctx, rng.standard_normal((n, cols)), "f32")
    y, yb, _ = R.rows_on(ctx, np.zeros((n, rows)), "f32")
    gemm = LoraGemm(ctx, w, bank, n)
    ctx.device_status()
    for _ in range(2):
        gemm.ws.upload(np.full(gemm.ws.shape, 0x7F, np.uint8))
        gemm(x, plan, y, in_order=True)
        want = xe @ we.T
        want[k:n - 1] += xe[k:n - 1] @ ae.T @ be.T
        got = R.read_rows(yb, y)[0]
        assert ctx.device_status() == 0 and np.linalg.norm(got - want) <= 2e-5 * np.linalg.norm(want)


def test_slots_are_replaced_and_emptied(ctx, oracle):
    from hawking_amd.rows import LoraBank, LoraGemm, RowGroups
    rng = np.random.default_rng(9)
    rows, cols, n = 32, 128, 6
    w, we = R.make_organ(ctx, oracle, "q4", rows, cols, 8100)
    bank = LoraBank(ctx, w, 2, 32)
    plan = RowGroups(ctx, n, 2).build(ctx.to_device(np.array([0, 1, 0, 1, -1, 0], np.int32)))
    x, _, xe = R.rows_on(ctx, rng.standard_normal((n, cols)), "f32")
    y, yb, _ = R.rows_on(ctx, np.zeros((n, rows)), "f32")
    gemm = LoraGemm(ctx, w, bank, n)
    base = xe @ we.T

    def close(want):
        gemm(x, plan, y)
        got = R.read_rows(yb, y)[0]
        assert np.linalg.norm(got - want) <= 2e-5 * np.linalg.norm(want)

    close(base)  # a new bank is empty
    a, b, ae, be = _adapter(ctx, rng, 32, rows, cols, "bf16")
    bank.set(0, 32, a, b)
    want = base.copy()
    want[[0, 2, 5]] += xe[[0, 2, 5]] @ ae.T @ be.T
    close(want)
    a2, b2, ae2, be2 = _adapter(ctx, rng, 3, rows, cols, "bf16")  # a smaller one over it
    bank.set(0, 3, a2, b2, scale=-2.0)
    want = base.copy()
    want[[0, 2, 5]] += -2.0 * (xe[[0, 2, 5]] @ ae2.T @ be2.T)
    close(want)
    bank.set(0, 0, None, None)
    close(base)


def test_nonfinite_adapter(ctx, oracle):
    from hawking_amd.rows import LoraBank, LoraGemm, RowGroups
    rng = np.random.default_rng(10)
    rows, cols, n = 32, 128, 4
    w, we = R.make_organ(ctx, oracle, "q4", rows, cols, 8200)
    bank = LoraBank(ctx, w, 2, 16)
    a, b, ae, be = _adapter(ctx, rng, 16, rows, cols, "bf16")
    bad, _ = R.to_type(np.where(np.arange(rows * 16).reshape(rows, 16) == 5, np.inf, 0.1), "bf16")
    ctx.device_status()
    bank.set(0, 16, a, b)
    assert ctx.device_status() == 0
    bank.set(1, 16, a, ctx.to_device(bad))
    assert ctx.device_status() & 1
    plan = RowGroups(ctx, n, 2).build(ctx.to_device(np.array([0, 1, -1, 0], np.int32)))
    x, _, xe = R.rows_on(ctx, rng.standard_normal((n, cols)), "f32")
    y, yb, _ = R.rows_on(ctx, np.zeros((n, rows)), "f32")
    LoraGemm(ctx, w, bank, n)(x, plan, y)
    got = R.read_rows(yb, y)[0]
    want = xe @ we.T
    want[[0, 3]] += xe[[0, 3]] @ ae.T @ be.T
    assert np.all(np.isnan(got[1])) and ctx.device_status() & 1
    assert np.linalg.norm(got[[0, 2, 3]] - want[[0, 2, 3]]) <= 2e-5 * np.linalg.norm(want)


def test_lora_refusals(ctx, oracle):
    from hawking_amd._lib import HK_E_GEOMETRY, HK_E_INVALID_ARG, HK_E_UNSUPPORTED, HawkingError
    from hawking_amd.organs import DenseF32Organ
    from hawking_amd.rows import LoraBank, LoraGemm, RowGroups
    w = R.make_organ(ctx, oracle, "q4", 32, 128, 8300)[0]

    def code(fn):
        with pytest.raises(HawkingError) as e:
            fn()
        return e.value.code

    assert code(lambda: LoraBank(ctx, w, 0, 16)) == HK_E_UNSUPPORTED
    assert code(lambda: LoraBank(ctx, w, 1, 257)) == HK_E_UNSUPPORTED
    assert code(lambda: LoraBank(ctx, DenseF32Organ(ctx, np.zeros((8, 128), np.float32)), 1, 16)) == HK_E_UNSUPPORTED
    bank = LoraBank(ctx, w, 2, 16)
    d = ctx.empty(4096, np.uint16)
    assert code(lambda: bank.set(2, 16, d, d)) == HK_E_INVALID_ARG
    assert code(lambda: bank.set(0, 17, d, d)) == HK_E_GEOMETRY
    assert code(lambda: bank.set(0, 16, d, d, "f32")) == HK_E_UNSUPPORTED
    assert code(lambda: bank.set(0, 16, None, d)) == HK_E_INVALID_ARG
    plan = RowGroups(ctx, 4, 2).build(ctx.to_device(np.zeros(4, np.int32)))
    x, _, _ = R.rows_on(ctx, np.zeros((4, 128)), "f32")
    y, _, _ = R.rows_on(ctx, np.zeros((4, 32)), "f32")
    y3, _, _ = R.rows_on(ctx, np.zeros((3, 32)), "f32")
    gemm = LoraGemm(ctx, w, bank, 4)
    assert code(lambda: gemm(x, RowGroups(ctx, 3, 2).build(ctx.to_device(np.zeros(3, np.int32))), y3)) == HK_E_GEOMETRY
    with pytest.raises(ValueError):
        gemm(x, plan, y3)
    with pytest.raises(ValueError):
        gemm(x, RowGroups(ctx, 4, 1).build(ctx.to_device(np.zeros(4, np.int32))), y)  # a bank of two slots
    with pytest.raises(ValueError):
        bank.set(0, 16, ctx.empty(16 * 128 - 1, np.uint16), d)
    other = R.make_organ(ctx, oracle, "q4", 32, 160, 8301)[0]
    assert code(lambda: ctx.call("hk_gemm_lora", other.h, bank.h, x.ref, None, plan.offsets.ptr, y.ref, gemm.ws.ptr,
                                 gemm.ws_bytes, None)) == HK_E_GEOMETRY
