"""Top logits, distillation and verification of drafts on the GPU against their float64 forms (tests/student.py).

Tolerances.  Indices, values, tokens and counts are exact.  Of the rest, with eps = 2^-24 (half a step of fp32):
  a term 2^((x - m) c) is off by 4 eps (the hardware's exponential) and by its argument's roundings: difference, product and c,
      3 eps |arg|, where terms that matter to a sum have arg of ln C + 1 on average
  a sum of them by the additions a thread makes in turn (64 in registers, a few hundred where a long row is walked in
      slices or streamed) and those of the tree above: `adds` eps
so a sum, and with it a probability or a normaliser, is off by SUM(C, adds) = eps (4 + 3 (ln C + 1) + adds).
"""
import numpy as np
import pytest

from zigrad_b200 import abi, opspec
from zigrad_b200.device import CudaDevice, DeviceSlice

from . import student
from .backends import GpuBackend

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24
HALF_STEP = {"f32": EPS, "bf16": 2.0 ** -8}


def rng(seed):
    return np.random.Generator(np.random.PCG64(seed))


def sum_error(C, adds):
    return EPS * (4 + 3 * (np.log(C) + 1) + adds)


def adds_for(C):
    return 80 + C // 256  # one thread of 256 over a whole row at worst


def up(be, a, dtype=None, offset=0):
    """A slice whose first element lies `offset` elements behind a 256-byte boundary."""
    a = np.ascontiguousarray(a) if dtype is None else np.ascontiguousarray(a, dtype)
    s = be.up(np.concatenate([np.zeros(offset, a.dtype), a.ravel()]), a.dtype)
    return s.view(offset, a.size)


def rows_with_ld(a, ld, fill):
    out = np.full((a.shape[0], ld), fill, a.dtype)
    out[:, :a.shape[1]] = a
    return out


def logits(g, rows, C):
    x = g.standard_normal((rows, C)) * 2
    at = g.integers(0, C, (rows, min(C, 12)))
    np.put_along_axis(x, at, g.random(at.shape) * 12, 1)
    return x.astype(np.float32)


# ------------------------------------------------------------------------------------------------ top logits
def run_top(gpu, x, k, dtype, T=1.0, ld=None, offset=0, lse=True):
    rows, C = x.shape
    raw, held = student.stored(x, dtype)
    ld = ld or C
    be = GpuBackend(gpu)
    nan = np.uint16(0x7FC0) if dtype == "bf16" else np.float32(np.nan)  # between the rows: above everything, if it were read
    X = up(be, rows_with_ld(raw, ld, nan), offset=offset)
    V, I, L = up(be, np.zeros(rows * k, raw.dtype)), up(be, np.zeros(rows * k, np.uint64)), up(be, np.zeros(rows, np.float32))
    gpu.dispatch(opspec.top_logits(X, rows, C, k, V, I, lse=L if lse else None, temperature=T, ld=ld if ld != C else 0))
    v, i, l = gpu.to_numpy(V, (rows, k)), gpu.to_numpy(I, (rows, k)), gpu.to_numpy(L)
    be.down(L)
    return (student.bf16_values(v) if dtype == "bf16" else v), i, l, held


def check_top(gpu, x, k, dtype, T=1.0, **kw):
    v, i, l, held = run_top(gpu, x, k, dtype, T, **kw)
    wv, wi, wl = student.top_logits(held, k, T)
    np.testing.assert_array_equal(i, wi)
    np.testing.assert_array_equal(v, wv.astype(np.float32))
    if kw.get("lse", True):
        np.testing.assert_array_equal(np.isfinite(l), np.isfinite(wl))
        ok = np.isfinite(wl)
        assert (np.abs(l - wl)[ok] <= sum_error(x.shape[1], adds_for(x.shape[1])) + 2 * EPS * np.abs(wl[ok])).all(), np.abs(l - wl)[ok].max()


CLASSES = [1, 2, 7, 8, 9, 33, 64, 255, 257, 511, 512, 513, 1003, 2048, 4099, 9000, 20001, 50021]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("C", CLASSES)
def test_top_logits(gpu, dtype, C):
    g = rng(C)
    for rows, k in ((1, 1), (3, min(C, 5)), (5, min(C, 64)), (2, min(C, 300)), (17 if C < 3000 else 2, min(C, 1024))):
        check_top(gpu, logits(g, rows, C), k, dtype, T=float(g.choice([1.0, 2.5])), offset=int(g.integers(0, 9)), ld=C + int(g.integers(0, 3)))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,C,k", [(1, 131072, 8), (2, 200003, 64), (40, 30000, 20), (150, 9001, 40), (700, 1500, 10), (5000, 79, 4), (9, 150001, 1024)])
def test_top_logits_of_many_rows_and_long_ones(gpu, dtype, rows, C, k):
    check_top(gpu, logits(rng(rows + C), rows, C), k, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("C,k", [(40, 7), (600, 600), (5000, 33), (70001, 1000), (140000, 64)])
def test_top_logits_of_rows_that_give_no_bound(gpu, dtype, C, k):
    g = rng(C + k)
    far = logits(g, 1, C)[0]
    some = np.where(g.random(C) < 0.5 * k / C, far, -np.inf)            # fewer finite values than k, most likely
    period = np.where(np.arange(C) % 2048 < 8, np.abs(far) + 20, far)   # the large ones side by side
    with_nan = far.copy()
    with_nan[g.integers(0, C, 3)] = np.nan
    plus = far.copy()
    plus[g.integers(0, C, 2)] = np.inf
    low = np.full(C, np.finfo(np.float32).min, np.float32)              # a mask of the type's lowest value over almost everything
    low[: C // 50 + 1] = far[: C // 50 + 1]
    zeros = np.where(np.arange(C) % 3 == 0, -0.0, 0.0)
    x = np.stack([np.zeros(C), np.full(C, -np.inf), some, np.sort(far), np.sort(far)[::-1], period, np.round(far), low, zeros]).astype(np.float32)
    check_top(gpu, x, k, dtype, lse=False)
    check_top(gpu, x[[0, 2, 3, 4, 5, 6]], k, dtype)
    check_top(gpu, np.stack([with_nan, plus, np.full(C, np.nan)]).astype(np.float32), k, dtype, lse=False)
    l = run_top(gpu, np.stack([with_nan, plus, x[1]]).astype(np.float32), k, dtype)[2]
    assert np.isnan(l[0]) and l[1] == np.inf and l[2] == -np.inf


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,C,k", [(90, 40003, 50), (90, 9001, 1024), (300, 300, 20)])
def test_top_logits_of_many_rows_of_ties(gpu, dtype, rows, C, k):
    """As many rows as leave a row to one CTA (to one warp): the digits' search there."""
    k = min(k, C)
    g = rng(C)
    x = np.round(logits(g, rows, C) / 4)
    x[::3] = 0.0
    x[1::3] = np.where(g.random((len(x[1::3]), C)) < 0.5 * k / C, x[1::3], -np.inf)
    check_top(gpu, x.astype(np.float32), k, dtype, lse=False, offset=1)


# ------------------------------------------------------------------------------------------------ distillation
def teacher_lists(g, x, k, tail, T, ragged=False, t_dtype="f32"):
    rows, C = x.shape
    t = (x + g.standard_normal(x.shape)).astype(np.float32)
    v, i, _ = student.top_logits(t, k)
    raw, held = student.stored(v, t_dtype)
    if ragged:
        for r in range(rows):
            i[r, g.integers(0, k + 1):] = C + 3 if r % 2 else student.NO_TOKEN
    return raw, held, i, (student.lse(t.astype(np.float64) / T).astype(np.float32) if tail else None)


def run_distill(gpu, x, raw_u, i, t_lse, dtype, T=1.0, weight=None, loss_div=3.0, ld=None, offset=0, grad_offset=None, mode="write"):
    """-> loss, row losses, gradient [rows, C], what the gradient's buffer held before"""
    rows, C = x.shape
    raw, _ = student.stored(x, dtype)
    ld = ld or C
    be = GpuBackend(gpu)
    nan = np.uint16(0x7FC0) if dtype == "bf16" else np.float32(np.nan)
    X = up(be, rows_with_ld(raw, ld, nan), offset=offset)
    before = np.zeros((rows, C), np.float32)
    G = X if mode == "inplace" else None
    if mode in ("write", "add"):
        old, before = student.stored(rng(1).standard_normal((rows, C)).astype(np.float32), dtype)
        G = up(be, rows_with_ld(old, ld, nan), offset=offset if grad_offset is None else grad_offset)
    U, I = up(be, raw_u), up(be, i, np.uint64)
    L = up(be, t_lse) if t_lse is not None else None
    W = up(be, weight, np.float32) if weight is not None else None
    loss, row = up(be, np.full(1, 7.0, np.float32)), up(be, np.full(rows, 7.0, np.float32))
    gpu.dispatch(opspec.distill_ce(X, I, U, rows, C, i.shape[1], loss, row, grad=G, t_lse=L, row_weight=W, temperature=T, loss_div=loss_div,
                                   accumulate=mode == "add", ld=ld if ld != C else 0))
    got_loss, got_row = float(gpu.to_numpy(loss)[0]), gpu.to_numpy(row)
    got = None
    if G is not None:
        full = gpu.to_numpy(G, (rows, ld))
        if ld > C:  # what lies between the rows stays as it was
            np.testing.assert_array_equal(full[:, C:].view(np.uint8), rows_with_ld(raw, ld, nan)[:, C:].copy().view(np.uint8))
        got = np.ascontiguousarray(full[:, :C])
        got = student.bf16_values(got) if dtype == "bf16" else got
    be.down(row)
    return got_loss, got_row, got, before


def check_distill(gpu, x, raw_u, held_u, i, t_lse, dtype, T=1.0, weight=None, loss_div=3.0, mode="write", **kw):
    rows, C = x.shape
    _, held = student.stored(x, dtype)
    loss, row, grad, before = run_distill(gpu, x, raw_u, i, t_lse, dtype, T, weight, loss_div, mode=mode, **kw)
    want_row, want, part = student.distill(held, i, held_u, t_lse, weight, T, loss_div)
    w = np.ones(rows) if weight is None else np.asarray(weight, np.float64)
    d = sum_error(C, adds_for(C))
    dq = EPS * (4 + part["far"])                      # expf of an argument that was rounded to fp32
    every = part["mass"] + part["rest"]
    # the student's sums enter as log p; the list's masses with the logarithms of their quotients, which |row| + 30 covers, and
    # through rest = 1 - mass, whose term has the derivative log rest - log p_rest + 1
    row_tol = np.abs(w) * (2 * d * every + dq * part["mass"] * (np.abs(want_row) + 31 + part["log_quotient"])) + 2 * EPS * np.abs(want_row)
    assert (np.abs(row - want_row) <= row_tol).all(), (np.abs(row - want_row) / row_tol).max()
    assert abs(loss - want_row.sum() / loss_div) <= row_tol.sum() / abs(loss_div) + 2 * EPS * abs(loss)
    if mode == "none":
        return
    # p: both sums; in the list q; outside it p / p_rest of what mass and p_rest are off by
    scale = np.abs(w / (T * loss_div))[:, None]
    p, q = part["p"], part["q"]
    outside = part["share"] * ((part["rest"] > 0) * (part["mass"] * dq + 2 * d * (1 - part["p_rest"]) * every))[:, None]
    tol = scale * (3 * d * every[:, None] * p + dq[:, None] * q + outside) + 4 * EPS * np.abs(want)
    total = want if mode != "add" else want + np.where(w[:, None] == 0, 0.0, 1.0) * before + np.where(w[:, None] == 0, 1.0, 0.0) * before
    tol = tol + HALF_STEP[dtype] * np.abs(total) * 1.01 + 1e-37
    off = np.abs(grad - total)
    assert (off <= tol).all(), ((off / tol).max(), np.argwhere(off > tol)[:5])


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("C", CLASSES)
def test_distillation(gpu, dtype, C, tail):
    g = rng(C + tail)
    for rows, k in ((1, 1), (3, min(C, 5)), (9, min(C, 64)), (2, min(C, 700))):
        x, T, t_dtype = logits(g, rows, C), float(g.choice([1.0, 3.0])), str(g.choice(["f32", "bf16"]))
        raw, held, i, l = teacher_lists(g, x, k, tail, T, ragged=bool(g.integers(0, 2)), t_dtype=t_dtype)
        weight = np.where(g.random(rows) < 0.3, 0.0, g.random(rows) * 2).astype(np.float32) if g.random() < 0.5 else None
        mode = str(g.choice(["write", "add", "inplace", "none"]))
        offset = int(g.integers(0, 9))
        check_distill(gpu, x, raw, held, i, l, dtype, T, weight, mode=mode, offset=offset, ld=C + int(g.integers(0, 3)),
                      grad_offset=offset if g.random() < 0.5 else offset + 1)


@pytest.mark.parametrize("mode", ["write", "add", "inplace", "none"])
@pytest.mark.parametrize("dtype,rows,C,k,tail", [("bf16", 3, 131072, 64, True), ("f32", 2, 131073, 100, True), ("bf16", 2, 300007, 64, False),
                                                 ("f32", 200, 1000, 10, False), ("bf16", 160, 8000, 32, True), ("f32", 3000, 10, 3, True), ("f32", 310, 4097, 33, True)])
def test_distillation_of_many_rows_and_long_ones(gpu, dtype, rows, C, k, tail, mode):
    g = rng(rows + C)
    x = logits(g, rows, C)
    raw, held, i, l = teacher_lists(g, x, k, tail, 1.0)
    check_distill(gpu, x, raw, held, i, l, dtype, mode=mode, loss_div=float(rows))


@pytest.mark.parametrize("mode", ["write", "add", "inplace", "none"])
@pytest.mark.parametrize("dtype,C,k,tail", [("f32", 376841, 1024, True), ("f32", 800003, 64, False), ("bf16", 753671, 33, True), ("bf16", 1500007, 1024, False)])
def test_distillation_of_rows_longer_than_a_clusters_shared_memory(gpu, dtype, C, k, tail, mode):
    g = rng(C)
    x = logits(g, 3, C)
    raw, held, i, l = teacher_lists(g, x, k, tail, 2.0)
    i[0, 3] = i[0, k - 1]                      # twice, in one slice or in two entries far apart
    i[1, :] = np.roll(i[1], 7)
    if l is not None:
        l = l + np.float32(3.0)                # the mass stays below one
    x[2] = np.nan                              # and a row that is not read
    check_distill(gpu, x, raw, held, i, l, dtype, 2.0, np.array([1, 0.5, 0], np.float32), mode=mode, offset=3, ld=C + 2)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("C", [12, 200, 3001, 40000])
def test_lists_in_any_order_with_a_class_more_than_once(gpu, dtype, C, tail):
    g = rng(C)
    x = logits(g, 4, C)
    raw, held, i, l = teacher_lists(g, x, 10, tail, 1.0)
    for r in range(4):
        o = g.permutation(10)
        raw[r], held[r], i[r] = raw[r][o], held[r][o], i[r][o]
    i[0, 7], i[1, :] = i[0, 2], i[1, 0]
    i[2, 0] = i[2, 5] = i[2, 9]
    if l is not None:
        l = l + np.float32(3.0)  # so that lists with repeated classes have a mass below one
    for mode in ("write", "add", "inplace"):
        check_distill(gpu, x, raw, held, i, l, dtype, mode=mode)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("C", [20, 700, 9000, 140001])
def test_masked_students_teachers_and_empty_lists(gpu, dtype, C):
    g = rng(C)
    x = logits(g, 6, C)
    raw, held, i, l = teacher_lists(g, x, 8, True, 1.0)
    lowest = np.float32(-3.3895314e38)  # bf16's lowest value
    at = i.astype(np.int64)
    outside = np.ones((6, C), bool)
    np.put_along_axis(outside, at, False, 1)
    x[0] = np.where(outside[0], -np.inf, x[0])      # the student knows nothing but the list
    x[1] = np.where(outside[1], lowest, x[1])
    x[2, : C // 2] = -np.inf                         # half of the classes are masked, the list's not
    x[2, at[2]] = 1.0
    x[3] = lowest                                    # nothing but the lowest value
    i[4, :] = student.NO_TOKEN                       # an empty list
    held[5, 2:], raw[5, 2:] = -np.inf, student.stored(np.float32(-np.inf), "f32")[0]
    for t_lse in (l, None):
        check_distill(gpu, x, raw, held, i, t_lse, dtype)
    # the student gives a listed class nothing: an infinite divergence, a finite gradient
    x[2, at[2, 0]] = -np.inf
    loss, row, grad, _ = run_distill(gpu, x, raw, i, None, dtype)
    assert row[2] == np.inf and loss == np.inf and np.isfinite(grad).all()
    _, _, want = (None, None, student.distill(student.stored(x, dtype)[1], i, held, None, None, 1.0, 3.0)[1])
    assert abs(grad[2, at[2, 0]] - want[2, at[2, 0]]) <= abs(want[2, at[2, 0]]) * (HALF_STEP[dtype] + 1e-5)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("C", [20, 900, 30000])
def test_rows_that_count_nothing_are_not_read(gpu, dtype, C):
    g = rng(C)
    x = logits(g, 5, C)
    raw, held, i, l = teacher_lists(g, x, 6, True, 1.0)
    weight = np.array([1, 0, 2, 0, 0.5], np.float32)
    x[[1, 3]] = np.nan
    l[1], i[3, :] = np.nan, 5
    for mode in ("write", "add", "inplace"):
        check_distill(gpu, x, raw, held, i, l, dtype, weight=weight, mode=mode)


@pytest.mark.parametrize("mode", ["none", "write"])
@pytest.mark.parametrize("C,k,near", [(700, 5, 0.05), (5003, 30, 0.02), (50021, 12, 0.02), (131072, 64, 0.01)])
def test_small_divergences_keep_their_digits(gpu, C, k, near, mode):
    """Where student and teacher nearly agree the row is a small difference of large logarithms.  An error d of the sum outside the
    list changes it by d (mass - (1 - p_rest)), the rounding of log2(e) / T by EPS max|z - m| times what the masses differ by; the list
    is summed in 64 bits."""
    g = rng(C)
    x = logits(g, 6, C)
    t = (x + near * g.standard_normal(x.shape)).astype(np.float32)
    u, i, _ = student.top_logits(t, k)
    l = student.lse(t.astype(np.float64)).astype(np.float32)
    _, row, _, _ = run_distill(gpu, x, u.astype(np.float32), i, l, "f32", mode=mode)
    want, _, part = student.distill(x, i, u, l)
    p_listed = 1 - part["p_rest"]
    apart = np.abs(part["mass"] - p_listed) + np.abs(part["q"] - np.where(part["q"] > 0, part["p"], 0)).sum(1)
    span = np.abs(x - x.max(1, keepdims=True)).max(1)
    tol = 2 * sum_error(C, adds_for(C)) * np.abs(part["mass"] - p_listed) + EPS * span * apart + 2 * EPS * np.abs(want) + 1e-12
    assert (np.abs(row - want) <= tol).all(), (np.abs(row - want) / tol, want)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("t_dtype,T", [("f32", 1.0), ("bf16", 1.0), ("f32", 2.5), ("bf16", 0.7)])
@pytest.mark.parametrize("dtype,rows,C,k", [("f32", 6, 900, 12), ("bf16", 700, 2003, 20), ("f32", 4, 9001, 200), ("bf16", 160, 50021, 33), ("f32", 3, 140001, 64),
                                            ("f32", 2, 800003, 100), ("bf16", 2, 1500007, 64)])
def test_rows_are_off_by_the_sum_over_all_classes_alone(gpu, dtype, rows, C, k, t_dtype, T, tail):
    """What the row is made of, the list's terms and logarithms of sums, is in 64 bits but for the sum of fp32 terms that the workers
    make: of the classes outside the list (of all of them without t_lse), taken to the largest of all by one more exponential.  A
    relative error d of that sum changes the row by d |(mass + rest) p_rest - rest|.  Additions per thread: at most one per word of four, the
    tree's and a dozen rescalings, below 60 + C / 4096 (rows this long are shared by CTAs).  Beside that the row's own rounding."""
    g = rng(C + k + int(10 * T) + tail)
    for near in (0.03, 1.0):
        x = student.stored(logits(g, rows, C), dtype)[1]
        t = (x + near * g.standard_normal(x.shape)).astype(np.float32)
        u, i, _ = student.top_logits(t, k)
        raw, held = student.stored(u, t_dtype)
        l = student.lse(t.astype(np.float64) / T).astype(np.float32) if tail else None
        row = run_distill(gpu, x, raw, i, l, dtype, T=T, mode="none")[1]
        want, _, part = student.distill(x, i, held, l, None, T)
        down = np.zeros(rows)
        if tail:
            outside = x.astype(np.float64)
            np.put_along_axis(outside, i.astype(np.int64), -np.inf, 1)
            down = (x.max(1) - outside.max(1)) / T
        every = part["mass"] + part["rest"]
        weighs = np.abs(every * part["p_rest"] - part["rest"])
        d = sum_error(C, 60 + C / 4096) + EPS * (4 + 3 * down)
        tol = d * weighs + 2 * EPS * np.abs(want) + 1e-12
        assert (np.abs(row - want) <= tol).all(), (np.abs(row - want) / tol).max()


def test_whole_list(gpu):
    """A list of all classes: the divergence of two softmaxes."""
    g = rng(3)
    x = logits(g, 5, 64)
    raw, held, i, l = teacher_lists(g, x, 64, True, 1.0)
    check_distill(gpu, x, raw, held, i, l, "f32")
    check_distill(gpu, x, raw, held, i, None, "f32")


def test_gradient_against_differences_of_the_loss(gpu):
    """The directional derivative along d, |d| <= 1: truncation h^2 / 6 times a third cumulant of at most 8, and twice the
    loss's own error over 2 h."""
    g = rng(9)
    C, h = 3001, 0.02
    x = logits(g, 4, C)
    raw, held, i, l = teacher_lists(g, x, 20, True, 1.0)
    d = g.uniform(-1, 1, x.shape).astype(np.float32)
    hi, lo = (x + np.float32(h) * d).astype(np.float32), (x - np.float32(h) * d).astype(np.float32)
    grad = run_distill(gpu, x, raw, i, l, "f32", loss_div=1.0)[2].astype(np.float64)
    f = [run_distill(gpu, y, raw, i, l, "f32", loss_div=1.0, mode="none")[1].astype(np.float64) for y in (hi, lo)]
    step = (hi.astype(np.float64) - lo)  # what was really moved
    for r in range(4):
        assert abs((f[0][r] - f[1][r]) - (grad[r] * step[r]).sum()) <= 2 * h * (8 * h * h / 6) + 2 * (2 * sum_error(C, 80) + EPS * 40)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("C", [6, 700, 9001, 140001, 800003])
def test_gradient_of_a_student_that_knows_nothing_but_the_list(gpu, dtype, C):
    """Everything outside the list is -infinity and the teacher has mass there: the gradient is that of the loss returned, and sums to
    zero.  Differences: truncation and the loss's error as above (the list is summed in 64 bits: the row's rounding alone); the
    gradient's own error, p and q of which are off by EPS (4 + 3 |arg|), |arg| <= 20, and its rounding."""
    g = rng(C)
    k, rows = 4, 3
    i = np.stack([g.permutation(C)[:k] for _ in range(rows)]).astype(np.uint64)
    u = g.standard_normal((rows, k)).astype(np.float32)
    l = (student.lse(u.astype(np.float64)) + np.array([0.7, 0.1, 3.0])).astype(np.float32)  # masses of 0.5, 0.9, 0.05
    at = i.astype(np.int64)
    x = np.full((rows, C), -np.inf, np.float32)
    np.put_along_axis(x, at, g.standard_normal((rows, k)).astype(np.float32) * 2, 1)
    d = np.zeros_like(x)
    np.put_along_axis(d, at, g.uniform(-0.03, 0.03, (rows, k)).astype(np.float32), 1)
    hi, lo = (student.stored(y, dtype)[1] for y in (x + d, x - d))
    grad = run_distill(gpu, x, u, i, l, dtype, loss_div=1.0)[2].astype(np.float64)
    f = [run_distill(gpu, y, u, i, l, dtype, loss_div=1.0, mode="none")[1].astype(np.float64) for y in (hi, lo)]
    own = EPS * (4 + 3 * 20) + HALF_STEP[dtype]
    for r in range(rows):
        mid, step = (np.take_along_axis(a.astype(np.float64), at, 1)[r] for a in (student.stored(x, dtype)[1], hi))
        step = step - np.take_along_axis(lo.astype(np.float64), at, 1)[r]
        centre = np.abs(np.take_along_axis(hi, at, 1)[r] + np.take_along_axis(lo, at, 1)[r] - 2 * mid).max() / 2  # what rounding moved the middle by
        h, size = np.abs(step).max() / 2, np.abs(grad[r]).sum()
        tol = 2 * h * (8 * h * h / 6 + centre) + 2 * (EPS * 40) + 2 * h * own * (size + 2)
        assert abs((f[0][r] - f[1][r]) - (grad[r, at[r]] * step).sum()) <= tol
        assert abs(grad[r].sum()) <= own * (size + 2)
        assert np.count_nonzero(grad[r]) <= k


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("C", [20, 900, 30001, 140001])
def test_bad_values_stay_in_their_row(gpu, dtype, C, tail):
    """A NaN or +infinity among a row's logits, a NaN in its list: no finite loss for that row, and the others' as if it were not there."""
    g = rng(C + tail)
    x = logits(g, 9, C)
    raw, held, i, l = teacher_lists(g, x, 6, tail, 1.0)
    outside = int(np.setdiff1d(np.arange(C), i[:5].astype(np.int64))[-1])
    x[0, outside], x[1, outside] = np.nan, np.inf
    x[2, int(i[2, 1])], x[3, int(i[3, 5])] = np.nan, np.inf
    raw[4, 2] = held[4, 2] = np.nan
    bad = [0, 1, 2, 3, 4]
    if tail:
        l[5] = np.nan
        i[6, :] = student.NO_TOKEN    # all of the teacher's mass is compared with the student's
        x[6, C // 2] = np.nan
        bad += [5, 6]
    good = [r for r in range(9) if r not in bad]
    weight = np.ones(9, np.float32)
    loss, row, grad, _ = run_distill(gpu, x, raw, i, l, dtype, weight=weight, mode="write")
    assert not np.isfinite(row[bad]).any() and not np.isfinite(loss), row
    _, one, alone, _ = run_distill(gpu, x[good], raw[good], i[good], None if l is None else l[good], dtype, weight=weight[good], mode="write")
    assert np.isfinite(one).all() and np.isfinite(alone).all()
    want_row, want, part = student.distill(student.stored(x[good], dtype)[1], i[good], held[good], None if l is None else l[good], None, 1.0, 3.0)
    np.testing.assert_allclose(row[good], want_row, rtol=1e-5, atol=1e-5)
    d = HALF_STEP[dtype] * 1.01 * np.abs(want) + 1e-5
    assert (np.abs(grad[good] - want) <= d).all()


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("C", [12, 900, 30001, 140001, 800003])
def test_a_student_whose_mask_leaves_nothing(gpu, dtype, C, tail):
    """Nothing but -infinity: p = 0 everywhere, the row infinite where the list has mass, its gradient -q; an empty list asks nothing."""
    g = rng(C + tail)
    x = logits(g, 3, C)
    raw, held, i, l = teacher_lists(g, x, 6, tail, 2.0)
    x[:2] = -np.inf
    i[1, :] = student.NO_TOKEN
    loss, row, grad, _ = run_distill(gpu, x, raw, i, l, dtype, T=2.0, mode="write")
    assert row[0] == np.inf and row[1] == 0 and np.isfinite(row[2]) and loss == np.inf
    u = held[0].astype(np.float64) / 2
    q = np.exp(u - (float(l[0]) if tail else student.lse(u[None])[0]))
    want = np.zeros(C)
    want[i[0].astype(np.int64)] = -q / (2.0 * 3.0)
    # six roundings in fp32 at most (q, the list's sum, its inverse, their product, the scale, the product with it), one to the type
    assert (np.abs(grad[0] - want) <= np.abs(want) * (HALF_STEP[dtype] * 1.01 + 6.1 * EPS)).all()
    assert (grad[1] == 0).all()
    _, alone, dx, _ = run_distill(gpu, x[2:], raw[2:], i[2:], None if l is None else l[2:], dtype, T=2.0, mode="write")
    assert np.isfinite(alone).all() and np.isfinite(dx).all() and np.isfinite(grad[2]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("C", [20, 3001, 140001])
def test_a_listed_class_without_mass_is_no_part_of_the_rest(gpu, dtype, C):
    """p_r is the student's mass outside the list, whatever the teacher gives the list's classes."""
    g = rng(C)
    x = logits(g, 3, C)
    raw, held, i, l = teacher_lists(g, x, 6, True, 1.0)
    raw[:, 3:] = held[:, 3:] = -np.inf
    check_distill(gpu, x, raw, held, i, l, dtype)
    short = i.copy()
    short[:, 3:] = student.NO_TOKEN
    at = i[:, 3:].astype(np.int64)
    x2 = x.copy()
    np.put_along_axis(x2, at, -np.inf, 1)      # the rest's comparison does not see them: without them the total alone changes
    listed, _, part = student.distill(student.stored(x, dtype)[1], i, held, l)
    bare, _, part2 = student.distill(student.stored(x2, dtype)[1], short, held, l)
    p = np.take_along_axis(part["p"], at, 1).sum(1)
    np.testing.assert_allclose(listed - bare, -(part["mass"] + part["rest"]) * np.log1p(-p), rtol=1e-9, atol=1e-12)


def test_no_rows(gpu):
    loss, one = gpu.from_numpy(np.full(1, 5.0, np.float32)), gpu.from_numpy(np.zeros(8, np.float32))
    idx = gpu.from_numpy(np.zeros(8, np.uint64))
    gpu.dispatch(opspec.distill_ce(one, idx, one, 0, 8, 2, loss, one))
    assert gpu.to_numpy(loss)[0] == 0.0
    gpu.dispatch(opspec.top_logits(one, 0, 8, 2, one, idx))
    gpu.dispatch(opspec.verify_drafts(one, idx, one, 0, 2, 4, idx, idx))
    assert (gpu.to_numpy(idx) == 0).all() and (gpu.to_numpy(one) == 0).all()


# ------------------------------------------------------------------------------------------------ verification
def run_verify(gpu, target, draft, tokens, lengths, u, dtype, ld_t=None, ld_d=None, offset=0):
    B, n1, C = target.shape
    n = n1 - 1
    be = GpuBackend(gpu)
    nan = np.uint16(0x7FC0) if dtype == "bf16" else np.float32(np.nan)
    raw_t, held_t = student.stored(target, dtype)
    ld_t, ld_d = ld_t or C, ld_d or C
    T = up(be, rows_with_ld(raw_t.reshape(-1, C), ld_t, nan), offset=offset)
    D, held_d = None, None
    if draft is not None:
        raw_d, held_d = student.stored(draft, dtype)
        D = up(be, rows_with_ld(raw_d.reshape(-1, C), ld_d, nan), offset=offset + 1)
    K, U = up(be, tokens, np.uint64), up(be, u, np.float32)
    N = up(be, lengths, np.uint64) if lengths is not None else None
    out, acc = up(be, np.full(B * n1, 77, np.uint64)), up(be, np.full(B, 77, np.uint64))
    gpu.dispatch(opspec.verify_drafts(T, K, U, B, n, C, out, acc, draft=D, lengths=N, ld_target=ld_t if ld_t != C else 0, ld_draft=ld_d if ld_d != C else 0))
    o, a = gpu.to_numpy(out, (B, n1)), gpu.to_numpy(acc)
    be.down(acc)
    return o, a, held_t, held_d


def check_verify(gpu, target, draft, tokens, lengths, u, dtype, **kw):
    u = np.asarray(u, np.float32)
    o, a, held_t, held_d = run_verify(gpu, target, draft, tokens, lengths, u, dtype, **kw)
    wo, wa = student.verify(held_t, held_d, tokens, lengths, u)
    np.testing.assert_array_equal(a, wa)
    np.testing.assert_array_equal(o, wo)


def softmax(x):
    e = np.exp(x - x.max(-1, keepdims=True))
    return (e / e.sum(-1, keepdims=True)).astype(np.float32)


def drafted(g, B, n, C, close=0.7):
    q = softmax(logits(g, max(1, B * n), C).reshape(-1, C)[: B * n].reshape(B, n, C).astype(np.float64))
    extra = softmax(logits(g, B, C).astype(np.float64))[:, None]
    p = np.concatenate([softmax(np.log(q.astype(np.float64) + 1e-9) + close * g.standard_normal((B, n, C))), extra], 1)
    tokens = np.argmax(q / g.exponential(1.0, q.shape), 2).reshape(B, n).astype(np.uint64)
    return p.astype(np.float32), q.astype(np.float32), tokens, g.random((B, n + 1)).astype(np.float32)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("C", [1, 2, 9, 33, 255, 256, 257, 1003, 4099, 20001])
def test_verification(gpu, dtype, C):
    g = rng(C)
    for B, n in ((1, 1), (1, 4), (7, 3), (40 if C < 5000 else 5, 2), (3, 0), (2, 40 if C < 2000 else 9)):
        p, q, tokens, u = drafted(g, B, n, C, close=0.3)
        lengths = g.integers(0, n + 3, B).astype(np.uint64) if g.random() < 0.5 else None
        kw = dict(offset=int(g.integers(0, 8)), ld_t=C + int(g.integers(0, 3)), ld_d=C + int(g.integers(0, 2)))
        check_verify(gpu, p, q, tokens, lengths, u, dtype, **kw)
        check_verify(gpu, p, None, tokens, lengths, u, dtype, **kw)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,n,C", [(1, 4, 131072), (2, 2, 250007), (160, 2, 3001), (80, 3, 9000), (400, 1, 300)])
def test_verification_of_long_rows_and_many_sequences(gpu, dtype, B, n, C):
    g = rng(B + C)
    p, q, tokens, u = drafted(g, B, n, C)
    check_verify(gpu, p, q, tokens, None, u, dtype)


@pytest.mark.parametrize("C", [6, 900, 40000])
def test_verification_at_the_borders(gpu, C):
    g = rng(C)
    one = np.zeros((1, 2, C), np.float32)
    one[0, 0, :4] = [0.5, 0.25, 0.125, 0.125]
    one[0, 1, C - 1] = 1.0
    q = np.zeros((1, 1, C), np.float32)
    q[0, 0, :4] = [0.25, 0.5, 0.125, 0.125]
    tok = lambda t: np.array([[t]], np.uint64)
    cases = []
    for t in (0, 1, 2, 4, C, C + 9, int(student.NO_TOKEN)):
        for a in (0.0, 0.25, 0.5, 0.4999999, 1 - 2.0 ** -24):
            for b in (0.0, 0.5, 0.25, 1 - 2.0 ** -24):
                cases.append((tok(t), np.array([[a, b]])))
    B = len(cases)
    tokens, u = np.concatenate([c[0] for c in cases]), np.concatenate([c[1] for c in cases])
    P, Q = np.repeat(one, B, 0), np.repeat(q, B, 0)
    check_verify(gpu, P, Q, tokens, None, u, "f32")          # u q = p exactly: the draft falls
    check_verify(gpu, P, None, tokens, None, u, "f32")
    check_verify(gpu, P, P[:, :1].copy(), tokens, None, u, "f32")   # nothing beyond the draft: the target's row
    check_verify(gpu, np.zeros_like(P), Q, tokens, None, u, "bf16")  # no mass at all
    bad = P.copy()
    bad[:, :, 1] = np.nan
    bad[:, 0, 3] = -1.0
    check_verify(gpu, bad, Q, tokens, None, u, "f32")
    # random numbers outside [0, 1) end at the last class that has mass
    o, a, _, _ = run_verify(gpu, P, Q, tokens, None, np.full((B, 2), 2.0, np.float32), "f32")
    assert (a == 0).all() and (o[:, 1] == student.NO_TOKEN).all() and np.isin(o[:, 0], [0, 1, 2, 3]).all()
    o, a, _, _ = run_verify(gpu, P, Q, tokens, None, np.full((B, 2), np.nan, np.float32), "f32")
    assert (a == 0).all() and np.isin(o[:, 0], [0, 1, 2, 3]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("C", [33, 1003, 4096, 40001])
def test_verification_with_nans_among_the_drafts_probabilities(gpu, dtype, C):
    """At the drafted token: it falls, however probable to the target.  Elsewhere: the class is never drawn behind a draft that fell."""
    g = rng(C)
    B, n = 24, 2
    p, q, tokens, u = drafted(g, B, n, C, close=0.3)
    u[:, 0] = 0.0                                              # stands wherever the target gives it anything
    b = np.arange(B)
    q[b[::2], 0, tokens[::2, 0].astype(np.int64)] = np.nan     # every second sequence's first draft falls
    q[b[:, None], 0, g.integers(0, C, (B, 5))] = np.nan
    q[:, 1, :: 3] = np.nan
    q[:4] = np.nan                                             # nothing beyond it: the target's own row
    check_verify(gpu, p, q, tokens, None, u, dtype)
    o, a, _, _ = run_verify(gpu, p, q, tokens, None, u, dtype)
    assert (a[::2] == 0).all() and (a[:4] == 0).all() and (a > 0).any()
    for r in range(4, B):
        if a[r] < n:
            assert not np.isnan(q[r, int(a[r]), int(o[r, int(a[r])])])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_past_32_bits_of_offset(gpu, dtype):
    """Three rows 2^31 elements apart: what lies between them is not touched, and need not be there for the test to be quick."""
    g = rng(12)
    C, k, ld = 1003, 7, 1 << 31
    x = logits(g, 3, C)
    raw, held = student.stored(x, dtype)
    big = gpu.mem_alloc(abi.BF16 if dtype == "bf16" else abi.SINGLE, 2 * ld + C)
    grad = gpu.mem_alloc(abi.BF16 if dtype == "bf16" else abi.SINGLE, 2 * ld + C)
    try:
        for r in range(3):
            gpu.mem_transfer_htod(raw[r].copy(), big.view(r * ld, C))
        V, I, L = gpu.from_numpy(np.zeros((3, k), raw.dtype)), gpu.from_numpy(np.zeros((3, k), np.uint64)), gpu.from_numpy(np.zeros(3, np.float32))
        loss, row = gpu.from_numpy(np.zeros(1, np.float32)), gpu.from_numpy(np.zeros(3, np.float32))
        gpu.dispatch(opspec.top_logits(big, 3, C, k, V, I, lse=L, ld=ld))
        v, i, l = student.top_logits(held, k)
        np.testing.assert_array_equal(gpu.to_numpy(I, (3, k)), i)
        U = gpu.from_numpy((v + 0.5).astype(np.float32))
        gpu.dispatch(opspec.distill_ce(big, I, U, 3, C, k, loss, row, grad=grad, t_lse=L, loss_div=1.0, accumulate=False, ld=ld))
        want, dx, _ = student.distill(held, i, (v + 0.5).astype(np.float32), gpu.to_numpy(L))
        np.testing.assert_allclose(gpu.to_numpy(row), want, rtol=1e-4, atol=1e-5)
        for r in range(3):
            got = gpu.to_numpy(grad.view(r * ld, C))
            got = student.bf16_values(got) if dtype == "bf16" else got
            np.testing.assert_allclose(got, dx[r], atol=1e-5, rtol=2 * HALF_STEP[dtype])
        p = softmax(x.astype(np.float64))
        raw_p, held_p = student.stored(p, dtype)
        for r in range(3):
            gpu.mem_transfer_htod(raw_p[r].copy(), big.view(r * ld, C))
        tokens, u = np.array([[3, 5]], np.uint64), np.array([[0.0, 0.999, 0.37]], np.float32)
        out, acc = gpu.from_numpy(np.zeros(3, np.uint64)), gpu.from_numpy(np.zeros(1, np.uint64))
        gpu.dispatch(opspec.verify_drafts(big, gpu.from_numpy(tokens), gpu.from_numpy(u), 1, 2, C, out, acc, ld_target=ld))
        wo, wa = student.verify(held_p[None], None, tokens, None, u)
        np.testing.assert_array_equal(gpu.to_numpy(out, (1, 3)), wo)
    finally:
        gpu.sync()
        gpu.mem_free(big)
        gpu.mem_free(grad)


def test_many_short_rows(gpu):
    """More rows than one pass of the kernel that adds their losses up, and than a grid of verification has clusters."""
    g = rng(21)
    some, C, k, rows = 997, 37, 4, 120011
    of = np.arange(rows) % some
    x = logits(g, some, C)
    raw, held, i, l = teacher_lists(g, x, k, True, 1.0)
    weight = (g.random(some) < 0.8).astype(np.float32)
    loss, row, grad, _ = run_distill(gpu, x[of], raw[of], i[of], l[of], "f32", weight=weight[of], loss_div=float(rows))
    want_row, want, _ = student.distill(x, i, held, l, weight, 1.0, float(rows))
    # Rows of 37 start 0, 4, 8 or 12 bytes behind a 16-byte boundary, in turn, which groups their sums differently: every fourth turn of
    # the 997 a row stands as it did before, and gives the same bits wherever it is in the grid.
    again = np.arange(rows) % (4 * some)
    np.testing.assert_array_equal(row, row[:4 * some][again])
    np.testing.assert_array_equal(grad, grad[:4 * some][again])
    np.testing.assert_allclose(row[:some], want_row, rtol=1e-5, atol=1e-5)
    np.testing.assert_allclose(grad[:some] * rows, want * rows, atol=1e-5)
    assert abs(loss - row.astype(np.float64).sum() / rows) <= 2 * EPS * abs(loss)
    v, j, lse, _ = run_top(gpu, x[of], k, "f32")
    wv, wj, wl = student.top_logits(x, k)
    np.testing.assert_array_equal(j, wj[of])
    np.testing.assert_array_equal(v, wv.astype(np.float32)[of])
    np.testing.assert_allclose(lse, wl[of], rtol=1e-5)
    B, C = (1 << 20) + 1009, 3
    of = np.arange(B) % some
    p, q, tokens, u = drafted(g, some, 1, C, close=1.5)
    o, a, held_p, held_q = run_verify(gpu, p[of], q[of], tokens[of], None, u[of], "f32")
    wo, wa = student.verify(p, q, tokens, None, u)
    np.testing.assert_array_equal(a, wa[of])
    np.testing.assert_array_equal(o, wo[of])


# ------------------------------------------------------------------------------------------------ together
@pytest.fixture()
def fresh(gpu):
    d = CudaDevice(0)
    yield d
    d.deinit()


def test_first_calls_inside_a_capture(fresh):
    """None of the three needs work space: a stream's first call may be a captured one, and its replays read new inputs."""
    g = rng(4)
    rows, C, k = 37, 5003, 16
    x, x2 = logits(g, rows, C), logits(g, rows, C)
    X, V, I, L = fresh.from_numpy(x), fresh.from_numpy(np.zeros(rows * k, np.float32)), fresh.from_numpy(np.zeros(rows * k, np.uint64)), fresh.from_numpy(np.zeros(rows, np.float32))
    Z, G = fresh.from_numpy(logits(g, rows, C)), fresh.from_numpy(np.zeros((rows, C), np.float32))
    loss, row = fresh.from_numpy(np.zeros(1, np.float32)), fresh.from_numpy(np.zeros(rows, np.float32))
    p, q, tokens, u = drafted(g, 3, 2, C)
    P, Q, K, U = (fresh.from_numpy(a) for a in (p, q, tokens, u))
    out, acc = fresh.from_numpy(np.zeros(9, np.uint64)), fresh.from_numpy(np.zeros(3, np.uint64))
    fresh.capture.open()
    fresh.dispatch(opspec.top_logits(X, rows, C, k, V, I, lse=L))
    fresh.dispatch(opspec.distill_ce(Z, I, V, rows, C, k, loss, row, grad=G, t_lse=L, accumulate=False))
    fresh.dispatch(opspec.verify_drafts(P, K, U, 3, 2, C, out, acc, draft=Q))
    fresh.capture.save()
    seen = []
    for y in (x, x2, x):
        fresh.mem_transfer_htod(y, X)
        fresh.capture.run()
        v, i, l = student.top_logits(y, k)
        np.testing.assert_array_equal(fresh.to_numpy(I, (rows, k)), i)
        want, grad, _ = student.distill(fresh.to_numpy(Z, (rows, C)), i, v, fresh.to_numpy(L))
        np.testing.assert_allclose(fresh.to_numpy(row), want, rtol=1e-5, atol=1e-5)
        np.testing.assert_allclose(fresh.to_numpy(G, (rows, C)) * rows, grad, atol=1e-5)
        np.testing.assert_array_equal(fresh.to_numpy(out, (3, 3)), student.verify(p, q, tokens, None, u)[0])
        seen.append((fresh.to_numpy(loss), fresh.to_numpy(G), fresh.to_numpy(L)))
    for a, b in zip(seen[0], seen[2]):  # bit for bit the same
        np.testing.assert_array_equal(a, b)


FIRST_IN_A_PROCESS = """
import numpy as np
from tests import student
from tests.test_gpu_student_ops import logits, rng, drafted
from zigrad_b200 import opspec
from zigrad_b200.device import CudaDevice
d, g = CudaDevice(0), rng(8)
rows, C, k = 3, 400003, 40    # a cluster a row, more shared memory than a kernel has unasked
x, t = logits(g, rows, C), logits(g, rows, C)
X, Z, G = d.from_numpy(t), d.from_numpy(x), d.from_numpy(np.ones((rows, C), np.float32))
V, I, L = d.from_numpy(np.zeros(rows * k, np.float32)), d.from_numpy(np.zeros(rows * k, np.uint64)), d.from_numpy(np.zeros(rows, np.float32))
loss, row = d.from_numpy(np.zeros(1, np.float32)), d.from_numpy(np.zeros(rows, np.float32))
p, q, tokens, u = drafted(g, 2, 2, 50021)
P, Q, K, U = (d.from_numpy(a) for a in (p, q, tokens, u))
out, acc = d.from_numpy(np.zeros(6, np.uint64)), d.from_numpy(np.zeros(2, np.uint64))
d.capture.open()
d.dispatch(opspec.top_logits(X, rows, C, k, V, I, lse=L))
d.dispatch(opspec.distill_ce(Z, I, V, rows, C, k, loss, row, grad=G, t_lse=L, loss_div=1.0))
d.dispatch(opspec.verify_drafts(P, K, U, 2, 2, 50021, out, acc, draft=Q))
d.capture.save()
for n in (1, 2):
    d.capture.run()
    v, i, l = student.top_logits(t, k)
    np.testing.assert_array_equal(d.to_numpy(I, (rows, k)), i)
    want, grad, _ = student.distill(x, i, v, d.to_numpy(L))
    np.testing.assert_allclose(d.to_numpy(row), want, rtol=1e-5, atol=1e-5)
    np.testing.assert_allclose(d.to_numpy(G, (rows, C)), 1 + n * grad, atol=1e-5)
    np.testing.assert_array_equal(d.to_numpy(out, (2, 3)), student.verify(p, q, tokens, None, u)[0])
print("captured")
"""


def test_first_calls_of_a_process_inside_a_capture(gpu):
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", FIRST_IN_A_PROCESS], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "captured" in done.stdout, done.stderr[-2000:]


def test_calls_on_two_streams_at_once(gpu):
    g = rng(6)
    rows, C, k = 300, 20000, 32
    jobs = []
    for s in range(2):
        x = logits(g, rows, C)
        raw, held, i, l = teacher_lists(g, x, k, True, 1.0)
        ups = [gpu.from_numpy(a) for a in (x, raw, i, l, np.zeros((rows, C), np.float32), np.zeros(1, np.float32), np.zeros(rows, np.float32),
                                           np.zeros(rows * k, np.float32), np.zeros(rows * k, np.uint64), np.zeros(rows, np.float32))]
        jobs.append((x, held, i, l, ups))

    def issue(job):
        X, U, I, L, G, loss, row, V, J, N = job[4]
        gpu.dispatch(opspec.distill_ce(X, I, U, rows, C, k, loss, row, grad=G, t_lse=L, accumulate=False))
        gpu.dispatch(opspec.top_logits(X, rows, C, k, V, J, lse=N))

    for _ in range(10):
        with gpu.branch(0):
            issue(jobs[0])
        issue(jobs[1])
        gpu.join()
    for x, held, i, l, (X, U, I, L, G, loss, row, V, J, N) in jobs:
        want, grad, _ = student.distill(x, i, held, l)
        np.testing.assert_allclose(gpu.to_numpy(row), want, rtol=1e-5, atol=1e-5)
        np.testing.assert_allclose(gpu.to_numpy(G, (rows, C)) * rows, grad, atol=1e-5)
        np.testing.assert_array_equal(gpu.to_numpy(J, (rows, k)), student.top_logits(x, k)[1])
        for s in (X, U, I, L, G, loss, row, V, J, N):
            gpu.mem_cache_free(s)


@pytest.mark.parametrize("C", [50, 2003])
def test_a_student_learns_from_a_teacher_and_drafts_for_it(gpu, C):
    """The ops as they are used together: the teacher's lists, SGD steps on a student's logits, softmax, drafts verified."""
    g = rng(C)
    B, n, k = 6, 3, 16
    rows = B * (n + 1)
    teacher, x = logits(g, rows, C), np.zeros((rows, C), np.float32)
    be = GpuBackend(gpu)
    Tl, X, G = be.up(teacher), be.up(x), be.up(np.zeros((rows, C)))
    V, I, L = be.up(np.zeros(rows * k)), be.up(np.zeros(rows * k, np.uint64), np.uint64), be.up(np.zeros(rows))
    loss, row = be.up(np.zeros(1)), be.up(np.zeros(rows))
    gpu.dispatch(opspec.top_logits(Tl, rows, C, k, V, I, lse=L))
    v, i, l = student.top_logits(teacher, k)
    held_l = gpu.to_numpy(L)
    mine, lr = x.astype(np.float64), 2.0
    for _ in range(5):
        gpu.dispatch(opspec.distill_ce(X, I, V, rows, C, k, loss, row, grad=G, t_lse=L, loss_div=1.0, accumulate=False))
        gpu.dispatch(opspec.sgd(X, G, [(0, rows * C)], lr))
        want, grad, _ = student.distill(mine, i, v, held_l)
        np.testing.assert_allclose(gpu.to_numpy(row), want, rtol=1e-5, atol=2e-5)
        mine = mine - lr * grad
    np.testing.assert_allclose(gpu.to_numpy(X, (rows, C)), mine, atol=2e-5)
    q = softmax(gpu.to_numpy(X, (B, n + 1, C)).astype(np.float64))[:, :n]
    p = softmax(teacher.astype(np.float64)).reshape(B, n + 1, C)
    tokens = np.argmax(q / g.exponential(1.0, q.shape), 2).astype(np.uint64)
    check_verify(gpu, p, q, tokens, None, g.random((B, n + 1)), "f32")
    be.down(row)


@pytest.mark.parametrize("C", [10, 37])
def test_a_network_learns_from_labels_and_a_teacher(gpu, C):
    """Softmax cross-entropy against hard labels and, added to its gradient, the divergence from the teacher's list, through the
    network's backward pass and an SGD step.  Each of the step's products is off by 2^-20 of its terms' magnitudes at most, six of them
    follow on one another, and a sum cancels to no less than an eighth of its terms' magnitude at the matrix's largest entry: 1e-4."""
    from zigrad_b200.mlp import MlpTrainer, kaiming_uniform
    g = rng(C)
    dims, B, k, T, lr = [24, 48, C], 32, 4, 2.0, 0.5
    ws, bs = kaiming_uniform(dims, 3)
    bs = [g.uniform(-0.1, 0.1, np.shape(b)).astype(np.float32) for b in bs]
    tr = MlpTrainer(gpu, dims, B, ws, bs, lr=lr, index_labels=True, pad_logits=False)
    X, y = g.standard_normal((B, dims[0])).astype(np.float32), g.integers(0, C, B)
    teacher = logits(g, B, C)
    be = GpuBackend(gpu)
    Xd, Y, Tl = be.up(X), be.up(y.astype(np.uint64), np.uint64), be.up(teacher)
    V, I, L = be.up(np.zeros(B * k)), be.up(np.zeros(B * k, np.uint64), np.uint64), be.up(np.zeros(B))
    loss, row = be.up(np.zeros(1)), be.up(np.zeros(B))
    gpu.dispatch(opspec.top_logits(Tl, B, C, k, V, I, lse=L, temperature=T))
    v, i, _ = student.top_logits(teacher, k)
    held_l = gpu.to_numpy(L)
    W, b = [np.asarray(w, np.float64).reshape(dims[n + 1], dims[n]) for n, w in enumerate(ws)], [np.asarray(x, np.float64).ravel() for x in bs]
    close = lambda got, want: np.abs(got - want).max() <= 1e-4 * np.abs(want).max()
    for _ in range(3):
        tr.forward(Xd)
        gpu.dispatch(opspec.softmax_ce(tr.act[-1], Y, B, C, tr.loss, tr.dact[-1], float(B), accumulate=False, ld=tr.ld_out))
        gpu.dispatch(opspec.distill_ce(tr.act[-1], I, V, B, C, k, loss, row, grad=tr.dact[-1], t_lse=L, temperature=T, loss_div=B / T ** 2, ld=tr.ld_out))
        tr.backward(Xd, last_bias_done=False)
        dW, db = tr.get_grads()
        tr.update()
        pre = X @ W[0].T + b[0]
        h = np.maximum(pre, 0)
        z = h @ W[1].T + b[1]
        p = np.exp(z - student.lse(z)[:, None])
        hard = -np.log(p[np.arange(B), y]).mean()
        want_row, soft, _ = student.distill(z, i, v, held_l, None, T, B / T ** 2)
        dz = (p - np.eye(C)[y]) / B + soft
        dh = (dz @ W[1]) * (pre > 0)
        want = [(dh.T @ X, dh.sum(0)), (dz.T @ h, dz.sum(0))]
        assert abs(tr.read_loss() - hard) <= 1e-4 * abs(hard) and close(gpu.to_numpy(row), want_row)
        assert abs(gpu.to_numpy(loss)[0] - want_row.sum() * T ** 2 / B) <= 1e-4 * want_row.sum() * T ** 2 / B
        assert close(tr.act_numpy(1, grad=True), dz)
        for n in range(2):
            assert close(dW[n], want[n][0]) and close(db[n], want[n][1])
            W[n], b[n] = W[n] - lr * want[n][0], b[n] - lr * want[n][1]
        got_W, got_b = tr.get_params()
        assert all(close(got_W[n], W[n]) and close(got_b[n], b[n]) for n in range(2))
    be.down(row)
    tr.free()
