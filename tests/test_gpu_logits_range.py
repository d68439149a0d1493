"""The operators over rows of logits where numbers go far: large logits, small temperatures, rows whose
beginning lies far below the rest, infinities, for every type.  References and tolerances are those of
tests/_logits.py and tests/test_gpu_logits.py, in which the errors of a softmax are counted."""
from unittest import mock

import numpy as np
import pytest

from tests import _logits as L
from tests import test_gpu_logits as G

pytestmark = pytest.mark.gpu

DTYPES = ["f32", "f16", "bf16"]
INF, NAN = float("inf"), float("nan")
# one length for each way that a row of a distillation is read: few vectors, a workgroup's registers, streamed
LENGTHS = [40, 4000, 20001, 70001, 140000]


def _far_rows(far, temperature, n, rng):
    """Rows whose maximum is `far` temperatures or so from zero, on either side."""
    m, near = far * temperature, lambda: temperature * rng.normal(0, 2, n)
    one = near()
    one[rng.integers(n)] = m
    low = np.full(n, -m)
    low[rng.integers(0, n, 3)] = temperature * rng.normal(0, 1, 3)
    return np.array([np.full(n, -m), np.full(n, m), near() - m, near() + m, one, low,
                     m * rng.random(n) * rng.choice([-1.0, 1.0], n)])


_ref_distill = L.ref_distill


def _ref_with_infinities(z, t, idx, temperature, *rest):
    """The reference for rows that hold +inf as well: the sum is +inf, so q = 0 for a finite logit whatever it
    is.  exp(z / T) itself passes the largest 64-bit number from z / T = 710 on, and inf / inf is NaN."""
    z = z.astype(np.float64)
    beside = np.isposinf(z).any(axis=1, keepdims=True) & np.isfinite(z)
    return _ref_distill(np.where(beside, np.minimum(z, 0.0), z), t, idx, temperature, *rest)


def _distill(x, dtype, temperature, calls, rng, k=8, scale=None, listed=True):
    """Loss and gradient against the 64-bit reference; the teacher lists the maximum, or only others."""
    view, _ = G._put(x, dtype, pad=len(x[0]) % 3)
    best = np.nan_to_num(G._host(view), nan=-INF).argmax(1)
    rows, n = x.shape
    k = min(k, n)
    idx = np.array([rng.permutation(n)[:k] for _ in range(rows)], dtype=np.int32)
    if listed:
        idx = np.where((idx == best[:, None]).any(1)[:, None] | (np.arange(k) > 0), idx, best[:, None])
    else:
        idx = np.where(idx == best[:, None], -1, idx)
    t = temperature * rng.normal(0, 2, (rows, k))
    with mock.patch.object(L, "ref_distill", _ref_with_infinities):
        G._check_distill(view, t, idx.astype(np.int32), temperature, scale or temperature, calls=calls)


# |max| / T where the product with log2(e) / T leaves no bits for a softmax: its rounding is 2^-8 and more
FAR = [("f32", 2e5, 1.0), ("f32", 5e9, 1.0), ("f32", 1e10, 1.0), ("f32", 1e12, 1.0), ("f32", 1e20, 1.0),
       ("f32", 5e29, 1.0), ("f32", 3333e6, 1e-6), ("f32", 2e5, 1e-4), ("f32", 1e12, 1e6),
       ("bf16", 2e5, 1.0), ("bf16", 5e9, 1.0), ("bf16", 1e10, 0.5), ("bf16", 1e20, 1.0), ("bf16", 3333e6, 1e-6),
       ("f16", 2.4e5, 0.25), ("f16", 3333e6, 1e-6)]


@pytest.mark.parametrize("dtype,far,temperature", FAR)
def test_log_sum_exp_far_from_zero(gpu, dtype, far, temperature):
    rng = np.random.default_rng(1)
    for n in (1, 9, 300, 5000, 70001):
        view, _ = G._put(_far_rows(far, temperature, n, rng), dtype)
        G._check_top_k(view, min(n, 5), temperature=temperature)


@pytest.mark.parametrize("dtype,far,temperature", FAR)
@pytest.mark.parametrize("calls", [1, 2])
def test_distill_far_from_zero(gpu, dtype, far, temperature, calls):
    rng = np.random.default_rng(2)
    for n in LENGTHS:
        _distill(_far_rows(far, temperature, n, rng), dtype, temperature, calls, rng)


@pytest.mark.parametrize("far,temperature", [(100.0, 1.0), (1e3, 1.0), (1e4, 1.0), (8e4, 1.0), (8e4, 1e-4), (2e4, 50.0)])
@pytest.mark.parametrize("calls", [1, 2])
def test_distill_does_not_depend_on_a_common_shift(gpu, far, temperature, calls):
    """What the constant log2(e) / T is off by counts for the distances from the maximum alone, and a reference's
    rounding not at all."""
    rng = np.random.default_rng(3)
    for n in LENGTHS:
        _distill(_far_rows(far, temperature, n, rng), "f32", temperature, calls, rng)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("temperature", [1.0, 0.25])
def test_rows_that_begin_far_below_the_rest(gpu, dtype, temperature):
    """All that a thread sees first lies far below what comes later, or is masked.  A reference taken from it
    makes the sum of exponentials so large that the gradient's factor sinks below the normal numbers, and then
    beyond the largest number."""
    rng = np.random.default_rng(5)
    per = 4 if dtype == "f32" else 8  # elements of a vector
    for n in (1000 * per - 5, 4000 * per + 3, 8100 * per, 16300 * per + 1):
        late = np.arange(n) > 0.9 * n
        x = []
        for gap in (15.0, 25.0, 40.0, 60.0, 78.0, 82.0, 86.0, 88.3, 91.0):
            whole = temperature * rng.normal(0, 1.5, n)
            whole[late] += gap * temperature       # a whole part lies high
            one = temperature * rng.normal(0, 1.5, n)
            one[n - n // 50] = gap * temperature   # a single logit does
            x += [whole, one]
        masked = temperature * rng.normal(80, 1.5, n)
        masked[~late] = -INF
        x += [masked, np.where(late, rng.normal(21, 0.3, n), -INF)]
        x = np.array(x)
        _distill(x, dtype, temperature, 1, rng, scale=1 / 4096)
        _distill(x, dtype, temperature, 1, rng, scale=1 / 4096, listed=False)


def test_many_rows_that_begin_far_below_the_rest(gpu):
    """The same where workgroups of 8 waves take the rows."""
    rng = np.random.default_rng(6)
    rows, n = 520, 12000
    x = rng.normal(0, 1.5, (rows, n))
    x[np.arange(rows), n - 1 - np.arange(rows)] = rng.uniform(20, 95, rows)
    _distill(x, "f32", 1.0, 1, rng, scale=1 / 4096, listed=False)


@pytest.mark.parametrize("dtype,far,temperature", [
    ("f16", 100.0, 1.0), ("f16", 6e3, 1.0), ("f16", 6e4, 1.0), ("f16", 2e4, 1e-3), ("f16", 8e4, 1e-2),
    ("bf16", 100.0, 1.0), ("bf16", 6e3, 1.0), ("bf16", 5e4, 1.0), ("bf16", 8e4, 1.0), ("bf16", 8e4, 1e-4)])
@pytest.mark.parametrize("calls", [1, 2])
def test_16_bit_gradient_of_large_logits(gpu, dtype, far, temperature, calls):
    """A factor of the gradient that went into the exponent would be rounded at the size of max / T."""
    rng = np.random.default_rng(4)
    for n in LENGTHS:
        for listed in (True, False):
            _distill(_far_rows(far, temperature, n, rng), dtype, temperature, calls, rng, listed=listed)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("calls", [1, 2])
def test_infinite_logit_beside_large_ones(gpu, dtype, calls):
    """A logit of +inf leaves q = 0 for all others, however large, and NaN for itself."""
    rng = np.random.default_rng(7)
    for n in LENGTHS:
        x = rng.normal(0, 2, (4, n))
        x[0] += 120.0
        x[1] -= 400.0
        x[2, rng.random(n) < 0.5] = 500.0
        x[3, rng.random(n) < 0.5] = -INF
        x[np.arange(4), rng.integers(0, n, 4)] = INF
        for temperature in (1.0, 0.8):
            _distill(x, dtype, temperature, calls, rng)
            _distill(x, dtype, temperature, calls, rng, listed=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("calls", [1, 2])
def test_distill_patterns(gpu, dtype, calls):
    """Infinities, NaN, lowest values, equal ones, in every type of the gradient."""
    rng = np.random.default_rng(8)
    for n in LENGTHS:
        x = G._patterns(n, rng)
        x[np.abs(x) == 3.3e38] *= {"f32": 1.0, "f16": 65504 / 3.3e38, "bf16": 1.0}[dtype]
        _distill(x, dtype, 1.0, calls, rng)
        _distill(x, dtype, 0.5, calls, rng, listed=False)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("calls", [1, 2])
@pytest.mark.parametrize("n", [40, 5000, 140000])
def test_16_bit_masked_and_odd_values(gpu, dtype, calls, n):
    """-inf, the lowest value, NaN and +inf among 16-bit logits; listed tokens among them or not."""
    rng = np.random.default_rng(n)
    low = -65504.0 if dtype == "f16" else -3.3e38
    x = rng.normal(0, 1, (10, n))
    idx = np.array([rng.permutation(n)[:6] for _ in range(10)], dtype=np.int32)
    t = rng.normal(0, 2, (10, 6))
    x[0, rng.random(n) < 0.5] = -INF
    x[0, idx[0]] = 1.0
    x[1, idx[1, 0]] = -INF
    x[2] = -INF
    x[2, idx[2]] = rng.normal(0, 1, 6)
    x[3, rng.random(n) < 0.9] = low
    x[4] = low
    x[5, n // 2] = NAN
    x[6, n // 3] = INF
    x[7] = -INF
    idx[7] = -1
    x[8, 0] = NAN
    idx[8] = -1
    t[9, 1] = -INF
    view, _ = G._put(x, dtype)
    G._check_distill(view, t, idx, 1.0, 1.0, calls=calls, t_dtype=dtype)
    G._check_distill(view, t, idx, 0.25, 1.0, calls=calls, t_dtype=dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [9, 5000, 40003])
def test_sample_keeps_one_token_below_any_mass(gpu, dtype, n):
    """top_p at and below zero leaves the token that ranks first, with top_k and min_p or without."""
    rng = np.random.default_rng(n)
    view, _ = G._put(rng.normal(0, 0.5, (5, n)), dtype)
    top_p = np.array([0.0, -0.0, -1e-30, -1e30, -INF])
    for _ in range(2):
        G._check_sample(view, rng.random(5), top_p=top_p)
        G._check_sample(view, rng.random(5), top_p=top_p, top_k=np.full(5, 400), min_p=np.full(5, 1e-3))
