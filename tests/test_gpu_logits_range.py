"""The operators over rows of logits where numbers go far: large logits, small temperatures, rows whose
beginning lies far below the rest, infinities, for every type.  References and tolerances are those of
tests/_logits.py and tests/test_gpu_logits.py, in which the errors of a softmax are counted."""
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
