"""rmi_top_k, rmi_distill_loss / rmi_distill_grad and rmi_sample on the GPU against plain
implementations in 64 bits (tests/_logits.py)."""
import numpy as np
import pytest

from tests import _logits as L

pytestmark = pytest.mark.gpu

DTYPES = ["f32", "f16", "bf16"]
INF, NAN = float("inf"), float("nan")


def _torch(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def _put(values, dtype, pad=0, offset=0):
    """The values, rounded to `dtype`, as a view of rows `pad` elements apart that starts `offset`
    elements into its memory; and the memory, whose other places hold a pattern."""
    import torch
    v = torch.as_tensor(np.asarray(values, dtype=np.float32)).to(_torch(dtype))
    rows, n = v.shape
    memory = torch.full((offset + rows * (n + pad) + 16,), 77.0, dtype=v.dtype).cuda()
    view = memory[offset:offset + rows * (n + pad)].view(rows, n + pad)[:, :n]
    view.copy_(v)
    return view, memory


def _host(x):
    return x.detach().float().cpu().numpy()


def _patterns(n, rng):
    """Rows of one length that a selection can go wrong on."""
    x = [rng.normal(0, 2.5, n) for _ in range(3)]
    x.append(np.zeros(n))                                             # all equal
    x.append(np.where(rng.random(n) < 0.5, -0.0, 0.0))                # -0 and +0 are equal
    x.append(np.arange(n, dtype=np.float64))                          # ascending
    x.append(-np.arange(n, dtype=np.float64))                         # descending
    x.append(np.where(rng.random(n) < 0.9, 1.0, 2.0))                 # two values
    x.append(np.full(n, -INF))                                        # nothing
    few = np.full(n, -INF)
    few[rng.integers(0, n, 3)] = rng.normal(0, 1, 3)
    x.append(few)                                                     # a handful among -inf
    x.append(np.full(n, NAN))
    x.append(np.where(rng.random(n) < 0.3, NAN, rng.normal(0, 1, n)))
    x.append(np.where(rng.random(n) < 0.1, INF, rng.normal(0, 1, n)))
    low = np.full(n, -3.3e38)                                         # lowest values in masked places
    low[rng.integers(0, n, 2)] = 5.0
    x.append(low)
    x.append(np.full(n, -3.3e38))
    x.append(rng.normal(0, 1, n) * 1e-30)
    x.append(np.where(rng.random(n) < 0.01, 60.0, -60.0))
    return np.array(x)


# ---- top_k ----------------------------------------------------------------------------------------


def _check_top_k(view, k, temperature=1.0, with_lse=True):
    import torch

    from raft_amd import device
    rows, n = view.shape
    values = torch.full((rows, k), 55.0, dtype=view.dtype, device="cuda")
    indices = torch.full((rows, k), -7, dtype=torch.int32, device="cuda")
    lse = torch.full((rows,), 55.0, device="cuda") if with_lse else None
    device.top_k(view, values, indices, lse, temperature=temperature)
    x = _host(view)
    want, want_lse = L.ref_top_k(x, k, temperature)
    got = indices.cpu().numpy()
    bad = np.flatnonzero((got != want).any(axis=1))
    assert len(bad) == 0, (bad[:5], got[bad[0]][:8], want[bad[0]][:8])
    rest = np.take_along_axis(x, want.astype(np.int64), 1)
    np.testing.assert_array_equal(_host(values), rest)
    if with_lse:
        got = lse.cpu().numpy().astype(np.float64)
        finite = np.isfinite(want_lse)
        np.testing.assert_array_equal(np.isnan(got), np.isnan(want_lse))
        np.testing.assert_array_equal(got[~finite & ~np.isnan(want_lse)], want_lse[~finite & ~np.isnan(want_lse)])
        # the half step of the result's own rounding comes on top
        tol = L.lse_error(n) + 2.0 ** -23 * np.abs(want_lse[finite])
        assert (np.abs(got[finite] - want_lse[finite]) <= tol).all(), np.abs(got[finite] - want_lse[finite]).max()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 31, 64, 65, 255, 256, 257, 1000, 2047, 2049, 4100, 9001])
def test_top_k_lengths_and_patterns(gpu, dtype, n):
    rng = np.random.default_rng(n)
    view, _ = _put(_patterns(n, rng), dtype)
    for k in sorted({1, min(2, n), min(n, 7), min(n, 64), min(n, 300), min(n, 1024)}):
        _check_top_k(view, k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,n,k", [(1, 32000, 8), (5, 32000, 64), (3, 50001, 256), (2, 131072, 1024), (2, 131071, 50),
                                      (300, 1500, 33), (1, 300007, 100), (1, 1 << 20, 64)])
def test_top_k_long_rows(gpu, dtype, rows, n, k):
    rng = np.random.default_rng(n + k)
    view, _ = _put(rng.normal(0, 2, (rows, n)), dtype, pad=3)
    _check_top_k(view, k, temperature=0.7)


@pytest.mark.parametrize("dtype", DTYPES)
def test_top_k_long_patterns(gpu, dtype):
    rng = np.random.default_rng(5)
    view, _ = _put(_patterns(40003, rng), dtype)
    for k in (1, 50, 700):
        _check_top_k(view, k, temperature=2.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pad,offset", [(0, 1), (1, 0), (5, 3), (8, 8), (64, 7)])
def test_top_k_strides_and_offsets(gpu, dtype, pad, offset):
    rng = np.random.default_rng(pad * 10 + offset)
    for n in (100, 777, 5003):
        view, memory = _put(rng.normal(0, 2, (9, n)), dtype, pad, offset)
        before = memory.clone()
        _check_top_k(view, 17, with_lse=bool(pad % 2))
        assert (memory == before).all()


@pytest.mark.parametrize("dtype,quiet", [("f32", 0x7f800001), ("bf16", 0x7f81), ("f16", 0x7c01)])
@pytest.mark.parametrize("n", [12, 300, 5000, 70000])
def test_signalling_nans_rank_last_too(gpu, dtype, quiet, n):
    """NaN bit patterns that no arithmetic makes, among the largest elements of their vectors."""
    import torch
    rng = np.random.default_rng(n)
    view, _ = _put(rng.normal(0, 1, (4, n)), dtype)
    bits = view.view(torch.int32 if dtype == "f32" else torch.int16)
    places = torch.as_tensor(rng.random((4, n)) < 0.2).cuda()
    places[3, :] = True
    places[3, 5] = False
    bits[places] = quiet
    for k in (1, 10, min(n, 200)):
        _check_top_k(view, k)
    u = rng.random(4)
    _check_sample(view, u)
    _check_sample(view, u, top_k=np.full(4, 20), top_p=np.full(4, 0.9))


def test_top_k_offsets_past_32_bits(gpu):
    """Rows that start more than 2^32 elements into the matrix."""
    import torch
    ld = (1 << 31) + 11
    memory = torch.zeros(2 * ld + 5000, dtype=torch.bfloat16, device="cuda")
    view = memory.as_strided((3, 5000), (ld, 1))
    view.copy_(torch.randn(3, 5000, generator=torch.Generator().manual_seed(1)))
    _check_top_k(view, 20)


# ---- distillation -----------------------------------------------------------------------------------


def _teacher(rng, rows, n, k, short=True):
    """Values and different tokens of every row; some entries unused, one row without any."""
    idx = np.full((rows, k), -1, dtype=np.int32)
    for i in range(rows):
        m = min(k, n)
        idx[i, :m] = rng.permutation(n)[:m]
    t = rng.normal(0, 2, (rows, k))
    if short and rows > 2:
        idx[1] = -1
        idx[2, k // 2:] = n + 5
    return t, idx


def _check_distill(z, t, idx, temperature, scale, t_lse=None, row_grad=None, pad=0, calls=1, t_dtype="f32", in_place=False):
    import torch

    from raft_amd import device
    rows, n = z.shape
    k = idx.shape[1]
    tt = torch.as_tensor(np.asarray(t, dtype=np.float32)).to(_torch(t_dtype)).cuda()
    ti = torch.as_tensor(idx).cuda()
    tl = torch.as_tensor(np.asarray(t_lse, dtype=np.float32)).cuda() if t_lse is not None else None
    rg = torch.as_tensor(np.asarray(row_grad, dtype=np.float32)).cuda() if row_grad is not None else None
    loss = torch.full((rows,), 55.0, device="cuda")
    x = _host(z)
    if in_place:
        grad, memory, outside = z, None, None
    else:
        memory = torch.full((rows * (n + pad) + 16,), 77.0, dtype=z.dtype, device="cuda")
        grad = memory[:rows * (n + pad)].view(rows, n + pad)[:, :n]
    how = dict(temperature=temperature, scale=scale, teacher_lse=tl)
    if calls == 1:
        device.distill_loss(z, tt, ti, loss, grad=grad, row_grad=rg, **how)
    else:
        stats = torch.full((rows, 2), 55.0, device="cuda")
        device.distill_loss(z, tt, ti, loss, stats, **how)
        device.distill_grad(z, tt, ti, stats, grad, row_grad=rg, **how)
    want, dz, q, mass = L.ref_distill(x, _host(tt), idx, temperature, scale,
                                      None if tl is None else tl.cpu().numpy(), row_grad if rg is None else _host(rg))
    got, g = _host(loss).astype(np.float64), _host(grad).astype(np.float64)
    if memory is not None:
        kept = memory[:rows * (n + pad)].view(rows, n + pad)[:, n:]
        assert (kept == 77.0).all() and (memory[rows * (n + pad):] == 77.0).all()
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    with np.errstate(over="ignore"):  # the loss is an fp32 number: 3.3e38 / 0.25 is beyond its range
        want = np.where(np.isinf(want.astype(np.float32)), np.copysign(INF, want), want)
    inf = np.isinf(want)
    np.testing.assert_array_equal(got[inf], want[inf])
    ok = np.isfinite(want)
    e = L.lse_error(n)
    # log q is off by e (and by the rounding of z / T in 64 bits, nothing); the loss is rounded once
    tol = abs(scale) * mass[ok] * e + 2.0 ** -23 * np.abs(want[ok])
    assert (np.abs(got[ok] - want[ok]) <= tol).all(), (np.abs(got[ok] - want[ok]) / tol).max()
    up = np.ones(rows) if rg is None else np.abs(_host(rg).astype(np.float64))
    c = abs(scale) / temperature * up * mass
    with np.errstate(all="ignore"):
        a = np.where(np.isfinite(x), (np.nanmax(np.where(np.isfinite(x), x, -INF), axis=1, keepdims=True, initial=-INF) - x)
                     / temperature * 1.4427, 0.0)
        a = np.minimum(a, 200.0)
    # q is off by e, by the rounding of the two saved statistics (log s below 16: 16 half steps), by
    # its own argument's rounding and one step each of exp2 and the product; then one rounding
    eps = {"torch.float32": 2.0 ** -24, "torch.float16": 2.0 ** -11, "torch.bfloat16": 2.0 ** -8}[str(z.dtype)]
    tiny = 2.0 ** -25 if eps == 2.0 ** -11 else 2.0 ** -120
    q = np.where(mass[:, None] == 0, 0.0, q)  # without a teacher the gradient is 0, also where q is NaN
    with np.errstate(all="ignore"):
        bound = eps * np.abs(dz) * 1.001 + c[:, None] * q * (e + (2 * a + 24) * 2.0 ** -24) + tiny * np.maximum(1.0, c[:, None])
    np.testing.assert_array_equal(np.isnan(g), np.isnan(dz))
    fine = np.isfinite(dz)
    over = np.abs(g - dz)[fine] - bound[fine]
    assert (over <= 0).all(), (over.max(), np.argwhere((np.abs(g - dz) > bound) & fine)[:4])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,k", [(1, 1), (2, 2), (7, 3), (8, 8), (9, 1), (65, 64), (255, 300), (1000, 17), (2049, 64),
                                 (4100, 1024), (9001, 33), (16385, 20)])
@pytest.mark.parametrize("calls", [1, 2])
def test_distill_lengths(gpu, dtype, n, k, calls):
    rng = np.random.default_rng(n + k)
    z, _ = _put(rng.normal(0, 2.5, (5, n)), dtype, pad=n % 3)
    t, idx = _teacher(rng, 5, n, k)
    _check_distill(z, t, idx, 2.0, 4.0, pad=n % 5, calls=calls, t_dtype=dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,n,k", [(3, 32000, 64), (2, 50001, 100), (2, 131072, 64), (3, 131071, 7), (1, 300007, 50),
                                      (600, 1200, 20), (33, 32000, 8)])
@pytest.mark.parametrize("calls", [1, 2])
def test_distill_long_rows(gpu, dtype, rows, n, k, calls):
    rng = np.random.default_rng(n + k)
    z, _ = _put(rng.normal(0, 2, (rows, n)), dtype, pad=1)
    t, idx = _teacher(rng, rows, n, k)
    t_lse = np.log(np.exp(t).sum(1)) + 0.1
    _check_distill(z, t, idx, 1.0, 0.5, t_lse=t_lse, row_grad=rng.normal(0, 1, rows), pad=2, calls=calls)


@pytest.mark.parametrize("calls", [1, 2])
@pytest.mark.parametrize("n", [40, 5000, 140000])
def test_distill_masked_and_odd_values(gpu, calls, n):
    """-inf, the lowest value, NaN and +inf among the logits; listed tokens among them or not."""
    rng = np.random.default_rng(n)
    x = rng.normal(0, 1, (10, n))
    t, idx = _teacher(rng, 10, n, 6, short=False)
    x[0, rng.random(n) < 0.5] = -INF
    x[0, idx[0]] = 1.0                      # masked places that the teacher does not list
    x[1, idx[1, 0]] = -INF                  # a listed token that is masked: the loss is infinite
    x[2] = -INF
    x[2, idx[2]] = rng.normal(0, 1, 6)      # nothing but the listed ones
    x[3, rng.random(n) < 0.9] = -3.3e38
    x[4] = -3.3e38                          # every value the lowest
    x[5, n // 2] = NAN
    x[6, n // 3] = INF
    x[7] = -INF                             # no token at all, and no teacher either
    idx[7] = -1
    x[8, 0] = NAN                           # NaN in a row without a teacher
    idx[8] = -1
    t[9, 1] = -INF                          # a teacher's entry without probability
    z, _ = _put(x, "f32")
    _check_distill(z, t, idx, 1.0, 1.0, calls=calls)
    _check_distill(z, t, idx, 0.25, 1.0, calls=calls)


@pytest.mark.parametrize("dtype", DTYPES)
def test_distill_the_same_token_twice(gpu, dtype):
    rng = np.random.default_rng(3)
    z, _ = _put(rng.normal(0, 1, (4, 300)), dtype)
    t = rng.normal(0, 1, (4, 40))
    idx = rng.integers(0, 12, (4, 40)).astype(np.int32)
    idx[1] = 299
    _check_distill(z, t, idx, 1.5, 1.0, calls=1)
    _check_distill(z, t, idx, 1.5, 1.0, calls=2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [50, 3001, 32000, 140001])
@pytest.mark.parametrize("calls", [1, 2])
def test_distill_gradient_in_place(gpu, dtype, n, calls):
    rng = np.random.default_rng(n)
    z, memory = _put(rng.normal(0, 2, (6, n)), dtype, pad=3, offset=1)
    t, idx = _teacher(rng, 6, n, 12)
    _check_distill(z, t, idx, 1.0, 1.0, calls=calls, in_place=True)
    pads = memory[1:1 + 6 * (n + 3)].view(6, n + 3)[:, n:]
    assert (pads == 77.0).all() and memory[0] == 77.0


def test_distill_without_teacher_entries(gpu):
    """k = 0: no loss, no gradient."""
    import torch

    from raft_amd import device
    z = torch.randn(3, 100, device="cuda")
    loss, grad = torch.full((3,), 5.0, device="cuda"), torch.full((3, 100), 5.0, device="cuda")
    none = torch.empty(3, 0, device="cuda")
    device.distill_loss(z, none, none.int(), loss, grad=grad)
    assert (loss == 0).all() and (grad == 0).all()


def test_distill_gradient_by_differences(gpu):
    """The gradient against central differences of the loss.  With h = 1/16 the third derivative of
    log-sum-exp (below 0.2 for T = 1) leaves h^2 / 6 * 0.2 of the teacher's mass; the two losses are
    off by lse_error and a rounding each, divided by 2 h."""
    import torch

    from raft_amd import device
    rng = np.random.default_rng(9)
    n, k, h = 60, 8, 1 / 16
    base = rng.normal(0, 1, n).astype(np.float32)
    t, idx = _teacher(rng, 1, n, k)
    z = np.repeat(base[None], 2 * n, axis=0)
    z[np.arange(n), np.arange(n)] += h
    z[n + np.arange(n), np.arange(n)] -= h
    step = (z[np.arange(n), np.arange(n)].astype(np.float64) - z[n + np.arange(n), np.arange(n)])
    zt = torch.as_tensor(z).cuda()
    tt = torch.as_tensor(np.repeat(t, 2 * n, 0).astype(np.float32)).cuda()
    ti = torch.as_tensor(np.repeat(idx, 2 * n, 0)).cuda()
    loss = torch.empty(2 * n, device="cuda")
    device.distill_loss(zt, tt, ti, loss)
    got = loss.double().cpu().numpy()
    slope = (got[:n] - got[n:]) / step
    one = torch.as_tensor(base[None]).cuda()
    grad, l1 = torch.empty_like(one), torch.empty(1, device="cuda")
    device.distill_loss(one, tt[:1], ti[:1], l1, grad=grad)
    tol = h * h / 6 * 0.2 + (L.lse_error(n) + 2.0 ** -23 * np.abs(got).max()) / h
    assert np.abs(slope - grad.double().cpu().numpy()[0]).max() <= tol


def test_distill_offsets_past_32_bits(gpu):
    import torch

    from raft_amd import device
    ld = (1 << 31) + 9
    memory = torch.zeros(2 * ld + 4000, dtype=torch.bfloat16, device="cuda")
    z = memory.as_strided((3, 4000), (ld, 1))
    rng = np.random.default_rng(2)
    z.copy_(torch.as_tensor(rng.normal(0, 2, (3, 4000)).astype(np.float32)))
    t, idx = _teacher(rng, 3, 4000, 9, short=False)
    _check_distill(z, t, idx, 1.0, 1.0, calls=2)
    _check_distill(z, t, idx, 1.0, 1.0, in_place=True)
    del memory, z
    torch.cuda.empty_cache()


# ---- sampling ---------------------------------------------------------------------------------------


def _check_sample(view, u, allowed=None, **how):
    import torch

    from raft_amd import device
    rows, n = view.shape
    token = torch.full((rows,), -9, dtype=torch.int32, device="cuda")
    logprob = torch.full((rows,), 5.0, device="cuda")
    kw = {}
    for name, v in how.items():
        if v is not None:
            kw[name] = torch.as_tensor(np.asarray(v, dtype=np.int32 if name == "top_k" else np.float32)).cuda()
    if allowed is not None:
        kw["allowed"] = torch.as_tensor(L.pack_bits(allowed)).cuda()
    device.sample(view, torch.as_tensor(np.asarray(u, dtype=np.float32)).cuda(), token, logprob, **kw)
    as32 = {k: None if v is None else np.asarray(v, dtype=np.int64 if k == "top_k" else np.float32) for k, v in how.items()}
    want, lp, w = L.ref_sample(_host(view), np.asarray(u, dtype=np.float32), allowed=allowed, **as32)
    got = token.cpu().numpy()
    bad = np.flatnonzero(got != want)
    assert len(bad) == 0, (bad[:5], got[bad[:5]], want[bad[:5]], {k: None if v is None else v[bad[:5]] for k, v in as32.items()})
    g = logprob.cpu().numpy().astype(np.float64)
    none = np.isinf(lp)
    np.testing.assert_array_equal(g[none], lp[none])
    # the token's weight is off by half a step, the sum of all n by n half steps of a sum that is at
    # least 1; the result is rounded once
    step = L.weight_step(n)
    tol = 2.0 ** -24 * np.abs(lp[~none]) * 1.001 + step / w[~none] + n * step
    assert (np.abs(g[~none] - lp[~none]) <= tol).all(), (np.abs(g[~none] - lp[~none]) / tol).max()


def _settings(rng, rows, n):
    """Every combination of the settings, the off values among them, dealt over the rows."""
    pick = lambda *v: np.array([v[rng.integers(len(v))] for _ in range(rows)])  # noqa: E731
    return dict(temperature=pick(1.0, 0.7, 1.5, 0.0, -1.0, 0.05, 30.0, NAN, INF),
                top_k=pick(0, -3, 1, 2, 5, 40, 300, 2000, max(1, n - 1), n, n + 5),
                top_p=pick(1.0, 0.9, 0.5, 0.1, 0.999, 0.0, -1.0, 2.0, NAN, 0.95),
                min_p=pick(0.0, 0.0, 0.05, 0.5, 1.0, 2.0, 1e-6, NAN, -1.0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 33, 64, 255, 257, 1000, 2049, 5000, 9001])
def test_sample_lengths_and_settings(gpu, dtype, n):
    rng = np.random.default_rng(n)
    rows = 60
    view, _ = _put(rng.normal(0, 2, (rows, n)), dtype, pad=n % 4)
    u = rng.random(rows)
    _check_sample(view, u)
    _check_sample(view, u, **_settings(rng, rows, n))
    allowed = rng.random((rows, n)) < 0.4
    allowed[5] = False
    allowed[6] = False
    allowed[6, n - 1] = True
    _check_sample(view, u, allowed, **_settings(rng, rows, n))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [5, 300, 5001, 40003])
def test_sample_patterns(gpu, dtype, n):
    """Equal values at every border, -inf, NaN and +inf; u at both ends of its range and outside."""
    rng = np.random.default_rng(n)
    x = np.repeat(_patterns(n, rng), 6, axis=0)
    view, _ = _put(x, dtype)
    rows = len(x)
    u = np.tile([0.0, 0.3, 0.5, 1 - 2.0 ** -24, 1.0, -0.5], rows // 6)
    _check_sample(view, u)
    _check_sample(view, u, top_k=np.full(rows, 3))
    _check_sample(view, u, top_p=np.full(rows, 0.5))
    _check_sample(view, u, top_p=np.full(rows, 0.75), top_k=np.full(rows, 64))
    _check_sample(view, u, min_p=np.full(rows, 0.5))
    _check_sample(view, u, temperature=np.zeros(rows))
    _check_sample(view, u, **_settings(rng, rows, n))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,n", [(1, 131072), (6, 131071), (40, 32000), (3, 300007), (2, 1 << 20)])
@pytest.mark.parametrize("spread", [0.3, 4.0])
def test_sample_long_rows(gpu, dtype, rows, n, spread):
    rng = np.random.default_rng(rows + n)
    view, _ = _put(rng.normal(0, spread, (rows, n)), dtype, pad=1)
    for _ in range(2):
        _check_sample(view, rng.random(rows))
        _check_sample(view, rng.random(rows), top_k=rng.integers(1, 100, rows), top_p=0.5 + 0.5 * rng.random(rows))
        _check_sample(view, rng.random(rows), top_p=rng.random(rows))
        _check_sample(view, rng.random(rows), **_settings(rng, rows, n))
        _check_sample(view, rng.random(rows), rng.random((rows, n)) < 0.2, top_p=rng.random(rows), min_p=0.1 * rng.random(rows))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("times", [5, 140])
def test_sample_a_row_does_not_depend_on_the_others(gpu, dtype, masked, times):
    """The same 60 rows of every setting once and many times over: more rows than CUs, then more than
    8192, of which most need more than one pass."""
    import torch

    from raft_amd import device
    rng = np.random.default_rng(times)
    rows, n = 60, 8200
    x = rng.normal(0, 0.3, (rows, n))
    x[7] = -INF
    view, _ = _put(x, dtype)
    u, settings = rng.random(rows), _settings(rng, rows, n)
    allowed = rng.random((rows, n)) < 0.5 if masked else None
    _check_sample(view, u, allowed, **settings)
    got = []
    for count in (1, times):
        kw = {k: torch.as_tensor(v.astype(np.int32 if k == "top_k" else np.float32)).cuda().repeat(count)
              for k, v in settings.items()}
        if masked:
            kw["allowed"] = torch.as_tensor(L.pack_bits(allowed)).cuda().repeat(count, 1)
        token = torch.full((rows * count,), -9, dtype=torch.int32, device="cuda")
        logprob = torch.full((rows * count,), 5.0, device="cuda")
        device.sample(view.repeat(count, 1), torch.as_tensor(u.astype(np.float32)).cuda().repeat(count), token, logprob, **kw)
        got.append((token.cpu().numpy(), logprob.cpu().numpy()))
    for once, many in zip(*got):
        np.testing.assert_array_equal(np.tile(once, times), many)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,n", [(8, 131072), (300, 9001)])
def test_sample_top_p_and_min_p(gpu, dtype, rows, n):
    """Either cut first, and both near one another."""
    rng = np.random.default_rng(n)
    view, _ = _put(rng.normal(0, 1.0, (rows, n)), dtype)
    for min_p in (0.3, 0.05, 0.02, 1e-3):
        for top_p in (0.02, 0.3, 0.9, 0.999):
            _check_sample(view[:8], rng.random(8), top_p=np.full(8, top_p), min_p=np.full(8, min_p))
    _check_sample(view, rng.random(rows), top_p=rng.random(rows), min_p=rng.random(rows) ** 4)


def test_sample_follows_the_distribution(gpu):
    """One row with many random numbers: the counts of the tokens against their probabilities.  A count
    of N p is off by sqrt(N p) on average; six of those and one are allowed."""
    import torch

    from raft_amd import device
    n, many = 50, 20000
    x = torch.randn(n, generator=torch.Generator().manual_seed(4)).cuda()
    view = x.expand(many, n).contiguous()
    u = torch.rand(many, generator=torch.Generator().manual_seed(5)).cuda()
    token = torch.empty(many, dtype=torch.int32, device="cuda")
    device.sample(view, u, token)
    counts = torch.bincount(token.long(), minlength=n).double().cpu().numpy()
    p = torch.softmax(x.double().cpu(), 0).numpy()
    assert (np.abs(counts - many * p) <= 6 * np.sqrt(many * p) + 1).all()


def test_sample_without_a_vocabulary(gpu):
    import torch

    from raft_amd import device
    token, logprob = torch.full((3,), 5, dtype=torch.int32, device="cuda"), torch.zeros(3, device="cuda")
    device.sample(torch.empty(3, 0, device="cuda"), torch.zeros(3, device="cuda"), token, logprob)
    assert (token == -1).all() and (logprob == -INF).all()


@pytest.mark.parametrize("rows", [(1 << 20) + 1, (1 << 24) + 3])
def test_more_rows_than_one_grid_dimension_holds(gpu, rows):
    """2^20 workgroups are one line of the grid; 2^24 of 256 threads would be 2^32 threads."""
    import torch

    from raft_amd import device
    n = 3
    x = torch.randn(rows, n, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).half()
    best = x.float().max(1)
    values, indices = torch.empty(rows, 1, dtype=torch.float16, device="cuda"), torch.full((rows, 1), -1, dtype=torch.int32, device="cuda")
    device.top_k(x, values, indices)
    assert (values[:, 0].float() == best.values).all()
    token = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    zero = torch.zeros(rows, device="cuda")
    device.sample(x, zero, token, temperature=zero)
    assert (x.gather(1, token.long()[:, None])[:, 0].float() == best.values).all()
    loss, stats, grad = torch.full((rows,), -1.0, device="cuda"), torch.empty(rows, 2, device="cuda"), torch.empty_like(x)
    device.distill_loss(x, values, indices, loss, stats)
    # one listed token has p = 1, so the loss is -log q
    want = -torch.log_softmax(x.float(), 1).gather(1, indices.long())[:, 0]
    assert (loss - want).abs().max() < 1e-5
    device.distill_grad(x, values, indices, stats, grad)
    assert grad.float().sum(1).abs().max() < 3 * 2.0 ** -11  # q - p sums to 0; three roundings


# ---- together ---------------------------------------------------------------------------------------


def test_teacher_student_and_sampling_together(gpu):
    """A teacher's logits are reduced to their best, a student is trained on them by its own logits'
    gradient, and its logits are sampled: the losses against the 64-bit chain."""
    import torch

    from raft_amd import device
    rng = np.random.default_rng(12)
    rows, n, k, temperature = 48, 4001, 32, 2.0
    teacher, _ = _put(rng.normal(0, 3, (rows, n)), "bf16", pad=7)
    values = torch.empty(rows, k, dtype=torch.bfloat16, device="cuda")
    indices = torch.empty(rows, k, dtype=torch.int32, device="cuda")
    lse = torch.empty(rows, device="cuda")
    student = torch.randn(rows, n, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    loss, grad = torch.empty(rows, device="cuda"), torch.empty_like(student)
    token, logprob = torch.empty(rows, dtype=torch.int32, device="cuda"), torch.empty(rows, device="cuda")
    u = torch.rand(rows, device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    first = None
    for _ in range(4):
        device.top_k(teacher, values, indices, lse, temperature=temperature)
        device.distill_loss(student, values, indices, loss, grad=grad, temperature=temperature,
                            scale=temperature ** 2, teacher_lse=lse)
        want, dz, _, mass = L.ref_distill(_host(student), _host(values), indices.cpu().numpy(), temperature,
                                          temperature ** 2, lse.cpu().numpy())
        tol = temperature ** 2 * mass * L.lse_error(n) + 2.0 ** -23 * np.abs(want)
        assert (np.abs(_host(loss) - want) <= tol).all()
        first = want.sum() if first is None else first
        student -= 0.5 * grad
        device.sample(student, u, token, logprob, top_k=torch.full((rows,), 20, dtype=torch.int32, device="cuda"))
        t, _, _ = L.ref_sample(_host(student), u.cpu().numpy(), top_k=np.full(rows, 20))
        np.testing.assert_array_equal(token.cpu().numpy(), t)


def test_replayed_graph_and_another_stream(gpu):
    """The calls recorded into one HIP graph on a side stream, replayed over new contents with eager
    work on the same buffers between the replays, give the eager results bit for bit."""
    import torch

    from raft_amd import device
    gen = torch.Generator("cuda").manual_seed(3)
    shapes = [(4, 32000, torch.bfloat16), (1, 131072, torch.float32), (300, 2000, torch.float16)]
    state = []
    for rows, n, dt in shapes:
        f = lambda *s, d=torch.float32: torch.zeros(*s, dtype=d, device="cuda")  # noqa: E731
        api_ws = None
        state.append(dict(x=f(rows, n, d=dt), v=f(rows, 16, d=dt), i=f(rows, 16, d=torch.int32), lse=f(rows), loss=f(rows),
                          stats=f(rows, 2), g=f(rows, n, d=dt), g2=f(rows, n, d=dt), u=f(rows),
                          tok=f(rows, d=torch.int32), lp=f(rows), p=torch.full((rows,), 0.9, device="cuda"), ws=api_ws))

    def run():
        for s in state:
            device.top_k(s["x"], s["v"], s["i"], s["lse"])
            device.distill_loss(s["x"], s["v"], s["i"], s["loss"], s["stats"], s["g"])
            device.distill_grad(s["x"], s["v"], s["i"], s["stats"], s["g2"], teacher_lse=s["lse"])
            device.sample(s["x"], s["u"], s["tok"], s["lp"], top_p=s["p"])

    def outputs():
        return [s[k].clone() for s in state for k in ("v", "i", "lse", "loss", "stats", "g", "g2", "tok", "lp")]

    def fill():
        for s in state:
            s["x"].copy_(2 * torch.randn(s["x"].shape, device="cuda", generator=gen))
            s["u"].copy_(torch.rand(s["u"].shape, device="cuda", generator=gen))

    fill()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        run()
    for _ in range(4):
        fill()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        replayed = outputs()
        run()
        torch.cuda.synchronize()
        for a, b in zip(replayed, outputs()):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_two_streams_at_once(gpu):
    """Calls on two streams, each with outputs of its own, at the same time."""
    import torch

    from raft_amd import device
    gen = torch.Generator("cuda").manual_seed(8)
    x = [2 * torch.randn(64, 20000, device="cuda", generator=gen) for _ in range(2)]
    u = torch.rand(64, device="cuda", generator=gen)
    p = torch.full((64,), 0.8, device="cuda")
    torch.cuda.synchronize()
    out, streams = {}, [torch.cuda.Stream(), torch.cuda.Stream()]
    for rep in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                o = [torch.empty(64, 40, device="cuda"), torch.empty(64, 40, dtype=torch.int32, device="cuda"),
                     torch.empty(64, dtype=torch.int32, device="cuda"), torch.empty(64, device="cuda")]
                device.top_k(x[i], o[0], o[1])
                device.sample(x[i], u, o[2], o[3], top_p=p)
                out[rep, i] = o
    torch.cuda.synchronize()
    for i in range(2):
        want, _ = L.ref_top_k(_host(x[i]), 40)
        tok, _, _ = L.ref_sample(_host(x[i]), u.cpu().numpy(), top_p=np.full(64, 0.8, dtype=np.float32))
        for rep in range(5):
            np.testing.assert_array_equal(out[rep, i][1].cpu().numpy(), want)
            np.testing.assert_array_equal(out[rep, i][2].cpu().numpy(), tok)
