"""Refusals of the operators over rows of logits (rmi_top_k, rmi_distill_*, rmi_sample): every one
of these calls returns before anything is launched, so no GPU is needed."""
import pytest

from raft_amd import _capi as api

P = 0x1000  # stands for a device address; never dereferenced by a refused call


def _call(name, change):
    lib = api.load()
    args = {
        "rmi_top_k": dict(dtype=api.F32, n_rows=2, n_cols=100, ld=100, k=5, temperature=1.0, logits=P, values=P,
                          indices=P, lse=P, stream=None),
        "rmi_distill_loss": dict(dtype=api.F32, t_dtype=api.F32, n_rows=2, n_cols=100, ld=100, k=5, temperature=1.0,
                                 scale=1.0, logits=P, t_values=P, t_indices=P, t_lse=P, loss=P, stats=P, row_grad=P,
                                 grad=P, ld_grad=100, stream=None),
        "rmi_distill_grad": dict(dtype=api.F32, t_dtype=api.F32, n_rows=2, n_cols=100, ld=100, k=5, temperature=1.0,
                                 scale=1.0, logits=P, t_values=P, t_indices=P, t_lse=P, stats=P, row_grad=P, grad=P,
                                 ld_grad=100, stream=None),
        "rmi_sample": dict(dtype=api.F32, n_rows=2, n_cols=100, ld=100, logits=P, allowed=P, ld_allowed=4,
                           temperature=P, top_k=P, top_p=P, min_p=P, u=P, token=P, logprob=P, ws=P, ws_bytes=1 << 20,
                           stream=None),
    }[name]
    assert set(change) <= set(args)
    args.update(change)
    return getattr(lib, name)(*args.values())


ALL = ["rmi_top_k", "rmi_distill_loss", "rmi_distill_grad", "rmi_sample"]
COMMON = [
    (dict(dtype=api.F64), api.ERR_UNSUPPORTED),
    (dict(dtype=api.I32), api.ERR_UNSUPPORTED),
    (dict(dtype=77), api.ERR_BAD_ENUM),
    (dict(dtype=-1), api.ERR_BAD_ENUM),
    (dict(n_rows=-1), api.ERR_BAD_SHAPE),
    (dict(n_cols=-1), api.ERR_BAD_SHAPE),
    (dict(n_cols=1 << 31, ld=1 << 31), api.ERR_BAD_SHAPE),
    (dict(n_rows=1 << 31), api.ERR_BAD_SHAPE),
    (dict(ld=99), api.ERR_BAD_SHAPE),
    (dict(logits=None), api.ERR_NULL),
    (dict(logits=P + 2), api.ERR_ALIGNMENT),
    (dict(dtype=api.BF16, logits=P + 1), api.ERR_ALIGNMENT),
]


@pytest.mark.parametrize("name", ALL)
@pytest.mark.parametrize("change,status", COMMON)
def test_refused_by_all(name, change, status):
    assert _call(name, change) == status


@pytest.mark.parametrize("change,status", [
    (dict(k=0), api.ERR_BAD_SHAPE), (dict(k=101), api.ERR_BAD_SHAPE),
    (dict(k=api.TOP_K_MAX + 1, n_cols=5000, ld=5000), api.ERR_BAD_SHAPE),
    (dict(n_cols=0, ld=0), api.ERR_BAD_SHAPE),
    (dict(temperature=0.0), api.ERR_UNSUPPORTED), (dict(temperature=float("nan")), api.ERR_UNSUPPORTED),
    (dict(temperature=1e7), api.ERR_UNSUPPORTED), (dict(temperature=-1.0), api.ERR_UNSUPPORTED),
    (dict(values=None), api.ERR_NULL), (dict(indices=None), api.ERR_NULL),
    (dict(values=P + 1), api.ERR_ALIGNMENT), (dict(indices=P + 2), api.ERR_ALIGNMENT), (dict(lse=P + 2), api.ERR_ALIGNMENT),
    (dict(n_rows=0, logits=None, values=None, indices=None), api.OK),
])
def test_top_k_refusals(change, status):
    assert _call("rmi_top_k", change) == status


@pytest.mark.parametrize("name", ["rmi_distill_loss", "rmi_distill_grad"])
@pytest.mark.parametrize("change,status", [
    (dict(t_dtype=api.F64), api.ERR_UNSUPPORTED), (dict(t_dtype=99), api.ERR_BAD_ENUM),
    (dict(k=-1), api.ERR_BAD_SHAPE), (dict(k=api.DISTILL_MAX + 1), api.ERR_BAD_SHAPE),
    (dict(ld_grad=99), api.ERR_BAD_SHAPE),
    (dict(temperature=0.0), api.ERR_UNSUPPORTED), (dict(temperature=float("inf")), api.ERR_UNSUPPORTED),
    (dict(scale=float("nan")), api.ERR_UNSUPPORTED), (dict(scale=float("inf")), api.ERR_UNSUPPORTED),
    (dict(t_values=None), api.ERR_NULL), (dict(t_indices=None), api.ERR_NULL),
    (dict(t_values=P + 2), api.ERR_ALIGNMENT), (dict(t_indices=P + 1), api.ERR_ALIGNMENT),
    (dict(t_lse=P + 1), api.ERR_ALIGNMENT), (dict(row_grad=P + 2), api.ERR_ALIGNMENT),
    (dict(grad=P + 2), api.ERR_ALIGNMENT), (dict(stats=P + 2), api.ERR_ALIGNMENT),
])
def test_distill_refusals(name, change, status):
    assert _call(name, change) == status


def test_distill_refusals_of_one_call():
    assert _call("rmi_distill_loss", dict(loss=None)) == api.ERR_NULL
    assert _call("rmi_distill_loss", dict(loss=P + 2)) == api.ERR_ALIGNMENT
    assert _call("rmi_distill_loss", dict(n_rows=0, logits=None, loss=None, t_values=None, t_indices=None)) == api.OK
    assert _call("rmi_distill_grad", dict(stats=None)) == api.ERR_NULL
    assert _call("rmi_distill_grad", dict(grad=None)) == api.ERR_NULL
    assert _call("rmi_distill_grad", dict(n_cols=0, ld=0, logits=None, grad=None, stats=None)) == api.OK


@pytest.mark.parametrize("change,status", [
    (dict(ld_allowed=3), api.ERR_BAD_SHAPE), (dict(u=None), api.ERR_NULL), (dict(token=None), api.ERR_NULL),
    (dict(allowed=P + 2), api.ERR_ALIGNMENT), (dict(temperature=P + 1), api.ERR_ALIGNMENT),
    (dict(top_k=P + 1), api.ERR_ALIGNMENT), (dict(top_p=P + 2), api.ERR_ALIGNMENT),
    (dict(min_p=P + 2), api.ERR_ALIGNMENT), (dict(u=P + 2), api.ERR_ALIGNMENT),
    (dict(token=P + 2), api.ERR_ALIGNMENT), (dict(logprob=P + 2), api.ERR_ALIGNMENT),
    (dict(ws=None), api.ERR_WORKSPACE), (dict(ws_bytes=65536 + 71), api.ERR_WORKSPACE), (dict(ws=P + 8), api.ERR_WORKSPACE),
    (dict(n_rows=0, logits=None, u=None, token=None), api.OK),
])
def test_sample_refusals(change, status):
    assert _call("rmi_sample", change) == status


def test_workspace_queries_of_bad_shapes():
    lib = api.load()
    assert lib.rmi_sample_workspace_bytes(api.F64, 400, 1 << 20) == 0
    assert lib.rmi_sample_workspace_bytes(99, 400, 1 << 20) == 0
    assert lib.rmi_sample_workspace_bytes(api.F32, -4, 1 << 20) == 0
    assert lib.rmi_sample_workspace_bytes(api.F32, 4, -1) == 0


def test_wrappers_refuse_what_does_not_fit():
    torch = pytest.importorskip("torch")
    from raft_amd import device
    x = torch.zeros(2, 8)
    with pytest.raises(ValueError):  # not on the GPU
        device.top_k(x, torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.int32))
    with pytest.raises(ValueError):  # no such type
        device.sample(x.double(), torch.zeros(2), torch.zeros(2, dtype=torch.int32))
