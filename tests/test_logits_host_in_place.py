"""A gradient in the logits' own memory whose rows lie another distance apart is refused before anything is
launched: no GPU is needed."""
import pytest

from raft_amd import _capi as api
from tests.test_logits_host import P, _call


@pytest.mark.parametrize("name", ["rmi_distill_loss", "rmi_distill_grad"])
@pytest.mark.parametrize("ld,ld_grad", [(100, 101), (128, 100), (1 << 20, 100)])
def test_in_place_with_another_row_stride(name, ld, ld_grad):
    # t_indices is refused after that: an accepted shape would end there
    assert _call(name, dict(ld=ld, ld_grad=ld_grad, t_indices=P + 2)) == api.ERR_BAD_SHAPE


@pytest.mark.parametrize("name", ["rmi_distill_loss", "rmi_distill_grad"])
@pytest.mark.parametrize("change", [dict(ld=128, ld_grad=128), dict(n_rows=1, ld=128, ld_grad=100),
                                    dict(ld=128, ld_grad=100, grad=P + (1 << 20))])
def test_in_place_and_apart(name, change):
    assert _call(name, dict(change, t_indices=P + 2)) == api.ERR_ALIGNMENT
