"""The operators around a decoder's cache as ``torch.ops.natten_b200``, what needs no GPU."""
import pytest
import torch
import torch.autograd.forward_ad as fw

import natten_mps_b200  # noqa: F401  (registers the operators)
from natten_mps_b200 import functional as F
from tests._decoder_calls import misfits


@pytest.mark.parametrize("name,call", misfits("meta"), ids=lambda x: x if isinstance(x, str) else "")
def test_shapes_that_do_not_fit_are_refused(name, call):
    with pytest.raises(ValueError, match="natten_b200"):
        call()


def _dual_calls():
    """Calls of every kind of operator on small ``meta`` tensors, by what they do with one of their arguments."""
    z = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device="meta")  # noqa: E731
    k, f, rpb = z(2, 5, 2, 8), z(4, dtype=torch.float64), z(4, 5)
    kc, table, lens = z(6, 4, 2, 8), z(2, 3, dtype=torch.int32), z(2, dtype=torch.int32)
    return {
        "rotary": lambda x: F.na1d_rotary(x, k, f), "rotary key": lambda x: F.na1d_rotary(x, x, f),
        "append": lambda x: F.na1d_append(x[:, :, :2], k, kc, kc.clone(), table, lens),
        "append query": lambda x: F.na1d_append(k, k, kc, kc.clone(), table, lens, query=x),
        "paged": lambda x: F.na1d_paged(x, kc, kc, table, lens, 3), "paged, all": lambda x: F.na1d_paged(x, kc, kc, table, lens),
        "fused": lambda x: F.na1d(x, k, k, 3),
        "qk": lambda x: F.na1d_qk(x, x, 3), "av": lambda x: F.na1d_av(x[..., :3], x, 3),
        "rpb": lambda x: F.na1d_qk_rpb(x, x, rpb, 3),
        "registered": lambda x: torch.ops.natten_b200.na1d_rotary(x, k, f, None, False, 1.0, False),
    }


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("name", _dual_calls())
def test_forward_mode_tangents_are_refused_not_lost(name, grad):
    x = torch.zeros(2, 5, 4, 8, device="meta")
    call = _dual_calls()[name]
    call(x)
    with fw.dual_level(), torch.set_grad_enabled(grad):
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(fw.make_dual(x, torch.ones_like(x)))
        call(x)


def test_forward_mode_tangents_of_caches_and_frequencies_are_refused():
    x, kc, f = torch.zeros(2, 5, 2, 8, device="meta"), torch.zeros(6, 4, 2, 8, device="meta"), torch.ones(4, device="meta").double()
    table, lens = torch.zeros(2, 3, dtype=torch.int32, device="meta"), torch.zeros(2, dtype=torch.int32, device="meta")
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: F.na1d_rotary(x, x, dual(f)), lambda: F.na1d_paged(x, kc, dual(kc), table, lens),
                     lambda: F.na1d_append(x, x, dual(kc), kc, table, lens)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
