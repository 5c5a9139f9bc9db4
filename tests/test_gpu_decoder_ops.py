"""The operators around a decoder's cache as ``torch.ops.natten_b200``."""
import pytest

from natten_mps_b200 import _cabi, functional  # noqa: F401  (registers the operators)
from tests._decoder_calls import misfits

pytestmark = pytest.mark.gpu


def test_shapes_that_do_not_fit_are_refused_before_a_launch():
    calls = misfits("cuda")
    before = _cabi.launch_count()
    for name, call in calls:
        with pytest.raises(ValueError, match="natten_b200"):
            call()
            pytest.fail(name)
    assert _cabi.launch_count() == before
