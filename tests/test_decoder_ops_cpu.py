"""The operators around a decoder's cache as ``torch.ops.natten_b200``, what needs no GPU."""
import pytest

import natten_mps_b200  # noqa: F401  (registers the operators)
from natten_mps_b200 import functional  # noqa: F401
from tests._decoder_calls import misfits


@pytest.mark.parametrize("name,call", misfits("meta"), ids=lambda x: x if isinstance(x, str) else "")
def test_shapes_that_do_not_fit_are_refused(name, call):
    with pytest.raises(ValueError, match="natten_b200"):
        call()
