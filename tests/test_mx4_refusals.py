"""What mx4.linear refuses before it looks at any memory."""
import pytest
import torch

from chpl_b200 import _lib, mx4


@pytest.mark.parametrize("how", [{}, dict(stream=0), dict(stream=0, act="none")], ids=str)
def test_weights_that_are_not_coded(how):
    x = torch.empty(1, 32, dtype=torch.bfloat16)
    for w in (x, None, (x, x)):
        with pytest.raises(_lib.ChplError) as err:
            mx4.linear(x, w, **how)
        assert err.value.code == _lib.CHPL_ERR_INVALID
