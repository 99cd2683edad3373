"""What the library refuses comes from rotate_heads as the error of the other calls, with the status, with and without a gradient."""
import pytest
import torch

import jaxmodules_b200 as jm
from jaxmodules_b200 import _native as nat

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("gradient", [False, True])
def test_too_many_tokens(gradient):
    q = torch.ones((1, 1, 1, 1), device="cuda", dtype=torch.bfloat16).expand(1, 1 << 30, 1, 1)
    w = torch.ones(1, device="cuda", requires_grad=gradient)
    with pytest.raises(nat.BmaError) as e:
        jm.rotate_heads(q, None, q_weight=w)
    assert e.value.status == nat.BMA_ERR_LIMIT
