"""append_kv writes into the tensors of a cache, and torch is told."""
import pytest
import torch

import jaxmodules_b200 as jm

pytestmark = pytest.mark.gpu


def append(c):
    x = torch.ones((1, 1, 1, 32), device="cuda", dtype=torch.bfloat16)
    jm.append_kv(c, x, x, torch.ones(1, dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("kind", [torch.bfloat16, "4bit"])
def test_versions(kind):
    c = jm.PagedCache.empty(2, 4, 1, 32, torch.zeros((1, 1), dtype=torch.int32, device="cuda"), kind)
    tensors = [x for x in (c.k, c.v, c.k_scale, c.v_scale) if x is not None]
    before, table = [x._version for x in tensors], c.page_table._version
    append(c)
    assert [x._version for x in tensors] == [n + 1 for n in before] and c.page_table._version == table


def test_a_graph_that_saved_pages_notices():
    c = jm.PagedCache.empty(2, 4, 1, 32, torch.zeros((1, 1), dtype=torch.int32, device="cuda"), torch.bfloat16)
    w = torch.ones((), device="cuda", requires_grad=True)
    y = (c.k[:1] * w).sum()
    append(c)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_a_cache_made_in_inference_mode():
    with torch.inference_mode():
        c = jm.PagedCache.empty(2, 4, 1, 32, torch.zeros((1, 1), dtype=torch.int32, device="cuda"), torch.bfloat16)
        append(c)
    append(c)
    assert c.k.float().sum() == 32
