"""Derivatives that the calls around the paged cache do not have are refused, in reverse and in forward mode, before anything else is looked at."""
import pytest
import torch
import torch.autograd.forward_ad as forward

import jaxmodules_b200 as jm

F = torch.zeros(4, dtype=torch.float64)


def heads(H=2):
    return torch.zeros((2, 3, H, 8))


def cache(**kw):
    c = jm.PagedCache.empty(5, 4, 2, 8, torch.zeros((2, 3), dtype=torch.int32), torch.float32)
    return jm.PagedCache(**{**c.__dict__, **kw})


LENGTHS = torch.zeros(2, dtype=torch.int32)
PAGES = torch.zeros(5, 4, 2, 8)
W = torch.ones(8)
# the call with one tensor of its own, and that tensor
CALLS = {
    "rotate_heads, q": (lambda x: jm.rotate_heads(x, heads(), None, F), heads()),
    "rotate_heads, k": (lambda x: jm.rotate_heads(heads(), x, None, F), heads()),
    "rotate_heads, q_weight": (lambda x: jm.rotate_heads(heads(), heads(), None, F, q_weight=x), W),
    "rotate_heads, k_weight": (lambda x: jm.rotate_heads(heads(), heads(), None, F, k_weight=x), W),
    "rotate_heads, frequencies": (lambda x: jm.rotate_heads(heads(), None, None, x), F),
    "append_kv, k": (lambda x: jm.append_kv(cache(), x, heads(), LENGTHS), heads()),
    "append_kv, v": (lambda x: jm.append_kv(cache(), heads(), x, LENGTHS), heads()),
    "append_kv, q": (lambda x: jm.append_kv(cache(), heads(), heads(), LENGTHS, q=x, frequencies=F), heads(4)),
    "append_kv, q_weight": (lambda x: jm.append_kv(cache(), heads(), heads(), LENGTHS, q=heads(4), q_weight=x), W),
    "append_kv, k_weight": (lambda x: jm.append_kv(cache(), heads(), heads(), LENGTHS, k_weight=x), W),
    "append_kv, frequencies": (lambda x: jm.append_kv(cache(), heads(), heads(), LENGTHS, frequencies=x), F),
    "append_kv, pages": (lambda x: jm.append_kv(cache(k=x), heads(), heads(), LENGTHS), PAGES),
    "read_kv, pages of keys": (lambda x: jm.read_kv(cache(k=x), LENGTHS, 4), PAGES),
    "read_kv, pages of values": (lambda x: jm.read_kv(cache(v=x), LENGTHS, 4), PAGES),
    "paged_attention, q": (lambda x: jm.paged_attention(x, cache(), LENGTHS), heads(4)),
    "paged_attention, pages of keys": (lambda x: jm.paged_attention(heads(4), cache(k=x), LENGTHS), PAGES),
    "paged_attention, pages of values": (lambda x: jm.paged_attention(heads(4), cache(v=x), LENGTHS), PAGES),
}


@pytest.mark.parametrize("name", CALLS)
def test_dual_tensors_are_refused(name):
    call, x = CALLS[name]
    with forward.dual_level():
        with pytest.raises(ValueError, match="forward mode"):
            call(forward.make_dual(x, torch.ones_like(x)))
        with torch.no_grad(), pytest.raises(ValueError, match="forward mode"):      # (which leaves forward mode on)
            call(forward.make_dual(x, torch.ones_like(x)))
    with pytest.raises(RuntimeError, match="CUDA"):
        call(x)


# (rotate_heads has gradients of the others)
@pytest.mark.parametrize("name", [n for n in CALLS if not n.startswith("rotate_heads") or n.endswith("frequencies")])
def test_gradients_that_there_are_not_are_refused(name):
    call, x = CALLS[name]
    x = x.clone().requires_grad_()
    with pytest.raises(ValueError, match="not differentiable"):
        call(x)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
        call(x)
