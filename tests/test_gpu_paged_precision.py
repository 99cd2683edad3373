"""How near paged_attention over a bfloat16 cache comes to float64: as near as float32 arithmetic, not as near as bfloat16 weights would.

Tolerances, per component, in units of sum p |v|: weights go through the product as two bfloat16 numbers, the first cut off after 8 bits, the second what is left (less than 2^-7 of
the weight) and rounded by 2^-8 of itself: 2^-15, with 2^-20 that is added to keep both above zero.  Sums and exponentials in float32 2^-17, as for float32 caches.  A logit is a sum of d products: d 2^-24 of the sum of their sizes at worst, which
counts twice (in its weight, and in the sum of all)."""
import math

import pytest
import torch

import jaxmodules_b200 as jm
from jaxmodules_b200 import attention as A
from oracle import paged_oracle as po

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lengths,T,Hq,H,d,window", [
    ([1], 1, 1, 1, 64, None), ([1500], 1, 16, 2, 64, None), ([700, 33, 64, 5], 1, 32, 8, 128, None), ([300, 41], 3, 8, 2, 128, None), ([300, 41], 7, 16, 4, 64, 100),
    ([6000], 4, 28, 4, 128, None), ([20000, 9], 1, 8, 8, 128, None), ([250, 16], 2, 5, 1, 72, 40),
])
def test_bfloat16(lengths, T, Hq, H, d, window):
    g = torch.Generator(device="cuda").manual_seed(T + d)
    page, B = 16, len(lengths)
    width = -(-max(lengths) // page)
    table = torch.randperm(B * width, generator=torch.Generator().manual_seed(d)).int().reshape(B, width).cuda()
    pages = [torch.randn((B * width, page, H, d), device="cuda", generator=g).bfloat16() for _ in range(2)]
    c = jm.PagedCache(*pages, table)
    q = torch.randn((B, T, Hq, d), device="cuda", generator=g).bfloat16()
    new = [min(T, n) for n in lengths]
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    o, lse = jm.paged_attention(q, c, ints(lengths), new_lengths=ints(new), window=window, return_lse=True)
    half = jm.paged_attention(q, c, ints(lengths), new_lengths=ints(new), window=window, out_dtype=torch.bfloat16)
    assert o.dtype == torch.float32 and A.device_status() == 0
    ks, vs = ([po.context(x.double(), table, b, n, page) for b, n in enumerate(lengths)] for x in pages)
    want, want_lse, size = po.attend(q.double(), ks, vs, lengths, new, window=window)
    most = max((q[b].double().abs().reshape(T, H, -1, d).transpose(1, 2).reshape(-1, H, d).unsqueeze(1) * ks[b].abs()).sum(-1).max() for b in range(B))
    off = float(most) * d * 2.0 ** -24 / math.sqrt(d)
    assert off < 2.0 ** -12
    bound = (2.0 ** -15 + 2.0 ** -20 + 2.0 ** -17 + 2 * off) * size
    assert ((o.double() - want).abs() <= bound + 1e-30).all(), ((o.double() - want).abs() / (bound + 1e-30)).max()
    assert ((half.double() - want).abs() <= 2.0 ** -8 * want.abs() + bound * (1 + 2.0 ** -8) + 1e-30).all()
    seen = want_lse > -torch.inf
    assert ((lse.double() - want_lse).abs()[seen] <= off + 2.0 ** -17).all()


@pytest.mark.parametrize("T", [1, 3])
@pytest.mark.parametrize("where", [0, 17, 99])
def test_infinite_values(where, T):
    """A weight makes an infinity of an infinity, whatever its bits, in every row that sees it."""
    n, H, d = 100, 2, 64
    g = torch.Generator(device="cuda").manual_seed(where)
    pages = [torch.randn((7, 16, H, d), device="cuda", generator=g).bfloat16() for _ in range(2)]
    pages[1][where // 16, where % 16, :, 5], pages[1][where // 16, where % 16, :, 6] = torch.inf, -torch.inf
    c = jm.PagedCache(*pages, torch.arange(7, dtype=torch.int32, device="cuda")[None])
    q = torch.randn((1, T, 8, d), device="cuda", generator=g).bfloat16()
    q[:, :, ::2] = 0                                 # weights of 1
    o = jm.paged_attention(q, c, torch.tensor([n], dtype=torch.int32, device="cuda"))
    sees = torch.arange(n - T, n, device="cuda") >= where
    assert (o[0, sees][..., 5] == torch.inf).all() and (o[0, sees][..., 6] == -torch.inf).all()
    assert o[0, ~sees].isfinite().all() and o[..., :5].isfinite().all() and o[..., 7:].isfinite().all()
