"""The very codes that append_kv writes into a 4-bit cache, wherever float64 leaves no doubt about them.

Normed and rotated keys are float32 numbers: off by 2^-18 of the largest of the head, as in the tests of rotate_heads.  A power of two is in doubt where the largest of its 32
components is that near to 6 times a power, a code where its value is that near to the border between two.  Elsewhere both are those of float64;
in doubt they are one of the two that meet there.  Values are not changed before they are rounded: no doubt about any."""
import pytest
import torch

import jaxmodules_b200 as jm
from jaxmodules_b200 import attention as A
from oracle import paged_oracle as po

pytestmark = pytest.mark.gpu

BORDERS = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64)


def magnitudes(pages):
    """Codes of the magnitudes, 0 to 7, and signs, [..., d]."""
    codes = torch.stack((pages & 15, pages >> 4), -1).flatten(-2)
    return (codes & 7).int(), (codes >> 3).bool()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d,dim,layout,norm,spread", [
    (128, 128, "half", True, 0), (128, 128, "interleaved", False, 0), (64, 64, "half", False, 40), (32, 32, "half", True, 0), (96, 96, "interleaved", True, 20),
    (128, 36, "half", True, 0), (64, 20, "interleaved", True, 0), (96, 0, "half", False, 100),
])
def test_codes(d, dim, layout, norm, spread, dtype):
    B, T, H, page = 3, 170, 2, 16
    g = torch.Generator(device="cuda").manual_seed(d + dim)
    width = -(-2 * T // page)
    table = torch.randperm(B * width, generator=torch.Generator().manual_seed(1)).int().reshape(B, width).cuda()
    c = jm.PagedCache.empty(B * width, page, H, d, table, "4bit")
    powers = torch.randint(-spread // 2, spread // 2 + 1, (B, T, H, 1), device="cuda", generator=g)
    k, v = ((torch.randn((B, T, H, d), device="cuda", generator=g) * torch.exp2(powers)).to(dtype) for _ in range(2))
    w = (1 + torch.randn(d, device="cuda", generator=g) / 4).to(dtype) if norm else None
    f = jm.rotary_frequencies(dim) if dim else None
    lengths = [T + 150, T, 2 * T]
    jm.append_kv(c, k, v, torch.tensor(lengths, dtype=torch.int32, device="cuda"), frequencies=f, layout=layout, k_weight=w)
    doubtful = total = 0
    for b, n in enumerate(lengths):
        at = torch.arange(n - T, n, device="cuda")
        slots = table[b].long()[at // page], at % page
        for pages, scales, want, doubt in ((c.k, c.k_scale, po.rotate(k[b].double(), at[:, None], f, layout, 1.0, None if w is None else w.double()), 2.0 ** -18),
                                           (c.v, c.v_scale, v[b].double(), 0.0)):
            if not dim and not norm:
                doubt = 0.0                        # (nothing is done to these keys)
            near = doubt * want.abs().amax(-1, keepdim=True)
            low, high = (po.to_4bit((want.abs() + x).clamp(min=0))[1].int() for x in (-near, near))          # powers of what float32 may have made of it
            byte = scales[slots].int()
            assert ((byte >= low) & (byte <= high)).all()
            unit = torch.exp2(byte.double() - 127).repeat_interleave(32, -1)
            code, sign = magnitudes(pages[slots])
            y, off = want.abs() / unit, near / unit
            borders = BORDERS.cuda()
            least, most = (torch.searchsorted(borders, x.contiguous()) for x in (y - off, y + off))
            if doubt == 0.0:                       # ties go to the even code
                tie = (y[..., None] == borders).any(-1)
                least = torch.where(tie & (least % 2 == 1), least + 1, least)
                most = least
            assert ((code >= least) & (code <= most)).all()
            assert (sign == (want < 0))[want.abs() > near].all()
            doubtful += (least != most).sum().item()
            total += code.numel()
    assert doubtful <= 1e-3 * total and A.device_status() == 0
