"""paged_attention over 4-bit caches whose powers of two go through the whole range of the format, against float64.

Tolerances.  A component's weights are float16 numbers: off by 2^-11 of themselves, or by 2^-40 of the largest weight times power (of the component's group of 32 where
powers are far apart, of the head's largest group where they are not), once as a weight and once more times its power, times a code of at most 6.  Logits are sums of d
products in float32, d 2^-24 of the sum of their sizes at worst, and a component of a query is off by 2^-40 of the largest of its row: d 2^-40 max |q| max |k| in all; an error of a
logit is one of its weight, and, through the sum of the weights, of all.  2^-17 for exponentials and sums, as for the other caches."""
import math

import pytest
import torch

import jaxmodules_b200 as jm
from jaxmodules_b200 import attention as A
from oracle import paged_oracle as po

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def cache(lengths, H, d, page=16, seed=0, scale_pad=0):
    """Random codes, powers of 1; `scale_pad`: bytes between the powers of a head and the next's."""
    width = max(-(-n // page) for n in lengths)
    B = len(lengths)
    table = torch.randperm(B * width, generator=torch.Generator().manual_seed(seed)).int().reshape(B, width).cuda()
    c = jm.PagedCache.empty(B * width, page, H, d, table, "4bit")
    for x in (c.k, c.v):
        x.copy_(torch.randint(0, 256, x.shape, device="cuda", generator=gen(seed + 1), dtype=torch.uint8))
    scales = [torch.zeros((B * width, page, H, d // 32 + scale_pad), dtype=torch.uint8, device="cuda")[..., :d // 32] for _ in range(2)]
    for s in scales:
        s.fill_(127)
    scales[0].fill_(125)
    return jm.PagedCache(c.k, c.v, c.page_table, *scales)


def at(c, b, positions):
    """Index of the slots of positions of sequence b."""
    positions = torch.as_tensor(positions, device="cuda")
    return c.page_table[b].long()[positions // c.k.shape[1]], positions % c.k.shape[1]


def check(q, c, lengths, apart, window=None):
    """`apart`: every tile of keys has a head whose powers are far apart."""
    B, T, Hq, d = q.shape
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    o, lse = jm.paged_attention(q, c, n, window=window, return_lse=True)
    assert A.device_status() == 0
    kv, vv = po.held_values(c.k, c.k_scale), po.held_values(c.v, c.v_scale)
    G = Hq // c.k.shape[2]
    for b, length in enumerate(lengths):
        slots = at(c, b, list(range(length)))
        k, v, e = (x[slots].repeat_interleave(G, 1) for x in (kv, vv, torch.exp2(c.v_scale.double() - 127)))
        if not apart:
            e = e.amax(-1, keepdim=True).expand(e.shape)
        for t in range(T):
            end = length - T + t + 1
            lo = 0 if window is None else max(0, end - 1 - window)
            x = q[b, t].double()
            logits = torch.einsum("hd,lhd->hl", x, k[lo:end]) / math.sqrt(d)
            sizes = torch.einsum("hd,lhd->hl", x.abs(), k[lo:end].abs()).amax(-1) * d * 2.0 ** -24
            off = (sizes + d * 2.0 ** -40 * x.abs().amax(-1) * k[lo:end].abs().amax((0, 2))) / math.sqrt(d)      # of a logit
            assert off.max() < 2.0 ** -8          # (what the inputs are chosen for)
            p = torch.softmax(logits, -1)
            want, size = (torch.einsum("hl,lhd->hd", p, y) for y in (v[lo:end], v[lo:end].abs()))
            most = (p[..., None] * e[lo:end].transpose(0, 1)).amax(1).repeat_interleave(32, -1)
            bound = (2.0 ** -11 + 2.0 ** -17 + 2 * off[:, None]) * size + 12 * (end - lo) * 2.0 ** -40 * most + 2.0 ** -100
            got = o[b, t].double()
            assert (got - want).abs().div(bound).max() <= 1, (b, t, (got - want).abs().div(bound).max())
            assert ((lse[b, :, t].double() - torch.logsumexp(logits, -1)).abs() <= off + 2.0 ** -17).all()


def queries(B, T, H, d, seed=5):
    return torch.randn((B, T, H, d), device="cuda", generator=gen(seed)).bfloat16()


@pytest.mark.parametrize("power", [-126, -100, -60, -41, 41, 60, 76, 100, 120])
@pytest.mark.parametrize("where", [0, 40, 99])
def test_one_key_of_large_or_small_values(where, power):
    """The others count in the sum of weights whatever its power, and the small ones of the others in their components."""
    lengths = [100, 37]
    c = cache(lengths, 2, 128)
    c.v_scale[at(c, 0, where)] = 127 + power
    c.v[at(c, 0, where)] |= 0x11                    # (codes other than zero)
    beside = at(c, 0, (where + 1) % 100)            # a zero value, with the least power, as append_kv writes it
    c.v[beside], c.v_scale[beside] = 0, 0
    check(queries(2, 1, 4, 128), c, lengths, False)


@pytest.mark.parametrize("d,T,Hq,H", [(128, 1, 4, 1), (128, 3, 8, 2), (64, 1, 4, 2), (64, 5, 6, 2), (96, 2, 3, 3)])
@pytest.mark.parametrize("spread", [15, 25, 60, 90])
def test_groups_of_a_head_far_apart(spread, d, T, Hq, H):
    """Each group of 32 is as good as if it stood alone."""
    lengths = [200, 64, 5]
    c = cache(lengths, H, d, seed=spread)
    powers = torch.randint(0, 5, c.v_scale.shape, device="cuda", generator=gen(9), dtype=torch.uint8) + 127 - spread // 2
    powers[..., ::2] += spread + 4
    c.v_scale.copy_(powers)
    check(queries(3, T, Hq, d), c, lengths, True)
    check(queries(3, T, Hq, d), c, lengths, True, window=70)


def test_powers_at_the_limit():
    """Spread and largest powers just inside of what one maximum for both serves."""
    lengths = [130]
    for top, spread in ((40, 14), (-40, 14), (0, 14), (40, 0), (-40, 0), (-26, 14)):
        c = cache(lengths, 1, 128)
        c.v_scale[:] = 127 + top
        c.v_scale[..., 1] -= spread
        check(queries(1, 2, 4, 128), c, lengths, False)


@pytest.mark.parametrize("scale_pad", [0, 3, 4])
@pytest.mark.parametrize("far", [False, True])
def test_powers_that_are_not_words(far, scale_pad):
    """A head's four powers read at once, and byte by byte."""
    lengths = [150, 33]
    c = cache(lengths, 3, 128, scale_pad=scale_pad)
    c.v_scale.copy_(torch.randint(120, 130, c.v_scale.shape, device="cuda", generator=gen(2), dtype=torch.uint8))
    if far:
        c.v_scale[..., 2] = 90
    check(queries(2, 2, 6, 128), c, lengths, far)


@pytest.mark.parametrize("parts", [20000, 3000])
def test_parts_of_one_sequence(parts):
    """Runs with and without such a key, put together again."""
    lengths = [parts, 12]
    c = cache(lengths, 2, 128)
    for where, power in ((parts // 3, 90), (parts // 3 + 1, -90), (parts - 2, 60)):
        c.v_scale[at(c, 0, where)] = 127 + power
    check(queries(2, 1, 4, 128), c, lengths, False)


@pytest.mark.parametrize("e", [-126, -100, 90, 110])
def test_powers_of_keys(e):
    """Keys of very small and very large powers, and queries that make ordinary logits of them."""
    lengths = [90]
    c = cache(lengths, 2, 128)
    c.k_scale[:] = 127 + e
    q = (queries(1, 2, 4, 128).double() * 2.0 ** (-e - 2)).bfloat16()
    check(q, c, lengths, False)
    c.k_scale[at(c, 0, 50)] = 0                     # 2^-127
    check(q, c, lengths, False)


@pytest.mark.parametrize("down", [8, 20, 26])
def test_small_components_of_a_query(down):
    """A group of small components, which meets keys of large powers, counts as much as the other."""
    lengths = [90]
    c = cache(lengths, 1, 64)
    q = queries(1, 1, 4, 64)
    q[..., 32:] *= 2.0 ** -down
    c.k_scale[..., 0], c.k_scale[..., 1] = 125 - 10, 125 + down - 4
    check(q, c, lengths, False)


@pytest.mark.parametrize("size", [1, 40, 200])
def test_rows_that_see_nothing_of_a_tile(size):
    """Far below zero as the logits of all that such a row has seen may be.  (So many sequences that a warp has all tiles of some of them.)"""
    B, T = 500, 3
    lengths = [33 + i % 3 for i in range(B)]
    c = cache(lengths, 4, 64)
    c.k[:] = 0x22                                    # ones
    c.k_scale[:] = 127
    c.v_scale[..., 1] = 90
    q = torch.full((B, T, 8, 64), -float(size), device="cuda").bfloat16()
    o, lse = jm.paged_attention(q, c, torch.tensor(lengths, dtype=torch.int32, device="cuda"), return_lse=True)
    # logits are -8 size, exactly, so that all weights of a row are the same
    values = po.held_values(c.v, c.v_scale).repeat_interleave(2, 2)
    for b, length in enumerate(lengths):
        v = values[at(c, b, list(range(length)))]
        for t in range(T):
            end = length - T + t + 1
            assert ((o[b, t].double() - v[:end].mean(0)).abs() <= (2.0 ** -11 + 2.0 ** -17) * v[:end].abs().mean(0)).all()
            assert ((lse[b, :, t].double() + 8 * size - math.log(end)).abs() <= 2.0 ** -22 * 8 * size + 2.0 ** -17).all()


def test_an_appended_infinity():
    """It is kept as 6 * 2^126: where its weight is small enough the result is finite."""
    n = 64
    c = jm.PagedCache.empty(4, 16, 1, 32, torch.arange(4, dtype=torch.int32, device="cuda")[None], "4bit")
    k, v = torch.zeros((1, n, 1, 32), device="cuda"), torch.ones((1, n, 1, 32), device="cuda")
    k[0, 20] = -6                                    # a logit of -480 / sqrt(32), a weight of 2^-122
    v[0, 20, 0, 3] = torch.inf
    jm.append_kv(c, k, v, torch.tensor([n], dtype=torch.int32, device="cuda"))
    q = torch.full((1, 1, 1, 32), 2.5, device="cuda", dtype=torch.bfloat16)
    check(q, c, [n], False)


def test_a_head_of_zeros_is_ordinary():
    """Heads and groups of zeros have the least power, which changes nothing but rounding."""
    lengths = [500]
    c = cache(lengths, 2, 128)
    heads, groups = at(c, 0, list(range(0, 500, 7))), at(c, 0, list(range(3, 500, 5)))
    c.v[heads] = 0
    c.v[groups[0], groups[1], :, 16:32] = 0
    q = queries(1, 2, 4, 128)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    want = jm.paged_attention(q, c, n)
    c.v_scale[heads] = 0
    c.v_scale[groups[0], groups[1], :, 1] = 0
    assert (jm.paged_attention(q, c, n) - want).abs().max() <= 2.0 ** -10 * want.abs().max()
    check(q, c, lengths, False)
