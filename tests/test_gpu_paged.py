"""The paged cache: append_kv, read_kv and paged_attention against their definitions in float64, and a run of all of them together.

Tolerances of attention, per component, in units of sum p |v| (what the weights could sum to): float32 sums and exponentials 2^-17 over contexts of these
lengths; the weights of bfloat16 and 4-bit caches are rounded to 16 bits before the product with the values, off by half a step of bfloat16, 2^-8, at most;
a bfloat16 result by 2^-8 of itself.  The log-sum-exp has the error of a logit, 128 products in float32 of which each sums to about 8: 2^-24 * 128 * 8 at worst.
float32 results as a whole: 2e-6 in the 2-norm, as for the other float32 calls.

A 4-bit cache's weights go through float16 as w = p 2^E / max p 2^E, 2^E the largest power of two of the key's value, times 2^15: 2^-12 of themselves down to
w = 2^-29, and below, where float16 has steps of 2^-24, off by at most 2^-25 2^-15 = 2^-40.  Each of the n keys adds that times max p 2^E <= max 2^E times a value of
at most 6 in units of 2^E: n 6 2^-40 max 2^E in all, which is seen where the keys of large weight have a code of 0 in a component."""
import pytest
import torch

import jaxmodules_b200 as jm
from jaxmodules_b200 import _native as nat, attention as A
from oracle import paged_oracle as po

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
KINDS = {"bf16": BF16, "f32": F32, "4bit": "4bit"}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def make(kind, lengths, H, d, page, seed=0, spare=2, order="shuffled", fill=True):
    """A cache with random content, and entries of the table that no position reaches out of range."""
    g = gen(seed)
    B = len(lengths)
    width = max(1, max(-(-n // page) for n in lengths))
    need = [-(-n // page) for n in lengths]
    pages = sum(need) + spare
    perm = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).int()
    table = torch.full((B, width), 1 << 30, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    c = jm.PagedCache.empty(pages, page, H, d, table.cuda(), KINDS[kind])
    if fill:
        for name in ("k", "v"):
            x = torch.randn((pages, page, H, d), device="cuda", generator=g)
            if kind == "4bit":
                getattr(c, name).copy_(torch.randint(0, 256, c.k.shape, device="cuda", generator=g, dtype=torch.uint8))
                getattr(c, name + "_scale").copy_(torch.randint(123, 128, c.k_scale.shape, device="cuda", generator=g, dtype=torch.uint8))
            else:
                getattr(c, name).copy_(x)
    return c


def causal_from(first):
    return lambda b, h, i, j: j <= i + first


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def contexts(c, lengths):
    page = c.k.shape[1]
    return [[po.context(po.held_values(x, s), c.page_table, b, n, page) for b, n in enumerate(lengths)] for x, s in ((c.k, c.k_scale), (c.v, c.v_scale))]


def check(q, c, lengths, new=None, **kw):
    B, T = q.shape[:2]
    out_dtype = kw.pop("out_dtype", None)
    o, lse = jm.paged_attention(q, c, ints(lengths), new_lengths=None if new is None else ints(new), return_lse=True, out_dtype=out_dtype, **kw)
    want, want_lse, size = po.attend(q.double(), *contexts(c, lengths), lengths, [T] * B if new is None else new, **kw)
    assert o.dtype == (out_dtype or F32) and o.shape == q.shape and lse.shape == (B, q.shape[2], T)
    slack = 2.0 ** -17 if c.k.dtype == F32 else 2.0 ** -8 + 2.0 ** -17
    off = (o.double() - want).abs()
    bound = slack * size + (2.0 ** -8 * want.abs() if o.dtype == BF16 else 0)
    if c.v_scale is not None:
        bound = bound + 6 * max(lengths) * 2.0 ** (int(c.v_scale.max()) - 127 - 40)
    assert o.isfinite().all() and (off <= bound + 1e-30).all(), (off / (bound + 1e-30)).max()
    if c.k.dtype == F32 and o.dtype == F32:
        assert (o.double() - want).norm() <= 2e-6 * want.norm()
    empty = want_lse == -torch.inf
    assert torch.equal(lse == -torch.inf, empty) and (torch.where(empty, 0, lse.double() - want_lse).abs() <= 128 * 8 * 2.0 ** -24).all()
    assert not o.permute(0, 2, 1, 3)[empty].any()
    assert A.device_status() == 0
    return o


def queries(B, T, H, d, kind, seed=1):
    return torch.randn((B, T, H, d), device="cuda", generator=gen(seed)).to(F32 if kind == "f32" else BF16)


# lengths, T, Hq, Hkv, d, page
ATTEND = [
    ([1], 1, 1, 1, 64, 16),
    ([15, 16, 17, 0, 1], 1, 4, 2, 128, 16),
    ([100, 3, 64, 65, 129, 1, 31, 32, 33], 1, 8, 2, 64, 8),
    ([1000, 250, 77], 1, 32, 4, 128, 16),
    ([300, 299], 1, 12, 1, 128, 7),               # pages that end inside every tile
    ([300, 511, 5], 3, 8, 2, 128, 64),
    ([130, 40], 7, 16, 2, 64, 16),                # 56 rows to a kv head
    ([40, 64, 9], 5, 7, 1, 128, 16),              # 35 rows
    ([260, 20], 1, 64, 1, 128, 32),               # 64 query heads to one
    ([90, 17], 1, 3, 3, 96, 16),
    ([90, 17], 2, 4, 2, 32, 1),                   # one token to a page
    ([5000, 4097], 1, 8, 8, 128, 128),
    ([20000], 1, 16, 2, 128, 16),
    ([20000], 2, 4, 1, 64, 256),
    ([33], 33, 4, 1, 64, 16),                     # a whole prompt
    (list(range(0, 480, 8)), 1, 8, 4, 128, 16),   # many sequences: four kv heads to a CTA
    (list(range(1, 400, 6)), 3, 4, 2, 64, 16),    # two kv heads
    (list(range(1, 300, 5)) + [9000], 2, 32, 8, 128, 16),      # a long one among them
    ([i * 7 % 50 for i in range(300)], 1, 4, 2, 64, 16),       # more sequences than a CTA has threads
    ([i * 13 % 90 for i in range(700)] + [3000], 1, 6, 3, 64, 16),
]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("case", ATTEND, ids=lambda c: f"{min(c[0])}..{max(c[0])}x{len(c[0])}-" + "-".join(map(str, c[1:])))
def test_attention(case, kind):
    lengths, T, Hq, Hkv, d, page = case
    lengths = [max(n, T) if n else 0 for n in lengths]
    new = [T if n else 0 for n in lengths]
    c = make(kind, lengths, Hkv, d, page, seed=len(lengths) + T)
    check(queries(len(lengths), T, Hq, d, kind), c, lengths, new)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T,Hq,Hkv,d", [(1, 4, 2, 64), (2, 6, 1, 128)])
@pytest.mark.parametrize("long", [400, 3000, 20000])
def test_a_long_sequence_among_many_short_ones(long, T, Hq, Hkv, d, kind):
    """Its walk is cut into 7 to 280 parts, those of the others into one or two."""
    lengths = [T + i * 5 % 40 for i in range(230)]
    lengths[101] = long
    check(queries(len(lengths), T, Hq, d, kind), make(kind, lengths, Hkv, d, 16, seed=long), lengths)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("d", [8, 40, 72, 120])
def test_head_dimensions(d, kind):
    lengths = [77, 300]
    check(queries(2, 2, 6, d, kind), make(kind, lengths, 3, d, 16, seed=d), lengths)


def test_4bit_powers_far_apart():
    """Powers of two from 2^-30 to 2^20 in one head, and a head of zeros: codes under 2^-24 of the head's largest may be dropped, 6 * 2^-25 of the largest power at
    most, of weights that sum to one."""
    lengths = [200, 64]
    c = make("4bit", lengths, 2, 128, 16, seed=5)
    for s in (c.k_scale, c.v_scale):
        s.copy_(torch.randint(97, 148, s.shape, device="cuda", generator=gen(3), dtype=torch.uint8))
    c.k_scale.clamp_(max=124)
    c.v[0], c.v_scale[0] = 0, 0
    q = queries(2, 2, 4, 128, "4bit")
    o, lse = jm.paged_attention(q, c, ints(lengths), return_lse=True)
    want, want_lse, size = po.attend(q.double(), *contexts(c, lengths), lengths, [2, 2])
    assert ((o.double() - want).abs() <= (2.0 ** -8 + 2.0 ** -17) * size + 6 * 2.0 ** (20 - 25) + 6 * 200 * 2.0 ** (20 - 40)).all()
    assert (lse.double() - want_lse).abs().max() <= 128 * 8 * 2.0 ** -24 * 4


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window", [0, 1, 15, 16, 100, 10 ** 9])
@pytest.mark.parametrize("T", [1, 4])
def test_window(window, T, kind):
    lengths = [1000, 64, 65, 4]
    c = make(kind, lengths, 2, 64, 16, seed=window % 1000)
    check(queries(4, T, 6, 64, kind), c, lengths, window=window)


@pytest.mark.parametrize("kind", KINDS)
def test_padded_batch(kind):
    """Fewer real tokens than given, none, more than there are, negative counts: zeros, nothing out of range."""
    lengths, new = [50, 20, 3, 0, 7], [3, 0, 3, 0, 1]
    c = make(kind, lengths, 2, 128, 16)
    check(queries(5, 4, 8, 128, kind), c, lengths, new)
    q = queries(5, 4, 8, 128, kind)
    a = jm.paged_attention(q, c, ints(lengths), new_lengths=ints([3, -5, 3, 0, 1]))
    assert torch.equal(a, jm.paged_attention(q, c, ints(lengths), new_lengths=ints(new)))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
def test_scale_and_out_dtype(scale, kind):
    lengths = [70, 300]
    c = make(kind, lengths, 2, 64, 16)
    q = queries(2, 2, 4, 64, kind) / (4 if abs(scale) == 2 else 1)
    for dtype in (None, BF16):
        check(q, c, lengths, scale=scale, out_dtype=dtype)


@pytest.mark.parametrize("kind", KINDS)
def test_large_logits(kind):
    """Weights that underflow all but at the largest logit, which comes last, first, and in the middle."""
    lengths = [600, 600, 600]
    c = make(kind, lengths, 1, 64, 16)
    q = queries(3, 1, 2, 64, kind)
    for b, at in enumerate((599, 0, 300)):
        page, slot = c.page_table[b, at // 16], at % 16
        if kind == "4bit":
            c.k_scale[page, slot] = 127 + 6
        else:
            c.k[page, slot] *= 100
    o = check(q, c, lengths)
    assert o.isfinite().all()


@pytest.mark.parametrize("kind", KINDS)
def test_what_lies_outside_reaches_nothing(kind):
    """NaN and infinities behind the length, before the window, after a row's token, in pages of nobody: the bits without them."""
    lengths, T, window = [77, 40, 200], 3, 20
    c = make(kind, lengths, 2, 64, 16, seed=3)
    q = queries(3, T, 4, 64, kind)
    clean = jm.paged_attention(q, c, ints(lengths), window=window)
    dirty = jm.PagedCache(c.k.clone(), c.v.clone(), c.page_table, *(None if s is None else s.clone() for s in (c.k_scale, c.v_scale)))
    seen = torch.zeros(c.k.shape[:2], dtype=torch.bool, device="cuda")
    for b, n in enumerate(lengths):
        at = torch.arange(max(0, n - T - window), n, device="cuda")
        seen[c.page_table[b].long()[at // 16], at % 16] = True
    for name in ("k", "v"):
        if kind == "4bit":
            getattr(dirty, name + "_scale")[~seen] = 255
        else:
            getattr(dirty, name)[~seen] = torch.nan if name == "k" else torch.inf
    assert torch.equal(clean, jm.paged_attention(q, dirty, ints(lengths), window=window))
    # the last token's: rows of the tokens before keep their bits, its own row is not finite
    last = c.page_table[0, 76 // 16], 76 % 16
    if kind == "4bit":
        dirty.v_scale[last] = 255
    else:
        dirty.v[last] = torch.inf
    o = jm.paged_attention(q, dirty, ints(lengths), window=window)
    assert torch.equal(o[0, :2], clean[0, :2]) and torch.equal(o[1:], clean[1:]) and not o[0, 2].isfinite().any()
    # the first key of the first row's window: only that row sees it
    first = c.page_table[0, (74 - 20) // 16], (74 - 20) % 16
    if kind == "4bit":
        dirty.v_scale[last], dirty.v_scale[first] = c.v_scale[last], 255
    else:
        dirty.v[last], dirty.v[first] = c.v[last], torch.nan
    o = jm.paged_attention(q, dirty, ints(lengths), window=window)
    assert torch.equal(o[0, 1:], clean[0, 1:]) and o[0, 0].isnan().all()


@pytest.mark.parametrize("kind", KINDS)
def test_layouts(kind):
    """Heads before slots, pages that are part of larger ones, queries of [B, H, T, d], wide tables: the bits of the plain layout."""
    lengths = [100, 33]
    c = make(kind, lengths, 2, 64, 16)
    q = queries(2, 3, 4, 64, kind)
    want = jm.paged_attention(q, c, ints(lengths))
    turned = lambda x: None if x is None else x.transpose(1, 2).contiguous().transpose(1, 2)
    part = lambda x: None if x is None else torch.cat((x, x), 2)[:, :, 2:]
    for how in (turned, part):
        other = jm.PagedCache(how(c.k), how(c.v), torch.cat((c.page_table, c.page_table), 1)[:, :c.page_table.shape[1]],
                              *(how(s) for s in (c.k_scale, c.v_scale)))
        assert torch.equal(want, jm.paged_attention(q.transpose(1, 2).contiguous().transpose(1, 2), other, ints(lengths)))
        assert all(torch.equal(a, b) for a, b in zip(jm.read_kv(other, ints(lengths), 100), jm.read_kv(c, ints(lengths), 100)))


@pytest.mark.parametrize("kind", KINDS)
def test_bad_pages(kind):
    """Pages outside the cache and positions outside the table: nothing is read or written there, and the status word says so."""
    lengths = [40, 40]
    c = make(kind, lengths, 1, 64, 16)
    q = queries(2, 1, 2, 64, kind)
    kv = torch.ones((2, 1, 1, 64), device="cuda", dtype=q.dtype)
    good = jm.paged_attention(q, c, ints(lengths))
    for bad in (-1, c.k.shape[0], -(1 << 31), (1 << 31) - 1):
        t = c.page_table.clone()
        t[1, 2] = bad
        other = jm.PagedCache(c.k, c.v, t, c.k_scale, c.v_scale)
        o = jm.paged_attention(q, other, ints(lengths))
        assert torch.equal(o[0], good[0]) and A.device_status() == 803
        held = c.k.clone(), c.v.clone()
        jm.append_kv(other, kv, kv, ints([0, 41]), new_lengths=ints([0, 1]))
        assert torch.equal(c.k, held[0]) and torch.equal(c.v, held[1]) and A.device_status() == 801
        k, v = jm.read_kv(other, ints(lengths), 45)
        assert not k[1, 32:].any() and not v[1, 32:].any() and A.device_status() == 802
    o = jm.paged_attention(q, c, ints([40, 1000]))                  # longer than the table
    assert torch.equal(o[0], good[0]) and A.device_status() == 803
    jm.append_kv(c, kv, kv, ints([0, 1000]), new_lengths=ints([0, 1]))
    assert A.device_status() == 801
    jm.append_kv(c, kv, kv, ints([0, 0]), new_lengths=ints([0, 1]))  # before the first position
    assert A.device_status() == 801 and torch.equal(c.k, held[0])


# kind, input dtype, T, Hq, Hkv, d, page, layout, norm, dim
APPEND = [
    ("bf16", BF16, 1, 8, 2, 128, 16, "half", True, 128),
    ("f32", F32, 1, 0, 1, 64, 16, "half", False, 64),
    ("4bit", BF16, 1, 8, 2, 128, 16, "half", True, 128),
    ("4bit", F32, 5, 4, 2, 32, 3, "half", False, 32),
    ("4bit", BF16, 40, 0, 3, 96, 16, "interleaved", True, 96),
    ("4bit", F32, 9, 3, 1, 128, 16, "half", True, 36),
    ("4bit", BF16, 9, 3, 1, 64, 16, "interleaved", True, 20),
    ("bf16", BF16, 40, 4, 4, 72, 16, "half", True, 36),
    ("bf16", BF16, 7, 0, 1, 8, 1, "half", False, 0),
    ("f32", F32, 33, 2, 2, 40, 5, "interleaved", True, 20),
]


@pytest.mark.parametrize("case", APPEND, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_append(case):
    """Rotated keys within the tolerances of rotate_heads; values as they are; 4 bits: within half a step, where the float64 value is no nearer to a border
    than float32 leaves it (2^-18) the very code; everything else in the cache untouched."""
    kind, dtype, T, Hq, Hkv, d, page, layout, norm, dim = case
    lengths, new = [T + 13, T, 2 * T + 1, 0, T + 3], [T, T, max(1, T // 2), 0, 0]
    c = make(kind, lengths, Hkv, d, page, seed=T + d)
    g = gen(T)
    randn = lambda *s: torch.randn(s, device="cuda", generator=g).to(dtype)
    k, v, q = randn(5, T, Hkv, d), randn(5, T, Hkv, d), randn(5, T, Hq, d) if Hq else None
    qw, kw = (1 + randn(d) / 4, 1 + randn(d) / 4) if norm else (None, None)
    f = jm.rotary_frequencies(dim) if dim else None
    before = [po.held_values(x, s).clone() for x, s in ((c.k, c.k_scale), (c.v, c.v_scale))]
    raw = [x.clone() for x in (c.k, c.v)]
    out = jm.append_kv(c, k, v, ints(lengths), new_lengths=ints(new), q=q, frequencies=f, layout=layout, q_weight=qw if Hq else None, k_weight=kw, magnitude=0.75)
    after = [po.held_values(x, s) for x, s in ((c.k, c.k_scale), (c.v, c.v_scale))]
    written = torch.zeros(c.k.shape[:2], dtype=torch.bool, device="cuda")
    for b, (n, t) in enumerate(zip(lengths, new)):
        at = torch.arange(n - t, n, device="cuda")
        where = c.page_table[b].long()[at // page], at % page
        written[where] = True
        for x, got, w in ((k, after[0][where], kw), (v, after[1][where], None)):
            want = x[b, :t].double()
            if x is k:
                want = po.rotate(want, at[:, None], f, layout, 0.75, None if w is None else w.double())
            if not t:
                continue
            if kind == "4bit":
                exact, byte = po.to_4bit(want)
                step = torch.exp2(byte.double() - 127).repeat_interleave(32, -1)
                assert ((got - want).abs() <= step * (1 + 2.0 ** -15)).all()              # half of the widest step, 4 to 6
                differ = got != exact
                if x is v:
                    assert not differ.any()
                else:
                    assert differ.double().mean() <= 1e-3
            else:
                half = 2.0 ** -8 if kind == "bf16" else 2.0 ** -24
                if x is v:
                    assert torch.equal(got, want)
                else:
                    assert ((got - want).abs() <= half * want.abs() + 2.0 ** -18 * want.abs().amax(-1, keepdim=True)).all()
        if Hq:
            want = po.rotate(q[b, :t].double(), at[:, None], f, layout, 0.75, None if qw is None else qw.double())
            half = 2.0 ** -8 if dtype == BF16 else 2.0 ** -24
            if t:
                assert ((out[b, :t].double() - want).abs() <= half * want.abs() + 2.0 ** -18 * want.abs().amax(-1, keepdim=True)).all()
            assert not out[b, t:].any()
    assert out is None or Hq
    for x, r in zip((c.k, c.v), raw):
        assert torch.equal(x[~written], r[~written])
    for a, b in zip(after, before):
        assert torch.equal(a[~written].nan_to_num(0), b[~written].nan_to_num(0))
    assert A.device_status() == 0


def test_append_is_rotate_heads():
    """The same bits as rotate_heads at the same positions."""
    c = make("bf16", [90, 80], 2, 128, 16)
    g = gen(0)
    q, k = (torch.randn((2, 80, h, 128), device="cuda", generator=g).to(BF16) for h in (4, 2))
    w = torch.rand(128, device="cuda") + 0.5
    f = jm.rotary_frequencies(128)
    positions = torch.stack((torch.arange(10, 90), torch.arange(80))).cuda()
    want = jm.rotate_heads(q, k, positions, f, q_weight=w, k_weight=w)
    out = jm.append_kv(c, k, k, ints([90, 80]), q=q, frequencies=f, q_weight=w, k_weight=w)
    ks, vs = jm.read_kv(c, ints([90, 80]), 90)
    assert torch.equal(out, want[0]) and torch.equal(ks[0, 10:], want[1][0]) and torch.equal(ks[1, :80], want[1][1]) and torch.equal(vs[0, 10:], k[0])


def test_4bit_special_values():
    c = make("4bit", [4], 1, 64, 4, fill=False)
    x = torch.randn((1, 4, 1, 64), device="cuda")
    x[0, 0, 0, 0], x[0, 1, 0, 0], x[0, 1, 0, 1] = torch.nan, torch.inf, -torch.inf
    x[0, 2] = 0
    x[0, 3, 0, :32] = 1e-42          # below 2^-127 * 0.25: zeros
    x[0, 3, 0, 32:] = 3e38
    jm.append_kv(c, x, x, ints([4]))
    k, _ = jm.read_kv(c, ints([4]), 4)
    assert k[0, 0, 0, :32].isnan().all() and torch.equal(k[0, 0, 0, 32:].double(), po.to_4bit(x[0, 0, 0].double())[0][32:])
    assert k[0, 1, 0, 0] == 6 * 2.0 ** 126 and k[0, 1, 0, 1] == -6 * 2.0 ** 126 and not k[0, 1, 0, 2:32].any()
    assert not k[0, 2].any() and not k[0, 3, 0, :32].any() and (k[0, 3, 0, 32:] == 4 * 2.0 ** 126).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H,d,page", [(2, 128, 16), (1, 64, 5), (8, 128, 64), (3, 32, 1)])
def test_read(H, d, page, kind):
    lengths = [37, 0, 1, 64]
    c = make(kind, lengths, H, d, page, seed=d)
    ks, vs = contexts(c, lengths)
    for L in (1, 40, 64, 100):
        k, v = jm.read_kv(c, ints(lengths), L)
        assert k.shape == (4, L, H, d) and k.dtype == (F32 if kind == "f32" else BF16)
        for b, n in enumerate(lengths):
            m = min(n, L)
            assert torch.equal(k[b, :m].double(), ks[b][:m]) and torch.equal(v[b, :m].double(), vs[b][:m]) and not k[b, m:].any() and not v[b, m:].any()


@pytest.mark.parametrize("kind", KINDS)
def test_prompt_and_decoding_together(kind):
    """A model's two layers: the prompts in chunks through read_kv and masked_attention_via_map, then token by token through the cache; every row against
    attention in float64 over the whole context of the keys and values that the cache holds."""
    B, Hq, Hkv, d, page, layers = 2, 4, 2, 64, 16, 2
    prompt, chunk, steps = [50, 33], 25, 4
    dtype = F32 if kind == "f32" else BF16
    f = jm.rotary_frequencies(d)
    g = gen(7)
    total = max(prompt) + steps
    width = -(-total // page)
    table = torch.randperm(B * width, generator=torch.Generator().manual_seed(0)).int().reshape(B, width).cuda()
    caches = [jm.PagedCache.empty(B * width, page, Hkv, d, table, KINDS[kind]) for _ in range(layers)]
    randn = lambda *s: torch.randn(s, device="cuda", generator=g).to(dtype)
    qw, kw = 1 + randn(d) / 8, 1 + randn(d) / 8
    rows = [[[None] * total for _ in range(B)] for _ in range(layers)]
    asked = [[[None] * total for _ in range(B)] for _ in range(layers)]
    for start in list(range(0, max(prompt), chunk)):
        new = [max(0, min(chunk, n - start)) for n in prompt]
        lengths = [min(n, start + chunk) for n in prompt]
        for i, c in enumerate(caches):
            q = jm.append_kv(c, randn(B, chunk, Hkv, d), randn(B, chunk, Hkv, d), ints(lengths), new_lengths=ints(new), q=randn(B, chunk, Hq, d), frequencies=f,
                             q_weight=qw, k_weight=kw)
            k, v = jm.read_kv(c, ints(lengths), max(lengths))
            for b in range(B):
                if not new[b]:
                    continue
                first = lengths[b] - new[b]
                o = jm.masked_attention_via_map(q[b:b + 1, :new[b]], k[b:b + 1, :lengths[b]], v[b:b + 1, :lengths[b]],
                                                mask_fn=causal_from(first), block_size=1)
                for t in range(new[b]):
                    rows[i][b][first + t], asked[i][b][first + t] = o[0, t], q[b, t]
    lengths = ints(prompt)
    for _ in range(steps):
        lengths += 1
        for i, c in enumerate(caches):
            q = jm.append_kv(c, randn(B, 1, Hkv, d), randn(B, 1, Hkv, d), lengths, q=randn(B, 1, Hq, d), frequencies=f, q_weight=qw, k_weight=kw)
            o = jm.paged_attention(q, c, lengths)
            for b, n in enumerate(lengths.tolist()):
                rows[i][b][n - 1], asked[i][b][n - 1] = o[b, 0], q[b, 0]
    for i, c in enumerate(caches):
        n = lengths.tolist()
        ks, vs = contexts(c, n)
        for b in range(B):
            q = torch.stack(asked[i][b][:n[b]])[None].double()
            want, _, size = po.attend(q, [ks[b]], [vs[b]], [n[b]], [n[b]])
            off = (torch.stack(rows[i][b][:n[b]])[None].double() - want).abs()
            assert (off <= (2.0 ** -17 if kind == "f32" else 2.0 ** -7) * size + 1e-30).all()
    assert A.device_status() == 0


@pytest.mark.parametrize("kind", KINDS)
def test_decoding_step_captured(kind):
    """A captured step replayed as the sequences grow, two graphs of one pool at work in turn, and a call on another stream: the bits of eager calls."""
    lengths = ints([30, 100])
    c = make(kind, [60, 130], 2, 64, 16)
    f = jm.rotary_frequencies(64)
    q, k, v = queries(2, 1, 8, 64, kind), queries(2, 1, 2, 64, kind, 2), queries(2, 1, 2, 64, kind, 3)

    def step():
        lengths.add_(1)
        return jm.paged_attention(jm.append_kv(c, k, v, lengths, q=q, frequencies=f), c, lengths)

    step()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            outs.append(step())
        graphs.append(graph)
    state = [x.clone() for x in (lengths, c.k, c.v)]
    got = []
    for i in (0, 1, 1, 0):
        graphs[i].replay()
        got.append(outs[i].clone())
    for x, s in zip((lengths, c.k, c.v), state):
        x.copy_(s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [step() for _ in range(4)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_calls_at_once_on_two_streams():
    """Workspaces are a call's own."""
    lengths = [3000, 1500]
    c = make("bf16", lengths, 2, 128, 16)
    qs = [queries(2, 1, 8, 128, "bf16", s) for s in range(2)]
    want = [jm.paged_attention(q, c, ints(lengths)) for q in qs]
    n = ints(lengths)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(jm.paged_attention(qs[i], c, n))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])


def test_a_long_cache():
    """Offsets beyond 2^31 values and 2^32 bytes: the last pages of a cache of 5.4 GB."""
    page, H, d = 16, 8, 128
    pages = (1 << 31) // (page * H * d) + 100
    table = torch.arange(pages - 64, pages, dtype=torch.int32, device="cuda")[None]
    c = jm.PagedCache(*(torch.empty((pages, page, H, d), device="cuda", dtype=BF16) for _ in range(2)), table)
    for x in (c.k, c.v):
        x[-64:] = torch.randn((64, page, H, d), device="cuda", generator=gen(1)).to(BF16)
    check(queries(1, 1, 8, d, "bf16"), c, [1000])
    jm.append_kv(c, torch.ones((1, 1, H, d), device="cuda", dtype=BF16), torch.ones((1, 1, H, d), device="cuda", dtype=BF16), ints([1024]))
    assert (c.k[-1, -1] == 1).all() and (c.v[-1, -1] == 1).all()
    k, _ = jm.read_kv(c, ints([1024]), 1024)
    assert torch.equal(k[0], c.k[-64:].reshape(1024, H, d))
