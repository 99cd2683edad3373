"""rotate_heads against its definition in float64.

Tolerances.  Everything is float32 until one rounding at the end.  Cosine and sine are off by at most 2^-22 (a phase of 32 bits, sincospi), the norm by
2^-21 of the value (a sum of at most 256 squares over lanes, rsqrt, two products), a pair's sum of two products by another 2^-22 of |a| + |b|: together less
than 2^-19 of |a| + |b|; a bfloat16 result is off by half a step more, 2^-8 of it.  The gradient of x has one more product and a mean of as many terms,
all at most |g w| inv + |x^| mean|g w x^| inv in magnitude: 2^-18 of that.  The gradients of the weights add n = tokens * heads terms with at most n / 4 of them
in one chain: 2^-18 + n 2^-26 of the sum of their magnitudes."""
import pytest
import torch

import jaxmodules_b200 as jm
from jaxmodules_b200 import _native as nat
from oracle import paged_oracle as po

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def close(got, want, size, slack):
    half = 2.0 ** -8 if got.dtype == BF16 else 2.0 ** -24
    off = (got.double() - want).abs()
    assert (off <= half * want.abs() + slack * size + 1e-30).all(), (off / (half * want.abs() + slack * size + 1e-30)).max()


def inputs(seed, B, L, Hq, Hkv, d, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(s, device="cuda", generator=g).to(dtype)
    return randn(B, L, Hq, d), randn(B, L, Hkv, d), 1 + randn(d) / 4, 1 + randn(d) / 4, randn(B, L, Hq, d), randn(B, L, Hkv, d)


def pair_sizes(x, frequencies, layout):
    """|a| + |b| of the pair that each component belongs to."""
    if frequencies is None:
        return x.abs()
    n = frequencies.numel()
    one = torch.arange(n) if layout == "half" else 2 * torch.arange(n)
    two = one + n if layout == "half" else one + 1
    out = x.abs().clone()
    out[..., one] = out[..., two] = x[..., one].abs() + x[..., two].abs()
    return out


CASES = [
    # B, L, Hq, Hkv, d, dim, layout, norm
    (2, 5, 4, 2, 128, 128, "half", True),
    (1, 1, 1, 1, 64, 64, "half", True),
    (3, 7, 8, 1, 128, 64, "half", False),
    (1, 33, 6, 2, 96, 96, "half", True),
    (2, 4, 5, 3, 80, 80, "half", True),
    (1, 9, 3, 3, 72, 36, "half", True),          # halves in the middle of 16-byte chunks
    (2, 3, 2, 2, 64, 32, "interleaved", True),
    (1, 6, 4, 4, 40, 20, "interleaved", True),    # ends in the middle of a chunk
    (1, 5, 2, 1, 256, 256, "half", True),
    (1, 4, 2, 1, 256, 100, "interleaved", False),
    (2, 3, 2, 1, 6, 4, "half", True),
    (1, 3, 2, 1, 7, 2, "interleaved", True),      # an odd head
    (1, 3, 2, 1, 1, 0, "half", True),
    (2, 300, 3, 1, 128, 0, "half", True),         # a norm alone
    (1, 2000, 32, 8, 128, 128, "half", True),
]


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_values_and_gradients(case, dtype):
    B, L, Hq, Hkv, d, dim, layout, norm = case
    q, k, qw, kw, gq, gk = inputs(sum(case[:6]), B, L, Hq, Hkv, d, dtype)
    f = jm.rotary_frequencies(dim) if dim else None
    positions = torch.randint(0, 1 << 20, (B, L), device="cuda")
    leaves = [t.requires_grad_(True) for t in ((q, k, qw, kw) if norm else (q, k))]
    out = jm.rotate_heads(q, k, positions, f, layout=layout, q_weight=qw if norm else None, k_weight=kw if norm else None, magnitude=1.25)
    grads = torch.autograd.grad(out, leaves, [gq, gk])
    exact = [t.detach().double().requires_grad_(True) for t in leaves]
    for i, (x, g) in enumerate(((q, gq), (k, gk))):
        w = exact[2 + i] if norm else None
        y = po.rotate(exact[i], positions[..., None], f, layout, 1.25, w)
        h = exact[i].detach()
        if norm:
            h = h / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-6)
        size = pair_sizes(h * w.detach() if norm else h, f, layout) * 1.25
        close(out[i], y.detach(), size, 2.0 ** -19)
        assert out[i].shape == x.shape and out[i].dtype == dtype and out[i].is_contiguous()
        dx, *dw = torch.autograd.grad(y, [exact[i]] + ([w] if norm else []), g.double())
        size = pair_sizes(g.double(), f, layout) * 1.25
        if norm:
            inv = 1 / torch.sqrt((exact[i].detach() ** 2).mean(-1, keepdim=True) + 1e-6)
            back = po.rotate(g.double(), -positions[..., None], f, layout, 1.25)
            close(grads[2 + i], dw[0], (size * h.abs()).sum((0, 1, 2)), 2.0 ** -18 + B * L * x.shape[2] * 2.0 ** -26)
            assert torch.allclose(dw[0], (back * h).sum((0, 1, 2)), rtol=1e-9, atol=1e-9)
            gws = size * w.detach().abs()
            size = inv * (gws + h.abs() * (gws * h.abs()).mean(-1, keepdim=True))
        close(grads[i], dx, size, 2.0 ** -18)


def test_gradients_against_differences():
    """Directional differences in float32: a step of 2^-9 leaves 2^-18 of curvature and 2^-24 / 2^-9 of rounding, of a sum of 2 * 48 terms of order 1."""
    q, k, qw, kw, gq, gk = inputs(3, 1, 2, 1, 1, 48, F32)
    f = jm.rotary_frequencies(48)
    leaves = [t.requires_grad_(True) for t in (q, k, qw, kw)]
    call = lambda *x: jm.rotate_heads(x[0], x[1], None, f, q_weight=x[2], k_weight=x[3])
    grads = torch.autograd.grad(call(*leaves), leaves, [gq, gk])
    for i, (leaf, grad) in enumerate(zip(leaves, grads)):
        way = torch.randn(leaf.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(i))
        moved = [[t.detach() + (sign * 2.0 ** -9 * way if j == i else 0) for j, t in enumerate(leaves)] for sign in (1, -1)]
        (qa, ka), (qb, kb) = (call(*m) for m in moved)
        slope = (((qa - qb).double() * gq).sum() + ((ka - kb).double() * gk).sum()) / 2.0 ** -8
        assert abs(slope - (grad.double() * way).sum()) <= 4e-3 * grad.double().norm() * way.norm() / 8


@pytest.mark.parametrize("kind", ["int32", "one row", "none", "expanded"])
def test_positions(kind):
    q, k, *_ = inputs(5, 2, 11, 2, 1, 64, F32)
    f = jm.rotary_frequencies(64)
    positions = {"int32": torch.randint(-100, 1 << 30, (2, 11), device="cuda", dtype=torch.int32), "one row": torch.arange(7, 18, device="cuda"),
                 "none": None, "expanded": torch.tensor([[3], [1 << 25]], device="cuda").expand(2, 11)}[kind]
    out = jm.rotate_heads(q, k, positions, f)
    at = torch.arange(11, device="cuda") if positions is None else positions
    for got, x in zip(out, (q, k)):
        want = po.rotate(x.double(), at.expand(2, 11)[..., None], f)
        # (beyond 2^25 the oracle's own float64 angle is off by up to 2^30 * 2^-53 of a radian: nothing next to 2^-19)
        close(got, want, pair_sizes(x.double(), f, "half"), 2.0 ** -19)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_strides_and_alignment(dtype):
    """Views of one projection, [B, H, L, d] storage, rows that no 16-byte access fits, components that lie apart: the bits of contiguous tensors (the sum of
    squares of narrow accesses is taken in another order: 2^-19)."""
    B, L, Hq, Hkv, d = 2, 9, 4, 2, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    f = jm.rotary_frequencies(d)
    qkv = torch.randn((B, L, Hq + 2 * Hkv, d), device="cuda", generator=g).to(dtype)
    q, k = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hkv]
    qw = torch.rand(d, device="cuda", generator=g) + 0.5
    want = jm.rotate_heads(q.contiguous(), k.contiguous(), None, f, q_weight=qw, k_weight=qw)
    odd = torch.zeros((B, L, Hq, d + 1), device="cuda", dtype=dtype)
    odd[..., 1:] = q
    views = {"projection": (q, True), "heads first": (q.transpose(1, 2).contiguous().transpose(1, 2), True), "odd": (odd[..., 1:], False),
             "apart": (q.transpose(2, 3).contiguous().transpose(2, 3), True)}
    for name, (view, same) in views.items():
        got = jm.rotate_heads(view, k, None, f, q_weight=qw, k_weight=qw)
        for a, b in zip(got, want):
            assert torch.equal(a, b) if same else ((a.double() - b.double()).abs() <= (2.0 ** -7 if dtype == BF16 else 2.0 ** -19) * (b.abs() + b.abs().amax())).all(), name
    # cotangents that are expanded, and of one side only
    x = q.contiguous().requires_grad_(True)
    y, _ = jm.rotate_heads(x, k, None, f, q_weight=qw, k_weight=qw)
    (a,) = torch.autograd.grad(y.sum(), [x])
    y, _ = jm.rotate_heads(x, k, None, f, q_weight=qw, k_weight=qw)
    (b,) = torch.autograd.grad(y, [x], torch.ones_like(y))
    assert torch.equal(a, b)
    kk = k.contiguous().requires_grad_(True)
    _, z = jm.rotate_heads(x, kk, None, f, q_weight=qw, k_weight=qw)
    gx, gk = torch.autograd.grad(z, [x, kk], torch.ones_like(z), allow_unused=True)
    assert not gx.any() and gk.any()


def test_no_keys_one_norm_and_float32_weights():
    q, k, qw, kw, gq, gk = inputs(9, 2, 6, 4, 2, 128, BF16)
    f = jm.rotary_frequencies(128)
    both = jm.rotate_heads(q, k, None, f, q_weight=qw.float())
    alone, none = jm.rotate_heads(q, None, None, f, q_weight=qw.float())
    plain, _ = jm.rotate_heads(k, None, None, f)
    assert none is None and torch.equal(both[0], alone) and torch.equal(both[1], plain)
    w = qw.float().requires_grad_(True)
    x, y = q.clone().requires_grad_(True), k.clone().requires_grad_(True)
    out = jm.rotate_heads(x, y, None, f, q_weight=w)
    dx, dy, dw = torch.autograd.grad(out, [x, y, w], [gq, gk])
    assert dw.dtype == F32 and dx.dtype == BF16
    exact = [t.detach().double().requires_grad_(True) for t in (x, y, w)]
    at = torch.arange(6, device="cuda")[None, :, None]
    o = po.rotate(exact[0], at, f, weight=exact[2]), po.rotate(exact[1], at, f)
    want = torch.autograd.grad(o, exact, [gq.double(), gk.double()])
    for got, e in zip((dx, dy, dw), want):
        assert (got.double() - e).norm() <= 2.0 ** -8 * e.norm()
    (only,) = torch.autograd.grad(jm.rotate_heads(x, None, None, f, q_weight=w)[0], [x], gq)
    assert torch.equal(only, dx)


def test_broadcast_inputs_and_shared_tensors():
    """One head expanded over several, and one tensor as queries and keys: gradients add up."""
    q, k, qw, kw, gq, gk = inputs(4, 2, 5, 4, 4, 64, F32)
    f = jm.rotary_frequencies(64)
    one = q[:, :, :1].contiguous().requires_grad_(True)
    y, _ = jm.rotate_heads(one.expand(2, 5, 4, 64), None, None, f, q_weight=qw)
    (got,) = torch.autograd.grad(y, [one], gq)
    whole = q[:, :, :1].expand(2, 5, 4, 64).contiguous().requires_grad_(True)
    z, _ = jm.rotate_heads(whole, None, None, f, q_weight=qw)
    (each,) = torch.autograd.grad(z, [whole], gq)
    assert torch.equal(y, z) and torch.allclose(got, each.sum(2, keepdim=True), rtol=1e-5, atol=1e-5)
    x = q.clone().requires_grad_(True)
    a, b = jm.rotate_heads(x, x, None, f, q_weight=qw, k_weight=kw)
    (both,) = torch.autograd.grad([a, b], [x], [gq, gk])
    x1, x2 = (q.clone().requires_grad_(True) for _ in range(2))
    d1, d2 = torch.autograd.grad(jm.rotate_heads(x1, x2, None, f, q_weight=qw, k_weight=kw), [x1, x2], [gq, gk])
    assert torch.equal(both, d1 + d2)


def test_second_derivatives_are_refused():
    q, k, qw, *_ = inputs(4, 1, 5, 2, 2, 64, F32)
    q.requires_grad_(True)
    y, _ = jm.rotate_heads(q, None, None, jm.rotary_frequencies(64), q_weight=qw)
    with pytest.raises(RuntimeError, match="second"):
        torch.autograd.grad(y.square().sum(), [q], create_graph=True)


def test_a_training_step_with_attention():
    """Norm, rotation and causal attention, and back: every gradient against float64."""
    B, L, Hq, Hkv, d = 2, 70, 4, 2, 64
    q, k, qw, kw, gq, gk = inputs(6, B, L, Hq, Hkv, d, F32)
    v = torch.randn_like(k)
    f = jm.rotary_frequencies(d)
    leaves = [t.requires_grad_(True) for t in (q, k, v, qw, kw)]
    o = jm.masked_attention_via_map(*jm.rotate_heads(q, k, None, f, q_weight=qw, k_weight=kw), v, is_causal=True)
    grads = torch.autograd.grad(o, leaves, gq)
    e = [t.detach().double().requires_grad_(True) for t in leaves]
    at = torch.arange(L, device="cuda")[None, :, None]
    rq, rk = po.rotate(e[0], at, f, weight=e[3]), po.rotate(e[1], at, f, weight=e[4])
    logits = torch.einsum("bqhd,bkhd->bhqk", rq, rk.repeat_interleave(Hq // Hkv, 2)) / d ** 0.5
    logits = logits.masked_fill(torch.ones(L, L, device="cuda").triu(1).bool(), -torch.inf)
    want = torch.einsum("bhqk,bkhd->bqhd", logits.softmax(-1), e[2].repeat_interleave(Hq // Hkv, 2))
    assert (o.double() - want).norm() <= 3e-6 * want.norm()
    for got, w in zip(grads, torch.autograd.grad(want, e, gq.double())):        # (2e-6 of attention, and of rotation the same)
        assert (got.double() - w).norm() <= 5e-6 * w.norm()


def test_components_that_are_not_rotated_keep_infinities():
    q = torch.ones((1, 2, 1, 64), device="cuda")
    q[..., 40], q[..., 41] = torch.inf, torch.nan
    for layout in ("half", "interleaved"):
        y, _ = jm.rotate_heads(q, None, None, jm.rotary_frequencies(32), layout=layout)
        assert torch.equal(y[..., 32:].nan_to_num(7), q[..., 32:].nan_to_num(7)) and y[..., :32].isfinite().all()


def test_zero_heads_and_eps():
    q = torch.zeros((1, 3, 2, 64), device="cuda")
    y, _ = jm.rotate_heads(q, None, q_weight=torch.ones(64, device="cuda"))
    assert not y.any()
    y, _ = jm.rotate_heads(q, None, q_weight=torch.ones(64, device="cuda"), eps=0.0)     # 0 * inf, as the definition has it
    assert y.isnan().all()


def test_repeated_streams_and_capture():
    q, k, qw, kw, gq, gk = inputs(2, 2, 257, 8, 2, 128, BF16)
    f = jm.rotary_frequencies(128)
    leaves = [t.requires_grad_(True) for t in (q, k, qw, kw)]
    step = lambda: torch.autograd.grad(jm.rotate_heads(q, k, None, f, q_weight=qw, k_weight=kw), leaves, [gq, gk])
    first = step()
    assert all(torch.equal(a, b) for a, b in zip(first, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, other))
    with torch.no_grad():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = jm.rotate_heads(q, k, None, f, q_weight=qw, k_weight=kw)
        q.mul_(-2)
        graph.replay()
        want = jm.rotate_heads(q, k, None, f, q_weight=qw, k_weight=kw)
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_captured_backward():
    q, k, qw, kw, gq, gk = inputs(8, 2, 33, 4, 2, 64, F32)
    f = jm.rotary_frequencies(64)
    leaves = [t.requires_grad_(True) for t in (q, k, qw, kw)]
    step = lambda: torch.autograd.grad(jm.rotate_heads(q, k, None, f, q_weight=qw, k_weight=kw), leaves, [gq, gk])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    gq.mul_(-0.5)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_many_tokens():
    """More (token, head) rows than 2^31 / 256: offsets in 64 bits."""
    B, L, H, d = 1, 70000, 128, 256
    q = torch.zeros((B, L, H, d), device="cuda", dtype=BF16)
    q[0, -1, -1] = 1
    y, _ = jm.rotate_heads(q, None, torch.zeros(L, dtype=torch.int32, device="cuda"), jm.rotary_frequencies(d))
    assert (y[0, -1, -1] == 1).all() and not y[0, -1, :-1].any() and not y[0, :1000].any()


def test_launches():
    q, k, qw, kw, gq, gk = inputs(2, 2, 3, 8, 2, 128, BF16)
    f = jm.rotary_frequencies(128)
    before = nat.lib().bma_launch_count()
    jm.rotate_heads(q, k, None, f, q_weight=qw, k_weight=kw)
    assert nat.lib().bma_launch_count() == before + 1
