"""Timed calls of the operators around a cache of keys and values: rotation (and norm) of heads, appending to pages, reading pages back,
and attention over pages, of bfloat16, float32 and 4-bit caches.

A case is a dict of plain values.  ``prepare`` makes what a program has in hand, ``run`` makes one pass: where ``own`` is false in elementary
torch operations, where it is true through the package's entry points.  ``exact`` is the definition in 64 bits.
"""
import math

import numpy as np
import torch

own = False

BASE = 10000.0
EPS = 1e-6
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


# ---- cases ----------------------------------------------------------------------------------------------------------
def _rotate(name, B, L, Hq, Hkv, d, dim, dtype, layout, norm, grad):
    return dict(name=name, op="rotate", B=B, L=L, Hq=Hq, Hkv=Hkv, d=d, dim=dim, dtype=dtype, layout=layout, norm=norm, grad=grad)


def _append(name, op, B, T, L, Hq, Hkv, d, page, dtype, layout, norm):
    return dict(name=name, op=op, B=B, T=T, L=L, Hq=Hq, Hkv=Hkv, d=d, page=page, dtype=dtype, layout=layout, norm=norm)


def _attend(name, B, T, L, Hq, Hkv, d, page, dtype, window=0):
    return dict(name=name, op="attend", B=B, T=T, L=L, Hq=Hq, Hkv=Hkv, d=d, page=page, dtype=dtype, window=window)


def listed():
    return [
        # one new token of each of 64 sequences, far into their contexts: norms and rotation of a decoding step
        _rotate("rotate_decode", 64, 1, 32, 8, 128, 128, "bfloat16", "half", True, False),
        # a training step's norms and rotation: the heads of the dense causal workload, and their gradients
        _rotate("rotate_train", 4, 4096, 32, 32, 128, 128, "bfloat16", "half", True, True),
        # float32, pairs side by side, half of the head rotated, an odd length
        _rotate("rotate_partial", 2, 2049, 8, 8, 64, 32, "float32", "interleaved", False, True),
        # decoding: each of 128 sequences appends one token, the queries rotated in the same call
        _append("append_decode", "append", 128, 1, 2048, 32, 8, 128, 16, "bfloat16", "half", False),
        # prefill: prompts of different lengths in a padded batch
        _append("append_prompts", "append", 8, 2500, 2500, 0, 8, 128, 64, "bfloat16", "half", True),
        # a chunk of prompt goes into a 4-bit cache, and the whole context is read back for the chunk's attention
        _append("append_read_4bit", "append_read", 4, 1024, 6000, 0, 8, 128, 16, "4bit", "half", False),
        # contexts read back as dense keys and values
        dict(name="read_bf16", op="read", B=16, L=5001, Hkv=8, d=128, page=16, dtype="bfloat16"),
        # one short sequence: the time of a launch
        _attend("attend_one", 1, 1, 1500, 16, 2, 64, 16, "bfloat16"),
        # a serving batch in mid-flight, every sequence of another length
        _attend("attend_batch", 64, 1, 8192, 32, 8, 128, 16, "bfloat16"),
        # float32, a sliding window, no shared heads
        _attend("attend_f32", 8, 1, 6000, 16, 16, 64, 32, "float32", 2048),
        # the same serving batch on a 4-bit cache
        _attend("attend_4bit_batch", 64, 1, 8192, 32, 8, 128, 16, "4bit"),
        # one long context, four draft tokens verified at once, on a 4-bit cache
        _attend("attend_4bit_long", 1, 4, 131072, 32, 8, 128, 64, "4bit"),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    Hkv = rng.choice((1, 2, 3, 4, 8, 8))
    return Hkv * rng.choice((1, 2, 3, 4, 4, 8)), Hkv


def draw(rng):
    kind = rng.choice(("rotate", "rotate", "append", "append_read", "read", "attend", "attend", "attend", "attend_4bit", "attend_4bit"))
    Hq, Hkv = _heads(rng)
    d = rng.choice((64, 128, 128))
    page = rng.choice((8, 16, 16, 32, 64, 128))
    if kind == "rotate":
        dtype = rng.choice(("bfloat16", "bfloat16", "float32"))
        B = _spread(rng, 1, 64)
        L = _spread(rng, 1, max(2, 500000 // (B * (Hq + Hkv))))
        d = rng.choice((64, 80, 96, 128, 128))
        dim = rng.choice((d, d, d // 2))
        norm = rng.random() < 0.5
        return dict(op="rotate", B=B, L=L, Hq=Hq, Hkv=Hkv, d=d, dim=dim, dtype=dtype, layout=rng.choice(("half", "half", "interleaved")), norm=norm,
                    grad=rng.random() < 0.5)
    if kind in ("append", "append_read"):
        dtype = "4bit" if kind == "append_read" else rng.choice(("bfloat16", "bfloat16", "float32"))
        B = _spread(rng, 1, 128)
        T = 1 if rng.random() < 0.4 else _spread(rng, 2, max(3, 20000 // B))
        L = min(T + _spread(rng, 1, 4096), max(T, 60000 // B))
        return dict(op=kind, B=B, T=T, L=L, Hq=rng.choice((0, Hq)), Hkv=Hkv, d=d, page=page, dtype=dtype, layout=rng.choice(("half", "half", "interleaved")),
                    norm=rng.random() < 0.5)
    if kind == "read":
        B = _spread(rng, 1, 64)
        return dict(op="read", B=B, L=_spread(rng, 1, 80000 // B), Hkv=Hkv, d=d, page=page, dtype=rng.choice(("bfloat16", "float32", "4bit")))
    B = _spread(rng, 1, 128)
    T = rng.choice((1, 1, 1, 2, 4, 7))
    L = T + _spread(rng, 1, min(131072, 400000 // B))
    dtype = "4bit" if kind == "attend_4bit" else rng.choice(("bfloat16", "bfloat16", "bfloat16", "float32"))
    return dict(op="attend", B=B, T=T, L=L, Hq=Hq, Hkv=Hkv, d=d, page=page, dtype=dtype, window=rng.choice((0, 0, 0, _spread(rng, 16, 4096))))


def _lengths(c):
    """(lengths, new tokens) of the sequences: the first the longest, the second with nothing before its new tokens, the last slot empty."""
    B, L, T = c["B"], c["L"], c.get("T", 1)
    rs = np.random.RandomState(B * 7919 + L)
    lengths = rs.randint(max(T, L // 4), L + 1, B)
    new = np.full(B, T)
    if c["op"] != "attend" and T > 1:
        new = rs.randint(max(1, T // 4), T + 1, B)
    lengths[0] = L
    if B >= 4:
        lengths[1] = new[1]
    if B >= 8:
        lengths[-1] = new[-1] = 0
    return lengths, np.minimum(new, lengths)


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _frequencies(dim):
    return torch.from_numpy(BASE ** (-np.arange(0, dim, 2, dtype=np.float64) / dim)).cuda()


def _cache(c, seed, gen):
    """Pages in shuffled order, a few more than are used; entries of the table that no sequence reaches are -1."""
    lengths, new = _lengths(c)
    B, page, Hkv, d = c["B"], c["page"], c["Hkv"], c["d"]
    width = max(1, -(-c["L"] // page))
    need = -(-lengths // page)
    pages = int(need.sum()) + 3
    order = np.random.RandomState(seed % (1 << 31)).permutation(pages)
    table = np.full((B, width), -1, dtype=np.int32)
    at = 0
    for b in range(B):
        table[b, : need[b]] = order[at : at + need[b]]
        at += need[b]
    s = dict(page_table=torch.from_numpy(table).cuda(), lengths=torch.from_numpy(lengths.astype(np.int32)).cuda(),
             new_lengths=torch.from_numpy(new.astype(np.int32)).cuda(), k_scale=None, v_scale=None)
    for name in ("k", "v"):
        x = torch.randn((pages, page, Hkv, d), generator=gen, device="cuda", dtype=torch.bfloat16 if c["dtype"] != "float32" else torch.float32)
        if c["dtype"] == "4bit":
            x, s[name + "_scale"] = _to_4bit(x.float())
        s[name] = x
    return s


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = torch.float32 if c["dtype"] == "float32" else torch.bfloat16
    randn = lambda *shape: torch.randn(shape, generator=gen, device="cuda", dtype=dtype)  # noqa: E731
    weight = lambda: (1 + 0.1 * torch.randn((c["d"],), generator=gen, device="cuda")).to(dtype)  # noqa: E731
    s = dict(case=c)
    if c["op"] == "rotate":
        B, L, Hq, Hkv, d = (c[n] for n in ("B", "L", "Hq", "Hkv", "d"))
        s["q"], s["k"] = randn(B, L, Hq, d), randn(B, L, Hkv, d)
        s["frequencies"] = _frequencies(c["dim"])
        start = torch.randint(0, 100000, (B, 1), generator=gen, device="cuda")
        s["positions"] = start + torch.arange(L, device="cuda")
        s["q_weight"], s["k_weight"] = (weight(), weight()) if c["norm"] else (None, None)
        if c["grad"]:
            s["dq"], s["dk"] = randn(B, L, Hq, d), randn(B, L, Hkv, d)
            s["leaves"] = [s[n].requires_grad_(True) for n in ("q", "k", "q_weight", "k_weight") if s[n] is not None]
        return s
    s.update(_cache(c, seed, gen))
    if c["op"] in ("append", "append_read"):
        B, T, Hq, Hkv, d = (c[n] for n in ("B", "T", "Hq", "Hkv", "d"))
        s["new_k"], s["new_v"] = randn(B, T, Hkv, d), randn(B, T, Hkv, d)
        s["q"] = randn(B, T, Hq, d) if Hq else None
        s["frequencies"] = _frequencies(d)
        s["k_weight"] = weight() if c["norm"] else None
        s["q_weight"] = weight() if c["norm"] and Hq else None
    if c["op"] == "attend":
        s["q"] = randn(c["B"], c["T"], c["Hq"], c["d"])
    return s


# ---- plain forms ----------------------------------------------------------------------------------------------------
def _to_4bit(x):
    """(codes, scales): of every 32 values e2m1 codes, the earlier value in the lower half of a byte, and the smallest power of two, from
    2^-127 to 2^126 and biased by 127, that lets the largest be at most 6; 255 where one is NaN."""
    g = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    top = g.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(torch.where(torch.isfinite(top) & (top > 0), top, torch.where(top > 0, 3e38, 1e-45)))
    e = (e - 3 + (m > 0.75).to(e.dtype)).clamp(-127, 126)
    y = (g.abs().double() * torch.exp2(-e.double())).float()
    code = ((y > 0.25).to(torch.uint8) + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5) + (y >= 3.5) + (y > 5)).to(torch.uint8)
    code = code | (g.signbit().to(torch.uint8) << 3)
    code = code.reshape(*x.shape[:-1], x.shape[-1] // 2, 2)
    scale = torch.where(torch.isnan(top), 255, e + 127).to(torch.uint8).squeeze(-1)
    return code[..., 0] | (code[..., 1] << 4), scale


def _values(codes, scales):
    """float32 values of a 4-bit cache."""
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    x = table[torch.stack((codes & 15, codes >> 4), -1).long()].reshape(*codes.shape[:-1], codes.shape[-1] // 16, 32)
    factor = torch.where(scales == 255, torch.nan, torch.exp2(scales.double() - 127).float())
    return (x * factor[..., None]).flatten(-2)


def _angles(positions, frequencies):
    """cos and sin as float32, of angles in 64 bits: at position 100000 an angle in 32 bits is off by 0.004."""
    a = positions.double()[..., None] * frequencies
    return a.cos().float()[..., None, :], a.sin().float()[..., None, :]


def _turn(x, cos, sin, layout):
    """Rotates the first 2 * cos.shape[-1] components of each head."""
    r = 2 * cos.shape[-1]
    head, rest = x[..., :r], x[..., r:]
    if layout == "half":
        a, b = head[..., : r // 2], head[..., r // 2 :]
        out = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    else:
        a, b = head[..., 0::2], head[..., 1::2]
        out = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    return torch.cat((out, rest), -1) if rest.shape[-1] else out


def _normed(x, weight):
    inv = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return x * inv * weight.float(), inv


def _rotated(x, weight, cos, sin, layout):
    x = x.float()
    if weight is not None:
        x = _normed(x, weight)[0]
    return _turn(x, cos, sin, layout)


def _rotate_back(x, weight, g, cos, sin, layout):
    """Gradients of _rotated in x and weight."""
    x, g = x.float(), _turn(g.float(), cos, -sin, layout)
    if weight is None:
        return g, None
    inv = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    h = x * inv
    gw = g * weight.float()
    return inv * (gw - h * (gw * h).mean(-1, keepdim=True)), (g * h).flatten(0, -2).sum(0, dtype=torch.float64)


def _rotate_plain(s):
    c = s["case"]
    with torch.no_grad():
        cos, sin = _angles(s["positions"], s["frequencies"])
        outs = {}
        for n in ("q", "k"):
            x, w = s[n], s[n + "_weight"]
            outs[n] = _rotated(x, w, cos, sin, c["layout"]).to(x.dtype)
            if c["grad"]:
                dx, dw = _rotate_back(x, w, s["d" + n], cos, sin, c["layout"])
                outs["grad_" + n] = dx.to(x.dtype)
                if dw is not None:
                    outs["grad_" + n + "_weight"] = dw.to(w.dtype)
        return outs


def _append_plain(s):
    c = s["case"]
    T, page = c["T"], c["page"]
    i = torch.arange(T, device="cuda")
    positions = (s["lengths"] - s["new_lengths"])[:, None] + i
    cos, sin = _angles(positions, s["frequencies"])
    there = i < s["new_lengths"][:, None]
    b, t = torch.nonzero(there, as_tuple=True)
    at = positions[b, t]
    pages, slots = s["page_table"][b, at // page].long(), at % page
    for name, x in (("k", _rotated(s["new_k"], s["k_weight"], cos, sin, c["layout"])), ("v", s["new_v"].float())):
        x = x[b, t]
        if c["dtype"] == "4bit":
            s[name][pages, slots], s[name + "_scale"][pages, slots] = _to_4bit(x)
        else:
            s[name][pages, slots] = x.to(s[name].dtype)
    if s["q"] is None:
        return None
    return torch.where(there[..., None, None], _rotated(s["q"], s["q_weight"], cos, sin, c["layout"]), 0).to(s["q"].dtype)


def _pages(s, name, dtype=torch.float32):
    """[B, positions, Hkv, d] of the cache."""
    table = s["page_table"].long()
    x = s[name][table]
    x = _values(x, s[name + "_scale"][table]) if s["case"]["dtype"] == "4bit" else x
    return x.to(dtype).flatten(1, 2)


def _read_plain(s):
    there = (torch.arange(s["case"]["L"], device="cuda") < s["lengths"][:, None])[..., None, None]
    dtype = torch.bfloat16 if s["case"]["dtype"] == "4bit" else s["k"].dtype
    return [torch.where(there, _pages(s, name)[:, : s["case"]["L"]], 0).to(dtype) for name in ("k", "v")]


def _attend_plain(s, dtype=torch.float32):
    c = s["case"]
    B, T, Hq, Hkv, d = (c[n] for n in ("B", "T", "Hq", "Hkv", "d"))
    k, v = _pages(s, "k", dtype), _pages(s, "v", dtype)
    i, j = torch.arange(T, device="cuda"), torch.arange(k.shape[1], device="cuda")
    at = torch.where(i < s["new_lengths"][:, None], (s["lengths"] - s["new_lengths"])[:, None] + i, -1)[..., None]
    ok = (j <= at) & (j >= at - c["window"]) if c["window"] else j <= at
    q = s["q"].to(dtype).reshape(B, T, Hkv, Hq // Hkv, d)
    logits = torch.matmul(q.permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, d), k.permute(0, 2, 3, 1)) / math.sqrt(d)
    logits = torch.where(ok[:, None, None], logits.reshape(B, Hkv, -1, T, k.shape[1]), -math.inf).reshape(B, Hkv, -1, k.shape[1])
    top = logits.amax(-1, keepdim=True)
    p = torch.exp(logits - torch.where(torch.isfinite(top), top, 0))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v.transpose(1, 2)) / torch.where(total > 0, total, 1)
    lse = (torch.log(total) + top).reshape(B, Hq, T)
    return o.reshape(B, Hq, T, d).transpose(1, 2), lse


def _own(s):
    import jaxmodules_b200 as jm

    c = s["case"]
    if c["op"] == "rotate":
        q, k = jm.rotate_heads(s["q"], s["k"], s["positions"], s["frequencies"], layout=c["layout"], q_weight=s["q_weight"], k_weight=s["k_weight"], eps=EPS)
        outs = dict(q=q, k=k)
        if c["grad"]:
            names = [n for n in ("q", "k", "q_weight", "k_weight") if s[n] is not None]
            outs.update(zip(["grad_" + n for n in names], torch.autograd.grad([q, k], s["leaves"], [s["dq"], s["dk"]])))
        return outs
    cache = jm.PagedCache(s["k"], s["v"], s["page_table"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    if c["op"] in ("append", "append_read"):
        q = jm.append_kv(cache, s["new_k"], s["new_v"], s["lengths"], new_lengths=s["new_lengths"], q=s["q"], frequencies=s["frequencies"], layout=c["layout"],
                         q_weight=s["q_weight"], k_weight=s["k_weight"], eps=EPS)
        if c["op"] == "append":
            return dict(q=q, k=s["k"], v=s["v"])
        return dict(zip(("k", "v"), jm.read_kv(cache, s["lengths"], c["L"])), q=q)
    if c["op"] == "read":
        return dict(zip(("k", "v"), jm.read_kv(cache, s["lengths"], c["L"])))
    o, lse = jm.paged_attention(s["q"], cache, s["lengths"], new_lengths=s["new_lengths"], window=c["window"] or None, out_dtype=s["q"].dtype, return_lse=True)
    return dict(o=o, lse=lse)


def run(state):
    if own:
        return _own(state)
    s = state
    op = s["case"]["op"]
    if op == "rotate":
        return _rotate_plain(s)
    if op == "append":
        q = _append_plain(s)
        return dict(q=q, k=s["k"], v=s["v"])
    if op == "append_read":
        q = _append_plain(s)
        return dict(zip(("k", "v"), _read_plain(s)), q=q)
    if op == "read":
        return dict(zip(("k", "v"), _read_plain(s)))
    o, lse = _attend_plain(s)
    return dict(o=o.to(s["q"].dtype), lse=lse)


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------
def _exact_heads(x, weight, positions, frequencies, layout):
    """Each pair as a complex number, turned by exp(i * angle)."""
    x = x.detach().double()
    if weight is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.detach().double()
    n = frequencies.numel()
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device), positions.double()[..., None, None] * frequencies)
    one, two = (slice(0, n), slice(n, 2 * n)) if layout == "half" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    z = torch.complex(x[..., one], x[..., two]) * turn
    out = x.clone()
    out[..., one], out[..., two] = z.real, z.imag
    return out


def _exact_4bit(x):
    """The 4-bit values nearest to float64 values (ties to the even code)."""
    g = x.reshape(*x.shape[:-1], -1, 32)
    top = g.abs().amax(-1, keepdim=True)
    unit = torch.exp2(torch.ceil(torch.log2(torch.clamp(top, min=1e-30) / 6)).clamp(-127, 126))
    y = g / unit
    step = torch.where(y.abs() < 2, 0.5, torch.where(y.abs() < 4, 1.0, 2.0)).double()
    return ((torch.round(y / step) * step).clamp(-6, 6) * unit).reshape(x.shape)


def _exact_cache(s):
    """(k, v) [pages, page, Hkv, d] in 64 bits after the append, and the rotated queries."""
    c = s["case"]
    lengths, new = s["lengths"].tolist(), s["new_lengths"].tolist()
    four = c["dtype"] == "4bit"
    k, v = ((_values(s[n], s[n + "_scale"]) if four else s[n]).double() for n in ("k", "v"))
    positions = (s["lengths"] - s["new_lengths"])[:, None] + torch.arange(c["T"], device="cuda")
    q = None if s["q"] is None else _exact_heads(s["q"], s["q_weight"], positions, s["frequencies"], c["layout"])
    for b in range(c["B"]):
        t = new[b]
        if q is not None:
            q[b, t:] = 0
        if not t:
            continue
        at = torch.arange(lengths[b] - t, lengths[b], device="cuda")
        pages, slots = s["page_table"][b].long()[at // c["page"]], at % c["page"]
        nk = _exact_heads(s["new_k"][b, :t], s["k_weight"], at, s["frequencies"], c["layout"])
        nv = s["new_v"][b, :t].double()
        k[pages, slots], v[pages, slots] = (_exact_4bit(nk), _exact_4bit(nv)) if four else (nk, nv)
    return k, v, q


def _exact_read(s, k, v):
    L, page = s["case"]["L"], s["case"]["page"]
    outs = []
    for x in (k, v):
        out = torch.zeros((s["case"]["B"], L, *x.shape[2:]), dtype=torch.float64, device="cuda")
        for b, n in enumerate(s["lengths"].tolist()):
            at = torch.arange(n, device="cuda")
            out[b, :n] = x[s["page_table"][b].long()[at // page], at % page]
        outs.append(out)
    return dict(zip(("k", "v"), outs))


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["op"] == "rotate":
        leaves = {n: s[n].detach().double().requires_grad_(c["grad"]) for n in ("q", "k", "q_weight", "k_weight") if s[n] is not None}
        outs = {}
        for n in ("q", "k"):
            outs[n] = _exact_grad_heads(leaves[n], leaves.get(n + "_weight"), s["positions"], s["frequencies"], c["layout"])
        if c["grad"]:
            grads = torch.autograd.grad([outs["q"], outs["k"]], list(leaves.values()), [s["dq"].double(), s["dk"].double()])
            outs.update(zip(["grad_" + n for n in leaves], grads))
        return {n: x.detach() for n, x in outs.items()}
    if c["op"] in ("append", "append_read"):
        k, v, q = _exact_cache(s)
        if c["op"] == "append":
            return dict(q=q, k=k, v=v)
        return dict(_exact_read(s, k, v), q=q)
    values = [(_values(s[n], s[n + "_scale"]) if c["dtype"] == "4bit" else s[n]) for n in ("k", "v")]
    if c["op"] == "read":
        return _exact_read(s, *(x.double() for x in values))
    B, T, Hq, Hkv, d, page = (c[n] for n in ("B", "T", "Hq", "Hkv", "d", "page"))
    o = torch.zeros((B, T, Hq, d), dtype=torch.float64, device="cuda")
    lse = torch.full((B, Hq, T), -math.inf, dtype=torch.float64, device="cuda")
    for b, (n, new) in enumerate(zip(s["lengths"].tolist(), s["new_lengths"].tolist())):
        at = torch.arange(n, device="cuda")
        rows = s["page_table"][b].long()[at // page], at % page
        kb, vb = (x[rows].double().repeat_interleave(Hq // Hkv, 1) for x in values)
        for t in range(new):
            end = n - new + t + 1
            lo = max(0, end - 1 - c["window"]) if c["window"] else 0
            logits = torch.einsum("hd,lhd->hl", s["q"][b, t].double(), kb[lo:end]) / math.sqrt(d)
            lse[b, :, t] = torch.logsumexp(logits, -1)
            o[b, t] = torch.einsum("hl,lhd->hd", torch.softmax(logits, -1), vb[lo:end])
    return dict(o=o, lse=lse)


def _exact_grad_heads(x, weight, positions, frequencies, layout):
    """_exact_heads by products with cosines and sines, for differentiation."""
    if weight is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * weight
    angle = positions.double()[..., None, None] * frequencies
    n = frequencies.numel()
    cos, sin = angle.cos(), angle.sin()
    if layout == "half":
        a, b = x[..., :n], x[..., n : 2 * n]
        parts = [a * cos - b * sin, a * sin + b * cos]
        return torch.cat(parts + [x[..., 2 * n :]], -1)
    a, b = x[..., 0 : 2 * n : 2], x[..., 1 : 2 * n : 2]
    return torch.cat((torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2), x[..., 2 * n :]), -1)


# ---- what a pass cannot do without --------------------------------------------------------------------------------------
def work(case):
    c = case
    size = 4 if c["dtype"] == "float32" else 2
    if c["op"] == "rotate":
        values = c["B"] * c["L"] * (c["Hq"] + c["Hkv"]) * c["d"]
        passes = 2 if not c["grad"] else 5 if c["norm"] else 4
        return dict(bytes=values * size * passes + 8 * c["B"] * c["L"], flops=values * (6 if not c["grad"] else 20))
    lengths, new = _lengths(c)
    held = c["d"] * size if c["dtype"] != "4bit" else c["d"] // 2 + c["d"] // 32        # bytes of one head of one token in the cache
    heads = 2 * c["Hkv"]                                                              # keys and values
    context = int(lengths.sum())
    if c["op"] == "read":
        return dict(bytes=context * heads * held + c["B"] * c["L"] * heads * c["d"] * size, flops=0)
    if c["op"] in ("append", "append_read"):
        n = int(new.sum())
        moved = n * heads * (c["d"] * size + held) + (n + c["B"] * c["T"]) * c["Hq"] * c["d"] * size
        if c["op"] == "append_read":
            moved += context * heads * held + c["B"] * c["L"] * heads * c["d"] * size
        return dict(bytes=moved, flops=n * (c["Hq"] + c["Hkv"]) * c["d"] * 6)
    pairs = tokens = 0
    for n, t in zip(lengths.tolist(), new.tolist()):
        if not t:
            continue
        ends = np.arange(n - t + 1, n + 1)
        starts = np.maximum(0, ends - 1 - c["window"]) if c["window"] else np.zeros_like(ends)
        pairs += int((ends - starts).sum())
        tokens += int(ends[-1] - starts[0])
    io = 2 * c["B"] * c["T"] * c["Hq"] * c["d"] * size
    return dict(bytes=tokens * heads * held + io, flops=4 * pairs * c["Hq"] * c["d"])
