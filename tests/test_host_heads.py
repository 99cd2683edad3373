"""Heads and the paged cache on the host: frequencies, what the calls refuse, the layouts of the argument structures, the 4-bit oracle."""
import ctypes as C
import math
import subprocess
from pathlib import Path

import pytest
import torch

import jaxmodules_b200 as jm
from jaxmodules_b200 import _native as nat
from oracle import paged_oracle as po

ROOT = Path(__file__).resolve().parents[1]


def test_struct_layouts(tmp_path):
    names = {"bma_rotary": nat.Rotary, "bma_rotate_args": nat.RotateArgs, "bma_paged_cache": nat.PagedCacheArgs, "bma_append_args": nat.AppendArgs,
             "bma_paged_attn_args": nat.PagedAttnArgs}
    lines, want = [], []
    for name, mirror in names.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(C.sizeof(mirror))
        for field, _ in mirror._fields_:
            lines.append(f'printf("%zu\\n", offsetof({name}, {field}));')
            want.append(getattr(mirror, field).offset)
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "bma.h"\nint main(void){' + "".join(lines) + "return 0;}\n")
    subprocess.run(["gcc", "-std=c99", "-I", str(ROOT / "include"), str(src), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split()
    assert [int(x) for x in out] == want


def test_frequencies():
    f = jm.rotary_frequencies(8, 100.0, device="cpu")
    assert f.dtype == torch.float64 and torch.allclose(f, torch.tensor([1, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=torch.float64), rtol=1e-15, atol=0)
    assert torch.allclose(jm.rotary_frequencies(8, 100.0, scaling="linear", factor=4, device="cpu"), f / 4, rtol=1e-15, atol=0)
    g = jm.rotary_frequencies(8, 100.0, scaling="base", factor=4, device="cpu")
    assert g[0] == 1 and abs(g[-1] * 4 / f[-1] - 1) < 1e-14
    # turns within 2 pi * 40 positions: 40, 12.6, 4, 1.26; kept above 13, divided below 4, the second nearly kept
    p = jm.rotary_frequencies(8, 100.0, scaling="parts", factor=8, original_length=2 * math.pi * 40, low=4.0, high=13.0, device="cpu")
    keep = (40 * 100 ** -0.25 - 4) / 9
    assert p[0] == f[0] and abs(p[1] / f[1] - (keep + (1 - keep) / 8)) < 1e-14 and torch.allclose(p[2:], f[2:] / 8, rtol=1e-13, atol=0)
    for bad in (dict(dim=7), dict(dim=0), dict(dim=2, scaling="base"), dict(dim=8, scaling="other"), dict(dim=8, factor=0.0), dict(dim=8, scaling="parts"),
                dict(dim=8, scaling="parts", original_length=10, low=2.0, high=2.0)):
        with pytest.raises(ValueError):
            jm.rotary_frequencies(**bad, device="cpu")


def heads(B=2, L=3, H=4, d=8, dtype=torch.float32):
    return torch.zeros((B, L, H, d), dtype=dtype)


F = torch.zeros(4, dtype=torch.float64)


@pytest.mark.parametrize("error,call", {
    "no cpu path": (RuntimeError, lambda: jm.rotate_heads(heads(), heads(), None, F)),
    "no cpu path, autograd": (RuntimeError, lambda: jm.rotate_heads(heads().requires_grad_(), heads(), None, F)),
    "layout": (ValueError, lambda: jm.rotate_heads(heads(), None, None, F, layout="other")),
}.values(), ids=lambda x: None if callable(x) else x.__name__)
def test_rotate_heads_refuses_before_native_code(error, call):
    with pytest.raises(error):
        call()


def rotate(q=heads(), k=heads(), positions=None, frequencies=F, layout=0, magnitude=1.0, q_weight=None, k_weight=None, eps=1e-6):
    return nat.host().rotate(q, k, positions, frequencies, layout, magnitude, q_weight, k_weight, eps)


# What is wrong with the tensors is said before where they are (the native checks are reached with CPU tensors; none gets past them).
@pytest.mark.parametrize("error,kwargs", [
    (RuntimeError, {}),
    (ValueError, dict(q=torch.zeros(2, 3, 8))),
    (ValueError, dict(q=heads(L=0))),
    (ValueError, dict(q=heads(d=512), k=None)),
    (TypeError, dict(q=heads(dtype=torch.float16), k=None)),
    (TypeError, dict(k=heads(dtype=torch.bfloat16))),
    (ValueError, dict(k=heads(L=4))),
    (ValueError, dict(k=heads(d=16))),
    (TypeError, dict(frequencies=F.float())),
    (ValueError, dict(frequencies=torch.zeros(5, dtype=torch.float64))),
    (ValueError, dict(frequencies=torch.zeros(0, dtype=torch.float64))),
    (ValueError, dict(frequencies=torch.zeros(8, dtype=torch.float64)[::2])),
    (ValueError, dict(frequencies=None)),
    (ValueError, dict(k=None, k_weight=torch.ones(8))),
    (ValueError, dict(frequencies=None, q_weight=torch.ones(7))),
    (TypeError, dict(frequencies=None, q_weight=torch.ones(8, dtype=torch.float64))),
])
def test_rotate_refuses(error, kwargs):
    with pytest.raises(error):
        rotate(**kwargs)


def cache(dtype=torch.float32, pages=5, page=4, H=2, d=32, B=2, width=3, **kw):
    table = torch.zeros((B, width), dtype=torch.int32)
    c = jm.PagedCache.empty(pages, page, H, d, table, dtype)
    return jm.PagedCache(**{**c.__dict__, **kw})


def attend(c=None, q=None, lengths=torch.zeros(2, dtype=torch.int32), new_lengths=None, window=None):
    c = cache() if c is None else c
    q = heads(d=32) if q is None else q
    return nat.host().paged(c.k, c.v, c.page_table, c.k_scale, c.v_scale, q, lengths, new_lengths, None, window, False, False)


@pytest.mark.parametrize("error,kwargs", [
    (RuntimeError, lambda: {}),
    (ValueError, lambda: dict(c=cache(k=torch.zeros(5, 4, 2, 16)))),
    (ValueError, lambda: dict(c=cache(d=12), q=heads(d=12))),
    (ValueError, lambda: dict(c=cache(d=136), q=heads(d=136))),
    (ValueError, lambda: dict(c=cache(k_scale=torch.zeros(5, 4, 2, 1, dtype=torch.uint8)))),
    (ValueError, lambda: dict(c=cache("4bit", k_scale=None))),
    (ValueError, lambda: dict(c=cache("4bit", k_scale=torch.zeros(5, 4, 2, 2, dtype=torch.uint8)))),
    (TypeError, lambda: dict(c=cache("4bit", k_scale=torch.zeros(5, 4, 2, 1)))),
    (TypeError, lambda: dict(c=cache(k=torch.zeros(5, 4, 2, 32).half(), v=torch.zeros(5, 4, 2, 32).half()))),
    (ValueError, lambda: dict(c=cache(k=torch.zeros(5, 4, 2, 33)[..., 1:], v=torch.zeros(5, 4, 2, 33)[..., 1:]))),
    (ValueError, lambda: dict(c=cache(k=torch.zeros(5, 2, 4, 32).transpose(1, 2)))),           # v has other strides
    (ValueError, lambda: dict(c=cache(k=torch.zeros(5, 4, 32, 2).transpose(2, 3), v=torch.zeros(5, 4, 32, 2).transpose(2, 3)))),
    (TypeError, lambda: dict(c=cache(page_table=torch.zeros((2, 3), dtype=torch.int64)))),
    (ValueError, lambda: dict(c=cache(page_table=torch.zeros(6, dtype=torch.int32)))),
    (ValueError, lambda: dict(c=cache(page_table=torch.zeros((3, 2), dtype=torch.int32).t()))),
    (ValueError, lambda: dict(c=cache(page_table=torch.zeros((2, 0), dtype=torch.int32)))),
    (TypeError, lambda: dict(lengths=torch.zeros(2, dtype=torch.int64))),
    (ValueError, lambda: dict(lengths=torch.zeros(3, dtype=torch.int32))),
    (ValueError, lambda: dict(new_lengths=torch.zeros((2, 1), dtype=torch.int32))),
    (ValueError, lambda: dict(q=heads(H=3, d=32))),
    (ValueError, lambda: dict(q=heads(B=3, d=32))),
    (ValueError, lambda: dict(q=heads(d=16))),
    (TypeError, lambda: dict(q=heads(d=32, dtype=torch.bfloat16))),
    (TypeError, lambda: dict(c=cache("4bit"), q=heads(d=32))),
    (ValueError, lambda: dict(window=-1)),
])
def test_paged_attention_refuses(error, kwargs):
    with pytest.raises(error):
        attend(**kwargs())


@pytest.mark.parametrize("error,kwargs", [
    (RuntimeError, {}),
    (ValueError, dict(v=heads(H=2, L=4, d=32))),
    (ValueError, dict(k=heads(H=3, d=32))),
    (TypeError, dict(k=heads(H=2, d=32, dtype=torch.bfloat16))),
    (ValueError, dict(q=heads(L=4, d=32))),
    (ValueError, dict(q=heads(d=32), frequencies=None)),
    (ValueError, dict(q_weight=torch.ones(32))),
    (ValueError, dict(frequencies=torch.zeros(17, dtype=torch.float64))),
])
def test_append_refuses(error, kwargs):
    c = cache()
    a = dict(k=heads(H=2, d=32), v=heads(H=2, d=32), lengths=torch.zeros(2, dtype=torch.int32), new_lengths=None, q=None, frequencies=F, q_weight=None) | kwargs
    with pytest.raises(error):
        nat.host().append(c.k, c.v, c.page_table, c.k_scale, c.v_scale, a["k"], a["v"], a["lengths"], a["new_lengths"], a["q"], a["frequencies"], 0, 1.0, a["q_weight"],
                          None, 1e-6)


def test_read_refuses():
    c = cache()
    lengths = torch.zeros(2, dtype=torch.int32)
    for error, L in ((ValueError, 0), (RuntimeError, 4)):
        with pytest.raises(error):
            nat.host().read(c.k, c.v, c.page_table, c.k_scale, c.v_scale, lengths, L)
    with pytest.raises(RuntimeError, match="CUDA"):
        jm.read_kv(c, lengths, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        jm.paged_attention(heads(d=32), c, lengths)
    with pytest.raises(ValueError, match="not differentiable"):
        jm.paged_attention(heads(d=32).requires_grad_(), c, lengths)
    with pytest.raises(ValueError, match="not differentiable"):
        jm.append_kv(c, heads(H=2, d=32).requires_grad_(), heads(H=2, d=32), lengths)
    with pytest.raises((TypeError, ValueError)):
        jm.PagedCache.empty(1, 1, 1, 16, c.page_table, "4bit")


def test_entry_points_refuse_without_a_device():
    """Rejected arguments return before any CUDA call."""
    lib = nat.lib()
    assert lib.bma_rotate(None, None) == nat.BMA_ERR_ARG and lib.bma_rotate_bwd(None, None, 0, None) == nat.BMA_ERR_ARG
    assert lib.bma_append_kv(None, None, None) == lib.bma_paged_attn(None, None, None, 0, None) == lib.bma_read_kv(None, None, 1, None, None, None) == nat.BMA_ERR_ARG
    a = nat.RotateArgs(B=1, L=1, Hq=1, Hkv=0, d=8)
    a.rotary.dim = 10
    assert lib.bma_rotate(C.byref(a), None) == nat.BMA_ERR_ARG          # more components rotated than there are
    a.rotary.dim, a.d = 0, 512
    assert lib.bma_rotate(C.byref(a), None) == nat.BMA_ERR_UNSUPPORTED
    assert lib.bma_rotate_bwd_workspace_bytes(C.byref(a)) == 0
    c = nat.PagedCacheArgs(k=16, v=16, page_table=16, pages=1, page_size=1, Hkv=2, d=64, B=1, width=1, dtype=nat.BMA_DTYPE_BF16)
    p = nat.PagedAttnArgs(T=1, Hq=3, lengths=16)
    assert lib.bma_paged_attn(C.byref(c), C.byref(p), None, 0, None) == nat.BMA_ERR_ARG      # heads
    c.d = 100
    assert lib.bma_paged_attn(C.byref(c), C.byref(p), None, 0, None) == nat.BMA_ERR_UNSUPPORTED
    c.d, c.stride_slot = 64, 3
    assert lib.bma_paged_attn(C.byref(c), C.byref(p), None, 0, None) == nat.BMA_ERR_UNSUPPORTED
    c.stride_slot, c.page_size, c.width = 64, 1 << 16, 1 << 16
    assert lib.bma_paged_attn(C.byref(c), C.byref(p), None, 0, None) == nat.BMA_ERR_LIMIT


def test_negative_strides_of_a_cache_are_refused():
    lib = nat.lib()
    lengths = 16
    p = nat.PagedAttnArgs(T=1, Hq=2, lengths=lengths)
    p.q.dtype = nat.BMA_DTYPE_BF16
    for dtype, field in [(nat.BMA_DTYPE_BF16, "stride_page"), (nat.BMA_DTYPE_BF16, "stride_slot"), (nat.BMA_DTYPE_BF16, "stride_head"),
                         (nat.BMA_DTYPE_MXFP4, "scale_stride_page"), (nat.BMA_DTYPE_MXFP4, "scale_stride_slot"), (nat.BMA_DTYPE_MXFP4, "scale_stride_head")]:
        c = nat.PagedCacheArgs(k=16, v=16, k_scale=16, v_scale=16, page_table=16, pages=1, page_size=1, Hkv=2, d=128, B=1, width=1, dtype=dtype)
        setattr(c, field, -64)
        k = nat.Tensor(ptr=16, dtype=nat.BMA_DTYPE_BF16)
        assert lib.bma_paged_attn(C.byref(c), C.byref(p), None, 0, None) == nat.BMA_ERR_ARG, field
        assert lib.bma_read_kv(C.byref(c), C.c_void_p(lengths), 1, C.byref(k), C.byref(k), None) == nat.BMA_ERR_ARG, field
        a = nat.AppendArgs(T=1, lengths=lengths, k=k, v=k)
        assert lib.bma_append_kv(C.byref(c), C.byref(a), None) == nat.BMA_ERR_ARG, field


def test_4bit_oracle():
    """Known answers of the format: exact values stay, ties go to the even code, the power of two is the smallest that fits."""
    exact = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
    x = torch.zeros(5, 32, dtype=torch.float64)
    x[0, :8], x[0, 8:16] = exact, -exact
    x[1, :8] = torch.tensor([6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5])
    x[2, 0] = 6.0001
    x[3, 0] = 3.0 * 2.0 ** -40
    v, byte = po.to_4bit(x)
    assert torch.equal(v[0], x[0]) and v[1, :8].tolist() == [6, 0, 1, 1, 2, 2, 4, 4] and v[2, 0] == 6
    assert byte.squeeze(-1).tolist() == [127, 127, 128, 127 - 41, 0] and v[3, 0] == 3.0 * 2.0 ** -40 and not v[4].any()
