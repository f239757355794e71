"""CPU: what the draw, the 4-bit products and the gradient norm refuse before any launch, and the quantiser of 4-bit weights."""
import ctypes as C

import pytest
import torch

import albatross_b200 as ab
from albatross_b200 import _lib

BAD = -1


def message():
    return _lib.lib.ab_last_error().decode()


def test_operators_refuse_tensors_on_the_host():
    with pytest.raises(RuntimeError, match="CUDA"):
        ab.sampler_batch(torch.zeros(2, 10), torch.zeros(2))
    with pytest.raises(RuntimeError, match="CUDA"):
        ab.linear_int4(torch.zeros(1, 128).half(), torch.zeros(4, 64, dtype=torch.uint8), torch.ones(4, 1).half())
    with pytest.raises(RuntimeError, match="gradient 0"):
        ab.clip_grad_norm([torch.zeros(3)], 1.0)
    with pytest.raises(RuntimeError, match="no gradients"):
        ab.grad_norm([])


def sample(dtype=0, rows=1, vocab=100, stride=100, T=1.0, p=1.0, m=0.0, logits=256, uniform=256, ids=256, logp=256, filters=True):
    s = _lib.Sampling(None, None, None, None, T, p, m, 0, 0)
    return _lib.lib.ab_sample_filtered(dtype, rows, vocab, logits, stride, uniform, C.byref(s) if filters else None, ids, logp, None)


def test_draw_refuses_bad_arguments():
    nan = float("nan")
    for bad in (dict(dtype=3), dict(rows=-1), dict(vocab=0), dict(vocab=(1 << 18) + 1), dict(stride=-1), dict(T=-1.0), dict(T=nan), dict(p=-1.0), dict(p=nan), dict(m=-0.5), dict(m=nan),
                dict(logits=None), dict(uniform=None), dict(ids=None), dict(logp=None), dict(filters=False), dict(logits=257), dict(uniform=258), dict(ids=260), dict(logp=258),
                dict(dtype=2, logits=258)):
        assert sample(**bad) == BAD, bad
        assert "ab_sample_filtered" in message()
    assert sample(rows=0, logits=None, uniform=None, ids=None, logp=None) == 0


def int4(rows=1, x=256, stride=128, y=256, **more):
    m = _lib.Int4(**{**dict(dtype=0, n_out=16, k=128, group=128, w=256, scale=256, zero=None), **more})
    return _lib.lib.ab_linear_int4(C.byref(m), rows, x, stride, y, None)


def test_4_bit_products_refuse_bad_arguments():
    for bad in (dict(dtype=2), dict(rows=-1), dict(rows=65536), dict(n_out=0), dict(k=0), dict(k=-128), dict(group=16), dict(group=0), dict(group=-128), dict(group=96, k=192), dict(group=64, k=96), dict(k=100),
                dict(w=None), dict(scale=None), dict(x=None), dict(y=None), dict(w=264), dict(scale=257), dict(x=257), dict(y=257), dict(stride=-1)):
        assert int4(**bad) == BAD, bad
        assert "ab_linear_int4" in message()
    assert _lib.lib.ab_linear_int4(None, 1, 256, 0, 256, None) == BAD
    assert int4(rows=0, x=None, y=None) == 0


def clip(tensors, scale=1.0, limit=1.0, norm=256, scratch=256):
    list_ = (_lib.Grad * len(tensors))(*[_lib.Grad(**{**dict(g=4096, out=4096, n=8, dtype=0, out_dtype=0), **t}) for t in tensors])
    return _lib.lib.ab_clip_grad_norm(list_, len(tensors), scale, limit, norm, scratch, None)


def test_gradient_norm_refuses_bad_arguments():
    nan, inf = float("nan"), float("inf")
    for bad in (dict(scale=0.0), dict(scale=-1.0), dict(scale=nan), dict(scale=inf), dict(limit=-1.0), dict(limit=nan), dict(norm=None), dict(scratch=None), dict(norm=258), dict(scratch=260)):
        assert clip([{}], **bad) == BAD, bad
    for bad in ([dict(dtype=3)], [dict(out_dtype=-1)], [dict(n=-1)], [dict(n=(1 << 40) + 1)], [dict(g=None)], [dict(g=4097)], [dict(out=4097)], [dict(), dict(g=8192, out=None)],
                # outputs on one another, or on other gradients
                [dict(), dict()], [dict(), dict(g=4104, out=4104)], [dict(g=8192, out=4096), dict(g=12288, out=4100)], [dict(g=8192, out=4096), dict(g=4096, out=8192)],
                [dict(g=4096, out=4098)], [dict(out_dtype=2)], [dict(g=4096, out=8192), dict(g=16384, out=4110)], [dict(n=100, g=4096, out=20000), dict(n=1, g=30000, out=4294)],
                [dict(g=40000, out=4096), dict(g=4100, out=50000), dict(g=4000, out=60000)]):
        assert clip(bad) == BAD, bad
        assert "ab_clip_grad_norm" in message()
    assert _lib.lib.ab_clip_grad_norm(None, 1, 1.0, 1.0, 256, 256, None) == BAD
    assert _lib.lib.ab_clip_grad_norm(None, -1, 1.0, 1.0, 256, 256, None) == BAD


def test_struct_layouts_match_the_header():
    assert C.sizeof(_lib.Grad) == 32 and C.sizeof(_lib.Int4) == 40 and C.sizeof(_lib.Sampling) == 64


def test_quantizer_of_4_bit_weights():
    torch.manual_seed(0)
    w = 0.02 * torch.randn(40, 256)
    w[7] = 0
    for zeros in (False, True):
        for group in (32, 64, 128, 256):
            for dtype in (torch.float16, torch.bfloat16):
                m = ab.quantize_int4(w, group, zeros, dtype)
                assert m.w.shape == (40, 128) and m.w.dtype == torch.uint8 and m.scale.shape == (40, 256 // group) and m.scale.dtype == dtype
                assert (m.zero is None) == (not zeros) and (m.zero is None or (m.zero.shape == m.scale.shape and int(m.zero.max()) <= 15))
                back = m.dequantize()
                # a bf16 scale is up to 2^-8 off: 7 or 15 steps of it are below 0.06 steps
                assert bool(((back - w).abs() <= 1.1 * m.scale.float().repeat_interleave(group, 1) + 1e-7).all()) and bool((back[7] == 0).all())
                code = (m.w[3, 5] & 15).float(), (m.w[3, 5] >> 4).float()
                z = 8.0 if m.zero is None else float(m.zero[3, 10 // group])
                assert float(back[3, 10]) == float((code[0] - z) * m.scale[3, 10 // group].float()) and float(back[3, 11]) == float((code[1] - z) * m.scale[3, 11 // group].float())
    for bad in (16, 96, 100, 512):
        with pytest.raises(ValueError):
            ab.quantize_int4(w, bad)
