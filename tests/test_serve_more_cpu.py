"""CPU: more of what the draw, the 4-bit products and the gradient norm refuse or hand on before any launch."""
import ctypes as C

import pytest
import torch

import albatross_b200 as ab
from albatross_b200 import _lib


def test_gradient_norm_refuses_scales_beyond_32_bits():
    one = (_lib.Grad * 1)(_lib.Grad(4096, 4096, 8, 0, 0))
    for scale in (1e39, 3.5e38, 1e300):
        assert _lib.lib.ab_clip_grad_norm(one, 1, scale, 1.0, 256, 256, None) == -1
        assert "scale" in _lib.lib.ab_last_error().decode()
