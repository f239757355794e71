"""CPU: the operators with gradients refuse what they cannot take, before any launch."""
import ctypes as C

import pytest
import torch

import albatross_b200 as ab
from albatross_b200 import _lib

P = 4096    # stands for a device pointer: nothing is launched here


def _seq(**kw):
    s = _lib.Wkv7Seq(_lib.DT_F16, 2, 5, 3)
    for i in range(6):
        s.x[i], s.batch_stride[i], s.step_stride[i] = P, 5 * 192, 192
    s.checkpoints = P
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def _fwd(s, y=P, out=P):
    return _lib.lib.ab_wkv7_seq_fwd(C.byref(s), y, out, None)


def _bwd(s, dx=None, dy=P):
    return _lib.lib.ab_wkv7_seq_bwd(C.byref(s), dy, 960, 192, None, (C.c_void_p * 6)(*(dx or [P] * 6)), P, None)


def test_checkpoint_bytes():
    for T, chunks in ((0, 0), (1, 1), (16, 1), (17, 2), (1024, 64)):
        assert _lib.lib.ab_wkv7_checkpoint_bytes(C.byref(_seq(T=T))) == 2 * 3 * chunks * 16384
    assert _lib.lib.ab_wkv7_checkpoint_bytes(C.byref(_seq(B=70000, T=70000, H=64))) == 70000 * 64 * 4375 * 16384
    assert -(-1024 // _lib.WKV_CHUNK) == 64


@pytest.mark.parametrize("kw", [{"dtype": _lib.DT_F32}, {"dtype": 7}, {"B": 0}, {"T": -1}, {"H": 0}, {"state": P + 4}, {"checkpoints": P + 8}, {"lengths": P + 2},
                                {"B": 1 << 20, "H": 1 << 12}])
def test_recurrence_refuses(kw):
    assert _fwd(_seq(**kw)) == -1 and _lib.lib.ab_last_error()
    assert _bwd(_seq(**kw)) == -1


def test_recurrence_refuses_missing_or_crooked_pointers():
    s = _seq()
    s.x[4] = None
    assert _fwd(s) == -1
    s = _seq()
    s.x[2] = P + 8
    assert _fwd(s) == -1
    s = _seq()
    s.step_stride[5] = 196
    assert _fwd(s) == -1 and b"16-byte" in _lib.lib.ab_last_error()
    assert _fwd(_seq(), y=None) == -1 and _fwd(_seq(), out=None) == -1 and _fwd(_seq(), y=P + 8) == -1
    assert _bwd(_seq(checkpoints=None)) == -1 and _bwd(_seq(), dx=[P, P, P + 2, P, P, P]) == -1 and _bwd(_seq(), dy=P + 1) == -1


@pytest.mark.parametrize("args", [(3, 3, 4, 64, 1), (0, 1, 4, 64, 1), (2, 0, 4, 64, 1), (0, 0, 4, 64, 3), (0, 0, 4, 0, 1), (0, 0, -1, 64, 1), (0, 0, 4, 64, 0)])
def test_norm_refuses(args):
    dtype, wtype, n, Cn, groups = args
    assert _lib.lib.ab_layer_norm_fwd(dtype, wtype, n, Cn, groups, P, Cn, P, P, 1e-5, P, None, None, None) == -1
    assert _lib.lib.ab_layer_norm_bwd(dtype, wtype, n, Cn, groups, P, Cn, P, P, P, P, Cn, P, P, P, P, None) == -1


def test_norm_refuses_pointers():
    fwd = lambda x=P, y=P, w=P, mean=None, rstd=None, stride=64: _lib.lib.ab_layer_norm_fwd(0, 0, 4, 64, 1, x, stride, w, P, 1e-5, y, mean, rstd, None)  # noqa: E731
    assert fwd(x=None) == -1 and fwd(y=None) == -1 and fwd(x=P + 1) == -1 and fwd(w=P + 1) == -1 and fwd(mean=P) == -1 and fwd(stride=-64) == -1
    assert _lib.lib.ab_layer_norm_bwd(0, 0, 4, 64, 1, P, 64, P, P, P, P, 64, P, P, P, None, None) == -1 and b"scratch" in _lib.lib.ab_last_error()
    assert _lib.lib.ab_layer_norm_scratch_bytes(-1, 64) == 0 and _lib.lib.ab_layer_norm_scratch_bytes(100, 64) > 0


def _rows(**kw):
    t = _lib.LogitRows(_lib.DT_BF16, 100, 6, 100, P, P, None)
    for k, v in kw.items():
        setattr(t, k, v)
    return t


def _policy(**kw):
    p = _lib.Policy(P, P, None, 0.2, 0.2, 0.0, 0.0)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw", [{"dtype": 3}, {"vocab": 0}, {"rows": -1}, {"stride": 99}, {"logits": None}, {"ids": None}, {"logits": P + 1}, {"ids": P + 4},
                                {"rows": 1 << 31}])
def test_losses_refuse_rows(kw):
    t = _rows(**kw)
    assert _lib.lib.ab_token_logp_fwd(C.byref(t), P, P, None, None) == -1
    assert _lib.lib.ab_token_logp_bwd(C.byref(t), P, P, 1, None, P, None) == -1
    assert _lib.lib.ab_policy_loss_fwd(C.byref(t), C.byref(_policy()), P, P, P, P, P, None) == -1
    assert _lib.lib.ab_policy_loss_grad(C.byref(t), C.byref(_policy()), 1.0, P, P, P, P, None) == -1
    assert _lib.lib.ab_preference_loss_fwd(C.byref(t), 1, 3, P, 0.1, 0.0, P, P, P, P, P, None) == -1


@pytest.mark.parametrize("kw", [{"advantages": None}, {"clip_low": -0.1}, {"clip_low": 1.1}, {"clip_high": -1.0}, {"clip_low": float("nan")}, {"denom": -1.0},
                                {"denom": float("nan")}])
def test_policy_loss_refuses(kw):
    assert _lib.lib.ab_policy_loss_fwd(C.byref(_rows()), C.byref(_policy(**kw)), P, P, P, P, P, None) == -1


def test_losses_refuse_the_rest():
    t = _rows()
    assert _lib.lib.ab_token_logp_fwd(C.byref(t), None, None, None, None) == -1
    assert _lib.lib.ab_token_logp_bwd(C.byref(t), P, P, 0, None, P, None) == -1 and _lib.lib.ab_token_logp_bwd(C.byref(t), P, None, 1, None, P, None) == -1
    assert _lib.lib.ab_policy_loss_fwd(C.byref(t), C.byref(_policy()), P, P, P, P, None, None) == -1
    wide = _rows(stride=128)
    assert _lib.lib.ab_policy_loss_grad(C.byref(wide), C.byref(_policy()), 1.0, P, P, P, P, None) == -1 and b"in place" in _lib.lib.ab_last_error()
    for pairs, steps, smoothing in ((2, 2, 0.0), (0, 3, 0.0), (1, 3, 1.5), (1, 3, float("nan"))):
        assert _lib.lib.ab_preference_loss_fwd(C.byref(t), pairs, steps, P, 0.1, smoothing, P, P, P, P, P, None) == -1


def test_gradients_over_other_rows_logits_are_refused():
    for t, at in ((_rows(stride=128), P + 16), (_rows(), P + 2), (_rows(), P + 1198), (_rows(stride=128), P - 1198)):     # (6 rows of 100 values of 2 bytes)
        assert _lib.lib.ab_policy_loss_grad(C.byref(t), C.byref(_policy()), 1.0, P, P, at, P, None) == -1 and b"overlaps" in _lib.lib.ab_last_error()
        assert _lib.lib.ab_token_logp_bwd(C.byref(t), P, P, 1, None, at, None) == -1 and b"overlaps" in _lib.lib.ab_last_error()


def test_python_entries_refuse_tensors_on_the_host():
    x = torch.zeros(2, 3, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError):
        ab.RWKV7_TRAIN_OP(None, x, x, x, x, x, x)
    with pytest.raises(RuntimeError):
        ab.layer_norm(x)
    ids = torch.zeros(2, 3, dtype=torch.int64)
    for f in (lambda: ab.token_logp(x, ids), lambda: ab.policy_loss(x, ids, None, ids.float()), lambda: ab.policy_loss_grad(x, ids, None, ids.float()),
              lambda: ab.preference_loss(x, ids, torch.zeros(2))):
        with pytest.raises(RuntimeError):
            f()


def test_python_entries_refuse_forward_mode_derivatives():
    """Before anything else of the arguments is looked at, so that it shows on the host."""
    import torch.autograd.forward_ad as forward_ad
    x, ids, one = torch.zeros(2, 3, 64), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        for f in (lambda: ab.RWKV7_TRAIN_OP(None, x, x, x, x, x, d), lambda: ab.layer_norm(x, None, d), lambda: ab.token_logp(d, ids), lambda: ab.policy_loss(x, ids, d, ids),
                  lambda: ab.policy_loss_grad(x, ids, None, x, ref_logp=d), lambda: ab.preference_loss(d, ids, one)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                f()


def test_python_entries_refuse_to_be_traced():
    """Tensors without memory, ahead of every other check."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x, ids, one = torch.empty(2, 3, 64, device="cuda", dtype=torch.float16), torch.empty(2, 3, device="cuda", dtype=torch.int64), torch.empty(2, device="cuda")
        for f in (lambda: ab.RWKV7_TRAIN_OP(None, x, x, x, x, x, x), lambda: ab.layer_norm(x), lambda: ab.token_logp(x, ids), lambda: ab.policy_loss(x, ids, None, one),
                  lambda: ab.policy_loss_grad(x, ids, None, one), lambda: ab.preference_loss(x, ids, one)):
            with pytest.raises(RuntimeError, match="cannot be traced"):
                f()


def test_struct_layouts_match_the_header():
    assert C.sizeof(_lib.Wkv7Seq) == 16 + 48 + 96 + 24 and C.sizeof(_lib.LogitRows) == 48 and C.sizeof(_lib.Policy) == 40


def test_the_range_checking_build_holds_asynchronous_copies_against_their_arrays():
    """What no loop bound stands next to: bulk copies, staged vectors and prefetches ask the extent of the caller's array for their final address."""
    import os
    from albatross_b200 import build
    seen = 0
    for name in ("loss.cu", "norm.cu", "wkv_train.cu"):
        lines = open(os.path.join(build.CSRC, name)).read().split("\n")
        for i, line in enumerate(lines):
            if any(op in line for op in ("bulk_g2s(", "prefetch.global", "bulk.prefetch", "cp.async.cg")):
                assert ".holds(" in " ".join(lines[max(0, i - 5):i + 2]), (name, i + 1)
                seen += 1
    assert seen >= 6
