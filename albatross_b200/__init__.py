"""albatross_b200 — sm_100a kernels for the RWKV-7 decode hot path behind the reference's model API.

`RWKV_x070`, `RWKV7_OP` and `RWKV7_BATCH_OP` mirror reference/rwkv7.py; `RWKV7_TRAIN_OP`, `layer_norm`, `token_logp`, `policy_loss`,
`policy_loss_grad` and `preference_loss` are operators with gradients, `grad_norm` and `clip_grad_norm` what comes after them (train.py);
`sampler_batch`, `linear_int4` and `quantize_int4` serve a token (serve.py); `synth` builds seeded
synthetic checkpoints in the reference's key schema; `build` compiles the CUDA library.
Importing the model needs the built library (python -m albatross_b200.build).
"""
import importlib

_TRAIN = ["RWKV7_TRAIN_OP", "layer_norm", "token_logp", "policy_loss", "policy_loss_grad", "preference_loss", "grad_norm", "clip_grad_norm"]
_SERVE = ["sampler_batch", "linear_int4", "quantize_int4", "Int4Matrix"]
__all__ = ["RWKV_x070", "RWKV7_OP", "RWKV7_BATCH_OP", "sampler_simple_batch"] + _TRAIN + _SERVE


def __getattr__(name):
    if name not in __all__:
        raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
    value = getattr(importlib.import_module(".train" if name in _TRAIN else ".serve" if name in _SERVE else ".rwkv7", __name__), name)
    globals()[name] = value     # found directly from now on
    return value
