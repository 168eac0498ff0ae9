"""neural_block_textures_b200: a B200 (sm_100a) Evolution Strategies training backend for
neural_block_textures, behind the reference's ntc_cuda::Trainer interface.

The product is libntc_b200.so (CUDA kernels + host engine + C ABI + the C++ class). This package
builds it (build.py), binds it (abi.py, trainer.py) and describes models and benchmark
configurations (model.py, synth.py, dct.py). The operators on the caller's own device tensors (symbols.py:
log probabilities of symbols and their gradient; optim.py: AdamW) take torch tensors and load torch on first use.
"""
from .abi import DctDesc, ModelDesc, QesDesc, load_library
from .model import CONFIGS, LevelSpec, ModelSpec, TrainConfig, config, qat_grid_table
from .trainer import Trainer

__all__ = ["Trainer", "ModelDesc", "QesDesc", "DctDesc", "load_library", "ModelSpec", "LevelSpec", "TrainConfig",
           "CONFIGS", "config", "qat_grid_table"]

# by name only: `import *` must not load torch
_TORCH_NAMES = {"symbol_logprobs": "symbols", "symbol_logprobs_grad": "symbols", "SymbolLogprobs": "symbols", "AdamW": "optim"}


def __getattr__(name):
    if name in _TORCH_NAMES:
        from importlib import import_module
        value = globals()[name] = getattr(import_module("." + _TORCH_NAMES[name], __name__), name)
        return value
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")


def __dir__():
    return sorted({*globals(), *_TORCH_NAMES})
