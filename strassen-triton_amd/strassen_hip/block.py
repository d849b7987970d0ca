"""The operators around the Linear layers of a decoder block, on the kernels of libstrassen_hip.so: the product with bias,
activation and residual in its epilogue (linear_act), layer norm (layer_norm) and rotary positions (rotary), each with its
gradients.  The reference leaves them to torch (model/model.py:4-32, model/layers.py:59-221).

Argument checks, memory and the autograd nodes are in csrc/sthip_torch.cpp (module _sthip_torch).  As in ops.py torch supplies
device memory, streams and the autograd graph only, and there is no CPU path.  Calls run on the current stream of their
tensors' device; workspaces come from torch's allocator at every call, so captured graphs share none.  Wrong arguments raise
ValueError or TypeError, a failing C-ABI call SthipError; gradients cannot be differentiated again.  Forward-mode derivatives,
torch.func transforms, traces and tensor subclasses are refused (RuntimeError): the operators would count as constants in them.  Under capture, a
leaf that a living eager graph on the default stream uses is refused (RuntimeError), whether it is an operand or one was computed
from it: torch's engine would end the process over it.
"""
from __future__ import annotations

import importlib.machinery
import importlib.util
import math
import os

import torch

from . import _capi

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
_LAYOUTS = {"half": False, "interleaved": True}
TORCH_LIB_PATH = os.path.join(os.path.dirname(_capi.LIB_PATH), "_sthip_torch.so")

_module = None


def _ext():
    """_sthip_torch, loaded once, with the C-ABI library before it."""
    global _module
    if _module is None:
        _capi.load()
        if not os.path.exists(TORCH_LIB_PATH):
            raise ImportError(f"{TORCH_LIB_PATH} is missing: build it with `python strassen-triton_amd/build.py`. "
                              "There is no fallback implementation.")
        loader = importlib.machinery.ExtensionFileLoader("_sthip_torch", TORCH_LIB_PATH)
        module = importlib.util.module_from_spec(importlib.util.spec_from_file_location("_sthip_torch", TORCH_LIB_PATH, loader=loader))
        loader.exec_module(module)
        _module = module
    return _module


def linear_act(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *, activation: str = "none",
               residual: torch.Tensor | None = None) -> torch.Tensor:
    """residual + activation(x @ weight.T + bias), differentiable, as one product whose epilogue does the rest
    (sthip_linear_act_forward).  x: (..., in_features), weight: (out_features, in_features), residual: (..., out_features);
    all of one type (float32, float16, bfloat16).  activation: "none", "relu", "gelu", "gelu_tanh" or "silu".  The product is a
    classical one (no Strassen levels); everything after it happens on its fp32 sums, which are rounded once."""
    try:
        act = ACTIVATIONS[activation]
    except KeyError:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}") from None
    return (_module or _ext()).linear_act(x, weight, bias, residual, act)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, *, eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(variance + eps) * weight + bias over the last dimension, differentiable (sthip_layer_norm_forward).
    weight and bias: one element a column, of x's type or both float32; either may be None.  Statistics and sums are fp32; the
    gradients of weight and bias are summed over the rows in a fixed order."""
    return (_module or _ext()).layer_norm(x, weight, bias, eps)


def rotary_frequencies(rotary_dim: int, *, base: float = 10000.0, scaling: str = "none", factor: float = 1.0, trained_length: int = 4096,
                       fast_turns: float = 32.0, slow_turns: float = 1.0, device="cuda") -> tuple[torch.Tensor, float]:
    """Radians a position of each of the rotary_dim / 2 pairs (float64, on `device`) and the factor that cosine and sine are
    multiplied with, for rotary().  Pair i turns by base ** (-2 i / rotary_dim); for contexts `factor` times trained_length:

    "linear"  every frequency divided by factor (position interpolation);
    "ntk"     base multiplied by factor ** (rotary_dim / (rotary_dim - 2)), which divides the slowest frequency by factor and
              leaves the fastest;
    "yarn"    a frequency that makes fast_turns or more turns within trained_length stays, one that makes slow_turns or fewer is
              divided by factor, linear between; the second result is 0.1 ln(factor) + 1."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and at least 2, got {rotary_dim}")
    if scaling not in ("none", "linear", "ntk", "yarn"):
        raise ValueError(f"scaling must be none, linear, ntk or yarn, got {scaling!r}")
    if not (base > 0 and factor >= 1 and trained_length > 0 and fast_turns > slow_turns):
        raise ValueError("base and trained_length must be positive, factor at least 1, fast_turns above slow_turns")
    if scaling == "ntk" and rotary_dim > 2:
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    f = [base ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)]
    gain = 1.0
    if scaling == "linear":
        f = [v / factor for v in f]
    elif scaling == "yarn":
        def mixed(v):
            keep = min(max((trained_length * v / (2 * math.pi) - slow_turns) / (fast_turns - slow_turns), 0.0), 1.0)
            return v * keep + v / factor * (1 - keep)
        f, gain = [mixed(v) for v in f], 0.1 * math.log(factor) + 1.0
    return torch.tensor(f, dtype=torch.float64).to(device), gain


def rotary(q: torch.Tensor, k: torch.Tensor | None, frequencies: torch.Tensor, positions: torch.Tensor | None = None, *,
           layout: str = "half", gain: float = 1.0, first_position: int = 0, inplace: bool = False):
    """q and k with rotary positions (sthip_rotary), differentiable, in one launch.  q: (batch, tokens, heads, head_dim) or
    (tokens, heads, head_dim); k the same with its own number of heads, or None.  The first 2 * len(frequencies) elements of a
    head turn, the others are copied; layout "half" pairs i with i + len(frequencies), "interleaved" 2 i with 2 i + 1.
    frequencies, gain: rotary_frequencies.  positions: int32 or int64, (tokens,) or (batch, tokens); None counts from
    first_position.  Angles are formed in 64 bits: below 2^29 radians they keep
    fp32's accuracy, beyond they are off by their size times 2^-53.  inplace=True turns q and k where they lie, without a
    gradient: unit stride within a head, any other strides, and no element twice, neither within a tensor nor in both
    (ValueError).  Returns (q, k), or q alone where k is None."""
    try:
        interleaved = _LAYOUTS[layout]
    except KeyError:
        raise ValueError(f"layout must be one of {sorted(_LAYOUTS)}, got {layout!r}") from None
    out = (_module or _ext()).rotary(q, k, frequencies, positions, interleaved, gain, first_position, inplace)
    return out[0] if k is None else out
