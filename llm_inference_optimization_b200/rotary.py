"""Rotary positions: the frequencies of a model and the rotation of query and key rows by them.

The reference leaves both to Hugging Face (benchmarks/llama_integration_benchmark.py:152-160).  A ``RotaryEmbedding``
holds one model's frequencies on one device; ``apply`` rotates rows (or takes the gradient back through the rotation), and
``paged.append_tokens`` takes the object to rotate tokens on their way into a cache.
"""
from __future__ import annotations

import math

import torch
from torch import Tensor

from . import _C, _lib, _workspace

_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
_SCALING_KEYS = {"linear": {"factor"}, "ntk": {"factor"},
                 "llama3": {"factor", "low_freq_factor", "high_freq_factor", "original_max_position"},
                 "yarn": {"factor", "original_max_position"}}
_SCALING_OPTIONAL = {"yarn": {"beta_fast", "beta_slow", "attention_factor"}}


def frequencies(rotary_dim: int, theta: float, scaling: dict | None = None) -> tuple[list[float], float]:
    """Angle per position of every pair (radians, 64-bit floats) and the factor on the rotated values.

    ``scaling`` stretches a model to contexts beyond the one it was trained on; ``type`` is one of

    * ``"linear"``: all frequencies divided by ``factor``;
    * ``"ntk"``: ``theta`` grown by ``factor ** (R / (R - 2))``, so that the slowest pair is slowed by ``factor``;
    * ``"llama3"``: pairs that turn more than ``high_freq_factor`` times over ``original_max_position`` tokens are kept, those
      that turn less than ``low_freq_factor`` times divided by ``factor``, those between blended;
    * ``"yarn"``: a ramp over the pairs between ``beta_fast`` (32) and ``beta_slow`` (1) turns over
      ``original_max_position`` tokens, and values multiplied by ``attention_factor`` (``0.1 ln(factor) + 1``, 1 for factors
      up to 1).
    """
    R = rotary_dim
    if not theta > 1.0 or not math.isfinite(theta):
        raise RuntimeError("rope theta must be finite and exceed 1")
    kind = None if scaling is None else scaling.get("type")
    if scaling is not None:
        if kind not in _SCALING_KEYS:
            raise RuntimeError(f"unknown rope scaling {kind!r}: one of {sorted(_SCALING_KEYS)}")
        given = set(scaling) - {"type"}
        need, may = _SCALING_KEYS[kind], _SCALING_OPTIONAL.get(kind, set())
        if not need <= given or not given <= need | may:
            raise RuntimeError(f"rope scaling {kind!r} takes {sorted(need)} and may take {sorted(may)}, got {sorted(given)}")
        try:   # (an optional value that is None counts as not given)
            scaling = {k: float(scaling[k]) for k in given if scaling[k] is not None or k in need}
        except (TypeError, ValueError) as e:
            raise RuntimeError(f"rope scaling values must be numbers: {e}") from None
        if any(not (v > 0.0 and math.isfinite(v)) for v in scaling.values()):
            raise RuntimeError("rope scaling values must be positive and finite")
    if kind == "ntk" and R > 2:
        theta = theta * scaling["factor"] ** (R / (R - 2))
    f = [theta ** (-2.0 * i / R) for i in range(R // 2)]
    if kind == "linear":
        return [x / scaling["factor"] for x in f], 1.0
    if kind == "llama3":
        low, high = scaling["low_freq_factor"], scaling["high_freq_factor"]
        if not high > low:
            raise RuntimeError("high_freq_factor must exceed low_freq_factor")

        def mix(x):
            turns = scaling["original_max_position"] * x / (2 * math.pi)
            keep = min(1.0, max(0.0, (turns - low) / (high - low)))
            return x * keep + x / scaling["factor"] * (1 - keep)
        return [mix(x) for x in f], 1.0
    if kind == "yarn":
        def pair(turns):   # the (fractional) pair that turns this often over the trained context
            return R * math.log(scaling["original_max_position"] / (2 * math.pi * turns)) / (2 * math.log(theta))
        low = max(math.floor(pair(scaling.get("beta_fast") or 32.0)), 0)
        high = min(math.ceil(pair(scaling.get("beta_slow") or 1.0)), R - 1)
        width = max(high - low, 0.001)
        ramp = [min(1.0, max(0.0, (i - low) / width)) for i in range(R // 2)]
        factor = scaling.get("attention_factor") or 0.1 * math.log(max(scaling["factor"], 1.0)) + 1.0
        return [x / scaling["factor"] * r + x * (1 - r) for x, r in zip(f, ramp)], factor
    return f, 1.0


class RotaryEmbedding:
    """The rotation of one model on one device.

    ``layout`` ``"half"`` pairs channel i with ``i + rotary_dim/2`` (Llama and most others), ``"interleaved"`` pairs
    neighbours ``(2i, 2i+1)``; ``rotary_dim`` (default: the whole head) is the part of the head that turns; ``scaling`` as for
    :func:`frequencies`.  Frequencies are kept as 64-bit fixed-point fractions of a turn per position, and their product with a
    position is exact.  What an angle is off by is the frequency's own rounding times the position: 2^-51 of the frequency and
    2^-65 of a turn, which is below the rounding of a 32-bit sine up to positions of about 2^26 (1e-3 radians at 2^41)."""

    def __init__(self, head_dim: int, theta: float = 10000.0, *, rotary_dim: int | None = None, layout: str = "half",
                 scaling: dict | None = None, device="cuda"):
        R = head_dim if rotary_dim is None else int(rotary_dim)
        _C._require(layout in ("half", "interleaved"), "layout must be 'half' or 'interleaved'")
        _C._require(0 < R <= head_dim and R % 2 == 0, f"rotary_dim must be even and in 2..{head_dim}")
        self.head_dim, self.rotary_dim, self.layout, self.theta = int(head_dim), R, layout, float(theta)
        freqs, self.factor = frequencies(R, float(theta), scaling)
        # round(f / 2 pi * 2^64), modulo a whole turn, as the signed 64-bit numbers torch holds
        turns = [round(math.ldexp(f / (2 * math.pi), 64)) % (1 << 64) for f in freqs]
        self.turns = torch.tensor([t - (1 << 64) if t >> 63 else t for t in turns], dtype=torch.int64, device=device)

    def kernel_args(self, head_dim: int, device: torch.device):
        """What the kernels take of this object, for rows of ``head_dim`` channels on ``device``."""
        if self.head_dim != head_dim or self.turns.device != device:
            raise RuntimeError(f"the rotation is for head_dim {self.head_dim} on {self.turns.device}, not {head_dim} on {device}")
        return self.turns.data_ptr(), self.rotary_dim, self.layout == "interleaved", self.factor

    def apply(self, positions: Tensor, q: Tensor, k: Tensor | None = None, *, adjoint: bool = False, inplace: bool = False):
        """Rotate ``q [T,Hq,D]`` (and ``k [T,Hk,D]``) at ``positions [T]`` (int32 or int64) in one launch.

        fp16, bf16 or fp32 (both alike; arithmetic in fp32), any strides with contiguous channels, for example slices of a
        fused projection.  Returns new contiguous tensors, or the inputs with ``inplace`` (whose rows must not share memory).  ``adjoint`` applies the
        transposed map: given gradients of the outputs it returns those of the inputs.  No autograd graph is recorded, and
        inputs that would need one are refused."""
        _C._require(q.is_cuda and q.dim() == 3 and q.dtype in _DTYPES, "q must be an fp16, bf16 or fp32 CUDA tensor [T,H,head_dim]")
        dev = q.device
        T, Hq, D = q.shape
        st, sh, sd = q.stride()
        freqs, R, inter, factor = self.kernel_args(D, dev)
        pos64 = positions.dtype is torch.int64
        _C._require((pos64 or positions.dtype is torch.int32) and positions.shape == (T,) and positions.is_contiguous()
                    and positions.device == dev, "positions must be a contiguous int32 or int64 [T] tensor on q's device")
        _C._require(sd == 1 or D == 1, "the channels of q must be contiguous")
        _C._require(not (torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad))),
                    "apply records no autograd graph: call it under no_grad and use adjoint=True for the gradient")
        qo = q if inplace else torch.empty_like(q, memory_format=torch.contiguous_format)
        Hk, kp, kop, ko, strides = 0, None, None, None, (0, 0)
        if k is not None:
            _C._require(k.dim() == 3 and k.dtype is q.dtype and k.shape[0] == T and k.shape[2] == D and k.stride(2) == 1
                        and k.device == dev, "k must be [T,Hk,head_dim] of q's dtype on q's device with contiguous channels")
            Hk, kp = k.shape[1], k.data_ptr()
            ko = k if inplace else torch.empty_like(k, memory_format=torch.contiguous_format)
            kop, strides = ko.data_ptr(), k.stride()[:2]
        if Hq + Hk:
            rc = _lib.load().skv_rotary(
                q.data_ptr(), kp, qo.data_ptr(), kop, _DTYPES[q.dtype], positions.data_ptr(), pos64, freqs, T, Hq, Hk, D, R, inter,
                factor, adjoint, st, sh, *strides, *((st, sh) if inplace else (Hq * D, D)), *(strides if inplace else (Hk * D, D)),
                dev.index, _workspace.stream(dev.index))
            if rc:
                _lib.check(rc, "rotary")
        if inplace:   # autograd then refuses a backward pass that needs the rows as they were
            torch.autograd.graph.increment_version(q if k is None else (q, k))
        return qo if k is None else (qo, ko)
