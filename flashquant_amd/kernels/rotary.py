"""Rotary positions: the frequencies, the rotation of queries and keys with its gradient, and the rotation that stores keys and
values into a 16-bit paged cache.  The reference has none of its own: keys reach its cache rotated
(src/flashquant/vllm/impl.py:220-263)."""
from __future__ import annotations

import math
from typing import Optional, Sequence, Tuple

import torch

from flashquant_amd.kernels._native import native, require_gpu


def rotary_frequencies(
    rotary_dim: int,
    base: float = 10000.0,
    scaling: str = "none",
    *,
    factor: float = 1.0,
    original_max_position: int = 0,
    beta_fast: float = 32.0,
    beta_slow: float = 1.0,
    low_freq_factor: float = 1.0,
    high_freq_factor: float = 4.0,
    factors: Optional[Sequence[float]] = None,
    device: Optional[torch.device] = None,
) -> Tuple[torch.Tensor, float]:
    """``(inv_freq, scale)`` for ``rotary_embedding``: float64 ``base ** (-2 i / rotary_dim)``, i < rotary_dim / 2, and the factor
    on queries and keys, for contexts ``factor`` times as long as a model was trained with (``original_max_position``):

    * ``none``
    * ``linear``: all frequencies divided by ``factor``
    * ``ntk``: the base times ``factor ** (rotary_dim / (rotary_dim - 2))``, which divides the lowest frequency by ``factor``
    * ``yarn``: a pair that turns more than ``beta_fast`` times over the original length keeps its frequency, one that turns less
      than ``beta_slow`` times has it divided, with a ramp over the pairs between; queries and keys times 0.1 ln(factor) + 1
    * ``bands``: the same by wavelength, from original / ``high_freq_factor`` (kept) to original / ``low_freq_factor`` (divided)
    * ``factors``: pair i divided by ``factors[i]``; queries and keys times sqrt(1 + ln(factor) / ln(original))
    """
    if rotary_dim < 2 or rotary_dim % 2 != 0:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    if not base > 0.0 or not factor > 0.0:
        raise ValueError("base and factor must be positive")
    if scaling in ("yarn", "bands") and original_max_position <= 0:
        raise ValueError(f"scaling '{scaling}' needs original_max_position")
    half = rotary_dim // 2
    pair = torch.arange(half, dtype=torch.float64)
    if scaling == "ntk":
        if rotary_dim == 2:
            raise ValueError("scaling 'ntk' needs a rotary_dim above 2")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    inv_freq = base ** (-pair / half)
    scale = 1.0
    if scaling in ("none", "ntk"):
        pass
    elif scaling == "linear":
        inv_freq = inv_freq / factor
    elif scaling == "yarn":
        if base == 1.0 or not beta_fast > 0.0 or not beta_slow > 0.0:
            raise ValueError("scaling 'yarn' needs a base other than 1 and positive beta_fast and beta_slow")

        def pair_of(turns: float) -> float:      # the pair that turns so many times over the original length
            return rotary_dim * math.log(original_max_position / (turns * 2 * math.pi)) / (2 * math.log(base))

        low, high = max(math.floor(pair_of(beta_fast)), 0), min(math.ceil(pair_of(beta_slow)), rotary_dim - 1)
        divided = ((pair - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
        inv_freq = inv_freq * (1.0 - divided) + inv_freq / factor * divided
        scale = 0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0
    elif scaling == "bands":
        if not high_freq_factor > low_freq_factor:
            raise ValueError("high_freq_factor must be above low_freq_factor")
        turns = original_max_position * inv_freq / (2 * math.pi)
        kept = ((turns - low_freq_factor) / (high_freq_factor - low_freq_factor)).clamp(0.0, 1.0)
        inv_freq = inv_freq * kept + inv_freq / factor * (1.0 - kept)
    elif scaling == "factors":
        if factors is None or len(factors) != half:
            raise ValueError(f"scaling 'factors' needs {half} factors")
        inv_freq = inv_freq / torch.tensor(list(factors), dtype=torch.float64)
        if factor > 1.0:
            if original_max_position <= 1:
                raise ValueError("scaling 'factors' with a factor above 1 needs original_max_position")
            scale = math.sqrt(1.0 + math.log(factor) / math.log(original_max_position))
    else:
        raise ValueError(f"unknown scaling '{scaling}'")
    return inv_freq.to(device) if device is not None else inv_freq, scale


def rotary_embedding(
    q: torch.Tensor,
    k: Optional[torch.Tensor],
    positions: torch.Tensor,
    inv_freq: torch.Tensor,
    *,
    interleaved: bool = False,
    scale: float = 1.0,
    inverse: bool = False,
    out: Optional[Tuple[torch.Tensor, Optional[torch.Tensor]]] = None,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Rotary positions on ``q`` (tokens, H_Q, D) and ``k`` (tokens, H_K, D) or None, float16, bfloat16 or float32, or both with a
    batch before the tokens: each pair i of the first ``2 * len(inv_freq)`` coordinates of a head, ``(i, i + len(inv_freq))`` or, where
    ``interleaved``, ``(2 i, 2 i + 1)``, is turned by ``positions * inv_freq[i]`` (``inverse``: back) and multiplied by ``scale``; the
    rest of the head is copied.  ``positions`` (tokens,) or (batch, tokens), int32 or int64; ``inv_freq`` float64, from
    ``rotary_frequencies``.  Rows may be strided (slices of one matrix product).

    ``out`` = (q_out, k_out): written instead of new tensors; either may be its input itself.  Differentiable with respect to q and
    k, any number of times and in forward mode too, where ``out`` is not given.  As with torch's own operators, a backward pass is
    captured in a graph only while no record of the same leaves from outside the capture is alive."""
    require_gpu(q, "q")
    q_out, k_out = (None, None) if out is None else out
    return native().rotary_embedding(q, k, positions, inv_freq, interleaved, scale, inverse, q_out, k_out)


def rotary_paged_store(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    positions: torch.Tensor,
    slot_mapping: torch.Tensor,
    inv_freq: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    *,
    interleaved: bool = False,
    scale: float = 1.0,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """``rotary_embedding`` of ``q`` (tokens, H_Q, D) and ``k`` (tokens, H_KV, D), with the rotated keys and ``v`` written into
    ``key_cache`` / ``value_cache`` (num_blocks, block_size, H_KV, D) at flat slot ``slot_mapping[i]``, in one launch; returns the
    rotated queries (``out``: new memory, or ``q`` itself).  Tokens beyond ``len(slot_mapping)`` and slots outside the cache are not
    stored.  float16 or bfloat16.  The caches may be strided (halves of one tensor, heads before tokens); they may not share memory
    with the other operands.  No gradient is recorded."""
    require_gpu(q, "q")
    return native().rotary_paged_store(q, k, v, positions, slot_mapping, inv_freq, key_cache, value_cache, interleaved, scale, out)
