"""Per-head norms and position rotation of query and key rows on the GPU.

``qk_norm_rope`` normalises every query and key head (RMS norm, where a weight
is given) and rotates it by its token's position, in one launch;
``paged_kv_write_rope`` does the same on the way into the paged cache, as
``paged_kv_write`` stores rows that are already rotated.  They stand in front
of the decode entry points in a serving step; the reference's models run these
as torch operations.  The checks and the launch are one call of the torch
binding (fasterkernels_amd/csrc/fsk_torch.cpp).  Inference only: inputs that
want gradients are refused.
"""
from __future__ import annotations

import torch

from fasterkernels_amd import native as nat

from .decode import _stream


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor | None, sin: torch.Tensor | None,
                 positions: torch.Tensor | None = None, *, q_weight: torch.Tensor | None = None,
                 k_weight: torch.Tensor | None = None, eps: float = 1e-6, interleaved: bool = False):
    """``(q_out, k_out)``: every head row of ``q`` [n, Hq, D] and ``k``
    [n, Hkv, D] (f16, bf16 or f32; any strides, e.g. views of one projection's
    output) normalised and rotated, as new contiguous tensors of the same type.

    Per row x: y = x / sqrt(mean(x^2) + eps) * weight (``q_weight`` /
    ``k_weight`` [D]; None: y = x), then the pairs (t, t + R/2) of its first R
    dims, or (2t, 2t + 1) when ``interleaved``, turned by the angle of
    ``cos`` / ``sin`` [rows, R/2] at the token's row: (a cos - b sin, b cos +
    a sin).  R is a multiple of 16; dims past it keep y.  Computed in fp32 (a row
    whose sum of squares leaves its range, values past about 2^60, normalises to
    zero) and rounded once.  ``positions`` (int64 or int32 [n]; values outside the table
    take its first or last row) gives each token's row; None: token i takes row
    i mod rows (tables made for these very tokens, or for one of several
    sequences of the same length).  ``cos = sin = None``: norms only.
    """
    return nat.ext().qk_norm_rope(q, k, cos, sin, positions, q_weight, k_weight, float(eps), bool(interleaved),
                                  _stream(q))


def paged_kv_write_rope(q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, k_pool: torch.Tensor,
                        v_pool: torch.Tensor, slot_mapping: torch.Tensor, cos: torch.Tensor | None,
                        sin: torch.Tensor | None, positions: torch.Tensor | None = None, *,
                        q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
                        eps: float = 1e-6, interleaved: bool = False, k_scale: torch.Tensor | None = None,
                        v_scale: torch.Tensor | None = None, block_table: torch.Tensor | None = None,
                        bt_updates: torch.Tensor | None = None) -> torch.Tensor | None:
    """``paged_kv_write`` of ``k`` and ``v`` [n, Hkv, D] with the norm and
    rotation of ``qk_norm_rope`` applied to ``k`` on the way (rounded once, to
    the pool's type) and to ``q`` [n, Hq, D], which is returned as a new tensor
    (None in, None out).  ``v`` is stored as it is.

    Slots, scales and block-table updates are ``paged_kv_write``'s; a token
    whose slot is negative or past the pool is not stored, but its query is
    still rotated.  One launch on the current stream.
    """
    if not isinstance(k_pool, torch.Tensor):
        raise TypeError("k_pool must be a torch.Tensor")
    index = k_pool.get_device()
    return nat.ext().kv_write_rope(q, k, v, k_pool, v_pool, slot_mapping, cos, sin, positions, q_weight, k_weight,
                                   float(eps), bool(interleaved), k_scale, v_scale, block_table, bt_updates,
                                   nat.raw_stream(index) if index >= 0 else 0)
