"""``LatentAttnDecode``: the decode step of latent attention (MLA) in its absorbed form, the
cache side of fastkernels/tasks/baseline/L2/mla_attention_impl.py.

The cache holds one row a token, [latent | rotated key], which all heads share;
``RotaryEmbedding.forward_store_latent`` writes it.  The projections on either side (the
queries into the latent space, the output out of it) are the caller's matrix products.
"""
from __future__ import annotations

import sys
from pathlib import Path

import torch
import torch.nn as nn

try:
    import fastkernels_amd  # noqa: F401
except ImportError:  # loaded by file path from the reference harness
    sys.path.insert(0, str(Path(__file__).resolve().parents[3]))
from fastkernels_amd import ops


class LatentAttnDecode(nn.Module):
    def __init__(self, num_heads: int, softmax_scale: float, latent_size: int = 512,
                 rope_size: int = 64):
        super().__init__()
        if (latent_size, rope_size) != (512, 64):
            raise NotImplementedError(f"LatentAttnDecode (gfx950): {latent_size} + {rope_size} is "
                                      "not built (512 + 64)")
        self.num_heads = num_heads
        self.softmax_scale = float(softmax_scale)
        self.latent_size = latent_size

    def forward(self, q, cache, cache_seqlens, block_table, cache_scale=None, cu_seqlens_q=None,
                max_seqlen_q: int | None = None, out=None, lse=None):
        """q [rows, num_heads, 576] over the latent cache [num_blocks, block_size, 576] (bf16, or
        float8_e4m3fn times cache_scale); returns [rows, num_heads, 512], and writes lse (float32
        [num_heads, rows]) if given.  One row per sequence, or the rows of cu_seqlens_q, at most
        max_seqlen_q (then required) per sequence."""
        if q.dim() != 3 or q.shape[1] != self.num_heads:
            raise ValueError(f"LatentAttnDecode: q must be [rows, {self.num_heads}, 576]")
        if out is None:
            out = q.new_empty((q.shape[0], self.num_heads, self.latent_size))
        call = torch.ops.fastkernels_amd.latent_decode if torch.compiler.is_compiling() \
            else ops.latent_decode
        call(out, q, cache, block_table.to(torch.int32), cache_seqlens.to(torch.int32),
             self.softmax_scale, cache_scale, cu_seqlens_q, max_seqlen_q, lse)
        return out
