"""sampling.py -- drawing the next token on the GPU (no counterpart in the
reference, whose generate() samples in Python)."""
from __future__ import annotations

from typing import Optional

import torch

import custom_ecc_cuda as ops


class Sampler:
    """Settings of ``custom_ecc_cuda.sample_tokens`` and the source of its
    uniform numbers.  Each setting is one number or a [B] tensor on the GPU.

        sampler = Sampler(temperature=0.7, top_k=50, top_p=0.9)
        token = sampler(logits)                       # [B] int64

    ``generator``: a CUDA generator for the numbers (default: torch's)."""

    def __init__(self, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, generator: Optional[torch.Generator] = None):
        self.temperature = temperature
        self.top_k = top_k
        self.top_p = top_p
        self.min_p = min_p
        self.generator = generator

    def uniform(self, out: torch.Tensor) -> torch.Tensor:
        """Fills ``out`` (float32, on the GPU) with numbers in [0, 1)."""
        return out.uniform_(generator=self.generator)

    def __call__(self, logits: torch.Tensor, uniform: Optional[torch.Tensor] = None,
                 return_logprobs: bool = False):
        """Tokens [B] of logits [B, V]; -1 for a row without a logit above -inf."""
        if uniform is None:
            uniform = self.uniform(torch.empty(logits.shape[0], dtype=torch.float32, device=logits.device))
        return ops.sample_tokens(logits, uniform, temperature=self.temperature, top_k=self.top_k, top_p=self.top_p,
                                 min_p=self.min_p, return_logprobs=return_logprobs)
