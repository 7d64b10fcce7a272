"""How a generation loop draws its tokens (``SelectiveRunner.generate``,
``MambaIntegerModel.generate``)."""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Union

import torch

from . import ops


@dataclass
class Sampling:
    """Parameters of ``ops.sample_tokens``: numbers, or tensors with a value a sequence (float32,
    top_k int32) where requests differ.  ``generator`` (of the logits' device) makes the random
    numbers; None: torch's own."""
    temperature: Union[float, torch.Tensor] = 1.0
    top_k: Union[int, torch.Tensor] = 0
    top_p: Union[float, torch.Tensor] = 1.0
    min_p: Union[float, torch.Tensor] = 0.0
    generator: Optional[torch.Generator] = None

    def draw(self, logits: torch.Tensor, scale: float = 1.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Tokens int64 [B] (in ``out``) from logits [B, V] (int32 ones count in ``scale``); a row
        without a token to draw gives -1, which is no token to go on with."""
        u = torch.rand(logits.shape[0], device=logits.device, generator=self.generator)
        return ops.sample_tokens(logits, u, temperature=self.temperature, top_k=self.top_k, top_p=self.top_p, min_p=self.min_p,
                                 scale=scale, out=out)
