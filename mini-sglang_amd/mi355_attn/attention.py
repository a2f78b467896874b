"""The operator boundary the Llama layers call (reference layers/attention.py:6-36): per-layer constants plus a
dispatch to `batch.attn_backend.forward(q=, k=, v=, layer=, batch=)`."""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn


class Attention(nn.Module):
    def __init__(self, layer_id: int, num_heads: int, num_kv_heads: int, head_dim: int, scale: Optional[float] = None, *,
                 logit_cap: float = 0.0, window: int = 0, slopes: Optional[torch.Tensor] = None):
        """logit_cap > 0 caps the scores (s -> logit_cap * tanh(s / logit_cap)), window > 0 lets a token see that many keys, its
        own included, and slopes (fp32 [num_heads], on the device) biases them by -slope * distance.  The reference's layers
        have none of the three.  A layer with any of them multiplies its scores by `scale` where that is given (1.0 too) and by
        head_dim^-0.5 otherwise; a layer with none does the latter whatever `scale` says, as the reference's backends do, which
        never pass it on."""
        super().__init__()
        self.layer_id = layer_id
        self.num_heads = num_heads
        self.num_kv_heads = num_kv_heads
        self.head_dim = head_dim
        self.scale = 1.0 if scale is None else scale          # the reference's attribute and its default
        self.score_scale = scale
        self.logit_cap = float(logit_cap)
        self.window = int(window)
        self.slopes = slopes

    def forward(self, q, k, v, batch):
        return batch.attn_backend.forward(q=q, k=k, v=v, layer=self, batch=batch)
