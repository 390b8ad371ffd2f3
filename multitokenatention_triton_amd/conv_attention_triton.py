"""Fused conv-attention forward (HIP-backed).

Mirrors TritonConvAttention (conv_attention_triton.py:476-502) and TritonAttention
(:359-452) of the reference.  O = softmax(mask(conv(mask0(Q K^T))) * scale) V is computed
by ``mta_conv_attn_fwd`` with score tiles kept in LDS; causal fp32 forwards without
gradients run as scores, conv, softmax and P V where that is faster, by way of at most
512 MB of scores in scratch tensors.  The reference also returns the (B,H,S,S) QK scratch it fills in global
memory; this build keeps none and returns ``None`` in its place (the reference's own harness accepts that,
compare_conv_attention2.py:171-187).
"""
from __future__ import annotations

import torch
import torch.nn as nn

from . import _lib, ops


class TritonAttention(torch.autograd.Function):
    """apply(Q, K, V, W, causal, softmax_scale) -> (O, None); Q,K,V are (B,H,S,D), W is (H,R,S)."""

    @staticmethod
    def forward(ctx, Q, K, V, W, causal, softmax_scale):
        # shape checks of conv_attention_triton.py:369-370
        assert W.shape[0] == Q.shape[1]
        assert Q.shape[-1] == K.shape[-1] and K.shape[-1] == V.shape[-1]
        # the row-wise log-sum-exp is what the reference keeps for a backward pass (its `M`,
        # conv_attention_triton.py:402-404, 445); it is kept on ctx the same way
        out, lse = ops.conv_attn_fwd(Q, K, V, W, causal, softmax_scale, return_lse=True)
        ctx.save_for_backward(Q, K, V, out, lse)
        ctx.softmax_scale = softmax_scale
        ctx.causal = causal
        ctx.mark_non_differentiable(out)
        return out, None

    @staticmethod
    def backward(ctx, dO, dQK):
        # the reference's backward is itself a stub that calls kernels it never defines
        # (conv_attention_triton.py:455-473)
        raise NotImplementedError("TritonAttention has no backward (neither has the reference: "
                                  "conv_attention_triton.py:455-473)")


class TritonConvAttention(nn.Module):
    def __init__(self, channels, kernel_size, causal=False):
        super().__init__()
        self.channels = channels
        self.kernel_size = tuple(kernel_size) if isinstance(kernel_size, (tuple, list)) else (kernel_size, kernel_size)
        self.causal = causal
        self.weight = nn.Parameter(torch.empty(channels, *self.kernel_size))
        self._init_parameters()

    def _init_parameters(self):
        # the reference's default (conv_attention_triton.py:494-499): 1.0 at [R//2, S//2]
        with torch.no_grad():
            self.weight.zero_()
            self.weight[:, self.kernel_size[0] // 2, self.kernel_size[1] // 2] = 1.0

    def forward(self, Q, K, V, causal, softmax_scale):
        weight = self.weight
        if torch.is_grad_enabled() and (Q.requires_grad or K.requires_grad or V.requires_grad or weight.requires_grad):
            return TritonAttention.apply(Q, K, V, weight, causal, softmax_scale)
        # (nothing to differentiate: no row statistic is written)
        assert weight.size(0) == Q.size(1)
        return _lib.host().conv_attn(Q, K, V, weight, causal, softmax_scale), None

    @property
    def decode_query_rows(self) -> int:
        """Queries per sequence that ``decode`` needs a cache to keep."""
        return self.kernel_size[0]

    def decode(self, cache, softmax_scale=None, window=0):
        """The row of the newest token of every slot of a ``PagedCache`` that got tokens in its last ``extend``: (slots, H, 1, D),
        zeros for the other slots.  Causal, whatever ``self.causal`` says (forward() takes it as an argument and does not read
        that either); ``window``: a row sees that many keys at most, itself included (0: all).  What forward() rounds to the dtype
        between its stages stays in fp32 here.  No gradients."""
        return _lib.host().conv_attn_decode(cache.k, cache.v, cache.q, cache.table, cache.state, cache.longest, self.weight.detach(), softmax_scale, window)
