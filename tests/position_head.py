"""The attention head with its optional position bias and residual norm, in plain torch operations on the CPU."""
import math

import torch
import torch.nn as nn

from oracle import effnet_b3 as O


class PositionHead(O.MultiHeadAttentionClassifier):
    """Same parameters as heads.MultiHeadAttentionClassifier with relative_position_buckets and residual_norm; the buckets of
    one axis are worked out here again, distance by distance."""

    def __init__(self, feature_dim, num_heads, num_classes, dropout=0.0, buckets=0, distance=128, norm=None):
        super().__init__(feature_dim, num_heads, num_classes, dropout)
        self.buckets, self.distance, self.norm = buckets, distance, norm
        if buckets:
            self.relative_position_table = nn.Parameter(torch.zeros(buckets * buckets, num_heads))
        if norm:
            self.residual_scale = nn.Parameter(torch.ones(feature_dim))
            self.residual_norm_weight = nn.Parameter(torch.ones(feature_dim))
            if norm == "layer":
                self.residual_norm_bias = nn.Parameter(torch.zeros(feature_dim))

    def _axis_bucket(self, d):
        half, exact = self.buckets // 2, self.buckets // 4
        n = abs(d)
        if n >= exact:
            n = min(half - 1, exact + int(math.log(n / exact) / math.log(self.distance / exact) * (half - exact)))
        return n + (half if d > 0 else 0)

    def bias(self, H, W):
        rows = [[self._axis_bucket(j // W - i // W) * self.buckets + self._axis_bucket(j % W - i % W) for j in range(H * W)] for i in range(H * W)]
        return self.relative_position_table[torch.tensor(rows)].permute(2, 0, 1)

    def forward(self, x):
        x = self.cbam(x)
        B, C, H, W = x.shape
        t = x.reshape(B, C, H * W).permute(0, 2, 1)
        sp = lambda y: y.reshape(B, H * W, self.num_heads, self.head_dim).transpose(1, 2)      # noqa: E731
        q, k, v = sp(self.query(t)), sp(self.key(t)), sp(self.value(t))
        s = q @ k.transpose(-2, -1) / math.sqrt(self.head_dim)
        if self.buckets:
            s = s + self.bias(H, W)
        a = self.output_projection((torch.softmax(s, -1) @ v).transpose(1, 2).reshape(B, H * W, C))
        if not self.norm:
            y = t + a
        else:
            y = t + self.residual_scale * a
            if self.norm == "layer":
                y = y - y.mean(-1, keepdim=True)
            y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + 1e-6) * self.residual_norm_weight
            if self.norm == "layer":
                y = y + self.residual_norm_bias
        return self.classifier(y.permute(0, 2, 1).reshape(B, C, H, W))
