"""Classification heads of the reference on the gfx950 kernels, NHWC in.

State-dict keys equal the reference's (src/model.py:11-175, :308-316):
  cbam.ChannelGate.mlp.{1,3}.*, cbam.SpatialGate.spatial.{conv.weight,bn.*},
  query/key/value/output_projection.*, classifier.{2,4,7}.* (attention head);
  relative_position_table, residual_scale, residual_norm_{weight,bias} only where its options ask for them;
  {3,6}.* (simple head, an nn.Sequential).
"""
import math

import torch
import torch.nn as nn
import torch.nn.functional as F


class _BasicConv(nn.Module):
    def __init__(self):
        super().__init__()
        self.conv = nn.Conv2d(2, 1, 7, 1, 3, bias=False)
        self.bn = nn.BatchNorm2d(1, eps=1e-5, momentum=0.01, affine=True)


class _ChannelGate(nn.Module):
    def __init__(self, c, r=16):
        super().__init__()
        self.mlp = nn.Sequential(nn.Identity(), nn.Linear(c, c // r), nn.ReLU(), nn.Linear(c // r, c))


class _SpatialGate(nn.Module):
    def __init__(self):
        super().__init__()
        self.spatial = _BasicConv()


class CBAM(nn.Module):
    """Channel gate then spatial gate (src/model.py:96-108); x: NHWC."""

    def __init__(self, c, r=16):
        super().__init__()
        self.ChannelGate = _ChannelGate(c, r)
        self.SpatialGate = _SpatialGate()

    def forward(self, x):
        from . import head_ops
        return head_ops.cbam_forward(self, x)


class MultiHeadAttentionClassifier(nn.Module):
    """CBAM -> 8-head self-attention over H*W tokens with residual -> avgpool -> LayerNorm -> MLP
    (src/model.py:112-175); x: NHWC feature map, returns fp32 logits [B, num_classes].

    Beyond the reference, off by default (the state dict then has the reference's keys):
      relative_position_buckets=n  adds a learned bias to every attention score by the bucket of (dy, dx) between the two
          positions, n buckets an axis up to relative_position_distance (relpos.RelativePositionBuckets). The table
          `relative_position_table` [n * n, heads] starts at zero, so a head loaded from a checkpoint without it starts as it
          was, and maps of any size up to the operator's limits are taken where the default path holds 256 tokens.
      residual_norm="rms" or "layer"  scales the attention branch by a learned `residual_scale` per channel (from 1) and pools
          the norm of the residual stream instead of the stream itself (block_norm.gated_residual_norm)."""

    def __init__(self, feature_dim, num_heads=8, num_classes=1, dropout=0.2, relative_position_buckets=0,
                 relative_position_distance=128, residual_norm=None):
        super().__init__()
        assert feature_dim % num_heads == 0, "feature_dim must be divisible by num_heads"
        self._check_options(feature_dim, num_heads, relative_position_buckets, relative_position_distance, residual_norm)
        self.feature_dim, self.num_heads, self.head_dim = feature_dim, num_heads, feature_dim // num_heads
        self.cbam = CBAM(feature_dim)
        self.query = nn.Linear(feature_dim, feature_dim)
        self.key = nn.Linear(feature_dim, feature_dim)
        self.value = nn.Linear(feature_dim, feature_dim)
        self.attention_dropout = nn.Dropout(dropout)
        self.output_projection = nn.Linear(feature_dim, feature_dim)
        self.classifier = nn.Sequential(
            nn.AdaptiveAvgPool2d(1), nn.Flatten(), nn.LayerNorm(feature_dim), nn.Dropout(dropout),
            nn.Linear(feature_dim, 512), nn.ReLU(), nn.Dropout(dropout), nn.Linear(512, num_classes))
        self.relative_position_buckets = int(relative_position_buckets or 0)
        self.relative_position_distance = int(relative_position_distance)
        self.residual_norm = residual_norm
        n = self.relative_position_buckets
        self.relative_position_table = nn.Parameter(torch.zeros(n * n, num_heads)) if n else None
        self.residual_scale = nn.Parameter(torch.ones(feature_dim)) if residual_norm else None
        self.residual_norm_weight = nn.Parameter(torch.ones(feature_dim)) if residual_norm else None
        self.residual_norm_bias = nn.Parameter(torch.zeros(feature_dim)) if residual_norm == "layer" else None
        self._position_plans = {}

    @staticmethod
    def _check_options(feature_dim, num_heads, buckets, distance, norm):
        if buckets:
            head_dim = feature_dim // num_heads
            if head_dim % 8 or head_dim > 128:
                raise ValueError(f"relative_position_buckets needs heads whose width is a multiple of 8 up to 128 (got {head_dim})")
            if buckets < 4 or buckets % 4 or distance <= buckets // 4:
                raise ValueError(f"relative_position_buckets must be a multiple of 4 and relative_position_distance beyond its quarter (got {buckets}, {distance})")
        if norm not in (None, "rms", "layer"):
            raise ValueError(f"residual_norm is 'rms', 'layer' or None (got {norm!r})")

    def position_plan(self, height, width, device):
        """The buckets of a height x width map, built the first time a map of that size comes and kept."""
        key = (height, width, device)
        if key not in self._position_plans:
            from .relpos import RelativePositionBuckets
            n = self.relative_position_buckets
            plan = RelativePositionBuckets(height, width, n, self.relative_position_distance, device=device)
            if height == 1:      # one row of buckets: the same table serves it
                plan = RelativePositionBuckets.from_index(height, width, plan.index, n * n, device=device)
            self._position_plans[key] = plan
        return self._position_plans[key]

    def forward(self, x):
        from . import head_ops
        return head_ops.mha_head_forward(self, x)


class SimpleHead(nn.Sequential):
    """AdaptiveAvgPool2d(1) -> Flatten -> Dropout -> Linear(C,512) -> ReLU -> Dropout -> Linear(512,n)
    (src/model.py:308-316); same child indices as the reference's nn.Sequential."""

    def __init__(self, feature_dim, num_classes, dropout=0.2):
        super().__init__(nn.AdaptiveAvgPool2d(1), nn.Flatten(), nn.Dropout(dropout), nn.Linear(feature_dim, 512),
                         nn.ReLU(), nn.Dropout(dropout), nn.Linear(512, num_classes))

    def forward(self, x):
        from . import head_ops
        return head_ops.simple_head_forward(self, x)
