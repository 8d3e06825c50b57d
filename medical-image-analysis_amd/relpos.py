"""Multi-head attention with a learned relative position bias, on the gfx950 kernels of csrc/relpos.hip: maps of up to 2 ** 22
tokens and series of up to 2 ** 26, masked keys, few queries against many keys, gradients of everything including the bias table
(whose backward holds up to L * L / 32 floats an image and head on a map of L tokens, L * L / 64 on a series)."""
import math

import numpy as np
import torch

from . import ops
from ._lib import nodes
from .ops import _DT


class RelativePositionBuckets:
    """Which bucket (= row of a bias table) every offset between two positions of an H x W map falls into; a sequence is a map
    of height 1. Positions are numbered row by row, and the offset (dy, dx) = position of the key - position of the query has
    the number (dy + H - 1) * (2 W - 1) + dx + W - 1 in `index`.

    The constructor buckets each axis on its own: half of num_buckets for each direction, half of those one distance each, the
    rest logarithmic up to max_distance and one for everything beyond; a map of several rows has num_buckets ** 2 rows of
    bias, a sequence num_buckets. from_index takes any assignment (one bucket per offset, shared buckets, ...).
    Built once and kept, like the weights: it holds the index and the offsets sorted by bucket on the device."""

    def __init__(self, height, width, num_buckets=32, max_distance=128, device="cuda"):
        if num_buckets < 4 or num_buckets % 4:
            raise ValueError(f"num_buckets must be a multiple of 4 (got {num_buckets})")
        if max_distance <= num_buckets // 4:
            raise ValueError(f"max_distance must exceed the {num_buckets // 4} exact distances (got {max_distance})")
        self._check_map(height, width)
        rows = 1 if height == 1 else num_buckets
        by, bx = self._axis(height, num_buckets, max_distance), self._axis(width, num_buckets, max_distance)
        index = by[:, None] * num_buckets + bx[None, :]
        self._set(height, width, index.reshape(-1), rows * num_buckets, device)

    @staticmethod
    def _axis(n, buckets, max_distance):
        if n == 1:
            return torch.zeros(1, dtype=torch.int64)
        d = torch.arange(1 - n, n, dtype=torch.float64)
        half, exact = buckets // 2, buckets // 4
        far = exact + ((d.abs().clamp(min=exact) / exact).log() / math.log(max_distance / exact) * (half - exact)).floor()
        return torch.where(d.abs() < exact, d.abs(), far.clamp(max=half - 1)).long() + half * (d > 0).long()

    @classmethod
    def from_index(cls, height, width, index, num_buckets=None, device="cuda"):
        """index: (2H - 1)(2W - 1) integers (any shape) on any device; num_buckets defaults to the largest + 1."""
        cls._check_map(height, width)
        index = torch.as_tensor(index)
        if index.dtype.is_floating_point or index.dtype.is_complex or index.dtype == torch.bool:
            raise TypeError(f"index holds integers (got {index.dtype})")
        self = cls.__new__(cls)
        self._set(height, width, index.detach().cpu().long().reshape(-1), num_buckets, device)
        return self

    @staticmethod
    def _check_map(height, width):
        if height < 1 or width < 1 or (height > 1 and (width > 896 or height * width > 1 << 22)) or (2 * height - 1) * (2 * width - 1) > 1 << 27:
            raise ValueError(f"a map of {height} x {width} is not supported (several rows: at most 896 wide and 2 ** 22 tokens; at most 2 ** 27 offsets)")

    def _set(self, height, width, index, num_buckets, device):
        n = (2 * height - 1) * (2 * width - 1)
        if index.numel() != n:
            raise ValueError(f"a map of {height} x {width} has {n} offsets (got an index of {index.numel()})")
        low, high = map(int, index.aminmax())
        num_buckets = high + 1 if num_buckets is None else int(num_buckets)
        if low < 0 or high >= num_buckets:
            raise ValueError(f"buckets {low}..{high} are not all in 0..{num_buckets - 1}")
        self.height, self.width, self.num_buckets = int(height), int(width), num_buckets
        count = torch.bincount(index, minlength=num_buckets)
        # 16-bit keys are sorted by radix: 0.2 ms for the 22201 offsets of a 75 x 75 map, 1.9 ms by torch's sort
        keys = index.numpy()
        order = torch.from_numpy((keys.astype(np.int16) if num_buckets <= 1 << 15 else keys).argsort(kind="stable"))
        packed = torch.cat((index, order, count.cumsum(0) - count, torch.tensor([n]))).to(torch.int32).to(device)
        self.index, self.order, self.start = packed[:n], packed[n:2 * n], packed[2 * n:]

    @property
    def device(self):
        return self.index.device


def _attend(name, q, k, v, B, Lq, Lk, heads, D, table, buckets, key_mask, scale, q_start, dropout_p, seed):
    dtype = q.dtype
    if dtype not in _DT or (k is not None and (k.dtype != dtype or v.dtype != dtype)):
        raise TypeError(f"{name}: queries, keys and values are all fp32 or all bf16 (got {', '.join(str(t.dtype) for t in (q, k, v) if t is not None)})")
    if D % 8 or not 8 <= D <= 128:
        raise ValueError(f"{name}: the head width must be a multiple of 8 up to 128 (got {D})")
    tokens = buckets.height * buckets.width
    q_start = int(q_start)
    if Lk > tokens or q_start < 0 or q_start + Lq > tokens:
        raise ValueError(f"{name}: {Lk} keys and {Lq} queries from {q_start} on do not fit a map of {buckets.height} x {buckets.width}")
    if table.shape != (buckets.num_buckets, heads) or table.dtype != torch.float32:
        raise ValueError(f"{name}: the table must be fp32 {(buckets.num_buckets, heads)} (got {table.dtype} {tuple(table.shape)})")
    if key_mask is not None and (key_mask.shape != (B, Lk) or key_mask.dtype not in (torch.bool, torch.uint8)):
        raise ValueError(f"{name}: key_mask must be bool {(B, Lk)}, true where a key counts (got {key_mask.dtype} {tuple(key_mask.shape)})")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 1e-30 < scale < 1e30:
        raise ValueError(f"{name}: scale must be positive (got {scale})")
    dropout_p = float(dropout_p)
    if not 0.0 <= dropout_p < 1.0:
        raise ValueError(f"{name}: dropout must be in [0, 1) (got {dropout_p})")
    device = q.get_device()
    for t in (q, k, v, table, buckets.index, key_mask):
        if t is not None and (device < 0 or t.get_device() != device):
            raise RuntimeError(f"{name} needs its tensors (and its buckets) on one MI355X device; there is no CPU path (got {t.device})")
    if dropout_p > 0.0 and seed is None:
        from .head_ops import _seed
        seed = _seed()
    return nodes().relpos(q, k, v, table, buckets.index, buckets.order, buckets.start, key_mask, buckets.height, buckets.width, buckets.num_buckets,
                          scale, q_start, dropout_p, int(seed or 0) & 0xFFFFFFFFFFFFFFFF, ops.seed_offset() or 0)


def relpos_attention(q, k, v, table, buckets, key_mask=None, scale=None, q_start=0, dropout_p=0.0, seed=None):
    """out[b, i, h] = sum_j softmax_j(scale * q[b, i, h] . k[b, j, h] + table[bucket(position of j - position of i), h]) v[b, j, h]

    q [B, Lq, heads, D], k and v [B, Lk, heads, D], fp32 or bf16, any strides (read in place when heads are contiguous rows at
    multiples of 16 bytes); D a multiple of 8 up to 128. buckets: a RelativePositionBuckets over a map of at least Lk tokens;
    key j is at token j, query i at token q_start + i (a new token against a series: q_start = Lk - 1). table: fp32
    [buckets.num_buckets, heads]. key_mask: bool [B, Lk], false = the key does not exist (what its rows hold is never read into a
    result); a query without any key gives zeros. scale defaults to 1/sqrt(D). dropout_p drops attention weights with the
    counter-based mask of the library's other dropouts. Returns [B, Lq, heads, D]; differentiable (once, backward) in q, k, v and table,
    the same bits every time."""
    for what, t in (("q", q), ("k", k), ("v", v)):
        if t.dim() != 4:
            raise ValueError(f"relpos_attention: {what} must be [batch, tokens, heads, D] (got {tuple(t.shape)})")
    if k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[2:] != k.shape[2:]:
        raise ValueError(f"relpos_attention: shapes do not belong together: {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    B, Lq, heads, D = q.shape
    return _attend("relpos_attention", q, k, v, B, Lq, k.shape[1], heads, D, table, buckets, key_mask, scale, q_start, dropout_p, seed)


def relpos_self_attention(qkv, table, buckets, key_mask=None, scale=None, dropout_p=0.0, seed=None):
    """relpos_attention of a packed projection qkv [B, L, 3, heads, D] over the first L tokens of the map; its gradient comes
    back packed as well."""
    if qkv.dim() != 5 or qkv.shape[2] != 3:
        raise ValueError(f"relpos_self_attention: qkv must be [batch, tokens, 3, heads, D] (got {tuple(qkv.shape)})")
    B, L, _, heads, D = qkv.shape
    return _attend("relpos_self_attention", qkv, None, None, B, L, L, heads, D, table, buckets, key_mask, scale, 0, dropout_p, seed)
