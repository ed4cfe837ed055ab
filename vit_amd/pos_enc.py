"""Position encoders added to the patch tokens (reference: vit/pos_enc.py).

Fourier: the batch-independent (1, N, D) table is built once per step: a K=2 product and sin/cos in fp32
(host-side set-up, as in the reference with autocast disabled), then the D x D projection runs through
libvitk's GEMM (ops.linear).  The "+ pos" itself is fused into the patch-embedding GEMM epilogue."""
from __future__ import annotations

import math
from typing import Optional, Sequence

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch import Tensor

from . import ops
from .initialization import INIT_STD, init_linear, trunc_normal_

PositionEncoder = str  # "fourier" | "learnable" | "none" | "rope"


_GRIDS: dict = {}   # (dims, dtype, device, normalize) -> coordinate grid: constants, built once per process


def create_grid(dims: Sequence[int], dtype=torch.float32, device="cpu", normalize: bool = True) -> Tensor:
    key = (tuple(dims), dtype, str(device), normalize)
    grid = _GRIDS.get(key)
    if grid is None:
        axes = [torch.linspace(-1, 1, d, device=device, dtype=dtype) if normalize else torch.arange(d, device=device, dtype=dtype)
                for d in dims]
        grid = torch.stack(torch.meshgrid(axes, indexing="ij"), dim=-1).view(1, -1, len(dims))
        if len(_GRIDS) < 64:
            _GRIDS[key] = grid
    return grid


def fourier_position(dims: Sequence[int], w_fourier: Tensor, w_fc1: Tensor, b_fc1: Optional[Tensor]) -> Tensor:
    grid = create_grid(dims, device=w_fourier.device)
    if len(dims) <= 3 and w_fourier.dtype == torch.float32:   # other dtypes fail below exactly as they do in the reference
        # features in fp32 arithmetic, rounded once to the dtype the projection computes in (what its input cast does)
        feats = ops.FourierFeaturesFn.apply(grid, w_fourier, ops.compute_dtype(w_fc1.dtype))
    else:
        with torch.autocast(device_type=w_fourier.device.type, enabled=False):
            feats = grid @ w_fourier
            feats = torch.cat([feats.sin(), feats.cos()], dim=-1) / math.sqrt(w_fourier.shape[-1])
    return ops.linear(feats, w_fc1, b_fc1)


class FourierPosition(nn.Module):
    def __init__(self, hidden_size: int, spatial_size: Sequence[int], device=None, dtype=None):
        super().__init__()
        self.spatial_size = spatial_size
        self.w_fourier = nn.Parameter(torch.empty(len(spatial_size), hidden_size // 2, device=device, dtype=dtype))
        self.w_fc1 = nn.Linear(hidden_size, hidden_size, device=device, dtype=dtype)
        self.reset_parameters()

    def reset_parameters(self, std: float = 1.0) -> None:
        nn.init.normal_(self.w_fourier, std=std)
        init_linear(self.w_fc1)

    def forward(self, dims: Optional[Sequence[int]]) -> Tensor:
        return fourier_position(dims or self.spatial_size, self.w_fourier, self.w_fc1.weight, self.w_fc1.bias)


@torch.no_grad()
def fourier_features_(param: Tensor, std: float = 1.0) -> None:
    *dims, hidden = param.shape
    if hidden % 2:
        raise ValueError(f"Hidden size must be even, got {hidden}")
    w = param.new_empty(len(dims), hidden // 2).normal_(std=std)
    f = create_grid(dims, dtype=param.dtype, device=param.device).squeeze(0) @ w
    param.data.copy_((torch.cat([f.sin(), f.cos()], dim=-1) / math.sqrt(hidden)).view_as(param))


class LearnablePosition(nn.Module):
    """Learned table with bicubic resize; a (1, N, D) parameter-sized tensor, batch independent, so the resize and
    the table dropout stay torch ops (set-up work), exactly as the reference orders them (vit/pos_enc.py:79-90)."""

    def __init__(self, hidden_size: int, spatial_size: Sequence[int], fourier_init: bool = True, dropout: float = 0.0,
                 device=None, dtype=None):
        super().__init__()
        self.spatial_size = spatial_size
        self.positions = nn.Parameter(torch.empty(math.prod(spatial_size), hidden_size, device=device, dtype=dtype))
        self.dropout = nn.Dropout(dropout)
        self.reset_parameters(fourier_init)

    @torch.no_grad()
    def reset_parameters(self, fourier_init: bool = True) -> None:
        if fourier_init:
            fourier_features_(self.positions.view(*self.spatial_size, self.positions.shape[-1]))
            self.positions.data.sub_(self.positions.mean()).mul_(INIT_STD / self.positions.std())
        else:
            trunc_normal_(self.positions)

    def forward(self, dims: Optional[Sequence[int]]) -> Tensor:
        dims = tuple(dims or self.spatial_size)
        pos, L_ = self.positions, math.prod(dims)
        if dims != tuple(self.spatial_size):
            p = pos.view(1, *self.spatial_size, -1).movedim(-1, 1)
            pos = F.interpolate(p, size=dims, mode="bicubic", antialias=False).movedim(1, -1).reshape(1, L_, -1)
        return F.dropout(pos, p=self.dropout.p, training=self.training).view(1, L_, -1)


def create_position_encoder(pos_enc: str, hidden_size: int, spatial_size: Sequence[int], **kwargs):
    if pos_enc == "learnable":
        kwargs.setdefault("dropout", 0.1)
        return LearnablePosition(hidden_size, spatial_size, **kwargs)
    if pos_enc == "fourier":
        return FourierPosition(hidden_size, spatial_size, **kwargs)
    if pos_enc == "none":
        return None
    if pos_enc == "rope":
        raise ValueError("Please create RoPE position encoder manually")
    raise ValueError(f"Invalid position encoder: {pos_enc}")


# ------------------------------------------------------------------------------------------------------------------------
# relative positions
# ------------------------------------------------------------------------------------------------------------------------
class RelativeBuckets:
    """Bucket number of every (query, key) pair, and the order in which the gradient of a bias table sums the pairs.

    ``index`` [Lq, Lk] holds integers in [0, num_buckets), num_buckets <= 65536.  The plan is built once (it reads the
    index on the host) and used by every call of every layer with these positions: ``index16`` the numbers in 16 bits,
    ``order`` the pairs sorted by bucket, ``piece`` / ``bucket_piece`` the runs of at most ``piece_length`` pairs that are
    summed at a time and the runs of each bucket."""

    def __init__(self, index: Tensor, num_buckets: int):
        if index.dim() != 2 or index.dtype in (torch.bool, torch.uint16, torch.uint32, torch.uint64) or index.is_floating_point() \
                or index.is_complex():
            raise ValueError(f"bucket index must be an integer tensor [Lq, Lk], got {index.dtype} {tuple(index.shape)}")
        if index.numel() == 0:
            raise ValueError("bucket index is empty")
        if index.numel() >= 2 ** 31:
            raise ValueError(f"bucket index of {index.numel()} pairs is too large (2^31)")
        if not 1 <= num_buckets <= 65536:
            raise ValueError(f"num_buckets must be in [1, 65536], got {num_buckets}")
        flat = index.detach().reshape(-1).to(torch.int32)
        lo, hi = (int(v) for v in torch.stack([index.min(), index.max()]).tolist())
        if lo < 0 or hi >= num_buckets:
            raise ValueError(f"bucket numbers must be in [0, {num_buckets}), got {lo} .. {hi}")
        self.shape = tuple(index.shape)
        self.num_buckets = int(num_buckets)
        self.index16 = torch.where(flat >= 32768, flat - 65536, flat).to(torch.int16).view(self.shape)
        self.order = torch.sort(flat, stable=True).indices.to(torch.int32)
        counts = torch.bincount(flat, minlength=num_buckets).cpu()
        # short runs keep many waves busy; the number of runs stays within what the second sum takes in a few steps
        self.piece_length = length = min(4096, max(256, 1 << (flat.numel() // 8192).bit_length()))
        pieces = (counts + length - 1) // length
        bucket_piece = torch.cat([pieces.new_zeros(1), pieces.cumsum(0)])
        starts = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
        owner = torch.repeat_interleave(torch.arange(num_buckets, device="cpu"), pieces)          # bucket of every piece
        within = torch.arange(int(bucket_piece[-1]), device="cpu") - bucket_piece[owner]
        piece = torch.cat([starts[owner] + within * length, starts[-1:]])
        self.num_pieces = int(bucket_piece[-1])
        self.piece = piece.to(torch.int32).to(index.device)
        self.bucket_piece = bucket_piece.to(torch.int32).to(index.device)

    @property
    def device(self) -> torch.device:
        return self.index16.device

    def to(self, device) -> "RelativeBuckets":
        """The same plan on another device."""
        new = object.__new__(RelativeBuckets)
        new.__dict__.update({k: v.to(device) if isinstance(v, Tensor) else v for k, v in self.__dict__.items()})
        return new

    def record_stream(self, stream) -> None:
        """``Tensor.record_stream`` for the plan: its memory is not given away before what ``stream`` has been asked to do until
        the plan is dropped."""
        for t in (self.index16, self.order, self.piece, self.bucket_piece):
            t.record_stream(stream)

    @classmethod
    def grid(cls, dims: Sequence[int], num_prefix_tokens: int = 0, device=None, table_dims: Optional[Sequence[int]] = None):
        """Tokens of a grid behind ``num_prefix_tokens`` prefix tokens: a bucket for every offset between two grid tokens of
        a ``table_dims`` grid (default: ``dims`` itself), and with a prefix three more, for grid token after prefix token
        (query, key) pairs: prefix to grid, grid to prefix, prefix to prefix."""
        dims = tuple(int(d) for d in dims)
        table_dims = tuple(int(d) for d in (table_dims or dims))
        if len(dims) != len(table_dims) or any(d < 1 or d > t for d, t in zip(dims, table_dims)):
            raise ValueError(f"a table for grids up to {table_dims} does not cover a {dims} grid")
        pos = torch.stack(torch.meshgrid([torch.arange(d, device="cpu") for d in dims], indexing="ij"), dim=-1).view(-1, len(dims))
        num = cls.grid_buckets(table_dims, num_prefix_tokens)
        idx = torch.zeros((pos.shape[0], pos.shape[0]), dtype=torch.int64, device="cpu")
        for axis, t in enumerate(table_dims):
            idx = idx * (2 * t - 1) + (pos[:, None, axis] - pos[None, :, axis] + t - 1)
        n = int(num_prefix_tokens)
        if n:
            full = torch.empty((n + pos.shape[0],) * 2, dtype=torch.int64, device="cpu")
            full[n:, n:], full[:n, n:], full[n:, :n], full[:n, :n] = idx, num - 3, num - 2, num - 1
            idx = full
        return cls(idx.to(torch.get_default_device() if device is None else device), num)

    @staticmethod
    def grid_buckets(table_dims: Sequence[int], num_prefix_tokens: int = 0) -> int:
        return math.prod(2 * int(t) - 1 for t in table_dims) + (3 if num_prefix_tokens else 0)

    @classmethod
    def log_distance(cls, num_queries: int, num_keys: int, num_buckets: int = 32, max_distance: int = 128, device=None):
        """Buckets of the signed distance key - query in a sequence: half of them for keys behind the query; of each half
        the first half are single distances, the others grow logarithmically up to ``max_distance``."""
        half = num_buckets // 2
        exact = half // 2
        if num_buckets % 4 or num_buckets < 4 or max_distance <= exact:
            raise ValueError(f"log_distance needs num_buckets a multiple of 4 and max_distance > num_buckets / 4, got "
                             f"{num_buckets}, {max_distance}")
        far = max(num_queries, num_keys)
        device = torch.get_default_device() if device is None else device
        d = torch.arange(max(far, 1), dtype=torch.float64, device="cpu")
        log = exact + torch.floor(torch.log(d.clamp_min(1) / exact) / math.log(max_distance / exact) * (half - exact) + 1e-9)
        table = torch.where(d < exact, d, log.clamp_max(half - 1)).to(torch.int64).to(device)
        rel = torch.arange(num_keys, device=device)[None, :] - torch.arange(num_queries, device=device)[:, None]
        return cls(table[rel.abs()] + half * (rel > 0), num_buckets)
