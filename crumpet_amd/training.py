"""The operators of a Swin block's training step on MI355X.

The rest of the package computes a block's forward pass; these four have
gradients, and with them a training step of the block runs in hand-written
kernels:

* ``relative_position_bias``: the learned bias table gathered by buckets
  (``BiasBuckets``), with the table's gradient;
* ``window_attention``: attention over the packed qkv of each window, with
  bias and mask, and the gradients of qkv and of the bias;
* ``residual_norm``: the residual sum of a branch (gate, drop-path scale, a
  norm after the branch) and the norm before the next one;
* ``linear_8bit``: a linear layer, with the GELU before it if there is one,
  that keeps its input in 8 bits for the backward pass.

The reference is forward-only (README.md:152): its patch falls back to eager
PyTorch for training (torch-ext/crumpet/monai_patch.py:138-142).  Everything
here runs on HIP devices only and raises elsewhere; sums, softmax statistics
and norms are fp32 and in a fixed order, so results repeat bit for bit.  The
calls run on the current stream, can be captured into a graph with their
backward passes (while no eager autograd graph of the same leaves is alive), and
have first derivatives only.  Meta and fake tensors are
supported for tracing.
"""

from __future__ import annotations

from typing import Sequence

import torch

from . import _native
from ._geometry import WindowGrid

_NORMS = {"layer": 0, "rms": 1}
_ACTIVATIONS = {"none": 0, "gelu": 1}


def _ops(t: torch.Tensor, what: str):
    if t.device.type not in ("cuda", "meta"):
        raise RuntimeError(f"{what}: crumpet_amd runs only on HIP (MI355X) devices; got a tensor on '{t.device}'")
    return _native.ops()


class BiasBuckets:
    """The buckets of a bias table, ``index[i, j]`` for query i and key j, made
    ready for ``relative_position_bias`` and its gradient: the index itself
    and the pairs sorted by bucket.

    Make one where the index is made and keep it with it, as a module keeps
    its ``relative_position_index``: it copies the index (later writes into it
    are not seen) and checks it, which waits for the device.  ``num_buckets``
    is the table's length; every index must lie in ``0 .. num_buckets - 1``.
    """

    def __init__(self, index: torch.Tensor, num_buckets: int):
        if index.dim() != 2:
            raise ValueError("index must have shape [queries, keys]")
        if index.dtype not in (torch.int64, torch.int32, torch.int16, torch.uint8, torch.int8):
            raise ValueError(f"index must hold integers, got {index.dtype}")
        num_buckets = int(num_buckets)
        if num_buckets < 1 or num_buckets >= 2**31 or index.numel() >= 2**31:
            raise ValueError("num_buckets and the pairs must lie in 1 .. 2**31 - 1")
        if index.device.type != "cuda":
            raise RuntimeError(f"BiasBuckets: crumpet_amd runs only on HIP (MI355X) devices; got '{index.device}'")
        self.num_buckets = num_buckets
        self.shape = tuple(index.shape)
        flat = index.detach().reshape(-1).long()
        if flat.numel() and (int(flat.min()) < 0 or int(flat.max()) >= num_buckets):
            raise ValueError(f"index must lie in 0 .. {num_buckets - 1}")
        self.index = flat.int().reshape(self.shape)
        if self.index.data_ptr() == index.data_ptr():
            self.index = self.index.clone()
        self.order = torch.sort(flat, stable=True).indices.int()
        counts = torch.bincount(flat, minlength=num_buckets)
        ends = counts.cumsum(0)
        longest = int(_native.hip_library().crumpet_bucket_segment())
        if int(counts.max()) <= longest:
            self.segments = torch.stack([ends - counts, ends], 1).int().contiguous()
            self.firsts = None
            return
        pieces = (counts + longest - 1) // longest
        lasts = pieces.cumsum(0)
        bucket = torch.repeat_interleave(torch.arange(num_buckets, device=flat.device), pieces)
        piece = torch.arange(int(lasts[-1]), device=flat.device) - (lasts - pieces)[bucket]
        start = (ends - counts)[bucket] + piece * longest
        self.segments = torch.stack([start, torch.minimum(start + longest, ends[bucket])], 1).int().contiguous()
        self.firsts = torch.cat([lasts.new_zeros(1), lasts]).int()

    @property
    def device(self) -> torch.device:
        return self.index.device


def relative_position_bias(table: torch.Tensor, buckets: BiasBuckets) -> torch.Tensor:
    """``[heads, queries, keys]``: ``table[index[i, j], h]`` of a learned table
    ``[num_buckets, heads]`` (float32, float16 or bfloat16), in its type.

    The gradient is the sum over the pairs of each bucket, in fp32 and in the
    pairs' order, rounded once; a bucket without pairs gets zeros.
    """
    if not isinstance(buckets, BiasBuckets):
        raise TypeError("buckets must be a BiasBuckets")
    ops = _ops(table, "relative_position_bias")
    if table.dim() != 2 or table.shape[0] != buckets.num_buckets:
        raise ValueError(f"table must have shape [{buckets.num_buckets}, heads], got {list(table.shape)}")
    return ops.bucket_bias(table, buckets.index, buckets.order, buckets.segments, buckets.firsts)


def window_attention(
    qkv: torch.Tensor,  # [windows, N, 3 * heads * head_dim]
    bias: torch.Tensor,  # [heads, N, N]
    num_heads: int,
    mask: torch.Tensor | None = None,  # [masks, N, N]
    volume: Sequence[int] | None = None,
    window_size: Sequence[int] | None = None,
    shift_size: Sequence[int] | None = None,
    scale: float | None = None,
) -> torch.Tensor:
    """``[windows, N, heads * head_dim]``: softmax(scale q k^T + bias + mask) v
    of each window and head, with gradients for ``qkv`` and ``bias``.

    ``qkv`` is the qkv projection's output (channel ``s C + h head_dim + d``),
    float32, float16 or bfloat16, head_dim 16, 32, 64 or 128, up to 16384
    tokens a window; rows of unit stride are read in place.  ``scale`` is
    ``head_dim ** -0.5`` by default.  ``bias`` may have any of the types and
    receives its gradient in its own, summed in fp32.

    ``mask`` is added to the scores, window b reads ``mask[b mod masks]`` (the
    windows are a multiple of the masks); it has no gradient.  Or ``volume``, ``window_size`` and ``shift_size`` give
    the shifted-window mask of the volume whose windows, in the order of
    ``fused_shift_partition_3d``, ``qkv`` holds (outer batch first), without a
    tensor.  A query whose scores are all -inf gets zeros, and no gradient
    flows through it.  The gradients of the scores are rounded to ``qkv``'s type
    on their way into those of q and k: in float16 they overflow past 65504.
    """
    ops = _ops(qkv, "window_attention")
    if qkv.dim() != 3:
        raise ValueError("qkv must have shape [windows, N, 3 * heads * head_dim]")
    num_heads = int(num_heads)
    if num_heads < 1 or qkv.shape[2] % (3 * num_heads) != 0:
        raise ValueError(f"qkv's last axis ({qkv.shape[2]}) must be 3 * num_heads * head_dim")
    region: list[int] = []
    given = [a is not None for a in (volume, window_size, shift_size)]
    if any(given):
        if not all(given):
            raise ValueError("volume, window_size and shift_size belong together")
        if mask is not None:
            raise ValueError("a mask tensor and a shifted volume exclude each other")
        if len(volume) != 3:
            raise ValueError("volume must have three sizes")
        grid = WindowGrid.checked(*(int(v) for v in volume), window_size, shift_size)
        region = [*grid.dims, *grid.window, *grid.shift]
    if scale is None:
        scale = (qkv.shape[2] // (3 * num_heads)) ** -0.5
    return ops.window_attention(qkv, bias, num_heads, mask, region, float(scale))


def residual_norm(
    x: torch.Tensor,  # [samples, ..., C]
    y: torch.Tensor,  # like x
    norm: str = "layer",
    weight: torch.Tensor | None = None,  # [C]
    bias: torch.Tensor | None = None,  # [C]
    post: bool = False,
    post_weight: torch.Tensor | None = None,  # [C]
    post_bias: torch.Tensor | None = None,  # [C]
    gate: torch.Tensor | None = None,  # [C] or [samples, C]
    scale: torch.Tensor | None = None,  # [samples]
    eps: float = 1e-5,
) -> tuple[torch.Tensor, torch.Tensor]:
    """``(x1, h)``: the residual sum ``x1 = x + scale[sample] gate y'`` and
    ``h = norm(x1) weight + bias``, ``y'`` being ``y`` or, with ``post``,
    ``norm(y) post_weight + post_bias``.

    ``norm`` is "layer" (LayerNorm) or "rms".  ``x`` (the residual stream) and
    ``x1`` are float32 or of ``y``'s type, ``h`` has ``y``'s; ``h`` and the
    gradients come from the unrounded sum.  ``scale`` is the drop-path factor
    of each sample (0 where its branch is dropped) and has no gradient;
    everything else has one.  ``C`` up to 8192, or 4096 where it is no
    multiple of 8.  The backward pass keeps ``x`` and ``y`` only.
    """
    ops = _ops(x, "residual_norm")
    if norm not in _NORMS:
        raise ValueError(f"norm must be one of {sorted(_NORMS)}, got {norm!r}")
    return ops.residual_norm(x, y, _NORMS[norm], bool(post), post_weight, post_bias, gate, scale, weight, bias,
                             float(eps))


def linear_8bit(
    x: torch.Tensor,  # [..., K]
    weight: torch.Tensor,  # [n_out, K]
    bias: torch.Tensor | None = None,  # [n_out]
    activation: str = "none",
) -> torch.Tensor:
    """``act(x) @ weight.T + bias``, ``activation`` "none" or "gelu" (exact),
    keeping for the backward pass only an 8-bit copy of ``x``: whole numbers
    up to 127 times a power of two for every 32 channels of a row, 33/32
    bytes a value.  The forward pass computes with ``x`` itself.

    The gradients are those at the copy: ``weight`` receives ``dy^T act(copy)``
    and ``x`` receives ``(dy weight) act'(copy)``; without an activation
    ``x``'s and ``bias``'s are exact.  Channels with an infinity or NaN among
    their 32 are kept as NaN.

    float16 and bfloat16; K and n_out multiples of 16.  Under autocast, x,
    weight and bias are converted to its type, as for a Linear; otherwise they
    must share one.
    """
    ops = _ops(x, "linear_8bit")
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(_ACTIVATIONS)}, got {activation!r}")
    if torch.is_autocast_enabled("cuda"):
        dtype = torch.get_autocast_dtype("cuda")
        x, weight = x.to(dtype), weight.to(dtype)
        bias = None if bias is None else bias.to(dtype)
    return ops.linear_8bit(x, weight, bias, _ACTIVATIONS[activation])


__all__ = ["BiasBuckets", "relative_position_bias", "window_attention", "residual_norm", "linear_8bit"]
