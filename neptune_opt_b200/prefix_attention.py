"""Attention of new tokens behind a prefix that the whole batch shares (nb200_prefix_attention).

A server's decode step: every sequence brings a few new tokens, all sequences begin with the same prefix
(a system prompt, a document) that is kept once, and each has its own cache behind it.

    o = softmax(scale * q K^T) V,   K, V = the whole prefix, then the sequence's own tokens up to the
                                    query's own position

q is [batch, heads, tokens, D], prefix_k and prefix_v [kv_heads, prefix, D], k and v [batch, kv_heads,
cache, D], all bfloat16 or all float16, D 64 or 128; query head h reads key/value head
h // (heads // kv_heads). seq_lens [batch] int32 counts each sequence's own tokens, the new ones (already
in k and v) included; without it every sequence fills its cache. Query t stands at own position
seq_lens[b] - tokens + t and sees the prefix and the own tokens up to there. A query before its
sequence's first token (a free slot of the batch) reads out as zero with a log-sum-exp of -inf, and so
does a row whose every score is -inf. What the caches hold behind a sequence does not matter, nor what a
later new token holds to an earlier one. Tensors whose rows the kernels' copies cannot read (an expanded
batch, a base off the 16-byte boundary) are copied first, in every call. prefix or cache may be 0: without a
prefix this is attention against a cache. Any number of new tokens is right, but the caches' side is laid out
for few: every 32 query rows read a sequence's cache once more.

The prefix is read once for the queries of all sequences, and every key range is split as far as the GPU
has room; the partial results are merged as the split plan merges its states (the reference's merge
certificate, neptune_codegen/algebra.py:348-403), in a fixed order. Scores, sums and merges are fp32;
probabilities are rounded to the inputs' type for the product with V.

No gradient: one that is asked for is refused (NotImplementedError). Errors follow the backend's
convention: TypeError for dtypes, ValueError for devices, shapes and scale, NotImplementedError for head
dimensions the kernels are not built for.
"""
from __future__ import annotations

import math

from neptune_opt_b200.torch_op import run_cxx

HEAD_DIMS = (64, 128)


def validate_prefix_attention_inputs(q, prefix_k, prefix_v, k, v, seq_lens, scale):
    """Metadata-only contract."""
    import torch

    what = "prefix_attention"
    for name, t, dims in (("q", q, 4), ("prefix_k", prefix_k, 3), ("prefix_v", prefix_v, 3), ("k", k, 4), ("v", v, 4)):
        if not isinstance(t, torch.Tensor) or t.layout != torch.strided:
            raise TypeError(f"{what}: {name} must be a strided tensor")
        if t.dtype not in (torch.bfloat16, torch.float16) or t.dtype != q.dtype:
            raise TypeError(f"{what}: {name} must share q's bfloat16/float16 dtype, got {t.dtype}")
        if t.dim() != dims:
            raise ValueError(f"{what}: {name} must have {dims} dimensions, got {tuple(t.shape)}")
        if t.device != q.device:
            raise ValueError(f"{what}: {name} must be on the device of q")
    if q.device.type not in ("cuda", "meta"):
        raise ValueError(f"{what}: inputs must be CUDA tensors, got {q.device}")
    if (k.shape != v.shape or prefix_k.shape != prefix_v.shape or q.shape[0] != k.shape[0]
            or k.shape[1] != prefix_k.shape[0] or not q.shape[-1] == k.shape[-1] == prefix_k.shape[-1]):
        raise ValueError(f"{what}: shapes differ: q {tuple(q.shape)}, prefix {tuple(prefix_k.shape)} and "
                         f"{tuple(prefix_v.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    if q.shape[1] != k.shape[1] and (k.shape[1] == 0 or q.shape[1] % k.shape[1]):
        raise ValueError(f"{what}: {q.shape[1]} query heads cannot share {k.shape[1]} key/value heads")
    if seq_lens is not None:
        if not isinstance(seq_lens, torch.Tensor) or seq_lens.dtype != torch.int32:
            raise TypeError(f"{what}: seq_lens must be an int32 tensor")
        if tuple(seq_lens.shape) != (q.shape[0],) or seq_lens.device != q.device or not seq_lens.is_contiguous():
            raise ValueError(f"{what}: seq_lens must be a contiguous [batch] tensor on the device of q")
    if not (math.isfinite(scale) and scale > 0.0):
        raise ValueError(f"{what}: scale must be finite and positive, got {scale}")
    if q.shape[-1] not in HEAD_DIMS:
        raise NotImplementedError(f"{what}: head_dim {q.shape[-1]} is not supported (built for {HEAD_DIMS})")


def prefix_attention(q, prefix_k, prefix_v, k, v, seq_lens=None, *, scale=None, return_lse: bool = False):
    """Fresh contiguous O [batch, heads, tokens, D] and, when asked, the natural log-sum-exp of each query's
    scaled scores, fp32 [batch, heads, tokens]. scale is 1/sqrt(D) by default."""
    if scale is None:
        scale = 1.0 / math.sqrt(max(q.shape[-1], 1)) if getattr(q, "shape", ()) else 1.0
    o, lse = run_cxx("prefix_attention", q, (q, prefix_k, prefix_v, k, v, seq_lens, scale, return_lse),
                     validate_prefix_attention_inputs, q, prefix_k, prefix_v, k, v, seq_lens, scale)
    return (o, lse) if return_lse else o
