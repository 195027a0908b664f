"""Token embedding: lookup with scaling, and the table's gradient by sorted tokens.

`embed_tokens` stands in for the call of `nn.Embedding` and the cast of its result to the compute dtype (modeling/model.py:227
of the reference; 185-193 for the embedding that trains). The lookup is one pass over the rows that are asked for. The
gradient is a dense matrix, written once: tokens are sorted by id, every row of the table sums its tokens' gradients in
token order, in fp32, without atomics, so repeated calls agree bit for bit.
"""

import torch

from .. import _lib


_INTEGERS = frozenset((torch.int64, torch.int32, torch.int16, torch.uint8))


def _ids(ids, other):
    _lib.require_cuda(ids, other)
    if ids.dtype not in _INTEGERS:
        raise TypeError(f"token ids must be integers, not {ids.dtype}")
    if ids.device != other.device:
        raise ValueError("token ids and the table must be on one device")
    return (ids if ids.dtype == torch.int64 else ids.to(torch.int64)).contiguous()


def embedding_lookup(ids, weight, *, scale=1.0, dtype=None):
    """round(scale * weight[ids]) in `dtype` (default: the table's), [*ids.shape, width]. An id outside the table gives a row
    of zeros and makes the next `_lib.check_device` raise."""
    if weight.ndim != 2:
        raise ValueError("the embedding table must be a matrix")
    ids = _ids(ids, weight)
    weight = weight.detach().contiguous()
    dtype = weight.dtype if dtype is None else dtype
    codes = _lib.code_of(weight.dtype), _lib.code_of(dtype)
    out = torch.empty((*ids.shape, weight.shape[1]), device=weight.device, dtype=dtype)
    with _lib.on_device(weight):
        _lib.check(_lib.load().ct_embedding_forward(
            ids.data_ptr(), weight.data_ptr(), out.data_ptr(), ids.numel(), *weight.shape, float(scale), *codes,
            _lib.stream_of(weight)))
    return out


def embedding_gradient(dy, ids, rows, *, scale=1.0, padding_idx=None, dtype=torch.float32):
    """The [rows, width] gradient of the table from `dy` [*ids.shape, width]: per row, scale times the sum of its tokens'
    gradients; zeros for the other rows and for `padding_idx` (negative: counted from the end, as nn.Embedding does)."""
    ids = _ids(ids, dy)
    if dy.shape[:-1] != ids.shape:
        raise ValueError("dy must have one row per token id")
    if padding_idx is not None:
        if not -rows <= padding_idx < rows:
            raise ValueError(f"padding_idx {padding_idx} lies outside the table")
        padding_idx %= rows
    width = dy.shape[-1]
    flat = dy.reshape(-1, width)
    if flat.stride(1) != 1 or (flat.shape[0] > 1 and flat.stride(0) < width):
        flat = flat.contiguous()
    stride = flat.stride(0) if flat.shape[0] > 1 else width
    codes = _lib.code_of(dy.dtype), _lib.code_of(dtype)
    out = torch.empty((rows, width), device=dy.device, dtype=dtype)
    library = _lib.load()
    with _lib.on_device(dy):
        size = library.ct_embedding_gradient_workspace(ids.numel(), rows, width)
        workspace = torch.empty(size, device=dy.device, dtype=torch.uint8)
        _lib.check(library.ct_embedding_gradient(
            flat.data_ptr(), stride, ids.data_ptr(), out.data_ptr(), ids.numel(), rows, width, float(scale),
            -1 if padding_idx is None else padding_idx, *codes, workspace.data_ptr(), _lib.stream_of(dy)))
    return out


class Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, ids, scale, dtype, padding_idx):
        ctx.save_for_backward(ids)
        ctx.rows, ctx.scale, ctx.table_dtype, ctx.padding_idx = weight.shape[0], scale, weight.dtype, padding_idx
        return embedding_lookup(ids, weight, scale=scale, dtype=dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        ids, = ctx.saved_tensors
        return embedding_gradient(dy, ids, ctx.rows, scale=ctx.scale, padding_idx=ctx.padding_idx,
                                  dtype=ctx.table_dtype), None, None, None, None


def embed_tokens(ids, weight, *, scale=1.0, dtype=None, padding_idx=None):
    """`embedding_lookup`, differentiable in `weight`; `padding_idx` is the row that gets no gradient."""
    if not (torch.is_grad_enabled() and weight.requires_grad):
        return embedding_lookup(ids, weight, scale=scale, dtype=dtype)
    return Embedding.apply(weight, ids, float(scale), dtype, padding_idx)
