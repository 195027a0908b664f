"""Causal attention inside the documents of packed rows, forward and backward.

The kernels behind `Runtime.attention = "documents"`, beside the library call of kernels/attention.py (58-93 of the
reference). Documents need not tile the rows and nothing is gathered: a plan, made once per batch and shared by all
layers and by checkpoint replays, lists the tiles of every document, longest work first.

    y      = softmax(scale * q k^T, keys of the same document up to the query) v       zeros outside documents
    dv     = P^T dy,   dS = P * (dy v^T - sum(dy * y)),   dq = scale dS k,   dk = scale dS^T q

The backward pass recomputes P from q, k and the row's log-sum. Every sum has a fixed order: the query gradients are one
kernel, the key and value gradients another whose pieces are added in plan order, so repeated calls agree bit for bit.
bf16 and fp16 run on the tensor cores; fp32, and operands whose rows are not 16-byte aligned, on FMA units.
A NaN or infinity outside the documents reaches nothing; one inside a document reaches that document only.
"""

import ctypes
from dataclasses import dataclass, field

import torch

from .. import _lib

KEY_TILE = 128              # keys of one piece of the key-gradient pass (include/ct_b200.h)


@dataclass(frozen=True)
class DocumentPlan:
    """Tiles of the documents of one batch, for one number of heads. Made by `prepare_documents`."""
    shape: tuple                    # (rows, width)
    heads: int
    kv_heads: int
    spans: tuple
    table: torch.Tensor             # int32 [records, 4] on the device
    sections: tuple                 # ((first record, count), ...) of the six sections
    key_slots: int
    host_sections: ctypes.Array = field(repr=False, compare=False, default=None)
    stream: int = 0                 # raw handle of the stream on which the table was made


def prepare_documents(shape, spans, device, heads, kv_heads=1):
    """The plan of a [rows, width] batch whose documents are `spans`, ((row, start, end), ...) as `segments.runs` gives
    them: any order, gaps allowed, no token in two documents. A captured graph reads the plan's table when it is replayed:
    keep the plan as long as the graph."""
    rows, width = (int(n) for n in shape)
    if heads < 1 or kv_heads < 1 or heads % kv_heads:
        raise ValueError(f"{heads} heads cannot share {kv_heads} key heads")
    tokens = rows * width
    if tokens >= 2 ** 31 - 256:
        raise NotImplementedError(f"{tokens} tokens in one batch")
    spans = tuple(spans)
    for row, start, end in spans:
        if not (0 <= row < rows and 0 <= start <= end <= width):
            raise ValueError(f"the document span {(row, start, end)} lies outside the batch")
    count = len(spans)
    starts = (ctypes.c_int64 * count)(*[row * width + start for row, start, _ in spans])
    lengths = (ctypes.c_int64 * count)(*[end - start for _, start, end in spans])
    library = _lib.load()
    tile_tokens = library.ct_attention_tile_tokens(heads, kv_heads)
    # at least the records there can be: query tiles of three sizes, key pieces (two records each), sums, gaps
    capacity = 2 * tokens // tile_tokens + tokens // 16 + 10 * count + 2048
    records = torch.empty((capacity, 4), dtype=torch.int32)
    host, slots = (ctypes.c_int64 * 12)(), ctypes.c_int64()
    used = library.ct_attention_plan(starts, lengths, count, tokens, heads, kv_heads, records.data_ptr(), capacity, host,
                                     ctypes.byref(slots))
    if used < 0:
        _lib.check(used)
    if used > capacity:
        raise RuntimeError(f"the plan has {used} records, room was made for {capacity}")
    table = records[:used].to(device, copy=True)
    sections = tuple((host[2 * i], host[2 * i + 1]) for i in range(6))
    return DocumentPlan((rows, width), heads, kv_heads, spans, table, sections, slots.value, host,
                        _lib.stream_of(table) if table.is_cuda else 0)


def _stream(plan, tensor):
    """The stream to launch on. A plan may be dropped as soon as the host has issued the calls that read it: where that is
    another stream than the table's own, the allocator is told."""
    stream = _lib.stream_of(tensor)
    if stream != plan.stream and not torch.cuda.is_current_stream_capturing():
        plan.table.record_stream(torch.cuda.current_stream(tensor.device))
    return stream


def _check(q, k, v, plan):
    _lib.require_cuda(q, k, v)
    if q.ndim != 4 or k.ndim != 4 or v.shape != k.shape or k.shape[:2] != q.shape[:2] or k.shape[3] != q.shape[3]:
        raise ValueError("document attention takes q [rows, width, heads, head_dim] and k, v [rows, width, kv_heads, head_dim]")
    if q.dtype != k.dtype or q.dtype != v.dtype:
        raise TypeError("q, k and v must have one dtype")
    _lib.code_of(q.dtype)
    if not q.device == k.device == v.device == plan.table.device:
        raise ValueError("q, k, v and the plan must be on one device")
    if tuple(q.shape[:2]) != plan.shape or q.shape[2] != plan.heads or k.shape[2] != plan.kv_heads:
        raise ValueError(f"the plan is for a batch of {plan.shape} tokens with {plan.heads} / {plan.kv_heads} heads")
    if q.shape[3] > 128:
        raise NotImplementedError(f"head_dim {q.shape[3]} is above 128")


def _rows(tensor):
    """(tensor, token stride, head stride) of [rows, width, heads, head_dim] as [tokens, heads, head_dim] with contiguous
    channels, copied only where the strides demand it; strides of dimensions of one element are made regular."""
    rows, width, heads, dim = tensor.shape
    if not tensor.is_contiguous():
        row, token, head, channel = tensor.stride()
        if ((channel != 1 and dim > 1) or (rows > 1 and width > 1 and row != width * token) or (heads > 1 and head <= 0)
                or (width > 1 and token <= 0) or (rows > 1 and row <= 0)):
            tensor = tensor.contiguous()
        else:
            head = head if heads > 1 else dim
            return tensor, token if width > 1 else row if rows > 1 else heads * head, head
    return tensor, heads * dim, dim


def _operands(*tensors):
    """The (copied where necessary) tensors, and (pointer, token stride, head stride) of each."""
    views = [_rows(tensor) for tensor in tensors]
    return [view[0] for view in views], [n for tensor, *strides in views for n in (tensor.data_ptr(), *strides)]


def _aligned(tensor):
    """A contiguous form whose first element is 16-byte aligned."""
    tensor = tensor.contiguous()
    return tensor if tensor.data_ptr() % 16 == 0 else tensor.clone()


def attention_forward(q, k, v, plan, *, scale=None, keep_lse=True):
    """(y, lse): the attention output, shaped like q, and the rows' base-2 log-sums [tokens, heads] (None without
    `keep_lse`). `scale` defaults to head_dim ** -0.5."""
    _check(q, k, v, plan)
    rows, width, heads, dim = q.shape
    tokens = rows * width
    kept, operands = _operands(q, k, v)
    out = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    lse = torch.empty((tokens, heads), device=q.device, dtype=torch.float32) if keep_lse else None
    if out.numel() == 0:
        return out, lse
    library, code = _lib.load(), _lib.code_of(q.dtype)
    scale = dim ** -0.5 if scale is None else float(scale)
    with _lib.on_device(q):
        _lib.check(library.ct_attention_forward(
            *operands, out.data_ptr(), _lib.pointer(lse), plan.table.data_ptr(), plan.host_sections, tokens, heads, plan.kv_heads,
            dim, scale, code, _lib.PATH_SIMT if _lib.gemm_path == _lib.PATH_SIMT else _lib.PATH_AUTO, _stream(plan, q)))
    return out, lse


def _path(library, operands, heads, kv_heads, dim, scale, code):
    if _lib.gemm_path == _lib.PATH_SIMT:
        return _lib.PATH_SIMT
    return library.ct_attention_path(*operands, heads, kv_heads, dim, scale, code)


def attention_backward(dy, q, k, v, y, lse, plan, *, scale=None):
    """(dq, dk, dv) from the upstream gradient `dy` of `y` and what `attention_forward` returned."""
    _check(q, k, v, plan)
    if dy.shape != q.shape or y.shape != q.shape:
        raise ValueError("dy and y must be shaped like q")
    if dy.device != q.device or y.device != q.device or lse.device != q.device:
        raise ValueError("dy, y and lse must be on the device of q")
    if lse.shape != (q.shape[0] * q.shape[1], q.shape[2]) or lse.dtype != torch.float32 or not lse.is_contiguous():
        raise ValueError("lse must be the contiguous fp32 [tokens, heads] of the forward pass")
    rows, width, heads, dim = q.shape
    tokens = rows * width
    kept, operands = _operands(q, k, v)
    dy, y = _aligned(dy.to(q.dtype)), _aligned(y.to(q.dtype))
    dq, dk, dv = (torch.empty(t.shape, device=t.device, dtype=t.dtype) for t in (q, k, v))
    if dq.numel() == 0:
        return dq, dk, dv
    library, code = _lib.load(), _lib.code_of(q.dtype)
    scale = dim ** -0.5 if scale is None else float(scale)
    with _lib.on_device(q):
        path = _path(library, operands, heads, plan.kv_heads, dim, scale, code)
        size = library.ct_attention_backward_workspace(tokens, heads, plan.kv_heads, dim, plan.key_slots, path)
        workspace = torch.empty(size, device=q.device, dtype=torch.uint8)
        _lib.check(library.ct_attention_backward(
            *operands, y.data_ptr(), lse.data_ptr(), dy.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
            plan.table.data_ptr(), plan.host_sections, tokens, heads, plan.kv_heads, dim, scale, code, path, workspace.data_ptr(),
            _stream(plan, q)))
    return dq, dk, dv


class DocumentAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, plan, scale):
        keep = any(ctx.needs_input_grad[:3])
        y, lse = attention_forward(q, k, v, plan, scale=scale, keep_lse=keep)
        ctx.plan, ctx.scale = plan, scale
        if keep:
            ctx.save_for_backward(q, k, v, y, lse)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        q, k, v, y, lse = ctx.saved_tensors
        return (*attention_backward(dy, q, k, v, y, lse, ctx.plan, scale=ctx.scale), None, None)


def document_attention(q, k, v, plan, *, scale=None):
    """Causal attention inside the plan's documents: q [rows, width, heads, head_dim], k and v
    [rows, width, kv_heads, head_dim] -> shaped like q, differentiable in all three."""
    if not (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)):
        return attention_forward(q, k, v, plan, scale=scale, keep_lse=False)[0]
    return DocumentAttention.apply(q, k, v, plan, scale)
