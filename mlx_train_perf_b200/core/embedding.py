"""`embedding_lookup`: scaled rows of a table, and the table's gradient by sorted tokens (csrc/embedding.cu).

The reference's trunk calls the model's own embedding module (adapters/mlx_lm.py:140-164), and so do the adapters here; where
the table is trained its gradient is this operator's.  The gradient adds the rows of equal ids in fp32 and in a fixed order, rounds
once, and is the same bits for equal calls.
"""
from __future__ import annotations

import ctypes as C

import torch

from mlx_train_perf_b200 import _lib
from mlx_train_perf_b200.core.loss import VJP_CALLS, has_tangent, index_status
from mlx_train_perf_b200.errors import EmbeddingInputError

_DTYPES = (torch.float32, torch.bfloat16)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """(N, D) with adjacent columns."""
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _look_up(weight: torch.Tensor, ids: torch.Tensor, scale: float, padding: int) -> torch.Tensor:
    """One launch; `ids` contiguous."""
    v, d = weight.shape
    dev, dtype, shape = weight.device, weight.dtype, ids.shape
    rows = _rows(weight)
    out = (torch.empty_strided((shape[0], d), (d, 1), dtype=dtype, device=dev) if len(shape) == 1
           else torch.empty((*shape, d), dtype=dtype, device=dev))
    a = _lib.EmbeddingArgs(ids.data_ptr(), ids.numel(), v, d, dtype is torch.bfloat16, ids.dtype is torch.int64, scale, rows.stride(0),
                           padding)
    with _lib.on(dev):
        rc = _lib.load().b200tp_embedding_fwd(C.byref(a), rows.data_ptr(), out.data_ptr(), _lib.stream(dev),
                                              index_status(dev).data_ptr())
    _lib.check(rc)
    return out


class _Lookup(torch.autograd.Function):
    """(weight, (ids, scale, padding, rows or None)) -> ids.shape + (D,)."""

    @staticmethod
    def forward(ctx, weight, call):
        ids, scale, padding, rows = call
        ctx.save_for_backward(ids)
        ctx.rule = *weight.shape, weight.dtype, scale, padding
        return _look_up(weight, ids, scale, padding) if rows is None else rows

    @staticmethod
    def backward(ctx, d_out):
        if torch.is_grad_enabled():
            raise EmbeddingInputError("embedding_lookup has no second derivative (create_graph=True)")
        VJP_CALLS["embedding_lookup"] = VJP_CALLS.get("embedding_lookup", 0) + 1
        ids, = ctx.saved_tensors
        v, d, dtype, scale, padding = ctx.rule
        dev = ids.device
        lib = _lib.load()
        if d_out.ndim != 2:
            d_out = d_out.reshape(-1, d)
        rows = _rows(d_out)
        grad = torch.empty_strided((v, d), (d, 1), dtype=dtype, device=dev)
        a = _lib.EmbeddingArgs(ids.data_ptr(), ids.numel(), v, d, dtype is torch.bfloat16, ids.dtype is torch.int64, scale, rows.stride(0),
                               padding)
        with _lib.on(dev):
            nbytes = lib.b200tp_embedding_bwd_workspace_bytes(C.byref(a))     # goes by the device's SMs
            ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
            rc = lib.b200tp_embedding_bwd(C.byref(a), rows.data_ptr(), grad.data_ptr(), None if ws is None else ws.data_ptr(), nbytes,
                                          _lib.stream(dev), index_status(dev).data_ptr())
        _lib.check(rc)
        return grad, None


def embedding_lookup(ids: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0, padding_idx: int | None = None,
                     validate_ids: bool = False) -> torch.Tensor:
    """`scale * weight[ids]`, shaped `ids.shape + (D,)`, fp32 arithmetic rounded once to the table's dtype (fp32 or bf16).

    ids: integers of any shape on the table's device (int32 and int64 are read as they are).  `padding_idx`: that row gets no gradient.  An id
    outside [0, V) gives a row of zeros and no gradient, and `core.loss.check_device_status()` reports it; `validate_ids=True`
    raises before the launch, with a host synchronisation.  The gradient is dense (V, D)."""
    shape = weight.shape
    if len(shape) != 2 or 0 in shape:
        raise EmbeddingInputError(f"weight must be (V, D), got {tuple(shape)}")
    if has_tangent(weight):
        raise EmbeddingInputError("embedding_lookup has no forward-mode derivative")
    if not weight.is_cuda:
        raise EmbeddingInputError(f"weight must be a CUDA tensor (the operator has no CPU path); got {weight.device}")
    if weight.dtype not in _DTYPES:
        raise EmbeddingInputError(f"weight must be fp32 or bf16, got {weight.dtype}")
    if ids.get_device() != weight.get_device():
        raise EmbeddingInputError(f"ids are on {ids.device}, weight on {weight.device}")
    if ids.dtype not in (torch.int64, torch.int32):
        if ids.dtype.is_floating_point or ids.dtype.is_complex or ids.dtype == torch.bool:
            raise EmbeddingInputError(f"ids must be an integer dtype, got {ids.dtype}")
        ids = ids.to(torch.int64)
    v, padding = shape[0], -1
    if padding_idx is not None:
        if not -v <= padding_idx < v:
            raise EmbeddingInputError(f"padding_idx must lie in [-{v}, {v}), got {padding_idx}")
        padding = int(padding_idx) % v
    if validate_ids and ids.numel() > 0:
        lo, hi = int(ids.min()), int(ids.max())
        if lo < 0 or hi >= v:
            raise EmbeddingInputError(f"ids must satisfy 0 <= id < V={v}; got range [{lo}, {hi}]")
    if not ids.is_contiguous():
        ids = ids.contiguous()
    if weight.requires_grad and torch.is_grad_enabled():
        return _Lookup.apply(weight, (ids, float(scale), padding, None))
    return _look_up(weight, ids, float(scale), padding)     # without autograd's function around it: 6 us of some 17


def module_lookup(mod: torch.nn.Embedding, ids: torch.Tensor) -> torch.Tensor:
    """`mod(ids)` with `embedding_lookup`'s gradient for its table, for the adapters' walk.  The rows are the module's own forward's,
    which also stops at an id outside the table as it always did; `ids` int32 or int64 beside the table."""
    with torch.no_grad():
        rows = mod(ids)
    padding = -1 if mod.padding_idx is None else mod.padding_idx % mod.weight.shape[0]
    return _Lookup.apply(mod.weight, (ids.contiguous(), 1.0, padding, rows))
