"""Features and labels of Gaussians or pixels over the C ABI of libsplat_b200.so
(include/splat_labels.h): the embedding of codebook tokens with its gradient, and the label
head (cross entropy over a label vocabulary without stored logits, its gradient, prediction).
No counterpart in the reference, which learns colour only.

Tensors are CUDA tensors of the handle's element type (torch.float32 or torch.bfloat16) with unit
column stride and any row stride of at least the column count; tokens and targets are int32 or
int64 and contiguous. A call runs on the context's stream; made from another torch stream it is
ordered after that stream's work and that stream after it. Calls enqueue only; `check()` waits.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass

from . import _lib
from .rasterizer import CUDA_STREAM_LEGACY, Context, _torch

SP_F32, SP_BF16 = 0, 1
SP_INDEX32, SP_INDEX64 = 0, 1


class _Handle:
    """What the two handles share: element type, argument checks, stream order, lifetime."""

    _create = _destroy = _check = ""

    def __init__(self, ctx: Context, dtype, *sizes):
        torch = _torch()
        elements = {torch.float32: SP_F32, torch.bfloat16: SP_BF16}
        if dtype not in elements:
            raise ValueError(f"element type {dtype}: torch.float32 or torch.bfloat16")
        self.ctx, self.dtype, self.lib = ctx, dtype, ctx.lib
        self._torch = torch
        self._stream = ctx.stream
        self._indices = {torch.int32: SP_INDEX32, torch.int64: SP_INDEX64}
        handle = ctypes.c_void_p()
        status = getattr(self.lib, self._create)(
            ctx.handle, *sizes[:2], elements[dtype], *sizes[2:], ctypes.byref(handle)
        )
        self.handle = handle.value
        _lib.check(status, ctx.handle, self._create)

    def _matrix(self, x, columns: int, what: str) -> tuple[int, int]:
        """(pointer, row stride) of a matrix argument."""
        if x.dtype != self.dtype or x.dim() != 2 or x.shape[1] != columns:
            raise ValueError(f"{what}: a {self.dtype} matrix of {columns} columns, got {x.dtype} {tuple(x.shape)}")
        if not x.is_cuda or x.device.index != self.ctx.device:
            raise ValueError(f"{what}: on cuda:{self.ctx.device}, got {x.device}")
        rows, (row_stride, column_stride) = x.shape[0], x.stride()
        if column_stride != 1 and columns > 1:
            raise ValueError(f"{what}: unit column stride, got {x.stride()}")
        if rows <= 1:
            row_stride = max(row_stride, columns)
        return x.data_ptr(), row_stride

    def _vector(self, x, what: str, dtype=None) -> int:
        if x.dim() != 1 or not x.is_contiguous() or (dtype is not None and x.dtype != dtype):
            raise ValueError(f"{what}: a contiguous vector{'' if dtype is None else f' of {dtype}'}, "
                             f"got {x.dtype} {tuple(x.shape)}")
        if not x.is_cuda or x.device.index != self.ctx.device:
            raise ValueError(f"{what}: on cuda:{self.ctx.device}, got {x.device}")
        return x.data_ptr()

    def _index(self, x, what: str) -> tuple[int, int]:
        if x.dtype not in self._indices:
            raise ValueError(f"{what}: int32 or int64, got {x.dtype}")
        return self._vector(x, what), self._indices[x.dtype]

    def _empty(self, *shape, dtype=None):
        return self._torch.empty(shape, dtype=dtype or self.dtype, device=f"cuda:{self.ctx.device}")

    def _output(self, out, rows: int, columns: int, what: str):
        if out is None:
            return self._empty(rows, columns)
        if out.shape != (rows, columns):
            raise ValueError(f"{what}: shape {(rows, columns)}, got {tuple(out.shape)}")
        return out

    def _call(self, function: str, *args) -> None:
        """The call on the context's stream, ordered with the current torch stream on both sides."""
        torch = self._torch
        current = torch.cuda.current_stream(self.ctx.device)
        if (current.cuda_stream or CUDA_STREAM_LEGACY) == self._stream:
            status = getattr(self.lib, function)(self.handle, *args)
        else:
            device = self.ctx.device
            legacy = self._stream == CUDA_STREAM_LEGACY
            own = torch.cuda.default_stream(device) if legacy else torch.cuda.ExternalStream(self._stream, device=device)
            own.wait_stream(current)
            status = getattr(self.lib, function)(self.handle, *args)
            current.wait_stream(own)
        if status != _lib.SP_OK:
            _lib.check(status, self.ctx.handle, function)

    def check(self) -> None:
        """Waits for the stream; raises where a device wait of an earlier call gave up."""
        _lib.check(getattr(self.lib, self._check)(self.handle), self.ctx.handle, self._check)

    def close(self) -> None:
        if getattr(self, "handle", None) and getattr(self.ctx, "handle", None):
            getattr(self.lib, self._destroy)(self.handle)
        self.handle = None

    def __del__(self):
        self.close()


class Embedding(_Handle):
    """A table of `entries` feature rows of width `dim`, looked up by token, and its gradient; at
    most `max_tokens` tokens a call. A token outside [0, entries) is none: a zero row, no gradient."""

    _create, _destroy, _check = "sp_embedding_create", "sp_embedding_destroy", "sp_embedding_check"

    def __init__(self, ctx: Context, entries: int, dim: int, dtype, max_tokens: int):
        self.entries, self.dim, self.max_tokens = entries, dim, max_tokens
        super().__init__(ctx, dtype, entries, dim, max_tokens)

    def lookup(self, table, tokens, scale: float = 1.0, out=None):
        """scale * table[tokens], in the element type."""
        table_at, table_stride = self._matrix(table, self.dim, "table")
        if table.shape[0] != self.entries:
            raise ValueError(f"table: {self.entries} rows, got {table.shape[0]}")
        tokens_at, index = self._index(tokens, "tokens")
        count = tokens.shape[0]
        out = self._output(out, count, self.dim, "out")
        out_at, out_stride = self._matrix(out, self.dim, "out")
        self._call("sp_embedding_lookup", table_at, table_stride, tokens_at, index, count, scale, out_at, out_stride)
        return out

    def gradient(self, out_gradient, tokens, scale: float = 1.0, out=None):
        """The gradient of the table from that of `lookup`'s result: every entry's row written."""
        gradient_at, gradient_stride = self._matrix(out_gradient, self.dim, "out_gradient")
        tokens_at, index = self._index(tokens, "tokens")
        count = tokens.shape[0]
        if out_gradient.shape[0] != count:
            raise ValueError(f"out_gradient: {count} rows, got {out_gradient.shape[0]}")
        out = self._output(out, self.entries, self.dim, "out")
        out_at, out_stride = self._matrix(out, self.dim, "out")
        self._call("sp_embedding_gradient", gradient_at, gradient_stride, tokens_at, index, count, scale, out_at,
                   out_stride)
        return out


@dataclass
class LabelLoss:
    """`LabelHead.loss`: the mean over the rows with a target (a 0-d tensor), and per row the loss
    and log sum exp of the logits (0 for a row without a target)."""

    mean: object
    losses: object
    log_normalizers: object


class LabelHead(_Handle):
    """Classifies feature rows of width `dim` against `labels` label rows (the weight); at most
    `max_rows` rows a call. `training` reserves what `gradient` needs. A target outside [0, labels)
    is none: its row is skipped, whatever its features hold."""

    _create, _destroy, _check = "sp_label_head_create", "sp_label_head_destroy", "sp_label_head_check"

    def __init__(self, ctx: Context, labels: int, dim: int, dtype, max_rows: int, training: bool = True):
        self.labels, self.dim, self.max_rows, self.training = labels, dim, max_rows, training
        super().__init__(ctx, dtype, labels, dim, max_rows, 1 if training else 0)

    def _inputs(self, features, weight) -> tuple[int, int, int, int]:
        features_at, feature_stride = self._matrix(features, self.dim, "features")
        weight_at, weight_stride = self._matrix(weight, self.dim, "weight")
        if weight.shape[0] != self.labels:
            raise ValueError(f"weight: {self.labels} rows, got {weight.shape[0]}")
        return features_at, feature_stride, weight_at, weight_stride

    def _targets(self, targets, rows: int) -> tuple[int, int]:
        targets_at, index = self._index(targets, "targets")
        if targets.shape[0] != rows:
            raise ValueError(f"targets: {rows}, got {targets.shape[0]}")
        return targets_at, index

    def loss(self, features, weight, targets, logit_scale: float = 1.0) -> LabelLoss:
        """Cross entropy of softmax(logit_scale * features @ weight.T) at each row's target."""
        inputs = self._inputs(features, weight)
        rows = features.shape[0]
        targets_at, index = self._targets(targets, rows)
        # One allocation: losses, log normalizers, mean.
        out = self._empty(2 * rows + 1, dtype=self._torch.float32)
        at = out.data_ptr()
        self._call("sp_label_head_loss", *inputs, targets_at, index, rows, logit_scale, at + 8 * rows, at, at + 4 * rows)
        return LabelLoss(out[2 * rows], out[:rows], out[rows : 2 * rows])

    def gradient(self, features, weight, targets, log_normalizers, logit_scale: float = 1.0, row_gradient=None,
                 feature_gradient=None, weight_gradient=None):
        """(gradient of the features, of the weight) of the mean loss, or with `row_gradient` (one
        float32 per row) of sum(row_gradient * losses). `log_normalizers` as `loss` returned them."""
        inputs = self._inputs(features, weight)
        rows = features.shape[0]
        targets_at, index = self._targets(targets, rows)
        float32 = self._torch.float32
        normalizers_at = self._vector(log_normalizers, "log_normalizers", float32)
        row_at = None if row_gradient is None else self._vector(row_gradient, "row_gradient", float32)
        if log_normalizers.shape[0] != rows or (row_gradient is not None and row_gradient.shape[0] != rows):
            raise ValueError(f"log_normalizers, row_gradient: {rows} each")
        feature_gradient = self._output(feature_gradient, rows, self.dim, "feature_gradient")
        weight_gradient = self._output(weight_gradient, self.labels, self.dim, "weight_gradient")
        self._call("sp_label_head_gradient", *inputs, targets_at, index, rows, logit_scale, normalizers_at, row_at,
                   *self._matrix(feature_gradient, self.dim, "feature_gradient"),
                   *self._matrix(weight_gradient, self.dim, "weight_gradient"))
        return feature_gradient, weight_gradient

    def predict(self, features, weight, logit_scale: float = 1.0):
        """(label int32, log-probability float32) of each row's most probable label."""
        inputs = self._inputs(features, weight)
        rows = features.shape[0]
        labels = self._empty(rows, dtype=self._torch.int32)
        log_probabilities = self._empty(rows, dtype=self._torch.float32)
        self._call("sp_label_head_predict", *inputs, rows, logit_scale, labels.data_ptr(), log_probabilities.data_ptr())
        return labels, log_probabilities
