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
    _functions: tuple[str, ...] = ()

    def __init__(self, ctx: Context, dtype, *sizes):
        torch = _torch()
        elements = {torch.float32: SP_F32, torch.bfloat16: SP_BF16}
        if dtype not in elements:
            raise ValueError(f"element type {dtype}: torch.float32 or torch.bfloat16")
        self.ctx, self.dtype, self.lib = ctx, dtype, ctx.lib
        self._torch = torch
        # The current stream's handle, without the stream object (1.2 us of a 7 us call).
        self._current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
            lambda device: torch.cuda.current_stream(device).cuda_stream
        )
        self._stream = ctx.stream
        self._indices = {torch.int32: SP_INDEX32, torch.int64: SP_INDEX64}
        self._entry = {name: getattr(self.lib, name) for name in self._functions}
        handle = ctypes.c_void_p()
        status = getattr(self.lib, self._create)(
            ctx.handle, *sizes[:2], elements[dtype], *sizes[2:], ctypes.byref(handle)
        )
        self.handle = handle.value
        _lib.check(status, ctx.handle, self._create)

    def _matrix(self, x, columns: int, what: str, rows: int | None = None) -> tuple[int, int]:
        """(pointer, row stride) of a matrix argument."""
        shape = x.shape
        if x.dtype is not self.dtype or len(shape) != 2 or shape[1] != columns or (rows is not None and shape[0] != rows):
            raise ValueError(f"{what}: a {self.dtype} matrix of {'any' if rows is None else rows} x {columns}, "
                             f"got {x.dtype} {tuple(shape)}")
        if x.get_device() != self.ctx.device:
            raise ValueError(f"{what}: on cuda:{self.ctx.device}, got {x.device}")
        row_stride, column_stride = x.stride()
        if column_stride != 1 and columns > 1:
            raise ValueError(f"{what}: unit column stride, got {x.stride()}")
        if row_stride < columns and shape[0] <= 1:
            row_stride = columns
        return x.data_ptr(), row_stride

    def _vector(self, x, what: str, count: int | None = None, dtype=None) -> int:
        shape = x.shape
        if (len(shape) != 1 or not x.is_contiguous() or (dtype is not None and x.dtype is not dtype)
                or (count is not None and shape[0] != count)):
            raise ValueError(f"{what}: a contiguous vector of {'any number of' if count is None else count} "
                             f"{'values' if dtype is None else dtype}, got {x.dtype} {tuple(shape)}")
        if x.get_device() != self.ctx.device:
            raise ValueError(f"{what}: on cuda:{self.ctx.device}, got {x.device}")
        return x.data_ptr()

    def _index(self, x, what: str, count: int | None = None) -> tuple[int, int]:
        index = self._indices.get(x.dtype)
        if index is None:
            raise ValueError(f"{what}: int32 or int64, got {x.dtype}")
        return self._vector(x, what, count), index

    def _call(self, function: str, *args) -> None:
        """The call on the context's stream, ordered with the current torch stream on both sides."""
        entry, device = self._entry[function], self.ctx.device
        if (self._current_stream(device) or CUDA_STREAM_LEGACY) == self._stream:
            status = entry(self.handle, *args)
        else:
            torch = self._torch
            current = torch.cuda.current_stream(device)
            legacy = self._stream == CUDA_STREAM_LEGACY
            own = torch.cuda.default_stream(device) if legacy else torch.cuda.ExternalStream(self._stream, device=device)
            own.wait_stream(current)
            status = entry(self.handle, *args)
            current.wait_stream(own)
        if status:
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
    _functions = ("sp_embedding_lookup", "sp_embedding_gradient")

    def __init__(self, ctx: Context, entries: int, dim: int, dtype, max_tokens: int):
        self.entries, self.dim, self.max_tokens = entries, dim, max_tokens
        super().__init__(ctx, dtype, entries, dim, max_tokens)

    def lookup(self, table, tokens, scale: float = 1.0, out=None):
        """scale * table[tokens], in the element type."""
        table_at, table_stride = self._matrix(table, self.dim, "table", self.entries)
        tokens_at, index = self._index(tokens, "tokens")
        count = tokens.shape[0]
        if out is None:
            out = table.new_empty((count, self.dim))
            out_at, out_stride = out.data_ptr(), self.dim
        else:
            out_at, out_stride = self._matrix(out, self.dim, "out", count)
        self._call("sp_embedding_lookup", table_at, table_stride, tokens_at, index, count, scale, out_at, out_stride)
        return out

    def gradient(self, out_gradient, tokens, scale: float = 1.0, out=None):
        """The gradient of the table from that of `lookup`'s result: every entry's row written."""
        tokens_at, index = self._index(tokens, "tokens")
        count = tokens.shape[0]
        gradient_at, gradient_stride = self._matrix(out_gradient, self.dim, "out_gradient", count)
        if out is None:
            out = out_gradient.new_empty((self.entries, self.dim))
            out_at, out_stride = out.data_ptr(), self.dim
        else:
            out_at, out_stride = self._matrix(out, self.dim, "out", self.entries)
        self._call("sp_embedding_gradient", gradient_at, gradient_stride, tokens_at, index, count, scale, out_at,
                   out_stride)
        return out


@dataclass
class LabelLoss:
    """`LabelHead.loss`: the mean over the rows with a target (a 0-d tensor), and per row the loss
    and, in float64, the log sum exp of the logits (0 for a row without a target)."""

    mean: object
    losses: object
    log_normalizers: object


class LabelHead(_Handle):
    """Classifies feature rows of width `dim` against `labels` label rows (the weight); at most
    `max_rows` rows a call. `training` reserves what `gradient` needs. A target outside [0, labels)
    is none: its row is skipped, whatever its features hold."""

    _create, _destroy, _check = "sp_label_head_create", "sp_label_head_destroy", "sp_label_head_check"
    _functions = ("sp_label_head_loss", "sp_label_head_gradient", "sp_label_head_predict")

    def __init__(self, ctx: Context, labels: int, dim: int, dtype, max_rows: int, training: bool = True):
        self.labels, self.dim, self.max_rows, self.training = labels, dim, max_rows, training
        super().__init__(ctx, dtype, labels, dim, max_rows, 1 if training else 0)

    def _inputs(self, features, weight) -> tuple[int, int, int, int]:
        return *self._matrix(features, self.dim, "features"), *self._matrix(weight, self.dim, "weight", self.labels)

    def loss(self, features, weight, targets, logit_scale: float = 1.0) -> LabelLoss:
        """Cross entropy of softmax(logit_scale * features @ weight.T) at each row's target."""
        inputs = self._inputs(features, weight)
        rows = features.shape[0]
        targets_at, index = self._index(targets, "targets", rows)
        losses = features.new_empty(rows, dtype=self._torch.float32)
        normalizers, mean = losses.new_empty(rows, dtype=self._torch.float64), losses.new_empty(())
        self._call("sp_label_head_loss", *inputs, targets_at, index, rows, logit_scale, mean.data_ptr(),
                   losses.data_ptr(), normalizers.data_ptr())
        return LabelLoss(mean, losses, normalizers)

    def gradient(self, features, weight, targets, log_normalizers, logit_scale: float = 1.0, row_gradient=None,
                 feature_gradient=None, weight_gradient=None):
        """(gradient of the features, of the weight) of the mean loss, or with `row_gradient` (one
        float32 per row) of sum(row_gradient * losses). `log_normalizers` as `loss` of this head returned
        them (those of a head not made for training may be of differently rounded logits)."""
        inputs = self._inputs(features, weight)
        rows = features.shape[0]
        targets_at, index = self._index(targets, "targets", rows)
        float32 = self._torch.float32
        normalizers_at = self._vector(log_normalizers, "log_normalizers", rows, self._torch.float64)
        row_at = None if row_gradient is None else self._vector(row_gradient, "row_gradient", rows, float32)
        # Fresh gradients are dense; only the caller's own are checked.
        if feature_gradient is None:
            feature_gradient = features.new_empty((rows, self.dim))
            to_features = feature_gradient.data_ptr(), self.dim
        else:
            to_features = self._matrix(feature_gradient, self.dim, "feature_gradient", rows)
        if weight_gradient is None:
            weight_gradient = weight.new_empty((self.labels, self.dim))
            to_weight = weight_gradient.data_ptr(), self.dim
        else:
            to_weight = self._matrix(weight_gradient, self.dim, "weight_gradient", self.labels)
        self._call("sp_label_head_gradient", *inputs, targets_at, index, rows, logit_scale, normalizers_at, row_at,
                   *to_features, *to_weight)
        return feature_gradient, weight_gradient

    def predict(self, features, weight, logit_scale: float = 1.0):
        """(label int32, log-probability float32) of each row's most probable label."""
        inputs = self._inputs(features, weight)
        rows = features.shape[0]
        labels = features.new_empty(rows, dtype=self._torch.int32)
        log_probabilities = features.new_empty(rows, dtype=self._torch.float32)
        self._call("sp_label_head_predict", *inputs, rows, logit_scale, labels.data_ptr(), log_probabilities.data_ptr())
        return labels, log_probabilities
