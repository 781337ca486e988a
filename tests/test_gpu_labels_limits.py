"""The label operators at the ends of their types' ranges and of their sizes: operands near the largest
finite value and infinite ones, labels out of use, gradients weighted by row, wide features, the
workspace. Against plain 64-bit results, with the bounds of test_gpu_labels."""

from __future__ import annotations

import pytest
import torch

import splat_b200 as sb
from test_gpu_labels import A, TYPES, Bounds, close, matrix, tokens_for

pytestmark = pytest.mark.gpu

# Rows of one call, and whether the head trains: the few-row pass, and the tiles' (a training head's loss
# and more than 64 rows).
PASSES = [(20, False), (64, True), (200, True), (300, False)]


def labels_out_of_use(rows, labels, dim, dtype, off, value, bias):
    """Features whose first column is `bias`, a weight whose `off` rows are `value` there and 0 elsewhere and
    whose other rows are 0 there, targets among the others; and the bounds over those alone."""
    features, weight = matrix(rows, dim, dtype, 1), matrix(labels, dim, dtype, 2)
    features[:, 0], weight[:, 0] = bias, 0.0
    weight[off] = 0.0
    weight[off, 0] = value
    keep = torch.ones(labels, dtype=torch.bool, device="cuda")
    keep[off] = False
    kept = torch.nonzero(keep)[:, 0]
    targets = kept[tokens_for("all", rows, len(kept), torch.int64, 3)]
    return features, weight, targets, kept, Bounds(features, weight[kept], torch.searchsorted(kept, targets), 1.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,training", PASSES)
@pytest.mark.parametrize("value,bias", [("lowest", 1.0), ("lowest", 0.7001), ("lowest", 700.3), ("lowest", 123_456.7),
                                        ("-inf", 1.0), ("-inf", 0.7001)])
def test_labels_out_of_use_have_no_probability(ctx, rows, training, value, bias, dtype):
    """A logit of the type's lowest value, or below it, leaves the other labels' loss and gradient alone
    (the gradient of the features meets an infinite weight times a slope of 0: only without one)."""
    labels, dim = 300, 32
    off = torch.arange(1, labels, 3, device="cuda")
    low = torch.finfo(dtype).min if value == "lowest" else float("-inf")
    features, weight, targets, kept, b = labels_out_of_use(rows, labels, dim, dtype, off, low, bias)
    head = sb.LabelHead(ctx, labels, dim, dtype, rows, training=training)
    loss = head.loss(features, weight, targets)
    close(loss.losses, b.losses, b.loss_error)
    if training:
        to_features, to_weight = head.gradient(features, weight, targets, loss.log_normalizers)
        assert to_weight[off].count_nonzero() == 0
        close(to_weight[kept], b.to_weight, b.weight_error)
        if value == "lowest":
            close(to_features, b.to_features, b.features_error)
    best = b.z.amax(1)
    got, log_probabilities = head.predict(features, weight)
    close(log_probabilities, best - b.normalizers, 2 * b.z_error + b.exp_error + 4 * A * b.normalizers.abs())
    assert torch.isin(got, kept.int()).all()
    head.check()


@pytest.mark.parametrize("rows,training", PASSES)
@pytest.mark.parametrize("which", ["features", "weight"])
def test_f32_operands_up_to_the_largest_value(ctx, rows, training, which):
    """Operands up to f32's largest value, past bf16's (3.39e38), with logits in range."""
    labels, dim = 300, 32
    features, weight = matrix(rows, dim, torch.float32, 1), matrix(labels, dim, torch.float32, 2)
    large, small = (features, weight) if which == "features" else (weight, features)
    large *= 1e38
    small *= 1e-3
    large.clamp_(-3.4e38, 3.4e38)
    large[0, :4] = torch.tensor([3.4e38, -3.4e38, torch.finfo(torch.float32).max, torch.finfo(torch.float32).min])
    targets = tokens_for("all", rows, labels, torch.int32, 3)
    scale = 2e-36
    b = Bounds(features, weight, targets, scale)
    assert 0.3 < b.z.std() < 3
    head = sb.LabelHead(ctx, labels, dim, torch.float32, rows, training=training)
    close(head.loss(features, weight, targets, scale).losses, b.losses, b.loss_error)
    _, log_probabilities = head.predict(features, weight, scale)
    close(log_probabilities, b.z.amax(1) - b.normalizers, 2 * b.z_error + b.exp_error + 4 * A * b.normalizers.abs())
    head.check()
