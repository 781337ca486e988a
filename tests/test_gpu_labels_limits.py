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


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,training", PASSES)
@pytest.mark.parametrize("scale", [1.0, 0.3, 0.45, 0.05, 7.0])
def test_blocks_of_labels_out_of_use(ctx, rows, training, scale, dtype):
    """Every label that a thread sees first, or last, is out of use: whatever the scale makes of the type's
    lowest value (in units of 2 it may pass f32's range, or be off by a rounding of 1e31)."""
    labels, dim = 700, 32
    off = torch.cat([torch.arange(0, 70), torch.arange(256, 400), torch.arange(600, 700)]).cuda()
    features, weight, targets, kept, _ = labels_out_of_use(rows, labels, dim, dtype, off, torch.finfo(dtype).min, 1.0)
    b = Bounds(features, weight[kept], torch.searchsorted(kept, targets), scale)
    head = sb.LabelHead(ctx, labels, dim, dtype, rows, training=training)
    loss = head.loss(features, weight, targets, scale)
    close(loss.losses, b.losses, b.loss_error)
    if training:
        to_features, to_weight = head.gradient(features, weight, targets, loss.log_normalizers, scale)
        assert to_weight[off].count_nonzero() == 0
        close(to_weight[kept], b.to_weight, b.weight_error)
        close(to_features, b.to_features, b.features_error)
    best = b.z.amax(1)
    got, log_probabilities = head.predict(features, weight, scale)
    close(log_probabilities, best - b.normalizers, 2 * b.z_error + b.exp_error + 4 * A * b.normalizers.abs())
    assert torch.isin(got, kept.int()).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,training", PASSES)
@pytest.mark.parametrize("scale", [1.0, 0.3, 0.45])
@pytest.mark.parametrize("logit", [1e6, -1e6, 3e9, -3e9, 1e30, "lowest", "largest"])
def test_equal_logits_of_any_size(ctx, rows, training, scale, logit, dtype):
    """All labels' logits are one value, up to the type's lowest (every label out of use): the loss is ln
    labels and the slopes are 1 / labels, as far as the normalizer in 64 bits still tells them apart."""
    labels, dim = 500, 40
    ends = {"lowest": torch.finfo(dtype).min, "largest": torch.finfo(dtype).max}
    features, weight = matrix(rows, dim, dtype, 1), torch.zeros(labels, dim, dtype=dtype, device="cuda")
    features[:, 3], weight[:, 3] = 1.0, ends.get(logit, logit)
    targets = tokens_for("all", rows, labels, torch.int32, 3)
    head = sb.LabelHead(ctx, labels, dim, dtype, rows, training=training)
    loss = head.loss(features, weight, targets, scale)
    want = torch.full((rows,), float(labels), dtype=torch.float64, device="cuda").log()
    # The sum of the labels' ones is exact; the exponentials of 0 are good to 2^-21, the loss is rounded.
    close(loss.losses, want, 2.0**-20 + 4 * A * want)
    got, log_probabilities = head.predict(features, weight, scale)
    close(log_probabilities, -want, 2.0**-20 + 4 * A * want)
    assert got.count_nonzero() == 0
    if training and isinstance(logit, float) and abs(logit) < 1e10:
        _, to_weight = head.gradient(features, weight, targets, loss.log_normalizers, scale)
        # The normalizers are good to 2^-53 of 3e9 and of ln labels; then as in Bounds, with logits that are exact.
        slopes = torch.full((rows, labels), 1.0 / labels, dtype=torch.float64, device="cuda")
        slopes[torch.arange(rows, device="cuda"), targets.long()] -= 1.0
        slopes *= float(torch.tensor(scale)) / rows
        h, element = features.double(), 2.0**-24 if dtype == torch.float32 else 2.0**-8
        products = 6 if dtype == torch.float32 else 1
        each = element + 2.0**-20 + 2 * A * (products * (rows / 16 + 1) + 8)
        close(to_weight, slopes.T @ h, slopes.abs().T @ h.abs() * each + (slopes.T @ h).abs() * element * 1.01)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,training", PASSES)
def test_rows_without_any_logit_have_no_softmax(ctx, rows, training, dtype):
    """Every logit of a row is -inf, as after a mask that leaves nothing: NaN, in that row alone."""
    labels, dim = 500, 40
    features, weight = matrix(rows, dim, dtype, 1), matrix(labels, dim, dtype, 2)
    features[:, 0], weight[:, 0] = 0.0, torch.finfo(dtype).min
    bare = torch.zeros(rows, dtype=torch.bool, device="cuda")
    bare[::7] = True
    features[bare] = 0.0
    features[bare, 0] = 3.0  # past f32's range
    targets = tokens_for("all", rows, labels, torch.int32, 3)
    b = Bounds(features, weight, targets, 1.0)
    head = sb.LabelHead(ctx, labels, dim, dtype, rows, training=training)
    loss = head.loss(features, weight, targets)
    assert loss.losses[bare].isnan().all() and loss.log_normalizers[bare].isnan().all() and loss.mean.isnan()
    close(loss.losses[~bare], b.losses[~bare], b.loss_error[~bare])
    _, log_probabilities = head.predict(features, weight)
    assert log_probabilities[bare].isnan().all()
    assert log_probabilities[~bare].isfinite().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [5, 20, 40, 64, 65, 300])
def test_predicted_labels_are_labels(ctx, rows, dtype):
    """Rows of NaN, of logits all -inf and of an infinite logit: the label of the largest that is a number, 0
    if there is none, and a log-probability of NaN."""
    labels, dim = 500, 40
    features, weight = matrix(rows, dim, dtype, 1), matrix(labels, dim, dtype, 2)
    features[:, 0], weight[:, 0] = 0.0, torch.finfo(dtype).min
    features[0] = float("nan")
    features[2], features[2, 0] = 0.0, 3.0  # -inf throughout
    weight[:, 1] = -1.0
    weight[[77, 402], 1] = 1.0
    features[4], features[4, 1] = 0.0, float("inf")  # +inf twice, -inf elsewhere
    head = sb.LabelHead(ctx, labels, dim, dtype, rows, training=False)
    got, log_probabilities = head.predict(features, weight)
    assert got[[0, 2, 4]].tolist() == [0, 0, 77]
    assert log_probabilities[[0, 2, 4]].isnan().all()
    ordinary = torch.ones(rows, dtype=torch.bool, device="cuda")
    ordinary[[0, 2, 4]] = False
    want = Bounds(features[ordinary], weight, None, 1.0)
    picked = want.z.gather(1, got[ordinary].long()[:, None])[:, 0]
    assert (want.z.amax(1) - picked <= 2 * want.z_error).all()
    assert log_probabilities[ordinary].isfinite().all()


def test_sizes_as_the_header_states_them(ctx):
    """The largest dim goes through, the next ones are refused, as are counts past theirs."""
    f32, dim = torch.float32, (1 << 20) - 1
    e = sb.Embedding(ctx, 3, dim, f32, 4)
    table, tokens = matrix(3, dim, f32, 1), torch.tensor([2, 0, 2, -1], device="cuda")
    assert torch.equal(e.lookup(table, tokens, 2.0)[:3], 2.0 * table[tokens[:3]])
    upstream = matrix(4, dim, f32, 2)
    assert torch.equal(e.gradient(upstream, tokens), torch.stack([upstream[1], 0 * upstream[1], upstream[0] + upstream[2]]))
    for sizes in ((3, 1 << 20, 4), (1 << 31, 4, 4), (3, 4, 1 << 30)):
        with pytest.raises(sb.SplatError):
            sb.Embedding(ctx, sizes[0], sizes[1], f32, sizes[2])
    for sizes in ((3, 1 << 20, 4), ((1 << 31) - 512, 4, 4), (3, 4, (1 << 31) - 512)):
        with pytest.raises(sb.SplatError):
            sb.LabelHead(ctx, sizes[0], sizes[1], f32, sizes[2])
