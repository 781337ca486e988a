"""The label operators at the ends of their types' ranges and of their sizes: operands near the largest
finite value and infinite ones, labels out of use, gradients weighted by row, wide features, the
workspace. Against plain 64-bit results, with the bounds of test_gpu_labels."""

from __future__ import annotations

import re
from pathlib import Path

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


@pytest.mark.parametrize("rows,labels,dim,factor", [(129, 300, 64, "uniform"), (256, 1000, 64, "uniform"),
                                                    (1000, 300, 72, "random"), (1000, 300, 72, "uniform"),
                                                    (3001, 65, 200, "by label")])
def test_bf16_weight_gradient_of_weighted_rows_is_rounded_once(ctx, rows, labels, dim, factor):
    """Each value is within half a unit in the last place (8 bits) of its exact sum, give or take its terms'
    2^-15 (a slope in two parts is off by 2^-17, and by as much again where its logit is, with logits up to 16)
    and the f32 sum of both parts over the rows. One rounding of slopes of one factor would be up to 2^-9 of the
    terms, all of one sign."""
    head = sb.LabelHead(ctx, labels, dim, torch.bfloat16, rows)
    features, weight = matrix(rows, dim, torch.bfloat16, 1), matrix(labels, dim, torch.bfloat16, 2)
    targets = tokens_for("some", rows, labels, torch.int64, 3)
    held = (targets >= 0) & (targets < labels)
    at = targets.clamp(0, labels - 1)
    factors = {"uniform": torch.full((rows,), 1.0 / rows, device="cuda"),
               "random": torch.rand(rows, device="cuda", generator=torch.Generator("cuda").manual_seed(4)) - 0.3,
               "by label": torch.rand(labels, device="cuda", generator=torch.Generator("cuda").manual_seed(5))[at]}
    loss = head.loss(features, weight, targets, 0.2)
    to_features, to_weight = head.gradient(features, weight, targets, loss.log_normalizers, 0.2, factors[factor])
    h, w = features.double(), weight.double()
    logits = 0.2 * h @ w.T
    assert logits.abs().max() < 16
    slopes = torch.softmax(logits, 1)
    slopes[torch.arange(rows, device="cuda"), at] -= 1
    slopes *= (float(torch.tensor(0.2)) * factors[factor].double() * held)[:, None]
    want, terms = slopes.T @ h, slopes.T.abs() @ h.abs()
    half = torch.ldexp(torch.ones_like(want), torch.frexp(want).exponent - 9)
    assert (((to_weight.double() - want).abs() - half) <= (2.0**-15 + 2 * A * (2 * (rows / 16 + 1) + 8)) * terms).all()
    b = Bounds(features, weight, targets, 0.2, factors[factor])
    close(to_features, b.to_features, b.features_error)
    again = head.gradient(features, weight, targets, loss.log_normalizers, 0.2, factors[factor])
    assert torch.equal(again[0], to_features) and torch.equal(again[1], to_weight)


@pytest.mark.parametrize("rows", [100, 129, 700])
def test_confident_weighted_rows_keep_their_slopes(ctx, rows):
    """As test_confident_rows_keep_their_small_losses_and_slopes, bf16 with a factor a row: the slopes are made in
    tiles of another shape than the loss's, of the same logits bit for bit."""
    labels, dim, scale = 40, 256, 20.0
    weight = matrix(labels, dim, torch.bfloat16, 2)
    weight /= weight.float().norm(dim=1, keepdim=True).to(torch.bfloat16)
    targets = tokens_for("all", rows, labels, torch.int32, 3)
    features = (weight[targets.long()].float() + 0.05 * matrix(rows, dim, torch.float32, 4) / dim**0.5).bfloat16()
    factors = matrix(1, rows, torch.float32, 5)[0].contiguous()
    exact = Bounds(features, weight, targets, scale, factors)
    assert (torch.exp(-exact.losses) > 0.999).float().mean() > 0.5
    head = sb.LabelHead(ctx, labels, dim, torch.bfloat16, rows)
    loss = head.loss(features, weight, targets, scale)
    to_features, to_weight = head.gradient(features, weight, targets, loss.log_normalizers, scale, factors)
    # Two roundings to bf16 (slopes, result), each at most 2^-9 of a value; the logits' errors are far below.
    for got, want in ((to_features, exact.to_features), (to_weight, exact.to_weight)):
        assert float((got.double() - want).norm() / want.norm()) <= 2.0**-8


@pytest.mark.parametrize("kind", ["all", "some", "none after row 200"])
def test_weighted_rows_in_chunks(ctx, kind):
    """Slopes in two parts of half as many rows a time: several chunks of rows with factors of their own."""
    rows, labels, dim = 6200, 70_000, 24
    head = sb.LabelHead(ctx, labels, dim, torch.bfloat16, rows)
    features, weight = matrix(rows, dim, torch.bfloat16, 1), matrix(labels, dim, torch.bfloat16, 2)
    targets = tokens_for("some" if kind == "some" else "all", rows, labels, torch.int64, 3)
    if kind == "none after row 200":
        targets[200:] = -1
    factors = matrix(1, rows, torch.float32, 5)[0].contiguous()
    loss = head.loss(features, weight, targets, 0.3)
    to_features, to_weight = head.gradient(features, weight, targets, loss.log_normalizers, 0.3, factors)
    want_weight = torch.zeros(labels, dim, dtype=torch.float64, device="cuda")
    weight_error = torch.zeros_like(want_weight)
    for first in range(0, rows, 1000):
        part = slice(first, min(rows, first + 1000))
        b = Bounds(features[part], weight, targets[part], 0.3, factors[part])
        want_weight += b.to_weight
        weight_error += b.weight_error
        close(to_features[part], b.to_features, b.features_error)
    close(to_weight, want_weight, weight_error * 1.1)  # the chunks' sums add f32 roundings
    again = head.gradient(features, weight, targets, loss.log_normalizers, 0.3, factors)
    assert torch.equal(again[0], to_features) and torch.equal(again[1], to_weight)
    head.check()


@pytest.mark.parametrize("rows,labels,dim", [(129, 300, 64), (256, 1000, 64), (2000, 1000, 72), (1023, 2050, 40)])
def test_bf16_weight_gradient_of_a_small_batch_is_rounded_once(ctx, rows, labels, dim):
    """The mean's call, bounded as test_bf16_weight_gradient_of_weighted_rows_is_rounded_once."""
    head = sb.LabelHead(ctx, labels, dim, torch.bfloat16, rows)
    features, weight = matrix(rows, dim, torch.bfloat16, 1), matrix(labels, dim, torch.bfloat16, 2)
    targets = tokens_for("all", rows, labels, torch.int64, 3)
    loss = head.loss(features, weight, targets, 0.2)
    _, to_weight = head.gradient(features, weight, targets, loss.log_normalizers, 0.2)
    h, w = features.double(), weight.double()
    logits = float(torch.tensor(0.2)) * h @ w.T
    assert logits.abs().max() < 16
    slopes = torch.softmax(logits, 1)
    slopes[torch.arange(rows, device="cuda"), targets] -= 1
    slopes *= float(torch.tensor(0.2)) / rows
    want, terms = slopes.T @ h, slopes.T.abs() @ h.abs()
    half = torch.ldexp(torch.ones_like(want), torch.frexp(want).exponent - 9)
    assert (((to_weight.double() - want).abs() - half) <= (2.0**-15 + 2 * A * (2 * (rows / 16 + 1) + 8)) * terms).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,training", PASSES)
@pytest.mark.parametrize("dim", [64, 768, 4096, 65_536])
def test_exact_logits_of_wide_features(ctx, rows, training, dim, dtype):
    """Features of a single 1: each logit is a weight, as it is. What is given back for the truncation of sums, an
    eighth of 2^-23 an addition of 16 columns, is not lost here; it stays bounded however wide the features are."""
    head = sb.LabelHead(ctx, 1, dim, dtype, rows, training=training)
    features, weight = torch.zeros(rows, dim, dtype=dtype, device="cuda"), matrix(1, dim, dtype, 2)
    column = torch.arange(rows, device="cuda") * 977 % dim
    features[torch.arange(rows, device="cuda"), column] = 1.0
    targets = torch.zeros(rows, dtype=torch.int32, device="cuda")
    loss = head.loss(features, weight, targets)
    want = weight[0, column].double()  # of one label, the normalizer is its logit
    given = (min(dim // 16, 256) + 1) / 8
    # f32 roundings of the scale and of the sums of three parts beside what is given back.
    assert ((loss.log_normalizers - want).abs() <= want.abs() * (given + 3) * 2.0**-23).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,labels,dim", [(1, 2, 16), (100, 100, 768), (300, 150, 1024), (60_000, 20, 512), (20, 60_000, 512)])
def test_workspace_follows_the_sizes(ctx, rows, labels, dim, dtype):
    """A head made for little holds little: copies of its operands, their slopes, and sums of the gradients in at
    most as many pieces as their inner dimension has steps of 256 (f32: of 2048 at least), beside 32 MB."""
    sb.LabelHead(ctx, 2, 16, dtype, 1).close()  # what the first head of a process loads
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    head = sb.LabelHead(ctx, labels, dim, dtype, rows)
    used = before - torch.cuda.mem_get_info()[0]
    up = lambda k, to: -(-k // to) * to  # noqa: E731
    parts = 3 if dtype == torch.float32 else 1
    operands = (up(rows, 256) + labels) * up(dim, 64) * 2 * parts
    slopes = 2 * up(rows, 256) * up(labels, 256) * 2 * parts
    sums = (rows * (1 + labels // 256) + labels * (1 + rows // 256)) * up(dim, 4) * 4
    assert used <= operands + slopes + min(sums, 2 * (4 * 148 * 128 + rows + labels) * up(dim, 4) * 4) + (32 << 20)
    head.close()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [0, 9, 32_768, 32_769])
@pytest.mark.parametrize("scale", [float("inf"), float("nan"), -2.0])
def test_entries_without_tokens_have_zero_rows_whatever_the_scale(ctx, n, scale, dtype):
    entries, dim = 50, 24
    e = sb.Embedding(ctx, entries, dim, dtype, max(n, 1))
    tokens = torch.arange(n, device="cuda") % 7
    upstream = torch.ones(n, dim, dtype=dtype, device="cuda")
    got = e.gradient(upstream, tokens, scale)
    assert got[min(n, 7):].count_nonzero() == 0
    count = torch.bincount(tokens, minlength=entries)[: min(n, 7), None].float() * scale
    assert torch.equal(got[: min(n, 7)].nan_to_num(nan=7.0), count.to(dtype).expand(-1, dim).nan_to_num(nan=7.0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,labels,dim", [(5000, 150, 45), (3001, 4099, 64), (20_003, 257, 24), (700, 9000, 300)])
def test_predict_of_many_rows(ctx, rows, labels, dim, dtype):
    """As test_predict, at the sizes of a scene: several tiles of rows, labels cut into pieces or not."""
    head = sb.LabelHead(ctx, labels, dim, dtype, rows, training=False)
    features, weight = matrix(rows, dim, dtype, 1), matrix(labels, dim, dtype, 2)
    b = Bounds(features, weight, None, 0.4)
    got, log_probabilities = head.predict(features, weight, 0.4)
    best = b.z.amax(1)
    close(log_probabilities, best - b.normalizers, 2 * b.z_error + b.exp_error + 4 * A * b.normalizers.abs())
    top = torch.topk(b.z, 2, 1).values
    clear = top[:, 0] - top[:, 1] > 2 * b.z_error
    assert clear.float().mean() > 0.9
    assert torch.equal(got[clear].long(), b.z.argmax(1)[clear])


@pytest.mark.parametrize("dtype", TYPES)
def test_gradient_beyond_the_budget_of_slopes(ctx, dtype):
    """Rows past what the budget holds at once, whatever the budget is: the weight's gradient over the chunks."""
    source = (Path(__file__).resolve().parents[1] / "splatting-rs_b200/csrc/label_head.cu").read_text()
    factor, shift = re.search(r"kSlopeBudget = (\d+)ull << (\d+);", source).groups()
    labels, dim, parts = 150_000, 16, 3 if dtype == torch.float32 else 1
    limit = (int(factor) << int(shift)) // (-(-labels // 256) * 256 * parts) // 256 * 256
    rows = limit + 300
    head = sb.LabelHead(ctx, labels, dim, dtype, rows)
    features, weight = matrix(rows, dim, dtype, 1), matrix(labels, dim, dtype, 2)
    targets = tokens_for("some", rows, labels, torch.int32, 3)
    loss = head.loss(features, weight, targets, 0.3)
    to_features, to_weight = head.gradient(features, weight, targets, loss.log_normalizers, 0.3)
    count = int(((targets >= 0) & (targets < labels)).sum())
    want_weight = torch.zeros(labels, dim, dtype=torch.float64, device="cuda")
    weight_error = torch.zeros_like(want_weight)
    for first in range(0, rows, 500):
        part = slice(first, min(rows, first + 500))
        b = Bounds(features[part], weight, targets[part], 0.3, torch.full((part.stop - first,), 1.0 / count, device="cuda"))
        want_weight += b.to_weight
        weight_error += b.weight_error
        close(to_features[part], b.to_features, b.features_error)
    close(to_weight, want_weight, weight_error * 1.1)  # the chunks' sums add f32 roundings
