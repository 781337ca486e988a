"""The label operators where they change the way they go, and the example that runs them together:
sizes on both sides of each rule, operands that cannot be read in place, offsets past 32 bits, a
context with a stream of its own. Against plain 64-bit results, with the bounds of test_gpu_labels."""

from __future__ import annotations

import sys
from pathlib import Path

import pytest
import torch

import splat_b200 as sb
from test_gpu_labels import A, TYPES, U, Bounds, close, matrix, tokens_for

pytestmark = pytest.mark.gpu


def gradient_bound(upstream, tokens, entries, scale):
    """(table gradient, error bound) as in test_embedding_gradient."""
    held = (tokens >= 0) & (tokens < entries)
    at, rows = tokens[held].long(), upstream[held].double()
    dim = upstream.shape[1]
    want = torch.zeros(entries, dim, dtype=torch.float64, device="cuda").index_add_(0, at, rows)
    size = torch.zeros(entries, dim, dtype=torch.float64, device="cuda").index_add_(0, at, rows.abs())
    count = torch.bincount(at, minlength=entries)[:, None]
    return want * scale, scale * (size * (count + 1) * A + want.abs() * U[upstream.dtype]) * (1 + 1e-3)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize(
    "n,entries,dim,kind",
    [(32_768, 40, 24, "some"), (32_769, 40, 24, "some"),  # one kernel, and the sorted list
     (32_768, 3, 200, "all"), (40_000, 30, 200, "all"),   # few entries: column tiles, a warp per join
     (64, 1, 64, "all"), (65, 1, 64, "all"),              # a run of one group, and of all of them
     (500, 20_000, 40, "some"), (2000, 90_000, 16, "all"),  # many entries a block, mostly without rows
     (75_775, 7, 33, "skewed"), (75_776, 7, 33, "skewed"),  # pieces of 16 and of 32
     (151_552, 500, 12, "skewed"), (303_104, 2, 16, "skewed"), (310_000, 70_000, 8, "some")],
)
def test_embedding_gradient_paths(ctx, n, entries, dim, kind, dtype):
    e = sb.Embedding(ctx, entries, dim, dtype, n)
    upstream, tokens = matrix(n, dim, dtype, 3), tokens_for(kind, n, entries, torch.int32, 4)
    want, bound = gradient_bound(upstream, tokens, entries, 1.0)
    got = e.gradient(upstream, tokens)
    close(got, want, bound)
    assert torch.equal(got, e.gradient(upstream, tokens))
    e.check()


def test_one_handle_for_calls_of_all_sizes(ctx):
    """Workspaces are shared by the calls of a handle, whatever way each goes."""
    entries, dim = 300, 64
    e = sb.Embedding(ctx, entries, dim, torch.float32, 200_000)
    for n in (200_000, 10, 33_000, 0, 160_000, 32_768, 1):
        upstream, tokens = matrix(n, dim, torch.float32, n), tokens_for("skewed", n, entries, torch.int64, n + 1)
        want, bound = gradient_bound(upstream, tokens, entries, 1.0)
        close(e.gradient(upstream, tokens), want, bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [16, 17, 64, 65, 128, 129])
@pytest.mark.parametrize("pad,shift,dim", [(0, 0, 72), (1, 0, 72), (0, 1, 64), (3, 5, 200)])
def test_predict_and_loss_around_the_few_row_pass(ctx, rows, pad, shift, dim, dtype):
    labels = 1500
    head = sb.LabelHead(ctx, labels, dim, dtype, 200, training=False)
    features = matrix(rows, dim, dtype, 1, pad, shift, spread=dim**-0.25)
    weight = matrix(labels, dim, dtype, 2, shift=0 if shift == 1 else shift, pad=pad, spread=dim**-0.25)
    b = Bounds(features, weight, None, 1.3)
    got, log_probabilities = head.predict(features, weight, 1.3)
    best = b.z.amax(1)
    close(log_probabilities, best - b.normalizers, 2 * b.z_error + b.exp_error + 4 * A * b.normalizers.abs())
    assert (best - b.z.gather(1, got.long()[:, None])[:, 0] <= 2 * b.z_error).all()
    targets = tokens_for("some", rows, labels, torch.int32, 3)
    b = Bounds(features, weight, targets, 1.3)
    loss = head.loss(features, weight, targets, 1.3)
    close(loss.losses, b.losses, b.loss_error)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,labels,dim", [(1030, 20_000, 40), (3000, 259, 33), (20_500, 130, 16), (66, 40_000, 16)])
def test_loss_and_gradient_in_pieces(ctx, rows, labels, dim, dtype):
    """Label tiles cut into pieces, row targets counted by groups, gradients summed from pieces."""
    head = sb.LabelHead(ctx, labels, dim, dtype, rows)
    features, weight = matrix(rows, dim, dtype, 1, spread=0.5), matrix(labels, dim, dtype, 2, spread=0.5)
    targets = tokens_for("some", rows, labels, torch.int64, 3)
    b = Bounds(features, weight, targets, 1.0)
    loss = head.loss(features, weight, targets)
    close(loss.losses, b.losses, b.loss_error)
    assert abs(loss.mean.double() - b.losses.sum() / len(b.rows)) <= b.loss_error.sum() / len(b.rows) + A * abs(loss.mean)
    to_features, to_weight = head.gradient(features, weight, targets, loss.log_normalizers)
    close(to_features, b.to_features, b.features_error)
    close(to_weight, b.to_weight, b.weight_error)


def test_logits_that_grow_along_the_vocabulary(ctx):
    """Each label tile raises the largest logit by more than the sums' range: the base moves on."""
    rows, labels, dim = 130, 2000, 16
    for dtype in TYPES:
        head = sb.LabelHead(ctx, labels, dim, dtype, rows)
        features = torch.ones(rows, dim, dtype=dtype, device="cuda")
        weight = torch.arange(labels, device="cuda")[:, None].expand(labels, dim).to(dtype).contiguous()
        targets = tokens_for("all", rows, labels, torch.int32, 3)
        for few in (False, True):
            some = slice(0, 40) if few else slice(0, rows)
            b = Bounds(features[some], weight, targets[some], 1.0)
            loss = head.loss(features[some], weight, targets[some])
            close(loss.losses, b.losses, b.loss_error)


def test_lowest_values_of_the_type_as_labels_out_of_use(ctx):
    """Label rows that push their logits to the type's lowest values have probability 0 and no gradient."""
    rows, labels, dim = 200, 300, 32
    head = sb.LabelHead(ctx, labels, dim, torch.bfloat16, rows)
    features, weight = matrix(rows, dim, torch.bfloat16, 1), matrix(labels, dim, torch.bfloat16, 2)
    features[:, 0] = 1.0
    off = torch.arange(0, labels, 3, device="cuda")
    weight[off] = 0
    weight[off, 0] = torch.finfo(torch.bfloat16).min
    keep = torch.ones(labels, dtype=torch.bool, device="cuda")
    keep[off] = False
    targets = torch.nonzero(keep)[:, 0][torch.randint(0, int(keep.sum()), (rows,), device="cuda")]
    b = Bounds(features, weight[keep], torch.searchsorted(torch.nonzero(keep)[:, 0], targets), 1.0)
    loss = head.loss(features, weight, targets)
    close(loss.losses, b.losses, b.loss_error)
    _, to_weight = head.gradient(features, weight, targets, loss.log_normalizers)
    assert to_weight[off].count_nonzero() == 0
    close(to_weight[keep], b.to_weight, b.weight_error)


def test_offsets_past_32_bits(ctx):
    """Rows further apart than 2^31 elements in all."""
    rows, stride, dim = 70_000, 32_768, 16
    wide = torch.zeros(rows, stride, dtype=torch.bfloat16, device="cuda")
    far = wide[:, :dim]
    far.copy_(torch.randn(rows, dim, device="cuda"))
    packed = far.contiguous()
    tokens = tokens_for("some", 4000, rows, torch.int64, 1)
    e = sb.Embedding(ctx, rows, dim, torch.bfloat16, 4000)
    found = e.lookup(packed, tokens)
    assert torch.equal(e.lookup(far, tokens), found)
    want = e.gradient(found, tokens).clone()
    e.gradient(found, tokens, out=far)
    assert torch.equal(far, want)
    far.copy_(packed)
    head = sb.LabelHead(ctx, 64, dim, torch.bfloat16, rows)
    weight, targets = matrix(64, dim, torch.bfloat16, 2), tokens_for("some", rows, 64, torch.int32, 3)
    near, away = head.loss(packed, weight, targets), head.loss(far, weight, targets)
    assert torch.equal(near.losses, away.losses)
    to_near, _ = head.gradient(packed, weight, targets, near.log_normalizers)
    head.gradient(packed, weight, targets, near.log_normalizers, feature_gradient=far)
    assert torch.equal(far, to_near)
    targets = tokens_for("all", 90, rows, torch.int32, 4)
    codes = sb.LabelHead(ctx, rows, dim, torch.bfloat16, 90)
    far.copy_(packed)
    assert torch.equal(codes.loss(packed[:90], far, targets).losses, codes.loss(packed[:90], packed, targets).losses)


def test_a_context_with_a_stream_of_its_own():
    stream = torch.cuda.Stream()
    own = sb.Context(0, stream=stream.cuda_stream)
    rows, labels, dim = 300, 400, 64
    weight, targets = matrix(labels, dim, torch.float32, 2), tokens_for("some", rows, labels, torch.int32, 3)
    head, e = sb.LabelHead(own, labels, dim, torch.float32, rows), sb.Embedding(own, labels, dim, torch.float32, rows)
    for _ in range(5):
        torch.cuda._sleep(200_000)  # the operands are late on the current stream
        table = weight * 1
        features = e.lookup(table, targets)
        loss = head.loss(features, table, targets)
        to_features, _ = head.gradient(features, table, targets, loss.log_normalizers)
        back = e.gradient(to_features, targets) * 1
        b = Bounds(features, weight, targets, 1.0)
        close(loss.losses, b.losses, b.loss_error)
        close(to_features, b.to_features, b.features_error)
        want, bound = gradient_bound(to_features, targets, labels, 1.0)
        close(back, want, bound)
    e.close(), head.close()


@pytest.mark.parametrize("dtype", TYPES)
def test_the_example_learns_its_scene(dtype):
    sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))
    import label_scene

    result = label_scene.train(steps=60, dtype=dtype, scale=0.1)
    # It starts at the loss of a uniform guess among 100 labels (small random weights: within 0.1 of
    # ln 100) and ends far below it; a token's Gaussians mostly share their region.
    assert abs(result["first_loss"] - 4.605) < 0.1
    assert result["last_loss"] < 0.5 * result["first_loss"]
    assert result["accuracy"] > 0.5


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,labels,dim", [(5, 20, 256), (300, 40, 300), (700, 900, 64), (3000, 30, 128)])
def test_confident_rows_keep_their_small_losses_and_slopes(ctx, rows, labels, dim, dtype):
    """Targets of probability close to 1: the loss and the slopes are what the other labels leave, and
    keep their relative precision (f32: a few roundings of logits of size 20, exp makes them relative)."""
    weight = matrix(labels, dim, dtype, 2)
    weight /= weight.float().norm(dim=1, keepdim=True).to(dtype)
    targets = tokens_for("all", rows, labels, torch.int32, 3)
    features = (weight[targets.long()].float() + 0.05 * torch.randn(rows, dim, device="cuda") / dim**0.5).to(dtype)
    scale = 20.0
    exact = Bounds(features, weight, targets, scale)
    p = torch.exp(-exact.losses)
    assert (p > 0.9).float().mean() > 0.5
    head = sb.LabelHead(ctx, labels, dim, dtype, rows)
    loss = head.loss(features, weight, targets, scale)
    # Each other label's share of the loss: exp of a difference of two logits.
    products = 6 if dtype == torch.float32 else 1
    each = 2 * A * 2 * (products * (dim / 16 + 1) + 4) * scale * (features.double().abs() @ weight.double().abs().T).amax(1)
    each = each + 8 * A * 20 * 2 + 2.0**-20
    close(loss.losses, exact.losses, exact.losses * each * 2)
    to_features, to_weight = head.gradient(features, weight, targets, loss.log_normalizers, scale)
    if dtype == torch.float32:
        for got, want in ((to_features, exact.to_features), (to_weight, exact.to_weight)):
            error = float((got.double() - want).norm() / want.norm())
            assert error <= float(2 * each.max()), f"relative error {error:.1e}"
    probe = sb.LabelHead(ctx, labels, dim, dtype, rows, training=False)
    close(probe.loss(features, weight, targets, scale).losses, exact.losses, exact.losses * each * 2)
    labels_found, log_probabilities = probe.predict(features, weight, scale)
    assert torch.equal(labels_found, targets)
    close(log_probabilities, -exact.losses, exact.losses * each * 2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["all", "some", "none after row 200"])
def test_gradient_of_more_slopes_than_the_workspace_holds(ctx, dtype, kind):
    """Above 671 million slopes (f32: a third of that) the rows go in chunks, and the weight's gradient is
    summed over them; a chunk without targets adds nothing."""
    rows, labels, dim = (10_300, 70_000, 24) if dtype == torch.bfloat16 else (3700, 70_000, 24)
    head = sb.LabelHead(ctx, labels, dim, dtype, rows)
    features, weight = matrix(rows, dim, dtype, 1), matrix(labels, dim, dtype, 2)
    targets = tokens_for("some" if kind == "some" else "all", rows, labels, torch.int64, 3)
    if kind == "none after row 200":
        targets[200:] = -1
    loss = head.loss(features, weight, targets, 0.3)
    to_features, to_weight = head.gradient(features, weight, targets, loss.log_normalizers, 0.3)
    count = int(((targets >= 0) & (targets < labels)).sum())
    want_weight = torch.zeros(labels, dim, dtype=torch.float64, device="cuda")
    weight_error = torch.zeros_like(want_weight)
    for first in range(0, rows, 1000):
        part = slice(first, min(rows, first + 1000))
        g = torch.full((part.stop - first,), 1.0 / count, device="cuda")
        b = Bounds(features[part], weight, targets[part], 0.3, g)
        want_weight += b.to_weight
        weight_error += b.weight_error
        close(loss.losses[part], b.losses, b.loss_error)
        close(to_features[part], b.to_features, b.features_error)
    close(to_weight, want_weight, weight_error * 1.1)  # the chunks' sums add f32 roundings
    again = head.gradient(features, weight, targets, loss.log_normalizers, 0.3)
    assert torch.equal(again[0], to_features) and torch.equal(again[1], to_weight)
    head.check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,pad,shift", [(45, 0, 0), (45, 3, 1), (64, 0, 1), (64, 8, 0), (6, 2, 2), (300, 4, 0)])
def test_embedding_gradient_writes_every_row_and_nothing_else(ctx, dim, pad, shift, dtype):
    """The sorted list's way: rows of zeros for entries without tokens, in 16-byte, 4-byte and 2-byte
    units, dense or not; what lies between the rows and around them stays."""
    n, entries = 40_000, 999
    e = sb.Embedding(ctx, entries, dim, dtype, n)
    upstream, tokens = matrix(n, dim, dtype, 3), tokens_for("some", n, entries, torch.int32, 4)
    tokens[(tokens > 300) & (tokens < 700)] = -1  # a gap, and ones at both ends
    tokens[(tokens < 5) | (tokens > 990)] = 9
    whole = torch.full((shift + entries * (dim + pad) + 8,), -7.0, dtype=dtype, device="cuda")
    out = whole[shift:shift + entries * (dim + pad)].view(entries, dim + pad)[:, :dim]
    want, bound = gradient_bound(upstream, tokens, entries, 0.5)
    close(e.gradient(upstream, tokens, 0.5, out=out), want, bound)
    assert out[301:700].count_nonzero() == 0 and out[:5].count_nonzero() == 0 and out[991:].count_nonzero() == 0
    out.zero_()
    assert (whole == -7).sum() == whole.numel() - entries * dim, "wrote outside its rows"
    e.check()


@pytest.mark.parametrize("n", [40_000, 75_000, 400_000])
def test_embedding_gradient_of_runs_over_many_stretches(ctx, n):
    """One token for nearly all rows, at the list's begin, middle or end, and runs that begin and end at
    the stretches' borders."""
    entries, dim = 64, 24
    e = sb.Embedding(ctx, entries, dim, torch.float32, n)
    upstream = matrix(n, dim, torch.float32, 5)
    place = torch.arange(n, device="cuda")
    cases = [torch.full((n,), v, device="cuda") for v in (0, 31, 63)]
    cases += [place // length % entries for length in (512, 1024, 2048, 4096)]
    cases += [torch.where(place < k, 3, 40) for k in (1, 2047, 2048, 2049, n - 1)]
    cases += [torch.where(place < n // 2, 7, -1), torch.full((n,), -1, device="cuda")]
    for tokens in cases:
        want, bound = gradient_bound(upstream, tokens, entries, 1.0)
        close(e.gradient(upstream, tokens), want, bound)
    e.check()


@pytest.mark.parametrize("rows,labels,dim", [(1, 700, 40), (2, 21, 242), (15, 1186, 33), (90, 5117, 156), (128, 398, 64)])
def test_bf16_weight_gradient_of_few_rows_is_rounded_once(ctx, rows, labels, dim):
    """Each value is within half a unit in the last place (8 bits) of its exact sum, give or take 2^-15 of
    the sum's terms: a slope in two parts is off by 2^-17, and by as much again where its logit is (logits up
    to 16, f32 sums over at most 256 columns, exponentials to 2^-21). One rounding of the slopes to bf16 would
    be 2^-9 of the terms."""
    head = sb.LabelHead(ctx, labels, dim, torch.bfloat16, rows)
    features, weight = matrix(rows, dim, torch.bfloat16, 1), matrix(labels, dim, torch.bfloat16, 2)
    targets = tokens_for("all", rows, labels, torch.int64, 3)
    loss = head.loss(features, weight, targets, 0.2)
    _, to_weight = head.gradient(features, weight, targets, loss.log_normalizers, 0.2)
    h, w = features.double(), weight.double()
    logits = 0.2 * h @ w.T
    assert logits.abs().max() < 16
    slopes = torch.softmax(logits, 1)
    slopes[torch.arange(rows), targets] -= 1
    want, terms = 0.2 / rows * slopes.T @ h, 0.2 / rows * slopes.T.abs() @ h.abs()
    half = torch.ldexp(torch.ones_like(want), torch.frexp(want).exponent - 9)
    assert (((to_weight.double() - want).abs() - half) <= 2.0**-15 * terms).all()
