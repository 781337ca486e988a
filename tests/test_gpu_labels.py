"""The label operators on a GPU against their definitions in 64 bits: the embedding of tokens and
its gradient, the label head's loss, gradient and prediction.

Tolerances are bounds on the rounding errors, element by element, from the definitions' own
magnitudes (`Bounds`): U is half a unit in the last place of the element type, A the error of one
f32 addition (2^-24; 2^-23 on the tensor cores, which truncate).
"""

from __future__ import annotations

import pytest
import torch

import splat_b200 as sb

pytestmark = pytest.mark.gpu

A = 2.0**-24
U = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8}
TYPES = [torch.float32, torch.bfloat16]


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def matrix(rows, columns, dtype, seed, pad=0, shift=0, spread=1.0):
    """Random rows; `pad` more elements of row stride, `shift` elements off the allocation's base."""
    g = generator(seed)
    flat = torch.full((shift + rows * (columns + pad) + 8,), float("nan"), dtype=dtype, device="cuda")
    view = flat[shift : shift + rows * (columns + pad)].view(rows, columns + pad)[:, :columns]
    view.copy_(torch.randn(rows, columns, generator=g, device="cuda") * spread)
    return view


def tokens_for(kind, n, entries, dtype, seed):
    g = generator(seed)
    t = torch.randint(0, entries, (n,), generator=g, device="cuda")
    if kind == "one":
        t = torch.full_like(t, entries - 1)
    elif kind == "none":
        t = torch.full_like(t, -1)
    elif kind == "some":
        gone = torch.rand(n, generator=g, device="cuda")
        t = torch.where(gone < 0.3, torch.full_like(t, -1), t)
        t = torch.where(gone > 0.9, torch.full_like(t, entries), t)  # past the end is none too
    elif kind == "skewed":
        t = torch.minimum(t, torch.randint(0, entries, (n,), generator=g, device="cuda") // 7)
    return t.to(dtype)


def close(got, want, tolerance):
    got, want = got.double(), want.double()
    assert torch.isfinite(got).all()
    worst = ((got - want).abs() - tolerance).max() if got.numel() else torch.tensor(-1.0)
    assert worst <= 0, f"beyond the bound by {worst.item():.3e}"


# ------------------------------------------------------------------ embedding


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize(
    "n,entries,dim,pad,shift,kind",
    [(1, 1, 1, 0, 0, "all"), (5, 3, 7, 2, 1, "some"), (1000, 37, 45, 0, 0, "some"), (777, 1000, 64, 8, 0, "all"),
     (4099, 300, 256, 0, 0, "skewed"), (300, 50, 1100, 4, 0, "some"), (64, 10, 24, 0, 3, "none")],
)
def test_lookup(ctx, n, entries, dim, pad, shift, kind, dtype):
    e = sb.Embedding(ctx, entries, dim, dtype, n)
    table = matrix(entries, dim, dtype, 1, pad, shift)
    for index in (torch.int32, torch.int64):
        tokens = tokens_for(kind, n, entries, index, 2)
        got = e.lookup(table, tokens, 1.7)
        held = (tokens >= 0) & (tokens < entries)
        want = torch.zeros(n, dim, dtype=torch.float64, device="cuda")
        want[held] = table.double()[tokens[held].long()] * float(torch.tensor(1.7))
        # The f32 product and its rounding to the element type.
        close(got, want, want.abs() * (U[dtype] + 2 * A))
        assert got[~held].count_nonzero() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize(
    "n,entries,dim,pad,shift,kind",
    [(1, 1, 1, 0, 0, "all"), (1, 900, 8, 0, 0, "none"), (15, 4, 7, 2, 1, "some"), (16, 4, 64, 0, 0, "one"),
     (17, 300, 45, 0, 0, "all"), (3001, 300, 100, 0, 0, "some"), (5000, 70, 256, 8, 0, "one"),
     (20_000, 1000, 64, 0, 0, "skewed"), (100_000, 40, 48, 0, 0, "skewed"), (90_000, 70_000, 20, 0, 0, "some"),
     (80_000, 2, 260, 0, 0, "one"), (700, 90, 1100, 4, 0, "some")],
)
def test_embedding_gradient(ctx, n, entries, dim, pad, shift, kind, dtype):
    e = sb.Embedding(ctx, entries, dim, dtype, n)
    upstream = matrix(n, dim, dtype, 3, pad, shift)
    for index in (torch.int32, torch.int64):
        tokens = tokens_for(kind, n, entries, index, 4)
        held = (tokens >= 0) & (tokens < entries)
        upstream[~held] = float("nan")  # rows without a token are not read into any sum
        got = e.gradient(upstream, tokens, 0.3)
        at, rows = tokens[held].long(), upstream[held].double()
        want = torch.zeros(entries, dim, dtype=torch.float64, device="cuda").index_add_(0, at, rows)
        size = torch.zeros(entries, dim, dtype=torch.float64, device="cuda").index_add_(0, at, rows.abs())
        count = torch.bincount(at, minlength=entries)[:, None]
        scale = float(torch.tensor(0.3))
        # count additions in f32 at most, the scaling, the rounding to the element type.
        close(got, want * scale, scale * (size * (count + 1) * A + want.abs() * U[dtype]) * (1 + 1e-3))
        assert torch.equal(got, e.gradient(upstream, tokens, 0.3)), "two runs differ"
        upstream[~held] = 0
    e.check()


def test_embedding_of_nothing(ctx):
    e = sb.Embedding(ctx, 5, 8, torch.float32, 4)
    table = matrix(5, 8, torch.float32, 1)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    assert e.lookup(table, none).shape == (0, 8)
    assert e.gradient(torch.empty(0, 8, device="cuda"), none).count_nonzero() == 0


def test_embedding_gradient_against_differences(ctx):
    """<dT, D> equals the change of <R, lookup(T)> along D (the lookup is linear in T)."""
    n, entries, dim = 500, 60, 33
    e = sb.Embedding(ctx, entries, dim, torch.float32, n)
    tokens = tokens_for("some", n, entries, torch.int32, 1)
    table, direction, r = (matrix(k, dim, torch.float32, s) for k, s in ((entries, 2), (entries, 3), (n, 4)))
    change = (r.double() * (e.lookup(table + direction, tokens, 2.0).double() - e.lookup(table, tokens, 2.0).double())).sum()
    along = (e.gradient(r, tokens, 2.0).double() * direction.double()).sum()
    held = (tokens >= 0) & (tokens < entries)
    at = tokens[held].long()
    # table + direction is rounded, and so are both lookups; the gradient's sums as above.
    size = (r[held].abs().double() * 2.0 * (table[at].abs() + direction[at].abs()).double()).sum()
    assert abs(change - along) <= size * A * (4 + torch.bincount(at).max())


# ----------------------------------------------------------------- label head


class Bounds:
    """The loss, its gradient and their error bounds in 64 bits, for rows [n], labels [v]."""

    def __init__(self, features, weight, targets, scale, row_gradient=None):
        dtype, dim = features.dtype, features.shape[1]
        v = weight.shape[0]
        products = 6 if dtype == torch.float32 else 1
        scale = float(torch.tensor(scale))
        self.counted = (targets >= 0) & (targets < v) if targets is not None else torch.ones(
            features.shape[0], dtype=torch.bool, device="cuda")
        rows = torch.nonzero(self.counted)[:, 0]
        h, w = features[rows].double(), weight.double()
        z, size = scale * (h @ w.T), scale * (h.abs() @ w.abs().T)
        # Each logit: products accumulated 16 at a time with truncation, the parts left out of f32
        # products (2^-23 of each), the scaling; and in the exponent form one more rounding of z.
        per_z = size * (2 * A * (products * (dim / 16 + 1) + 4))
        self.z_error = per_z.amax(1) + 4 * A * z.abs().amax(1)
        self.rows, self.z = rows, z
        self.normalizers = torch.logsumexp(z, 1)
        # ex2.approx is good to 2^-22; the running sum adds at most v / 32 + 40 times.
        self.exp_error = 2.0**-21 + A * (v / 32 + 40)
        if targets is None:
            return
        at = targets[rows].long()
        self.losses = torch.zeros(features.shape[0], dtype=torch.float64, device="cuda")
        self.losses[rows] = self.normalizers - z.gather(1, at[:, None])[:, 0]
        self.loss_error = torch.zeros_like(self.losses)
        self.loss_error[rows] = (2 * self.z_error + self.exp_error + 4 * A * (self.normalizers.abs() + z.abs().amax(1)))
        count = max(1, len(rows))
        g = torch.full((len(rows),), 1.0 / count, dtype=torch.float64, device="cuda")
        if row_gradient is not None:
            g = row_gradient[rows].double()
        p = torch.exp(z - self.normalizers[:, None])
        p_error = p * (2 * self.z_error[:, None] + self.exp_error + 8 * A * (1 + self.normalizers.abs()[:, None]))
        slopes = p.clone()
        slopes[torch.arange(len(rows), device="cuda"), at] -= 1.0
        weights = (scale * g)[:, None]
        slope_error = weights.abs() * (p_error + slopes.abs() * (U[dtype] + 4 * A))
        slopes = slopes * weights
        n, d = features.shape
        add = lambda k: 2 * A * (products * (k / 16 + 1) + 8)  # noqa: E731
        self.to_features = torch.zeros(n, d, dtype=torch.float64, device="cuda")
        self.to_features[rows] = slopes @ w
        self.features_error = torch.zeros_like(self.to_features)
        self.features_error[rows] = slope_error @ w.abs() + add(v) * (slopes.abs() @ w.abs())
        self.features_error += self.to_features.abs() * U[dtype] * 1.01
        self.to_weight = slopes.T @ h
        self.weight_error = slope_error.T @ h.abs() + add(len(rows)) * (slopes.abs().T @ h.abs())
        self.weight_error += self.to_weight.abs() * U[dtype] * 1.01


HEADS = [
    # rows, labels, dim, pad, shift, targets, scale
    (1, 1, 1, 0, 0, "all", 1.0),
    (1, 130, 64, 0, 0, "all", 1.0),
    (3, 2, 5, 3, 1, "some", 2.0),
    (127, 127, 64, 0, 0, "all", 1.0),
    (128, 128, 128, 0, 0, "some", 0.5),
    (129, 129, 65, 0, 0, "all", 1.0),
    (300, 1000, 200, 8, 0, "some", 1.0),
    (257, 3001, 72, 0, 0, "some", 1.0),
    (5000, 150, 45, 0, 0, "some", 1.0),
    (700, 259, 520, 0, 8, "all", 1.0),
    (260, 5003, 129, 1, 0, "skewed", 4.0),
    (200, 300, 64, 0, 0, "none", 1.0),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,labels,dim,pad,shift,kind,scale", HEADS)
def test_loss_and_gradient(ctx, rows, labels, dim, pad, shift, kind, scale, dtype):
    head = sb.LabelHead(ctx, labels, dim, dtype, rows + 3)
    features = matrix(rows, dim, dtype, 1, pad, shift, spread=dim**-0.25)
    weight = matrix(labels, dim, dtype, 2, pad, shift, spread=dim**-0.25)
    for index, row_gradient in ((torch.int32, None), (torch.int64, matrix(1, rows, torch.float32, 5)[0].contiguous())):
        targets = tokens_for(kind, rows, labels, index, 3)
        held = (targets >= 0) & (targets < labels)
        features[~held] = float("nan")
        if rows > 1:
            features[~held, 0] = float("inf")
        b = Bounds(features, weight, targets, scale, row_gradient)
        loss = head.loss(features, weight, targets, scale)
        close(loss.losses, b.losses, b.loss_error)
        mean = b.losses.sum() / max(1, len(b.rows))
        assert abs(loss.mean.double() - mean) <= b.loss_error.sum() / max(1, len(b.rows)) + A * abs(mean)
        assert loss.losses[~held].count_nonzero() == 0 and loss.log_normalizers[~held].count_nonzero() == 0
        to_features, to_weight = head.gradient(features, weight, targets, loss.log_normalizers, scale, row_gradient)
        close(to_features, b.to_features, b.features_error)
        close(to_weight, b.to_weight, b.weight_error)
        assert to_features[~held].count_nonzero() == 0
        again = head.gradient(features, weight, targets, loss.log_normalizers, scale, row_gradient)
        assert torch.equal(again[0], to_features) and torch.equal(again[1], to_weight), "two runs differ"
        features[~held] = 0
    head.check()


@pytest.mark.parametrize("dtype", TYPES)
def test_gradient_over_several_chunks_of_rows(ctx, dtype):
    """More slopes than the workspace holds at once: the rows go in chunks, the weight's gradient
    is summed over them, and chunks that the missing targets leave without rows add nothing."""
    rows, labels, dim = (9000, 70_000, 24) if dtype == torch.bfloat16 else (3100, 70_000, 24)
    head = sb.LabelHead(ctx, labels, dim, dtype, rows)
    features, weight = matrix(rows, dim, dtype, 1), matrix(labels, dim, dtype, 2)
    for kind in ("all", "some", "few"):
        targets = tokens_for("all" if kind == "few" else kind, rows, labels, torch.int32, 3)
        if kind == "few":
            targets[200:] = -1
        loss = head.loss(features, weight, targets, 0.3)
        to_features, to_weight = head.gradient(features, weight, targets, loss.log_normalizers, 0.3)
        chosen = torch.arange(0, rows, max(1, rows // 100), device="cuda")  # rows of dH checked in full
        step = 1000
        want_weight = torch.zeros(labels, dim, dtype=torch.float64, device="cuda")
        weight_error = torch.zeros_like(want_weight)
        count = int((targets >= 0).logical_and(targets < labels).sum())
        for first in range(0, rows, step):
            part = slice(first, min(rows, first + step))
            g = torch.full((part.stop - first,), 1.0 / count, device="cuda")
            b = Bounds(features[part], weight, targets[part], 0.3, g)
            want_weight += b.to_weight
            weight_error += b.weight_error
            close(loss.losses[part], b.losses, b.loss_error)
            here = chosen[(chosen >= first) & (chosen < part.stop)]
            close(to_features[here], b.to_features[here - first], b.features_error[here - first])
        # The chunks' sums add f32 roundings (each at most the bound's own additions).
        close(to_weight, want_weight, weight_error * 1.1)


@pytest.mark.parametrize("dtype", TYPES)
def test_gradient_against_differences(ctx, dtype):
    """Central differences of the loss along random directions."""
    rows, labels, dim, scale = 90, 201, 40, 1.5
    head = sb.LabelHead(ctx, labels, dim, torch.float32, rows)
    typed = sb.LabelHead(ctx, labels, dim, dtype, rows)
    features, weight = matrix(rows, dim, dtype, 1, spread=0.5), matrix(labels, dim, dtype, 2, spread=0.5)
    targets = tokens_for("some", rows, labels, torch.int64, 3)
    loss = typed.loss(features, weight, targets, scale)
    to_features, to_weight = typed.gradient(features, weight, targets, loss.log_normalizers, scale)
    b = Bounds(features, weight, targets, scale)
    step = 2.0**-7
    for which, seed in ((0, 11), (1, 12)):
        base = (features, weight)[which].float()
        direction = matrix(*base.shape, torch.float32, seed)
        means = []
        for sign in (1, -1):
            moved = [features.float(), weight.float()]
            moved[which] = base + sign * step * direction
            means.append(head.loss(moved[0], moved[1], targets, scale).mean.double())
        difference = (means[0] - means[1]) / (2 * step)
        gradient = (to_features, to_weight)[which].double()
        error = (b.features_error, b.weight_error)[which]
        # The third derivative of log sum exp along z' is below 2 max|z'|^3 per row; the means' roundings.
        slope = scale * (direction @ weight.float().T if which == 0 else features.float() @ direction.T)
        third = 2 * float(slope[b.counted].abs().amax()) ** 3
        tolerance = (error * direction.abs().double()).sum() + third * step**2 / 6 + 2 * float(b.loss_error.max()) / step
        assert abs(difference - (gradient * direction.double()).sum()) <= tolerance


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,labels,dim,pad,shift", [(1, 1, 3, 0, 0), (1, 5000, 64, 0, 0), (7, 130, 33, 1, 1),
                                                       (64, 20_011, 100, 0, 0), (300, 2000, 128, 8, 0)])
def test_predict(ctx, rows, labels, dim, pad, shift, dtype):
    head = sb.LabelHead(ctx, labels, dim, dtype, rows, training=False)
    features, weight = matrix(rows, dim, dtype, 1, pad, shift), matrix(labels, dim, dtype, 2, pad, shift)
    half = labels // 2
    weight[half : 2 * half] = weight[:half].clone()  # pairs of equal label rows: the lower is the answer
    b = Bounds(features, weight, None, 0.7)
    got, log_probabilities = head.predict(features, weight, 0.7)
    best = b.z.amax(1)
    error = 2 * b.z_error + b.exp_error + 4 * A * b.normalizers.abs()
    close(log_probabilities, best - b.normalizers, error)
    picked = b.z.gather(1, got.long()[:, None])[:, 0]
    assert (best - picked <= 2 * b.z_error).all()
    assert not ((got >= half) & (got < 2 * half)).any() or labels == 1
    top = torch.topk(b.z[:, list(range(half)) + list(range(2 * half, labels))], min(2, labels - half), 1).values
    clear = top[:, 0] - top[:, -1] > 2 * b.z_error
    want = b.z.argmax(1)
    want = torch.where((want >= half) & (want < 2 * half), want - half, want)
    assert torch.equal(got[clear].long(), want[clear])


def test_large_logits_do_not_overflow(ctx):
    """Logits of thousands: the running maximum keeps the exponentials in range."""
    rows, labels, dim = 140, 300, 16
    head = sb.LabelHead(ctx, labels, dim, torch.float32, rows)
    features, weight = matrix(rows, dim, torch.float32, 1, spread=30.0), matrix(labels, dim, torch.float32, 2, spread=30.0)
    targets = tokens_for("all", rows, labels, torch.int32, 3)
    b = Bounds(features, weight, targets, 1.0)
    loss = head.loss(features, weight, targets)
    close(loss.losses, b.losses, b.loss_error)


def test_nonfinite_logits_stay_in_their_rows(ctx):
    rows, labels, dim = 200, 260, 32
    head = sb.LabelHead(ctx, labels, dim, torch.bfloat16, rows)
    features, weight = matrix(rows, dim, torch.bfloat16, 1), matrix(labels, dim, torch.bfloat16, 2)
    targets = tokens_for("all", rows, labels, torch.int32, 3)
    clean = head.loss(features, weight, targets).losses.clone()
    features[5] = float("nan")
    features[77, 3] = float("inf")
    losses = head.loss(features, weight, targets).losses
    bad = torch.zeros(rows, dtype=torch.bool, device="cuda")
    bad[5] = bad[77] = True
    assert losses[bad].isnan().all()
    assert torch.equal(losses[~bad], clean[~bad])


def test_no_rows(ctx):
    head = sb.LabelHead(ctx, 50, 16, torch.float32, 8)
    features, weight = torch.empty(0, 16, device="cuda"), matrix(50, 16, torch.float32, 2)
    targets = torch.empty(0, dtype=torch.int32, device="cuda")
    loss = head.loss(features, weight, targets)
    assert float(loss.mean) == 0 and loss.losses.numel() == 0
    to_features, to_weight = head.gradient(features, weight, targets, loss.log_normalizers)
    assert to_features.shape == (0, 16) and to_weight.count_nonzero() == 0
    assert head.predict(features, weight)[0].numel() == 0


def test_fewer_rows_than_a_call_before(ctx):
    """The workspace holds an earlier call's rows: none of them may show."""
    head = sb.LabelHead(ctx, 140, 48, torch.float32, 1000)
    weight = matrix(140, 48, torch.float32, 2)
    fresh = sb.LabelHead(ctx, 140, 48, torch.float32, 1000)
    for rows, kind in ((1000, "all"), (130, "some"), (3, "all"), (400, "some")):
        features, targets = matrix(rows, 48, torch.float32, rows), tokens_for(kind, rows, 140, torch.int32, rows)
        if rows == 1000:
            features[::2] = float("nan")
            head.loss(features, weight, targets)
            continue
        loss, other = head.loss(features, weight, targets), fresh.loss(features, weight, targets)
        assert torch.equal(loss.losses, other.losses)
        for x, y in zip(head.gradient(features, weight, targets, loss.log_normalizers),
                        fresh.gradient(features, weight, targets, loss.log_normalizers)):
            assert torch.equal(x, y)


def test_calls_from_another_stream_are_ordered(ctx):
    rows, labels, dim = 2000, 700, 64
    head = sb.LabelHead(ctx, labels, dim, torch.bfloat16, rows)
    e = sb.Embedding(ctx, labels, dim, torch.bfloat16, rows)
    weight, targets = matrix(labels, dim, torch.bfloat16, 2), tokens_for("all", rows, labels, torch.int32, 3)
    want = head.loss(e.lookup(weight, targets), weight, targets).losses.clone()
    want_gradient = e.gradient(e.lookup(weight, targets), targets).clone()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(20):
            # Made late on the side stream, read by the context's, and used on the side stream again.
            late = weight.clone()
            torch.cuda._sleep(100_000)
            late.copy_(weight)
            features = e.lookup(late, targets)
            late.zero_()
            losses = head.loss(features, weight, targets).losses * 1
            back = e.gradient(features, targets) * 1
            features.zero_()
            assert torch.equal(losses, want) and torch.equal(back, want_gradient)


def test_refusals(ctx):
    f32, i32 = torch.float32, torch.int32
    with pytest.raises(ValueError):
        sb.Embedding(ctx, 5, 8, torch.float16, 4)
    for sizes in ((0, 8, 4), (5, 0, 4), (5, 8, 0), (5, 8, 1 << 30), (1 << 31, 8, 4)):
        with pytest.raises(sb.SplatError):
            sb.Embedding(ctx, sizes[0], sizes[1], f32, sizes[2])
    for sizes in ((0, 8, 4), (5, 0, 4), (5, 8, 0), (1 << 31, 8, 4)):
        with pytest.raises(sb.SplatError):
            sb.LabelHead(ctx, sizes[0], sizes[1], f32, sizes[2])
    e, head = sb.Embedding(ctx, 5, 8, f32, 4), sb.LabelHead(ctx, 5, 8, f32, 4, training=False)
    table, rows = matrix(5, 8, f32, 1), matrix(4, 8, f32, 2)
    tokens = torch.zeros(4, dtype=i32, device="cuda")
    for call in (
        lambda: e.lookup(table.to(torch.bfloat16), tokens),
        lambda: e.lookup(table[:4], tokens),
        lambda: e.lookup(table[:, :7], tokens),
        lambda: e.lookup(table, tokens.short()),
        lambda: e.lookup(table, tokens.cpu()),
        lambda: e.lookup(table.cpu(), tokens),
        lambda: e.lookup(matrix(8, 5, f32, 1).T, tokens),
        lambda: e.lookup(table, tokens[::2]),
        lambda: e.lookup(table, tokens, out=torch.empty(3, 8, device="cuda")),
        lambda: e.gradient(rows[:3], tokens),
        lambda: head.loss(rows, table[:4], tokens),
        lambda: head.loss(rows, table, tokens[:3]),
        lambda: head.loss(rows[:, :7], table, tokens),
    ):
        with pytest.raises(ValueError):
            call()
    many = torch.zeros(5, dtype=i32, device="cuda")
    loss = head.loss(rows, table, tokens)
    for call in (
        lambda: e.lookup(table, many),
        lambda: e.gradient(torch.zeros(5, 8, device="cuda"), many),
        lambda: e.gradient(rows[:1].expand(4, 8), tokens),  # row stride 0
        lambda: head.loss(torch.zeros(5, 8, device="cuda"), table, many),
        lambda: head.loss(rows, table, tokens, 0.0),
        lambda: head.loss(rows, table, tokens, float("inf")),
        lambda: head.loss(rows, table, tokens, float("nan")),
        lambda: head.gradient(rows, table, tokens, loss.log_normalizers),  # not made for training
    ):
        with pytest.raises(sb.SplatError) as refused:
            call()
        assert "SP_ERR_INVALID" in str(refused.value)
