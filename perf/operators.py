"""The label operators' measured cases: the embedding of codebook tokens and its gradient, and
the label head's cross entropy, gradient and prediction.

A scene's Gaussians (or an image's pixels) each carry a token of a feature codebook; the
features are classified against a vocabulary of labels given by one weight row each. The
sizes are those of this repository's scenes (20,000 and 500,000 Gaussians, images of
256 x 256 and 1024 x 768 pixels) or generic ones for feature widths and vocabularies.

`own` false computes an operator in elementary torch operations in 32 bits; true calls
`splat_b200`.
"""

import math
import os
import sys

import numpy as np
import torch

own = False

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}
TOKENS = {"int32": torch.int32, "int64": torch.int64}


def case(name, operator, rows, entries, dim, dtype, index="int32", skew=0.0, absent=0.0):
    """One case. `entries`: codebook entries or labels. `skew`: exponent of the power law that
    tokens and labels follow (0: uniform). `absent`: share of rows without a token or label."""
    made = {"operator": operator, "rows": rows, "entries": entries, "dim": dim, "dtype": dtype, "index": index,
            "skew": skew, "absent": absent}
    return {"name": name, **made} if name else made


def listed():
    return [
        # A handful of picked Gaussians' features, odd width: the latency of a call.
        case("lookup_picked", "lookup", 37, 150, 45, "float32"),
        # Every Gaussian of a 500,000-Gaussian scene takes its feature from an 8192-entry codebook.
        case("lookup_scene", "lookup", 500_000, 8192, 256, "bfloat16", skew=0.7),
        # The codebook's gradient for a small scene's 20,000 Gaussians.
        case("embedding_gradient_small", "embedding_gradient", 20_000, 1000, 64, "float32"),
        # ... for a 500,000-Gaussian scene, popular entries holding much of it.
        case("embedding_gradient_scene", "embedding_gradient", 500_000, 8192, 256, "bfloat16", skew=1.0),
        # ... for one token per pixel of a 1024 x 768 image (less one), a third of them uncovered.
        case("embedding_gradient_pixels", "embedding_gradient", 786_431, 65_521, 100, "float32", index="int64", skew=0.5,
             absent=0.33),
        # Scoring the labels of a few probe points.
        case("loss_probe", "loss", 200, 150, 45, "float32"),
        # Validation loss over a 256 x 256 image with a large label vocabulary.
        case("loss_image", "loss", 65_536, 4096, 512, "bfloat16", index="int64", absent=0.2),
        # A training step on a small batch of Gaussians and a thousand labels.
        case("train_small", "train", 256, 1000, 64, "bfloat16"),
        # A training step in 32 bits, odd vocabulary, a third of the rows unlabelled.
        case("train_masked_f32", "train", 4096, 8191, 256, "float32", skew=0.7, absent=0.33),
        # A training step of 20,000 Gaussians against an open vocabulary.
        case("train_open_vocabulary", "train", 20_000, 32_768, 512, "bfloat16", index="int64", skew=1.0),
        # Labelling one clicked point against an open vocabulary: latency and the weights' bytes.
        case("predict_one", "predict", 1, 65_536, 512, "bfloat16"),
        # Labelling a few dozen picked points in 32 bits.
        case("predict_few_f32", "predict", 60, 20_011, 768, "float32"),
    ]


def spread(rng, low, high):
    """A whole number from low to high, even over the logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    operator = rng.choice(["lookup", "embedding_gradient", "loss", "train", "predict"])
    dtype = rng.choice(["float32", "bfloat16"])
    index = rng.choice(["int32", "int64"])
    skew = rng.choice([0.0, 0.5, 0.7, 1.0])
    absent = rng.choice([0.0, 0.0, 0.2, 0.5])
    if operator in ("lookup", "embedding_gradient"):
        return case("", operator, spread(rng, 1, 786_432), spread(rng, 2, 65_536), spread(rng, 16, 256), dtype, index, skew,
                    absent)
    entries, dim = spread(rng, 20, 65_536), spread(rng, 16, 768)
    if operator == "predict":
        return case("", operator, spread(rng, 1, 64), entries, dim, dtype)
    # At most the products of the largest listed training step, in 32 bits a quarter of them.
    most = 20_000 * 32_768 * 512 // (4 if dtype == "float32" else 1)
    rows = spread(rng, 1, max(1, min(65_536, most // (entries * dim))))
    return case("", operator, rows, entries, dim, dtype, index, skew, absent)


def make_tokens(c, generator):
    """Tokens (or labels) of a power law over shuffled entries, -1 where a row has none."""
    n, v = c["rows"], c["entries"]
    if c["skew"]:
        mass = torch.arange(1, v + 1, dtype=torch.float64, device="cuda").pow(-c["skew"])
        cumulative = torch.cumsum(mass / mass.sum(), 0)
        u = torch.rand(n, generator=generator, dtype=torch.float64, device="cuda")
        ranked = torch.searchsorted(cumulative, u).clamp(max=v - 1)
        tokens = torch.randperm(v, generator=generator, device="cuda")[ranked]
    else:
        tokens = torch.randint(0, v, (n,), generator=generator, device="cuda")
    if c["absent"]:
        gone = torch.rand(n, generator=generator, device="cuda") < c["absent"]
        tokens = torch.where(gone, torch.full_like(tokens, -1), tokens)
    return tokens.to(TOKENS[c["index"]])


def make_inputs(c, seed):
    """The case's tensors, from the seed alone."""
    generator = torch.Generator(device="cuda")
    generator.manual_seed(int(seed) * 7919 + 17)
    n, v, d, dtype = c["rows"], c["entries"], c["dim"], TYPES[c["dtype"]]

    def normal(rows, columns):
        return torch.randn(rows, columns, generator=generator, device="cuda")

    if c["operator"] == "lookup":
        return {"table": normal(v, d).to(dtype), "tokens": make_tokens(c, generator), "scale": math.sqrt(d)}
    if c["operator"] == "embedding_gradient":
        return {"upstream": normal(n, d).to(dtype), "tokens": make_tokens(c, generator), "scale": math.sqrt(d)}
    # A head some way into its training: unit-norm label rows, features that lean towards their label's row, and
    # the logits' scale that spreads them over a few units.
    weight = normal(v, d)
    weight = weight / weight.norm(dim=1, keepdim=True)
    lean = make_tokens(c, generator).long()
    features = normal(n, d) / math.sqrt(d)
    features = torch.where((lean >= 0)[:, None], features + 0.7 * weight[lean.clamp(min=0)], features)
    state = {"features": features.to(dtype), "weight": weight.to(dtype), "logit_scale": 10.0}
    if c["operator"] != "predict":
        state["targets"] = lean.to(TOKENS[c["index"]])
    return state


def prepare(c, seed):
    state = {"case": c, **make_inputs(c, seed)}
    if own:
        root = os.path.join(os.getcwd(), "splatting-rs_b200")
        if root not in sys.path:
            sys.path.insert(0, root)
        import splat_b200 as sb

        state["context"] = sb.Context(0)
        dtype = TYPES[c["dtype"]]
        if c["operator"] in ("lookup", "embedding_gradient"):
            state["embedding"] = sb.Embedding(state["context"], c["entries"], c["dim"], dtype, c["rows"])
        else:
            state["head"] = sb.LabelHead(state["context"], c["entries"], c["dim"], dtype, c["rows"],
                                         training=c["operator"] == "train")
    return state


def run(state):
    return (run_own if own else run_plain)(state, state["case"]["operator"])


def run_own(s, operator):
    if operator == "lookup":
        return s["embedding"].lookup(s["table"], s["tokens"], s["scale"])
    if operator == "embedding_gradient":
        return s["embedding"].gradient(s["upstream"], s["tokens"], s["scale"])
    head, features, weight = s["head"], s["features"], s["weight"]
    if operator == "predict":
        labels, log_probabilities = head.predict(features, weight, s["logit_scale"])
        return {"labels": labels, "log_probabilities": log_probabilities}
    loss = head.loss(features, weight, s["targets"], s["logit_scale"])
    if operator == "loss":
        return {"mean": loss.mean, "losses": loss.losses}
    to_features, to_weight = head.gradient(features, weight, s["targets"], loss.log_normalizers, s["logit_scale"])
    return {"mean": loss.mean, "losses": loss.losses, "features": to_features, "weight": to_weight}


def run_plain(s, operator):
    c = s["case"]
    dtype = TYPES[c["dtype"]]
    if operator in ("lookup", "embedding_gradient"):
        tokens = s["tokens"].long()
        present = (tokens >= 0) & (tokens < c["entries"])
        at = torch.where(present, tokens, torch.zeros_like(tokens))
        if operator == "lookup":
            rows = s["table"][at].float() * s["scale"]
            return torch.where(present[:, None], rows, torch.zeros_like(rows)).to(dtype)
        rows = s["upstream"].float()
        rows = torch.where(present[:, None], rows, torch.zeros_like(rows))
        total = torch.zeros(c["entries"], c["dim"], dtype=torch.float32, device="cuda")
        total.index_add_(0, at, rows)
        return (total * s["scale"]).to(dtype)
    features, weight = s["features"].float(), s["weight"].float()
    logits = (features @ weight.T) * s["logit_scale"]
    largest = logits.amax(1)
    weights = torch.exp(logits - largest[:, None])
    sums = weights.sum(1)
    if operator == "predict":
        columns = torch.arange(c["entries"], device="cuda")
        first = torch.where(logits == largest[:, None], columns, c["entries"]).amin(1)
        return {"labels": first.int(), "log_probabilities": -torch.log(sums)}
    targets = s["targets"].long()
    counted = (targets >= 0) & (targets < c["entries"])
    at = torch.where(counted, targets, torch.zeros_like(targets))
    picked = logits.gather(1, at[:, None])[:, 0]
    losses = torch.where(counted, torch.log(sums) + largest - picked, torch.zeros_like(sums))
    count = counted.sum().clamp(min=1)
    mean = losses.sum() / count
    if operator == "loss":
        return {"mean": mean, "losses": losses}
    per_row = torch.where(counted, s["logit_scale"] / count.float(), torch.zeros_like(sums))
    weights = weights / sums[:, None]
    weights[torch.arange(c["rows"], device="cuda"), at] -= 1.0
    weights = weights * per_row[:, None]
    return {"mean": mean, "losses": losses, "features": (weights @ weight).to(dtype),
            "weight": (weights.T @ features).to(dtype)}


def work(c):
    """Each input read once, each output written once, and the products of the definition; for a training step the
    logits' product twice, since they are not kept."""
    n, v, d = c["rows"], c["entries"], c["dim"]
    size = 4 if c["dtype"] == "float32" else 2
    token = 4 if c["index"] == "int32" else 8
    present = n * (1.0 - c["absent"])
    if c["operator"] == "lookup":
        return {"bytes": token * n + size * d * (min(v, n) + n), "flops": present * d}
    if c["operator"] == "embedding_gradient":
        return {"bytes": token * n + size * d * (present + v), "flops": present * d}
    if c["operator"] == "predict":
        return {"bytes": size * d * (n + v) + 8 * n, "flops": 2.0 * n * v * d}
    rows = present
    if c["operator"] == "loss":
        return {"bytes": token * n + size * d * (rows + v) + 4 * n, "flops": 2.0 * rows * v * d}
    return {"bytes": token * n + size * d * (2 * (rows + v) + n - rows) + 4 * n, "flops": 8.0 * rows * v * d}


def exact(c, seed):
    """The definitions in 64 bits, rows in blocks."""
    s = make_inputs(c, seed)
    operator, n, v = c["operator"], c["rows"], c["entries"]
    if operator == "lookup":
        found = np.zeros((n, c["dim"]))
        tokens = s["tokens"].cpu().numpy().astype(np.int64)
        held = (tokens >= 0) & (tokens < v)
        found[held] = s["table"].double().cpu().numpy()[tokens[held]] * s["scale"]
        return torch.from_numpy(found)
    if operator == "embedding_gradient":
        # Sorted by token, then differences of running sums would cancel: sums of each run instead.
        order = torch.argsort(s["tokens"].long(), stable=True)
        sorted_tokens = s["tokens"].long()[order]
        order = order[(sorted_tokens >= 0) & (sorted_tokens < v)]
        lengths = torch.bincount(s["tokens"].long()[order], minlength=v)
        rows = s["upstream"].double()[order]
        if rows.shape[0] == 0:
            return torch.zeros(v, c["dim"], dtype=torch.float64)
        return torch.segment_reduce(rows, "sum", lengths=lengths, initial=0.0) * s["scale"]
    weight = s["weight"].double()
    labels, losses, logs, to_features = [], [], [], []
    to_weight = torch.zeros_like(weight)
    targets = s["targets"].long() if operator != "predict" else None
    count = max(1, int(((targets >= 0) & (targets < v)).sum())) if targets is not None else 0
    block = max(1, min(n, (1 << 27) // v))
    for begin in range(0, n, block):
        features = s["features"][begin:begin + block].double()
        logits = s["logit_scale"] * torch.einsum("nd,vd->nv", features, weight)
        normalizers = torch.logsumexp(logits, 1)
        if operator == "predict":
            best, which = logits.max(1)
            labels.append(which.int())
            logs.append(best - normalizers)
            continue
        target = targets[begin:begin + block]
        counted = (target >= 0) & (target < v)
        rows = torch.nonzero(counted)[:, 0]
        loss = torch.zeros_like(normalizers)
        loss[rows] = normalizers[rows] - logits[rows, target[rows]]
        losses.append(loss)
        if operator == "train":
            slope = torch.exp(logits[rows] - normalizers[rows, None])
            slope[torch.arange(len(rows), device="cuda"), target[rows]] -= 1.0
            slope *= s["logit_scale"] / count
            back = torch.zeros_like(features)
            back[rows] = slope @ weight
            to_features.append(back)
            to_weight += slope.T @ features[rows]
    if operator == "predict":
        return {"labels": torch.cat(labels), "log_probabilities": torch.cat(logs)}
    losses = torch.cat(losses)
    found = {"mean": losses.sum() / count, "losses": losses}
    if operator == "train":
        found |= {"features": torch.cat(to_features), "weight": to_weight}
    return found
