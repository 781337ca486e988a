"""Labels for a scene's Gaussians: a feature codebook and a label head trained together.

Every Gaussian carries a token of a feature codebook. Views of the scene have a label per pixel
(here a checkerboard of the scene's regions, as a segmentation of photographs would give); a view
labels the Gaussians that are visible in it by the pixel under their projected centre, and the others
carry no target in that step. One step:

    features  = embedding.lookup(codebook, tokens)             one row per Gaussian
    loss      = head.loss(features, weight, targets)           over the label vocabulary
    gradients = head.gradient(...)                             of features and label weights
    codebook gradient = embedding.gradient(features' gradient, tokens)

    python examples/label_scene.py [--steps 60] [--dtype bfloat16]
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import numpy as np
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "splatting-rs_b200"))

import splat_b200 as sb  # noqa: E402
from splat_b200 import scenes  # noqa: E402


def region_of(positions: np.ndarray, labels: int) -> np.ndarray:
    """The region each point of the scene lies in, one of `labels`: cells of a grid, numbered."""
    side = max(1, int(np.ceil(labels ** (1 / 3))))
    cell = np.clip(((positions + 1.0) * 0.5 * side).astype(np.int64), 0, side - 1)
    return (cell[:, 0] * side * side + cell[:, 1] * side + cell[:, 2]) % labels


def visible_targets(rast: sb.Rasterizer, camera: sb.PinholeCamera, label_image: np.ndarray) -> torch.Tensor:
    """Per Gaussian the label of the pixel under its projected centre, -1 where it is not in view."""
    rast.set_camera(camera)
    rast.encode_forward()
    projected = rast.read_projected()
    x, y = np.floor(projected["mean"][:, 0]).astype(np.int64), np.floor(projected["mean"][:, 1]).astype(np.int64)
    seen = (projected["radius"] > 0) & (x >= 0) & (x < camera.width) & (y >= 0) & (y < camera.height)
    targets = np.full(len(projected), -1, np.int64)
    targets[seen] = label_image[y[seen], x[seen]]
    return torch.from_numpy(targets).cuda()


def label_image_of(rast: sb.Rasterizer, camera: sb.PinholeCamera, regions: np.ndarray) -> np.ndarray:
    """The camera's label image: at each Gaussian's projected centre its region, nearest last; -1 elsewhere."""
    rast.set_camera(camera)
    rast.encode_forward()
    projected = rast.read_projected()
    image = np.full((camera.height, camera.width), -1, np.int64)
    for i in np.argsort(-projected["depth"], kind="stable"):
        x, y = int(projected["mean"][i, 0]), int(projected["mean"][i, 1])
        if projected["radius"][i] > 0 and 0 <= x < camera.width and 0 <= y < camera.height:
            image[y, x] = regions[i]
    return image


def train(steps: int = 60, dtype: torch.dtype = torch.bfloat16, scale: float = 0.2, labels: int = 100, dim: int = 64,
          rate: float = 0.05) -> dict[str, float]:
    """Trains the codebook and the label weights; the first and last losses and the final accuracy."""
    scene = scenes.config(0, scale=scale)
    cloud, n = scene.cloud, len(scene.cloud)
    ctx = sb.Context(0)
    params = torch.from_numpy(cloud.to_packed()).cuda()
    first = scene.cameras[0]
    ground_truth = torch.zeros(first.width * first.height * 4, device="cuda")
    rast = sb.Rasterizer(ctx, params, n, first.width, first.height, ground_truth, 1)
    positions = np.asarray(cloud.positions, np.float64)
    regions = region_of(positions, labels)
    images = [label_image_of(rast, camera, regions) for camera in scene.cameras]

    # Tokens: finer cells than the regions, so that a token's Gaussians share a label as a rule.
    entries = 4 * labels
    tokens = torch.from_numpy(region_of(positions, entries).astype(np.int32)).cuda()
    generator = torch.Generator(device="cuda").manual_seed(0)
    master = [0.1 * torch.randn(rows, dim, generator=generator, device="cuda") for rows in (entries, labels)]
    adam = torch.optim.Adam([p.requires_grad_() for p in master], lr=rate)
    embedding = sb.Embedding(ctx, entries, dim, dtype, n)
    head = sb.LabelHead(ctx, labels, dim, dtype, n)

    losses = []
    targets = [visible_targets(rast, camera, image) for camera, image in zip(scene.cameras, images)]
    for step in range(steps):
        target = targets[step % len(targets)]
        codebook, weight = (p.detach().to(dtype) for p in master)
        features = embedding.lookup(codebook, tokens)
        loss = head.loss(features, weight, target)
        to_features, to_weight = head.gradient(features, weight, target, loss.log_normalizers)
        master[0].grad = embedding.gradient(to_features, tokens).float()
        master[1].grad = to_weight.float()
        adam.step()
        losses.append(loss.mean)
    codebook, weight = (p.detach().to(dtype) for p in master)
    predicted, _ = head.predict(embedding.lookup(codebook, tokens), weight)
    embedding.check()
    head.check()
    wanted = torch.from_numpy(regions).cuda()
    seen = torch.stack([t >= 0 for t in targets]).any(0)
    return {"first_loss": float(losses[0]), "last_loss": float(losses[-1]),
            "accuracy": float((predicted.long() == wanted)[seen].float().mean())}


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--steps", type=int, default=60)
    parser.add_argument("--dtype", choices=("float32", "bfloat16"), default="bfloat16")
    args = parser.parse_args()
    result = train(args.steps, getattr(torch, args.dtype))
    print(f"loss {result['first_loss']:.3f} -> {result['last_loss']:.3f}, "
          f"{100 * result['accuracy']:.1f} % of the seen Gaussians labelled with their region")


if __name__ == "__main__":
    main()
