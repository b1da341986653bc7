"""Training a small voxel network for semantic segmentation with the operators around its convolutions: group norm per scene
with its activation (``SegmentedGroupNorm``), a head that gives the loss without its logits (``LinearCrossEntropy``) and
``AdamW`` in one launch, moments in 32 or 8 bits.

    python -m warpconvnet_b200.examples.train_segmentation --scenes 4 --voxels 60000 --classes 200 --state-bits 8

Scenes are synthetic rooms; a voxel's class is the cell of a coarse grid that it lies in, which its features (noisy coordinates)
tell.  Prints one JSON line: the loss at the first and the last steps and milliseconds per step (CUDA events).
"""
from __future__ import annotations

import argparse
import json
from typing import List, Tuple

import numpy as np
import torch
import torch.nn as nn
from torch import Tensor

from .. import LinearCrossEntropy, SegmentedGroupNorm, Sequential, SparseConv3d, Voxels, cat
from .._native import check_device_status
from ..datasets import synthetic
from ..optim import AdamW


def _norm(channels: int) -> SegmentedGroupNorm:
    return SegmentedGroupNorm(8, channels, activation="silu")


class SegmentationNet(nn.Module):
    """Two levels of a U-Net; ``forward`` gives the loss of a batch, :meth:`features` what the head is applied to."""

    def __init__(self, in_channels: int, num_classes: int, width: int = 32):
        super().__init__()
        self.stem = Sequential(SparseConv3d(in_channels, width, 3, bias=False), _norm(width))
        self.down = Sequential(SparseConv3d(width, 2 * width, 2, stride=2, bias=False), _norm(2 * width),
                               SparseConv3d(2 * width, 2 * width, 3, bias=False), _norm(2 * width))
        self.up = SparseConv3d(2 * width, width, 2, stride=2, transposed=True, bias=False)
        self.mix = Sequential(SparseConv3d(2 * width, 2 * width, 3, bias=False), _norm(2 * width))
        self.head = LinearCrossEntropy(2 * width, num_classes)

    def features(self, x: Voxels) -> Voxels:
        fine = self.stem(x)
        return self.mix(cat(self.up(self.down(fine), fine), fine))

    def forward(self, x: Voxels, labels: Tensor) -> Tensor:
        return self.head(self.features(x), labels)


def make_batch(scenes: int, voxels: int, classes: int, seed: int, device) -> Tuple[Voxels, Tensor]:
    """Rooms in Morton order, and their voxels' classes (some unlabelled)."""
    rng = np.random.default_rng(seed)
    rooms = [synthetic.room_scene(voxels, 0.05 if voxels <= 40000 else 0.02, seed + i, "raster_crop") for i in range(scenes)]
    xyz = np.concatenate(rooms).astype(np.int32)
    offsets = np.concatenate([[0], np.cumsum([len(r) for r in rooms])])
    place = np.concatenate([(r - r.min(0)) / (np.ptp(r, axis=0) + 1) for r in rooms])
    side = int(np.ceil(classes ** (1 / 3)))
    cell = (place * side).astype(np.int64)
    labels = ((cell[:, 0] * side + cell[:, 1]) * side + cell[:, 2]) % classes
    labels[rng.random(len(labels)) < 0.05] = -100
    feats = np.concatenate([place * 4 - 2, rng.normal(size=(len(place), 1))], 1) + 0.1 * rng.normal(size=(len(place), 4))
    vox = Voxels(torch.from_numpy(xyz).to(device), torch.from_numpy(feats).float().to(device), offsets=torch.from_numpy(offsets)).sort()
    return vox, torch.from_numpy(labels).to(device)[vox.extra_attributes["perm"]]


def train(scenes: int = 2, voxels: int = 20000, classes: int = 40, steps: int = 30, state_bits: int = 32, dtype=torch.bfloat16,
          lr: float = 4e-3, seed: int = 0, device="cuda:0") -> Tuple[List[float], float]:
    """(loss of every step, milliseconds per step after the first five)"""
    torch.manual_seed(seed)
    net = SegmentationNet(4, classes).to(device)
    opt = AdamW(net.parameters(), lr=lr, state_bits=state_bits)
    scaler = torch.amp.GradScaler("cuda", enabled=dtype == torch.float16)
    batches = [make_batch(scenes, voxels, classes, seed + 100 * i, device) for i in range(2)]
    losses, began, ended = [], torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    for i in range(steps):
        if i == 5:
            began.record()
        vox, labels = batches[i % len(batches)]
        opt.zero_grad()
        with torch.autocast("cuda", dtype=dtype, enabled=dtype != torch.float32):
            loss = net(vox, labels)
        scaler.scale(loss).backward()
        scaler.step(opt)
        scaler.update()
        losses.append(loss.detach())
    ended.record()
    check_device_status(device)
    return torch.stack(losses).tolist(), began.elapsed_time(ended) / max(1, steps - 5)


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--scenes", type=int, default=4)
    ap.add_argument("--voxels", type=int, default=60000)
    ap.add_argument("--classes", type=int, default=200)
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--state-bits", type=int, default=32, choices=(8, 32))
    ap.add_argument("--dtype", default="bf16", choices=("fp32", "fp16", "bf16"))
    a = ap.parse_args()
    dtype = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}[a.dtype]
    losses, ms = train(a.scenes, a.voxels, a.classes, a.steps, a.state_bits, dtype)
    print(json.dumps({"scenes": a.scenes, "voxels_per_scene": a.voxels, "classes": a.classes, "state_bits": a.state_bits, "dtype": a.dtype,
                      "first_loss": round(losses[0], 4), "last_loss": round(losses[-1], 4), "ms_per_step": round(ms, 3)}))


if __name__ == "__main__":
    main()
