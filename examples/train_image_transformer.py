"""Trains a small image transformer on batches of the loader, with the operators of ``ffcv_b200.training``:

    python examples/train_image_transformer.py                       # on synthetic images, a minute on one GPU
    python examples/train_image_transformer.py --data train.beton --classes 1000 --width 384 --layers 12

The loader decodes, crops, flips and mixes the images on the GPU and hands the mixed labels over as [label, partner's
label, lambda] rows, which the loss reads as they are.  The resolution grows from epoch to epoch; patches have rotary
positions by row and column, which do not depend on it.  Every residual join is one kernel with the norm before the
next block; AdamW keeps 32-bit masters of the bfloat16 weights and moments in 8 bits.
"""
import argparse
import json
import os
import sys
import tempfile

import numpy as np
import torch
from torch import nn
from torch.nn import functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

MEAN = np.array([0.485, 0.456, 0.406]) * 255
STD = np.array([0.229, 0.224, 0.225]) * 255


class Colours:
    """Noise around a colour of the class's own: a set that a small network learns in a minute."""

    def __init__(self, count, classes):
        self.count, self.classes = count, classes

    def __len__(self):
        return self.count

    def __getitem__(self, k):
        rng = np.random.default_rng(k)
        label = k % self.classes
        colour = np.random.default_rng([7, label]).integers(60, 196, 3)
        h, w = rng.integers(100, 180, 2)
        return np.clip(rng.normal(colour, 30, (h, w, 3)), 0, 255).astype(np.uint8), label


def write(path, count, classes):
    from ffcv_b200 import DatasetWriter
    from ffcv_b200.fields import IntField, RGBImageField
    DatasetWriter(path, {'image': RGBImageField(write_mode='jpg', jpeg_quality=90), 'label': IntField()},
                  num_workers=1).from_indexed_dataset(Colours(count, classes))


def loader_of(path, batch, side, mixup, seed):
    from ffcv_b200 import Loader, OrderOption
    from ffcv_b200.fields.decoders import IntDecoder, RandomResizedCropRGBImageDecoder
    from ffcv_b200.transforms import (ImageMixup, LabelMixup, NormalizeImage, RandomHorizontalFlip, ToDevice, ToTensor,
                                      ToTorchImage)
    device = torch.device('cuda', torch.cuda.current_device())
    image = [RandomResizedCropRGBImageDecoder((side, side)), RandomHorizontalFlip(), ImageMixup(mixup, False), ToTensor(),
             ToDevice(device), ToTorchImage(), NormalizeImage(MEAN, STD, np.float16)]
    label = [IntDecoder(), LabelMixup(mixup, False), ToTensor(), ToDevice(device)]
    return Loader(path, batch_size=batch, order=OrderOption.RANDOM, seed=seed, pipelines={'image': image, 'label': label})


class Block(nn.Module):
    """Attention and a perceptron.  Each is given the normed stream and followed by the join with the stream and the
    norm of what comes next."""

    def __init__(self, width, heads, rotary):
        from ffcv_b200.training import NormResidual
        super().__init__()
        self.heads, self.rotary = heads, rotary
        self.qkv, self.out = nn.Linear(width, 3 * width), nn.Linear(width, width)
        self.up, self.down = nn.Linear(width, 4 * width), nn.Linear(4 * width, width)
        self.join_attention, self.join_perceptron = NormResidual(width, scale=0.1), NormResidual(width, scale=0.1)

    def forward(self, stream, normed, positions):
        batch, tokens, width = stream.shape
        qkv = self.qkv(normed).view(batch, tokens, 3 * self.heads, width // self.heads)
        q, k = self.rotary(qkv[:, :, :self.heads], qkv[:, :, self.heads:2 * self.heads], positions)
        mixed = F.scaled_dot_product_attention(q.transpose(1, 2), k.transpose(1, 2), qkv[:, :, 2 * self.heads:].transpose(1, 2))
        stream, normed = self.join_attention(stream, self.out(mixed.transpose(1, 2).reshape(batch, tokens, width)))
        return self.join_perceptron(stream, self.down(F.gelu(self.up(normed))))


class ImageTransformer(nn.Module):
    def __init__(self, classes, patch, width, layers, heads):
        from ffcv_b200.training import NormResidual, RotaryPositions
        super().__init__()
        self.patch, self.embed = patch, nn.Linear(3 * patch * patch, width)
        self.first = NormResidual(width)
        rotary = RotaryPositions(width // heads, axes=2)
        self.blocks = nn.ModuleList([Block(width, heads, rotary) for _ in range(layers)])
        self.head = nn.Linear(width, classes)

    def forward(self, images):
        from ffcv_b200.training import patch_positions
        batch, channels, height, width = images.shape
        rows, cols = height // self.patch, width // self.patch
        patches = images.reshape(batch, channels, rows, self.patch, cols, self.patch).permute(0, 2, 4, 1, 3, 5)
        stream, normed = self.first(self.embed(patches.reshape(batch, rows * cols, -1)))
        positions = patch_positions(rows, cols, images.device)
        for block in self.blocks:
            stream, normed = block(stream, normed, positions)
        return self.head(normed.mean(1))


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument('--data', help='a .beton with fields image and label; default: synthetic images')
    ap.add_argument('--classes', type=int, default=10)
    ap.add_argument('--count', type=int, default=2048, help='synthetic images')
    ap.add_argument('--batch', type=int, default=128)
    ap.add_argument('--epochs', type=int, default=6)
    ap.add_argument('--sides', type=int, nargs=2, default=(64, 112), help="images' side in the first and the last epoch")
    ap.add_argument('--patch', type=int, default=16)
    ap.add_argument('--width', type=int, default=192)
    ap.add_argument('--layers', type=int, default=4)
    ap.add_argument('--heads', type=int, default=3)
    ap.add_argument('--lr', type=float, default=1e-3)
    ap.add_argument('--mixup', type=float, default=0.2)
    ap.add_argument('--state-bits', type=int, default=8, choices=(8, 32))
    a = ap.parse_args()

    own = None
    if a.data is None:  # (before the process touches the GPU: the writer forks)
        own = tempfile.TemporaryDirectory(dir='/dev/shm' if os.path.isdir('/dev/shm') else None)
        a.data = os.path.join(own.name, 'colours.beton')
        write(a.data, a.count, a.classes)

    from ffcv_b200.training import AdamW, MixupCrossEntropy
    torch.manual_seed(0)
    model = ImageTransformer(a.classes, a.patch, a.width, a.layers, a.heads).cuda().bfloat16()
    matrices = [p for p in model.parameters() if p.dim() > 1]
    vectors = [p for p in model.parameters() if p.dim() <= 1]
    opt = AdamW([dict(params=matrices), dict(params=vectors, weight_decay=0.0)], lr=a.lr, weight_decay=0.05,
                state_bits=a.state_bits, max_grad_norm=1.0)
    loss_of = MixupCrossEntropy(label_smoothing=0.1)
    means = []
    for epoch in range(a.epochs):
        share = epoch / max(1, a.epochs - 1)
        side = int(round((a.sides[0] + share * (a.sides[1] - a.sides[0])) / a.patch)) * a.patch
        losses = []
        for images, labels in loader_of(a.data, a.batch, side, a.mixup, epoch):
            loss = loss_of(model(images.bfloat16()), labels)
            opt.zero_grad()
            loss.backward()
            opt.step()
            losses.append(loss.detach())
        means.append(float(torch.stack(losses).mean()))
        print(f'epoch {epoch}: {len(losses)} steps of {a.batch} images of {side} x {side}, loss {means[-1]:.3f}, '
              f'gradient norm {float(opt.grad_norm):.3f}', flush=True)
    print(json.dumps({'losses': means}))
    if own is not None:
        own.cleanup()


if __name__ == '__main__':
    main()
