"""ResNet-50 (bottleneck v1.5) written out in torch.nn, for the data-parallel
benchmark: 161 trainable tensors, 25,557,032 parameters.  torchvision is not
needed.

`norm="group"` takes group normalisation (32 groups) in the place of batch normalisation: the
same tensors and parameters, but no statistics of a rank's own batch, so that a step does not
depend on how the batch is split over the ranks.  On CUDA tensors the normalisation, the
activation and the shortcut are one operator of this package (ops.group_norm)."""
import torch
from torch import nn
from torch.nn import functional as F

from ..ops import group_norm


class GroupNormAct(nn.Module):
    """Group normalisation with what follows it: the shortcut, if one is given, and the activation."""

    def __init__(self, channels, activation="relu", groups=32, eps=1e-5):
        super().__init__()
        self.groups, self.eps, self.activation = groups, eps, activation
        self.weight = nn.Parameter(torch.ones(channels))
        self.bias = nn.Parameter(torch.zeros(channels))

    def forward(self, x, residual=None):
        if x.is_cuda:
            return group_norm(x, self.groups, self.weight, self.bias, eps=self.eps,
                              activation=self.activation, residual=residual)
        y = F.group_norm(x, self.groups, self.weight, self.bias, self.eps)
        y = y if residual is None else y + residual
        return y if self.activation is None else getattr(F, self.activation)(y)


class GroupNormBottleneck(nn.Module):
    def __init__(self, inplanes, planes, stride, downsample):
        super().__init__()
        self.conv1 = nn.Conv2d(inplanes, planes, 1, bias=False)
        self.norm1 = GroupNormAct(planes)
        self.conv2 = nn.Conv2d(planes, planes, 3, stride=stride, padding=1, bias=False)
        self.norm2 = GroupNormAct(planes)
        self.conv3 = nn.Conv2d(planes, planes * 4, 1, bias=False)
        self.norm3 = GroupNormAct(planes * 4)
        self.downsample = downsample

    def forward(self, x):
        idt = x if self.downsample is None else self.downsample(x)
        y = self.norm2(self.conv2(self.norm1(self.conv1(x))))
        return self.norm3(self.conv3(y), residual=idt)


class Bottleneck(nn.Module):
    def __init__(self, inplanes, planes, stride, downsample):
        super().__init__()
        self.conv1 = nn.Conv2d(inplanes, planes, 1, bias=False)
        self.bn1 = nn.BatchNorm2d(planes)
        self.conv2 = nn.Conv2d(planes, planes, 3, stride=stride, padding=1, bias=False)
        self.bn2 = nn.BatchNorm2d(planes)
        self.conv3 = nn.Conv2d(planes, planes * 4, 1, bias=False)
        self.bn3 = nn.BatchNorm2d(planes * 4)
        self.relu = nn.ReLU(inplace=True)
        self.downsample = downsample

    def forward(self, x):
        idt = x if self.downsample is None else self.downsample(x)
        y = self.relu(self.bn1(self.conv1(x)))
        y = self.relu(self.bn2(self.conv2(y)))
        y = self.bn3(self.conv3(y))
        return self.relu(y + idt)


class ResNet50(nn.Module):
    def __init__(self, num_classes=1000, norm="batch"):
        super().__init__()
        if norm not in ("batch", "group"):
            raise ValueError(f"unknown norm {norm!r}")
        group = norm == "group"
        self.conv1 = nn.Conv2d(3, 64, 7, stride=2, padding=3, bias=False)
        self.bn1 = GroupNormAct(64) if group else nn.BatchNorm2d(64)
        self.relu = nn.Identity() if group else nn.ReLU(inplace=True)
        self.maxpool = nn.MaxPool2d(3, stride=2, padding=1)
        layers, inplanes = [], 64
        for planes, blocks, stride in ((64, 3, 1), (128, 4, 2), (256, 6, 2), (512, 3, 2)):
            for b in range(blocks):
                s = stride if b == 0 else 1
                down = None
                if b == 0:
                    down = nn.Sequential(nn.Conv2d(inplanes, planes * 4, 1, stride=s, bias=False),
                                         GroupNormAct(planes * 4, None) if group
                                         else nn.BatchNorm2d(planes * 4))
                layers.append((GroupNormBottleneck if group else Bottleneck)(inplanes, planes, s, down))
                inplanes = planes * 4
        self.layers = nn.Sequential(*layers)
        self.avgpool = nn.AdaptiveAvgPool2d(1)
        self.fc = nn.Linear(2048, num_classes)

    def forward(self, x):
        x = self.maxpool(self.relu(self.bn1(self.conv1(x))))
        x = self.layers(x)
        return self.fc(torch.flatten(self.avgpool(x), 1))
