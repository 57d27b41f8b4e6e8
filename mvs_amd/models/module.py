"""Building blocks with the reference's names and state_dict layout
(MVSNet/models/module.py), backed by the HIP kernels of libmvs_hip.so.

`homo_warping` and `depth_regression` keep the reference signatures
(module.py:46, module.py:91); the convolution blocks are ordinary nn.Modules so
that `state_dict()` keys (`conv.weight`, `bn.running_mean`, ...) are identical
and reference checkpoints load unchanged.
"""
import torch
import torch.nn as nn
import torch.nn.functional as F

from .. import ops


class _ConvNorm(nn.Module):
    """conv (no bias) + batch-norm, optional ReLU; `conv`/`bn` child names are
    the checkpoint contract (module.py:6-43)."""
    conv_cls = nn.Conv2d
    norm_cls = nn.BatchNorm2d
    act = True

    def __init__(self, in_channels, out_channels, kernel_size=3, stride=1, pad=1):
        super().__init__()
        self.conv = self.conv_cls(in_channels, out_channels, kernel_size, stride=stride,
                                  padding=pad, bias=False)
        self.bn = self.norm_cls(out_channels)

    def forward(self, x):
        y = self.bn(self.conv(x))
        return F.relu(y, inplace=True) if self.act else y


class ConvBnReLU(_ConvNorm):
    pass


class ConvBn(_ConvNorm):
    act = False


class ConvBnReLU3D(_ConvNorm):
    conv_cls = nn.Conv3d
    norm_cls = nn.BatchNorm3d


class ConvBn3D(_ConvNorm):
    conv_cls = nn.Conv3d
    norm_cls = nn.BatchNorm3d
    act = False


def homo_warping(src_fea, src_proj, ref_proj, depth_values, align_corners=False, proj_where="host"):
    """Drop-in for module.py:46-87 (and CasMVSNet/models/module.py:245-280 when
    depth_values is [B,D,H,W]).  Returns the warped volume [B,C,D,H,W];
    differentiable w.r.t. src_fea (the grid carries no gradient, module.py:62).

    align_corners=False is what the reference's un-annotated grid_sample call
    computes on torch >= 1.3 -- the behaviour the parity gate is defined on."""
    rt = ops.rot_trans(src_proj, ref_proj, where=proj_where)
    return ops.homo_warp(src_fea, rt, depth_values, align_corners)


def depth_regression(p, depth_values):
    """module.py:91-103: expectation of depth_values under p along dim 1.
    p is already a probability volume here, so this is a plain reduction."""
    if depth_values.dim() == 2:
        depth_values = depth_values.view(*depth_values.shape, 1, 1)
    return torch.sum(p * depth_values, 1)


def matching_cells(depth, src_proj, ref_proj, mask=None):
    """The source view's feature cell that every reference cell's point falls on: depth [B,h,w] of the reference view at feature
    resolution, projection matrices [B,4,4] as in homo_warping -> int64 [B, h*w], y * w + x of the nearest cell, -1 where the point
    lies behind the camera or outside the map, where depth is not positive and where mask ([B,h,w]) is not > 0.5."""
    B, h, w = depth.shape
    rt = ops.rot_trans_all(torch.stack((ref_proj, src_proj), 1), "device")[0].view(B, 3, 4)
    y, x = torch.meshgrid(torch.arange(h, device=depth.device, dtype=torch.float32), torch.arange(w, device=depth.device, dtype=torch.float32), indexing="ij")
    ray = torch.stack((x, y, torch.ones_like(x)), -1).view(1, h * w, 3, 1)
    p = (rt[:, None, :, :3] * ray.transpose(2, 3)).sum(-1) * depth.reshape(B, h * w, 1) + rt[:, None, :, 3]
    u, v = torch.round(p[..., 0] / p[..., 2]), torch.round(p[..., 1] / p[..., 2])
    seen = (depth.reshape(B, h * w) > 0) & (p[..., 2] > 0) & (u >= 0) & (u <= w - 1) & (v >= 0) & (v <= h - 1)
    if mask is not None:
        seen = seen & (mask.reshape(B, h * w) > 0.5)
    u, v = (torch.where(seen, t, 0.0).to(torch.int64) for t in (u, v))      # (whole from here on: v * w + u may pass 2^24)
    return (v * w + u).masked_fill(~seen, -1)


def matching_sums(ref_fea, src_fea, ref_cells, src_cells, temperature=1.0):
    """feature_matching_loss as (sum over the pairs there are, their number): 0 of 0, with gradients of zero, where there is none."""
    B, C, h, w = src_fea.shape
    total = 0.0
    for b in range(B):
        rows = [f[b].permute(1, 2, 0).reshape(-1, C) for f in (ref_fea, src_fea)]
        paired = (ref_cells[b] >= 0) & (src_cells[b] >= 0)
        target = torch.where(paired, src_cells[b].masked_fill(ref_cells[b] >= rows[0].shape[0], h * w), -100)
        total = total + ops.linear_cross_entropy(ops.lookup_rows(rows[0], ref_cells[b]), rows[1], target, scale=1.0 / temperature,
                                                 reduction="sum")
    return total, ((ref_cells >= 0) & (src_cells >= 0)).sum()


def feature_matching_loss(ref_fea, src_fea, ref_cells, src_cells, temperature=1.0):
    """Cross entropy of finding a point's cell in the source view by its feature in the reference view: over the pairs (point) of
    ref_cells, src_cells [B,P] (cell numbers y * w + x; -1 on either side: no such pair; a number beyond its map: NaN), the softmax of
    <ref feature, source feature> / temperature over ALL cells of the source map, averaged over the pairs there are (NaN if there is
    none, with gradients of zero).
    ref_fea, src_fea [B,C,h,w]; differentiable in both.  The [P, h*w] scores are never stored (ops.linear_cross_entropy), several
    points may share a cell (ops.lookup_rows)."""
    total, pairs = matching_sums(ref_fea, src_fea, ref_cells, src_cells, temperature)
    return total / pairs
