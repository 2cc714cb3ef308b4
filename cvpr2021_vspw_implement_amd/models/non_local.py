"""Non-local block (modes 'dot' and 'differential') on the HIP kernels, mirroring reference models/non_local.py:7-151.

y = (theta^T phi / N) g is evaluated by ONE fused kernel (csrc/nonlocal.hip, ops.non_local_dot) over the [B, N, C]
pixel-row matrices that NHWC memory provides for free (N = H*W, or T*H*W for the spatio-temporal block): 32-key tiles of
phi / g stream through LDS, the affinity tile lives in MFMA accumulators and feeds the second product directly, so the
N x N affinity (2.5 GB per sample at T = 7) never exists in memory - forward or backward.

Mode 'differential' (no reference counterpart: the reference's block has no softmax here) replaces the affinity by the
difference of two softmax maps per head with a learned weight (csrc/diff_attn.hip, ops.diff_attention), normalises every
head (csrc/group_norm.hip) and drops features (csrc/dropout.hip) before the same W_z and residual:
    theta, phi -> two queries / keys of width D per head, g -> values of width 2 D;   Ci = heads * 2 D
    y = Dropout(GroupNorm_heads((softmax(q1 k1^T / sqrt(D)) - lam softmax(q2 k2^T / sqrt(D))) v));   z = x + BN(W_z y)
    lam = exp(lq1.lk1) - exp(lq2.lk2) + lambda_init;   GroupNorm's weights start at 1 - lambda_init
"""
import torch
import torch.nn as nn

from .. import nn as vnn
from .. import ops


class NLBlockND(nn.Module):
    def __init__(self, in_channels, inter_channels=None, mode="embedded", dimension=3, bn_layer=True, heads=2, dropout=0.0,
                 lambda_init=0.8, frame_causal=False):
        """heads, dropout, lambda_init, frame_causal: mode 'differential' only; frame_causal (dimension 3): positions of a frame
        see their own and earlier frames."""
        super().__init__()
        assert dimension in [1, 2, 3]
        if mode not in ["gaussian", "embedded", "dot", "concatenate", "differential"]:
            raise ValueError("`mode` must be one of `gaussian`, `embedded`, `dot`, `concatenate` or `differential`")
        if mode not in ("dot", "differential"):
            raise NotImplementedError("only mode='dot' (the one the VSPW heads use) and 'differential' are on the HIP path")
        if not bn_layer or dimension == 1:
            raise NotImplementedError("only the bn_layer=True, 2-D / 3-D block of the VSPW heads is on the HIP path")
        self.mode = mode
        self.dimension = dimension
        self.in_channels = in_channels
        self.inter_channels = inter_channels
        if self.inter_channels is None:
            self.inter_channels = max(in_channels // 2, 1)
        if dimension == 3:
            conv_nd = lambda cin, cout: vnn.Conv3d1x1(in_channels=cin, out_channels=cout, kernel_size=1)  # noqa: E731
        else:
            conv_nd = lambda cin, cout: vnn.Conv2d(in_channels=cin, out_channels=cout, kernel_size=1)  # noqa: E731
        # the reference instantiates SynchronizedBatchNorm3d for both the 2-D and the 3-D block (non_local.py:42-46)
        bn = vnn.SynchronizedBatchNorm3d
        self.g = conv_nd(self.in_channels, self.inter_channels)
        self.W_z = nn.Sequential(conv_nd(self.inter_channels, self.in_channels), bn(self.in_channels))
        nn.init.constant_(self.W_z[1].weight, 0)
        nn.init.constant_(self.W_z[1].bias, 0)
        self.theta = conv_nd(self.in_channels, self.inter_channels)
        self.phi = conv_nd(self.in_channels, self.inter_channels)
        if mode == "differential":
            d, rest = divmod(self.inter_channels, 2 * heads)
            if rest or not ops.diff_attention_supported(d):
                raise ValueError("%d inner channels do not divide into %d heads of two maps of width 16, 32 or 64"
                                 % (self.inter_channels, heads))
            if frame_causal and dimension != 3:
                raise ValueError("frame_causal needs the spatio-temporal block (dimension=3)")
            self.heads, self.lambda_init, self.frame_causal = heads, float(lambda_init), bool(frame_causal)
            for name in ("lambda_q1", "lambda_k1", "lambda_q2", "lambda_k2"):
                self.register_parameter(name, nn.Parameter(0.1 * torch.randn(heads, d)))
            self.norm = vnn.GroupNorm(heads, self.inter_channels)
            nn.init.constant_(self.norm.weight, 1.0 - self.lambda_init)
            self.drop = vnn.Dropout(dropout)

    def _differential(self, th, ph, g, shape, n_pos):
        b, h = shape[0], self.heads
        lam = ops.diff_lambda(self.lambda_q1, self.lambda_k1, self.lambda_q2, self.lambda_k2, self.lambda_init)
        frame = n_pos // shape[2] if self.frame_causal else 0
        y = ops.diff_attention(th.view(b, n_pos, h, 2, -1), ph.view(b, n_pos, h, 2, -1), g.view(b, n_pos, h, -1), lam, frame=frame)
        return self.norm(ops.from_pixels(y.view(b, n_pos, self.inter_channels), n_pos, 1), "none", self.drop)

    @staticmethod
    def _w2d(conv):
        return conv.weight.reshape(conv.out_channels, conv.in_channels, 1, 1)

    def forward(self, x):
        shape = x.shape
        b, c = shape[0], shape[1]
        n_pos = 1
        for s in shape[2:]:
            n_pos *= s
        xr = ops.as_nhwc(x.reshape(b, c, n_pos, 1))  # [B,C,N,1]: rows = positions
        g = ops.pixels_view(ops.conv2d(xr, self._w2d(self.g), self.g.bias))  # [B,N,Ci]
        th = ops.pixels_view(ops.conv2d(xr, self._w2d(self.theta), self.theta.bias))
        ph = ops.pixels_view(ops.conv2d(xr, self._w2d(self.phi), self.phi.bias))
        if self.mode == "differential":
            y = self._differential(th, ph, g, shape, n_pos)
        elif ops.nl_dot_supported(self.inter_channels):
            # fused: theta phi^T is streamed through registers, never written (csrc/nonlocal.hip); f / N happens on the
            # affinity tile, where the reference applies it
            y = ops.from_pixels(ops.non_local_dot(th, ph, g, 1.0 / n_pos), n_pos, 1)  # [B,Ci,N,1]
        else:  # other channel counts: two dense GEMMs over a materialised [B,N,N] affinity
            f = ops.bmm_nt(th, ph)  # [B,N,N]
            gT = ops.transpose_last2(ops.scale(g, 1.0 / n_pos))  # [B,Ci,N]
            y = ops.from_pixels(ops.bmm_nt(f, gT), n_pos, 1)  # [B,Ci,N,1]
        wz, bnz = self.W_z[0], self.W_z[1]
        z = ops.conv_bn_act(y, self._w2d(wz), wz.bias, bnz.weight, bnz.bias, bnz.running_mean, bnz.running_var,
                            residual=xr, mask=None, stride=1, pad=0, dil=1, training=bnz.training,
                            momentum=bnz.momentum, eps=bnz.eps, relu=False)
        return z.reshape(shape)
