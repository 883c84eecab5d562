"""Multi-head self-attention over the positions of a map, with positions: query / key norm + rotation by row and column, a learned bias by
buckets of the row and column distance, dropout in front of the residual (ops_tokens).  The second entry of ATTENTION_TYPES beside the
SAGAN block (which has one head and no notion of position); takes and returns a map like that one."""
import torch
from torch import nn

from ... import ops, ops_tokens
from ..layers import HipConv2d, HipDropout


def _head_size(channels):
    """The largest even head size up to 64 that divides `channels`."""
    for d in range(min(64, channels), 1, -1):
        if channels % d == 0 and d % 2 == 0:
            return d
    raise ValueError(f"RelativeAttention needs an even number of channels (got {channels})")


class RelativeAttention(nn.Module):
    """x + dropout(proj(attention(q', k', v))), q' and k' normed and rotated per head.  num_buckets: of one axis (the table has its square
    per head); distances from max_distance on share the last bucket.  dropout, stream:
    see HipDropout."""

    def __init__(self, in_dim, activation=None, num_buckets=16, max_distance=32, dropout=0.0, stream=None):
        super().__init__()
        self.head_dim = _head_size(in_dim)
        self.heads = in_dim // self.head_dim
        self.num_buckets, self.max_distance = num_buckets, max_distance
        self.activation = activation  # accepted and ignored, as by SelfAttention
        self.qkv_conv = HipConv2d(in_dim, 3 * in_dim, kernel_size=1)
        self.out_conv = HipConv2d(in_dim, in_dim, kernel_size=1)
        self.query_norm = nn.Parameter(torch.ones(self.head_dim))
        self.key_norm = nn.Parameter(torch.ones(self.head_dim))
        self.bias_table = nn.Parameter(torch.zeros(num_buckets * num_buckets, self.heads))
        self.dropout = HipDropout(dropout, stream)
        self._plans = {}      # (H, W, device) -> (RelativePositions, cos, sin): constants of the map's shape

    def _plan(self, h, w, device):
        key = (h, w, device)
        if key not in self._plans:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError(f"RelativeAttention meets {h} x {w} maps for the first time inside a stream capture; run one eager "
                                   "step first")
            self._plans[key] = (ops_tokens.RelativePositions((h, w), self.num_buckets, self.max_distance, device=device),
                                *ops_tokens.rotary_table((h, w), self.head_dim, device=device))
        return self._plans[key]

    def forward(self, x):
        b, c, h, w = x.shape
        plan, cos, sin = self._plan(h, w, x.device)
        qkv = self.qkv_conv(x).permute(0, 2, 3, 1).reshape(b, h * w, 3 * self.heads, self.head_dim)
        q, k, v = qkv.split(self.heads, 2)
        q, k = ops_tokens.qk_norm_rotary(q, k, self.query_norm, self.key_norm, cos, sin)
        o = ops_tokens.attention(q, k, v, relative=plan, bias_table=self.bias_table)
        y = self.out_conv(o.reshape(b, h, w, c).permute(0, 3, 1, 2))
        return self.dropout(y, residual=x) if self.dropout.active() else ops.add(x, y)
