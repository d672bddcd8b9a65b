"""The encoder operators in elementary torch operations on any device, rounded where ops.py's say they round: what the encoder's own
tests run on without a GPU."""
import torch

import ops_reference as ref

ACT = {"none": lambda z: z, "gelu": torch.nn.functional.gelu, "gelu_tanh": lambda z: torch.nn.functional.gelu(z, approximate="tanh"), "relu": torch.relu}


def linear(x, weight, bias=None, activation="none", residual=None):
    assert all(t is None or t.dtype == x.dtype for t in (weight, bias, residual))
    y = ACT[activation](x.float() @ weight.float().t() + (0 if bias is None else bias.float()))
    return (y if residual is None else y + residual.float()).to(x.dtype)


def bucketed_attention(qkv, table, offsets, scale=None, max_distance=128):
    assert table.dtype == qkv.dtype and table.shape[1] == qkv.shape[2]
    scale = qkv.shape[3] ** -0.5 if scale is None else scale
    out, ends = torch.zeros_like(qkv[:, 0]), offsets.tolist()
    for lo, hi in zip(ends, ends[1:]):
        if lo < hi:
            q, k, v = qkv[lo:hi].float().permute(1, 2, 0, 3)
            bias = table.float().t()[:, ref.buckets_of(hi - lo, table.shape[0], max_distance)]
            out[lo:hi] = (torch.softmax(scale * (q @ k.transpose(1, 2)) + bias, -1) @ v).transpose(0, 1).to(out.dtype)
    return out


def mean_pool(hidden, offsets, normalize=True):
    ends = offsets.tolist()
    mean = torch.stack([hidden[lo:hi].float().mean(0) if lo < hi else torch.zeros(hidden.shape[1]) for lo, hi in zip(ends, ends[1:])])
    return mean / mean.norm(dim=1, keepdim=True).clamp(min=1e-12) if normalize else mean
