"""MPNet's encoder on the framework's own operators (ops.py): what MPNetEmbedder(engine="hip") runs.

The reference's embedding model (src/vectordb.py:13-69, src/config.py:36) is an MPNet: token and position embeddings, then
layers of  x = LN(attention(x) + x);  x = LN(W2 gelu(W1 x + b1) + b2 + x)  with one relative position bias table shared by
all layers, then the mean over a text's tokens, to unit length.  Here the tokens of a batch are packed without padding, the
three projections of a layer run as one product, bias, activation and residual are part of their product's kernel, and the
position bias never becomes a matrix."""
from __future__ import annotations

from typing import Sequence

import torch
import torch.nn.functional as F

from . import ops

#: names of the transformers configuration -> ops.linear's
_ACTIVATIONS = {"gelu": "gelu", "gelu_new": "gelu_tanh", "gelu_pytorch_tanh": "gelu_tanh", "relu": "relu"}
#: the model's bucketing, whatever its configuration says: it uses a larger table's first rows, and fails on a smaller one
BUCKETS, MAX_DISTANCE = 32, 128


class MPNetEncoder:
    """Runs a transformers MPNetModel's weights.  dtype: what the products and the attention compute in (float32, bfloat16, float16);
    the embedding look-up, the sums x + f(x) between the layers, the normalisations and the pooled vector are float32, as under
    torch.autocast.  There is no dropout, as in eval()."""

    def __init__(self, model: torch.nn.Module, dtype: torch.dtype = torch.float32):
        cfg = model.config
        if getattr(cfg, "model_type", None) != "mpnet":
            raise ValueError(f"only MPNet models are supported; got {type(model).__name__}")
        if cfg.hidden_act not in _ACTIVATIONS:
            raise ValueError(f"hidden_act {cfg.hidden_act!r} is not one of {sorted(_ACTIVATIONS)}")
        if cfg.hidden_size % cfg.num_attention_heads or cfg.hidden_size // cfg.num_attention_heads > 128:
            raise ValueError(f"heads of {cfg.hidden_size}/{cfg.num_attention_heads} values are not supported (whole, at most 128)")
        if model.encoder.relative_attention_bias.weight.shape[0] < BUCKETS:
            raise ValueError(f"a position bias of {model.encoder.relative_attention_bias.weight.shape[0]} buckets is not supported (the model looks up {BUCKETS})")
        self.model = model
        self.dtype = dtype
        self.activation = _ACTIVATIONS[cfg.hidden_act]
        self.eps = float(cfg.layer_norm_eps)
        self.heads = int(cfg.num_attention_heads)
        self.pad = int(model.embeddings.padding_idx)      # positions count from behind it; the model takes 1 whatever cfg.pad_token_id says
        self.max_positions = int(model.embeddings.position_embeddings.weight.shape[0])

    # -- weights -------------------------------------------------------------
    def _modules(self):
        for layer in self.model.encoder.layer:
            a = layer.attention.attn
            up, down = layer.intermediate.dense, layer.output.dense
            for m in (a.q, a.k, a.v, a.o, up, down):
                if type(m).forward is not torch.nn.Linear.forward:     # an adapter or a quantised layer: its weight alone is not what it computes
                    raise ValueError(f"layers must be torch.nn.Linear; got {type(m).__name__}")
            yield a, layer.attention.LayerNorm, up, down, layer.output.LayerNorm

    def _table(self):
        return self.model.encoder.relative_attention_bias.weight[:BUCKETS]

    def _layers(self):
        """The weights as the operators take them, differentiable."""
        dt = self.dtype
        layers = []
        for a, norm, up, down, norm2 in self._modules():
            layers.append((
                torch.cat([a.q.weight, a.k.weight, a.v.weight]).to(dt), torch.cat([a.q.bias, a.k.bias, a.v.bias]).to(dt),
                a.o.weight.to(dt), a.o.bias.to(dt), norm.weight.float(), norm.bias.float(), up.weight.to(dt), up.bias.to(dt),
                down.weight.to(dt), down.bias.to(dt), norm2.weight.float(), norm2.bias.float()))
        return self._table().to(dt), layers

    def lay_out(self):
        """The same without gradients: what encode() computes with under no_grad, and takes as its `weights` where a program runs
        several batches on the same ones.  All copies go into one buffer by one call (12 layers of 768: 0.2 ms of host time in fp32, where
        only the three projections are joined, 0.27 in 16 bits; 0.38 and 1.13 tensor by tensor).  They are made anew for every call, from
        what the parameters hold then, on the stream that uses them: nothing tells reliably whether a parameter has changed (fused
        optimisers and replayed graphs count no version), and copies kept for later would have to be waited for by other streams
        and outlive the graphs captured with them."""
        dt = self.dtype
        sources, places, layers = [], [], []
        at = 0

        def copied(*parts):
            """-> (offset, shape) of the parts one behind the other, the first on a 16-byte border."""
            nonlocal at
            at = (at + 7) & -8
            begin = at
            for p in parts:
                sources.append(p)
                places.append(at)
                at += p.numel()
            return begin, (sum(p.shape[0] for p in parts), *parts[0].shape[1:])

        def taken(p):
            return p if p.dtype == dt else copied(p)

        with torch.no_grad():
            table = taken(self._table())
            for a, norm, up, down, norm2 in self._modules():
                layers.append((copied(a.q.weight, a.k.weight, a.v.weight), copied(a.q.bias, a.k.bias, a.v.bias),
                               taken(a.o.weight), taken(a.o.bias), norm.weight.float(), norm.bias.float(), taken(up.weight), taken(up.bias),
                               taken(down.weight), taken(down.bias), norm2.weight.float(), norm2.bias.float()))
            flat = torch.empty(at, dtype=dt, device=self._table().device)

            def view(begin, shape):
                return flat.as_strided(shape, (shape[1], 1) if len(shape) == 2 else (1,), begin)
            if sources:
                torch._foreach_copy_([view(b, p.shape) for b, p in zip(places, sources)], sources)
            return (table if isinstance(table, torch.Tensor) else view(*table),
                    [tuple(w if isinstance(w, torch.Tensor) else view(*w) for w in layer) for layer in layers])

    def refresh(self) -> None:
        """Nothing to do: the weights are laid out for every call.  Here for programs that ask for it after a change."""

    # -- forward -------------------------------------------------------------
    def pack(self, token_lists: Sequence[Sequence[int]], device) -> tuple:
        """Token ids, positions and offsets of a batch, on the device in one copy."""
        ids, places, ends = [], [], [0]
        for tokens in token_lists:
            at = self.pad                      # positions count from pad + 1; a pad token inside a text takes pad and is not counted
            for t in tokens:
                if t != self.pad:
                    at += 1
                ids.append(t)
                places.append(at if t != self.pad else self.pad)
            if at >= self.max_positions:
                raise ValueError(f"a text of {len(tokens)} tokens: the model has {self.max_positions - self.pad - 1} positions")
            ends.append(len(ids))
        n = len(ids)
        flat = torch.tensor(ids + places + ends, dtype=torch.int64).to(device)
        return flat[:n], flat[n:2 * n], flat[2 * n:]

    def encode(self, ids: torch.Tensor, places: torch.Tensor, offsets: torch.Tensor, weights=None) -> torch.Tensor:
        """Packed tokens -> float32 [n_texts, hidden], unit length.  With gradients enabled it is differentiable in the model's
        parameters (unless weights, of lay_out(), are given)."""
        emb = self.model.embeddings
        table, layers = weights or (self._layers() if torch.is_grad_enabled() else self.lay_out())
        x = emb.word_embeddings(ids).float() + emb.position_embeddings(places).float()
        hidden = x.shape[1]
        x = F.layer_norm(x, (hidden,), emb.LayerNorm.weight.float(), emb.LayerNorm.bias.float(), self.eps)
        for wqkv, bqkv, wo, bo, g1, c1, w1, b1, w2, b2, g2, c2 in layers:
            qkv = ops.linear(x.to(self.dtype), wqkv, bqkv).view(-1, 3, self.heads, hidden // self.heads)
            ctx = ops.bucketed_attention(qkv, table, offsets, max_distance=MAX_DISTANCE).view(-1, hidden)
            x = F.layer_norm(self._added(x, ctx, wo, bo), (hidden,), g1, c1, self.eps)
            up = ops.linear(x.to(self.dtype), w1, b1, self.activation)
            x = F.layer_norm(self._added(x, up, w2, b2), (hidden,), g2, c2, self.eps)
        return ops.mean_pool(x, offsets)

    def _added(self, x, inner, weight, bias):
        """x + inner weight^T + bias in 32 bits: inside the product's kernel in float32.  A 16-bit product's residual would be 16 bits too:
        the vectors of a 12-layer, 768-wide encoder (random weights, 14 tokens, bf16) were off by 0.0077 in the 2-norm that way, by
        0.0039 this way; transformers under autocast 0.0041.  The price is two more launches a sum: 64 texts of 302 tokens 5.0 -> 5.8 ms."""
        if self.dtype == torch.float32:
            return ops.linear(inner, weight, bias, residual=x)
        return x + ops.linear(inner, weight, bias)
