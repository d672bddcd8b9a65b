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
#: the model's bucketing ends here whatever its configuration says (its number of buckets is the table's)
MAX_DISTANCE = 128


class MPNetEncoder:
    """Runs a transformers MPNetModel's weights.  dtype: what the layers compute in (float32, bfloat16, float16); the embedding
    look-up and the pooled vector are float32.  There is no dropout, as in eval()."""

    def __init__(self, model: torch.nn.Module, dtype: torch.dtype = torch.float32):
        cfg = model.config
        if cfg.hidden_act not in _ACTIVATIONS:
            raise ValueError(f"hidden_act {cfg.hidden_act!r} is not one of {sorted(_ACTIVATIONS)}")
        if cfg.hidden_size % cfg.num_attention_heads or cfg.hidden_size // cfg.num_attention_heads > 128:
            raise ValueError(f"heads of {cfg.hidden_size}/{cfg.num_attention_heads} values are not supported (whole, at most 128)")
        self.model = model
        self.dtype = dtype
        self.activation = _ACTIVATIONS[cfg.hidden_act]
        self.eps = float(cfg.layer_norm_eps)
        self.heads = int(cfg.num_attention_heads)
        self.pad = int(cfg.pad_token_id)
        self.max_positions = int(model.embeddings.position_embeddings.weight.shape[0])
        self._laid_out = None
        self._stamp = None

    # -- weights -------------------------------------------------------------
    def _layers(self):
        """The weights as the operators take them, differentiable."""
        enc, dt = self.model.encoder, self.dtype
        layers = []
        for layer in enc.layer:
            a = layer.attention.attn
            layers.append((
                torch.cat([a.q.weight, a.k.weight, a.v.weight]).to(dt), torch.cat([a.q.bias, a.k.bias, a.v.bias]).to(dt),
                a.o.weight.to(dt), a.o.bias.to(dt), layer.attention.LayerNorm.weight.to(dt), layer.attention.LayerNorm.bias.to(dt),
                layer.intermediate.dense.weight.to(dt), layer.intermediate.dense.bias.to(dt),
                layer.output.dense.weight.to(dt), layer.output.dense.bias.to(dt), layer.output.LayerNorm.weight.to(dt), layer.output.LayerNorm.bias.to(dt)))
        return enc.relative_attention_bias.weight.to(dt), layers

    def refresh(self) -> None:
        """Lay the weights out again.  encode() does so by itself after an in-place change (an optimiser's step, load_state_dict)
        or a replaced parameter; only writes through `parameter.data` go unseen."""
        self._stamp = None

    def _frozen(self):
        stamp = tuple((id(p), p.data_ptr(), -1 if p.is_inference() else p._version) for p in self.model.encoder.parameters())
        if stamp != self._stamp:
            with torch.no_grad():
                self._laid_out = self._layers()
            self._stamp = stamp
        return self._laid_out

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

    def encode(self, ids: torch.Tensor, places: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
        """Packed tokens -> float32 [n_texts, hidden], unit length.  With gradients enabled it is differentiable in the model's
        parameters."""
        emb = self.model.embeddings
        table, layers = self._layers() if torch.is_grad_enabled() else self._frozen()
        x = emb.word_embeddings(ids) + emb.position_embeddings(places)
        hidden = x.shape[1]
        x = F.layer_norm(x, (hidden,), emb.LayerNorm.weight, emb.LayerNorm.bias, self.eps).to(self.dtype)
        for wqkv, bqkv, wo, bo, g1, c1, w1, b1, w2, b2, g2, c2 in layers:
            qkv = ops.linear(x, wqkv, bqkv).view(-1, 3, self.heads, hidden // self.heads)
            ctx = ops.bucketed_attention(qkv, table, offsets, max_distance=MAX_DISTANCE).view(-1, hidden)
            x = F.layer_norm(ops.linear(ctx, wo, bo, residual=x), (hidden,), g1, c1, self.eps)
            up = ops.linear(x, w1, b1, self.activation)
            x = F.layer_norm(ops.linear(up, w2, b2, residual=x), (hidden,), g2, c2, self.eps)
        return ops.mean_pool(x, offsets)
