"""Actor and critic (reference: ``src/rlsp/agents/models.py:55-154``).

Actor (graph mode): ``emb = GNN(obs)``; ``MLP([emb | mask]) * mask`` with PyG ``MLP`` semantics
(ReLU between layers, plain last layer, no norm) and **no output squashing** (Q6).
Critic: ``MLP([GNN(obs) | mask | action]) -> Q``.

Flat mode (``graph_mode: False``, reference ``models.py:115-122, 151``): the reference sizes the
actor's first layer for ``obs + action`` inputs but feeds only the flattened observation (Q13, a
shape error at the first forward).  Here flat mode is the evident intent: actor
``MLP(flatten(obs)) -> action``, critic ``MLP([flatten(obs) | action]) -> Q`` (no embedder, no mask
inputs; the actor output is still multiplied by the topology's action mask so padded nodes
schedule nothing).

The action mask is a per-topology constant, so its contribution to the first layer,
``mask @ W1[:, H:H+A]^T``, is evaluated once per topology and added like a bias instead of
multiplying a ``[B, A]`` block of known zeros/ones (bit-for-bit the same function and the same
gradients — autograd sees the mask columns of ``W1`` through that per-topology product).

Optional hidden parts (keys of the agent config with an ``actor_`` or ``critic_`` prefix; absent: the reference's MLP):

    hidden_layer_norm: layer       hidden activation = dropout(relu(layer_norm(h)))
    feedforward_blocks: N          N residual blocks behind the last hidden activation,
                                   h <- h + dropout(W_d gated_linear(layer_norm(h)) + b_d)
    feedforward_expansion: 4       width of a block's gated layer, in widths of the last hidden layer
    feedforward_activation: silu   of the gated layer (silu, gelu, sigmoid)
    dropout: p                     in training mode only; the mask is a function of the site and of the learner's update

They run on :mod:`gsc_amd.ops` (HIP kernels on the GPU, PyTorch references on the CPU).
"""
from __future__ import annotations

from typing import List, Sequence

import math

import numpy as np
import torch
import torch.nn as nn
import torch.nn.functional as F

from gsc_amd.ops import dropout, gated_linear, layer_norm
from gsc_amd.ops.gated import ACTIVATIONS
from gsc_amd.ops.linear import composed_projection, linear, shadow
from .gnn import GNNEmbedder
from .graphs import GraphSet


def select_rows(table: torch.Tensor, topo: torch.Tensor) -> torch.Tensor:
    """``table[topo]`` for a per-topology table ``[T, D]``.

    A single topology broadcasts (no [B, D] materialisation, and the backward is a plain column
    sum); several topologies use a one-hot GEMM, whose backward is again a GEMM instead of an
    atomic scatter-add of B rows into T rows."""
    if table.shape[0] == 1:
        return table
    onehot = F.one_hot(topo, table.shape[0]).to(table.dtype)
    return onehot @ table


class LayerNorm(nn.Module):
    """Scale and shift of :func:`gsc_amd.ops.layer_norm` over ``width`` features."""

    def __init__(self, width: int):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(width))
        self.bias = nn.Parameter(torch.zeros(width))

    def forward(self, x):
        return layer_norm(x, self.weight, self.bias)


class FeedForwardBlock(nn.Module):
    """``h + drop(W_d gated_linear(layer_norm(h)) + b_d)``: gate and up rows of the gated layer in one ``[2 hidden, width]``
    weight, initialised like ``nn.Linear``."""

    def __init__(self, width: int, hidden: int, activation: str):
        super().__init__()
        self.activation = activation
        self.norm = LayerNorm(width)
        bound = 1.0 / math.sqrt(width)
        self.weight = nn.Parameter(torch.empty(2 * hidden, width).uniform_(-bound, bound))
        self.bias = nn.Parameter(torch.empty(2 * hidden).uniform_(-bound, bound))
        self.down = nn.Linear(hidden, width)

    def forward(self, h, drop):
        g = gated_linear(self.norm(h), self.weight, self.bias, activation=self.activation)
        return drop(linear(g, self.down.weight, self.down.bias).to(h.dtype), residual=h)


def hidden_options(cfg: dict, net: str) -> dict:
    """The optional hidden parts of ``net`` ("actor" or "critic") in an agent config, checked."""
    get = lambda key, default: cfg.get(f"{net}_{key}", default)
    norm = get("hidden_layer_norm", "none") or "none"
    if norm not in ("none", "layer"):
        raise ValueError(f"{net}_hidden_layer_norm must be none|layer, got {norm}")
    blocks, expansion = get("feedforward_blocks", 0) or 0, get("feedforward_expansion", 4)
    if int(blocks) != blocks or blocks < 0 or int(expansion) != expansion or expansion < 1:
        raise ValueError(f"{net}_feedforward_blocks must be >= 0 and {net}_feedforward_expansion >= 1 (whole numbers), got "
                         f"{blocks} and {expansion}")
    act = get("feedforward_activation", "silu")
    if act not in ACTIVATIONS:
        raise ValueError(f"{net}_feedforward_activation must be {'|'.join(ACTIVATIONS)}, got {act}")
    p = float(get("dropout", 0.0) or 0.0)
    if not 0.0 <= p < 1.0:
        raise ValueError(f"{net}_dropout must be in [0, 1), got {p}")
    if (blocks or norm == "layer" or p) and not cfg[f"{net}_hidden_layer_nodes"]:
        raise ValueError(f"{net}_hidden_layer_norm, {net}_feedforward_blocks and {net}_dropout need a hidden layer")
    return {"norm": norm == "layer", "blocks": int(blocks), "expansion": int(expansion), "activation": act, "dropout": p}


class MaskedInputMLP(nn.Module):
    """PyG-style MLP whose input is ``[dense | mask(topology) | extra]``; mask block folded per topology.

    ``norm`` / ``blocks`` / ``expansion`` / ``activation`` / ``dropout``: the optional hidden parts (module docstring).
    Dropout is active in training mode; its masks follow ``drop_step`` (:meth:`advance_dropout`), a device counter, so
    captured graphs draw new ones on every replay."""

    def __init__(self, dense_dim: int, mask_dim: int, extra_dim: int, hidden: Sequence[int], out_dim: int, norm: bool = False,
                 blocks: int = 0, expansion: int = 4, activation: str = "silu", dropout: float = 0.0):
        super().__init__()
        self.dense_dim, self.mask_dim, self.extra_dim = dense_dim, mask_dim, extra_dim  # mask_dim 0: no mask input
        dims = [dense_dim + mask_dim + extra_dim, *hidden, out_dim]
        self.layers = nn.ModuleList([nn.Linear(dims[i], dims[i + 1]) for i in range(len(dims) - 1)])
        self.norms = nn.ModuleList([LayerNorm(w) for w in hidden]) if norm else None
        self.blocks = (nn.ModuleList([FeedForwardBlock(hidden[-1], expansion * hidden[-1], activation) for _ in range(blocks)])
                       if blocks else None)
        self.dropout, self.drop_seed = float(dropout), 0
        if self.dropout:
            self.register_buffer("drop_step", torch.zeros(1, dtype=torch.int64), persistent=False)

    @property
    def plain(self) -> bool:
        """Only linear layers and ReLU (what the native learner's kernels cover)."""
        return self.norms is None and self.blocks is None and not self.dropout

    def seed_dropout(self, seed: int) -> None:
        self.drop_seed = int(seed) & 0xFFFFFFFFFFFFFFFF

    def advance_dropout(self) -> None:
        """New masks from here on (one device addition, recorded in captured graphs)."""
        if self.dropout:
            self.drop_step.add_(1)

    def _drop(self, x, site: int, residual=None):
        """Dropout site ``site`` (plus ``residual``): hidden layer i is site i, block j site -1 - j."""
        if not (self.training and self.dropout):
            return x if residual is None else residual + x
        seed = (self.drop_seed + site * 0x9E3779B97F4A7C15) & 0xFFFFFFFFFFFFFFFF   # odd multiplier: a seed per site
        return dropout(x, self.dropout, seed, self.drop_step, residual=residual)

    def _hidden_activation(self, h, i: int):
        """Activation of hidden layer ``i`` from its linear output; behind the last one, the feed-forward blocks."""
        if self.norms is not None:
            h = self.norms[i](h)
        h = self._drop(F.relu(h), i)
        if i == len(self.layers) - 2 and self.blocks is not None:
            for j, block in enumerate(self.blocks):
                h = block(h, lambda x, residual, j=j: self._drop(x, -1 - j, residual))
        return h

    @property
    def first(self) -> nn.Linear:
        return self.layers[0]

    def first_layer(self, dense, topo, masks, extra=None):
        W = self.first.weight
        W16 = shadow(W)
        sl = lambda a, b: (W[:, a:b], W16[:, a:b] if W16 is not None else None)
        D, A = self.dense_dim, self.mask_dim
        w, w16 = sl(0, D)
        h = linear(dense, w, self.first.bias, w16=w16)
        if A > 0:
            w, w16 = sl(D, D + A)
            topo_bias = linear(masks, w, w16=w16)            # [T, h1]
            h = h + select_rows(topo_bias, topo)
        if extra is not None:
            w, w16 = sl(D + A, W.shape[1])
            h = h + linear(extra, w, w16=w16)
        return h

    def forward(self, dense, topo, masks, extra=None, out_mask=None, out_mask16=None):
        """``out_mask`` [out_dim]: multiply the output by a constant 0/1 vector, folded into the last
        layer's weight rows and bias (same values as masking the ``[B, out]`` output, no extra pass)."""
        h = self.first_layer(dense, topo, masks, extra)
        last = len(self.layers) - 1
        for i, layer in enumerate(self.layers):
            if i == 0:
                continue
            h = self._hidden_activation(h, i - 1)
            if i == last and out_mask is not None:
                h = linear(h, layer.weight, layer.bias, row_mask=out_mask, row_mask16=out_mask16)
            else:
                h = linear(h, layer.weight, layer.bias)
        if last == 0 and out_mask is not None:
            h = h * out_mask
        return h

    def hidden(self, dense, topo, masks, extra=None):
        """Input of the last layer (activation of the last hidden layer)."""
        h = self.first_layer(dense, topo, masks, extra)
        for i, layer in enumerate(self.layers[1:-1]):
            h = linear(self._hidden_activation(h, i), layer.weight, layer.bias)
        return self._hidden_activation(h, len(self.layers) - 2)

    def from_first(self, h):
        """Output from the first layer's linear output."""
        for i, layer in enumerate(self.layers[1:]):
            h = linear(self._hidden_activation(h, i), layer.weight, layer.bias)
        return h

    def forward_full(self, x):
        """Unfolded reference: ``x`` is the explicit concatenation (used by tests)."""
        h = x
        for i, layer in enumerate(self.layers):
            h = layer(h if i == 0 else self._hidden_activation(h, i - 1))
        return h


def _embedder(cfg: dict, in_dim: int) -> GNNEmbedder:
    return GNNEmbedder(input_dim=in_dim, hidden_dim=int(cfg["GNN_features"]), num_layers=int(cfg["GNN_num_layers"]),
                       aggr=cfg.get("GNN_aggr", "mean"), num_iter=int(cfg["GNN_num_iter"]))


def _flat_dim(cfg: dict, obs_dim: int, action_dim: int) -> int:
    """Flattened observation size in flat mode: n_pad x obs features (n_pad from the action size)."""
    P = int(cfg.get("max_nodes", 24))
    return P * obs_dim


class Actor(nn.Module):
    def __init__(self, cfg: dict, obs_dim: int, action_dim: int, low=0.0, high=1.0):
        super().__init__()
        self.graph_mode = bool(cfg.get("graph_mode", True))
        self.action_dim = action_dim
        if self.graph_mode:
            self.embedder = _embedder(cfg, obs_dim)
            H, mdim = self.embedder.hidden_dim, action_dim
        else:
            self.embedder = None
            H, mdim = _flat_dim(cfg, obs_dim, action_dim), 0
        self.mlp = MaskedInputMLP(H, mdim, 0, list(cfg["actor_hidden_layer_nodes"]), action_dim,
                                  **hidden_options(cfg, "actor"))
        self.low, self.high = float(low), float(high)
        # reference: no output squashing (Q6); new optional key ``actor_output_activation: sigmoid``
        # bounds the policy to the [0, 1] action box (keeps the critic from being queried far outside
        # the replayed actions, where its linear extrapolation drives the actor loss to -inf)
        act = cfg.get("actor_output_activation", "none") or "none"
        if act not in ("none", "sigmoid"):
            raise ValueError(f"actor_output_activation must be none|sigmoid, got {act}")
        self.squash = act == "sigmoid"

    def embed(self, x, topo, graphs: GraphSet):
        return self.embedder(x, topo, graphs) if self.graph_mode else x.reshape(x.shape[0], -1)

    def forward(self, x, topo, graphs: GraphSet, masks: torch.Tensor):
        emb = self.embed(x, topo, graphs)
        if self.squash:
            return torch.sigmoid(self.mlp(emb, topo, masks)) * select_rows(masks, topo)
        if masks.shape[0] == 1:  # one topology: fold the output mask into the last layer
            m16 = shadow(masks)
            return self.mlp(emb, topo, masks, out_mask=masks[0], out_mask16=m16[0] if m16 is not None else None)
        out = self.mlp(emb, topo, masks)
        return out * select_rows(masks, topo)

    def hidden(self, x, topo, graphs: GraphSet, masks: torch.Tensor):
        """Last hidden activation ``z`` with ``forward(x) = (z W^T + b) * mask`` (W, b = last layer)."""
        return self.mlp.hidden(self.embed(x, topo, graphs), topo, masks)

    def scale_action(self, a):
        return 2.0 * ((a - self.low) / (self.high - self.low)) - 1.0

    def unscale_action(self, a):
        return self.low + (0.5 * (a + 1.0) * (self.high - self.low))


class QNetwork(nn.Module):
    def __init__(self, cfg: dict, obs_dim: int, action_dim: int):
        super().__init__()
        self.graph_mode = bool(cfg.get("graph_mode", True))
        if self.graph_mode:
            self.embedder = _embedder(cfg, obs_dim)
            H, mdim = self.embedder.hidden_dim, action_dim
        else:
            self.embedder = None
            H, mdim = _flat_dim(cfg, obs_dim, action_dim), 0
        self.mlp = MaskedInputMLP(H, mdim, action_dim, list(cfg["critic_hidden_layer_nodes"]), 1,
                                  **hidden_options(cfg, "critic"))

    def embed(self, x, topo, graphs: GraphSet):
        return self.embedder(x, topo, graphs) if self.graph_mode else x.reshape(x.shape[0], -1)

    def forward(self, x, topo, graphs: GraphSet, masks: torch.Tensor, action: torch.Tensor):
        emb = self.embed(x, topo, graphs)
        return self.mlp(emb, topo, masks, action)


    def forward_on_actor(self, x, topo, graphs: GraphSet, masks: torch.Tensor, actor: "Actor", z: torch.Tensor):
        """``forward(x, ..., actor(x))`` for one topology without materialising the ``[B, A]`` action.

        With one topology the actor output is ``a = z W2m^T + b2m`` (``W2m``, ``b2m``: last layer with
        the constant mask folded in), so the critic's action projection re-associates:
        ``a Wa^T = z (Wa W2m)^T + Wa b2m``.  Same function (up to rounding order); the ``[B, A]``
        actor output and its two large GEMMs (plus their backward) are replaced by an ``[H1, A] x
        [A, h]`` product and a ``[B, h] x [h, H1]`` GEMM.  Gradients reach the actor through
        ``W2m``, ``b2m`` and ``z`` exactly as through ``a``."""
        assert masks.shape[0] == 1, "composed critic/actor path needs a single topology"
        mlp = self.mlp
        D, A = mlp.dense_dim, mlp.mask_dim
        W1 = mlp.first.weight
        Wa = W1[:, D + A:]                                   # [h1, A]
        W16 = shadow(W1)
        if W16 is not None:
            Wa._bf16 = W16[:, D + A:]
        last = actor.mlp.layers[-1]
        m16 = shadow(masks)
        Mc, cb = composed_projection(Wa, last.weight, last.bias, masks[0],
                                     m16[0] if m16 is not None else None)   # [h1, z], [h1]
        emb = self.embed(x, topo, graphs)
        return mlp.from_first(mlp.first_layer(emb, topo, masks) + linear(z, Mc, cb))


def count_params(m: nn.Module) -> int:
    return sum(p.numel() for p in m.parameters())
