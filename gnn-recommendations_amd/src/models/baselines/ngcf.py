"""NGCF as implemented by the reference (src/models/baselines/ngcf.py), MI355X kernels.

Per layer (ngcf.py:52-86, the code's form, not the paper's):
    n = A x;   out = Dropout(LeakyReLU_0.2(W1 n + b1 + W2 (x * n) + b2))
and the model output is cat(x0, x1, ..., xK) along features (ngcf.py:186).

On a ROCm operand in inference (no autograd, dropout inactive) each layer is ONE kernel:
SpMM + both Linear layers on MFMA + bias + LeakyReLU (gnnrec_spmm_ngcf_f32). With autograd
on, the SpMM stays native (differentiable) and the two 64x64 Linear layers run through torch.

Two options that the reference does not have, off by default:
* ``counter_dropout``: on a ROCm device the LeakyReLU and the dropout are one native pass with a
  counter-based mask that is never stored (ops.dropout) instead of torch's;
* ``layer_norm``: a layer's output is LayerNorm(x + Dropout(LeakyReLU(...))) (without the
  residual x where the widths differ), one native pass each way (ops.dropout_add_layer_norm),
  the mask counter-based as well. It keeps stacked hops from drifting to one direction and scale.
Their masks' seed is drawn from torch's generator for every training forward, or read from
``model.dropout_seed`` where that is set (a one-element int64 tensor on the device; a captured
training step needs it, to draw new masks on replay); the layer's number is the mask's site.
"""
from typing import List, Optional, Tuple

import torch
import torch.nn as nn
import torch.nn.functional as F

from ..base import BaseRecommender
from ... import ops
from ...ops.graph import CsrGraph


class NGCFLayer(nn.Module):
    """One NGCF propagation layer (ngcf.py:19-86)."""

    def __init__(self, in_dim: int, out_dim: int, dropout: float = 0.0,
                 counter_dropout: bool = False, layer_norm: bool = False):
        super().__init__()
        self.W1 = nn.Linear(in_dim, out_dim, bias=True)
        self.W2 = nn.Linear(in_dim, out_dim, bias=True)
        self.dropout = nn.Dropout(dropout)
        self.activation = nn.LeakyReLU(negative_slope=0.2)
        self.counter_dropout = counter_dropout
        self.norm = nn.LayerNorm(out_dim) if layer_norm else None
        self.single_kernel = False  # True: gather + MFMA in one launch (see ops.ngcf_layer)

    def __setstate__(self, state):
        """A layer that was saved whole before it had the options is one without them."""
        super().__setstate__(state)
        self.__dict__.setdefault("counter_dropout", False)
        if not hasattr(self, "norm"):
            self.norm = None

    def _fused_ok(self, x: torch.Tensor, a) -> bool:
        return (isinstance(a, CsrGraph) and not (torch.is_grad_enabled() and (
            x.requires_grad or self.W1.weight.requires_grad))
            and (not self.training or self.dropout.p == 0.0)
            and self.W1.in_features == self.W1.out_features
            and self.W1.in_features in (32, 64, 128))

    def normalised(self, z: torch.Tensor, x: torch.Tensor, p: float = 0.0, seed=0,
                   site: int = 0, negative_slope: float = 1.0) -> torch.Tensor:
        """LayerNorm(x + Dropout_p(LeakyReLU(z))); the layer's rows only, so a row shard may
        call it with its own. Under autocast z is in half precision: the sum and the norm are in
        x's fp32, which the next hop gathers."""
        z = z.to(torch.promote_types(z.dtype, x.dtype))
        res = x if x.shape == z.shape else None
        if z.is_cuda:
            return ops.dropout_add_layer_norm(z, res, self.norm.weight, self.norm.bias, p, seed,
                                              site=site, negative_slope=negative_slope,
                                              eps=self.norm.eps)[0]
        out = F.dropout(F.leaky_relu(z, negative_slope), p, training=p > 0)
        return self.norm(out if res is None else res + out)

    def forward(self, x: torch.Tensor, adj_matrix, gas: Optional[nn.Module] = None, seed=None,
                site: int = 0) -> torch.Tensor:
        """seed: of the counter-based mask (see the module's text), needed where one is drawn."""
        a = ops.as_operand(adj_matrix)
        if self._fused_ok(x, a) and (gas is None or gas.fusable()):
            fuse_gas = gas is not None and self.norm is None
            blocks, perm = (gas.blocks(), gas.perm) if fuse_gas else (None, None)
            out = ops.ngcf_layer(a, x, self.W1.weight, self.W1.bias, self.W2.weight,
                                 self.W2.bias, self.activation.negative_slope,
                                 gas_blocks=blocks, gas_perm=perm, fused=self.single_kernel)
            if self.norm is None:
                return out
            out = self.normalised(out, x)
            return gas(out) if gas is not None else out
        n = ops.sparse_mm(a, x)
        if isinstance(a, CsrGraph):   # device path: row-chunked weight gradients (training)
            lin = ops.functional.linear_rows
            out = lin(n, self.W1) + lin(x * n, self.W2)
        else:
            out = self.W1(n) + self.W2(x * n)
        p = self.dropout.p if self.dropout.training else 0.0
        slope = self.activation.negative_slope
        if p > 0 and out.is_cuda and seed is None and (self.counter_dropout
                                                       or self.norm is not None):
            raise ValueError("NGCFLayer: the counter-based dropout needs a seed")
        if self.norm is not None:
            out = self.normalised(out, x, p, seed if p > 0 else 0, site, slope)
        elif self.counter_dropout and p > 0 and out.is_cuda:
            out = ops.dropout(out, p, seed, site=site, negative_slope=slope)
        else:
            out = self.dropout(self.activation(out))
        return gas(out) if gas is not None else out


class NGCF(BaseRecommender):
    dropout_seed: Optional[torch.Tensor] = None     # see the module's text

    def __init__(self, n_users: int, n_items: int, embedding_dim: int = 64,
                 layer_sizes: Optional[List[int]] = None, dropout: float = 0.1,
                 init_scale: float = 0.01, counter_dropout: bool = False,
                 layer_norm: bool = False):
        super().__init__(n_users, n_items, embedding_dim)
        layer_sizes = [64, 64, 64] if layer_sizes is None else list(layer_sizes)
        self.layer_sizes = layer_sizes
        self.n_layers = len(layer_sizes)
        self.dropout = dropout
        self.init_scale = init_scale
        self.user_embedding = nn.Embedding(n_users, embedding_dim)
        self.item_embedding = nn.Embedding(n_items, embedding_dim)
        dims = [embedding_dim] + layer_sizes
        self.layers = nn.ModuleList(NGCFLayer(dims[k], dims[k + 1], dropout, counter_dropout,
                                              layer_norm)
                                    for k in range(self.n_layers))
        self.reset_parameters()

    def reset_parameters(self):
        # ngcf.py:143-155
        nn.init.normal_(self.user_embedding.weight, mean=0.0, std=self.init_scale)
        nn.init.normal_(self.item_embedding.weight, mean=0.0, std=self.init_scale)
        for layer in self.layers:
            for lin in (layer.W1, layer.W2):
                nn.init.xavier_uniform_(lin.weight)
                nn.init.zeros_(lin.bias)
            if layer.norm is not None:
                layer.norm.reset_parameters()

    def _mask_seed(self):
        """The seed of one training forward's counter-based masks, None where none is drawn."""
        if not any(layer.dropout.training and layer.dropout.p > 0
                   and (layer.counter_dropout or layer.norm is not None) for layer in self.layers):
            return None
        if self.dropout_seed is not None:
            return self.dropout_seed
        if self.user_embedding.weight.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("NGCF: a captured step needs model.dropout_seed (an int64 tensor "
                               "on the device); a seed drawn now would be every replay's")
        return int(torch.randint(0, 2 ** 63 - 1, (1,)).item())

    def _mask_arguments(self):
        """What each layer is told of its mask; nothing where none is drawn."""
        seed = self._mask_seed()
        return [{} if seed is None else {"seed": seed, "site": k} for k in range(len(self.layers))]

    def forward(self, adj_matrix) -> Tuple[torch.Tensor, torch.Tensor]:
        x_final = self._native_concat_forward(adj_matrix, [None] * self.n_layers)
        if x_final is None:
            x = self._initial_table()
            outs = [x]
            mask = self._mask_arguments()
            for layer, kw in zip(self.layers, mask):
                x = layer(x, adj_matrix, **kw)
                outs.append(x)
            x_final = torch.cat(outs, dim=1)
        user_emb, item_emb = torch.split(x_final, [self.n_users, self.n_items], dim=0)
        return user_emb, item_emb

    def _native_concat_forward(self, adj_matrix, gs_layers):
        """Inference on a ROCm operand: every layer's fused kernel reads its input from, and
        writes its output into, its column block of the final [N, (K+1) d] table, so
        torch.cat(outs, dim=1) (ngcf.py:186) costs no extra pass over 2 GB at G100M. Same
        values as the layer-by-layer form (the kernels do not depend on row strides).
        None when a layer cannot take the fused path."""
        a = ops.as_operand(adj_matrix)
        d = self.embedding_dim
        if not all(layer._fused_ok(self.user_embedding.weight, a) and layer.W1.in_features == d
                   and layer.norm is None
                   and (gs is None or gs.fusable())
                   for layer, gs in zip(self.layers, gs_layers)):
            return None
        n = self.n_users + self.n_items
        w = self.user_embedding.weight
        # placed so that the gathered blocks x0 .. x_{K-1} avoid the slow line offset
        # (ops.functional.gather_table); still a contiguous [N, (K+1) d] tensor
        out = ops.functional.gather_table(n, d * (self.n_layers + 1), d * self.n_layers,
                                          dtype=w.dtype, device=w.device)
        out[:self.n_users, :d].copy_(self.user_embedding.weight.detach())
        out[self.n_users:, :d].copy_(self.item_embedding.weight.detach())
        for k, (layer, gs) in enumerate(zip(self.layers, gs_layers)):
            blocks, perm = (gs.blocks(), gs.perm) if gs is not None else (None, None)
            ops.ngcf_layer(a, out[:, k * d:(k + 1) * d], layer.W1.weight, layer.W1.bias,
                           layer.W2.weight, layer.W2.bias, layer.activation.negative_slope,
                           gas_blocks=blocks, gas_perm=perm, fused=layer.single_kernel,
                           out=out[:, (k + 1) * d:(k + 2) * d])
        return out

    def predict(self, users, items, adj_matrix=None) -> torch.Tensor:
        if adj_matrix is None:
            raise ValueError("adj_matrix must be given for NGCF")
        user_emb, item_emb = self._serving_embeddings(adj_matrix)
        return self._score_pairs(user_emb, item_emb, users, items)

    def get_all_embeddings(self, adj_matrix=None) -> Tuple[torch.Tensor, torch.Tensor]:
        if adj_matrix is None:
            raise ValueError("adj_matrix must be given for NGCF")
        return self.forward(adj_matrix)


class NGCFGroupShuffle(NGCF):
    """NGCF with a Group-and-Shuffle transform after every layer,
    x_{l+1} = GS_l(NGCFLayer_l(x_l)); fused into one kernel per layer on a ROCm operand.
    The composition is defined by this build (the reference has no such model class); its
    oracle is composed from the reference's NGCFLayer and GroupShuffleLayer."""

    def __init__(self, n_users: int, n_items: int, embedding_dim: int = 64,
                 layer_sizes: Optional[List[int]] = None, dropout: float = 0.1,
                 init_scale: float = 0.01, block_size: int = 8, gs_init_scale: float = 0.01,
                 counter_dropout: bool = False, layer_norm: bool = False):
        super().__init__(n_users, n_items, embedding_dim, layer_sizes, dropout, init_scale,
                         counter_dropout, layer_norm)
        from ..orthogonal_bundle.group_shuffle_layer import GroupShuffleLayer
        self.gs_layers = nn.ModuleList(GroupShuffleLayer(d, block_size, gs_init_scale)
                                       for d in self.layer_sizes)

    def forward(self, adj_matrix) -> Tuple[torch.Tensor, torch.Tensor]:
        x_final = self._native_concat_forward(adj_matrix, list(self.gs_layers))
        if x_final is None:
            x = self._initial_table()
            outs = [x]
            mask = self._mask_arguments()
            for layer, gs, kw in zip(self.layers, self.gs_layers, mask):
                x = layer(x, adj_matrix, gas=gs, **kw)
                outs.append(x)
            x_final = torch.cat(outs, dim=1)
        user_emb, item_emb = torch.split(x_final, [self.n_users, self.n_items], dim=0)
        return user_emb, item_emb
