"""Stand-ins for the module upstream imports but does not ship (`ROF_models`:
ROF_evaluation/ROF_main.py:31): the `ROF_inputInfo` attribute bag, the `ROF_GCN` stack, and a
GIN stack for the sum-aggregation configuration.  Shapes and argument order are inferred from
the call sites (ROF_main.py:164-174, 192-200, 230; ROF_evaluation/cuda/middle-rof.py:496)."""
import numpy as np
import torch
import torch.nn.functional as F
from torch.nn.modules.module import _has_any_global_hook

from . import norm as N
from .plan import AggregationPlan, scale_rows
from .reuse_conv import ROF_GCNConv

_TENSOR_FIELDS = ("row_pointers", "column_index", "degrees", "part_pointers", "part2Node", "part_cache_flagindex",
                  "part_pointers_cache", "column_index_cache", "uniqpart_column_index", "uniqpart_pointers",
                  "part2Node_ptr", "part2Node_col")


class ROF_inputInfo:
    """Positional order of ROF_main.py:164-174."""

    def __init__(self, row_pointers, column_index, degrees, part_pointers, part2Node, partSize, warpPerBlock,
                 part_cache_flagindex, part_pointers_cache, column_index_cache, uniqpart_column_index=None,
                 uniqpart_pointers=None, part2Node_ptr=None, part2Node_col=None):
        self.row_pointers, self.column_index, self.degrees = row_pointers, column_index, degrees
        self.part_pointers, self.part2Node = part_pointers, part2Node
        self.partSize, self.warpPerBlock = partSize, warpPerBlock
        self.part_cache_flagindex = part_cache_flagindex
        self.part_pointers_cache, self.column_index_cache = part_pointers_cache, column_index_cache
        self.uniqpart_column_index, self.uniqpart_pointers = uniqpart_column_index, uniqpart_pointers
        self.part2Node_ptr, self.part2Node_col = part2Node_ptr, part2Node_col
        self.dimWorker = 32
        self.transform_order = "reference"
        self.part_result_cache = None
        self.transposed = None      # optional ROF_inputInfo of the transposed graph (exact backward, directed graphs)

    @classmethod
    def from_layouts(cls, indptr_dst, layouts, warpPerBlock=4, device=None):
        """Build from the dict of numpy arrays a reuse search returns (int32 / float32 casts of
        ROF_main.py:138-161)."""
        t = lambda a, dt=torch.int32: torch.from_numpy(np.ascontiguousarray(a)).to(dt)
        info = cls(t(np.asarray(indptr_dst).astype(np.int32)), t(layouts["column_index"]),
                   torch.from_numpy(np.diff(indptr_dst).astype(np.float32)), t(layouts["part_pointers"]),
                   t(layouts["part2Node"]), int(layouts["part_size"]), warpPerBlock,
                   t(layouts["part_cache_flagindex"]), t(layouts["part_pointers_cache"]),
                   t(layouts["column_index_cache"]), t(layouts["uniqpart_column_index"]),
                   t(layouts["uniqpart_pointers"]), t(layouts["part2Node_ptr"]), t(layouts["part2Node_col"]))
        return info.to(device) if device is not None else info

    @property
    def reuse_size(self):
        return int(self.part_pointers_cache.shape[0]) - 1

    def with_transposed(self, other):
        """attach the layouts of the transposed graph; `other.degrees` is replaced by this graph's
        in-degrees, because A_hat^T = D^-1/2 A^T D^-1/2 keeps the forward normalisation"""
        other.degrees = self.degrees
        self.transposed = other
        return self

    def to(self, device):
        if self.transposed is not None:
            self.transposed.to(device)
        for f in _TENSOR_FIELDS:
            v = getattr(self, f)
            if isinstance(v, torch.Tensor):
                setattr(self, f, v.to(device))
        return self

    def __repr__(self):
        parts = []
        for f in _TENSOR_FIELDS:
            v = getattr(self, f)
            parts.append(f"{f}={tuple(v.shape) if isinstance(v, torch.Tensor) else v}")
        return f"ROF_inputInfo(partSize={self.partSize}, warpPerBlock={self.warpPerBlock}, " + ", ".join(parts) + ")"


def _stands_alone(module, kind):
    """whether a call of `module` is `kind`'s forward and nothing else, so that a pass fused with it may take its place: no other class,
    no hooks"""
    return (getattr(module.forward, "__func__", None) is kind.forward and not module._forward_hooks and not module._forward_pre_hooks
            and not module._backward_hooks and not module._backward_pre_hooks and not _has_any_global_hook())


def _norm_relu_dropout(m, h, relu, drop):
    """dropout(relu?(m(h))) -> (its value, whether the ReLU and the dropout are in it): one pass where `m` is a LayerNorm of norm.py that
    stands alone, else the call of the module"""
    if _stands_alone(m, N.LayerNorm) and not m.relu and m.p == 0:
        return N.layer_norm(h, m.weight, m.bias, m.eps, relu=relu, **drop), True
    return m(h), False


class ROF_GCN(torch.nn.Module):
    """n_layers hidden ROF_GCNConv layers + one output layer; activation and dropout between
    layers (constructor keywords of ROF_main.py:192-200).  Two keywords upstream does not have:
    norm="layer" puts a layer norm in front of every activation; dropout_source="counter" draws the
    dropout from the counter-based generator of norm.py (seed, step, row_offset of forward(); layer i of the stack takes
    step + i * 2**40), in one pass with what stands before it when the activation is F.relu."""

    def __init__(self, in_feats, n_hidden, n_classes, n_layers, activation=F.relu, dropout=0.5, add_self_loops=False,
                 reuse_size=0, kernel_type="ROF_v1", weight_initializer="glorot", norm=None, dropout_source="torch"):
        super().__init__()
        if norm not in (None, "layer") or dropout_source not in ("torch", "counter"):
            raise ValueError("ROF_GCN: norm is None or 'layer', dropout_source 'torch' or 'counter'")
        kw = dict(add_self_loops=add_self_loops, reuse_size=reuse_size, kernel_type=kernel_type,
                  weight_initializer=weight_initializer)
        dims = [in_feats] + [n_hidden] * n_layers + [n_classes]
        self.layers = torch.nn.ModuleList(ROF_GCNConv(a, b, **kw) for a, b in zip(dims[:-1], dims[1:]))
        self.activation, self.dropout, self.dropout_source = activation, dropout, dropout_source
        # (not among the children without a norm: the state of such a stack keeps its names)
        self.norms = torch.nn.ModuleList(N.LayerNorm(d) for d in dims[1:-1]) if norm is not None else None

    def __setstate__(self, state):
        # (a stack that was saved whole before it could have these)
        super().__setstate__({"norms": None, "dropout_source": "torch", **state} if "norms" not in state["_modules"] else state)

    def _between(self, h, i, bias, drop):
        """what stands between layer i and the next: norm, activation, dropout (`drop`: its keywords, or None)"""
        relu = self.activation is F.relu
        if self.norms is not None:
            h, done = _norm_relu_dropout(self.norms[i], h, relu, drop if relu and drop is not None else {})
            if done and relu:
                return h
        if relu and drop is not None:
            return N.dropout(h, bias=bias, relu=True, **drop)
        h = self.activation(h)
        return h if drop is None else N.dropout(h, **drop)

    def forward(self, features, inputInfo, edge_index=None, seed=None, step=0, row_offset=0):
        h = features
        last = len(self.layers) - 1
        counter = self.dropout_source == "counter"
        # in training mode a pass without gradients drops too (a reentrant checkpoint's first pass is one); a stack without norm and
        # counter has always taken the pass of inference there, and keeps it
        due = self.training and self.dropout > 0 and (counter or self.norms is not None)
        if not torch.is_grad_enabled() and self.activation is F.relu and not due:
            # inference: bias and ReLU are fused into the store of the gather kernel (with a norm, the ReLU follows that)
            for i, layer in enumerate(self.layers):
                h = layer.forward_fused(h, inputInfo, relu=i < last and self.norms is None)
                if i < last and self.norms is not None:
                    h = self._between(h, i, None, None)
            return h
        if counter and seed is None and self.training and self.dropout > 0:
            seed = N.draw_seed()
        for i, layer in enumerate(self.layers):
            if i and not counter:
                h = F.dropout(h, self.dropout, self.training)
            # the fused pass adds the bias itself
            bare = i < last and counter and self.norms is None and self.activation is F.relu and _stands_alone(layer, ROF_GCNConv)
            h = layer.convolve(h, inputInfo) if bare else layer(h, inputInfo)
            if i == last:
                break
            if counter:
                drop = dict(p=self.dropout, seed=seed, step=step + (i << 40), row_offset=row_offset, training=self.training)
                h = self._between(h, i, layer.bias if bare else None, drop)
            elif self.norms is not None:
                h = self._between(h, i, None, None)
            else:
                h = self.activation(h)
        return h


class SumAggregate(torch.autograd.Function):
    """h -> self_scale * h + A h (sum) or self_scale * h + D^-1 A h (mean) over in-neighbours through an
    AggregationPlan, the self term fused into the store of the gather kernel.  The backward pass runs
    the transposed plan when given one, else the same plan (upstream's convention: exact for a
    symmetric graph).  For mean the gradient is A^T (D^-1 g): g is divided by the forward in-degrees
    first and then summed, never averaged by the degrees again."""

    @staticmethod
    def forward(ctx, h, plan, plan_t, degrees, mode, self_scale=0.0):
        if mode not in ("sum", "mean"):
            raise ValueError("SumAggregate: mode must be 'sum' or 'mean'")
        ctx.plan_t, ctx.degrees, ctx.mode, ctx.self_scale = (plan_t or plan), degrees, mode, self_scale
        h = h.contiguous()
        return plan.aggregate(h, degrees, mode, tiles="auto", self_x=h if self_scale else None,
                              self_scale=self_scale)

    @staticmethod
    def backward(ctx, g):
        g = g.contiguous()
        gs = scale_rows(g, ctx.degrees, "reciprocal") if ctx.mode == "mean" else g
        return (ctx.plan_t.aggregate(gs, None, "sum", tiles="auto", self_x=g if ctx.self_scale else None,
                                     self_scale=ctx.self_scale), None, None, None, None, None)


class ROF_GIN(torch.nn.Module):
    """GIN: h' = MLP((1 + eps) h + sum_{n in N(v)} h_n), 2-layer MLP per layer, eps fixed.  norm="layer" puts a
    layer norm in front of the ReLU between two layers; dropout > 0 a dropout behind it (norm.py, one pass)."""

    def __init__(self, in_feats, n_hidden, n_classes, n_layers=3, eps=0.0, norm=None, dropout=0.0):
        super().__init__()
        if norm not in (None, "layer"):
            raise ValueError("ROF_GIN: norm is None or 'layer'")
        dims = [in_feats] + [n_hidden] * (n_layers - 1) + [n_classes]
        self.mlps = torch.nn.ModuleList(
            torch.nn.Sequential(torch.nn.Linear(a, n_hidden), torch.nn.ReLU(), torch.nn.Linear(n_hidden, b))
            for a, b in zip(dims[:-1], dims[1:]))
        self.eps, self.dropout = eps, dropout
        self.norms = torch.nn.ModuleList(N.LayerNorm(d) for d in dims[1:-1]) if norm is not None else None

    def __setstate__(self, state):
        super().__setstate__({"norms": None, "dropout": 0.0, **state} if "norms" not in state["_modules"] else state)

    def forward(self, features, plan: AggregationPlan, plan_t=None, seed=None, step=0, row_offset=0):
        h = features
        if seed is None and self.training and self.dropout > 0:
            seed = N.draw_seed()
        for i, mlp in enumerate(self.mlps):
            h = mlp(SumAggregate.apply(h, plan, plan_t, None, "sum", 1.0 + self.eps))
            if i + 1 == len(self.mlps):
                break
            drop = dict(p=self.dropout, seed=seed, step=step + (i << 40), row_offset=row_offset, training=self.training)
            done = False
            if self.norms is not None:
                h, done = _norm_relu_dropout(self.norms[i], h, True, drop)
            if done:
                continue
            if self.dropout > 0:
                h = N.dropout(h, relu=True, **drop)
            else:
                h = F.relu(h)
        return h
