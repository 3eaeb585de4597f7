"""The operators between two graph layers: layer norm, dropout, and the two in one pass with the ReLU between
them (include/rof_b200.h: rof_layer_norm_*, rof_dropout_*), with their gradients.

Dropout draws from a counter-based generator: whether element e = (row_offset + row) * width + column of a matrix
stays is a function of (seed, step, e) and nothing else.  So no mask is stored (the backward pass computes it again),
a rank that holds a block of rows drops what a single GPU holding all rows would (`row_offset`), and a run is
repeated by its seed.  `seed` is a number; without one it is drawn from torch's default CPU generator, which
torch.manual_seed and torch.utils.checkpoint control.  `step` is a number or a one-element int64 CUDA tensor that
is read when the kernel runs: a captured graph that adds to it draws anew on every replay.  The backward pass
reads the tensor too: change it after the backward pass only (in eager mode autograd refuses a change in between).
Both passes can be captured into a CUDA graph; as with every torch operation, no eager graph of the same leaves may be
alive meanwhile (torch ties a leaf's gradient to the stream of the graph that lives).

All sums and statistics are held in 32 bits whatever the matrix's type (float32, bfloat16, float16); results
are rounded once and are the same bit for bit on every call.  As everywhere in this package there is no CPU path.
"""
import torch

from . import _native

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _check_matrix(x, name):
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not x.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    if x.dtype not in DTYPES:
        raise RuntimeError(f"{name} must be float32, bfloat16 or float16, got {x.dtype}")
    if x.dim() < 1:
        raise RuntimeError(f"{name} must have at least one dimension")


def _check_vector(v, name, x):
    if not isinstance(v, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if v.get_device() != x.get_device() or v.dim() != 1 or v.size(0) != x.size(-1):
        raise RuntimeError(f"{name} must be a vector of {x.size(-1)} entries on x's device, got {tuple(v.shape)} on {v.device}")
    if v.dtype is not torch.float32 and v.dtype is not x.dtype:
        raise RuntimeError(f"{name} must be float32 or of x's type, got {v.dtype}")


def draw_seed():
    """a seed from torch's default CPU generator; not under capture, where every replay would use the one drawn now"""
    if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("a captured dropout needs a seed: one drawn now would be the same on every replay "
                           "(give `seed`, and a `step` tensor that the graph adds to)")
    return int(torch.empty((), dtype=torch.int64).random_())


def _check_drop(p, seed, step, row_offset, training, x):
    """-> None (nothing is dropped) or (p, seed, step, step tensor or None, row_offset)"""
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p must be in [0, 1], got {p}")
    if not training or p == 0.0:
        return None
    tensor = None
    if isinstance(step, torch.Tensor):
        if step.dtype != torch.int64 or step.numel() != 1 or step.device != x.device:
            raise RuntimeError("step must be a number or a one-element int64 tensor on x's device")
        step, tensor = 0, step
    if seed is None:
        seed = draw_seed()
    for name, v, top in (("seed", seed, 2 ** 64), ("step", step, 2 ** 64), ("row_offset", row_offset, 2 ** 60)):
        if not 0 <= v < top:
            raise ValueError(f"{name} must be in [0, 2**{top.bit_length() - 1}), got {v}")
    return float(p), int(seed), int(step), tensor, int(row_offset)


def _rows(x):
    """x as [rows, width] with unit column stride: a view where its layout allows it, else a copy"""
    v = x if x.dim() == 2 else x.unsqueeze(0) if x.dim() == 1 else x.flatten(0, -2)
    if v.is_contiguous() or ((v.stride(1) == 1 or v.size(1) <= 1) and (v.stride(0) >= v.size(1) or v.size(0) <= 1)):
        return v
    return v.contiguous()


def _laid_like(t, v):
    """t with rows that lie against the 16-byte boundaries like v's: t itself, or a copy.  The backward kernels read both
    matrices in the same 16-byte vectors; a copy costs a third of what they lose on rows that lie differently."""
    per = 16 // t.element_size()
    off, step = v.data_ptr() % 16, v.stride(0) % per
    if t.data_ptr() % 16 == off and (t.stride(0) % per == step or t.size(0) <= 1):
        return t
    rows, width = t.shape
    if rows <= 1:
        step = 0
    ld = width + (step - width) % per
    out = t.new_empty(rows * ld + per).as_strided((rows, width), (ld, 1), off // t.element_size())
    return out.copy_(t)


def _drop_arg(drop, step):
    if drop is None:
        return None
    return _native.Dropout(drop[0], drop[1], drop[2], step.data_ptr() if step is not None else None, drop[4])


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _kind(weight, bias):
    """the one type in which both vectors go down: their own, or 32-bit where they differ"""
    if weight is None or bias is None:
        v = bias if weight is None else weight
        return torch.float32 if v is None else v.dtype
    return weight.dtype if weight.dtype is bias.dtype else torch.float32


def _vector(v, kind):
    if v is None or (v.dtype is kind and v.is_contiguous()):
        return v
    return v.to(kind).contiguous()


def _call(function, x, *args):
    """a C-ABI call that enqueues on the current stream of x's device"""
    index = x.get_device()
    if index == torch.cuda.current_device():
        _native.check(function(*args, torch._C._cuda_getCurrentRawStream(index)))
    else:
        with torch.cuda.device(index):
            _native.check(function(*args, torch._C._cuda_getCurrentRawStream(index)))


def _like(x):
    return torch.empty_like(x) if x.is_contiguous() else torch.empty_like(x, memory_format=torch.contiguous_format)


def _workspace(lib, rows, width, x):
    # torch's caching allocator returns 512-byte aligned blocks
    n = lib.rof_layer_norm_workspace_bytes(rows, width)
    return x.new_empty(n, dtype=torch.uint8), n


def _norm_forward(x, weight, bias, eps, relu, drop, want_stats):
    v = _rows(x)
    rows, width = v.shape
    y = _like(x)
    stats = x.new_empty((rows, 2), dtype=torch.float32) if want_stats else None
    kind = _kind(weight, bias)
    w, b = _vector(weight, kind), _vector(bias, kind)
    _call(_native.cuda().rof_layer_norm_forward, x, DTYPES[x.dtype], v.data_ptr(), v.stride(0), rows, width, DTYPES[kind],
          _ptr(w), _ptr(b), eps, relu, _drop_arg(drop, drop[3] if drop else None), y.data_ptr(), width, _ptr(stats))
    return v, y, stats


def _norm_backward(ctx, grad):
    v, weight, bias, stats, step = ctx.saved_tensors
    relu, drop = ctx.more
    need_x, need_w, need_b, _ = ctx.needs_input_grad
    rows, width = v.shape
    dy = _laid_like(_rows(grad), v)
    dx = _like(grad) if need_x else None
    kind = _kind(weight, bias)
    w, b = _vector(weight, kind), _vector(bias, kind)
    dw = torch.empty_like(w) if need_w else None
    db = torch.empty_like(b) if need_b else None
    lib = _native.cuda()
    ws, n = _workspace(lib, rows, width, v) if need_w or need_b else (None, 0)
    _call(lib.rof_layer_norm_backward, v, DTYPES[v.dtype], dy.data_ptr(), dy.stride(0), v.data_ptr(), v.stride(0), rows, width,
          DTYPES[kind], _ptr(w), _ptr(b), stats.data_ptr(), relu, _drop_arg(drop, step), _ptr(dx), width, _ptr(dw), _ptr(db),
          _ptr(ws), n)
    if need_w and dw.dtype is not weight.dtype:
        dw = dw.to(weight.dtype)
    if need_b and db.dtype is not bias.dtype:
        db = db.to(bias.dtype)
    return dx, dw, db, None


# The wrapper that refuses a second derivative costs 12 us a call: it is only gone through where a graph of the
# gradients is being made (create_graph).
_norm_backward_once = torch.autograd.function.once_differentiable(_norm_backward)


def _without_tensor(drop):
    """what the autograd node keeps of a drop: the step tensor is saved apart, where changes to it are seen"""
    return drop[:3] + (None, drop[4]) if drop is not None else None


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, more):
        eps, relu, drop = more
        v, y, stats = _norm_forward(x, weight, bias, eps, relu, drop, True)
        ctx.save_for_backward(v, weight, bias, stats, drop[3] if drop else None)
        ctx.more = relu, _without_tensor(drop)
        return y

    @staticmethod
    def backward(ctx, grad):
        return _norm_backward_once(ctx, grad) if torch.is_grad_enabled() else _norm_backward(ctx, grad)


def layer_norm(x, weight=None, bias=None, eps=1e-5, relu=False, p=0.0, seed=None, step=0, row_offset=0, training=True):
    """dropout(relu?(layer norm of x over its last dimension)) in one pass, and one back.

    x: a CUDA tensor [..., width] of float32, bfloat16 or float16 with any strides; weight, bias: vectors of `width`
    entries, float32 or of x's type, or None; eps >= 0.  relu: apply the ReLU.  p, seed, step, row_offset: the
    dropout behind it (see `dropout`), only where `training`.  Returns a contiguous tensor like x; gradients flow to x, weight
    and bias (once: a second derivative is not offered)."""
    _check_matrix(x, "x")
    if weight is not None:
        _check_vector(weight, "weight", x)
    if bias is not None:
        _check_vector(bias, "bias", x)
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    drop = _check_drop(p, seed, step, row_offset, training, x)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return _LayerNorm.apply(x, weight, bias, (eps, bool(relu), drop))
    return _norm_forward(x, weight, bias, eps, bool(relu), drop, False)[1]


def _dropout_forward(x, bias, relu, drop):
    v = _rows(x)
    rows, width = v.shape
    y = _like(x)
    kind = torch.float32 if bias is None else bias.dtype
    b = _vector(bias, kind)
    _call(_native.cuda().rof_dropout_forward, x, DTYPES[x.dtype], v.data_ptr(), v.stride(0), rows, width, DTYPES[kind], _ptr(b),
          relu, _drop_arg(drop, drop[3] if drop else None), y.data_ptr(), width)
    return y


def _dropout_backward(ctx, grad):
    y, step = ctx.saved_tensors
    relu, drop, kind = ctx.more
    need_x, need_b, _ = ctx.needs_input_grad
    dy = _rows(grad)
    rows, width = dy.shape
    dx = _like(grad) if need_x else None
    lib = _native.cuda()
    db, (ws, n) = None, (None, 0)
    if need_b:
        dy = _laid_like(dy, _rows(dx) if need_x else _rows(y) if relu else dy)
        db = dy.new_empty(width, dtype=kind)
        ws, n = _workspace(lib, rows, width, dy)
    _call(lib.rof_dropout_backward, dy, DTYPES[dy.dtype], dy.data_ptr(), dy.stride(0), _ptr(y), width, rows, width, DTYPES[kind],
          relu, _drop_arg(drop, step), _ptr(dx), width, _ptr(db), _ptr(ws), n)
    return dx, db, None


_dropout_backward_once = torch.autograd.function.once_differentiable(_dropout_backward)


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, bias, more):
        relu, drop = more
        y = _dropout_forward(x, bias, relu, drop)
        # behind a ReLU the output says which elements were kept and positive
        ctx.save_for_backward(y if relu else None, drop[3] if drop else None)
        ctx.more = relu, _without_tensor(drop), bias.dtype if bias is not None else torch.float32
        return y

    @staticmethod
    def backward(ctx, grad):
        return _dropout_backward_once(ctx, grad) if torch.is_grad_enabled() else _dropout_backward(ctx, grad)


def dropout(x, p=0.0, seed=None, step=0, row_offset=0, training=True, bias=None, relu=False):
    """dropout(relu?(x + bias)) in one pass, and one back.

    x: a CUDA tensor [..., width] of float32, bfloat16 or float16 with any strides; bias: a vector of `width` entries,
    float32 or of x's type, or None.  Each element is zeroed with probability p and scaled by 1 / (1 - p) otherwise, only where
    `training`; p = 1 zeroes everything.  The choice depends on (seed, step, element index) alone, the index counted from
    row `row_offset` of the whole matrix.  Returns a contiguous tensor like x."""
    _check_matrix(x, "x")
    if bias is not None:
        _check_vector(bias, "bias", x)
    drop = _check_drop(p, seed, step, row_offset, training, x)
    if torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad)):
        return _Dropout.apply(x, bias, (bool(relu), drop))
    return _dropout_forward(x, bias, bool(relu), drop)


class LayerNorm(torch.nn.Module):
    """layer_norm() with its weight and bias; relu and p: the ReLU and the dropout behind it, in the same pass."""

    def __init__(self, width, eps=1e-5, bias=True, relu=False, p=0.0):
        super().__init__()
        self.width, self.eps, self.relu, self.p = width, eps, relu, p
        self.weight = torch.nn.Parameter(torch.ones(width))
        if bias:
            self.bias = torch.nn.Parameter(torch.zeros(width))
        else:
            self.register_parameter("bias", None)

    def reset_parameters(self):
        torch.nn.init.ones_(self.weight)
        if self.bias is not None:
            torch.nn.init.zeros_(self.bias)

    def forward(self, x, seed=None, step=0, row_offset=0):
        return layer_norm(x, self.weight, self.bias, self.eps, self.relu, self.p, seed, step, row_offset, self.training)

    def extra_repr(self):
        return f"{self.width}, eps={self.eps}, bias={self.bias is not None}, relu={self.relu}, p={self.p}"


class Dropout(torch.nn.Module):
    """dropout() as a module"""

    def __init__(self, p=0.5, relu=False):
        super().__init__()
        self.p, self.relu = p, relu

    def forward(self, x, seed=None, step=0, row_offset=0, bias=None):
        return dropout(x, self.p, seed, step, row_offset, self.training, bias, self.relu)

    def extra_repr(self):
        return f"p={self.p}, relu={self.relu}"
