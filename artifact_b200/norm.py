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

Argument checks, memory and the autograd nodes are csrc/torch/norm_torch.cpp.  All sums and statistics are held in 32 bits whatever the matrix's type (float32, bfloat16, float16); results
are rounded once and are the same bit for bit on every call.  As everywhere in this package there is no CPU path.
"""
import torch

from . import _native


def draw_seed():
    """a seed from torch's default CPU generator; not under capture, where every replay would use the one drawn now"""
    if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("a captured dropout needs a seed: one drawn now would be the same on every replay "
                           "(give `seed`, and a `step` tensor that the graph adds to)")
    return int(torch.empty((), dtype=torch.int64, device="cpu").random_())


def _drop_args(p, seed, step, row_offset, training):
    """the generator's arguments as the native operators take them: p, seed, step, row_offset, step tensor"""
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p must be in [0, 1], got {p}")
    if p == 0.0 or not training:
        return 0.0, 0, 0, 0, None
    tensor = None
    if isinstance(step, torch.Tensor):
        step, tensor = 0, step
    if seed is None:
        seed = draw_seed()
    if not (0 <= seed < 2 ** 64 and 0 <= step < 2 ** 64 and 0 <= row_offset < 2 ** 60):
        raise ValueError(f"seed and step must be in [0, 2**64) and row_offset in [0, 2**60), got {seed}, {step}, {row_offset}")
    return float(p), int(seed), int(step), int(row_offset), tensor


def layer_norm(x, weight=None, bias=None, eps=1e-5, relu=False, p=0.0, seed=None, step=0, row_offset=0, training=True):
    """dropout(relu?(layer norm of x over its last dimension)) in one pass, and one back.

    x: a CUDA tensor [..., width] of float32, bfloat16 or float16 with any strides; weight, bias: vectors of `width`
    entries, float32 or of x's type, or None; eps >= 0.  relu: apply the ReLU.  p, seed, step, row_offset: the
    dropout behind it (see `dropout`), only where `training`.  Returns a contiguous tensor like x; gradients flow to x, weight
    and bias (once: a second derivative is not offered, nor are forward-mode derivatives and torch.jit.trace; all are refused)."""
    return _native.torch_ops().layer_norm(x, weight, bias, eps, bool(relu), *_drop_args(p, seed, step, row_offset, training))


def dropout(x, p=0.0, seed=None, step=0, row_offset=0, training=True, bias=None, relu=False):
    """dropout(relu?(x + bias)) in one pass, and one back.

    x: a CUDA tensor [..., width] of float32, bfloat16 or float16 with any strides; bias: a vector of `width` entries,
    float32 or of x's type, or None.  Each element is zeroed with probability p and scaled by 1 / (1 - p) otherwise, only where
    `training`; p = 1 zeroes everything.  The choice depends on (seed, step, element index) alone, the index counted from
    row `row_offset` of the whole matrix.  Returns a contiguous tensor like x.  Behind the ReLU a positive sum that rounds to zero
    (16-bit x beside a float32 bias) is returned as -0: its gradient is not zero, and the backward pass reads that from the output."""
    return _native.torch_ops().dropout(x, bias, bool(relu), *_drop_args(p, seed, step, row_offset, training))


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
