"""Operators and layers of a head behind the distance layers: layer norm, dropout whose mask is never stored, both joined on a
residual stream, and the matrix product in 8-bit integers that the head answers with.  The reference has none of them (its head
is linear, tanh, linear; core/modules/basic_modules.py:11-46).

Rows are the last dimension of a float32, float16 or bfloat16 CUDA tensor; a norm's weight and bias are float32 or of that type.
Statistics, sums and gradients' sums have 32 bits whatever the type, and results are rounded once.  Launches go to PyTorch's
current stream.  There is no other path: arguments that do not fit raise RuntimeError before anything is launched, and so do
function transforms, torch.compile and the tracer, which would not see the kernels.
"""
import torch
import torch.distributed as dist
import torch.nn as nn

from . import norm_dist_cuda as _C

__all__ = ["layer_norm", "dropout", "dropout_add_layer_norm", "quantize_rows", "layer_norm_quantized", "int8_linear", "LayerNorm",
           "Dropout", "Int8Linear", "ResidualHead", "QuantizedHead"]

_ACTIVATIONS = {"none": 0, "relu": 1, "tanh": 2}


def _native():
    ext = _C.native()
    if ext is None:
        raise RuntimeError("the head's operators need the compiled binding (python l_inf_dist_net_v2_b200/build.py) and run under no "
                           "function transform and not in torch.compile")
    return ext


def _draw(seed, offset):
    """(seed, offset, device words) as the binding takes them: 64 bits as Python's integers have them, signed."""
    if isinstance(seed, torch.Tensor):
        return 0, _signed(offset), seed
    return _signed(seed), _signed(offset), None


def _signed(v):
    if not 0 <= v < 1 << 64:
        raise ValueError("seed and offset are unsigned 64-bit numbers")
    return v - (1 << 64) if v >= 1 << 63 else v


def _padded(terms):
    """The distance of rows of integers that start at multiples of 16 bytes."""
    return (terms + 15) // 16 * 16


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension; gradients of x, weight and bias."""
    return _native().layer_norm(x, weight, bias, eps)


def dropout(x, p, seed, offset=0, residual=None):
    """[residual +] x / (1 - p) where an element is kept, 0 elsewhere.

    Element i (in the order of a contiguous tensor) is kept if word i % 4 of Philox4x32-10 with key `seed` and counter
    (i // 4, offset) is at least round(p * 2^32): the same seed, offset and shape give the same mask, on any device and in the
    backward pass.  `seed` may be a CUDA tensor of two int64 values, a seed and an offset that is added to `offset`: a recorded
    graph then draws what the tensor holds when it is replayed.
    """
    s, o, state = _draw(seed, offset)
    return _native().dropout(x, p, s, o, state, residual)


def dropout_add_layer_norm(x, residual, weight, bias, p, seed, offset=0, eps=1e-5):
    """(y, h): h = residual + dropout(x), in the type of x, and y = layer_norm(h), in one kernel each way."""
    s, o, state = _draw(seed, offset)
    return _native().dropout_add_layer_norm(x, residual, weight, bias, p, s, o, state, eps)


def quantize_rows(x):
    """(q, scale): scale = max(largest |x| of a row / 127, 2^-126), q = round(x / scale) as int8 whose rows start at multiples of 16
    bytes (what the integer product reads fastest).  A row with a value that is not finite answers with values that are not numbers."""
    return _native().quantize_rows(x)


def layer_norm_quantized(x, weight=None, bias=None, eps=1e-5):
    """quantize_rows(layer_norm(x)) without the norm's result in memory, and without its rounding."""
    return _native().layer_norm_quantized(x, weight, bias, eps)


def int8_linear(x, weight, bias=None, activation="none", out_dtype=None):
    """act(x @ weight.T + bias) in 8-bit integers, the sums exact: `weight` is the (q, scale) that `quantize_rows` gives of an
    (outputs, terms) weight; `x` is a tensor, quantised here, or such a pair.  activation: "none", "relu" or "tanh".  The result
    has the type of x (float32 for a pair) or out_dtype.  No gradient."""
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(_ACTIVATIONS)}, not {activation!r}")
    x, x_scale = (x, None) if isinstance(x, torch.Tensor) else x
    return _native().int8_linear(x, x_scale, weight[0], weight[1], bias, _ACTIVATIONS[activation], out_dtype)


class LayerNorm(nn.Module):
    def __init__(self, features, eps=1e-5, affine=True):
        super().__init__()
        self.features = features
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(features)) if affine else None
        self.bias = nn.Parameter(torch.zeros(features)) if affine else None

    def forward(self, x, residual=None, p=0.0, seed=0, offset=0):
        """The norm of x; with a residual (y, h) of `dropout_add_layer_norm`.  (Either is a call of the layer that has the parameters,
        as hooks on layers have to see: the data-parallel wrapper updates a layer in front of its call.)"""
        if residual is None:
            return layer_norm(x, self.weight, self.bias, self.eps)
        return dropout_add_layer_norm(x, residual, self.weight, self.bias, p, seed, offset, self.eps)

    def extra_repr(self):
        return f"{self.features}, eps={self.eps}, affine={self.weight is not None}"


class Dropout(nn.Module):
    """Dropout with a seed of its own (from torch's generator where none is given) and the number of calls so far as the offset, so
    that every call draws another mask; both are in the state_dict.  In a process group the ranks' offsets are 2^40 apart, so that ranks
    with one seed, as after loading one checkpoint, draw masks of their own.  In eval mode the identity.

    A call that torch.utils.checkpoint makes again in a backward pass draws the mask that it drew before: every call takes a number
    from torch's generator on the host, which the recomputation finds in the state that it had, and by it the layer knows its last
    4096 calls."""

    REMEMBERED = 4096

    def __init__(self, p=0.1, seed=None):
        super().__init__()
        if not 0 <= p <= 1:
            raise ValueError("p must be a probability")
        self.p = p
        self.seed = self._number() if seed is None else seed
        self.calls = 0
        self._offsets = {}  # of the last calls, by their numbers, and whether a backward pass has repeated them

    @staticmethod
    def _number():
        return int(torch.randint(1 << 62, (), device="cpu"))

    def draw(self):
        """(seed, offset) of a call."""
        number = self._number()
        known, repeated = self._offsets.pop(number, (None, True))
        if torch._C._current_graph_task_id() != -1:  # (in a backward pass)
            if known is None:
                raise RuntimeError("dropout in a backward pass does not find the call that it repeats: recomputation has to keep the "
                                   "generator's state (preserve_rng_state=True), to come within the layer's next 4096 calls, and to "
                                   "find no two calls of the layer with the generator in the same state")
            self._offsets[number] = (known, True)
            return self.seed, known
        rank = dist.get_rank() if dist.is_available() and dist.is_initialized() else 0
        offset = self.calls + (rank << 40)
        # (a program that seeds the generator anew for every step has the number again: the call before has been repeated, or it is
        # not known which of the two would be)
        self._offsets[number] = (offset if repeated else None, False)
        self.calls += 1
        if len(self._offsets) > self.REMEMBERED:
            del self._offsets[next(iter(self._offsets))]
        return self.seed, offset

    def get_extra_state(self):
        return dict(seed=self.seed, calls=self.calls)

    def set_extra_state(self, state):
        self.seed, self.calls = state["seed"], state["calls"]

    def forward(self, x, residual=None):
        if not self.training or self.p == 0:
            return x if residual is None else residual + x
        seed, offset = self.draw()
        return dropout(x, self.p, seed, offset, residual)

    def extra_repr(self):
        return f"p={self.p}"


class _Answers(nn.Module):
    """A module whose buffers of floating point have 32 bits wherever it is moved: the kernels take no other."""

    def _apply(self, fn, recurse=True):
        before = {name: t for name, t in self._buffers.items() if t is not None and t.is_floating_point()}
        super()._apply(fn, recurse)
        for name, t in before.items():
            self._buffers[name] = t.to(self._buffers[name].device)
        return self


class Int8Linear(_Answers):
    """A linear layer that answers in 8-bit integers: weight (outputs, terms) with a scale per output, rows quantised as they come.
    Wherever it is moved its rows start at multiples of 16 bytes, and scales and bias have 32 bits."""

    def __init__(self, weight, bias=None, activation="none"):
        super().__init__()
        if activation not in _ACTIVATIONS:
            raise ValueError(f"activation must be one of {sorted(_ACTIVATIONS)}, not {activation!r}")
        with torch.no_grad():
            q, scale = quantize_rows(weight)
        self.register_buffer("weight", q)
        self.register_buffer("weight_scale", scale)
        self.register_buffer("bias", None if bias is None else bias.detach().float().clone())
        self.activation = activation

    def _apply(self, fn, recurse=True):
        super()._apply(fn, recurse)
        rows, terms = self.weight.shape
        if self.weight.stride() != (_padded(terms), 1):  # (a copy of rows that are apart leaves them side by side)
            self.weight = self.weight.new_zeros(rows, _padded(terms))[:, :terms].copy_(self.weight)
        return self

    @classmethod
    def from_linear(cls, linear, activation="none"):
        """Of torch's linear layer, or of one of this package's with their scales."""
        w_scale, b_scale = getattr(linear, "w_scale", 1.0), getattr(linear, "b_scale", 1.0)
        bias = None if linear.bias is None else linear.bias.detach() * b_scale
        return cls(linear.weight.detach() * w_scale, bias, activation)

    def forward(self, x, out_dtype=None):
        return int8_linear(x, (self.weight, self.weight_scale), self.bias, self.activation, out_dtype)

    def extra_repr(self):
        return f"{self.weight.size(1)}, {self.weight.size(0)}, bias={self.bias is not None}, activation={self.activation}"


class ResidualHead(nn.Module):
    """A pre-norm residual feed-forward head: every block adds dropout(down(relu(up(norm(h))))) to the stream h, and the classes are a
    linear map of the last norm.  Between the products of neighbouring blocks there is one kernel each way: dropout, residual and the
    next block's norm.  It has no interval bounds, so what it answers is not certified.

    The stream has the type of the head's weights (features of distance layers have 32 bits, a head may have 16), under torch.autocast
    too, where the products may give another."""

    def __init__(self, width, hidden, num_classes=10, blocks=2, dropout=0.1, eps=1e-5, seed=None):
        super().__init__()
        self.up = nn.ModuleList(nn.Linear(width, hidden) for _ in range(blocks))
        self.down = nn.ModuleList(nn.Linear(hidden, width) for _ in range(blocks))
        self.norm = nn.ModuleList(LayerNorm(width, eps) for _ in range(blocks + 1))
        self.drop = nn.ModuleList(Dropout(dropout, None if seed is None else seed + i) for i in range(blocks))
        self.final = nn.Linear(width, num_classes)

    def forward(self, h):
        h = h.to(self.final.weight.dtype)
        y = self.norm[0](h)
        for up, down, norm, drop in zip(self.up, self.down, self.norm[1:], self.drop):
            p, (seed, offset) = (drop.p, drop.draw()) if self.training else (0.0, (0, 0))
            y, h = norm(down(torch.relu(up(y))).to(h.dtype), h, p, seed, offset)
        return self.final(y)

    def quantized(self):
        """The head as it answers in 8-bit integers, from the weights as they are now."""
        return QuantizedHead(self)


class QuantizedHead(_Answers):
    """A residual head whose products are in 8-bit integers: the norms' rows leave as integers, hidden rows are quantised in the product
    that takes them.  It answers only; the stream has the type that it comes in."""

    def __init__(self, head):
        super().__init__()
        self.eps = head.norm[0].eps
        self.up = nn.ModuleList(Int8Linear.from_linear(m, "relu") for m in head.up)
        self.down = nn.ModuleList(Int8Linear.from_linear(m) for m in head.down)
        self.final = Int8Linear.from_linear(head.final)
        for i, m in enumerate(head.norm):
            # (in 32 bits, which go with rows of any type)
            self.register_buffer(f"norm_weight{i}", m.weight.detach().float().clone())
            self.register_buffer(f"norm_bias{i}", m.bias.detach().float().clone())

    def _normed(self, i, h):
        return layer_norm_quantized(h, getattr(self, f"norm_weight{i}"), getattr(self, f"norm_bias{i}"), self.eps)

    @torch.no_grad()
    def forward(self, h):
        for i, (up, down) in enumerate(zip(self.up, self.down)):
            h = h + down(up(self._normed(i, h), out_dtype=h.dtype))
        return self.final(self._normed(len(self.up), h), out_dtype=h.dtype)
