"""``torch.nn`` layers on top of the fused kernels, with the reference's rank-from-compression-rate rules.

The reference builds its layers with ``conv2d_tensor`` / ``dense_tensor`` (test/layers.py:63-101,147-175): a
compression ``rate`` is turned into a CP rank by ``generate_params_*`` (pure integer arithmetic, restated here),
factor variables are created, and the layer is the sequential or the fused op.  These modules keep that
interface for the three CP layer families of the hot path; weights live in the layout the C ABI takes
(``[dim, R]`` factors for CP4, ``[c_k, t_k, R]`` for rCP, ``[i_k, o_k, R]`` for the dense layer).  Beside them stand
``AdaptedDense`` (a shared projection with low-rank adapters per request), ``GatedDense`` (the gated half of a feed-forward block), ``Embedding`` and
``LayerNorm`` (what is before and between such blocks).
"""
from __future__ import annotations

import math

import torch
from torch import nn

_ops_module = None


def _ops():
    """The operators, loaded with the library at the first forward (the rank rules need neither)."""
    global _ops_module
    if _ops_module is None:
        from . import ops
        _ops_module = ops
    return _ops_module


DEFAULT_COMPRESSION_RATE = 0.1        # test/layers.py:16
DEFAULT_FACTORIZATION_BASE = 16       # test/layers.py:17


def generate_shape(number, order=None, base=None, reverse=False):
    """Mode sizes of a power of two ``number = 2**e``, the rule of the reference's ``generate_shape``
    (test/layers.py:22-48), stated on the exponents.

    ``base = 2**b``: ``e = q*b + s`` gives ``q`` modes of size ``base``; the left-over ``2**s`` becomes a mode of its
    own when it is at least ``sqrt(base)`` (``2*s >= b``) or when there is no other mode, else it is folded into the
    first mode.  ``order``: the ``e`` twos are dealt to ``order`` modes in turn, so the first ``e % order`` modes get
    one more.  ``reverse`` flips the list.
    """
    if number <= 0 or number & (number - 1):
        raise ValueError("generate_shape supports powers of two only")
    if (order is None) == (base is None):
        raise ValueError("give either order or base")
    e = number.bit_length() - 1
    if order is not None:
        shape = [1 << (e // order + (1 if k < e % order else 0)) for k in range(order)]
    else:
        if base < 2 or base & (base - 1):
            raise ValueError("base must be a power of two")
        b = base.bit_length() - 1
        q, s = divmod(e, b)
        shape = [base] * q
        if q == 0 or 2 * s >= b:
            shape.append(1 << s)
        else:
            shape[0] <<= s
    return shape[::-1] if reverse else shape


def params_conv2d_cp4(in_channels, out_channels, kernel_size, rate=DEFAULT_COMPRESSION_RATE):
    """Rank of the four-factor CP conv: the rule of ``generate_params_conv2d_cp`` (test/layers.py:296-304) with the
    spatial factor counted as two separable vectors (2k parameters per rank instead of k*k)."""
    original = kernel_size * kernel_size * in_channels * out_channels
    unit = 2 * kernel_size + in_channels + out_channels
    return {"rank": int(math.ceil(rate * original / unit))}


def params_conv2d_cp(in_channels, out_channels, kernel_size, rate=DEFAULT_COMPRESSION_RATE):
    """``generate_params_conv2d_cp`` (test/layers.py:296-304): the three-factor CP conv, k*k + C + T parameters per rank."""
    original = kernel_size * kernel_size * in_channels * out_channels
    unit = kernel_size * kernel_size + in_channels + out_channels
    return {"rank": int(math.ceil(rate * original / unit))}


def params_conv2d_rcp(in_channels, out_channels, kernel_size, rate=DEFAULT_COMPRESSION_RATE, order=2):
    """``generate_params_conv2d_rcp`` (test/layers.py:816-851); the reference fixes ``order = 2``."""
    ishape = generate_shape(in_channels, order=order)
    oshape = generate_shape(out_channels, order=order)
    original = kernel_size ** 2 * in_channels * out_channels
    unit = (2 * kernel_size if kernel_size > 1 else 0) + sum(ishape) + sum(oshape)
    return {"input_shape": ishape, "output_shape": oshape, "rank": int(math.ceil(rate * original / unit))}


def params_dense_cp(in_features, out_features, rate=DEFAULT_COMPRESSION_RATE):
    """``generate_params_dense_cp`` (test/layers.py:491-507)."""
    ishape = generate_shape(in_features, base=DEFAULT_FACTORIZATION_BASE)
    if len(ishape) < 2:
        raise ValueError("in_features is too small to be factorized further")
    oshape = generate_shape(out_features, order=len(ishape), reverse=True)
    unit = sum(i * o for i, o in zip(ishape, oshape))
    return {"input_shape": ishape, "output_shape": oshape,
            "rank": int(math.ceil(in_features * out_features * rate / unit))}


class CP4Conv2d(nn.Module):
    """Rank-R CP4 conv2d, stride 1, same padding: ``K[t,c,y,x] = sum_r FT[t,r] FC[c,r] FY[y,r] FX[x,r]``
    (Cuda_kernels/Utils.cu:51-62) without ever forming ``K``."""

    def __init__(self, in_channels, out_channels, kernel_size=3, rank=None, rate=DEFAULT_COMPRESSION_RATE, bias=False,
                 flags=0):
        super().__init__()
        if kernel_size % 2 == 0:
            raise ValueError("same padding needs an odd kernel size")
        self.rank = rank or params_conv2d_cp4(in_channels, out_channels, kernel_size, rate)["rank"]
        self.pad, self.flags = (kernel_size - 1) // 2, flags
        # every factor gets the fourth root of the variance a dense filter of this fan-in would have per rank term
        std4 = (1.0 / (in_channels * kernel_size * kernel_size * self.rank)) ** 0.125
        mk = lambda d: nn.Parameter(torch.randn(d, self.rank) * std4)
        self.FT, self.FC, self.FY, self.FX = mk(out_channels), mk(in_channels), mk(kernel_size), mk(kernel_size)
        self.bias = nn.Parameter(torch.zeros(out_channels)) if bias else None

    def forward(self, x):
        y = _ops().CP4Conv2dFunction.apply(x.contiguous(), self.FT, self.FC, self.FY, self.FX, self.pad, self.flags)
        return y if self.bias is None else y + self.bias.view(1, -1, 1, 1)


class CPConv2d(nn.Module):
    """Three-factor CP conv2d, the layer ``conv2d_cp`` defines (test/layers.py:265-291): 1x1 conv C->R, per-rank k x k
    filter, 1x1 conv R->T, as one fused kernel; stride 1, same padding.  Training needs a 3x3 filter."""

    def __init__(self, in_channels, out_channels, kernel_size=3, rank=None, rate=DEFAULT_COMPRESSION_RATE, bias=False):
        super().__init__()
        if kernel_size % 2 == 0:
            raise ValueError("same padding needs an odd kernel size")
        self.rank = rank or params_conv2d_cp(in_channels, out_channels, kernel_size, rate)["rank"]
        self.pad = (kernel_size - 1) // 2
        std3 = (1.0 / (in_channels * kernel_size * kernel_size * self.rank)) ** (1.0 / 6.0)
        self.KT = nn.Parameter(torch.randn(out_channels, self.rank) * std3)
        self.KCin = nn.Parameter(torch.randn(in_channels, self.rank) * std3)
        self.KC = nn.Parameter(torch.randn(kernel_size, kernel_size, self.rank) * std3)
        self.bias = nn.Parameter(torch.zeros(out_channels)) if bias else None

    def forward(self, x):
        y = _ops().CP3Conv2dFunction.apply(x.contiguous(), self.KT, self.KCin, self.KC, self.pad)
        return y if self.bias is None else y + self.bias.view(1, -1, 1, 1)


class RCPConv2d(nn.Module):
    """Reshaped-CP conv2d (test/layers.py:687-789): channels factored into modes, one ``[c_k, t_k, R]`` factor per
    mode and a ``[k, k, R]`` spatial core; stride 1, same padding."""

    def __init__(self, in_channels, out_channels, kernel_size=3, rank=None, rate=DEFAULT_COMPRESSION_RATE,
                 input_shape=None, output_shape=None, bias=False):
        super().__init__()
        p = params_conv2d_rcp(in_channels, out_channels, kernel_size, rate)
        self.input_shape = list(input_shape or p["input_shape"])
        self.output_shape = list(output_shape or p["output_shape"])
        if math.prod(self.input_shape) != in_channels or math.prod(self.output_shape) != out_channels:
            raise ValueError("mode sizes must multiply to the channel counts")
        if len(self.input_shape) != len(self.output_shape):
            raise ValueError("input_shape and output_shape need the same number of modes")
        self.rank = rank or p["rank"]
        m = len(self.input_shape)
        std = (1.0 / (in_channels * kernel_size * kernel_size * self.rank)) ** (0.5 / (m + 1))
        self.factors = nn.ParameterList([nn.Parameter(torch.randn(c, t, self.rank) * std)
                                         for c, t in zip(self.input_shape, self.output_shape)])
        self.core = nn.Parameter(torch.randn(kernel_size, kernel_size, self.rank) * std)
        self.bias = nn.Parameter(torch.zeros(out_channels)) if bias else None

    def forward(self, x):
        y = _ops().RCPConv2dFunction.apply(x.contiguous(), self.core, *self.factors)
        return y if self.bias is None else y + self.bias.view(1, -1, 1, 1)


class CPDense(nn.Module):
    """CP dense layer (test/layers.py:430-469): ``W[i, o] = sum_r prod_k F_k[i_k, o_k, r]`` without forming ``W``."""

    def __init__(self, in_features, out_features, rank=None, rate=DEFAULT_COMPRESSION_RATE, input_shape=None,
                 output_shape=None, bias=False):
        super().__init__()
        if input_shape is None or output_shape is None:
            p = params_dense_cp(in_features, out_features, rate)
            input_shape, output_shape = p["input_shape"], p["output_shape"]
            rank = rank or p["rank"]
        self.input_shape, self.output_shape = list(input_shape), list(output_shape)
        if math.prod(self.input_shape) != in_features or math.prod(self.output_shape) != out_features:
            raise ValueError("mode sizes must multiply to the feature counts")
        if rank is None:
            rank = params_dense_cp(in_features, out_features, rate)["rank"]
        self.rank = rank
        m = len(self.input_shape)
        std = (1.0 / (in_features * self.rank)) ** (0.5 / m)
        self.factors = nn.ParameterList([nn.Parameter(torch.randn(i, o, self.rank) * std)
                                         for i, o in zip(self.input_shape, self.output_shape)])
        self.bias = nn.Parameter(torch.zeros(out_features)) if bias else None

    def forward(self, x):
        if x.dim() == 2:
            y = _ops().CPDenseFunction.apply(x.contiguous(), *self.factors)
        else:
            y = _ops().CPDenseFunction.apply(x.reshape(-1, x.shape[-1]).contiguous(), *self.factors).reshape(*x.shape[:-1], -1)
        return y if self.bias is None else y + self.bias


class AdaptedDense(nn.Module):
    """A shared projection with one low-rank adapter per request: ``shared(x) + scale[a] (x A[a]) B[a]`` for rows of adapter ``a``.

    ``shared``: a ``CPDense`` or any module ``[..., in_features] -> [..., out_features]``; its parameters are frozen unless ``freeze=False``.  ``count``
    adapters of rank ``rank`` start at zero (``B`` is zero), in the type of ``dtype`` (the shared layer's).  ``forward(x, adapters)``: ``adapters``
    holds the adapter of each row (any number outside ``0 .. count - 1``: none), or is an ``ops.AdapterPlan`` that all layers of a batch share."""

    def __init__(self, shared, count, rank, in_features=None, out_features=None, scale=1.0, freeze=True, dtype=None):
        super().__init__()
        if isinstance(shared, CPDense):
            in_features, out_features = math.prod(shared.input_shape), math.prod(shared.output_shape)
        in_features = in_features or getattr(shared, "in_features", None)
        out_features = out_features or getattr(shared, "out_features", None)
        if not in_features or not out_features:
            raise ValueError("in_features and out_features of the shared projection are needed")
        if count < 1 or not 1 <= rank <= 128:
            raise ValueError("at least one adapter, of a rank of 1 to 128")
        self.shared = shared
        if freeze:
            for p in shared.parameters():
                p.requires_grad_(False)
        if dtype is None:
            dtype = next((p.dtype for p in shared.parameters()), torch.float32)
        self.A = nn.Parameter((torch.randn(count, in_features, rank) * in_features ** -0.5).to(dtype))
        self.B = nn.Parameter(torch.zeros(count, rank, out_features, dtype=dtype))
        self.register_buffer("scale", torch.full((count,), float(scale), dtype=torch.float32))

    def _apply(self, fn, recurse=True):
        scale = self.scale
        super()._apply(fn, recurse)
        if self.scale.dtype != torch.float32:   # a type given to the module is that of the adapters; the scales stay as they are, in float32
            self.scale = scale.to(self.scale.device)
        return self

    def forward(self, x, adapters):
        return _ops().DenseAdaptersFunction.apply(self.shared(x), x, self.A, self.B, adapters, self.scale)


class GatedDense(nn.Module):
    """The gated half of a feed-forward block, ``act(x Wg) * (x Wu)`` as one kernel; bfloat16 or float16.  What follows it is any dense layer
    (``CPDense`` in float32, or a product of its own type)."""

    def __init__(self, in_features, hidden_features, activation="silu", dtype=torch.bfloat16):
        super().__init__()
        if activation not in ("silu", "gelu", "gelu_tanh"):
            raise ValueError("activation is silu, gelu or gelu_tanh")
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("dtype is bfloat16 or float16")
        self.activation = activation
        make = lambda: nn.Parameter((torch.randn(in_features, hidden_features) * in_features ** -0.5).to(dtype))  # noqa: E731
        self.Wg, self.Wu = make(), make()

    def forward(self, x):
        return _ops().DenseGatedFunction.apply(x, self.Wg, self.Wu, self.activation)


class Embedding(nn.Module):
    """Rows of a table by token, times ``scale``; a token outside ``0 .. count - 1`` is none (padding): zeros, and no gradient.  The table's gradient is dense and
    its sums are in a fixed order.  float32, bfloat16 or float16."""

    def __init__(self, count, features, scale=1.0, dtype=torch.float32):
        super().__init__()
        if count < 1 or features < 1:
            raise ValueError("at least one token and one feature")
        if dtype not in (torch.float32, torch.bfloat16, torch.float16):
            raise ValueError("dtype is float32, bfloat16 or float16")
        self.scale = float(scale)
        self.W = nn.Parameter((torch.randn(count, features) / abs(self.scale or 1.0)).to(dtype))

    def forward(self, tokens):
        return _ops().EmbeddingFunction.apply(tokens, self.W, self.scale)


class LayerNorm(nn.Module):
    """Layer norm over the last dimension.  ``forward(x)`` gives ``norm(x)``; ``forward(x, residual)`` gives ``(norm(h), h)`` with ``h = x + residual`` in the same pass:
    a block's output joins the stream, and the next block gets its input.  ``weight`` and ``bias`` (``affine=False``: neither, ``bias=False``: no bias) are float32 or of the rows' type."""

    def __init__(self, features, eps=1e-5, affine=True, bias=True, dtype=torch.float32):
        super().__init__()
        if features < 1 or not eps >= 0:
            raise ValueError("at least one feature, and eps may not be negative")
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(features, dtype=dtype)) if affine else None
        self.bias = nn.Parameter(torch.zeros(features, dtype=dtype)) if affine and bias else None

    def forward(self, x, residual=None):
        return _ops().LayerNormFunction.apply(x, self.weight, self.bias, self.eps, residual)
