"""What stands around the routed layers of a model: a norm in front of each, the embedding in front of the first.

    layer_norm(x, weight, bias, eps)             (x - mean) / sqrt(var + eps) * weight + bias over the last dimension   (autograd)
    rms_norm(x, weight, eps, residual)           h / sqrt(mean(h^2) + eps) * weight, h = x + residual                  (autograd)
    rms_norm_fp8(x, weight, eps, residual, ...)  the same in 8 bits, by the tensor's scale or one for every row
    embedding(ids, weight, scale, padding_idx)   scale * weight[ids]                                                   (autograd)

and the modules ``LayerNorm``, ``RMSNorm`` and ``Embedding`` that own their parameters.  The reference's users take these from torch;
here they are kernels of this package's library (csrc/layer_norm.hip, csrc/rms_norm.hip, csrc/embedding.hip) with a host path in
native code (csrc/host_layers.cpp).  Rows are bfloat16, float16 or float32; statistics and sums are kept in float32, a result is
rounded once, and gradients are the same bits from call to call.  A routed layer norms its own rows with ``layer_norm=True`` or
``rms_norm=True`` (:mod:`fp8_gmm_amd.moe`).

Autocast is not looked at: a call computes in the types of its tensors, as the grouped modules do.  Gradients can be taken once;
forward-mode differentiation (under ``no_grad`` too, where torch keeps tangents), ``torch.func`` transforms and tracing are refused.
"""
import torch

from . import native


def layer_norm(x, weight, bias=None, eps=1e-5):
    """Layer norm of ``x [..., columns]`` over its last dimension.  ``weight`` and ``bias`` (may be None) ``[columns]``, of the
    type of ``x`` or float32; the result has the type of ``x`` and is contiguous.  Rows may be strided as long as the columns
    are neighbours; others are copied first.  Differentiable in all three; a row whose variance is zero has ``rstd = 1 /
    sqrt(eps)``, one whose sum or squares pass float32's range is no number or its bias, and the rows of an empty ``x`` leave
    gradients of zeros."""
    return native.layer_norm(x, weight, bias, eps)


def rms_norm(x, weight, eps=1e-5, residual=None):
    """Root-mean-square norm of ``x [..., columns]`` over its last dimension: ``x / sqrt(mean(x^2) + eps) * weight``.  ``weight
    [columns]``, of the type of ``x`` or float32.  With ``residual`` (of the shape and type of ``x``) the norm is that of ``h = x +
    residual``, rounded to their type, and the call returns ``(y, h)``: ``h`` is the residual stream that goes on.  Results are
    contiguous.  Rows may be strided as long as the columns are neighbours; others are copied first.  Differentiable in all three:
    ``h`` is kept for the backward pass, so it may not be changed in place before that.  A row of zeros with an ``eps`` of 0 is no
    number, one whose squares pass float32's range is normed to zeros, and the rows of an empty ``x`` leave gradients of zeros."""
    return native.rms_norm(x, weight, eps, residual)


def rms_norm_fp8(x, weight, eps=1e-5, residual=None, scale=None, amax=None, dtype=torch.float8_e4m3fn):
    """The norm of ``rms_norm`` in 8 bits, rounded once, for a product in 8 bits: ``(q, scale_inv, h)``.  With ``scale`` (one float32
    on the device, of delayed scaling as the grouped modules use it: a slot of ``fp8_meta``) ``q = y * scale``, saturating, and ``amax``
    (one float32, may be None) is raised to ``max |y|``; ``scale_inv`` is None, the caller's.  Without, every row has its own scale:
    by ``most``, its largest ``|y|`` or 2^-100, and ``largest``, the largest number of ``dtype`` (``float8_e4m3fn`` or ``float8_e5m2``),
    ``q = y * (largest / most)``, saturating, and ``scale_inv [...] = most / largest`` (float32, without the columns), for a product of the
    caller's: the package's own take one scale for a tensor.  ``h`` is None without a residual.  A NaN stays one and leaves the maximum as
    it is; a row with an infinite ``y`` has an infinite scale.  No gradients are taken: tensors that require one are refused outside of
    ``torch.no_grad()``."""
    return native.rms_norm_fp8(x, weight, eps, residual, scale, amax, dtype)


def embedding(ids, weight, scale=1.0, padding_idx=None):
    """Rows of the table ``weight [rows, columns]`` (contiguous) by token id, times ``scale``: ``[*ids.shape, columns]`` in the
    table's type.  ``ids``: int64 or int32.  An id outside the table gives a row of zeros and takes no gradient (a table that is sharded by
    rows is looked up with ``ids - first_row`` and its results added up); the row ``padding_idx`` is read like any other and
    takes no gradient.  The table's gradient is dense, summed in float32 over every row's tokens in a fixed order."""
    return native.embedding(ids, weight, scale, padding_idx)


class LayerNorm(torch.nn.Module):
    """Layer norm over the last dimension with its own weight (ones) and bias (zeros; None without)."""

    def __init__(self, hidden, eps=1e-5, bias=True, dtype=torch.bfloat16, device="cuda"):
        super().__init__()
        self.hidden = hidden
        self.eps = eps
        self.weight = torch.nn.Parameter(torch.ones(hidden, dtype=dtype, device=device))
        self.bias = torch.nn.Parameter(torch.zeros(hidden, dtype=dtype, device=device)) if bias else None

    def forward(self, input):
        return layer_norm(input, self.weight, self.bias, self.eps)

    def extra_repr(self):
        return f"{self.hidden}, eps={self.eps}, bias={self.bias is not None}"


class RMSNorm(torch.nn.Module):
    """Root-mean-square norm over the last dimension with its own weight (ones); ``forward(x)`` or, the residual's addition in front,
    ``forward(x, residual)``, which returns the normed rows and the sum."""

    def __init__(self, hidden, eps=1e-5, dtype=torch.bfloat16, device="cuda"):
        super().__init__()
        self.hidden = hidden
        self.eps = eps
        self.weight = torch.nn.Parameter(torch.ones(hidden, dtype=dtype, device=device))

    def forward(self, input, residual=None):
        return rms_norm(input, self.weight, self.eps, residual)

    def extra_repr(self):
        return f"{self.hidden}, eps={self.eps}"


class Embedding(torch.nn.Module):
    """A table of ``num_embeddings`` rows of ``hidden`` columns, drawn from a normal distribution (the row ``padding_idx``
    zeros), and its scaled lookup."""

    def __init__(self, num_embeddings, hidden, scale=1.0, padding_idx=None, dtype=torch.bfloat16, device="cuda"):
        super().__init__()
        self.scale = scale
        self.padding_idx = padding_idx
        self.weight = torch.nn.Parameter(torch.randn(num_embeddings, hidden, dtype=dtype, device=device))
        if padding_idx is not None:
            with torch.no_grad():
                self.weight[padding_idx].zero_()

    def forward(self, ids):
        return embedding(ids, self.weight, self.scale, self.padding_idx)

    def extra_repr(self):
        return f"{self.weight.shape[0]}, {self.weight.shape[1]}, scale={self.scale}, padding_idx={self.padding_idx}"
