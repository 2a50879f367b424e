"""The Python reference's Linear layer on the HIP kernels.

core/layers.py:7-33 keeps the weight as [out_channels, in_features] and, in forward, first
materialises its transpose with permute([1, 0]) (a tensor_permute launch and a copy of the
weight) and then runs bmm(x, W^T) (:27-29). Here forward runs the same product as ONE NT GEMM
(B stored [N, K]: migemm_bmm_permute_tiled with transB and a broadcast weight), so no
transposed copy of the weight is ever made.

Like the reference's forward, this one returns x @ W^T and does not add the bias (layers.py:
21-33 never reads self.bias, which starts at zero, :16); LinearForward (the C# host's
NnClGlob.LinearForward) is the bias-epilogue form.
"""
import numpy as np
import torch

from .nncl_glob import NnClGlob, ShapeError, _check_typed, _closing, _require


class Linear:
    """Linear(in_features, out_channels, nnclglob) as core/layers.py:7-33."""

    def __init__(self, in_features, out_channels, nnclglob=None, weight=None, seed=None):
        self.nnclglob = nnclglob if nnclglob is not None else NnClGlob()
        self.in_features = int(in_features)
        self.out_channels = int(out_channels)
        dev = self.nnclglob.device
        if weight is None:
            # U(-1/sqrt(in), 1/sqrt(in)) of shape [out, in] (layers.py:14-15)
            bound = 1.0 / np.sqrt(self.in_features)
            rng = np.random.default_rng(seed)
            weight = rng.uniform(-bound, bound, size=(self.out_channels, self.in_features))
        w = torch.as_tensor(np.asarray(weight, dtype=np.float32)) if not isinstance(
            weight, torch.Tensor) else weight.to(torch.float32)
        _require(list(w.shape) == [self.out_channels, self.in_features],
                 f"weight must be [{self.out_channels}, {self.in_features}]")
        self.weight = w.to(dev).contiguous()
        self.bias = torch.zeros(self.out_channels, dtype=torch.float32, device=dev)  # :16

    def forward(self, x):
        """y[..., out] = x[..., in] @ weight^T, as one NT GEMM over all rows of x."""
        if x.shape[-1] != self.in_features:
            raise ShapeError(f"x must end in {self.in_features} features (got {list(x.shape)})")
        x3 = x.reshape(1, -1, self.in_features).contiguous()  # layers.py:23-24
        y = self.nnclglob.BmmPermute(x3, self.weight.unsqueeze(0), transA=False, transB=True)
        return y.reshape(list(x.shape[:-1]) + [self.out_channels])  # :31-33

    __call__ = forward

    def parameters(self):
        return [self.weight, self.bias]


class LinearInt8:
    """A Linear layer for serving, its weight held in 8 bits with a scale for each output:
    y[..., out] = x[..., in] @ weight^T (+ bias). weight [out, in] is a float tensor or array
    (e.g. Linear.weight), quantised here once; x and y are float32 or bfloat16. For inference: y
    carries no gradient. activation ("relu", "silu", "gelu", "gelu_tanh") and a residual given
    with x are applied in the product's launch; gated: weight [2 * out, in] holds the rows of a
    gate, then those that it multiplies: y = activation(gate) * up."""

    def __init__(self, weight, bias=None, nnclglob=None, activation=None, gated=False):
        self.nnclglob = nnclglob if nnclglob is not None else NnClGlob()
        dev = self.nnclglob.device
        w = weight if isinstance(weight, torch.Tensor) else torch.as_tensor(
            np.asarray(weight, dtype=np.float32))
        _require(w.dim() == 2, "weight must be [out, in]")
        rows, self.in_features = w.shape
        self.out_channels, _ = _closing(rows, activation, gated)
        self.activation, self.gated = activation, bool(gated)
        if w.dtype != torch.bfloat16:
            w = w.to(torch.float32)
        self.weight, self.scales = self.nnclglob.QuantizeRows(w.to(dev).contiguous())
        self.bias = None
        if bias is not None:
            b = bias if isinstance(bias, torch.Tensor) else torch.as_tensor(np.asarray(bias))
            self.bias = b.to(dev, torch.float32).contiguous()
            _check_typed("bias", self.bias, torch.float32, (rows,))

    def forward(self, x, residual=None):
        if not isinstance(x, torch.Tensor) or not x.dim() or x.shape[-1] != self.in_features:
            raise ShapeError(f"x must end in {self.in_features} features (got "
                             f"{list(getattr(x, 'shape', []))})")
        return self.nnclglob.LinearInt8(x, self.weight, self.scales, self.bias, self.activation,
                                        self.gated, residual)

    __call__ = forward

    def forwardRows(self, values, scales, dtype=torch.float32, residual=None):
        """The same layer over rows that are in 8 bits already (of QuantizeRows or NormInt8)."""
        return self.nnclglob.MatmulInt8(values, scales, self.weight, self.scales, self.bias, dtype,
                                        self.activation, self.gated, residual)

    def parameters(self):
        return [self.weight, self.scales] + ([self.bias] if self.bias is not None else [])
