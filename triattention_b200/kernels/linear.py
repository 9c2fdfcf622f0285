"""INT8 projections: rows of codes made from activations, and the products of such rows with INT8 weights.

The reference runs every matrix product of the model in bf16 through torch; only its attention is quantised.  Here a
decoder layer's projections may run on the tensor cores' INT8 path as well: symmetric codes, one scale per token and one per
output channel, exact 32-bit integer sums (``csrc/linear.cu``), and the kernels that make the tokens' codes as part of what
precedes a projection anyway (``csrc/rows.cu``): the root-mean-square norm with the residual's addition, the gated
activation, or plain rows.

``Int8Ops`` is the executor (it allocates, checks and calls the library, on the caller's current stream); ``Int8Linear``,
``Int8RMSNorm``, ``Int8MLP`` and ``Int8DecoderLayer`` put it into a Hugging Face model (``models.int8_projections``).
"""
from __future__ import annotations

import torch

from triattention_b200.kernels.extension import MAX_WIDTH

CODE_ALIGN = 16     # code rows start on 16-byte boundaries


class Int8Rows:
    """Codes int8 [..., H] and scales f32 [...]: row t stands for scales[t] * codes[t].  `dtype` is the type of the values the
    rows were made from, which `dequantize` and `linear` give back unless they are told otherwise."""

    __slots__ = ("codes", "scales", "dtype")

    def __init__(self, codes, scales, dtype=torch.bfloat16):
        if codes.dtype != torch.int8 or scales.dtype != torch.float32 or codes.shape[:-1] != scales.shape:
            raise RuntimeError("Int8Rows: int8 codes [..., H] and float32 scales [...]")
        self.codes, self.scales, self.dtype = codes, scales, dtype

    @property
    def shape(self):
        return self.codes.shape

    @property
    def device(self):
        return self.codes.device


def _flat(x):
    """[..., H] as [T, H] (a view wherever the rows lie one stride apart)."""
    return x if x.dim() == 2 else x.reshape(-1, x.shape[-1])


class Int8Ops:
    """Calls that end in rows of codes, and the product that starts from them.  Every call allocates its results and runs on the
    current stream of the inputs' device; nothing synchronises with the host.  Inference only: codes carry no gradient, and
    inputs that ask for one are refused while gradients are being recorded."""

    def __init__(self, module):
        self.module = module

    @staticmethod
    def _inference(*tensors):
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
            raise RuntimeError("the INT8 projections have no backward pass: call them under torch.no_grad() or inference_mode()")

    @staticmethod
    def _empty_codes(x):
        """Uninitialised codes [T, H], rows a multiple of 16 bytes apart, and scales [T]."""
        rows, width = x.shape
        if not 1 <= width <= MAX_WIDTH:
            raise RuntimeError(f"rows of 1..{MAX_WIDTH} features")
        pitch = -(-width // CODE_ALIGN) * CODE_ALIGN
        codes = torch.empty((rows, pitch), dtype=torch.int8, device=x.device)
        return (codes if pitch == width else codes[:, :width]), torch.empty(rows, dtype=torch.float32, device=x.device)

    @staticmethod
    def _shaped(codes, scales, like):
        if like.dim() != 2:
            codes, scales = codes.view(like.shape), scales.view(like.shape[:-1])
        return Int8Rows(codes, scales, like.dtype)

    def quantize_rows(self, x):
        """x [..., H] (bf16, fp16 or fp32) -> Int8Rows."""
        self._inference(x)
        flat = _flat(x)
        codes, scales = self._empty_codes(flat)
        self.module.quantize_rows(flat, codes, scales)
        return self._shaped(codes, scales, x)

    def silu_mul(self, gate, up):
        """silu(gate) * up -> Int8Rows; gate and up [..., H] may be the halves of one tensor."""
        self._inference(gate, up)
        if gate.shape != up.shape:
            raise RuntimeError("gate and up have one shape")
        flat = _flat(gate)
        codes, scales = self._empty_codes(flat)
        self.module.silu_mul_rows(flat, _flat(up), codes, scales)
        return self._shaped(codes, scales, gate)

    def rms_norm(self, x, weight, eps, residual=None):
        """h = x + residual (rounded to x's type); h / sqrt(mean h^2 + eps) * weight -> Int8Rows, or (Int8Rows, h) with a
        residual."""
        self._inference(x, weight, residual)
        if residual is not None and residual.shape != x.shape:
            raise RuntimeError("x and residual have one shape")
        flat = _flat(x)
        codes, scales = self._empty_codes(flat)
        if residual is None:
            self.module.rms_norm_rows(flat, weight, eps, codes, scales)
            return self._shaped(codes, scales, x)
        total = torch.empty(flat.shape, dtype=x.dtype, device=x.device)
        self.module.rms_norm_rows(flat, weight, eps, codes, scales, _flat(residual), total)
        return self._shaped(codes, scales, x), total.view(x.shape)

    def dequantize(self, rows, dtype=None):
        """The values that rows of codes stand for, in `dtype` (default: the type they were made from)."""
        flat = _flat(rows.codes)
        out = torch.empty(flat.shape, dtype=dtype or rows.dtype, device=flat.device)
        return self.module.dequantize_rows(flat, rows.scales.reshape(-1), out).view(rows.shape)

    def linear(self, rows, weight, bias=None, residual=None, dtype=None):
        """rows [..., K] . weight [N, K]^T (both Int8Rows) + bias [N] + residual [..., N], in `dtype` (default: the type the
        rows were made from; bias and residual have it too)."""
        self._inference(bias, residual)
        shape = rows.shape[:-1] + weight.shape[:1]
        if residual is not None and residual.shape != shape:
            raise RuntimeError("residual [..., N]")
        codes = _flat(rows.codes)
        out = torch.empty((codes.shape[0], weight.shape[0]), dtype=dtype or rows.dtype, device=codes.device)
        self.module.int8_linear(codes, rows.scales.reshape(-1), weight.codes, weight.scales, out, bias,
                                None if residual is None else _flat(residual))
        return out if len(shape) == 2 else out.view(shape)
