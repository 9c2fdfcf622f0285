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

    @classmethod
    def _of(cls, codes, scales, dtype):
        self = cls.__new__(cls)     # made by a call of this file: nothing to check
        self.codes, self.scales, self.dtype = codes, scales, dtype
        return self

    def _flat(self):
        """codes [T, H] and scales [T]."""
        if self.codes.dim() == 2:
            return self.codes, self.scales
        return self.codes.reshape(-1, self.codes.shape[-1]), self.scales.reshape(-1)

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
        if torch.is_grad_enabled():
            for t in tensors:
                if t is not None and t.requires_grad:
                    raise RuntimeError("the INT8 projections have no backward pass: call them under torch.no_grad() or "
                                       "inference_mode()")

    @staticmethod
    def _empty_codes(x):
        """Uninitialised codes [T,H], rows a multiple of 16 bytes apart, and scales [T], for the rows x [T,H]."""
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
        return Int8Rows._of(codes, scales, like.dtype)

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
        flat = _flat(x)
        if residual is None:
            codes, scales = self._empty_codes(flat)
            self.module.rms_norm_rows(flat, weight, eps, codes, scales)
            return self._shaped(codes, scales, x)
        if residual.shape != x.shape:
            raise RuntimeError("x and residual have one shape")
        codes, scales = self._empty_codes(flat)
        total = flat.new_empty(flat.shape)
        self.module.rms_norm_rows(flat, weight, eps, codes, scales, _flat(residual), total)
        return self._shaped(codes, scales, x), total if x.dim() == 2 else total.view(x.shape)

    def dequantize(self, rows, dtype=None):
        """The values that rows of codes stand for, in `dtype` (default: the type they were made from)."""
        codes, scales = rows._flat()
        out = torch.empty(codes.shape, dtype=dtype or rows.dtype, device=codes.device)
        self.module.dequantize_rows(codes, scales, out)
        return out if rows.codes.dim() == 2 else out.view(rows.shape)

    def linear(self, rows, weight, bias=None, residual=None, dtype=None):
        """rows [..., K] . weight [N, K]^T (both Int8Rows) + bias [N] + residual [..., N], in `dtype` (default: the type the
        rows were made from; bias and residual have it too)."""
        self._inference(bias, residual)
        codes, scales = rows._flat()
        if codes.dim() != 2 or weight.codes.dim() != 2:
            raise RuntimeError("rows [..., K] and weight [N, K]")
        flat = rows.codes.dim() == 2
        out = torch.empty((codes.shape[0], weight.codes.shape[0]), dtype=dtype or rows.dtype, device=codes.device)
        if residual is not None and not flat:
            if residual.shape != rows.shape[:-1] + out.shape[1:]:
                raise RuntimeError("residual [..., N]")
            residual = _flat(residual)
        self.module.int8_linear(codes, scales, weight.codes, weight.scales, out, bias, residual)
        return out if flat else out.view(rows.shape[:-1] + out.shape[1:])
