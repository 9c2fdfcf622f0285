"""INT8 projections: rows of codes made from activations, and the products of such rows with INT8 weights.

The reference runs every matrix product of the model in bf16 through torch; only its attention is quantised.  Here a
decoder layer's projections may run on the tensor cores' INT8 path as well: symmetric codes, one scale per token and one per
output channel, exact 32-bit integer sums (``csrc/linear.cu``), and the kernels that make the tokens' codes as part of what
precedes a projection anyway (``csrc/rows.cu``): the root-mean-square norm with the residual's addition, the gated
activation, or plain rows.

``Int8Ops`` is the executor (it allocates, checks and calls the library, on the caller's current stream); ``Int8Linear`` and
``Int8DecoderLayer`` put it into a Hugging Face model (``models.int8_projections``).
"""
from __future__ import annotations

import copy
import inspect

import torch
from torch.autograd import forward_ad

from triattention_b200.kernels.extension import MAX_OUTPUTS, MAX_WIDTH, ROW_TYPES

ATTENTION_PROJECTIONS = ("q_proj", "k_proj", "v_proj", "o_proj")
CODE_ALIGN = 16     # code rows start on 16-byte boundaries
# Rows that the calls make start on 128-byte boundaries, one cache line, where that is little memory: products read codes 128 bytes
# a row at a time, and rows that straddle lines cost up to a third (16384 x 4099 -> 4096: 262 us 16 bytes apart, 188 with 64, 179
# with 128; 1 x 4099 -> 6144: 11.9 and 9.7).
CODE_LINE, CODE_LINE_FROM = 128, 512


def code_pitch(width):
    """Bytes between the rows of codes that a call makes."""
    align = CODE_LINE if width > CODE_LINE_FROM else CODE_ALIGN
    return -(-width // align) * align


class Int8Rows:
    """Codes int8 [..., H] and scales f32 [...]: row t stands for scales[t] * codes[t].  `dtype` is the type of the values the
    rows were made from, which `dequantize` and `linear` give back unless they are told otherwise.  Those calls want code rows
    that start on 16-byte boundaries (`H` itself may be anything); on 128-byte boundaries products are fastest.

    Rows that a call of `Int8Ops` made lie in one allocation, codes first; the tensors `codes` and `scales` are made when they
    are first asked for (a call is as short as the host is, and most rows are only handed on)."""

    __slots__ = ("shape", "dtype", "device", "index", "rows", "width", "pitch", "codes_ptr", "scales_ptr", "_codes", "_scales", "_buffer")

    def __init__(self, codes, scales, dtype=torch.bfloat16):
        shape = codes.shape
        if codes.dtype != torch.int8 or scales.dtype != torch.float32 or not shape or scales.shape != shape[:-1]:
            raise RuntimeError("Int8Rows: int8 codes [..., H] and float32 scales [...]")
        self.shape, self.dtype, self.device, self.index = shape, dtype, codes.device, codes.get_device()
        if len(shape) != 2:
            codes, scales = codes.reshape(-1, shape[-1]), scales.reshape(-1)
            shape = codes.shape
        self.rows, self.width = rows, width = shape
        self.codes_ptr, self.scales_ptr = pointer, _ = codes.data_ptr(), scales.data_ptr()
        pitch, feature = codes.stride()
        if rows <= 1:
            pitch = -(-width // CODE_ALIGN) * CODE_ALIGN
        if (not 1 <= width <= MAX_WIDTH or pointer % CODE_ALIGN or pitch % CODE_ALIGN or (width > 1 and feature != 1) or
                (rows > 1 and not scales.is_contiguous())):
            pitch = -1      # rows that the calls refuse
        self.pitch, self._codes, self._scales, self._buffer = pitch, codes, scales, None
        if scales.get_device() != self.index:
            raise RuntimeError("Int8Rows: codes and scales on one device")

    @classmethod
    def _empty(cls, like, rows, width, index):
        """Uninitialised rows, of the shape and type of `like`, for a call to fill."""
        self = cls.__new__(cls)
        pitch = code_pitch(width)
        self.device = device = like.device
        self._buffer = buffer = torch.empty(rows * (pitch + 4), dtype=torch.int8, device=device)
        self.codes_ptr = pointer = buffer.data_ptr()
        self.scales_ptr = pointer + rows * pitch
        self.shape, self.dtype, self.index, self.rows, self.width, self.pitch = like.shape, like.dtype, index, rows, width, pitch
        self._codes = None
        return self

    @classmethod
    def _of_buffer(cls, buffer, shape, dtype):
        """Rows as a call makes them, in memory that holds them already."""
        self = cls.__new__(cls)
        self.shape, self.dtype, self.device, self.index = shape, dtype, buffer.device, buffer.get_device()
        self.rows, self.width, self.pitch = shape[:-1].numel(), shape[-1], code_pitch(shape[-1])
        self.codes_ptr, self._buffer, self._codes = buffer.data_ptr(), buffer, None
        self.scales_ptr = self.codes_ptr + self.rows * self.pitch
        return self

    def __reduce__(self):               # copies and saved rows are made anew from their tensors: addresses do not travel
        if self._buffer is not None:    # (one tensor: torch.save takes no two types of one allocation)
            return self._of_buffer, (self._buffer, self.shape, self.dtype)
        shared = self._codes.untyped_storage().data_ptr() == self._scales.untyped_storage().data_ptr()
        return type(self), (self.codes, self.scales.clone() if shared else self.scales, self.dtype)

    def _refuse(self, name):
        raise RuntimeError(f"{name}: rows of 1..{MAX_WIDTH} codes that start on 16-byte boundaries, with contiguous features and "
                           "scales, on a GPU")

    def _views(self):
        if self._codes is None:
            end = self.rows * self.pitch
            self._scales = self._buffer[end:].view(torch.float32)      # (first: who finds codes takes the scales for made)
            self._codes = self._buffer[:end].view(self.rows, self.pitch)[:, :self.width]
        return self._codes, self._scales

    @property
    def codes(self):
        return self._views()[0].view(self.shape)

    @property
    def scales(self):
        return self._views()[1].view(self.shape[:-1])


def _flat(x):
    """[..., H] as [T, H] (a view wherever the rows lie one stride apart)."""
    return x if x.dim() in (0, 2) else x.reshape(-1, x.shape[-1])


class Int8Ops:
    """Calls that end in rows of codes, and the product that starts from them.  Every call allocates its results and runs on the
    current stream of the inputs' device; nothing synchronises with the host.  Inference only: codes carry no gradient, and
    inputs that ask for one are refused while gradients are being recorded, and inputs with a forward-mode tangent always.

    A product whose bounded waits ran out (a GPU that others hold up for seconds) returns all the same, with void results, and says so
    in the GPU's error word: call ``ops.module.check_device_error()``, which waits for the current stream and raises, before results
    are relied on.  ``TriAttention.generate`` does."""

    def __init__(self, module):
        self.module, lib = module, module.lib
        self._launch, self._calls = module._launch, (lib.tri_quantize_rows, lib.tri_silu_mul_rows, lib.tri_rms_norm_rows,
                                                     lib.tri_dequantize_rows, lib.tri_int8_linear)

    def __copy__(self):                 # (the loaded library, and no data)
        return self

    def __deepcopy__(self, memo):
        return self

    def __reduce__(self):
        raise RuntimeError("Int8Ops holds the loaded library and cannot be saved, nor can layers that hold it: save their Int8Rows")

    @staticmethod
    def _inference(*tensors):
        if torch.is_grad_enabled():
            for t in tensors:
                if t is not None and t.requires_grad:
                    raise RuntimeError("the INT8 projections have no backward pass: call them under torch.no_grad() or "
                                       "inference_mode()")
        if forward_ad._current_level >= 0:
            for t in tensors:
                if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                    raise RuntimeError("the INT8 projections have no forward-mode derivative")

    def quantize_rows(self, x):
        """x [..., H] (bf16, fp16 or fp32) -> Int8Rows."""
        self._inference(x)
        flat = x if x.dim() == 2 else _flat(x)
        kind, index, rows, width, stride = self.module._rows(flat, "x")
        out = Int8Rows._empty(x, rows, width, index)
        self._launch(self._calls[0], index, flat.data_ptr(), kind, rows, width, stride, out.codes_ptr, out.pitch, out.scales_ptr)
        return out

    def silu_mul(self, gate, up):
        """silu(gate) * up -> Int8Rows; gate and up [..., H] may be the halves of one tensor."""
        self._inference(gate, up)
        if gate.shape != up.shape:
            raise RuntimeError("gate and up have one shape")
        flat, other = (gate, up) if gate.dim() == 2 else (_flat(gate), _flat(up))
        kind, index, rows, width, stride = self.module._rows(flat, "gate")
        other_stride = self.module._like(other, flat, index, "up")
        out = Int8Rows._empty(gate, rows, width, index)
        self._launch(self._calls[1], index, flat.data_ptr(), other.data_ptr(), kind, rows, width, stride, other_stride, out.codes_ptr,
                     out.pitch, out.scales_ptr)
        return out

    def rms_norm(self, x, weight, eps, residual=None):
        """h = x + residual (rounded to x's type); h / sqrt(mean h^2 + eps) * weight -> Int8Rows, or (Int8Rows, h) with a
        residual."""
        self._inference(x, weight, residual)
        if residual is not None and residual.shape != x.shape:
            raise RuntimeError("x and residual have one shape")
        m, flat = self.module, x if x.dim() == 2 else _flat(x)
        kind, index, rows, width, stride = m._rows(flat, "x")
        m._norm_weight(weight, flat, width, index)
        if residual is None:
            out = Int8Rows._empty(x, rows, width, index)
            self._launch(self._calls[2], index, flat.data_ptr(), None, weight.data_ptr(), kind, rows, width, stride, 0, eps, None, 0,
                         out.codes_ptr, out.pitch, out.scales_ptr)
            return out
        other = residual if residual.dim() == 2 else _flat(residual)
        other_stride = m._like(other, flat, index, "residual")
        out = Int8Rows._empty(x, rows, width, index)
        total = torch.empty_like(x) if x.is_contiguous() else x.new_empty(*x.shape)
        self._launch(self._calls[2], index, flat.data_ptr(), other.data_ptr(), weight.data_ptr(), kind, rows, width, stride,
                     other_stride, eps, total.data_ptr(), width, out.codes_ptr, out.pitch, out.scales_ptr)
        return out, total

    def dequantize(self, rows, dtype=None):
        """The values that rows of codes stand for, in `dtype` (default: the type they were made from)."""
        dtype = dtype or rows.dtype
        out, kind = torch.empty(*rows.shape, dtype=dtype, device=rows.device), ROW_TYPES.get(dtype)
        if rows.pitch < 0 or rows.index < 0:
            rows._refuse("dequantize")
        if kind is None:
            raise RuntimeError("dequantize: bf16, fp16 or fp32 values")
        self._launch(self._calls[3], rows.index, rows.codes_ptr, rows.pitch, rows.scales_ptr, kind, rows.rows, rows.width,
                     out.data_ptr(), rows.width)
        return out

    def linear(self, rows, weight, bias=None, residual=None, dtype=None):
        """rows [..., K] . weight [N, K]^T (both Int8Rows) + bias [N] + residual [..., N], in `dtype` (default: the type the
        rows were made from; bias and residual have it too)."""
        self._inference(bias, residual)
        m, index, outputs = self.module, rows.index, weight.rows
        if rows.pitch < 0 or index < 0:
            rows._refuse("linear")
        if weight.pitch < 0:
            weight._refuse("weight")
        if rows.width != weight.width or len(weight.shape) != 2 or weight.index != index or not 1 <= outputs <= MAX_OUTPUTS:
            raise RuntimeError("codes [..., K] and weight [N, K] on one GPU")
        dtype = dtype or rows.dtype
        shape = (rows.rows, outputs) if len(rows.shape) == 2 else (*rows.shape[:-1], outputs)
        out, kind = torch.empty(*shape, dtype=dtype, device=rows.device), ROW_TYPES.get(dtype)
        if kind is None:
            raise RuntimeError("linear: bf16, fp16 or fp32 outputs")
        if bias is not None:
            m._bias(bias, dtype, outputs, index)
        residual_ptr, residual_stride = None, 0
        if residual is not None:
            if residual.shape != out.shape:
                raise RuntimeError("residual [..., N]")
            residual = _flat(residual)
            if residual.dtype != out.dtype or residual.get_device() != index or (residual.stride(1) != 1 and outputs != 1):
                raise RuntimeError("residual of the output's type, on its device, with contiguous features")
            residual_ptr, residual_stride = residual.data_ptr(), residual.stride(0)
        self._launch(self._calls[4], index, rows.codes_ptr, rows.pitch, rows.scales_ptr, weight.codes_ptr, weight.pitch,
                     weight.scales_ptr, None if bias is None else bias.data_ptr(), residual_ptr, residual_stride, out.data_ptr(),
                     outputs, kind, rows.rows, outputs, rows.width, m._error_pointer(index))
        return out


class Int8Linear(torch.nn.Module):
    """A projection with INT8 weights (one scale per output channel).  Takes rows of codes as they are, quantises anything else.
    The weights are plain attributes, made on the device of the layer they replace: for inference, not for saving or moving."""

    def __init__(self, ops, weight, bias=None):
        super().__init__()
        self.ops, self.rows, self.bias_row = ops, ops.quantize_rows(weight.detach()), None if bias is None else bias.detach()

    @classmethod
    def of(cls, ops, *linears):
        """One projection of torch.nn.Linear layers that read the same rows; their outputs come side by side."""
        if any(type(l) is not torch.nn.Linear for l in linears):
            raise RuntimeError("Int8Linear: torch.nn.Linear layers (one of these is something else, or shared and replaced already)")
        biases = [l.bias for l in linears]
        if any(b is None for b in biases) and any(b is not None for b in biases):
            biases = [torch.zeros_like(l.weight[:, 0]) if b is None else b for l, b in zip(linears, biases)]
        weight = linears[0].weight if len(linears) == 1 else torch.cat([l.weight.detach() for l in linears])
        bias = None if biases[0] is None else biases[0] if len(linears) == 1 else torch.cat([b.detach() for b in biases])
        return cls(ops, weight, bias)

    def forward(self, x, residual=None):
        rows = self.ops.quantize_rows(x) if isinstance(x, torch.Tensor) else x
        return self.ops.linear(rows, self.rows, bias=self.bias_row, residual=residual)


def _stand_in(module, **children):
    """An object of the module's class with its settings, but other children: its forward can be run without touching the model."""
    made = type(module).__new__(type(module))
    made.__dict__.update(vars(module), training=False, _modules={**module._modules, **children})
    return made


def _run(module, values, **more):
    """The class's forward on `values`, as a decoder layer's modules are called; arguments that it cannot do without are None."""
    names = inspect.signature(type(module).forward).parameters.values()
    given = [p.name for p in names if p.kind is p.POSITIONAL_OR_KEYWORD][2:]
    anything = any(p.kind is p.VAR_KEYWORD for p in names)
    missing = {p.name: None for p in list(names)[2:] if p.default is p.empty and p.kind in (p.POSITIONAL_OR_KEYWORD, p.KEYWORD_ONLY)}
    return type(module).forward(module, values, **{**missing, **{n: v for n, v in more.items() if anything or n in given or n in missing}})


def _same(got, want):
    return type(got) is torch.Tensor and got.shape == want.shape and torch.allclose(got, want, rtol=1e-9, atol=1e-9)


def _trial():
    """What forwards are tried on: small and large numbers of both signs (a clamp or a factor shows), in float64."""
    even = dict(dtype=torch.float64, device="cpu")
    return (torch.linspace(-1, 1, 24, **even) * 10.0 ** torch.arange(-3, 5, **even).repeat(3)).reshape(2, 3, 4)


def _layer_adds_up(layer):
    """x + attention(norm(x)), and the feed-forward block of its norm added to that; a tensor, not a tuple."""
    def attention(hidden_states, *args, **kwargs):
        return torch.sin(hidden_states), None
    norm, other, block = lambda x: 2 * x + 1, lambda x: x / 3 - 2, lambda x: 5 * torch.cos(x)
    x = _trial()
    h = x + torch.sin(norm(x))
    got = _run(_stand_in(layer, self_attn=attention, input_layernorm=norm, post_attention_layernorm=other, mlp=block), x)
    return _same(got, h + block(other(h)))


def _block_is_gated(mlp):
    """down(act(gate(x)) * up(x))."""
    x, gate, up, down, act = _trial(), lambda x: 2 * x + 1, lambda x: x / 3 - 2, lambda x: 5 * x - 7, torch.atan
    return _same(_run(_stand_in(mlp, gate_proj=gate, up_proj=up, down_proj=down, act_fn=act), x), down(act(gate(x)) * up(x)))


def _norm_is_rms(norm):
    """weight * x / sqrt(mean x^2 + eps), on the norm's own width in fp32."""
    width, at = norm.weight.shape[0], dict(dtype=torch.float32, device="cpu")
    x, weight = torch.cos(torch.arange(2 * width, **at)).reshape(2, width) * 0.01, torch.sin(torch.arange(width, **at))
    made = _stand_in(norm)
    made.__dict__["_parameters"] = {**norm._parameters, "weight": weight}
    want = x / (x.square().mean(1, keepdim=True) + norm.variance_epsilon).sqrt() * weight
    got = _run(made, x)
    return type(got) is torch.Tensor and torch.allclose(got, want, rtol=1e-4, atol=1e-6)


def _attention_takes_rows(attention):
    """Whether its forward gets by on rows of codes, which have a shape, a type and a device and are otherwise there for the three
    projections.  Run on two tokens with the model's plain attention (whichever is set keeps what it holds)."""
    like, width = attention.o_proj.weight, attention.q_proj.in_features
    rows = Int8Rows(torch.zeros(1, 2, width, dtype=torch.int8, device="cpu"), torch.zeros(1, 2, dtype=torch.float32, device="cpu"), like.dtype)
    rows.device = like.device

    def projection(linear):
        def project(x):
            if x is not rows:
                raise TypeError("not the rows")
            return like.new_zeros(1, 2, linear.out_features)
        return project

    def output(x):
        if type(x) is not torch.Tensor or x.shape != (1, 2, attention.o_proj.in_features):
            raise TypeError("not the heads' outputs")
        return x.new_zeros(1, 2, attention.o_proj.out_features)

    made = _stand_in(attention, o_proj=output, **{n: projection(getattr(attention, n)) for n in ("q_proj", "k_proj", "v_proj")})
    if hasattr(attention, "config"):
        made.config = copy.deepcopy(attention.config)
        made.config._attn_implementation = "eager"
    turn, places = like.new_zeros(1, 2, attention.head_dim), torch.arange(2, device=like.device)
    out = _run(made, rows, position_embeddings=(turn, turn), attention_mask=None, position_ids=places[None], cache_position=places)
    return isinstance(out, tuple) and type(out[0]) is torch.Tensor and out[0].shape == (1, 2, attention.o_proj.out_features)


class Int8DecoderLayer(torch.nn.Module):
    """A decoder layer of the Llama kind (two RMS norms, q / k / v / o projections, a gated SiLU feed-forward block) whose
    projections run on INT8 codes.  Both norms, the addition of the attention's output to the residual stream and the gated
    activation end in the codes that the next projection reads; the down projection adds the residual stream itself.  The
    attention in between is the model's own module, with its projections replaced: whatever attention implementation the model
    is set to runs as before."""

    def __init__(self, ops, layer):
        super().__init__()
        attention, mlp, norms = layer.self_attn, layer.mlp, (layer.input_layernorm, layer.post_attention_layernorm)
        projections = [getattr(attention, n) for n in ATTENTION_PROJECTIONS]
        if len({(w.dtype, w.device) for m in (*projections, *norms, mlp.gate_proj, mlp.up_proj, mlp.down_proj) for w in m.parameters()}) > 1:
            raise RuntimeError("Int8DecoderLayer: the projections' and norms' weights and biases have one type and lie on one device")
        made = [Int8Linear.of(ops, p) for p in projections]
        self.gate_up, self.down = Int8Linear.of(ops, mlp.gate_proj, mlp.up_proj), Int8Linear.of(ops, mlp.down_proj)
        self.norm_weights, self.eps = [n.weight.detach() for n in norms], [n.variance_epsilon for n in norms]
        for name, projection in zip(ATTENTION_PROJECTIONS, made):       # (nothing is replaced before all is made)
            setattr(attention, name, projection)
        self.ops, self.self_attn = ops, attention
        for name, value in vars(layer).items():         # what the model looks up on its layers (attention_type and the like)
            if not name.startswith("_") and name not in self.__dict__:
                setattr(self, name, value)
        self.train(layer.training)

    @staticmethod
    def fits(layer):
        """Whether `layer` is built like that, with nothing in it that would be lost: no module or factor more (scaled residuals,
        norms inside the block), no hooks and no forward of an object's own on what is replaced or is handed rows of codes in place
        of values; and whether it computes that, which its forwards show by what they make of stand-ins for the modules (names
        alone say little: norms behind the blocks, factors, clamped activations and tuples as results go by the same ones)."""
        bare = lambda m: not ("forward" in vars(m) or m._forward_hooks or m._forward_pre_hooks)
        plain = lambda m: bare(m) and not any(isinstance(v, (float, torch.Tensor)) for v in vars(m).values()) and not m._parameters and not m._buffers
        linear = lambda m: type(m) is torch.nn.Linear and bare(m)
        norm = lambda m: ("RMSNorm" in type(m).__name__ and hasattr(m, "variance_epsilon") and bare(m) and
                          [n for n, w in m.named_parameters() if w is not None] == ["weight"])
        attention, mlp = getattr(layer, "self_attn", None), getattr(layer, "mlp", None)
        if not (isinstance(attention, torch.nn.Module) and isinstance(mlp, torch.nn.Module) and bare(attention) and
                all(linear(getattr(attention, n, None)) for n in ATTENTION_PROJECTIONS) and
                all(linear(getattr(mlp, n, None)) for n in ("gate_proj", "up_proj", "down_proj")) and
                type(getattr(mlp, "act_fn", None)).__name__ in ("SiLU", "SiLUActivation") and
                all(norm(getattr(layer, n, None)) for n in ("input_layernorm", "post_attention_layernorm")) and
                plain(layer) and plain(mlp) and len(layer._modules) == 4 and len(mlp._modules) == 4):
            return False
        try:
            return (_layer_adds_up(layer) and _block_is_gated(mlp) and _attention_takes_rows(attention) and
                    all(_norm_is_rms(n) for n in (layer.input_layernorm, layer.post_attention_layernorm)))
        except torch.OutOfMemoryError:
            raise
        except Exception:       # a forward that wants something else
            return False

    def forward(self, hidden_states, **kwargs):
        ops = self.ops
        attended = self.self_attn(hidden_states=ops.rms_norm(hidden_states, self.norm_weights[0], self.eps[0]), **kwargs)[0]
        rows, hidden_states = ops.rms_norm(attended, self.norm_weights[1], self.eps[1], residual=hidden_states)
        both = self.gate_up(rows)
        inner = both.shape[-1] // 2
        return self.down(ops.silu_mul(both[..., :inner], both[..., inner:]), residual=hidden_states)
