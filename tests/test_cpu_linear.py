"""INT8 projections without a GPU: what the entry points refuse (before any CUDA call) and how rows of codes are held."""
import pytest
import torch

from triattention_b200.kernels import extension
from triattention_b200.kernels.extension import MAX_WIDTH, Module, load_library
from triattention_b200.kernels.linear import Int8Ops, Int8Rows, code_pitch

P = 4096            # a 16-byte aligned address that a refused call never touches


@pytest.fixture(scope="module")
def lib():
    return load_library()


def refused(lib, status, what):
    assert status == -1 and what in lib.tri_last_error().decode(), lib.tri_last_error()


def test_row_entry_points_refuse_bad_arguments(lib):
    def quantize(x=P, type=0, rows=4, width=64, stride=64, codes=P, pitch=64, scales=P):
        return lib.tri_quantize_rows(x, type, rows, width, stride, codes, pitch, scales, None)

    for bad in (dict(width=0), dict(width=MAX_WIDTH + 1), dict(width=-5), dict(type=3), dict(type=-1), dict(rows=-1), dict(rows=1 << 31)):
        refused(lib, quantize(**bad), "quantize_rows: rows, width")
    for bad in (dict(x=None), dict(codes=None), dict(scales=None)):
        refused(lib, quantize(**bad), "null")
    for bad in (dict(codes=P + 8), dict(pitch=72), dict(pitch=48)):
        refused(lib, quantize(**bad), "16-byte")
    for bad in (dict(x=P + 1), dict(x=P + 2, type=2), dict(stride=-64)):
        refused(lib, quantize(**bad), "input rows")
    assert quantize(rows=0, x=None, codes=None, scales=None) == 0          # an empty batch is no work

    def gated(gate=P, up=P, type=1, rows=4, width=64, codes=P, pitch=64):
        return lib.tri_silu_mul_rows(gate, up, type, rows, width, 128, 128, codes, pitch, P, None)

    refused(lib, gated(up=None), "silu_mul_rows: null")
    refused(lib, gated(up=P + 1), "silu_mul_rows: input rows")
    refused(lib, gated(pitch=63), "silu_mul_rows: code rows")
    refused(lib, gated(width=MAX_WIDTH + 1), "silu_mul_rows: rows, width")
    assert gated(rows=0) == 0

    def norm(x=P, residual=P, weight=P, rows=4, width=64, eps=1e-6, out=P, out_stride=64, codes=P):
        return lib.tri_rms_norm_rows(x, residual, weight, 0, rows, width, 64, 64, eps, out, out_stride, codes, 64, P, None)

    refused(lib, norm(weight=None), "rms_norm_rows: null")
    refused(lib, norm(residual=None), "both or none")
    refused(lib, norm(out=None), "both or none")
    for eps in (-1e-9, 1.5, float("nan")):
        refused(lib, norm(eps=eps), "eps")
    refused(lib, norm(out_stride=63), "overlap")
    refused(lib, norm(weight=P + 1), "input rows")
    refused(lib, norm(codes=P + 4), "16-byte")
    assert norm(rows=0) == 0

    def values(codes=P, pitch=64, type=0, rows=2, width=64, out=P, out_stride=64):
        return lib.tri_dequantize_rows(codes, pitch, P, type, rows, width, out, out_stride, None)

    refused(lib, values(codes=None), "dequantize_rows: null")
    refused(lib, values(pitch=65), "16-byte")
    refused(lib, values(out_stride=60), "output rows")
    refused(lib, values(out=P + 2, type=2), "output rows")
    assert values(rows=0) == 0


def test_linear_entry_point_refuses_bad_arguments(lib):
    def linear(codes=P, pitch=64, scales=P, weight=P, weight_pitch=64, weight_scales=P, bias=None, residual=None, residual_stride=0,
               out=P, out_stride=32, type=0, tokens=4, outputs=32, width=64, error=P):
        return lib.tri_int8_linear(codes, pitch, scales, weight, weight_pitch, weight_scales, bias, residual, residual_stride, out,
                                   out_stride, type, tokens, outputs, width, error, None)

    for bad in (dict(width=0), dict(width=MAX_WIDTH + 1), dict(outputs=0), dict(tokens=-1), dict(tokens=1 << 31), dict(type=5)):
        refused(lib, linear(**bad), "int8_linear: tokens, outputs, width")
    for name in ("codes", "scales", "weight", "weight_scales", "out", "error"):
        refused(lib, linear(**{name: None}), "int8_linear: null")
    for bad in (dict(codes=P + 1), dict(weight=P + 8), dict(pitch=80 + 8), dict(weight_pitch=63), dict(pitch=48), dict(weight_pitch=0)):
        refused(lib, linear(**bad), "16-byte")
    for bad in (dict(out=P + 1), dict(bias=P + 1), dict(residual=P + 2, type=2)):
        refused(lib, linear(**bad), "alignment")
    for bad in (dict(out_stride=31), dict(residual=P, residual_stride=-1)):
        refused(lib, linear(**bad), "output and residual rows")
    assert linear(tokens=0) == 0


def test_module_and_ops_refuse_host_tensors_and_shapes(lib):
    module, ops = Module(lib), Int8Ops(Module(lib))
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="on a GPU"):
        ops.quantize_rows(x)
    with pytest.raises(RuntimeError, match="on a GPU"):
        ops.silu_mul(x, x)
    with pytest.raises(RuntimeError, match="on a GPU"):
        ops.rms_norm(x, x[0], 1e-6)
    with pytest.raises(RuntimeError, match="on a GPU"):
        ops.linear(Int8Rows(x.to(torch.int8), torch.ones(4)), Int8Rows(x.to(torch.int8), torch.ones(4)))
    with pytest.raises(RuntimeError, match="on a GPU"):
        module.dequantize_rows(x.to(torch.int8), torch.ones(4), x)
    with pytest.raises(RuntimeError, match="one shape"):
        ops.silu_mul(x, x[:, :32])
    with pytest.raises(RuntimeError, match="one shape"):
        ops.rms_norm(x, x[0], 1e-6, residual=x[:1])
    with pytest.raises(RuntimeError, match="rows of 1"):
        ops.quantize_rows(torch.zeros(1, MAX_WIDTH + 1))
    with pytest.raises(RuntimeError, match="rows of 1"):
        ops.quantize_rows(torch.zeros(3, 0))
    with pytest.raises(RuntimeError, match="no backward"):
        ops.quantize_rows(x.requires_grad_())


def test_rows_of_codes_are_checked():
    codes = torch.zeros(2, 3, 16, dtype=torch.int8)
    rows = Int8Rows(codes, torch.ones(2, 3))
    assert rows.shape == (2, 3, 16) and rows.dtype == torch.bfloat16 and rows.device == codes.device
    for bad in ((codes.float(), torch.ones(2, 3)), (codes, torch.ones(2, 3).double()), (codes, torch.ones(6)), (codes, torch.ones(2, 3, 1))):
        with pytest.raises(RuntimeError, match="Int8Rows"):
            Int8Rows(*bad)


def test_rows_that_calls_make_start_on_cache_lines():
    for width, pitch in ((1, 16), (65, 80), (512, 512), (513, 640), (4096, 4096), (4099, 4224), (MAX_WIDTH, 131072)):
        assert code_pitch(width) == pitch
        rows = Int8Rows._empty(torch.zeros(3, width), 3, width, -1)
        assert rows.pitch == pitch and rows.codes.shape == (3, width) and rows.codes.stride() == (pitch, 1)
        assert rows.scales.shape == (3,) and rows.scales.data_ptr() == rows.codes_ptr + 3 * pitch == rows.scales_ptr


def test_a_library_without_an_entry_point_asks_to_be_rebuilt(monkeypatch):
    monkeypatch.setitem(extension.SIGNATURES, "tri_not_there", [])
    with pytest.raises(RuntimeError, match="tri_not_there: rebuild"):
        load_library()


# ---- in a model ------------------------------------------------------------------------------------------------------

class ExactOps:
    """The interface of Int8Ops without any quantisation: rows are the values themselves."""

    class Rows:
        def __init__(self, values):
            self.values, self.shape = values, values.shape

    def quantize_rows(self, x):
        return self.Rows(x)

    def silu_mul(self, gate, up):
        return self.Rows(torch.nn.functional.silu(gate) * up)

    def rms_norm(self, x, weight, eps, residual=None):
        h = x if residual is None else x + residual
        rows = self.Rows(h / (h.square().mean(-1, keepdim=True) + eps).sqrt() * weight)
        return rows if residual is None else (rows, h)

    def linear(self, rows, weight, bias=None, residual=None, dtype=None):
        y = torch.nn.functional.linear(rows.values, weight.values, bias)
        return y if residual is None else y + residual


def toy(kind, **more):
    import transformers
    torch.manual_seed(0)
    config = getattr(transformers, kind + "Config")(hidden_size=96, intermediate_size=160, num_hidden_layers=3, num_attention_heads=4,
                                                    num_key_value_heads=2, head_dim=32, vocab_size=200, **more)
    return getattr(transformers, kind + "ForCausalLM")(config).eval()


@pytest.mark.parametrize("kind,more", [("Llama", {}), ("Llama", dict(attention_bias=True, mlp_bias=True)), ("Qwen2", {}), ("Mistral", {}),
                                       ("Qwen3", {})])
def test_wrapped_layers_compute_the_model(kind, more):
    """Every weight, bias, norm and residual in its place: with operators that do not quantise, the wrapped model is the model.
    fp32 sums in another order: 3 layers of products over at most 160 terms, far below 1e-4 of logits of order one."""
    from triattention_b200.models import int8_projections
    model = toy(kind, **more)
    with torch.no_grad():
        for p in model.parameters():           # (norm weights of one and biases of zero would hide a mix-up)
            p.add_(0.1 * torch.randn_like(p))
        ids = torch.randint(0, 200, (2, 11))
        want = model(input_ids=ids, use_cache=False).logits
        assert int8_projections(model, ExactOps()) is model
        got = model(input_ids=ids, use_cache=False).logits
        torch.testing.assert_close(got, want, rtol=1e-4, atol=1e-4 * float(want.abs().max()))
        # and with a cache of its own, token by token
        out = model(input_ids=ids[:, :10], use_cache=True)
        step = model(input_ids=ids[:, 10:], past_key_values=out.past_key_values, use_cache=True).logits
        torch.testing.assert_close(step[:, 0], want[:, 10], rtol=1e-3, atol=1e-3 * float(want.abs().max()))


def test_models_without_such_layers_are_refused():
    import transformers
    from triattention_b200.models import int8_projections
    other = transformers.GPT2LMHeadModel(transformers.GPT2Config(n_embd=32, n_layer=1, n_head=2, vocab_size=50))
    with pytest.raises(RuntimeError, match="no decoder layer"):
        int8_projections(other, ExactOps())
    with pytest.raises(RuntimeError, match="no decoder layer"):
        int8_projections(toy("Llama", hidden_act="gelu"), ExactOps())
    wrapped = int8_projections(toy("Llama"), ExactOps())
    with pytest.raises(RuntimeError, match="no decoder layer"):
        int8_projections(wrapped, ExactOps())   # once is enough


@pytest.mark.parametrize("what", ["scaled residual", "norm in the block", "factor of the block", "scaled norm", "layer norm", "hook",
                                  "pre-hook", "own forward", "hook on a projection", "parameter", "buffer"])
def test_layers_with_something_more_are_refused(what):
    """What the wrapped layer would drop: it computes the plain decoder layer and nothing else."""
    from triattention_b200.models import int8_projections
    model = toy("Llama")
    for layer in model.model.layers:
        norm = layer.input_layernorm
        if what == "scaled residual":
            layer.residual_multiplier = 0.5
        elif what == "norm in the block":
            layer.mlp.inner_norm = torch.nn.RMSNorm(8)
        elif what == "factor of the block":
            layer.mlp.multiplier = 2.0
        elif what == "scaled norm":
            norm.bias = torch.nn.Parameter(torch.zeros_like(norm.weight))
        elif what == "layer norm":
            layer.input_layernorm = torch.nn.LayerNorm(norm.weight.shape[0])
            layer.input_layernorm.variance_epsilon = 1e-6
        elif what == "hook":
            layer.register_forward_hook(lambda *a: None)
        elif what == "pre-hook":
            layer.mlp.register_forward_pre_hook(lambda *a: None)
        elif what == "own forward":
            layer.forward = lambda *a, **k: None
        elif what == "hook on a projection":
            layer.self_attn.q_proj.register_forward_hook(lambda *a: None)
        elif what == "parameter":
            layer.gain = torch.nn.Parameter(torch.ones(1))
        elif what == "buffer":
            layer.mlp.register_buffer("gain", torch.ones(1))
    with pytest.raises(RuntimeError, match="no decoder layer"):
        int8_projections(model, ExactOps())
    assert all(type(layer.self_attn.q_proj) is torch.nn.Linear for layer in model.model.layers)


def test_wrapped_layers_keep_the_mode():
    from triattention_b200.models import int8_projections
    model = toy("Llama").eval()
    int8_projections(model, ExactOps())
    assert not any(m.training for m in model.modules())


def test_rows_without_a_feature_axis_are_refused(lib):
    with pytest.raises(RuntimeError, match="rows of 1"):
        Int8Ops(Module(lib)).quantize_rows(torch.zeros(()))


def test_a_layer_used_twice_stays_one_layer():
    from triattention_b200.models import int8_projections
    model = toy("Llama")
    model.model.layers[2] = model.model.layers[0]
    ids = torch.arange(12)[None]
    with torch.no_grad():
        want = model(input_ids=ids, use_cache=False).logits
        int8_projections(model, ExactOps())
        torch.testing.assert_close(model(input_ids=ids, use_cache=False).logits, want, rtol=1e-4, atol=1e-4 * float(want.abs().max()))
    assert model.model.layers[2] is model.model.layers[0] is not model.model.layers[1]


def test_more_channels_than_32_bits_count_are_refused(lib):
    """(The C call takes an int: 2^32 + 5 channels must not become 5.)"""
    rows, weight = Int8Rows(torch.zeros(1, 16, dtype=torch.int8), torch.ones(1)), Int8Rows(torch.zeros(1, 16, dtype=torch.int8), torch.ones(1))
    rows.index = weight.index = 0           # as if on a GPU: the refusal comes before anything is allocated or launched
    weight.rows = (1 << 32) + 5
    with pytest.raises(RuntimeError, match="weight"):
        Int8Ops(Module(lib)).linear(rows, weight)


def test_infer_flag(monkeypatch):
    """--int8-projections wraps the model before the engine is made; without it nothing is wrapped."""
    import sys
    from triattention_b200 import infer
    done = []

    class Engine:
        def __init__(self, model, *args):
            done.append("engine")

        def generate(self, *args):
            return [1, 2]

    class Tokenizer:
        def __call__(self, *args, **kwargs):
            import types
            return types.SimpleNamespace(input_ids=types.SimpleNamespace(cuda=lambda: None))

        def decode(self, tokens, **kwargs):
            return "text"

    monkeypatch.setattr(infer, "load_tokenizer", lambda path: Tokenizer())
    monkeypatch.setattr(infer, "load_model", lambda path: "model")
    monkeypatch.setattr(infer, "render_prompt", lambda *a: "")
    monkeypatch.setattr(infer, "eos_ids", lambda *a: set())
    monkeypatch.setattr(infer, "TriAttention", Engine)
    monkeypatch.setattr(infer, "int8_projections", lambda model: done.append("int8"))
    for flags, want in (([], ["engine"]), (["--int8-projections"], ["int8", "engine"])):
        done.clear()
        monkeypatch.setattr(sys, "argv", ["infer", "--model", "m", "--prompt", "p", *flags])
        infer.main()
        assert done == want


# ---- copies --------------------------------------------------------------------------------------------------------------

def copies(rows):
    import copy
    import io
    import pickle
    saved = io.BytesIO()
    torch.save(rows, saved)
    saved.seek(0)
    yield "deepcopy", copy.deepcopy(rows)
    yield "pickle", pickle.loads(pickle.dumps(rows))
    yield "save", torch.load(saved, weights_only=False)
    yield "copy", copy.copy(rows)


def test_copied_and_saved_rows_hold_their_own_memory():
    """Calls read rows by address: a copy's addresses are those of the copy's tensors, and its pitch theirs."""
    made = Int8Rows._empty(torch.zeros(2, 3, 600, dtype=torch.float16), 6, 600, -1)      # as a call makes them, 640 bytes apart
    made._buffer.copy_(torch.arange(made._buffer.numel()) % 61)
    pitched = torch.arange(5 * 64).reshape(5, 64).to(torch.int8)
    for rows in (made, Int8Rows(pitched[:, :50], torch.arange(5.0)), Int8Rows(pitched[2], torch.tensor(3.0), torch.float32),
                 Int8Rows(pitched[:, :50].view(5, 1, 50), torch.ones(5, 1)), Int8Rows(pitched[:0], torch.ones(0)),
                 Int8Rows(pitched[:, 1:50], torch.ones(5)),                              # (this one is refused by the calls)
                 Int8Rows(made.codes[:1], made.scales[:1])):                             # one allocation, two types
        codes, scales = rows.codes.clone(), rows.scales.clone()
        for how, other in copies(rows):
            assert type(other) is Int8Rows and (other.shape, other.dtype, other.index, other.rows, other.width, other.pitch) == (
                rows.shape, rows.dtype, rows.index, rows.rows, rows.width, rows.pitch), how
            assert torch.equal(other.codes, codes) and torch.equal(other.scales, scales), how
            assert other.codes_ptr == other.codes.data_ptr() and other.scales_ptr == other.scales.data_ptr(), how
            assert how == "copy" or not rows.rows or other.codes_ptr != rows.codes_ptr, how
    import copy
    other = copy.deepcopy(made)
    made._buffer.fill_(9)
    assert not torch.equal(other.codes, made.codes)


def test_copies_of_the_executor(lib):
    """It holds the loaded library and no data: copies of a model share it, and saving it is refused in words."""
    import copy
    import pickle
    ops = Int8Ops(Module(lib))
    assert copy.deepcopy(ops) is ops and copy.deepcopy([ops])[0] is ops and copy.copy(ops) is ops
    with pytest.raises(RuntimeError, match="Int8Rows"):
        pickle.dumps(ops)


def test_rows_shown_to_two_threads_at_once():
    """The tensors of rows that a call made are made when first asked for: a second thread that asks meanwhile gets them too."""
    import threading
    rows = Int8Rows._empty(torch.zeros(3, 40), 3, 40, -1)
    inside, go_on = threading.Event(), threading.Event()

    class Slow:             # the first thread that comes to the scales stops there
        def __init__(self, buffer):
            self.buffer = buffer

        def __getitem__(self, part):
            if part.start is not None and not inside.is_set():
                inside.set()
                go_on.wait(20)
            return self.buffer[part]

    rows._buffer = Slow(rows._buffer)
    first = []
    thread = threading.Thread(target=lambda: first.append(rows.scales))
    thread.start()
    try:
        assert inside.wait(20)
        assert rows.scales.shape == (3,) and rows.codes.shape == (3, 40)
    finally:
        go_on.set()
        thread.join()
    assert first[0].data_ptr() == rows.scales.data_ptr() == rows.scales_ptr


# ---- which layers are taken: by what they compute ----------------------------------------------------------------------------

def behaving(kind):
    """A toy model whose layers have the names, modules and settings of the Llama kind, and one thing that they compute otherwise."""
    from transformers.models.llama.modeling_llama import LlamaAttention, LlamaDecoderLayer, LlamaMLP, LlamaRMSNorm
    model = toy("Llama")

    class Scaled(LlamaDecoderLayer):            # an integer factor: no float among the settings
        def forward(self, hidden_states, **kwargs):
            hidden_states = hidden_states + self.times * self.self_attn(hidden_states=self.input_layernorm(hidden_states), **kwargs)[0]
            return hidden_states + self.mlp(self.post_attention_layernorm(hidden_states))

    class Behind(LlamaDecoderLayer):            # norms behind the blocks
        def forward(self, hidden_states, **kwargs):
            hidden_states = hidden_states + self.input_layernorm(self.self_attn(hidden_states=hidden_states, **kwargs)[0])
            return hidden_states + self.post_attention_layernorm(self.mlp(hidden_states))

    class Beside(LlamaDecoderLayer):            # both blocks on the layer's input
        def forward(self, hidden_states, **kwargs):
            attended = self.self_attn(hidden_states=self.input_layernorm(hidden_states), **kwargs)[0]
            return hidden_states + attended + self.mlp(self.post_attention_layernorm(hidden_states))

    class Tuple(LlamaDecoderLayer):
        def forward(self, hidden_states, **kwargs):
            return (super().forward(hidden_states, **kwargs),)

    class Clamped(LlamaMLP):
        def forward(self, x):
            return self.down_proj(self.act_fn(self.gate_proj(x).clamp(max=7)) * self.up_proj(x))

    class Swapped(LlamaMLP):
        def forward(self, x):
            return self.down_proj(self.gate_proj(x) * self.act_fn(self.up_proj(x)))

    class OneMoreRMSNorm(LlamaRMSNorm):         # weights around zero
        def forward(self, x):
            return x * (x.square().mean(-1, keepdim=True) + self.variance_epsilon).rsqrt() * (1 + self.weight)

    class Gate(LlamaAttention):                 # values of its own made of what it is given
        def forward(self, hidden_states, **kwargs):
            out, weights = super().forward(hidden_states, **kwargs)
            return out * hidden_states.mean(-1, keepdim=True), weights

    for layer in model.model.layers:
        layer.times = 2
        if kind in ("Scaled", "Behind", "Beside", "Tuple"):
            layer.__class__ = locals()[kind]
        elif kind in ("Clamped", "Swapped"):
            layer.mlp.__class__ = locals()[kind]
        elif kind == "OneMore":
            layer.post_attention_layernorm.__class__ = OneMoreRMSNorm
        elif kind == "Gate":
            layer.self_attn.__class__ = Gate
        elif kind == "hook":
            layer.self_attn.register_forward_hook(lambda *a: None)
        elif kind == "pre-hook":
            layer.self_attn.register_forward_pre_hook(lambda *a: None)
        elif kind == "own forward":
            layer.self_attn.forward = layer.self_attn.forward
    return model


@pytest.mark.parametrize("kind", ["Scaled", "Behind", "Beside", "Tuple", "Clamped", "Swapped", "OneMore", "Gate", "hook", "pre-hook", "own forward"])
def test_layers_that_compute_something_else_are_refused(kind):
    from triattention_b200.models import int8_projections
    model = behaving(kind)
    before = [(n, type(m)) for n, m in model.named_modules()]
    with pytest.raises(RuntimeError, match="no decoder layer"):
        int8_projections(model, ExactOps())
    assert [(n, type(m)) for n, m in model.named_modules()] == before
    assert all("forward" not in vars(m) for m in model.modules()) or kind == "own forward"


def test_models_whose_attention_wants_values_are_refused_whole():
    """DiffLlama, the text model of Qwen2.5-VL, Mllama's and Chameleon's layers ask the hidden states for their size (and Chameleon's norms
    stand behind, its results are tuples): refused before anything is replaced, and they run as before."""
    import transformers
    from transformers.models.chameleon import modeling_chameleon as chameleon
    from transformers.models.mllama import modeling_mllama as mllama
    from triattention_b200.kernels.linear import Int8DecoderLayer
    from triattention_b200.models import int8_projections
    small = dict(hidden_size=96, intermediate_size=160, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, vocab_size=200)
    ids = torch.arange(7)[None]
    for model in (toy("DiffLlama"), transformers.Qwen2_5_VLTextModel(transformers.Qwen2_5_VLTextModel.config_class(
            **small, rope_parameters=dict(rope_type="default", rope_theta=1e4, mrope_section=[2, 4, 6]))).eval()):
        with torch.no_grad():
            want = model(input_ids=ids, use_cache=False)[0]
            with pytest.raises(RuntimeError, match="no decoder layer"):
                int8_projections(model, ExactOps())
            assert torch.equal(model(input_ids=ids, use_cache=False)[0], want)
    config = transformers.ChameleonConfig(**small)
    for layer in (chameleon.ChameleonDecoderLayer(config, 0), chameleon.ChameleonSwinDecoderLayer(config, 0)):
        assert not Int8DecoderLayer.fits(layer)
    config = mllama.MllamaTextConfig(**small)
    config._attn_implementation = "eager"
    assert not Int8DecoderLayer.fits(mllama.MllamaSelfAttentionDecoderLayer(config, 0))


@pytest.mark.parametrize("kind", ["Ministral", "SmolLM3", "Cwm", "Ernie4_5"])
def test_other_models_of_the_kind_are_taken(kind):
    from triattention_b200.models import int8_projections
    model, ids = toy(kind, pad_token_id=0, bos_token_id=1, eos_token_id=2), torch.arange(3, 15)[None]
    with torch.no_grad():
        want = model(input_ids=ids, use_cache=False).logits
        got = int8_projections(model, ExactOps())(input_ids=ids, use_cache=False).logits
    torch.testing.assert_close(got, want, rtol=1e-4, atol=1e-4 * float(want.abs().max()))


def test_trying_a_layer_leaves_the_model_alone():
    """Whatever attention the model is set to is not called, and no setting of the model changes."""
    from transformers.modeling_utils import ALL_ATTENTION_FUNCTIONS
    from triattention_b200.models import int8_projections
    calls = []
    ALL_ATTENTION_FUNCTIONS["counted"] = lambda module, query, *a, **k: (calls.append(1), (query.transpose(1, 2).contiguous(), None))[1]
    model = toy("Llama").train()
    model.set_attn_implementation("counted")
    settings, weights = repr(model.config), [(n, p.data_ptr()) for n, p in model.named_parameters()]
    from triattention_b200.kernels.linear import Int8DecoderLayer
    assert all(Int8DecoderLayer.fits(layer) for layer in model.model.layers)
    assert not calls and repr(model.config) == settings and [(n, p.data_ptr()) for n, p in model.named_parameters()] == weights
    assert model.config._attn_implementation == "counted" and all(m.training for m in model.modules())
    int8_projections(model, ExactOps())
    assert not calls
    model(input_ids=torch.arange(4)[None], use_cache=False)
    assert len(calls) == 3


# ---- all of the model or nothing of it ---------------------------------------------------------------------------------------

def unchanged_by(model, ops, match):
    """int8_projections(model, ops) fails, and the model is what it was."""
    from triattention_b200.models import int8_projections
    before, ids = [(n, id(m)) for n, m in model.named_modules()], torch.arange(9)[None]
    with torch.no_grad():
        want = model(input_ids=ids, use_cache=False).logits
        with pytest.raises(RuntimeError, match=match):
            int8_projections(model, ops)
        assert [(n, id(m)) for n, m in model.named_modules()] == before
        assert torch.equal(model(input_ids=ids, use_cache=False).logits, want)


@pytest.mark.parametrize("at", [0, 1, 4, 5, 6, 11, 17])
def test_a_conversion_that_fails_leaves_the_model_whole(at):
    class Failing(ExactOps):
        calls = 0

        def quantize_rows(self, x):
            if self.calls == at:
                raise RuntimeError("no memory")
            self.calls += 1
            return super().quantize_rows(x)

    unchanged_by(toy("Llama", attention_bias=True), Failing(), "no memory")


def test_weights_of_several_types_are_refused():
    """Calls want the norm's weight and a bias in the type of the rows: said before anything is replaced, not by the first forward."""
    model = toy("Llama")
    model.model.layers[2].post_attention_layernorm.bfloat16()
    unchanged_by(model, ExactOps(), "one type")


def test_layers_that_share_an_attention_are_refused():
    model = toy("Llama")
    model.model.layers[1].self_attn = model.model.layers[0].self_attn
    unchanged_by(model, ExactOps(), "torch.nn.Linear")


def test_two_threads_get_one_error_word(lib, monkeypatch):
    """A word that nothing holds any more would be written to by kernels under way, and read by nobody."""
    import threading
    module, both, zeros = Module(lib), threading.Barrier(2, timeout=5), torch.zeros
    module._errors = {}

    def slow(*args, device=None, **kwargs):
        try:
            both.wait()
        except threading.BrokenBarrierError:        # (one thread alone)
            pass
        return zeros(*args, **kwargs)

    monkeypatch.setattr(extension.torch, "zeros", slow)
    words = []
    threads = [threading.Thread(target=lambda: words.append(module.error_word("cuda:0"))) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert words[0] is words[1] is module.error_word(torch.device("cuda", 0))


def test_error_words_are_the_process_s(lib, monkeypatch):
    """The projections of a model and the engine around it each loaded the library for themselves: what one's kernels report, the
    other's check (generate's, or any) must see."""
    one, other = Module(lib), Module(lib)
    monkeypatch.setitem(one._errors, 5, torch.tensor([1], dtype=torch.int32))
    with pytest.raises(RuntimeError, match="device error 1 on cuda:5"):
        other.check_device_error()
    other.check_device_error()                  # reported once


def test_an_error_word_made_in_inference_mode_is_reported_outside(lib):
    module = Module(lib)
    with torch.inference_mode():
        module._errors = {5: torch.tensor([1], dtype=torch.int32), 6: torch.zeros(1, dtype=torch.int32)}
    with pytest.raises(RuntimeError, match="device error 1 on cuda:5"):
        module.check_device_error()
    module.check_device_error()


def test_forward_mode_tangents_are_refused(lib):
    """Codes carry no tangent either: it would be dropped without a word, under no_grad as well (which is about the other mode)."""
    import torch.autograd.forward_ad as forward
    ops, x = Int8Ops(Module(lib)), torch.zeros(4, 64)
    weight, rows = torch.ones(64), Int8Rows(torch.zeros(4, 64, dtype=torch.int8), torch.ones(4))
    with forward.dual_level(), torch.no_grad():
        dual = forward.make_dual(x, torch.ones_like(x))
        for call in (lambda: ops.quantize_rows(dual), lambda: ops.silu_mul(x, dual), lambda: ops.rms_norm(x, weight, 1e-6, residual=dual),
                     lambda: ops.linear(rows, rows, residual=dual)):
            with pytest.raises(RuntimeError, match="no forward-mode"):
                call()
        with pytest.raises(RuntimeError, match="on a GPU"):     # (one without a tangent goes on to the next check)
            ops.quantize_rows(x)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda x: ops.quantize_rows(x).scales, (x,), (torch.ones_like(x),))
