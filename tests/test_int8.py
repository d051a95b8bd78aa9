"""8-bit integer layers on the CPU: the definition of the rows, refusals, training through the layers, serving through the engine."""
import copy

import pytest
import torch

from levanter_b200.nn import Linear, RmsNorm, linear_many, norm_for
from levanter_b200.ops import int8 as I
from levanter_b200.quantization import QuantizationConfig, quantize_for_serving, quantize_linear_layers
from levanter_b200.utils.activation import ActivationFunctionEnum as Act

BF = torch.bfloat16


def llama(**kw):
    from levanter_b200.models.llama import LlamaConfig

    cfg = dict(seq_len=64, hidden_dim=64, intermediate_dim=128, num_layers=2, num_heads=4, num_kv_heads=2, gradient_checkpointing=False)
    return LlamaConfig(**{**cfg, **kw})


def test_rows_and_back():
    torch.manual_seed(0)
    x = torch.randn(5, 3, 70) * torch.logspace(-3, 3, 3)[:, None]
    rows = I.quantize_rows(x)
    assert rows.shape == x.shape and rows.scale.shape == (5, 3) and rows.values.stride(1) % 16 == 0
    top = x.abs().amax(-1, keepdim=True)
    assert ((rows.dequantize(torch.float32) - x).abs() <= top / 254 * (1 + 1e-5)).all()
    assert (rows.values.abs().amax(-1) == 127).all()


def test_ties_go_to_the_even_number():
    x = torch.tensor([[127.0, 63.5, 0.5, 1.5, 2.5, -0.5, -1.5, -126.5], [1.0, 0.5, -0.5, 0, 0, 0, 0, 0]])
    assert I.quantize_rows(x).values.tolist() == [[127, 64, 0, 2, 2, 0, -2, -126], [127, 64, -64, 0, 0, 0, 0, 0]]


def test_special_rows():
    x = torch.zeros(5, 8)
    x[1, 2] = 1e-31
    x[2, 3] = float("nan")
    x[3, 4] = -float("inf")
    x[4, 5] = 2.0
    rows = I.quantize_rows(x)
    assert rows.scale[:2].tolist() == [0, 0] and rows.scale[2:4].isnan().all() and not rows.values[:4].any() and rows.values[4, 5] == 127


@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_rows_of_the_largest_numbers(dtype):
    m = torch.finfo(dtype).max  # as masks have it
    x = torch.tensor([[m, m / 2, -m / 2, m / 4, -m, m / 127 * 3, 1.0, 0.0], [-m] * 8], dtype=dtype)
    rows = I.quantize_rows(x)
    assert torch.equal(rows.values.double(), (127 * x.double() / x.double().abs().amax(-1, keepdim=True)).round())
    back = rows.dequantize(torch.float32)
    assert bool(back.isfinite().all()) and bool(((back[:, 4].double() + m).abs() <= 2.0 ** -22 * m).all())


def test_norm_with_its_residual_and_gated_activation():
    torch.manual_seed(1)
    x, r, w = torch.randn(6, 48).to(BF), torch.randn(6, 48).to(BF), (1 + 0.1 * torch.randn(48)).to(BF)
    rows, h = I.rms_norm_int8(x, w, 1e-5, residual=r)
    assert torch.equal(h, (x.float() + r.float()).to(BF))
    y = h.float() * torch.rsqrt(h.float().square().mean(-1, keepdim=True) + 1e-5) * w.float()
    assert ((rows.dequantize(torch.float32) - y).abs() <= y.abs().amax(-1, keepdim=True) / 254 * (1 + 1e-5)).all()
    assert I.rms_norm_int8(x, None)[1] is None
    y = torch.nn.functional.silu(x.float()) * r.float()
    assert ((I.gated_activation_int8(x, r, "silu").dequantize(torch.float32) - y).abs() <= y.abs().amax(-1, keepdim=True) / 254 * (1 + 1e-5)).all()


def test_product_is_exact_in_whole_numbers():
    torch.manual_seed(2)
    a = I.Int8Rows(torch.randint(-128, 128, (4, 300), dtype=torch.int8), torch.ones(4))
    b = I.Int8Rows(torch.randint(-128, 128, (7, 300), dtype=torch.int8), torch.ones(7))
    bias, res = torch.randn(7), torch.randn(4, 7)
    want = (a.values.long() @ b.values.long().t()).float()
    assert torch.equal(I.int8_product(a, b, out_dtype=torch.float32), want)
    assert torch.equal(I.int8_product(a, b, bias, res, out_dtype=torch.float32), want + bias + res)


@pytest.mark.parametrize("call, error", [
    (lambda x, w: I.quantize_rows(x.half()), TypeError),
    (lambda x, w: I.quantize_rows(x.int()), TypeError),
    (lambda x, w: I.quantize_rows(torch.tensor(1.0)), ValueError),
    (lambda x, w: I.quantize_rows(torch.zeros(3, 0)), ValueError),
    (lambda x, w: I.quantize_rows(x.clone().requires_grad_()), RuntimeError),
    (lambda x, w: I.quantize_rows(x).dequantize(torch.float16), TypeError),
    (lambda x, w: I.rms_norm_int8(x, torch.ones(7)), ValueError),
    (lambda x, w: I.rms_norm_int8(x, torch.ones(1, 16)), ValueError),
    (lambda x, w: I.rms_norm_int8(x, torch.ones(16).half()), ValueError),
    (lambda x, w: I.rms_norm_int8(x, torch.ones(16), residual=x[:2]), ValueError),
    (lambda x, w: I.rms_norm_int8(x, torch.ones(16), residual=x.to(BF)), ValueError),
    (lambda x, w: I.rms_norm_int8(x, torch.ones(16, requires_grad=True)), RuntimeError),
    (lambda x, w: I.gated_activation_int8(x, x[:, :8], Act.silu), ValueError),
    (lambda x, w: I.gated_activation_int8(x, x.to(BF), Act.silu), ValueError),
    (lambda x, w: I.gated_activation_int8(x, x, "no such thing"), ValueError),
    (lambda x, w: I.int8_product(I.Int8Rows(x, torch.ones(4)), w), TypeError),
    (lambda x, w: I.int8_product(I.Int8Rows(w.values, w.scale.double()), w), TypeError),
    (lambda x, w: I.int8_product(I.Int8Rows(w.values, w.scale[:3]), w), ValueError),
    (lambda x, w: I.int8_product(I.Int8Rows(w.values[:, :8], w.scale), w), ValueError),
    (lambda x, w: I.int8_product(w, I.Int8Rows(w.values[0], w.scale[0])), ValueError),
    (lambda x, w: I.int8_product(w, w, bias=torch.ones(5)), ValueError),
    (lambda x, w: I.int8_product(w, w, bias=torch.ones(4).half()), ValueError),
    (lambda x, w: I.int8_product(w, w, residual=torch.ones(4, 5)), ValueError),
    (lambda x, w: I.int8_product(w, w, residual=torch.ones(4, 4, requires_grad=True)), RuntimeError),
    (lambda x, w: I.int8_product(w, w, out_dtype=torch.float16), TypeError),
    (lambda x, w: I.int8_product(I.Int8Rows(torch.zeros(1, I.MAX_COLS + 1, dtype=torch.int8), torch.ones(1)),
                                 I.Int8Rows(torch.zeros(1, I.MAX_COLS + 1, dtype=torch.int8), torch.ones(1))), ValueError),
    (lambda x, w: I.int8_linear_many(x, []), ValueError),
    (lambda x, w: I.int8_linear_many(x, [torch.ones(3, 16)], []), ValueError),
    (lambda x, w: I.int8_linear(x, torch.ones(3, 17)), ValueError),
    (lambda x, w: I.int8_linear(x, torch.ones(3, 16), torch.ones(4)), ValueError),
    (lambda x, w: I.int8_linear(x.double(), torch.ones(3, 16)), TypeError),
    (lambda x, w: I.Int8ServingLinear(torch.ones(3, 16).half(), None), ValueError),
    (lambda x, w: quantize_for_serving(Linear(8, 8), QuantizationConfig(int8=True)), ValueError),
    (lambda x, w: quantize_for_serving(Linear(8, 8), QuantizationConfig(fp8=True)), ValueError),
    (lambda x, w: quantize_linear_layers(Linear(8, 8), QuantizationConfig(fp8=True, int8=True)), ValueError),
])
def test_refusals(call, error):
    torch.manual_seed(3)
    with pytest.raises(error):
        call(torch.randn(4, 16), I.quantize_rows(torch.randn(4, 16)))


def test_gradients_are_those_of_the_product_of_what_is_held():
    torch.manual_seed(4)
    x, w, b = torch.randn(2, 5, 24), torch.randn(7, 24), torch.randn(7)
    x, w, b = (t.requires_grad_() for t in (x, w, b))
    dy = torch.randn(2, 5, 7)
    y = I.int8_linear(x, w, b)
    gx, gw, gb = torch.autograd.grad(y, [x, w, b], dy)
    xh, wh = (I.quantize_rows(t.detach()).dequantize(torch.float32) for t in (x, w))
    torch.testing.assert_close(y, xh @ wh.t() + b, atol=2e-5, rtol=1e-5)
    torch.testing.assert_close(gx, dy @ wh, atol=2e-5, rtol=1e-5)
    torch.testing.assert_close(gw, dy.flatten(0, 1).t() @ xh.flatten(0, 1), atol=2e-5, rtol=1e-5)
    torch.testing.assert_close(gb, dy.sum((0, 1)), atol=2e-5, rtol=1e-5)


def test_quantize_linear_layers_trains_in_int8_under_the_same_names():
    from levanter_b200.models.lm_model import LmExample, compute_next_token_loss

    model = llama().build(100, seed=0)
    names = [n for n, _ in model.named_parameters()]
    plain = copy.deepcopy(model)
    quantize_linear_layers(model, QuantizationConfig(int8=True))
    assert [n for n, _ in model.named_parameters()] == names
    assert sum(isinstance(m, I.Int8Linear) for m in model.modules()) == 2 * 7 and type(model.lm_head) is Linear
    ex = LmExample.causal(torch.randint(0, 100, (2, 64), dtype=torch.int32))
    loss, want = compute_next_token_loss(model, ex), compute_next_token_loss(plain, ex)
    assert abs(loss.item() - want.item()) < 0.02
    loss.backward()
    want.backward()
    for (n, p), q in zip(model.named_parameters(), plain.parameters()):
        assert (p.grad - q.grad).norm() <= 0.2 * q.grad.norm() + 1e-6, n


def test_targets_choose_the_layers():
    model = quantize_linear_layers(llama().build(100, seed=0), QuantizationConfig(int8=True, targets="mlp"))
    assert isinstance(model.transformer.layers[0].mlp.gate_proj, I.Int8Linear) and type(model.transformer.layers[0].self_attn.q_proj) is Linear
    model = quantize_for_serving(llama().build(100, seed=0), QuantizationConfig(int8=True, targets=["down_proj"]))
    assert sum(isinstance(m, I.Int8ServingLinear) for m in model.modules()) == 2


def test_one_quantisation_for_all_readers(monkeypatch):
    calls = []
    monkeypatch.setattr(I, "_quantize", lambda x, real=I._quantize: calls.append(1) or real(x))
    mods = [I.Int8ServingLinear(torch.randn(n, 32), torch.randn(n) if n == 8 else None) for n in (8, 16, 4)]
    calls.clear()
    x = torch.randn(3, 32)
    with torch.no_grad():
        ys = linear_many(x, *mods)
    assert len(calls) == 1
    for m, y in zip(mods, ys):
        assert torch.equal(y, m(x))


def test_norm_for_makes_rows_only_for_readers_of_rows():
    norm, x, r = RmsNorm(32).to(BF), torch.randn(3, 32).to(BF), torch.randn(3, 32).to(BF)
    mods = [I.Int8ServingLinear(torch.randn(8, 32).to(BF), None) for _ in range(2)]
    with torch.no_grad():
        rows, h = norm_for(norm, x, mods, residual=r)
        assert isinstance(rows, I.Int8Rows) and torch.equal(h, x + r)
        assert isinstance(norm_for(norm, x, mods)[0], I.Int8Rows) and norm_for(norm, x, mods)[1] is x
        for others in ([], mods[:1] + [Linear(32, 8)]):
            y, h = norm_for(norm, x, others, residual=r)
            assert torch.equal(y, norm(x + r)) and torch.equal(h, x + r)
        mods[0].register_forward_hook(lambda *a: None)  # a hook has to see a tensor
        assert isinstance(norm_for(norm, x, mods)[0], torch.Tensor)
    assert isinstance(norm_for(norm, x, mods[1:])[0], torch.Tensor)  # gradients are recorded


def test_serving_weights_survive_moves_and_state_dicts():
    m = I.Int8ServingLinear(torch.randn(8, 20), torch.randn(8))
    x = torch.randn(3, 20)
    with torch.no_grad():
        y = m(x)
    scale = m.weight_scale.clone()
    m.to(BF)
    assert m.weight.dtype == torch.int8 and torch.equal(m.weight_scale, scale) and m.bias.dtype == BF
    other = I.Int8ServingLinear(torch.zeros(8, 20), torch.zeros(8))
    other.load_state_dict({k: v.float() if k == "bias" else v for k, v in m.state_dict().items()})
    with torch.no_grad():
        assert (other(x) - y).abs().max() <= 2.0 ** -8 * 4


@pytest.mark.parametrize("kw", [dict(), dict(hybrid_norm=True), dict(use_bias=True), dict(head_dim=24)])
def test_engine_serves_weights_held_in_8_bits(kw):
    """The engine's tokens are those that the quantised model gives without a cache."""
    from levanter_b200.data.passthrough_tokenizer import PassthroughTokenizer
    from levanter_b200.inference.engine import InferenceEngine, InferenceEngineConfig, Request
    from levanter_b200.inference.jit_scheduler import SeqDecodingParams
    from levanter_b200.layers.attention import AttentionMask

    model = llama(**kw).build(100, seed=0).eval()
    bytes_before = sum(p.nbytes for p in model.parameters())
    cfg = InferenceEngineConfig(max_pages=32, max_seqs=4, page_size=8, max_pages_per_seq=8, compute_dtype=torch.float32, quantization=QuantizationConfig(int8=True))
    with torch.no_grad():
        engine = InferenceEngine.from_model_with_config(model, PassthroughTokenizer(100), cfg)
        assert sum(isinstance(m, I.Int8ServingLinear) for m in model.modules()) == 2 * 7
        assert sum(p.nbytes for p in model.parameters()) < 0.5 * bytes_before
        prompts = [[3, 14, 15, 92], [65, 35, 8, 9, 79, 32, 38]]
        reqs = [Request(prompt_tokens=p, request_id=i, decode_params=SeqDecodingParams(len(p) + 6, None, 0.0, i), n_generations=1) for i, p in enumerate(prompts)]
        got = engine.generate(reqs).tokens
        for p, out in zip(prompts, got):
            seq = list(p)
            for t in out:
                logits = model(torch.tensor([seq], dtype=torch.int32), AttentionMask.causal())
                logits = getattr(logits, "array", logits)[0, -1].float()
                assert logits[t] >= logits.max() - 0.02  # (a cache of other widths sums in another order)
                seq.append(int(t))
    assert quantize_for_serving(model, cfg.quantization) is model


@pytest.mark.parametrize("kw, targets", [(dict(), None), (dict(hybrid_norm=True), None), (dict(use_bias=True), None), (dict(), ["gate_proj", "up_proj"]), (dict(), ["q_proj", "down_proj"]),
                                         (dict(), ["q_proj", "k_proj", "v_proj", "o_proj"]), (dict(), ["up_proj"])])
def test_bf16_engine_takes_rows_from_the_norms_where_all_readers_do(kw, targets):
    from levanter_b200.data.passthrough_tokenizer import PassthroughTokenizer
    from levanter_b200.inference.engine import InferenceEngine, InferenceEngineConfig, Request
    from levanter_b200.inference.jit_scheduler import SeqDecodingParams
    from levanter_b200.layers.attention import AttentionMask

    quant = QuantizationConfig(int8=True) if targets is None else QuantizationConfig(int8=True, targets=targets)
    model = quantize_for_serving(llama(**kw).build(100, seed=0).eval(), quant).to(BF)  # (a conversion after the weights were quantised)
    cfg = InferenceEngineConfig(max_pages=32, max_seqs=4, page_size=8, max_pages_per_seq=8, compute_dtype=BF)
    with torch.no_grad():
        engine = InferenceEngine.from_model_with_config(model, PassthroughTokenizer(100), cfg)
        prompts = [[3, 14, 15, 92], [65, 35, 8, 9, 79, 32, 38]]
        reqs = [Request(prompt_tokens=p, request_id=i, decode_params=SeqDecodingParams(len(p) + 4, None, 0.0, i), n_generations=1) for i, p in enumerate(prompts)]
        for p, out in zip(prompts, engine.generate(reqs).tokens):
            logits = model(torch.tensor([p], dtype=torch.int32), AttentionMask.causal())
            logits = getattr(logits, "array", logits)[0, -1].float()
            # the paged path forms its norms in 32 bits ahead of the 8 bits, the other rounds them to bf16: some steps of 2^-8 per layer, of logits below 1
            assert logits.abs().max() < 1 and logits[out[0]] >= logits.max() - 0.05


def test_results_have_the_type_of_the_rows():
    m = I.Int8ServingLinear(torch.randn(8, 32), None)
    x = torch.randn(3, 32)
    with torch.no_grad():
        assert m(x).dtype == torch.float32 and m(x.to(BF)).dtype == BF and m(I.quantize_rows(x)).dtype == BF
        assert [y.dtype for y in linear_many(x, m, m)] == [torch.float32] * 2


@pytest.mark.parametrize("call", [lambda r: r.dequantize(), lambda r: I.int8_product(r, r), lambda r: I.int8_product(I.Int8Rows(r.values, r.scale.detach()), r)])
def test_scales_that_want_a_gradient_are_refused(call):
    rows = I.quantize_rows(torch.randn(4, 16))
    rows = I.Int8Rows(rows.values, rows.scale.requires_grad_())
    with pytest.raises(RuntimeError):
        call(rows)
    with torch.no_grad():
        call(rows)


def test_a_single_row_without_a_leading_dimension():
    x, w, bias = torch.randn(20), I.quantize_rows(torch.randn(7, 20)), torch.randn(7)
    row = I.quantize_rows(x)
    assert row.scale.shape == () and I.int8_product(row, w, bias).shape == (7,)
    assert torch.equal(I.int8_product(row, w, bias), I.int8_product(I.quantize_rows(x[None]), w, bias)[0])
    assert torch.equal(I.rms_norm_int8(x, None, residual=x)[1], x + x) and row.dequantize().shape == (20,)


def test_rows_without_elements_come_back_empty():
    assert I.Int8Rows(torch.empty(3, 0, dtype=torch.int8), torch.empty(3)).dequantize().shape == (3, 0)
    assert I.quantize_rows(torch.empty(0, 16)).dequantize().shape == (0, 16)


def test_weights_of_a_model_that_was_not_quantised_are_quantised_as_they_load():
    plain = llama().build(100, seed=1)
    want = quantize_for_serving(copy.deepcopy(plain), QuantizationConfig(int8=True))
    model = quantize_for_serving(llama().build(100, seed=0), QuantizationConfig(int8=True))
    state = plain.state_dict()
    before = {k: v.clone() for k, v in state.items()}
    model.load_state_dict(state)
    assert state.keys() == before.keys() and all(torch.equal(state[k], before[k]) for k in state)
    for (n, a), (_, b) in zip(model.state_dict().items(), want.state_dict().items()):
        assert a.dtype == b.dtype and torch.equal(a, b), n
    with pytest.raises(RuntimeError):
        I.Int8ServingLinear(torch.zeros(8, 20), None).load_state_dict({"weight": torch.zeros(8, 21)})


def test_engine_config_takes_the_quantization_from_a_file():
    from levanter_b200.config import decode
    from levanter_b200.inference.engine import InferenceEngineConfig

    cfg = decode(InferenceEngineConfig, {"max_seqs": 2, "quantization": {"int8": True, "targets": ["mlp"]}})
    assert cfg.quantization.int8 and cfg.quantization.matches("layers.0.mlp.up_proj") and not cfg.quantization.matches("layers.0.self_attn.q_proj")


@pytest.mark.parametrize("family", ["fedolorn", "zadepel", "zosipel", "mumizen"])
@pytest.mark.parametrize("name", ["mixed", "odd"])
def test_other_decoders_serve_weights_held_in_8_bits(family, name, tmp_path):
    """Attention without positions, with gates, windows, differences and mixed values: the tokens are those of the same layers as training computes them."""
    import importlib
    import json

    import test_fedolorn as F
    from levanter_b200.inference.engine import Request
    from levanter_b200.inference.jit_scheduler import SeqDecodingParams
    from levanter_b200.layers.attention import Attention
    from levanter_b200.models.llama import LlamaMlp
    from safetensors.torch import save_file

    cfg = importlib.import_module(f"test_{family}")._config(name)
    (tmp_path / "config.json").write_text(json.dumps(cfg))
    save_file(importlib.import_module(f"{family}_oracle").random_weights(cfg, seed=3), str(tmp_path / "model.safetensors"))
    place = ("cpu", torch.float32)
    tokens, counts = [], []
    with torch.no_grad():
        for serving in (False, True):
            model = F._load(str(tmp_path), place)
            if serving:
                quantize_for_serving(model, QuantizationConfig(int8=True))
            else:
                for m in [m for m in model.modules() if isinstance(m, (Attention, LlamaMlp))]:
                    for child_name, child in list(m.named_children()):
                        if type(child) is Linear:
                            setattr(m, child_name, I.Int8Linear.from_linear(child))
            counts.append(sum(isinstance(m, (I.Int8Linear, I.Int8ServingLinear)) for m in model.modules()))
            prompts = [[1, 2, 3, 4, 5, 6, 7], [9, 8, 7]]
            reqs = [Request(prompt_tokens=p, request_id=i, decode_params=SeqDecodingParams(len(p) + 6, None, 0.0, i), n_generations=1) for i, p in enumerate(prompts)]
            tokens.append(F._engine(model, place).generate(reqs).tokens)
    assert counts[0] == counts[1] > 0 and tokens[0] == tokens[1]


def test_checkpoints_neither_read_nor_write_weights_held_in_8_bits(tmp_path):
    from levanter_b200.checkpoint import load_model_params, save_checkpoint
    from levanter_b200.compat.hf_checkpoints import load_hf_state_dict, to_hf_state_dict

    model = llama().build(100, seed=0)
    state = to_hf_state_dict(model)
    quantize_for_serving(model, QuantizationConfig(int8=True))
    for call in (lambda: to_hf_state_dict(model), lambda: load_hf_state_dict(model, state), lambda: load_model_params(model, str(tmp_path)),
                 lambda: save_checkpoint(model, 0, str(tmp_path / "out"))):
        with pytest.raises(ValueError, match="held in 8 bits"):
            call()


@pytest.mark.parametrize("swap", [False, True])
def test_product_of_the_largest_numbers(swap):
    """Scales as rows of up to 3e38 have them: results that fit into fp32 are right, the others infinite, zeros stay zeros."""
    torch.manual_seed(5)
    a = I.Int8Rows(torch.randint(-127, 128, (5, 64), dtype=torch.int8), torch.tensor([I.MOST_SCALE, 2.0 ** 100, 2.0 ** 64, 1.0, 2.0 ** -60]))
    b = I.Int8Rows(torch.randint(-127, 128, (6, 64), dtype=torch.int8), torch.tensor([2.0 ** -60, 1e-9, 0.01, 1.0, 2.0 ** 40, 0.0]))
    a.values[:, :] = a.values.abs()
    b.values[:5] = b.values[:5].abs()  # sums of some 2^18 and more
    a, b = (b, a) if swap else (a, b)
    got = I.int8_product(a, b, out_dtype=torch.float32).double()
    want = (a.values.double() @ b.values.double().t()) * a.scale.double()[:, None] * b.scale.double()
    fits = want.abs() < torch.finfo(torch.float32).max
    assert 20 < int(fits.sum()) < 30 and bool(((got - want).abs() <= 3 * 2.0 ** -24 * want.abs())[fits].all()) and got[~fits].isinf().all()  # three roundings


@pytest.mark.parametrize("size, eps", [(1e20, 1e-6), (1e30, 1e-6), (3e37, 1e-6), (1e-15, 0.0), (1e-22, 0.0), (1e-30, 0.0)])
@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_norms_whose_squares_leave_the_range_of_fp32(size, eps, dtype):
    torch.manual_seed(6)
    x, w = (torch.randn(4, 96).clamp(-5, 5) * size).to(dtype), 1 + 0.1 * torch.randn(96)
    x[1] = 0
    x[2] = torch.randn(96).to(dtype)  # an ordinary row
    rows, _ = I.rms_norm_int8(x, w, eps if eps else 0.0)
    d = x.double()
    y = (d * torch.rsqrt(d.square().mean(-1, keepdim=True) + eps)).nan_to_num() * w.double()
    live = [0, 2, 3]
    assert ((rows.dequantize(torch.float32).double() - y).abs() <= y.abs().amax(-1, keepdim=True) / 254 * (1 + 1e-5))[live].all()
    assert (rows.values.abs().amax(-1) == 127)[live].all()
    x[3, 5], x[0, 7] = float("inf"), float("nan")
    assert I.rms_norm_int8(x, w, eps)[0].scale.isnan().tolist()[0::3] == [True, True]


def test_norms_of_zeros_without_an_eps():
    rows, _ = I.rms_norm_int8(torch.zeros(3, 40), None, 0.0)
    assert not rows.values.any() and not rows.scale.any()  # (as on the GPU)
    rows, _ = I.rms_norm_int8(torch.randn(3, 40), torch.zeros(40), 0.0)
    assert not rows.values.any() and not rows.scale.any()


def test_memory_accesses_in_assembly_keep_their_place():
    """Kernels start before the kernel ahead of them has finished: a load that is not volatile could move ahead of the wait for what it reads."""
    import re
    from pathlib import Path

    import levanter_b200.ops

    csrc = Path(levanter_b200.ops.__file__).parent / "csrc"
    free = [f"{p.name}: {m.group(1)}" for p in sorted(csrc.glob("*.cu*")) for m in re.finditer(r'\basm\s*\(\s*"([^"]*)', p.read_text())]
    assert free and not [f for f in free if re.search(r": (\{|\\n|\\t|\s)*(ld|st|atom|red|cp)\.", f)]


@pytest.mark.parametrize("bias", [False, True])
def test_products_without_a_kernel_round_once(bias):
    """The operands stay what the whole numbers stand for; the result is rounded to the rows' type, and so are the gradients."""
    torch.manual_seed(7)
    x, w, b = torch.randn(64, 100).to(BF), torch.randn(31, 100).to(BF), torch.randn(31).to(BF) if bias else None
    xh, wh = (I.quantize_rows(t).dequantize(torch.float32).double() for t in (x, w))
    x.requires_grad_(), w.requires_grad_()
    y, dy = I.int8_linear(x, w, b), torch.randn(64, 31).to(BF)
    gx, gw = torch.autograd.grad(y, [x, w], dy)
    want = xh @ wh.t() + (b.double() if bias else 0)
    size = xh.abs() @ wh.abs().t() + 10
    # sums of 101 numbers in fp32 (and what is held, off by two roundings of the dequantisation and two of the difference), one rounding to bf16
    assert y.dtype == BF and ((y.double() - want).abs() <= 2.0 ** -8 * want.abs() + 110 * 2.0 ** -24 * size).all()
    d = dy.double()
    assert gx.dtype == BF and ((gx.double() - d @ wh).abs() <= 2.0 ** -8 * (d @ wh).abs() + 110 * 2.0 ** -24 * (d.abs() @ wh.abs())).all()
    assert ((gw.double() - d.t() @ xh).abs() <= 2.0 ** -8 * (d.t() @ xh).abs() + 110 * 2.0 ** -24 * (d.abs().t() @ xh.abs())).all()


def test_fp32_streams_get_results_that_were_not_rounded_to_bf16():
    """What ends a block is added to an fp32 stream, or normed in fp32, as the product's epilogue has it."""
    from levanter_b200.layers.attention import Attention, AttentionConfig
    from levanter_b200.models.llama import LlamaMlp

    torch.manual_seed(8)
    x, stream = torch.randn(5, 64).to(BF), torch.randn(5, 64)
    with torch.no_grad():
        mlp = quantize_for_serving(LlamaMlp(64, 96, Act.silu, init_std=0.2), QuantizationConfig(int8=True, targets=["down_proj"])).to(BF)
        down = mlp.down_proj
        want = I.int8_product(I.quantize_rows(mlp._inner(x)), down.rows, out_dtype=torch.float32)
        assert not torch.equal(want, want.to(BF).float())
        assert torch.equal(mlp.forward_fp32(x), want) and torch.equal(mlp.add_to_stream(stream, x), want + stream)
        assert torch.equal(mlp.add_to_stream(stream.view(1, 5, 64), x.view(1, 5, 64)), (want + stream).view(1, 5, 64))
        attn = quantize_for_serving(Attention(AttentionConfig(64, 4, 2)), QuantizationConfig(int8=True)).to(BF)
        attn._paged_heads = lambda *a: (x, None)
        want = I.int8_product(I.quantize_rows(x), attn.o_proj.rows, out_dtype=torch.float32)
        assert torch.equal(attn.paged_decode_mixing_values(x, None, None, None)[0], want)
        assert torch.equal(attn.paged_decode_stream(x, None, None, None, stream)[0], want + stream)


@pytest.mark.parametrize("act", ["silu", "tanh"])
def test_blocks_on_an_fp32_stream_quantise_their_rows_once(act, monkeypatch):
    """Once for gate and up, and the gated activation as it is made, in 32 bits."""
    from levanter_b200.models.llama import LlamaMlp

    torch.manual_seed(9)
    x, stream = torch.randn(5, 64).to(BF), torch.randn(5, 64)
    mlp = quantize_for_serving(LlamaMlp(64, 96, Act(act), init_std=0.2), QuantizationConfig(int8=True)).to(BF).eval()
    with torch.no_grad():
        gate, up = linear_many(x, mlp.gate_proj, mlp.up_proj)
        want = I.int8_product(I.gated_activation_int8(gate, up, mlp.act), mlp.down_proj.rows, out_dtype=torch.float32)
        calls = []
        monkeypatch.setattr(I, "_quantize", lambda x, real=I._quantize: calls.append(1) or real(x))
        assert torch.equal(mlp.forward_fp32(x), want) and torch.equal(mlp.add_to_stream(stream, x), want + stream)
        assert len(calls) == (2 if act == "silu" else 4)  # (an activation without a kernel of its own is quantised as it comes)
        calls.clear()
        mlp.down_proj.register_forward_hook(lambda *a: None)  # then it has to see the rows
        mlp.forward_fp32(x)
        assert len(calls) == 2
    model = LlamaMlp(64, 96, Act(act))
    quantize_linear_layers(model, QuantizationConfig(int8=True))
    calls, many = [], I._straight_through
    monkeypatch.setattr(I, "_straight_through", lambda x: calls.append(x.shape) or many(x))
    with torch.no_grad():
        model.forward_fp32(torch.randn(5, 64))
    assert calls.count((5, 64)) == 1 and calls.count((5, 96)) == 1


@pytest.mark.parametrize("watch", ["pre_hook", "hook", "subclass", "instance", "attention subclass", "attention instance"])
def test_layers_that_are_watched_get_tensors(watch):
    """Rows in 8 bits are handed to the layers' own code only."""
    from levanter_b200.data.passthrough_tokenizer import PassthroughTokenizer
    from levanter_b200.inference.engine import InferenceEngine, InferenceEngineConfig, Request
    from levanter_b200.inference.jit_scheduler import SeqDecodingParams
    from levanter_b200.layers.attention import Attention
    from levanter_b200.models.llama import LlamaMlp

    seen = []

    class Mlp(LlamaMlp):
        def forward(self, x, residual=None):
            seen.append(x)
            return super().forward(x, residual)

    class Attn(Attention):
        def paged_decode(self, x, *args, **kw):
            seen.append(x)
            return super().paged_decode(x, *args, **kw)

    model = quantize_for_serving(llama().build(100, seed=0).eval(), QuantizationConfig(int8=True)).to(BF)
    layer = model.transformer.layers[1]
    if watch == "pre_hook":
        layer.mlp.register_forward_pre_hook(lambda m, args: seen.append(args[0]))
    elif watch == "hook":
        layer.mlp.register_forward_hook(lambda m, args, out: seen.append(args[0]))
    elif watch == "subclass":
        layer.mlp.__class__ = Mlp
    elif watch == "instance":
        layer.mlp.forward = lambda x, residual=None: (seen.append(x), LlamaMlp.forward(layer.mlp, x, residual))[1]
    elif watch == "attention subclass":
        layer.self_attn.__class__ = Attn
    else:
        layer.self_attn.paged_decode = lambda x, *a, **kw: (seen.append(x), Attention.paged_decode(layer.self_attn, x, *a, **kw))[1]
    with torch.no_grad():
        engine = InferenceEngine.from_model_with_config(model, PassthroughTokenizer(100), InferenceEngineConfig(max_pages=32, max_seqs=4, page_size=8, max_pages_per_seq=8, compute_dtype=BF))
        engine.generate([Request(prompt_tokens=[3, 4, 5], request_id=0, decode_params=SeqDecodingParams(6, None, 0.0, 0), n_generations=1)])
    assert seen and all(type(x) is torch.Tensor and x.dtype == BF for x in seen)


@pytest.mark.parametrize("no_grad", [False, True])
def test_tangents_are_refused_or_kept_but_not_dropped(no_grad):
    import contextlib

    import torch.autograd.forward_ad as ad

    torch.manual_seed(10)
    x, t, w = torch.randn(4, 16), torch.randn(4, 16), I.quantize_rows(torch.randn(16, 16))
    rows = I.quantize_rows(x)
    with torch.no_grad() if no_grad else contextlib.nullcontext(), ad.dual_level():
        d, s = ad.make_dual(x, t), ad.make_dual(rows.scale, rows.scale)
        for call in (lambda: I.quantize_rows(d), lambda: I.rms_norm_int8(d, None), lambda: I.rms_norm_int8(x, None, residual=d), lambda: I.rms_norm_int8(x, d[0]),
                     lambda: I.gated_activation_int8(d, x, Act.silu), lambda: I.gated_activation_int8(x, d, "tanh"), lambda: I.int8_product(rows, w, residual=d),
                     lambda: I.int8_product(rows, w, bias=d[0]), lambda: I.int8_product(I.Int8Rows(rows.values, s), w), lambda: I.Int8Rows(rows.values, s).dequantize()):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        I.int8_product(I.quantize_rows(x), w, residual=x)  # others go on as ever
        weight = torch.randn(5, 16)
        y = ad.unpack_dual(I.int8_linear(d, weight))
        torch.testing.assert_close(y.tangent, t @ I.quantize_rows(weight).dequantize(torch.float32).t(), atol=2e-5, rtol=1e-5)
    assert torch.equal(I.quantize_rows(x).values, rows.values)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda a: I.quantize_rows(a).scale, (x,), (t,))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda a: I.quantize_rows(a).scale.sum())(x)


def test_weights_of_any_width_stay_where_products_read_them(tmp_path):
    """Rows of a width that is no multiple of 16 lie apart; moves, copies and loads keep them so."""
    torch.manual_seed(11)
    m = I.Int8ServingLinear(torch.randn(8, 20), None)
    values, x = m.weight.clone(), torch.randn(3, 20)
    with torch.no_grad():
        y = m(x)
    state = m.state_dict()
    torch.save(state, tmp_path / "state.pt")
    packed = {k: v.contiguous() for k, v in torch.load(tmp_path / "state.pt").items()}
    steps = [lambda: m._apply(lambda t: t.contiguous().clone()), lambda: m.load_state_dict(packed), lambda: m.load_state_dict(packed, assign=True), lambda: m.load_state_dict(state, assign=True), lambda: m.to(BF),
             lambda: copy.deepcopy(m), lambda: m.to("meta") and m.to_empty(device="cpu").load_state_dict(packed)]
    for step in steps:
        got = step()
        for mod in (m, got) if isinstance(got, I.Int8ServingLinear) else (m,):
            assert mod.weight.stride() == (32, 1)
            if mod.weight.device.type != "meta":
                assert torch.equal(mod.weight, values)
    with torch.no_grad():
        assert torch.equal(m(x), y)
    wide = I.Int8ServingLinear(torch.randn(8, 32), None)
    assert wide.to(BF).weight is wide.weight and wide.weight.stride() == (32, 1)


def test_the_launcher_module_is_built_where_it_can_be(tmp_path, monkeypatch):
    """Missing or of another source: built when it is first wanted.  What cannot be built keeps nothing else from being built."""
    from levanter_b200.ops import build as B
    from levanter_b200.ops import lib

    src = B.CSRC / "host" / "launcher.c"
    (tmp_path / "csrc" / "host").mkdir(parents=True)
    mine = tmp_path / "csrc" / "host" / "launcher.c"
    mine.write_bytes(src.read_bytes())
    monkeypatch.setattr(B, "CSRC", tmp_path / "csrc")
    monkeypatch.setattr(B, "LIBDIR", tmp_path / "lib")
    module = lib._launcher.__wrapped__()
    assert module is not None and (tmp_path / "lib" / B.LAUNCHER).exists()
    first = (tmp_path / "lib" / B.LAUNCHER).stat().st_mtime_ns
    assert B.build_launcher() is not None and (tmp_path / "lib" / B.LAUNCHER).stat().st_mtime_ns == first
    mine.write_text(mine.read_text() + "\n// another\n")
    assert B.build_launcher() is not None and (tmp_path / "lib" / B.LAUNCHER).stat().st_mtime_ns != first
    mine.write_text("#error no such calling convention\n")
    with pytest.warns(UserWarning, match="ctypes"):
        assert B.build_launcher() is None
    with pytest.warns(UserWarning):
        assert lib._launcher.__wrapped__() is None  # not the module of the other source
    monkeypatch.setattr(B.shutil, "which", lambda name: None)
    assert B.build_launcher() is None


def test_what_a_graph_reads_one_by_one_stays_where_it_is():
    """Laying weights out moves nothing of a layer whose weights a recorded graph reads where they lie."""
    from levanter_b200.layers.attention import Attention, AttentionConfig
    from levanter_b200.models.llama import LlamaMlp

    attn = quantize_for_serving(Attention(AttentionConfig(64, 4, 2, head_dim=64, use_bias=True)), QuantizationConfig(int8=True))
    mods = attn._projections()
    attn._rows._held.update(m.weight.data_ptr() for m in mods)  # as hold() notes them under capture
    attn._scale_rows._held.update(m.weight_scale.data_ptr() for m in mods)
    mlp = quantize_for_serving(LlamaMlp(64, 96, Act.silu), QuantizationConfig(int8=True))
    mlp._rows._held.update((mlp.gate_proj.weight.data_ptr(),))
    tensors = [t for m in mods + [mlp.gate_proj, mlp.up_proj] for t in (m.weight, m.weight_scale, m.bias) if t is not None]
    before = [t.data_ptr() for t in tensors]
    attn.lay_out_for_serving()
    mlp.lay_out_for_serving()
    assert [t.data_ptr() for t in tensors] == before


@pytest.mark.parametrize("path", ["forward", "forward_fp32", "add_to_stream"])
@pytest.mark.parametrize("targets", [None, ["gate_proj", "up_proj"]])
def test_weights_read_one_by_one_are_noted(path, targets, monkeypatch):
    from levanter_b200.models.llama import LlamaMlp
    from levanter_b200.nn import FusedRows

    noted = []
    monkeypatch.setattr(FusedRows, "hold", lambda self, params: noted.extend(p.data_ptr() for p in params))
    mlp = quantize_for_serving(LlamaMlp(64, 96, Act.silu), QuantizationConfig(int8=True, targets=targets)).eval()
    x = torch.randn(300, 64)
    with torch.no_grad():
        mlp.add_to_stream(x, x) if path == "add_to_stream" else getattr(mlp, path)(x)
    assert {t.data_ptr() for m in (mlp.gate_proj, mlp.up_proj) for t in (m.weight, m.weight_scale)} <= set(noted)


def test_what_is_refused_is_left_as_it_was():
    """Quantising for serving changes a model in place: not before all of it can be done."""
    from levanter_b200.data.passthrough_tokenizer import PassthroughTokenizer
    from levanter_b200.inference.engine import InferenceEngine, InferenceEngineConfig
    from levanter_b200.models.gemma import GemmaConfig

    def untouched(model):
        return not any(isinstance(m, I.Int8ServingLinear) for m in model.modules())

    model = llama().build(100, seed=0)
    model.transformer.layers[1].mlp.half()
    with pytest.raises(ValueError, match="float16"):
        quantize_for_serving(model, QuantizationConfig(int8=True))
    assert untouched(model)
    model = GemmaConfig(seq_len=64, hidden_dim=64, intermediate_dim=128, num_layers=1, num_heads=4, num_kv_heads=2, gradient_checkpointing=False).build(100, seed=0)
    cfg = InferenceEngineConfig(max_pages=32, max_seqs=4, page_size=8, max_pages_per_seq=8, compute_dtype=torch.float32, quantization=QuantizationConfig(int8=True))
    with pytest.raises(AttributeError):  # the engine has no cache for it
        InferenceEngine.from_model_with_config(model, PassthroughTokenizer(100), cfg)
    assert untouched(model)
