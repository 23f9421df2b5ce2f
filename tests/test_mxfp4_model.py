"""A base in 4 bits under adapters and behind the engine (CPU): it computes what the same model with the quantised values in 16 (here
32) bits computes, its files and counts stay whole, and what cannot be quantised is refused."""
import copy

import pytest
import torch

from lumen.lora import LoraConfig, apply_lora, count_parameters, merge_lora, quantize_base
from lumen.models import build_model
from lumen.models.layers import Linear
from lumen.ops.mxfp4 import MXFP4, mxfp4_quantize


def pair(name="tiny-llama-gqa", lora=True, seed=0):
    """(a model with its base in 4 bits, the same model with the values of that base)."""
    torch.manual_seed(seed)
    m = build_model(name, dtype=torch.float32, init="random", seed=seed)
    if lora:
        apply_lora(m, LoraConfig(r=4, lora_dropout=0.0))
        with torch.no_grad():
            for p in m.parameters():
                if p.requires_grad:
                    p.normal_(0, 0.1)
    plain = copy.deepcopy(m)
    freed = quantize_base(m)
    assert freed > 0
    with torch.no_grad():
        for (n, q), (_, p) in zip(m.named_modules(), plain.named_modules()):
            if isinstance(q, Linear) and not n.endswith("lm_head"):
                assert type(q.qweight) is MXFP4 and q.weight.numel() == 0
                p.weight.copy_(q.qweight.dequantize(torch.float32))
            elif isinstance(q, Linear):
                assert q.qdata is None
    return m, plain


def close(a, b):
    """Equal but for the order of fp32 sums: 1e-5 of the largest value (sums of up to 700 terms, 2^-24 each, through four layers)."""
    assert (a - b).abs().max() <= 1e-5 * b.abs().max()


@pytest.mark.parametrize("name", ["tiny-llama-gqa", "tiny-opt"])
@pytest.mark.parametrize("policy", ["none", "true"])
def test_loss_and_adapter_gradients(name, policy):
    m, plain = pair(name)
    ids = torch.randint(3, m.config.vocab_size, (2, 24))
    grads = []
    for model in (m, plain):
        model.train()
        model.gradient_checkpointing = policy
        loss = model(ids, labels=torch.roll(ids, -1, 1))
        loss.backward()
        grads.append((loss.detach(), [p.grad for p in model.parameters() if p.requires_grad]))
    close(grads[0][0], grads[1][0])
    assert len(grads[0][1]) == len(grads[1][1]) > 0
    for a, b in zip(grads[0][1], grads[1][1]):
        close(a, b)


def test_counts_files_and_merge(tmp_path):
    m, plain = pair()
    assert count_parameters(m) == count_parameters(plain)
    from lumen.models.loading import load_hf_weights, save_hf_weights

    save_hf_weights(m, str(tmp_path))
    again = build_model("tiny-llama-gqa", dtype=torch.float32, init="random", seed=9)
    load_hf_weights(again, str(tmp_path))
    for k, v in again.state_dict().items():
        assert torch.equal(v, plain.state_dict()[k])
    merge_lora(m), merge_lora(plain)
    assert all(getattr(x, "qdata", None) is None for x in m.modules() if isinstance(x, Linear) and x.seg_names == ["o_proj"])
    for (n, p) in plain.named_modules():
        if n.endswith("qkv_proj"):
            close(dict(m.named_modules())[n].weight, p.weight)


def test_quantised_bases_move_copy_and_come_back():
    m, plain = pair(lora=False)
    lin = m.layers[0].mlp.down_proj
    assert copy.deepcopy(lin).qweight.shape == lin.qweight.shape == (256, 688)
    assert lin.to(torch.bfloat16).qdata.dtype == torch.uint8
    codes = lin.qweight.codes
    quantize_base(m)                                      # a second time: nothing to do
    assert torch.equal(lin.qweight.codes, codes)
    lin.dequantize_base()
    assert lin.qdata is None and torch.equal(lin.weight.float(), plain.layers[0].mlp.down_proj.weight)
    lin.quantize_base()
    assert torch.equal(lin.qweight.codes, codes)          # quantised values stay what they are


def test_state_dict_holds_the_base():
    m, _ = pair(lora=False, seed=3)
    other, _ = pair(lora=False, seed=4)
    other.load_state_dict(m.state_dict())
    for a, b in zip(m.modules(), other.modules()):
        if isinstance(a, Linear) and a.qdata is not None:
            assert torch.equal(a.qdata, b.qdata)
    whole = build_model("tiny-llama-gqa", dtype=torch.float32, init="random", seed=5)
    with pytest.raises(RuntimeError):
        whole.load_state_dict(m.state_dict())
    with pytest.raises(RuntimeError):
        m.load_state_dict(whole.state_dict())


def engine(model, **kw):
    from lumen.serve.engine import EngineConfig, LLMEngine

    return LLMEngine(EngineConfig(model="tiny-llama-gqa", device="cpu", max_model_len=128, block_size=16, num_blocks=64, **kw), model=model)


def answers(eng):
    from lumen.serve.sequence import SamplingParams

    seqs = [eng.add_request(p, SamplingParams(max_tokens=8, temperature=0.0, ignore_eos=True)) for p in ([5, 9, 33, 7] * 6, [42, 43], list(range(3, 30)))]
    while eng.has_work:
        eng.step()
    return [s.output_ids for s in seqs]


def test_engine_answers_as_with_the_quantised_values():
    torch.manual_seed(1)
    base = build_model("tiny-llama-gqa", dtype=torch.float32, init="random", seed=1)
    m, plain = pair(lora=False, seed=1)
    want = answers(engine(plain))
    eng = engine(base, quantization="mxfp4")
    assert type(eng.weights.layers[0].qkv) is MXFP4 and not isinstance(eng.weights.lm_head, MXFP4)
    assert base.layers[0].self_attn.o_proj.weight.numel() > 0        # the caller's model stays whole
    assert answers(eng) == want
    assert answers(engine(m, quantization="mxfp4")) == want          # a base that is in 4 bits already
    assert answers(engine(m)) == want


def test_engine_with_inputs_in_4_bits_too():
    """Against full forwards of the model with the quantised values whose projections see quantised rows."""
    _, plain = pair(lora=False, seed=1)
    for n, lin in plain.named_modules():
        if isinstance(lin, Linear) and not n.endswith("lm_head"):
            lin.register_forward_pre_hook(lambda mod, a: (mxfp4_quantize(a[0]).dequantize(torch.float32),))
    plain.eval()
    torch.manual_seed(1)
    eng = engine(build_model("tiny-llama-gqa", dtype=torch.float32, init="random", seed=1), quantization="mxfp4_a4")
    got = answers(eng)
    for p, out in zip(([5, 9, 33, 7] * 6, [42, 43], list(range(3, 30))), got):
        ids = list(p)
        for tok in out:
            with torch.no_grad():
                assert int(plain(torch.tensor([ids])).view(len(ids), -1)[-1].argmax()) == tok
            ids.append(tok)


def test_engine_adds_adapters_to_projections_in_4_bits(tmp_path):
    """A batch of plain and adapted requests against engines whose weights are the quantised values, adapters merged."""
    from lumen.lora import load_adapter, save_adapter
    from lumen.serve.sequence import SamplingParams

    m, plain = pair(lora=False, seed=1)
    adapted = copy.deepcopy(plain)
    apply_lora(adapted, LoraConfig(r=4, lora_dropout=0.0, target_modules=["q_proj", "v_proj", "o_proj", "up_proj", "down_proj"]))
    with torch.no_grad():
        for p in adapted.parameters():
            if p.requires_grad:
                p.normal_(0, 0.1)
    save_adapter(adapted, str(tmp_path / "a"), "tiny-llama-gqa")
    eng = engine(m, quantization="mxfp4", lora_modules={"a": str(tmp_path / "a")}, max_loras=2)
    params = dict(max_tokens=8, temperature=0.0, ignore_eos=True)
    prompts = ([5, 9, 33, 7] * 6, [42, 43], list(range(3, 30)))
    which = (None, "a", "a")
    seqs = [eng.add_request(p, SamplingParams(**params), lora=w) for p, w in zip(prompts, which)]
    while eng.has_work:
        eng.step()
    load_adapter(plain_a := copy.deepcopy(plain), str(tmp_path / "a"))
    merge_lora(plain_a)
    for p, w, s in zip(prompts, which, seqs):
        assert s.output_ids == answers(engine(plain if w is None else plain_a))[prompts.index(p)]


def test_engine_frees_the_model_that_it_builds():
    eng = engine(None, quantization="mxfp4", init="random")
    assert type(eng.weights.layers[0].down) is MXFP4 and len(answers(eng)) == 3


def test_training_run_from_the_command_line(tmp_path):
    from lumen.cli.train import main

    main("baseline", ["--model_name", "tiny-llama", "--synthetic", "--synthetic_samples", "8", "--max_steps", "2", "--max_length", "32",
                      "--device", "cpu", "--per_device_train_batch_size", "2", "--gradient_accumulation_steps", "1",
                      "--output_dir", str(tmp_path / "o"), "--metrics_csv", str(tmp_path / "m.csv"), "--base_quantization", "mxfp4",
                      "--save_strategy", "no", "--init", "random"])


def test_refusals():
    m = build_model("tiny-llama", dtype=torch.float32, init="random")
    with pytest.raises(ValueError):
        quantize_base(m, "int4")
    with pytest.raises(ValueError):
        engine(m, quantization="awq")
    m.layers[0].mlp.down_proj.weight.requires_grad_(True)
    with pytest.raises(ValueError):
        quantize_base(m)
    with pytest.raises(ValueError):
        m.layers[0].mlp.down_proj.quantize_base()
    assert m.layers[0].self_attn.qkv_proj.qdata is None   # refused before anything was quantised
    odd = Linear(60, 8, dtype=torch.float32)
    with pytest.raises(ValueError):
        quantize_base(odd)
    with pytest.raises(ValueError):
        quantize_base(torch.nn.Linear(64, 64))


def test_hybrid_models_and_zero3_refuse(tmp_path):
    from lumen.parallel.dist import init
    from lumen.serve.engine import EngineConfig, LLMEngine
    from lumen.train.config import load_ds_config
    from lumen.train.engine import ZeroEngine
    from lumen.train.trainer import TrainArgs, Trainer

    with pytest.raises(ValueError, match="quantization"):
        LLMEngine(EngineConfig(model="tiny-gedatar", device="cpu", init="random", quantization="mxfp4"))
    env = init(device="cpu")
    m, _ = pair()
    ds = load_ds_config({"zero_optimization": {"stage": 3}}, 2, 1, 1, 2e-4, dtype_override="fp32")
    with pytest.raises(ValueError, match="4 bits"):
        ZeroEngine(m, ds, env)
    with pytest.raises(ValueError, match="ZeRO-3"):
        Trainer(TrainArgs(model_name="tiny-llama", init="random", synthetic=True, base_quantization="mxfp4"), ds, env)


@pytest.mark.parametrize("lora", [False, True])
def test_a_bias_that_trains(lora):
    """Its gradient is the column sums of dy, with and without adapters."""
    lin = Linear(64, 24, bias=True, dtype=torch.float32, seg_names=["fc1"])
    torch.manual_seed(0)
    with torch.no_grad():
        lin.weight.normal_(0, 0.05), lin.bias.normal_()
        if lora:
            lin.add_lora(["fc1"], 4, 8.0, 0.0)
    frozen = copy.deepcopy(lin)
    lin.bias.requires_grad_(True)
    lin.quantize_base(), frozen.quantize_base()
    x, dy = torch.randn(5, 64), torch.randn(5, 24)
    y = lin(x)
    y.backward(dy)
    close(y.detach(), frozen(x).detach())
    close(lin.bias.grad, dy.sum(0))


def test_counts_of_copies():
    """Copied, pickled and reloaded models count a 4-bit weight as the weight that it is."""
    import io
    import pickle

    m, plain = pair()
    want = count_parameters(plain)
    buf = io.BytesIO()
    torch.save(m.state_dict(), buf)
    buf.seek(0)
    again = copy.deepcopy(m)
    again.load_state_dict(torch.load(buf, weights_only=True), assign=True)
    assert count_parameters(m) == want
    for c in (copy.deepcopy(m), pickle.loads(pickle.dumps(m)), m.to(torch.bfloat16)):
        assert count_parameters(c) == want
    assert count_parameters(again)[1] == want[1]          # (what trains is not part of the state)
    m.layers[0].mlp.down_proj.dequantize_base()
    assert count_parameters(m) == want


@pytest.mark.parametrize("name,cut", [("tiny-llama-tp8", False), ("tiny-llama-gqa", True)])
def test_ranks_keep_the_values_of_a_4_bit_base(name, cut):
    """Every rank's slice holds the base's own values; a base whose blocks the ranks would share is refused (688 / 2 is no multiple
    of 32), and served from its 16-bit values."""
    from lumen.serve.model_runner import ServeWeights

    m, plain = pair(name, lora=False)
    for rank in range(2):
        if cut:
            with pytest.raises(ValueError, match="inside a block"):
                ServeWeights(m, rank, 2, "mxfp4")
        whole = ServeWeights(plain, rank, 2)
        got = ServeWeights(m, rank, 2, None if cut else "mxfp4")
        for a, b in zip(got.layers, whole.layers):
            for n in ("qkv", "o", "gate_up", "down"):
                w = getattr(a, n)
                assert torch.equal(w if cut else w.dequantize(torch.float32), getattr(b, n))
