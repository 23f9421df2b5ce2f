"""A base in 4 bits on the GPU: adapters train on it, the engine serves it (graphs too), as the same model with the quantised values in 16
bits does."""
import copy

import pytest
import torch

from lumen.lora import LoraConfig, apply_lora, quantize_base
from lumen.models import build_model
from lumen.models.layers import Linear

pytestmark = pytest.mark.gpu
HALF = [torch.bfloat16, torch.float16]


def pair(name, dtype, lora=True):
    m = build_model(name, dtype=dtype, device="cuda", init="random", seed=3)
    if lora:
        apply_lora(m, LoraConfig(r=16, lora_dropout=0.0))
        g = torch.Generator(device="cuda").manual_seed(1)
        with torch.no_grad():
            for p in m.parameters():
                if p.requires_grad:
                    p.normal_(0, 0.05, generator=g)
    plain = copy.deepcopy(m)
    quantize_base(m)
    with torch.no_grad():
        for q, p in zip(m.modules(), plain.modules()):
            if isinstance(q, Linear) and q.qdata is not None:
                p.weight.copy_(q.qweight.dequantize(dtype))
    return m, plain


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("T", [1, 70, 600])
def test_adapted_linear(T, dtype):
    """The base's product and its gradient differ from the 16-bit one's in the order of fp32 sums alone: a step of the type where that
    turns a rounding, once in the product and once where the adapter's part joins it."""
    q = Linear(256, 384, dtype=dtype, device="cuda", seg_sizes=[256, 128], seg_names=["q_proj", "k_proj"])
    g = torch.Generator(device="cuda").manual_seed(T)
    with torch.no_grad():
        q.weight.normal_(0, 0.05, generator=g)
        q.add_lora(["q_proj", "k_proj"], 16, 32.0, 0.0)
        q.lora.lora_B.normal_(0, 0.05, generator=g)
    q.quantize_base()
    p = copy.deepcopy(q)
    p.dequantize_base()
    x = torch.randn(T, 256, device="cuda", generator=g).to(dtype)
    dy = torch.randn(T, 384, device="cuda", generator=g).to(dtype)
    out = []
    for lin in (q, p):
        leaf = x.clone().requires_grad_()
        y = lin(leaf)
        dx, dA, dB = torch.autograd.grad(y, (leaf, lin.lora.lora_A, lin.lora.lora_B), dy)
        out.append((y.detach().double(), dx.double(), dA, dB))
    W = p.weight.double()
    for i, base in ((0, x.double() @ W.t()), (1, dy.double() @ W)):
        tol = torch.finfo(dtype).eps * (out[1][i].abs() + base.abs()) * 1.01 + 1e-6
        assert ((out[0][i] - out[1][i]).abs() <= tol).all()
    for i in (2, 3):                                      # of x and dy alone: T terms in another order
        assert (out[0][i] - out[1][i]).abs().max() <= (T + 16) * 2.0 ** -22 * (out[1][i].abs().max() + 30)


def test_loss_and_gradients_of_a_model():
    """Norm-wise within 3 %: every layer rounds some ten times to bf16 (rms 2^-9 / sqrt 3 each, about 0.4 % a layer)."""
    m, plain = pair("small-llama", torch.bfloat16)
    ids = torch.randint(3, m.config.vocab_size, (2, 128), device="cuda")
    got = []
    for model in (m, plain):
        model.train()
        loss = model(ids, labels=torch.roll(ids, -1, 1))
        loss.backward()
        got.append((float(loss.detach()), [p.grad.clone() for p in model.parameters() if p.requires_grad]))
    assert abs(got[0][0] - got[1][0]) <= 3e-2 * abs(got[1][0])
    for a, b in zip(got[0][1], got[1][1]):
        assert (a - b).norm() <= 3e-2 * b.norm()


def test_a_training_step_through_the_engine():
    from lumen.parallel.dist import init
    from lumen.train.config import load_ds_config
    from lumen.train.engine import ZeroEngine

    m, _ = pair("small-llama", torch.bfloat16)
    m.train()
    eng = ZeroEngine(m, load_ds_config({"zero_optimization": {"stage": 1}}, 2, 1, 1, 2e-4), init())
    ids = torch.randint(3, m.config.vocab_size, (2, 128), device="cuda")
    codes = m.layers[0].mlp.down_proj.qdata.clone()
    before = [p.detach().clone() for p in m.parameters() if p.requires_grad]
    for _ in range(2):
        eng.backward(eng.forward({"input_ids": ids, "labels": torch.roll(ids, -1, 1), "n_valid": ids.numel()}))
        assert eng.step()
    after = [p.detach() for p in m.parameters() if p.requires_grad]
    assert any(not torch.equal(a, b) for a, b in zip(after, before)) and all(torch.isfinite(a).all() for a in after)
    assert torch.equal(m.layers[0].mlp.down_proj.qdata, codes)


@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("name", ["tiny-llama", "tiny-llama-gqa"])
def test_engine_logits(name, graphs):
    """Decode steps of an engine in 4 bits against the full forward of the model with the quantised values (norm-wise 3 %, as above)."""
    from lumen.serve.engine import EngineConfig, LLMEngine
    from lumen.serve.sequence import SamplingParams

    m, plain = pair(name, torch.bfloat16, lora=False)
    m.eval(), plain.eval()
    eng = LLMEngine(EngineConfig(model=name, device="cuda", max_model_len=256, block_size=16, num_blocks=128, use_graphs=graphs,
                                 quantization="mxfp4"), model=m)
    prompts = [list(range(10, 40)), [7, 8, 9] * 20, [42]]
    seqs = [eng.add_request(p, SamplingParams(max_tokens=6, temperature=0, ignore_eos=True)) for p in prompts]
    got, orig = [], eng.runner.decode

    def spy(inp):
        out = orig(inp)
        got.append((inp.positions.cpu().tolist(), out.float().clone()))
        return out
    eng.runner.decode = spy
    while eng.has_work:
        eng.step()
    assert got
    for positions, logits in got:
        for i, (s, pos) in enumerate(zip(seqs, positions)):
            ids = torch.tensor([s.all_ids[:pos + 1]], device="cuda")
            with torch.no_grad():
                ref = plain(ids).float().view(pos + 1, -1)[-1]
            assert (logits[i] - ref).norm() <= 3e-2 * ref.norm()


@pytest.mark.parametrize("graphs", [False, True])
def test_engine_with_inputs_in_4_bits_too(graphs):
    """Decode steps against the full forward of the model whose projections see quantised rows.  Both round in 16 bits before they
    quantise, and a value within that rounding v 2^-8 of a tie may take the other code.  v is some four steps at most, so two
    hundredths of the values do, a step each: 0.02 step^2 against the step^2 / 12 of quantisation itself, half its norm.  Allowed
    is the whole distance that quantising the rows makes, and the 3 % of 16-bit arithmetic."""
    from lumen.ops.mxfp4 import mxfp4_quantize
    from lumen.serve.engine import EngineConfig, LLMEngine
    from lumen.serve.sequence import SamplingParams

    m, plain = pair("tiny-llama-gqa", torch.bfloat16, lora=False)
    m.eval(), plain.eval()
    rows = copy.deepcopy(plain)
    for n, lin in rows.named_modules():
        if isinstance(lin, Linear) and not n.endswith("lm_head"):
            lin.register_forward_pre_hook(
                lambda mod, a: (mxfp4_quantize(a[0].reshape(-1, a[0].shape[-1])).dequantize(a[0].dtype).view(a[0].shape),))
    eng = LLMEngine(EngineConfig(model="tiny-llama-gqa", device="cuda", max_model_len=256, block_size=16, num_blocks=128, use_graphs=graphs,
                                 quantization="mxfp4_a4"), model=m)
    prompts = [list(range(10, 40)), [7, 8, 9] * 20, [42]]
    seqs = [eng.add_request(p, SamplingParams(max_tokens=6, temperature=0, ignore_eos=True)) for p in prompts]
    got, orig = [], eng.runner.decode

    def spy(inp):
        out = orig(inp)
        got.append((inp.positions.cpu().tolist(), out.float().clone()))
        return out
    eng.runner.decode = spy
    while eng.has_work:
        eng.step()
    assert got
    for positions, logits in got:
        for i, (s, pos) in enumerate(zip(seqs, positions)):
            ids = torch.tensor([s.all_ids[:pos + 1]], device="cuda")
            with torch.no_grad():
                with_q, without = (mod(ids).float().view(pos + 1, -1)[-1] for mod in (rows, plain))
            assert (logits[i] - with_q).norm() <= (with_q - without).norm() + 3e-2 * without.norm()


@pytest.mark.parametrize("lora", [False, True])
@pytest.mark.parametrize("grad", [False, True])
def test_a_quantised_linear_refuses_other_rows(lora, grad):
    lin = Linear(256, 128, dtype=torch.bfloat16, device="cuda", seg_names=["q_proj"])
    with torch.no_grad():
        lin.weight.normal_(0, 0.05)
        if lora:
            lin.add_lora(["q_proj"], 16, 32.0, 0.0)
    lin.quantize_base()
    for K in (248, 264, 128):
        x = torch.randn(6, K, device="cuda").bfloat16().requires_grad_(grad)
        with pytest.raises(ValueError):
            lin(x)
    assert lin(torch.randn(6, 256, device="cuda").bfloat16()).shape == (6, 128)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("lora", [False, True])
def test_a_bias_is_added_before_the_rounding(lora, dtype):
    """A quantised projection with a bias gives mxfp4_linear's own bits: fp32 sums and the bias, one rounding."""
    from lumen.ops.mxfp4 import mxfp4_linear

    lin = Linear(256, 384, bias=True, dtype=dtype, device="cuda", seg_names=["fc1"])
    g = torch.Generator(device="cuda").manual_seed(5)
    with torch.no_grad():
        lin.weight.normal_(0, 0.05, generator=g)
        lin.bias.normal_(0, 1, generator=g)
        if lora:                                          # lora_B is zero: the adapter adds nothing
            lin.add_lora(["fc1"], 16, 32.0, 0.0)
    lin.quantize_base()
    for T in (1, 70, 600):
        x = torch.randn(T, 256, device="cuda", generator=g).to(dtype)
        same = torch.equal(lin(x), mxfp4_linear(x, lin.qweight, lin.bias))
        assert same


def test_memory_of_the_16_bit_projections_is_given_back():
    """Freed projections are the device's again, so that the automatic number of cache blocks goes by what is left."""
    import gc

    from lumen.serve.engine import EngineConfig, LLMEngine
    from lumen.serve.model_runner import ServeWeights

    gc.collect()                                          # (what earlier tests left)
    name = "llama2-70b-2l"                                # 3.4 GB of projections
    m = build_model(name, dtype=torch.bfloat16, device="cuda", init="random")
    held = sum(p.numel() * 2 for n, p in m.named_parameters() if "_proj" in n)
    torch.cuda.empty_cache()
    before = torch.cuda.mem_get_info()[0]
    w = ServeWeights(m, quantization="mxfp4", release=True)
    kept = sum(q.nbytes for L in w.layers for q in (L.qkv, L.o, L.gate_up, L.down))
    assert torch.cuda.mem_get_info()[0] - before >= held - kept - (128 << 20)     # (segments are rounded up)
    del m, w
    gc.collect()
    torch.cuda.empty_cache()
    free, total = torch.cuda.mem_get_info()               # (of 14 GiB of what is free the engine leaves 4 to activations)
    share = 1 - (free - (14 << 30)) / total
    blocks = {}
    for how in (None, "mxfp4"):
        eng = LLMEngine(EngineConfig(model=name, device="cuda", max_model_len=4096, max_num_seqs=256, block_size=16, init="random",
                                     use_graphs=False, quantization=how, gpu_memory_utilization=share))
        blocks[how] = eng.blocks.num_blocks
        del eng
        gc.collect()
        torch.cuda.empty_cache()
    per_block = 16 * 2 * 2 * 8 * 128 * 2                  # tokens, keys and values, layers, heads, values, bytes
    assert (blocks["mxfp4"] - blocks[None]) * per_block >= held - kept - (128 << 20)


def test_engine_quantises_its_inputs_or_leaves_them():
    """Prompts' last logits of ``mxfp4_a4`` lie nearer to the full forward on quantised rows than to the one on 16-bit rows, those of
    ``mxfp4`` the other way round.  (Both are off by roundings that know nothing of the distance d between the two: |e|^2 of one beside
    |e|^2 + |d|^2 of the other.)"""
    from lumen.ops.mxfp4 import mxfp4_quantize
    from lumen.serve.engine import EngineConfig, LLMEngine
    from lumen.serve.sequence import SamplingParams

    m, plain = pair("tiny-llama-gqa", torch.bfloat16, lora=False)
    m.eval(), plain.eval()
    rows = copy.deepcopy(plain)
    for n, lin in rows.named_modules():
        if isinstance(lin, Linear) and not n.endswith("lm_head"):
            lin.register_forward_pre_hook(
                lambda mod, a: (mxfp4_quantize(a[0].reshape(-1, a[0].shape[-1])).dequantize(a[0].dtype).view(a[0].shape),))
    prompts = [list(range(10, 40)), [7, 8, 9] * 20, [42], list(range(100, 400, 3))]
    for how, graphs in (("mxfp4", False), ("mxfp4", True), ("mxfp4_a4", False), ("mxfp4_a4", True)):
        eng = LLMEngine(EngineConfig(model="tiny-llama-gqa", device="cuda", max_model_len=256, block_size=16, num_blocks=128,
                                     use_graphs=graphs, quantization=how), model=m)
        seqs = [eng.add_request(p, SamplingParams(max_tokens=6, temperature=0, ignore_eos=True)) for p in prompts]
        got, orig = [], eng.runner.decode

        def spy(inp):
            out = orig(inp)
            got.append((inp.positions.cpu().tolist(), out.float().clone()))
            return out
        eng.runner.decode = spy
        while eng.has_work:
            eng.step()
        assert got
        quantised = left = 0.0
        for positions, logits in got:
            for i, (s, pos) in enumerate(zip(seqs, positions)):
                ids = torch.tensor([s.all_ids[:pos + 1]], device="cuda")
                with torch.no_grad():
                    quantised += float((logits[i] - rows(ids).float().view(pos + 1, -1)[-1]).norm() ** 2)
                    left += float((logits[i] - plain(ids).float().view(pos + 1, -1)[-1]).norm() ** 2)
        assert (quantised < left) == (how == "mxfp4_a4")
