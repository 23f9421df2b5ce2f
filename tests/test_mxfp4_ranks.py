"""A base in 4 bits on two ranks (gloo, CPU): adapters train on it as on one, tensor-parallel engines answer as a model with each rank's
quantised values does."""
import pytest
import torch
import torch.multiprocessing as mp

from lumen.models.layers import Linear
from lumen.ops.mxfp4 import mxfp4_quantize
from tests._dist_worker import _tp_test_model, serve_tp_worker
from tests.test_serving_cpu import naive_greedy
from tests.test_zero_gloo import _close, _port, _run


@pytest.mark.parametrize("stage", [1, 2])
def test_training(stage, tmp_path):
    four = {"base_quantization": "mxfp4"}
    want = _run(1, 0, str(tmp_path / "one"), model="tiny-llama", micro=4, accum=1, steps=3, extra=four)
    got = _run(2, stage, str(tmp_path / "two"), model="tiny-llama", micro=2, accum=1, steps=3, extra=four)
    assert len(got["losses"]) == len(want["losses"]) == 3
    for a, b in zip(got["losses"], want["losses"]):
        assert abs(a - b) < 1e-3
    _close(got["sd"], want["sd"])
    assert any(v.abs().sum() > 0 for k, v in got["sd"].items() if "lora_B" in k)
    whole = _run(1, 0, str(tmp_path / "whole"), model="tiny-llama", micro=4, accum=1, steps=3)
    assert any(not torch.equal(whole["sd"][k], v) for k, v in want["sd"].items())       # (the base was quantised)


def test_resuming_on_fewer_ranks(tmp_path):
    four = {"base_quantization": "mxfp4"}
    ck = str(tmp_path / "ck")
    want = _run(1, 0, str(tmp_path / "one"), model="tiny-llama", micro=4, accum=1, steps=4, extra=four)
    _run(2, 2, str(tmp_path / "a"), model="tiny-llama", micro=2, accum=1, steps=2, extra=dict(four, save_steps=2, ckdir=ck))
    got = _run(1, 2, str(tmp_path / "b"), model="tiny-llama", micro=4, accum=1, steps=4,
               extra=dict(four, save_steps=100, ckdir=ck, resume=True))
    _close(got["sd"], want["sd"])


def by_rank(x, n):
    """x [rows, K] quantised and back, each of n slices of its columns by itself."""
    return torch.cat([mxfp4_quantize(p.contiguous()).dequantize(torch.float32) for p in x.chunk(n, 1)], 1)


@pytest.mark.parametrize("how", ["mxfp4", "mxfp4_a4"])
def test_tensor_parallel_engine(how, tmp_path):
    mp.start_processes(serve_tp_worker, args=(2, _port(), str(tmp_path), None, True, None, {"quantization": how}), nprocs=2, join=True,
                       start_method="spawn")
    got = torch.load(tmp_path / "tp_out.pt", weights_only=True)
    plain = _tp_test_model()
    for n, lin in plain.named_modules():
        if isinstance(lin, Linear) and not n.endswith("lm_head"):
            parts = 2 if n.endswith(("o_proj", "down_proj")) else 1     # cut along the inputs, the others along the outputs
            with torch.no_grad():
                lin.weight.copy_(by_rank(lin.weight, parts))
            if how == "mxfp4_a4":
                lin.register_forward_pre_hook(lambda mod, a, parts=parts: (by_rank(a[0].reshape(-1, a[0].shape[-1]), parts),))
    for p, out in zip([[5, 9, 33, 7], list(range(3, 30)), [42, 43]], got):
        assert out == naive_greedy(plain, p, 8), p
