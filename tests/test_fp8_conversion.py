"""Converting an encoder to 8-bit products: once, as a whole, and what it keeps after."""

import argparse
import dataclasses
import json

import pytest
import torch

from vilbert_multi_task_amd.config import ViLBertConfig
from vilbert_multi_task_amd.engine.runner import GraphRunner
from vilbert_multi_task_amd.models import VILBertForVLTasks
from vilbert_multi_task_amd.models.fp8 import (
    BlockFp8LayerNorm,
    BlockFp8Linear,
    _block_pack,
    convert_encoder_to_fp8,
    convert_encoder_to_fp8_block,
)
from vilbert_multi_task_amd.models.vilbert import FusedLayerNorm
from vilbert_multi_task_amd.serve.main import build_worker


def _model():
    torch.manual_seed(0)
    return VILBertForVLTasks(ViLBertConfig.tiny()).eval()


@pytest.mark.parametrize("first", [convert_encoder_to_fp8, convert_encoder_to_fp8_block])
@pytest.mark.parametrize("second", [convert_encoder_to_fp8, convert_encoder_to_fp8_block])
def test_a_second_conversion_is_refused_and_changes_nothing(first, second):
    model = _model()
    first(model)
    parts = dict(model.named_modules())
    held = {
        (name, key): value for name, m in parts.items()
        for key, value in vars(m).items() if isinstance(value, torch.Tensor)}
    held = {at: (t, t.clone()) for at, t in held.items()}
    with pytest.raises(RuntimeError, match="already"):
        second(model)
    assert dict(model.named_modules()) == parts
    for (name, key), (t, before) in held.items():
        assert getattr(parts[name], key) is t
        assert torch.equal(t.float(), before.float())


def _linears(model):
    return [m for m in model.modules() if isinstance(m, BlockFp8Linear)]


@pytest.mark.parametrize("cast", [
    lambda m: m.to(torch.bfloat16), lambda m: m.bfloat16(), lambda m: m.half(), lambda m: m.double(),
    lambda m: m.to("cpu"), lambda m: m.to(torch.bfloat16).float(), lambda m: m.type(torch.bfloat16),
    lambda m: m.share_memory()])
def test_casts_leave_8_bit_weights_and_their_scales(cast):
    model = _model()
    convert_encoder_to_fp8_block(model)
    before = [(m.w8.clone(), m.w_scales.clone()) for m in _linears(model)]
    cast(model)
    assert before
    for m, (w8, scales) in zip(_linears(model), before):
        assert m.w8.dtype == torch.float8_e4m3fn and m.w_scales.dtype == torch.bfloat16
        assert torch.equal(m.w8.float(), w8.float()) and torch.equal(m.w_scales, scales)
        assert {"w8", "w_scales", "bias"} == set(m.state_dict())


def test_a_cast_module_answers_in_its_new_type():
    torch.manual_seed(1)
    for bias in (True, False):
        m = BlockFp8Linear(torch.nn.Linear(96, 200, bias=bias))
        x = torch.randn(5, 96)
        want = m(x)
        assert want.dtype == torch.float32
        q, s = m.to(torch.bfloat16).gelu8(x.bfloat16())
        assert m(x.bfloat16()).dtype == torch.bfloat16
        wide = BlockFp8Linear(torch.nn.Linear(200, 8)).to(torch.bfloat16)
        assert wide((q, s)).dtype == torch.bfloat16  # a pair has no type of its own
        assert torch.equal(m.float()(x), want) or bias  # a bias was rounded on the way


def test_a_state_dict_is_taken_up_again():
    a, b = _model(), _model()
    convert_encoder_to_fp8_block(a)
    with torch.no_grad():
        for p in b.parameters():
            p.mul_(1.5)
    convert_encoder_to_fp8_block(b)
    b.load_state_dict(a.state_dict())
    for m, n in zip(_linears(a), _linears(b)):
        assert torch.equal(m.w8.float(), n.w8.float()) and torch.equal(m.w_scales, n.w_scales)


@pytest.mark.gpu
def test_a_module_moves_to_the_gpu_as_it_is():
    torch.manual_seed(1)
    m = BlockFp8Linear(torch.nn.Linear(100, 60))  # rows that are no multiple of 16 bytes
    x = torch.randn(7, 100)
    want = m(x)
    got = m.cuda()(x.cuda())
    assert got.dtype == want.dtype
    # both round once to bf16; the 8-bit instruction drops 2^-13 of the largest of eight
    # products for 7 of them, of sizes that add up to about 4
    assert torch.allclose(got.cpu(), want, rtol=2.0 ** -7, atol=7 * 2.0 ** -13 * 4)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_what_is_written_over_is_quantised_anew(device):
    """The norm's 8-bit form stands for the values that it was made with alone."""
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    torch.manual_seed(1)
    norm = BlockFp8LayerNorm(FusedLayerNorm(96, 1e-5)).to(device, dtype)
    linear = BlockFp8Linear(torch.nn.Linear(96, 40).to(device, dtype))
    x = torch.randn(5, 96, device=device, dtype=dtype)
    change = [
        lambda y: y.mul_(3), lambda y: y[1:].zero_(), lambda y: y.copy_(x), lambda y: y.view(-1)[7:9].fill_(50)]
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            for f in change:
                y = norm(x)
                f(y)
                assert torch.equal(linear(y), linear(y.clone()))
                q, s = linear.gelu8(y)
                rq, rs = linear.gelu8(y.clone())
                assert torch.equal(q.float(), rq.float()) and torch.equal(s, rs)


def test_the_norms_8_bit_form_is_what_is_used():
    norm = BlockFp8LayerNorm(FusedLayerNorm(96, 1e-5))
    linear = BlockFp8Linear(torch.nn.Linear(96, 40))
    with torch.no_grad():
        y = norm(torch.randn(5, 96))
        assert _block_pack(y)[0] is y._fp8b[0] and _block_pack(y)[1] is y._fp8b[1]
        linear(y)


@pytest.mark.parametrize("fp8", [None, False, 0, "", True, 1, "block"])
def test_runner_takes_what_says_yes_or_no(fp8):
    GraphRunner(_model(), device="cpu", fp8=fp8)


@pytest.mark.parametrize("fp8", ["tensor", "blocks", 2, object()])
def test_runner_refuses_other_modes(fp8):
    with pytest.raises(ValueError, match="fp8"):
        GraphRunner(_model(), device="cpu", fp8=fp8)


@pytest.mark.parametrize("more", [{}, {"fp8_block": True}])
def test_a_worker_is_built_with_and_without_the_mode(more, tmp_path):
    """Callers that were there before the mode say nothing of it."""
    config = tmp_path / "tiny.json"
    config.write_text(json.dumps(dataclasses.asdict(ViLBertConfig.tiny())))
    args = argparse.Namespace(
        config=str(config), checkpoint="", device=-1, fp8=False, detector=False,
        queue=str(tmp_path / "q"), db=str(tmp_path / "d"), hub_port=0, vqa_answers="", gqa_answers="",
        max_batch=4, **more)
    assert build_worker(args).runner is not None
