"""Converting an encoder to 8-bit products: once, as a whole, and what it keeps after."""

import pytest
import torch

from vilbert_multi_task_amd.config import ViLBertConfig
from vilbert_multi_task_amd.models import VILBertForVLTasks
from vilbert_multi_task_amd.models.fp8 import (
    convert_encoder_to_fp8,
    convert_encoder_to_fp8_block,
)


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
