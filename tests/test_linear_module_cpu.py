"""The cell of linear attention as a module: its decays stay float32 and go where the module goes, also from the meta device."""
import copy

import pytest
import torch

from acctransformer_b200 import LinearAttention

DECAYS = [-0.1, -0.0123456]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float64])
def test_casts(dtype):
    cell = LinearAttention(2, 64, log_decay=DECAYS).to(dtype)
    assert cell.log_decay.dtype == torch.float32 and torch.equal(cell.log_decay, torch.tensor(DECAYS))
    assert "log_decay" in cell.state_dict() and "log_decay" in dict(cell.named_buffers())


def test_from_the_meta_device():
    cell = torch.nn.Sequential(LinearAttention(2, 64, log_decay=DECAYS).to("meta"))
    assert cell[0].log_decay.is_meta
    cell.to(torch.bfloat16)
    assert cell[0].log_decay.dtype == torch.float32
    cell.to_empty(device="cpu")
    assert cell[0].log_decay.dtype == torch.float32 and not cell[0].log_decay.is_meta
    cell.load_state_dict({"0.log_decay": torch.tensor(DECAYS)})
    assert torch.equal(cell[0].log_decay, torch.tensor(DECAYS))


def test_made_on_the_meta_device():
    with torch.device("meta"):
        cell = LinearAttention(2, 64)
    assert cell.log_decay.is_meta
    cell.to_empty(device="cpu")
    cell.load_state_dict(LinearAttention(2, 64, log_decay=DECAYS).state_dict())
    assert torch.equal(cell.log_decay, torch.tensor(DECAYS))


def test_copies_are_apart():
    cell = LinearAttention(2, 64, log_decay=DECAYS)
    other = copy.deepcopy(cell).half()
    other.log_decay.zero_()
    assert torch.equal(cell.log_decay, torch.tensor(DECAYS))
