"""CPU: a moving average has no meaning over 8-bit integers and their scales; an update that would meet them is refused before
anything is written.  A quantised copy of the teacher leaves the teacher itself in floats."""
import copy

import pytest
import torch

from datr_amd.ema import CosineEMA, ModelEMA
from datr_amd.int8 import quantize_ffn_
from helpers_int8 import host_layer


class Block(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.linear1, self.linear2 = torch.nn.Linear(8, 16), torch.nn.Linear(16, 8)


@pytest.mark.parametrize("average", [ModelEMA, CosineEMA])
def test_an_update_of_a_quantised_teacher_is_refused(monkeypatch, average):
    host_layer(monkeypatch, 4, 4)                        # quantize_rows on the host from here on
    student = torch.nn.Sequential(torch.nn.Linear(8, 8), Block())
    teacher = average(student)
    assert quantize_ffn_(teacher.ema) == 1
    before = {k: v.clone() for k, v in teacher.ema.state_dict().items()}
    with torch.no_grad():
        for p in student.parameters():
            p.add_(1.0)
    with pytest.raises(RuntimeError, match="8-bit"):
        teacher.update(student)
    assert all(torch.equal(v, before[k]) for k, v in teacher.ema.state_dict().items())
    # both sides in integers: the scales would be averaged and the integers not
    quantize_ffn_(student)
    with pytest.raises(RuntimeError, match="8-bit"):
        teacher.update(student)
    with pytest.raises(RuntimeError, match="8-bit"):
        average(student).update(student)


def test_a_quantised_copy_leaves_the_teacher_as_it_is(monkeypatch):
    host_layer(monkeypatch, 4, 4)
    student = torch.nn.Sequential(torch.nn.Linear(8, 8), Block())
    teacher = ModelEMA(student)
    assert quantize_ffn_(copy.deepcopy(teacher.ema)) == 1
    with torch.no_grad():
        for p in student.parameters():
            p.add_(1.0)
    before = teacher.ema[1].linear1.weight.clone()
    teacher.update(student)
    assert not torch.equal(teacher.ema[1].linear1.weight, before)
