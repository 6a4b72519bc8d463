"""GPU: the engine's evaluation and its teacher-student epoch with a detector whose feed-forward products are in 8-bit integers."""
import copy
import types

import numpy as np
import pytest
import torch

from helpers import build_model, load_npz
from test_selftrain_cpu import batch

pytestmark = pytest.mark.gpu


def quantised(model):
    from datr_amd.int8 import Int8Linear, quantize_ffn_
    small = copy.deepcopy(model).eval()
    layers = quantize_ffn_(small)
    assert layers == 12 and sum(isinstance(m, Int8Linear) for m in small.modules()) == 24
    return small


@pytest.mark.parametrize("amp", [False, True])
def test_evaluation(amp):
    import synth
    from datr_amd.detector import PostProcess
    from datr_amd.engine import evaluate
    from datr_amd.nested import nested_tensor_from_tensor_list
    dev = torch.device("cuda:0")
    args, model, criterion, _ = build_model("cuda:0")
    criterion.to(dev)
    args.use_dn, args.amp = False, amp
    imgs, _ = synth.synth_batch()
    targets = tuple({"boxes": torch.tensor([[0.4, 0.5, 0.2, 0.3]], device=dev), "labels": torch.tensor([1], device=dev),
                     "image_id": torch.tensor([n], device=dev), "orig_size": torch.tensor([480.0, 600.0], device=dev),
                     "iscrowd": torch.zeros(1, dtype=torch.long, device=dev)} for n in (1, 2))
    loader = [(nested_tensor_from_tensor_list([i.to(dev) for i in imgs]), None, targets)]
    stats, _ = evaluate(quantised(model), criterion, {"bbox": PostProcess(num_select=100)}, loader, None, dev, args=args)
    assert len(stats["coco_eval_bbox"]) == 12 and np.isfinite(stats["loss"]) and stats["loss"] > 0


def test_a_teacher_student_epoch_with_a_quantised_copy_of_the_teacher():
    from datr_amd.config import get_param_dict
    from datr_amd.ema import ModelEMA
    from datr_amd.engine import train_one_epoch_with_self_training
    dev = torch.device("cuda:0")
    args, model, criterion, _ = build_model("cuda:0")
    criterion.to(dev)
    args.pseudo_label_threshold = float(load_npz("selftrain_step.npz")["threshold"])
    teacher = ModelEMA(model, decay=args.ema_decay_teacher)
    optimizer = torch.optim.AdamW(get_param_dict(args, model), lr=args.lr, weight_decay=args.weight_decay)
    before = teacher.ema.state_dict()["transformer.encoder.layers.0.linear1.weight"].clone()
    moved = model.transformer.encoder.layers[0].linear1.weight.detach().clone()
    loader = batch()
    stats = train_one_epoch_with_self_training(model, types.SimpleNamespace(ema=quantised(teacher.ema)), criterion, loader, loader,
                                               optimizer, dev, 0, args.clip_max_norm, args=args)
    assert np.isfinite(stats["loss"]) and not torch.equal(moved, model.transformer.encoder.layers[0].linear1.weight)
    # the teacher itself is in floats and takes its update
    teacher.update(model)
    after = teacher.ema.state_dict()["transformer.encoder.layers.0.linear1.weight"]
    assert after.dtype is torch.float32 and not torch.equal(before, after)
