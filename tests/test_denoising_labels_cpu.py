"""CPU: the de-noising queries draw labels from as many classes as the label table has rows for; fewer rows are refused before the
draw, on every device alike."""
import pytest
import torch

from datr_amd.denoising import prepare_for_cdn
from datr_amd.embedding import FastEmbedding


def targets():
    return [{"labels": torch.tensor([1, 2]), "boxes": torch.rand(2, 4) * 0.3 + 0.2}]


@pytest.mark.parametrize("table", [torch.nn.Embedding, FastEmbedding])
def test_a_table_with_too_few_rows(table):
    for rows in (9, 10):
        q = prepare_for_cdn((targets(), 100, 0.5, 1.0), True, 20, 9, 16, table(rows, 16))[0]
        assert q.shape[0] == 1 and q.shape[2] == 16
    with pytest.raises(ValueError, match="9 classes.*8 rows"):
        prepare_for_cdn((targets(), 100, 0.5, 1.0), True, 20, 9, 16, table(8, 16))
    # no label is drawn: the targets' own are all there are
    assert prepare_for_cdn((targets(), 100, 0.0, 1.0), True, 20, 9, 16, table(3, 16))[0].shape[2] == 16
