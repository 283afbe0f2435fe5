"""ScaledEmbedding as a subclass of nn.Embedding: construction from a given table, checks that do not hang on gradients."""
import pytest
import torch

from distributed_tensorflow_amd.ops import embedding as em
from token_utils import devices


@pytest.mark.parametrize("dev", devices())
def test_from_a_given_table(dev):
    table, ids = torch.randn(9, 8, device=dev), torch.tensor([[0, 8], [3, 3]], device=dev)
    m = em.ScaledEmbedding.from_pretrained(table, padding_idx=3)
    assert m.scale == 1.0 and not m.weight.requires_grad and torch.equal(m(ids), table[ids])
    m = em.ScaledEmbedding.from_pretrained(table.clone(), freeze=False, padding_idx=3, scale=2.0)
    y = m(ids)
    assert torch.equal(y, 2.0 * table[ids])
    y.sum().backward()
    assert not m.weight.grad[3].any() and torch.equal(m.weight.grad[8], torch.full((8,), 2.0, device=dev))
    assert em.ScaledEmbedding(9, 8, max_norm=None, scale_grad_by_freq=False, sparse=False).scale == 1.0
    for bad in (dict(max_norm=1.0), dict(max_norm=0.0), dict(sparse=True), dict(scale_grad_by_freq=True)):
        with pytest.raises(ValueError):
            em.ScaledEmbedding(9, 8, **bad)
        with pytest.raises(ValueError):
            em.ScaledEmbedding.from_pretrained(table, **bad)


@pytest.mark.parametrize("dev", devices())
@pytest.mark.parametrize("grad", [False, True])
def test_a_padding_index_outside_the_table_is_refused_with_and_without_gradients(grad, dev):
    table, ids = torch.randn(9, 8, device=dev, requires_grad=grad), torch.zeros(2, dtype=torch.int64, device=dev)
    for bad in (9, -10):
        with pytest.raises(ValueError, match="padding_idx"):
            em.embedding(ids, table, padding_idx=bad)
    assert torch.equal(em.embedding(ids, table, padding_idx=-9), table[ids])
