"""The CPU statement of the vocabulary cross entropy under autocast."""
import torch

from distributed_tensorflow_amd.ops.vocab_xent import vocab_xent


def test_the_cpu_statement_keeps_float32_logits_under_autocast():
    """Forward under autocast, backward outside as usual: both on the same logits."""
    g = torch.Generator().manual_seed(2)
    x, w, b = torch.randn(30, 64, generator=g), torch.randn(90, 64, generator=g), torch.randn(90, generator=g)
    lab = torch.randint(0, 90, (30,), generator=g)
    results = []
    for enabled in (False, True):
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
        with torch.autocast("cpu", dtype=torch.bfloat16, enabled=enabled):
            loss, _ = vocab_xent(leaves[0], leaves[1], lab, leaves[2])
            loss.backward()
        results.append([loss.detach()] + [t.grad for t in leaves])
    assert all(torch.equal(a, c) for a, c in zip(*results))
