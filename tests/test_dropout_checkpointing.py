"""FusedDropout inside activation checkpointing: the recomputation draws the mask of the forward pass it repeats."""
import copy
import io

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from distributed_tensorflow_amd.ops import dropout as dp
from token_utils import devices


def block(m, t):
    return m(t).square() * 0.5 + m(t, t)           # two calls; the square's gradient reads the recomputed values


def gradients(m, xs, wrap):
    """Forward passes of all inputs, then the backward passes in reverse order."""
    leaves = [x.clone().requires_grad_(True) for x in xs]
    losses = [wrap(lambda t: block(m, t), leaf * 1.5).sum() for leaf in leaves]
    for loss in reversed(losses):
        loss.backward()
    return [leaf.grad for leaf in leaves]


@pytest.mark.parametrize("dev", devices())
@pytest.mark.parametrize("reentrant", [False, True])
@pytest.mark.parametrize("batches", [1, 3])
def test_gradients_are_those_without_checkpointing(batches, reentrant, dev):
    xs = [torch.randn(40, 33, generator=torch.Generator().manual_seed(k)).to(dev) for k in range(batches)]
    m = dp.FusedDropout(0.4, 77).to(dev)
    for first in (0, 5):                           # the second round with a counter set from outside
        m.step.fill_(first)
        want = gradients(m, xs, lambda f, t: f(t))
        assert int(m.step) == first + 2 * batches
        m.step.fill_(first)
        got = gradients(m, xs, lambda f, t: checkpoint(f, t, use_reentrant=reentrant))
        assert int(m.step) == first + 2 * batches  # recomputing does not advance it
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dev", devices())
def test_nested_checkpoints_and_a_second_backward_pass(dev):
    m, x = dp.FusedDropout(0.5, 3).to(dev), torch.randn(200, device=dev)
    want = gradients(m, [x], lambda f, t: f(t))
    m.step.zero_()
    got = gradients(m, [x], lambda f, t: checkpoint(lambda u: checkpoint(f, u, use_reentrant=False), t, use_reentrant=False))
    assert torch.equal(got[0], want[0])
    m.step.zero_()
    leaf = x.clone().requires_grad_(True)
    loss = checkpoint(lambda t: block(m, t), leaf * 1.5, use_reentrant=False).sum()
    for _ in range(2):
        assert torch.equal(torch.autograd.grad(loss, leaf, retain_graph=True)[0], want[0])


@pytest.mark.parametrize("dev", devices())
def test_a_generator_seeded_anew_for_every_step(dev):
    m, x = dp.FusedDropout(0.5, 3).to(dev), torch.randn(200, device=dev)
    for k in range(3):
        m.step.fill_(2 * k)
        want = gradients(m, [x], lambda f, t: f(t))
        m.step.fill_(2 * k)
        torch.manual_seed(11)
        got = gradients(m, [x], lambda f, t: checkpoint(f, t, use_reentrant=False))
        assert torch.equal(got[0], want[0])
    # two forward passes that the generator cannot tell apart: refused, not guessed
    leaf, losses = x.clone().requires_grad_(True), []
    for _ in range(2):
        torch.manual_seed(11)
        losses.append(checkpoint(lambda t: block(m, t), leaf * 1.5, use_reentrant=False).sum())
    for loss in losses:
        with pytest.raises(RuntimeError, match="FusedDropout"):
            loss.backward(retain_graph=True)


@pytest.mark.parametrize("dev", devices())
def test_a_recomputation_that_cannot_be_recognised_is_refused(dev):
    m, leaf = dp.FusedDropout(0.5, 3).to(dev), torch.randn(200, device=dev, requires_grad=True)
    torch.manual_seed(0)
    loss = checkpoint(lambda t: block(m, t), leaf * 1.5, use_reentrant=False, preserve_rng_state=False).sum()
    with pytest.raises(RuntimeError, match="preserve_rng_state"):
        loss.backward()
    # the function with a step of its own works there
    f = lambda t: dp.dropout(t, 0.5, 3, 9).square().sum()  # noqa: E731
    want = torch.autograd.grad(f(leaf), leaf)[0]
    assert torch.equal(torch.autograd.grad(checkpoint(f, leaf, use_reentrant=False, preserve_rng_state=False), leaf)[0], want)


@pytest.mark.parametrize("dev", devices())
def test_what_the_module_remembers_is_bounded_and_not_part_of_its_copies(dev):
    m, x = dp.FusedDropout(0.5, 3).to(dev), torch.ones(8, device=dev)
    for _ in range(dp.REMEMBERED + 50):
        m(x)
    assert len(m._steps) == dp.REMEMBERED
    other = copy.deepcopy(m)
    buffer = io.BytesIO()
    torch.save(m, buffer)
    assert len(other._steps) == 0 and buffer.tell() < 1 << 15
    assert torch.equal(other(x), m(x)) and set(m.state_dict()) == {"step"}
