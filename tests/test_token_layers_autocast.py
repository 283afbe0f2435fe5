"""The token-model layers under autocast, by themselves and in a module that the framework's program trains."""
import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from distributed_tensorflow_amd.models.resnet import TorchModuleProgram
from distributed_tensorflow_amd.ops.dropout import FusedDropout, dropout_apply
from distributed_tensorflow_amd.ops.embedding import ScaledEmbedding
from distributed_tensorflow_amd.ops.layernorm import FusedLayerNorm, layer_norm
from distributed_tensorflow_amd.parallel.sync_replicas import SyncReplicasEngine
from token_utils import U32, assert_within, devices


def autocast(dev, dtype=torch.bfloat16):
    return torch.autocast(dev.split(":")[0], dtype=dtype)


@pytest.mark.parametrize("dev", devices())
@pytest.mark.parametrize("low", [torch.bfloat16, torch.float16])
def test_a_branch_in_low_precision_meets_a_float32_stream(low, dev):
    """As ``x + residual`` does, in either order of types: both in the wider one."""
    g = torch.Generator().manual_seed(1)
    x, r, up = (torch.randn(7, 40, generator=g).to(dev) for _ in range(3))
    w, b = torch.rand(40, generator=g).to(dev) + 0.5, torch.randn(40, generator=g).to(dev)
    for a, c in ((x.to(low), r), (x, r.to(low))):
        leaves = [t.detach().requires_grad_(True) for t in (a, c)]
        with autocast(dev, low):
            y, h = layer_norm(leaves[0], w, b, residual=leaves[1])
            z = FusedDropout(0.25, 9).to(dev)(leaves[0], leaves[1])
        want_y, want_h = layer_norm(a.float(), w, b, residual=c.float())
        assert y.dtype == h.dtype == z.dtype == torch.float32
        assert torch.equal(y, want_y) and torch.equal(h, want_h)
        assert torch.equal(z, dropout_apply(a.float(), 0.25, 9, 0, residual=c.float()))
        ((y + z) * up).sum().backward()
        wide = [t.detach().float().requires_grad_(True) for t in (a, c)]
        want = layer_norm(wide[0], w, b, residual=wide[1])[0]
        (want * up).sum().backward()
        wide[0].grad += dropout_apply(up, 0.25, 9, 0)
        wide[1].grad += up
        for leaf, exp in zip(leaves, wide):
            assert leaf.grad.dtype == leaf.dtype
            # two float32 gradients, each rounded to the leaf's type before or after their sum
            eps = torch.finfo(leaf.dtype).eps
            assert_within(leaf.grad, exp.grad.double(), 2 * eps * (exp.grad.double().abs() + 2 * up.double().abs() + 4) * (1 if eps > 1e-4 else 8))
    with pytest.raises(ValueError):                # outside autocast as before
        layer_norm(x.bfloat16(), w, b, residual=r)


class Net(nn.Module):
    """Tokens -> embedding -> two residual blocks with dropout and layer norm -> classes."""

    def __init__(self, vocab=50, d=48, classes=10):
        super().__init__()
        self.embed = ScaledEmbedding(vocab, d, scale=d ** 0.5)
        self.drop = nn.ModuleList(FusedDropout(0.1, seed=k) for k in range(2))
        self.norm = nn.ModuleList(FusedLayerNorm(d) for _ in range(2))
        self.hidden = nn.ModuleList(nn.Linear(d, d) for _ in range(2))
        self.out = nn.Linear(d, classes)
        with torch.no_grad():
            self.embed.weight.normal_(0, d ** -0.5)

    def forward(self, ids):
        y = h = self.embed(ids)
        for lin, drop, norm in zip(self.hidden, self.drop, self.norm):
            y, h = norm(drop(torch.relu(lin(y))), h)
        return self.out(y.mean(1))


@pytest.mark.parametrize("dev", devices())
@pytest.mark.parametrize("cast", [None, torch.bfloat16])
def test_the_layers_in_the_frameworks_module_program(cast, dev):
    torch.manual_seed(4)
    ids, labels = torch.randint(0, 50, (64, 12)), torch.randint(0, 10, (64,))
    net = Net()
    prog = TorchModuleProgram(net, dev, ids, labels, batch=16, optimizer="sgd", lr=0.05, channels_last=False, autocast=cast)
    before = prog.state.params.clone()
    SyncReplicasEngine(prog, prog.state).run(4)
    assert torch.isfinite(prog.log[:4]).all() and torch.isfinite(prog.state.params).all()
    assert not torch.equal(before, prog.state.params) and [int(d.step) for d in net.drop] == [4, 4]
    # the gradient of the step against the same step on float64, layer by layer stock PyTorch with the same masks
    x, y = prog.images[:8], prog.labels[:8]
    net.zero_grad()
    with torch.autocast(dev.split(":")[0], dtype=cast or torch.bfloat16, enabled=cast is not None):
        logits = net(x)
    grads = torch.autograd.grad(F.cross_entropy(logits.float(), y), list(net.parameters()))
    wide = {n: p.detach().double().requires_grad_(True) for n, p in net.named_parameters()}
    n = h = wide["embed.weight"][x] * 48 ** 0.5
    for k in range(2):
        a = torch.relu(n @ wide[f"hidden.{k}.weight"].t() + wide[f"hidden.{k}.bias"])
        keep = dropout_apply(torch.ones_like(a, dtype=torch.float32), 0.1, k, 4).double()
        h = h + a * keep
        n = F.layer_norm(h, (48,), wide[f"norm.{k}.weight"], wide[f"norm.{k}.bias"])
    loss = F.cross_entropy(n.mean(1) @ wide["out.weight"].t() + wide["out.bias"], y)
    want = torch.autograd.grad(loss, list(wide.values()))
    # a chain of a dozen operators on values of order one to ten: 2000 roundings in float32; with bfloat16 products twelve of
    # those (forward and backward), each of half a step 2^-8 and grown by at most four behind the layer norms
    for name, g, e in zip(wide, grads, want):
        assert_within(g, e, (12 * 4 * 2.0 ** -8 if cast else 2000 * U32) * e.abs().max(), name)
