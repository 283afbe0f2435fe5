"""TorchModuleProgram with a module that brings its own loss: a token model whose head is the vocabulary cross entropy."""
import copy
import math

import pytest
import torch
import torch.nn as nn

from distributed_tensorflow_amd.models.resnet import TorchModuleProgram
from distributed_tensorflow_amd.ops.dropout import FusedDropout
from distributed_tensorflow_amd.ops.embedding import ScaledEmbedding
from distributed_tensorflow_amd.ops.layernorm import FusedLayerNorm
from distributed_tensorflow_amd.ops.vocab_xent import vocab_xent
from distributed_tensorflow_amd.parallel.sync_replicas import SyncReplicasEngine
from token_utils import U32, assert_within, devices

V, D, T, PAD = 97, 32, 12, 0


class TokenModel(nn.Module):
    def __init__(self):
        super().__init__()
        self.embed = ScaledEmbedding(V, D, scale=math.sqrt(D), padding_idx=PAD)
        self.drop, self.norm, self.hidden = FusedDropout(0.1, seed=3), FusedLayerNorm(D), nn.Linear(D, D)
        with torch.no_grad():
            self.embed.weight.normal_(0, 1 / math.sqrt(D))

    def forward(self, ids):
        h = self.embed(ids)
        y, _ = self.norm(self.drop(torch.relu(self.hidden(h))), h)
        return y

    def training_loss(self, ids, labels):
        return vocab_xent(self(ids).reshape(-1, D), self.embed.weight, labels.reshape(-1), ignore_index=PAD)


def data():
    g = torch.Generator().manual_seed(5)
    ids = torch.randint(1, V, (40, T), generator=g)
    ids[::3, -4:] = PAD
    return ids, torch.roll(ids, -1, 1)


@pytest.mark.parametrize("dev", devices())
def test_steps_are_those_of_a_plain_loop(dev):
    ids, labels = data()
    torch.manual_seed(2)
    model = TokenModel()
    plain = copy.deepcopy(model).to(dev)
    prog = TorchModuleProgram(model, dev, ids, labels, batch=8, optimizer="sgd", lr=0.1, channels_last=False)
    SyncReplicasEngine(prog, prog.state).run(5)
    recs = prog.read_log(0, 5)
    for s, rec in enumerate(recs):
        lo = (s * 8) % 33
        loss, hits = plain.training_loss(ids[lo:lo + 8].to(dev), labels[lo:lo + 8].to(dev))
        grads = torch.autograd.grad(loss, list(plain.parameters()))
        assert abs(rec.loss - float(loss.detach())) < 1e-4 and rec.train_correct == int(hits)
        with torch.no_grad():
            for p, g in zip(plain.parameters(), grads):
                p -= 0.1 * g
    for p, q in zip(model.parameters(), plain.parameters()):          # five steps of a dozen operators
        assert_within(p, q.detach().double(), 5 * 2000 * U32 * q.detach().double().abs().max())
    assert int(model.drop.step) == 5


@pytest.mark.gpu
@pytest.mark.parametrize("cast", [None, torch.bfloat16])
def test_captured_steps_follow_the_eager_ones(cast, monkeypatch):
    ids, labels = data()
    logs = []
    for graph in ("0", "1"):
        monkeypatch.setenv("DTF_MODULE_GRAPH", graph)
        torch.manual_seed(2)
        model = TokenModel()
        prog = TorchModuleProgram(model, "cuda:0", ids, labels, batch=8, optimizer="adam", lr=1e-2, channels_last=False, autocast=cast)
        SyncReplicasEngine(prog, prog.state).run(8)
        torch.cuda.synchronize()
        assert (prog._graph is not None) == (graph == "1") and int(model.drop.step) == 8
        logs.append([r.loss for r in prog.read_log(0, 8)])
    # the hidden layer's library product may choose another order of sums in a graph; Adam turns that into steps' last bits
    assert all(abs(a - b) < 2e-2 for a, b in zip(*logs))
