"""Forward-mode derivatives of the token-model operators: right on the CPU (plain PyTorch), refused by the kernels."""
import pytest
import torch
from torch.autograd import forward_ad

from distributed_tensorflow_amd.ops import _token
from distributed_tensorflow_amd.ops.dropout import dropout, dropout_apply
from distributed_tensorflow_amd.ops.embedding import embedding
from distributed_tensorflow_amd.ops.layernorm import layer_norm, layer_norm_fwd
from distributed_tensorflow_amd.ops.vocab_xent import vocab_xent, vocab_xent_fwd


def calls(dev):
    """name -> (function of one tensor, that tensor)"""
    g = torch.Generator().manual_seed(3)
    draw = lambda *s: torch.randn(s, generator=g, dtype=torch.float32).to(dev)  # noqa: E731
    x, w, b, table = draw(6, 16), draw(16), draw(16), draw(20, 16)
    ids = torch.tensor([3, 0, 3, 7, 19, 1], device=dev)
    return {
        "layer_norm of x": (lambda t: layer_norm(t, w, b), x), "layer_norm of weight": (lambda t: layer_norm(x, t, b), w),
        "layer_norm of bias": (lambda t: layer_norm(x, w, t), b), "layer_norm of residual": (lambda t: layer_norm(x, w, b, residual=t)[0], x + 1),
        "layer_norm_fwd": (lambda t: layer_norm_fwd(t, w, b).y, x),
        "dropout of x": (lambda t: dropout(t, 0.3, 5), x), "dropout of residual": (lambda t: dropout(x, 0.3, 5, residual=t), x + 1),
        "dropout_apply": (lambda t: dropout_apply(t, 0.3, 5), x),
        "embedding": (lambda t: embedding(ids, t, 2.0), table),
        "vocab_xent of features": (lambda t: vocab_xent(t, table, ids)[0], x), "vocab_xent of weight": (lambda t: vocab_xent(x, t, ids)[0], table),
        "vocab_xent of bias": (lambda t: vocab_xent(x, table, ids, t)[0], draw(20)),
        "vocab_xent_fwd": (lambda t: vocab_xent_fwd(t, table, ids).loss, x),
    }


@pytest.mark.parametrize("name", list(calls("cpu")))
def test_tangents_on_the_cpu(name):
    f, x = calls("cpu")[name]
    d = torch.randn(x.shape, generator=torch.Generator().manual_seed(4))
    with forward_ad.dual_level():
        tangent = forward_ad.unpack_dual(f(forward_ad.make_dual(x, d))).tangent
    h = 2.0 ** -7          # central differences of values of order one: 1e-6 of noise over the step, third-order term 1e-4
    want = (f(x + h * d).double() - f(x - h * d).double()) / (2 * h)
    assert (tangent.double() - want).abs().max() < 5e-3 * (1 + want.abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(calls("cpu")))
def test_tangents_are_refused_on_the_gpu(name):
    f, x = calls("cuda:0")[name]
    want = f(x)
    with forward_ad.dual_level():
        assert torch.equal(f(x), want)                     # no tangent: as ever
        with pytest.raises(NotImplementedError, match="forward-mode"):
            f(forward_ad.make_dual(x, torch.ones_like(x)))
    for leaf in (x.clone().requires_grad_(True),):         # with a backward pass as well: PyTorch's refusal or this one
        with forward_ad.dual_level(), pytest.raises(RuntimeError):
            f(forward_ad.make_dual(leaf, torch.ones_like(leaf)))


def test_the_refusal_itself():
    x = torch.ones(3)
    _token.refuse_tangents("f", x, None)
    with forward_ad.dual_level():
        _token.refuse_tangents("f", x, None)
        with pytest.raises(NotImplementedError, match="f: no forward-mode"):
            _token.refuse_tangents("f", x, None, forward_ad.make_dual(x, x))
