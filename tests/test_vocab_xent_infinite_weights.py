"""float32 vocabulary cross entropy with weight rows of infinities or of the type's lowest value (classes that are masked out):
the same results at every size, whichever kernels the size selects."""
import pytest
import torch

from distributed_tensorflow_amd.ops import vocab_xent as vx
from test_large_vocab_xent import draw, exact, run
from token_utils import assert_within, devices

# one tile of 16 rows a workgroup, two, four; planes in the 128x128 blocks, in the 256x256 ones; more than 448 rows beside them
SIZES = [(40, 300, 24), (20, 33000, 9), (40, 33000, 300), (448, 6001, 95), (500, 16401, 130), (600, 16001, 520), (1000, 9001, 257)]


def masked(n, v, d, dev, value):
    x, w, lab, b = (t.to(dev) for t in draw(n, v, d, torch.float32, pad=0.0))
    x = x.abs() + 0.1                              # every product with the masked rows is negative
    keep = torch.ones(v, dtype=torch.bool, device=dev)
    keep[10::20] = False
    keep[-1] = False
    lab = torch.where(keep[lab], lab, 0)
    rank = torch.cumsum(keep, 0) - 1               # a kept class' index among the kept ones
    want = exact(x, w[keep], rank[lab], b[keep])
    w[~keep] = value
    return x, w, lab, b, keep, want


def compare(dev, x, w, lab, b, keep, want, finite):
    r, (dx, dw, db) = run(x, w, lab, b, dev)
    assert_within(r.loss_rows, *want["rows"], "loss rows")
    assert_within(r.lse, *want["lse"], "lse")
    assert int(r.hits) == want["hits"]
    assert_within(dw[keep], *want["dw"], "dweight")
    assert_within(db[keep], *want["db"], "dbias")
    assert not dw[~keep].any() and not db[~keep].any()
    if finite:
        assert_within(dx, *want["dx"], "dfeatures")
    else:
        assert torch.isnan(dx).all()               # 0 times infinity


@pytest.mark.parametrize("dev", devices())
@pytest.mark.parametrize("n,v,d", SIZES)
def test_rows_of_infinities(n, v, d, dev):
    compare(dev, *masked(n, v, d, dev, -float("inf")), finite=False)


@pytest.mark.parametrize("dev", devices())
@pytest.mark.parametrize("n,v,d", SIZES)
def test_rows_of_the_lowest_value(n, v, d, dev):
    """Finite, though not in bfloat16: their logits are -inf or near it, their share of dfeatures is 0 times a number."""
    compare(dev, *masked(n, v, d, dev, torch.finfo(torch.float32).min), finite=True)


@pytest.mark.parametrize("dev", devices())
@pytest.mark.parametrize("n,v,d", SIZES)
def test_a_row_of_nan_features_stays_alone(n, v, d, dev):
    x, w, lab, b = (t.to(dev) for t in draw(n, v, d, torch.float32, pad=0.0))
    clean, (cx, _, _) = run(x, w, lab, b, dev)
    x[5, d // 2] = float("nan")
    r, (dx, dw, _) = run(x, w, lab, b, dev)
    others = torch.arange(n) != 5
    assert torch.isnan(r.loss_rows[5]) and torch.isnan(dx[5]).all() and torch.isnan(dw).all()
    assert torch.equal(r.loss_rows[others], clean.loss_rows[others]) and torch.equal(dx[others], cx[others])


@pytest.mark.gpu
def test_one_infinity_of_a_row_reaches_one_column_of_dfeatures():
    for n, v, d in SIZES:
        x, w, lab, b, keep, _ = masked(n, v, d, "cuda:0", 0.5)
        w[~keep, d // 3] = -float("inf")
        r = vx.vocab_xent_fwd(x, w, lab, b)
        dx, dw, db = vx.vocab_xent_bwd(r, x, w, lab, b)
        others = torch.arange(d) != d // 3
        assert torch.isfinite(r.loss_rows).all() and torch.isfinite(dw).all() and torch.isfinite(db).all()
        assert torch.isnan(dx[:, d // 3]).all() and torch.isfinite(dx[:, others]).all()
