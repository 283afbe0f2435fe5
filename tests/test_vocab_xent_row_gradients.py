"""Gradients of a vocabulary cross entropy with one upstream gradient for each row (reduction "none")."""
import pytest
import torch

from distributed_tensorflow_amd.ops import vocab_xent as vx
from test_large_vocab_xent import IGN, draw, exact, run
from token_utils import U32, assert_within, devices, half_step

# sizes at which the products read dz rounded to bfloat16, by each of the logits' kernels: shared K, 128x128, 256x256
# blocks, the last two also over several K ranges and at widths that go through copies
SIZES = [(40, 300, 64), (300, 16400, 40), (260, 49999, 320), (777, 16001, 1024), (700, 4003, 71)]


def slope(got, want):
    """How large ``got`` is along ``want``, relative to it: 1 if the errors have no direction in common."""
    got, want = got.detach().double().flatten(), want.double().flatten()
    return float((got @ want) / (want @ want))


@pytest.mark.gpu
@pytest.mark.parametrize("n,v,d", SIZES)
@pytest.mark.parametrize("wdtype", [torch.bfloat16, torch.float32])
def test_equal_row_gradients_carry_no_common_rounding(n, v, d, wdtype):
    """1 / 8160 lies half-way between two bfloat16 numbers: rounded with it, the label's elements of dz would all be off by
    2^-8 of themselves in the same direction, and so would the gradients.  The rounding of p - 1, the final one and those of X
    have no common sign: each at most 2^-9 of its element, over at least 30 rows of labels 2^-9 / sqrt(30) = 2^-11.4 of
    the whole; and a probability below 2^-9 that is lost beside 1 (a label's, 1 / V or so where it is not the maximum) 2^-12
    at the mean.  2^-10 bounds the sum, a quarter of what the common rounding does."""
    x, w, lab, _ = (t if t is None else t.cuda() for t in draw(n, v, d, torch.bfloat16, wdtype, bias=False))
    g = torch.full((n,), 1 / 8160, device="cuda")
    r = vx.vocab_xent_fwd(x, w, lab, ignore_index=IGN, reduction="none")
    dx, dw, _ = vx.vocab_xent_bwd(r, x, w, lab, dloss=g)
    want = exact(x, w, lab, None, "none", g, torch.bfloat16)
    assert abs(slope(dx, want["dx"][0]) - 1) < 2.0 ** -10 and abs(slope(dw, want["dw"][0]) - 1) < 2.0 ** -10
    # the same as the sum's gradient times the factor: nothing but that product and the last rounding may differ
    s = vx.vocab_xent_fwd(x, w, lab, ignore_index=IGN, reduction="sum")
    sx, sw, _ = vx.vocab_xent_bwd(s, x, w, lab, dloss=g[0])
    for a, b in ((dx, sx), (dw, sw)):
        assert_within(a, b.double(), (2 * half_step(a.dtype) + 2 * U32) * b.double().abs())


@pytest.mark.parametrize("dev", devices())
@pytest.mark.parametrize("dtype,wdtype", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32)])
@pytest.mark.parametrize("n,v,d", SIZES[:2] + [(20, 500, 48), (700, 4003, 71)])
def test_row_gradients_of_many_sizes(n, v, d, dtype, wdtype, dev):
    """Values over eight decades, zeros and both signs; bias gradients too.  Above the bounds of ``exact`` comes half a step for
    X times its row's factor, which the product dW reads in the operands' type, and 4 U32 for that factor."""
    x, w, lab, b = draw(n, v, d, dtype, wdtype)
    g = torch.Generator().manual_seed(n)
    up = torch.randn(n, generator=g) * 10.0 ** (torch.rand(n, generator=g) * 8 - 6)
    up[::7] = 0.0
    x, w, lab, b, up = (t.to(dev) for t in (x, w, lab, b, up))
    compute = dtype if dev != "cpu" else wdtype
    want = exact(x, w, lab, b, "none", up, compute)
    _, (dx, dw, db) = run(x, w, lab, b, dev, "none", up)
    xd, wd = x.double(), w.to(compute).double()
    z = xd @ wd.t() + b.double()
    p = torch.softmax(z, 1)
    p[torch.arange(n), lab.clamp_min(0)] -= 1
    dz = (p * torch.where(lab != IGN, up.double(), 0.0)[:, None]).abs()
    step = (half_step(compute) if compute == torch.bfloat16 else 0.0) + 4 * U32
    assert_within(dx, want["dx"][0], want["dx"][1] + step * (dz @ wd.abs()), "dfeatures")
    assert_within(dw, want["dw"][0], want["dw"][1] + step * (dz.t() @ xd.abs()), "dweight")
    assert_within(db, want["db"][0], want["db"][1] + 4 * U32 * dz.sum(0), "dbias")
    assert not dx[up == 0].any()


@pytest.mark.parametrize("dev", devices())
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,v", [(20, 100), (60, 300), (300, 16400), (500, 8300)])
def test_an_infinite_row_gradient_stays_in_its_row_of_dfeatures(n, v, dtype, dev):
    """And what the padding rows' gradients hold does not matter at all."""
    x, w, lab, b = (t.to(dev) for t in draw(n, v, 40, dtype, pad=0.0))
    lab[::5] = IGN
    up = torch.rand(n, generator=torch.Generator().manual_seed(1)).to(dev)
    r = vx.vocab_xent_fwd(x, w, lab, b, reduction="none")
    clean = vx.vocab_xent_bwd(r, x, w, lab, b, dloss=up)
    junk = up.clone()
    junk[::5] = float("nan")
    for a, c in zip(vx.vocab_xent_bwd(r, x, w, lab, b, dloss=junk), clean):
        assert torch.equal(a, c)
    junk[6] = float("inf")
    dx, dw, db = vx.vocab_xent_bwd(r, x, w, lab, b, dloss=junk)
    others = torch.arange(n) != 6
    assert not torch.isfinite(dx[6]).any() and torch.equal(dx[others], clean[0][others])
    assert not torch.isfinite(dw).all() and not torch.isfinite(db).all()


@pytest.mark.gpu
@pytest.mark.parametrize("wdtype", [torch.bfloat16, torch.float32])
def test_row_gradients_over_pieces_of_the_vocabulary(wdtype):
    """40 000 columns at 16 416 tokens are more than one piece; dfeatures is scaled row by row behind the last one."""
    n, v, d = 16416, 40001, 24
    x, w, lab, b = (t.cuda() for t in draw(n, v, d, torch.bfloat16, wdtype))
    r = vx.vocab_xent_fwd(x, w, lab, b, ignore_index=IGN, reduction="none")
    s = vx.vocab_xent_fwd(x, w, lab, b, ignore_index=IGN, reduction="sum")
    ones = vx.vocab_xent_bwd(s, x, w, lab, b)
    for a, c in zip(vx.vocab_xent_bwd(r, x, w, lab, b, dloss=torch.full((n,), 1 / 8160, device="cuda")), ones):
        c = c.double() / 8160
        assert_within(a, c, (2 * half_step(a.dtype) + 2 * U32) * c.abs())
    up = torch.randn(n, generator=torch.Generator().manual_seed(9)).cuda()
    dx, dw, db = vx.vocab_xent_bwd(r, x, w, lab, b, dloss=up)
    want = ones[0].double() * up.double()[:, None]                 # a row of dfeatures is linear in its gradient
    assert_within(dx, want, (2 * half_step(dx.dtype) + 4 * U32) * want.abs())
    g = torch.where(lab != IGN, up, 0.0).double()
    z = x.double() @ w.to(torch.bfloat16).double().t()[:, :64] + b.double()[:64]
    p = torch.exp(z - r.lse.double()[:, None]) - (lab[:, None] == torch.arange(64, device="cuda")).double()
    size = (p * g[:, None]).abs()
    # p off by less than 1e-4 of itself (sums of 24 and 40 001 terms), then dz and X rounded to bfloat16
    bound = (2 * half_step(torch.bfloat16) + 1e-4) * (size.t() @ x.double().abs()) + half_step(dw.dtype) * dw[:64].double().abs()
    assert_within(dw[:64], (p * g[:, None]).t() @ x.double(), bound)
    assert_within(db[:64], (p * g[:, None]).sum(0), 1e-4 * size.sum(0))


@pytest.mark.gpu
def test_row_gradients_in_replayed_graphs():
    x, w, lab, b = (t.cuda() for t in draw(300, 1111, 128, torch.bfloat16))
    up = torch.rand(300, device="cuda")

    def step():
        r = vx.vocab_xent_fwd(x, w, lab, b, reduction="none")
        return (r.loss_rows, *vx.vocab_xent_bwd(r, x, w, lab, b, dloss=up))
    step()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for k in range(3):
        up.copy_(torch.randn(300, generator=torch.Generator().manual_seed(k)) * 10.0 ** k)
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = step()
        for _, out in graphs:
            assert all(torch.equal(a, c) for a, c in zip(want, out))
