"""Softmax cross entropy over a vocabulary without kept logits (ops/vocab_xent.py) against the definition in 64 bits."""
import math

import pytest
import torch

from distributed_tensorflow_amd.ops import vocab_xent as vx
from token_utils import U32, assert_within, devices, half_step

IGN = -100


def draw(n, v, d, dtype, wdtype=None, bias=True, seed=0, pad=0.15):
    g = torch.Generator().manual_seed(seed + 7 * n + v)
    x = torch.randn((n, d), generator=g).to(dtype)
    w = (torch.randn((v, d), generator=g) * 2 / math.sqrt(d)).to(wdtype or dtype)
    b = torch.randn(v, generator=g) * 0.3 if bias else None
    lab = torch.randint(0, v, (n,), generator=g)
    best = (x.double() @ w.double().t() + (0 if b is None else b.double())).argmax(1) if n * v * d < 1 << 28 else lab
    lab = torch.where(torch.rand(n, generator=g) < 0.4, best, lab)             # some rows hit
    lab = torch.where(torch.rand(n, generator=g) < pad, IGN, lab)
    return x, w, lab, b


def exact(x, w, lab, b, reduction="mean", dloss=None, compute=None):
    """Values and element-wise error bounds in float64.  ``compute``: the type the products run in (a float32 weight under
    bfloat16 features is rounded to bfloat16 first).

    Bounds.  A logit is a sum of D products in fp32, accumulated in any order: off by at most
    e_z = (D + 2) U32 (sum |x w| + |b|).  exp, log and the sums over V in strips and joins add at most 96 U32 relative to the
    sum, plus U32 |z - lse| for the exponent's argument (times 2: log2 e and its rounding).  So lse is off by e_l = max e_z +
    (96 + 2 max|z - ref|) U32, p by p (e_z + e_l + 4 |z - lse| U32), dz additionally by half a step of the operands' type,
    and a product of K terms by K U32 and the factors' errors, each times the sum of absolute products."""
    compute = compute or x.dtype
    xd, wd = x.double(), w.to(compute).double()
    z = xd @ wd.t() + (0 if b is None else b.double())
    valid = lab != IGN
    l0 = torch.where(valid, lab, 0)
    lse = torch.logsumexp(z, 1)
    rows = torch.where(valid, lse - z.gather(1, l0[:, None])[:, 0], 0.0)
    count = int(valid.sum())
    e_z = (x.shape[1] + 2) * U32 * (xd.abs() @ wd.abs().t() + (0 if b is None else b.double().abs()))
    top = e_z.amax(1)
    e_l = top + (96 + 2 * torch.clamp(z.amax(1) - z.mean(1), max=100)) * U32 + U32 * lse.abs()
    out = {"rows": (rows, e_l + top + 2 * U32 * (lse.abs() + z.abs().amax(1)))}
    total, e_total = rows.sum(), out["rows"][1].sum() + 16 * U32 * rows.abs().sum() + x.shape[0] / 64 * U32 * rows.abs().sum()
    scale = 1.0 / max(count, 1) if reduction == "mean" else 1.0
    out["loss"] = (total * scale, e_total * scale + 2 * U32 * abs(total * scale))
    out["lse"] = (lse, e_l + U32 * lse.abs())
    out["hits"] = int(((z.argmax(1) == l0) & valid).sum())
    out["count"] = count
    up = torch.ones(x.shape[0], dtype=torch.float64, device=x.device) if dloss is None else dloss.double().expand(x.shape[0])
    gr = torch.where(valid, up * scale, 0.0)[:, None]
    p = torch.exp(z - lse[:, None])
    one = torch.zeros_like(p).scatter_(1, l0[:, None], 1.0)
    dz = (p - one) * gr
    e_p = p * (e_z + e_l[:, None] + 4 * (z - lse[:, None]).abs() * U32 + 4 * U32)
    e_dz = (e_p + 2 * U32 * (p + one)) * gr.abs() + 2 * U32 * dz.abs()
    step = half_step(compute) if compute == torch.bfloat16 else 0.0
    e_op = e_dz + step * dz.abs()                       # as operand of the two products
    n, v = p.shape
    for name, val, err, size, like in (("dx", dz @ wd, e_op @ wd.abs(), (v + 40) * (dz.abs() @ wd.abs()), x),
                                       ("dw", dz.t() @ xd, e_op.t() @ xd.abs(), (n + 40) * (dz.abs().t() @ xd.abs()), w)):
        out[name] = (val, err + U32 * size + (half_step(like.dtype)) * val.abs())
    if b is not None:
        out["db"] = (dz.sum(0), e_dz.sum(0) + (n + 8) * U32 * dz.abs().sum(0))
    return out


def run(x, w, lab, b, dev, reduction="mean", dloss=None):
    to = lambda t: None if t is None else t.to(dev)  # noqa: E731
    a = (to(x), to(w), to(lab), to(b))
    r = vx.vocab_xent_fwd(*a, ignore_index=IGN, reduction=reduction)
    return r, vx.vocab_xent_bwd(r, *a, dloss=to(dloss))


def check(n, v, d, dtype, dev, wdtype=None, bias=True, reduction="mean", dloss=None, seed=0, data=None):
    x, w, lab, b, dloss = (None if t is None else t.to(dev) for t in (*(data or draw(n, v, d, dtype, wdtype, bias, seed)), dloss))
    want = exact(x, w, lab, b, reduction, dloss, dtype if dev != "cpu" else (wdtype or dtype))
    r, (dx, dw, db) = run(x, w, lab, b, dev, reduction, dloss)
    assert_within(r.loss_rows, *want["rows"], "loss rows")
    assert_within(r.lse, *want["lse"], "lse")
    assert_within(r.loss.reshape(1), want["loss"][0].reshape(1), want["loss"][1], "loss")
    assert int(r.hits) == want["hits"] and int(r.count) == want["count"]
    assert dx.dtype == x.dtype and dw.dtype == w.dtype
    assert_within(dx, *want["dx"], "dfeatures")
    assert_within(dw, *want["dw"], "dweight")
    if b is not None:
        assert_within(db, *want["db"], "dbias")
    else:
        assert db is None
    pad = lab == IGN
    assert not dx[pad].any() and not r.loss_rows[pad].any()


SIZES = [(1, 1, 1), (1, 2, 8), (1, 1000, 64), (2, 63, 16), (3, 64, 24), (5, 65, 40), (7, 129, 100), (17, 257, 7), (100, 1000, 256),
         (127, 10, 33), (128, 128, 128), (129, 300, 264), (300, 77, 72), (260, 515, 20),
         (16, 16500, 24), (17, 16500, 40), (32, 8200, 33), (33, 8200, 33), (48, 16500, 40), (49, 16500, 40), (64, 16500, 130), (65, 16500, 130),
         (255, 9001, 48), (256, 9001, 48)]


@pytest.mark.parametrize("dev", devices())
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,v,d", SIZES)
def test_sizes(n, v, d, dtype, dev):
    check(n, v, d, dtype, dev, bias=v % 2 == 0)


@pytest.mark.gpu
@pytest.mark.parametrize("n,v,d", [(3001, 5003, 264), (1024, 12544, 512), (777, 16001, 1024), (2048, 8192, 256), (260, 49999, 320)])
def test_sizes_of_the_large_blocks(n, v, d):
    """Token and vocabulary counts at which the 256x256 blocks run, ragged and whole."""
    check(n, v, d, torch.bfloat16, "cuda:0", bias=n % 2 == 0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,wdtype,n,v,d", [
    (torch.float32, torch.float32, 20, 33000, 9), (torch.float32, torch.float32, 33, 33000, 33), (torch.float32, torch.float32, 40, 33000, 300),
    (torch.float32, torch.float32, 200, 8300, 130), (torch.float32, torch.float32, 255, 20001, 257), (torch.float32, torch.float32, 96, 16500, 64),
    (torch.bfloat16, torch.bfloat16, 20, 33000, 700), (torch.bfloat16, torch.float32, 31, 33000, 701), (torch.float32, torch.float32, 700, 130, 1030),
    (torch.float32, torch.float32, 448, 6001, 95), (torch.float32, torch.float32, 449, 6001, 96), (torch.float32, torch.float32, 18, 33001, 31),
    (torch.float32, torch.float32, 300, 17000, 32), (torch.float32, torch.float32, 6, 140000, 66)])
def test_sizes_of_the_kernels_of_few_rows(dtype, wdtype, n, v, d):
    """Sizes at which a workgroup takes one, two and four tiles of 16 rows; widths of whole and of broken 16-byte pieces."""
    check(n, v, d, dtype, "cuda:0", wdtype=wdtype, bias=n % 2 == 0)


@pytest.mark.gpu
@pytest.mark.parametrize("n,v,d", [(449, 9001, 33), (500, 16401, 130), (600, 16001, 520), (1000, 9001, 257), (1030, 700, 64)])
def test_float32_sizes_of_the_planes(n, v, d):
    check(n, v, d, torch.float32, "cuda:0", bias=n % 2 == 0)


@pytest.mark.gpu
def test_a_weight_row_of_infinities_behind_a_broken_piece():
    """Width 5: the 16-byte piece that ends a row reaches into the next one, whose logits are -inf here and stay apart."""
    x, w, lab, b = draw(40, 300, 5, torch.float32, pad=0.0)
    x, lab = x.abs() + 0.1, lab % 7
    w[10::20] = -float("inf")
    r, (dx, dw, db) = run(x, w, lab, b, "cuda:0")
    keep = torch.ones(300, dtype=torch.bool)
    keep[10::20] = False
    want = exact(x, w[keep], lab, b[keep])
    assert_within(r.loss_rows.cpu(), *want["rows"], "loss rows")
    assert_within(dw.cpu()[keep], *want["dw"], "dweight")
    assert not dw.cpu()[~keep].any() and not db.cpu()[~keep].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,wdtype", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32)])
def test_pieces_of_the_vocabulary(dtype, wdtype):
    """40 000 columns at 16 416 tokens are more than one piece (1 GiB of dz and dz^T), the last one ragged.  Column and row
    subsets are compared: the whole in 64 bits would take minutes."""
    n, v, d = 16416, 40001, 24
    x, w, lab, b = draw(n, v, d, dtype, wdtype)
    r, (dx, dw, db) = run(x, w, lab, b, "cuda:0")
    xd, wd, bd = x.cuda().double(), w.cuda().to(dtype).double(), b.cuda().double()
    lse = torch.cat([torch.logsumexp(xd[i:i + 2048] @ wd.t() + bd, 1) for i in range(0, n, 2048)])
    assert (r.lse.double() - lse).abs().max() < 4e-5          # (24 + 2 + 96 + 40) U32 times values up to 4
    valid = (lab != IGN).cuda()
    g = valid.double() / valid.sum()
    cols = torch.cat([torch.arange(0, 300), torch.arange(15000, 17000, 7), torch.arange(v - 300, v)]).cuda()
    one = (lab.cuda()[:, None] == cols[None, :]).double()
    dz = (torch.exp(xd @ wd[cols].t() + bd[cols] - lse[:, None]) - one) * g[:, None]
    want, size = dz.t() @ xd, dz.abs().t() @ xd.abs()
    step = half_step(torch.bfloat16) if dtype == torch.bfloat16 else 2e-5          # fp32: p off by (e_z + e_l) < 2e-5
    assert_within(dw[cols], want, step * size + 1e-4 * size / 16 + half_step(dw.dtype) * want.abs(), "dweight")
    assert_within(db[cols], dz.sum(0), 1e-4 * dz.abs().sum(0), "dbias")
    rows = torch.arange(0, n, 97).cuda()
    dzr = torch.exp(xd[rows] @ wd.t() + bd - lse[rows, None])
    dzr[torch.arange(len(rows)), lab.cuda()[rows].clamp_min(0)] -= 1
    dzr *= g[rows, None]
    want, size = dzr @ wd, dzr.abs() @ wd.abs()
    assert_within(dx[rows], want, step * size + 1e-4 * size / 16 + half_step(dx.dtype) * want.abs(), "dfeatures")


@pytest.mark.parametrize("dev", devices())
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_reductions_and_upstream_gradients(reduction, dev):
    g = torch.Generator().manual_seed(4)
    up = torch.randn(70, generator=g) if reduction == "none" else torch.tensor(-1.75)
    check(70, 200, 48, torch.float32, dev, reduction=reduction, dloss=up)


@pytest.mark.parametrize("dev", devices())
def test_float32_weight_under_bfloat16_features(dev):
    check(90, 333, 72, torch.bfloat16, dev, wdtype=torch.float32)
    check(40, 333, 71, torch.bfloat16, dev, wdtype=torch.float32)


@pytest.mark.parametrize("dev", devices())
def test_no_rows_and_no_labels(dev):
    w = torch.randn(50, 16, device=dev)
    b = torch.randn(50, device=dev)
    x0, l0 = torch.empty((0, 16), device=dev), torch.empty(0, dtype=torch.int64, device=dev)
    for x, lab in ((x0, l0), (torch.randn(9, 16, device=dev), torch.full((9,), IGN, device=dev))):
        r = vx.vocab_xent_fwd(x, w, lab, b)
        dx, dw, db = vx.vocab_xent_bwd(r, x, w, lab, b)
        assert float(r.loss) == 0 and int(r.hits) == 0 and int(r.count) == 0
        assert dx.shape == x.shape and not dx.any() and not dw.any() and not db.any()


@pytest.mark.parametrize("dev", devices())
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_ties_go_to_the_lowest_index(dtype, dev):
    """Equal logits: whole rows (zero features), within a strip, across strips, across blocks."""
    v, d = 700, 32
    x = torch.zeros(8, d)
    w = torch.randn(v, d, generator=torch.Generator().manual_seed(1))
    x[4:] = 1.0
    w[[5, 9, 70, 300, 699]] = 2.0                               # the same, largest logit five times
    lab = torch.tensor([0, 1, 64, 699, 5, 9, 70, 699])
    r = vx.vocab_xent_fwd(x.to(dtype).to(dev), w.to(dtype).to(dev), lab.to(dev))
    assert int(r.hits) == 2
    alone = [int(vx.vocab_xent_fwd(x[i:i + 1].to(dtype).to(dev), w.to(dtype).to(dev), lab[i:i + 1].to(dev)).hits) for i in range(8)]
    assert alone == [1, 0, 0, 0, 1, 0, 0, 0]


@pytest.mark.parametrize("dev", devices())
def test_masked_vocabulary_and_large_logits(dev):
    """A bias of -inf takes classes (here whole strips) out; logits of some thousands do not overflow."""
    x, w, _, b = draw(33, 300, 40, torch.float32)
    b[64:192] = float("-inf")
    b[299] = float("-inf")
    lab = torch.randint(0, 64, (33,), generator=torch.Generator().manual_seed(2))
    x[3] *= 2000.0
    r, (dx, dw, db) = run(x, w, lab, b, dev)
    keep = torch.isfinite(b)
    want = exact(x, w[keep], lab, b[keep])
    assert_within(r.loss_rows, *want["rows"], "rows")
    assert_within(dx, want["dx"][0], want["dx"][1], "dx")
    assert not dw[~keep].any() and not db[~keep].any()
    assert_within(dw[keep], *want["dw"], "dw")


@pytest.mark.parametrize("dev", devices())
def test_nan_stays_in_its_row(dev):
    x, w, lab, b = draw(40, 200, 24, torch.float32, pad=0.0)
    clean, _ = run(x, w, lab, b, dev)
    x[7, 3] = float("nan")
    r, (dx, _, _) = run(x, w, lab, b, dev)
    others = torch.arange(40) != 7
    assert torch.isnan(r.loss_rows[7]) and torch.isnan(r.loss) and torch.isnan(dx[7]).all()
    assert torch.equal(r.loss_rows[others], clean.loss_rows[others]) and torch.isfinite(dx[others]).all()


@pytest.mark.parametrize("dev", devices())
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,v", [(20, 100), (60, 300), (100, 300), (300, 16400), (70, 33000), (500, 8300)])
def test_padding_rows_may_hold_nan_and_infinity(n, v, dtype, dev):
    """Every path of the backward pass: rows with the ignored label are as good as rows of zeros."""
    x, w, lab, b = draw(n, v, 40, dtype)
    lab[::3] = IGN
    zero, junk = x.clone(), x.clone()
    zero[::3] = 0
    junk[0::6], junk[3::6] = float("nan"), float("inf")
    r0, g0 = run(zero, w, lab, b, dev)
    r1, g1 = run(junk, w, lab, b, dev)
    assert torch.equal(r0.loss, r1.loss) and torch.equal(r0.loss_rows, r1.loss_rows) and torch.equal(r0.counts, r1.counts)
    for a, c in zip(g0, g1):
        assert torch.isfinite(c).all() and torch.equal(a, c)


def test_labels_outside_the_vocabulary_raise_on_the_cpu():
    x, w, lab, b = draw(6, 20, 8, torch.float32)
    for bad in (20, -1, 1 << 40):
        lab[2] = bad
        with pytest.raises(IndexError):
            vx.vocab_xent_fwd(x, w, lab, b)


@pytest.mark.gpu
def test_labels_outside_the_vocabulary_are_nan_on_the_gpu():
    x, w, lab, b = draw(6, 20, 8, torch.float32, pad=0.0)
    good = lab.clone()
    for bad in (20, -1, 63, 1 << 40, -(1 << 40)):
        lab = good.clone()
        lab[2] = bad
        r, (dx, dw, db) = run(x, w, lab, b, "cuda:0")
        assert torch.isnan(r.loss) and torch.isnan(r.loss_rows[2]) and int(torch.isnan(r.loss_rows).sum()) == 1
        assert not dx[2].any() and torch.isfinite(dx).all() and torch.isfinite(dw).all() and torch.isfinite(db).all()


@pytest.mark.parametrize("dev", devices())
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [50, 90])
def test_strides_alignment_and_label_views(n, dtype, dev):
    x, w, lab, b = (t.to(dev) for t in draw(n, 150, 64, dtype))
    base = vx.vocab_xent_fwd(x, w, lab, b)
    grads = vx.vocab_xent_bwd(base, x, w, lab, b)
    wide_x, wide_w = torch.zeros(n, 131, device=dev, dtype=dtype), torch.zeros(150, 80, device=dev, dtype=dtype)
    wide_x[:, 3:67], wide_w[:, 8:72] = x, w
    two = torch.stack([lab, lab], 1)
    for xv, wv, lv in ((wide_x[:, 3:67], wide_w[:, 8:72], two[:, 0]), (x.t().contiguous().t(), w.t().contiguous().t(), lab)):
        r = vx.vocab_xent_fwd(xv, wv, lv, b)
        assert torch.equal(r.loss_rows, base.loss_rows)
        for a, c in zip(vx.vocab_xent_bwd(r, xv, wv, lv, b), grads):
            assert torch.equal(a, c)


@pytest.mark.parametrize("dev", devices())
def test_autograd_and_selected_gradients(dev):
    x, w, lab, b = (t.to(dev) for t in draw(60, 210, 40, torch.float32))
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    loss, hits = vx.vocab_xent(leaves[0], leaves[1], lab, leaves[2])
    (3.0 * loss).backward()
    r = vx.vocab_xent_fwd(x, w, lab, b)
    want = vx.vocab_xent_bwd(r, x, w, lab, b, dloss=torch.tensor(3.0, device=dev))
    for leaf, t in zip(leaves, want):
        assert torch.equal(leaf.grad, t)
    assert int(hits) == int(r.hits)
    only = w.clone().requires_grad_(True)
    vx.vocab_xent(x, only, lab, b, reduction="none")[0].sum().backward()
    full = vx.vocab_xent_bwd(vx.vocab_xent_fwd(x, w, lab, b, reduction="none"), x, w, lab, b)
    assert torch.equal(only.grad, full[1])
    assert not vx.vocab_xent(x, w, lab, b)[0].requires_grad


@pytest.mark.parametrize("dev", devices())
def test_gradient_against_differences(dev):
    """Central differences along random directions with step 2^-6: noise (64 U32 of a loss near 6) over the step and the
    third-order term stay below 3e-3 of |gradient| |direction|."""
    x, w, lab, b = (t.to(dev) for t in draw(40, 120, 32, torch.float32))
    f = lambda *a: vx.vocab_xent_fwd(a[0], a[1], lab, a[2], reduction="none").loss_rows.double().sum()  # noqa: E731
    r = vx.vocab_xent_fwd(x, w, lab, b, reduction="sum")
    args, h = [x, w, b], 2.0 ** -6
    for k, g in enumerate(vx.vocab_xent_bwd(r, x, w, lab, b)):
        d = torch.randn(args[k].shape, generator=torch.Generator().manual_seed(k)).to(dev)
        d *= 4.0 / d.norm()
        plus, minus = list(args), list(args)
        plus[k], minus[k] = args[k] + h * d, args[k] - h * d
        slope = (f(*plus) - f(*minus)) / (2 * h)
        assert abs(float(slope - (g.double() * d.double()).sum())) < 3e-3 * float(g.norm() * d.norm())


@pytest.mark.parametrize("dev", devices())
def test_refusals(dev):
    x, w, lab, b = (t.to(dev) for t in draw(6, 20, 8, torch.float32))
    r = vx.vocab_xent_fwd(x, w, lab, b)
    bad = [lambda: vx.vocab_xent(x.half(), w.half(), lab), lambda: vx.vocab_xent(x, w.bfloat16(), lab), lambda: vx.vocab_xent(x, w[:, :4], lab),
           lambda: vx.vocab_xent(x, w, lab[:3]), lambda: vx.vocab_xent(x, w, lab.int()), lambda: vx.vocab_xent(x, w, lab, b[:5]),
           lambda: vx.vocab_xent(x, w, lab, b, reduction="median"), lambda: vx.vocab_xent(x, w[:0], lab), lambda: vx.vocab_xent(x[:, :0], w[:, :0], lab),
           lambda: vx.vocab_xent(x[None], w, lab), lambda: vx.vocab_xent_bwd(r, x, w, lab, b, dloss=torch.ones(6, device=dev)),
           lambda: vx.vocab_xent_bwd(r, x[:3], w, lab[:3], b)]
    for call in bad:
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("dev", devices())
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,v", [(20, 100), (100, 300), (300, 16400), (500, 8300)])
def test_selected_gradients_are_those_of_a_full_call(n, v, dtype, dev):
    x, w, lab, b = (t.to(dev) for t in draw(n, v, 40, dtype))
    r = vx.vocab_xent_fwd(x, w, lab, b)
    full = vx.vocab_xent_bwd(r, x, w, lab, b)
    for k in range(1, 8):
        want = [bool(k >> i & 1) for i in range(3)]
        for got, one, take in zip(vx.vocab_xent_bwd(r, x, w, lab, b, want=want), full, want):
            assert torch.equal(got, one) if take else got is None


@pytest.mark.parametrize("dev", devices())
def test_sizes_of_more_than_32_bits_are_refused(dev):
    one = torch.zeros((1, 1), device=dev)
    lab = torch.zeros(1, dtype=torch.int64, device=dev)
    with pytest.raises(ValueError, match="range"):
        vx.vocab_xent_fwd(one.expand(2 ** 32 + 4, 1), one, lab.expand(2 ** 32 + 4))
    with pytest.raises(ValueError, match="range"):
        vx.vocab_xent_fwd(one.expand(1, 2 ** 32 + 4), one.expand(3, 2 ** 32 + 4), lab)


@pytest.mark.gpu
def test_more_blocks_of_logits_than_one_launch_may_have():
    """2^20 x 2^19 logits are 2^25 blocks of 128 x 128 and 2^33 threads; 64 distinct rows stand for all."""
    n, v, d = 1 << 20, 1 << 19, 8
    g = torch.Generator(device="cuda").manual_seed(4)
    x, w = torch.randn((64, d), generator=g, device="cuda").bfloat16(), torch.randn((v, d), generator=g, device="cuda").bfloat16()
    lab = torch.randint(0, v, (64,), generator=g, device="cuda")
    r = vx.vocab_xent_fwd(x.repeat(n // 64, 1), w, lab.repeat(n // 64))
    z = x.double() @ w.double().t()
    want = torch.logsumexp(z, 1) - z.gather(1, lab[:, None])[:, 0]
    # sum |x w| stays below 100, so a logit is off by at most 10 U32 * 100 = 6e-5; lse by that and 150 U32
    assert float((x.double().abs() @ w.double().abs().t()).max()) < 100
    assert float((r.loss_rows.double().reshape(-1, 64) - want).abs().max()) < 2e-4
    assert int(r.count) == n and int(r.hits) == int((z.argmax(1) == lab).sum()) * (n // 64)


@pytest.mark.gpu
def test_operands_of_two_gibibytes_are_refused():
    x = torch.empty((1, 8), dtype=torch.bfloat16, device="cuda").expand(1 << 27, 8)
    lab = torch.empty(1, dtype=torch.int64, device="cuda").expand(1 << 27)
    a = vx._Args(N=1 << 27, D=8, V=10, ldx=8, ldw=8, dtype=1, w_dtype=1)
    assert vx._kernels().dtf_vocab_xent_ws_bytes(vx.C.byref(a), 0) == -1
    with pytest.raises(ValueError):
        vx._workspace(a, 0, "cuda")
    del x, lab


@pytest.mark.gpu
def test_same_bits_again_on_another_stream_and_in_replayed_graphs():
    x, w, lab, b = (t.cuda() for t in draw(300, 1111, 128, torch.bfloat16))

    def step():
        r = vx.vocab_xent_fwd(x, w, lab, b)
        return (r.loss, r.loss_rows, r.counts) + vx.vocab_xent_bwd(r, x, w, lab, b)
    first = [t.clone() for t in step()]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = step()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, c) for a, c in zip(first, other))
    graphs = []
    for _ in range(2):                                          # two graphs, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for k in range(3):
        x.copy_(draw(300, 1111, 128, torch.bfloat16, seed=50 + k)[0])
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = step()
        for _, out in graphs:
            assert all(torch.equal(a, c) for a, c in zip(want, out))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_millions_of_columns(dtype):
    """More than 65535 tiles of 64 vocabulary rows."""
    n, v, d = 2, 4_300_000, 8
    g = torch.Generator(device="cuda").manual_seed(3)
    x, w = torch.randn((n, d), generator=g, device="cuda").to(dtype), torch.randn((v, d), generator=g, device="cuda").to(dtype)
    lab = torch.tensor([17, v - 1], device="cuda")
    r = vx.vocab_xent_fwd(x, w, lab)
    dx, dw, _ = vx.vocab_xent_bwd(r, x, w, lab)
    xd = x.double().requires_grad_(True)
    wd = w.double().requires_grad_(True)
    loss = torch.nn.functional.cross_entropy(xd @ wd.t(), lab)
    loss.backward()
    # sum |x w| stays below 60 here, so a logit is off by at most 10 U32 * 60 = 4e-5, lse by that and 150 U32, and a
    # probability by 1e-4 of itself; both gradients are sums of terms dz x and dz w, bounded by 1e-4 (and the operands'
    # rounding) of the sum of the terms' sizes, not of the sum, in which the rows' terms may cancel
    assert float((xd.detach().abs() @ wd.detach().abs().t()).max()) < 60
    assert abs(float(r.loss) - float(loss.detach())) < 1e-4
    step = half_step(dtype)
    dz = torch.softmax(xd.detach() @ wd.detach().t(), 1) / n
    dz[torch.arange(n), lab] -= 1 / n
    assert_within(dw, wd.grad, (2 * step + 1e-4) * (dz.abs().t() @ xd.detach().abs()))
    assert_within(dx, xd.grad, (2 * step + 1e-4) * (dz.abs() @ wd.detach().abs()))


@pytest.mark.gpu
def test_weight_rows_so_far_apart_that_a_piece_must_be_shorter():
    """40 000 rows 65 536 elements apart are 5 GB from end to end: beyond one launch's 32-bit offsets."""
    x, w, lab, b = (t.cuda() for t in draw(50, 40000, 64, torch.bfloat16))
    far = torch.zeros((40000, 65536), dtype=torch.bfloat16, device="cuda")[:, 256:320]
    far.copy_(w)
    # shorter pieces may run on another kernel, with another order of sums: held to the definition, not to the other's bits
    want = exact(x, w, lab, b)
    r = vx.vocab_xent_fwd(x, far, lab, b)
    assert_within(r.loss_rows, *want["rows"], "loss rows")
    assert int(r.hits) == want["hits"]
    for got, name in zip(vx.vocab_xent_bwd(r, x, far, lab, b), ("dx", "dw", "db")):
        assert_within(got, *want[name], name)
