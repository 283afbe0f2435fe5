"""Layer normalisation (ops/layernorm.py) against the definition in 64 bits, on the CPU path and on the kernels."""
import pytest
import torch
import torch.nn as nn

from distributed_tensorflow_amd.ops import layernorm as ln
from token_utils import U32, assert_within, devices, half_step

EPS = 1e-5


def exact(x, w, b, residual=None, dy=None, dh=None, eps=EPS):
    """Outputs and error bounds in float64.  The bounds: sums run over at most 64 additions in a row per element (16 in
    a thread, 6 + 4 across lanes and waves; at most C / 1024 < 48 where rows are streamed), so a sum of n terms is off by
    at most 64 U32 times the sum of its absolute terms; the last rounding is half a step of the type."""
    h = x.double() if residual is None else (x.float() + residual.float()).to(x.dtype).double()
    c = h.shape[-1]
    mean = h.mean(-1, keepdim=True)
    var = ((h - mean) ** 2).mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    xhat = (h - mean) * rstd
    ww = torch.ones(c, dtype=torch.float64) if w is None else w.double()
    y = xhat * ww + (0 if b is None else b.double())
    step = half_step(x.dtype)
    # xhat: mean off by 64 U32 mean|h|, the subtraction and product by 2 U32; rstd relative 64 U32 + the mean's part
    e_hat = 130 * U32 * ((h.abs().amax(-1, keepdim=True)) * rstd + xhat.abs() + 1)
    out = {"h": h, "y": (y, e_hat * ww.abs() + 2 * U32 * y.abs() + step * y.abs())}
    if dy is not None:
        d = dy.double()
        g = d * ww
        m1, m2 = g.mean(-1, keepdim=True), (g * xhat).mean(-1, keepdim=True)
        dx = rstd * (g - m1 - xhat * m2)
        gm, xm = g.abs().amax(-1, keepdim=True), xhat.abs().amax(-1, keepdim=True)
        em = e_hat.amax(-1, keepdim=True)
        e_dx = rstd * (gm * (70 * U32 * (1 + xm) ** 2 + em * (2 + 2 * xm))) + 130 * U32 * dx.abs()
        if dh is not None:
            dx = dx + dh.double()
        out["dx"] = (dx, e_dx + (step + U32) * dx.abs())
        d2, x2, e2 = d.reshape(-1, c), xhat.reshape(-1, c), e_hat.expand_as(xhat).reshape(-1, c)
        n = 64 + d2.shape[0] / 64                       # additions in a row for one column
        out["dw"] = ((d2 * x2).sum(0), n * U32 * (d2 * x2).abs().sum(0) + (d2.abs() * e2).sum(0))
        out["db"] = (d2.sum(0), n * U32 * d2.abs().sum(0))
    return out


def draw(shape, dtype, seed=0, mean=0.3, std=1.4):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std + mean).to(dtype)


def check(shape, dtype, dev, wdtype=torch.float32, residual=False, affine=True, seed=1, change=None):
    x, dy = draw(shape, dtype, seed), draw(shape, dtype, seed + 1, 0.0, 1.0)
    r = draw(shape, dtype, seed + 2) if residual else None
    dh = draw(shape, dtype, seed + 3) if residual else None
    w = draw(shape[-1:], wdtype, seed + 4, 1.0, 0.2) if affine else None
    b = draw(shape[-1:], wdtype, seed + 5, 0.0, 0.2) if affine else None
    if change:
        change(x)
    want = exact(x, w, b, r, dy, dh)
    to = lambda t: None if t is None else t.to(dev)  # noqa: E731
    fwd = ln.layer_norm_fwd(to(x), to(w), to(b), EPS, residual=to(r))
    dx, dw, db = ln.layer_norm_bwd(to(dy), fwd, to(w), dh=to(dh))
    assert fwd.y.shape == x.shape and fwd.y.dtype == dtype and dx.shape == x.shape
    if residual:
        assert torch.equal(fwd.h.double().cpu(), want["h"])
    assert_within(fwd.y, *want["y"], "y")
    assert_within(dx, *want["dx"], "dx")
    for name, t in (("dw", dw), ("db", db)):
        ref, bound = want[name]
        assert t.dtype == (wdtype if affine else torch.float32)
        assert_within(t, ref, bound + half_step(t.dtype) * ref.abs(), name)


# widths on both sides of every change of kernel: 16 elements a thread on 64 / 256 / 512 / 1024 threads, then streamed
WIDTHS = [1, 2, 7, 8, 63, 64, 100, 511, 512, 513, 784, 1000, 1001, 1024, 1025, 1032, 4096, 4097, 4104, 8192, 8193, 8200, 16384, 16385]


@pytest.mark.parametrize("dev", devices())
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cols", WIDTHS)
def test_widths(cols, dtype, dev):
    check((5, cols), dtype, dev)


@pytest.mark.parametrize("dev", devices())
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", [(1, 4096), (17, 512), (4099, 40), (8200, 33), (1030, 1032), (300, 8200), (3, 20000), (130, 17000)])
def test_rows_with_residual(rows, cols, dtype, dev):
    check((rows, cols), dtype, dev, residual=True)


@pytest.mark.parametrize("dev", devices())
@pytest.mark.parametrize("wdtype,affine", [(torch.bfloat16, True), (torch.float32, False)])
def test_parameter_types_and_leading_axes(wdtype, affine, dev):
    check((3, 5, 7, 264), torch.bfloat16, dev, wdtype=wdtype, affine=affine)


@pytest.mark.parametrize("dev", devices())
def test_constant_and_offset_rows(dev):
    """A constant row has variance 0 (y = bias); a row far from zero keeps the accuracy of its spread."""
    def change(x):
        x[0] = 3.25
        x[1] += 4096.0
    check((4, 1000), torch.float32, dev, change=change)
    check((4, 20000), torch.float32, dev, change=change)


@pytest.mark.parametrize("dev", devices())
def test_rows_with_nan_and_infinity_stay_alone(dev):
    x = draw((6, 520), torch.float32)
    y0 = ln.layer_norm_fwd(x.to(dev)).y
    x[2, 3], x[4, 519] = float("nan"), float("inf")
    y = ln.layer_norm_fwd(x.to(dev)).y
    assert torch.isnan(y[2]).all() and torch.isnan(y[4]).all()
    for r in (0, 1, 3, 5):
        assert torch.equal(y[r], y0[r])


@pytest.mark.parametrize("dev", devices())
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_and_misaligned_rows(dtype, dev):
    wide = draw((6, 300), dtype).to(dev)
    w, b = torch.ones(256, device=dev), torch.zeros(256, device=dev)
    dy = draw((6, 256), dtype, 9).to(dev)
    for x in (wide[:, :256], wide[:, 3:259], wide[:, 8:264], draw((256, 6), dtype).to(dev).t(), wide[:1, :256].expand(6, 256)):
        a, c = ln.layer_norm_fwd(x, w, b), ln.layer_norm_fwd(x.contiguous(), w, b)
        assert_within(a.y, c.y.double(), 4 * half_step(dtype) * c.y.double().abs() + 64 * U32)   # another kernel: another order of sums
        for g, h in zip(ln.layer_norm_bwd(dy, a, w), ln.layer_norm_bwd(dy, c, w)):
            assert_within(g, h.double(), 4 * half_step(g.dtype) * h.double().abs() + 2e-5)


@pytest.mark.parametrize("dev", devices())
def test_no_rows(dev):
    x = torch.empty((0, 16), device=dev)
    w = torch.ones(16, device=dev)
    r = ln.layer_norm_fwd(x, w, w)
    dx, dw, db = ln.layer_norm_bwd(x, r, w)
    assert r.y.shape == (0, 16) and dx.shape == (0, 16)
    assert torch.equal(dw.cpu(), torch.zeros(16)) and torch.equal(db.cpu(), torch.zeros(16))


@pytest.mark.parametrize("dev", devices())
@pytest.mark.parametrize("residual", [False, True])
def test_autograd_and_module(residual, dev):
    torch.manual_seed(3)
    ref, mod = nn.LayerNorm(72).double(), ln.FusedLayerNorm(72)
    with torch.no_grad():
        ref.weight.uniform_(0.5, 1.5)
        ref.bias.normal_()
    mod.load_state_dict({k: v.float() for k, v in ref.state_dict().items()})
    ref.load_state_dict({k: v.double() for k, v in mod.state_dict().items()})
    mod = mod.to(dev)
    x, r = draw((4, 9, 72), torch.float32, 5), draw((4, 9, 72), torch.float32, 6)
    xs = [t.to(dev, copy=True).requires_grad_(True) for t in (x, r)]
    xd = [t.double().requires_grad_(True) for t in (x, r)]
    up = draw((4, 9, 72), torch.float32, 7)
    if residual:
        y, h = mod(*xs)
        hd = (x + r).double() + (xd[0] - x.double()) + (xd[1] - r.double())      # the sum as stored, differentiable
        loss, want = ((y * up.to(dev)).sum() + (h * 0.5 * up.to(dev)).sum()), (ref(hd) * up).sum() + (hd * 0.5 * up).sum()
    else:
        loss, want = (mod(xs[0]) * up.to(dev)).sum(), (ref(xd[0]) * up).sum()
    loss.backward()
    want.backward()
    pairs = [(xs[0].grad, xd[0].grad), (mod.weight.grad, ref.weight.grad), (mod.bias.grad, ref.bias.grad)]
    if residual:
        pairs.append((xs[1].grad, xd[1].grad))
    for got, exp in pairs:                       # unit-scale data, 36 rows: below 200 roundings of values up to ~30
        assert_within(got, exp, 200 * U32 * (exp.abs() + 30))


@pytest.mark.parametrize("dev", devices())
def test_gradient_against_differences(dev):
    """Central differences of the forward pass along random directions; the forward's float32 noise (1e-6 of values of
    order 1, averaged over 600 elements) over the step 2^-7 and the third-order term stay below 2e-3 of the slope."""
    x, w, b, up = (draw(s, torch.float32, i).to(dev) for i, s in enumerate([(6, 100), (100,), (100,), (6, 100)]))
    fwd = ln.layer_norm_fwd(x, w, b)
    grads = ln.layer_norm_bwd(up, fwd, w)
    f = lambda *a: (ln.layer_norm_fwd(*a).y.double() * up.double()).sum()  # noqa: E731
    args, h = [x, w, b], 2.0 ** -7
    for k, g in enumerate(grads):
        d = draw(args[k].shape, torch.float32, 20 + k, 0.0, 1.0).to(dev)
        plus, minus = list(args), list(args)
        plus[k], minus[k] = args[k] + h * d, args[k] - h * d
        slope = (f(*plus) - f(*minus)) / (2 * h)
        want = (g.double() * d.double()).sum()
        size = (g.double().norm() * d.double().norm())
        assert abs(slope - want) < 2e-3 * size


@pytest.mark.parametrize("dev", devices())
def test_only_the_sum_or_only_some_inputs_need_gradients(dev):
    x = draw((5, 64), torch.float32).to(dev).requires_grad_(True)
    r = draw((5, 64), torch.float32, 1).to(dev)
    _, h = ln.layer_norm(x, residual=r)
    h.sum().backward()
    assert torch.equal(x.grad, torch.ones_like(x))
    w = torch.ones(64, device=dev, requires_grad=True)
    y = ln.layer_norm(r, w)
    y.sum().backward()
    assert r.grad is None and w.grad.shape == (64,)


@pytest.mark.parametrize("dev", devices())
def test_refusals(dev):
    x = torch.zeros((4, 16), device=dev)
    w = torch.ones(16, device=dev)
    bad = [lambda: ln.layer_norm(x.half()), lambda: ln.layer_norm(x, w[:8]), lambda: ln.layer_norm(x, w.half(), w.half()),
           lambda: ln.layer_norm(x, w, w.bfloat16()), lambda: ln.layer_norm(x, w, w, -1.0), lambda: ln.layer_norm(x[:, :0]),
           lambda: ln.layer_norm(x, w, w, residual=x[:2]), lambda: ln.layer_norm(x, w, w, residual=x.bfloat16()),
           lambda: ln.layer_norm(x, torch.ones(32, device=dev)[::2]), lambda: ln.layer_norm_bwd(x[:2], ln.layer_norm_fwd(x, w), w),
           lambda: ln.FusedLayerNorm((4, 16)), lambda: ln.FusedLayerNorm(8)(x)]
    for call in bad:
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("dev", devices())
def test_an_axis_of_more_than_32_bits_is_refused(dev):
    """Not taken modulo 2^32."""
    with pytest.raises(ValueError, match="range"):
        ln.layer_norm(torch.zeros((1, 1), device=dev).expand(1, 2 ** 32 + 4))


@pytest.mark.gpu
def test_same_bits_again_on_another_stream_and_in_a_replayed_graph():
    x, dy = draw((700, 1024), torch.bfloat16).cuda(), draw((700, 1024), torch.bfloat16, 1).cuda()
    w, b = torch.ones(1024, device="cuda"), torch.zeros(1024, device="cuda")

    def step():
        r = ln.layer_norm_fwd(x, w, b, residual=dy)
        return (r.y, r.h) + ln.layer_norm_bwd(dy, r, w)
    first = [t.clone() for t in step()]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = step()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, c) for a, c in zip(first, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        x.copy_(draw((700, 1024), torch.bfloat16, 10 + k))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(step(), out))


@pytest.mark.gpu
def test_more_rows_than_one_launch_index_holds():
    """70 million rows of four: a row takes a wave, and 2^32 threads are more than one grid dimension may have."""
    rows = 70_000_001
    x = torch.randint(-3, 4, (rows, 4), device="cuda", dtype=torch.int8).to(torch.bfloat16)
    r = ln.layer_norm_fwd(x)
    dx, dw, db = ln.layer_norm_bwd(torch.ones_like(x), r)
    for part in (slice(0, 1000), slice(1 << 26, (1 << 26) + 1000), slice(rows - 1000, rows)):
        want = exact(x[part].cpu(), None, None)
        assert_within(r.y[part], *want["y"], "y")
    assert torch.equal(db, torch.full((4,), float(rows), device="cuda"))
    assert dx.abs().max() < 1e-2                     # dy = 1: nothing but the rounding of sums of four is left
