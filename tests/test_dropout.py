"""Dropout from the counter-based generator (ops/dropout.py): the mask against an independent statement of the generator
with Python integers, values, statistics, the step counter, captured graphs."""
import pytest
import torch

from distributed_tensorflow_amd.ops import dropout as dp
from distributed_tensorflow_amd.ops import reference
from token_utils import U32, assert_within, devices, half_step


def philox(counter, key):
    """Philox4x32-10 on Python integers (Salmon et al. 2011)."""
    c, (k0, k1) = list(counter), key
    for _ in range(10):
        p0, p1 = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(p1 >> 32) ^ c[1] ^ k0, p1 & 0xFFFFFFFF, (p0 >> 32) ^ c[3] ^ k1, p0 & 0xFFFFFFFF]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return c


def keeps(n, rate, seed, step):
    out = []
    for q in range(-(-n // 8)):
        w = philox((q & 0xFFFFFFFF, q >> 32, step & 0xFFFFFFFF, step >> 32), (seed & 0xFFFFFFFF, seed >> 32))
        out += [(x >> s) & 0xFFFF for x in w for s in (0, 16)]
    return torch.tensor(out[:n]) >= round(rate * 65536)


def test_generator_known_answers():
    """The published test vectors of Philox4x32-10: all-zero and all-one counter and key."""
    assert philox((0, 0, 0, 0), (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = 0xFFFFFFFF
    assert philox((ones,) * 4, (ones, ones)) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert reference.philox_words(1, 0, 0)[0].tolist() == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]


@pytest.mark.parametrize("dev", devices())
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 7, 8, 9, 2047, 2048, 2049, 5000])
@pytest.mark.parametrize("rate", [0.0, 0.1, 0.5, 0.97])
def test_values(n, rate, dtype, dev):
    seed, step = 0xFEDCBA9876543210, (5 << 32) + 77
    x = torch.randn(n, generator=torch.Generator().manual_seed(n)).to(dtype)
    r = torch.randn(n, generator=torch.Generator().manual_seed(n + 1)).to(dtype)
    keep = keeps(n, rate, seed, step)
    want = torch.where(keep, x.double() * (65536 / (65536 - round(rate * 65536))), 0.0)
    got = dp.dropout_apply(x.to(dev), rate, seed, step)
    assert_within(got, want, (half_step(dtype) + 3 * U32) * want.abs())
    assert torch.equal((got == 0).cpu(), ~keep | (x == 0))
    both = dp.dropout_apply(x.to(dev), rate, seed, step, residual=r.to(dev))
    total = want + r.double()
    assert_within(both, total, half_step(dtype) * total.abs() + 3 * U32 * (want.abs() + total.abs()))


@pytest.mark.parametrize("dev", devices())
def test_views_and_masked_values(dev):
    """Any view gives what its contiguous copy gives; what is dropped is zero, whatever it was."""
    wide = torch.randn(65, 130, device=dev)
    for v in (wide[:, 1:], wide.t(), wide[3:7, ::2], wide.flatten()[1:1000], wide[0, 0]):
        assert torch.equal(dp.dropout_apply(v, 0.3, 11, 2), dp.dropout_apply(v.clone(memory_format=torch.contiguous_format), 0.3, 11, 2))
    x = torch.full((4096,), float("inf"), device=dev)
    x[::2] = float("nan")
    y = dp.dropout_apply(x, 0.5, 1)
    keep = keeps(4096, 0.5, 1, 0)
    assert torch.equal((y == 0).cpu(), ~keep) and torch.equal(torch.isnan(y).cpu(), keep & torch.isnan(x).cpu())


@pytest.mark.parametrize("dev", devices())
def test_rates_zero_and_one_and_no_elements(dev):
    x = torch.randn(1000, device=dev)
    assert torch.equal(dp.dropout_apply(x, 0.0, 5), x)
    assert torch.equal(dp.dropout_apply(x, 1.0, 5), torch.zeros_like(x))
    assert torch.equal(dp.dropout_apply(x, 1.0, 5, residual=x), x)
    assert dp.dropout_apply(x[:0], 0.5, 5).shape == (0,)
    assert dp.dropout(x, 0.5, 5, training=False) is x


@pytest.mark.parametrize("dev", devices())
def test_masks_of_other_seeds_and_steps_are_unrelated(dev):
    """Kept counts and agreements of 2^18 independent draws: within six standard deviations of their means."""
    n, rate = 1 << 18, 0.25
    x = torch.ones(n, device=dev)
    a = [dp.dropout_apply(x, rate, s, t) != 0 for s, t in ((1, 0), (2, 0), (1, 1), (1 + (1 << 32), 0), (1, 1 << 32))]
    for m in a:
        assert abs(float(m.double().sum()) - 0.75 * n) < 6 * (n * 0.75 * 0.25) ** 0.5
    p = 0.75 ** 2 + 0.25 ** 2
    for m in a[1:]:
        assert abs(float((m == a[0]).double().sum()) - p * n) < 6 * (n * p * (1 - p)) ** 0.5


@pytest.mark.parametrize("dev", devices())
def test_gradient_uses_the_forward_mask_even_if_the_counter_moved(dev):
    x = torch.randn(33, 65, device=dev, requires_grad=True)
    r = torch.randn(33, 65, device=dev, requires_grad=True)
    step = torch.tensor([41], device=dev)
    y = dp.dropout(x, 0.4, 9, step, residual=r)
    step.add_(1)
    up = torch.randn(33, 65, device=dev)
    y.backward(up)
    assert torch.equal(x.grad, dp.dropout_apply(up, 0.4, 9, 41)) and torch.equal(r.grad, up)
    # the map is linear: differences give its slope exactly up to rounding
    d = torch.randn(33, 65, device=dev)
    f = lambda t: (dp.dropout_apply(t, 0.4, 9, 41).double() * up.double()).sum()  # noqa: E731
    slope = (f(x.detach() + d) - f(x.detach() - d)) / 2
    assert abs(float(slope - (x.grad.double() * d.double()).sum())) < 1e-5 * float(x.grad.norm() * d.norm())


@pytest.mark.parametrize("dev", devices())
def test_module_advances_its_counter(dev):
    m = dp.FusedDropout(0.5, 123).to(dev)
    x = torch.ones(5000, device=dev)
    a, b = m(x), m(x)
    assert torch.equal(a, dp.dropout_apply(x, 0.5, 123, 0)) and torch.equal(b, dp.dropout_apply(x, 0.5, 123, 1))
    assert int(m.step) == 2
    m.eval()
    assert torch.equal(m(x), x) and torch.equal(m(x, x), 2 * x) and int(m.step) == 2


@pytest.mark.parametrize("dev", devices())
def test_refusals(dev):
    x = torch.ones(8, device=dev)
    t = torch.zeros(1, dtype=torch.int64, device=dev)
    bad = [lambda: dp.dropout_apply(x.half(), 0.5, 1), lambda: dp.dropout_apply(x, -0.1, 1), lambda: dp.dropout_apply(x, 1.5, 1),
           lambda: dp.dropout_apply(x, float("nan"), 1), lambda: dp.dropout_apply(x, 0.5, -1), lambda: dp.dropout_apply(x, 0.5, 1 << 64),
           lambda: dp.dropout_apply(x, 0.5, 1, -1), lambda: dp.dropout_apply(x, 0.5, 1, t.int()),
           lambda: dp.dropout_apply(x, 0.5, 1, torch.zeros(2, dtype=torch.int64, device=dev)),
           lambda: dp.dropout_apply(x, 0.5, 1, residual=x[:4]), lambda: dp.dropout_apply(x, 0.5, 1, residual=x.bfloat16()),
           lambda: dp.dropout_apply(x, 0.5, 1, t, used=t), lambda: dp.FusedDropout(2.0, 1)]
    for call in bad:
        with pytest.raises(ValueError):
            call()


@pytest.mark.gpu
def test_captured_training_step_draws_a_new_mask_in_every_replay():
    m = dp.FusedDropout(0.3, 77).cuda()
    x = torch.randn(300, 257, device="cuda")
    up = torch.randn(300, 257, device="cuda")

    def step():
        leaf = x.detach().requires_grad_(True)
        y = m(leaf)
        return y, torch.autograd.grad(y, leaf, up)[0]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, dx = step()
    m.step.zero_()
    for k in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, dp.dropout_apply(x, 0.3, 77, k)) and torch.equal(dx, dp.dropout_apply(up, 0.3, 77, k))
    assert int(m.step) == 4


@pytest.mark.gpu
def test_device_mask_equals_host_mask_and_spans_many_blocks():
    n = (1 << 22) + 5
    x = torch.ones(n)
    assert torch.equal(dp.dropout_apply(x.cuda(), 0.1, 3, 9).cpu(), dp.dropout_apply(x, 0.1, 3, 9))
