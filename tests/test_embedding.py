"""Embedding lookup and the table's gradient by sorted tokens (ops/embedding.py) against 64-bit sums."""
import pytest
import torch

from distributed_tensorflow_amd.ops import embedding as em
from token_utils import U32, assert_within, devices, half_step


def tokens(n, v, kind="zipf", seed=0):
    g = torch.Generator().manual_seed(seed + n)
    if kind == "zipf":
        return (torch.exp(torch.rand(n, generator=g, dtype=torch.float64) * torch.log(torch.tensor(v + 1.0, dtype=torch.float64))) - 1).long().clamp_(0, v - 1)
    if kind == "same":
        return torch.full((n,), v // 2)
    if kind == "few":
        return torch.randint(0, v, (3,), generator=g)[torch.randint(0, 3, (n,), generator=g)]
    return torch.randint(0, v, (n,), generator=g)


def sums(dy, ids, v, scale, skip=None):
    """Gradient and bound: a row's sum of m terms takes at most m additions in a row, then scale and the last rounding."""
    flat, d = ids.reshape(-1), dy.double().reshape(-1, dy.shape[-1])
    keep = (flat >= 0) & (flat < v) & (flat != (skip if skip is not None else -1))
    flat, d = flat[keep], d[keep]
    zero = torch.zeros((v, d.shape[1]), dtype=torch.float64)
    want = zero.index_add(0, flat, d) * scale
    size = zero.index_add(0, flat, d.abs()) * abs(scale)
    m = torch.bincount(flat, minlength=v).double()[:, None]
    return want, m * U32 * size + 2 * U32 * want.abs() + half_step(dy.dtype) * want.abs()


def check(n, v, d, dtype, dev, kind="zipf", scale=1.7, skip=None, idtype=torch.int64):
    ids = tokens(n, v, kind).to(idtype)
    g = torch.Generator().manual_seed(d)
    table, dy = torch.randn((v, d), generator=g).to(dtype), torch.randn((n, d), generator=g).to(dtype)
    y = em.embedding_fwd(ids.to(dev), table.to(dev), scale)
    want = table.double()[ids.long()] * scale
    assert y.dtype == dtype
    assert_within(y, want, (half_step(dtype) + 2 * U32) * want.abs(), "y")
    got = em.embedding_bwd(dy.to(dev), ids.to(dev), v, scale, skip)
    assert got.shape == (v, d) and got.dtype == dtype
    assert_within(got, *sums(dy, ids.long(), v, scale, skip), "dtable")


@pytest.mark.parametrize("dev", devices())
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,v,d", [(1, 1, 1), (1, 5, 8), (2, 2, 3), (8, 1000, 64), (63, 31, 100), (64, 32, 40), (65, 33, 7), (500, 511, 264), (700, 512, 16),
                                   (1025, 513, 24), (3000, 50001, 8), (300, 17, 1032), (257, 40, 4100)])
def test_sizes(n, v, d, dtype, dev):
    check(n, v, d, dtype, dev)


@pytest.mark.parametrize("dev", devices())
@pytest.mark.parametrize("kind", ["zipf", "same", "few", "uniform"])
@pytest.mark.parametrize("n", [64, 65, 129, 2000, 8191, 8192, 8193, 16384, 40000])
def test_token_counts_and_hot_rows(n, kind, dev):
    """Both sides of the one-workgroup sort, and rows that take part of a chunk, one, or many."""
    check(n, 300, 24, torch.float32, dev, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("v", [1, 511, 512, 262143, 262144, 300000])
@pytest.mark.parametrize("n", [5000, 20000])
def test_key_widths_of_the_sort(n, v):
    """One, two and three passes, at the borders of 9-bit digits."""
    check(n, v, 8, torch.bfloat16, "cuda:0", "uniform")


@pytest.mark.gpu
def test_very_long_rows_are_split_into_larger_chunks():
    check(70000, 9, 40, torch.float32, "cuda:0", "few")
    check(530000, 7, 8, torch.bfloat16, "cuda:0", "zipf")
    check(1100000, 1000, 8, torch.float32, "cuda:0", "zipf")          # more than 256 blocks of the sort: scanned by a launch of its own


@pytest.mark.parametrize("dev", devices())
@pytest.mark.parametrize("idtype", [torch.int32, torch.int64])
def test_padding_index_and_id_types(idtype, dev):
    check(900, 50, 40, torch.float32, dev, skip=0, idtype=idtype)
    ids = tokens(900, 50)
    dy = torch.randn(900, 40)
    a = em.embedding_bwd(dy.to(dev), ids.to(dev), 50, 1.0, -50)
    assert not a[0].any()
    dy[ids == 0] = float("nan")                      # what padding tokens bring does not matter
    assert torch.equal(em.embedding_bwd(dy.to(dev), ids.to(dev), 50, 1.0, 0), a)


@pytest.mark.parametrize("dev", devices())
@pytest.mark.parametrize("v,d", [(1, 1), (2, 2), (1, 4), (3, 2), (2, 8)])
def test_tables_of_a_few_bytes_under_many_tokens(v, d, dev, monkeypatch):
    """Fewer 16-byte pieces than the sort has launches: rows without tokens are zeros all the same."""
    empty = torch.empty
    # new memory may hold anything: here bytes of ones, NaN in either type
    def poisoned(*args, **kw):
        t = empty(*args, **kw)
        t.view(torch.uint8).fill_(255)
        return t

    monkeypatch.setattr(torch, "empty", poisoned)
    for dtype in (torch.float32, torch.bfloat16):
        got = em.embedding_bwd(torch.ones(10000, d, dtype=dtype, device=dev), torch.zeros(10000, dtype=torch.int64, device=dev), v)
        assert torch.equal(got[1:], torch.zeros_like(got[1:]))
        assert torch.equal(got[0].float(), torch.full((d,), 10000.0, device=dev).to(dtype).float())


@pytest.mark.parametrize("dev", devices())
def test_no_tokens_and_leading_axes(dev):
    table = torch.randn(11, 16, device=dev)
    y = em.embedding_fwd(torch.empty((0, 3), dtype=torch.int64, device=dev), table)
    assert y.shape == (0, 3, 16)
    assert torch.equal(em.embedding_bwd(y, torch.empty((0, 3), dtype=torch.int64, device=dev), 11), torch.zeros(11, 16, device=dev))
    ids = tokens(24, 11).reshape(2, 3, 4).to(dev)
    assert torch.equal(em.embedding_fwd(ids, table), table[ids])
    assert em.embedding_fwd(ids[0, 0, 0], table).shape == (16,)


@pytest.mark.parametrize("dev", devices())
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_alignment(dtype, dev):
    wide, up = torch.randn(40, 70, device=dev).to(dtype), torch.randn(100, 70, device=dev).to(dtype)
    both = torch.stack([tokens(100, 40), tokens(100, 40)], 1).to(dev)
    for sl in (slice(0, 64), slice(3, 67), slice(6, 70)):
        t, dy, ids = wide[:, sl], up[:, sl], both[:, 1]
        assert torch.equal(em.embedding_fwd(ids, t, 2.0), em.embedding_fwd(ids.clone(), t.clone(), 2.0))
        assert torch.equal(em.embedding_bwd(dy, ids, 40), em.embedding_bwd(dy.clone(), ids.clone(), 40))
    assert torch.equal(em.embedding_fwd(both[:, 0], wide.t().contiguous().t()), em.embedding_fwd(both[:, 0], wide))


def test_ids_outside_the_table_raise_on_the_cpu():
    table = torch.randn(10, 8)
    for bad in (10, -1):
        with pytest.raises((IndexError, RuntimeError)):
            em.embedding_fwd(torch.tensor([1, bad]), table)


@pytest.mark.gpu
def test_ids_outside_the_table_are_zero_rows_on_the_gpu():
    table = torch.randn(10, 8, device="cuda")
    ids = torch.tensor([1, 10, -1, 9, 1 << 40, -(1 << 40)], device="cuda")
    y = em.embedding_fwd(ids, table)
    assert torch.equal(y[[0, 3]], table[[1, 9]]) and not y[[1, 2, 4, 5]].any()
    g = em.embedding_bwd(torch.ones(6, 8, device="cuda"), ids, 10)
    assert float(g.sum()) == 16 and (g[[1, 9]] == 1).all()


@pytest.mark.parametrize("dev", devices())
def test_autograd_module_and_differences(dev):
    m = em.ScaledEmbedding(30, 24, scale=3.0, padding_idx=2).to(dev)
    assert set(m.state_dict()) == {"weight"}
    ids = tokens(77, 30).to(dev)
    up = torch.randn(77, 24, device=dev)
    y = m(ids)
    y.backward(up)
    assert torch.equal(y, em.embedding_fwd(ids, m.weight, 3.0))
    assert torch.equal(m.weight.grad, em.embedding_bwd(up, ids, 30, 3.0, 2)) and not m.weight.grad[2].any()
    # linear in the table: a difference along any direction (zero in the padding row) is the slope up to rounding
    d = torch.randn(30, 24, device=dev)
    d[2] = 0
    f = lambda w: (em.embedding_fwd(ids, w, 3.0).double() * up.double()).sum()  # noqa: E731
    slope = (f(m.weight.detach() + d) - f(m.weight.detach() - d)) / 2
    assert abs(float(slope - (m.weight.grad.double() * d.double()).sum())) < 1e-5 * float(m.weight.grad.norm() * d.norm())


@pytest.mark.parametrize("dev", devices())
def test_refusals(dev):
    t, ids, dy = torch.zeros(5, 8, device=dev), torch.zeros(3, dtype=torch.int64, device=dev), torch.zeros(3, 8, device=dev)
    bad = [lambda: em.embedding_fwd(ids.float(), t), lambda: em.embedding_fwd(ids, t.half()), lambda: em.embedding_fwd(ids, t[0]),
           lambda: em.embedding_fwd(ids, t[:0]), lambda: em.embedding_bwd(dy[:2], ids, 5), lambda: em.embedding_bwd(dy, ids, 0),
           lambda: em.embedding_bwd(dy, ids, 5, padding_idx=5), lambda: em.embedding_bwd(dy.half(), ids, 5), lambda: em.embedding_bwd(dy, ids.to(torch.int16), 5),
           lambda: em.ScaledEmbedding(5, 8, max_norm=1.0), lambda: em.ScaledEmbedding(5, 8, dtype=torch.float16)]
    for call in bad:
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("dev", devices())
def test_a_width_of_more_than_32_bits_is_refused(dev):
    ids, far = torch.zeros(1, dtype=torch.int64, device=dev), torch.zeros((1, 1), device=dev).expand(1, 2 ** 32 + 4)
    with pytest.raises(ValueError, match="range"):
        em.embedding_fwd(ids, far)
    with pytest.raises(ValueError, match="range"):
        em.embedding_bwd(far, ids, 3)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [3000, 30000])
def test_same_bits_again_on_another_stream_and_in_replayed_graphs(n):
    ids, dy = tokens(n, 2000).cuda(), torch.randn(n, 64, device="cuda")
    step = lambda: em.embedding_bwd(dy, ids, 2000, 0.5)  # noqa: E731
    first = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = step()
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(first, other)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for k in range(3):
        ids.copy_(tokens(n, 2000, seed=5 + k))
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(want, out) for _, out in graphs)
