"""kernels.sample against its 64-bit statement.

Weights are rounded to multiples of 2^-42 of the largest one, by 2^-43 at most, after an exponential that is
within 3e-13 of itself, so a cumulated weight of V tokens is within e = V 2^-43 / kept + 3e-13 of the kept weight.  A decision
compares two of them: tokens have to be equal wherever the statement's nearest decision is further than 2 e from
falling otherwise, and no row of these tests is nearer.  A probability is off by 2 e and its rounding to 32 bits."""

import numpy as np
import pytest
import torch

from oracle import sampling as osm
from wanferenz_amd import kernels

pytestmark = pytest.mark.gpu


def check(logits, u, got, t=1.0, k=0, p=1.0, m=0.0):
    x = logits.float().cpu().numpy()
    n, V = x.shape
    f = lambda v: np.broadcast_to(v.cpu().numpy() if isinstance(v, torch.Tensor) else np.float32(v), (n,))  # noqa: E731
    t, k, p, m = f(t), np.broadcast_to(k.cpu().numpy() if isinstance(k, torch.Tensor) else k, (n,)), f(p), f(m)
    tok, prob = got[0].cpu().numpy(), got[1].double().cpu().numpy()
    for r in range(n):
        token, pr, slack, kept = osm.sample(x[r], float(u[r]), float(t[r]), int(k[r]), float(p[r]), float(m[r]))
        e = V * 2.0 ** -43 / max(kept, 1.0) + 3e-13
        # (an exact tie is one of equal weights, whole numbers on both sides)
        assert slack == 0 or slack > 2 * e, ("a decision too near to be tested", r, slack, e)
        assert tok[r] == token, (r, tok[r], token, slack)
        assert abs(prob[r] - pr) <= pr * (2.0 ** -24 + 2 * e) + 2.0 ** -43, (r, prob[r], pr)


def heads(seed, n, V, dtype, gpu):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, V, generator=g) * 2
    for _ in range(3):
        x[torch.arange(n), torch.randint(0, V, (n,), generator=g)] += 8 + 4 * torch.rand(n, generator=g)
    return x.to(dtype).to(gpu), torch.rand(n, generator=g)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [1, 2, 3, 7, 64, 1000, 4097, 32768, 50001])
@pytest.mark.parametrize("t,k,p,m", [(1.0, 0, 1.0, 0.0), (0.7, 50, 0.9, 0.0), (1.3, 0, 0.95, 0.0), (0.9, 0, 1.0, 0.05),
                                     (1.0, 1, 1.0, 0.0), (0.0, 5, 0.5, 0.1), (1.1, 2000, 0.8, 0.01), (0.5, 1024, 1.0, 0.0),
                                     (2.0, 1025, 0.99, 0.0)])
def test_filters(gpu, t, k, p, m, V, dtype):
    x, u = heads(V + k, 24, V, dtype, gpu)
    got = kernels.sample(x, u.to(gpu), temperature=t, top_k=k, top_p=p, min_p=m)
    assert got[0].dtype == torch.int32 and got[1].dtype == torch.float32
    check(x, u, got, t, k, p, m)


def test_uniform_numbers_over_the_whole_range(gpu):
    """One row many times, with u on a fine grid, at 0 and just below 1: the tokens come in order, in proportion."""
    g = torch.Generator().manual_seed(0)
    row = torch.randn(3001, generator=g) * 1.5
    u = torch.cat([torch.linspace(0, 1, 800)[:-1], torch.tensor([0.0, 1 - 2.0 ** -24, 2.0 ** -24])])
    x = row.expand(len(u), -1).contiguous().to(gpu)
    got = kernels.sample(x, u.to(gpu), temperature=0.8)
    check(x, u, got, 0.8)
    z = row[got[0][:799].cpu().long()]
    assert (z[1:] <= z[:-1]).all()
    # numbers that are none of [0, 1): below 0 and NaN as 0, 1 and above as the last below 1
    odd = torch.tensor([-1.0, float("nan"), 1.0, 7.0, float("inf")])
    got = kernels.sample(x[:5], odd.to(gpu), temperature=0.8)
    check(x[:5], torch.tensor([0.0, 0.0] + [1 - 2.0 ** -24] * 3), got, 0.8)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,levels", [(5000, 1), (40000, 1), (40000, 2), (9001, 3), (70001, 40)])
@pytest.mark.parametrize("k,p,m", [(0, 1.0, 0.0), (0, 0.37, 0.0), (4500, 1.0, 0.0), (7, 0.9, 0.0), (6000, 0.61, 0.0),
                                   (0, 0.8, 0.3)])
def test_equal_logits(gpu, k, p, m, V, levels, dtype):
    """Rows of a few values, so that thousands of tokens are equal: they go by index."""
    g = torch.Generator().manual_seed(V + levels)
    x = (torch.randint(0, levels, (6, V), generator=g).float() * 0.25).to(dtype).to(gpu)
    u = torch.tensor([0.0, 0.123, 0.5001, 0.77, 0.9301, 1 - 2.0 ** -24])
    check(x, u, kernels.sample(x, u.to(gpu), top_k=k, top_p=p, min_p=m), 1.0, k, p, m)


@pytest.mark.parametrize("V", [300, 60001])
def test_flat_rows(gpu, V):
    """High temperatures and narrow spreads: most of the tokens lie in a few bins."""
    g = torch.Generator().manual_seed(V)
    x = torch.randn(12, V, generator=g)
    x[4:8] *= 1e-3
    x[8:] *= 1e-6
    u = torch.rand(12, generator=g)
    x = x.to(gpu)
    for t, k, p in ((1.0, 0, 1.0), (50.0, 0, 0.9), (3e38, 0, 1.0), (float("inf"), 100, 0.5), (1.0, 30000, 0.7)):
        check(x, u, kernels.sample(x, u.to(gpu), temperature=t, top_k=k, top_p=p), t, k, p)


def test_values_that_are_not_finite(gpu):
    inf, nan = float("inf"), float("nan")
    rows = torch.tensor([[nan, -inf, nan, -inf, nan], [-inf] * 5, [nan, 1.0, -inf, 2.0, nan], [inf, 5.0, inf, -inf, nan],
                         [3e38, -3e38, 3e38, 0.0, 1.0], [-0.0, 0.0, -0.0, 0.0, -inf], [nan, nan, nan, nan, -3.4e38],
                         [torch.finfo(torch.float32).min, 0.0, 1e-45, -1e-45, 1e-38]])
    u = torch.full((8,), 0.6)
    for args in (dict(), dict(top_k=2), dict(top_p=0.5), dict(min_p=0.9), dict(temperature=0.0), dict(temperature=1e-30),
                 dict(temperature=1e-45, top_p=0.9)):
        got = kernels.sample(rows.to(gpu), u.to(gpu), **args)
        check(rows, u, got, args.get("temperature", 1.0), args.get("top_k", 0), args.get("top_p", 1.0), args.get("min_p", 0.0))
        assert got[0].tolist()[:2] == [-1, -1] and got[1].tolist()[:2] == [0, 0]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_rows_that_are_not_finite(gpu, dtype):
    """Rows that several workgroups share: nothing to choose from, an infinity or many, ties of the largest over all
    parts of a row, a NaN beside each."""
    inf, nan = float("inf"), float("nan")
    g = torch.Generator().manual_seed(2)
    x = torch.randn(9, 40001, generator=g)
    x[0], x[1], x[2] = nan, -inf, nan
    x[2, 33333] = 1.5
    x[3, 17000] = inf
    x[4, ::97] = inf
    x[5, ::101] = 9.0
    x[6, ::2] = nan
    x[7] = -3e38
    x[8] = 0.0
    x[3:6, 5] = nan
    x, u = x.to(dtype), torch.rand(9, generator=g)
    for args in (dict(), dict(top_k=7), dict(top_p=0.5), dict(min_p=0.2), dict(temperature=0.0), dict(top_k=3000, top_p=0.9)):
        got = kernels.sample(x.to(gpu), u.to(gpu), **args)
        check(x, u, got, args.get("temperature", 1.0), args.get("top_k", 0), args.get("top_p", 1.0), args.get("min_p", 0.0))
        assert got[0].tolist()[:4] == [-1, -1, 33333, 17000]
    mixed = torch.tensor([1.0, 0, 1, 0, 0, 0, 0, 0, 1])
    got = kernels.sample(x.to(gpu), u.to(gpu), temperature=mixed.to(gpu))
    check(x, u, got, mixed)
    assert got[0].tolist()[4:6] == [0, 0]


@pytest.mark.parametrize("V", [1000, 40001])
def test_temperatures_and_logits_below_the_normal_range(gpu, V):
    """Differences of logits that are a normal number of temperatures, and far more of them than a weight has, at the
    smallest temperatures."""
    g = torch.Generator().manual_seed(5)
    x = torch.stack([-1e-36 * torch.rand(V, generator=g), -1e-37 * torch.rand(V, generator=g),
                     -1e-43 * torch.rand(V, generator=g), -torch.rand(V, generator=g)])
    x[:, V // 2] = 0
    u = torch.rand(4, generator=g)
    for t in (1e-44, 1e-40, 1e-38, 1e-37, 3e-37, 1e-36, 1e-30):
        for k, p, m in ((0, 1.0, 0.0), (50, 1.0, 0.0), (0, 0.9, 0.0), (2000, 0.9, 0.1)):
            got = kernels.sample(x.to(gpu), u.to(gpu), temperature=t, top_k=k, top_p=p, min_p=m)
            check(x, u, got, t, k, p, m)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_parameters_of_each_row(gpu, dtype):
    n, V = 70, 2003
    x, u = heads(5, n, V, dtype, gpu)
    g = torch.Generator().manual_seed(6)
    t = torch.where(torch.rand(n, generator=g) < 0.2, 0.0, 0.3 + torch.rand(n, generator=g))
    t[3] = -1.0
    k = torch.randint(-2, 60, (n,), generator=g).to(torch.int32)
    p = torch.where(torch.rand(n, generator=g) < 0.3, 1.0, torch.rand(n, generator=g))
    p[:3] = torch.tensor([0.0, 2.0, 1e-30])
    m = torch.where(torch.rand(n, generator=g) < 0.5, 0.0, 0.2 * torch.rand(n, generator=g))
    m[4:6] = torch.tensor([1.0, -1.0])
    got = kernels.sample(x, u.to(gpu), t.to(gpu), k.to(gpu), p.to(gpu), m.to(gpu))
    check(x, u, got, t, k, p, m)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_at_any_stride_and_alignment(gpu, dtype):
    """Slices of a padded vocabulary and of rows that begin off 16 bytes: what lies around a row does not count."""
    for lo, V, width in ((0, 997, 1000), (1, 997, 999), (3, 1500, 1503), (5, 8, 31), (2, 1, 7)):
        x, u = heads(lo, 9, V, dtype, gpu)
        wide = torch.full((9, width), float("inf"), dtype=dtype, device=gpu)
        wide[:, lo:lo + V] = x
        view = wide[:, lo:lo + V]
        for args in (dict(top_p=0.9), dict(top_k=5), dict(temperature=0.0)):
            got = kernels.sample(view, u.to(gpu), **args)
            check(x, u, got, args.get("temperature", 1.0), args.get("top_k", 0), args.get("top_p", 1.0))
    x, u = heads(9, 4, 640, dtype, gpu)
    got = kernels.sample(x.t().contiguous().t(), u.to(gpu), top_p=0.9)
    check(x, u, got, p=0.9)


@pytest.mark.parametrize("n", [1, 2, 5, 300])
def test_same_result_in_every_call_and_batch(gpu, n):
    """A row's token depends on the row alone, and is the same in every call."""
    V = 33333  # shared by several workgroups up to 128 rows
    x, u = heads(3, n, V, torch.float32, gpu)
    u = u.to(gpu)
    first = [kernels.sample(x, u, top_p=p, top_k=k) for p, k in ((0.9, 0), (1.0, 0), (0.9, 40))]
    for _ in range(3):
        for a, (p, k) in zip(first, ((0.9, 0), (1.0, 0), (0.9, 40))):
            b = kernels.sample(x, u, top_p=p, top_k=k)
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
            i = n // 2
            one = kernels.sample(x[i:i + 1], u[i:i + 1], top_p=p, top_k=k)
            assert one[0][0] == a[0][i] and one[1][0] == a[1][i]


@pytest.mark.parametrize("n,V", [(3, 40000), (600, 6000)])
def test_lists_of_every_length(gpu, n, V):
    """top-k from 1 to the most that is gathered by its count, where lists are sorted in one way or another."""
    x, u = heads(11, n, V, torch.float32, gpu)
    rows = min(n, 8)
    for k in (1, 2, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 512, 513, 1000, 1024):
        got = kernels.sample(x, u.to(gpu), temperature=3.0, top_k=k)
        check(x[:rows], u[:rows], [y[:rows] for y in got], 3.0, k)


def test_long_rows(gpu):
    """A row of 2^21 logits, and its top half alone."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(2, 2 ** 21, generator=g).to(gpu)
    u = torch.tensor([0.3, 0.9])
    for args in (dict(p=1.0), dict(p=0.5), dict(k=100), dict(k=5000, p=0.9)):
        got = kernels.sample(x, u.to(gpu), top_p=args.get("p", 1.0), top_k=args.get("k", 0))
        check(x, u, got, 1.0, args.get("k", 0), args.get("p", 1.0))


def test_refusals_and_outputs(gpu):
    x, u = torch.zeros(3, 10, device=gpu), torch.zeros(3, device=gpu)
    for bad, match in ((dict(temperature=-1.0), "temperature"), (dict(top_k=-1), "top_k"), (dict(top_p=1.5), "top_p"),
                       (dict(min_p=-0.1), "min_p"), (dict(top_p=float("nan")), "top_p"), (dict(top_k=u), "top_k must be"),
                       (dict(temperature=u[:2]), "temperature must be"), (dict(min_p=u.cpu()), "min_p must be"),
                       (dict(out=(u, u)), "out")):
        with pytest.raises(ValueError, match=match):
            kernels.sample(x, u, **bad)
    with pytest.raises(TypeError, match="float32 or bf16"):
        kernels.sample(x.half(), u)
    with pytest.raises(ValueError, match="uniform must be"):
        kernels.sample(x, u[:2])
    with pytest.raises(ValueError, match="logits must be"):
        kernels.sample(x[0], u)
    with pytest.raises(ValueError, match="logits must be"):
        kernels.sample(x[:, :0], u)
    out = torch.empty(3, dtype=torch.int32, device=gpu), torch.empty(3, device=gpu)
    assert kernels.sample(x, u, out=out) is out and out[0].tolist() == [0, 0, 0]
    assert kernels.sample(x[:0], u[:0])[0].shape == (0,)
