"""GPU tests of sample_filtered_batched against a plain form (step_refs.sample).

Tokens are whole numbers and equal. Both sides' weights are whole numbers of
float64 exponentials, which differ by a unit of 2^-40 in a few of a hundred at
most; a token would differ only where a threshold falls within such units of
a token's border, one row in 10^8 or fewer at these sizes."""

import numpy as np
import pytest
import torch

import fusedtok_amd as ft
from tests import step_refs as refs

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
# both sides of each form's sizes: registers of 4, 8, 16, 32 tokens, slices
SIZES = [1, 2, 5, 64, 1000, 4096, 4097, 8192, 8193, 16384, 20001, 32768, 32769, 40963, 70000]


def dev(x, dtype=None):
    return torch.as_tensor(np.ascontiguousarray(x)).to(DEV, dtype=dtype)


def check(x, u, temp=1.0, k=0, p=1.0, minp=0.0):
    """x: a GPU tensor [rows, n]; the parameters numbers or arrays."""
    rows = x.shape[0]

    def given(v, dtype):
        return dev(np.asarray(v), dtype) if np.ndim(v) else v

    got = ft.sample_filtered_batched(
        x, dev(u, torch.float32), temperature=given(temp, torch.float32),
        top_k=given(k, torch.int32), top_p=given(p, torch.float32),
        min_p=given(minp, torch.float32))
    assert got.dtype == torch.int64 and got.shape == (rows,) and got.is_cuda
    f32 = lambda v: np.broadcast_to(np.asarray(v, np.float32), rows)
    xs = x.float().cpu().numpy()
    want = [refs.sample(xs[r], np.float32(u[r]), f32(temp)[r],
                        int(np.broadcast_to(k, rows)[r]), f32(p)[r], f32(minp)[r])
            for r in range(rows)]
    assert got.tolist() == want
    return got


def logits(seed, rows, n, dtype, width=2.0):
    rng = np.random.default_rng(seed)
    return dev(rng.standard_normal((rows, n)) * width, dtype), rng.random(rows).astype(np.float32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", SIZES)
def test_sizes(n, dtype):
    x, u = logits(n, 4, n, dtype)
    check(x, u)
    check(x, u, 0.7, 40, 0.9, 0.01)
    check(x, u, 0.0)
    check(x, u, 1.3, 0, 0.95)


@pytest.mark.parametrize("n", [900, 20000, 50257])
@pytest.mark.parametrize("k", [0, 1, 2, 50, 1000, 2 ** 31 - 1])
@pytest.mark.parametrize("p", [1.0, 0.999, 0.9, 0.3, 1e-6])
@pytest.mark.parametrize("minp", [0.0, 0.05, 1.0])
def test_filters(minp, p, k, n):
    x, u = logits(7, 6, n, torch.float32)
    check(x, u, 1.0, k, p, minp)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [3000, 33000])
def test_each_row_its_own(n, dtype):
    rows = 40
    x, u = logits(n, rows, n, dtype)
    r = np.random.default_rng(1)
    check(x, u, r.choice([0.0, 0.3, 1.0, 2.5], rows), r.choice([0, 1, 7, 300], rows),
          r.choice([0.1, 0.8, 0.99, 1.0], rows), r.choice([0.0, 0.0, 0.1, 1.0], rows))


@pytest.mark.parametrize("n", [5000, 20000, 50000])
@pytest.mark.parametrize("steps", [1, 2, 5, 40])
def test_equal_logits(steps, n):
    """A few values only, thousands of tokens each: ties go by index."""
    rng = np.random.default_rng(steps)
    x = dev(rng.integers(0, steps, (9, n)) * 0.25, torch.bfloat16)
    u = rng.random(9)
    for k in (0, 1, 100, n // 2, n - 1):
        for p in (1.0, 0.7, 0.01):
            check(x, u, 1.0, k, p)
            check(x, u, 0.2, k, p, 0.3)


def test_signed_zeros_are_equal():
    x = torch.zeros(64, 500, device=DEV)
    x[:, ::2] = -0.0
    check(x, np.arange(64) / 64, 1.0, 10, 0.9)
    assert (ft.sample_filtered_batched(x, torch.zeros(64, device=DEV), temperature=0.0) == 0).all()


@pytest.mark.parametrize("n", [700, 40000])
def test_infinities_and_nan(n):
    x, u = logits(3, 8, n, torch.float32)
    x[0] = -float("inf")                       # nothing at all
    x[1] = float("nan")
    x[2, :] = -float("inf")
    x[2, n - 3] = -80.0                        # one token
    x[3, ::2] = float("nan")
    x[4, 1::3] = -float("inf")                 # a mask
    x[5, 10] = x[5, n - 1] = float("inf")      # infinite ones share the mass
    x[6, :] = torch.finfo(torch.float32).min   # the type's lowest value everywhere
    x[7, 5:] = torch.finfo(torch.float32).min
    for k, p, m in ((0, 1.0, 0.0), (3, 1.0, 0.0), (0, 0.8, 0.0), (5, 0.6, 0.1)):
        got = check(x, u, 0.9, k, p, m)
        assert got[:2].tolist() == [-1, -1] and got[2] == n - 3
    check(x, u, 0.0)


@pytest.mark.parametrize("n", [2000, 36000])
def test_ends_of_the_random_numbers(n):
    x, _ = logits(5, 5, n, torch.float32)
    u = np.array([0.0, np.nextafter(np.float32(1), np.float32(0)), 2.0 ** -149, 0.5, 0.25])
    for k, p in ((0, 1.0), (7, 1.0), (0, 0.5), (1, 0.5)):
        check(x, u, 1.0, k, p)
    # outside [0, 1): the first or the last kept token
    last = ft.sample_filtered_batched(x, dev(np.full(5, u[1]), torch.float32), top_k=4)
    for bad in (1.0, 7.0, float("inf")):
        assert torch.equal(ft.sample_filtered_batched(x, torch.full((5,), bad, device=DEV),
                                                      top_k=4), last)
    first = ft.sample_filtered_batched(x, torch.zeros(5, device=DEV), top_k=4)
    for bad in (-1.0, float("nan"), -float("inf")):
        assert torch.equal(ft.sample_filtered_batched(x, torch.full((5,), bad, device=DEV),
                                                      top_k=4), first)


@pytest.mark.parametrize("n", [2000, 36000])
@pytest.mark.parametrize("temp", [1e-30, 1e-4, 0.01, 30.0, 1e30])
def test_temperatures(temp, n):
    x, u = logits(6, 6, n, torch.float32)
    check(x, u, temp, 0, 0.9)
    check(x, u, temp, 20)


@pytest.mark.parametrize("n", [900, 20000, 50257, 140000])
@pytest.mark.parametrize("k", [1, 30, 112, 113, 256, 257, 700])
def test_where_the_first_k_lie(k, n):
    """k on both sides of the parts whose largest logits bound the first k;
    the largest logits all in one part, a part each, equal, or too few."""
    rng = np.random.default_rng(k)
    x = rng.standard_normal((8, n)).astype(np.float32)
    x[1] = np.sort(x[1])[::-1]                   # the first k side by side
    x[2] = np.sort(x[2])
    x[3] = np.round(4 * x[3])                    # many equal at any bound
    x[4] = -3.0
    x[5, k // 2 + 1:] = -np.inf                  # fewer than k have weight
    x[6, rng.permutation(n)[:k + 5]] = np.inf    # more than k share it all
    x[7] = -np.finfo(np.float32).max
    x[7, n // 2] = 1.0
    u = rng.random(8).astype(np.float32)
    check(dev(x), u, 0.9, k)
    check(dev(x), u, 1.1, k, 0.8, 0.02)


@pytest.mark.parametrize("n", [2000, 36000])
@pytest.mark.parametrize("temp", [1e-44, 1e-30, 1e-9, 1e-5])
def test_cold_neighbours(temp, n):
    """Logits a rounding apart and far, under temperatures that make either
    far: no distance runs over into the bins."""
    rng = np.random.default_rng(n)
    x = rng.standard_normal((4, n)).astype(np.float32) * 1e-3 + 20.0
    x[1] = np.nextafter(np.float32(7.0), np.float32(np.inf)) - np.float32(2 ** -22) * (
        np.arange(n) % 9)
    x[2] *= np.float32(1e36)
    x[3, ::2] = -np.finfo(np.float32).max
    u = rng.random(4).astype(np.float32)
    for k, p in ((0, 0.9), (3, 1.0), (50, 0.7), (0, 1.0)):
        check(dev(x), u, temp, k, p)


@pytest.mark.parametrize("n", [2000, 36000])
def test_values_of_vectors_are_safe(n):
    x, u = logits(8, 8, n, torch.float32)
    nan, inf = float("nan"), float("inf")
    got = ft.sample_filtered_batched(
        x, dev(u, torch.float32), temperature=dev([nan, -1, 1, 1, 1, 1, 1, 1.0], torch.float32),
        top_k=dev([0, 0, -5, 2 ** 31 - 1, 3, 3, 0, 0], torch.int32),
        top_p=dev([1, 1, nan, inf, 1, 1, 0, -2.0], torch.float32),
        min_p=dev([0, 0, 0, -1, 5, 0, 0, 0.0], torch.float32))
    best = x.argmax(1).tolist()
    want = [best[0], best[1]] + [refs.sample(x[r].cpu().numpy(), u[r], 1.0, k, 1.0, 0.0)
                                 for r, k in ((2, 0), (3, 0))]
    want += [best[4], refs.sample(x[5].cpu().numpy(), u[5], 1.0, 3, 1.0, 0.0), best[6], best[7]]
    assert got.tolist() == want


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad,n", [(1, 4095), (3, 33001), (64, 32768), (47, 50257)])
def test_rows_inside_wider_ones(pad, n, dtype):
    wide, u = logits(2, 7, n + pad, dtype)
    wide[:, n:] = 1e4   # never seen
    check(wide[:, :n], u, 1.1, 60, 0.9)
    check(wide[1:, :n], u[1:])


def test_a_row_depends_on_itself_alone():
    x, u = logits(4, 20, 40000, torch.bfloat16)
    all_of_them = ft.sample_filtered_batched(x, dev(u, torch.float32), top_k=99, top_p=0.9)
    for r in (0, 13):
        one = ft.sample_filtered_batched(x[r:r + 1], dev(u[r:r + 1], torch.float32), top_k=99,
                                         top_p=0.9)
        assert one[0] == all_of_them[r]


def test_a_large_vocabulary_and_many_rows():
    x, u = logits(11, 2, 1 << 20, torch.float32, 1.0)
    check(x, u, 1.0, 0, 0.97)
    x, u = logits(12, 700, 1100, torch.float16)
    check(x, u, 0.8, 30, 0.9)


def test_draws_follow_the_weights():
    """Evenly spaced random numbers: each token as often as its share, to one
    (a share's ends may each fall between two of them)."""
    x = torch.tensor([[0.0, 1.0, -1.0, 2.0, 0.5]], device=DEV)
    m = 20000
    got = ft.sample_filtered_batched(x.expand(m, 5).contiguous(),
                                     (torch.arange(m, device=DEV) + 0.5) / m)
    want = torch.softmax(x[0].double(), 0) * m
    assert (torch.bincount(got, minlength=5) - want).abs().max() <= 1.01


def test_streams_and_graphs_at_once():
    x = [logits(s, 16, 50000, torch.float32) for s in (1, 2)]
    args = [(a, dev(u, torch.float32)) for a, u in x]
    kw = dict(temperature=0.8, top_k=50, top_p=0.9, min_p=0.01)
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in args]
    ft.sample_filtered_batched(*args[0], **kw)
    torch.cuda.synchronize()
    for a in args:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ft.sample_filtered_batched(*a, **kw))
        graphs.append(graph)
    for turn in range(4):
        for a in args:   # new logits in the same place
            a[0].mul_(0.9)
        want = [ft.sample_filtered_batched(*a, **kw) for a in args]
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        eager = ft.sample_filtered_batched(*args[turn % 2], **kw)
        torch.cuda.synchronize()
        assert torch.equal(eager, want[turn % 2])
        assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_refusals():
    x, u = logits(0, 3, 100, torch.float32)
    u, f = dev(u, torch.float32), ft.sample_filtered_batched
    for bad, exc, word in [
            (lambda: f(x.cpu(), u), TypeError, "GPU"),
            (lambda: f(x.double(), u), TypeError, "float32"),
            (lambda: f(x[0], u), ValueError, "2-D"),
            (lambda: f(x.t(), u), ValueError, "contiguous"),
            (lambda: f(x[:, :0], u), ValueError, "empty"),
            (lambda: f(x, u.cpu()), TypeError, "uniforms"),
            (lambda: f(x, [0.1, 0.2, 0.3]), TypeError, "uniforms"),
            (lambda: f(x, u.double()), TypeError, "uniforms"),
            (lambda: f(x, u[:2]), ValueError, "uniforms"),
            (lambda: f(x, u, temperature=-0.1), ValueError, "temperature"),
            (lambda: f(x, u, temperature=float("nan")), ValueError, "temperature"),
            (lambda: f(x, u, temperature=u.half()), TypeError, "temperature"),
            (lambda: f(x, u, top_k=-1), ValueError, "top_k"),
            (lambda: f(x, u, top_k=1.5), TypeError, "top_k"),
            (lambda: f(x, u, top_k=u), TypeError, "top_k"),
            (lambda: f(x, u, top_p=0.0), ValueError, "top_p"),
            (lambda: f(x, u, top_p=1.01), ValueError, "top_p"),
            (lambda: f(x, u, min_p=-0.5), ValueError, "min_p"),
            (lambda: f(x, u, min_p=1.5), ValueError, "min_p"),
            (lambda: f(x, u, min_p=u[:1]), ValueError, "min_p")]:
        with pytest.raises(exc, match=word):
            bad()
    assert f(x[:0], u[:0]).shape == (0,)
