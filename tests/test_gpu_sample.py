"""rtd_sample on the GPU against an integer statement of its rule in numpy: the ids are
equal, for every filter, type, size and for rows at the rule's edges."""
import numpy as np
import pytest
import torch

from runtimed_b200 import _lib, sampling
from runtimed_b200.errors import ConfigError, ShapeError
from runtimed_b200.weights import Context

pytestmark = pytest.mark.gpu

UNIT = float(1 << 44)


def pick(x, u, t=1.0, k=0, p=1.0, m=0.0):
    """The rule of include/rtd.h for one row (x f32 [V]): Python integers, f64 weights."""
    x = x.astype(np.float64)
    ok = ~np.isnan(x)
    if not ok.any():
        return 0
    top = x[ok].max()
    arg = int(np.nonzero(x == top)[0][0])
    if not np.isfinite(top) or not t > 0 or k == 1:
        return arg
    with np.errstate(all="ignore"):
        e = np.exp((x - top) / t)
    e[~ok | (x == -np.inf)] = 0
    w = np.rint(e * UNIT).astype(np.int64)
    order = np.lexsort((np.arange(len(x)), -np.where(ok, x, -np.inf), ~ok))
    order = order[:ok.sum()]
    if 0 < k:
        order = order[:k]
    if p < 1:
        c = np.cumsum(w[order])
        enough = max(1, int(np.floor(np.float64(p) * np.float64(c[-1]))))
        order = order[:1 + int(np.searchsorted(c, enough, "left"))]
    keep = np.zeros(len(x), bool)
    keep[order] = True
    if m > 0:
        keep &= w.astype(np.float64) >= np.float64(min(np.float32(m), 1.0)) * UNIT
    c = np.cumsum(np.where(keep, w, 0))
    at = min(int(np.floor(np.float64(max(u, 0.0)) * np.float64(c[-1]))), int(c[-1]) - 1)
    return int(np.searchsorted(c, at, "right"))


def check(x, u, t=None, k=None, p=None, m=None):
    """x a torch tensor [T, V] on the CPU; filters numpy arrays or None."""
    T = x.shape[0]
    on = lambda a, dt: None if a is None else torch.from_numpy(np.asarray(a, dt)).cuda()  # noqa: E731
    got = sampling.sample(x.cuda(), on(u, np.float32), on(t, np.float32), on(k, np.int32), on(p, np.float32), on(m, np.float32))
    at = lambda a, r, d, dt: d if a is None else dt(np.asarray(a)[r])  # noqa: E731
    f = x.float().numpy()
    want = [pick(f[r], np.float32(u[r]), np.float64(at(t, r, 1.0, np.float32)), at(k, r, 0, int), np.float64(at(p, r, 1.0, np.float32)),
                 at(m, r, 0.0, np.float32)) for r in range(T)]
    assert got.cpu().tolist() == want


def logits(T, V, seed, std=2.0):
    g = torch.Generator().manual_seed(seed)
    x = std * torch.randn((T, V), generator=g)
    at = torch.randint(0, V, (T, min(V, 20)), generator=g)
    return x.scatter_add(1, at, 6 + 3 * torch.randn(at.shape, generator=g))


@pytest.mark.parametrize("V", [1, 2, 31, 33, 1000, 8192, 8193, 40001, 151936, 1 << 19])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
def test_filters(V, dt):
    T = 6
    rng = np.random.default_rng(V)
    x = logits(T, V, V).to(dt)
    for k, p, m in [(None, None, None), (50, None, None), (None, 0.9, None), (None, None, 0.02), (40, 0.95, 0.01), (1, 0.5, None),
                    (2000, 0.999, None)]:
        f = lambda v: None if v is None else np.full(T, v)  # noqa: E731
        check(x, rng.random(T, dtype=np.float32), rng.uniform(0.3, 2.0, T), f(k), f(p), f(m))


def test_each_row_has_its_own_filters():
    T, V = 40, 5000
    rng = np.random.default_rng(0)
    check(logits(T, V, 1), rng.random(T, dtype=np.float32), rng.choice([0.0, 0.2, 1.0, 5.0, np.inf, np.nan, -1.0], T),
          rng.choice([-3, 0, 1, 2, 17, 1023, 1024, 4999, 5000, 9999], T), rng.choice([-1.0, 0.0, 1e-6, 0.3, 0.999, 1.0, 2.0], T),
          rng.choice([-1.0, 0.0, 0.001, 0.5, 1.0, 7.0], T))


@pytest.mark.parametrize("V", [100, 9000, 100000])
def test_ties(V):
    # few distinct values: thresholds fall inside runs of equal logits, lowest index first
    T = 12
    rng = np.random.default_rng(V)
    x = torch.from_numpy(rng.integers(0, 4, (T, V)).astype(np.float32))
    x[1] = 0.0        # one value alone
    x[2] = -0.0
    x[3, ::2] = 0.0   # both zeros are one value
    x[3, 1::2] = -0.0
    for k, p in [(V // 3, None), (None, 0.4), (V // 2, 0.7), (V - 1, 0.2), (3, 0.9)]:
        f = lambda v: None if v is None else np.full(T, v)  # noqa: E731
        check(x, rng.random(T, dtype=np.float32), np.full(T, 0.8), f(k), f(p))


def test_flat_rows_keep_large_nuclei():
    # nearly uniform rows: thousands of entries share a histogram bin
    T, V = 4, 150000
    rng = np.random.default_rng(5)
    x = torch.from_numpy((rng.random((T, V)) * 1e-3).astype(np.float32))
    x[1] += 1e6  # the differences are a few ulp: thousands of equal values
    x[2] *= 1e-30
    for k, p in [(70000, None), (None, 0.5), (100000, 0.9)]:
        f = lambda v: None if v is None else np.full(T, v)  # noqa: E731
        check(x, rng.random(T, dtype=np.float32), np.ones(T), f(k), f(p))


def test_edges_of_u():
    T, V = 5, 3000
    x = logits(T, V, 9)
    u = np.array([0.0, 1 - 2.0 ** -24, 1.0, -0.5, np.nan], np.float32)
    got = sampling.sample(x.cuda(), torch.from_numpy(u).cuda()).cpu().tolist()
    f = x.numpy()
    assert got == [pick(f[r], v) for r, v in enumerate([0.0, np.float32(1 - 2.0 ** -24), 1.0, 0.0, 0.0])]


def test_infinite_and_nan_logits():
    V = 20000
    x = logits(8, V, 3)
    x[0] = float("nan")
    x[1] = -float("inf")
    x[2] = -float("inf")
    x[2, 777] = -3.0
    x[3, 500] = x[3, 9000] = float("inf")
    x[4, ::3] = float("nan")
    x[5, 5:] = -float("inf")
    x[6] = float("nan")
    x[6, 11] = -float("inf")
    x[7, 10:] = float("nan")
    rng = np.random.default_rng(3)
    for k, p in [(None, None), (50, 0.9), (None, 0.6)]:
        f = lambda v: None if v is None else np.full(8, v)  # noqa: E731
        check(x, rng.random(8, dtype=np.float32), None, f(k), f(p))


def test_equal_seeds_draw_the_distribution():
    # inverse sampling at evenly spaced numbers: each id comes as often as its share, +- 1
    V, n = 50, 4000
    x = logits(1, V, 8, std=1.0)
    u = (np.arange(n) + 0.5) / n
    got = sampling.sample(x.expand(n, V).contiguous().cuda(), torch.from_numpy(u.astype(np.float32)).cuda()).cpu().numpy()
    p = np.exp(x[0].double().numpy())
    p /= p.sum()
    assert np.all(np.abs(np.bincount(got, minlength=V) - n * p) <= 1.01)


def test_strided_rows_out_and_a_captured_graph():
    T, V = 3, 12345
    rng = np.random.default_rng(2)
    wide = torch.zeros((T, V + 55), device="cuda")
    x = logits(T, V, 4)
    wide[:, 7:7 + V] = x.cuda()
    u = torch.from_numpy(rng.random(T, dtype=np.float32)).cuda()
    p = torch.full((T,), 0.9, device="cuda")
    want = sampling.sample(x.cuda(), u, top_p=p)
    assert torch.equal(sampling.sample(wide[:, 7:7 + V], u, top_p=p), want)
    out = torch.empty(T, dtype=torch.int32, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        sampling.sample(wide[:, 7:7 + V], u, top_p=p, out=out)
    for _ in range(3):
        out.fill_(-1)
        g.replay()
        assert torch.equal(out, want)
        u.copy_(torch.from_numpy(rng.random(T, dtype=np.float32)))
        want = sampling.sample(x.cuda(), u, top_p=p)


def test_agrees_with_argmax_at_temperature_zero():
    x = logits(7, 151936, 6).cuda()
    u = torch.full((7,), 0.7, device="cuda")
    ids = torch.empty(7, dtype=torch.int32, device="cuda")
    L, c = _lib.lib(), Context.for_device("cuda:0").handle
    assert L.rtd_argmax(c, x.data_ptr(), x.shape[1], 7, x.shape[1], ids.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(sampling.sample(x, u, temperature=torch.zeros(7, device="cuda")), ids)


def test_refusals():
    x, u = torch.zeros((2, 10), device="cuda"), torch.zeros(2, device="cuda")
    for bad, err in [(lambda: sampling.sample(x[0], u), ShapeError), (lambda: sampling.sample(x.double(), u), ConfigError),
                     (lambda: sampling.sample(x, u[:1]), ShapeError), (lambda: sampling.sample(x, u.double()), ConfigError),
                     (lambda: sampling.sample(x, u, top_k=u), ConfigError), (lambda: sampling.sample(x.t(), u), ConfigError),
                     (lambda: sampling.sample(x, u.cpu()), ConfigError),
                     (lambda: sampling.sample(torch.zeros((1, (1 << 19) + 1), device="cuda"), u[:1]), ConfigError)]:
        with pytest.raises(err):
            bad()
    L, h = _lib.lib(), Context.for_device("cuda:0").handle
    a = [h, x.data_ptr(), 0, 10, 2, 10, None, None, None, None, u.data_ptr(), u.data_ptr(), None]
    for at, value, code in [(1, None, 1), (2, 5, 1), (3, 9, 2), (4, -1, 2), (5, 0, 2), (5, (1 << 19) + 1, 2), (10, None, 1), (11, None, 1)]:
        bad = list(a)
        bad[at] = value
        assert L.rtd_sample(*bad) == code
    assert sampling.sample(x[:0], u[:0]).numel() == 0


@pytest.mark.parametrize("T,k", [(2, 100), (2, 128), (2, 129), (2, 257), (2, 513), (2, 1000), (150, 129), (150, 256)])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_sizes_of_top_k(T, k, dt):
    # candidates counted (up to 128) and sorted (up to 1024), one CTA a row and eight; in bf16
    # many are equal at the k-th place
    V = 30000
    x = logits(T, V, k).to(dt)
    rng = np.random.default_rng(k)
    for p, m in [(None, None), (0.97, 0.001)]:
        f = lambda v: None if v is None else np.full(T, v)  # noqa: E731
        check(x, rng.random(T, dtype=np.float32), rng.uniform(1.0, 4.0, T), f(k), f(p), f(m))


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_the_largest_rows_one_cta_each(dt):
    T, V, some = 150, 1 << 19, [0, 74, 149]
    x = logits(3, V, 5).to(dt)
    wide = torch.zeros((T, V), dtype=dt, device="cuda")
    wide[some] = x.cuda()
    u = np.random.default_rng(1).random(T, dtype=np.float32)
    for k, p, m in [(50, 0.9, 0.01), (0, 0.9, 0.0), (0, 1.0, 0.0), (1, 1.0, 0.0)]:
        full = lambda v, t: torch.full((T,), v, dtype=t, device="cuda")  # noqa: E731
        got = sampling.sample(wide, torch.from_numpy(u).cuda(), None, full(k, torch.int32), full(p, torch.float32), full(m, torch.float32))
        want = [pick(x[i].float().numpy(), u[r], 1.0, k, np.float64(np.float32(p)), np.float32(m)) for i, r in enumerate(some)]
        assert got.cpu()[some].tolist() == want


@pytest.mark.parametrize("T,k", [(2, 20), (2, 100), (2, 256), (150, 20), (150, 100), (150, 256)])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_top_k_of_logits_that_few_threads_hold(T, k, dt):
    # The largest lie side by side (a masked vocabulary) or far above the rest (a low temperature):
    # the threads' maxima do not bound the k-th largest, and the histogram of the whole row follows
    # at once.  Equal calls give equal ids, those of the rule.
    V = 30000
    rng = np.random.default_rng(k)
    x = torch.full((T, V), -float("inf"))
    x[:, 5000:5000 + 2 * k] = torch.from_numpy(rng.normal(0, 1, (T, 2 * k)).astype(np.float32))
    low = logits(T, V, k)
    for rows, t in [(x, None), (low, np.full(T, 0.02, np.float32))]:
        rows = rows.to(dt)
        for _ in range(3 if T < 10 else 1):
            check(rows, rng.random(T, dtype=np.float32), t, np.full(T, k), np.full(T, 0.99), None)
        d, u, kk = rows.cuda(), torch.from_numpy(rng.random(T, dtype=np.float32)).cuda(), torch.full((T,), k, dtype=torch.int32, device="cuda")
        tt = None if t is None else torch.from_numpy(t).cuda()
        first = sampling.sample(d, u, tt, kk)
        for _ in range(50):
            assert torch.equal(sampling.sample(d, u, tt, kk), first)
