"""The 4-bit paged KV cache (rtd_kv_plan, rtd_rope_kv4_append, rtd_kv4_read,
rtd_attention_kv4) on the GPU against float64 / integer numpy statements of the rules in
include/rtd.h.  Block tables are compared with the host's PagedKvCache, exactly; codes of
unrotated values are compared bit by bit; attention by bounds on its roundings.
"""
import math

import numpy as np
import pytest
import torch

from runtimed_b200 import _lib, kv4
from runtimed_b200.errors import ConfigError, ShapeError
from runtimed_b200.qwen2 import PagedKvCache, Qwen2Config
from runtimed_b200.weights import Context

pytestmark = pytest.mark.gpu

HEADS = [(14, 2, 64), (64, 8, 128), (28, 4, 128), (4, 4, 32), (12, 4, 96), (40, 2, 64)]


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def i32(a):
    return dev(np.asarray(a, np.int32))


def status():
    """The device status word's code, cleared."""
    try:
        Context.for_device("cuda:0").check_device_status()
    except ConfigError as e:
        return str(e)
    return ""


@pytest.fixture(autouse=True)
def clean_status():
    status()
    yield
    assert status() == ""


# ------------------------------------------------------------------ the format in numpy
def quantise(x):
    """x f32 [..., D] -> (codes, d, m): groups of 32, in 32-bit arithmetic as stated."""
    g = np.asarray(x, np.float32).reshape(*x.shape[:-1], -1, 32)
    lo, hi = g.min(-1), g.max(-1)
    with np.errstate(all="ignore"):
        d = ((hi - lo) / np.float32(15)).astype(np.float16)
        m = lo.astype(np.float16)
        bad = ~(np.isfinite(g).all(-1) & np.isfinite(d) & np.isfinite(m))
        df, mf = d.astype(np.float32)[..., None], m.astype(np.float32)[..., None]
        c = np.where(df > 0, np.clip(np.rint((g - mf) / df), 0, 15), 0)
        c = np.where(bad[..., None], 0, c)
    d[bad] = np.nan
    m[bad] = np.nan
    return c.astype(np.int64).reshape(x.shape), d, m


def values(c, d, m):
    """f64 values of codes and headers."""
    g = c.reshape(*c.shape[:-1], -1, 32)
    return (g * d.astype(np.float64)[..., None] + m.astype(np.float64)[..., None]).reshape(c.shape)


def page_of(kc, kd, km, vc, vd, vm):
    """Bytes [20 D] of one page from [16, D] codes and [16, NG] headers, by the stated layout."""
    D = kc.shape[1]
    ng = D // 32
    out = np.zeros(20 * D, np.uint8)
    for t in range(16):
        for d in range(D):
            g, r = divmod(d, 32)
            byte = t * (D // 2) + ((r // 8) * ng + g) * 4 + (r % 8) // 2
            out[byte] |= kc[t, d] << (4 * (d % 2))
            n, p = divmod(r, 4)
            if ng == 4:
                at = ((2 * n + g // 2) ^ (8 if t & 2 else 0)) * 4 + (g % 2) * 2
            elif ng % 2 and g == ng - 1:
                at = ((ng - 1) * 8 + n) * 2
            else:
                at = n * 4 + (g % 2) * 2
            out[10 * D + t * (D // 2) + at + p // 2] |= vc[t, d] << (4 * (d % 2))
        for g in range(ng):
            for base, dd, mm in ((8 * D, kd, km), (18 * D, vd, vm)):
                at = base + (t * ng + g) * 4
                out[at:at + 4] = np.array([dd[t, g], mm[t, g]], np.float16).view(np.uint8)
    return out


# ------------------------------------------------------------------ block tables
def make_state(n_seq, max_blocks, n_blocks, seed):
    rng = np.random.default_rng(seed)
    return dict(length=i32(np.zeros(n_seq)), table=i32(np.zeros((n_seq, max_blocks))), free_list=i32(rng.permutation(n_blocks)),
                free_count=i32([n_blocks]))


def host_cache(n_seq, max_blocks, n_blocks, free):
    cfg = Qwen2Config(0, 32, 1, 1, 32, 32, 32, 1e-6, 1e4, False)
    c = PagedKvCache(cfg, n_blocks, n_seq, max_blocks * 16, "cpu")
    c._free = [int(v) for v in free]
    return c


@pytest.mark.parametrize("n_seq,max_blocks,n_blocks,steps", [(1, 1, 1, 6), (3, 4, 9, 30), (64, 20, 900, 12), (1500, 3, 4000, 6)])
def test_plan_follows_the_host_cache(n_seq, max_blocks, n_blocks, steps):
    rng = np.random.default_rng(n_seq)
    st = make_state(n_seq, max_blocks, n_blocks, n_seq)
    host = host_cache(n_seq, max_blocks, n_blocks, st["free_list"].cpu().numpy())
    lens = np.zeros(n_seq, np.int64)
    for step in range(steps):
        kind = rng.integers(0, 4, n_seq)
        want = np.where(kind == 0, 0, np.where(kind == 1, lens, np.where(kind == 2, np.minimum(lens + 1, max_blocks * 16),
                                                                       rng.integers(0, max_blocks * 16 + 1, n_seq))))
        # keep within the pool
        while sum(-(-int(w) // 16) for w in want) > n_blocks:
            want[rng.integers(0, n_seq)] = 0
        new = np.maximum(want - lens, 0)
        total = int(new.sum())
        cap = total + int(rng.integers(0, 40))
        start, seq, pos, slot = kv4.plan(i32(want), **st, max_tokens=cap)
        for s in range(n_seq):
            if want[s] < lens[s]:
                host.truncate(s, int(want[s]))
        for s in range(n_seq):
            if want[s] > lens[s]:
                host.reserve(s, int(want[s]))
        assert st["length"].cpu().tolist() == want.tolist()
        n = int(st["free_count"].cpu()[0])
        assert st["free_list"].cpu().tolist()[:n] == host._free
        t = st["table"].cpu().numpy()
        for s in range(n_seq):
            nb = -(-int(want[s]) // 16)
            assert t[s, :nb].tolist() == host._blocks.get(s, [])
        want_tok = [(s, p, int(t[s, p // 16]) * 16 + p % 16) for s in range(n_seq) for p in range(int(lens[s]), int(want[s]))]
        got = list(zip(seq.cpu().tolist(), pos.cpu().tolist(), slot.cpu().tolist()))
        assert got == want_tok + [(-1, -1, -1)] * (cap - total)
        assert start.cpu().tolist() == np.concatenate([[0], np.cumsum(new)]).tolist()
        lens = want
    assert status() == ""


@pytest.mark.parametrize("what", ["negative", "too long", "too many tokens", "no blocks", "bad count"])
def test_plan_refuses_whole(what):
    # nothing changes, the lists are empty and the status word tells
    st = make_state(5, 8, 12, 3)
    kv4.plan(i32([20, 0, 33, 16, 1]), **st)
    want = {"negative": [20, 0, -1, 16, 1], "too long": [20, 129, 33, 16, 1], "too many tokens": [60, 0, 33, 16, 1],
            "no blocks": [20, 128, 33, 16, 1], "bad count": [21, 0, 33, 16, 1]}[what]
    if what == "bad count":
        st["free_count"].fill_(13)
    before = {k: v.clone() for k, v in st.items()}
    out = kv4.plan(i32(want), **st, max_tokens=130 if what != "too many tokens" else 39)
    for k, v in st.items():
        assert torch.equal(v, before[k]), k
    assert out[0].cpu().tolist() == [0] * 6
    assert all((o == -1).all() for o in out[1:])
    assert "paged cache" in status()


def test_plan_of_no_sequences_and_no_tokens():
    st = make_state(1, 4, 4, 0)
    kv4.plan(i32([7]), **st)
    out = kv4.plan(i32([7]), **st, max_tokens=0)
    assert out[0].cpu().tolist() == [0, 0] and out[1].numel() == 0
    empty = dict(length=i32([]), table=i32(np.zeros((0, 4))), free_list=st["free_list"], free_count=st["free_count"])
    out = kv4.plan(i32([]), **empty, max_tokens=3)
    assert out[0].cpu().tolist() == [0] and (out[3] == -1).all()


# ------------------------------------------------------------------ append and read
def rope64(x, pos, inv):
    half = len(inv)
    ang = pos.astype(np.float64)[:, None, None] * inv[None, None]
    c, s = np.cos(ang), np.sin(ang)
    a, b = x[..., :half], x[..., half:2 * half]
    return np.concatenate([a * c - b * s, b * c + a * s, x[..., 2 * half:]], -1)


@pytest.mark.parametrize("n_head,n_kv,D", HEADS)
@pytest.mark.parametrize("T,dt", [(1, torch.float32), (37, torch.bfloat16), (400, torch.float16)])
def test_append_without_rope_is_exact(n_head, n_kv, D, T, dt):
    # no rotation: the pages hold exactly what the rule says, byte by byte
    g = torch.Generator().manual_seed(T + D)
    q, k, v = (torch.randn((T, h, D), generator=g).to(dt) for h in (n_head, n_kv, n_kv))
    k = k * 3 + 1
    blocks = -(-T // 16) + 3
    slots = np.random.default_rng(T).permutation(blocks * 16)[:T].astype(np.int32)
    pages = kv4.alloc_pages(blocks, n_kv, D)
    none = torch.empty(0, dtype=torch.float64, device="cuda")
    qo = kv4.append(q.cuda(), k.cuda(), v.cuda(), none, i32(np.arange(T)), i32(slots), pages)
    assert torch.equal(qo.cpu(), q.float())
    K = np.zeros((blocks, 16, n_kv, D), np.int64), np.zeros((blocks, 16, n_kv, D // 32), np.float16), np.zeros((blocks, 16, n_kv, D // 32), np.float16)
    V = tuple(a.copy() for a in K)
    for X, x in ((K, k), (V, v)):
        for a, b in zip(X, quantise(x.float().numpy())):
            a[slots // 16, slots % 16] = b
    want = np.stack([np.stack([page_of(*(a[b, :, h] for a in K), *(a[b, :, h] for a in V)) for h in range(n_kv)])
                     for b in range(blocks)])
    assert np.array_equal(pages.cpu().numpy(), want)
    # and the reader gives the values they stand for
    kk, vv = kv4.read(pages, i32(slots))
    for got, x in ((kk, k), (vv, v)):
        w = values(*quantise(x.float().numpy()))
        # one fma: half a step of the value
        assert np.all(np.abs(got.cpu().numpy() - w) <= np.abs(w) * 2.0 ** -24 + 1e-45)
    h, _ = kv4.read(pages, i32(slots), torch.bfloat16)
    assert torch.equal(h, kk.to(torch.bfloat16))


@pytest.mark.parametrize("rot", [64, 32, 10, 0])
def test_append_rotates_far_positions(rot):
    n_head, n_kv, D, T = 6, 2, 64, 50
    rng = np.random.default_rng(rot)
    pos = rng.integers(0, 1 << 20, T).astype(np.int32)
    inv = 1e6 ** (-2.0 * np.arange(rot // 2) / max(rot, 1))
    q, k, v = (rng.normal(0, 1, (T, h, D)).astype(np.float32) for h in (n_head, n_kv, n_kv))
    slots = rng.permutation(80)[:T].astype(np.int32)
    slots[7] = -1
    pages = kv4.alloc_pages(5, n_kv, D)
    qo = kv4.append(dev(q), dev(k), dev(v), dev(inv), i32(pos), i32(slots), pages).cpu().numpy()
    # cos, sin, two products and a sum, each off by half a step of at most |x1| + |x2|
    want = rope64(q.astype(np.float64), pos, inv)
    assert np.max(np.abs(qo - want)) <= 5 * 2.0 ** -24 * 2 * np.abs(q).max()
    kk, vv = (x.cpu().numpy() for x in kv4.read(pages, i32(slots)))
    kw = rope64(k.astype(np.float64), pos, inv)
    for got, w in ((kk, kw), (vv, v.astype(np.float64))):
        g = w.reshape(T, n_kv, -1, 32)
        step = (g.max(-1) - g.min(-1))[..., None] / 15
        # half a step, the minimum's rounding (2^-11), the step's rounding over 15 codes, f32 slack
        bound = step / 2 + np.abs(g).max(-1, keepdims=True) * (2.0 ** -11 + 2.0 ** -20) + 15 * step * 2.0 ** -11
        err = np.abs(got.reshape(g.shape) - g)
        live = slots >= 0
        assert np.all(err[live] <= np.broadcast_to(bound, err.shape)[live])
        assert not got[7].any()  # a padded row reads as zeros ...
    untouched = np.setdiff1d(np.arange(80), slots).astype(np.int32)
    assert not torch.stack(kv4.read(pages, i32(untouched))).any()  # ... and wrote nowhere


def test_append_of_constants_and_non_finite_groups():
    D = 64
    x = np.zeros((6, 1, D), np.float32)
    x[1] = 5.0                        # a constant group: step 0
    x[2, 0, 3] = np.inf
    x[3, 0, 40] = np.nan
    x[4, 0, 0], x[4, 0, 1] = -60000, 60000
    x[5, 0, 0], x[5, 0, 1] = -3e6, 3e6  # the header overflows f16
    pages = kv4.alloc_pages(1, 1, D)
    none = torch.empty(0, dtype=torch.float64, device="cuda")
    kv4.append(dev(x), dev(x), dev(x), none, i32(np.zeros(6)), i32(np.arange(6)), pages)
    for got in kv4.read(pages, i32(np.arange(6))):
        got = got.cpu().numpy()[:, 0]
        assert not got[0].any() and (got[1] == 5.0).all()
        assert np.isnan(got[2, :32]).all() and not got[2, 32:].any()
        assert np.isnan(got[3, 32:]).all() and not got[3, :32].any()
        assert np.isfinite(got[4]).all() and abs(got[4, 1] - 60000) <= 60000 * 2.0 ** -9
        assert np.isnan(got[5, :32]).all()


def test_append_takes_strided_rows_and_reports_bad_slots():
    T, H, G, D = 9, 4, 2, 64
    rng = np.random.default_rng(3)
    row = (H + 2 * G) * D + 24
    qkv = dev(rng.normal(0, 1, (T, row)).astype(np.float32))
    q, k, v = (qkv[:, a:a + n * D].unflatten(1, (n, D)) for a, n in ((0, H), (H * D, G), ((H + G) * D, G)))
    inv = kv4.rope_frequencies(D, 1e4)
    slots = np.arange(T) * 3
    out = []
    for args in ((q, k, v), (q.contiguous(), k.contiguous(), v.contiguous())):
        pages = kv4.alloc_pages(2, G, D)
        out.append((kv4.append(*args, inv, i32(np.arange(T)), i32(slots), pages), pages))
    assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1])
    bad = slots.copy()
    bad[4] = 32  # the pool has slots 0 .. 31
    pages = kv4.alloc_pages(2, G, D)
    kv4.append(q, k, v, inv, i32(np.arange(T)), i32(bad), pages)
    assert "paged cache" in status()
    good = np.delete(slots, 4)
    for a, b in zip(kv4.read(pages, i32(good)), kv4.read(out[1][1], i32(good))):
        assert torch.equal(a, b)
    k2, v2 = kv4.read(pages, i32([32, 3]))
    assert "paged cache" in status() and not k2[0].any()


# ------------------------------------------------------------------ attention
class Case:
    """A pool with sequences of the given lengths, and its values in 64 bits."""

    def __init__(self, lens, n_kv, D, seed, k_std=1.0, v_std=1.0, spare=2, bias=1.0, big=None):
        rng = np.random.default_rng(seed)
        self.lens, self.n_kv, self.D = list(lens), n_kv, D
        nb = [-(-max(0, n) // 16) for n in lens]
        used = sum(nb)
        total = used + spare
        perm = rng.permutation(total) if big is None else big - 1 - rng.permutation(total)
        self.table = np.zeros((len(lens), max(1, max(nb))), np.int32)
        # unused table entries and unwritten slots hold anything
        self.table[:] = np.int32(2 ** 31 - 1)
        at = 0
        self.K, self.V, slots = [], [], []
        pool = total if big is None else big
        self.pages = torch.empty((pool, n_kv, kv4.page_bytes(D)), dtype=torch.uint8, device="cuda")
        if big is None:
            self.pages.fill_(255)
        else:
            self.pages[big - total:].fill_(255)
        ks, vs = [], []
        off = rng.normal(0, bias, (n_kv, D))
        for s, n in enumerate(lens):
            self.table[s, :nb[s]] = perm[at:at + nb[s]]
            at += nb[s]
            ks.append((rng.normal(0, k_std, (n, n_kv, D)) + off).astype(np.float32))
            vs.append(rng.normal(0, v_std, (n, n_kv, D)).astype(np.float32))
            p = np.arange(n)
            slots.append(self.table[s, p // 16] * 16 + p % 16)
        self.slots = [np.asarray(x, np.int32) for x in slots]
        self.write(np.concatenate(ks), np.concatenate(vs), np.concatenate(self.slots).astype(np.int32))

    def write(self, k, v, slots):
        none = torch.empty(0, dtype=torch.float64, device="cuda")
        if len(slots):
            kv4.append(dev(k), dev(k), dev(v), none, i32(np.zeros(len(slots))), i32(slots), self.pages)
        self.load()

    def load(self):
        self.K, self.V = [], []
        for x in self.slots:
            k, v = kv4.read(self.pages, i32(x))
            self.K.append(k.cpu().numpy().astype(np.float64))
            self.V.append(v.cpu().numpy().astype(np.float64))

    def want(self, q, new, scale):
        """(rows in 64 bits, their error bounds for exact f32 outputs)."""
        out, tol = np.zeros(q.shape), np.zeros(q.shape)
        row = 0
        H = q.shape[1]
        for s, n in enumerate(new):
            for i in range(n):
                seen = max(0, self.lens[s] - n + i + 1)
                for h in range(H):
                    g = h * self.n_kv // H
                    if seen:
                        K, V = self.K[s][:seen, g], self.V[s][:seen, g]
                        x = K @ q[row, h] * scale
                        w = np.exp(x - x.max())
                        w /= w.sum()
                        out[row, h] = w @ V
                        # a score is off by 2^-21 of sum |q| |k| (queries in 22 bits, 32-bit
                        # sums with minimum and step apart: at most 4 times sum |q k|), which
                        # moves the output by twice that; p d in 22 bits; each 16 keys a
                        # 32-bit sum more, warps and chunks a few more
                        a = np.abs(q[row, h]) @ (np.abs(K).max(0)) * scale * 4
                        d = 2 * a * 2.0 ** -21 + 2.0 ** -19 + (seen / 16 + 8) * 2.0 ** -23
                        tol[row, h] = d * np.abs(V).max(0).max()
                row += 1
        return out, tol


def run_attention(c, q, new, scale=None, out_dtype=torch.float32, out=None, max_q=None, max_ctx=None, ctx=None):
    start = np.concatenate([[0], np.cumsum(new)])
    return kv4.attention(q, c.pages, i32(c.table), i32(start), i32(c.lens if ctx is None else ctx), max_q or max(1, max(new)),
                         max_ctx or max(1, max(c.lens)), scale=scale, out_dtype=out_dtype, out=out)


def check(c, new, H, out_dtype=torch.float32, q_dtype=torch.float32, q_std=1.0, seed=0, **kw):
    rng = np.random.default_rng(seed)
    q = torch.from_numpy(rng.normal(0, q_std, (sum(new), H, c.D)).astype(np.float32)).to(q_dtype)
    got = run_attention(c, q.cuda(), new, out_dtype=out_dtype, **kw)
    want, tol = c.want(q.double().numpy(), new, 1 / math.sqrt(c.D))
    if out_dtype != torch.float32:
        # rounding the output: half a step; 16-bit queries and weights behind it, 2^-11 each
        half = torch.finfo(out_dtype).eps / 2
        tol = tol + np.abs(want) * half + 2.0 ** -24
        tol = tol + tol_16bit(c, q, new)
    err = np.abs(got.double().cpu().numpy() - want)
    assert np.all(err <= tol), (err.max(), (err / np.maximum(tol, 1e-300)).max())
    return got


def tol_16bit(c, q, new):
    """What queries, keys and weights of 11 bits may add: 2^-11 of sum |q| |k| in a score."""
    scale = 1 / math.sqrt(c.D)
    out = []
    for s, n in enumerate(new):
        K = np.abs(c.K[s]).max(0).max(0) if len(c.K[s]) else np.zeros(c.D)
        V = np.abs(c.V[s]).max() if len(c.V[s]) else 0.0
        out += [(4 * K.max() * scale * 2.0 ** -11 + 2.0 ** -10, V)] * n
    a = np.array([x for x, _ in out])[:, None, None] * np.maximum(1, np.abs(q.double().numpy()).sum(-1, keepdims=True))
    return a * np.array([v for _, v in out])[:, None, None]


@pytest.mark.parametrize("H,n_kv,D", HEADS)
@pytest.mark.parametrize("lens", [[1], [15, 16, 17], [160], [33, 700, 2, 64]])
def test_decode(H, n_kv, D, lens):
    check(Case(lens, n_kv, D, seed=D + len(lens)), [1] * len(lens), H)


@pytest.mark.parametrize("H,n_kv,D", HEADS)
@pytest.mark.parametrize("lens,new", [([5], [5]), ([40, 21], [3, 5]), ([300, 7, 90], [130, 7, 1]), ([64], [17])])
def test_several_queries(H, n_kv, D, lens, new):
    check(Case(lens, n_kv, D, seed=H), new, H)


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("q_dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,new", [([700, 31], [1, 1]), ([200], [150]), ([2100, 100], [64, 100])])
def test_types(out_dtype, q_dtype, lens, new):
    check(Case(lens, 2, 64, seed=5), new, 8, out_dtype=out_dtype, q_dtype=q_dtype)


@pytest.mark.parametrize("n", [4000, 20011])
def test_long_contexts_split_and_join_alike(n):
    c = Case([n, 700], 2, 128, seed=n)
    a = check(c, [1, 1], 16)
    rng = np.random.default_rng(0)
    q = dev(rng.normal(0, 1, (2, 16, 128)).astype(np.float32))
    assert torch.equal(run_attention(c, q, [1, 1]), a)  # equal calls, equal bits


def test_rows_that_see_nothing_and_rows_of_no_sequence():
    c = Case([0, 20, 2], 2, 64, seed=1)
    rng = np.random.default_rng(2)
    new = [1, 0, 4]  # an empty sequence, one without queries, one whose first two rows come before its start
    q = rng.normal(0, 1, (8, 8, 64)).astype(np.float32)
    out = torch.full((8, 8, 64), 7.0, device="cuda")
    got = run_attention(c, dev(q), new, out=out).cpu().numpy()
    want, tol = c.want(q[:5].astype(np.float64), new, 1 / 8)
    assert np.all(np.abs(got[:5] - want) <= tol)
    assert not got[:3].any() and (got[5:] == 7.0).all()


@pytest.mark.parametrize("std", [1e-3, 300.0])
def test_small_and_large_values(std):
    # steps of V far below and above one
    check(Case([500, 77], 2, 64, seed=3, v_std=std), [1, 2], 8)


def test_sharp_scores():
    # one key far above the others, met late: the running maximum rises again and again
    c = Case([900], 1, 64, seed=4)
    k = np.stack([np.full((1, 64), (i / 900) * 3.0, np.float32) for i in range(900)])
    v = np.random.default_rng(0).normal(0, 1, (900, 1, 64)).astype(np.float32)
    c.write(k, v, c.slots[0])
    q = np.ones((1, 8, 64), np.float32) * np.linspace(-8, 8, 8, dtype=np.float32)[None, :, None]
    got = run_attention(c, dev(q), [1]).cpu().numpy()
    want, tol = c.want(q.astype(np.float64), [1], 1 / 8)
    assert np.all(np.abs(got - want) <= tol)


def test_nan_is_seen_only_by_rows_that_see_its_key():
    # keys 36 (V) and 38 (K) hold a NaN group; rows before them stay clean
    c = Case([40], 2, 64, seed=6)
    k, v = c.K[0].astype(np.float32), c.V[0].astype(np.float32)
    v[36, 1, 40] = np.nan
    k[38, 0, 3] = np.nan
    c.write(k, v, c.slots[0])
    q = np.random.default_rng(1).normal(0, 1, (6, 4, 64)).astype(np.float32)
    got = run_attention(c, dev(q), [6]).cpu().numpy()  # positions 34 .. 39
    assert np.isfinite(got[:2]).all()
    assert np.isfinite(got[2:4, :2]).all() and np.isnan(got[4:, :2]).all()      # kv head 0: K at 38
    assert np.isfinite(got[2:, 2:, :32]).all() and np.isnan(got[2:, 2:, 32:]).all()  # kv head 1: V group 1 at 36
    want, tol = c.want(q.astype(np.float64)[:2], [2], 1 / 8)
    c.lens = [36]
    c.load()
    want, tol = c.want(q.astype(np.float64)[:2], [2], 1 / 8)
    assert np.all(np.abs(got[:2] - want) <= tol)


def test_strided_queries_and_outputs():
    c = Case([90, 30], 2, 64, seed=7)
    rng = np.random.default_rng(3)
    wide = dev(rng.normal(0, 1, (3, 1000)).astype(np.float32))
    q = wide[:, 3:3 + 512].unflatten(1, (8, 64))
    store = torch.zeros((3, 700), device="cuda")
    out = store[:, 5:5 + 512].unflatten(1, (8, 64))
    run_attention(c, q, [2, 1], out=out)
    assert torch.equal(out, run_attention(c, q.contiguous(), [2, 1]))
    assert not store[:, :5].any() and not store[:, 517:].any()


def test_pool_beyond_4_gib():
    blocks = (1 << 32) // (2 * kv4.page_bytes(128)) + 500
    c = Case([70, 20], 2, 128, seed=8, big=blocks)
    assert c.table[c.table < 2 ** 31 - 1].min() > (1 << 32) // (2 * kv4.page_bytes(128))
    check(c, [2, 1], 8)


def test_bad_blocks_and_lengths_are_reported():
    c = Case([50, 40], 2, 64, seed=9)
    q = dev(np.random.default_rng(4).normal(0, 1, (2, 8, 64)).astype(np.float32))
    clean = run_attention(c, q, [1, 1])
    keep = c.table[0, 1]
    for wrong in (-1, c.pages.shape[0], 2 ** 31 - 1):
        c.table[0, 1] = wrong
        got = run_attention(c, q, [1, 1])
        assert "paged cache" in status()
        assert torch.isnan(got[0]).all() and torch.equal(got[1], clean[1])
    c.table[0, 1] = keep
    got = run_attention(c, q, [1, 1], ctx=[50, 49], max_ctx=48)  # both beyond their bound
    assert "paged cache" in status() and not got.any()
    # more queries than max_q, or offsets outside the rows: the sequence is left out
    out = torch.full_like(clean, 3.0)
    start = i32([0, 2, 2])
    kv4.attention(q, c.pages, i32(c.table), start, i32(c.lens), 1, 50, out=out)
    assert "paged cache" in status() and (out == 3.0).all()
    kv4.attention(q, c.pages, i32(c.table), i32([-1, 1, 7]), i32(c.lens), 8, 50, out=out)
    assert "paged cache" in status() and (out == 3.0).all()


def test_another_stream_and_a_captured_graph():
    c = Case([400, 90], 2, 64, seed=10)
    rng = np.random.default_rng(5)
    qs = [dev(rng.normal(0, 1, (2, 8, 64)).astype(np.float32)) for _ in range(3)]
    want = [run_attention(c, q, [1, 1]) for q in qs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(run_attention(c, qs[0], [1, 1]), want[0])
    torch.cuda.current_stream().wait_stream(side)
    q, out = qs[0].clone(), torch.empty_like(want[0])
    args = (i32(c.table), i32([0, 1, 2]), i32(c.lens))
    graphs = []
    for _ in range(2):  # two graphs that share the context's workspace
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            kv4.attention(q, c.pages, *args, 1, 400, out=out)
        graphs.append(g)
    for i in range(6):
        q.copy_(qs[i % 3])
        out.zero_()
        graphs[i % 2].replay()
        assert torch.equal(out, want[i % 3])


# ------------------------------------------------------------------ refusals
def test_refusals():
    c = Case([20], 2, 64, seed=11)
    q = torch.zeros((1, 8, 64), device="cuda")
    t, s, n = i32(c.table), i32([0, 1]), i32([20])
    ok = dict(max_q=1, max_ctx=20)
    for bad, err in [
        (lambda: kv4.attention(q[..., :32], c.pages, t, s, n, **ok), ShapeError),          # page size of another head_dim
        (lambda: kv4.attention(q.cpu(), c.pages, t, s, n, **ok), ConfigError),
        (lambda: kv4.attention(q.double(), c.pages, t, s, n, **ok), ConfigError),
        (lambda: kv4.attention(torch.zeros((1, 7, 64), device="cuda"), c.pages, t, s, n, **ok), ConfigError),
        (lambda: kv4.attention(q, c.pages, t.long(), s, n, **ok), ConfigError),
        (lambda: kv4.attention(q, c.pages, t, s[:1], n, **ok), ShapeError),
        (lambda: kv4.attention(q, c.pages, t, s, n, max_q=0, max_ctx=20), ConfigError),
        (lambda: kv4.attention(q, c.pages, t, s, n, max_q=1, max_ctx=100), ConfigError),   # beyond the table
        (lambda: kv4.attention(q.transpose(1, 2).contiguous().transpose(1, 2), c.pages, t, s, n, **ok), ConfigError),
        (lambda: kv4.read(c.pages[:, :, :-20].contiguous(), n), ConfigError),              # head_dim 63
        (lambda: kv4.append(q, q[:, :2], q[:, :1], kv4.rope_frequencies(64, 1e4), n, n, c.pages), ShapeError),
        (lambda: kv4.append(q, q[:, :2], q[:, :2].half(), kv4.rope_frequencies(64, 1e4), n, n, c.pages), ConfigError),
        (lambda: kv4.append(q, q[:, :2], q[:, :2], kv4.rope_frequencies(64, 1e4).float(), n, n, c.pages), ConfigError),
        (lambda: kv4.plan(i32([1, 2]), n, t, i32([0]), i32([1])), ShapeError),
    ]:
        with pytest.raises(err):
            bad()
    L, h = _lib.lib(), Context.for_device("cuda:0").handle
    p, z = c.pages.data_ptr(), torch.zeros(64, dtype=torch.int32, device="cuda").data_ptr()
    f = q.data_ptr()
    att = [h, f, 0, 512, 1, 8, 2, 64, 0.1, z, z, 1, z, 2, 1, 20, p, 4, f, 0, 512, None]
    for at, value, code in [(2, 9, _lib.RTD_ERR_INVALID), (3, 511, _lib.RTD_ERR_SHAPE), (4, -1, _lib.RTD_ERR_SHAPE),
                            (5, 7, _lib.RTD_ERR_SHAPE), (7, 80, _lib.RTD_ERR_SHAPE), (7, 256, _lib.RTD_ERR_SHAPE),
                            (9, None, _lib.RTD_ERR_INVALID), (13, 0, _lib.RTD_ERR_INVALID), (16, p + 8, _lib.RTD_ERR_INVALID),
                            (17, 0, _lib.RTD_ERR_SHAPE), (19, 3, _lib.RTD_ERR_INVALID), (20, 500, _lib.RTD_ERR_SHAPE)]:
        bad = list(att)
        bad[at] = value
        assert L.rtd_attention_kv4(*bad) == code, (at, value)
    assert L.rtd_kv_plan(h, z, 8193, z, z, 1, z, z, 1, None, None, None, None, 0, None) == _lib.RTD_ERR_SHAPE
    assert L.rtd_kv_plan(h, z, 1, z, z, 1, z, z, 1, z, None, None, None, 4, None) == _lib.RTD_ERR_INVALID
    assert L.rtd_rope_kv4_append(h, f, 512, f, 128, f, 128, 0, 1, 8, 2, 64, 66, z, z, z, p, 4, f, None) == _lib.RTD_ERR_SHAPE
