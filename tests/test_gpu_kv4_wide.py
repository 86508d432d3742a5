"""rtd_attention_kv4 for prompt chunks with 16-bit outputs (many query rows of a sequence on
the tcgen05 tensor cores) against float64, by bounds on its roundings, and what it shares a
call with: decoding sequences, rows without keys, rows of no sequence.
"""
import math

import numpy as np
import pytest
import torch

from runtimed_b200 import _lib, kv4
from runtimed_b200.errors import ConfigError
from runtimed_b200.weights import Context
from test_gpu_kv4 import Case, clean_status, dev, i32, run_attention, status  # noqa: F401

pytestmark = pytest.mark.gpu

HEADS = [(64, 8, 128), (14, 2, 64), (40, 2, 64), (3, 3, 128)]  # 8, 7, 20 and 1 heads a group
WIDE = 96  # rows (queries x heads of the group) from which a sequence is a chunk


def expected(c, q, new, out_dtype):
    """(rows in 64 bits, bounds): q f64 [T, H, D]."""
    H = q.shape[1]
    G, scale = H // c.n_kv, 1 / math.sqrt(c.D)
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    at = 0
    for s, n in enumerate(new):
        ctx = c.lens[s]
        see = np.arange(ctx)[None] <= ctx - n + np.arange(n)[:, None]  # [n, ctx]
        some = see.any(1)
        chunk = n * G >= WIDE
        for h in range(H if ctx and n else 0):
            K, V, Q = c.K[s][:, h // G], c.V[s][:, h // G], q[at:at + n, h]
            x = np.where(see, Q @ K.T * scale, -np.inf)
            with np.errstate(invalid="ignore"):
                w = np.exp(x - np.where(some, x.max(1), 0)[:, None])
                w = np.where(some[:, None], w / w.sum(1, keepdims=True), 0)
            # A chunk's scores: queries and keys rounded to f16, 2^-11 each, and 32-bit sums and
            # exponentials.  Otherwise the products are with codes, |q| |d c| <= |q| (|k| + |m|),
            # at most four times the group's largest value.
            a = np.abs(Q) @ np.abs(K).T * scale if chunk else \
                4 * np.abs(Q).sum(1, keepdims=True) * np.abs(K).max() * scale * np.ones((1, ctx))
            e = np.where(see, np.expm1(np.minimum(a * 1.02 * 2.0 ** -10 + 2.0 ** -16, 50)), 0)
            v = np.abs(V) if chunk else np.full_like(V, 3 * np.abs(V).max())
            # weights and values rounded to f16, 2^-11 each; sums of 16 keys in 32 bits
            wv = w @ v
            err = (w * e) @ v + (w * e).sum(1, keepdims=True) * wv + (1.01 * 2.0 ** -10 + ctx * 2.0 ** -26 + 2.0 ** -14) * wv
            # whatever the weights, result and mean lie within the values (each rounded): where
            # scores are so large that their roundings alone decide, this is the bound
            err = np.minimum(err, 2.01 * np.abs(V).max())
            out[at:at + n, h] = w @ V
            half = torch.finfo(out_dtype).eps / 2
            tol[at:at + n, h] = err * (1 + half) + np.abs(w @ V) * half + 2.0 ** -24
        at += n
    return out, tol


def check(c, new, H, out_dtype=torch.float16, q_dtype=torch.float32, q_std=1.0, out=None, q=None):
    rng = np.random.default_rng(len(new))
    if q is None:
        q = torch.from_numpy(rng.normal(0, q_std, (sum(new), H, c.D)).astype(np.float32)).to(q_dtype).cuda()
    got = run_attention(c, q, new, out_dtype=out_dtype, out=out)
    want, tol = expected(c, q.double().cpu().numpy(), new, out_dtype)
    err = np.abs(got.double().cpu().numpy() - want)
    assert np.all(err <= tol), (err.max(), (err / np.maximum(tol, 1e-300)).max(), np.argwhere(err > tol)[:5])
    return got


@pytest.mark.parametrize("H,n_kv,D", HEADS)
@pytest.mark.parametrize("lens,new", [
    ([130], [130]),                                     # a whole prompt
    ([700, 31, 64, 50, 513], [100, 1, 64, 0, 300]),     # with a decoding sequence and one without queries
    ([1025, 97], [97, 97]),
    ([2049], [33]),
])
def test_chunks(H, n_kv, D, lens, new):
    check(Case(lens, n_kv, D, seed=D + len(lens)), new, H)


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("q_dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_types(out_dtype, q_dtype):
    check(Case([400, 90], 2, 64, seed=5), [120, 3], 14, out_dtype=out_dtype, q_dtype=q_dtype)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("ctx,n", [(1, 300), (17, 130), (63, 63), (64, 64), (65, 65), (96, 33), (127, 50), (333, 129), (334, 65)])
def test_every_key_counts_once(D, ctx, n):
    # Scores near zero, and key i's value is 1 at dim i % D alone (15 steps of f16(1 / 15)):
    # a missing or doubled key changes that dim by a sixth at least, against a bound of 1 %.
    c = Case([ctx], 1, D, seed=ctx, k_std=0.05, bias=0.0)
    v = np.zeros((ctx, 1, D), np.float32)
    v[np.arange(ctx), 0, np.arange(ctx) % D] = 1
    c.write(c.K[0].astype(np.float32), v, c.slots[0])
    check(c, [n], 8, q_std=0.05)


def test_rows_that_see_nothing_and_rows_of_no_sequence():
    c = Case([20, 0, 40], 2, 64, seed=1)
    new = [90, 30, 0]  # 70 queries before the sequence's start, a chunk of an empty sequence
    q = dev(np.random.default_rng(2).normal(0, 1, (125, 14, 64)).astype(np.float32))
    out = torch.full((125, 14, 64), 7.0, device="cuda", dtype=torch.float16)
    start = i32([0, 90, 120, 120])
    got = kv4.attention(q, c.pages, i32(c.table), start, i32(c.lens), 90, 40, out=out)
    want, tol = expected(c, q[:120].double().cpu().numpy(), new, torch.float16)
    assert np.all(np.abs(got[:120].double().cpu().numpy() - want) <= tol)
    assert not got[:70].any() and not got[90:120].any() and (got[120:] == 7.0).all()


def test_nan_keys_and_values():
    # keys 130 (K, kv head 0) and 135 (V, kv head 1, the second group) hold a NaN group
    c = Case([200], 2, 64, seed=6)
    k, v = c.K[0].astype(np.float32), c.V[0].astype(np.float32)
    k[130, 0, 3] = np.nan
    v[135, 1, 40] = np.nan
    c.write(k, v, c.slots[0])
    q = np.random.default_rng(1).normal(0, 1, (100, 14, 64)).astype(np.float32)  # positions 100 .. 199
    got = run_attention(c, dev(q), [100], out_dtype=torch.bfloat16).float().cpu().numpy()
    assert np.isfinite(got[:30]).all() and np.isnan(got[30:, :7]).all()
    assert np.isfinite(got[:35, 7:]).all() and np.isnan(got[35:, 7:, 32:]).all()
    # before the chunk's own tokens: the group alone
    c = Case([200], 2, 64, seed=6)
    v = c.V[0].astype(np.float32)
    v[20, 1, 40] = np.nan
    c.write(c.K[0].astype(np.float32), v, c.slots[0])
    got = run_attention(c, dev(q), [100], out_dtype=torch.bfloat16).float().cpu().numpy()
    assert np.isfinite(got[:, :7]).all() and np.isfinite(got[:, 7:, :32]).all() and np.isnan(got[:, 7:, 32:]).all()
    # and a query's NaN stays in its row and head
    c = Case([200], 2, 64, seed=6)
    q[50, 3, 9] = np.nan
    got = run_attention(c, dev(q), [100], out_dtype=torch.bfloat16).float().cpu().numpy()
    assert np.isnan(got[50, 3]).all()
    got[50, 3] = 0
    assert np.isfinite(got).all()


def test_rising_scores():
    # each key above those before it: the running maximum is found again and again
    n = 600
    c = Case([n], 1, 64, seed=4)
    k = np.stack([np.full((1, 64), i / n * 8.0, np.float32) for i in range(n)])
    v = np.random.default_rng(0).normal(0, 1, (n, 1, 64)).astype(np.float32)
    c.write(k, v, c.slots[0])
    q = np.ones((60, 8, 64), np.float32) * np.linspace(-8, 8, 8, dtype=np.float32)[None, :, None]
    check(c, [60], 8, q=dev(q))


@pytest.mark.parametrize("std", [1e-3, 300.0])
def test_small_and_large_values(std):
    check(Case([300], 2, 128, seed=3, v_std=std), [64], 8, out_dtype=torch.bfloat16)


def test_large_queries():
    check(Case([300], 2, 64, seed=3), [64], 8, q_std=1e5, out_dtype=torch.bfloat16)
    check(Case([300], 2, 64, seed=3), [64], 8, q_std=1e-12, out_dtype=torch.bfloat16)


def test_strided_queries_and_outputs():
    c = Case([150, 300], 2, 64, seed=7)
    wide = dev(np.random.default_rng(3).normal(0, 1, (200, 1000)).astype(np.float32))
    q = wide[:, 3:3 + 896].unflatten(1, (14, 64))
    for off in (5, 8):  # unaligned and aligned rows of the output
        store = torch.zeros((200, 1000), device="cuda", dtype=torch.bfloat16)
        out = store[:, off:off + 896].unflatten(1, (14, 64))
        run_attention(c, q, [80, 120], out=out)
        assert torch.equal(out, run_attention(c, q.contiguous(), [80, 120], out_dtype=torch.bfloat16))
        assert not store[:, :off].any() and not store[:, off + 896:].any()


def test_bad_blocks_and_lengths_are_reported():
    c = Case([250, 240], 2, 64, seed=9)
    q = dev(np.random.default_rng(4).normal(0, 1, (200, 8, 64)).astype(np.float32))
    clean = run_attention(c, q, [100, 100], out_dtype=torch.float16)
    keep = c.table[0, 3]
    for wrong in (-1, c.pages.shape[0], 2 ** 31 - 1):
        c.table[0, 3] = wrong
        got = run_attention(c, q, [100, 100], out_dtype=torch.float16)
        assert "paged cache" in status()
        assert torch.isnan(got[:100]).all() and torch.equal(got[100:], clean[100:])
    c.table[0, 3] = keep
    for ctx in ([250, 241], [-1, 241]):  # beyond their bound, before any token
        got = run_attention(c, q, [100, 100], out_dtype=torch.float16, ctx=ctx, max_ctx=240)
        assert "paged cache" in status() and not got.any()
    out = torch.full_like(clean, 3.0)  # more queries than max_q
    kv4.attention(q, c.pages, i32(c.table), i32([0, 100, 200]), i32(c.lens), 99, 250, out=out)
    assert "paged cache" in status() and (out == 3.0).all()


def test_equal_calls_another_stream_and_graphs():
    c = Case([1500, 90, 40], 2, 128, seed=10)
    new = [200, 40, 1]
    rng = np.random.default_rng(5)
    qs = [dev(rng.normal(0, 1, (241, 16, 128)).astype(np.float32)) for _ in range(3)]
    want = [run_attention(c, q, new, out_dtype=torch.bfloat16) for q in qs]
    for q, w in zip(qs, want):
        assert torch.equal(run_attention(c, q, new, out_dtype=torch.bfloat16), w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(run_attention(c, qs[0], new, out_dtype=torch.bfloat16), want[0])
    torch.cuda.current_stream().wait_stream(side)
    q, out = qs[0].clone(), torch.empty_like(want[0])
    args = (i32(c.table), i32(np.concatenate([[0], np.cumsum(new)])), i32(c.lens))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            kv4.attention(q, c.pages, *args, 200, 1500, out=out)
        graphs.append(g)
    for i in range(6):
        q.copy_(qs[i % 3])
        out.zero_()
        graphs[i % 2].replay()
        assert torch.equal(out, want[i % 3])


@pytest.mark.parametrize("S,at", [(700, 350), (2000, 1999), (33, 0)])
def test_a_long_chunk_among_many_short_sequences(S, at):
    rng = np.random.default_rng(S)
    lens, new = rng.integers(1, 40, S).tolist(), [1] * S
    lens[at], new[at] = 300, 70
    if S > at + 2:
        lens[at + 2], new[at + 2] = 64, 12  # 96 rows: the least that is a chunk
    c = Case(lens, 1, 64, seed=S)
    check(c, new, 8)


def test_no_tokens_and_no_heads():
    c = Case([20], 2, 64, seed=1)
    n = i32([])
    none = torch.empty((0, 8, 64), device="cuda")
    f = kv4.rope_frequencies(64, 1e4)
    assert kv4.append(none, none[:, :2], none[:, :2], f, n, n, c.pages).shape == (0, 8, 64)
    assert kv4.read(c.pages, n)[0].shape == (0, 2, 64)
    assert kv4.attention(none, c.pages, i32(c.table), i32([0, 0]), i32([20]), 1, 20, out_dtype=torch.float16).shape == (0, 8, 64)
    q = torch.ones((3, 8, 64), device="cuda")
    out = torch.full((3, 8, 64), 2.0, device="cuda")
    kv4.attention(q, c.pages, i32(np.zeros((0, 2))), i32([0]), n, 1, 20, out=out)  # no sequences
    assert (out == 2.0).all()
    headless = torch.zeros((4, 0, 1280), dtype=torch.uint8, device="cuda")
    for call in (lambda: kv4.read(headless, n), lambda: kv4.attention(q, headless, i32(c.table), i32([0, 3]), i32([20]), 3, 20),
                 lambda: kv4.append(q, q[:, :0], q[:, :0], f, n, n, headless)):
        with pytest.raises(ConfigError):
            call()


def test_sizes_beyond_32_bits_are_refused():
    c = Case([20], 2, 64, seed=1)
    L, h = _lib.lib(), Context.for_device("cuda:0").handle
    p, f = c.pages.data_ptr(), torch.zeros((1, 8, 64), device="cuda").data_ptr()
    z = torch.zeros(64, dtype=torch.int32, device="cuda").data_ptr()
    att = [h, f, 0, 512, 1, 8, 2, 64, 0.1, z, z, 1, z, 2, 1, 20, p, 4, f, 0, 512, None]
    for at, value in [(4, 2 ** 31 // 8), (13, 2 ** 26), (15, 33)]:  # T * heads, blocks of the table, max_ctx
        bad = list(att)
        bad[at] = value
        assert L.rtd_attention_kv4(*bad) == _lib.RTD_ERR_SHAPE, (at, value)
