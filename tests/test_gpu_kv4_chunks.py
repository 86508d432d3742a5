"""rtd_attention_kv4: the edge cases of prompt chunks at sizes where the chunk kernel takes them
(4096 rows of queries x heads in all at head_dim 128, 6144 at 64), and on both sides of that
bound.  Oracle and bounds are test_gpu_kv4_wide.py's.
"""
import numpy as np
import pytest
import torch

from runtimed_b200 import kv4
from test_gpu_kv4 import Case, clean_status, dev, i32, run_attention, status  # noqa: F401
from test_gpu_kv4_wide import check, expected

pytestmark = pytest.mark.gpu

H, N_KV = 64, 8
ROWS = {64: 6144, 128: 4096}


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("less", [1, 0])
def test_both_sides_of_the_bound(D, less):
    n = ROWS[D] // H - less
    check(Case([n + 37, 50], N_KV, D, seed=n), [n, 1], H)
    # short of the bound by the decoding sequence's rows, which do not count
    check(Case([n + 37] + [9] * 40, N_KV, D, seed=n), [n] + [1] * 40, H)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("ctx,n", [(1, 300), (17, 130), (63, 63), (64, 64), (65, 65), (96, 33), (127, 50), (128, 12), (333, 129), (334, 65)])
def test_every_key_counts_once(D, ctx, n):
    # Scores near zero, and key i's value is 1 at dim i % D alone (15 steps of f16(1 / 15)):
    # a missing or doubled key changes that dim by a sixth at least, against a bound of 1 %.
    copies = -(-ROWS[D] // (n * H))
    c = Case([ctx] * copies, N_KV, D, seed=ctx, k_std=0.05, bias=0.0)
    v = np.zeros((ctx, N_KV, D), np.float32)
    v[np.arange(ctx), :, np.arange(ctx) % D] = 1
    c.write(np.concatenate(c.K).astype(np.float32), np.tile(v, (copies, 1, 1)), np.concatenate(c.slots))
    check(c, [n] * copies, H, q_std=0.05)


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("q_dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_types(out_dtype, q_dtype):
    check(Case([400, 90], N_KV, 64, seed=5), [120, 3], H, out_dtype=out_dtype, q_dtype=q_dtype)


def test_rows_that_see_nothing_and_rows_of_no_sequence():
    c = Case([20, 0, 40], N_KV, 64, seed=1)
    new = [90, 30, 0]  # 70 queries before the sequence's start, a chunk of an empty sequence
    q = dev(np.random.default_rng(2).normal(0, 1, (125, H, 64)).astype(np.float32))
    out = torch.full((125, H, 64), 7.0, device="cuda", dtype=torch.float16)
    got = kv4.attention(q, c.pages, i32(c.table), i32([0, 90, 120, 120]), i32(c.lens), 90, 40, out=out)
    want, tol = expected(c, q[:120].double().cpu().numpy(), new, torch.float16)
    assert np.all(np.abs(got[:120].double().cpu().numpy() - want) <= tol)
    assert not got[:70].any() and not got[90:120].any() and (got[120:] == 7.0).all()


def test_nan_keys_values_and_queries():
    # keys 130 (K, kv head 0) and 135 (V, kv head 1, the second group) hold a NaN group
    def case(k=None, v=None):
        c = Case([200], N_KV, 64, seed=6)
        kk, vv = c.K[0].astype(np.float32), c.V[0].astype(np.float32)
        for x, at in ((kk, k), (vv, v)):
            if at is not None:
                x[at] = np.nan
        c.write(kk, vv, c.slots[0])
        return c

    q = np.random.default_rng(1).normal(0, 1, (100, H, 64)).astype(np.float32)  # positions 100 .. 199
    run = lambda c: run_attention(c, dev(q), [100], out_dtype=torch.bfloat16).float().cpu().numpy()  # noqa: E731
    got = run(case((130, 0, 3), (135, 1, 40)))
    assert np.isfinite(got[:30]).all() and np.isnan(got[30:, :8]).all()
    assert np.isfinite(got[:35, 8:]).all() and np.isnan(got[35:, 8:16, 32:]).all() and np.isfinite(got[:, 16:]).all()
    got = run(case(v=(20, 1, 40)))  # before the chunk's own tokens: the group alone
    assert np.isnan(got[:, 8:16, 32:]).all() and np.isfinite(got[:, 8:16, :32]).all()
    assert np.isfinite(got[:, :8]).all() and np.isfinite(got[:, 16:]).all()
    q[50, 3, 9] = np.nan  # a query's stays in its row and head
    got = run(case())
    assert np.isnan(got[50, 3]).all()
    got[50, 3] = 0
    assert np.isfinite(got).all()


def test_rising_scores():
    # each key above those before it: the running maximum is found again and again
    n = 600
    c = Case([n], N_KV, 64, seed=4)
    k = np.stack([np.full((N_KV, 64), i / n * 8.0, np.float32) for i in range(n)])
    c.write(k, np.random.default_rng(0).normal(0, 1, (n, N_KV, 64)).astype(np.float32), c.slots[0])
    q = np.ones((100, H, 64), np.float32) * np.linspace(-8, 8, H, dtype=np.float32)[None, :, None]
    check(c, [100], H, q=dev(q))


@pytest.mark.parametrize("v_std,q_std", [(1e-3, 1.0), (300.0, 1.0), (1.0, 1e5), (1.0, 1e-12)])
def test_small_and_large_values(v_std, q_std):
    check(Case([300], N_KV, 128, seed=3, v_std=v_std), [64], H, q_std=q_std, out_dtype=torch.bfloat16)


def test_strided_queries_and_outputs():
    c = Case([150, 300], N_KV, 64, seed=7)
    wide = dev(np.random.default_rng(3).normal(0, 1, (200, 4200)).astype(np.float32))
    q = wide[:, 3:3 + 4096].unflatten(1, (H, 64))
    for off in (5, 8):  # unaligned and aligned rows of the output
        store = torch.zeros((200, 4200), device="cuda", dtype=torch.bfloat16)
        out = store[:, off:off + 4096].unflatten(1, (H, 64))
        run_attention(c, q, [80, 120], out=out)
        assert torch.equal(out, run_attention(c, q.contiguous(), [80, 120], out_dtype=torch.bfloat16))
        assert not store[:, :off].any() and not store[:, off + 4096:].any()


def test_bad_blocks_and_lengths_are_reported():
    c = Case([250, 240], N_KV, 64, seed=9)
    q = dev(np.random.default_rng(4).normal(0, 1, (200, H, 64)).astype(np.float32))
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
    c = Case([1500, 90, 40], N_KV, 128, seed=10)
    new = [200, 40, 1]
    rng = np.random.default_rng(5)
    qs = [dev(rng.normal(0, 1, (241, H, 128)).astype(np.float32)) for _ in range(3)]
    want = [run_attention(c, q, new, out_dtype=torch.bfloat16) for q in qs]
    for q, w in zip(qs, want):
        assert torch.equal(run_attention(c, q, new, out_dtype=torch.bfloat16), w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(run_attention(c, qs[0], new, out_dtype=torch.bfloat16), want[0])
    torch.cuda.current_stream().wait_stream(side)
    q, out = qs[0].clone(), torch.empty_like(want[0])
    starts, lens, table = i32(np.concatenate([[0], np.cumsum(new)])), i32(c.lens), i32(c.table)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            kv4.attention(q, c.pages, table, starts, lens, 241, 1500, out=out)
        graphs.append(g)
    for i in range(6):
        q.copy_(qs[i % 3])
        out.zero_()
        graphs[i % 2].replay()
        assert torch.equal(out, want[i % 3])
    # the same graph with other lengths: no chunk is left, the decoding sequences stay
    starts.copy_(i32([0, 1, 2, 3]))
    out.zero_()
    graphs[0].replay()
    alone = kv4.attention(q[:3], c.pages, table, starts, lens, 1, 1500, out_dtype=torch.bfloat16)
    assert torch.allclose(out[:3].float(), alone.float(), rtol=2 ** -6, atol=2 ** -8) and not out[3:].any()


@pytest.mark.parametrize("S,at", [(700, 350), (2000, 1999), (33, 0)])
def test_a_long_chunk_among_many_short_sequences(S, at):
    rng = np.random.default_rng(S)
    lens, new = rng.integers(1, 40, S).tolist(), [1] * S
    lens[at], new[at] = 300, 100
    if S > at + 2:
        lens[at + 2], new[at + 2] = 64, 12  # 96 rows: the least that is a chunk
    check(Case(lens, N_KV, 64, seed=S), new, H)
