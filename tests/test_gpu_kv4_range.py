"""rtd_attention_kv4: prompt chunks with 16-bit outputs whose keys or values have no place in the
chunk kernel's f16 tiles (beyond 65504, NaN that only some rows see), against 64 bits.
"""
import math

import numpy as np
import pytest
import torch

from runtimed_b200 import kv4
from test_gpu_kv4 import Case, clean_status, dev, i32, run_attention  # noqa: F401

pytestmark = pytest.mark.gpu

H, N_KV, N = 64, 8, 100  # 6400 rows, all of them a chunk's
CTX = 200                # positions 100 .. 199 are the call's own


def case(D, k=None, v=None, value=1e5, seed=6):
    c = Case([CTX], N_KV, D, seed=seed)
    kk, vv = c.K[0].astype(np.float32), c.V[0].astype(np.float32)
    for x, at in ((kk, k), (vv, v)):
        if at is not None:
            x[at] = value
    c.write(kk, vv, c.slots[0])
    return c


def close(c, q, got, out_dtype):
    """f16 outputs by the bound on exact ones and their own rounding; bf16's by 11-bit queries
    and weights and their own rounding, each 2^-9 at most, over a row and head."""
    want, tol = c.want(q.astype(np.float64), [N], 1 / math.sqrt(c.D))
    err = np.abs(got.double().cpu().numpy() - want)
    if out_dtype == torch.float16:
        tol = tol + np.abs(want) * 2.0 ** -11 + 2.0 ** -25
        assert np.all(err <= tol), (err.max(), np.argwhere(err > tol)[:5])
    else:
        rel = np.linalg.norm(err, axis=-1) / np.linalg.norm(want, axis=-1)
        assert rel.max() <= 2.0 ** -7, rel.max()


@pytest.mark.parametrize("out_dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
def test_values_beyond_f16(D, out_dtype):
    # one of the call's own tokens, and one before them
    q = np.random.default_rng(1).normal(0, 1, (N, H, D)).astype(np.float32)
    for at in (135, 20):
        c = case(D, v=(at, 1, 40))
        assert np.abs(c.V[0]).max() > 65504 and np.isfinite(c.V[0]).all()
        close(c, q, run_attention(c, dev(q), [N], out_dtype=out_dtype), out_dtype)


@pytest.mark.parametrize("out_dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
def test_keys_beyond_f16(D, out_dtype):
    q = np.random.default_rng(1).normal(0, 1e-4, (N, H, D)).astype(np.float32)
    for at in (130, 20):
        c = case(D, k=(at, 0, 3))
        assert np.abs(c.K[0]).max() > 65504
        close(c, q, run_attention(c, dev(q), [N], out_dtype=out_dtype), out_dtype)


@pytest.mark.parametrize("D", [64, 128])
def test_nan_reaches_its_group_of_the_rows_that_see_it(D):
    q = np.random.default_rng(1).normal(0, 1, (N, H, D)).astype(np.float32)
    for out_dtype in (torch.float16, torch.bfloat16):
        got = run_attention(case(D, v=(135, 1, 40), value=np.nan), dev(q), [N], out_dtype=out_dtype).float().cpu().numpy()
        bad = np.zeros(got.shape, bool)
        bad[35:, 8:16, 32:64] = True
        assert np.array_equal(np.isnan(got), bad)


@pytest.mark.parametrize("D", [64, 128])
def test_other_chunks_and_later_calls_are_as_ever(D):
    # a sequence beyond f16 beside one within it, and a graph whose pages come and go
    c = Case([CTX, CTX], N_KV, D, seed=6)
    kv = [np.concatenate(x).astype(np.float32) for x in (c.K, c.V)]
    slots = np.concatenate(c.slots)
    c.write(*kv, slots)
    q = dev(np.random.default_rng(2).normal(0, 1, (2 * N, H, D)).astype(np.float32))
    clean = run_attention(c, q, [N, N], out_dtype=torch.bfloat16)
    out = torch.empty_like(clean)
    args = (i32(c.table), i32([0, N, 2 * N]), i32(c.lens))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kv4.attention(q, c.pages, *args, N, CTX, out=out)
    for _ in range(2):
        large = kv[1].copy()
        large[135, 1, 40] = 1e5  # sequence 0, kv head 1
        c.write(kv[0], large, slots)
        assert torch.equal(run_attention(c, q, [N, N], out_dtype=torch.bfloat16)[N:], clean[N:])
        out.zero_()
        g.replay()
        assert out.isfinite().all() and torch.equal(out[N:], clean[N:]) and not torch.equal(out[:N], clean[:N])
        c.write(*kv, slots)
        out.zero_()
        g.replay()
        assert torch.equal(out, clean)
        assert torch.equal(run_attention(c, q, [N, N], out_dtype=torch.bfloat16), clean)


@pytest.mark.parametrize("D", [64, 128])
def test_outputs_over_the_queries(D):
    q = np.random.default_rng(3).normal(0, 1, (N, H, D)).astype(np.float32)
    for c in (case(D), case(D, v=(135, 1, 40))):
        for dt in (torch.float16, torch.bfloat16):
            x = dev(q).to(dt)
            rows = x.float().cpu().numpy()
            close(c, rows, run_attention(c, x, [N], out=x), dt)


@pytest.mark.parametrize("D,low,high", [(64, 60000, 1e6), (128, -65000, 9e5), (32, 0, 65504 * 15), (96, 65504, 65504 * 16)])
def test_groups_whose_middle_is_beyond_f16(D, low, high):
    # step and minimum are f16, minimum + 8 steps is not: read with a 16th of the middle
    c = Case([70, 20], 2, D, seed=D)
    v = np.concatenate(c.V).astype(np.float32)
    v[33, 1, :32] = np.linspace(low, high, 32)
    c.write(np.concatenate(c.K).astype(np.float32), v, np.concatenate(c.slots))
    assert np.isfinite(c.V[0]).all() and c.V[0].max() > 8e5
    q = np.random.default_rng(4).normal(0, 1, (5, 8, D)).astype(np.float32)
    got = run_attention(c, dev(q), [4, 1]).cpu().numpy()
    want, tol = c.want(q.astype(np.float64), [4, 1], 1 / math.sqrt(D))
    assert np.all(np.abs(got - want) <= tol)
