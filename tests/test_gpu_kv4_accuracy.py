"""How near rtd_attention_kv4 comes to 64 bits: relative L2 errors over each sequence's rows, so
that lost low halves of queries or weights, a drift with the length or a grid that small values
meet are seen, at every head layout and output type.

f32 outputs.  Relative to the result, with weights of like size and unit values: scores of a few
bits in 32-bit sums of 2 NG terms (2^-24 of about 4 each, NG at most 4: 3e-7), the exponential
(2^-22 at most, 1e-7 on average), p d in 22 bits (1e-7), one 32-bit addition a page to a sum that
grows like the result (2^-25 sqrt(pages / 3): 2e-7 at 1000 tokens, 6e-7 at 20000); as
independent errors 4e-7 and 8e-7.  Allowed are 1e-6 up to 1000 tokens and 1.6e-6 beyond.
f16 outputs: those, and half a step of f16 a value.  bf16 outputs: queries and weights of 11
bits (2^-12 on average a score of 4 bits: 7e-4 of a weight; the weights' own 2e-4), half a step
of bf16 (2^-9 at most, 1.7e-3 over a binade): 1.9e-3 together; 2.6e-3 are allowed.
"""
import math

import numpy as np
import pytest
import torch

from test_gpu_kv4 import HEADS, Case, clean_status, dev, run_attention  # noqa: F401

pytestmark = pytest.mark.gpu


def wanted(c, q, new):
    """Rows in 64 bits of q f64 [T, H, D], sequence by sequence."""
    H, at, out = q.shape[1], 0, []
    G = H // c.n_kv
    for s, n in enumerate(new):
        K, V, ctx = c.K[s], c.V[s], c.lens[s]
        hidden = np.arange(ctx)[None] > ctx - n + np.arange(n)[:, None]
        rows = np.zeros((n, H, c.D))
        for h in range(H):
            x = q[at:at + n, h] @ K[:, h // G].T / math.sqrt(c.D)
            x[hidden] = -np.inf
            w = np.exp(x - x.max(1, keepdims=True))
            rows[:, h] = (w / w.sum(1, keepdims=True)) @ V[:, h // G]
        out.append(rows)
        at += n
    return out


def rel(err, want):
    return np.linalg.norm(err) / np.linalg.norm(want)


def check(c, new, H, out_dtype=torch.float32, q_std=1.0):
    q = np.random.default_rng(sum(c.lens)).normal(0, q_std, (sum(new), H, c.D)).astype(np.float32)
    got = run_attention(c, dev(q), new, out_dtype=out_dtype).double().cpu().numpy()
    at = 0
    for s, want in enumerate(wanted(c, q.astype(np.float64), new)):
        err = got[at:at + new[s]] - want
        at += new[s]
        limit = 1e-6 if c.lens[s] <= 1000 else 1.6e-6
        if out_dtype == torch.bfloat16:
            limit = 2.6e-3
        elif out_dtype == torch.float16:  # what half a step (2^-25 among subnormals) leaves
            err = np.maximum(0, np.abs(err) - np.abs(want) * 2.0 ** -11 - 2.0 ** -25)
        assert rel(err, want) <= limit, (s, rel(err, want), limit)


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,n_kv,D", HEADS)
@pytest.mark.parametrize("lens,new", [([160, 17], [1, 1]), ([700, 33], [5, 2]), ([900], [12]), ([3000, 40, 640], [1, 1, 1])])
def test_against_64_bits(H, n_kv, D, lens, new, out_dtype):
    check(Case(lens, n_kv, D, seed=D + len(lens)), new, H, out_dtype)


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [13376, 20011])
def test_long_contexts(n, out_dtype):
    check(Case([n, 700], 2, 128, seed=n), [1, 1], 16, out_dtype)


@pytest.mark.parametrize("H,n_kv,D", HEADS)
@pytest.mark.parametrize("v_std", [1e-2, 1e-3, 1e-4, 100.0])
def test_small_and_large_values(H, n_kv, D, v_std):
    check(Case([500, 77], n_kv, D, seed=3, v_std=v_std), [1, 2], H)


@pytest.mark.parametrize("first", [0.0, 1e-4, 1e-2])
def test_values_that_grow_after_the_first_pages(first):
    # the first 64 tokens hold small values (or none), the others ordinary and large ones
    c = Case([500], 2, 64, seed=9)
    v = c.V[0].astype(np.float32)
    v[:64] *= first
    v[300:] *= 30
    c.write(c.K[0].astype(np.float32), v, c.slots[0])
    check(c, [2], 8)


@pytest.mark.parametrize("out_dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,new", [([4000], [130]), ([9000, 2500], [40, 70]), ([300] * 8, [12] * 8), ([700] * 12, [8] * 12)])
def test_prompt_chunks(D, lens, new, out_dtype):
    # Queries, keys, weights and values of f16's 11 bits, 2e-4 each on average: with keys about one,
    # not zero, a score's two count 3e-4 each, 5e-4 in all, beside half a step of the output.
    # f16 outputs of the other kernel (12 x 8 queries of 8 heads a group) come closer.
    c = Case(lens, 8, D, seed=len(lens) + D)
    q = np.random.default_rng(1).normal(0, 1, (sum(new), 64, D)).astype(np.float32)
    got = run_attention(c, dev(q), new, out_dtype=out_dtype).double().cpu().numpy()
    limit = 8e-4 if out_dtype == torch.float16 else 2.6e-3
    at = 0
    for s, want in enumerate(wanted(c, q.astype(np.float64), new)):
        assert rel(got[at:at + new[s]] - want, want) <= limit, (s, rel(got[at:at + new[s]] - want, want))
        at += new[s]


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,n_kv,D", HEADS)
@pytest.mark.parametrize("what,v_std", [(np.nan, 1e-4), (np.nan, 1.0), (1e5, 1e-2), ("grown", 1e-3), ("grown", 1.0)])
def test_what_is_read_twice_loses_no_accuracy(H, n_kv, D, what, v_std, out_dtype):
    # a NaN, a value beyond f16, or values 1e5 times those of a warp's first page
    c = Case([700], n_kv, D, seed=3, v_std=v_std)
    v = c.V[0].astype(np.float32)
    if what == "grown":
        v[:80] *= 1e-5
    else:
        v[400, 0, D - 1] = what
    c.write(c.K[0].astype(np.float32), v, c.slots[0])
    q = np.random.default_rng(1).normal(0, 1, (2, H, D)).astype(np.float32)
    got = run_attention(c, dev(q), [2], out_dtype=out_dtype).double().cpu().numpy().reshape(2, H, D // 32, 32)
    want = wanted(c, q.astype(np.float64), [2])[0].reshape(got.shape)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    limit = {torch.float32: 1e-6, torch.float16: 1e-6, torch.bfloat16: 2.6e-3}[out_dtype]
    for g in range(D // 32):
        for h in range(n_kv):
            at = np.s_[:, h * (H // n_kv):(h + 1) * (H // n_kv), g]
            if np.isnan(want[at]).any():
                continue
            err = got[at] - want[at]
            if out_dtype == torch.float16:
                err = np.maximum(0, np.abs(err) - np.abs(want[at]) * 2.0 ** -11 - 2.0 ** -25)
            assert rel(err, want[at]) <= limit, (g, h, rel(err, want[at]))


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,n_kv,D", HEADS)
@pytest.mark.parametrize("small,large,nan", [(1e-4, 1e3, None), (1e-3, 1e5, None), (1e-4, 1.0, 37), (1.0, 1e5, 30)])
def test_large_values_of_keys_not_seen_yet(H, n_kv, D, small, large, nan, out_dtype):
    # row by row: those before token 21 see small values alone, the others of its page are large
    c = Case([40], n_kv, D, seed=5, v_std=1.0)
    v = c.V[0].astype(np.float32)
    v[:21] *= small
    v[21:] *= large / 4
    v[21:] = np.clip(v[21:], -60000, None)
    if nan is not None:
        v[nan, 0, 3] = np.nan
    c.write(c.K[0].astype(np.float32), v, c.slots[0])
    q = np.random.default_rng(2).normal(0, 1, (40, H, D)).astype(np.float32)
    got = run_attention(c, dev(q), [40], out_dtype=out_dtype).double().cpu().numpy()
    want = np.zeros(got.shape)
    for i in range(40):
        for h in range(H):
            x = q[i, h].astype(np.float64) @ c.K[0][:i + 1, h * n_kv // H].T / math.sqrt(D)
            w = np.exp(x - x.max())
            want[i, h] = (w / w.sum()) @ c.V[0][:i + 1, h * n_kv // H]
    assert np.array_equal(np.isnan(got), np.isnan(want))
    # Eight rows (token * G + head) are read together.  Where 8 divides G they see the same keys, and
    # each is as near as alone; elsewhere, as with G = 20, rows 416 .. 423 belong to tokens 20 and 21,
    # and what f16 pairs hold beside values 1e8 times as large is all that remains of the first.
    if H // n_kv % 8 == 0:
        limit = 2e-6 if out_dtype == torch.float32 else 8e-3
        ok = ~np.isnan(want).any(axis=(1, 2))
        err = np.linalg.norm((got - want)[ok], axis=(1, 2)) / np.linalg.norm(want[ok], axis=(1, 2))
        assert err.max() <= limit, (err.argmax(), err.max())
