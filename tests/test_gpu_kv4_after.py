"""What spoiled and refused calls leave behind: nothing that later calls trip over."""
import numpy as np
import pytest
import torch

from test_gpu_kv4 import Case, clean_status, dev, run_attention  # noqa: F401

pytestmark = pytest.mark.gpu


def test_calls_after_overlapping_ones():
    # Calls of one context at the same time are not allowed and spoil their outputs; nothing in the
    # kernel waits for another CTA, and every index comes from the call's own lengths.  Two shapes,
    # whose shared units span different CTAs.
    cases = [(Case([3000, 40, 3000], 2, 64, seed=1), [1, 1, 1], 8), (Case([5000, 700], 4, 128, seed=2), [3, 1], 32)]
    qs = [dev(np.random.default_rng(i).normal(0, 1, (sum(new), H, c.D)).astype(np.float32)) for i, (c, new, H) in enumerate(cases)]
    want = [run_attention(c, q, new) for (c, new, _), q in zip(cases, qs)]
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, st in enumerate(streams):
            c, new, _ = cases[i % 2]
            with torch.cuda.stream(st):
                for _ in range(3):
                    run_attention(c, qs[i % 2], new)
        torch.cuda.synchronize()
        for (c, new, _), q, w in zip(cases, qs, want):
            assert torch.equal(run_attention(c, q, new), w)
        torch.cuda.synchronize()


def test_refused_plans_keep_no_reference():
    import sys

    from runtimed_b200 import kv4
    from runtimed_b200.errors import ShapeError

    t = kv4.BlockTables(3, 2, 5, 4)
    out = (t.q_start, t.tok_seq, t.tok_pos, t.tok_slot)
    before = sys.getrefcount(out)
    for _ in range(10):
        try:
            kv4.plan(t.length[:2], t.length, t.table, t.free_list, t.free_count, out=out)
            raise AssertionError("not refused")
        except ShapeError:
            pass
    assert kv4.plan(t.length, t.length, t.table, t.free_list, t.free_count, out=out) is out
    assert sys.getrefcount(out) == before
