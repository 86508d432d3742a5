"""rtd_attention_kv4: calls of one context that ran at the same time, which is not allowed and
spoils their outputs, leave nothing behind that later calls trip over.  (Nothing in the kernel
waits for another CTA and every index comes from the call's own lengths.)"""
import numpy as np
import pytest
import torch

from test_gpu_kv4 import Case, clean_status, dev, run_attention  # noqa: F401

pytestmark = pytest.mark.gpu


def test_later_calls_are_right():
    # two shapes whose shared units span different CTAs
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
