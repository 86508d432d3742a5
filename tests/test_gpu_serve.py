"""The device-resident decode step on the Qwen2 decoder: the 4-bit KV cache behind the model's
own entry points, block tables on the device and sampling, together as they are used."""
import os
import tempfile

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def rel_l2(got, want):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    return float(np.linalg.norm(got - want) / max(np.linalg.norm(want), 1e-300))


@pytest.fixture(scope="module")
def gguf():
    from runtimed_b200 import fixtures

    with tempfile.TemporaryDirectory(prefix="rtd_serve_") as d:
        path = os.path.join(d, "small.gguf")
        fixtures.write_qwen2_gguf(path, fixtures.small_shape(n_layer=2, vocab=1000), seed=3)
        yield path


def model(path, kv, **kw):
    from runtimed_b200.qwen2 import Qwen2Model

    return Qwen2Model(path, max_seqs=4, max_ctx=256, kv_dtype=kv, exact_linears=True, **kw)


def prompts(*lens, seed=1):
    rng = np.random.default_rng(seed)
    return [list(rng.integers(0, 1000, n)) for n in lens]


def test_pages_hold_the_keys_and_values_of_the_f32_cache(gguf):
    # layer 0 sees the same input in both caches: its values differ by the 4-bit rounding
    p = prompts(50)[0]
    full, q4 = model(gguf, torch.float32), model(gguf, "q4")
    for m in (full, q4):
        m.forward(p, 0, seq=1)
    for want, got in zip(full.cache.values(0, 1), q4.cache.values(0, 1)):
        want, got = want.cpu().numpy(), got.cpu().numpy()
        g = want.reshape(50, want.shape[1], -1, 32)
        step = (g.max(-1) - g.min(-1))[..., None] / 15
        # half a step, the minimum's rounding, the step's over 15 codes; rope's angles are formed
        # in 32 bits for the f32 cache: off by up to 50 * 2^-24 and a few roundings
        bound = step / 2 + np.abs(g).max(-1, keepdims=True) * (2.0 ** -11 + 60 * 2.0 ** -24) + 15 * step * 2.0 ** -11
        assert np.all(np.abs(got.reshape(g.shape) - g) <= bound)
    # and attention through the model uses them: a prompt's logits stay close to the f32 cache's
    assert q4.cache.pages[0].numel() * 16 == full.cache.k[0].numel() * 2 * 4 * 10 // 4


def test_prefill_chunks_and_single_tokens_agree(gguf):
    # the cache quantises a token before any query reads it, so the prompt may come in any cut
    p = prompts(45)[0]
    whole = model(gguf, "q4")
    a = whole.forward(p, 0).cpu().numpy()
    cut = model(gguf, "q4")
    b = np.concatenate([cut.forward(p[i:j], i).cpu().numpy() for i, j in ((0, 17), (17, 18), (18, 40), (40, 45))])
    assert rel_l2(b, a) <= 1e-3
    one = model(gguf, "q4")
    c = np.concatenate([one.forward([t], i).cpu().numpy() for i, t in enumerate(p)])
    assert rel_l2(c, a) <= 1e-3
    # batched decode, a sequence twice in one call: positions 43 and 44 together
    two = model(gguf, "q4")
    two.forward(p[:43], 0, seq=2)
    d = two.decode_batch(p[43:45], [2, 2], [43, 44]).cpu().numpy()
    assert rel_l2(d, a[43:45]) <= 1e-3


def test_graph_and_speculative_decode_on_the_4_bit_cache(gguf):
    from runtimed_b200.qwen2 import Session
    from runtimed_b200.speculate import speculative_generate

    p = prompts(24, seed=4)[0]
    m = model(gguf, "q4")
    ids, _ = Session(m).greedy(p, 40)
    m.cache.release(0)
    out, g, replay = m.greedy_graph(p, 40)
    for _ in range(40):
        replay()
    torch.cuda.synchronize()
    assert out.cpu().tolist() == ids
    del g
    st = speculative_generate(model(gguf, "q4"), m, p, 40, k=4)
    assert st.tokens == ids and st.accepted == st.proposed


@pytest.mark.parametrize("kv", ["q4", torch.float16])
def test_generate_batch_is_the_step_by_step_loop(gguf, kv):
    from runtimed_b200 import sampling

    ps, steps = prompts(5, 33, 16), 40  # sequences cross block borders at different steps
    args = dict(temperature=0.8, top_k=50, top_p=0.9, min_p=0.01, seed=11)
    m = model(gguf, kv)
    got = m.generate_batch(ps, steps, **args).cpu()
    assert torch.equal(got, m.generate_batch(ps, steps, **args).cpu())
    assert torch.equal(got, model(gguf, kv).generate_batch(ps, steps, graph=False, **args).cpu())
    assert not torch.equal(got, m.generate_batch(ps, steps, **{**args, "seed": 12}).cpu())
    # the same by hand: host block tables, decode_batch, sample
    gen = torch.Generator(device="cuda")
    gen.manual_seed(11)
    u = torch.rand((steps, 3), generator=gen, dtype=torch.float32, device="cuda")
    on = lambda v, dt=torch.float32: torch.full((3,), v, dtype=dt, device="cuda")  # noqa: E731
    f = (on(0.8), on(50, torch.int32), on(0.9), on(0.01))
    ref = model(gguf, kv)
    logits = torch.cat([ref.forward(p, 0, seq=s, last_only=True) for s, p in enumerate(ps)])
    ids, pos = [], [len(p) for p in ps]
    for i in range(steps):
        ids.append(sampling.sample(logits, u[i], *f).cpu().tolist())
        if i + 1 < steps:
            logits = ref.decode_batch(ids[-1], [0, 1, 2], [q + i for q in pos])
    assert got.t().tolist() == ids


def test_generate_batch_leaves_the_cache_usable(gguf):
    m = model(gguf, "q4")
    m.forward(prompts(20, seed=9)[0], 0, seq=3)  # a sequence that takes no part
    kept = [x.cpu().numpy() for x in m.cache.values(1, 3)]
    ps = prompts(5, 33)
    got = m.generate_batch(ps, 30, temperature=0.0).cpu()
    assert m.cache.lengths == {0: 34, 1: 62, 3: 20}
    held = [b for s in (0, 1, 3) for b in m.cache._blocks[s]]
    assert sorted(held + m.cache._free) == list(range(m.cache.num_blocks))
    for a, b in zip(kept, m.cache.values(1, 3)):
        assert np.array_equal(a, b.cpu().numpy())
    # going on by hand gives what a fresh model gives for the whole text
    tail = m.decode_batch(got[:, -1].tolist(), [0, 1], [34, 62]).cpu().numpy()
    fresh = model(gguf, "q4")
    for s, p in enumerate(ps):
        want = fresh.forward(p + got[s].tolist(), 0, seq=s)[-1].cpu().numpy()
        assert rel_l2(tail[s], want) <= 1e-3
    # and temperature 0 is the greedy decode
    from runtimed_b200.qwen2 import Session

    assert got[0].tolist() == Session(fresh).greedy(ps[0], 30)[0]


def test_generate_batch_refuses_what_does_not_fit(gguf):
    from runtimed_b200.errors import ConfigError

    m = model(gguf, "q4", kv_blocks=6)
    for bad in (dict(prompts=prompts(5, 5, 5, 5, 5), steps=2), dict(prompts=[[]], steps=2), dict(prompts=prompts(5), steps=0),
                dict(prompts=prompts(90), steps=20), dict(prompts=prompts(250), steps=20)):
        with pytest.raises(ConfigError):
            m.generate_batch(**bad)
    assert m.generate_batch(prompts(5), 2).shape == (1, 2)


def test_a_step_without_free_blocks_is_reported(gguf):
    from runtimed_b200 import kv4
    from runtimed_b200.errors import ConfigError
    from runtimed_b200.weights import Context

    m = model(gguf, "q4", kv_blocks=4)
    m.forward(prompts(32)[0], 0, seq=0)
    m.forward(prompts(32)[0], 0, seq=1)
    t = kv4.BlockTables.from_cache(m.cache, 4)
    t.step(t.length + 1)  # two more blocks are wanted (and two for empty sequences), none is free
    with pytest.raises(ConfigError, match="paged cache"):
        Context.for_device("cuda:0").check_device_status()
    assert (t.tok_seq == -1).all() and t.length.tolist() == [32, 32, 0, 0]
    t.set_lengths(torch.tensor([32, 0, 0, 0], dtype=torch.int32, device="cuda"))
    t.step(torch.tensor([33, 0, 0, 1], dtype=torch.int32, device="cuda"))
    assert t.tok_seq.tolist() == [0, 3, -1, -1] and t.q_start.tolist() == [0, 1, 1, 1, 2]
    t.into(m.cache)
    assert m.cache.lengths == {0: 33, 3: 1} and len(m.cache._free) == 0
    Context.for_device("cuda:0").check_device_status()


@pytest.mark.parametrize("kv", [torch.float16, torch.float32])
def test_padded_rows_of_a_plan_leave_the_16_and_32_bit_caches_alone(kv):
    # rtd_kv_plan pads its lists with -1 (all of them when it refuses): such a row appends nothing
    # and its attention is zero, whichever cache the step runs on
    from runtimed_b200 import _lib, kv4
    from runtimed_b200.errors import ConfigError
    from runtimed_b200.weights import Context

    L, h, abi = _lib.lib(), Context.for_device("cuda:0"), _lib.DT_F16 if kv == torch.float16 else _lib.DT_F32
    st = torch.cuda.current_stream().cuda_stream
    rng = np.random.default_rng(0)
    T, H, G, D = 6, 4, 2, 64
    x = [torch.from_numpy(rng.normal(0, 1, (T, n * D)).astype(np.float32)).cuda() for n in (H, G, G)]

    def run(t, T, max_ctx=32):
        cache = [torch.full((5, G, 16, D), 3.0, dtype=kv, device="cuda") for _ in range(2)]
        q, o = (torch.full((T, H * D), 9.0, device="cuda") for _ in range(2))
        assert L.rtd_rope_kv_append(h.handle, x[0].data_ptr(), H * D, x[1].data_ptr(), G * D, x[2].data_ptr(), G * D, T, H, G, D, D,
                                    1e4, t.tok_seq.data_ptr(), t.tok_pos.data_ptr(), t.table.data_ptr(), 2, cache[0].data_ptr(),
                                    cache[1].data_ptr(), abi, q.data_ptr(), st) == 0
        assert L.rtd_attention_paged(h.handle, q.data_ptr(), T, H, G, D, 0.125, t.tok_seq.data_ptr(), t.tok_pos.data_ptr(),
                                     t.table.data_ptr(), 2, max_ctx, cache[0].data_ptr(), cache[1].data_ptr(), abi, o.data_ptr(),
                                     _lib.DT_F32, H * D, st) == 0
        return cache, o

    def tables(max_tokens):
        t = kv4.BlockTables(3, 2, 5, max_tokens)
        t.step(torch.tensor([2, 0, 1], dtype=torch.int32, device="cuda"))
        return t

    padded, whole = tables(T), tables(3)
    assert padded.tok_seq.tolist() == [0, 0, 2, -1, -1, -1]
    (cache, o), (want, o3) = run(padded, T), run(whole, 3)
    for a, b in zip(cache, want):
        assert torch.equal(a, b)
        assert (a != 3.0).any() and (a == 3.0).sum() == a.numel() - 3 * G * D  # three tokens, and nothing else
    assert torch.equal(o[:3], o3) and not o[3:].any()
    padded.step(torch.tensor([33, 0, 1], dtype=torch.int32, device="cuda"))  # more than the table holds: refused
    with pytest.raises(ConfigError, match="paged cache"):
        h.check_device_status()
    assert (padded.tok_seq == -1).all()
    cache, o = run(padded, T)
    assert all((c == 3.0).all() for c in cache) and not o.any()


@pytest.mark.parametrize("kv", ["q4", torch.float16])
@pytest.mark.parametrize("graph", [True, False])
def test_generate_batch_raises_what_a_step_reported(gguf, kv, graph, monkeypatch):
    # a free stack that is empty on the device: the second step wants a block for each sequence
    from runtimed_b200 import kv4
    from runtimed_b200.errors import ConfigError

    take_over = kv4.BlockTables.from_cache.__func__

    def none_free(cls, cache, max_tokens):
        t = take_over(cls, cache, max_tokens)
        t.free_count.zero_()
        return t

    m = model(gguf, kv)
    monkeypatch.setattr(kv4.BlockTables, "from_cache", classmethod(none_free))
    with pytest.raises(ConfigError, match="paged cache"):
        m.generate_batch(prompts(16, 32), 3, graph=graph)
    assert m.cache.lengths == {0: 16, 1: 32}
    monkeypatch.undo()
    m.ctx.check_device_status()  # told once
    fresh = model(gguf, kv)
    assert torch.equal(fresh.generate_batch(prompts(16, 32), 3, graph=graph), model(gguf, kv).generate_batch(prompts(16, 32), 3))


def test_a_refused_generate_batch_leaves_its_sequences(gguf):
    from runtimed_b200.errors import ConfigError

    m = model(gguf, "q4", kv_blocks=6)
    p = prompts(40)[0]
    m.forward(p, 0, seq=0)
    kept = [x.clone() for x in m.cache.values(1, 0)]
    with pytest.raises(ConfigError):
        m.generate_batch(prompts(90), 20)
    assert m.cache.lengths == {0: 40} and all(torch.equal(a, b) for a, b in zip(kept, m.cache.values(1, 0)))
    assert m.generate_batch(prompts(70), 20).shape == (1, 20)  # six blocks, three of them sequence 0's own
    assert m.cache.lengths == {0: 89}
