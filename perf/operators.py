"""The operators of a decode step that never leaves the device, and their plain forms.

Four operators serve a batch of sequences over a paged KV cache held in 4 bits:

  plan       block tables, sequence lengths and the tokens' slots, built from the lengths wanted
  append     NeoX rope on queries and keys, keys and values quantised into the pages, read back
  attention  causal GQA over the 4-bit pages, for single tokens, verified drafts and prompt chunks
  sample     temperature, top-k, top-p and min-p from given random numbers

``run`` calls the framework's entry points where ``own`` is true and computes the same in
elementary torch operations where it is false.  ``exact`` computes it once more in 64 bits.

A page holds 16 tokens of one kv head in 20 * D bytes (D = head size): K codes, K headers,
V codes, V headers.  Every 32 dims of a token share a header (f16 step d, f16 minimum m) and
stand for d * code + m.  Where a code lies is said by `_places`.
"""
import math

import numpy as np
import torch

own = False

BLOCK, GROUP = 16, 32


def listed():
    return [
        # one new token for each of 64 sequences in decode, then the rollback of a rejected token
        dict(name="plan 64 decode", op="plan", seqs=64, ctx=4096, new=1, busy=1.0),
        # 1000 sequence slots of a busy server: prompts arrive, sequences decode, end and roll back
        dict(name="plan 1000 mixed", op="plan", seqs=1000, ctx=1500, new=120, busy=0.6),
        # one decode token of the 0.5B-shaped decoder (14 / 2 heads of 64)
        dict(name="append 1 of 14/2", op="append", tokens=1, heads=14, kv=2, dim=64, ctx=4096, type="f32"),
        # a prompt chunk of the 70B-shaped decoder (64 / 8 heads of 128)
        dict(name="append 2000 of 64/8", op="append", tokens=2000, heads=64, kv=8, dim=128, ctx=8192, type="f32"),
        # one short sequence of the 0.5B-shaped decoder: latency is all there is
        dict(name="attn 1x160 14/2", op="attention", seqs=1, ctx=160, new=1, heads=14, kv=2, dim=64, out="f32"),
        # batched decode of the 70B-shaped decoder, ragged lengths up to 4096
        dict(name="attn 64x4096 64/8", op="attention", seqs=64, ctx=4096, new=1, heads=64, kv=8, dim=128, out="f32"),
        # a few long documents in decode
        dict(name="attn 3x60000 64/8", op="attention", seqs=3, ctx=60000, new=1, heads=64, kv=8, dim=128, out="bf16"),
        # speculative verify: five positions of each sequence, the 7B-shaped decoder (28 / 4 heads)
        dict(name="attn 8x2000 verify 28/4", op="attention", seqs=8, ctx=2000, new=5, heads=28, kv=4, dim=128, out="f32"),
        # a 512-token prompt chunk of a long prompt
        dict(name="attn 2x4000 chunk 64/8", op="attention", seqs=2, ctx=4000, new=512, heads=64, kv=8, dim=128, out="bf16"),
        # one row of the 0.5B-shaped decoder's logits
        dict(name="sample 1x151936", op="sample", rows=1, vocab=151936, type="f32", k=50, p=0.95, m=0.0),
        # a batch with the nucleus alone: no top-k to bound it
        dict(name="sample 64x152064 top-p", op="sample", rows=64, vocab=152064, type="f32", k=0, p=0.9, m=0.0),
        # a batch of bf16 logits under every filter
        dict(name="sample 200x151936 all", op="sample", rows=200, vocab=151936, type="bf16", k=200, p=0.95, m=0.02),
    ]


def _log(rng, low, high):
    """A whole number spread over the logarithm of its range."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


HEADS = ((14, 2, 64), (28, 4, 128), (64, 8, 128), (8, 8, 64), (8, 1, 128), (5, 5, 32), (12, 4, 96))


def draw(rng):
    op = rng.choice(("plan", "append", "attention", "attention", "sample"))
    if op == "plan":
        return dict(op=op, seqs=_log(rng, 1, 1000), ctx=_log(rng, 16, 4000), new=_log(rng, 1, 120), busy=rng.choice((1.0, 0.6)))
    heads, kv, dim = rng.choice(HEADS)
    if op == "append":
        return dict(op=op, tokens=_log(rng, 1, 1900), heads=heads, kv=kv, dim=dim, ctx=_log(rng, 2000, 100000),
                    type=rng.choice(("f32", "bf16", "f16")))
    if op == "attention":
        kind = rng.choice(("decode", "decode", "verify", "chunk"))
        out = rng.choice(("f32", "bf16", "f16"))
        if kind == "decode":
            ctx = _log(rng, 1, 50000)
            return dict(op=op, seqs=max(1, min(_log(rng, 1, 64), 150000 // ctx)), ctx=ctx, new=1, heads=heads, kv=kv, dim=dim, out=out)
        if kind == "verify":
            return dict(op=op, seqs=_log(rng, 1, 16), ctx=_log(rng, 8, 4000), new=rng.randint(2, 8), heads=heads, kv=kv, dim=dim, out=out)
        new = _log(rng, 16, 500)
        return dict(op=op, seqs=rng.randint(1, 2), ctx=new + _log(rng, 1, 3400), new=new, heads=heads, kv=kv, dim=dim, out=out)
    return dict(op=op, rows=_log(rng, 1, 64), vocab=_log(rng, 1000, 152064), type=rng.choice(("f32", "bf16", "f16")),
                k=rng.choice((0, 1, 20, 200)), p=rng.choice((1.0, 0.95, 0.5)), m=rng.choice((0.0, 0.05)))


def _dtype(name):
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


# ---------------------------------------------------------------- the pages' layout
_tables = {}


def _places(dim, device):
    """For K and V: the byte and the shift of (token, dim)'s code within its page, int64 [16, dim].

    K: a token's row is dim / 2 bytes; word i * NG + g (NG = dim / 32) holds dims 32 g + 8 i ..
    + 7 of group g, lowest nibble first.  V: word n holds, in its low and high half, dims 4 n ..
    + 3 of two neighbouring groups; with four groups the words of both pairs alternate and
    tokens with bit 1 set have words 8 apart exchanged; a last odd group fills half words."""
    key = (dim, str(device))
    if key not in _tables:
        ng, t, d = dim // GROUP, np.arange(BLOCK)[:, None], np.arange(dim)[None, :]
        g, r = d // 32, d % 32
        kbyte = ((r // 8) * ng + g) * 4 + (r % 8) // 2 + t * (dim // 2)
        n, p = r // 4, r % 4
        word = (n * 2 + g // 2) ^ (8 * ((t >> 1) & 1)) if ng == 4 else n + 0 * t
        vbyte = word * 4 + (g % 2) * 2 + p // 2
        if ng % 2:
            vbyte = np.where(g == ng - 1, ((ng - 1) * 8 + n) * 2 + p // 2, vbyte)
        vbyte = vbyte + t * (dim // 2) + 10 * dim
        shift = 4 * (d % 2) + 0 * t
        _tables[key] = [torch.from_numpy(np.ascontiguousarray(a)).to(device) for a in (kbyte, vbyte, shift)]
    return _tables[key]


def _quantise(x):
    """(codes, steps, minima) of x f32 [..., dim] in groups of 32: steps and minima in f16."""
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    low, high = g.amin(-1), g.amax(-1)
    step, least = ((high - low) / 15.0).half(), low.half()
    bad = ~(torch.isfinite(step) & torch.isfinite(least) & torch.isfinite(low) & torch.isfinite(high))
    step, least = (torch.where(bad, torch.nan, v) for v in (step, least))
    s = step.float()[..., None]
    codes = torch.where(s > 0, torch.clamp(torch.round((g - least.float()[..., None]) / s), 0, 15), 0.0)
    return codes.to(torch.uint8).reshape(x.shape), step, least


def _store(pages, slots, x, values):
    """Write x f32 [n, kv, dim] into the K or V half of the pages at `slots` (all >= 0)."""
    n, kv, dim = x.shape
    kbyte, vbyte, shift = _places(dim, x.device)
    at, base = (vbyte, 18 * dim) if values else (kbyte, 8 * dim)
    codes, step, least = _quantise(x)
    block, tok = slots.long() // BLOCK, slots.long() % BLOCK
    head = torch.arange(kv, device=x.device)[None, :, None]
    lo = torch.nonzero(torch.arange(dim, device=x.device) % 2 == 0).reshape(-1)
    both = codes[..., lo] | (codes[..., lo + 1] << 4)
    pages[block[:, None, None], head, at[tok][:, None, :][..., lo]] = both
    headers = torch.stack([step, least], -1).view(torch.uint8).reshape(n, kv, -1)
    width = headers.shape[-1]
    pages[block[:, None, None], head, base + tok[:, None, None] * width + torch.arange(width, device=x.device)] = headers


def _load(pages, values):
    """f32 [..., 16, dim] of the K or V half of pages [..., 20 * dim]."""
    dim = pages.shape[-1] // 20
    kbyte, vbyte, shift = _places(dim, pages.device)
    at, base = (vbyte, 18 * dim) if values else (kbyte, 8 * dim)
    codes = (pages[..., at.reshape(-1)] >> shift.reshape(-1).to(torch.uint8)) & 15
    codes = codes.reshape(*pages.shape[:-1], BLOCK, dim // GROUP, GROUP).float()
    headers = pages[..., base:base + 2 * dim].contiguous().view(torch.float16).reshape(*pages.shape[:-1], BLOCK, dim // GROUP, 2).float()
    return (codes * headers[..., :1] + headers[..., 1:]).reshape(*pages.shape[:-1], BLOCK, dim)


# ---------------------------------------------------------------- inputs
def _table(gen, blocks_of, total):
    """(table, free stack): the blocks of every sequence from one shuffled pool of `total`."""
    perm = gen.permutation(total).astype(np.int32)
    width = max(1, max(blocks_of))
    table = np.zeros((len(blocks_of), width), np.int32)
    at = 0
    for s, n in enumerate(blocks_of):
        table[s, :n] = perm[at:at + n]
        at += n
    return table, perm[at:]


def prepare(case, seed):
    device = torch.device("cuda")
    gen = np.random.default_rng([seed, 20])
    gpu = torch.Generator(device=device)
    gpu.manual_seed(seed)
    to = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(device)  # noqa: E731
    if case["op"] == "plan":
        n = case["seqs"]
        length = gen.integers(0, case["ctx"] + 1, n)
        grown = length + (1 if case["new"] == 1 else gen.integers(1, case["new"] + 1, n))
        kind = gen.random(n)
        want = np.where(kind < case["busy"], grown, np.where(kind < 0.7, length, np.where(kind < 0.85, 0, np.maximum(0, length - 5))))
        most = -(-(case["ctx"] + case["new"]) // BLOCK)
        total = n * (-(-case["ctx"] // BLOCK) + -(-case["new"] // BLOCK))
        table, free = _table(gen, [-(-int(v) // BLOCK) for v in length], total)
        wide = np.zeros((n, most), np.int32)
        wide[:, :min(most, table.shape[1])] = table[:, :most]
        stack = np.full(total, -1, np.int32)
        stack[:len(free)] = free
        tokens = n * case["new"]
        return dict(op="plan", length=to(length.astype(np.int32)), want=to(want.astype(np.int32)), back=to(length.astype(np.int32)),
                    table=to(wide), free_list=to(stack), free_count=to(np.array([len(free)], np.int32)), tokens=tokens)
    if case["op"] == "append":
        n, dt = case["tokens"], _dtype(case["type"])
        blocks = -(-n // BLOCK) * 2 + 4
        slots = gen.permutation(blocks * BLOCK)[:n].astype(np.int32)
        # a prompt chunk's positions, far into a long context
        pos = (case["ctx"] - n + np.arange(n)).clip(0).astype(np.int32)
        if n > 4:
            slots[n // 2] = -1  # a padded row
        mk = lambda h: torch.randn((n, h, case["dim"]), device=device, generator=gpu)  # noqa: E731
        k = mk(case["kv"]) + 2 * torch.randn((case["kv"], case["dim"]), device=device, generator=gpu)  # keys carry a bias per channel
        inv = 1e6 ** (-np.arange(0, case["dim"], 2, dtype=np.float64) / case["dim"])
        pages = torch.zeros((blocks, case["kv"], 20 * case["dim"]), dtype=torch.uint8, device=device)
        return dict(op="append", q=mk(case["heads"]).to(dt), k=k.to(dt), v=mk(case["kv"]).to(dt), inv_freq=to(inv), pos=to(pos),
                    slots=to(slots), pages=pages)
    if case["op"] == "attention":
        n, dim, kv = case["seqs"], case["dim"], case["kv"]
        ctx = np.maximum(case["new"], (case["ctx"] * (1 - 0.9 * gen.random(n) ** 2)).astype(np.int64))
        ctx[0] = case["ctx"]
        new = np.full(n, case["new"])
        blocks_of = [-(-int(c) // BLOCK) for c in ctx]
        total = sum(blocks_of) + 3
        table, free = _table(gen, blocks_of, total)
        pages = torch.empty((total, kv, 20 * dim), dtype=torch.uint8, device=device)
        bias = 2 * torch.randn((kv, 1, dim), device=device, generator=gpu)
        step = max(1, (1 << 26) // (kv * BLOCK * dim))
        every = torch.arange(step * BLOCK, device=device, dtype=torch.int32)
        for b in range(0, total, step):
            m = min(step, total - b)
            for half in (False, True):
                x = torch.randn((m, kv, BLOCK, dim), device=device, generator=gpu)
                x = x if half else x + bias
                _store(pages[b:b + m], every[:m * BLOCK], x.transpose(1, 2).reshape(m * BLOCK, kv, dim), half)
        tail = torch.full((n, kv, dim), torch.nan, device=device)  # the slot behind each sequence was never written
        behind = np.array([table[s, c // BLOCK] * BLOCK + c % BLOCK for s, c in enumerate(ctx) if c % BLOCK], np.int32)
        for half in (False, True) if len(behind) else ():
            _store(pages, to(behind), tail[:len(behind)], half)
        q = torch.randn((int(new.sum()), case["heads"], dim), device=device, generator=gpu)
        start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        return dict(op="attention", q=q, pages=pages, table=to(table), start=to(start), ctx=to(ctx.astype(np.int32)), scale=1.0 / math.sqrt(dim),
                    max_q=int(new.max()), max_ctx=int(ctx.max()), out=_dtype(case["out"]))
    rows, vocab = case["rows"], case["vocab"]
    # a language model's logits: a broad body and a few strong candidates
    x = 2.0 * torch.randn((rows, vocab), device=device, generator=gpu)
    peaks = torch.randint(0, vocab, (rows, 30), device=device, generator=gpu)
    x.scatter_add_(1, peaks, 8 + 3 * torch.randn((rows, 30), device=device, generator=gpu))
    x[:, vocab // 2] = -torch.inf  # a token that is never allowed
    some = lambda low, high: (low + (high - low) * torch.rand(rows, device=device, generator=gpu)).float()  # noqa: E731
    k = torch.full((rows,), case["k"], dtype=torch.int32, device=device)
    return dict(op="sample", logits=x.to(_dtype(case["type"])), u=some(0, 1), t=some(0.6, 1.1), k=k if case["k"] else None,
                p=some(case["p"] - 0.02, case["p"]) if case["p"] < 1 else None,
                m=some(0.5 * case["m"], case["m"]) if case["m"] else None)


# ---------------------------------------------------------------- one pass
def run(s):
    return {"plan": _plan, "append": _append, "attention": _attention, "sample": _sample}[s["op"]](s)


def _plan(s):
    """The lengths wanted, with the new tokens' places; then the rollback to the lengths before."""
    if own:
        from runtimed_b200 import kv4
        start, seq, pos, slot = kv4.plan(s["want"], s["length"], s["table"], s["free_list"], s["free_count"], max_tokens=s["tokens"])
        kv4.plan(s["back"], s["length"], s["table"], s["free_list"], s["free_count"])
    else:
        start, seq, pos, slot = _plan_plain(s, s["want"], s["tokens"])
        _plan_plain(s, s["back"], 0)
    return dict(start=start, seq=seq, pos=pos, slot=slot, length=s["length"], table=s["table"], free_list=s["free_list"], free_count=s["free_count"])


def _plan_plain(s, want, tokens):
    """Sequences that shrink push their blocks, last block first, in sequence order; then those
    that grow pop theirs.  Tokens are listed by sequence and position; rows behind them hold -1."""
    length, table, free, count = s["length"], s["table"], s["free_list"], s["free_count"]
    dev, total = length.device, free.shape[0]
    n, most = table.shape
    have, need = (length.long() + BLOCK - 1) // BLOCK, (want.long() + BLOCK - 1) // BLOCK
    gone, taken = (have - need).clamp(min=0), (need - have).clamp(min=0)
    col = torch.arange(most, device=dev)[None, :]
    # the freed blocks in order
    goes = (col >= need[:, None]) & (col < have[:, None])
    rank = (gone.cumsum(0) - gone)[:, None] + (have[:, None] - 1 - col)
    freed = torch.zeros(total + 1, dtype=torch.int32, device=dev)
    freed[torch.where(goes, rank, total).reshape(-1)] = table.reshape(-1)
    top = count.long() + gone.sum()
    place = torch.arange(total, device=dev)
    stack = torch.where(place < count, free, freed[(place - count).clamp(0, total)])
    # the blocks taken from the top
    comes = (col >= have[:, None]) & (col < need[:, None])
    rank = (taken.cumsum(0) - taken)[:, None] + (col - have[:, None])
    table.copy_(torch.where(comes, stack[(top - 1 - rank).clamp(0, total - 1)], table))
    left = top - taken.sum()
    free.copy_(torch.where((place >= count) & (place < left), stack, free))
    old = length.clone()
    count.copy_(left.to(torch.int32))
    length.copy_(want)
    # the tokens
    new = (want - old).long().clamp(min=0)
    start = torch.cat([torch.zeros(1, dtype=torch.long, device=dev), new.cumsum(0)])
    if not tokens:
        return None
    t = torch.arange(tokens, device=dev)
    seq = torch.searchsorted(start, t, right=True) - 1
    here = seq < n
    seq = seq.clamp(max=n - 1)
    pos = old.long()[seq] + t - start[seq]
    slot = table[seq, (pos // BLOCK).clamp(0, most - 1)].long() * BLOCK + pos % BLOCK
    return (start.to(torch.int32), *(torch.where(here, v, -1).to(torch.int32) for v in (seq, pos, slot)))


def _append(s):
    if own:
        from runtimed_b200 import kv4
        q = kv4.append(s["q"], s["k"], s["v"], s["inv_freq"], s["pos"], s["slots"], s["pages"])
        k, v = kv4.read(s["pages"], s["slots"], torch.float16)
        return dict(q=q, k=k, v=v)
    angle = s["pos"].double()[:, None] * s["inv_freq"]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def rope(x):
        a, b = x.float().chunk(2, -1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    slots = s["slots"]
    there = slots >= 0
    q, k = rope(s["q"]), rope(s["k"])
    _store(s["pages"], slots[there], k[there], False)
    _store(s["pages"], slots[there], s["v"].float()[there], True)
    block, tok = (slots.clamp(min=0).long() // BLOCK), slots.clamp(min=0).long() % BLOCK
    every = torch.arange(len(slots), device=slots.device)
    read = [torch.where(there[:, None, None], _load(s["pages"][block], half)[every, :, tok], 0.0).half() for half in (False, True)]
    return dict(q=q, k=read[0], v=read[1])


def _attention(s):
    if own:
        from runtimed_b200 import kv4
        return kv4.attention(s["q"], s["pages"], s["table"], s["start"], s["ctx"], scale=s["scale"], max_q=s["max_q"], max_ctx=s["max_ctx"],
                             out_dtype=s["out"])
    q, start, ctx = s["q"], s["start"].long(), s["ctx"].long()
    tokens, heads, dim = q.shape
    kv, n, dev = s["pages"].shape[1], len(ctx), q.device
    new = start[1:] - start[:-1]
    most, longest = s["max_q"], s["max_ctx"]
    blocks = -(-longest // BLOCK)
    key = torch.arange(blocks * BLOCK, device=dev)
    behind = (key >= ctx[:, None])[:, None, :, None]
    table = s["table"][:, :blocks].long()

    def values(half):
        x = _load(s["pages"][table], half).transpose(1, 2).reshape(n, kv, blocks * BLOCK, dim)
        return x.masked_fill_(behind, 0.0)

    row = start[:-1, None] + torch.arange(most, device=dev)
    there = torch.arange(most, device=dev) < new[:, None]
    padded = q[row.clamp(max=tokens - 1)].reshape(n, most, kv, heads // kv, dim).permute(0, 2, 3, 1, 4).reshape(n, kv, -1, dim)
    score = (padded * s["scale"]) @ values(False).transpose(-1, -2)
    pos = (ctx - new)[:, None] + torch.arange(most, device=dev)
    seen = (key <= pos[:, :, None])[:, None, None]
    score = score.reshape(n, kv, heads // kv, most, -1).masked_fill_(~seen, -torch.inf)
    score = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-1e30))
    total = score.sum(-1, keepdim=True)
    out = (score.reshape(n, kv, -1, blocks * BLOCK) @ values(True)).reshape(n, kv, heads // kv, most, dim)
    out = torch.where(total > 0, out / total, 0.0)
    out = out.permute(0, 3, 1, 2, 4).reshape(n, most, heads, dim)
    return out[there].to(s["out"])


def _sample(s):
    if own:
        from runtimed_b200 import sampling
        return sampling.sample(s["logits"], s["u"], temperature=s["t"], top_k=s["k"], top_p=s["p"], min_p=s["m"])
    x = s["logits"].float()
    rows, vocab = x.shape
    # weights in units of 2^-44 of the largest: whole numbers, so that no order of sums matters
    unit = float(1 << 44)
    d = x.double()
    w = torch.round(torch.exp((d - d.amax(1, keepdim=True)) / s["t"].double()[:, None]) * unit).long()
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    ranked = w.gather(1, order)
    if s["k"] is not None:
        ranked = torch.where(torch.arange(vocab, device=x.device) < s["k"][:, None], ranked, 0)
    if s["p"] is not None:
        run_ = ranked.cumsum(1)
        enough = torch.floor(s["p"].double()[:, None] * run_[:, -1:].double()).long().clamp(min=1)
        ranked = torch.where(run_ - ranked < enough, ranked, 0)
    if s["m"] is not None:
        ranked = torch.where(ranked.double() >= s["m"].double()[:, None] * unit, ranked, 0)
    kept = torch.zeros_like(w).scatter_(1, order, ranked)
    run_ = kept.cumsum(1)
    total = run_[:, -1]
    at = torch.minimum(torch.floor(s["u"].double() * total.double()).long(), total - 1)
    return (run_ <= at[:, None]).sum(1).to(torch.int32)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["op"] == "plan":
        n, tokens = case["seqs"], case["seqs"] * case["new"]
        blocks = n * (1 + case["new"] // BLOCK)
        return dict(bytes=2 * (12 * n + 8 * blocks) + 4 * n + 12 * tokens, flops=0)
    if case["op"] == "append":
        n, dim, kv, heads = case["tokens"], case["dim"], case["kv"], case["heads"]
        size = 4 if case["type"] == "f32" else 2
        stored = n * kv * dim * 2 * 5 // 8
        return dict(bytes=n * (heads + 2 * kv) * dim * size + n * heads * dim * 4 + 2 * stored + 4 * n * kv * dim + 8 * n, flops=n * (heads + 2 * kv) * dim * 6)
    if case["op"] == "attention":
        # the mean of the lengths that prepare draws is 0.7 of the longest
        n, new, dim = case["seqs"], case["new"], case["dim"]
        ctx = case["ctx"] * (1 + 0.7 * (n - 1))
        size = 4 if case["out"] == "f32" else 2
        seen = new * (ctx - n * (new - 1) / 2)
        return dict(bytes=ctx * case["kv"] * dim * 2 * 5 / 8 + n * new * case["heads"] * dim * (4 + size), flops=4 * seen * case["heads"] * dim)
    return dict(bytes=case["rows"] * case["vocab"] * (4 if case["type"] == "f32" else 2), flops=2 * case["rows"] * case["vocab"])


# ---------------------------------------------------------------- in 64 bits
def _decode64(page, dim):
    """(K, V) f64 [16, dim] each of a batch of pages uint8 [..., 20 dim], word by word."""
    ng = dim // 32
    lead = page.shape[:-1]
    out = []
    for half in (0, 1):
        base = 10 * dim * half
        words = page[..., base:base + 8 * dim].contiguous().view(torch.int16).to(torch.int64) & 0xFFFF
        words = words.reshape(*lead, 16, dim // 4)  # half words of four codes
        codes = torch.zeros((*lead, 16, dim), dtype=torch.float64, device=page.device)
        for g in range(ng):
            for r in range(8):  # four dims from 32 g + 4 r
                if not half:
                    at = [2 * ((r // 2) * ng + g) + r % 2] * 16
                elif ng == 4:
                    at = [2 * ((2 * r + g // 2) ^ (8 if t & 2 else 0)) + g % 2 for t in range(16)]
                elif ng % 2 and g == ng - 1:
                    at = [8 * g + r] * 16
                else:
                    at = [2 * r + g] * 16
                w = torch.stack([words[..., t, a] for t, a in enumerate(at)], -1)
                for j in range(4):
                    codes[..., 32 * g + 4 * r + j] = ((w >> (4 * j)) & 15).double()
        head = page[..., base + 8 * dim:base + 10 * dim].contiguous().view(torch.float16).double().reshape(*lead, 16, ng, 2)
        out.append(codes * head[..., 0].repeat_interleave(32, -1) + head[..., 1].repeat_interleave(32, -1))
    return out


def exact(case, seed):
    s = prepare(case, seed)
    host = lambda t: t.detach().cpu().numpy()  # noqa: E731
    if case["op"] == "plan":
        return None  # whole numbers: held to the plain form's
    if case["op"] == "append":
        x = {k: host(s[k].float()).astype(np.float64) for k in ("q", "k", "v")}
        half = case["dim"] // 2
        turn = np.exp(1j * (host(s["pos"]).astype(np.float64)[:, None] * host(s["inv_freq"])[None]))[:, None]
        slots = host(s["slots"])
        got = {}
        for name in ("q", "k", "v"):
            v = x[name]
            if name != "v":
                z = (v[..., :half] + 1j * v[..., half:]) * turn
                v = np.concatenate([z.real, z.imag], -1)
            if name != "q":
                g = v.reshape(*v.shape[:2], -1, 32)
                m = g.min(-1, keepdims=True).astype(np.float16).astype(np.float64)
                d = ((g.max(-1, keepdims=True) - g.min(-1, keepdims=True)) / 15).astype(np.float16).astype(np.float64)
                c = np.clip(np.rint((g - m) / np.where(d > 0, d, 1)), 0, 15) * (d > 0)
                v = (c * d + m).reshape(v.shape) * (slots >= 0)[:, None, None]
            got[name] = torch.from_numpy(v)
        return got
    if case["op"] == "attention":
        start, ctx, dim, kv = host(s["start"]), host(s["ctx"]), case["dim"], case["kv"]
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
        for b in range(len(ctx)):
            c, rows = int(ctx[b]), slice(int(start[b]), int(start[b + 1]))
            n = rows.stop - rows.start
            pages = s["pages"][s["table"][b, :-(-c // 16)].long()]
            pos = torch.arange(c - n, c, device=out.device)
            for h in range(kv):
                k, v = (x.reshape(-1, dim)[:c] for x in _decode64(pages[:, h], dim))
                q = s["q"][rows].double().reshape(n, kv, -1, dim)[:, h]
                e = torch.einsum("nhd,cd->nhc", q, k) * s["scale"]
                e.masked_fill_((torch.arange(c, device=out.device) > pos[:, None])[:, None], -torch.inf)
                out[rows].view(n, kv, -1, dim)[:, h] = torch.einsum("nhc,cd->nhd", torch.softmax(e, -1), v)
        return out
    ids = []
    for r in range(case["rows"]):
        x = host(s["logits"][r].float()).astype(np.float64)
        e = np.exp((x - x.max()) / float(s["t"][r]))
        order = np.lexsort((np.arange(len(x)), -x))
        keep = np.zeros(len(x), bool)
        if s["k"] is not None:
            order = order[:int(s["k"][r])]
        if s["p"] is not None:
            c = np.cumsum(e[order])
            order = order[:1 + int(np.searchsorted(c, float(s["p"][r]) * c[-1], "left"))]
        keep[order] = True
        if s["m"] is not None:
            keep &= e >= float(s["m"][r])
        c = np.cumsum(np.where(keep, e, 0.0))
        ids.append(int(np.searchsorted(c, float(s["u"][r]) * c[-1], "right")))
    return torch.tensor(ids, dtype=torch.int32)
