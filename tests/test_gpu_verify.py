"""verify_tokens against a plain loop in 64 bits, and the decode-step operators together.

Tokens are whole numbers and have to be equal.  Both sides sum in f64, so they
can differ only where a draw lies within about 1e-13 of a token's edge; the
draws of the edge tests are set 1e-9 or more from it.
"""
import math

import numpy as np
import pytest
import torch

from commitllm_b200 import _lib
from commitllm_b200 import commit as C
from commitllm_b200 import decode as D
from oracle import commit_oracle as O

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def draw(w, u):
    run = np.cumsum(w)
    at = int((run <= u * run[-1]).sum())
    return min(at, int(np.nonzero(w > 0)[0][-1]))


def plain(logits, drafts, uniforms, temperature, probs=None):
    """(tokens, counts) of one batch, all numpy, one position at a time."""
    S, N, V = logits.shape
    tokens = np.full((S, N), -1, np.int32)
    counts = np.zeros(S, np.int32)
    for s in range(S):
        t = float(temperature[s])
        for i in range(N):
            row = logits[s, i].astype(np.float64)
            top = row.max()
            x = int(drafts[s, i]) if i < N - 1 else -1
            there = 0 <= x < V
            if not np.isfinite(top):
                break
            w = np.exp((row - top) / t) if t > 0 else (np.arange(V) == row.argmax()).astype(np.float64)
            if probs is None or t <= 0:
                token = draw(w, uniforms[s, i]) if t > 0 else int(row.argmax())
                keep = there and token == x
            else:
                p = w / w.sum()
                keep = there and uniforms[s, i] * float(probs[s, i, x]) < p[x]
                if not keep:
                    if there:
                        over = np.maximum(p - probs[s, i].astype(np.float64), 0)
                        w = over if over.sum() > 0 else w
                    token = draw(w, uniforms[s, N - 1])
            counts[s] += 1
            tokens[s, i] = x if keep else token
            if not keep:
                break
    return tokens, counts


def check(ctx, logits, drafts, uniforms, temperature, probs=None):
    """logits, probs: CUDA tensors (any strides); the rest numpy."""
    S, N, V = logits.shape
    tok, cnt = D.verify_tokens(ctx, logits, torch.tensor(drafts, dtype=torch.int32, device="cuda").reshape(S, N - 1),
                               torch.tensor(uniforms, dtype=torch.float64, device="cuda"),
                               torch.tensor(temperature, dtype=torch.float32, device="cuda"), draft_probs=probs)
    ctx.sync(60000)
    want, n = plain(logits.double().cpu().numpy(), drafts, uniforms, np.asarray(temperature, np.float32),
                    None if probs is None else probs.cpu().numpy())
    assert np.array_equal(cnt.cpu().numpy(), n)
    assert np.array_equal(tok.cpu().numpy(), want)
    return want, n


def inputs(seed, S, k, V, dtype, with_probs, peak=True, sharp=1.0):
    rng = np.random.default_rng(seed)
    l = rng.standard_normal((S, k + 1, V)).astype(np.float32) * 3
    likely = rng.integers(0, V, (S, k + 1))
    if peak:
        l[np.arange(S)[:, None], np.arange(k + 1)[None], likely] += rng.uniform(4, 18, (S, k + 1)).astype(np.float32)
    if V > 10:
        l[:, :, 3::17] = -np.inf
    logits = torch.tensor(l, device="cuda").to(DT[dtype])
    probs = None
    drafts = np.where(rng.random((S, k)) < 0.8, likely[:, :k], rng.integers(0, V, (S, k))).astype(np.int32)
    if with_probs:
        probs = torch.softmax(torch.tensor(l[:, :k] + sharp * rng.standard_normal((S, k, V)).astype(np.float32),
                                           device="cuda"), -1)
        if k:
            drafts = torch.multinomial(probs.reshape(S * k, V).double(), 1).reshape(S, k).cpu().numpy().astype(np.int32)
    temperature = rng.uniform(0.5, 1.5, S).astype(np.float32)
    temperature[::4] = 0
    return logits, drafts, rng.random((S, k + 1)), temperature, probs


@pytest.mark.parametrize("with_probs", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("S,k,V", [(1, 0, 1), (3, 2, 2), (5, 3, 7), (9, 4, 100), (4, 1, 4096), (6, 5, 4097),
                                   (7, 7, 32001), (5, 3, 50257), (9, 4, 128256), (2, 2, 200001)])
def test_verify_shapes(ctx, dtype, S, k, V, with_probs):
    check(ctx, *inputs(S + k + V, S, k, V, dtype, with_probs))


@pytest.mark.parametrize("with_probs", [False, True])
def test_verify_flat_rows_and_many_sequences(ctx, with_probs):
    """Without likely tokens every draw falls between close edges; 300 sequences."""
    check(ctx, *inputs(5, 300, 2, 3001, "f32", with_probs, peak=False))


def test_verify_largest_vocabulary(ctx):
    check(ctx, *inputs(6, 1, 1, 1 << 20, "bf16", False))
    check(ctx, *inputs(7, 1, 1, 1 << 20, "bf16", True))


@pytest.mark.parametrize("with_probs", [False, True])
def test_verify_strided_rows(ctx, with_probs):
    """Logits and probabilities as views of wider, oddly strided buffers."""
    logits, drafts, u, t, probs = inputs(8, 5, 3, 999, "f32", with_probs)
    wide = torch.zeros(4, 5, 1003, device="cuda")
    wide[:, :, 3:1002] = logits.transpose(0, 1)
    if with_probs:
        pw = torch.zeros(5, 3, 1001, device="cuda")
        pw[:, :, 1:1000] = probs
        probs = pw[:, :, 1:1000]
    check(ctx, wide[:, :, 3:1002].transpose(0, 1), drafts, u, t, probs)


def test_verify_ties_go_to_the_lowest_index(ctx):
    V = 40000
    l = np.zeros((3, 2, V), np.float32)
    l[0, 0, [39999, 17, 20000]] = 5
    l[1, 0, [0, 39999]] = 1
    l[0, 1, 9:] = -1e-30
    t = np.zeros(3, np.float32)
    d = np.array([[17], [39999], [0]], np.int32)
    u = np.full((3, 2), 0.5)
    want, n = check(ctx, torch.tensor(l, device="cuda"), d, u, t)
    assert want.tolist() == [[17, 0], [0, -1], [0, 0]]
    q = torch.full((3, 1, V), 1.0 / V, device="cuda")
    got, _ = check(ctx, torch.tensor(l, device="cuda"), d, u, t, q)
    assert np.array_equal(got, want)


def test_verify_numbers_at_the_ends(ctx):
    """u = 0 takes the first possible token, u just under 1 the last one."""
    V = 9001
    rng = np.random.default_rng(3)
    l = rng.standard_normal((4, 1, V)).astype(np.float32)
    l[:, :, :5] = -np.inf
    l[:, :, -3:] = -np.inf
    l[2:, :, -4] = -200.0           # still possible
    u = np.array([[0.0], [1 - 2.0 ** -53], [1 - 2.0 ** -53], [0.0]])
    want, _ = check(ctx, torch.tensor(l, device="cuda"), np.zeros((4, 0), np.int32), u, np.ones(4, np.float32))
    assert want[0, 0] == 5 and want[3, 0] == 5


@pytest.mark.parametrize("side", [-1, 1])
@pytest.mark.parametrize("gap", [1e-9, 1e-7, 3e-6])
def test_verify_draws_next_to_an_edge(ctx, side, gap):
    """Numbers set next to where a draft is just kept, or just drawn: what f32 sums leave open."""
    V, S = 30011, 24
    logits, drafts, u, t, probs = inputs(11, S, 1, V, "f32", True)
    t = np.full(S, 0.9, np.float32)
    l = logits.double().cpu().numpy()
    w = np.exp((l[:, 0] - l[:, 0].max(-1, keepdims=True)) / float(np.float32(0.9)))
    p = w / w.sum(-1, keepdims=True)
    q = probs.cpu().numpy().astype(np.float64)
    at = np.arange(S)
    # with probabilities: u q = p (1 +- gap), where the draft is likelier than the target has it
    ratio = p[at, drafts[:, 0]] / q[at, 0, drafts[:, 0]]
    u[:, 0] = np.where(ratio < 0.99, ratio * (1 + side * gap), u[:, 0])
    assert (ratio < 0.99).sum() > 3
    _, n = check(ctx, logits, drafts, u, t, probs)
    assert ((n == 2) == (side < 0))[ratio < 0.99].all()
    # without: u at the upper edge of the first token likelier than twenty gaps, where as much lies behind it
    d = np.array([int(np.nonzero(r > 20 * gap)[0][0]) for r in p], np.int32)[:, None]
    edge = np.cumsum(p, -1)[at, d[:, 0]]
    fits = edge < 1 - 20 * gap
    assert fits.sum() > 3
    u[:, 0] = np.where(fits, edge + side * gap, u[:, 0])
    _, n = check(ctx, logits, d, u, t)
    assert ((n == 2) == (side < 0))[fits].all()


def test_verify_rows_that_cannot_be_used(ctx):
    """NaN, +inf, nothing above -inf: the sequence ends there; behind the end they do not matter."""
    for with_probs in (False, True):
        logits, drafts, u, t, probs = inputs(12, 8, 2, 5000, "f32", with_probs)
        best = logits.argmax(-1).cpu().numpy()
        drafts[:] = best[:, :2]
        t[:] = 0
        logits[0, 0, 77] = math.nan
        logits[1, 1, 4999] = math.inf
        logits[2, 2] = -math.inf
        logits[3, 2, 0] = math.nan
        drafts[3, 1] = (best[3, 1] + 1) % 5000     # ends before the NaN row
        logits[4, 1] = -math.inf
        t[4:6] = 1.0
        _, n = check(ctx, logits, drafts, u, t, probs)
        assert n[:4].tolist() == [0, 1, 2, 2]


def test_verify_sequences_with_fewer_drafts(ctx):
    for with_probs in (False, True):
        logits, drafts, u, t, probs = inputs(13, 6, 4, 3000, "f32", with_probs)
        drafts[1, 0] = -1
        drafts[2, 2] = 3000
        drafts[4, 3] = 2 ** 31 - 1
        check(ctx, logits, drafts, u, t, probs)


@pytest.mark.parametrize("k", [15, 16, 17, 40])
def test_verify_many_drafts(ctx, k):
    """Runs of kept drafts past 16 positions, ended at every kind of place."""
    rng = np.random.default_rng(k)
    S, V = 12, 600
    l = rng.standard_normal((S, k + 1, V)).astype(np.float32)
    best = rng.integers(0, V, (S, k + 1))
    l[np.arange(S)[:, None], np.arange(k + 1)[None], best] += 25.0
    drafts = best[:, :k].astype(np.int32)
    for s, end in enumerate((0, 1, 14, 15, 16, 17, 31, 32, 33, k - 1)):
        if end < k:
            drafts[s, end] = (drafts[s, end] + 1) % V
    t = np.where(np.arange(S) % 3 == 0, 0.0, 1.0).astype(np.float32)
    u = rng.random((S, k + 1))
    _, n = check(ctx, torch.tensor(l, device="cuda"), drafts, u, t)
    assert n[-1] == k + 1 and n[3] == min(16, k + 1)
    probs = torch.softmax(torch.tensor(l[:, :k], device="cuda") + 1, -1)
    check(ctx, torch.tensor(l, device="cuda"), drafts, u, t, probs)


def test_verify_draft_distribution_equal_to_the_targets(ctx):
    """Nothing of p lies above q: a refused draft's replacement comes from p itself."""
    V = 64
    l = np.zeros((2, 2, V), np.float32)
    l[:, 0, 1:] = -np.inf                      # all on token 0
    q = torch.zeros(2, 1, V, device="cuda")
    q[:, 0, 0] = 1.0
    d = np.array([[5], [0]], np.int32)         # 5 was never possible
    u = np.full((2, 2), 0.5)
    want, n = check(ctx, torch.tensor(l, device="cuda"), d, u, np.ones(2, np.float32), q)
    assert want[0].tolist() == [0, -1] and n.tolist() == [1, 2]


def test_verify_extreme_temperatures(ctx):
    logits, drafts, u, t, probs = inputs(14, 6, 2, 2000, "f32", False)
    t = np.array([1e-38, 1e-6, 1e6, 3e38, 1e-3, 100.0], np.float32)
    logits[torch.isinf(logits)] = -30.0
    check(ctx, logits, drafts, u, t)


@pytest.mark.parametrize("t", [1e-9, 1.03e-8, 1.1e-8, 1e-7, 1e-5])
def test_verify_neighbouring_logits_at_small_temperatures(ctx, t):
    """Logits one f32 step apart, where a step is from a fraction of the temperature to hundreds of it."""
    V = 5000
    l = np.full((8, 1, V), 100.0, np.float32)
    step = np.nextafter(np.float32(100), np.float32(0)) - np.float32(100)
    l[:, 0] += step * np.random.default_rng(19).integers(0, 4, (8, V)).astype(np.float32)
    l[:, 0, 17:2000] -= 1
    u = np.linspace(0, 0.999, 8)[:, None] + 1e-5 * np.pi
    check(ctx, torch.tensor(l, device="cuda"), np.zeros((8, 0), np.int32), u, np.full(8, t, np.float32))


def test_verify_is_captured_and_replayed(ctx):
    stream = torch.cuda.Stream()
    c2 = C.Context(0, stream)
    logits, drafts, u, t, probs = inputs(15, 4, 3, 9000, "f32", True)
    dev = dict(l=logits, d=torch.tensor(drafts, device="cuda"), u=torch.tensor(u, device="cuda"),
               t=torch.tensor(t, device="cuda"), p=probs)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        D.verify_tokens(c2, dev["l"], dev["d"], dev["u"], dev["t"], draft_probs=dev["p"])
        stream.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=stream):
            tok, cnt = D.verify_tokens(c2, dev["l"], dev["d"], dev["u"], dev["t"], draft_probs=dev["p"])
    for seed in (16, 17):
        logits, drafts, u, t, probs = inputs(seed, 4, 3, 9000, "f32", True)
        dev["l"].copy_(logits), dev["d"].copy_(torch.tensor(drafts)), dev["u"].copy_(torch.tensor(u))
        dev["t"].copy_(torch.tensor(t)), dev["p"].copy_(probs)
        torch.cuda.synchronize()
        gr.replay()
        torch.cuda.synchronize()
        want, n = plain(logits.double().cpu().numpy(), drafts, u, t, probs.cpu().numpy())
        assert np.array_equal(tok.cpu().numpy(), want) and np.array_equal(cnt.cpu().numpy(), n)
    del gr
    c2.close()


def test_verify_refusals(ctx):
    logits, drafts, u, t, probs = inputs(18, 2, 2, 50, "f32", True)
    d, uu, tt = (torch.tensor(x, device="cuda") for x in (drafts, u, t))
    for bad in (dict(l=logits.double()), dict(l=logits[0]), dict(l=logits.cpu()), dict(l=logits.transpose(1, 2)),
                dict(l=logits[:, :, :0]), dict(d=d.long()), dict(d=d[:, :1]), dict(u=uu.float()), dict(u=uu[:, :2]),
                dict(t=tt.double()), dict(t=tt[:1]), dict(p=probs.double()), dict(p=probs[:, :1]),
                dict(p=probs.transpose(1, 2).contiguous().transpose(1, 2)),
                dict(u=None), dict(t=u), dict(d=None), dict(p=drafts),
                dict(w=torch.empty(8, dtype=torch.uint8, device="cuda"))):
        kw = dict(l=logits, d=d, u=uu, t=tt, p=probs, w=None)
        kw.update(bad)
        with pytest.raises(ValueError):
            D.verify_tokens(ctx, kw["l"], kw["d"], kw["u"], kw["t"], draft_probs=kw["p"], workspace=kw["w"])
    with pytest.raises(_lib.VcError, match="vocab"):
        D.verify_tokens(ctx, torch.zeros(1, 1, (1 << 20) + 1, device="cuda"), d[:1, :0].contiguous(),
                        uu[:1, :1].contiguous(), tt[:1])
    a, b = D.verify_tokens(ctx, logits[:0], d[:0], uu[:0], tt[:0])
    assert a.shape == (0, 3) and b.shape == (0,)


# ----------------------------------------------------------- a run of them all

class Model:
    """One attention layer over token tables: what a token contributes does not depend on the batch it is in."""

    def __init__(self, ctx, vocab, heads, kv, dim, seed):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g, device="cuda")
        self.q, self.k, self.v = r(vocab, heads, dim), r(vocab, kv, dim), r(vocab, kv, dim)
        self.out = r(heads * dim, vocab).double() * 0.3
        self.rope = D.rope_table(ctx, C.RopeConfig(theta=500000.0, scaling="llama3"), dim)

    def step(self, cache, tokens, positions, lens, seq_ids):
        """tokens, positions [S, N]; float32 logits [S, N, vocab], as the capture keeps them."""
        S, N = tokens.shape
        t = tokens.reshape(-1).long().clamp(min=0)
        q = D.rope_append(cache, 0, self.q[t], self.k[t], self.v[t], positions.reshape(-1).contiguous(), self.rope,
                          seq_ids=seq_ids)
        o = D.paged_attention(cache, 0, q.view(S, N, *q.shape[1:]), lens)
        return (o.reshape(S, N, -1).double() @ self.out).float()


def test_drafted_decoding_commits_what_plain_decoding_commits(ctx):
    """Greedy and drawn requests decoded one by one, and with four drafts a step of which many are wrong: the same
    tokens, and the same kv_roots over the pages (the oracle's, over the rows read back)."""
    vocab, heads, kv, dim, page, S, steps, k = 300, 8, 2, 64, 16, 4, 40, 4
    model = Model(ctx, vocab, heads, kv, dim, 3)
    rng = np.random.default_rng(4)
    prompts = [rng.integers(0, vocab, n) for n in (5, 33, 1, 16)]
    U = torch.tensor(rng.random((S, 200)), device="cuda")
    temp = torch.tensor([0.0, 0.8, 1.0, 0.5], device="cuda")
    seqs = torch.arange(S, dtype=torch.int32, device="cuda")

    def new_cache():
        kvs = torch.zeros(2, 40, page, kv, dim, device="cuda")
        perm = torch.tensor(rng.permutation(40).astype(np.int32), device="cuda").view(S, 10)
        return D.PagedCache(ctx, [kvs[0]], [kvs[1]], perm.contiguous())

    def prefill(cache):
        # every prompt token but the last, in one ragged call
        toks = np.concatenate([p[:-1] for p in prompts])
        pos = np.concatenate([np.arange(len(p) - 1) for p in prompts])
        ids = np.concatenate([np.full(len(p) - 1, s) for s, p in enumerate(prompts)])
        t = torch.tensor(toks, device="cuda")
        i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")
        D.rope_append(cache, 0, model.q[t], model.k[t], model.v[t], i32(pos), model.rope, seq_ids=i32(ids))

    first = torch.tensor([[p[-1]] for p in prompts], dtype=torch.int32, device="cuda")
    start = torch.tensor([len(p) - 1 for p in prompts], dtype=torch.int32, device="cuda")
    # one by one
    plain_cache = new_cache()
    prefill(plain_cache)
    last, pos, text = first, start.clone(), []
    no_drafts = torch.zeros(S, 0, dtype=torch.int32, device="cuda")
    for _ in range(steps):
        logits = model.step(plain_cache, last, pos[:, None], (pos + 1).contiguous(), seqs)
        tok, cnt = D.verify_tokens(ctx, logits, no_drafts, U.gather(1, pos[:, None].long()), temp)
        assert bool((cnt == 1).all())
        text.append(tok[:, 0])
        last, pos = tok, pos + 1
    text = torch.stack(text, 1)                       # [S, steps]
    # drafted: the right continuation with every third token or so replaced
    cache = new_cache()
    prefill(cache)
    wrong = torch.tensor(rng.random((S, 200)) < 0.3, device="cuda")
    future = torch.cat([text, torch.zeros(S, 100, dtype=torch.int32, device="cuda")], 1)
    future = torch.where(wrong[:, : future.shape[1]], (future + 7) % vocab, future)
    ids = seqs.repeat_interleave(k + 1)
    got = torch.full((S, steps + 100), -1, dtype=torch.int32, device="cuda")
    done = torch.zeros(S, dtype=torch.int64, device="cuda")
    last, rounds = first, 0
    span = torch.arange(k + 1, device="cuda")
    while int(done.min()) < steps:
        drafts = future.gather(1, done[:, None] + span[None, :k]).to(torch.int32)
        base = start.long() + done
        p = (base[:, None] + span[None]).to(torch.int32)
        logits = model.step(cache, torch.cat([last, drafts], 1), p, (base + k + 1).to(torch.int32), ids)
        tok, cnt = D.verify_tokens(ctx, logits, drafts.contiguous(), U.gather(1, p.long()), temp)
        got.scatter_(1, done[:, None] + span[None], tok)
        done += cnt
        last = tok.gather(1, (cnt.long() - 1)[:, None])
        rounds += 1
    ctx.sync(60000)
    assert torch.equal(got[:, :steps], text)
    assert rounds < steps                              # drafts were kept
    lens = [len(p) - 1 + steps for p in prompts]
    r1, _ = C.kv_commit(ctx, plain_cache.view(lens), keep_trees=False)
    r2, _ = C.kv_commit(ctx, cache.view(lens), keep_trees=False)
    ctx.sync(60000)
    assert torch.equal(r1, r2)
    s = 1
    rows = torch.arange(lens[s], device="cuda")
    pg = cache.block_tables[s].long()[rows // page]
    kr, vr = (t[0][pg, rows % page].reshape(lens[s], -1).double().cpu().numpy() for t in (cache.k_layers, cache.v_layers))
    assert bytes(r2[s, 0].cpu().numpy()) == O.compute_root([O.hash_kv_entry(0, i, kr[i], vr[i]) for i in range(lens[s])])
