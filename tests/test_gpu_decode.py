"""Decode-step operators (rope_append, paged_attention) against plain 64-bit forms.

Tolerances.  A value rounded to a type with machine epsilon ``eps`` is off by at
most ``eps / 2`` of itself.  Rotations: the f32 cos and sin are off by 2^-24 of
1 each, the two products and the sum by 2^-24 each, so a rotated element is off
by at most 4 * 2^-24 * (|x1| + |x2|) * factor before its own rounding.
Attention: an output is a weighted mean of V rows.  The f32 score of a row is
off by at most (D + 4) * 2^-24 * scale * sum|q_d k_d| (D fused or tensor-core
additions, the scaling, the maximum's subtraction), its weight by that plus 2^-21
(exp2's two units, and the split of a weight in two 16-bit numbers, 2^-16 of it
for bf16 inputs, 2^-21 for f16), and the sums of n terms by n * 2^-24 in the
worst case; each bounds the error relative to sum(p |v|).  Then one rounding.
"""
import math

import numpy as np
import pytest
import torch

from commitllm_b200 import commit as C
from commitllm_b200 import decode as D

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def make_cache(ctx, seed, lens, kv_heads, dim, page, dtype, layers=1, spare=2, hnd=False, fill=None):
    """(PagedCache, generator): permuted pages, unused table entries junk, unused slots `fill` or noise."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    need = [(n + page - 1) // page for n in lens]
    total = sum(need) + spare
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(max(need), 1)), -9, dtype=torch.int32, device="cuda")
    at = 0
    for s, k in enumerate(need):
        table[s, :k] = order[at:at + k]
        at += k
    kv = []
    for _ in range(2 * layers):
        shape = (total, kv_heads, page, dim) if hnd else (total, page, kv_heads, dim)
        t = torch.randn(shape, generator=g, device="cuda").to(dtype)
        if hnd:
            t = t.permute(0, 2, 1, 3)
        if fill is not None:
            t.fill_(fill)
        kv.append(t)
    return D.PagedCache(ctx, kv[:layers], kv[layers:], table), g


def rows_of(cache, layer, s, n):
    """K and V rows 0..n-1 of sequence s, float64 [n, kv_heads, dim]."""
    p = torch.arange(n, device="cuda")
    page = cache.block_tables[s].long()[p // cache.block_size]
    return (cache.k_layers[layer][page, p % cache.block_size].double(),
            cache.v_layers[layer][page, p % cache.block_size].double())


def reference(cache, layer, q, lens, scale=None):
    """(out, lse, allowed error of out, of lse), float64."""
    S, N, H, Dm = q.shape
    G = cache.n_kv_heads
    scale = Dm ** -0.5 if scale is None else scale
    eps = torch.finfo(q.dtype).eps
    split = 2.0 ** -16 if q.dtype == torch.bfloat16 else 2.0 ** -21
    out = torch.zeros(S, N, H, Dm, dtype=torch.float64, device="cuda")
    lse = torch.full((S, N, H), -math.inf, dtype=torch.float64, device="cuda")
    tol, tol_l = torch.zeros_like(out), torch.zeros_like(lse)
    for s in range(S):
        k, v = rows_of(cache, layer, s, int(lens[s]))
        for j in range(N):
            m = int(lens[s]) - N + 1 + j
            if m <= 0:
                continue
            for h in range(H):
                kk, vv = k[:m, h // (H // G)], v[:m, h // (H // G)]
                x = q[s, j, h].double()
                sc = (kk @ x) * scale
                p = torch.softmax(sc, 0)
                out[s, j, h] = p @ vv
                lse[s, j, h] = torch.logsumexp(sc, 0)
                off = (Dm + 4) * 2.0 ** -24 * abs(scale) * float((kk.abs() @ x.abs()).max())
                rel = 2 * off + 2.0 ** -21 + split + 2 * m * 2.0 ** -24
                tol[s, j, h] = rel * (p @ vv.abs()) + eps / 2 * out[s, j, h].abs() + 1e-30
                tol_l[s, j, h] = off + 2.0 ** -20 + m * 2.0 ** -24 + 2.0 ** -23 * lse[s, j, h].abs()
    return out, lse, tol, tol_l


def check_attention(ctx, cache, q, lens, layer=0, scale=None):
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out, lse = D.paged_attention(cache, layer, q, n, scale=scale, return_lse=True)
    ctx.sync(60000)
    ro, rl, to, tl = reference(cache, layer, q, lens, scale)
    sub = torch.finfo(q.dtype).smallest_normal      # below it a type keeps fewer bits
    assert bool(((out.double() - ro).abs() <= to + sub).all()), float(((out.double() - ro).abs() - to).max())
    empty = torch.isneginf(rl)
    assert torch.equal(torch.isneginf(lse), empty)
    assert bool(((lse.double() - rl).abs()[~empty] <= tl[~empty]).all())
    assert bool((out[empty] == 0).all())
    return out, lse


def queries(g, S, N, H, dim, dtype, amp=2.0):
    return (torch.randn(S, N, H, dim, generator=g, device="cuda") * amp).to(dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("lens", [[1], [2, 1, 0, 63], [64, 65, 15, 16, 17], [700], [129, 0, 1000, 3]])
def test_attention_lengths(ctx, dtype, lens):
    cache, g = make_cache(ctx, 1 + len(lens), lens, 2, 128, 16, DT[dtype])
    check_attention(ctx, cache, queries(g, len(lens), 1, 8, 128, DT[dtype]), lens)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim", [2, 8, 20, 64, 72, 80, 96, 128, 136, 192, 256])
def test_attention_head_sizes(ctx, dtype, dim):
    lens = [50, 131]
    cache, g = make_cache(ctx, dim, lens, 2, dim, 16, DT[dtype])
    check_attention(ctx, cache, queries(g, 2, 1, 6, dim, DT[dtype]), lens)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads,kv", [(1, 1), (8, 8), (7, 1), (28, 4), (12, 4), (32, 2), (40, 1)])
@pytest.mark.parametrize("new", [1, 3, 5])
def test_attention_head_layouts_and_drafts(ctx, dtype, heads, kv, new):
    lens = [200, new, new - 1, 77]       # the third sequence's first tokens see nothing
    cache, g = make_cache(ctx, heads + new, lens, kv, 64, 24, DT[dtype])
    check_attention(ctx, cache, queries(g, 4, new, heads, 64, DT[dtype]), lens)


@pytest.mark.parametrize("page", [1, 3, 16, 64, 100, 1024])
@pytest.mark.parametrize("hnd", [False, True])
def test_attention_pages(ctx, page, hnd):
    lens = [333, 1, 90]
    cache, g = make_cache(ctx, page, lens, 4, 128, page, torch.bfloat16, layers=2, hnd=hnd)
    check_attention(ctx, cache, queries(g, 3, 2, 8, 128, torch.bfloat16), lens, layer=1)


def test_attention_long_split_and_scale(ctx):
    lens = [30001, 5, 9000]
    cache, g = make_cache(ctx, 4, lens, 1, 128, 16, torch.bfloat16)
    check_attention(ctx, cache, queries(g, 3, 1, 4, 128, torch.bfloat16, amp=1.0), lens, scale=0.3)
    check_attention(ctx, cache, queries(g, 3, 1, 4, 128, torch.bfloat16), lens, scale=-0.05)
    check_attention(ctx, cache, queries(g, 3, 1, 4, 128, torch.bfloat16), lens, scale=0.0)


def test_attention_many_sequences(ctx):
    rng = np.random.default_rng(7)
    lens = [int(x) for x in rng.integers(0, 90, 300)]
    cache, g = make_cache(ctx, 5, lens, 2, 64, 16, torch.bfloat16)
    check_attention(ctx, cache, queries(g, 300, 1, 4, 64, torch.bfloat16), lens)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_attention_unaligned_and_strided(ctx, dtype):
    """Rows that start at odd elements, and queries strided over a fused projection."""
    dt = DT[dtype]
    g = torch.Generator(device="cuda")
    g.manual_seed(9)
    base = torch.randn(2, 6 * 16 * 2 * 67 + 1, generator=g, device="cuda").to(dt)
    k, v = (b[1:].view(6, 16, 2, 67)[..., :66] for b in base)
    table = torch.tensor([[3, 1, 5], [0, 2, 4]], dtype=torch.int32, device="cuda")
    cache = D.PagedCache(ctx, [k], [v], table)
    fused = torch.randn(2, 3, 5 * 66 + 1, generator=g, device="cuda").to(dt)
    q = fused[:, :2, 1:1 + 4 * 66].unflatten(2, (4, 66))
    check_attention(ctx, cache, q, [40, 33])


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads,dim", [(12, 128), (4, 128), (8, 64), (4, 256), (12, 64), (2, 66)])
def test_attention_ignores_what_is_masked(ctx, dtype, heads, dim):
    """NaN and infinities in unused slots, past the length, and in rows that only later drafts see."""
    dt = DT[dtype]
    lens = [70, 16, 130]
    new = 4
    cache, g = make_cache(ctx, 10, lens, 2, dim, 16, dt)
    for s, n in enumerate(lens):      # slots past the length
        last = int(cache.block_tables[s, (n - 1) // 16])
        for t, x in ((cache.k_layers[0], math.inf), (cache.v_layers[0], math.nan)):
            t[last, (n - 1) % 16 + 1:] = x
    q = queries(g, 3, new, heads, dim, dt)
    check_attention(ctx, cache, q, lens)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for s, ln in enumerate(lens):     # the last two drafts' own rows
        for p, kx, vx in ((ln - 1, math.nan, math.inf), (ln - 2, -math.inf, math.nan)):
            page = int(cache.block_tables[s, p // 16])
            cache.k_layers[0][page, p % 16] = kx
            cache.v_layers[0][page, p % 16] = vx
    out = D.paged_attention(cache, 0, q, n)
    ctx.sync(60000)
    ro, _, to, _ = reference(cache, 0, q, lens)
    seen = slice(0, new - 2)
    assert bool(((out[:, seen].double() - ro[:, seen]).abs() <= to[:, seen]).all())
    assert bool(torch.isnan(out[:, new - 2:]).all())


def test_attention_extreme_scores(ctx):
    """Scores far apart: the largest takes all, and a masked maximum does not count."""
    lens = [100]
    cache, g = make_cache(ctx, 11, lens, 1, 64, 16, torch.float32)
    cache.k_layers[0].mul_(1000)
    q = queries(g, 1, 1, 2, 64, torch.float32, amp=100)
    k, v = rows_of(cache, 0, 0, 100)
    sc = torch.einsum("hd,nd->hn", q[0, 0].double(), k[:, 0])
    out = D.paged_attention(cache, 0, q, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    ctx.sync(60000)
    assert torch.equal(out[0, 0].double(), v[sc.argmax(1), 0])


def test_attention_same_result_every_time(ctx):
    lens = [5000, 300, 0, 2000]
    cache, g = make_cache(ctx, 12, lens, 4, 128, 16, torch.bfloat16)
    q = queries(g, 4, 2, 16, 128, torch.bfloat16)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    first = D.paged_attention(cache, 0, q, n, return_lse=True)
    for _ in range(5):
        again = D.paged_attention(cache, 0, q, n, return_lse=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_attention_leaves_rows_behind_the_batch(ctx):
    """A batch of fewer sequences than the table: outputs past it stay as they were."""
    lens = [30, 40, 50]
    cache, g = make_cache(ctx, 13, lens, 2, 64, 16, torch.bfloat16)
    q = queries(g, 3, 1, 4, 64, torch.bfloat16)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    whole = D.paged_attention(cache, 0, q, n)
    buf = torch.full((3, 1, 4, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    D.paged_attention(cache, 0, q[:2], n[:2], out=buf[:2])
    ctx.sync(60000)
    assert torch.equal(buf[:2], whole[:2]) and bool((buf[2] == 7).all())


def test_attention_bad_pages_are_reported(ctx):
    lens = [40, 20]
    cache, g = make_cache(ctx, 14, lens, 2, 64, 16, torch.bfloat16)
    q = queries(g, 2, 1, 4, 64, torch.bfloat16)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    good = D.paged_attention(cache, 0, q, n)
    keep = cache.block_tables.clone()
    for bad in (-1, cache.n_pages, 2 ** 31 - 1):
        cache.block_tables.copy_(keep)
        cache.block_tables[0, 1] = bad
        out = D.paged_attention(cache, 0, q, n)
        with pytest.raises(Exception, match="block table"):
            ctx.sync(60000)
        assert torch.equal(out[1], good[1])
    cache.block_tables.copy_(keep)
    # a length beyond the table is held to the table
    D.paged_attention(cache, 0, q, torch.tensor([40, 4000], dtype=torch.int32, device="cuda"))
    with pytest.raises(Exception, match="block table"):
        ctx.sync(60000)
    out = D.paged_attention(cache, 0, q, n)
    ctx.sync(60000)
    assert torch.equal(out, good)


def test_attention_lengths_past_the_table_are_reported(ctx):
    cache, g = make_cache(ctx, 16, [48, 48], 2, 64, 16, torch.bfloat16)
    q = queries(g, 2, 1, 4, 64, torch.bfloat16)
    want = D.paged_attention(cache, 0, q, torch.tensor([48, 30], dtype=torch.int32, device="cuda"))
    ctx.sync(60000)
    out = D.paged_attention(cache, 0, q, torch.tensor([49, 30], dtype=torch.int32, device="cuda"))
    with pytest.raises(Exception, match="block table"):
        ctx.sync(60000)
    assert torch.equal(out, want)
    # a negative length is an empty sequence
    out = D.paged_attention(cache, 0, q, torch.tensor([-5, 30], dtype=torch.int32, device="cuda"))
    ctx.sync(60000)
    assert bool((out[0] == 0).all()) and torch.equal(out[1], want[1])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rows_past_32_bits(ctx, dtype):
    """A cache of more than 2^32 elements, used at its far end and at its start."""
    dt, dim, kv, page = DT[dtype], 128, 8, 16
    pages = (1 << 32) // (page * kv * dim) + 40
    k, v = (torch.empty(pages, page, kv, dim, dtype=dt, device="cuda") for _ in range(2))
    table = torch.tensor([[pages - 1, 3, pages - 30, pages - 2], [7, pages - 3, 0, pages - 4]], dtype=torch.int32,
                         device="cuda")
    g = torch.Generator(device="cuda")
    g.manual_seed(21)
    for p in table.flatten().tolist():
        for t in (k, v):
            t[p] = torch.randn(page, kv, dim, generator=g, device="cuda").to(dt)
    cache = D.PagedCache(ctx, [k], [v], table)
    check_attention(ctx, cache, queries(g, 2, 2, 16, dim, dt), [64, 50])
    x = torch.randn(3, 2, kv, dim, generator=g, device="cuda").to(dt)
    pos = torch.tensor([5, 63], dtype=torch.int32, device="cuda")
    D.rope_append(cache, 0, x[0], x[1], x[2], pos, D.rope_table(ctx, C.RopeConfig(), dim),
                  seq_ids=torch.tensor([0, 1], dtype=torch.int32, device="cuda"))
    ctx.sync(60000)
    inv, f = D.rope_frequencies(C.RopeConfig(), dim)
    want, tol = rope_reference(x[1], pos, inv, f, False)
    for t, (p, slot) in enumerate(((pages - 1, 5), (pages - 4, 15))):
        assert close_rows(k[p, slot], want[t], tol[t]) and torch.equal(v[p, slot], x[2, t])


def test_attention_graph_replay_grows_with_its_tensors(ctx):
    """A captured step replayed with other lengths, queries and pages; two graphs, replayed on two streams."""
    stream = torch.cuda.Stream()
    c2 = C.Context(0, stream)
    lens = [500, 40]
    cache, g = make_cache(c2, 15, [3000, 3000], 2, 128, 16, torch.bfloat16)
    q = queries(g, 2, 1, 8, 128, torch.bfloat16)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        D.paged_attention(cache, 0, q, n)
        stream.synchronize()
        graphs, outs = [], []
        for _ in range(2):
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=stream):
                outs.append(D.paged_attention(cache, 0, q, n, return_lse=True))
            graphs.append(gr)
    for new_lens in ([500, 40], [2999, 0], [1, 1500]):
        q.copy_(queries(g, 2, 1, 8, 128, torch.bfloat16))
        n.copy_(torch.tensor(new_lens, dtype=torch.int32))
        torch.cuda.synchronize()
        other = torch.cuda.Stream()
        for _ in range(3):
            with torch.cuda.stream(stream):
                graphs[0].replay()
            with torch.cuda.stream(other):
                graphs[1].replay()
        torch.cuda.synchronize()
        ro, rl, to, _ = reference(cache, 0, q, new_lens)
        for out, _lse in outs:
            assert bool(((out.double() - ro).abs() <= to).all())
        assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
    del graphs
    c2.close()


# ------------------------------------------------------------------- rotary

def rope_reference(x, pos, inv, factor, interleaved):
    """float64 rotation of [n, heads, dim] at each token's position, and its allowed error before rounding."""
    r = 2 * len(inv)
    y = x.double().clone()
    ang = pos.double()[:, None] * torch.tensor(inv, dtype=torch.float64, device="cuda")[None]
    cos, sin = torch.cos(ang)[:, None] * factor, torch.sin(ang)[:, None] * factor
    i1, i2 = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    a, b = x[..., i1].double(), x[..., i2].double()
    y[..., i1], y[..., i2] = a * cos - b * sin, b * cos + a * sin
    tol = torch.zeros_like(y)
    tol[..., i1] = tol[..., i2] = 4 * 2.0 ** -24 * factor * (a.abs() + b.abs())
    pad = (pos < 0)[:, None, None]
    return torch.where(pad, x.double(), y), torch.where(pad, torch.zeros_like(tol), tol)


def close_rows(got, want, tol):
    eps = torch.finfo(got.dtype).eps
    return bool(((got.double() - want).abs() <= tol + eps / 2 * (want.abs() + tol) + 2.0 ** -25).all())


CONFIGS = {"none": C.RopeConfig(), "llama3": C.RopeConfig(theta=500000.0, scaling="llama3"),
           "linear": C.RopeConfig(scaling="linear", factor=4.0),
           "yarn": C.RopeConfig(theta=1e6, scaling="yarn", factor=8.0)}


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rot", [(128, 128), (128, 64), (64, 2), (80, 20), (256, 256), (6, 4), (96, 96), (20, 12)])
def test_rope_append_layouts(ctx, dtype, interleaved, dim, rot):
    dt = DT[dtype]
    lens = [70000, 40, 9, 3]
    kv, heads = 2, 6
    cache, g = make_cache(ctx, dim + rot, [64] * 4, kv, dim, 16, dt, layers=2, spare=3, fill=5.0)
    # sequence 0's rows live far out: its table is long, with pages only at the end
    table = torch.full((4, 5000), -1, dtype=torch.int32, device="cuda")
    table[0, 4370:4376] = torch.tensor([15, 3, 8, 1, 12, 6], dtype=torch.int32)
    table[1, :3] = torch.tensor([0, 9, 2], dtype=torch.int32)
    table[2, :1] = 5
    table[3, :1] = 14
    cache = D.PagedCache(ctx, cache.k_layers, cache.v_layers, table)
    pos = torch.tensor([69999, 70000, 69920, -1, 0, 39, 38, 8, 2, -5], dtype=torch.int32, device="cuda")
    ids = torch.tensor([0, 0, 0, 0, 1, 1, 1, 2, 3, 3], dtype=torch.int32, device="cuda")
    n = pos.numel()
    fused = torch.randn(n, (heads + 2 * kv) * dim, generator=g, device="cuda").to(dt)
    q = fused[:, : heads * dim].unflatten(1, (heads, dim))
    k = fused[:, heads * dim:(heads + kv) * dim].unflatten(1, (kv, dim))
    v = fused[:, (heads + kv) * dim:].unflatten(1, (kv, dim))
    cfg = CONFIGS[["none", "llama3", "linear", "yarn"][(dim + rot) // 2 % 4]]
    inv, factor = D.rope_frequencies(cfg, rot)
    rope = D.rope_table(ctx, cfg, rot)
    before = [t.clone() for t in cache.k_layers + cache.v_layers]
    q_in = q.clone()
    out = D.rope_append(cache, 1, q, k, v, pos, rope, seq_ids=ids, interleaved=interleaved)
    ctx.sync(60000)
    wq, tq = rope_reference(q, pos, inv, factor, interleaved)
    wk, tk = rope_reference(k, pos, inv, factor, interleaved)
    assert torch.equal(q, q_in)
    assert close_rows(out, wq, tq)
    assert torch.equal(out[..., rot:], q[..., rot:]) and torch.equal(out[[3, 9]], q[[3, 9]])
    touched = torch.zeros(cache.n_pages, 16, dtype=torch.bool, device="cuda")
    for t in range(n):
        p = int(pos[t])
        if p < 0:
            continue
        page, slot = int(table[int(ids[t]), p // 16]), p % 16
        touched[page, slot] = True
        assert close_rows(cache.k_layers[1][page, slot], wk[t], tk[t])
        assert torch.equal(cache.v_layers[1][page, slot], v[t])
    for now, was in zip(cache.k_layers + cache.v_layers, before):
        assert torch.equal(now[~touched], was[~touched])
    assert torch.equal(cache.k_layers[0], before[0]) and torch.equal(cache.v_layers[0], before[2])
    # in place, through the same fused tensor
    D.rope_append(cache, 1, q, k, v, pos, rope, seq_ids=ids, interleaved=interleaved, q_out=q)
    ctx.sync(60000)
    assert torch.equal(q, out)


def test_rope_append_unaligned_rows(ctx):
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    base = torch.zeros(2, 4 * 8 * 2 * 65 + 1, dtype=torch.bfloat16, device="cuda")
    k, v = (b[1:].view(4, 8, 2, 65)[..., :64] for b in base)
    cache = D.PagedCache(ctx, [k], [v], torch.tensor([[2, 0]], dtype=torch.int32, device="cuda"))
    x = torch.randn(3, 8 * 64 + 1, generator=g, device="cuda").to(torch.bfloat16)[:, 1:].unflatten(1, (8, 64))
    pos = torch.tensor([0, 9, 15], dtype=torch.int32, device="cuda")
    ids = torch.zeros(3, dtype=torch.int32, device="cuda")
    for interleaved in (False, True):
        rope = D.rope_table(ctx, C.RopeConfig(), 64)
        out = D.rope_append(cache, 0, x[:, :4], x[:, 4:6], x[:, 6:], pos, rope, seq_ids=ids, interleaved=interleaved)
        ctx.sync(60000)
        inv, f = D.rope_frequencies(C.RopeConfig(), 64)
        assert close_rows(out, *rope_reference(x[:, :4], pos, inv, f, interleaved))
        wk, tk = rope_reference(x[:, 4:6], pos, inv, f, interleaved)
        kk, vv = rows_of(cache, 0, 0, 16)
        assert close_rows(kk[pos.long()].to(torch.bfloat16), wk, tk)
        assert torch.equal(vv[pos.long()], x[:, 6:].double())


def test_rope_append_many_tokens_and_default_sequences(ctx):
    dim, S = 128, 700
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    kv = torch.zeros(2, S, 4, 2, dim, dtype=torch.bfloat16, device="cuda")
    table = torch.randperm(S, generator=g, device="cuda").to(torch.int32)[:, None].contiguous()
    cache = D.PagedCache(ctx, [kv[0]], [kv[1]], table)
    x = torch.randn(3, S, 2, dim, generator=g, device="cuda").to(torch.bfloat16)
    pos = (torch.arange(S, device="cuda") % 4).to(torch.int32)
    cfg = CONFIGS["llama3"]
    out = D.rope_append(cache, 0, x[0], x[1], x[2], pos, D.rope_table(ctx, cfg, dim))
    ctx.sync(60000)
    inv, f = D.rope_frequencies(cfg, dim)
    assert close_rows(out, *rope_reference(x[0], pos, inv, f, False))
    got = kv[0][table[:, 0].long(), pos.long()]
    assert close_rows(got, *rope_reference(x[1], pos, inv, f, False))
    assert torch.equal(kv[1][table[:, 0].long(), pos.long()], x[2])


def test_rope_append_is_captured_and_replayed(ctx):
    """A captured step replayed with other tokens, positions and pages."""
    stream = torch.cuda.Stream()
    c2 = C.Context(0, stream)
    cache, g = make_cache(c2, 22, [64, 64], 2, 64, 16, torch.bfloat16, fill=0.0)
    x = torch.zeros(3, 2, 2, 64, dtype=torch.bfloat16, device="cuda")
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    rope = D.rope_table(c2, CONFIGS["yarn"], 64)
    inv, f = D.rope_frequencies(CONFIGS["yarn"], 64)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        D.rope_append(cache, 0, x[0], x[1], x[2], pos, rope)
        stream.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=stream):
            out = D.rope_append(cache, 0, x[0], x[1], x[2], pos, rope)
    for p in ([3, 40], [63, 0]):
        x.copy_(torch.randn(3, 2, 2, 64, generator=g, device="cuda"))
        pos.copy_(torch.tensor(p, dtype=torch.int32))
        cache.block_tables.copy_(cache.block_tables.flip(0))
        torch.cuda.synchronize()
        gr.replay()
        torch.cuda.synchronize()
        assert close_rows(out, *rope_reference(x[0], pos, inv, f, False))
        wk, tk = rope_reference(x[1], pos, inv, f, False)
        for s in range(2):
            page, slot = int(cache.block_tables[s, p[s] // 16]), p[s] % 16
            assert close_rows(cache.k_layers[0][page, slot], wk[s], tk[s])
            assert torch.equal(cache.v_layers[0][page, slot], x[2, s])
    del gr
    c2.close()


def test_contexts_on_two_streams_at_once(ctx):
    """Two contexts on their own streams, neither the current one, working at the same time: the results of one
    after the other."""
    lens = [3000, 170, 0, 1024]
    ctxs = [C.Context(0, torch.cuda.Stream()) for _ in range(2)]
    made = [make_cache(c, 40 + i, lens, 2, 128, 16, torch.bfloat16) for i, c in enumerate(ctxs)]
    qs = [queries(g, 4, 2, 8, 128, torch.bfloat16) for _, g in made]
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    want = []
    for (cache, _), q in zip(made, qs):
        want.append(D.paged_attention(cache, 0, q, n, return_lse=True))
        cache.ctx.sync(60000)
    got = [[], []]
    for _ in range(10):
        for i, ((cache, _), q) in enumerate(zip(made, qs)):
            got[i].append(D.paged_attention(cache, 0, q, n, return_lse=True))
    for c in ctxs:
        c.sync(60000)
    for i in range(2):
        for out, lse in got[i]:
            assert torch.equal(out, want[i][0]) and torch.equal(lse, want[i][1])
        check_attention(ctxs[i], made[i][0], qs[i], lens)
    for c in ctxs:
        c.close()


def test_rope_append_reports_rows_outside_the_cache(ctx):
    cache, g = make_cache(ctx, 20, [32, 32], 1, 64, 16, torch.bfloat16, fill=0.0)
    x = torch.randn(3, 1, 64, generator=g, device="cuda").to(torch.bfloat16)
    rope = D.rope_table(ctx, C.RopeConfig(), 64)

    def call(pos, ids):
        D.rope_append(cache, 0, x, x, x, torch.tensor(pos, dtype=torch.int32, device="cuda"), rope,
                      seq_ids=torch.tensor(ids, dtype=torch.int32, device="cuda"))

    for pos, ids in (([0, 1, 32], [0, 0, 0]), ([0, 1, 2 ** 31 - 1], [0, 0, 0]), ([0, 1, 2], [0, 0, 2]),
                     ([0, 1, 2], [0, 0, -1])):
        call(pos, ids)
        with pytest.raises(Exception, match="block table"):
            ctx.sync(60000)
    cache.block_tables[1, 0] = cache.n_pages
    call([0, 1, 3], [0, 0, 1])
    with pytest.raises(Exception, match="block table"):
        ctx.sync(60000)
    call([0, 1, 17], [0, 0, 1])
    ctx.sync(60000)
    assert int((cache.v_layers[0].abs().sum(-1) != 0).sum()) == 3


# ----------------------------------------------------------------- refusals

def test_decode_refusals(ctx):
    cache, g = make_cache(ctx, 30, [32, 32], 2, 64, 16, torch.bfloat16)
    q = queries(g, 2, 1, 4, 64, torch.bfloat16)
    n = torch.tensor([3, 4], dtype=torch.int32, device="cuda")
    ok = D.paged_attention(cache, 0, q, n)
    assert ok.shape == q.shape
    for bad in (dict(q=q.float()), dict(q=q[..., :32]), dict(q=q[0]), dict(q=q.cpu()), dict(n=n.long()),
                dict(n=n[:1]), dict(n=n.cpu()), dict(q=queries(g, 2, 1, 3, 64, torch.bfloat16)), dict(layer=1),
                dict(layer=-1), dict(scale=math.nan), dict(scale=math.inf), dict(out=q.float()),
                dict(out=ok.transpose(0, 1)), dict(workspace=torch.empty(16, dtype=torch.uint8, device="cuda")),
                dict(q=queries(g, 3, 1, 4, 64, torch.bfloat16), n=torch.ones(3, dtype=torch.int32, device="cuda")),
                dict(q=q.transpose(2, 3).contiguous().transpose(2, 3))):
        kw = dict(layer=0, q=q, n=n, scale=None, out=None, workspace=None)
        kw.update(bad)
        with pytest.raises(ValueError):
            D.paged_attention(cache, kw["layer"], kw["q"], kw["n"], scale=kw["scale"], out=kw["out"],
                              workspace=kw["workspace"])
    k = cache.k_layers[0]
    for bad in (([k], [], cache.block_tables), ([k], [k[:1]], cache.block_tables), ([k.double()], [k.double()], cache.block_tables),
                ([k[0]], [k[0]], cache.block_tables), ([k], [k], cache.block_tables.long()),
                ([k], [k], cache.block_tables[0]), ([k.cpu()], [k.cpu()], cache.block_tables),
                ([k.transpose(2, 3)], [k.transpose(2, 3)], cache.block_tables)):
        with pytest.raises(ValueError):
            D.PagedCache(ctx, *bad)
    x = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device="cuda")
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    rope = D.rope_table(ctx, C.RopeConfig(), 64)
    big = D.rope_table(ctx, C.RopeConfig(), 128)
    half = D.RopeTable(rope.inv_freq.float(), 1.0)
    for bad in (dict(q=x.float()), dict(k=x[:, :1]), dict(v=x[:1]), dict(pos=pos.long()), dict(pos=pos[:1]),
                dict(ids=pos[:1]), dict(rope=big), dict(rope=half), dict(q_out=x[:, :1]), dict(q=x[0]), dict(layer=7)):
        kw = dict(layer=0, q=x, k=x, v=x, pos=pos, rope=rope, ids=None, q_out=None)
        kw.update(bad)
        with pytest.raises(ValueError):
            D.rope_append(cache, kw["layer"], kw["q"], kw["k"], kw["v"], kw["pos"], kw["rope"], seq_ids=kw["ids"],
                          q_out=kw["q_out"])
    # more tokens than sequences need seq_ids; overlapping rows cannot be written
    y = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError):
        D.rope_append(cache, 0, y, y, y, torch.zeros(3, dtype=torch.int32, device="cuda"), rope)
    shared = D.PagedCache(ctx, [k[:, :, :1].expand(-1, -1, 2, -1)], [k[:, :, :1].expand(-1, -1, 2, -1)],
                          cache.block_tables)
    with pytest.raises(ValueError):
        D.rope_append(shared, 0, x, x, x, pos, rope)
    endless = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16, device="cuda").expand(1, (1 << 30) + 1, 1, 64)
    with pytest.raises(Exception, match="2\\^30"):
        D.paged_attention(D.PagedCache(ctx, [endless], [endless], pos[:1, None].contiguous()), 0, q[:1, :, :1], n[:1])
    with pytest.raises(ValueError):
        D.rope_append(cache, 0, x, None, x, pos, rope)
    odd = torch.zeros(2, 16, 1, 7, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(Exception):
        D.paged_attention(D.PagedCache(ctx, [odd], [odd], cache.block_tables), 0, odd[:2, :1, :1], n)
    ctx.sync(60000)


def test_empty_calls(ctx):
    cache, g = make_cache(ctx, 31, [32], 2, 64, 16, torch.bfloat16)
    x = torch.zeros(0, 2, 64, dtype=torch.bfloat16, device="cuda")
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert D.rope_append(cache, 0, x, x, x, none, D.rope_table(ctx, C.RopeConfig(), 64)).shape == x.shape
    assert D.paged_attention(cache, 0, x[:, None], none).shape == (0, 1, 2, 64)
