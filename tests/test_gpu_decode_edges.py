"""The decode step's operators at their edges: batches wider than a block, every attention kernel, masks of the lowest
value, weights of few bits, arguments that overlap.  References and tolerances are those of ``test_gpu_decode``
and ``test_gpu_verify`` where nothing else is said."""
import numpy as np
import pytest
import torch

from tests import test_gpu_decode as base
from commitllm_b200 import commit as C
from commitllm_b200 import decode as D

pytestmark = pytest.mark.gpu

DT = base.DT


# ------------------------------------------------- batches wider than a block

# (dtype, query heads, KV heads, new tokens, head size): one of each worker kernel, whose blocks scan the lengths of
# 128 (4 warps), 128 and 192 sequences at a time
WORKERS = [("bf16", 2, 1, 1, 64), ("f16", 6, 1, 4, 64), ("bf16", 8, 1, 5, 64), ("f32", 2, 1, 1, 64), ("bf16", 2, 1, 1, 66)]


@pytest.mark.parametrize("S", [128, 129, 192, 193, 256, 400])
@pytest.mark.parametrize("dtype,heads,kv,new,dim", WORKERS)
def test_attention_batches_wider_than_a_block(ctx, dtype, heads, kv, new, dim, S):
    rng = np.random.default_rng(S)
    lens = [int(x) for x in rng.integers(0, 150, S)]
    lens[1] = 0
    lens[-1] = 149                    # the last sequence has tiles
    cache, g = base.make_cache(ctx, S + dim, lens, kv, dim, 16, DT[dtype])
    q = base.queries(g, S, new, heads, dim, DT[dtype])
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = D.paged_attention(cache, 0, q, n)
    ctx.sync(60000)
    # the same sequences in batches that one pass over the lengths covers.  Their ranges are cut elsewhere, so the
    # sums run in another order: each side is within the reference's tolerance of the 64-bit values
    some = sorted(set([0, 1, 126, 127, S - 2, S - 1] + [x for x in (128, 191, 192, 255, 256) if x < S]))
    small = D.PagedCache(ctx, cache.k_layers, cache.v_layers, cache.block_tables[some].contiguous())
    ro, _, to, _ = base.reference(small, 0, q[some], [lens[s] for s in some])
    sub = torch.finfo(q.dtype).smallest_normal
    assert bool(((out[some].double() - ro).abs() <= to + sub).all())
    for a in range(0, S, 100):
        part = D.PagedCache(ctx, cache.k_layers, cache.v_layers, cache.block_tables[a:a + 100].contiguous())
        got = D.paged_attention(part, 0, q[a:a + 100], n[a:a + 100])
        ctx.sync(60000)
        # both within rel * (weighted mean of |v|) <= rel * max |v| and their rounding: rel as in the reference, with
        # scores of at most 150 keys
        e = torch.finfo(q.dtype).eps
        vmax = float(cache.v_layers[0].abs().max())
        kmax = float(cache.k_layers[0].abs().sum(-1).max()) * float(q.abs().max()) * dim ** -0.5
        rel = 2 * (dim + 4) * 2.0 ** -24 * kmax + 2.0 ** -21 + 2.0 ** -16 + 300 * 2.0 ** -24
        diff = (got.double() - out[a:a + 100].double()).abs()
        assert bool((diff <= 2 * rel * vmax + e * got.double().abs() + e * rel * vmax + sub).all())


# ----------------------------------------------------- every attention kernel

def kernel_of(dtype, rows, dim, wide):
    """Number of the kernel that ``variant_for`` in csrc/paged_attn.cu takes for this call: the rule restated."""
    size = 0 if dim <= 64 else 1 if dim <= 128 else 2
    if not wide:
        return {"f32": 25, "bf16": 27, "f16": 29}[dtype] + (size == 2)
    if dtype == "f32":
        return (23 if rows > 4 and size < 2 else 20) + size
    first = 0 if dtype == "bf16" else 10
    if rows <= 8:
        return first + size
    if rows <= 16 or size == 2:
        return first + 3 + size
    return first + (6 if -(-rows // 32) <= -(-rows // 48) else 8) + size


# (query heads, KV heads, new tokens): 4, 7, 12, 16, 24, 35, 48, 49 and 100 query rows of a KV head
LAYOUTS = [(8, 2, 1), (14, 2, 1), (6, 2, 4), (8, 2, 4), (12, 2, 4), (14, 2, 5), (24, 2, 4), (14, 2, 7), (40, 2, 5)]
DIMS = [64, 80, 128, 136, 256, 58, 66, 130, 250]      # the last four put rows off 16-byte boundaries
CALLS = [(dtype, *layout, dim) for dtype in ("bf16", "f16", "f32") for layout in LAYOUTS for dim in DIMS
         if dim in (64, 128, 256) or layout in ((8, 2, 1), (14, 2, 5))]


def rows_and_width(dtype, heads, kv, new, dim):
    return new * heads // kv, dim * (4 if dtype == "f32" else 2) % 16 == 0


@pytest.mark.parametrize("dtype,heads,kv,new,dim", CALLS)
def test_attention_every_kernel(ctx, dtype, heads, kv, new, dim):
    """Three sequences, split over many ranges and joined; then the same ones forty times over, most of them in one
    range each."""
    lens = [200, new - 1, 77]
    cache, g = base.make_cache(ctx, heads + dim, lens, kv, dim, 24, DT[dtype])
    q = base.queries(g, 3, new, heads, dim, DT[dtype])
    base.check_attention(ctx, cache, q, lens)
    many = D.PagedCache(ctx, cache.k_layers, cache.v_layers, cache.block_tables.repeat(40, 1))
    n = torch.tensor(lens * 40, dtype=torch.int32, device="cuda")
    out, lse = D.paged_attention(many, 0, q.repeat(40, 1, 1, 1), n, return_lse=True)
    ctx.sync(60000)
    ro, rl, to, tl = (x.repeat(40, *[1] * (x.dim() - 1)) for x in base.reference(cache, 0, q, lens))
    assert bool(((out.double() - ro).abs() <= to + torch.finfo(q.dtype).smallest_normal).all())
    empty = torch.isneginf(rl)
    assert torch.equal(torch.isneginf(lse), empty) and bool(((lse.double() - rl).abs()[~empty] <= tl[~empty]).all())


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads,dim", [(6, 64), (6, 128), (6, 256), (18, 64), (18, 128), (24, 128), (50, 128), (2, 130), (2, 256)])
def test_attention_kernels_ignore_what_is_masked(ctx, dtype, heads, dim):
    base.test_attention_ignores_what_is_masked(ctx, dtype, heads, dim)


# -------------------------------------------------------- weights of few bits

@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("heads,kv,new,dim", [(64, 64, 1, 64), (32, 32, 1, 128), (48, 4, 1, 128), (96, 4, 1, 64), (160, 4, 1, 128)])
def test_attention_small_weights_next_to_a_large_one(ctx, dtype, heads, kv, new, dim):
    """A key that takes almost all of the softmax and whose value is zero, and keys 15 - 20 nats below it: the output
    is theirs alone.

    Tolerance: the reference's, and what two 16-bit numbers leave of a weight.  The kernel's f16 weights are relative to
    a reference that the large key, the first one, sets to 2^-7 of itself, or that has come down to 2^-7 of the largest
    of a warp's 16 or 32 keys; rounding to a multiple of 2^-24 is off by at most 2^-25, so by 2^-32 of the large
    key's weight among its neighbours, and by 2^-18 of the largest weight among its own 32 keys elsewhere.
    """
    dt, S, L = DT[dtype], 8, 2048
    cache, g = base.make_cache(ctx, heads + dim, [L] * S, kv, dim, 16, dt, fill=0.0)
    k, v = cache.k_layers[0], cache.v_layers[0]
    # the score of a key is its first element
    k[..., 0] = (torch.rand(k.shape[:-1], generator=g, device="cuda") * 5).to(dt)
    v.copy_(torch.rand(v.shape, generator=g, device="cuda") * 1000 + 500)
    for s in range(S):
        k[int(cache.block_tables[s, 0]), 0, :, 0] = 20.0
        v[int(cache.block_tables[s, 0]), 0] = 0.0
    q = torch.zeros(S, new, heads, dim, dtype=dt, device="cuda")
    q[..., 0] = 1.0
    lens = [L] * S
    lens[3] = 700
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = D.paged_attention(cache, 0, q, n, scale=1.0)
    ctx.sync(60000)
    few = [0, 3]
    small = D.PagedCache(ctx, [k], [v], cache.block_tables[few].contiguous())
    ro, _, to, _ = base.reference(small, 0, q[few], [lens[s] for s in few], scale=1.0)
    for i, s in enumerate(few):
        kk, vv = base.rows_of(small, 0, i, lens[s])
        p = torch.softmax(kk[:, :, 0], 0)                                  # [keys, kv heads]
        pad = -len(p) % 32
        top = torch.nn.functional.pad(p, (0, 0, 0, pad)).view(-1, 32, kv).amax(1).repeat_interleave(32, 0)[:len(p)]
        unit = 2.0 ** -18 * top
        unit[:32] = 2.0 ** -32 * p[0]
        extra = torch.einsum("ng,ngd->gd", unit, vv.abs()).repeat_interleave(heads // kv, 0)
        assert float(ro[i].abs().min()) > 1e-3                             # well above f16's smallest numbers
        assert bool(((out[s].double() - ro[i]).abs() <= to[i] + extra).all()), float(((out[s].double() - ro[i]) / ro[i]).abs().max())


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("heads,kv,dim", [(16, 16, 128), (40, 2, 128)])
def test_attention_scores_that_rise_and_fall(ctx, dtype, heads, kv, dim):
    """Runs of 64 keys by turns 40 nats above and below each other, falling all the way, and rising all the way."""
    dt, S, L = DT[dtype], 3, 1600
    cache, g = base.make_cache(ctx, heads, [L] * S, kv, dim, 16, dt)
    k = cache.k_layers[0]
    run = torch.arange(L, device="cuda") // 64
    level = [run % 2 * 40.0, -3.0 * run, 3.0 * run]
    for s in range(S):
        p = torch.arange(L, device="cuda")
        page = cache.block_tables[s].long()[p // 16]
        k[page, p % 16] = 0.0
        k[page, p % 16, :, 0] = (level[s][:, None] + torch.rand(L, kv, generator=g, device="cuda")).to(dt)
    q = torch.zeros(S, 1, heads, dim, dtype=dt, device="cuda")
    q[..., 0] = 1.0
    base.check_attention(ctx, cache, q, [L, L, L - 5], scale=1.0)


# ------------------------------------------------------------------ refusals


@pytest.mark.parametrize("layer", [2 ** 32, -2 ** 32, 2 ** 31, 2 ** 40])
def test_layers_past_32_bits_are_refused(ctx, layer):
    cache, g = base.make_cache(ctx, 51, [32, 32], 2, 64, 16, torch.bfloat16)
    before = [t.clone() for t in (cache.k_layers[0], cache.v_layers[0])]
    x = torch.randn(2, 2, 64, generator=g, device="cuda").to(torch.bfloat16)
    pos = torch.ones(2, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        D.rope_append(cache, layer, x, x, x, pos, D.rope_table(ctx, C.RopeConfig(), 64))
    with pytest.raises(ValueError):
        D.paged_attention(cache, layer, x[:, None].contiguous(), pos)
    ctx.sync(60000)
    assert torch.equal(before[0], cache.k_layers[0]) and torch.equal(before[1], cache.v_layers[0])


def test_cache_sizes_past_32_bits_are_refused(ctx):
    one = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16, device="cuda")
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    D.PagedCache(ctx, [one], [one], table)
    for shape in ((1, 2 ** 32 + 16, 1, 64), (1, 1, 2 ** 32 + 1, 64), (1, 2 ** 31, 1, 64)):
        with pytest.raises(ValueError, match="2\\^31"):
            D.PagedCache(ctx, [one.expand(shape)], [one.expand(shape)], table)


def test_rope_append_refuses_rows_that_overlap(ctx):
    """Outputs that share memory among themselves: queries expanded over heads or tokens, K and V in one buffer."""
    cache, g = base.make_cache(ctx, 50, [32, 32], 2, 64, 16, torch.bfloat16)
    x = torch.randn(2, 2, 64, generator=g, device="cuda").to(torch.bfloat16)
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    rope = D.rope_table(ctx, C.RopeConfig(), 64)
    one = torch.zeros(1, 1, 64, dtype=torch.bfloat16, device="cuda")
    flat = torch.zeros(64 * 4, dtype=torch.bfloat16, device="cuda")
    for bad in (one.expand(2, 2, 64), flat[:128].view(1, 2, 64).expand(2, -1, -1), flat[:128].view(2, 1, 64).expand(-1, 2, -1),
                flat.as_strided((2, 2, 64), (128, 32, 1)), flat.as_strided((2, 2, 64), (32, 128, 1)),
                flat.as_strided((2, 2, 64), (64, 64, 1))):
        with pytest.raises(ValueError, match="overlap"):
            D.rope_append(cache, 0, x, x, x, pos, rope, q_out=bad)
    for good in (flat.as_strided((2, 2, 64), (64, 128, 1)), flat.view(2, 2, 64)):
        D.rope_append(cache, 0, x, x, x, pos, rope, q_out=good)
        ctx.sync(60000)
        assert torch.equal(good, x)                       # position 0 turns nothing
    same = D.PagedCache(ctx, [cache.k_layers[0]], [cache.k_layers[0]], cache.block_tables)
    with pytest.raises(ValueError, match="overlap"):
        D.rope_append(same, 0, x, x, x, pos, rope)
    D.paged_attention(same, 0, x[:, None].contiguous(), pos)          # reading one buffer as both is fine
    ctx.sync(60000)
