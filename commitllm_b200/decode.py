"""The decode step over the committed paged cache.

What a serving engine does between two commits, on the same
``[num_pages, block_size, n_kv_heads, head_dim]`` cache that
:func:`commitllm_b200.commit.kv_commit` hashes in place:

* :func:`rope_append` -- rotary positions of the new tokens' queries and keys,
  K and V rows into their pages;
* :func:`paged_attention` -- attention of each sequence's newest tokens over its
  pages (one token, or the last token and its drafts);
* :func:`verify_tokens` -- how many drafted tokens the target's logits keep, and
  the token after them, from given random numbers.

Lengths, positions, block tables and draws are read on the device, and a call
allocates only its outputs and workspace (through torch's caching allocator),
so a step can be captured in a CUDA graph on the context's stream and replayed
while its tensors change in place.  Serving only: outputs carry no gradients.  As everywhere in this package, calls are
ordered on the context's stream: inputs made on another stream need that
stream's work ordered before them.
"""
from __future__ import annotations

import ctypes
import math
import struct
from dataclasses import dataclass
from typing import Optional, Sequence

import torch

from . import _lib
from ._lib import KvDesc, check, lib
from .commit import Context, KvCacheView, RopeConfig, _ptrs

_CACHE_DTYPES = {torch.bfloat16: _lib.VC_DTYPE_BF16, torch.float16: _lib.VC_DTYPE_F16,
                 torch.float32: _lib.VC_DTYPE_F32}


# A decode step runs these calls layer by layer, often on a batch of one, where the
# host's share of a call is longer than the GPU's.  So the arguments go over in one
# packed buffer, each call tests everything in one expression, and looks for what to
# complain about only when that fails.
_ROPE = struct.Struct("21qdq")
_ATTEND = struct.Struct("11qd4q")
_VERIFY = struct.Struct("18q")
_VERIFY_ROW_BYTES = 1024        # vc_verify_tokens_workspace: this many for each logits row
_decode_call = None


def _call(which: int, n: int, slots: bytes) -> None:
    global _decode_call
    if _decode_call is None:
        _decode_call = lib().vc_decode_call
    status = _decode_call(which, n, slots)
    if status:
        check(status)


def _handle(ctx: Context) -> int:
    return ctx._h.value or ctx.handle.value


def _empty(ctx: Context, like: torch.Tensor, shape, dtype=None) -> torch.Tensor:
    # Context.empty without the stream switch when the stream is current already;
    # new_empty costs two thirds of torch.empty
    if torch._C._cuda_getCurrentRawStream(ctx.device) == ctx.stream.cuda_stream:
        return like.new_empty(shape) if dtype is None else like.new_empty(shape, dtype=dtype)
    return ctx.empty(shape, dtype=dtype or like.dtype)


def _empty_like(ctx: Context, t: torch.Tensor) -> torch.Tensor:
    if torch._C._cuda_getCurrentRawStream(ctx.device) == ctx.stream.cuda_stream:
        return torch.empty_like(t, memory_format=torch.contiguous_format)
    return ctx.empty(t.shape, dtype=t.dtype)


def _on(ctx: Context, t: torch.Tensor, name: str) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.get_device() != ctx.device:
        raise ValueError(f"{name} must be a CUDA tensor on device {ctx.device}")


def _index(ctx: Context, t: torch.Tensor, name: str, shape) -> int:
    """Address of a contiguous int32 tensor of this shape."""
    if not (isinstance(t, torch.Tensor) and t.dtype is torch.int32 and t.get_device() == ctx.device and t.shape == shape
            and t.is_contiguous()):
        _on(ctx, t, name)
        raise ValueError(f"{name} must be a contiguous int32 tensor of shape {list(shape)}")
    return t.data_ptr()


class PagedCache:
    """The paged K/V cache of a range of layers, its descriptor built once.

    ``k_layers[l]`` / ``v_layers[l]``: CUDA tensors ``[num_pages, block_size,
    n_kv_heads, head_dim]`` of one dtype (bfloat16, float16 or float32), shape
    and strides, contiguous within a head; ``block_tables``: int32 CUDA
    ``[n_seqs, max_blocks]``, read on the device by every call (update it in
    place).  A contiguous cache ``[n_seqs, max_len, heads, dim]`` is one page a
    sequence: ``block_tables = arange(n_seqs)[:, None]``.  Only the addresses
    are kept with the tensors; replacing a tensor needs a new ``PagedCache``.
    """

    def __init__(self, ctx: Context, k_layers: Sequence[torch.Tensor], v_layers: Sequence[torch.Tensor],
                 block_tables: torch.Tensor):
        if len(k_layers) == 0 or len(k_layers) != len(v_layers):
            raise ValueError("k_layers and v_layers must be non-empty and of equal length")
        k0 = k_layers[0]
        for t in list(k_layers) + list(v_layers):
            _on(ctx, t, "K/V layer")
            if t.dtype != k0.dtype or t.shape != k0.shape or t.stride() != k0.stride():
                raise ValueError("all K/V layers must share one dtype, shape and strides")
        if k0.dtype not in _CACHE_DTYPES:
            raise ValueError(f"unsupported cache dtype {k0.dtype}")
        if k0.dim() != 4 or 0 in k0.shape:
            raise ValueError("K/V layers must be [num_pages, block_size, n_kv_heads, head_dim]")
        if k0.stride(3) != 1 and k0.shape[3] > 1:
            raise ValueError("head_dim must be contiguous")
        _on(ctx, block_tables, "block_tables")
        if block_tables.dtype != torch.int32 or block_tables.dim() != 2 or 0 in block_tables.shape \
                or not block_tables.is_contiguous():
            raise ValueError("block_tables must be a contiguous int32 [n_seqs, max_blocks] tensor")
        self.ctx = ctx
        self.k_layers, self.v_layers, self.block_tables = list(k_layers), list(v_layers), block_tables
        self.n_layers = len(k_layers)
        self.dtype = k0.dtype
        self.n_pages, self.block_size, self.n_kv_heads, self.head_dim = (int(x) for x in k0.shape)
        self.n_seqs, self.max_blocks = (int(x) for x in block_tables.shape)
        if max(self.n_layers, *k0.shape[1:], *block_tables.shape) >= 1 << 31:      # the descriptor's integers
            raise ValueError("layers, block_size, n_kv_heads, head_dim, n_seqs and max_blocks must be below 2^31")
        d = KvDesc()
        d.n_layers, d.n_kv_heads, d.head_dim = self.n_layers, self.n_kv_heads, self.head_dim
        d.dtype, d.n_seqs = _CACHE_DTYPES[k0.dtype], self.n_seqs
        d.block_tables, d.block_size, d.max_blocks_per_seq = block_tables.data_ptr(), self.block_size, self.max_blocks
        d.stride_page, d.stride_row, d.stride_head = k0.stride(0), k0.stride(1), k0.stride(2)
        # Elements reachable from the base pointer of each layer buffer.
        d.cache_elems = sum((s - 1) * st for s, st in zip(k0.shape, k0.stride())) + 1
        kp = _ptrs([t.data_ptr() for t in self.k_layers])
        vp = _ptrs([t.data_ptr() for t in self.v_layers])
        self._keep = (kp, vp)
        d.k_layers = ctypes.cast(kp, ctypes.POINTER(ctypes.c_void_p))
        d.v_layers = ctypes.cast(vp, ctypes.POINTER(ctypes.c_void_p))
        self.desc = d
        self._ref = ctypes.byref(d)
        self._addr = ctypes.addressof(d)
        self._workspace = {}        # (n_new, n_heads) -> bytes

    def view(self, seq_lens: Sequence[int], layer_base: int = 0) -> KvCacheView:
        """The rows 0..seq_lens[s]-1 of the first ``len(seq_lens)`` sequences, for
        :func:`commitllm_b200.commit.kv_commit` (which takes bfloat16 and float32)."""
        return KvCacheView(k_layers=self.k_layers, v_layers=self.v_layers, seq_lens=seq_lens,
                           block_tables=self.block_tables, layer_base=layer_base)

    def workspace_bytes(self, n_new: int, n_heads: int) -> int:
        """Workspace of :func:`paged_attention` for this many new tokens and query heads."""
        n = self._workspace.get((n_new, n_heads))
        if n is None:
            out = ctypes.c_size_t()
            check(lib().vc_paged_attention_workspace(self.ctx.handle, self._ref, n_new, n_heads, ctypes.byref(out)))
            n = self._workspace[(n_new, n_heads)] = out.value
        return n


# ---------------------------------------------------------------------------
# Rotary positions
# ---------------------------------------------------------------------------

@dataclass
class RopeTable:
    """Angle per position of each rotated pair (float64, on the device) and the
    factor on cos and sin."""
    inv_freq: torch.Tensor
    factor: float

    @property
    def rotary_dim(self) -> int:
        return 2 * int(self.inv_freq.numel())


def rope_frequencies(cfg: RopeConfig, rotary_dim: int, beta_fast: float = 32.0, beta_slow: float = 1.0,
                     attention_factor: Optional[float] = None):
    """``(inv_freq list, factor)`` of ``cfg`` for ``rotary_dim`` rotated elements.

    theta^(-2i/rotary_dim), then by ``cfg.scaling``: None unscaled;
    ``"linear"`` over ``factor``; ``"llama3"`` as the transcript scales it
    (crates/verilm-core/src/constants.rs:253-297); ``"yarn"`` over ``factor``
    for pairs that turn less than ``beta_slow`` times in the original length,
    unscaled above ``beta_fast`` turns, linear in the pair's index between, with
    cos and sin times ``attention_factor`` (default 0.1 ln(factor) + 1).
    """
    r = int(rotary_dim)
    if r < 2 or r % 2:
        raise ValueError(f"rotary_dim {r} must be even and at least 2")
    if not cfg.theta > 0:
        raise ValueError("theta must be positive")
    inv = [1.0 / math.pow(cfg.theta, (2 * i) / r) for i in range(r // 2)]
    factor = 1.0
    if cfg.scaling in (None, ""):
        return inv, factor
    if not cfg.factor > 0:
        raise ValueError("factor must be positive")
    length = float(cfg.original_max_position_embeddings)
    if cfg.scaling == "linear":
        inv = [f / cfg.factor for f in inv]
    elif cfg.scaling == "llama3":
        if not 0 < cfg.low_freq_factor < cfg.high_freq_factor:
            raise ValueError("llama3 scaling needs 0 < low_freq_factor < high_freq_factor")
        out = []
        for f in inv:
            wave = 2.0 * math.pi / f
            if wave > length / cfg.low_freq_factor:
                f = f / cfg.factor
            elif not wave < length / cfg.high_freq_factor:
                smooth = (length / wave - cfg.low_freq_factor) / (cfg.high_freq_factor - cfg.low_freq_factor)
                f = f * ((1.0 - smooth) / cfg.factor + smooth)
            out.append(f)
        inv = out
    elif cfg.scaling == "yarn":
        if not (cfg.theta > 1 and length > 0 and 0 < beta_slow < beta_fast):
            raise ValueError("yarn scaling needs theta > 1, a positive original length and 0 < beta_slow < beta_fast")

        def index(turns):      # the pair that turns this often in the original length
            return r * math.log(length / (turns * 2.0 * math.pi)) / (2.0 * math.log(cfg.theta))
        lo = max(math.floor(index(beta_fast)), 0)
        hi = min(math.ceil(index(beta_slow)), r - 1)
        span = max(hi - lo, 1e-3)
        inv = [f * (1.0 - s) + f / cfg.factor * s
               for f, s in ((f, min(max((i - lo) / span, 0.0), 1.0)) for i, f in enumerate(inv))]
        factor = 0.1 * math.log(cfg.factor) + 1.0 if cfg.factor > 1 else 1.0
        if attention_factor is not None:
            factor = float(attention_factor)
    else:
        raise ValueError(f"unknown rope scaling {cfg.scaling!r}")
    return inv, factor


def rope_table(ctx: Context, cfg: RopeConfig, rotary_dim: int, **kw) -> RopeTable:
    """:func:`rope_frequencies` on the device, for :func:`rope_append` (``kw``: the yarn options)."""
    inv, factor = rope_frequencies(cfg, rotary_dim, **kw)
    return RopeTable(ctx.to_device(torch.tensor(inv, dtype=torch.float64)), factor)


def _rows(ctx: Context, t: torch.Tensor, name: str, n: int, heads: Optional[int], dim: int, dtype) -> None:
    _on(ctx, t, name)
    if t.dtype != dtype or t.dim() != 3 or t.shape[0] != n or t.shape[2] != dim or \
            (heads is not None and t.shape[1] != heads):
        raise ValueError(f"{name} must be {dtype} [{n}, {'heads' if heads is None else heads}, {dim}]")
    if t.stride(2) != 1:
        raise ValueError(f"{name} must be contiguous within a head")


def rope_append(cache: PagedCache, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                positions: torch.Tensor, rope: RopeTable, seq_ids: Optional[torch.Tensor] = None,
                interleaved: bool = False, q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotate the queries and keys of ``n`` tokens and write their K and V rows.

    q: ``[n, n_heads, head_dim]``; k, v: ``[n, n_kv_heads, head_dim]``, in the
    cache's dtype, any token and head strides (views of one fused projection);
    positions: int32 ``[n]``, the row of each token in its sequence (negative:
    padding, its query is copied and nothing is written); seq_ids: int32 ``[n]``,
    the token's sequence (default: token t is sequence t's).  The first
    ``rope.rotary_dim`` elements of each head are rotated, in halves ``(i, i +
    rotary_dim/2)`` or, ``interleaved``, in neighbours ``(2i, 2i+1)``.  Returns
    the rotated queries (``q_out``, which may be ``q`` and otherwise overlaps no
    input; its rows may not overlap, nor a layer's K and V; new by default).  Two
    tokens of a call must not share a row.  A position or page outside the
    cache is raised by the next ``ctx.sync()``.
    """
    ctx = cache.ctx
    if not isinstance(q, torch.Tensor) or q.dim() != 3:
        raise ValueError("q must be [n_tokens, n_heads, head_dim]")
    n, heads, _ = q.shape
    dev, dt, dim = ctx.device, cache.dtype, cache.head_dim
    kv = (n, cache.n_kv_heads, dim)
    if not (isinstance(k, torch.Tensor) and isinstance(v, torch.Tensor)):
        raise ValueError("k and v must be CUDA tensors")
    qs, ks, vs = q.stride(), k.stride(), v.stride()
    if not (q.dtype is dt and k.dtype is dt and v.dtype is dt and q.shape[2] == dim and k.shape == kv and v.shape == kv
            and qs[2] == 1 and ks[2] == 1 and vs[2] == 1 and q.get_device() == dev and k.get_device() == dev
            and v.get_device() == dev):
        _rows(ctx, q, "q", n, None, dim, dt)
        _rows(ctx, k, "k", n, cache.n_kv_heads, dim, dt)
        _rows(ctx, v, "v", n, cache.n_kv_heads, dim, dt)
    pos = _index(ctx, positions, "positions", (n,))
    ids = 0 if seq_ids is None else _index(ctx, seq_ids, "seq_ids", (n,))
    inv = rope.inv_freq
    if not (inv.dtype is torch.float64 and inv.get_device() == dev and inv.is_contiguous()):
        raise ValueError(f"rope.inv_freq must be a contiguous float64 tensor on device {dev}")
    if q_out is None:
        q_out = _empty_like(ctx, q)
    else:
        _rows(ctx, q_out, "q_out", n, heads, dim, dt)
    if n == 0:
        return q_out
    os = q_out.stride()
    _call(_lib.VC_CALL_ROPE_APPEND, 23,
          _ROPE.pack(_handle(ctx), cache._addr, layer, n, pos, ids, heads, q.data_ptr(), qs[0], qs[1], q_out.data_ptr(),
                     os[0], os[1], k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], inv.data_ptr(),
                     2 * inv.numel(), rope.factor, interleaved))
    return q_out


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------

def paged_attention(cache: PagedCache, layer: int, q: torch.Tensor, seq_lens: torch.Tensor,
                    scale: Optional[float] = None, return_lse: bool = False, out: Optional[torch.Tensor] = None,
                    workspace: Optional[torch.Tensor] = None):
    """Attention of the newest ``n_new`` tokens of each sequence over its cached rows.

    q: ``[n_seqs, n_new, n_heads, head_dim]`` in the cache's dtype, any strides
    outside a head (``n_heads`` a multiple of the cache's KV heads; sequence s is
    row s of the block table); seq_lens: int32 ``[n_seqs]`` on the device, the
    cached rows of each sequence with the new tokens' own (0 or less: a padding row of
    the batch; more than the block table holds: raised by the next ``ctx.sync()``).
    New token j sees rows ``p < seq_lens[s] - n_new + 1 + j``; a token that sees none
    gets zeros, and what a token does not see cannot reach its output.  Sums are f32
    in an order that depends on n_new and on the batch's lengths: a token's output
    may differ in its last bits between batches, not between equal calls.
    ``scale`` defaults to ``head_dim ** -0.5``.  Returns ``out`` (shaped as q),
    or ``(out, lse)`` with the float32 natural log of each softmax's sum
    ``[n_seqs, n_new, n_heads]`` (-inf where nothing is seen), from which shards of
    one sequence on several GPUs are joined.  ``workspace``: a uint8 CUDA tensor
    of at least ``cache.workspace_bytes(n_new, n_heads)`` that no concurrent call
    uses (new by default).
    """
    ctx = cache.ctx
    if not isinstance(q, torch.Tensor) or q.dim() != 4:
        raise ValueError("q must be [n_seqs, n_new, n_heads, head_dim]")
    S, N, H, D = q.shape
    qs = q.stride()
    if not (q.dtype is cache.dtype and D == cache.head_dim and qs[3] == 1 and S <= cache.n_seqs and N > 0 and H > 0
            and q.get_device() == ctx.device):
        _on(ctx, q, "q")
        if q.dtype != cache.dtype or D != cache.head_dim:
            raise ValueError(f"q must be {cache.dtype} [n_seqs, n_new, n_heads, {cache.head_dim}]")
        if qs[3] != 1:
            raise ValueError("q must be contiguous within a head")
        if S > cache.n_seqs:
            raise ValueError(f"{S} sequences, the block table has {cache.n_seqs}")
        raise ValueError("n_new and n_heads must be at least 1")
    lens = _index(ctx, seq_lens, "seq_lens", (S,))
    if out is None:
        out = _empty_like(ctx, q)
    else:
        _on(ctx, out, "out")
        if out.dtype != cache.dtype or out.shape != q.shape or not out.is_contiguous():
            raise ValueError("out must be contiguous, of q's shape and dtype")
    lse = _empty(ctx, q, (S, N, H), torch.float32) if return_lse else None
    need = cache._workspace.get((N, H)) or cache.workspace_bytes(N, H)
    if workspace is None:
        workspace = _empty(ctx, seq_lens, need // 4)        # (a multiple of 16 bytes)
    else:
        _on(ctx, workspace, "workspace")
        if workspace.dtype != torch.uint8 or not workspace.is_contiguous():
            raise ValueError("workspace must be a contiguous uint8 tensor")
        need = workspace.numel()
    if S:
        _call(_lib.VC_CALL_PAGED_ATTENTION, 16,
              _ATTEND.pack(_handle(ctx), cache._addr, layer, S, N, H, q.data_ptr(), qs[0], qs[1], qs[2], lens,
                           D ** -0.5 if scale is None else scale, out.data_ptr(), 0 if lse is None else lse.data_ptr(),
                           workspace.data_ptr(), need))
    return (out, lse) if return_lse else out


# ---------------------------------------------------------------------------
# Drafted tokens
# ---------------------------------------------------------------------------

def verify_tokens(ctx: Context, logits: torch.Tensor, drafts: torch.Tensor, uniforms: torch.Tensor,
                  temperature: torch.Tensor, draft_probs: Optional[torch.Tensor] = None,
                  workspace: Optional[torch.Tensor] = None):
    """The drafted tokens that the target keeps and the token after them.

    logits: ``[n_seqs, n_draft + 1, vocab]`` float32, bfloat16 or float16, row i
    the target's at draft i (any strides between rows); drafts: int32 ``[n_seqs,
    n_draft]`` (a value outside the vocabulary, such as -1, ends a sequence's
    drafts); uniforms: float64 ``[n_seqs, n_draft + 1]`` in [0, 1); temperature:
    float32 ``[n_seqs]``, 0 for greedy.  With ``draft_probs`` (float32 ``[n_seqs,
    n_draft, vocab]``, the distributions the drafts were drawn from) draft i is kept
    while ``uniforms[i] * q_i(x_i) < p_i(x_i)``, and the next token is drawn with
    the last uniform from ``max(p - q, 0)`` where a draft was refused, else from
    ``p``.  Without, the token at i is the one ``p_i`` gives for ``uniforms[i]``, and
    drafts are kept while they equal it: the tokens are then those drawn one by one
    from the same logits, whatever was drafted.  A draw from weights w is the lowest v whose
    running sum passes ``u * sum(w)``.

    Returns ``(tokens int32 [n_seqs, n_draft + 1], counts int32 [n_seqs])``: each
    sequence's new tokens, padded with -1.  A reached row with a NaN, a +inf or
    nothing above -inf ends its sequence without a drawn token.  Rejected drafts'
    K/V rows stay in their pages until the next step writes them; commit with the
    lengths that ``counts`` gives.
    """
    if not isinstance(logits, torch.Tensor) or logits.dim() != 3:
        raise ValueError("logits must be [n_seqs, n_draft + 1, vocab]")
    S, N, V = logits.shape
    ls = logits.stride()
    dev = ctx.device
    if not (logits.dtype in _CACHE_DTYPES and N > 0 and V > 0 and (ls[2] == 1 or V == 1) and logits.get_device() == dev):
        _on(ctx, logits, "logits")
        raise ValueError("logits must be float32, bfloat16 or float16 [n_seqs, n_draft + 1, vocab], contiguous within a row")
    x = _index(ctx, drafts, "drafts", (S, N - 1))
    for t in (uniforms, temperature) if draft_probs is None else (uniforms, temperature, draft_probs):
        if not isinstance(t, torch.Tensor):
            raise ValueError("uniforms, temperature and draft_probs must be CUDA tensors")
    if not (uniforms.dtype is torch.float64 and uniforms.shape == (S, N) and uniforms.get_device() == dev
            and uniforms.is_contiguous()):
        raise ValueError(f"uniforms must be contiguous float64 [{S}, {N}] on device {dev}")
    if not (temperature.dtype is torch.float32 and temperature.shape == (S,) and temperature.get_device() == dev
            and temperature.is_contiguous()):
        raise ValueError(f"temperature must be contiguous float32 [{S}] on device {dev}")
    probs, ps = 0, (0, 0)
    if draft_probs is not None:
        ps = draft_probs.stride()
        if not (draft_probs.dtype is torch.float32 and draft_probs.shape == (S, N - 1, V) and (ps[2] == 1 or V == 1)
                and draft_probs.get_device() == dev):
            raise ValueError(f"draft_probs must be float32 [{S}, {N - 1}, {V}] on device {dev}, contiguous within a row")
        probs = draft_probs.data_ptr()
    tokens = _empty(ctx, drafts, (S, N))
    counts = _empty(ctx, drafts, (S,))
    if S == 0:
        return tokens, counts
    if workspace is None:
        need = S * N * _VERIFY_ROW_BYTES
        workspace = _empty(ctx, drafts, need // 4)
    else:
        _on(ctx, workspace, "workspace")
        if workspace.dtype != torch.uint8 or not workspace.is_contiguous():
            raise ValueError("workspace must be a contiguous uint8 tensor")
        need = workspace.numel()
    _call(_lib.VC_CALL_VERIFY_TOKENS, 18,
          _VERIFY.pack(_handle(ctx), S, N - 1, V, logits.data_ptr(), _CACHE_DTYPES[logits.dtype], ls[0], ls[1], probs, ps[0],
                       ps[1], x, uniforms.data_ptr(), temperature.data_ptr(), tokens.data_ptr(), counts.data_ptr(),
                       workspace.data_ptr(), need))
    return tokens, counts
