"""The decode-step operators over the committed paged KV cache, as measured cases.

Three operators of one serving step: rotary positions on the new tokens' queries and keys with the K/V
rows put into their cache pages (``rope_append``), attention of the new tokens over the pages
(``paged_attention``), and verification of drafted tokens against the target's logits from given random
numbers (``verify_tokens``).  ``run`` computes each in elementary torch operations, or through
``commitllm_b200.decode`` where ``own`` is true.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
TARGET_BYTES = 1_400_000_000      # no drawn case moves more than the largest listed one


# ------------------------------------------------------------------ cases

def listed():
    return [
        # one short request alone on the GPU: latency of a decode step's attention (8B shape)
        {"name": "attend_one", "op": "attend", "seqs": 1, "new": 1, "longest": 700, "even": True, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "dtype": "bf16", "lse": False},
        # a full decode batch of ragged requests, one of them padding (8B shape)
        {"name": "attend_batch", "op": "attend", "seqs": 64, "new": 1, "longest": 8192, "even": False, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "dtype": "bf16", "lse": False},
        # two long documents (70B shape), with the log-sum that joins position shards of several GPUs
        {"name": "attend_long", "op": "attend", "seqs": 2, "new": 1, "longest": 131072, "even": True, "heads": 64,
         "kv_heads": 8, "dim": 128, "page": 16, "dtype": "bf16", "lse": True},
        # four drafted tokens and the last accepted one, verified in one pass (7B shape with 4 KV heads)
        {"name": "attend_drafts", "op": "attend", "seqs": 16, "new": 5, "longest": 8192, "even": False, "heads": 28,
         "kv_heads": 4, "dim": 128, "page": 16, "dtype": "f16", "lse": False},
        # a float32 validation run with a head size and a page size that are no powers of two
        {"name": "attend_f32", "op": "attend", "seqs": 5, "new": 2, "longest": 2500, "even": False, "heads": 12,
         "kv_heads": 4, "dim": 80, "page": 24, "dtype": "f32", "lse": True},
        # one token of one request: latency of the position step
        {"name": "rope_one", "op": "rope", "tokens": 1, "seqs": 1, "farthest": 8191, "heads": 32, "kv_heads": 8,
         "dim": 128, "rotary": 128, "interleaved": False, "scaling": "llama3", "page": 16, "dtype": "bf16"},
        # one token each of a full decode batch (70B shape)
        {"name": "rope_batch", "op": "rope", "tokens": 256, "seqs": 256, "farthest": 32767, "heads": 64,
         "kv_heads": 8, "dim": 128, "rotary": 128, "interleaved": False, "scaling": "llama3", "page": 16,
         "dtype": "bf16"},
        # a prefill chunk at the far end of a stretched context (70B shape)
        {"name": "rope_prefill", "op": "rope", "tokens": 8192, "seqs": 2, "farthest": 131071, "heads": 64,
         "kv_heads": 8, "dim": 128, "rotary": 128, "interleaved": False, "scaling": "yarn", "page": 16,
         "dtype": "bf16"},
        # neighbouring pairs over part of the head, in float32, with an odd number of tokens
        {"name": "rope_part", "op": "rope", "tokens": 1001, "seqs": 3, "farthest": 20000, "heads": 28, "kv_heads": 4,
         "dim": 128, "rotary": 64, "interleaved": True, "scaling": "linear", "page": 24, "dtype": "f32"},
        # one request's four drafts: latency of the acceptance step
        {"name": "verify_one", "op": "verify", "seqs": 1, "drafts": 4, "vocab": 128256, "dtype": "f32", "probs": True},
        # a batch's drafts against a draft model's distributions
        {"name": "verify_batch", "op": "verify", "seqs": 64, "drafts": 4, "vocab": 128256, "dtype": "f32",
         "probs": True},
        # drafts without a distribution (copied from the prompt), kept while they equal the token drawn
        {"name": "verify_match", "op": "verify", "seqs": 32, "drafts": 7, "vocab": 152064, "dtype": "bf16",
         "probs": False},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attend", "rope", "verify"])
    if op == "attend":
        kv_heads = rng.choice([1, 2, 4, 8])
        c = {"op": op, "seqs": _log(rng, 1, 96), "new": rng.choice([1, 1, 1, 2, 3, 5, 8]),
             "longest": _log(rng, 1, 131072), "even": rng.random() < 0.25, "heads": kv_heads * rng.choice([1, 3, 4, 7, 8]),
             "kv_heads": kv_heads, "dim": rng.choice([64, 80, 96, 128, 128, 128, 256]),
             "page": rng.choice([1, 8, 16, 16, 24, 32, 64, 100]), "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]),
             "lse": rng.random() < 0.5}
        # the padded float32 copies of the plain form bound the sizes too
        while work(c)["bytes"] > TARGET_BYTES or c["seqs"] * c["longest"] * c["kv_heads"] * c["dim"] > 600_000_000:
            c["longest"] = max(1, c["longest"] // 2)
        return c
    if op == "rope":
        kv_heads = rng.choice([1, 2, 4, 8])
        dim = rng.choice([64, 80, 96, 128, 128, 128, 256])
        c = {"op": op, "tokens": _log(rng, 1, 8192), "seqs": _log(rng, 1, 256), "farthest": _log(rng, 8192, 131072),
             "heads": kv_heads * rng.choice([1, 3, 4, 7, 8]), "kv_heads": kv_heads, "dim": dim,
             "rotary": rng.choice([dim, dim, dim // 2, dim // 4]), "interleaved": rng.random() < 0.4,
             "scaling": rng.choice(["none", "llama3", "linear", "yarn"]), "page": rng.choice([1, 8, 16, 16, 24, 32, 64]),
             "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}
        c["rotary"] -= c["rotary"] % 2
        c["seqs"] = min(c["seqs"], c["tokens"])
        return c
    c = {"op": op, "seqs": _log(rng, 1, 64), "drafts": rng.choice([0, 1, 2, 3, 4, 4, 5, 7]),
         "vocab": rng.choice([32000, 32001, 50257, 128256, 151936, 152064, _log(rng, 2, 200000)]),
         "dtype": rng.choice(["f32", "f32", "bf16", "f16"]), "probs": rng.random() < 0.5}
    return c


def work(case):
    c = case
    if c["op"] == "attend":
        # every cached K and V row once, the queries, the outputs; two products of 2 * dim operations
        rows = c["seqs"] * c["longest"] if c["even"] else c["seqs"] * c["longest"] * 5 // 8
        e = SIZE[c["dtype"]]
        q = c["seqs"] * c["new"] * c["heads"] * c["dim"] * e
        return {"bytes": 2 * rows * c["kv_heads"] * c["dim"] * e + 2 * q + 4 * (rows // c["page"]),
                "flops": 4 * rows * c["new"] * c["heads"] * c["dim"]}
    if c["op"] == "rope":
        # queries, keys and values read once and written once; three operations an element
        n = c["tokens"] * (c["heads"] + 2 * c["kv_heads"]) * c["dim"]
        return {"bytes": 2 * n * SIZE[c["dtype"]] + 8 * c["tokens"],
                "flops": 3 * c["tokens"] * (c["heads"] + c["kv_heads"]) * c["rotary"]}
    # every logits row once, and one row of draft probabilities a sequence (the refused position's)
    rows = c["seqs"] * (c["drafts"] + 1)
    e = SIZE[c["dtype"]]
    return {"bytes": rows * c["vocab"] * e + (c["seqs"] * c["vocab"] * 4 if c["probs"] and c["drafts"] else 0),
            "flops": 4 * rows * c["vocab"]}


# ----------------------------------------------------------------- inputs

def _pages(gen, lens, page, spare):
    """A block table of permuted pages: int32 [n_seqs, max pages], -1 where a sequence has no page."""
    need = [(n + page - 1) // page for n in lens]
    total = sum(need) + spare
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(max(need), 1)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, k in enumerate(need):
        table[s, :k] = order[at:at + k]
        at += k
    return table, total


def _lens(case, gen):
    c = case
    if c["even"]:
        return [c["longest"]] * c["seqs"]
    x = torch.rand(c["seqs"], generator=gen, device="cuda").cpu().tolist()
    lens = [max(1, int(c["longest"] * (0.25 + 0.75 * v))) for v in x]
    if c["seqs"] > 2:
        lens[1] = 0              # a padding row of a fixed batch
    return lens


def prepare(case, seed):
    c, dt = case, DTYPES.get(case["dtype"])
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)

    st = {"case": c}
    if c["op"] == "attend":
        lens = _lens(c, gen)
        table, pages = _pages(gen, lens, c["page"], 2)
        shape = (pages, c["page"], c["kv_heads"], c["dim"])
        st["k"] = torch.empty(shape, dtype=dt, device="cuda").normal_(generator=gen)
        st["v"] = torch.empty(shape, dtype=dt, device="cuda").normal_(generator=gen)
        st["q"] = (normal(c["seqs"], c["new"], c["heads"], c["dim"]) * 2).to(dt)
        st["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        st["table"] = table
    elif c["op"] == "rope":
        # consecutive positions of each sequence, ending somewhere before the farthest one
        n, S = c["tokens"], c["seqs"]
        per = [n // S + (1 if s < n % S else 0) for s in range(S)]
        ends = torch.rand(S, generator=gen, device="cuda").cpu().tolist()
        first = [int((c["farthest"] + 1 - k) * (0.75 + 0.25 * e)) for k, e in zip(per, ends)]
        need = [f + k for f, k in zip(first, per)]
        mb = max((m + c["page"] - 1) // c["page"] for m in need)
        # only the pages that the call writes are held: a long context's other pages are someone else's
        lo = [f // c["page"] for f in first]
        hi = [(m + c["page"] - 1) // c["page"] for m in need]
        total = sum((k + c["page"] - 1) // c["page"] + 1 for k in per) + 2
        order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
        table = torch.full((S, mb), -1, dtype=torch.int32, device="cuda")
        at = 0
        for s in range(S):
            table[s, lo[s]:hi[s]] = order[at:at + hi[s] - lo[s]]
            at += hi[s] - lo[s]
        pos = [f + i for f, k in zip(first, per) for i in range(k)]
        if n > 8:
            pos[n // 2] = -1     # a padding token
        st["positions"] = torch.tensor(pos, dtype=torch.int32, device="cuda")
        st["seq_ids"] = torch.tensor([s for s, k in enumerate(per) for _ in range(k)], dtype=torch.int32, device="cuda")
        st["table"] = table
        shape = (total, c["page"], c["kv_heads"], c["dim"])
        st["k_cache"] = torch.zeros(shape, dtype=dt, device="cuda")
        st["v_cache"] = torch.zeros(shape, dtype=dt, device="cuda")
        # views of one projection's output, as the model's fused product leaves them
        h, g, d = c["heads"], c["kv_heads"], c["dim"]
        qkv = normal(n, (h + 2 * g) * d).to(dt)
        st["q"] = qkv[:, : h * d].unflatten(1, (h, d))
        st["k"] = qkv[:, h * d: (h + g) * d].unflatten(1, (g, d))
        st["v"] = qkv[:, (h + g) * d:].unflatten(1, (g, d))
    else:
        n, k, V = c["seqs"], c["drafts"], c["vocab"]
        logits = normal(n, k + 1, V) * 3
        # most positions have one likely token, some are open; part of the vocabulary is ruled out
        likely = torch.randint(V, (n, k + 1), generator=gen, device="cuda")
        height = torch.rand(n, k + 1, 1, generator=gen, device="cuda") * 16 + 6
        logits.scatter_add_(2, likely[..., None], height)
        logits[:, :, 1::97] = -math.inf
        st["logits"] = logits.to(dt)
        temperature = torch.rand(n, generator=gen, device="cuda") * 0.8 + 0.6
        temperature[2::5] = 0.0
        st["temperature"] = temperature
        st["uniforms"] = torch.rand(n, k + 1, generator=gen, device="cuda", dtype=torch.float64)
        st["draft_probs"] = None
        if c["probs"]:
            guess = logits[:, :k] + normal(n, k, V)
            st["draft_probs"] = torch.softmax(guess, -1)
            drafts = (torch.multinomial(st["draft_probs"].reshape(n * k, V), 1, generator=gen).reshape(n, k)
                      if n * k else torch.zeros(n, k, dtype=torch.int64, device="cuda"))
        else:
            wrong = torch.randint(V, (n, k), generator=gen, device="cuda")
            drafts = torch.where(torch.rand(n, k, generator=gen, device="cuda") < 0.85, likely[:, :k], wrong)
        if n > 3 and k > 1:
            drafts[3, k - 1:] = -1      # a sequence with fewer drafts
        st["drafts"] = drafts.to(torch.int32)
    if own:
        from commitllm_b200 import commit as C
        from commitllm_b200 import decode as D
        st["ctx"] = C.Context()
        if c["op"] == "attend":
            st["cache"] = D.PagedCache(st["ctx"], [st["k"]], [st["v"]], st["table"])
        elif c["op"] == "rope":
            st["cache"] = D.PagedCache(st["ctx"], [st["k_cache"]], [st["v_cache"]], st["table"])
            st["rope"] = D.rope_table(st["ctx"], C.RopeConfig(**_rope_config(c)), c["rotary"])
    return st


# ------------------------------------------------------------- plain forms

def _rope_config(c):
    base = {"theta": 500000.0, "original_max_position_embeddings": 8192}
    return {"none": {"theta": 10000.0}, "llama3": {**base, "scaling": "llama3", "factor": 8.0},
            "linear": {"theta": 10000.0, "scaling": "linear", "factor": 4.0},
            "yarn": {**base, "scaling": "yarn", "factor": 16.0}}[c["scaling"]]


def _frequencies(c):
    """Angle per position of each rotated pair, float64, and the factor on both cos and sin."""
    cfg, half = _rope_config(c), c["rotary"] // 2
    i = torch.arange(half, dtype=torch.float64, device="cuda")
    inv = cfg["theta"] ** (-2.0 * i / c["rotary"])
    kind = cfg.get("scaling")
    if kind == "linear":
        return inv / cfg["factor"], 1.0
    if kind == "llama3":
        # wavelengths up to a quarter of the trained length stay, those over all of it stretch, linear between
        turns = cfg["original_max_position_embeddings"] * inv / (2 * math.pi)
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return inv * ((1 - keep) / cfg["factor"] + keep), 1.0
    if kind == "yarn":
        # pairs that turn over 32 times in the trained length stay, those under once stretch, linear in the index between
        def index(turns):
            return c["rotary"] * math.log(cfg["original_max_position_embeddings"] / (turns * 2 * math.pi)) / (2 * math.log(cfg["theta"]))
        lo, hi = max(math.floor(index(32.0)), 0), min(math.ceil(index(1.0)), c["rotary"] - 1)
        stretch = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        return inv * ((1 - stretch) + stretch / cfg["factor"]), 0.1 * math.log(cfg["factor"]) + 1.0
    return inv, 1.0


def _plain_rope(st):
    c = st["case"]
    inv, factor = _frequencies(c)
    pos = st["positions"]
    real = (pos >= 0)[:, None, None]
    angle = pos.double()[:, None] * inv[None, :]
    cos = (torch.cos(angle) * factor).float()[:, None, :]
    sin = (torch.sin(angle) * factor).float()[:, None, :]
    rot, half = c["rotary"], c["rotary"] // 2

    def turned(x):
        f = x.float()
        a, b = (f[..., 0:rot:2], f[..., 1:rot:2]) if c["interleaved"] else (f[..., :half], f[..., half:rot])
        x1, x2 = a * cos - b * sin, b * cos + a * sin
        y = torch.stack([x1, x2], -1).flatten(-2) if c["interleaved"] else torch.cat([x1, x2], -1)
        return torch.where(real, torch.cat([y, f[..., rot:]], -1), f).to(x.dtype)

    q, k = turned(st["q"]), turned(st["k"])
    at = torch.nonzero(pos >= 0)[:, 0]
    p = pos[at].long()
    page = st["table"][st["seq_ids"][at].long(), p // c["page"]].long()
    st["k_cache"][page, p % c["page"]] = k[at]
    st["v_cache"][page, p % c["page"]] = st["v"][at]
    return q, st["k_cache"], st["v_cache"]


def _plain_attend(st):
    c = st["case"]
    S, N, H, G, d = c["seqs"], c["new"], c["heads"], c["kv_heads"], c["dim"]
    table = st["table"].long().clamp(min=0)
    k = st["k"][table].reshape(S, -1, G, d).float()
    v = st["v"][table].reshape(S, -1, G, d).float()
    L = k.shape[1]
    q = st["q"].float().reshape(S, N, G, H // G, d).permute(0, 2, 1, 3, 4).reshape(S, G, N * (H // G), d)
    score = torch.matmul(q, k.permute(0, 2, 3, 1)) / math.sqrt(d)
    seen = st["lens"][:, None].long() - N + 1 + torch.arange(N, device="cuda")[None, :]
    seen = seen[:, None, :, None].expand(S, G, N, H // G).reshape(S, G, N * (H // G), 1)
    hidden = torch.arange(L, device="cuda")[None, None, None, :] >= seen
    score = score.masked_fill(hidden, -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    e = torch.exp(score - top)
    total = e.sum(-1, keepdim=True)
    out = torch.matmul(e, v.permute(0, 2, 1, 3)) / torch.where(total > 0, total, torch.ones_like(total))
    out = out.reshape(S, G, N, H // G, d).permute(0, 2, 1, 3, 4).reshape(S, N, H, d).to(st["q"].dtype)
    if not c["lse"]:
        return out
    lse = (torch.log(total) + top).reshape(S, G, N, H // G).permute(0, 2, 1, 3).reshape(S, N, H)
    return out, lse


def _plain_verify(st):
    # 64 bits throughout: a drawn token must not depend on how the sums were rounded
    c = st["case"]
    n, k, V = c["seqs"], c["drafts"], c["vocab"]
    logits, u = st["logits"].double(), st["uniforms"]
    greedy = (st["temperature"] == 0)[:, None]
    best = logits.argmax(-1)
    top = logits.amax(-1, keepdim=True)
    usable = torch.isfinite(top)[..., 0]
    t = st["temperature"].double()[:, None, None]
    w = torch.exp((logits - top) / torch.where(t > 0, t, torch.ones_like(t)))
    total = w.sum(-1)

    def drawn(weight, at):
        """The lowest index whose running sum passes at * sum."""
        run = torch.cumsum(weight, -1)
        x = (run <= at[..., None] * run[..., -1:]).sum(-1)
        last = V - 1 - torch.argmax((weight.flip(-1) > 0).to(torch.uint8), -1)
        return torch.minimum(x, last)

    x = st["drafts"].long()
    there = (x >= 0) & (x < V)
    xs = x.clamp(0, V - 1)
    if st["draft_probs"] is None:
        token = torch.where(greedy, best, drawn(w, u))
        kept = there & usable[:, :k] & (token[:, :k] == x)
        count = torch.cumprod(kept.long(), 1).sum(1)
        final = token.gather(1, count[:, None])[:, 0]
    else:
        probs = st["draft_probs"]
        p = torch.where(greedy, (best[:, :k] == xs).double(), w[:, :k].gather(2, xs[..., None])[..., 0] / total[:, :k])
        q = probs.gather(2, xs[..., None])[..., 0].double()
        kept = there & usable[:, :k] & (u[:, :k] * q < p)
        count = torch.cumprod(kept.long(), 1).sum(1)
        row = count[:, None, None].expand(n, 1, V)
        pw = w.gather(1, row)[:, 0] / total.gather(1, count[:, None])
        # at a refused draft the part of p above q is drawn from, elsewhere p itself
        refused = torch.cat([there, torch.zeros(n, 1, dtype=torch.bool, device="cuda")], 1).gather(1, count[:, None])
        if k:
            over = pw - probs.gather(1, row.clamp(max=k - 1))[:, 0].double()
            over = torch.where(over > 0, over, torch.zeros_like(over))
            pw = torch.where(refused & (over.sum(-1, keepdim=True) > 0), over, pw)
        final = torch.where(greedy[:, 0], best.gather(1, count[:, None])[:, 0], drawn(pw, u[:, k]))
    ends = usable.gather(1, count[:, None])[:, 0]
    final = torch.where(ends, final, torch.full_like(final, -1))
    at = torch.arange(k + 1, device="cuda")[None, :]
    padded = torch.cat([x, torch.full((n, 1), -1, device="cuda", dtype=x.dtype)], 1)
    tokens = torch.where(at < count[:, None], padded, torch.where(at == count[:, None], final[:, None], torch.full_like(padded, -1)))
    return tokens.to(torch.int32), (count + ends).to(torch.int32)


def run(state):
    st, c = state, state["case"]
    if own:
        from commitllm_b200 import decode as D
        if c["op"] == "attend":
            if c["lse"]:
                return D.paged_attention(st["cache"], 0, st["q"], st["lens"], return_lse=True)
            return D.paged_attention(st["cache"], 0, st["q"], st["lens"])
        if c["op"] == "rope":
            q = D.rope_append(st["cache"], 0, st["q"], st["k"], st["v"], st["positions"], st["rope"],
                              seq_ids=st["seq_ids"], interleaved=c["interleaved"])
            return q, st["k_cache"], st["v_cache"]
        return D.verify_tokens(st["ctx"], st["logits"], st["drafts"], st["uniforms"], st["temperature"],
                               draft_probs=st["draft_probs"])
    return {"attend": _plain_attend, "rope": _plain_rope, "verify": _plain_verify}[c["op"]](st)


# --------------------------------------------------- the definitions, in 64 bits

def exact(case, seed):
    c = case
    if c["op"] == "verify":
        return None                   # whole numbers: compared with the plain form
    st = prepare(c, seed)
    if c["op"] == "attend":
        S, N, H, G, d = c["seqs"], c["new"], c["heads"], c["kv_heads"], c["dim"]
        out = torch.zeros(S, N, H, d, dtype=torch.float64, device="cuda")
        lse = torch.full((S, N, H), -math.inf, dtype=torch.float64, device="cuda")
        lens = st["lens"].tolist()
        for s in range(S):
            rows = torch.arange(lens[s], device="cuda")
            page = st["table"][s].long()[rows // c["page"]]
            for g in range(G):
                k = st["k"][page, rows % c["page"], g].double()
                v = st["v"][page, rows % c["page"], g].double()
                for j in range(N):
                    m = lens[s] - N + 1 + j
                    if m <= 0:
                        continue
                    heads = slice(g * (H // G), (g + 1) * (H // G))
                    score = st["q"][s, j, heads].double() @ k[:m].T / math.sqrt(d)
                    lse[s, j, heads] = torch.logsumexp(score, -1)
                    out[s, j, heads] = torch.softmax(score, -1) @ v[:m]
        return (out, lse) if c["lse"] else out
    inv, factor = _frequencies(c)
    pos = st["positions"].tolist()
    ids = st["seq_ids"].tolist()
    on = torch.tensor([p >= 0 for p in pos], device="cuda")
    spin = torch.polar(torch.where(on[:, None], torch.full_like(inv, factor)[None, :], torch.ones_like(inv)[None, :]),
                       st["positions"].clamp(min=0).double()[:, None] * inv)[:, None, :]
    rot, half = c["rotary"], c["rotary"] // 2

    def turned(x):
        y = x.double().clone()
        first, second = (slice(0, rot, 2), slice(1, rot, 2)) if c["interleaved"] else (slice(0, half), slice(half, rot))
        z = torch.complex(y[..., first], y[..., second]) * spin
        y[..., first], y[..., second] = z.real, z.imag
        return y

    k_cache, v_cache = st["k_cache"].double(), st["v_cache"].double()
    rows = [i for i, p in enumerate(pos) if p >= 0]
    at = torch.tensor(rows, dtype=torch.long, device="cuda")
    seqs = torch.tensor([ids[i] for i in rows], dtype=torch.long, device="cuda")
    block = torch.tensor([pos[i] // c["page"] for i in rows], dtype=torch.long, device="cuda")
    slot = torch.tensor([pos[i] % c["page"] for i in rows], dtype=torch.long, device="cuda")
    page = st["table"][seqs, block].long()
    k_cache[page, slot] = turned(st["k"])[at]
    v_cache[page, slot] = st["v"].double()[at]
    return turned(st["q"]), k_cache, v_cache
