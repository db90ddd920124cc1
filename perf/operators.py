"""Cases of the paged serving operators (``hf_attention_normalizers_b200.serving``).

Three operators work on one paged KV cache, in the order a serving step calls them:

* ``append``  the new tokens' K/V rows go into their sequences' pages;
* ``chunk``   a ragged chunk of new tokens per sequence (one token, a prompt piece, or a mix)
              attends over the whole cached context, optionally adding every key's attention
              weight to the cache's accumulators;
* ``evict``   every KV head of a sequence keeps its ``budget`` most attended keys (and the most
              recent ones), moved to the front of the sequence's pages.

``own = False`` computes them from elementary torch operations in 32 bits, ``own = True`` calls the
framework.  Sequence lengths come from the case alone, values and page order from the seed.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _case(name, op, batch, new, context, hkv=8, group=4, dim=128, page=32, dtype="bf16", **kw):
    """``new`` and ``context``: the longest sequence's new tokens and keys (the new ones included); with
    ``ragged`` the others are shorter, down to one token on an almost empty cache."""
    c = dict(op=op, batch=batch, new=new, context=context, hkv=hkv, group=group, dim=dim, page=page, dtype=dtype,
             ragged=True, norm="softmax1", weights=False, budget=0, recent=0)
    c.update(kw)
    if name is not None:
        c["name"] = name
    return c


def listed():
    return [
        # one decode step's writes: 64 sequences, a token each (latency)
        _case("append-decode-64", "append", 64, 1, 4096),
        # a prefill step's writes: 8 prompt pieces of up to 2048 tokens
        _case("append-prefill-8x2048", "append", 8, 2048, 8192, ragged=False),
        # the smallest attention call: a few sequences decode on short contexts (latency)
        _case("chunk-decode-4x2k", "chunk", 4, 1, 2048, norm="softmax1"),
        # one long document is decoded: few rows, the key axis has to be split
        _case("chunk-decode-1x32k", "chunk", 1, 1, 32768, ragged=False),
        # a mixed batch: decoding sequences beside prompt pieces, odd lengths
        _case("chunk-mixed-16x255x8k", "chunk", 16, 255, 8191),
        # a prompt piece on a long document, the largest attention call
        _case("chunk-prefill-1x1024x32k", "chunk", 1, 1024, 32768, ragged=False),
        # sparse normalizers on prompt pieces, the second with 64-wide heads, fp16 and 16-token pages
        _case("chunk-sparsemax-4x256x8k", "chunk", 4, 256, 8192, norm="sparsemax"),
        _case("chunk-entmax15-8x130x3k", "chunk", 8, 130, 3001, norm="entmax15", hkv=4, group=7, dim=64, page=16,
              dtype="fp16"),
        # decoding while the keys' weights are collected for eviction
        _case("weights-decode-32x8k", "chunk", 32, 1, 8192, weights=True),
        # prompt pieces with collected weights
        _case("weights-prefill-2x512x8k", "chunk", 2, 512, 8192, weights=True, ragged=False),
        # a few sequences fall back to their budget while they decode (latency)
        _case("evict-4x2k-to-1k", "evict", 4, 0, 2049, budget=1024, recent=64),
        # a full batch of long contexts is cut to a quarter
        _case("evict-32x16k-to-4k", "evict", 32, 0, 16384, budget=4096, recent=128, ragged=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: sizes log-uniform over the ranges that the listed cases span."""
    op = rng.choice(["append", "chunk", "chunk", "chunk", "evict"])
    hkv, group, dim = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 5, 7, 8]), rng.choice([64, 128])
    kw = dict(hkv=hkv, group=group, dim=dim, page=rng.choice([16, 32, 64]), dtype=rng.choice(["bf16", "fp16"]),
              ragged=rng.random() < 0.7)
    if op == "append":
        new = _log(rng, 1, 2048)
        batch = _log(rng, 1, max(1, min(64, 16384 // new)))
        return _case(None, op, batch, new, _log(rng, new, 8192), **kw)
    if op == "evict":
        context = _log(rng, 256, 16384)
        batch = _log(rng, 1, max(1, min(32, 32 * 16384 // context)))
        budget = _log(rng, 64, context)
        return _case(None, op, batch, 0, context, budget=budget, recent=rng.randint(0, budget // 4), **kw)
    norm = rng.choice(["softmax1", "softmax1", "sparsemax", "entmax15"])
    most = (1 << 30) if norm == "softmax1" else (1 << 28)  # score elements
    new = 1 if rng.random() < 0.3 else _log(rng, 2, 1024)
    context = _log(rng, max(64, new), 32768)
    context = max(new, min(context, most // (new * hkv * group)))
    batch = _log(rng, 1, max(1, min(64, most // (new * hkv * group * context))))
    return _case(None, op, batch, new, context, norm=norm, weights=rng.random() < 0.4, **kw)


def _lengths(case):
    """(new tokens, keys) of every sequence, from the case alone: the first has both in full."""
    rng = random.Random("%(batch)d/%(new)d/%(context)d/%(page)d" % case)
    new, ctx = [], []
    for i in range(case["batch"]):
        n, c = case["new"], case["context"]
        if case["ragged"] and i > 0:
            n = rng.randint(1, n) if n else 0
            c = max(n, rng.randint(max(1, c // 8), c))
        new.append(n)
        ctx.append(c)
    return new, ctx


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def prepare(case, seed):
    dev, dt = "cuda", DTYPES[case["dtype"]]
    g = torch.Generator(device=dev).manual_seed(seed)
    new, ctx = _lengths(case)
    ps, hkv, dim, b = case["page"], case["hkv"], case["dim"], case["batch"]
    pages = [-(-c // ps) for c in ctx]
    order = torch.randperm(sum(pages) + 3, generator=g, device=dev).to(torch.int32)  # the pool has pages of nobody too
    at = torch.tensor([0] + pages, device=dev).cumsum(0)
    col = torch.arange(max(pages), device=dev)
    idx = (at[:-1, None] + col[None, :]).clamp(max=sum(pages) - 1)
    table = torch.where(col[None, :] < torch.tensor(pages, device=dev)[:, None], order[idx], torch.zeros_like(order[idx]))
    slots = (sum(pages) + 3) * ps
    cu = torch.tensor([0] + new, device=dev).cumsum(0).to(torch.int32)

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device=dev, dtype=torch.float32) * scale).to(dt)

    s = {"op": case["op"], "norm": case["norm"], "page": ps, "group": case["group"], "dtype": dt,
         "max_q": max(new), "max_k": max(ctx), "budget": case["budget"], "recent": case["recent"],
         "key_cache": normal(slots, hkv, dim), "value_cache": normal(slots, hkv, dim),
         "table": table.contiguous(), "cu": cu, "lens": torch.tensor(ctx, device=dev, dtype=torch.int32),
         "key_weights": None}
    if case["op"] != "chunk" or case["weights"]:
        # what earlier steps collected: most keys got little, a few got much
        u = torch.rand(hkv, slots, generator=g, device=dev)
        s["key_weights"] = (-torch.log(u.clamp_min(1e-7))) ** 3 / 8.0
    if case["op"] == "append":
        s["key"], s["value"] = normal(sum(new), hkv, dim), normal(sum(new), hkv, dim)
    if case["op"] == "chunk":
        # normalised queries with a gain of two: scores of standard deviation two
        s["query"] = normal(sum(new), hkv * case["group"], dim, scale=2.0)
    return s


# ---------------------------------------------------------------------------
# the operators' plain forms
# ---------------------------------------------------------------------------
def _slots(s):
    """Physical cache row and validity of every logical position, [B, max_k]."""
    pos = torch.arange(s["max_k"], device=s["table"].device)
    phys = s["table"].long()[:, pos // s["page"]] * s["page"] + pos % s["page"]
    return pos, phys, pos[None, :] < s["lens"][:, None]


def _owner(s, total):
    """Sequence and offset within it of every packed row."""
    row = torch.arange(total, device=s["cu"].device)
    b = torch.searchsorted(s["cu"][1:].contiguous(), row.to(torch.int32), right=True)
    return b, row - s["cu"].long()[b]


def _plain_append(s):
    b, i = _owner(s, s["key"].shape[0])
    n = (s["cu"][1:] - s["cu"][:-1]).long()
    pos = s["lens"].long()[b] - n[b] + i
    row = s["table"].long()[b, pos // s["page"]] * s["page"] + pos % s["page"]
    s["key_cache"][row] = s["key"]
    s["value_cache"][row] = s["value"]
    s["key_weights"][:, row] = 0.0
    return s["key_cache"], s["value_cache"], s["key_weights"]


def _plain_probabilities(x, norm):
    """Rows of scores (-inf: masked) to probabilities."""
    if norm == "softmax1":
        m = x.amax(-1, keepdim=True).clamp_min(0.0)
        e = torch.exp(x - m)
        return e / (e.sum(-1, keepdim=True) + torch.exp(-m))
    z = x if norm == "sparsemax" else x * 0.5
    top = z.amax(-1, keepdim=True)
    z = z - torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    y = z.sort(dim=-1, descending=True).values.clamp_min(-8.0)  # the threshold is at least the maximum minus one
    k = torch.arange(1, y.shape[-1] + 1, device=y.device, dtype=y.dtype)
    s1 = y.cumsum(-1)
    if norm == "sparsemax":
        t = (s1 - 1.0) / k
    else:
        mean = s1 / k
        d = (1.0 - ((y * y).cumsum(-1) - s1 * mean)) / k
        t = mean - torch.sqrt(d.clamp_min(0.0))
    n = (t <= y).sum(-1, keepdim=True).clamp_min(1)
    p = (z - t.gather(-1, n - 1)).clamp_min(0.0)
    return p if norm == "sparsemax" else p * p


def _plain_chunk(s):
    pos, phys, valid = _slots(s)
    q, kc, vc = s["query"], s["key_cache"], s["value_cache"]
    total, hq, dim = q.shape
    hkv, g = kc.shape[1], s["group"]
    batch, n = phys.shape[0], s["max_q"]
    k = torch.where(valid[:, :, None, None], kc[phys].float(), 0.0).permute(0, 2, 3, 1)      # [B, Hkv, D, L]
    v = torch.where(valid[:, :, None, None], vc[phys].float(), 0.0).transpose(1, 2)          # [B, Hkv, L, D]
    start, count = s["cu"].long()[:-1], (s["cu"][1:] - s["cu"][:-1]).long()
    i = torch.arange(n, device=q.device)
    rows = (start[:, None] + i[None, :]).clamp(max=total - 1)
    qp = q[rows].float().view(batch, n, hkv, g, dim).permute(0, 2, 3, 1, 4).reshape(batch, hkv, g * n, dim)
    x = torch.matmul(qp, k).mul_(dim ** -0.5).view(batch, hkv, g, n, -1)
    limit = (s["lens"].long() - count)[:, None] + i[None, :]                                 # last visible key of a row
    see = (pos[None, None, :] <= limit[:, :, None]) & valid[:, None, :] & (i[None, :] < count[:, None])[:, :, None]
    x = x.masked_fill_(~see[:, None, None], float("-inf"))
    p = _plain_probabilities(x, s["norm"])
    out = torch.matmul(p.view(batch, hkv, g * n, -1), v).view(batch, hkv, g, n, dim)
    bi, ii = _owner(s, total)
    out = out.permute(0, 3, 1, 2, 4)[bi, ii].reshape(total, hq, dim).to(s["dtype"])
    if s["key_weights"] is None:
        return out
    s["key_weights"][:, phys[valid]] += p.sum((2, 3)).permute(1, 0, 2)[:, valid]
    return out, s["key_weights"]


def _plain_evict(s):
    pos, phys, valid = _slots(s)
    kc, vc, kw, budget = s["key_cache"], s["value_cache"], s["key_weights"], s["budget"]
    hkv = kc.shape[1]
    w = kw[:, phys].transpose(0, 1)                                                            # [B, Hkv, L]
    late = pos[None, :] >= (s["lens"] - s["recent"])[:, None]
    w = torch.where((late & valid)[:, None], float("inf"), torch.where(valid[:, None], w, float("-inf")))
    kept = w.sort(dim=-1, descending=True, stable=True).indices[..., :budget]                  # ties: the lowest position
    kept = kept.sort(dim=-1).values
    head = torch.arange(hkv, device=kc.device)[None, :, None].expand_as(kept)
    live = kept < s["lens"][:, None, None]
    src = phys[:, None].expand(-1, hkv, -1).gather(-1, kept)[live]
    dst = phys[:, None, :budget].expand(-1, hkv, -1)[live]
    head = head[live]
    kc[dst, head] = kc[src, head]
    vc[dst, head] = vc[src, head]
    kw[head, dst] = kw[head, src]
    kept = torch.where(live, kept, -1).to(torch.int32)
    return s["lens"].clamp(max=budget), kept, kc, vc, kw


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    s = state
    if not own:
        return {"append": _plain_append, "chunk": _plain_chunk, "evict": _plain_evict}[s["op"]](s)
    from hf_attention_normalizers_b200 import serving

    if s["op"] == "append":
        serving.paged_append(s["key"], s["value"], s["key_cache"], s["value_cache"], s["table"], s["cu"], s["lens"],
                             s["page"], key_weights=s["key_weights"])
        return s["key_cache"], s["value_cache"], s["key_weights"]
    if s["op"] == "chunk":
        out = serving.paged_chunk_attention(s["query"], s["key_cache"], s["value_cache"], s["table"], s["cu"],
                                            s["lens"], s["page"], normalizer=s["norm"], key_weights=s["key_weights"],
                                            max_seqlen_q=s["max_q"], max_seqlen_k=s["max_k"])
        return out if s["key_weights"] is None else (out, s["key_weights"])
    lens, kept = serving.paged_evict(s["key_cache"], s["value_cache"], s["key_weights"], s["table"], s["lens"],
                                     s["page"], s["budget"], recent=s["recent"], max_seqlen_k=s["max_k"])
    return lens, kept, s["key_cache"], s["value_cache"], s["key_weights"]


# ---------------------------------------------------------------------------
# floors and exact values
# ---------------------------------------------------------------------------
def work(case):
    new, ctx = _lengths(case)
    hkv, hq, d = case["hkv"], case["hkv"] * case["group"], case["dim"]
    table = 4 * sum(-(-c // case["page"]) for c in ctx)
    if case["op"] == "append":  # K and V rows read and written, the accumulators cleared
        return {"bytes": sum(new) * hkv * (8 * d + 4) + table, "flops": 0}
    if case["op"] == "evict":
        # every weight read once; the kept K/V rows and weights read and written
        kept = sum(min(c, case["budget"]) for c in ctx if c > case["budget"])
        return {"bytes": hkv * (4 * sum(ctx) + kept * (8 * d + 4) + 4 * case["batch"] * case["budget"]) + table,
                "flops": 0}
    pairs = sum(n * c - n * (n - 1) // 2 for n, c in zip(new, ctx))  # visible (token, key) pairs
    nbytes = 4 * d * hq * sum(new) + 4 * d * hkv * sum(ctx) + table
    if case["weights"]:
        nbytes += 8 * hkv * sum(ctx)
    return {"bytes": nbytes, "flops": 4 * d * hq * pairs}


def _threshold64(x, norm):
    """Row thresholds by Newton's method from the left, from max - 1 (float64; the sums are convex in t)."""
    z = x if norm == "sparsemax" else x / 2
    t = z.amax(-1, keepdim=True) - 1.0
    for _ in range(60):
        r = (z - t).clamp_min(0.0)
        if norm == "sparsemax":
            step = (r.sum(-1, keepdim=True) - 1.0) / (r > 0).sum(-1, keepdim=True).clamp_min(1)
        else:
            step = (r.square().sum(-1, keepdim=True) - 1.0) / (2.0 * r.sum(-1, keepdim=True)).clamp_min(1e-300)
        t = t + step.clamp_min(0.0)
        if float(step.abs().max()) < 1e-15:
            break
    return (z - t).clamp_min(0.0)


def exact(case, seed):
    """Outputs and accumulators of the attention from its definition, float64, a sequence and KV head at a time.
    The other operators only move values."""
    if case["op"] != "chunk":
        return None
    s = prepare(case, seed)
    new, ctx = _lengths(case)
    g, dim = case["group"], case["dim"]
    out = torch.zeros(s["query"].shape, dtype=torch.float64, device="cuda")
    weights = None if s["key_weights"] is None else s["key_weights"].double()
    at = 0
    for b, (n, c) in enumerate(zip(new, ctx)):
        j = torch.arange(c, device="cuda")
        slot = s["table"][b].long()[j // case["page"]] * case["page"] + j % case["page"]
        hidden = j[None, :] > (c - n + torch.arange(n, device="cuda"))[:, None]
        for h in range(case["hkv"]):
            k, v = s["key_cache"][slot, h].double(), s["value_cache"][slot, h].double()
            for e in range(h * g, (h + 1) * g):
                x = (s["query"][at:at + n, e].double() @ k.T) / math.sqrt(dim)
                x = x.masked_fill(hidden, float("-inf"))
                if case["norm"] == "softmax1":
                    e_x = torch.exp(x)  # |scores| stay far below 700
                    p = e_x / (1.0 + e_x.sum(-1, keepdim=True))
                else:
                    p = _threshold64(x, case["norm"])
                    p = p if case["norm"] == "sparsemax" else p.square()
                out[at:at + n, e] = p @ v
                if weights is not None:
                    weights[h, slot] += p.sum(0)
        at += n
    return out if weights is None else (out, weights)
