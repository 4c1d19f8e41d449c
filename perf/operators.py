"""Workloads of the paged-cache serving operators: page plan, QK-norm + rotation + cache append, and
single-token attention over the paged cache.

A case is one call of one operator. ``run`` computes it in plain fp32 torch operations, or, with
``own`` set, through ``mint_b200.ops``. Request lengths are spread evenly between the case's bounds
and shuffled by the seed, so a case moves the same bytes whatever its seed. Pages of a request are
scattered over the pool, as they are after requests have come and gone.

Caches are ``[pages, kv heads, page size, head dim]``.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
DEVICE = "cuda"


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decoding step of a small batch, two requests already finished: pure latency
        {"name": "plan_decode", "op": "plan", "requests": 32, "lo": 1, "hi": 2047, "new_lo": 1, "new_hi": 1,
         "idle": 2, "page": 16},
        # admission of many prompts at once: 256 prompts, about 131 thousand tokens
        {"name": "plan_prompts", "op": "plan", "requests": 256, "lo": 0, "hi": 0, "new_lo": 1, "new_hi": 1023,
         "idle": 0, "page": 16},
        # one interactive user of the 12-layer model (6 heads of 128): latency
        {"name": "append_one", "op": "append", "tokens": 1, "hq": 6, "hkv": 6, "dim": 128, "page": 16, "span": 2048,
         "type": "bf16"},
        # a decoding batch of the 2B model (16 query heads over 4)
        {"name": "append_decode", "op": "append", "tokens": 64, "hq": 16, "hkv": 4, "dim": 128, "page": 16,
         "span": 4096, "type": "bf16"},
        # a few prompts together, odd token count, fp16, heads of 64
        {"name": "append_prompts_fp16", "op": "append", "tokens": 4093, "hq": 8, "hkv": 2, "dim": 64, "page": 32,
         "span": 512, "type": "fp16"},
        # the largest prompt batch: 16 full rows of the 2B model
        {"name": "append_prefill", "op": "append", "tokens": 65536, "hq": 16, "hkv": 4, "dim": 128, "page": 64,
         "span": 4096, "type": "bf16"},
        # one short conversation on the 12-layer model: latency
        {"name": "attend_short", "op": "attend", "tokens": 1, "lo": 37, "hi": 37, "hq": 6, "hkv": 6, "dim": 128,
         "page": 16, "window": -1, "alibi": False, "type": "bf16"},
        # one long document: a single query per head has to fill the whole GPU
        {"name": "attend_long", "op": "attend", "tokens": 1, "lo": 131072, "hi": 131072, "hq": 16, "hkv": 4,
         "dim": 128, "page": 64, "window": -1, "alibi": False, "type": "bf16"},
        # a windowed layer of the 12-layer model (window = a quarter of 2048), ragged batch
        {"name": "attend_window", "op": "attend", "tokens": 32, "lo": 1, "hi": 2048, "hq": 6, "hkv": 6, "dim": 128,
         "page": 16, "window": 512, "alibi": False, "type": "bf16"},
        # an ordinary ragged batch on the 2B model
        {"name": "attend_batch", "op": "attend", "tokens": 24, "lo": 64, "hi": 4096, "hq": 16, "hkv": 4, "dim": 128,
         "page": 16, "window": -1, "alibi": False, "type": "bf16"},
        # multi-query attention with the linear distance bias, fp16, heads of 64, many short requests
        {"name": "attend_mqa_alibi", "op": "attend", "tokens": 128, "lo": 1, "hi": 1000, "hq": 12, "hkv": 1,
         "dim": 64, "page": 32, "window": -1, "alibi": True, "type": "fp16"},
        # long contexts in a full batch: about a million cached tokens, 2.2 GB
        {"name": "attend_large", "op": "attend", "tokens": 64, "lo": 1024, "hi": 32768, "hq": 16, "hkv": 4,
         "dim": 128, "page": 16, "window": -1, "alibi": False, "type": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("plan", "append", "attend", "attend"))
    page = rng.choice((8, 16, 32, 64, 128))
    if op == "plan":
        n = _log(rng, 1, 1024)
        if rng.random() < 0.5:
            return {"op": op, "requests": n, "lo": 1, "hi": _log(rng, 2, 8192), "new_lo": 1, "new_hi": 1,
                    "idle": rng.randint(0, n // 4), "page": page}
        hi = _log(rng, 2, max(3, 200000 // n))
        return {"op": op, "requests": n, "lo": 0, "hi": rng.choice((0, 300)), "new_lo": 1, "new_hi": hi,
                "idle": rng.randint(0, n // 4), "page": page}
    dim = rng.choice((64, 128, 128, 256))
    hkv = rng.choice((1, 2, 4, 6, 8))
    group = rng.choice((1, 2, 3, 4, 8, 12))
    kind = rng.choice(("bf16", "bf16", "fp16"))
    if op == "append":
        most = max(2, min(65536, 200_000_000 // (hkv * (group + 2) * dim)))
        return {"op": op, "tokens": _log(rng, 1, most), "hq": hkv * group, "hkv": hkv, "dim": dim, "page": page,
                "span": _log(rng, 64, 16384), "type": kind}
    n = _log(rng, 1, 256)
    most = max(2, min(131072, 400_000_000 // (n * hkv * dim)))
    hi = _log(rng, 1, most)
    return {"op": op, "tokens": n, "lo": rng.randint(1, hi), "hi": hi, "hq": hkv * group, "hkv": hkv, "dim": dim,
            "page": page, "window": rng.choice((-1, -1, _log(rng, 1, 4096))), "alibi": rng.random() < 0.25,
            "type": kind}


# ----------------------------------------------------------------------------------------- inputs
def _spread(n, lo, hi):
    """n lengths, evenly spread over [lo, hi]."""
    return [lo + int((hi - lo) * (i + 0.5) / n) if hi > lo else lo for i in range(n)]


def _pages(length, page):
    return -(-length // page)


def _shuffled(values, gen):
    order = torch.randperm(len(values), generator=gen)
    return torch.tensor(values, dtype=torch.int64)[order]


def _normal(shape, gen, dtype):
    return torch.randn(shape, generator=gen, device=DEVICE, dtype=dtype)


def _block_tables(lens, page, gen):
    """[requests, width] int32 tables over a shuffled pool, and the pool's size in pages."""
    counts = (lens + page - 1) // page
    total = int(counts.sum())
    pool = total + max(4, total // 16)
    ids = torch.randperm(pool, generator=gen)[:total]
    width = int(counts.max())
    at = torch.arange(width)[None, :]
    first = torch.cumsum(counts, 0) - counts
    table = ids[(first[:, None] + at).clamp(max=total - 1)]
    table = torch.where(at < counts[:, None], table, torch.zeros_like(table))
    return table.to(torch.int32), pool


def prepare(case, seed):
    host = torch.Generator().manual_seed(seed)
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    page = case["page"]
    if case["op"] == "plan":
        n = case["requests"]
        seq = _shuffled(_spread(n, case["lo"], case["hi"]), host)
        new = _shuffled([0] * case["idle"] + _spread(n - case["idle"], case["new_lo"], case["new_hi"]), host)
        n_tokens = n if case["new_hi"] == 1 else int(new.sum())  # a decoding step keeps its padded shape
        width = int(((seq + new + page - 1) // page).max()) + 1
        have = (seq + page - 1) // page
        pool = int(have.sum()) + int(((seq + new + page - 1) // page).sum()) + 8
        ids = torch.randperm(pool, generator=host)
        used = int(have.sum())
        first = torch.cumsum(have, 0) - have
        at = torch.arange(width)[None, :]
        table = torch.where(at < have[:, None], ids[(first[:, None] + at).clamp(max=max(used - 1, 0))], -1)
        head = torch.tensor([used], dtype=torch.int32, device=DEVICE)
        return {"op": "plan", "seq_lens": seq.to(DEVICE, torch.int32), "new_lens": new.to(DEVICE, torch.int32),
                "tables": table.to(DEVICE, torch.int32), "free_pages": ids.to(DEVICE, torch.int32),
                "free_head": head, "page": page, "n_tokens": n_tokens}
    dtype = DTYPES[case["type"]]
    hq, hkv, dim, n = case["hq"], case["hkv"], case["dim"], case["tokens"]
    if case["op"] == "append":
        span = case["span"]
        pool = _pages(n, page) + 4
        freq = 1.0 / (10000.0 ** (torch.arange(0, dim, 2, dtype=torch.float32, device=DEVICE) / dim))
        angle = torch.arange(span, dtype=torch.float32, device=DEVICE)[:, None] * freq[None, :]
        start = int(torch.randint(span, (1,), generator=host))
        positions = (torch.arange(n) + start) % span
        slots = torch.randperm(pool, generator=host)[:, None] * page + torch.arange(page)[None, :]
        slots = slots.reshape(-1)[:n]
        return {"op": "append", "qkv": _normal((n, (hq + 2 * hkv) * dim), gen, dtype), "hq": hq, "hkv": hkv,
                "dim": dim, "page": page,
                "q_scale": 0.1 * _normal((dim,), gen, torch.float32), "k_scale": 0.1 * _normal((dim,), gen, torch.float32),
                "cos": angle.cos(), "sin": angle.sin(),
                "positions": positions.to(DEVICE, torch.int32), "slots": slots.to(DEVICE, torch.int32),
                "k_pages": _normal((pool, hkv, page, dim), gen, dtype),
                "v_pages": _normal((pool, hkv, page, dim), gen, dtype)}
    lens = _shuffled(_spread(n, case["lo"], case["hi"]), host)
    table, pool = _block_tables(lens, page, host)
    slopes = None
    if case["alibi"]:
        slopes = torch.exp2(-8.0 * torch.arange(1, hq + 1, dtype=torch.float32, device=DEVICE) / hq)
    return {"op": "attend", "q": _normal((n, hq, dim), gen, dtype),
            "k_pages": _normal((pool, hkv, page, dim), gen, dtype),
            "v_pages": _normal((pool, hkv, page, dim), gen, dtype),
            "tables": table.to(DEVICE), "positions": (lens - 1).to(DEVICE, torch.int32),
            "window": case["window"], "slopes": slopes, "page": page}


# ------------------------------------------------------------------------------------ plain forms
def _plan(s):
    page = s["page"]
    seq, new = s["seq_lens"].long(), s["new_lens"].long()
    have = (seq + page - 1) // page
    need = (seq + new + page - 1) // page - have
    before = torch.cumsum(need, 0) - need
    ends = torch.cumsum(new, 0)
    at = torch.arange(s["tables"].shape[1], device=seq.device)[None, :]
    k = at - have[:, None]
    fresh = (k >= 0) & (k < need[:, None])
    pick = (s["free_head"].long() + before[:, None] + k).clamp(0, s["free_pages"].numel() - 1)
    s["tables"].copy_(torch.where(fresh, s["free_pages"][pick], s["tables"]))
    i = torch.arange(s["n_tokens"], device=seq.device)
    rows = torch.searchsorted(ends, i, right=True)
    live = rows < seq.numel()
    r = rows.clamp(max=seq.numel() - 1)
    pos = seq[r] + i - (ends[r] - new[r])
    pos = torch.where(live, pos, 0)
    slots = s["tables"][r, pos // page].long() * page + pos % page
    neg = torch.full_like(pos, -1)
    out = {"positions": torch.where(live, pos, neg), "slots": torch.where(live, slots, neg),
           "rows": torch.where(live, r, neg), "ends": ends, "seq_lens": seq + new,
           "free_head": s["free_head"] + need.sum()}
    return {**{name: t.to(torch.int32) for name, t in out.items()}, "tables": s["tables"]}


def _norm(x, scale):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * (1.0 + scale)


def _rotate(x, cos, sin):
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)


def _append(s):
    hq, hkv, page = s["hq"], s["hkv"], s["page"]
    x = s["qkv"].view(s["qkv"].shape[0], hq + 2 * hkv, s["dim"])
    pos = s["positions"].long()
    cos, sin = s["cos"][pos][:, None, :], s["sin"][pos][:, None, :]
    q = _rotate(_norm(x[:, :hq].float(), s["q_scale"]), cos, sin)
    k = _rotate(_norm(x[:, hq : hq + hkv].float(), s["k_scale"]), cos, sin)
    slots = s["slots"].long()
    s["k_pages"][slots // page, :, slots % page] = k.to(x.dtype)
    s["v_pages"][slots // page, :, slots % page] = x[:, hq + hkv :]
    return {"q": q.to(x.dtype), "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _attend(s):
    q, tables, page = s["q"].float(), s["tables"].long(), s["page"]
    n, hq, dim = q.shape
    hkv, keys = s["k_pages"].shape[1], tables.shape[1] * page
    k = s["k_pages"][tables].float().permute(0, 2, 1, 3, 4).reshape(n, hkv, keys, dim)
    scores = (q.view(n, hkv, hq // hkv, dim) @ k.transpose(-1, -2)) / math.sqrt(dim)
    del k
    back = s["positions"].long()[:, None] - torch.arange(keys, device=q.device)[None, :]
    seen = back >= 0
    if s["window"] >= 0:
        seen = seen & (back <= s["window"])
    if s["slopes"] is not None:
        scores = scores - s["slopes"].view(1, hkv, hq // hkv, 1) * back[:, None, None, :].float()
    scores = scores.masked_fill(~seen[:, None, None, :], float("-inf"))
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    v = s["v_pages"][tables].float().permute(0, 2, 1, 3, 4).reshape(n, hkv, keys, dim)
    return (p @ v).reshape(n, hq, dim).to(s["q"].dtype)


# ------------------------------------------------------------------------------- the framework's
def _own(s):
    from mint_b200.ops import paged_attention, paged_plan, qk_norm_rope_paged

    if s["op"] == "plan":
        p = paged_plan(s["seq_lens"], s["new_lens"], s["tables"], s["free_pages"], s["free_head"],
                       page_size=s["page"], n_tokens=s["n_tokens"])
        return {"positions": p.positions, "slots": p.slots, "rows": p.rows, "ends": p.ends,
                "seq_lens": p.seq_lens, "free_head": p.free_head, "tables": s["tables"]}
    if s["op"] == "append":
        q = qk_norm_rope_paged(s["qkv"], s["hq"], s["hkv"], s["dim"], s["q_scale"], s["k_scale"], s["cos"], s["sin"],
                               s["positions"], s["slots"], s["k_pages"], s["v_pages"])
        return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    return paged_attention(s["q"], s["k_pages"], s["v_pages"], s["tables"], s["positions"],
                           window_left=s["window"], alibi_slopes=s["slopes"])


def run(state):
    if own:
        return _own(state)
    return {"plan": _plan, "append": _append, "attend": _attend}[state["op"]](state)


# ------------------------------------------------------------------------------------------- work
def work(case):
    page = case["page"]
    if case["op"] == "plan":
        n = case["requests"]
        new = _spread(n - case["idle"], case["new_lo"], case["new_hi"])
        tokens = n if case["new_hi"] == 1 else sum(new)
        fresh = sum(new) / page  # pages handed out: read from the free list, written to the tables
        return {"bytes": 4 * (2 * n + 2 * n + 3 * tokens + 2 * fresh + 2), "flops": 0}
    hq, hkv, dim, n = case["hq"], case["hkv"], case["dim"], case["tokens"]
    if case["op"] == "append":
        rows = n * (hq + 2 * hkv) * dim
        tables = min(n, case["span"]) * dim * 4
        return {"bytes": 4 * rows + tables + 8 * n + 8 * dim, "flops": 10 * n * (hq + hkv) * dim}
    lens = _spread(n, case["lo"], case["hi"])
    if case["window"] >= 0:
        lens = [min(v, case["window"] + 1) for v in lens]
    keys = sum(lens)
    pages = sum(_pages(v, page) for v in lens)
    return {"bytes": keys * hkv * dim * 4 + n * hq * dim * 4 + 4 * pages + 4 * n, "flops": 4 * keys * hq * dim}


# ---------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "plan":
        return None  # whole numbers only
    if s["op"] == "append":
        hq, hkv, dim, page = s["hq"], s["hkv"], s["dim"], s["page"]
        x = s["qkv"].double().view(-1, hq + 2 * hkv, dim)
        where = s["positions"].long()
        turn = torch.complex(s["cos"].double(), s["sin"].double())[where].unsqueeze(1)
        outs = []
        for part, scale in ((x[:, :hq], s["q_scale"]), (x[:, hq : hq + hkv], s["k_scale"])):
            y = part / (part.pow(2).sum(-1, keepdim=True) / dim + 1e-6).sqrt() * (scale.double() + 1.0)
            z = torch.complex(y[..., : dim // 2], y[..., dim // 2 :]) * turn
            outs.append(torch.cat([z.real, z.imag], -1))
        slot = s["slots"].long()
        page_of, line = torch.div(slot, page, rounding_mode="floor"), slot.remainder(page)
        kp, vp = s["k_pages"].double(), s["v_pages"].double()
        kp[page_of, :, line] = outs[1]
        vp[page_of, :, line] = x[:, hq + hkv :]
        return {"q": outs[0], "k_pages": kp, "v_pages": vp}
    n, hq, dim = s["q"].shape
    hkv, page = s["k_pages"].shape[1], s["page"]
    group = hq // hkv
    out = torch.zeros(n, hq, dim, dtype=torch.float64, device=DEVICE)
    for i in range(n):
        last = int(s["positions"][i])
        first = max(0, last - s["window"]) if s["window"] >= 0 else 0
        ids = s["tables"][i, first // page : last // page + 1].long()
        cut = slice(first % page, first % page + last - first + 1)
        k = s["k_pages"][ids].transpose(0, 1).reshape(hkv, -1, dim)[:, cut].double()
        v = s["v_pages"][ids].transpose(0, 1).reshape(hkv, -1, dim)[:, cut].double()
        logits = torch.einsum("hgd,hkd->hgk", s["q"][i].double().view(hkv, group, dim), k) * dim**-0.5
        if s["slopes"] is not None:
            away = torch.arange(first - last, 1, dtype=torch.float64, device=DEVICE)
            logits = logits + s["slopes"].double().view(hkv, group, 1) * away
        out[i] = torch.einsum("hgk,hkd->hgd", torch.softmax(logits, -1), v).reshape(hq, dim)
    return out
