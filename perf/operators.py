"""Operators of a served decoder whose requests have different lengths: pages of the key / value cache handed out on the GPU, rows written into
them, attention of one new token per request over them, and what a request's settings do to its logits before a token is picked.

`prepare` makes what a program holds before the call, `run` is one pass (plain torch, or the framework's kernels where `own` is true), `exact`
the same results in 64 bits. Heads, widths and vocabularies are those of the palettized Qwen3-4B model (32 query and 8 key / value heads of
128, vocabulary 151936) and of the hybrid decoders (vocabulary 32768), and ranges around both.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

DEV = "cuda"
# query heads, key / value heads, head size
HEADS = ((32, 8, 128), (16, 8, 128), (16, 16, 64), (12, 2, 64), (20, 4, 128), (32, 2, 128), (8, 2, 256), (7, 1, 128))
PAGES = (1, 8, 16, 24, 32, 64, 128)
VOCABS = (1001, 32768, 50257, 151936)


def _ops():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen-palettize_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import plz_ops
    return plz_ops


def _seq():
    _ops()
    import seq_ops
    return seq_ops


# ---- cases ---------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # pages for a step of token decode: every request brings one token, a few of them start a page
        {"name": "plan_decode_64", "kind": "plan", "B": 64, "cached": 4096, "new": 1, "rows": 64, "page": 16, "prompts": 0.0},
        # a batch of fresh prompts of ragged lengths
        {"name": "plan_prompts_8x2048", "kind": "plan", "B": 8, "cached": 0, "new": 2048, "rows": 16384, "page": 16, "prompts": 1.0},
        # a large server's step: a thousand requests, some with a portion of their prompt, the others with one token
        {"name": "plan_mixed_1000", "kind": "plan", "B": 1000, "cached": 8192, "new": 512, "rows": 32768, "page": 64, "prompts": 0.1},
        # keys and values of one decode step, and of a step full of prompts whose last rows are padding
        {"name": "write_decode_64", "kind": "write", "rows": 64, "width": 1024, "page": 16, "type": "bf16", "padding": 0.0},
        {"name": "write_prompts_16383", "kind": "write", "rows": 16383, "width": 1024, "page": 16, "type": "bf16", "padding": 0.05},
        # one user's token over a cache of ordinary length
        {"name": "attn_1x2049", "kind": "attn", "B": 1, "T": 2049, "heads": 0, "page": 16, "ragged": False},
        # a full batch of users, lengths from nothing to 4096
        {"name": "attn_64x4096_ragged", "kind": "attn", "B": 64, "T": 4096, "heads": 0, "page": 16, "ragged": True},
        # many short requests, a key / value head per query head
        {"name": "attn_256x300_ragged", "kind": "attn", "B": 256, "T": 300, "heads": 2, "page": 64, "ragged": True},
        # two users with very long documents
        {"name": "attn_2x131072", "kind": "attn", "B": 2, "T": 131072, "heads": 0, "page": 64, "ragged": False},
        # one user's logits: penalties over what was said, a few biases
        {"name": "logits_1x32768", "kind": "logits", "rows": 1, "V": 32768, "history": 500, "biases": 4, "mask": False, "type": "fp32"},
        # a few users who want structured output after long documents
        {"name": "logits_8x151936_grammar", "kind": "logits", "rows": 8, "V": 151936, "history": 30000, "biases": 0, "mask": True, "type": "fp32"},
        # a full batch with everything, as the model's head writes it
        {"name": "logits_64x151936_all", "kind": "logits", "rows": 64, "V": 151936, "history": 4096, "biases": 100, "mask": True, "type": "bf16"},
    ]


def _log(rng, lo, hi):
    """Whole number from lo to hi, spread over the logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(("plan", "write", "attn", "attn", "attn", "logits", "logits"))
    if kind == "plan":
        B = _log(rng, 1, 1000)
        new = _log(rng, 1, min(4096, 32768 // B))
        return {"kind": kind, "B": B, "cached": rng.choice((0, _log(rng, 1, 8192))), "new": new, "rows": B * new, "page": rng.choice(PAGES[1:]), "prompts": rng.choice((0.0, 0.2, 1.0))}
    if kind == "write":
        return {"kind": kind, "rows": _log(rng, 1, 16383), "width": rng.choice((64, 128, 512, 1024)), "page": rng.choice(PAGES), "type": rng.choice(("bf16", "fp32")),
                "padding": rng.choice((0.0, 0.1))}
    if kind == "attn":
        heads = rng.randrange(len(HEADS))
        _, hk, d = HEADS[heads]
        T = _log(rng, 1, 131072)
        most = max(1, 2 * 131072 * 8 * 128 // (T * hk * d))
        return {"kind": kind, "B": _log(rng, 1, min(256, most)), "T": T, "heads": heads, "page": rng.choice(PAGES), "ragged": rng.random() < 0.7}
    return {"kind": kind, "rows": _log(rng, 1, 64), "V": rng.choice(VOCABS), "history": rng.choice((0, _log(rng, 1, 4096))), "biases": rng.choice((0, _log(rng, 1, 300))),
            "mask": rng.random() < 0.5, "type": rng.choice(("fp32", "bf16"))}


# ---- inputs --------------------------------------------------------------------------------------------------------------
def _ints(lo, hi, shape, g, dtype=torch.int32):
    return torch.randint(lo, hi, shape, generator=g, device=DEV, dtype=torch.int64).to(dtype)


def _pages_of(T, page):
    return (T + page - 1) // page


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return {"plan": _prepare_plan, "write": _prepare_write, "attn": _prepare_attn, "logits": _prepare_logits}[case["kind"]](case, g)


def _prepare_plan(c, g):
    """Requests that hold the pages of their cached tokens, a shuffled stack of free pages, and how many tokens each brings."""
    B, page = c["B"], c["page"]
    cached = _ints(0, c["cached"] + 1, (B,), g)
    prompt = torch.rand(B, generator=g, device=DEV) < c["prompts"]
    new = torch.where(prompt, _ints(1, c["new"] + 1, (B,), g), torch.ones_like(cached))
    width = _pages_of(c["cached"] + c["new"], page)
    pool = B * width + 7
    order = torch.randperm(pool, generator=g, device=DEV).to(torch.int32)
    table = order[: B * width].view(B, width).clone()
    held = _pages_of(cached, page)
    at = torch.arange(width, device=DEV, dtype=torch.int32)
    taken = at[None, :] < held[:, None]
    loose = torch.cat([torch.where(taken, -1, table).reshape(-1), order[B * width:]])
    by = torch.argsort((loose < 0).to(torch.int8), stable=True)          # free pages first
    return {"kind": "plan", "cached": cached, "new": new, "table": torch.where(taken, table, -1), "free": loose[by].contiguous(), "n_free": (loose >= 0).sum().to(torch.int32).view(1),
            "page": page, "rows": c["rows"], "lengths_out": torch.empty_like(cached), "n_free_out": torch.empty(1, dtype=torch.int32, device=DEV)}


def _prepare_write(c, g):
    n, W, page = c["rows"], c["width"], c["page"]
    t = {"bf16": torch.bfloat16, "fp32": torch.float32}[c["type"]]
    pages = _pages_of(n + 1, page) + 3
    k, v = (torch.randn(n, W, generator=g, device=DEV).to(t) for _ in range(2))
    kp, vp = (torch.randn(pages, page, W, generator=g, device=DEV).to(t) for _ in range(2))
    slots = torch.randperm(pages * page - 1, generator=g, device=DEV)[:n].to(torch.int32)       # the last slot stays out of it
    keep = torch.arange(n, device=DEV) < n - int(n * c["padding"])
    return {"kind": "write", "k": k, "v": v, "slots": torch.where(keep, slots, -1), "k_pages": kp, "v_pages": vp}


def _lengths(B, T, ragged, g):
    n = _ints(1, T + 1, (B,), g) if ragged else torch.full((B,), T, dtype=torch.int32, device=DEV)
    n[0] = T
    if ragged and B >= 4:
        n[B // 2] = 0                                 # a request without a token yet
    return n


def _prepare_attn(c, g):
    hq, hk, d = HEADS[c["heads"]]
    B, T, page = c["B"], c["T"], c["page"]
    width = _pages_of(T, page)
    n_pages = B * width + 1
    table = torch.randperm(n_pages, generator=g, device=DEV)[: B * width].to(torch.int32).view(B, width)
    kp, vp = (torch.randn(n_pages, page, hk * d, generator=g, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    q = torch.randn(B, hq * d, generator=g, device=DEV, dtype=torch.bfloat16)
    return {"kind": "attn", "q": q, "k_pages": kp, "v_pages": vp, "table": table, "lengths": _lengths(B, T, c["ragged"], g), "hq": hq, "hk": hk, "d": d}


def _prepare_logits(c, g):
    B, V, L = c["rows"], c["V"], c["history"]
    t = {"bf16": torch.bfloat16, "fp32": torch.float32}[c["type"]]
    logits = (3.0 * torch.randn(B, V, generator=g, device=DEV)).to(t)
    # text repeats itself: low numbers are common, the square of a uniform draw
    tokens = (torch.rand(B, max(L, 1), generator=g, device=DEV) ** 2 * V).long().clamp(max=V - 1)
    n = _ints(L // 2, L + 1, (B,), g)
    s = {"kind": "logits", "logits": logits, "tokens": tokens, "lengths": n, "prompt_lengths": n // 3,
         "repetition": 1.0 + 0.3 * torch.rand(B, generator=g, device=DEV), "presence": torch.rand(B, generator=g, device=DEV), "frequency": 0.2 * torch.rand(B, generator=g, device=DEV),
         "bias_ids": None, "bias": None, "mask": None}
    if c["biases"]:
        s["bias_ids"] = _ints(-1, V, (B, c["biases"]), g, torch.int64)      # -1: no bias in this place
        s["bias"] = 5.0 * torch.randn(B, c["biases"], generator=g, device=DEV)
    if c["mask"]:
        # a grammar allows few tokens inside a word of the language and many in free text
        share = torch.rand(B, 1, generator=g, device=DEV) ** 2
        bits = (torch.rand(B, (V + 31) // 32 * 32, generator=g, device=DEV) < share).view(B, -1, 32).long()
        words = (bits << torch.arange(32, device=DEV)).sum(-1)
        s["mask"] = torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)
    return s


# ---- one pass ------------------------------------------------------------------------------------------------------------
def run(s):
    return {"plan": _run_plan, "write": _run_write, "attn": _run_attn, "logits": _run_logits}[s["kind"]](s)


def _run_plan(s):
    if own:
        p = _ops().plan_pages(s["cached"], s["new"], s["table"], s["free"], s["n_free"], s["page"], s["rows"], lengths_out=s["lengths_out"], n_free_out=s["n_free_out"])
        return p.lengths, p.n_free, p.starts, p.slots, p.positions, p.status, s["table"]
    cached, new, table, free, page, rows = s["cached"].long(), s["new"].long(), s["table"].long(), s["free"].long(), s["page"], s["rows"]
    B, width = table.shape
    n_free = s["n_free"].long()
    ends = torch.cumsum(new, 0)
    starts = torch.cat([torch.zeros_like(ends[:1]), ends])
    total, held = cached + new, (cached + page - 1) // page
    fits = (total <= width * page) & (ends <= rows)
    need = torch.where(fits, (total + page - 1) // page - held, 0)
    upto = torch.cumsum(need, 0)
    served = fits & ((need == 0) | (upto <= n_free))
    status = torch.where(served, 0, torch.where(fits, 1, 2))
    at = torch.arange(width, device=table.device)
    fresh = (at >= held[:, None]) & (at < (held + need)[:, None]) & served[:, None]
    pick = n_free - 1 - ((upto - need)[:, None] + at - held[:, None])
    table = torch.where(fresh, free[pick.clamp(0, free.numel() - 1)], table)
    r = torch.arange(rows, device=table.device)
    b = torch.searchsorted(ends, r, right=True).clamp(max=B - 1)
    live = (r < ends[-1]) & served[b]
    pos = cached[b] + r - starts[b]
    slot = table[b, (pos // page).clamp(0, width - 1)] * page + pos % page
    taken = torch.where(served, need, 0).sum()
    out = (torch.where(served, total, cached), n_free - taken, starts, torch.where(live, slot, -1), torch.where(live, pos, -1), status, table)
    return tuple(map(torch.Tensor.int, out))


def _run_write(s):
    if own:
        _ops().write_pages(s["k"], s["v"], s["slots"], s["k_pages"], s["v_pages"])
        return s["k_pages"], s["v_pages"]
    at = s["slots"].long()                            # padding, -1, lands in the last slot, which gets its own row back
    kp, vp = s["k_pages"].flatten(0, 1), s["v_pages"].flatten(0, 1)
    k_last, v_last = kp[-1].clone(), vp[-1].clone()
    kp[at] = s["k"]
    vp[at] = s["v"]
    kp[-1] = k_last
    vp[-1] = v_last
    return s["k_pages"], s["v_pages"]


def _run_attn(s):
    hq, hk, d = s["hq"], s["hk"], s["d"]
    if own:
        return _ops().attention_decode_paged(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], hq, hk, d)
    B = s["q"].shape[0]
    at = s["table"].long()
    q = s["q"].float().view(B, hk, hq // hk, d)
    k = s["k_pages"][at].view(B, -1, hk, d).permute(0, 2, 3, 1).float()
    v = s["v_pages"][at].view(B, -1, hk, d).permute(0, 2, 1, 3).float()
    here = (torch.arange(k.shape[3], device=q.device) < s["lengths"][:, None])[:, None, None, :]
    score = torch.where(here, q @ k * d ** -0.5, -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    w = torch.exp(score - top)
    total = w.sum(-1, keepdim=True)
    return ((w @ v) / torch.where(total > 0, total, 1)).reshape(B, hq * d).to(s["q"].dtype)


def _run_logits(s):
    if own:
        return _seq().adjust_logits(s["logits"], tokens=s["tokens"], lengths=s["lengths"], prompt_lengths=s["prompt_lengths"], repetition=s["repetition"], presence=s["presence"],
                                    frequency=s["frequency"], bias_ids=s["bias_ids"], bias=s["bias"], mask=s["mask"])
    x = s["logits"].float()
    B, V = x.shape
    place = torch.arange(s["tokens"].shape[1], device=x.device)
    said = place < s["lengths"][:, None]
    own_words = said & (place >= s["prompt_lengths"][:, None])
    seen = torch.zeros_like(x).scatter_add_(1, s["tokens"], said.float()) > 0
    count = torch.zeros_like(x).scatter_add_(1, s["tokens"], own_words.float())
    r, p, f = s["repetition"][:, None], s["presence"][:, None], s["frequency"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = torch.where(count > 0, x - f * count - p, x)
    if s["bias_ids"] is not None:
        at = s["bias_ids"]
        x = x.scatter_add(1, at.clamp(min=0), torch.where(at >= 0, s["bias"], 0))
    if s["mask"] is not None:
        tok = torch.arange(V, device=x.device)
        x = torch.where((s["mask"][:, tok >> 5] >> (tok & 31)) & 1 != 0, x, -math.inf)
    return x.to(s["logits"].dtype)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------
def work(c):
    if c["kind"] == "plan":
        # per request: length in and out, new tokens, start, status, one table entry; per row: slot and position; per page handed out: an entry of the stack and of the table
        rows = c["B"] * (c["prompts"] * (c["new"] + 1) / 2 + 1 - c["prompts"])
        return {"bytes": int(24 * c["B"] + 8 * c["rows"] + 8 * rows / c["page"] + 8), "flops": 0}
    if c["kind"] == "write":
        n = c["rows"] - int(c["rows"] * c["padding"])
        return {"bytes": 4 * c["rows"] + 4 * n * c["width"] * {"bf16": 2, "fp32": 4}[c["type"]], "flops": 0}
    if c["kind"] == "attn":
        hq, hk, d = HEADS[c["heads"]]
        tokens = c["B"] * (c["T"] + 1) / 2 if c["ragged"] else c["B"] * c["T"]
        return {"bytes": int(tokens * hk * d * 4 + 4 * tokens / c["page"] + 4 * c["B"] * hq * d + 4 * c["B"]), "flops": int(4 * tokens * hq * d)}
    B, V, L = c["rows"], c["V"], c["history"]
    size = {"bf16": 2, "fp32": 4}[c["type"]]
    return {"bytes": int(2 * B * V * size + B * 6 * L + (B * (V + 31) // 32 * 4 if c["mask"] else 0) + 12 * B * c["biases"] + 20 * B), "flops": 6 * B * V}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------------
def exact(case, seed):
    if case["kind"] == "plan":
        return None                                  # whole numbers
    s = prepare(case, seed)
    if case["kind"] == "write":
        out = []
        good = s["slots"] >= 0
        for rows, pool in ((s["k"], s["k_pages"]), (s["v"], s["v_pages"])):
            full = pool.double()
            full.view(-1, rows.shape[1]).index_copy_(0, s["slots"][good].long(), rows[good].double())
            out.append(full)
        return tuple(out)
    if case["kind"] == "attn":
        hq, hk, d = s["hq"], s["hk"], s["d"]
        page = s["k_pages"].shape[1]
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        for b, n in enumerate(s["lengths"].tolist()):
            if n == 0:
                continue
            ids = s["table"][b, : _pages_of(n, page)].long()
            k = s["k_pages"][ids].reshape(-1, hk, d)[:n].double()
            v = s["v_pages"][ids].reshape(-1, hk, d)[:n].double()
            for h in range(hk):
                q = s["q"][b].view(hq, d)[h * (hq // hk):(h + 1) * (hq // hk)].double()
                w = torch.softmax(q @ k[:, h].T / math.sqrt(d), -1)
                out[b].view(hq, d)[h * (hq // hk):(h + 1) * (hq // hk)] = w @ v[:, h]
        return out
    x = s["logits"].double()
    B, V = x.shape
    for b in range(B):
        n, n_prompt = int(s["lengths"][b]), int(s["prompt_lengths"][b])
        all_words = torch.bincount(s["tokens"][b, :n], minlength=V)
        spoken = torch.bincount(s["tokens"][b, n_prompt:n], minlength=V)
        r, p, f = (float(s[name][b]) for name in ("repetition", "presence", "frequency"))
        row = x[b]
        hit = all_words > 0
        row[hit] = torch.where(row[hit] > 0, row[hit] / r, row[hit] * r)
        row -= f * spoken.double() + p * (spoken > 0).double()
        if s["bias_ids"] is not None:
            good = s["bias_ids"][b] >= 0
            row.index_add_(0, s["bias_ids"][b][good], s["bias"][b][good].double())
        if s["mask"] is not None:
            bits = (s["mask"][b][:, None].long() >> torch.arange(32, device=DEV)) & 1
            row[bits.view(-1)[:V] == 0] = -math.inf
    return x
