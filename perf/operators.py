"""The operators of serving from a paged key-value cache: what is measured and what they compute.

One serving step makes all four: `plan` (which page and slot every new token gets, built on the GPU from the requests'
lengths; and the pages of finished requests given back), `append` (rotary positions on q and k, k and v written to their
slots), `attend` (the new tokens over their requests' pages) and `logprobs` (log-probabilities of given tokens, entropy,
rank and the top alternatives). Sizes are those of the repository's benchmark configurations (12 query heads over 4,
16 over 2, 12 over 12, head_dim 64; vocabularies of 32000, 50257 and 151936 tokens) and generic ones with 128-wide heads.

`draw` gives more of the same ranges: 1..1024 requests, up to 262144 rows in one plan; 1..8192 rows appended; 1..256
attended rows of 1..131072 positions, 1..8 kv heads with 1..8 query heads each, head_dim 32..256 in steps of 8, pages of
8..256 positions; 1..2048 rows of 100..200000 logits with 0..32 alternatives. Activations, caches and logits are f32, f16
or bf16.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
_device = None


def _dev():
    """The library's device handle, kept for the process as a server keeps it."""
    global _device
    if _device is None:
        from ferrum_gpu_b200 import Device
        _device = Device.open(0)
    return _device


# ---- cases -------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one user's next token: a table entry and a slot, nothing but latency
        {"name": "plan_1_decode", "op": "plan", "way": "extend", "requests": 1, "page": 16, "longest": 700, "prompts": 0, "grow": 1, "rows": 1},
        # a busy server's step: 512 requests, every eighth a prompt that enters, the others one token each; padded rows
        {"name": "plan_512_mixed", "op": "plan", "way": "extend", "requests": 512, "page": 16, "longest": 4000, "prompts": 64, "grow": 2001,
         "rows": 131072},
        # 200 requests end at once: their pages go back
        {"name": "release_200", "op": "plan", "way": "release", "requests": 200, "page": 16, "longest": 8000, "prompts": 0, "grow": 0, "rows": 0},
        # a few users' tokens of the 12-over-4-head model, neighbouring pairs, f32 rows into an f16 cache
        {"name": "append_6_decode", "op": "append", "rows": 6, "heads": 12, "kv_heads": 4, "head_dim": 64, "rope_dim": 64, "neox": False,
         "act": "f32", "cache": "f16", "page": 16, "positions": 2048},
        # a chunk of prompts, half layout over three quarters of a 128-wide head, long positions
        {"name": "append_8192_prompt", "op": "append", "rows": 8192, "heads": 32, "kv_heads": 8, "head_dim": 128, "rope_dim": 96, "neox": True,
         "act": "bf16", "cache": "bf16", "page": 16, "positions": 131072},
        # the first words of one stream of the small model without grouped heads, in f32
        {"name": "attend_1x17_f32", "op": "attend", "rows": 1, "longest": 17, "heads": 6, "kv_heads": 6, "head_dim": 64, "act": "f32",
         "cache": "f32", "page": 16},
        # a full server of the 16-over-2-head model: texts of all lengths up to 1999 positions, the cache in f32 as the resident models keep it
        {"name": "attend_64x1999_f32", "op": "attend", "rows": 64, "longest": 1999, "heads": 16, "kv_heads": 2, "head_dim": 64, "act": "f32",
         "cache": "f32", "page": 32},
        # one very long text: the cache's length split over the whole GPU
        {"name": "attend_1x131071_f16", "op": "attend", "rows": 1, "longest": 131071, "heads": 32, "kv_heads": 8, "head_dim": 128, "act": "f32",
         "cache": "f16", "page": 64},
        # many long texts in 16 bits
        {"name": "attend_48x8000_bf16", "op": "attend", "rows": 48, "longest": 8000, "heads": 32, "kv_heads": 8, "head_dim": 128, "act": "bf16",
         "cache": "bf16", "page": 16},
        # the answer's tokens of one user: probability of the pick and five alternatives
        {"name": "logprobs_1x32000", "op": "logprobs", "rows": 1, "vocab": 32000, "pad": 0, "top": 5, "logits": "f32", "masked": False},
        # a full server with a large vocabulary and a grammar that forbids most tokens, twenty alternatives
        {"name": "logprobs_64x151936", "op": "logprobs", "rows": 64, "vocab": 151936, "pad": 0, "top": 20, "logits": "f32", "masked": True},
        # a prompt's own log-probabilities, odd vocabulary in padded rows of f16
        {"name": "logprobs_1500x50257_f16", "op": "logprobs", "rows": 1500, "vocab": 50257, "pad": 47, "top": 1, "logits": "f16", "masked": False},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "append", "attend", "attend", "logprobs", "logprobs"])
    page = rng.choice([8, 16, 16, 32, 64, 128, 256])
    if op == "plan":
        n = _log_int(rng, 1, 1024)
        longest = _log_int(rng, 1, 16000)
        if rng.random() < 0.3:
            return {"op": op, "way": "release", "requests": n, "page": page, "longest": longest, "prompts": 0, "grow": 0, "rows": 0}
        prompts = rng.randint(0, max(1, n // 4))
        grow = _log_int(rng, 1, min(8000, max(2, (262144 - n) // max(1, prompts))))
        return {"op": op, "way": "extend", "requests": n, "page": page, "longest": longest, "prompts": prompts, "grow": grow,
                "rows": n + prompts * grow + rng.randint(0, 100)}
    head_dim = 8 * rng.choice([4, 8, 8, 10, 12, 16, 16, 24, 32, rng.randint(4, 32)])
    kv_heads = rng.randint(1, 8)
    heads = kv_heads * rng.randint(1, 8)
    act, cache = rng.choice([("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")])
    if op == "append":
        rope_dim = rng.choice([head_dim, head_dim, 2 * rng.randint(1, head_dim // 2)])
        return {"op": op, "rows": _log_int(rng, 1, 8192 * 6144 // max(6144, (heads + 2 * kv_heads) * head_dim)), "heads": heads,
                "kv_heads": kv_heads, "head_dim": head_dim, "rope_dim": rope_dim, "neox": rng.random() < 0.5, "act": act, "cache": cache,
                "page": page, "positions": _log_int(rng, 256, 131072)}
    if op == "attend":
        rows = _log_int(rng, 1, 256)
        most = int(0.49e9 / (rows * kv_heads * head_dim * BYTES[cache]))  # (a gigabyte of k and v)
        return {"op": op, "rows": rows, "longest": _log_int(rng, 1, min(131072, most)), "heads": heads, "kv_heads": kv_heads,
                "head_dim": head_dim, "act": act, "cache": cache, "page": page}
    vocab = _log_int(rng, 100, 200000)
    return {"op": op, "rows": _log_int(rng, 1, min(2048, 1500 * 50257 // vocab)), "vocab": vocab, "pad": rng.choice([0, 0, rng.randint(1, 63)]),
            "top": rng.choice([0, 1, 5, 20, 32]), "logits": rng.choice(["f32", "f32", "f16", "bf16"]), "masked": rng.random() < 0.3}


# ---- inputs ------------------------------------------------------------------------------------------------------

def _lengths(n, longest):
    """Lengths from a quarter of the longest one up, the longest among them."""
    low = max(1, longest // 4)
    return [longest - (i * 617) % max(1, longest - low + 1) for i in range(n)]


def _grows(case):
    """Tokens that each request adds: prompts spread among the requests, one token for the others."""
    n, p = case["requests"], case["prompts"]
    every = n // p if p else 0
    grow = [1] * n
    for i in range(p):
        grow[i * every] = case["grow"] - (i * 131) % max(1, case["grow"] // 2)
    return grow


def _pages(x, page):
    return -(-x // page)


def _tables(lens, page, most, n_pages, gen):
    """Page tables of requests of these lengths over a pool whose pages lie in no order, and the pages left over, as a stack."""
    order = torch.randperm(n_pages, device="cuda", generator=gen, dtype=torch.int64).to(torch.int32)
    held = torch.tensor([_pages(x, page) for x in lens], device="cuda")
    first = held.cumsum(0) - held
    at = torch.arange(most, device="cuda")
    has = at[None, :] < held[:, None]
    table = torch.where(has, order[(first[:, None] + at[None, :]).clamp(max=n_pages - 1)], -1).to(torch.int32)
    used = int(held.sum())
    free = torch.full((n_pages,), -1, dtype=torch.int32, device="cuda")
    free[:n_pages - used] = order[used:]
    return table, free, n_pages - used


def _rotary(case):
    """cos and sin of every position, pairs slowed down towards the long wavelengths as for a context eight times longer."""
    half = case["rope_dim"] // 2
    i = torch.arange(half, dtype=torch.float64, device="cuda")
    freq = 500000.0 ** (-2.0 * i / case["rope_dim"])
    wave = 2 * math.pi / freq
    keep = ((wave.log2() - 11.0) / 2.0).clamp(0.0, 1.0)
    freq = freq * (1 - keep) + freq / 8 * keep
    angle = torch.arange(case["positions"], dtype=torch.float64, device="cuda")[:, None] * freq[None, :]
    return angle.cos().float(), angle.sin().float()


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def normal(*shape, dtype="f32"):
        return torch.randn(*shape, device="cuda", generator=gen, dtype=DTYPES[dtype])

    if case["op"] == "plan":
        n, page = case["requests"], case["page"]
        lens, grow = _lengths(n, case["longest"]), _grows(case)
        rows_of = n + n // 4 + 1  # requests the server has places for; this step's are some of them, in no order
        place = torch.randperm(rows_of, device="cuda", generator=gen)[:n]
        most = max(_pages(a + b, page) for a, b in zip(lens, grow)) + 3
        n_pages = sum(_pages(a + b, page) for a, b in zip(lens, grow)) + 50
        table = torch.full((rows_of, most), -1, dtype=torch.int32, device="cuda")
        mine, free, n_free = _tables(lens, page, most, n_pages, gen)
        table[place] = mine
        all_lens = torch.zeros(rows_of, dtype=torch.int32, device="cuda")
        all_lens[place] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        return {"requests": place.to(torch.int32), "grow": torch.tensor(grow, dtype=torch.int32, device="cuda"), "table": table,
                "lens": all_lens, "free": free, "n_free": torch.tensor([n_free], dtype=torch.int32, device="cuda"), "n_pages": n_pages}
    if case["op"] == "append":
        rows, hd, page = case["rows"], case["head_dim"], case["page"]
        n_pages = _pages(rows, page) + _pages(rows, page) // 8 + 1
        cos, sin = _rotary(case)
        pool = (n_pages, case["kv_heads"], page, hd)
        if rows <= 64:  # a token of each of so many requests, each somewhere in a page of its own choosing
            slot = torch.randperm(n_pages * page, device="cuda", generator=gen)[:rows]
        else:  # a prompt: whole pages one after another, the pages in no order
            t = torch.arange(rows, device="cuda")
            slot = torch.randperm(n_pages, device="cuda", generator=gen)[t // page] * page + t % page
        first = torch.randint(0, max(1, case["positions"] - rows), (1,), device="cuda", generator=gen)
        position = ((first + torch.arange(rows, device="cuda")) % case["positions"]).to(torch.int32)
        return {"qkv": normal(rows, (case["heads"] + 2 * case["kv_heads"]) * hd, dtype=case["act"]), "k": normal(*pool, dtype=case["cache"]),
                "v": normal(*pool, dtype=case["cache"]), "slot": slot, "position": position, "cos": cos, "sin": sin}
    if case["op"] == "attend":
        rows, hd, page = case["rows"], case["head_dim"], case["page"]
        lens = _lengths(rows, case["longest"])
        most = max(_pages(x, page) for x in lens) + 2
        n_pages = sum(_pages(x, page) for x in lens) + 7
        table, _, _ = _tables(lens, page, most, n_pages, gen)
        pool = (n_pages, case["kv_heads"], page, hd)
        order = torch.randperm(rows, device="cuda", generator=gen)
        position = torch.tensor(lens, device="cuda", dtype=torch.int32)[order] - 1
        # (queries of twice the keys' size: some positions stand out, as after training)
        return {"q": normal(rows, case["heads"] * hd, dtype=case["act"]) * 2, "k": normal(*pool, dtype=case["cache"]),
                "v": normal(*pool, dtype=case["cache"]), "table": table, "request": order.to(torch.int32), "position": position}
    rows, vocab = case["rows"], case["vocab"]
    logits = normal(rows, vocab + case["pad"]) * 3
    # the token that was picked is likely, not any: the best of eight; the last row of a text has none
    some = torch.randint(0, vocab, (rows, 8), device="cuda", generator=gen)
    pick = some.gather(1, logits.gather(1, some).argmax(dim=1, keepdim=True))
    if case["masked"]:
        allowed = torch.rand(rows, vocab + case["pad"], device="cuda", generator=gen) < 0.05
        logits = torch.where(allowed.scatter(1, pick, True), logits, float("-inf"))
    target = pick[:, 0].to(torch.int32)
    if rows > 1:
        target[-1] = -1
    return {"logits": logits.to(DTYPES[case["logits"]]), "target": target}


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    rows = case["rows"]

    def ints(*shape, dtype=torch.int32):
        return torch.zeros(*shape, dtype=dtype, device="cuda")

    # what a program keeps between steps: the buffers that results land in, and the handle over the cache
    if case["op"] == "plan":
        state["new_lens"], state["new_n_free"], state["status"] = state["lens"].clone(), ints(1), ints(1)
        if case["way"] == "extend":
            state["starts"], state["slot"] = ints(case["requests"] + 1), ints(rows, dtype=torch.int64)
            state["position"], state["request"] = ints(rows), ints(rows)
    elif case["op"] == "append":
        state["q"] = torch.zeros(rows, case["heads"] * case["head_dim"], dtype=DTYPES[case["act"]], device="cuda")
    elif case["op"] == "attend":
        state["out"] = torch.zeros_like(state["q"])
    else:
        state["out"] = {"logprob": torch.zeros(rows, device="cuda"), "entropy": torch.zeros(rows, device="cuda"), "rank": ints(rows),
                        "top_index": ints(rows, case["top"]), "top_logprob": torch.zeros(rows, case["top"], device="cuda")}
    if own:
        _handles(state)
    torch.cuda.synchronize()
    return state


def _handles(state):
    """The library's view of the cache and of one step's rows: pointers and sizes, nothing of the data."""
    from ferrum_gpu_b200 import LogProbs, PagedCache, Rotary, Step
    case, op = state["case"], state["case"]["op"]
    if op == "plan":
        state["cache"] = PagedCache(_dev(), page=case["page"], table=state["table"], lens=state["lens"], free=state["free"],
                                    n_free=state["n_free"])
        if case["way"] == "extend":
            state["step"] = Step(starts=state["starts"], slot=state["slot"], position=state["position"], request=state["request"],
                                 status=state["status"])
    elif op == "append":
        state["cache"] = PagedCache(_dev(), page=case["page"], layers=[(state["k"], state["v"])])
        state["step"] = Step(slot=state["slot"], position=state["position"])
        state["rotary"] = Rotary(state["cos"], state["sin"], neox=case["neox"])
    elif op == "attend":
        state["cache"] = PagedCache(_dev(), page=case["page"], table=state["table"], layers=[(state["k"], state["v"])])
        state["step"] = Step(position=state["position"], request=state["request"])
    else:
        state["results"] = LogProbs(**state["out"])


# ---- one pass ----------------------------------------------------------------------------------------------------

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    case, op = state["case"], state["case"]["op"]
    if op == "plan":
        cache = state["cache"]
        if case["way"] == "release":
            cache.release(state["requests"], lens_out=state["new_lens"], n_free_out=state["new_n_free"], status=state["status"])
            return {"free": state["free"], "lens": state["new_lens"], "n_free": state["new_n_free"], "status": state["status"]}
        cache.extend(state["grow"], state["step"], requests=state["requests"], lens_out=state["new_lens"], n_free_out=state["new_n_free"])
        return {"starts": state["starts"], "slot": state["slot"], "position": state["position"], "request": state["request"],
                "table": state["table"], "lens": state["new_lens"], "n_free": state["new_n_free"], "status": state["status"]}
    if op == "append":
        state["cache"].append(0, state["qkv"], state["step"], state["q"], rotary=state["rotary"])
        return {"q": state["q"], "k": state["k"], "v": state["v"]}
    if op == "attend":
        state["cache"].attend(0, state["q"], state["step"], state["out"])
        return state["out"]
    from ferrum_gpu_b200 import logprobs
    logprobs(_dev(), state["logits"], state["target"], state["results"], vocab=case["vocab"])
    return state["out"]


def _run_plain(state):
    case, op = state["case"], state["case"]["op"]
    if op == "plan":
        return (_plain_release if case["way"] == "release" else _plain_extend)(state, case)
    return {"append": _plain_append, "attend": _plain_attend, "logprobs": _plain_logprobs}[op](state, case)


def _plain_extend(s, case):
    page, rows = case["page"], case["rows"]
    req, grow, n_free, table = s["requests"].long(), s["grow"].long(), s["n_free"].long(), s["table"]
    old = s["lens"][req].long()
    held, held_after = (old + page - 1) // page, (old + grow + page - 1) // page
    need = held_after - held
    first = need.cumsum(0) - need  # of the pages taken, the request's first
    end = grow.cumsum(0)
    short = (need.sum() - n_free).clamp(min=0)
    bad = (short > 0) | (end[-1] > rows)
    good = ~bad
    # rows -> (request, position, slot)
    t = torch.arange(rows, device="cuda")
    i = torch.searchsorted(end, t, right=True).clamp(max=len(end) - 1)
    here = good & (t < end[-1])
    position = old[i] + t - (end - grow)[i]
    p = position // page
    fresh = p >= held[i]
    taken = (n_free - 1 - (first[i] + p - held[i])).clamp(min=0)
    at = torch.where(fresh, s["free"][taken].long(), table[req[i], p.clamp(max=table.shape[1] - 1)].long())
    # the pages that the table gets
    col = torch.arange(table.shape[1], device="cuda")[None, :]
    new = good & (col >= held[:, None]) & (col < held_after[:, None])
    page_id = s["free"][(n_free - 1 - (first[:, None] + col - held[:, None])).clamp(0, s["n_pages"] - 1)]
    table, lens = table.clone(), s["lens"].clone()
    table[req] = torch.where(new, page_id, table[req])
    lens[req] = torch.where(good, old + grow, old).to(torch.int32)
    starts = torch.cat([end.new_zeros(1), torch.where(good, end, 0)])
    return {"starts": starts.to(torch.int32), "slot": torch.where(here, at * page + position % page, -1),
            "position": torch.where(here, position, -1).to(torch.int32), "request": torch.where(here, req[i], -1).to(torch.int32),
            "table": table, "lens": lens, "n_free": torch.where(good, n_free - need.sum(), n_free).to(torch.int32),
            "status": torch.where(end[-1] > rows, -1, short).to(torch.int32)}


def _plain_release(s, case):
    req, n_free, table = s["requests"].long(), s["n_free"].long(), s["table"]
    held = (s["lens"][req].long() + case["page"] - 1) // case["page"]
    first = held.cumsum(0) - held
    col = torch.arange(table.shape[1], device="cuda")[None, :]
    to = torch.where(col < held[:, None], n_free + first[:, None] + col, s["n_pages"])  # (one place past the end for the others)
    free = torch.cat([s["free"], s["free"].new_zeros(1)])
    free[to] = table[req]
    lens = s["lens"].clone()
    lens[req] = 0
    return {"free": free[:-1], "lens": lens, "n_free": (n_free + held.sum()).to(torch.int32), "status": torch.zeros_like(s["status"])}


def _plain_append(s, case):
    rows, heads, kv, hd, rd = case["rows"], case["heads"], case["kv_heads"], case["head_dim"], case["rope_dim"]
    x = s["qkv"].float().view(rows, heads + 2 * kv, hd)
    qk, v = x[:, :heads + kv], x[:, heads + kv:]
    at = s["position"].long()
    cos, sin = s["cos"][at][:, None, :], s["sin"][at][:, None, :]
    if case["neox"]:
        a, b = qk[..., :rd // 2], qk[..., rd // 2:rd]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    else:
        a, b = qk[..., 0:rd:2], qk[..., 1:rd:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    qk = torch.cat([turned, qk[..., rd:]], dim=-1)
    page, offset = s["slot"] // case["page"], s["slot"] % case["page"]
    k, cache_v = s["k"].clone(), s["v"].clone()
    k[page, :, offset] = qk[:, heads:].to(k.dtype)
    cache_v[page, :, offset] = v.to(k.dtype)
    return {"q": qk[:, :heads].reshape(rows, heads * hd).to(s["qkv"].dtype), "k": k, "v": cache_v}


def _plain_attend(s, case):
    rows, heads, kv, hd = case["rows"], case["heads"], case["kv_heads"], case["head_dim"]
    used = (case["longest"] + case["page"] - 1) // case["page"]
    pages = s["table"][s["request"].long()][:, :used].long().clamp(min=0)
    k = s["k"][pages].float().transpose(1, 2).reshape(rows, kv, -1, hd)  # [row, kv head, position, hd]
    v = s["v"][pages].float().transpose(1, 2).reshape(rows, kv, -1, hd)
    q = s["q"].float().view(rows, kv, heads // kv, hd)
    score = q @ k.transpose(2, 3) / math.sqrt(hd)
    seen = torch.arange(k.shape[2], device="cuda")[None, :] <= s["position"][:, None].long()
    score = torch.where(seen[:, None, None, :], score, float("-inf"))
    p = (score - score.amax(dim=-1, keepdim=True)).exp()
    p = p / p.sum(dim=-1, keepdim=True)
    v = torch.where(seen[:, None, :, None], v, 0.0)
    return (p @ v).reshape(rows, heads * hd).to(s["q"].dtype)


def _plain_logprobs(s, case):
    vocab, top = case["vocab"], case["top"]
    x = s["logits"][:, :vocab].float()
    t = s["target"].long()
    has = t >= 0
    m = x.amax(dim=1, keepdim=True)
    m = torch.where(m == float("-inf"), 0.0, m)  # (nothing is allowed: every log-probability is -inf, the entropy 0)
    d = x - m
    e = d.exp()
    total = e.sum(dim=1, keepdim=True)
    total = torch.where(total == 0, 1.0, total)
    log_total = total.log()
    of = torch.where(e > 0, e * d, 0.0).sum(dim=1, keepdim=True)
    entropy = (log_total - of / total)[:, 0]
    mine = x.gather(1, t.clamp(min=0)[:, None])
    index = torch.arange(vocab, device="cuda")[None, :]
    rank = ((x > mine) | ((x == mine) & (index < t[:, None]))).sum(dim=1)
    logprob = torch.where(has, (mine - m - log_total)[:, 0], float("nan"))
    value, order = torch.sort(x, dim=1, descending=True, stable=True)
    return {"logprob": logprob, "entropy": entropy, "rank": torch.where(has, rank, -1).to(torch.int32),
            "top_index": order[:, :top].to(torch.int32), "top_logprob": value[:, :top] - m - log_total}


# ---- the same from the definitions, in 64 bits --------------------------------------------------------------------

def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "plan":
        return None
    if case["op"] == "append":
        return _exact_append(s, case)
    return _exact_attend(s, case) if case["op"] == "attend" else _exact_logprobs(s, case)


def _exact_append(s, case):
    heads, kv, hd, half = case["heads"], case["kv_heads"], case["head_dim"], case["rope_dim"] // 2
    x = s["qkv"].double().view(case["rows"], -1, hd)
    out = x.clone()
    pair = torch.complex(s["cos"].double(), s["sin"].double())[s["position"].long()]  # a turn is a product of complex numbers
    one = torch.arange(half, device="cuda")
    re, im = (one, one + half) if case["neox"] else (2 * one, 2 * one + 1)
    for h in range(heads + kv):
        z = torch.complex(x[:, h, re], x[:, h, im]) * pair
        out[:, h, re], out[:, h, im] = z.real, z.imag
    k, v = s["k"].double(), s["v"].double()
    for h in range(kv):
        at = (s["slot"] // case["page"], torch.full_like(s["slot"], h), s["slot"] % case["page"])
        k[at] = out[:, heads + h]
        v[at] = x[:, heads + kv + h]
    return {"q": out[:, :heads].reshape(case["rows"], heads * hd), "k": k, "v": v}


def _exact_attend(s, case):
    rows, heads, kv, hd, page = case["rows"], case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    group = heads // kv
    q = s["q"].double().view(rows, heads, hd)
    out = torch.zeros(rows, heads, hd, dtype=torch.float64, device="cuda")
    for r, (request, last) in enumerate(zip(s["request"].tolist(), s["position"].tolist())):
        pages = s["table"][request][:last // page + 1].long()
        for h in range(kv):
            k = s["k"][pages, h].reshape(-1, hd)[:last + 1].double()
            v = s["v"][pages, h].reshape(-1, hd)[:last + 1].double()
            mine = slice(h * group, (h + 1) * group)
            out[r, mine] = torch.softmax(torch.einsum("gd,jd->gj", q[r, mine], k) * hd ** -0.5, dim=1) @ v
    return out.reshape(rows, heads * hd)


def _exact_logprobs(s, case):
    vocab, top = case["vocab"], case["top"]
    out = {"logprob": [], "entropy": [], "top_logprob": []}
    for row, t in zip(s["logits"], s["target"].tolist()):
        lp = row[:vocab].double()
        lp = lp - lp.logsumexp(dim=0) if bool((lp > float("-inf")).any()) else lp
        p = lp.exp()
        out["logprob"].append(lp[t] if t >= 0 else torch.full_like(lp[0], float("nan")))
        out["entropy"].append(-torch.special.xlogy(p, p).sum())
        out["top_logprob"].append(lp.sort(descending=True).values[:top])
    return {**{name: torch.stack(v) for name, v in out.items()}, "rank": None, "top_index": None}


# ---- what a pass cannot do without --------------------------------------------------------------------------------

def work(case):
    if case["op"] == "plan":
        n, page = case["requests"], case["page"]
        lens = _lengths(n, case["longest"])
        if case["way"] == "release":
            return {"bytes": 12.0 * n + 8.0 * sum(_pages(x, page) for x in lens), "flops": 0.0}
        grow = _grows(case)
        need = sum(_pages(a + b, page) - _pages(a, page) for a, b in zip(lens, grow))
        return {"bytes": 24.0 * n + 16.0 * case["rows"] + 8.0 * need, "flops": 0.0}
    if case["op"] == "append":
        rows, q, kv = case["rows"], case["heads"] * case["head_dim"], case["kv_heads"] * case["head_dim"]
        row = (2 * q + 2 * kv) * BYTES[case["act"]] + 2 * kv * BYTES[case["cache"]] + 4 * case["rope_dim"] + 12
        return {"bytes": float(rows * row), "flops": 3.0 * rows * (case["heads"] + case["kv_heads"]) * case["rope_dim"]}
    if case["op"] == "attend":
        cached = sum(_lengths(case["rows"], case["longest"]))
        q = case["heads"] * case["head_dim"]
        return {"bytes": 2.0 * cached * case["kv_heads"] * case["head_dim"] * BYTES[case["cache"]] + 2.0 * case["rows"] * q * BYTES[case["act"]]
                + 4.0 * cached / case["page"], "flops": 4.0 * cached * q}
    rows = case["rows"]
    return {"bytes": float(rows * (case["vocab"] * BYTES[case["logits"]] + 16 + 8 * case["top"])), "flops": 5.0 * rows * case["vocab"]}
