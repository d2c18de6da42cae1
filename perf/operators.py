"""What is measured of the paged 8-bit key / value cache: planning a step's pages and slots, writing new keys and
values into the cache, and attention over it, each over the sizes it meets in serving.

Layout of the cache.  Tokens live in pages of `page` tokens.  `k_cache` / `v_cache` are float8_e4m3fn
[pages, Hkv, page, D] (layout "head": a head's page is one block of memory; layout "token": stored [pages, page, Hkv, D]
and seen through a permutation), `k_scale` / `v_scale` are float32 [pages, Hkv]: a value is code * scale.  Row i of
`table` lists the pages of request i in order.
"""
import math
import random

import numpy as np
import torch

own = False

E4M3_MAX = 448.0
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---- cases --------------------------------------------------------------------------------------------------------

def listed():
    return [
        # a decode step of a full server: every request adds one token, one in sixteen needs a page
        dict(name="plan_decode", op="plan", B=64, cached=4096, new=1, page=16, ragged=True),
        # prompts of a batch being admitted, with some requests continuing
        dict(name="plan_prompts", op="plan", B=500, cached=512, new=1024, page=64, ragged=True),
        # the cache write of a decode step
        dict(name="append_decode", op="append", B=64, cached=4096, new=1, page=16, Hkv=8, D=128, dtype="bf16",
             layout="head", ragged=True),
        # the cache write of whole prompts
        dict(name="append_prompt", op="append", B=8, cached=0, new=4096, page=64, Hkv=8, D=128, dtype="bf16",
             layout="token", ragged=False),
        # chunks of prompts that begin and end inside pages, small heads
        dict(name="append_chunk", op="append", B=37, cached=700, new=701, page=48, Hkv=5, D=64, dtype="fp16",
             layout="head", ragged=True),
        # one user, a short conversation: latency
        dict(name="decode_one", op="attend", B=1, cached=1000, new=1, page=16, Hq=32, Hkv=8, D=128, dtype="bf16",
             layout="head", causal=True, ragged=False),
        # a full server, grouped heads, ragged contexts
        dict(name="decode_batch", op="attend", B=64, cached=4095, new=1, page=16, Hq=32, Hkv=8, D=128, dtype="bf16",
             layout="head", causal=True, ragged=True),
        # as many key heads as query heads, the attention benchmark's sizes with one query each
        dict(name="decode_mha", op="attend", B=8, cached=4095, new=1, page=64, Hq=32, Hkv=32, D=128, dtype="fp16",
             layout="token", causal=True, ragged=False),
        # few users, very long documents
        dict(name="decode_long", op="attend", B=2, cached=131071, new=1, page=128, Hq=32, Hkv=4, D=128, dtype="bf16",
             layout="head", causal=True, ragged=False),
        # several drafted tokens a request checked in one pass, small heads
        dict(name="verify_draft", op="attend", B=24, cached=2000, new=5, page=32, Hq=16, Hkv=4, D=64, dtype="fp16",
             layout="token", causal=True, ragged=True),
        # a chunk of a long prompt against what is cached of it
        dict(name="chunk", op="attend", B=3, cached=8191, new=513, page=16, Hq=32, Hkv=8, D=128, dtype="bf16",
             layout="head", causal=True, ragged=True),
        # whole prompts, read back from the cache they were just written to
        dict(name="prompt", op="attend", B=4, cached=0, new=4096, page=64, Hq=32, Hkv=8, D=128, dtype="bf16",
             layout="head", causal=True, ragged=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "append", "append", "attend", "attend", "attend", "attend"])
    page = rng.choice([16, 16, 32, 48, 64, 128])
    case = dict(op=op, page=page, ragged=rng.random() < 0.8)
    if op == "plan":
        case.update(B=_log(rng, 1, 2000), cached=rng.choice([0, _log(rng, 1, 8000)]),
                    new=rng.choice([1, _log(rng, 1, 1000)]))
        return case
    case.update(Hkv=rng.choice([1, 2, 3, 4, 5, 8, 16, 32]), D=rng.choice([64, 128, 128]),
                dtype=rng.choice(["bf16", "fp16"]), layout=rng.choice(["head", "token"]))
    if op == "append":
        tokens = _log(rng, 1, 30000)
        case["new"] = rng.choice([1, _log(rng, 1, min(tokens, 5000))])
        case["B"] = max(1, min(256, tokens // case["new"]))
        case["cached"] = rng.choice([0, _log(rng, 1, 4000)])
        while case["B"] * (case["cached"] + case["new"]) * case["Hkv"] * case["D"] > 250e6:
            case["B"] = max(1, case["B"] // 2)
            case["cached"] //= 2
            case["Hkv"] = max(1, case["Hkv"] // 2)
        return case
    group = rng.choice([1, 1, 2, 3, 4, 4, 7, 8])
    case["Hkv"] = min(case["Hkv"], 32 // group) or 1
    case["Hq"] = case["Hkv"] * group
    case["causal"] = rng.random() < 0.85
    kind = rng.choice(["decode", "decode", "draft", "chunk", "prompt"])
    if kind == "decode":
        case.update(new=1, B=_log(rng, 1, 128), cached=_log(rng, 1, 60000))
    elif kind == "draft":
        case.update(new=rng.randint(2, 9), B=_log(rng, 1, 64), cached=_log(rng, 1, 20000))
    elif kind == "chunk":
        case.update(new=_log(rng, 10, 1024), B=_log(rng, 1, 8), cached=_log(rng, 1, 16000))
    else:
        case.update(new=_log(rng, 2, 4096), B=_log(rng, 1, 4), cached=0)
    while (case["B"] * (case["cached"] + case["new"]) * case["Hkv"] * case["D"] > 270e6
           or case["B"] * (case["cached"] + case["new"]) * case["Hq"] * case["new"] > 2.1e9):
        case["B"] = max(1, case["B"] // 2)
        case["cached"] = case["cached"] * 2 // 3
        if case["B"] == 1:
            case["new"] = max(1, case["new"] * 2 // 3)
    return case


def _lengths(case):
    """(cached, new) of every request, as host lists; the case alone decides them."""
    r = random.Random("%d %d %d %d" % (case["B"], case["cached"], case["new"], case["page"]))
    cached, new = [], []
    for i in range(case["B"]):
        full = i == 0 or not case["ragged"]       # the longest request is always there
        cached.append(case["cached"] if full else r.randint(case["cached"] // 8, case["cached"]))
        new.append(case["new"] if full else r.randint(max(1, case["new"] // 8), case["new"]))
    return cached, new


# ---- inputs -------------------------------------------------------------------------------------------------------

def _scale_for(amax):
    """Smallest power of two s with amax / s <= 448 (float32), and at least 2^-110."""
    m, e = torch.frexp(amax)                      # amax = m * 2^e, m in [0.5, 1)
    e = torch.where(m > 0.875, e - 8, e - 9)      # 448 = 0.875 * 2^9
    e = torch.where(amax > 0, e, torch.full_like(e, -110)).clamp_min(-110)
    return torch.ldexp(torch.ones_like(amax), e)


def _filled(gen, pages, Hkv, page, D, layout, dev):
    """A cache whose pages hold keys (or values) of ordinary size, heads differing by a factor of a few."""
    x = torch.randn(pages, Hkv, page, D, generator=gen, device=dev, dtype=torch.float16)
    x *= torch.rand(1, Hkv, 1, 1, generator=gen, device=dev).mul_(2).exp_().half()
    scale = _scale_for(x.abs().amax(dim=(2, 3)).float())
    code = (x.float() / scale[:, :, None, None]).to(torch.float8_e4m3fn)
    if layout == "token":
        code = code.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    return code, scale


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    cached, new = _lengths(case)
    B, page = case["B"], case["page"]
    held = [-(-c // page) for c in cached]                          # pages before the step
    ends = [-(-(c + n) // page) for c, n in zip(cached, new)]       # and after it
    width, T = max(ends), sum(new)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    s = dict(op=case["op"], page=page, T=T, max_new=max(new), max_len=max(c + n for c, n in zip(cached, new)))
    pages = sum(ends) + 3
    order = torch.randperm(pages, generator=gen, device=dev).to(torch.int32)
    cols = torch.arange(width, device=dev, dtype=torch.int32)
    fill = held if case["op"] == "plan" else ends
    first = i32([sum(fill[:i]) for i in range(B)])
    at = first[:, None] + cols
    table = torch.where(cols < i32(fill)[:, None], order[at.clamp_max(pages - 1).long()], -1).to(torch.int32)
    if case["op"] == "plan":
        s.update(cached=i32(cached), new=i32(new), table=table, free_pages=order[sum(held):].contiguous(),
                 free_count=i32([pages - sum(held)]))
        return s
    Hkv, D, dtype = case["Hkv"], case["D"], DTYPES[case["dtype"]]
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    s["k_cache"], s["k_scale"] = _filled(gen, pages, Hkv, page, D, case["layout"], dev)
    s["v_cache"], s["v_scale"] = _filled(gen, pages, Hkv, page, D, case["layout"], dev)
    if case["op"] == "append":
        s["K"] = torch.randn(T, Hkv, D, generator=gen, device=dev).mul_(1.5).to(dtype)
        s["V"] = torch.randn(T, Hkv, D, generator=gen, device=dev).mul_(1.5).to(dtype)
        req = torch.repeat_interleave(torch.arange(B, device=dev), i32(new).long(), output_size=T)
        pos = torch.arange(T, device=dev) - i32(cu)[req] + i32(cached)[req]
        s["slots"] = table[req, pos // page].long() * page + pos % page
        # the first token of every run of tokens that share a page (the caller knows its requests' lengths)
        s["runs"] = torch.nonzero((pos % page == 0) | (pos == i32(cached)[req])).flatten()
        return s
    s.update(Q=torch.randn(T, case["Hq"], D, generator=gen, device=dev).to(dtype), table=table,
             lengths=i32([c + n for c, n in zip(cached, new)]), cu=i32(cu), scale=D ** -0.5, causal=case["causal"])
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------

def run(s):
    if own:
        from kernelcodegen_b200 import ops
        if s["op"] == "plan":
            lengths, cu, slots, left = ops.cache_plan(s["cached"], s["new"], s["table"], s["free_pages"],
                                                      s["free_count"], s["page"], s["T"])
            return dict(lengths=lengths, cu=cu, slots=slots, left=left, table=s["table"])
        if s["op"] == "append":
            ops.cache_append(s["K"], s["V"], s["slots"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
            return [s[k] for k in ("k_cache", "v_cache", "k_scale", "v_scale")]
        return ops.fmha_cached(s["Q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["table"],
                               s["lengths"], s["cu"], softmax_scale=s["scale"], causal=s["causal"],
                               max_new=s["max_new"])
    if s["op"] == "plan":
        return _plan(s)
    if s["op"] == "append":
        _append(s, s["K"], s["k_cache"], s["k_scale"])
        _append(s, s["V"], s["v_cache"], s["v_scale"])
        return [s[k] for k in ("k_cache", "v_cache", "k_scale", "v_scale")]
    return _attend(s)


def _plan(s):
    cached, new, page, table, T = s["cached"].long(), s["new"].long(), s["page"], s["table"], s["T"]
    width = table.shape[1]
    bad = (cached < 0) | (new < 0) | (cached + new > width * page)
    have = torch.div(cached + page - 1, page, rounding_mode="floor")
    need = torch.where(bad, 0, torch.div(cached + new + page - 1, page, rounding_mode="floor") - have)
    end, stop = need.cumsum(0), new.clamp_min(0).cumsum(0)
    served = ~bad & (stop <= T) & ((need == 0) | (end <= s["free_count"]))
    lengths = torch.where(served, cached + new, cached).to(torch.int32)
    taken = torch.where(served & (need > 0), end, 0).max()
    cu = torch.cat([stop.new_zeros(1), stop]).clamp_max(T)
    k = torch.arange(width, device=table.device) - have[:, None]
    at = (s["free_count"].long() - 1 - (end - need)[:, None] - k).clamp(0, s["free_pages"].numel() - 1)
    table.copy_(torch.where(served[:, None] & (k >= 0) & (k < need[:, None]), s["free_pages"][at], table))
    t = torch.arange(T, device=table.device)
    req = torch.searchsorted(stop, t, right=True).clamp_max(cached.numel() - 1)
    pos = cached[req] + t - cu[req]
    slot = table[req, torch.div(pos, page, rounding_mode="floor").clamp_max(width - 1)].long() * page + pos % page
    slot = torch.where((t < stop[-1]) & served[req], slot, -1)
    return dict(lengths=lengths, cu=cu.to(torch.int32), slots=slot, left=(s["free_count"] - taken).to(torch.int32),
                table=table)


def _append(s, x, cache, scale):
    page, slots = s["page"], s["slots"]
    at, off = torch.div(slots, page, rounding_mode="floor"), slots % page
    x = x.float()
    size = torch.where(torch.isfinite(x), x.abs(), 0).amax(dim=2)                               # [T, Hkv]
    most = torch.zeros_like(scale).scatter_reduce(0, at[:, None].expand_as(size), size, "amax")
    heads, begin = at[s["runs"]], off[s["runs"]]                                                # touched pages
    old = scale[heads]
    want = _scale_for(most[heads])
    new = torch.where((begin == 0)[:, None], want, torch.maximum(want, old))
    row = torch.arange(page, device=x.device)
    held = cache[heads].float()                                                                 # [R, Hkv, page, D]
    again = (held * (old / new)[:, :, None, None]).to(cache.dtype)
    keep = (row < begin[:, None])[:, None, :, None]
    cache[heads] = torch.where(keep, again.float(), held).to(cache.dtype)
    scale[heads] = new
    code = torch.where(torch.isfinite(x), x / scale[at][:, :, None], math.nan).to(cache.dtype)
    cache[at, :, off] = code


def _attend(s):
    page, T, n, S = s["page"], s["T"], s["max_new"], s["max_len"]
    Q, lengths, cu = s["Q"], s["lengths"].long(), s["cu"].long()
    Hq, D = Q.shape[1:]
    Hkv, G, B = s["k_cache"].shape[1], Hq // s["k_cache"].shape[1], lengths.numel()
    dev = Q.device
    new = cu[1:] - cu[:-1]
    j, key = torch.arange(n, device=dev), torch.arange(S, device=dev)
    live = j < new[:, None]                                                                     # [B, n]
    rows = (cu[:-1, None] + j).clamp_max(T - 1)
    q = Q.float()[rows].view(B, n, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * n, D)
    pages = s["table"][:, : -(-S // page)].long().clamp_min(0)

    def side(cache, scale):
        x = cache.permute(0, 2, 1, 3)[pages].float() * scale[pages][:, :, None, :, None]        # [B, W, page, Hkv, D]
        x = x.flatten(1, 2)[:, :S]
        return torch.where((key < lengths[:, None])[:, :, None, None], x, 0).transpose(1, 2)    # [B, Hkv, S, D]

    score = torch.matmul(q, side(s["k_cache"], s["k_scale"]).transpose(2, 3)) * s["scale"]
    seen = key < lengths[:, None, None]
    if s["causal"]:
        seen = seen & (key <= (lengths - new)[:, None, None] + j[:, None])                      # [B, n, S]
    seen = seen.expand(B, n, S).repeat(1, G, 1)[:, None]
    score = score.masked_fill_(~seen, -math.inf)
    p = (score - score.amax(dim=3, keepdim=True).clamp_min(-1e30)).exp_()
    o = torch.matmul(p, side(s["v_cache"], s["v_scale"])) / p.sum(dim=3, keepdim=True).clamp_min(1e-30)
    o = o.view(B, Hkv, G, n, D).permute(0, 3, 1, 2, 4).reshape(B, n, Hq, D)
    out = torch.empty_like(Q)
    req = torch.searchsorted(cu[1:], torch.arange(T, device=dev), right=True)
    out.copy_(o[req, torch.arange(T, device=dev) - cu[req]])
    return out


# ---- what a pass cannot do without --------------------------------------------------------------------------------

def work(case):
    cached, new = _lengths(case)
    T, page = sum(new), case["page"]
    if case["op"] == "plan":
        pages = sum(-(-(c + n) // page) - -(-c // page) for c, n in zip(cached, new))
        # cached, new, lengths, cu; the pages dealt (list and table); a slot a token and the table entry it names
        return {"bytes": 16 * case["B"] + 8 * pages + 8 * T + 4 * case["B"], "flops": 0}
    Hkv, D = case["Hkv"], case["D"]
    if case["op"] == "append":
        pages = sum(-(-(c + n) // page) - c // page for c, n in zip(cached, new))
        return {"bytes": 2 * T * Hkv * D * 3 + 8 * T + 2 * pages * Hkv * 8, "flops": 2 * T * Hkv * D * 2}
    pages = sum(-(-(c + n) // page) for c, n in zip(cached, new))
    keys = sum(c + n for c, n in zip(cached, new))
    seen = sum(n * (c + n) - (n * (n - 1) // 2 if case["causal"] else 0) for c, n in zip(cached, new))
    return {"bytes": 2 * keys * Hkv * D + pages * (8 * Hkv + 4) + 2 * 2 * T * case["Hq"] * D + 8 * case["B"],
            "flops": 4 * D * case["Hq"] * seen}


# ---- the definition, in 64 bits -----------------------------------------------------------------------------------

def _round_e4m3(y):
    """float64 to the nearest e4m3 value, ties to even; |y| <= 448 or NaN."""
    _, e = torch.frexp(y)
    step = torch.ldexp(torch.ones_like(y), (e - 1).clamp_min(-6) - 3)
    return torch.round(y / step) * step


def _exact_append(case, x, cache, scale, slots):
    page = case["page"]
    value, scale = cache.double(), scale.double()
    x, at, off = x.double(), (slots // page).cpu().numpy(), (slots % page).cpu().numpy()
    first = np.flatnonzero((np.diff(at, prepend=-1) != 0))           # a page's tokens stand together
    for a, b in zip(first, [*first[1:], len(at)]):
        p, o = int(at[a]), int(off[a])
        amax = x[a:b].abs().amax(dim=(0, 2))
        s = torch.ldexp(torch.ones_like(amax), torch.ceil(torch.log2(amax / E4M3_MAX)).int()).clamp_min(2.0 ** -110)
        s = torch.where(amax <= E4M3_MAX * s / 2, s / 2, s).clamp_min(2.0 ** -110)     # log2 of a power of two may round up
        if o:
            s = torch.maximum(s, scale[p])
            value[p, :, :o] = _round_e4m3(value[p, :, :o] * (scale[p] / s)[:, None, None])
        scale[p] = s
        value[p, :, o:o + b - a] = _round_e4m3(x[a:b] / s[:, None]).transpose(0, 1)
    return value, scale


def exact(case, seed):
    if case["op"] == "plan":
        return None
    s = prepare(case, seed)
    page = case["page"]
    if case["op"] == "append":
        if s["runs"].numel() > 6000:
            return None
        k, ks = _exact_append(case, s["K"], s["k_cache"], s["k_scale"], s["slots"])
        v, vs = _exact_append(case, s["V"], s["v_cache"], s["v_scale"], s["slots"])
        return [k, v, ks, vs]
    cached, new = _lengths(case)
    out, start = torch.zeros(s["Q"].shape, dtype=torch.float64, device=s["Q"].device), 0
    group = case["Hq"] // case["Hkv"]
    for i, (c, n) in enumerate(zip(cached, new)):
        ids = s["table"][i, : -(-(c + n) // page)].long()
        pos = torch.arange(n, device=out.device)[:, None] + c
        blind = (torch.arange(c + n, device=out.device) > pos) if case["causal"] else None
        for h in range(case["Hkv"]):
            K = (s["k_cache"][ids, h].double() * s["k_scale"][ids, h].double()[:, None, None]).reshape(-1, case["D"])
            V = (s["v_cache"][ids, h].double() * s["v_scale"][ids, h].double()[:, None, None]).reshape(-1, case["D"])
            for g in range(h * group, (h + 1) * group):
                z = s["Q"][start:start + n, g].double() @ K[: c + n].T * s["scale"]
                if blind is not None:
                    z = z.masked_fill(blind, -math.inf)
                out[start:start + n, g] = torch.softmax(z, dim=1) @ V[: c + n]
        start += n
    return out
