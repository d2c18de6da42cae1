"""The paged 8-bit key / value cache on the GPU: planning, appending and attention against their restatement in
64 bits (tests/cache_reference.py).  Planning and appending are compared bit for bit; attention element by element
within the error its arithmetic admits."""
import ctypes
import math
import random

import pytest
import torch

from tests import cache_reference as R
from tests.helpers import gen, sync_ok

pytestmark = pytest.mark.gpu


def ops():
    from kernelcodegen_b200 import ops as _ops
    return _ops


def i32(v):
    return torch.tensor(v, dtype=torch.int32)


# ---- planning -----------------------------------------------------------------------------------------------------

def run_plan(cached, new, page, max_tokens=None, width=None, free=None, extra_rows=0, in_place=False):
    B = len(cached)
    rng = random.Random(B * 1000 + page)
    held = [max(0, -(-c // page)) for c in cached]
    width = width or max([1] + [-(-(max(c, 0) + max(n, 0)) // page) for c, n in zip(cached, new)])
    pool = list(range(sum(held) + 5000))
    rng.shuffle(pool)
    table, at = [], 0
    for h in held:
        row = pool[at:at + h][:width]
        table.append(row + [-7] * (width - len(row)))
        at += h
    free_pages = pool[at:]
    free = len(free_pages) if free is None else free
    max_tokens = sum(max(n, 0) for n in new) if max_tokens is None else max_tokens
    table += [[-9] * width for _ in range(extra_rows)]
    tab = i32(table).cuda()
    c, n, f = i32(cached).cuda(), i32(new).cuda(), i32([free]).cuda()
    out = None
    if in_place:
        out = (c, torch.empty(B + 1, dtype=torch.int32, device="cuda"),
               torch.empty(max_tokens, dtype=torch.int64, device="cuda"), f)
    got = ops().cache_plan(c, n, tab, i32(free_pages).cuda(), f, page, max_tokens, out=out)
    want = R.plan(cached, new, table, free_pages, free, page, max_tokens)
    torch.cuda.synchronize()
    for g, w, name in zip(got, (*want[:3], [want[3]]), ("lengths", "cu_new", "slot_map", "free_left")):
        assert g.cpu().tolist() == list(w), name
    assert tab.cpu().tolist() == table


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("B,cached,new,page", [(1, 0, 1, 16), (1, 16, 1, 16), (3, 15, 2, 16), (64, 300, 1, 16),
                                              (700, 90, 9, 32), (37, 1000, 333, 48), (5, 0, 4096, 64), (1025, 3, 1, 1)])
def test_plan(B, cached, new, page, in_place):
    r = random.Random(B)
    run_plan([r.randint(0, cached) for _ in range(B)], [r.randint(0, new) for _ in range(B)], page, in_place=in_place)
    sync_ok()


def test_plan_with_no_request_and_with_padding():
    run_plan([], [], 16, max_tokens=5, width=3, extra_rows=2)
    run_plan([5, 0, 31], [1, 0, 1], 16, max_tokens=11, extra_rows=3)
    run_plan([0, 0], [0, 0], 16)
    sync_ok()


def test_plan_serves_in_order_until_the_pages_run_out():
    run_plan([0, 10, 0, 20, 5], [40, 3, 33, 1, 2], 16, free=3)        # the third goes without, the last two need none
    run_plan([0, 16, 16], [16, 1, 16], 16, free=1)
    run_plan([3, 3], [1, 1], 16, free=0)
    sync_ok()


def test_plan_cuts_at_the_token_limit_and_at_the_table_width():
    run_plan([0, 0, 0, 4], [10, 10, 10, 1], 16, max_tokens=25)
    run_plan([40, 10], [9, 5], 16, width=3)                            # 49 tokens do not fit three pages
    sync_ok()


def test_plan_reports_negative_counts():
    from kernelcodegen_b200 import _lib
    run_plan([4, -1, 7], [1, 3, 2], 16)
    assert _lib.device_status() == _lib.ERR_INVALID_ARG
    run_plan([4, 1, 7], [1, -3, 2], 16)
    assert _lib.device_status() == _lib.ERR_INVALID_ARG
    tab = i32([[0, 0]]).cuda()
    got = ops().cache_plan(i32([16]).cuda(), i32([1]).cuda(), tab, i32([3, 4]).cuda(), i32([9]).cuda(), 16, 1)
    torch.cuda.synchronize()
    assert _lib.device_status() == _lib.ERR_INVALID_ARG                # nine pages of a list of two: cut to two
    assert got[3].item() == 1 and tab.cpu().tolist() == [[0, 4]]


# ---- appending ----------------------------------------------------------------------------------------------------

def buffers(pages, Hkv, page, D, layout, seed, poison=True):
    """A pool of codes and scales, strided by `layout`, every byte NaN and every scale NaN where poison."""
    shape = (pages, Hkv, page, D) if layout == "head" else (pages, page, Hkv, D)
    raw = torch.full(shape, 0x7F, dtype=torch.uint8, device="cuda")
    code = raw.view(R.E4M3)
    if layout == "token":
        code = code.permute(0, 2, 1, 3)
    return code, torch.full((pages, Hkv), math.nan, device="cuda")


def same_codes(got, want):
    """float8 tensor against float64 code values, bit for bit up to the sign of zero."""
    g = got.cpu().to(torch.float64)
    return torch.equal(torch.isnan(g), torch.isnan(want)) and torch.equal(g.nan_to_num(), want.nan_to_num())


@pytest.mark.parametrize("layout", ["head", "token"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("page,Hkv,D", [(16, 2, 128), (48, 3, 64), (256, 1, 128)])
def test_append_step_by_step(page, Hkv, D, dtype, layout):
    """Requests grow over several steps: new pages, pages filled in parts, scales that grow and that stay."""
    steps = [[5, 0, 40], [1, 17, 1], [1, 1, 0], [300, 1, 2]]
    B = 3
    pages = 100
    free = list(range(pages))
    random.Random(page).shuffle(free)
    table = [[-1] * 30 for _ in range(B)]
    cached, left = [0] * B, pages
    k, ks = buffers(pages, Hkv, page, D, layout, 0)
    v, vs = buffers(pages, Hkv, page, D, layout, 1)
    want = [(x.cpu().double(), s.cpu().double()) for x, s in ((k, ks), (v, vs))]
    g = gen(page + D)
    for step, new in enumerate(steps):
        T = sum(new)
        cached, _, slots, left = R.plan(cached, new, table, free, left, page, T)
        size = 10.0 ** (2 * (step % 3) - 2)
        # a packed projection: K and V are strided views of it
        kv = (torch.randn((T, 2, Hkv, D), generator=g) * size).to(dtype)
        if step == 2:
            kv[:] = 0
        dev = kv.cuda()
        ops().cache_append(dev[:, 0], dev[:, 1], torch.tensor(slots).cuda(), k, v, ks, vs)
        for side in range(2):
            R.append(kv[:, side], slots, *want[side], page)
        sync_ok()
        for (code, scale), (wc, ws) in zip(((k, ks), (v, vs)), want):
            assert same_codes(code, wc)
            assert torch.equal(scale.cpu().double().nan_to_num(), ws.nan_to_num())


@pytest.mark.parametrize("T", [1, 33, 700, 9000])
def test_append_many_tokens(T):
    """From one warp per token to thirty-two tokens per warp."""
    page, Hkv, D = 32, 8, 64
    pages = -(-T // page) + 1
    k, ks = buffers(pages, Hkv, page, D, "head", 0)
    v, vs = buffers(pages, Hkv, page, D, "head", 1)
    g = gen(T)
    K, V = (torch.randn((T, Hkv, D), generator=g).to(torch.bfloat16) for _ in range(2))
    slots = [t + 7 for t in range(T)]          # begins inside a page that holds nothing yet
    ks[0], vs[0] = 0.25, 2.0 ** -20
    k.view(torch.uint8)[0, :, :7] = 0x38       # 1.0
    v.view(torch.uint8)[0, :, :7] = 0x38
    wk, wv = [(x.cpu().double(), s.cpu().double()) for x, s in ((k, ks), (v, vs))]
    ops().cache_append(K.cuda(), V.cuda(), torch.tensor(slots).cuda(), k, v, ks, vs)
    R.append(K, slots, *wk, page)
    R.append(V, slots, *wv, page)
    sync_ok()
    for (code, scale), (wc, ws) in zip(((k, ks), (v, vs)), (wk, wv)):
        assert same_codes(code, wc)
        assert torch.equal(scale.cpu().double().nan_to_num(), ws.nan_to_num())


def test_append_skips_and_special_values():
    from kernelcodegen_b200 import _lib
    page, Hkv, D = 16, 1, 64
    k, ks = buffers(3, Hkv, page, D, "head", 0)
    v, vs = buffers(3, Hkv, page, D, "head", 1)
    K = torch.zeros(6, Hkv, D, dtype=torch.float16)
    K[0, 0, 0], K[0, 0, 1], K[0, 0, 2] = math.inf, -3.0, math.nan
    K[2] = 65504.0
    K[3] = 6e-8
    K[4, 0, 5] = -math.inf
    V = -K
    slots = [16, -1, 17, 0, 32, -1]
    wk, wv = [(x.cpu().double(), s.cpu().double()) for x, s in ((k, ks), (v, vs))]
    ops().cache_append(K.cuda(), V.cuda(), torch.tensor(slots).cuda(), k, v, ks, vs)
    R.append(K, slots, *wk, page)
    R.append(V, slots, *wv, page)
    sync_ok()
    for (code, scale), (wc, ws) in zip(((k, ks), (v, vs)), (wk, wv)):
        assert same_codes(code, wc)
        assert torch.equal(scale.cpu().double().nan_to_num(), ws.nan_to_num())
    # gaps between a page's tokens: skipped tokens and rows that nobody writes
    K2 = torch.randn((80, Hkv, D), generator=gen(5)).to(torch.float16)
    slots2 = [-1] * 80
    for t, s in ((0, 3), (1, 5), (20, 6), (51, 15), (52, 16), (79, 47)):
        slots2[t] = s
    K2[2] = math.inf
    ops().cache_append(K2.cuda(), K2.cuda(), torch.tensor(slots2).cuda(), k, v, ks, vs)
    R.append(K2, slots2, *wk, page)
    R.append(K2, slots2, *wv, page)
    sync_ok()
    for (code, scale), (wc, ws) in zip(((k, ks), (v, vs)), (wk, wv)):
        assert same_codes(code, wc)
        assert torch.equal(scale.cpu().double().nan_to_num(), ws.nan_to_num())
    # slots outside the pool: skipped and reported
    before = k.view(torch.uint8).clone()
    for bad in (48, -2, 2 ** 62, -(2 ** 62)):
        ops().cache_append(K[:1].cuda(), V[:1].cuda(), torch.tensor([bad]).cuda(), k, v, ks, vs)
        torch.cuda.synchronize()
        assert _lib.device_status() == _lib.ERR_INVALID_ARG
    assert torch.equal(k.view(torch.uint8), before)


# ---- attention ----------------------------------------------------------------------------------------------------

def make(lengths, new, page, Hq, Hkv, D, dtype, layout="head", seed=0, spread=1.0, pow2=False, size=1.0):
    """Inputs on the host and on the GPU.  Everything that must not be read is NaN: rows behind a request's last
    token, pages of nobody, their scales, table entries behind the last page (-1)."""
    g = gen(seed)
    B = len(lengths)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    need = [-(-L // page) for L in lengths]
    pages = sum(need) + 2
    ids = torch.randperm(pages, generator=g).tolist()
    width = max([1] + need) + 1
    table, at = [], 0
    for n in need:
        table.append(ids[at:at + n] + [-1] * (width - n))
        at += n
    code, scale = [], []
    for _ in range(2):
        c = torch.randn((pages, Hkv, page, D), generator=g) * 60 * size
        c = c.clamp(-448, 448).to(R.E4M3)
        s = torch.exp(torch.randn((pages, Hkv), generator=g) * spread) / 60
        if pow2:
            s = torch.exp2(torch.round(torch.log2(s)))
        used = torch.zeros(pages, dtype=torch.bool)
        for i in range(B):
            for w in range(need[i]):
                used[table[i][w]] = True
                end = lengths[i] - w * page
                if end < page:
                    c.view(torch.uint8)[table[i][w], :, end:] = 0x7F
        c.view(torch.uint8)[~used] = 0x7F
        s[~used] = math.nan
        code.append(c)
        scale.append(s)
    Q = torch.randn((cu[-1], Hq, D), generator=g).to(dtype)
    dev = []
    for c in code:
        if layout == "token":
            c = c.permute(0, 2, 1, 3).contiguous().cuda().permute(0, 2, 1, 3)
        dev.append(c.cuda())
    return dict(Q=Q, code=code, scale=scale, table=table, lengths=lengths, cu=cu, page=page,
                args=(Q.cuda(), dev[0], dev[1], scale[0].cuda(), scale[1].cuda(), i32(table).cuda(), i32(lengths).cuda()),
                cu_dev=i32(cu).cuda())


def check(c, got, softmax_scale, causal, many=False):
    want, tol = R.attend(c["Q"], c["code"][0].double(), c["scale"][0].double(), c["code"][1].double(),
                         c["scale"][1].double(), c["table"], c["lengths"], c["cu"], c["page"], softmax_scale, causal, many)
    got = got.cpu().double()
    off = (got - want).abs()
    assert not torch.isnan(got).any()
    worst = (off / tol.clamp_min(1e-300)).max().item() if off.numel() else 0.0
    assert worst <= 1, f"{worst} of the allowed error"


CASES = [
    # lengths, new, page, Hq, Hkv, D
    ([1], [1], 16, 1, 1, 128),
    ([17], [1], 16, 4, 1, 64),
    ([128, 1, 129, 31, 32, 33], [1] * 6, 32, 8, 2, 128),
    ([700, 3, 250], [1, 1, 1], 48, 6, 2, 64),
    ([1500], [1], 64, 8, 1, 128),
    ([300, 5, 90, 64], [5, 5, 1, 3], 16, 6, 3, 128),      # several queries, all of a request's tokens new
    ([40, 0, 200], [3, 2, 0], 16, 4, 4, 64),              # a request without keys, one without queries
    ([260, 130], [40, 130], 128, 14, 2, 128),             # several row blocks
    ([2], [6], 16, 3, 1, 64),                             # rows before the first key
    ([513, 4000], [200, 77], 16, 8, 4, 128),
    ([1000], [1000], 64, 2, 1, 64),
]


@pytest.mark.parametrize("layout", ["head", "token"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention(case, causal, dtype, layout):
    lengths, new, page, Hq, Hkv, D = CASES[case]
    c = make(lengths, new, page, Hq, Hkv, D, dtype, layout, seed=case)
    got = ops().fmha_cached(*c["args"], c["cu_dev"], softmax_scale=D ** -0.5, causal=causal, max_new=max(new))
    sync_ok()
    check(c, got, D ** -0.5, causal, many=max(new) * Hq // Hkv > 48)


@pytest.mark.parametrize("max_new", [0, 1, 7, 10 ** 6])
def test_attention_max_new_is_only_a_hint(max_new):
    c = make([300, 90, 40], [60, 1, 40], 16, 8, 2, 128, torch.bfloat16, seed=3)
    got = ops().fmha_cached(*c["args"], c["cu_dev"], softmax_scale=0.1, causal=True, max_new=max_new)
    sync_ok()
    check(c, got, 0.1, True, many=True)


@pytest.mark.parametrize("B,length,new", [(300, 200, 1), (1, 40000, 1), (2000, 20, 1), (3, 9000, 2)])
def test_attention_work_split(B, length, new):
    """Many short requests, few long ones: items inside a block, items over many blocks, blocks without work."""
    r = random.Random(B)
    lengths = [r.randint(max(new, length // 4), length) for _ in range(B)]
    c = make(lengths, [new] * B, 16, 2, 1, 64, torch.float16, seed=B, pow2=True)
    got = ops().fmha_cached(*c["args"], c["cu_dev"], softmax_scale=0.125, causal=True, max_new=new)
    sync_ok()
    check(c, got, 0.125, True)
    again = ops().fmha_cached(*c["args"], softmax_scale=0.125, causal=True, max_new=new)   # T / B rows each
    sync_ok()
    assert torch.equal(got, again)


def test_attention_sharp_and_flat_scores():
    for scale in (0.0, 8.0, -3.0):
        c = make([777], [3], 16, 4, 2, 128, torch.float16, seed=11, spread=3.0)
        got = ops().fmha_cached(*c["args"], c["cu_dev"], softmax_scale=scale, causal=True)
        sync_ok()
        check(c, got, scale, True)


def test_attention_query_magnitudes():
    """bfloat16 queries reach far beyond float16's range, in both directions."""
    c = make([200], [4], 16, 4, 4, 64, torch.bfloat16, seed=12)
    Q = c["Q"] * torch.tensor([1e30, 1e-30, 1.0, 0.0]).to(torch.bfloat16)[None, :, None]
    c["Q"] = Q
    scale = [1e-31, 1e29, 0.2, 0.2]
    for h, s in enumerate(scale):
        got = ops().fmha_cached(Q.cuda(), *c["args"][1:], c["cu_dev"], softmax_scale=s, causal=False)
        sync_ok()
        want, tol = R.attend(Q, c["code"][0].double(), c["scale"][0].double(), c["code"][1].double(), c["scale"][1].double(),
                             c["table"], c["lengths"], c["cu"], 16, s, False)
        assert bool(((got.cpu().double() - want).abs()[:, h] <= tol[:, h]).all())


def test_attention_leaves_other_rows_and_takes_strided_operands():
    c = make([90, 20], [3, 2], 16, 4, 2, 128, torch.bfloat16, seed=13)
    T = 5
    wide = torch.full((T + 4, 3, 4, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    wide[:T, 1] = c["args"][0]
    out = torch.full((T + 4, 4, 2, 128), -5.0, dtype=torch.bfloat16, device="cuda").transpose(1, 2)[:, 0]
    cu = c["cu_dev"]
    got = ops().fmha_cached(wide[:, 1], *c["args"][1:], cu, softmax_scale=0.1, causal=True,
                            out=out)
    sync_ok()
    assert bool((got[T:] == -5).all())
    check(c, got[:T], 0.1, True)


def test_attention_bad_pages_and_lengths_are_reported_not_followed():
    from kernelcodegen_b200 import _lib
    c = make([100, 40], [1, 1], 16, 4, 2, 128, torch.float16, seed=14)
    good = ops().fmha_cached(*c["args"], c["cu_dev"], softmax_scale=0.1, causal=True)
    sync_ok()
    args = list(c["args"])
    for bad in (-1, 10 ** 6, 2 ** 31 - 1, -(2 ** 31)):
        table = args[5].clone()
        table[0, 2] = bad
        got = ops().fmha_cached(*args[:5], table, args[6], c["cu_dev"], softmax_scale=0.1, causal=True)
        torch.cuda.synchronize()
        assert _lib.device_status() == _lib.ERR_INVALID_ARG
        assert torch.equal(got[1], good[1]) and not torch.isnan(got).any()
        # the page's sixteen keys are left out
        ids = [p for w, p in enumerate(c["table"][0][:7]) if w != 2]
        left = dict(c, table=[ids, c["table"][1]], lengths=[84, 40])
        check(left, got, 0.1, True)
    lengths = args[6].clone()
    for bad in (10 ** 9, 2 ** 31 - 1, -5):
        lengths[0] = bad
        table = args[5].clamp_min(0)
        ops().fmha_cached(*args[:5], table, lengths, c["cu_dev"], softmax_scale=0.1, causal=True)
        torch.cuda.synchronize()
        assert _lib.device_status() == _lib.ERR_INVALID_ARG
    for cu in ([0, 5, 2], [-3, 1, 2], [0, 2 ** 31 - 1, 2], [2, 1, 0]):
        out = torch.zeros_like(args[0])
        ops().fmha_cached(*args, i32(cu).cuda(), softmax_scale=0.1, causal=True, out=out)
        torch.cuda.synchronize()
        assert _lib.device_status() == _lib.ERR_INVALID_ARG


def test_attention_nan_in_seen_places_reaches_the_result():
    c = make([40], [1], 16, 2, 1, 64, torch.float16, seed=15)
    k = c["args"][1].clone()
    k.view(torch.uint8)[c["table"][0][1], 0, 3, 5] = 0x7F
    got = ops().fmha_cached(c["args"][0], k, *c["args"][2:], c["cu_dev"], softmax_scale=0.1)
    sync_ok()
    assert bool(torch.isnan(got).all())
    v = c["args"][2].clone()
    v.view(torch.uint8)[c["table"][0][1], 0, 3, 5] = 0x7F
    got = ops().fmha_cached(*c["args"][:2], v, *c["args"][3:], c["cu_dev"], softmax_scale=0.1)
    sync_ok()
    assert bool(torch.isnan(got[:, :, 5]).all()) and not torch.isnan(got[:, :, :5]).any()


# ---- together -----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("graph", [False, True])
def test_serving_loop(graph):
    """Prompts, then single tokens: plan, append and attend on one stream, eagerly and as a graph replayed for every
    token with lengths and the free count updated in place; two graphs of the same step alternate."""
    B, page, Hq, Hkv, D, dtype = 3, 16, 4, 2, 64, torch.bfloat16
    prompts, steps = [37, 1, 16], 6
    g = gen(99)
    pages, width = 40, 8
    free = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((B, width), -1, dtype=torch.int32)
    host_table, host_free, cached, left = table.tolist(), free.tolist(), [0] * B, pages
    dev = torch.device("cuda")
    k, ks = buffers(pages, Hkv, page, D, "token", 0)
    v, vs = buffers(pages, Hkv, page, D, "token", 1)
    wk, wv = [(x.cpu().double(), s.cpu().double()) for x, s in ((k, ks), (v, vs))]
    d_table, d_free, d_left, d_len = table.to(dev), free.to(dev), i32([pages]).to(dev), torch.zeros(B, dtype=torch.int32, device=dev)
    d_one = torch.ones(B, dtype=torch.int32, device=dev)
    step_in = [torch.zeros((B, Hq + 2 * Hkv, D), dtype=dtype, device=dev) for _ in range(2)]
    step_out = [torch.zeros((B, Hq, D), dtype=dtype, device=dev) for _ in range(2)]
    cu_out = [torch.empty(B + 1, dtype=torch.int32, device=dev) for _ in range(2)]
    slot_out = [torch.empty(B, dtype=torch.int64, device=dev) for _ in range(2)]

    def step(which):
        x = step_in[which]
        _, cu, slots, _ = ops().cache_plan(d_len, d_one, d_table, d_free, d_left, page, B,
                                           out=(d_len, cu_out[which], slot_out[which], d_left))
        ops().cache_append(x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:], slots, k, v, ks, vs)
        ops().fmha_cached(x[:, :Hq], k, v, ks, vs, d_table, d_len, cu, softmax_scale=D ** -0.5, causal=True, max_new=1,
                          out=step_out[which])

    def verify(x, got, new, slots, cu):
        R.append(x[:, Hq:Hq + Hkv], slots, *wk, page)
        R.append(x[:, Hq + Hkv:], slots, *wv, page)
        c = dict(Q=x[:, :Hq], table=host_table, lengths=cached, cu=cu, page=page)
        want, tol = R.attend(c["Q"], wk[0], wk[1], wv[0], wv[1], host_table, cached, cu, page, D ** -0.5, True)
        assert bool(((got.cpu().double() - want).abs() <= tol).all())

    T = sum(prompts)
    x = torch.randn((T, Hq + 2 * Hkv, D), generator=g).to(dtype)
    dx = x.to(dev)
    lengths, cu, slots, left_dev = ops().cache_plan(d_len, i32(prompts).to(dev), d_table, d_free, d_left, page, T)
    ops().cache_append(dx[:, Hq:Hq + Hkv], dx[:, Hq + Hkv:], slots, k, v, ks, vs)
    got = ops().fmha_cached(dx[:, :Hq], k, v, ks, vs, d_table, lengths, cu, softmax_scale=D ** -0.5, causal=True)
    d_len.copy_(lengths)
    d_left.copy_(left_dev)
    sync_ok()
    cached, hcu, hslots, left = R.plan(cached, prompts, host_table, host_free, left, page, T)
    verify(x, got, prompts, hslots, hcu)

    graphs = []
    if graph:
        saved = [t.clone() for t in (d_len, d_left, d_table, k.view(torch.uint8), v.view(torch.uint8), ks, vs)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(0)
        torch.cuda.current_stream().wait_stream(side)
        for which in range(2):
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr):
                step(which)
            graphs.append(gr)
        for t, s in zip((d_len, d_left, d_table, k.view(torch.uint8), v.view(torch.uint8), ks, vs), saved):
            t.copy_(s)
    for n in range(steps):
        which = n % 2
        x = torch.randn((B, Hq + 2 * Hkv, D), generator=g).to(dtype) * (3 if n == 3 else 1)
        step_in[which].copy_(x)
        if graph:
            graphs[which].replay()
        else:
            step(which)
        sync_ok()
        cached, hcu, hslots, left = R.plan(cached, [1] * B, host_table, host_free, left, page, B)
        assert d_len.tolist() == cached and d_left.item() == left and d_table.tolist() == host_table
        verify(x, step_out[which], [1] * B, hslots, hcu)


def test_two_streams_at_once():
    """Calls in flight together do not share a workspace."""
    c = [make([3000 + i], [1], 16, 8, 2, 128, torch.float16, seed=20 + i) for i in range(2)]
    want = [ops().fmha_cached(*x["args"], x["cu_dev"], softmax_scale=0.1, max_new=1) for x in c]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in c]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops().fmha_cached(*c[i]["args"], c[i]["cu_dev"], softmax_scale=0.1, max_new=1))
    sync_ok()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


@pytest.mark.parametrize("new", [1, 6])
def test_attention_scales_of_other_requests_do_not_leak(new):
    """A request whose scales are NaN shares a block's buffers with one whose last half tile holds no keys."""
    B = 1200
    c = make([32, 10] * (B // 2), [new] * B, 16, 4, 1, 64, torch.float16, seed=61)
    want = ops().fmha_cached(*c["args"], c["cu_dev"], softmax_scale=0.1, causal=True, max_new=new)
    ks, vs = c["args"][3].clone(), c["args"][4].clone()
    for i in range(0, B, 2):
        ks[c["table"][i][1]] = math.nan
        vs[c["table"][i][1]] = math.nan
    got = ops().fmha_cached(*c["args"][:3], ks, vs, *c["args"][5:], c["cu_dev"], softmax_scale=0.1, causal=True, max_new=new)
    sync_ok()
    got, want = got.view(B, new, 4, 64), want.view(B, new, 4, 64)
    assert bool(torch.isnan(got[::2, -1]).all()) and torch.equal(got[1::2], want[1::2])


@pytest.mark.parametrize("word", [-1, 0, 1, 2 ** 30, 2 ** 31 - 1, 0x7FC00000])
def test_attention_workspace_may_hold_anything(word):
    from kernelcodegen_b200 import _lib
    size = ctypes.c_size_t()
    assert _lib.load().kcg_fmha_cached_workspace(64, ctypes.byref(size)) == 0
    for lengths, new in (([5, 200, 0, 3000], 1), ([40, 1000], 6), ([700, 60], 70)):
        c = make(lengths, [new] * len(lengths), 16, 4, 2, 64, torch.float16, seed=62)
        st2, st3 = (ctypes.c_int64 * 2)(256, 64), (ctypes.c_int64 * 3)(2048, 1024, 64)
        work = torch.full((size.value // 4,), word, dtype=torch.int32, device="cuda")
        Q, k, v, ks, vs, table, lens = c["args"]
        out = torch.empty_like(Q)
        rc = _lib.load().kcg_fmha_cached_fwd(_lib.F16, Q.shape[0], len(lengths), 4, 2, 64, new, 0.1, 1, Q.data_ptr(), st2, k.data_ptr(), st3,
                                             ks.data_ptr(), v.data_ptr(), st3, vs.data_ptr(), k.shape[0], 16, table.data_ptr(),
                                             table.shape[1], table.stride(0), lens.data_ptr(), None, out.data_ptr(), st2,
                                             work.data_ptr(), size.value, torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        sync_ok()
        check(c, out, 0.1, True, many=new * 2 > 48)
