"""Attention over the paged cache with many query rows per request on the GPU: the tile kernel, its items dealt whole or in
ranges of key blocks, at the places where it can go wrong; and both kernels on the same work."""
import math

import pytest
import torch

from tests import cache_reference as R
from tests.helpers import sync_ok
from tests.test_cache_gpu import check, i32, make, ops

pytestmark = pytest.mark.gpu

MANY = 10 ** 6          # max_new, taken as all rows of the batch: the tile kernel from 49 rows per key head on


def attend(c, scale=0.1, causal=True, max_new=MANY, **kw):
    got = ops().fmha_cached(*c["args"], c["cu_dev"], softmax_scale=scale, causal=causal, max_new=max_new, **kw)
    sync_ok()
    return got


# Items (256 rows of a request and key head, by max_new) that nearly fill one round of SMs, or make many, are dealt whole.
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths,new,page,Hq,Hkv,D,dtype", [
    ([131] * 70, [1, 33, 64, 0, 130, 64, 7] * 10, 16, 8, 2, 64, torch.float16),        # 140 or more items, several rounds' worth
    ([70, 300, 0, 129, 16] * 32, [70, 20, 3, 129, 1] * 32, 32, 4, 2, 128, torch.bfloat16),
    ([700, 260, 64, 1] * 25, [60, 50, 60, 60] * 25, 64, 4, 4, 64, torch.float16),       # the second tile of every pair is empty
    ([300, 256, 600], [257, 256, 10], 48, 40, 8, 64, torch.bfloat16),                   # groups of 5: rows that straddle tiles
])
def test_whole_items(lengths, new, page, Hq, Hkv, D, dtype, causal):
    c = make(lengths, new, page, Hq, Hkv, D, dtype, "token", seed=31)
    check(c, attend(c, D ** -0.5, causal, max(new)), D ** -0.5, causal, many=True)
    check(c, attend(c, D ** -0.5, causal), D ** -0.5, causal, many=True)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths,new,page,Hq,Hkv,D,dtype", [
    ([9000], [70], 16, 2, 1, 128, torch.bfloat16),                # one item over many blocks
    ([3000, 40, 1, 0, 700], [65, 40, 80, 3, 300], 64, 6, 2, 64, torch.float16),
    ([20000, 5, 60], [1, 0, 48], 32, 4, 4, 64, torch.bfloat16),   # one row against many keys
    ([129, 257, 385], [129, 257, 385], 16, 1, 1, 128, torch.float16),
    ([400, 1500, 3], [60, 60, 60], 32, 8, 8, 64, torch.float16),  # several parts and items per SM, second tiles empty
    ([60, 300, 20] * 20, [0, 100, 7] * 20, 16, 3, 1, 64, torch.bfloat16),
])
def test_ranges_of_blocks(lengths, new, page, Hq, Hkv, D, dtype, causal):
    c = make(lengths, new, page, Hq, Hkv, D, dtype, "head", seed=32, spread=2.0)
    got = attend(c, D ** -0.5, causal, max(new) if max(new) * Hq // Hkv > 48 else 49)
    check(c, got, D ** -0.5, causal, many=True)


@pytest.mark.parametrize("max_new", [1, 4, MANY])
def test_every_kernel_on_one_batch(max_new):
    """The same batch through each kernel."""
    c = make([257, 15, 16, 128], [9, 15, 1, 50], 16, 12, 2, 128, torch.bfloat16, seed=33)
    check(c, attend(c, 0.09, True, max_new), 0.09, True, many=max_new * 6 > 48)


def test_sharp_and_flat_scores():
    for scale in (0.0, 8.0, -3.0):
        c = make([777], [80], 16, 4, 2, 128, torch.float16, seed=34, spread=3.0)
        check(c, attend(c, scale), scale, True, many=True)


def test_query_magnitudes():
    c = make([200], [60], 16, 4, 4, 64, torch.bfloat16, seed=35)
    Q = c["Q"] * torch.tensor([1e30, 1e-30, 1.0, 0.0]).to(torch.bfloat16)[None, :, None]
    for h, s in enumerate([1e-31, 1e29, 0.2, 0.2]):
        got = ops().fmha_cached(Q.cuda(), *c["args"][1:], c["cu_dev"], softmax_scale=s, max_new=MANY)
        sync_ok()
        want, tol = R.attend(Q, c["code"][0].double(), c["scale"][0].double(), c["code"][1].double(), c["scale"][1].double(),
                             c["table"], c["lengths"], c["cu"], 16, s, False, True)
        assert bool(((got.cpu().double() - want).abs()[:, h] <= tol[:, h]).all())


@pytest.mark.parametrize("B", [1, 160])
def test_other_rows_stay_and_operands_may_be_strided(B):
    c = make([90] * B, [30] * B, 16, 4, 2, 128, torch.bfloat16, seed=36)
    T = 30 * B
    wide = torch.full((T + 4, 3, 4, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    wide[:T, 1] = c["args"][0]
    for out in (torch.full((T + 4, 4, 2, 128), -5.0, dtype=torch.bfloat16, device="cuda").transpose(1, 2)[:, 0],
                torch.full((T + 4, 4, 136), -5.0, dtype=torch.bfloat16, device="cuda")[:, :, 8:]):   # rows on 16 bytes, not 32
        got = ops().fmha_cached(wide[:, 1], *c["args"][1:], c["cu_dev"], softmax_scale=0.1, causal=True, max_new=30, out=out)
        sync_ok()
        assert bool((got[T:] == -5).all())
        check(c, got[:T], 0.1, True, many=True)


@pytest.mark.parametrize("B", [1, 160])
def test_bad_pages_and_lengths_are_reported_not_followed(B):
    from kernelcodegen_b200 import _lib
    c = make([100] + [40] * B, [30] * (B + 1), 16, 4, 2, 128, torch.float16, seed=37)
    good = attend(c)
    args = list(c["args"])
    for bad in (-1, 10 ** 6, 2 ** 31 - 1, -(2 ** 31)):
        table = args[5].clone()
        table[0, 2] = bad
        got = ops().fmha_cached(*args[:5], table, args[6], c["cu_dev"], softmax_scale=0.1, causal=True, max_new=MANY)
        torch.cuda.synchronize()
        assert _lib.device_status() == _lib.ERR_INVALID_ARG
        assert torch.equal(got[30:], good[30:]) and not torch.isnan(got).any()
        # all rows see keys 32 .. 47, which are left out
        ids = [p for w, p in enumerate(c["table"][0][:7]) if w != 2]
        left = dict(c, table=[ids] + c["table"][1:], lengths=[84] + [40] * B)
        check(left, got, 0.1, True, many=True)
    for bad in (10 ** 9, 2 ** 31 - 1, -5):
        lengths = args[6].clone()
        lengths[0] = bad
        ops().fmha_cached(*args[:5], args[5].clamp_min(0), lengths, c["cu_dev"], softmax_scale=0.1, causal=True, max_new=MANY)
        torch.cuda.synchronize()
        assert _lib.device_status() == _lib.ERR_INVALID_ARG
    for cu in ([0, 50, 20], [-3, 10, 20], [0, 2 ** 31 - 1, 20], [20, 10, 0]):
        ops().fmha_cached(*args, i32(cu + [20] * (B - 1)).cuda(), softmax_scale=0.1, causal=True, max_new=MANY)
        torch.cuda.synchronize()
        assert _lib.device_status() == _lib.ERR_INVALID_ARG


def test_nan_in_seen_places_reaches_the_result():
    c = make([200], [60], 16, 2, 1, 64, torch.float16, seed=38)
    for side in (1, 2):
        x = c["args"][side].clone()
        x.view(torch.uint8)[c["table"][0][1], 0, 3, 5] = 0x7F          # key 19, before every query
        args = [*c["args"][:side], x, *c["args"][side + 1:]]
        got = ops().fmha_cached(*args, c["cu_dev"], softmax_scale=0.1, causal=True, max_new=MANY)
        sync_ok()
        assert bool(torch.isnan(got if side == 1 else got[:, :, 5]).all())
        assert side == 1 or not torch.isnan(got[:, :, :5]).any()


def test_scales_of_zero_and_far_apart():
    """Pages whose scale is zero, and pages a factor of 2^14 apart, all of them seen by every row."""
    c = make([128], [64], 16, 4, 2, 64, torch.float16, seed=39, pow2=True)
    for side in range(2):
        s = c["scale"][side]
        for w, f in enumerate([1.0, 0.0, 2.0 ** -14, 1.0, 0.0, 1.0, 2.0 ** -7, 1.0]):
            s[c["table"][0][w]] *= f
    args = (*c["args"][:3], c["scale"][0].cuda(), c["scale"][1].cuda(), *c["args"][5:])
    c["args"] = args
    check(c, attend(c, 0.1, False), 0.1, False, many=True)
    check(c, attend(c, 0.1, False, 1), 0.1, False)


def test_repeatable_captured_and_on_two_streams():
    """Parts merge in a fixed order; a captured call replays to the same bits; calls in flight share nothing."""
    c = [make([2500 + 700 * i], [100], 16, 8, 2, 128, torch.float16, seed=40 + i) for i in range(2)]
    want = [attend(x) for x in c]
    streams, got = [torch.cuda.Stream() for _ in c], [[], []]
    torch.cuda.synchronize()
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops().fmha_cached(*c[i]["args"], c[i]["cu_dev"], softmax_scale=0.1, causal=True, max_new=MANY))
    sync_ok()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])
    graph, out = torch.cuda.CUDAGraph(), torch.zeros_like(want[0])
    with torch.cuda.graph(graph):
        ops().fmha_cached(*c[0]["args"], c[0]["cu_dev"], softmax_scale=0.1, causal=True, max_new=MANY, out=out)
    for _ in range(3):
        out.fill_(math.nan)
        graph.replay()
        sync_ok()
        assert torch.equal(out, want[0])


def test_no_work_at_all():
    """No request with queries or keys, in every kernel: rows stay or become zero."""
    c = make([0, 0, 7], [30, 20, 0], 16, 4, 2, 64, torch.float16, seed=42)
    for max_new in (1, 10, MANY):
        assert bool((attend(c, max_new=max_new) == 0).all())
    out = torch.full((50, 4, 64), 3.0, dtype=torch.float16, device="cuda")
    args = (out.clone(), *c["args"][1:])
    for max_new in (1, 10, MANY):
        ops().fmha_cached(*args, i32([0, 0, 0, 0]).cuda(), softmax_scale=0.1, max_new=max_new, out=out)
        sync_ok()
        assert bool((out == 3).all())


def test_cache_beyond_32_bit_offsets():
    """The last pages of a pool of more than 2^32 bytes, through append and each attention kernel."""
    pages, Hkv, page, D, n = 140000, 2, 128, 128, 300
    assert pages * Hkv * page * D > 2 ** 32
    k, v = (torch.zeros((pages, Hkv, page, D), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2))
    ks, vs = (torch.ones((pages, Hkv), device="cuda") for _ in range(2))
    ids = [pages - 1, 0, pages - 2]
    slots = [ids[t // page] * page + t % page for t in range(n)]
    g = torch.Generator().manual_seed(50)
    Q, K, V = (torch.randn((n, h, D), generator=g).to(torch.bfloat16) for h in (4, Hkv, Hkv))
    ops().cache_append(K.cuda(), V.cuda(), torch.tensor(slots).cuda(), k, v, ks, vs)
    # the pages in use, renumbered
    code = [x.view(torch.uint8)[ids].cpu().view(torch.float8_e4m3fn) for x in (k, v)]
    scale = [x[ids].cpu() for x in (ks, vs)]
    for x, c, s in ((K, code[0], scale[0]), (V, code[1], scale[1])):
        want = torch.zeros((3, Hkv, page, D), dtype=torch.float64), torch.ones((3, Hkv), dtype=torch.float64)
        R.append(x, list(range(n)), *want, page)
        assert torch.equal(c.double(), want[0]) and torch.equal(s.double(), want[1])
    for rows, max_new in ((n, MANY), (8, 8), (2, 2)):
        c = dict(Q=Q[:rows], code=code, scale=scale, table=[[0, 1, 2]], lengths=[n], cu=[0, rows], page=page)
        got = ops().fmha_cached(Q[:rows].cuda(), k, v, ks, vs, i32([ids]).cuda(), i32([n]).cuda(), softmax_scale=0.09, causal=True,
                                max_new=max_new)
        sync_ok()
        check(c, got, 0.09, True, many=rows > 24)


def test_table_without_columns():
    c = make([0, 0], [1, 30], 16, 4, 2, 64, torch.float16, seed=51)
    args = [*c["args"][:5], torch.empty((2, 0), dtype=torch.int32, device="cuda"), c["args"][6]]
    for max_new in (1, 10, MANY):
        got = ops().fmha_cached(*args, c["cu_dev"], softmax_scale=0.1, max_new=max_new)
        sync_ok()
        assert bool((got == 0).all())
