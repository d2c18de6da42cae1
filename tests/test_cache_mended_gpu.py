"""Calls of the paged-cache entry points that were once answered wrongly, or by a path that no other test reaches."""
import ctypes
import math

import pytest
import torch

from tests import cache_reference as R
from tests.helpers import sync_ok
from tests.test_cache_gpu import check, make, ops
from tests.test_cache_mended_cpu import check_pages, draft_steps, give_back

pytestmark = pytest.mark.gpu

MANY = 10 ** 6          # max_new, taken as all rows of the batch: the tile kernel from 49 rows per key head on


def attend_c(c, softmax_scale, causal, max_new, at=0, q=None, out=None, turned=False):
    """fmha_cached through the C ABI, with a workspace of exactly the bytes asked for, `at` bytes behind a 512-byte boundary.
    turned: the rows of q and out stand in memory in reverse order, reached by a negative stride."""
    from kernelcodegen_b200 import _lib
    lib = _lib.load()
    Q, k, v, ks, vs, table, lens = c["args"]
    Q = Q if q is None else q
    out = torch.empty_like(Q) if out is None else out
    strides = lambda t: (ctypes.c_int64 * (t.dim() - 1))(*t.stride()[:-1])  # noqa: E731
    rows = (lambda t: (ctypes.c_int64 * 2)(-t.stride(0), t.stride(1))) if turned else strides  # noqa: E731
    first = (lambda t: t[-1].data_ptr()) if turned else torch.Tensor.data_ptr  # noqa: E731
    size = ctypes.c_size_t()
    assert lib.kcg_fmha_cached_workspace(Q.shape[2], ctypes.byref(size)) == 0
    room = torch.full((size.value + 1024,), 0x5A, dtype=torch.uint8, device="cuda")
    room = room[-room.data_ptr() % 512:]
    _lib.check(lib.kcg_fmha_cached_fwd(_lib.F16 if Q.dtype == torch.float16 else _lib.BF16, Q.shape[0], lens.shape[0], Q.shape[1],
                                       k.shape[1], Q.shape[2], max_new, softmax_scale, causal, first(Q), rows(Q), k.data_ptr(),
                                       strides(k), ks.data_ptr(), v.data_ptr(), strides(v), vs.data_ptr(), k.shape[0], c["page"],
                                       table.data_ptr(), table.shape[1], table.stride(0), lens.data_ptr(), c["cu_dev"].data_ptr(),
                                       first(out), rows(out), room.data_ptr() + at, size.value,
                                       torch.cuda.current_stream().cuda_stream), "kcg_fmha_cached_fwd")
    sync_ok()
    assert bool((room[:at] == 0x5A).all()) and bool((room[at + size.value:] == 0x5A).all())
    return out


@pytest.mark.parametrize("at", [0, 16, 32, 48])
@pytest.mark.parametrize("D", [64, 128])
def test_workspace_at_any_multiple_of_16_bytes(D, at):
    """One chunk against a context, in ranges whose parts go through the workspace, and the same by the split kernel."""
    c = make([2300, 90], [60, 60], 16, 4, 2, D, torch.bfloat16, seed=71)
    want = ops().fmha_cached(*c["args"], c["cu_dev"], softmax_scale=0.1, causal=True, max_new=60)
    got = attend_c(c, 0.1, 1, 60, at)
    check(c, got, 0.1, True, many=True)
    assert torch.equal(got, want)
    c = make([2300, 90], [3, 3], 16, 4, 2, D, torch.bfloat16, seed=72)
    check(c, attend_c(c, 0.1, 1, 3, at), 0.1, True)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("big", [0, 9])                  # in a block before most pages, or in a later one
@pytest.mark.parametrize("below", [14, 15, 20, 25, 28, 33])
@pytest.mark.parametrize("side", ["K", "V"])
def test_pages_far_below_their_neighbours_keep_what_f16_holds(side, below, big, causal):
    """One page's scale is 1, all others 2^-below, and the rows' weight lies on the small ones: a code may be off by half of
    f16's smallest step, 2^-25 of the largest scale, and not by the code itself."""
    c = make([200], [64], 16, 4, 2, 64, torch.float16, seed=73, pow2=True)
    Q = c["Q"].abs()
    ids = c["table"][0][:13]
    k, v = (x.clone().float() for x in c["code"])
    ks, vs = (torch.full_like(x, math.nan) for x in c["scale"])
    factor = 2.0 ** -below
    if side == "V":                                       # ordinary keys, but for the big page's, which point away from Q
        ks[ids], vs[ids] = 2.0 ** -6, factor
        k[ids[big]], vs[ids[big]] = -448.0, 1.0
        v[ids] = (v[ids] * 3).clamp(-448, 448)
        scale = 0.1
    else:                                                 # a key is +-c in all dims; scores of small pages are of size 5
        ks[ids], vs[ids] = factor, 2.0 ** -6
        k[ids] = torch.where(k[ids][..., :1] < 0, -1.0, 1.0) * k[ids][..., :1].abs().clamp(40, 200)
        k[ids[big]], ks[ids[big]] = -448.0, 1.0
        scale = 5 / (200 * factor * 51)
    end = 200 - 12 * 16
    code = []
    for x in (k, v):
        x = x.to(torch.float8_e4m3fn)
        x.view(torch.uint8)[ids[12], :, end:] = 0x7F
        code.append(x)
    c.update(Q=Q, code=code, scale=[ks, vs])
    c["args"] = (Q.cuda(), code[0].cuda(), code[1].cuda(), ks.cuda(), vs.cuda(), *c["args"][5:])
    for max_new in (MANY, 1):
        got = ops().fmha_cached(*c["args"], c["cu_dev"], softmax_scale=scale, causal=causal, max_new=max_new)
        sync_ok()
        check(c, got, scale, causal, many=max_new == MANY)


def test_a_wait_that_runs_out_in_some_lanes_ends_in_all():
    """What the warps of the attention kernels do together behind a wait needs one answer in all of their lanes."""
    from kernelcodegen_b200 import _lib
    lib = _lib.load()
    answers = torch.full((1,), -1, dtype=torch.int32, device="cuda")
    assert lib.kcg_selftest_warp_wait(1_000_000, answers.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
    sync_ok()
    assert answers.item() == 0
    assert lib.kcg_selftest_warp_wait(0, answers.data_ptr(), None) == _lib.ERR_INVALID_ARG
    assert lib.kcg_selftest_warp_wait(1, None, None) == _lib.ERR_INVALID_ARG


@pytest.mark.parametrize("B", [1, 160])                  # ranges of key blocks, whole items
@pytest.mark.parametrize("rows", [2, 60])
def test_rows_of_q_and_o_in_reverse_order(rows, B):
    c = make([300] * B, [rows] * B, 16, 4, 2, 64, torch.float16, seed=74)
    got = attend_c(c, 0.1, 1, rows, q=c["args"][0].flip(0), turned=True)
    check(c, got.flip(0), 0.1, True, many=rows * 2 > 48)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("rows", [1, 130])
def test_as_many_requests_as_there_may_be(rows, causal):
    """The kernels walk past a million requests without queries, from one with work to the next."""
    B = 2 ** 20
    c = make([300, 77], [rows, 1], 16, 4, 2, 64, torch.float16, seed=75)
    at = (5, B - 1)                                       # the two that have work
    lengths = torch.full((B,), 3, dtype=torch.int32)
    cu = torch.zeros(B + 1, dtype=torch.int32)
    cu[at[0] + 1:] = rows
    cu[B] = rows + 1
    table = torch.full((B, c["args"][5].shape[1]), -1, dtype=torch.int32, device="cuda")
    for i, b in enumerate(at):
        lengths[b] = c["lengths"][i]
        table[b] = c["args"][5][i]
    got = ops().fmha_cached(*c["args"][:5], table, lengths.cuda(), cu.cuda(), softmax_scale=0.1, causal=causal, max_new=rows)
    sync_ok()
    check(c, got, 0.1, causal, many=rows * 2 > 48)


@pytest.mark.parametrize("max_new", [1, 4, MANY])        # 8, 16 rows a tile; 256
@pytest.mark.parametrize("where", ["key", "key scale", "value", "value scale"])
@pytest.mark.parametrize("lengths,new,page,Hq,Hkv,D,dtype", [
    ([200, 90], [60, 1], 16, 4, 2, 128, torch.bfloat16),
    ([300, 40], [300, 40], 32, 2, 1, 64, torch.float16),                # whole prompts, rows of both tiles
    ([700, 90] * 3, [400, 90] * 3, 48, 6, 1, 128, torch.float16),       # ranges that end inside an item
    ([330] * 90, [70] * 90, 16, 4, 2, 64, torch.bfloat16),              # whole items
])
def test_what_nan_reaches(lengths, new, page, Hq, Hkv, D, dtype, where, max_new):
    """A NaN key reaches the rows that see it and no others; a NaN value no other dim, head or request than its own."""
    c = make(lengths, new, page, Hq, Hkv, D, dtype, seed=76)
    want = ops().fmha_cached(*c["args"], c["cu_dev"], softmax_scale=0.1, causal=True, max_new=max_new)
    at = lengths[0] - new[0] // 2                        # a key that half of request 0's rows see
    p, r = c["table"][0][at // page], at % page
    k, v, ks, vs = (x.clone() for x in c["args"][1:5])
    dims = slice(None)
    if "scale" in where:
        (ks if where == "key scale" else vs)[p, 0] = math.nan
        at -= r
    elif where == "key":
        k.view(torch.uint8)[p, 0, r, 3] = 0xFF
    else:
        v.view(torch.uint8)[p, 0, r, [5, D - 1]] = 0x7F
        dims = [5, D - 1]
    got = ops().fmha_cached(c["args"][0], k, v, ks, vs, *c["args"][5:], c["cu_dev"], softmax_scale=0.1, causal=True, max_new=max_new)
    sync_ok()
    first = at - (lengths[0] - new[0])                   # the first row that sees it
    assert 0 < first < new[0]
    hit, clean = (torch.zeros(want.shape, dtype=torch.bool, device="cuda") for _ in range(2))
    hit[first:new[0], :Hq // Hkv, dims] = True
    clean[:] = True                                      # (rows before a NaN value's key may be NaN in its dims, as in a plain product)
    clean[0 if "value" in where else first:new[0], :Hq // Hkv, dims] = False
    assert bool(got[hit].isnan().all()) and bool(got[clean].isfinite().all())
    if "scale" in where:                                 # (other pages' codes may be relative to another scale)
        check(c, torch.where(clean, got, want), 0.1, True, many=True)
    else:
        assert torch.equal(got[clean], want[clean])


def test_rejected_drafts_give_their_pages_back():
    """Plans and returns in turn, nothing read on the host in between."""
    B, page, pages, width = 5, 16, 400, 110
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    table, free_pages, left, cached = torch.full((B, width), -1, dtype=torch.int32, device="cuda"), i32(list(range(pages)) + [-1]), i32([pages]), i32([0] * B)
    for new, kept in draft_steps(4):
        want = (cached + i32(new)).tolist()
        lengths, _, _, left = ops().cache_plan(cached, i32(new), table, free_pages, left, page, sum(new))
        assert lengths.tolist() == want
        cached = i32(kept)
        give_back(cached, lengths, table, free_pages, left, page)
        check_pages(kept, table.tolist(), free_pages.tolist(), left.item(), page, pages)
    sync_ok()


@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("max_new", [0, 1, 7, 12, 13, 10 ** 6])
def test_every_max_new_within_the_bound_of_its_kernel(max_new, pow2):
    """More rows than the kernel was chosen for, or fewer: each is held to its own arithmetic."""
    c = make([300, 90, 40], [60, 1, 40], 16, 8, 2, 128, torch.bfloat16, seed=77, pow2=pow2)
    got = ops().fmha_cached(*c["args"], c["cu_dev"], softmax_scale=0.1, causal=True, max_new=max_new)
    sync_ok()
    check(c, got, 0.1, True, many=(max_new or -(-101 // 3)) * 4 > 48)


@pytest.mark.parametrize("max_new", [0, 1, 512])
def test_one_call_with_a_chunk_and_single_tokens(max_new):
    """A step of a server: 40 requests with one token each, and two prompts in chunks, in one call."""
    new = [1] * 20 + [512] + [1] * 20 + [77]
    lengths = [37 * i + 1 for i in range(20)] + [1500] + [61 * i + 5 for i in range(20)] + [77]
    c = make(lengths, new, 16, 8, 2, 128, torch.bfloat16, seed=78, pow2=True)
    got = ops().fmha_cached(*c["args"], c["cu_dev"], softmax_scale=128 ** -0.5, causal=True, max_new=max_new)
    sync_ok()
    check(c, got, 128 ** -0.5, True, many=(max_new or -(-sum(new) // 42)) * 4 > 48)


@pytest.mark.parametrize("max_new", [1, MANY])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("softmax_scale", [2.0 ** 12, 2.0 ** 18, 2.0 ** 21, 2.0 ** 23, -2.0 ** 24, 2.0 ** 26, 2.0 ** 34])
def test_scores_of_any_size(softmax_scale, dtype, causal, max_new):
    """Scores of 2^15 to 2^40.  Queries and keys are whole numbers, so that scores are exact and the largest wins by 2^12 at least:
    a row's result is the value of the key with the largest score."""
    c = make([700, 300], [60, 60], 16, 4, 2, 64, dtype, seed=79, pow2=True)
    ids = [p for i in range(2) for p in c["table"][i] if p >= 0]
    g = torch.Generator().manual_seed(80)
    k = torch.randint(-8, 9, c["code"][0].shape, generator=g).float()
    nan = torch.isnan(c["code"][0].float())
    c["code"][0] = torch.where(nan, math.nan, k).to(torch.float8_e4m3fn)
    c["scale"][0][ids] = 1.0
    c["Q"] = torch.randint(-8, 9, c["Q"].shape, generator=g).to(dtype)
    got = ops().fmha_cached(c["Q"].cuda(), c["code"][0].cuda(), c["args"][2], c["scale"][0].cuda(), *c["args"][4:], c["cu_dev"],
                            softmax_scale=softmax_scale, causal=causal, max_new=max_new)
    sync_ok()
    want, _ = R.attend(c["Q"], c["code"][0].double(), c["scale"][0].double(), c["code"][1].double(), c["scale"][1].double(), c["table"],
                       c["lengths"], c["cu"], c["page"], softmax_scale, causal)
    # weights are 0, or equal among keys of equal score; a value is an e4m3 code times a power of two, their mean is rounded to
    # P's and O's types: (2^-11 + eps / 2) of the largest value, and fp32 sums
    size = max(float((c["code"][1].double().nan_to_num().amax() * c["scale"][1][p].max())) for p in ids)
    assert bool(((got.cpu().double() - want).abs() <= (2.0 ** -11 + torch.finfo(dtype).eps) * size).all())
