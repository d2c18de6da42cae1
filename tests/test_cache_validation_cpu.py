"""Refusals of the paged-cache entry points, without a GPU: operands that a kernel would read or write out of bounds with
stop in the Python wrappers, arguments that make no sense in the C ABI, and the host restatement that the GPU tests
compare with counts and rounds as it says."""
import ctypes
import random

import pytest
import torch

from kernelcodegen_b200 import _lib, ops
from tests import cache_reference as R


def cache(pages=4, Hkv=2, page=16, D=64):
    k = torch.zeros((pages, Hkv, page, D), dtype=torch.float8_e4m3fn)
    return k, k.clone(), torch.ones(pages, Hkv), torch.ones(pages, Hkv)


def i32(*v):
    return torch.tensor(v, dtype=torch.int32)


def test_attention_operands():
    k, v, ks, vs = cache()
    Q = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    table, lengths, cu = torch.zeros(2, 2, dtype=torch.int32), i32(5, 6), i32(0, 1, 3)
    good = [Q, k, v, ks, vs, table, lengths, cu]

    def bad(at, value, match):
        args = list(good)
        args[at] = value
        with pytest.raises(ValueError, match=match):
            ops.fmha_cached(*args)
    bad(0, torch.zeros(3, 4, 128, dtype=torch.bfloat16), "Q must be")
    bad(0, torch.zeros(3, 4, 64, 2, dtype=torch.bfloat16)[..., 0], "Q must be")
    bad(0, torch.zeros(3, 5, 64, dtype=torch.bfloat16), "do not divide")
    bad(1, k.to(torch.float16), "k_cache")
    bad(2, v[:3], "v_cache")
    bad(3, ks.double(), "k_scale")
    bad(4, torch.ones(2, 4).t(), "v_scale")
    bad(5, table.long(), "block_table")
    bad(5, table[:1], "block_table")
    bad(5, torch.zeros(2, 4, dtype=torch.int32)[:, ::2], "block_table")
    bad(6, lengths.long(), "lengths")
    bad(7, i32(0, 3), "cu_new")
    bad(7, None, "must divide")
    with pytest.raises(ValueError, match="CUDA"):
        ops.fmha_cached(*good)


def test_append_operands():
    k, v, ks, vs = cache()
    K = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    slots = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="K must be"):
        ops.cache_append(K[:, :1], K, slots, k, v, ks, vs)
    with pytest.raises(ValueError, match="V must be"):
        ops.cache_append(K, K[:2], slots, k, v, ks, vs)
    with pytest.raises(TypeError):
        ops.cache_append(K, K.float(), slots, k, v, ks, vs)
    with pytest.raises(ValueError, match="slot_map"):
        ops.cache_append(K, K, slots.int(), k, v, ks, vs)
    with pytest.raises(ValueError, match="expanded"):
        ops.cache_append(K, K, slots, k[:1].expand(4, 2, 16, 64), v, ks, vs)
    with pytest.raises(ValueError, match="CUDA"):
        ops.cache_append(K, K, slots, k, v, ks, vs)


def test_plan_operands():
    table = torch.zeros(2, 2, dtype=torch.int32)
    good = [i32(1, 2), i32(1, 1), table, i32(3, 4), i32(2), 16, 2]

    def bad(at, value, match):
        args = list(good)
        args[at] = value
        with pytest.raises(ValueError, match=match):
            ops.cache_plan(*args)
    bad(0, torch.tensor([1, 2]), "cached")
    bad(1, i32(1), "new")
    bad(2, table[:1], "block_table")
    bad(3, torch.tensor([1.0]), "free_pages")
    bad(4, i32(1, 2), "free_count")
    bad(5, 0, "page_size")
    bad(6, -1, "max_tokens")
    bad(0, i32(1, 2), "CUDA")


def test_c_abi_refusals(lib):
    st2, st3 = (ctypes.c_int64 * 2)(64, 64), (ctypes.c_int64 * 3)(4096, 1024, 64)

    def attend(dtype=_lib.BF16, T=1, B=1, Hq=2, Hkv=1, D=64, max_new=1, Q=16, pages=4, page=16, width=2, stride=2, cu=None,
               q=st2, kc=st3, work=16, nbytes=1 << 30):
        return lib.kcg_fmha_cached_fwd(dtype, T, B, Hq, Hkv, D, max_new, 1.0, 1, Q, q, 16, kc, 16, 16, kc, 16, pages, page, 16,
                                       width, stride, 16, cu, 16, q, work, nbytes, None)
    assert attend(T=-1) == _lib.ERR_INVALID_ARG
    assert attend(page=8) == attend(page=24) == attend(page=0) == _lib.ERR_INVALID_ARG
    assert attend(dtype=_lib.F32) == attend(D=96) == _lib.ERR_UNSUPPORTED
    assert attend(Hq=3, Hkv=2) == attend(Hkv=0) == _lib.ERR_INVALID_ARG
    assert attend(Q=None) == _lib.ERR_INVALID_ARG
    assert attend(T=3, B=2) == _lib.ERR_INVALID_ARG                       # no cu_new and no whole share
    assert attend(stride=1) == attend(pages=0) == _lib.ERR_INVALID_ARG
    assert attend(width=1 << 28, stride=1 << 28) == _lib.ERR_UNSUPPORTED
    assert attend(q=(ctypes.c_int64 * 2)(60, 64)) == attend(Q=8) == _lib.ERR_ALIGNMENT
    assert attend(kc=(ctypes.c_int64 * 3)(4096, 1024, 0)) == _lib.ERR_UNSUPPORTED
    assert attend(work=None) == attend(nbytes=10) == _lib.ERR_INVALID_ARG
    assert attend(T=0) == attend(B=0) == _lib.OK                          # nothing to do
    size = ctypes.c_size_t()
    assert lib.kcg_fmha_cached_workspace(96, ctypes.byref(size)) == _lib.ERR_UNSUPPORTED
    assert lib.kcg_fmha_cached_workspace(64, None) == _lib.ERR_INVALID_ARG

    def append(dtype=_lib.BF16, T=1, H=1, D=64, K=16, pages=4, page=16, k=st2, kc=st3):
        return lib.kcg_cache_append(dtype, T, H, D, K, k, 16, k, 16, pages, page, 16, kc, 16, kc, 16, 16, None)
    assert append(T=-1) == append(page=20) == append(K=None) == _lib.ERR_INVALID_ARG
    assert append(D=32) == append(dtype=_lib.I32) == _lib.ERR_UNSUPPORTED
    assert append(K=8) == append(kc=(ctypes.c_int64 * 3)(4096, 1024, 72)) == _lib.ERR_ALIGNMENT
    assert append(T=0) == _lib.OK

    def plan(B=1, page=16, tokens=1, cached=16, width=1, stride=1, count=16):
        return lib.kcg_cache_plan(B, page, tokens, cached, 16, 16, width, stride, 16, 1, count, 16, 16, 16, 16, None)
    assert plan(B=-1) == plan(page=0) == plan(stride=0) == plan(cached=None) == plan(count=None) == _lib.ERR_INVALID_ARG
    assert plan(B=16385) == _lib.ERR_UNSUPPORTED


def test_reference_rounding_is_that_of_the_storage_type():
    x = torch.cat([torch.linspace(-448, 448, 4001), torch.linspace(-0.05, 0.05, 4001)]).double()
    assert torch.equal(R.round_e4m3(x), x.float().to(torch.float8_e4m3fn).double())


def test_reference_plan_by_hand():
    table = [[7, -1, -1], [-1, -1, -1]]
    got = R.plan([15, 0], [2, 17], table, [1, 2, 3, 4], 4, 16, 20)
    assert got == ([17, 17], [0, 2, 19], [7 * 16 + 15, 4 * 16] + [3 * 16 + i for i in range(16)] + [2 * 16, -1], 1)
    assert table == [[7, 4, -1], [3, 2, -1]]


def test_pair_units_formula():
    """The many-row kernel counts the key blocks of a causal request's row pairs by a closed form; here it is against the sum."""
    def floor_sum(n, m, a, b):
        s = 0
        while n > 0:
            s += (n - 1) * n // 2 * (a // m) + n * (b // m)
            a, b = a % m, b % m
            top = a * n + b
            if top < m:
                break
            n, b, m, a = top // m, top % m, a, m
        return s

    def blocks(first, n, L, G):
        last = min(first + 128, n * G) - 1
        end = min(L, L - n + 1 + last // G) if last >= first else 0
        return -(-end // 128) if end > 0 else 0
    r = random.Random(1)
    for _ in range(500):
        G, n = r.randint(1, 20), r.randint(1, 2000)
        L = n + r.choice([0, r.randint(0, 5000)])
        pairs = -(-n * G // 256)
        k = r.randint(1, pairs)
        want = sum(max(blocks(256 * i, n, L, G), blocks(256 * i + 128, n, L, G)) for i in range(k))
        full = min(k, pairs - 1)
        got = floor_sum(full, 128 * G, 256, 255 + G * (L - n + 128))
        if k > full:
            got += max(blocks(256 * full, n, L, G), blocks(256 * full + 128, n, L, G))
        assert got == want
