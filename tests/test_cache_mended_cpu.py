"""Refusals and rules of the paged-cache entry points that came after their first tests, without a GPU."""
import ctypes
import inspect
import random

import torch

from kernelcodegen_b200 import _lib, ops
from tests import cache_reference as R


def test_more_requests_than_a_limited_wait_can_walk_past(lib):
    st2, st3 = (ctypes.c_int64 * 2)(64, 64), (ctypes.c_int64 * 3)(4096, 1024, 64)
    for T, cu in ((1, 16), (2 ** 20 + 1, None)):
        rc = lib.kcg_fmha_cached_fwd(_lib.BF16, T, 2 ** 20 + 1, 2, 1, 64, 1, 1.0, 1, 16, st2, 16, st3, 16, 16, st3, 16, 4, 16, 16, 2, 2, 16, cu,
                                     16, st2, 16, 1 << 30, None)
        assert rc == _lib.ERR_UNSUPPORTED and "requests" in lib.kcg_last_error().decode()


def give_back(kept, lengths, block_table, free_pages, free_left, page_size):
    """The lines that cache_plan's docstring gives for returning pages."""
    col = torch.arange(block_table.shape[1], device=kept.device)
    gone = ((col >= (kept[:, None] + page_size - 1) // page_size) &
            (col < (lengths[:, None] + page_size - 1) // page_size)).flatten()
    at = torch.where(gone, gone.cumsum(0) - 1 + free_left, free_pages.shape[0] - 1)
    free_pages.scatter_(0, at, block_table.flatten())
    free_left += gone.sum()


def check_pages(lengths, table, free_pages, free_left, page, pages):
    """Every page is held by one request or stands in the list."""
    held = [p for n, row in zip(lengths, table) for p in row[:-(-n // page)]]
    assert sorted(held + free_pages[:free_left]) == list(range(pages))


def draft_steps(seed, B=5, page=16, steps=40):
    """(new, kept) of each step: up to 40 tokens are added, some of the last ones rejected, and now and then a request ends."""
    r = random.Random(seed)
    cached, out = [0] * B, []
    for _ in range(steps):
        new = [r.randint(0, 40) for _ in range(B)]
        kept = [0 if r.random() < 0.1 else c + r.randint(0, n) for c, n in zip(cached, new)]
        cached = kept
        out.append((new, kept))
    return out


def test_rejected_drafts_give_their_pages_back():
    B, page, pages, width = 5, 16, 400, 110
    table, free_pages, left, cached = [[-1] * width for _ in range(B)], list(range(pages)) + [-1], pages, [0] * B
    for new, kept in draft_steps(3):
        lengths, _, _, left = R.plan(cached, new, table, free_pages, left, page, sum(new))
        assert lengths == [c + n for c, n in zip(cached, new)]
        check_pages(lengths, table, free_pages, left, page, pages)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
        f, n = i32(free_pages), i32([left])
        give_back(i32(kept), i32(lengths), i32(table), f, n, page)
        free_pages, left, cached = f.tolist(), n.item(), kept
        check_pages(cached, table, free_pages, left, page, pages)


def test_the_documented_lines_are_the_tested_ones():
    body = [line.strip() for line in inspect.getsource(give_back).splitlines()[2:]]
    assert body == [line.strip() for line in ops.cache_plan.__doc__.splitlines() if line.startswith(" " * 8)]
