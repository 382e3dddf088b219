"""Child process of test_window_serving_gpu.py: windowed attention and the operators on pages with MSA_BOUNDS_CHECK=1.

1. Valid inputs on every kernel that takes windows: no status, results within the tolerance.
2. A page number behind the pages that the library is told of (a view of the first pages of a larger pool): clamped, STATUS_BOUNDS.  Nothing can
   leave the buffers even if the check were wrong.
3. Page numbers of copies that are no pages: skipped and reported."""
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "msa-for-sail_b200", "python"))
sys.path.insert(0, os.path.join(ROOT, "tests"))

import msa_for_sail as msa                      # noqa: E402
from msa_for_sail import _lib, api              # noqa: E402
from test_window_gpu import BF, DEV, E4, Case, _i32   # noqa: E402

assert _lib.BOUNDS_CHECK and _lib.LIB_PATH.endswith("libmsa_b200_check.so")
SHAPES = [(8, 2, 1, BF, BF), (8, 1, 2, BF, E4), (32, 1, 1, BF, BF), (16, 1, 3, E4, E4), (40, 1, 2, BF, BF), (8, 2, 300, BF, BF), (8, 2, 300, E4, E4), (8, 2, 40, BF, E4)]


def part_valid():
    for hq, hk, n, qt, ct in SHAPES:
        for layout, page in (("hnd", 128), ("nhd", 32), ("ragged", 0)):
            for splits in (1, 3):
                Case([n, n], [1000, n + 200], hq, hk, 250, 5, layout, page, qt, ct).check(num_kv_splits=splits)
    print("valid windows: ok, status 0")


def part_bad_page():
    n, extra = 6, 4
    for hq, hk, rows, qt, ct in SHAPES:
        pool_k, pool_v = (torch.randn(n + extra, hk, 128, 128, device=DEV).to(ct) for _ in range(2))
        q = torch.randn(rows, hq, 128, device=DEV).to(qt)
        table = torch.arange(n, dtype=torch.int32)
        table[4] = n + 1
        plan = msa.fmha_sail_plan(_i32([rows], "cpu"), _i32([n * 128], "cpu"), hq, num_kv_heads=hk, page_size=128, window_size=200, num_sink_tokens=5, num_kv_splits=1)
        out, _ = msa.fmha_sail(q, pool_k[:n], pool_v[:n], plan, kv_indices=table.to(DEV))
        torch.cuda.synchronize()
        assert torch.isfinite(out.float()).all()
        st = api.last_status()
        assert st == _lib.STATUS_BOUNDS, f"expected STATUS_BOUNDS, got {st} ({hq}, {hk}, {rows}, {qt}, {ct})"
        table[4], table[2] = 4, n + 1                       # a page that no row sees is not looked up
        if rows == 1:
            msa.fmha_sail(q, pool_k[:n], pool_v[:n], plan, kv_indices=table.to(DEV))
            torch.cuda.synchronize()
            assert api.last_status() == 0
    print("a page number that is none: clamped and reported")


def part_pages():
    pool = torch.randn(10, 2, 16, 128, device=DEV).to(BF)
    was = pool.clone()
    msa.kv_pages_copy(pool[:6], _i32([0, 7, -1, 2]), _i32([1, 3, 4, 8]))
    torch.cuda.synchronize()
    was[1] = was[0]
    assert torch.equal(pool, was)
    assert api.last_status() == _lib.STATUS_BOUNDS
    print("copies of pages that are none: skipped and reported")


if __name__ == "__main__":
    part_valid()
    part_bad_page()
    part_pages()
    print("CHECKED_WINDOW_OK")
