"""Child process of test_kv4_copy_path_gpu.py: the build with bounds checks on a prompt over a 4-bit cache, whose pages are copied.

"pages": a number that is no page is reported where it counts, not behind the last page of a table that is longer than its use.
"table": places past the end of a table that the lengths outgrew are reported, on the copies and on a bf16 cache."""
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (os.path.join(ROOT, "msa-for-sail_b200", "python"), ROOT, os.path.join(ROOT, "tests")):
    sys.path.insert(0, p)

import torch                                    # noqa: E402

import msa_for_sail as msa                      # noqa: E402
from msa_for_sail import _lib, api              # noqa: E402
from test_kv4_attention_gpu import DEV, Batch   # noqa: E402

assert _lib.BOUNDS_CHECK and _lib.LIB_PATH.endswith("libmsa_b200_check.so")


def status():
    torch.cuda.synchronize()
    return api.last_status()


b = Batch(104, [200], [600], 8, 2)
q, k, v, table = b.cuda()
if sys.argv[1] == "pages":
    plan = b.plan()
    assert msa.fmha_sail(q, k, v, plan, kv_indices=table)[0].isfinite().all() and status() == _lib.STATUS_OK
    msa.fmha_sail(q, k, v, plan, kv_indices=torch.cat([table, torch.tensor([-1, 10 ** 6], dtype=torch.int32, device=DEV)]))
    assert status() == _lib.STATUS_OK
    bad = table.clone()
    bad[2] = 10 ** 6
    msa.fmha_sail(q, k, v, plan, kv_indices=bad)
    assert status() == _lib.STATUS_BOUNDS
else:
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    ws = msa.allocate_graph_workspace(1, 8, num_kv_heads=2, page_size=128, max_qo_len=200)
    plan = msa.fmha_sail_plan(i32([200]), i32([600]), 8, num_kv_heads=2, page_size=128, num_kv_splits=1, graph_safe=True, max_total_q=200,
                              max_qo_len_override=200, qo_len_uniform_override=True, max_kv_len_override=600, qo_offset=i32([-1]), given_workspace=ws)
    bf16 = [torch.randn(k.shape[0], 2, 128, 128, device=DEV).to(torch.bfloat16) for _ in range(2)]
    for kv in ([k, v], bf16):
        assert msa.fmha_sail(q, *kv, plan, kv_indices=table)[0].isfinite().all() and status() == _lib.STATUS_OK
        msa.fmha_sail(q, *kv, plan, kv_indices=table[:3].clone())
        assert status() == _lib.STATUS_BOUNDS
print("CHECKED_KV4_OK")
