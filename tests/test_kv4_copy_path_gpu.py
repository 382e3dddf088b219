"""Attention over a 4-bit cache where it runs on bf16 copies of the pages: queries of more than 128 rows, page scores, pages that many tokens
share.  What holds for the kernels that read 4 bits holds here too."""
import pytest
import torch

import serving_ref as ref
from test_kv4_attention_gpu import DEV, P_BF16, Batch

pytestmark = pytest.mark.gpu


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _empty_batch():
    """A call without a token, and one whose sequences have no key: neither has a page to read."""
    import msa_for_sail as msa
    k, v = (torch.zeros(3, 2, 128, 72, dtype=torch.uint8, device=DEV) for _ in range(2))
    return msa, k, v, torch.empty(0, dtype=torch.int32, device=DEV)


def test_a_table_shorter_than_a_host_made_plan():
    import msa_for_sail as msa
    b = Batch(101, [200, 1], [300, 200], 16, 2)
    q, k, v, table = b.cuda()
    for n in (4, 0):
        with pytest.raises(ValueError, match="kv_indices must have the 5 pages"):
            msa.fmha_sail(q, k, v, b.plan(), kv_indices=table[:n].clone())
    out, _ = msa.fmha_sail(q, k, v, b.plan(), kv_indices=table)
    ref.check_attention(out, None, b.want(), P_BF16, "the whole table")


def test_a_call_without_tokens():
    msa, k, v, none = _empty_batch()
    plan = msa.fmha_sail_plan(torch.tensor([0, 0]), torch.tensor([300, 200]), 16, num_kv_heads=2, page_size=128, use_kv4_cache=True)
    out, _ = msa.fmha_sail(torch.empty(0, 16, 128, dtype=torch.bfloat16, device=DEV), k, v, plan, kv_indices=none)
    assert out.shape == (0, 16, 128)


def test_offsets_of_any_type_and_stride():
    """An override may be int64, or every second entry of a tensor: it is what it says, entry by entry."""
    import msa_for_sail as msa
    b = Batch(102, [140, 3], [300, 200], 8, 2, offsets=[100, 150])
    q, k, v, table = b.cuda()
    plan = msa.fmha_sail_plan(torch.tensor(b.qo), torch.tensor(b.kv), 8, num_kv_heads=2, page_size=128, use_kv4_cache=True)
    wide = torch.tensor([100, -7, 150, -7], device=DEV)
    for off in (wide[::2], wide[::2].to(torch.int32), wide.to(torch.int32)[::2]):
        out, _ = msa.fmha_sail(q, k, v, plan, kv_indices=table, q_offset_override=off)
        ref.check_attention(out, None, b.want(), P_BF16, "offsets")
    with pytest.raises(ValueError, match="q_offset_override must be"):
        msa.fmha_sail(q, k, v, plan, kv_indices=table, q_offset_override=wide[:1])
