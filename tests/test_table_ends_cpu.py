"""Where kernels read the page table: a rule of the sources, since a table that ends too early must not be found out by reading behind it."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "msa-for-sail_b200", "csrc")


def code(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*|/\*.*?\*/", "", f.read(), flags=re.S)


@pytest.mark.parametrize("name", sorted(n for n in os.listdir(CSRC) if n.startswith(("fmha_", "score_"))))
def test_every_read_of_the_page_table_is_bounded(name):
    """Lengths on the device may outgrow the table: a read is page_entry(), or one with a bound beside it (4-bit kernels)."""
    for line in code(name).splitlines():
        if "p.kv_indices[" in line:
            assert "kv4" in name and ("p.num_logical_pages - 1)" in line or "p.kv_indices[at]" in line), line
    if "kv4" in name:
        assert "p.num_logical_pages - 1)" in code(name)


def test_a_read_past_the_end_is_the_last_entry():
    text = code("common.cuh").split("page_entry(const MsaFmhaParams& p, int at) {")[1].split("\n}")[0]
    assert "min(static_cast<unsigned>(at), static_cast<unsigned>(p.num_page_entries) - 1u)" in text and "p.kv_indices[place]" in text


def test_the_length_travels_with_the_table():
    import inspect
    from msa_for_sail import _lib, api
    assert [n for n, _ in _lib.MsaFmhaParams._fields_][-1] == "num_page_entries"
    assert "p.num_page_entries = kv_indices.data_ptr(), kv_indices.numel()" in inspect.getsource(api._fmha_sail)


def test_rows_of_a_decode_tile_are_bounded():
    """A sequence of a device-made plan may have more tokens than the plan was made for: the tile holds as many rows as were announced."""
    assert "ntok = min(p.qo_start[b + 1] - p.qo_start[b], p.decode_rows >> (__ffs(G) - 1));" in code("fmha_decode_tc.cu")
