"""What the attention kernels over trees and Q8_0 pools take (no GPU needed)."""
import pytest

pytest.importorskip("msgpack")

from tests.test_kernel_resources import kernels


@pytest.mark.parametrize("name", ["paged_attn_q8_kernel", "paged_attn_q8_shared_kernel", "paged_attn_shared_kernel",
                                  "paged_attn_kernel", "kv_store_q8_kernel", "kv_gather_q8_kernel", "kv_move_kernel",
                                  "lp_slice_kernel", "lp_row_kernel", "merge_kernel"])
def test_draft_kernels_use_next_to_no_scratch(name):
    """A register kept in scratch memory is waited for with the cache's loads in
    flight behind it, once per block. Two kernels hold some, and no more than they
    did when they were timed: workgroups of four waves over Q8_0 heads of 256, and
    trees over f16 heads of 128 (one item a wave)."""
    got = {n: k for n, k in kernels().items() if name + "I" in n or name + "E" in n}
    assert got
    for n, k in got.items():
        most = {"27paged_attn_q8_shared_kernelILi256ELi4E": 52, "17paged_attn_kernelILi128ELb0ELb1E": 56}
        room = max([v for m, v in most.items() if m in n], default=0)
        assert k[".private_segment_fixed_size"] <= room, (n, k[".private_segment_fixed_size"])
