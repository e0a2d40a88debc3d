"""The built library's metadata of the paged attention kernels: their accumulators, and the
rows on their way, have to stay in registers."""
import pytest

from tests.test_abi import _kernel_metadata


@pytest.mark.parametrize("kernel,forms", [("paged_decode_kernel", 16), ("paged_prefill_kernel", 32)])
def test_attention_keeps_its_sums_in_registers(kernel, forms):
    """bf16 or fp16, head_dim 64 or 128, 16- or 4-bit cache, pages of whole 16 keys or not,
    and 64 or 128 rows in the prefill form."""
    found = {n: k for n, k in _kernel_metadata().items() if kernel in n}
    assert len(found) == forms
    spills = {n: k[".private_segment_fixed_size"] for n, k in found.items() if k[".private_segment_fixed_size"]}
    assert not spills


@pytest.mark.parametrize("kernel", ["paged_plan_kernel", "paged_merge_kernel", "paged_batch_kernel",
                                    "qk_norm_rope_kernel", "kv_fp4_append_kernel", "kv_fp4_gather_kernel"])
def test_the_others_use_no_scratch_memory(kernel):
    found = {n: k[".private_segment_fixed_size"] for n, k in _kernel_metadata().items() if kernel in n}
    assert found and not any(found.values()), {n: v for n, v in found.items() if v}
