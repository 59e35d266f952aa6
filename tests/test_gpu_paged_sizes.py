"""Sizes past 32 bits are refused with the framework's own error, which names
them (empty tensors: nothing of that size is allocated)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_sizes_past_32_bits(rb):
    pages = torch.empty(2**31, 0, 16, 128, dtype=torch.bfloat16, device="cuda")
    q = torch.zeros(1, 8 * 128, dtype=torch.bfloat16, device="cuda")
    pos, table = (torch.zeros(*x, dtype=torch.int32, device="cuda") for x in ((1,), (1, 2)))
    with pytest.raises(rb.ConfigError, match="sizes"):
        rb.rope_paged_append(q, pos, table, pages, pages, torch.ones(64, device="cuda"))
    with pytest.raises(rb.ConfigError, match="sizes"):
        rb.paged_attention(q, pos, table, pages, pages)
    none = torch.zeros(0, device="cuda")
    with pytest.raises(rb.ConfigError, match="sizes"):
        rb.verify_draft(torch.empty(0, 1, 2**31, device="cuda"), None, None, none, none)
