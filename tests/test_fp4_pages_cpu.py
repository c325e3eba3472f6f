"""Shapes of 4-bit pages whose sizes the C ABI cannot hold are refused ahead of it."""

import pytest
import torch

from velox_voice_b200 import ops


@pytest.mark.parametrize("units", [2 ** 27, 2 ** 28, 2 ** 28 + 1, 2 ** 31 + 1])
def test_pages_of_too_many_tokens_are_refused(monkeypatch, units):
    """page_size is 32 bits: pages of 2^32 + 16 tokens would be taken for pages of 16."""
    monkeypatch.setattr(ops, "_require_cuda", lambda t, name: None)
    pages = torch.empty((1, 1, units, 144), dtype=torch.uint8, device="meta")
    for call in (lambda: ops._fp4_tensor(pages, "pages"), lambda: ops._kv_cache(pages, pages)):
        with pytest.raises(ValueError, match="2\\^31"):
            call()
    ops._fp4_tensor(torch.empty((1, 1, 2 ** 27 - 1, 144), dtype=torch.uint8, device="meta"), "pages")
