"""CPU test: an append into a cache in 8 bits whose pages, rows, heads or scales lie at one address (an expanded tensor) is
refused: the waves that write them would overwrite one another."""

import pytest
import torch

from test_cache8_host import E8M0, _refused
from tttj_2026_amd import _lib, ops


@pytest.mark.parametrize("field", ["kc_page", "vc_page", "kc_row", "vc_row", "kc_head", "vc_head", "s_page", "s_head"])
def test_one_address_is_refused(field):
    assert "one address" in _refused("tt_cache_rows8", **{field: 0})


def test_one_address_of_blocks_is_refused():
    assert "one address" in _refused("tt_cache_rows8", page_size=32, s_block=0)


def test_expanded_scales_are_refused(monkeypatch):
    """By the library, through ops.cache_append (host tensors: nothing is launched)."""
    monkeypatch.setattr(ops, "_typed", lambda t, name: (t.dtype, t.get_device()))
    monkeypatch.setattr(ops, "_call", lambda name, args, index: _lib.check(getattr(_lib.load(), name)(args, None), name))
    k = torch.zeros(4, 2, 64, dtype=torch.float16)
    table, starts = torch.zeros(1, 8, dtype=torch.int32), torch.tensor([0, 4], dtype=torch.int32)
    cache = [torch.zeros(9, 32, 2, 64).to(torch.float8_e4m3fn) for _ in range(2)]
    one = torch.zeros(9, 2, 1, dtype=torch.uint8).view(E8M0).expand(9, 2, 2)
    with pytest.raises(ValueError, match="one address"):
        ops.cache_append(k, k, *cache, table, starts[1:], starts, k_scales=one, v_scales=one)
