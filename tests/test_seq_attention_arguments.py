"""CPU tests of arguments that the packed attention's and the paged cache's argument structures cannot hold."""

import pytest
import torch

from tttj_2026_amd import _lib, ops


@pytest.fixture
def host(monkeypatch):
    """Host tensors pass for the device's, up to the library call, which fails the test."""
    def call(*args):
        raise AssertionError("reached the library")

    monkeypatch.setattr(ops, "_typed", lambda t, name: (t.dtype, t.get_device()))
    monkeypatch.setattr(ops, "_call", call)


def test_scale_beyond_a_float(host):
    """(A float beyond fp32 becomes an infinity there, which the library refuses.)"""
    scale = 10 ** 400
    q, k = torch.zeros(4, 8, 64, dtype=torch.float16), torch.zeros(4, 2, 64, dtype=torch.float16)
    starts, cache = torch.tensor([0, 4], dtype=torch.int32), torch.zeros(9, 16, 2, 64, dtype=torch.float16)
    table = torch.zeros(1, 8, dtype=torch.int32)
    with pytest.raises(ValueError, match="packed_attention"):
        ops.packed_attention(q, k, k, starts, scale=scale)
    with pytest.raises(ValueError, match="cache_attention"):
        ops.cache_attention(q, cache, cache, table, starts[1:], starts, scale=scale)


def test_more_tokens_and_pages_than_an_int32(host):
    starts, table = torch.tensor([0, 4], dtype=torch.int32), torch.zeros(1, 8, dtype=torch.int32)
    one = torch.zeros(1, 1, 8, dtype=torch.float16)
    cache = torch.zeros(9, 16, 1, 8, dtype=torch.float16)
    many = one.expand(1 << 31, 1, 8)
    with pytest.raises(ValueError, match="cache_append"):
        ops.cache_append(many, many, cache, cache, table, starts[1:], starts)
    pages = cache[:1].expand(1 << 31, 16, 1, 8)
    with pytest.raises(ValueError, match="cache_append"):
        ops.cache_append(one, one, pages, pages, table, starts[:1], torch.tensor([0, 1], dtype=torch.int32))
    with pytest.raises(ValueError, match="cache_attention"):
        ops.cache_attention(one, pages, pages, table, starts[:1])


@pytest.mark.parametrize("hd,waves", [(64, 2), (128, 2), (136, 1), (256, 1)])
def test_keys_are_dealt_out_after_16_rounds_of_a_block(hd, waves):
    """More blocks of 32 rows than CUs: a block of `waves` waves takes 16 rounds of 32 keys each alone."""
    size = _lib.cache_attention_workspace_bytes
    rows, longest = 300, 16 * 32 * waves
    assert size(rows, rows, 8, 2, hd, 16, 128, longest, True) == 0
    assert size(rows, rows, 8, 2, hd, 16, 128, longest + 1, True) > 0
