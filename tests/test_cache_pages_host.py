"""CPU tests of the host side of forks, compaction and copies of a cache's pages."""

import ctypes

import pytest
import torch

from test_cache8_host import P, _fields
from tttj_2026_amd import _lib, ops

CALLS = {"tt_cache_fork_pages": (_lib.CACHE_FORK, "tt_cache_fork"),
         "tt_cache_compact_pages": (_lib.CACHE_COMPACT, "tt_cache_compact"),
         "tt_cache_copy_pages": (_lib.CACHE_COPY, "tt_cache_copy")}
STATE = dict(table=P, lengths=P, uses=P, new_table=P, new_uses=P, workspace=P, workspace_bytes=1 << 40, table_row=8,
             part_count=1, batch=2, columns=8, pages=9, page_size=16)
GOOD = {"tt_cache_fork_pages": dict(STATE, parents=P, counts=P, new_lengths=P), "tt_cache_compact_pages": STATE,
        "tt_cache_copy_pages": dict(source=P, target=P, part_count=1, count=3, pages=9)}
PART = dict(data=P, page=4096, row=256, rows=16)


def _struct(name):
    return type(name, (ctypes.Structure,), {"_fields_": _fields(name)})


@pytest.mark.parametrize("name,packer", [*((n, p) for n, (p, _) in CALLS.items()), ("tt_cache_part", _lib.CACHE_PART)])
def test_structures_are_the_header_s(name, packer):
    values = {n: i + 1 for i, (n, _) in enumerate(_fields(name))}
    assert bytes(_struct(name)(**values)) == packer.pack(*values.values())


def _call(name, part=PART, **change):
    parts = _struct("tt_cache_part")(**part)
    values = {"size": CALLS[name][0].size, "parts": ctypes.addressof(parts), **GOOD[name], **change}
    return getattr(_lib.load(), CALLS[name][1])(ctypes.byref(_struct(name)(**values)), None)


@pytest.mark.parametrize("name", CALLS)
def test_refusals(name):
    fields = [n for n, _ in _fields(name)]
    assert getattr(_lib.load(), CALLS[name][1])(None, None) == _lib.TT_ERR_INVALID
    for change in (dict(size=8), dict(batch=-1), dict(columns=0), dict(pages=0), dict(pages=-1), dict(page_size=8),
                   dict(page_size=48), dict(page_size=1 << 20, columns=1 << 11), dict(batch=1 << 27), dict(table_row=-1),
                   dict(part_count=-1), dict(parts=None), dict(count=-1), dict(workspace=P + 8), dict(workspace_bytes=64)):
        change = {k: v for k, v in change.items() if k in fields}
        if change:
            assert _call(name, **change) == _lib.TT_ERR_INVALID, change
    for field, kind in _fields(name):
        if kind is ctypes.c_void_p and field not in ("parents", "counts"):
            assert _call(name, **{field: None}) == _lib.TT_ERR_INVALID, field
    for change in (dict(data=None), dict(rows=0), dict(row=0), dict(row=-16), dict(page=4095), dict(page=-1),
                   dict(row=1 << 40), dict(row=1 << 62, page=1 << 62)):
        assert _call(name, part={**PART, **change}) == _lib.TT_ERR_INVALID, change


def test_workspace():
    size = _lib.cache_pages_workspace_bytes
    assert size(2, 8, 9) == 4 * (4 * 2 + 2 * 9 + 9 + 3 * 4 + 1)
    assert _call("tt_cache_copy_pages", count=0) == _lib.TT_OK
    for bad in ((-1, 8, 9), (2, 0, 9), (2, 8, 0), (1 << 27, 8, 9)):
        with pytest.raises(ValueError):
            size(*bad)


@pytest.fixture
def host(monkeypatch):
    """Host tensors pass for the device's, up to the library call, whose tensors are counted."""
    calls = []
    real = ops._parts

    class Device:
        def __init__(self, t):
            self.t = t

        def __getattr__(self, name):
            return True if name == "is_cuda" else getattr(self.t, name)

    monkeypatch.setattr(ops, "_parts", lambda caches, *how: real([Device(t) for t in caches], *how))
    monkeypatch.setattr(ops, "_call", lambda name, args, index: calls.append(name))
    return calls


def test_tensors(host):
    caches = list(torch.zeros(3, 9, 32, 2, 8).half())
    i32 = dict(dtype=torch.int32)
    table, n, uses = torch.zeros(4, 6, **i32), torch.zeros(4, **i32), torch.zeros(9, **i32)
    good = [caches, [caches[0], torch.zeros(9, 2, 2, dtype=torch.uint8).view(torch.float8_e8m0fnu)], [torch.zeros(9, 2, 32, 2, 8)[:, 0]],
            [torch.zeros(9, 2, 32, 8).transpose(1, 2)], [torch.zeros(9, 32, 1, 8)], [torch.zeros(9, 32, 2, 8)[::1]]]
    for c in good:
        ops.cache_fork(c, table, n, uses, n, n), ops.cache_compact(c, table, n, uses), ops.cache_copy(c, n, n)
    assert len(host) == 3 * len(good)
    halves = torch.zeros(9, 2, 32, 2, 8)
    for c in ([caches[0], halves], [caches[0], torch.zeros(9, 2, 2)], [caches[0], torch.zeros(9, 5, 2)]):
        with pytest.raises(ValueError):
            ops.cache_fork(c, table, n, uses)
        with pytest.raises(ValueError):
            ops.cache_compact(c, table, n, uses)
        ops.cache_copy(c, n, n)
    del host[-3:]
    for c in ([], [torch.zeros(9)], [caches[0], torch.zeros(8, 32, 2)],
              [torch.zeros(9, 32, 2, 8)[..., :4]], [torch.zeros(9, 32, 2, 8)[:, ::2]], [torch.zeros(9, 0, 2)],
              [torch.zeros(0, 32, 2)], [torch.zeros(1, 32, 2).expand(9, 32, 2)],
              [torch.zeros(9, 32, 1).expand(9, 32, 4)], [torch.zeros(9, 32, 2, 8).transpose(0, 1)]):
        with pytest.raises(ValueError):
            ops.cache_fork(c, table, n, uses)
        with pytest.raises(ValueError):
            ops.cache_compact(c, table, n, uses)
        with pytest.raises(ValueError):
            ops.cache_copy(c, n, n)
    for state in ((table.long(), n, uses), (table[:3], n, uses), (table[:, :0], n, uses), (table[0], n, uses),
                  (table, n.long(), uses), (table, n, uses[:8]), (table, table, uses), (table, n, uses.long())):
        with pytest.raises(ValueError):
            ops.cache_fork(caches, *state)
        with pytest.raises(ValueError):
            ops.cache_compact(caches, *state)
    for how in (dict(parents=n[:3]), dict(counts=n[:3]), dict(parents=n.long()), dict(counts=n.float())):
        with pytest.raises(ValueError):
            ops.cache_fork(caches, table, n, uses, **how)
    for pair in ((n, n[:3]), (n.long(), n), (n, n.long()), (table, table)):
        with pytest.raises(ValueError):
            ops.cache_copy(caches, *pair)
    assert len(host) == 3 * len(good)


def test_host_tensors_are_refused():
    t, n = torch.zeros(9, 32, 2, 8), torch.zeros(4, dtype=torch.int32)
    for call in (lambda: ops.cache_fork([t], n.view(4, 1), n, n), lambda: ops.cache_compact([t], n.view(4, 1), n, n),
                 lambda: ops.cache_copy([t], n, n)):
        with pytest.raises(ValueError):
            call()
