"""CPU tests of the 8-bit cache's host side: argument structures, refusals before any launch, workspace sizes."""

import ctypes
import pathlib
import re

import pytest
import torch

from tttj_2026_amd import _lib, ops

HEADER = (pathlib.Path(__file__).resolve().parents[1] / "include" / "tttj_amd.h").read_text()
P = 1 << 20  # an aligned address that is never read
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _fields(name):
    body = re.search(r"typedef struct \{([^}]*)\} " + name + ";", HEADER).group(1)
    fields = []
    for line in body.split(";"):
        line = line.strip()
        if line:
            kind = ctypes.c_void_p if "*" in line else {"int64_t": ctypes.c_int64, "int32_t": ctypes.c_int32,
                                                        "float": ctypes.c_float}[line.split()[0]]
            names = re.sub(r"^(const\s+)?\w+", "", line).replace("*", "").split(",")
            fields += [(n.strip(), kind) for n in names]
    return fields


STRUCTS = {"tt_cache_rows8": (_lib.CACHE_ROWS8, "tt_cache_append8"),
           "tt_cache_attention8": (_lib.CACHE_ATTENTION8, "tt_cache_attention8_fwd")}
STRIDES = dict(s_page=2, s_block=2, s_head=1, table_row=8)
GOOD = {
    "tt_cache_rows8": dict(k=P, v=P, k_cache=P, v_cache=P, k_scales=P + 1, v_scales=P + 3, table=P, lengths=P, starts=P,
                           k_row=128, k_head=64, v_row=128, v_head=64, kc_page=2048, kc_row=128, kc_head=64,
                           vc_page=2048, vc_row=128, vc_head=64, **STRIDES, tokens=4, batch=2, kv_heads=2, head_dim=64,
                           pages=9, page_size=16, table_pages=8, block=16, dtype=0),
    "tt_cache_attention8": dict(q=P, k_cache=P, v_cache=P, k_scales=P + 1, v_scales=P + 3, table=P, lengths=P, starts=P,
                                out=P, workspace=P, workspace_bytes=1 << 40, q_row=512, q_head=64, k_page=2048,
                                k_row=128, k_head=64, v_page=2048, v_row=128, v_head=64, **STRIDES, tokens=4, batch=2,
                                heads=8, kv_heads=2, head_dim=64, pages=9, page_size=16, table_pages=8, max_length=100,
                                block=16, dtype=0, scale=0.125),
}


@pytest.mark.parametrize("name", STRUCTS)
def test_structures_are_the_header_s(name):
    fields, packer = _fields(name), STRUCTS[name][0]
    kind = type(name, (ctypes.Structure,), {"_fields_": fields})
    assert ctypes.sizeof(kind) == packer.size
    formats = {ctypes.c_void_p: "Q", ctypes.c_int64: "q", ctypes.c_int32: "i", ctypes.c_float: "f"}
    fmt = packer.format
    flat = re.sub(r"(\d+)(\w)", lambda m: m.group(2) * int(m.group(1)), fmt if isinstance(fmt, str) else fmt.decode())
    assert flat == "".join(formats[t] for _, t in fields)
    assert set(GOOD[name]) | {"size", "reserved"} >= {n for n, _ in fields}


def _call(name, **change):
    values = {**GOOD[name], **change}
    kind = type(name, (ctypes.Structure,), {"_fields_": _fields(name)})
    s = kind(**{k: v for k, v in values.items() if k != "size"})
    s.size = values.get("size", ctypes.sizeof(kind))
    return getattr(_lib.load(), STRUCTS[name][1])(ctypes.byref(s), None)


def _refused(name, **change):
    assert _call(name, **change) == _lib.TT_ERR_INVALID, (name, change)
    return _lib.last_error()


@pytest.mark.parametrize("name", STRUCTS)
def test_refusals(name):
    fields = [n for n, _ in _fields(name)]
    assert _lib.TT_ERR_INVALID == getattr(_lib.load(), STRUCTS[name][1])(None, None)
    assert name in _refused(name, size=8)
    for change in (dict(tokens=-1), dict(batch=-1), dict(kv_heads=0), dict(kv_heads=-2), dict(head_dim=0), dict(dtype=2),
                   dict(head_dim=24), dict(head_dim=272), dict(tokens=1 << 30, heads=8, kv_heads=8), dict(pages=0),
                   dict(table_pages=0), dict(page_size=8), dict(page_size=48), dict(page_size=1 << 20, table_pages=1 << 11),
                   dict(block=1 << 17, page_size=1 << 17), dict(block=8), dict(block=0), dict(block=32), dict(block=48, page_size=64), dict(block=-16),
                   dict(s_page=1 << 31), dict(s_block=1 << 31, page_size=32), dict(s_head=1 << 31), dict(s_page=1 << 28),
                   dict(s_page=(1 << 28) - 1, s_head=8), dict(s_page=1 << 62, s_head=1 << 62),
                   dict(table_row=-1), dict(starts=None)):
        _refused(name, **{k: v for k, v in change.items() if k in fields})
    for field, kind in _fields(name):
        if kind is ctypes.c_void_p and field not in ("starts", "workspace"):
            _refused(name, **{field: None})
        if kind is ctypes.c_void_p and field not in ("starts", "table", "lengths", "workspace", "k_scales", "v_scales"):
            _refused(name, **{field: P + 8})
        if field.endswith(("_row", "_head", "_page", "_block")):
            _refused(name, **{field: -64})
        if field.endswith(("_row", "_head", "_page")) and field[0] != "s" and field != "table_row":
            _refused(name, **{field: 68})
            if field not in ("q_row", "q_head") and (name == "tt_cache_attention8" or field[1] == "c"):
                _refused(name, **{field: 72})  # 8 bytes: rows of a cache in 8 bits are read 16 at a time
    for field in ("k_row", "v_row", "kc_row", "vc_row"):
        if field in fields:
            _refused(name, **{field: 1 << 26})
    if "heads" in fields:
        _refused(name, heads=3), _refused(name, heads=0), _refused(name, max_length=-1)
        for scale in (0.0, -1.0, float("nan"), float("inf")):
            _refused(name, scale=scale)


@pytest.mark.parametrize("name", STRUCTS)
def test_nothing_to_do_launches_nothing(name):
    for change in (dict(tokens=0), dict(batch=0)):
        assert _call(name, **change) == _lib.TT_OK


def test_workspace():
    size = _lib.cache_attention_workspace_bytes
    assert size(64, 64, 32, 8, 128, 16, 32, 300, True, True) == 0
    assert size(4, 4, 64, 8, 128, 64, 1600, 100000, True, True) > 0
    need = dict(tokens=2, starts=None, max_length=100000, table_pages=8000, page_size=16)
    assert size(2, 2, 8, 2, 64, 16, 8000, 100000, True, True) > 64
    assert "workspace" in _refused("tt_cache_attention8", **need, workspace_bytes=64)
    assert "workspace" in _refused("tt_cache_attention8", **need, workspace=None)
    assert "workspace" in _refused("tt_cache_attention8", **need, workspace=P + 8)
    for bad in ((1, 1, 8, 2, 72, 16, 8, 9, True, True), (1, 1, 8, 2, 64, 16, 8, -1, True, True)):
        with pytest.raises(ValueError):
            size(*bad)


@pytest.fixture
def host(monkeypatch):
    """Host tensors pass for the device's, up to the library call, which is counted."""
    calls = []
    monkeypatch.setattr(ops, "_typed", lambda t, name: (t.dtype, t.get_device()))
    monkeypatch.setattr(ops, "_call", lambda name, args, index: calls.append(name))
    return calls


def test_tensors(host):
    q, k = torch.zeros(4, 8, 64, dtype=torch.float16), torch.zeros(4, 2, 64, dtype=torch.float16)
    starts, table = torch.tensor([0, 4], dtype=torch.int32), torch.zeros(1, 8, dtype=torch.int32)
    length = starts[1:]
    cache, scales = torch.zeros(9, 32, 2, 64).to(E4M3), torch.zeros(9, 2, 2, dtype=torch.uint8).view(E8M0)
    good = dict(k_scales=scales, v_scales=scales)

    def both(k_cache=cache, v_cache=cache, **scales_):
        ops.cache_append(k, k, k_cache, v_cache, table, length, starts, **scales_)
        ops.cache_attention(q, k_cache, v_cache, table, length, starts, **scales_)

    both(**good)
    halves = torch.zeros(9, 2, 32, 2, 64).to(E4M3).unbind(1)
    both(*halves, **{n: torch.zeros(2, 9, 2, dtype=torch.uint8).view(E8M0).permute(1, 2, 0) for n in good})
    both(**{n: torch.zeros(9, 1, 2, dtype=torch.uint8).view(E8M0) for n in good})
    assert host == ["tt_cache_append8", "tt_cache_attention8_fwd"] * 3
    sixteen = cache.to(torch.float16)
    bad = [dict(k_scales=scales), dict(v_scales=scales), dict(good, k_cache=sixteen, v_cache=sixteen), {},
           dict(k_scales=scales.view(torch.uint8), v_scales=scales), dict(k_scales=scales, v_scales=scales.float()),
           dict(k_scales=scales[:8], v_scales=scales[:8]), dict(k_scales=scales[:, :1], v_scales=scales),
           dict(k_scales=scales[..., :1], v_scales=scales[..., :1]), dict(k_scales=scales[:, :0], v_scales=scales[:, :0]),
           dict(k_scales=scales[..., 0], v_scales=scales[..., 0]), dict(good, v_cache=cache[:8]),
           dict(good, k_cache=cache[..., :32], v_cache=cache[..., :32]),
           dict(good, k_cache=cache.transpose(2, 3), v_cache=cache.transpose(2, 3)),
           dict(good, v_cache=torch.zeros(cache.numel() + 8).to(E4M3)[8:].view(cache.shape)),
           {n: torch.zeros(9, 3, 2, dtype=torch.uint8).view(E8M0) for n in good},
           dict(k_scales=scales, v_scales=torch.zeros(2, 9, 2, dtype=torch.uint8).view(E8M0).permute(1, 2, 0))]
    for change in bad:
        change = {"k_cache": cache, "v_cache": cache, **change}
        caches = change.pop("k_cache"), change.pop("v_cache")
        with pytest.raises(ValueError):
            ops.cache_append(k, k, *caches, table, length, starts, **change)
        with pytest.raises(ValueError):
            ops.cache_attention(q, *caches, table, length, starts, **change)
    assert len(host) == 6


def test_host_tensors_are_refused():
    q, starts = torch.zeros(4, 8, 64, dtype=torch.float16), torch.tensor([0, 4], dtype=torch.int32)
    cache, scales = torch.zeros(9, 32, 8, 64).to(E4M3), torch.zeros(9, 2, 8, dtype=torch.uint8).view(E8M0)
    table = torch.zeros(1, 8, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.cache_append(q, q, cache, cache, table, starts[1:], starts, k_scales=scales, v_scales=scales)
    with pytest.raises(ValueError):
        ops.cache_attention(q, cache, cache, table, starts[1:], starts, k_scales=scales, v_scales=scales)
