"""The 8-bit cache where it can go wrong: bad pages and scales, values past fp16, strides, offsets past 32 bits, heads side
by side in a block, growing and exhausted scales, values of the append at the ends of their types, lengths cut to the
table, falling starts, captured graphs, streams and calls at once.  Bounds as in test_gpu_cache8.py."""

import threading

import pytest
import torch

from test_gpu_cache8 import BF16, E4M3, E8M0, F16, NAN, Cache, _attend, _check, _i32, _randn, _reference, _same, _starts
from tttj_2026_amd import ops

pytestmark = pytest.mark.gpu


def _run(q, cache, lengths, starts, dev=None, table=None, **how):
    dev = cache.device() if dev is None else dev
    return ops.cache_attention(q.cuda(), dev["k_cache"], dev["v_cache"], cache.table.cuda() if table is None else table,
                               _i32(lengths), starts, k_scales=dev["k_scales"], v_scales=dev["v_scales"], **how)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd", [16, 48, 64, 80, 128])
@pytest.mark.parametrize("h,hkv", [(4, 4), (16, 8), (6, 6), (9, 3), (2, 1), (20, 4)])
def test_heads_side_by_side(dtype, hd, h, hkv):
    """Narrow blocks (more tokens than CUs, or keys dealt out) whose waves share tiles for 1, 2 or 4 heads."""
    lengths = [1 + 7 * i % 70 for i in range(150)]
    cache = Cache(lengths, hkv, hd, 32, 16)
    q = _randn(1, len(lengths), h, hd, dtype=dtype)
    _check(_run(q, cache, lengths, None, max_length=70), *_reference(q, cache, [1] * len(lengths)))
    lengths, counts = [2100, 130, 3, 1300], [2, 1, 3, 1]
    cache = Cache(lengths, hkv, hd, 64, 32)
    q = _randn(2, sum(counts), h, hd, dtype=dtype)
    _check(_run(q, cache, lengths, _starts(counts)), *_reference(q, cache, counts))


@pytest.mark.parametrize("hd", [32, 64, 112, 128, 256])
@pytest.mark.parametrize("h,hkv", [(40, 1), (66, 2), (100, 1)])
def test_many_query_heads(hd, h, hkv):
    """More rows a token than a narrow block has, alone, in a batch and with keys dealt out."""
    for counts, lengths in (([1], [700]), ([1] * 5, [1, 64, 90, 2500, 17]), ([2, 9, 0], [300, 60, 5])):
        cache = Cache(lengths, hkv, hd, 32, 32)
        q = _randn(9, sum(counts), h, hd, dtype=BF16)
        starts = None if set(counts) == {1} else _starts(counts)
        _check(_run(q, cache, lengths, starts), *_reference(q, cache, counts))


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("hkv", [1, 2, 4])
@pytest.mark.parametrize("counts,lengths", [([4, 2, 3], [700, 3000, 33]), ([90, 2], [200, 1500])])
def test_bad_pages_and_scales(hd, hkv, counts, lengths):
    """A page outside the cache, and a block whose scale of K or V is none, are NaN for the rows that see a key of them and
    for no other."""
    for kind in ("page", "k", "v"):
        cache = Cache(lengths, hkv, hd, 16, 16)
        q = _randn(3, sum(counts), 2 * hkv, hd)
        clean = _run(q, cache, lengths, _starts(counts))
        # the block that holds the last keys of sequence 0, and one in the middle of sequence 1
        spoiled = {0: lengths[0] - 2, 1: lengths[1] // 2}
        head = hkv - 1
        for b, t in spoiled.items():
            page = int(cache.table[b, t // 16])
            if kind == "page":
                cache.table[b, t // 16] = [-1, 1 << 30][b]
            else:
                cache.scales["kv".index(kind)][page, 0, head] = 255
        for most in (None, 10):
            y = _run(q, cache, lengths, _starts(counts), max_length=most)
            first = 0
            for b, n in enumerate(counts):
                for i in range(n):
                    seen = b in spoiled and lengths[b] - n + i >= spoiled[b] // 16 * 16
                    got = y[first + i].view(hkv, -1)
                    if kind == "page":
                        bad = torch.full((hkv,), seen)
                    else:
                        bad = torch.tensor([seen and h == head for h in range(hkv)])
                    assert torch.equal(torch.isnan(got).any(1).cpu(), bad), (kind, b, i)
                    assert bool(torch.isnan(got[bad.cuda()]).all())
                    keep = ~bad.cuda()
                    # (where nothing is spoiled the sums are the same, part by part)
                    if most is None:
                        assert torch.equal(got[keep], clean[first + i].view(hkv, -1)[keep])
                first += n


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("counts,lengths", [([5, 3], [600, 90]), ([80, 1], [300, 40])])
def test_values_past_fp16(hd, counts, lengths):
    """Large scales, as bfloat16 writes them: in fp16 what lies past its largest is an infinity in V, for the rows that see
    it and no other; in bfloat16 it is what it is."""
    for e in (135, 137, 142, 150, 152, 160):
        cache = Cache(lengths, 2, hd, 32, 16, seed=e)
        for b, n in enumerate(counts):
            t = lengths[b] - max(n // 2, 1)  # some rows see it, some do not
            cache.scales[1][int(cache.table[b, t // 32]), t % 32 // 16, 1] = e
        q = _randn(4, sum(counts), 4, hd)
        dev = cache.device()
        refs, first = [], 0
        for b, n in enumerate(counts):
            v = cache.values(1, b).to(F16).double()
            limits = lengths[b] - n + torch.arange(1, n + 1)
            # two infinities of unlike sign make NaN, and so on: what fp32 sums make of them
            refs.append(_attend(q[first:first + n], cache.values(0, b), v, limits))
            first += n
        _check(_run(q, cache, lengths, _starts(counts), dev), *(torch.cat(x) for x in zip(*refs)))
        q = q.to(BF16)
        _check(_run(q, cache, lengths, _starts(counts), dev), *_reference(q, cache, counts))


@pytest.mark.parametrize("hd,hkv", [(64, 4), (128, 2), (96, 3)])
def test_strides(hd, hkv):
    """Both halves in one tensor, heads outside tokens, tokens with room behind them, scales in any order."""
    counts, lengths, page, block = [3, 40, 1], [1200, 64, 300], 64, 16
    cache = Cache(lengths, hkv, hd, page, block)
    q = _randn(5, sum(counts), 2 * hkv, hd, dtype=BF16)
    ref = _reference(q, cache, counts)
    pages = cache.shape[0]
    k, v = (x.cuda() for x in cache.bytes)
    ks, vs = (x.cuda() for x in cache.scales)
    both = torch.stack([k, v], 1)
    turned = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v)]
    roomy = torch.zeros(2, pages, page, hkv + 1, hd + 16, dtype=torch.uint8, device="cuda")
    roomy[:, :, :, :hkv, :hd] = torch.stack([k, v])
    scales = torch.stack([ks, vs], -1).permute(1, 2, 0, 3).contiguous().permute(2, 0, 1, 3)
    x = _randn(6, 2, sum(counts), hkv, hd, dtype=BF16).cuda()
    want = None
    for a, b in ((k, v), both.unbind(1), turned, roomy[:, :, :, :hkv, :hd].unbind(0)):
        for s, t in ((ks, vs), scales.unbind(-1)):
            a, b, s2, t2 = a.clone(memory_format=torch.preserve_format), b, s, t
            args = dict(k_scales=s.view(E8M0), v_scales=t.view(E8M0))
            y = ops.cache_attention(q.cuda(), a.view(E4M3), b.view(E4M3), cache.table.cuda(), _i32(lengths),
                                    _starts(counts), **args)
            _check(y, *ref)
            halves = [z.clone(memory_format=torch.preserve_format) for z in (a, b, s, t)]
            strides = [z.stride() for z in halves]
            ops.cache_append(x[0], x[1], halves[0].view(E4M3), halves[1].view(E4M3), cache.table.cuda(), _i32(lengths),
                             _starts(counts), k_scales=halves[2].view(E8M0), v_scales=halves[3].view(E8M0))
            assert strides == [z.stride() for z in halves]
            halves = [z.cpu() for z in halves]
            want = want or halves
            for z, w in zip(halves, want):
                assert torch.equal(z, w)
    assert not bool(roomy[:, :, :, hkv:].any()) and not bool(roomy[..., hd:].any())
    wide = torch.zeros(sum(counts), 4 * hkv, hd + 8, dtype=BF16, device="cuda")  # queries with room between them
    wide[:, :2 * hkv, :hd] = q.cuda()
    y = ops.cache_attention(wide[:, :2 * hkv, :hd], k.view(E4M3), v.view(E4M3), cache.table.cuda(), _i32(lengths),
                            _starts(counts), k_scales=ks.view(E8M0), v_scales=vs.view(E8M0))
    _check(y, *ref)


def test_offsets_past_32_bits():
    """A cache of more than 4 GiB a half, whose last pages are used."""
    page, hkv, hd = 256, 32, 128
    pages = (1 << 32) // (page * hkv * hd) + 3  # 4099 pages of 1 MiB
    k, v = (torch.zeros(pages, page, hkv, hd, dtype=torch.uint8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros(pages, page // 16, hkv, dtype=torch.uint8, device="cuda") for _ in range(2))
    table, lengths = _i32([[pages - 1, pages - 3]]), _i32([300])
    x = _randn(7, 2, 300, hkv, hd).cuda()
    args = k.view(E4M3), v.view(E4M3), table, lengths
    scales = dict(k_scales=ks.view(E8M0), v_scales=vs.view(E8M0))
    ops.cache_append(x[0], x[1], *args, _i32([0, 300]), **scales)
    assert not bool(k[:pages - 3].any()) and not bool(v[pages - 2].any())
    small = Cache([300], hkv, hd, page, 16)
    small.table[0, :2] = torch.tensor([1, 0], dtype=torch.int32)
    for half in range(2):
        small.append(half, 0, x[half].cpu(), 0, F16)
    for half, (y, s) in enumerate(((k, ks), (v, vs))):
        for at, there in ((pages - 1, 1), (pages - 3, 0)):
            n = 256 if there else 44
            assert torch.equal(y[at, :n].cpu(), small.bytes[half][there, :n])
            assert torch.equal(s[at, :-(-n // 16)].cpu(), small.scales[half][there, :-(-n // 16)])
    for counts in ([1], [5], [70]):
        q = _randn(8, counts[0], hkv, hd)
        y = ops.cache_attention(q.cuda(), *args, _starts(counts), **scales)
        _check(y, *_reference(q, small, counts))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_append_at_the_ends_of_the_types(dtype):
    """Zeros, subnormals, the largest values (which e4m3 would round past them), infinities and NaN, every value of the type
    in turn, and scales that grow over the whole range."""
    hkv, hd, page, block = 1, 64, 64, 16
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype).view(-1, hkv, hd)  # 1024 tokens
    blocks = [bits]
    top = torch.finfo(dtype).max
    for x in (0.0, -0.0, top, -top, torch.finfo(dtype).tiny, torch.finfo(dtype).smallest_normal / 8, float("inf"),
              float("nan"), 1.0, 448.0, 464.0, 465.0):
        y = torch.zeros(16, hkv, hd, dtype=dtype)
        y[3, 0, 5] = x
        blocks.append(y)
    x = torch.cat(blocks)
    cache = Cache([0], hkv, hd, page, block, room=[len(x)])
    dev = cache.device()
    ops.cache_append(x.cuda(), x.flip(0).cuda(), dev["k_cache"], dev["v_cache"], cache.table.cuda(), _i32([len(x)]),
                     _i32([0, len(x)]), k_scales=dev["k_scales"], v_scales=dev["v_scales"])
    cache.append(0, 0, x, 0, dtype), cache.append(1, 0, x.flip(0), 0, dtype)
    _same(cache, dev)
    # one token after another, each larger than the last, then smaller ones
    cache = Cache([0], hkv, hd, page, block, room=[64])
    dev = cache.device()
    powers = [-24, -20, -13, -9, -3, 0, 1, 5, 9, 12, 15, 14, 2, -20] if dtype == F16 else \
        [-133, -128, -120, -60, -9, -1, 3, 40, 90, 119, 120, 126, 127, 127, 1, -130]
    for t, p in enumerate(powers):
        y = (_randn(t, 1, hkv, hd, dtype=torch.float64).clamp(-1.99, 1.99) * 2.0 ** p).to(dtype)
        ops.cache_append(y.cuda(), -y.cuda(), dev["k_cache"], dev["v_cache"], cache.table.cuda(), _i32([t + 1]),
                         k_scales=dev["k_scales"], v_scales=dev["v_scales"])
        cache.append(0, 0, y, t, dtype), cache.append(1, 0, -y, t, dtype)
        _same(cache, dev)


@pytest.mark.parametrize("hd", [16, 256])
def test_append_large_blocks(hd):
    """One scale for 4096 tokens: far more pieces than a block's lanes keep, older ones among them."""
    cache = Cache([1000], 2, hd, 4096, 4096, room=[6000])
    dev = cache.device()
    x = (_randn(3, 2, 4500, 2, hd, dtype=torch.float32) * 6).to(BF16)
    ops.cache_append(x[0].cuda(), x[1].cuda(), dev["k_cache"], dev["v_cache"], cache.table.cuda(), _i32([5500]),
                     _i32([0, 4500]), k_scales=dev["k_scales"], v_scales=dev["v_scales"])
    for half in range(2):
        cache.append(half, 0, x[half], 1000, BF16)
    cache.lengths = [5500]
    _same(cache, dev)
    q = _randn(4, 3, 4, hd, dtype=BF16)
    _check(_run(q, cache, [5500], _starts([3])), *_reference(q, cache, [3]))


def test_append_to_a_block_without_a_scale():
    """A scale that is none stays none until its block is begun anew."""
    cache = Cache([20], 2, 32, 32, 16, room=[64])
    cache.scales[0][int(cache.table[0, 0]), 1, 0] = 255
    dev = cache.device()
    x = _randn(1, 3, 2, 32)
    ops.cache_append(x.cuda(), x.cuda(), dev["k_cache"], dev["v_cache"], cache.table.cuda(), _i32([23]), _i32([0, 3]),
                     k_scales=dev["k_scales"], v_scales=dev["v_scales"])
    assert int(dev["k_scales"].view(torch.uint8)[int(cache.table[0, 0]), 1, 0]) == 255
    x = _randn(2, 10, 2, 32)
    ops.cache_append(x.cuda(), x.cuda(), dev["k_cache"], dev["v_cache"], cache.table.cuda(), _i32([26]), _i32([0, 10]),
                     k_scales=dev["k_scales"], v_scales=dev["v_scales"])
    cache.append(1, 0, _randn(1, 3, 2, 32), 20, F16)
    for half in range(2):
        cache.append(half, 0, x, 16, F16)
    _same(cache, dev)


def test_what_is_not_written():
    """Tokens before position 0, behind the table or in no page, rows of no sequence, and what others hold stay."""
    cache = Cache([0, 40, 0], 2, 32, 32, 16, room=[40, 64, 64])
    cache.table[2, 1] = -7
    table = cache.table[:, :2].contiguous()
    cache.table = table
    dev = cache.device()
    counts, lengths, first = [50, 30, 40], [40, 70, 64], 4
    x = _randn(3, 2, sum(counts) + first + 5, 2, 32)
    starts = _i32([4, 54, 84, 124])
    ops.cache_append(x[0].cuda(), x[1].cuda(), dev["k_cache"], dev["v_cache"], table.cuda(), _i32(lengths), starts,
                     k_scales=dev["k_scales"], v_scales=dev["v_scales"])
    for half in range(2):
        at = first
        for b, n in enumerate(counts):
            cache.append(half, b, x[half, at:at + n], lengths[b] - n, F16)
            at += n
    _same(cache, dev)
    # falling starts: nothing outside the cache's own pages, and nothing hangs
    for s in ([0, 60, 20, 124], [200, -5, 1 << 30, 0], [124, 80, 40, 0]):
        ops.cache_append(x[0].cuda(), x[1].cuda(), dev["k_cache"], dev["v_cache"], table.cuda(), _i32(lengths), _i32(s),
                         k_scales=dev["k_scales"], v_scales=dev["v_scales"])
        q = _randn(4, 129, 4, 32)
        ops.cache_attention(q.cuda(), dev["k_cache"], dev["v_cache"], table.cuda(), _i32(lengths), _i32(s),
                            k_scales=dev["k_scales"], v_scales=dev["v_scales"])
    torch.cuda.synchronize()


def test_lengths_are_cut_to_the_table():
    cache = Cache([64, 64], 2, 64, 32, 16)
    table = cache.table[:, :2].contiguous()
    q = _randn(5, 2, 4, 64)
    for lengths in ([64, 64], [500, 2 ** 31 - 1]):
        y = _run(q, cache, lengths, None, table=table.cuda())
        _check(y, *_reference(q, cache, [1, 1]))
    y = _run(q, cache, [0, -5], None, table=table.cuda())
    assert not bool(y.any())


def test_rows_outside_sequences():
    cache = Cache([100, 30], 2, 64, 32, 16)
    q = _randn(6, 12, 4, 64)
    out = torch.full((12, 256), 7.0, dtype=F16, device="cuda")
    dev = cache.device()
    ops.cache_attention(q.cuda(), dev["k_cache"], dev["v_cache"], cache.table.cuda(), _i32([100, 30]), _i32([2, 5, 9]),
                        out=out, k_scales=dev["k_scales"], v_scales=dev["v_scales"])
    assert bool((out[:2] == 7).all()) and bool((out[9:] == 7).all())
    _check(out[2:9], *_reference(q[2:9], cache, [3, 4]))


@pytest.mark.parametrize("hkv,hd", [(2, 64), (2, 256)])
def test_graphs_and_streams(hkv, hd):
    """Growing lengths under a captured call, on another stream, and two captured calls of their own workspaces."""
    lengths = [3000, 40, 900]
    cache = Cache(lengths, hkv, hd, 64, 32)
    dev, table = cache.device(), cache.table.cuda()
    n, q = _i32([2000, 20, 300]), _randn(7, 3, 2 * hkv, hd, dtype=BF16).cuda()

    def call():
        return ops.cache_attention(q, dev["k_cache"], dev["v_cache"], table, n, max_length=3000, k_scales=dev["k_scales"],
                                   v_scales=dev["v_scales"])

    eager = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, eager)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(call())
    for more in ([0, 0, 0], [700, 3, 600], [300, 17, 0]):
        n.add_(_i32(more))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        eager = call()
        for y in outs:
            assert torch.equal(y, eager)
        _check(eager, *_lengths_reference(q, cache, n.tolist()))


def _lengths_reference(q, cache, lengths):
    refs = [_attend(q[b:b + 1], cache.values(0, b)[:n], cache.values(1, b)[:n], [n]) for b, n in enumerate(lengths)]
    return [torch.cat(x) for x in zip(*refs)]


def test_calls_at_once():
    """Two threads on streams of their own, over one cache."""
    lengths = [4000, 50]
    cache = Cache(lengths, 4, 64, 64, 32)
    dev, table, n = cache.device(), cache.table.cuda(), _i32(lengths)
    qs = [_randn(s, 2, 8, 64).cuda() for s in (1, 2)]
    want = [_run(q, cache, lengths, None, dev, table) for q in qs]
    torch.cuda.synchronize()
    got, failed = [None, None], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(50):
                    got[i] = ops.cache_attention(qs[i], dev["k_cache"], dev["v_cache"], table, n,
                                                 k_scales=dev["k_scales"], v_scales=dev["v_scales"])
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for g, w in zip(got, want):
        assert torch.equal(g, w)


def test_long_contexts_of_small_probabilities():
    """30000 keys a 2^-20th of the largest each: together they count."""
    n, hd = 30001, 64
    cache = Cache([n], 1, hd, 256, 256)
    k = torch.zeros(n, 1, hd, dtype=F16)
    k[0, 0, 0] = 8.0
    v = torch.ones(n, 1, hd, dtype=F16)
    v[0] = -1.0
    cache.append(0, 0, k, 0, F16), cache.append(1, 0, v, 0, F16)
    for dtype in (F16, BF16):
        q = torch.zeros(1, 1, hd, dtype=dtype)
        q[0, 0, 0] = 14.0  # 14 * 8 / 8 = 14: exp(-14) each, 30000 of them 0.025
        _check(_run(q, cache, [n], None), *_reference(q, cache, [1]))
