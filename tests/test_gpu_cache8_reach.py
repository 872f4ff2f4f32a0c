"""The 8-bit cache's attention on paths that take many sequences, wide heads between the tiles' or scales near the types' ends:
each way of dealing work out, on either side of its rules.  Bounds as in test_gpu_cache8.py."""

import pytest
import torch

import test_gpu_cache8 as base
import test_gpu_cache8_edges as edges
from test_gpu_cache8 import BF16, E4M3, E8M0, F16, Cache, _attend, _check, _i32, _randn, _reference, _starts
from tttj_2026_amd import ops

pytestmark = pytest.mark.gpu

# Heads above 128 that do not fill their tile of 256.
BETWEEN = [144, 208, 240]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd", BETWEEN)
@pytest.mark.parametrize("counts,lengths,h,hkv", [
    ([5, 1, 7], [1000, 40, 7], 4, 4),
    ([70, 100, 0, 1], [70, 900, 30, 500], 6, 2),
    ([200, 64], [200, 321], 8, 1),
    ([33], [32], 6, 2),
])
def test_wide_heads_between_tiles(dtype, hd, counts, lengths, h, hkv):
    base.test_chunks(dtype, hd, counts, lengths, h, hkv, 64, 32)


@pytest.mark.parametrize("hd", BETWEEN)
def test_wide_heads_in_parts(hd):
    base.test_split_keys(F16, hd)
    base.test_split_keys(BF16, hd)
    edges.test_many_query_heads(hd, 66, 2)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd", BETWEEN)
@pytest.mark.parametrize("counts,lengths", [([5, 1, 7], [2000, 40, 7]), ([70, 100], [70, 1500])])
def test_wide_heads_between_tiles_with_nan(dtype, hd, counts, lengths):
    base.test_masked_values(dtype, hd, counts, lengths)


@pytest.mark.parametrize("hd", BETWEEN)
@pytest.mark.parametrize("counts,lengths", [([4, 2, 3], [700, 3000, 33]), ([90, 2], [200, 1500])])
def test_wide_heads_between_tiles_with_bad_pages(hd, counts, lengths):
    edges.test_bad_pages_and_scales(hd, 2, counts, lengths)
    edges.test_values_past_fp16(hd, counts, lengths)


class Pool:
    """A cache of random bytes (no NaN) and scales that any number of sequences read, pages shared."""

    def __init__(self, batch, columns, hkv, hd, page=32, block=16, pages=97, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.page, self.block = page, block
        self.table = torch.randint(0, pages, (batch, columns), generator=g, dtype=torch.int32)
        shape = (2, pages, page, hkv, hd)
        x = torch.randn(shape, generator=g).to(E4M3)
        e = torch.randint(125, 129, (2, pages, page // block, hkv), generator=g).to(torch.uint8)
        self.values = x.double() * torch.exp2(e.double() - 127).repeat_interleave(block, 2)[..., None]
        self.k, self.v = x.cuda().unbind(0)
        self.k_scales, self.v_scales = e.cuda().view(E8M0).unbind(0)

    def rows(self, half, b, n):
        at = torch.arange(n)
        return self.values[half][self.table[b, at // self.page].long(), at % self.page]

    def attend(self, q, lengths, starts=None, **how):
        return ops.cache_attention(q.cuda(), self.k, self.v, self.table.cuda(), _i32(lengths), starts,
                                   k_scales=self.k_scales, v_scales=self.v_scales, **how)


def _sampled(pool, y, q, counts, lengths, sample):
    """Sequences of `sample`, first and last rows, against float64."""
    first = torch.tensor([0, *counts]).cumsum(0).tolist()
    for b in sample:
        n = counts[b]
        if n == 0:
            continue
        at = sorted({0, n // 2, n - 1})
        rows = [first[b] + i for i in at]
        limits = [max(lengths[b] - n + i + 1, 0) for i in at]
        _check(y[rows], *_attend(q[rows], pool.rows(0, b, lengths[b]), pool.rows(1, b, lengths[b]), limits))


@pytest.mark.parametrize("dtype,hd", [(F16, 64), (BF16, 128), (F16, 128), (BF16, 64), (BF16, 112)])
@pytest.mark.parametrize("hkv", [4, 8, 6])
@pytest.mark.parametrize("batch", [63, 65, 256, 257, 513])
def test_many_sequences(dtype, hd, hkv, batch):
    """Ragged lengths to 2000, with one token each and with a few: keys dealt out, and not, by the number of sequences and of
    heads that share a block."""
    lengths = [(1 + 311 * b % 1999) for b in range(batch)]
    lengths[1], lengths[batch // 2], lengths[-1] = 2000, 0, 1
    pool = Pool(batch, 63, hkv, hd, seed=batch)
    sample = [0, 1, 2, batch // 2 - 1, batch // 2, batch // 2 + 1, batch - 2, batch - 1]
    q = _randn(1, batch, 2 * hkv, hd, dtype=dtype)
    for most in (2000, 700):  # (what is longer than the caller expects is right too)
        _sampled(pool, pool.attend(q, lengths, max_length=most), q, [1] * batch, lengths, sample)
    counts = [1 + b % 4 for b in range(batch)]
    counts[2], counts[-1] = 0, 3  # (three rows of a sequence of one key: two see none)
    q = _randn(2, sum(counts), 2 * hkv, hd, dtype=dtype)
    _sampled(pool, pool.attend(q, lengths, _starts(counts), max_length=2000), q, counts, lengths, sample)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,h,hkv", [(64, 64, 16), (128, 32, 8), (80, 32, 8), (256, 16, 8), (208, 16, 8)])
def test_tiles_by_their_keys(dtype, hd, h, hkv):
    """Chunks of very different lengths whose tiles are more than the chip holds: the heaviest come first."""
    counts = [900, 13, 0, 1500, 1, 400, 37]
    lengths = [900, 2600, 100, 1700, 500, 390, 1337]
    pool = Pool(len(counts), 82, hkv, hd, seed=hd)
    q = _randn(3, sum(counts), h, hd, dtype=dtype)
    _sampled(pool, pool.attend(q, lengths, _starts(counts)), q, counts, lengths, range(len(counts)))
    # narrow blocks: many sequences of few tokens, too short to deal keys out
    counts, hkv = [3 - b % 3 for b in range(64)], 32
    lengths = [10 + 29 * b % 300 for b in range(64)]
    pool = Pool(64, 10, hkv, hd, seed=hd + 1)
    q = _randn(4, sum(counts), 2 * hkv, hd, dtype=dtype)
    _sampled(pool, pool.attend(q, lengths, _starts(counts), max_length=310), q, counts, lengths, range(0, 64, 5))


# fp32 sums hold products of V with probabilities of up to 1 (fp16: times 2^7; bfloat16: times 2^-24, so 65536 keys cannot
# overflow), and what is subnormal in fp32 may count for nothing: 2^-126 2^24 of a result in bfloat16.
FLOOR = {F16: 2.0 ** -25, BF16: 2.0 ** -102}


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("h", [2, 66])  # narrow and wide blocks
def test_one_key_at_any_scale(dtype, hd, h):
    """A row that sees one key gets its V: every byte of e4m3 at every scale, as a conversion to the type has it (nearest, ties
    to even; infinities past the largest)."""
    for scale in range(0, 255, 3):
        cache = Cache([1, 1], 2, hd, 16, 16, seed=scale)
        for b in range(2):
            page = int(cache.table[b, 0])
            x = torch.arange(2 * hd).add(b * 128).to(torch.uint8).view(2, hd)
            cache.bytes[1][page, 0] = torch.where((x & 0x7f) == 0x7f, 0, x)
            cache.scales[1][page, 0] = _u8([scale + b, max(scale - b, 0)])
        q = _randn(1, 2, h, hd, dtype=dtype)
        y = edges._run(q, cache, [1, 1], None).view(2, 2, h // 2, hd).double().cpu()
        want = torch.cat([cache.values(1, b) for b in range(2)]).to(dtype).double()[:, :, None].expand_as(y)
        near = want.abs() >= FLOOR[dtype] if dtype == BF16 else torch.ones_like(want, dtype=torch.bool)
        assert torch.equal(y[near], want[near]), scale
        assert bool((y[~near].abs() <= FLOOR[dtype]).all()), scale


def _u8(values):
    return torch.tensor(values, dtype=torch.uint8)


@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("counts,lengths", [([1, 1], [600, 90]), ([5, 3], [600, 90]), ([80, 1], [300, 40])])
def test_small_scales(half, hd, counts, lengths):
    """K or V whose products with their scales are subnormal in fp16 or below it, or small in bfloat16, the scale byte 0 among
    them: both are what a conversion to the type makes of them."""
    for dtype, exponents in ((F16, (96, 103, 106, 109, 112, 115)), (BF16, (0, 1, 4, 9, 20, 33, 64))):
        for e in exponents:
            cache = Cache(lengths, 2, hd, 32, 16, seed=e)
            cache.scales[half][:] = torch.randint(e, e + 3, cache.scales[half].shape,
                                                  generator=torch.Generator().manual_seed(e)).to(torch.uint8)
            # Scores of a size that tells keys apart: of K at most 448 2^(e - 125), times queries and the call's scale.  Those
            # are shared out so that products of bfloat16 stay normal in fp32.
            q, scale = _randn(4, sum(counts), 4, hd, dtype=dtype), None
            if half == 0:
                scale = 2.0 ** (117 - e)
                if dtype == BF16:
                    q, scale = q * 2.0 ** 60, scale * 2.0 ** -60
            dev = cache.device()
            refs, first = [], 0
            for b, n in enumerate(counts):
                k, v = (cache.values(i, b).to(dtype).double() for i in range(2))
                limits = lengths[b] - n + torch.arange(1, n + 1)
                refs.append(_attend(q[first:first + n], k, v, limits, scale))
                first += n
            ref, mag = (torch.cat(x) for x in zip(*refs))
            y = ops.cache_attention(q.cuda(), dev["k_cache"], dev["v_cache"], cache.table.cuda(), _i32(lengths),
                                    _starts(counts), scale=scale, k_scales=dev["k_scales"], v_scales=dev["v_scales"])
            err = (y.double().cpu() - ref).abs()
            bound = 4 * torch.finfo(dtype).eps / 2 * mag + FLOOR[dtype]
            assert bool((err <= bound).all()), (dtype, e, (err / bound).max().item())


@pytest.mark.parametrize("hd", [32, 128])
def test_falling_starts_leave_the_rest_alone(hd):
    """Starts that fall: pages that no row names, guard pages on either side and the scales of both stay as they are, and the
    attention writes its output alone."""
    page, hkv, pages = 32, 2, 12
    table = _i32([[3, 5], [4, 8], [9, -7]])
    named, lengths = [3, 4, 5, 8, 9], _i32([40, 70, 64])
    g = torch.Generator().manual_seed(1)
    whole = torch.randint(0, 256, (2, pages + 2, page, hkv, hd), generator=g, dtype=torch.uint8).cuda()
    wholes = torch.randint(0, 255, (2, pages + 2, page // 16, hkv), generator=g, dtype=torch.uint8).cuda()
    args = [x[1:-1].view(E4M3) for x in whole]
    scales = dict(zip(("k_scales", "v_scales"), (x[1:-1].view(E8M0) for x in wholes)))
    before, befores = whole.clone(), wholes.clone()
    x = _randn(3, 2, 129, hkv, hd).cuda()
    q = _randn(4, 129, 4, hd).cuda()
    out = torch.zeros(131, 4 * hd, dtype=F16, device="cuda")
    others = [p for p in range(pages + 2) if p - 1 not in named]
    for s in ([0, 60, 20, 124], [200, -5, 1 << 30, 0], [124, 80, 40, 0], [-3, 129, 0, 129]):
        ops.cache_append(x[0], x[1], *args, table, lengths, _i32(s), **scales)
        assert torch.equal(whole[:, others], before[:, others]) and torch.equal(wholes[:, others], befores[:, others])
        held, helds = whole.clone(), wholes.clone()
        ops.cache_attention(q, *args, table, lengths, _i32(s), out=out[1:-1], **scales)
        assert torch.equal(whole, held) and torch.equal(wholes, helds)
        assert not bool(out[0].any()) and not bool(out[-1].any())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,h,hkv,counts,lengths", [
    (64, 16, 16, [1], [500]), (128, 32, 8, [1] * 16, [67 + 500 * b for b in range(16)]),
    (128, 32, 8, [512, 300], [4608, 700]), (208, 8, 2, [5, 90, 1], [3000, 100, 900])])
def test_calls_repeat_themselves(dtype, hd, h, hkv, counts, lengths):
    """The same call gives the same bits, whatever ran between."""
    pool = Pool(len(lengths), -(-max(lengths) // 32), hkv, hd)
    q, starts = _randn(5, sum(counts), h, hd, dtype=dtype).cuda(), _starts(counts)
    want = pool.attend(q, lengths, starts)
    for i in range(8):
        if i % 2:
            pool.attend(q.flip(0), lengths, starts)
        assert torch.equal(pool.attend(q, lengths, starts), want), i
