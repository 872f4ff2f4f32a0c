"""Packed prompts and the paged cache with values that only some rows of a tile may see.  References and bounds as in
test_gpu_seq_attention_edges.py: what a row does not see does not count, whatever it holds."""

import pytest
import torch
from test_gpu_seq_attention_edges import (BF16, F16, _attend, _check, _i32, _over_cache, _over_prompts, _randn, _starts,
                                          _store, _write)

from tttj_2026_amd import ops

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd", [8, 64, 80, 128, 256])
@pytest.mark.parametrize("h", [128, 130, 256])
def test_prompts_whose_tiles_hold_one_token(dtype, hd, h):
    """So many query heads on one key head that all rows of a tile end at the same key: what lies behind it in the last
    32 or 64 keys belongs to later tokens."""
    counts = [6, 1, 70]
    q, k, v = (_randn(s, sum(counts), n, hd, dtype=dtype) for s, n in ((1, h), (2, 1), (3, 1)))
    v[5], v[4, 0, 1], v[47, 0, hd - 1], v[48, 0, hd - 1], v[76] = NAN, INF, -INF, INF, -INF
    _check(ops.packed_attention(q, k, v, _starts(counts)), *_over_prompts(q, k, v, counts))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd", [8, 64, 128, 200, 256])
@pytest.mark.parametrize("h,counts,lengths", [
    (128, [6, 3, 2], [700, 40, 2]), (130, [6, 3], [700, 40]), (256, [5], [1500]),  # tiles of 128 rows
    (32, [2, 0], [700, 5]), (32, [3, 0, 0], [90, 0, 9]), (40, [2, 0, 0], [2500, 3, 0]),  # tiles of 32 rows
    (32, [2, 0] * 130, [75, 9] * 130),  # ... more of them than CUs
])
def test_chunks_whose_tiles_hold_one_token(dtype, hd, h, counts, lengths):
    """The same over a cache, keys in one block or dealt to many."""
    kc, vc, table, k, v = _store(lengths, 1, hd, 16, dtype)
    for b, n in enumerate(lengths):
        if n > 1:
            v[b][n - 1], v[b][n - 2, 0, hd // 2] = NAN, INF
            _write(kc, vc, table.cpu(), b, 0, k[b], v[b])
    q = _randn(9, sum(counts), h, hd, dtype=dtype)
    ref = _over_cache(q, k, v, counts, lengths)
    for most in (None, 10):
        _check(ops.cache_attention(q, kc, vc, table, _i32(lengths), _starts(counts), max_length=most), *ref)


@pytest.mark.parametrize("number", [-1, 1 << 30])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("h,counts", [(128, [12]), (32, [2, 0])])
def test_bad_page_behind_a_row(number, hd, h, counts):
    """Rows that end before a page outside the cache stay as they are, with page 0 of the cache holding NaN."""
    lengths = [112 + counts[0] // 2, 20][:len(counts)]
    kc, vc, table, k, v = _store(lengths, 1, hd, 16)
    table = torch.where(table < len(kc), table + 1, table)  # another page before the others
    kc, vc = (torch.cat([torch.full_like(c[:1], NAN), c]) for c in (kc, vc))
    table[0, 7] = number  # positions 112 ... 127
    q = _randn(4, sum(counts), h, hd)
    y = ops.cache_attention(q, kc, vc, table, _i32(lengths), _starts(counts))
    fine = counts[0] - counts[0] // 2
    assert torch.isnan(y[fine:]).all()
    ref, mag = _over_cache(q, k, v, counts, lengths)
    _check(y[:fine], ref[:fine], mag[:fine])


def _far(n, hkv, hd, gap, rising, dtype, seed):
    """K whose first feature alone counts (for the q below): scores fall or rise by `gap` (log2) along the keys; V with an
    infinity in the 10th key, two that cancel and a NaN elsewhere."""
    k = _randn(seed, n, hkv, hd, dtype=dtype)
    at = torch.linspace(0, gap, n, device="cuda")[:, None]
    k[..., 0] = at if rising else -at
    v = _randn(seed + 1, n, hkv, hd, dtype=dtype)
    v[9 if rising else -10, :, 1], v[n // 2, :, 2] = INF, -INF
    v[9, :, 4], v[-10, :, 4], v[n // 3, 0, 5] = INF, -INF, NAN
    q = torch.zeros(n, 2 * hkv, hd, dtype=dtype, device="cuda")
    q[..., 0] = 1
    return q, k, v, 0.6931471805599453


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd", [32, 128, 256])
@pytest.mark.parametrize("gap", [60, 400])
@pytest.mark.parametrize("rising", [False, True])
def test_infinities_with_small_probabilities(dtype, hd, gap, rising):
    """A row that sees an infinity in V has it in its result, however small the key's probability: no probability is 0 by
    the definition."""
    q, k, v, scale = _far(700, 2, hd, gap, rising, dtype, 11)
    for causal in (True, False):
        y = ops.packed_attention(q, k, v, _starts([700]), causal=causal, scale=scale)
        _check(y, *_over_prompts(q, k, v, [700], causal, scale))
    lengths = [3000, 700]
    kc, vc, table, ks, vs = _store(lengths, 2, hd, 32, dtype)
    for b, n in enumerate(lengths):
        _, ks[b], vs[b], scale = _far(n, 2, hd, gap, rising, dtype, 21 + b)
        _write(kc, vc, table.cpu(), b, 0, ks[b], vs[b])
    for counts in ([1, 1], [5, 2], [300, 2]):
        for most in (None, 10):  # keys in shares or not
            y = ops.cache_attention(q[:sum(counts)], kc, vc, table, _i32(lengths), _starts(counts), scale=scale,
                                    max_length=most)
            _check(y, *_over_cache(q[:sum(counts)], ks, vs, counts, lengths, scale))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd", [32, 128, 256])
def test_rows_whose_scores_are_all_infinitely_low(dtype, hd):
    """... are +0.0, whatever V holds; the rows beside them see what they should."""
    q, k, v = (_randn(s, 300, n, hd, dtype=dtype) for s, n in ((1, 4), (2, 2), (3, 2)))
    k[..., 0] = -INF
    q[..., 0] = 0.5
    q[200:, :, 0] = -0.5  # scores of +infinity: NaN
    v[0, 0, 1], v[100, 1, 2] = INF, NAN
    starts, lengths = _starts([300]), _i32([300])
    kc, vc = (torch.full((10, 32, 2, hd), NAN, dtype=dtype, device="cuda") for _ in range(2))
    table = torch.arange(10, dtype=torch.int32, device="cuda")[None]
    ops.cache_append(k, v, kc, vc, table, lengths, starts)
    ys = [ops.packed_attention(q, k, v, starts), ops.cache_attention(q, kc, vc, table, lengths, starts),
          ops.cache_attention(q, kc, vc, table, lengths, starts, max_length=1)]
    for y in ys:
        assert not y[:200].view(torch.int16).any() and torch.isnan(y[200:]).all()
    one = ops.cache_attention(q[:1], kc, vc, table, lengths)
    assert not one.view(torch.int16).any()


def _all_forms(q, k, v, lengths, scale=None):
    """Outputs of the last 300 tokens of a prompt and of its last token over the cache, with their references: as a
    prompt, as a chunk and as a single token, keys in shares or not."""
    n, hkv, hd = k.shape
    limits = torch.arange(n - len(q) + 1, n + 1)
    yield ops.packed_attention(torch.cat([q.new_zeros(n - len(q), *q.shape[1:]), q]), k, v, _starts([n]),
                               scale=scale)[n - len(q):], *_attend(q, k, v, limits, scale)
    pages = -(-n // 32)
    kc, vc = (torch.zeros(pages, 32, hkv, hd, dtype=k.dtype, device="cuda") for _ in range(2))
    table = torch.arange(pages, dtype=torch.int32, device="cuda").flip(0)[None]
    ops.cache_append(k, v, kc, vc, table, _i32([n]), _starts([n]))
    for rows in (q, q[-1:]):
        for most in (None, 10):
            yield ops.cache_attention(rows, kc, vc, table, _i32([n]), _starts([len(rows)]), scale=scale,
                                      max_length=most), *_attend(rows, k, v, limits[-len(rows):], scale)


@pytest.mark.parametrize("hd", [32, 128, 256])
def test_large_and_small_values_of_bfloat16(hd):
    """V over bfloat16's range: its largest values do not overflow the sums, small ones are not lost, and large ones of keys
    with probabilities that are 0 in fp32 do not show.  Relative to sum p |v| alone: products p v are made with p times
    2^-24, so were those below fp32's 2^-126 lost, at 1e-24 = 2^-79.7 they would be 2500 of p below 2^-22 of the largest,
    0.0006 of the sum and a third of u."""
    q, k, v = (_randn(s, n, h, hd, dtype=BF16) for s, n, h in ((1, 300, 4), (2, 2500, 2), (3, 2500, 2)))
    u = torch.finfo(BF16).eps / 2
    for size in (8e37, 1e-24):
        for y, ref, mag in _all_forms(q, k, v.clamp(-4, 4) * size, 2500):
            assert bool(((y.double() - ref).abs() <= 4 * u * mag).all())
    k[..., 0] = 0
    q[..., 0] = 1
    k[[5, 1200, 2100], :, 0] = -1000.0 * hd ** 0.5
    v[[5, 1200, 2100]] = 3e38
    for y, ref, mag in _all_forms(q, k, v, 2500):
        _check(y, ref, mag)


@pytest.mark.parametrize("length", [5000, 1 << 27])
def test_falling_starts_with_keys_in_shares(length):
    """Starts that go up and down between the same rows give every second sequence all of them; with the longest lengths
    their units of keys pass 32 bits many times over.  Nothing outside the output is written, and rising starts in the
    same call's place are right again."""
    batch, tokens, page = 512, 512, 256
    kc, vc = _randn(1, 4, page, 1, 64), _randn(2, 4, page, 1, 64)
    table = torch.zeros(1, length // page + 1, dtype=torch.int32, device="cuda").expand(batch, -1)
    q = _randn(3, tokens, 8, 64)
    lengths = torch.full((batch,), length, dtype=torch.int32, device="cuda")
    around = torch.full((3 * tokens, 512), 7.0, dtype=F16, device="cuda")
    for starts in ([tokens * (b % 2) for b in range(batch + 1)], [tokens - b for b in range(batch + 1)]):
        ops.cache_attention(q, kc, vc, table, lengths, _i32(starts), out=around[tokens:2 * tokens])
        torch.cuda.synchronize()
        assert bool((around[:tokens] == 7).all()) and bool((around[2 * tokens:] == 7).all())
    lengths.fill_(page)
    y = ops.cache_attention(q, kc, vc, table, lengths, _i32(list(range(batch + 1))))
    limits = torch.full((tokens,), page)
    _check(y, *_attend(q, kc[0], vc[0], limits))


@pytest.mark.parametrize("dtype,hd", [(F16, 64), (BF16, 128), (BF16, 256)])
@pytest.mark.parametrize("counts,lengths", [
    ([600, 1, 1, 0, 3], [700, 9000, 1, 30, 5000]),                      # tiles of 128 rows, keys dealt out
    ([1, 2600, 1, 40], [7000, 2600, 90, 3000]),                         # ... more tiles than the chip holds
    ([300] + [1] * 200, [800] + [1 + 37 * b % 1900 for b in range(200)]),  # tiles of 32 rows
])
def test_chunks_and_single_tokens_in_one_call(dtype, hd, counts, lengths):
    """New tokens of prompts that are read in pieces beside single tokens over long contexts."""
    kc, vc, table, k, v = _store(lengths, 2, hd, 16, dtype)
    q = _randn(7, sum(counts), 8, hd, dtype=dtype)
    ref = _over_cache(q, k, v, counts, lengths)
    for most in (None, max(lengths), 1):
        y = ops.cache_attention(q, kc, vc, table, _i32(lengths), _starts(counts), max_length=most)
        _check(y, *ref)
        assert torch.equal(y, ops.cache_attention(q, kc, vc, table, _i32(lengths), _starts(counts), max_length=most))
