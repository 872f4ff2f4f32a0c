"""A paged cache in 8 bits: its append against the definition in 64 bits, bit by bit, and its attention against float64.

Bound of the attention, with u half a step of the type: what the cache stands for is exact in both types at these scales
(four significant bits, exponents far from their ends), so the bound is that of 16 bits: each probability is rounded once
(u of each term of the numerator, and u of the sum that divides it), the result once (u), and the fp32 scores' error times
ln 2 stays below another u.  Together 4 u sum p |v|, plus half a subnormal step of fp16 (2^-25)."""

import pytest
import torch

from tttj_2026_amd import ops

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
NAN = 0x7f


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _starts(counts):
    return _i32([0, *torch.tensor(counts).cumsum(0).tolist()])


def _randn(seed, *shape, dtype=F16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


class Cache:
    """A cache in host memory: bytes and scales as the definition has them, and its copy on the device.  It holds
    lengths[b] tokens of sequence b and has room for room[b]."""

    def __init__(self, lengths, hkv, hd, page, block, room=None, seed=0):
        g = torch.Generator().manual_seed(seed)
        need = [-(-n // page) for n in room or lengths]
        pages = sum(need) + 2
        order = torch.randperm(pages, generator=g).tolist()
        self.table = torch.full((len(lengths), max(need) + 1), 1 << 30, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
            at += n
        self.lengths, self.page, self.block, self.shape = lengths, page, block, (pages, page, hkv, hd)
        # what nobody has written yet: any bytes, NaN among them
        self.bytes = [torch.randint(0, 256, self.shape, generator=g, dtype=torch.uint8) for _ in range(2)]
        self.scales = [torch.randint(0, 256, (pages, page // block, hkv), generator=g, dtype=torch.uint8) for _ in range(2)]
        for b, n in enumerate(lengths):
            for half in range(2):
                self.append(half, b, _randn(seed + 100 * b + half, n, hkv, hd).mul(torch.exp(
                    _randn(seed + b + 7, 1, hkv, 1))), 0, F16)

    def append(self, half, b, x, first, dtype):
        """The definition: x [n, heads, hd] at positions from `first` on (they may begin before 0 or end behind the table)."""
        top = 1.875 * 2.0 ** (15 if dtype == F16 else 127)
        end = min(first + len(x), self.table.shape[1] * self.page)
        begin = max(first, 0)
        for p in range(begin // self.block * self.block, end if len(x) else 0, self.block):
            page = int(self.table[b, p // self.page])
            if not 0 <= page < self.shape[0]:
                continue
            rows = slice(p % self.page, p % self.page + self.block)
            lo, hi = max(p, begin), min(p + self.block, end)
            y = x[lo - first:hi - first].double()
            finite = torch.isfinite(y)
            largest = torch.where(finite, y, 0.0).abs().amax((0, 2))
            e = torch.frexp(largest)[1] - 9
            e = torch.where(largest > 448 * torch.exp2(e.double()), e + 1, e)
            e = torch.where(largest > 0, e, -127).clamp(min=-127) + 127
            held = self.scales[half][page, p % self.page // self.block]
            if lo > p:
                e = torch.maximum(e, held.int())
                old = self.bytes[half][page, rows][:lo - p]
                grown = (e > held.int())[:, None].expand(old.shape)
                less = torch.exp2((held.int() - e).double())[:, None]
                old[grown] = (old.view(E4M3).double() * less).float().to(E4M3).view(torch.uint8)[grown]
            z = (y.clamp(-top, top) * torch.exp2(127.0 - e.double())[:, None])
            z = torch.where(finite, z, float("nan")).float().to(E4M3).view(torch.uint8)
            self.bytes[half][page, rows][lo - p:hi - p] = z
            self.scales[half][page, p % self.page // self.block] = e.to(torch.uint8)

    def device(self):
        return dict(k_cache=self.bytes[0].cuda().view(E4M3), v_cache=self.bytes[1].cuda().view(E4M3),
                    k_scales=self.scales[0].cuda().view(E8M0), v_scales=self.scales[1].cuda().view(E8M0))

    def values(self, half, b):
        """[length, heads, hd] in 64 bits."""
        at = torch.arange(self.lengths[b])
        page = self.table[b, at // self.page].long()
        x = self.bytes[half].view(E4M3).double()[page, at % self.page]
        return x * torch.exp2(self.scales[half][page, at % self.page // self.block].double() - 127)[..., None]


def _same(cache, dev):
    """Bytes and scales, NaN of either sign alike."""
    for half, name in enumerate(("k", "v")):
        assert torch.equal(dev[name + "_scales"].view(torch.uint8).cpu(), cache.scales[half]), name
        a, b = dev[name + "_cache"].view(torch.uint8).cpu(), cache.bytes[half]
        a, b = (torch.where((t & 0x7f) == NAN, NAN, t) for t in (a, b))
        assert torch.equal(a, b), (name, (a != b).nonzero()[:5].tolist())


def _attend(q, k, v, limits, scale=None):
    """Row i of q [n, H, hd] over the first limits[i] of k, v [L, Hkv, hd] (64 bits): (o, sum p |v|).  Keys that a row does
    not see are left out whatever they hold."""
    n, h, hd = q.shape
    g, zero = h // k.shape[1], torch.zeros((), dtype=torch.float64)
    q = q.double().cpu()
    hidden = torch.arange(k.shape[0])[None, :] >= torch.as_tensor(limits)[:, None]
    out, mag = torch.zeros(n, h, hd, dtype=torch.float64), torch.zeros(n, h, hd, dtype=torch.float64)
    for i in range(h):
        s = q[:, i] @ k[:, i // g].T * (hd ** -0.5 if scale is None else scale)
        p = torch.softmax(s.masked_fill(hidden, float("-inf")), -1)
        p = torch.where(hidden, zero, p)
        x = v[:, i // g]
        fine = torch.isfinite(x)
        out[:, i] = p @ torch.where(fine, x, zero)
        mag[:, i] = p @ torch.where(fine, x, zero).abs()
        for j in (~fine).any(1).nonzero().flatten().tolist():
            seen = ~hidden[:, j]
            out[seen, i] += torch.where(fine[j], zero, x[j])
    return out.view(n, h * hd), mag.view(n, h * hd)


def _check(y, ref, mag):
    u = torch.finfo(y.dtype).eps / 2
    y = y.double().cpu()
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isnan(y), torch.isnan(ref))
    assert torch.equal(y[~fine].nan_to_num(7.0), ref[~fine].nan_to_num(7.0))
    err = (y - ref)[fine].abs()
    assert bool((err <= 4 * u * mag[fine] + 2.0 ** -25).all()), (err - 4 * u * mag[fine]).max().item()


def _reference(q, cache, counts, scale=None):
    refs, first = [], 0
    for b, n in enumerate(counts):
        length = cache.lengths[b]
        limits = (length - n + torch.arange(1, n + 1)).clamp(min=0)
        refs.append(_attend(q[first:first + n], cache.values(0, b), cache.values(1, b), limits, scale))
        first += n
    return [torch.cat(x) for x in zip(*refs)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd", [16, 64, 80, 128, 256])
@pytest.mark.parametrize("page,block", [(16, 16), (64, 16), (64, 64), (256, 128)])
@pytest.mark.parametrize("counts,lengths", [
    ([1, 1, 1], [1, 70, 300]),
    ([5, 0, 130, 17], [5, 40, 200, 16]),
    ([300], [290]),          # the first tokens have no place
    ([20, 3], [400, 290]),
])
def test_append(dtype, hd, page, block, counts, lengths):
    hkv = 3
    cache = Cache([max(n - c, 0) for n, c in zip(lengths, counts)], hkv, hd, page, block, room=lengths)
    dev = cache.device()
    size = torch.exp(2 * _randn(5, sum(counts), hkv, 1, dtype=torch.float32))  # some outgrow their block
    k, v = ((_randn(s, sum(counts), hkv, hd, dtype=torch.float32) * size).to(dtype) for s in (1, 2))
    ops.cache_append(k.cuda(), v.cuda(), dev["k_cache"], dev["v_cache"], cache.table.cuda(), _i32(lengths),
                     None if set(counts) == {1} else _starts(counts), k_scales=dev["k_scales"], v_scales=dev["v_scales"])
    first = 0
    for b, n in enumerate(counts):
        for half, x in enumerate((k, v)):
            cache.append(half, b, x[first:first + n], lengths[b] - n, dtype)
        first += n
    _same(cache, dev)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd", [16, 64, 80, 128, 144, 256])
@pytest.mark.parametrize("h,hkv", [(4, 4), (10, 2)])
@pytest.mark.parametrize("page,block", [(16, 16), (64, 16), (128, 128)])
def test_single_tokens(dtype, hd, h, hkv, page, block):
    lengths = [1, 300, 16, 17, 2, 129]
    cache = Cache(lengths, hkv, hd, page, block)
    q = _randn(3, len(lengths), h, hd, dtype=dtype)
    dev = cache.device()
    ref = _reference(q, cache, [1] * len(lengths))
    for most in (None, 300, 1):
        y = ops.cache_attention(q.cuda(), dev["k_cache"], dev["v_cache"], cache.table.cuda(), _i32(lengths),
                                max_length=most, k_scales=dev["k_scales"], v_scales=dev["v_scales"])
        _check(y, *ref)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("counts,lengths", [
    ([5, 1, 7], [1000, 40, 7]),
    ([70, 100, 0, 1], [70, 900, 30, 500]),
    ([200, 64], [200, 321]),
    ([33], [32]),
])
@pytest.mark.parametrize("h,hkv,page,block", [(4, 4, 32, 16), (6, 2, 64, 32), (8, 1, 256, 256)])
def test_chunks(dtype, hd, counts, lengths, h, hkv, page, block):
    cache = Cache(lengths, hkv, hd, page, block)
    q = _randn(4, sum(counts), h, hd, dtype=dtype)
    dev = cache.device()
    ref = _reference(q, cache, counts)
    for most in (None, 10):
        y = ops.cache_attention(q.cuda(), dev["k_cache"], dev["v_cache"], cache.table.cuda(), _i32(lengths),
                                _starts(counts), max_length=most, k_scales=dev["k_scales"], v_scales=dev["v_scales"])
        _check(y, *ref)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_split_keys(dtype, hd):
    """Keys dealt out over blocks, for single tokens, drafts and chunks."""
    for counts, lengths, h, hkv in (([1, 1], [9000, 3], 8, 1), ([4, 2], [7000, 5000], 4, 2), ([40], [6000], 8, 2)):
        cache = Cache(lengths, hkv, hd, 64, 32)
        q = _randn(5, sum(counts), h, hd, dtype=dtype)
        dev = cache.device()
        y = ops.cache_attention(q.cuda(), dev["k_cache"], dev["v_cache"], cache.table.cuda(), _i32(lengths),
                                _starts(counts), k_scales=dev["k_scales"], v_scales=dev["v_scales"])
        _check(y, *_reference(q, cache, counts))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("counts,lengths", [([5, 1, 7], [2000, 40, 7]), ([70, 100], [70, 1500])])
def test_masked_values(dtype, hd, counts, lengths):
    """NaN in the bytes of K and V reach exactly the rows that see them."""
    cache = Cache(lengths, 2, hd, 32, 32)
    for b, n in enumerate(counts):
        if n > 2:
            at = lengths[b] - 2, lengths[b] - 1
            page = [int(cache.table[b, t // 32]) for t in at]
            cache.bytes[1][page[0], at[0] % 32, 1, 4] = NAN
            cache.bytes[1][page[1], at[1] % 32, 0, 9] = NAN | 0x80
    q = _randn(9, sum(counts), 6, hd, dtype=dtype)
    dev = cache.device()
    ref = _reference(q, cache, counts)
    for most in (None, max(lengths), 10):
        _check(ops.cache_attention(q.cuda(), dev["k_cache"], dev["v_cache"], cache.table.cuda(), _i32(lengths),
                                   _starts(counts), max_length=most, k_scales=dev["k_scales"],
                                   v_scales=dev["v_scales"]), *ref)
    b = 0  # a key of the last token only
    t = lengths[b] - 1
    cache.bytes[0][int(cache.table[b, t // 32]), t % 32] = NAN
    dev = cache.device()
    y = ops.cache_attention(q.cuda(), dev["k_cache"], dev["v_cache"], cache.table.cuda(), _i32(lengths), _starts(counts),
                            k_scales=dev["k_scales"], v_scales=dev["v_scales"])
    row = counts[0] - 1
    assert bool(torch.isnan(y[row]).all())
    keep = [i for i in range(len(y)) if i != row]
    _check(y[keep], ref[0][keep], ref[1][keep])
