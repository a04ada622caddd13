"""The paged 4-bit KV cache: rows into and out of it, attention over it, and copies of its pages."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import mxfp4
from tests.serving import Cache, assert_within, attention64, cumulative, half_values, i32
from texelator_amd import _lib, layers

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


# ---------------------------------------------------------------------------------------------
# rows


def place(lengths, new, page_size, seed, spare=2):
    """A block table of scattered pages, and (page, offset) of every new token, which are each sequence's last ones."""
    rng = np.random.default_rng(seed)
    counts = [-(-n // page_size) for n in lengths]
    order = rng.permutation(sum(counts) + spare)
    table = np.full((len(lengths), max(1, max(counts)) + 1), -1, dtype=np.int32)
    at, where = 0, []
    for s, n in enumerate(lengths):
        table[s, :counts[s]] = order[at:at + counts[s]]
        at += counts[s]
        where += [(int(table[s, p // page_size]), p % page_size) for p in range(n - new[s], n)]
    return i32(table.reshape(-1)).view(table.shape), where, len(order)


def rows(tokens, kv_heads, dim, dtype, seed):
    """[tokens, 2, kv_heads, dim] of many magnitudes, zeros and groups at the type's borders among them."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, 2, kv_heads, dim, generator=g) * torch.exp(4 * torch.randn(tokens, 2, kv_heads, dim // 32, generator=g)).repeat_interleave(32, -1)
    x[0, 0, 0, :32] = 0
    x[-1, 1, -1, 32:64] = -0.0
    x[0, 1, 0, :32] = torch.arange(32) / 4 - 4  # exact ties
    x[-1, 0, 0, -32:] = torch.finfo(dtype).max
    x[tokens // 2, 0, -1, :32] = torch.finfo(dtype).smallest_normal / 64
    x[tokens // 2, 1, -1, -32:] = torch.finfo(dtype).tiny * torch.arange(32)
    return x.clamp(torch.finfo(dtype).min, torch.finfo(dtype).max).to(dtype)


CASES = [
    # lengths after the call, new tokens, kv heads, dim, page size
    ([1], None, 1, 64, 16),
    ([5, 700, 16, 33], None, 2, 128, 16),
    ([5, 0, 700], [5, 0, 1], 3, 128, 64),
    ([17, 16, 15, 256, 257], [17, 1, 15, 100, 257], 2, 64, 32),
    ([1000], [999], 5, 128, 1024),
    ([0, 0, 3], [0, 0, 3], 1, 64, 16),
    (list(range(1, 101)), [1 + n // 3 for n in range(1, 101)], 2, 128, 16),
    ([2] * 2500, [n % 3 for n in range(2500)], 1, 64, 16),  # more sequences than the search holds in LDS
]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("lengths,new,kv_heads,dim,page_size", CASES)
def test_rows_are_stored_and_read_back_to_the_bit(ext, lengths, new, kv_heads, dim, page_size, dtype):
    counts = new if new is not None else [1] * len(lengths)
    table, where, total = place(lengths, counts, page_size, len(lengths))
    tokens = sum(counts)
    x = rows(tokens, kv_heads, dim, dtype, tokens)
    half = page_size * dim * 17 // 32
    before = np.random.default_rng(5).integers(0, 256, size=(total, kv_heads, 2, half), dtype=np.uint8)
    pages, cu = torch.from_numpy(before.copy()).cuda(), cumulative(counts) if new is not None else None
    behind = torch.full((3, 2, kv_heads, dim), float("nan"), dtype=dtype) if new is not None else x[:0]
    gpu = torch.cat([x, behind]).cuda()  # rows behind the last sequence
    layers.kv4_append(gpu[:, 0], gpu[:, 1], pages, table, i32(lengths), cu=cu)
    want = before.copy()
    codes, exponents = mxfp4.quantize(x.float().numpy())
    packed = mxfp4.pack(codes)
    split = page_size * dim // 2
    for t, (page, offset) in enumerate(where):
        c = want[page, :, :, :split].reshape(kv_heads, 2, page_size, dim // 2)
        c[:, :, offset] = packed[t].transpose(1, 0, 2)
        want[page, :, :, :split] = c.reshape(kv_heads, 2, -1)
        e = want[page, :, :, split:].reshape(kv_heads, 2, page_size, dim // 32)
        e[:, :, offset] = exponents[t].transpose(1, 0, 2)
        want[page, :, :, split:] = e.reshape(kv_heads, 2, -1)
    assert np.array_equal(pages.cpu().numpy(), want)
    out = torch.full((tokens + len(behind), 2, kv_heads, dim), float("nan"), dtype=dtype, device="cuda")
    layers.kv4_read(pages, table, i32(lengths), dim, cu=cu, out=(out[:, 0], out[:, 1]))
    values = torch.from_numpy(mxfp4.dequantize(codes, exponents)).to(dtype)
    assert torch.equal(out[:tokens].cpu(), values) and torch.isnan(out[tokens:]).all()
    k, v = layers.kv4_read(pages, table, i32(lengths), dim, cu=cu, tokens=tokens, dtype=dtype)
    assert torch.equal(k.cpu(), values[:, 0]) and torch.equal(v.cpu(), values[:, 1])


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_every_code_and_scale_reads_as_defined(ext, dtype, dim):
    """All 256 scales with all codes: 255 is NaN, 0 is 2^-127; fp16 rounds what it cannot hold."""
    rng = np.random.default_rng(3)
    half = np.empty((4, 1, 2, 64 * dim * 17 // 32), dtype=np.uint8)
    half[..., :32 * dim] = rng.integers(0, 256, size=(4, 1, 2, 32 * dim), dtype=np.uint8)
    half[..., 32 * dim:] = np.resize(np.arange(256, dtype=np.uint8), (4, 1, 2, 2 * dim))
    pages = torch.from_numpy(half).cuda()
    table = i32([2, 0, 3, 1]).view(1, 4)
    k, v = layers.kv4_read(pages, table, i32([256]), dim, cu=i32([0, 256]), tokens=256, dtype=dtype)
    want = torch.from_numpy(half_values(half, 64, dim))[[2, 0, 3, 1]].permute(2, 0, 3, 1, 4).reshape(2, 256, 1, dim).to(dtype)
    for got, expected in zip((k, v), want):
        assert torch.equal(torch.nan_to_num(got.cpu(), 7.7, 8.8, 9.9), torch.nan_to_num(expected, 7.7, 8.8, 9.9))


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_a_group_that_is_not_finite_reads_as_nan_and_no_other(ext, dtype):
    x = torch.randn(4, 2, 1, 64, dtype=torch.float32).to(dtype)
    x[0, 0, 0, 5], x[1, 1, 0, 40], x[2, 0, 0, 0] = float("nan"), float("inf"), float("-inf")
    x[2, 0, 0, 1] = float("nan")
    pages = layers.kv4_pages(1, 1, 64, 16)
    gpu = x.cuda()
    layers.kv4_append(gpu[:, 0], gpu[:, 1], pages, i32([0]).view(1, 1), i32([4]), cu=i32([0, 4]))
    got = torch.stack(layers.kv4_read(pages, i32([0]).view(1, 1), i32([4]), 64, cu=i32([0, 4]), tokens=4, dtype=dtype), 1).cpu()
    bad = torch.zeros(4, 2, 1, 2, dtype=torch.bool)
    bad[0, 0, 0, 0] = bad[1, 1, 0, 1] = bad[2, 0, 0, 0] = True
    assert torch.equal(torch.isnan(got), bad.repeat_interleave(32, -1))


def test_tokens_without_a_place_are_skipped(ext):
    """Page ids outside the pool, lengths below the new tokens or past the table, tokens outside cu: nothing else is touched."""
    dim, page = 64, 16
    pages = layers.kv4_pages(3, 2, dim, page)
    k = torch.randn(12, 2, dim, device="cuda").to(BF16)
    #                sequence 0: page outside; 1: only its last token has a position; 2: longer than its row; 3: below zero
    table, lengths = i32([-1, 7, 0, 0, 1, 2, 2, -2 ** 31]).view(4, 2), i32([20, 1, 1000, -5])
    layers.kv4_append(k, k, pages, table, lengths, cu=i32([1, 4, 6, 8, 10]))
    taken = {(0, 0): 5, (2, 14): 6, (2, 15): 7}  # (page, offset) <- token; sequence 2 counts as 32 positions
    got = torch.from_numpy(half_values(pages.cpu().numpy(), page, dim))
    for p in range(3):
        for offset in range(page):
            token = taken.get((p, offset))
            want = torch.zeros(2, dim) if token is None else \
                torch.from_numpy(mxfp4.dequantize(*mxfp4.quantize(k[token].float().cpu().numpy())))
            assert torch.equal(got[p, :, 0, offset], want.double()) and torch.equal(got[p, :, 1, offset], want.double()), (p, offset)
    out = torch.full((2, 12, 2, dim), 3.0, dtype=BF16, device="cuda")
    layers.kv4_read(pages, table, lengths, dim, cu=i32([1, 4, 6, 8, 10]), out=(out[0], out[1]))
    assert all((out[:, t] == 3).all() for t in range(12) if t not in taken.values())
    assert all((out[:, t] != 3).any() for t in taken.values())


# ---------------------------------------------------------------------------------------------
# attention


ATTEND = [
    # lengths, heads, kv heads, dim, page size
    ([1], 8, 8, 128, 16),
    ([0], 2, 1, 64, 16),
    ([0, 0, 5, 0], 10, 2, 128, 32),
    ([15, 16, 17, 31, 32, 33], 8, 1, 64, 16),
    ([127, 128, 129, 1, 0, 255, 256, 257], 16, 2, 128, 64),
    ([700], 16, 2, 128, 16),
    ([1000, 3, 0, 2049], 40, 8, 128, 128),
    ([513, 2], 32, 2, 64, 1024),   # 16 queries a head: a full tile
    ([90, 600], 34, 2, 128, 64),   # 17: a second tile of one
    ([300], 40, 1, 64, 32),        # 40 queries on one head
    ([20011], 5, 1, 128, 256),
    ([9, 30000, 700, 1], 4, 4, 64, 64),
    ([(37 * i) % 301 for i in range(150)], 4, 2, 128, 16),  # more sequences than lanes
    ([(53 * i) % 1500 for i in range(70)], 12, 12, 64, 32),
    ([(29 * i) % 900 for i in range(80)], 16, 4, 128, 64),  # heads that fill the chip: a workgroup each up to 1024 positions
    ([(29 * i) % 400 for i in range(66)], 33, 1, 64, 16),
]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("lengths,heads,kv_heads,dim,page_size", ATTEND)
def test_attention_against_64_bits(ext, lengths, heads, kv_heads, dim, page_size, dtype):
    cache = Cache(lengths, kv_heads, dim, page_size, len(lengths) + heads, dtype)
    q = torch.randn(len(lengths), heads, dim, generator=torch.Generator().manual_seed(heads)).to(dtype).cuda()
    got = layers.kv4_attention(q, cache.pages, cache.table, cache.lengths, dim ** -0.5)
    assert_within(got, *cache.attention(q, dim ** -0.5))
    assert all(not got[s].any() for s, n in enumerate(lengths) if n == 0)
    assert torch.equal(layers.kv4_attention(q, cache.pages, cache.table, cache.lengths, dim ** -0.5), got)  # the same bits again


@pytest.mark.parametrize("scale", [1.0, -0.7, 0.0])
@pytest.mark.parametrize("lengths,heads,kv_heads,dim", [([3000, 40], 8, 2, 128), ([5000], 4, 1, 64)])
def test_scores_that_grow_along_the_keys(ext, lengths, heads, kv_heads, dim, scale):
    """Running maxima that rise block after block, large, negative and zero scales, and pieces whose maxima differ widely."""
    cache = Cache(lengths, kv_heads, dim, 64, 1, spread=lambda n: np.linspace(0.05, 4, n, dtype=np.float32))
    q = (torch.randn(len(lengths), heads, dim, generator=torch.Generator().manual_seed(2)) * 0.5).to(BF16).cuda()
    assert_within(layers.kv4_attention(q, cache.pages, cache.table, cache.lengths, scale), *cache.attention(q, scale))


def test_small_probabilities_keep_their_weight_in_fp16(ext):
    """One key far above thousands of others whose probabilities, 2^-20 of its own, make up the rest of the sum."""
    n, dim = 8192, 64
    pages = layers.kv4_pages(n // 64, 1, dim, 64)
    k, v = torch.zeros(n, 1, dim), torch.ones(n, 1, dim)
    k[0], v[0] = 1.0, -1.0  # q . k = 64 * q: exp(13.86) above the others' 0
    table, lengths, cu = i32(range(n // 64)).view(1, -1), i32([n]), i32([0, n])
    layers.kv4_append(k.half().cuda(), v.half().cuda(), pages, table, lengths, cu=cu)
    q = torch.full((1, 1, dim), math.log(2 ** 20) / dim * 8).half().cuda()
    p = math.exp(float(q[0, 0, 0]) / 8 * dim)
    want = (n - 1 - p) / (n - 1 + p)
    got = layers.kv4_attention(q, pages, table, lengths, 1 / 8)
    # want is about -0.98: the rest weighs 2^-7; half a step of it, and twice that of the probabilities' rounding
    assert float((got.double() - want).abs().max()) <= 3.5 * 2.0 ** -11 * abs(want)


def test_strided_queries_outputs_and_tables(ext):
    lengths, heads, kv_heads, dim = [100, 0, 333], 6, 2, 128
    cache = Cache(lengths, kv_heads, dim, 32, 4)
    q = torch.randn(3, heads, dim).to(BF16).cuda()
    want = layers.kv4_attention(q, cache.pages, cache.table, cache.lengths, 0.1)
    wide = torch.randn(3, heads + 2 * kv_heads, dim + 8).to(BF16).cuda()
    view = wide[:, 1:1 + heads, 8:]
    view.copy_(q)
    out = torch.full((3, 2 * heads, dim + 4), 9.0, dtype=BF16, device="cuda")
    table = torch.full((3, cache.table.shape[1] + 5), 2 ** 30, dtype=torch.int32, device="cuda")
    table[:, 3:3 + cache.table.shape[1]] = cache.table
    got = layers.kv4_attention(view, cache.pages, table[:, 3:], cache.lengths, 0.1, out=out[:, ::2, 4:])
    assert torch.equal(got, want) and (out[:, 1::2] == 9).all() and (out[..., :4] == 9).all()
    shared = cache.table[2:].expand(3, -1)  # one table row for all sequences
    same = layers.kv4_attention(q, cache.pages, shared, i32([333, 333, 333]), 0.1)
    assert torch.equal(same[2], want[2])


@pytest.mark.parametrize("heads", [1, 3])
def test_strides_of_dimensions_of_one(ext, heads):
    """One sequence, one head: whatever stride the tensor names there, in every call."""
    cache = Cache([77], 1, 64, 16, 5, extra_columns=0)
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(1, h, 64, generator=g).to(BF16).cuda() for h in (heads, 1, 1))

    def odd(t):
        return t.as_strided(t.shape, [s if n > 1 else o for n, s, o in zip(t.shape, t.stride(), (3, 5, 1))])

    pages = cache.pages.clone()
    layers.kv4_append(k, v, cache.pages, cache.table, cache.lengths)
    layers.kv4_append(odd(k), odd(v), pages, cache.table.as_strided(cache.table.shape, (7, 1)), cache.lengths)
    assert torch.equal(pages, cache.pages)
    want, rows = layers.kv4_attention(q, pages, cache.table, cache.lengths, 0.1), layers.kv4_read(pages, cache.table, cache.lengths, 64)
    out, back = torch.zeros_like(q), [torch.zeros_like(k) for _ in range(2)]
    layers.kv4_attention(odd(q), pages, cache.table, cache.lengths, 0.1, out=odd(out))
    layers.kv4_read(pages, cache.table, cache.lengths, 64, out=tuple(odd(t) for t in back))
    assert torch.equal(out, want) and want.any() and torch.equal(torch.stack(back), torch.stack(rows)) and back[0].any()


def test_pages_outside_the_pool_take_no_part(ext):
    """Unknown page ids are skipped wherever they occur, and lengths past the table or below zero are cut to it."""
    page, dim = 32, 64
    cache = Cache([160, 64, 96, 40], 1, dim, page, 6, extra_columns=0)
    q = torch.randn(4, 3, dim).to(BF16).cuda()
    table = cache.table.clone()
    table[0, 1], table[0, 3] = -1, 10 ** 6       # sequence 0 loses positions 32..63 and 96..127
    table[1, :2] = -7                            # sequence 1 has nothing left
    lengths = i32([160, 64, 10 ** 9, -3])        # sequence 2: the whole row, whose last columns are -1
    got = layers.kv4_attention(q, cache.pages, table, lengths, 0.2)
    kept = torch.cat([cache.values[0][:, :, a:b] for a, b in ((0, 32), (64, 96), (128, 160))], dim=2)
    cache.values[0] = kept
    cache.lengths_host[:] = [96, 0, 96, 0]
    want, bound = cache.attention(q, 0.2)
    assert_within(got[[0, 1, 2, 3]], want, bound)
    assert not got[1].any() and not got[3].any()


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_a_nan_reaches_its_own_sequence_and_head_alone(ext, dtype):
    lengths = [300, 900, 40]
    cache = Cache(lengths, 2, 128, 64, 8, dtype)
    q = torch.randn(3, 4, 128).to(dtype).cuda()
    want = layers.kv4_attention(q, cache.pages, cache.table, cache.lengths, 0.1)
    page = int(cache.table[1, 10])  # positions 640 .. 703
    cache.pages[page, 0, 0, 64 * 64 + 5 * 4] = 255       # a key's first group, head 0
    cache.pages[page, 1, 1, 64 * 64 + 63 * 4 + 3] = 255  # a value's last group, head 1
    got = layers.kv4_attention(q, cache.pages, cache.table, cache.lengths, 0.1)
    assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])
    assert torch.isnan(got[1, :2]).all() and torch.isnan(got[1, 2:, 96:]).all() and torch.equal(got[1, 2:, :96], want[1, 2:, :96])


@pytest.mark.parametrize("lengths,heads,kv_heads,dim,page", [([30, 7, 0, 90], 8, 2, 64, 16), ([700, 1, 0, 1024], 16, 2, 128, 64),
                                                             ([20000, 40, 0, 3000], 5, 1, 128, 128), ([3000, 8, 0, 9000], 8, 2, 64, 32)])
def test_scores_of_minus_infinity(ext, lengths, heads, kv_heads, dim, page):
    """Two thirds of sequence 0's positions and all of sequence 1's score -infinity for KV head 0: the first is what its other positions make
    it, the second has no softmax and gets NaN, the others and a sequence without any position in the pool are what they were."""
    sequences, scale, group = len(lengths), dim ** -0.5, heads // kv_heads
    g = torch.Generator().manual_seed(31)
    x = torch.randn(sum(lengths), 2, kv_heads, dim, generator=g).to(BF16)
    starts, struck = [sum(lengths[:s]) for s in range(sequences)], lengths[0] * 2 // 3
    low = torch.zeros(32)
    low[3] = -2.0 ** 100
    x[:lengths[0], 0, 0, :32] = 0   # these and the query's 2^100 make 0 or -2^200
    x[:struck, 0, 0, :32] = low.to(BF16)
    x[starts[1]:starts[2], 0, 0, :32] = low.to(BF16)
    q = torch.randn(sequences, heads, dim, generator=g).to(BF16)
    q[:2, :group, 3] = 2.0 ** 100
    counts = [-(-n // page) for n in lengths]
    table = torch.full((sequences + 1, max(counts)), -1, dtype=torch.int32)
    for s, n in enumerate(counts):
        table[s, :n] = torch.arange(sum(counts[:s]), sum(counts[:s]) + n)
    pages, table, positions = layers.kv4_pages(sum(counts), kv_heads, dim, page), table.cuda(), i32([*lengths, 50])
    gpu = x.cuda()
    layers.kv4_append(gpu[:, 0], gpu[:, 1], pages, table[:-1], positions[:-1], cu=cumulative(lengths))
    q = torch.cat([q, q[:1]]).cuda()  # the last sequence has positions, but no page
    got = layers.kv4_attention(q, pages, table, positions, scale)
    values = torch.from_numpy(mxfp4.dequantize(*mxfp4.quantize(x.float().numpy()))).cuda()
    for s, n in enumerate(lengths):
        for h in range(heads):
            first = struck if s == 0 and h < group else 0
            if s == 1 and h < group:
                assert torch.isnan(got[s, h]).all()
                continue
            seen = slice(starts[s] + first, starts[s] + n)
            k, v = values[seen, 0, h // group], values[seen, 1, h // group]
            query = q[s, h][None]
            if s == 0 and h < group:
                query = query.clone()
                query[:, :32] = 0  # as these keys are
            assert_within(got[s, h][None], *attention64(query, k, v, scale, n - first - 1))
    assert not got[sequences].any()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("lengths,heads,kv_heads,dim,page", [([30, 7, 0, 90], 8, 2, 64, 16), ([700, 1, 0, 1024], 16, 2, 128, 64),
                                                             ([20000, 40, 0, 3000], 5, 1, 128, 128), ([3000, 8, 0, 9000], 8, 2, 64, 32)])
def test_the_largest_values(ext, lengths, heads, kv_heads, dim, page, dtype):
    """Values of the largest magnitude that a cache of the type holds, all of one sign or of both, give finite averages."""
    g = torch.Generator().manual_seed(37)
    x = torch.randn(sum(lengths), 2, kv_heads, dim, generator=g).to(dtype)
    largest = 6 * 2.0 ** (125 if dtype == BF16 else 13)
    x[:, 1] = torch.where(x[:, 1] > 0, largest, -largest)
    x[:, 1, :, dim // 2:] = largest
    counts = [-(-n // page) for n in lengths]
    table = torch.full((len(lengths), max(counts)), -1, dtype=torch.int32)
    for s, n in enumerate(counts):
        table[s, :n] = torch.arange(sum(counts[:s]), sum(counts[:s]) + n)
    pages, table, gpu = layers.kv4_pages(sum(counts), kv_heads, dim, page), table.cuda(), x.cuda()
    layers.kv4_append(gpu[:, 0], gpu[:, 1], pages, table, i32(lengths), cu=cumulative(lengths))
    q = torch.randn(len(lengths), heads, dim, generator=g).to(dtype).cuda()
    got = layers.kv4_attention(q, pages, table, i32(lengths), dim ** -0.5)
    values = torch.from_numpy(mxfp4.dequantize(*mxfp4.quantize(x.float().numpy()))).cuda()
    assert torch.equal(values[:, 1].cpu(), x[:, 1].double())
    for s, n in enumerate(lengths):
        for h in range(heads):
            k, v = (values[sum(lengths[:s]):sum(lengths[:s + 1]), i, h // (heads // kv_heads)] for i in (0, 1))
            assert_within(got[s, h][None], *attention64(q[s, h][None], k, v, dim ** -0.5, n - 1))


def test_workspace_is_of_the_stated_size_and_needs_no_clearing(ext):
    cache = Cache([5000, 17, 900], 2, 128, 64, 9)
    q = torch.randn(3, 10, 128).to(BF16).cuda()
    size = layers.kv4_attention_workspace_bytes(cache.pages, cache.table, 10, 128)
    guarded = torch.full((size + 512,), 255, dtype=torch.uint8, device="cuda")  # NaN wherever it is read unwritten
    want = layers.kv4_attention(q, cache.pages, cache.table, cache.lengths, 0.1)
    assert torch.equal(layers.kv4_attention(q, cache.pages, cache.table, cache.lengths, 0.1, workspace=guarded[256:256 + size]), want)
    assert (guarded[:256] == 255).all() and (guarded[256 + size:] == 255).all()
    with pytest.raises(_lib.TexelatorError, match="too small"):
        layers.kv4_attention(q, cache.pages, cache.table, cache.lengths, 0.1, workspace=guarded[:size - 16])


def test_a_captured_step_serves_the_lengths_of_each_replay(ext):
    """Append and attention captured once; every replay finds the lengths, tables and rows of its time, with eager work
    between; a second graph shares the workspace on the same stream."""
    kv_heads, heads, dim, page = 2, 8, 128, 16
    cache = Cache([30, 0, 500, 127], kv_heads, dim, page, 11, extra_columns=8, spare=40)
    free = iter(sorted(set(range(cache.pages.shape[0])) - set(cache.table.flatten().tolist())))
    for s, n in enumerate([30, 0, 500, 127]):
        for column in range(-(-n // page), -(-n // page) + 3):
            cache.table[s, column] = next(free)
    q, k, v = (torch.zeros(4, h, dim, dtype=BF16, device="cuda") for h in (heads, kv_heads, kv_heads))
    size = layers.kv4_attention_workspace_bytes(cache.pages, cache.table, heads, dim)
    workspace = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    outs = [torch.zeros_like(q) for _ in range(2)]

    def step(out, scale):
        layers.kv4_append(k, v, cache.pages, cache.table, cache.lengths)
        layers.kv4_attention(q, cache.pages, cache.table, cache.lengths, scale, workspace=workspace, out=out)

    saved = cache.pages.clone()
    stream = torch.cuda.Stream()
    graphs = []
    with torch.cuda.stream(stream):
        for out, scale in zip(outs, (0.09, 0.05)):
            step(out, scale)
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                step(out, scale)
            graphs.append(graph)
        cache.pages.copy_(saved)
        for turn in range(20):
            cache.lengths += 1
            for t, h in ((q, heads), (k, kv_heads), (v, kv_heads)):
                t.copy_(torch.randn(4, h, dim, generator=torch.Generator().manual_seed(turn)))
            for graph, out, scale in zip(graphs, outs, (0.09, 0.05)):
                graph.replay()
                stream.synchronize()
                want = layers.kv4_attention(q, cache.pages, cache.table, cache.lengths, scale)
                got_k, got_v = layers.kv4_read(cache.pages, cache.table, cache.lengths, dim)
                assert torch.equal(out, want), turn
                expected = torch.from_numpy(mxfp4.dequantize(*mxfp4.quantize(torch.stack([k, v]).float().cpu().numpy())))
                assert torch.equal(torch.stack([got_k, got_v]).cpu().double(), expected)


def test_two_streams_at_once(ext):
    """Calls on two streams, each with its own workspace, give the bits of calls one after the other."""
    caches = [Cache([4000, 100], 2, 128, 64, 12), Cache([900, 2500, 3], 4, 64, 32, 13)]
    qs = [torch.randn(2, 8, 128).to(BF16).cuda(), torch.randn(3, 8, 64).to(BF16).cuda()]
    want = [layers.kv4_attention(q, c.pages, c.table, c.lengths, 0.1) for q, c in zip(qs, caches)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(10):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(layers.kv4_attention(qs[i], caches[i].pages, caches[i].table, caches[i].lengths, 0.1))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])


def test_pages_past_four_gib(ext):
    """Offsets of pages, of tokens' rows and of table rows beyond 32 bits."""
    page, dim, kv_heads = 1024, 128, 8
    pages = torch.zeros(4000, kv_heads, 2, page * dim * 17 // 32, dtype=torch.uint8, device="cuda")  # 4.4 GB
    assert pages.numel() > 2 ** 32
    ids = [3999, 0, 3950]
    table = i32(ids).view(1, 3)
    x = torch.randn(2500, 2, kv_heads, dim, generator=torch.Generator().manual_seed(1)).to(BF16).cuda()
    lengths, cu = i32([2500]), i32([0, 2500])
    layers.kv4_append(x[:, 0], x[:, 1], pages, table, lengths, cu=cu)
    k, v = layers.kv4_read(pages, table, lengths, dim, cu=cu, tokens=2500)
    values = torch.from_numpy(mxfp4.dequantize(*mxfp4.quantize(x.float().cpu().numpy())))
    assert torch.equal(torch.stack([k, v], 1).cpu().double(), values)
    small = layers.kv4_pages(3, kv_heads, dim, page)
    small.copy_(pages[ids])
    q = torch.randn(1, 16, dim).to(BF16).cuda()
    want = layers.kv4_attention(q, small, i32([0, 1, 2]).view(1, 3), lengths, 0.09)
    assert torch.equal(layers.kv4_attention(q, pages, table, lengths, 0.09), want) and want.any()
    layers.kv4_copy_pages(pages, [3999], [3998])
    assert torch.equal(pages[3998], pages[3999]) and not pages[3997].any()


# ---------------------------------------------------------------------------------------------
# pages


@pytest.mark.parametrize("layer_count,num_pages,kv_heads,dim,page,copies", [
    (None, 2, 1, 64, 16, 1), (3, 9, 2, 128, 64, 4), (1, 1000, 1, 64, 16, 500), (5, 40, 3, 128, 16, 20), (2, 7, 1, 128, 1024, 3)])
def test_copies_of_pages(ext, layer_count, num_pages, kv_heads, dim, page, copies):
    """Every byte, in every layer, of the pages named and of no others; more pairs than one launch takes among the cases."""
    rng = np.random.default_rng(copies)
    pages = layers.kv4_pages(num_pages, kv_heads, dim, page, layers=layer_count)
    pages.copy_(torch.from_numpy(rng.integers(0, 256, size=tuple(pages.shape), dtype=np.uint8)))
    chosen = rng.permutation(num_pages)
    src, dst = chosen[:copies].tolist(), chosen[copies:2 * copies].tolist()
    want = pages.cpu().clone()
    at = want if layer_count else want[None]
    at[:, dst] = at[:, src]
    layers.kv4_copy_pages(pages, src, dst)
    assert torch.equal(pages.cpu(), want)
    if copies > 1:  # one page to many
        layers.kv4_copy_pages(pages, [src[0]] * copies, dst)
        at[:, dst] = at[:, src[:1] * copies]
        assert torch.equal(pages.cpu(), want)
    with pytest.raises(_lib.TexelatorError, match="outside"):
        layers.kv4_copy_pages(pages, [0], [num_pages])
    with pytest.raises(_lib.TexelatorError, match="as many"):
        layers.kv4_copy_pages(pages, [0, 1], [1])
    with pytest.raises(_lib.TexelatorError, match="integers"):
        layers.kv4_copy_pages(pages, [0.5], [1])
    with pytest.raises(_lib.TexelatorError, match="integers"):
        layers.kv4_copy_pages(pages, bytes(8), bytes(range(8)))
    layers.kv4_copy_pages(pages, np.array([src[0]]), torch.tensor([dst[0]]))  # integers of other kinds
    assert torch.equal(pages.cpu(), want)


def test_wrong_tensors_are_refused(ext):
    pages = layers.kv4_pages(4, 2, 64, 16)
    table, lengths = torch.zeros(3, 2, dtype=torch.int32, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda")
    k = torch.zeros(3, 2, 64, dtype=BF16, device="cuda")
    q = torch.zeros(3, 6, 64, dtype=BF16, device="cuda")
    wide = torch.zeros(3, 2, 128, dtype=BF16, device="cuda")
    bad_append = [(k[:2], k, None), (k, k.half(), None), (k, k[:, :1], None), (wide, wide, None), (k.float(), k.float(), None),
                  (k[0, 0, 0], k[0, 0, 0], None), (k, k, i32([0, 3])), (k, k, i32([0, 1, 2, 3]).long()), (wide[:, :, ::2], k, None), (wide[:, :, 4:68], k, None)]
    for a, b, cu in bad_append:
        with pytest.raises(_lib.TexelatorError):
            layers.kv4_append(a, b, pages, table, lengths, cu=cu)
    bad_cache = [(pages.short(), table, lengths), (pages[:, :, :1], table, lengths), (pages[:, :1], table, lengths), (pages[0], table, lengths),
                 (pages, table.long(), lengths), (pages, table[0], lengths), (pages, table.t(), lengths), (pages, table[:, :0], lengths),
                 (pages, table, lengths.long()), (pages, table, lengths[:2]), (pages, table.cpu(), lengths), (pages, table, lengths.cpu())]
    for cache in bad_cache:
        with pytest.raises(_lib.TexelatorError):
            layers.kv4_attention(q, *cache, 1.0)
        with pytest.raises(_lib.TexelatorError):
            layers.kv4_read(*cache, 64)
    for a in (q[:2], q[:, :5], q.float(), wide, q.cpu(), q.transpose(1, 2)):
        with pytest.raises(_lib.TexelatorError):
            layers.kv4_attention(a, pages, table, lengths, 1.0)
    with pytest.raises(_lib.TexelatorError):
        layers.kv4_attention(q, pages, table, lengths, 1.0, out=q[:, :4])
    with pytest.raises(_lib.TexelatorError, match="tokens"):
        layers.kv4_read(pages, table, lengths, 64, cu=i32([0, 1, 2, 3]))
    with pytest.raises(_lib.TexelatorError):
        layers.kv4_read(pages, table, lengths, 64, dtype=torch.float32)
    empty = layers.kv4_attention(q[:0], pages, table[:0], lengths[:0], 1.0)
    assert empty.shape == (0, 6, 64)
    layers.kv4_append(k[:0], k[:0], pages, table[:0], lengths[:0])
    assert layers.kv4_read(pages, table[:0], lengths[:0], 64)[0].shape == (0, 2, 64) and not pages.any()
