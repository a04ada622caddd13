"""The operators of a drafted step: rotation on the way into the cache, attention of trees, verification, and the move of the
accepted rows; each against 64 bits or to the bit."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import mxfp4
from tests.drafts import Trees, masked_attention64, quantise64, random_parents, rounded64, seen_rows, turned64, verify64
from tests.serving import HALF_STEP, Cache, assert_within, cumulative, half_values, i32
from tests.test_gpu_kv4 import place, rows
from texelator_amd import _lib, layers

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def rope_tables(count, rotary, seed=0, scale=1.0):
    frequency = 1e6 ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)
    angles = torch.arange(count, dtype=torch.float64)[:, None] * frequency
    return (scale * angles.cos()).float().cuda(), (scale * angles.sin()).float().cuda()


# ---------------------------------------------------------------------------------------------
# rotation and storage

ROPE = [
    # lengths after the call, new tokens, heads, kv heads, dim, page size, rotary, interleaved, positions given
    ([1], None, 1, 1, 64, 16, 64, False, False),
    ([5, 700, 16, 33], None, 16, 2, 128, 16, 128, False, False),
    ([5, 700, 16, 33], None, 6, 3, 128, 16, 128, True, True),
    ([17, 16, 0, 256, 257], [17, 1, 0, 100, 64], 5, 1, 64, 32, 32, False, True),
    ([1000, 40], [999, 7], 4, 4, 128, 1024, 48, False, False),
    ([1000, 40], [999, 7], 3, 3, 64, 64, 16, True, True),
    ([64, 300], [64, 3], 7, 7, 128, 64, 112, False, True),
    (list(range(1, 101)), [1 + n // 3 for n in range(1, 101)], 2, 2, 128, 16, 64, True, False),
    ([2] * 2500, [n % 3 for n in range(2500)], 2, 1, 64, 16, 64, False, False),  # more sequences than the search holds in LDS
    # several heads a workgroup, queries, keys and values among them
    ([2000, 1300], [1999, 1200], 30, 5, 128, 64, 128, False, True),
    ([3000, 900, 2500], [2999, 800, 2400], 40, 8, 64, 256, 48, True, False),
]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("lengths,new,heads,kv_heads,dim,page_size,rotary,interleaved,given", ROPE)
def test_rotated_rows(ext, lengths, new, heads, kv_heads, dim, page_size, rotary, interleaved, given, dtype):
    """Cache bytes as the exact rotation quantizes, to the bit, wherever tokens go and nowhere else; queries and key rows within their
    roundings; q, k and v as columns of one buffer, rows behind the last sequence untouched."""
    counts = new if new is not None else [1] * len(lengths)
    table, where, total = place(lengths, counts, page_size, len(lengths))
    tokens, behind = sum(counts), 3 if new is not None else 0
    g = torch.Generator().manual_seed(tokens)
    kv = rows(tokens, kv_heads, dim, dtype, tokens).float().clamp(-1e4, 1e4).to(dtype)
    qkv = torch.cat([torch.randn(tokens, heads, dim, generator=g).to(dtype), kv[:, 0], kv[:, 1]], dim=1)
    qkv = torch.cat([qkv, torch.full((behind, *qkv.shape[1:]), float("nan"), dtype=dtype)]).cuda()
    q, k, v = qkv.split([heads, kv_heads, kv_heads], dim=1)
    places = [n - c + i for n, c in zip(lengths, counts) for i in range(c)]
    positions = [(7 * p + 3) % 5000 for p in places] if given else places
    cos, sin = rope_tables(max(positions) + 1, rotary, scale=1.1 if given else 1.0)
    half = page_size * dim * 17 // 32
    before = np.random.default_rng(5).integers(0, 256, size=(total, kv_heads, 2, half), dtype=np.uint8)
    pages, cu = torch.from_numpy(before.copy()).cuda(), cumulative(counts) if new is not None else None
    out = torch.full((tokens + behind, heads, dim), 7.0, dtype=dtype, device="cuda")
    k_out = torch.full((tokens + behind, kv_heads, dim), 7.0, dtype=dtype, device="cuda")
    at = i32(positions + [0] * behind) if given else None
    got = layers.kv4_append_rope(q, k, v, cos, sin, pages, table, i32(lengths), cu=cu, positions=at, interleaved=interleaved, out=out,
                                 k_out=k_out)
    assert got is out and (out[tokens:] == 7).all() and (k_out[tokens:] == 7).all()
    c, s = cos[positions].cpu(), sin[positions].cpu()
    exact_k = turned64(k[:tokens].cpu(), c, s, interleaved)
    want = before.copy()
    codes, exponents = quantise64(torch.stack([exact_k, v[:tokens].cpu().double()], dim=1).numpy())
    packed, split = mxfp4.pack(codes), page_size * dim // 2
    for t, (page, offset) in enumerate(where):
        part = want[page, :, :, :split].reshape(kv_heads, 2, page_size, dim // 2)
        part[:, :, offset] = packed[t].transpose(1, 0, 2)
        want[page, :, :, :split] = part.reshape(kv_heads, 2, -1)
        part = want[page, :, :, split:].reshape(kv_heads, 2, page_size, dim // 32)
        part[:, :, offset] = exponents[t].transpose(1, 0, 2)
        want[page, :, :, split:] = part.reshape(kv_heads, 2, -1)
    assert np.array_equal(pages.cpu().numpy(), want)
    assert torch.equal(k_out[:tokens].cpu().double(), rounded64(exact_k, dtype))  # one rounding, of the exact value
    # q: two products and their sum in 32 bits, then the type: (|a cos| + |b sin|) times 2 * 2^-24 and half a step of the result
    x = q[:tokens].cpu()
    exact_q = turned64(x, c, s, interleaved)
    spread = turned64(x.abs().double(), c.abs(), -s.abs(), interleaved).abs() + turned64(x.abs().double(), c.abs(), s.abs(), interleaved).abs()
    error = (out[:tokens].cpu().double() - exact_q).abs()
    tiny = float(torch.finfo(dtype).smallest_normal) * float(torch.finfo(dtype).eps) / 2
    assert (error <= HALF_STEP[dtype] * exact_q.abs() + 2 * 2.0 ** -24 * (1 + HALF_STEP[dtype]) * spread + tiny).all()
    fresh = layers.kv4_append_rope(q[:tokens], k[:tokens], v[:tokens], cos, sin, pages, table, i32(lengths), cu=cu,
                                   positions=None if at is None else at[:tokens], interleaved=interleaved)
    assert torch.equal(fresh, out[:tokens]) and np.array_equal(pages.cpu().numpy(), want)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_angle_zero_stores_what_append_stores(ext, dtype, interleaved):
    """Cosines of one and sines of zero: the bytes of kv4_append, at the type's borders too, and the queries' own bits."""
    x = rows(40, 2, 128, dtype, 3).cuda()
    cos, sin = torch.ones(50, 64, device="cuda"), torch.zeros(50, 64, device="cuda")
    table, lengths, cu = i32([2, 0, 1, 3]).view(2, 2), i32([20, 30]), i32([0, 15, 40])
    pages, want = layers.kv4_pages(4, 2, 128, 16), layers.kv4_pages(4, 2, 128, 16)
    layers.kv4_append(x[:, 0], x[:, 1], want, table, lengths, cu=cu)
    q = torch.randn(40, 3, 128, device="cuda").to(dtype)
    got = layers.kv4_append_rope(q, x[:, 0], x[:, 1], cos, sin, pages, table, lengths, cu=cu, interleaved=interleaved)
    assert torch.equal(pages, want) and torch.equal(got, q)


def test_slow_pairs_next_to_a_tie(ext):
    """Keys midway between two codes, turned by angles far below 2^-24: the exact value is off the middle, and decides."""
    k = torch.tensor([4.0, 5.0, 2.5, 3.5, 0.25, 0.75, 1.25, 1.75] * 4).repeat(2).view(1, 1, 64)  # scale 1, from the 4
    k[..., 32:] = torch.tensor([1.0, -1.0] * 16)
    cos, sin = torch.ones(2, 32, device="cuda"), torch.full((2, 32), 1e-9, device="cuda")
    for dtype in (BF16, FP16):
        x = k.to(dtype).cuda()
        pages = layers.kv4_pages(1, 1, 64, 16)
        layers.kv4_append_rope(x, x, x, cos, sin, pages, i32([0]).view(1, 1), i32([1]))
        codes, exponents = quantise64(turned64(x.cpu(), cos[:1].cpu(), sin[:1].cpu(), False).numpy())
        got = half_values(pages.cpu().numpy(), 16, 64)[0, 0, 0, 0]
        want = mxfp4.dequantize(codes, exponents)[0, 0]
        assert np.array_equal(got, want)
        plain = mxfp4.dequantize(*mxfp4.quantize(k.float().numpy()))[0, 0]
        assert not np.array_equal(want, plain)  # a rounding to 32 bits on the way would have stored these


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_what_is_not_finite_and_positions_without_a_row(ext, dtype):
    """A NaN or an infinity reaches its pair and, stored, its group; a position outside the tables turns to NaN; no page: q is
    turned all the same."""
    x = torch.randn(5, 3, 64, generator=torch.Generator().manual_seed(1)).to(dtype)
    x[1, 1, 3], x[1, 2, 40] = float("inf"), float("nan")
    gpu = x.cuda()
    q, k, v = gpu[:, :1], gpu[:, 1:2], gpu[:, 2:]
    cos, sin = rope_tables(10, 32)
    pages = layers.kv4_pages(2, 1, 64, 16)
    table, lengths = i32([0, 1, -1, 7]).view(2, 2), i32([4, 17])  # sequence 1's only token lies in no page
    at = i32([2, 9, 10, -1, 5])
    got = layers.kv4_append_rope(q, k, v, cos, sin, pages, table, lengths, cu=i32([0, 4, 5]), positions=at)
    turned = torch.isnan(got[:, 0]).cpu()
    assert not turned[[0, 1, 4]].any() and turned[2:4, :32].all() and not turned[2:4, 32:].any()
    assert torch.equal(got[2:4, 0, 32:], q[2:4, 0, 32:])
    values = half_values(pages.cpu().numpy(), 16, 64)[0, 0]
    nan = np.isnan(values)
    assert nan[0, 1, :32].all() and not nan[0, 1, 32:].any() and nan[1, 1, 32:].all() and not nan[1, 1, :32].any()  # k, v of token 1
    assert nan[0, 2:4, :32].all() and not nan[0, 2:4, 32:].any() and not nan[1, [0, 2, 3]].any() and not nan[0, 0].any()
    assert not pages[1].any()
    huge = torch.full((1, 1, 64), torch.finfo(dtype).max, dtype=dtype, device="cuda")
    layers.kv4_append_rope(huge, huge, huge, cos * 1e30, sin * 1e30, pages, table[:1], i32([1]))
    assert np.isnan(half_values(pages.cpu().numpy(), 16, 64)[0, 0, 0, 0, :32]).all() == (dtype == BF16)


def test_tables_as_columns_and_other_strides(ext):
    """Tables whose rows are parts of wider ones, expanded rows, strided outputs."""
    tokens, heads, kv_heads, dim = 9, 4, 2, 128
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(tokens, h, dim, generator=g).to(BF16).cuda() for h in (heads, kv_heads, kv_heads))
    cos, sin = rope_tables(40, dim)
    pages, other = layers.kv4_pages(2, kv_heads, dim, 16), layers.kv4_pages(2, kv_heads, dim, 16)
    table, lengths, cu = i32([0, 1]).view(1, 2), i32([30]), i32([0, tokens])
    want = layers.kv4_append_rope(q, k, v, cos, sin, pages, table, lengths, cu=cu)
    wide = torch.cat([cos, cos], dim=1), torch.cat([sin, sin], dim=1)
    out = torch.full((tokens, 2 * heads, dim + 8), 9.0, dtype=BF16, device="cuda")
    both = torch.cat([q, k], dim=1).transpose(0, 1).contiguous().transpose(0, 1)  # heads outermost
    got = layers.kv4_append_rope(both[:, :heads], both[:, heads:], v, wide[0][:, :64], wide[1][:, 64:], other, table, lengths, cu=cu,
                                 out=out[:, ::2, 8:])
    assert torch.equal(got, want) and torch.equal(other, pages) and (out[:, 1::2] == 9).all() and (out[..., :8] == 9).all()
    one = layers.kv4_append_rope(q, k, v, cos[5:6].expand(40, -1), sin[5:6].expand(40, -1), other, table, lengths, cu=cu)
    same = layers.kv4_append_rope(q, k, v, cos, sin, pages, table, lengths, cu=cu, positions=i32([5] * tokens))
    assert torch.equal(one, same) and torch.equal(other, pages)
    with pytest.raises(_lib.TexelatorError, match="overlap"):
        layers.kv4_append_rope(q, k, v, cos, sin, pages, table, lengths, cu=cu, out=q)


# ---------------------------------------------------------------------------------------------
# attention of trees

TREES = [
    # lengths, rows, heads, kv heads, dim, page size, chain
    ([1], [1], 8, 8, 128, 16, False),
    ([6], [6], 16, 2, 128, 16, False),
    ([700], [6], 16, 2, 128, 16, False),
    ([700], [64], 16, 2, 128, 32, True),
    ([90, 0, 33, 600], [5, 0, 33, 17], 10, 2, 64, 16, False),
    ([127, 128, 129, 1, 65, 255, 256, 257], [2, 3, 4, 1, 64, 10, 12, 7], 40, 8, 128, 64, False),
    ([127, 128, 129, 1, 65, 255, 256, 257], [2, 3, 4, 1, 64, 10, 12, 7], 4, 4, 64, 64, True),
    ([1000, 3, 9, 2049], [26, 3, 9, 1], 40, 8, 128, 128, False),
    ([513, 200], [64, 63], 34, 2, 64, 1024, False),   # 17 queries a row: 34 blocks
    ([300], [64], 40, 1, 64, 32, False),
    ([20011], [16], 5, 1, 128, 256, True),
    ([9, 30000, 700, 1], [9, 2, 64, 1], 4, 4, 64, 64, False),
    ([4 + (37 * i) % 301 for i in range(150)], [1 + i % 4 for i in range(150)], 4, 2, 128, 16, False),  # more sequences than lanes
    ([70 + (53 * i) % 1500 for i in range(70)], [i % 65 for i in range(70)], 12, 12, 64, 32, False),
    ([3, 2, 1], [5, 2, 7], 8, 2, 128, 16, False),     # fewer positions than rows
    # hundreds of queries a row
    ([90, 40], [3, 1], 300, 1, 64, 16, False),
    ([2000], [2], 601, 1, 128, 64, False),
    # as many short (sequence, head)s as fill the grid by themselves
    ([20 + (37 * i) % 300 for i in range(80)], [1 + i % 20 for i in range(80)], 24, 8, 128, 16, False),
    ([64 + (41 * i) % 200 for i in range(40)], [64 - i % 7 for i in range(40)], 32, 16, 64, 32, True),
    # long sequences among and behind the 64th
    ([30 + i for i in range(63)] + [20000, 40, 6000, 9], [1 + i % 3 for i in range(63)] + [40, 2, 7, 9], 4, 2, 128, 64, False),
]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("lengths,rows,heads,kv_heads,dim,page_size,chain", TREES)
def test_trees_against_64_bits(ext, lengths, rows, heads, kv_heads, dim, page_size, chain, dtype):
    trees = Trees(lengths, rows, kv_heads, dim, page_size, len(lengths) + heads, dtype, chain)
    q = torch.randn(sum(rows), heads, dim, generator=torch.Generator().manual_seed(heads)).to(dtype).cuda()

    def run():
        return layers.kv4_tree_attention(q, trees.pages, trees.table, trees.lengths, trees.cu, dim ** -0.5, parents=trees.parents)

    got = run()
    assert_within(got, *trees.tree_attention(q, dim ** -0.5))
    assert torch.equal(run(), got)  # the same bits again


@pytest.mark.parametrize("dim", [64, 128])
def test_tables_with_room_for_a_billion_positions(ext, dim):
    """Room for far more work than there is: a table of 2^20 pages of 1,024 positions, 64 queries a row and KV head."""
    lengths, rows = [20011, 900, 64, 1, 5000, 33], [16, 64, 3, 1, 40, 33]
    trees = Trees(lengths, rows, 2, dim, 1024, 11)
    table = torch.full((len(rows), 1 << 20), -1, dtype=torch.int32, device="cuda")
    table[:, :trees.table.shape[1]] = trees.table
    q = torch.randn(sum(rows), 128, dim, generator=torch.Generator().manual_seed(1)).to(BF16).cuda()

    def run():
        return layers.kv4_tree_attention(q, trees.pages, table, trees.lengths, trees.cu, dim ** -0.5, parents=trees.parents)

    got = run()
    assert_within(got, *trees.tree_attention(q, dim ** -0.5))
    assert torch.equal(run(), got)


def test_a_row_alone_is_single_token_attention(ext):
    """One row a sequence: within both calls' roundings of kv4_attention."""
    cache = Cache([700, 1, 9000, 33], 2, 128, 64, 3)
    q = torch.randn(4, 16, 128, generator=torch.Generator().manual_seed(1)).to(BF16).cuda()
    want, bound = cache.attention(q, 0.09)
    got = layers.kv4_tree_attention(q, cache.pages, cache.table, cache.lengths, i32(range(5)), 0.09)
    assert_within(got, want, bound)
    assert_within(layers.kv4_attention(q, cache.pages, cache.table, cache.lengths, 0.09), want, bound)


@pytest.mark.parametrize("scale", [1.0, -0.7, 0.0])
@pytest.mark.parametrize("lengths,rows,heads,kv_heads,dim", [([3000, 40], [7, 40], 8, 2, 128), ([5000], [20], 4, 1, 64)])
def test_scores_that_grow_along_the_keys(ext, lengths, rows, heads, kv_heads, dim, scale):
    trees = Trees(lengths, rows, kv_heads, dim, 64, 1, spread=lambda n: np.linspace(0.05, 4, n, dtype=np.float32))
    q = (torch.randn(sum(rows), heads, dim, generator=torch.Generator().manual_seed(2)) * 0.5).to(BF16).cuda()
    got = layers.kv4_tree_attention(q, trees.pages, trees.table, trees.lengths, trees.cu, scale, parents=trees.parents)
    assert_within(got, *trees.tree_attention(q, scale))


@pytest.mark.parametrize("dim", [64, 128])
def test_parents_of_every_kind(ext, dim):
    """Rows in any order, several roots, numbers outside the sequence, a row that is its own parent, and two that are each other's."""
    parents = [[-1, 0, 5, 1, -9, 4, 2, 70, 3], [1, 0, 2, 2 ** 31 - 1, -2 ** 31, 3, 1], [0]]
    trees = Trees([500, 30, 9], [len(t) for t in parents], 2, dim, 16, 4)
    trees.trees, trees.parents = parents, i32([p for tree in parents for p in tree])
    q = torch.randn(sum(trees.rows), 6, dim, generator=torch.Generator().manual_seed(3)).to(BF16).cuda()
    got = layers.kv4_tree_attention(q, trees.pages, trees.table, trees.lengths, trees.cu, 0.1, parents=trees.parents)
    assert_within(got, *trees.tree_attention(q, 0.1))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("lengths,rows,heads,kv_heads,dim", [([40, 300, 20], [9, 30, 20], 8, 2, 128), ([100, 1200], [33, 64], 4, 4, 64),
                                                             ([5000], [12], 40, 8, 128)])
def test_hidden_drafts_may_hold_anything(ext, lengths, rows, heads, kv_heads, dim, dtype):
    """Drafts whose keys or values are NaN (in fp16 infinite too) reach the rows that see them and no others, bit for bit; the
    context's reach all."""
    trees = Trees(lengths, rows, kv_heads, dim, 16, 6, dtype)
    q = torch.randn(sum(rows), heads, dim, generator=torch.Generator().manual_seed(5)).to(dtype).cuda()

    def run():
        return layers.kv4_tree_attention(q, trees.pages, trees.table, trees.lengths, trees.cu, 0.1, parents=trees.parents)

    clean, at, split, group = run(), 0, 16 * dim // 2, heads // kv_heads
    touched = torch.zeros(clean.shape, dtype=torch.bool)
    for s, (n, count, tree) in enumerate(zip(lengths, rows, trees.trees)):
        seen = torch.from_numpy(seen_rows(tree, count))
        for draft, half, scale, chunk in ((count - 1, 0, 255, 0), (count // 2, 1, 255, 1), (count // 3, 1, 250, dim // 32 - 1)):
            if scale == 250 and dtype == BF16:
                continue
            position = n - count + draft
            page = int(trees.table[s, position // 16])
            trees.pages[page, 1, half, split + position % 16 * (dim // 32) + chunk] = scale
            if scale == 250:
                trees.pages[page, 1, half, position % 16 * (dim // 2) + 16 * chunk:][:16] = 0x11  # 0.5 * 2^123: beyond fp16
            columns = slice(None) if half == 0 else slice(32 * chunk, 32 * chunk + 32)
            reached = touched[at:at + count, group:2 * group, columns]
            reached |= seen[:, draft, None, None]
        at += count
    got = run()
    assert torch.equal(torch.isfinite(got).cpu(), ~touched)
    assert torch.equal(got[~touched.cuda()], clean[~touched.cuda()])


def test_values_beyond_a_type_sum_as_infinities(ext):
    """fp16: a draft's value of 2^20 reads as infinity for the rows that see it; of both signs they make NaN."""
    trees = Trees([50], [4], 1, 64, 16, 7, FP16)
    trees.trees, trees.parents = [[-1, 0, 1, 0]], i32([-1, 0, 1, 0])
    q = torch.randn(4, 2, 64, generator=torch.Generator().manual_seed(1)).half().cuda()
    for draft, code in ((1, 0x22), (2, 0xAA)):  # 1.0 and -1.0
        page, offset = int(trees.table[0, (46 + draft) // 16]), (46 + draft) % 16
        trees.pages[page, 0, 1, 16 * 32 + offset * 2] = 127 + 20
        trees.pages[page, 0, 1, offset * 32:offset * 32 + 16] = code
    got = layers.kv4_tree_attention(q, trees.pages, trees.table, trees.lengths, trees.cu, 0.1, parents=trees.parents)
    assert torch.isfinite(got[[0, 3]]).all() and torch.isfinite(got[:, :, 32:]).all()
    assert (got[1, :, :32] == float("inf")).all() and torch.isnan(got[2, :, :32]).all()


def test_pages_outside_the_pool_and_odd_lengths(ext):
    """Unknown pages in the context and under the drafts, lengths past the table and below zero; rows that see nothing give zeros."""
    page, dim = 16, 64
    trees = Trees([160, 20, 64, 40], [6, 20, 3, 4], 1, dim, page, 6, extra_columns=0)
    q = torch.randn(sum(trees.rows), 3, dim, generator=torch.Generator().manual_seed(1)).to(BF16).cuda()
    table, lengths = trees.table.clone(), trees.lengths.clone()
    table[0, 2], table[0, 9] = -1, 10 ** 6  # positions 32..47 of the context; the drafts' 154..159
    table[1, 0] = -7                        # sequence 1: all but rows 16..19
    lengths[2], lengths[3] = 10 ** 9, -3
    got = layers.kv4_tree_attention(q, trees.pages, table, lengths, trees.cu, 0.2, parents=trees.parents)
    gone = [set(range(32, 48)) | set(range(144, 160)), set(range(16)), set(), set()]
    ends, at = [160, 20, 160, 0], 0  # the table's rows have ten columns
    for s, (end, count, tree) in enumerate(zip(ends, trees.rows, trees.trees)):
        seen, context = seen_rows(tree, count), end - count
        values = torch.zeros(1, 2, end, dim, dtype=torch.float64)
        values[:, :, :trees.values[s].shape[2]] = trees.values[s][:, :, :end]
        known = min(end, trees.lengths_host[s])
        hidden = torch.ones(count, end, dtype=torch.bool)
        for i in range(count):
            for p in range(known):
                hidden[i, p] = p in gone[s] or not (p < context or seen[i, p - context])
        for h in range(3):
            want, bound = masked_attention64(q[at:at + count, h], values[0, 0].cuda(), values[0, 1].cuda(), 0.2, hidden.cuda())
            assert_within(got[at:at + count, h], want, bound)
        at += count
    alone = [i for i in range(20) if not any(j >= 16 for j in np.flatnonzero(seen_rows(trees.trees[1], 20)[i]))]
    assert alone and not got[6:26][alone].any() and got[6 + 19].any() and not got[29:33].any()


@pytest.mark.parametrize("lengths,heads,kv_heads,dim", [([30, 20], 8, 2, 64), ([3000, 20], 5, 1, 128)])
def test_scores_of_minus_infinity(ext, lengths, heads, kv_heads, dim):
    """Rows whose visible scores are all -infinity get NaN; siblings that see another draft are what that draft makes them."""
    rows, page = [3, 2], 16
    counts = [-(-n // page) for n in lengths]
    table = torch.full((2, max(counts)), -1, dtype=torch.int32)
    for s, n in enumerate(counts):
        table[s, :n] = torch.arange(sum(counts[:s]), sum(counts[:s]) + n)
    x = torch.randn(sum(lengths), 2, kv_heads, dim, generator=torch.Generator().manual_seed(2)).to(BF16)
    x[:lengths[0], 0, :, :32] = 0
    x[:lengths[0], 0, :, 3] = -2.0 ** 100
    x[lengths[0] - 1, 0, :, 3] = 0  # the last row's own key
    pages, gpu = layers.kv4_pages(sum(counts), kv_heads, dim, page), x.cuda()
    layers.kv4_append(gpu[:, 0], gpu[:, 1], pages, table.cuda(), i32(lengths), cu=cumulative(lengths))
    q = torch.randn(5, heads, dim, generator=torch.Generator().manual_seed(3)).to(BF16)
    q[:3, :, 3] = 2.0 ** 100
    got = layers.kv4_tree_attention(q.cuda(), pages, table.cuda(), i32(lengths), i32([0, 3, 5]), dim ** -0.5, parents=i32([-1, 0, 0, -1, 0]))
    assert torch.isnan(got[:2]).all() and torch.isfinite(got[2:]).all()
    own = torch.from_numpy(mxfp4.dequantize(*mxfp4.quantize(x[lengths[0] - 1, 1].float().numpy()))).to(BF16)
    assert torch.equal(got[2].cpu(), own.repeat_interleave(heads // kv_heads, 0))  # a probability of one


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_the_largest_values(ext, dtype):
    for lengths, rows, heads, kv_heads, dim in (([90, 30], [5, 30], 8, 2, 64), ([9000], [16], 5, 1, 128)):
        page = 64
        counts = [-(-n // page) for n in lengths]
        table = torch.full((len(lengths), max(counts)), -1, dtype=torch.int32)
        for s, n in enumerate(counts):
            table[s, :n] = torch.arange(sum(counts[:s]), sum(counts[:s]) + n)
        x = torch.randn(sum(lengths), 2, kv_heads, dim, generator=torch.Generator().manual_seed(3)).to(dtype)
        largest = 6 * 2.0 ** (125 if dtype == BF16 else 13)
        x[:, 1] = largest
        pages, gpu = layers.kv4_pages(sum(counts), kv_heads, dim, page), x.cuda()
        layers.kv4_append(gpu[:, 0], gpu[:, 1], pages, table.cuda(), i32(lengths), cu=cumulative(lengths))
        q = torch.randn(sum(rows), heads, dim, generator=torch.Generator().manual_seed(4)).to(dtype).cuda()
        got = layers.kv4_tree_attention(q, pages, table.cuda(), i32(lengths), cumulative(rows), dim ** -0.5)
        assert ((got.double() / largest - 1).abs() <= 2 * HALF_STEP[dtype] + (9000 + 64) * 2.0 ** -23).all()


def test_rows_past_the_64th_and_outside_cu(ext):
    """Rows behind a sequence's 64th and rows of no sequence are left as they are; the 64 see what they see as drafts of all rows."""
    dim, page = 64, 16
    cache = Cache([200, 90], 2, dim, page, 5)
    q = torch.randn(100, 4, dim, generator=torch.Generator().manual_seed(1)).to(BF16).cuda()
    out = torch.full((100, 4, dim), 5.0, dtype=BF16, device="cuda")
    got = layers.kv4_tree_attention(q, cache.pages, cache.table, cache.lengths, i32([3, 83, 90]), 0.1, out=out)
    assert (out[:3] == 5).all() and (out[67:83] == 5).all() and (out[90:] == 5).all()
    for at, count, end, values in ((3, 64, 184, cache.values[0]), (83, 7, 90, cache.values[1])):
        hidden = torch.ones(count, end, dtype=torch.bool).triu(end - count + 1).cuda()
        for h in range(4):
            k, v = values[h // 2, :, :end].cuda()
            assert_within(got[at:at + count, h], *masked_attention64(q[at:at + count, h], k, v, 0.1, hidden))


def test_strided_rows_tables_and_the_workspace(ext):
    lengths, rows, heads, kv_heads, dim = [1000, 9, 333], [11, 9, 2], 6, 2, 128
    trees = Trees(lengths, rows, kv_heads, dim, 32, 4)
    q = torch.randn(sum(rows), heads, dim, generator=torch.Generator().manual_seed(1)).to(BF16).cuda()
    want = layers.kv4_tree_attention(q, trees.pages, trees.table, trees.lengths, trees.cu, 0.1, parents=trees.parents)
    wide = torch.randn(sum(rows), heads + 2 * kv_heads, dim + 8).to(BF16).cuda()
    view = wide[:, 1:1 + heads, 8:]
    view.copy_(q)
    out = torch.full((sum(rows), 2 * heads, dim + 4), 9.0, dtype=BF16, device="cuda")
    table = torch.full((3, trees.table.shape[1] + 5), 2 ** 30, dtype=torch.int32, device="cuda")
    table[:, 3:3 + trees.table.shape[1]] = trees.table
    got = layers.kv4_tree_attention(view, trees.pages, table[:, 3:], trees.lengths, trees.cu, 0.1, parents=trees.parents, out=out[:, ::2, 4:])
    assert torch.equal(got, want) and (out[:, 1::2] == 9).all() and (out[..., :4] == 9).all()
    size = layers.kv4_tree_attention_workspace_bytes(trees.pages, trees.table, sum(rows), heads, dim)
    guarded = torch.full((size + 512,), 255, dtype=torch.uint8, device="cuda")  # NaN wherever it is read unwritten
    again = layers.kv4_tree_attention(q, trees.pages, trees.table, trees.lengths, trees.cu, 0.1, parents=trees.parents,
                                      workspace=guarded[256:256 + size])
    assert size > 0 and torch.equal(again, want) and (guarded[:256] == 255).all() and (guarded[256 + size:] == 255).all()
    with pytest.raises(_lib.TexelatorError, match="too small"):
        layers.kv4_tree_attention(q, trees.pages, trees.table, trees.lengths, trees.cu, 0.1, workspace=guarded[:size - 16])
    with pytest.raises(_lib.TexelatorError, match="overlap"):
        layers.kv4_tree_attention(q, trees.pages, trees.table, trees.lengths, trees.cu, 0.1, out=q)


def test_trees_past_four_gib(ext):
    page, dim, kv_heads = 1024, 128, 8
    pages = torch.zeros(4000, kv_heads, 2, page * dim * 17 // 32, dtype=torch.uint8, device="cuda")
    assert pages.numel() > 2 ** 32
    ids = [3999, 0, 3950]
    table, lengths = i32(ids).view(1, 3), i32([2500])
    x = torch.randn(2500, 2, kv_heads, dim, generator=torch.Generator().manual_seed(1)).to(BF16).cuda()
    cos, sin = rope_tables(2500, dim)
    q = torch.randn(2500, 16, dim).to(BF16).cuda()
    turned = layers.kv4_append_rope(q, x[:, 0], x[:, 1], cos, sin, pages, table, lengths, cu=i32([0, 2500]))
    small, near = layers.kv4_pages(3, kv_heads, dim, page), i32([0, 1, 2]).view(1, 3)
    layers.kv4_append_rope(q, x[:, 0], x[:, 1], cos, sin, small, near, lengths, cu=i32([0, 2500]))
    assert torch.equal(small, pages[ids]) and not pages[3998].any()
    want = layers.kv4_tree_attention(turned[-9:], small, near, lengths, i32([0, 9]), 0.09)
    assert torch.equal(layers.kv4_tree_attention(turned[-9:], pages, table, lengths, i32([0, 9]), 0.09), want) and want.any()
    path, accepted = i32([0, 3, 8, -1, -1, -1, -1, -1, -1]), i32([2])
    for p, t in ((pages, table), (small, near)):
        assert layers.kv4_keep_path(p, t, lengths, i32([0, 9]), path, accepted, dim).tolist() == [2494]
    assert torch.equal(small, pages[ids])


# ---------------------------------------------------------------------------------------------
# verification


def drafted(rows, vocab, dtype, seed, kind="tree", width=None):
    """Target logits with a few likely tokens, drafts that mostly agree with them, and random numbers."""
    g, rng = torch.Generator().manual_seed(seed), np.random.default_rng(seed)
    total = sum(rows)
    trees = [random_parents(rng, n) if kind == "tree" else list(range(-1, n - 1)) for n in rows]
    logits = 1.5 * torch.randn(total, vocab, generator=g)
    logits.scatter_add_(1, torch.randint(0, vocab, (total, min(4, vocab)), generator=g), 5 + torch.randn(total, min(4, vocab), generator=g))
    draft = (logits + 0.7 * torch.randn(total, vocab, generator=g)).to(dtype)
    logits = logits.to(dtype)
    ids, at = torch.zeros(total, dtype=torch.int64), 0
    for tree in trees:
        tried = {}
        for i, parent in enumerate(tree):
            source, rank = at + max(parent, 0), tried.get(parent, 0)
            tried[parent] = rank + 1
            if kind == "sampled":
                ids[at + i] = torch.multinomial(torch.softmax(draft[source].float(), 0), 1, generator=g)[0]
            else:
                ids[at + i] = draft[source].float().topk(min(rank + 1, vocab)).indices[-1]
        at += len(tree)
    return trees, logits, draft if kind == "sampled" else None, ids, torch.rand(total, generator=g)


def check_verified(rows, trees, logits, draft, ids, uniforms, temperatures, kind, **more):
    want = verify64(logits, ids, uniforms, trees, temperatures, draft)
    parents = i32([p for tree in trees for p in tree]) if kind == "tree" else None
    heat = torch.tensor(temperatures, dtype=FP32, device="cuda") if len(set(temperatures)) != 1 else temperatures[0]
    got = layers.verify_drafts(logits.cuda(), ids.cuda(), uniforms.cuda(), cumulative(rows), parents=parents,
                               draft_logits=None if draft is None else draft.cuda(), temperature=heat, **more)
    assert [t.tolist() for t in got] == [list(w) for w in want]
    return got


VERIFY = [
    # rows, vocabulary, kind
    ([1], 1, "tree"),
    ([1], 700, "chain"),
    ([6], 151936, "tree"),
    ([8, 8, 1, 3], 32003, "sampled"),
    ([5, 0, 64, 17], 5003, "tree"),
    ([64, 63, 2], 2048, "chain"),
    ([9, 0, 30], 2047, "sampled"),
    ([3] * 100, 501, "tree"),
    ([i % 9 for i in range(130)], 257, "sampled"),
]


@pytest.mark.parametrize("temperature", [0.0, 0.7, 2.5, None])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("rows,vocab,kind", VERIFY)
def test_verified_as_one_draft_after_the_other(ext, rows, vocab, kind, dtype, temperature):
    trees, logits, draft, ids, uniforms = drafted(rows, vocab, dtype, vocab + len(rows), kind)
    temperatures = [temperature] * len(rows) if temperature is not None else [(0.0, 0.5, 1.0, -1.0)[i % 4] for i in range(len(rows))]
    check_verified(rows, trees, logits, draft, ids, uniforms, temperatures, kind)


def test_every_token_is_drawn_at_its_share(ext):
    """Random numbers on a grid: of N closing draws, each token gets N p of them, one more or less for each border; after a rejected
    draft the rest's share; and a draft is accepted for just the numbers below its probability."""
    vocab, grid = 37, 4096
    g = torch.Generator().manual_seed(1)
    logits = torch.randn(1, vocab, generator=g) * 2
    p = torch.softmax(logits.double() / 0.9, 1)[0]
    u = (torch.arange(grid) + 0.5) / grid
    # one sequence a number: a row and no draft
    cu = i32(range(grid + 1))
    _, _, tokens = layers.verify_drafts(logits.expand(grid, -1).cuda(), torch.zeros(grid, dtype=torch.int64, device="cuda"), u.cuda(), cu,
                                        temperature=0.9)
    share = torch.bincount(tokens.cpu(), minlength=vocab) / grid
    assert ((share - p).abs() <= 1.0 / grid).all()
    # a draft of token 5, its number on the grid, then the closing number on another
    pairs = torch.stack([u.flip(0), u], 1).flatten()
    two = logits.expand(2 * grid, -1).cuda()
    ids = torch.full((2 * grid,), 5, dtype=torch.int64, device="cuda")
    accepted, _, tokens = layers.verify_drafts(two, ids, pairs.cuda(), i32(range(0, 2 * grid + 1, 2)), temperature=0.9)
    assert torch.equal(accepted.cpu() == 1, u.double() < p[5])
    closing = tokens.view(-1, 2)[accepted == 0][:, 0].cpu()
    assert not (closing == 5).any()
    rest = torch.where(torch.arange(vocab) == 5, 0.0, p) / (1 - p[5])
    expected = torch.searchsorted(rest.cumsum(0), pairs.view(-1, 2)[accepted.cpu() == 0][:, 0].double(), right=True)
    assert torch.equal(closing, expected.clamp(max=vocab - 1))


@pytest.mark.parametrize("temperature", [0.6, 1.0, 2.0])
def test_sampled_drafts_leave_the_targets_distribution(ext, temperature):
    """A draft x drawn from q, then the call: the first new token is p's. Numbers on a grid: for each x the share a(x) of them that accept, then
    with x rejected the shares r(y | x) of the closing tokens. q(y) a(y) + sum over x of q(x) (1 - a(x)) r(y | x) is p(y) but for the grid,
    which is off by 1 / grid at most in each a and 1 / grid in each r (a token's numbers are an interval): 3 / grid in all."""
    vocab, grid = 11, 2048
    g = torch.Generator().manual_seed(4)
    logits, draft = (1.5 * torch.randn(1, vocab, generator=g) for _ in range(2))
    t = float(torch.tensor(temperature, dtype=FP32))
    p, q = (torch.softmax(x[0].double() / t, 0) for x in (logits, draft))
    u = ((torch.arange(grid) + 0.5) / grid).repeat(vocab)
    n = vocab * grid
    ids = torch.arange(vocab).repeat_interleave(grid).repeat_interleave(2).cuda()
    cu = i32(range(0, 2 * n + 1, 2))
    rows = [x.cuda().expand(2 * n, -1) for x in (logits, draft)]

    def call(tests, closing):
        accepted, _, tokens = layers.verify_drafts(rows[0], ids, torch.stack([closing, tests], 1).flatten().cuda(), cu, draft_logits=rows[1],
                                                   temperature=temperature)
        return accepted.cpu().view(vocab, grid), tokens.cpu().view(vocab, grid, 2)

    accepted, tokens = call(u, u.flip(0))
    assert torch.equal(tokens[accepted == 1][:, 0], torch.arange(vocab)[:, None].expand(-1, grid)[accepted == 1])
    share = accepted.double().mean(1)
    total = q * share
    rejected, tokens = call(torch.full((n,), 1 - 2.0 ** -24), u)
    for x in range(vocab):
        if share[x] == 1:
            continue
        assert p[x] < q[x] and not rejected[x].any()
        total += q[x] * (1 - share[x]) * torch.bincount(tokens[x, :, 0], minlength=vocab) / grid
    assert (share < 1).any() and ((total - p).abs() <= 3 / grid).all()


@pytest.mark.parametrize("temperature", [0.9, 1.3, 2.5])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_drafts_next_to_their_border(ext, dtype, temperature):
    """Numbers 9e-8 of a draft's probability below it accept, as far above it they do not. Terms in 32 bits are off by half of an
    exponential's last bit in common at most (2^-24 = 6e-8); their other roundings are each its own, and 2^-24 (2 + exponent) of thousands of
    terms that count make less than 1e-8 of the sum."""
    vocab, drafts, off = 151936, 200, 9e-8
    g = torch.Generator().manual_seed(3)
    logits = (2.5 * torch.randn(1, vocab, generator=g)).to(dtype)
    p = torch.softmax(logits[0].double() / float(torch.tensor(temperature, dtype=FP32)), 0)
    ids = torch.randint(0, vocab, (drafts,), generator=g)
    borders = p[ids].numpy()
    below, above = (borders * (1 - off)).astype(np.float32), (borders * (1 + off)).astype(np.float32)
    below = np.where(below.astype(np.float64) > borders * (1 - off), np.nextafter(below, np.float32(0)), below)
    above = np.where(above.astype(np.float64) < borders * (1 + off), np.nextafter(above, np.float32(1)), above)
    tokens, uniforms = torch.zeros(4 * drafts, dtype=torch.int64), torch.full((4 * drafts,), 0.5)
    tokens[1::2] = ids.repeat_interleave(2)
    uniforms[1::4], uniforms[3::4] = torch.from_numpy(below), torch.from_numpy(above)
    accepted, _, _ = layers.verify_drafts(logits.cuda().expand(4 * drafts, -1), tokens.cuda(), uniforms.cuda(), i32(range(0, 4 * drafts + 1, 2)),
                                          temperature=temperature)
    assert accepted[0::2].all() and not accepted[1::2].any()


def test_repeated_unknown_and_impossible_drafts(ext):
    """A token that a sibling had already, tokens outside the vocabulary, tokens without weight: never accepted, and not counted."""
    vocab = 50
    logits = torch.randn(6, vocab, generator=torch.Generator().manual_seed(2))
    logits[0, 7] = float("-inf")
    logits[0, 9] = 1.0
    trees, rows = [[-1, 0, 0, 0, 0, 0]], [6]
    for ids in ([0, 9, 9, 9, 9, 9], [0, 7, -1, 50, 2 ** 40, 9], [0, -2 ** 62, 9, 9, 7, 9]):
        for u in (0.001, 0.02, 0.3, 0.999):
            uniforms = torch.full((6,), u)
            uniforms[0] = 0.77
            check_verified(rows, trees, logits, None, torch.tensor(ids), uniforms, [1.0], "tree")
            check_verified(rows, trees, logits, None, torch.tensor(ids), uniforms, [0.0], "tree")


def test_rows_of_any_order_and_loose_ends(ext):
    """Parents behind their rows, rows that hang on nothing, on themselves or on each other: only what row 0 leads to is reached."""
    rows = [8, 5, 3]
    trees = [[3, 5, 0, 7, 2, 0, -1, 6], [-1, 2, 1, 0, 3], [9, 2, 2]]
    logits = torch.randn(16, 20, generator=torch.Generator().manual_seed(3))
    flat, at = [], 0
    ids = torch.zeros(16, dtype=torch.int64)
    for tree in trees:
        for i, p in enumerate(tree):
            ids[at + i] = logits[at + (p if 0 <= p < len(tree) else 0)].argmax()
        flat += tree
        at += len(tree)
    safe = [[-1] + t[1:] for t in trees]  # row 0 follows nothing whatever its entry says
    for temperature in (0.0, 0.3):
        uniforms = torch.rand(16, generator=torch.Generator().manual_seed(4)) * 0.5
        want = verify64(logits, ids, uniforms, safe, [temperature] * 3)
        got = layers.verify_drafts(logits.cuda(), ids.cuda(), uniforms.cuda(), cumulative(rows), parents=i32(flat), temperature=temperature)
        assert [t.tolist() for t in got] == [list(w) for w in want]


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("vocab", [40, 9001])
def test_probabilities_that_are_undefined(ext, vocab, dtype):
    """Rows with a NaN, an infinity or nothing above -infinity: nothing behind them is accepted and the token is -1, in their own
    sequence alone; -infinity elsewhere is no weight."""
    rows = [3, 3, 3, 3, 3, 3]
    trees, logits, _, ids, uniforms = drafted(rows, vocab, dtype, 5, "chain")
    uniforms = uniforms * 0.01
    logits[0, vocab // 2] = float("nan")
    logits[3 + 1] = float("-inf")
    logits[6 + 2, vocab - 1] = float("inf")
    logits[9:12, : vocab // 3] = float("-inf")
    logits[12 + 1, 0] = float("nan")
    for i in (2, 5, 8, 11, 14, 17):
        ids[i], ids[i - 1] = logits[i - 1].float().nan_to_num(-1e9, posinf=1e9).argmax(), logits[i - 2].float().nan_to_num(-1e9).argmax()
    for temperature in (0.0, 0.8):
        check_verified(rows, trees, logits, None, ids, uniforms, [temperature] * 6, "chain")
    draft = logits.clone()
    draft[12:] = torch.randn(6, vocab)
    draft[15, 3] = float("nan")  # the draft model's own: undefined as well
    logits[12:] = torch.randn(6, vocab)
    check_verified(rows, trees, logits, draft, ids, uniforms, [0.8] * 6, "sampled")


def test_temperatures_of_all_sizes(ext):
    """From the smallest, where all weight is on the largest logits, to infinity, where every token weighs the same."""
    rows, vocab = [4] * 6, 300
    trees, logits, _, ids, uniforms = drafted(rows, vocab, FP32, 6, "tree")
    temperatures = [1e-38, 1e-6, 0.05, 40.0, 1e30, float("inf")]
    check_verified(rows, trees, logits, None, ids, uniforms, temperatures, "tree")


@pytest.mark.parametrize("temperature", [float("inf"), 3e38])
@pytest.mark.parametrize("kind", ["tree", "sampled"])
def test_masked_tokens_at_the_largest_temperatures(ext, kind, temperature):
    """Every token above -infinity weighs the same, the others nothing: drafts are accepted at that share."""
    rows, vocab = [6, 3], 11
    trees, logits, draft, ids, uniforms = drafted(rows, vocab, FP32, 8, kind)
    logits[:, 4:9] = -np.inf
    ids[:] = torch.tensor([0, 1, 2, 3, 9, 10, 4, 0, 1])
    uniforms[:] = torch.tensor([0.9, 0.05, 0.1, 0.16, 0.05, 0.1, 0.5, 0.0, 0.1])
    check_verified(rows, trees, logits, draft, ids, uniforms, [temperature] * 2, kind)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("kind", ["tree", "sampled"])
def test_lowest_values_as_masks_and_the_widest_rows(ext, kind, dtype):
    """The type's lowest value in place of most logits, or of all; logits further apart than fp32's largest value; exponents far from zero."""
    rows, vocab, info = [3] * 5, 2500, torch.finfo(dtype)
    temperatures = [1.0, 1e-3, float("inf"), 2e-38, 0.9]
    trees, logits, draft, ids, uniforms = drafted(rows, vocab, dtype, 12, kind)
    logits[:, 100:2400] = info.min
    logits[3:6, ::2] = info.min  # spans with a maximum of their own
    logits[7] = info.min
    logits[8, ::3] = info.max
    logits[13:, :90] += 900.0 if dtype == FP16 else 1e5
    uniforms = uniforms * 0.02
    check_verified(rows, trees, logits, draft, ids, uniforms, temperatures, kind)


@pytest.mark.parametrize("temperature", [0.0, 1.3])
@pytest.mark.parametrize("kind", ["tree", "sampled"])
def test_the_largest_vocabulary(ext, kind, temperature):
    rows, vocab = [3, 2], 1 << 24
    trees, logits, draft, ids, uniforms = drafted(rows, vocab, FP16, 3, "tree")
    if kind == "sampled":
        trees, draft = [list(range(-1, n - 1)) for n in rows], torch.cat([logits[:, 5:], logits[:, :5]], dim=1)
    logits[0, -1] = 30.0  # the last token is drawn or drafted
    ids[1] = vocab - 1
    check_verified(rows, trees, logits, draft, ids, uniforms, [temperature] * 2, kind)


def test_the_same_tokens_whichever_workgroup_ends_last(ext):
    """Other numbers for the last draw between two calls that are alike: their sums lie in the same workspace."""
    rows, vocab = [5] * 12, 70001
    trees, logits, draft, ids, uniforms = drafted(rows, vocab, BF16, 9, "sampled")
    scratch = torch.empty(layers.verify_drafts_workspace_bytes(logits.cuda(), 12, sampled=True), dtype=torch.uint8, device="cuda")
    logits, draft, ids, cu = logits.cuda(), draft.cuda(), ids.cuda(), cumulative(rows)
    numbers = [uniforms.cuda(), (uniforms * 0.37).cuda()]

    def call(i, temperature):
        return layers.verify_drafts(logits, ids, numbers[i], cu, draft_logits=draft, temperature=temperature, workspace=scratch)

    want = [[t.tolist() for t in call(i, 1.0 + i)] for i in range(2)]
    for _ in range(60):
        for i in range(2):
            assert [t.tolist() for t in call(i, 1.0 + i)] == want[i]


def test_identical_models_and_the_largest_numbers(ext):
    """Draft and target alike: every draft is accepted, for numbers of 1 too (where q(x) is not below p(x)) nothing breaks."""
    rows, vocab = [5, 7], 3001
    trees, logits, _, ids, uniforms = drafted(rows, vocab, BF16, 7, "sampled")
    got = check_verified(rows, trees, logits, logits, ids, uniforms, [1.0] * 2, "sampled")
    assert got[0].tolist() == [4, 6]
    ones = torch.ones(12)
    accepted, path, tokens = layers.verify_drafts(logits.cuda(), ids.cuda(), ones.cuda(), cumulative(rows), draft_logits=logits.cuda())
    assert accepted.tolist() == [0, 0] and all(0 <= tokens[i] < vocab for i in (0, 5))


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_strided_logits_outputs_and_the_workspace(ext, dtype):
    """Rows of a wider buffer that begin anywhere; outputs and workspace given, rows of no sequence left alone."""
    rows, vocab = [5, 9], 4099
    trees, logits, draft, ids, uniforms = drafted(rows, vocab, dtype, 8, "sampled")
    want = layers.verify_drafts(logits.cuda(), ids.cuda(), uniforms.cuda(), cumulative(rows), draft_logits=draft.cuda())
    wide = torch.full((20, 2 * vocab + 7), float("nan"), dtype=dtype, device="cuda")
    views = wide[3:17, 1:1 + vocab], wide[3:17, vocab + 4:2 * vocab + 4]
    for view, source in zip(views, (logits, draft)):
        view.copy_(source)
    got = layers.verify_drafts(views[0], ids.cuda(), uniforms.cuda(), cumulative(rows), draft_logits=views[1])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    size = layers.verify_drafts_workspace_bytes(wide[:, :vocab], 2, sampled=True)
    guarded = torch.full((size + 512,), 255, dtype=torch.uint8, device="cuda")
    out = torch.full((2,), 77, dtype=torch.int32, device="cuda"), torch.full((20,), 77, dtype=torch.int32, device="cuda"), torch.full((20,), 77, device="cuda")
    more = torch.zeros(20, dtype=torch.int64, device="cuda"), torch.rand(20, device="cuda")
    more[0][3:17], more[1][3:17] = ids.cuda(), uniforms.cuda()
    layers.verify_drafts(wide[:, 1:1 + vocab], *more, i32([3, 8, 17]), draft_logits=wide[:, vocab + 4:2 * vocab + 4],
                         workspace=guarded[256:256 + size], out=out)
    assert torch.equal(out[0], want[0]) and torch.equal(out[1][3:17], want[1]) and torch.equal(out[2][3:17], want[2])
    assert all((t[:3] == 77).all() and (t[17:] == 77).all() for t in out[1:])
    assert (guarded[:256] == 255).all() and (guarded[256 + size:] == 255).all()


def test_rows_past_the_64th_take_no_part_in_a_path(ext):
    vocab = 100
    logits = torch.randn(70, vocab, generator=torch.Generator().manual_seed(1))
    ids = torch.cat([torch.zeros(1, dtype=torch.int64), logits[:-1].argmax(1)])
    out = torch.full((1,), 9, dtype=torch.int32, device="cuda"), torch.full((70,), 9, dtype=torch.int32, device="cuda"), torch.full((70,), 9, device="cuda")
    layers.verify_drafts(logits.cuda(), ids.cuda(), torch.zeros(70, device="cuda"), i32([0, 70]), temperature=0.0, out=out)
    assert out[0].item() == 63 and out[1][:64].tolist() == list(range(64)) and (out[1][64:] == 9).all() and (out[2][64:] == 9).all()
    assert out[2][:64].tolist() == ids[1:65].tolist()


# ---------------------------------------------------------------------------------------------
# the accepted rows


@pytest.mark.parametrize("layer_count,kv_heads,dim,page", [(None, 1, 64, 16), (3, 2, 128, 16), (2, 5, 64, 32), (1, 3, 128, 1024),
                                                          (100, 8, 64, 16), (101, 5, 128, 16)])
def test_accepted_rows_move_together(ext, layer_count, kv_heads, dim, page):
    """Every byte of every pool: the path's rows at their places, nothing else changed; paths in any order, whole, empty."""
    rng = np.random.default_rng(dim + kv_heads)
    rows = [9, 1, 64, 64, 5, 0, 7, 3]
    lengths = [100, 1, 64, 200, 30, 12, 16, 2]  # the last has fewer positions than rows
    paths = [[0, 2, 5, 8], [0], list(range(64)), [0] + sorted(rng.choice(np.arange(1, 64), 40, replace=False).tolist()), [0, 4, 2, 1, 3], [],
             [0, 6, 9, -4, 5], [0, 2]]
    counts = [-(-n // page) for n in lengths]
    order = rng.permutation(sum(counts) + 2)
    table = np.full((len(lengths), max(counts) + 1), -1, dtype=np.int32)
    for s, n in enumerate(counts):
        table[s, :n] = order[sum(counts[:s]):sum(counts[:s]) + n]
    shape = (layer_count or 1, len(order), kv_heads, 2, page * dim * 17 // 32)
    before = rng.integers(0, 256, size=shape, dtype=np.uint8)
    want, split = before.copy(), page * dim // 2
    codes, scales = (want[..., :split].reshape(*shape[:-1], page, dim // 2).copy(), want[..., split:].reshape(*shape[:-1], page, dim // 32).copy())
    for s, (n, count, path) in enumerate(zip(lengths, rows, paths)):
        moves = [(n - count + row, n - count + j) for j, row in enumerate(path) if j > 0 and 0 <= row < count]
        moves = [(a, b) for a, b in moves if a >= 0 and b >= 0]
        for part in (codes, scales):
            held = [part[:, table[s, a // page], :, :, a % page].copy() for a, _ in moves]
            for (_, b), row in zip(moves, held):
                part[:, table[s, b // page], :, :, b % page] = row
    want = np.concatenate([codes.reshape(*shape[:-1], -1), scales.reshape(*shape[:-1], -1)], axis=-1)
    flat = [r for count, path in zip(rows, paths) for r in (path + [-1] * count)[:count]]
    accepted = [len(path) - 1 for path in paths]
    pages = torch.from_numpy(before.copy()).cuda()
    given = pages if layer_count else pages[0]
    got = layers.kv4_keep_path(given, i32(table.reshape(-1)).view(table.shape), i32(lengths), cumulative(rows), i32(flat), i32(accepted), dim)
    assert got.tolist() == [n - count + a + 1 for n, count, a in zip(lengths, rows, accepted)]
    assert np.array_equal(pages.cpu().numpy(), want)


def test_moves_out_of_and_into_unknown_pages(ext):
    """Rows whose place or target lies in no page stay; counts beyond the rows are cut to them; rows past the 64th stay."""
    dim, page = 64, 16
    pages = torch.randint(0, 256, (4, 1, 2, page * dim * 17 // 32), dtype=torch.uint8, device="cuda")
    before = pages.clone()
    table, lengths = i32([-1, 0, 1, 99]).view(2, 2), i32([20, 30])
    out = layers.kv4_keep_path(pages, table, lengths, i32([0, 8, 14]), i32([0, 5, 3, 6, 1, 1, 1, 1] + [0, 3, 5, 5, 5, 5]), i32([3, 900]), dim)
    assert out.tolist() == [16, 30]
    # sequence 0: places 12..19, in page -1 up to 15: rows 5 -> 1, 3 -> 2 and 6 -> 3 have no place; sequence 1: 24..29 lie in page 99
    assert torch.equal(pages, before)
    many = i32([0, 70])
    path = i32([0, 66, 5] + [-1] * 67)
    table, lengths = i32([0, 1, 2, 3, 3]).view(1, 5), i32([70])
    out = torch.empty(1, dtype=torch.int32, device="cuda")
    layers.kv4_keep_path(pages, table, lengths, many, path, i32([2]), dim, out=out)
    assert out.item() == 3
    codes = pages[0, 0, :, :page * dim // 2].view(2, page, dim // 2)
    assert torch.equal(codes[:, 1], before[0, 0, :, :page * dim // 2].view(2, page, dim // 2)[:, 1])  # row 66 is none
    assert torch.equal(codes[:, 2], before[0, 0, :, :page * dim // 2].view(2, page, dim // 2)[:, 5])
    with pytest.raises(_lib.TexelatorError, match="overlap"):
        layers.kv4_keep_path(pages, table, lengths, many, path, i32([2]), dim, out=lengths)


# ---------------------------------------------------------------------------------------------
# streams and empty calls


def test_two_streams_at_once(ext):
    """Attention and verification on two streams, each call with its own workspace, give the bits of calls one after the other."""
    trees = [Trees([4000, 100], [16, 9], 2, 128, 64, 12), Trees([900, 2500, 3], [30, 5, 3], 4, 64, 32, 13)]
    qs = [torch.randn(sum(t.rows), 8, t.dim, generator=torch.Generator().manual_seed(1)).to(BF16).cuda() for t in trees]
    cases = [drafted(t.rows, 6007, BF16, 3, "tree") for t in trees]
    moved = [tuple(x.cuda() for x in (c[1], c[3], c[4])) + (i32([p for tree in c[0] for p in tree]),) for c in cases]

    def both(i):
        t, (logits, ids, uniforms, parents) = trees[i], moved[i]
        return (layers.kv4_tree_attention(qs[i], t.pages, t.table, t.lengths, t.cu, 0.1, parents=t.parents),
                *layers.verify_drafts(logits, ids, uniforms, t.cu, parents=parents))

    want = [both(i) for i in range(2)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(8):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(both(i))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for i in range(2) for result in got[i] for a, b in zip(result, want[i]))


def test_calls_without_rows(ext):
    pages = layers.kv4_pages(4, 2, 64, 16)
    table, lengths = torch.zeros(3, 2, dtype=torch.int32, device="cuda"), i32([3, 0, 20])
    none = torch.zeros(0, 2, 64, dtype=BF16, device="cuda")
    cu = i32([0, 0, 0, 0])
    cos, sin = rope_tables(4, 64)
    assert layers.kv4_append_rope(none, none, none, cos, sin, pages, table, lengths, cu=cu).shape == none.shape
    assert layers.kv4_tree_attention(none, pages, table, lengths, cu, 1.0).shape == none.shape
    empty = torch.zeros(0, dtype=torch.int64, device="cuda")
    accepted, path, tokens = layers.verify_drafts(torch.zeros(0, 9, device="cuda"), empty, empty.float(), cu)
    assert accepted.tolist() == [-1] * 3 and path.numel() == tokens.numel() == 0
    assert layers.kv4_keep_path(pages, table, lengths, cu, path, accepted, 64).tolist() == [3, 0, 20]
    assert layers.verify_drafts(torch.zeros(0, 9, device="cuda"), empty, empty.float(), cu[:1])[0].numel() == 0
    assert layers.kv4_keep_path(pages, table[:0], lengths[:0], cu[:1], path, accepted[:0], 64).numel() == 0
    assert not pages.any()
