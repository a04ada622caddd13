"""Causal attention of packed sequences at the edges of its tiles and under each split of its waves."""
from __future__ import annotations

import pytest
import torch

from tests.serving import assert_within, attention64, cumulative, i32
from texelator_amd import _lib, layers

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def inputs(new, old, heads, kv_heads, dim, dtype, seed, behind=0, spread=1.0):
    """q, k, v as views of one projection each, noise in the columns between, NaN rows behind the last sequence."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    tokens, keys = sum(new), sum(new) + sum(old)
    q = torch.randn(tokens + behind, heads + 1, dim, device="cuda", generator=g)
    kv = torch.randn(keys + behind, 2 * kv_heads + 1, dim, device="cuda", generator=g)
    q[:tokens] *= spread
    if behind:
        q[tokens:], kv[keys:] = float("nan"), float("nan")
    q, kv = q.to(dtype), kv.to(dtype)
    return q[:, :heads], kv[:, :kv_heads], kv[:, kv_heads:2 * kv_heads]


def reference(q, k, v, new, old, scale):
    heads, group = q.shape[1], q.shape[1] // k.shape[1]
    want = torch.zeros(sum(new), heads, q.shape[2], dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(want)
    q0 = k0 = 0
    for n, o in zip(new, old):
        for h in range(heads):
            want[q0:q0 + n, h], bound[q0:q0 + n, h] = attention64(q[q0:q0 + n, h], k[k0:k0 + n + o, h // group], v[k0:k0 + n + o, h // group],
                                                                  scale, o)
        q0, k0 = q0 + n, k0 + n + o
    return want, bound


def run(q, k, v, new, old, scale, **more):
    return layers.packed_attention(q, k, v, cumulative(new), scale, cu_k=cumulative([n + o for n, o in zip(new, old)]), **more)


CASES = [
    # new tokens, tokens before them (negative: fewer keys than queries), heads, kv heads
    ([1], [0], 1, 1),
    ([1, 1, 1], [0, 31, 700], 16, 2),
    ([31, 32, 33, 0, 64, 65], [0] * 6, 8, 1),
    ([0, 0, 5], [3, 0, 0], 5, 5),
    ([97, 128, 129, 127], [1, 30, 31, 33], 16, 2),
    ([50, 7, 90], [-50, -3, -33], 8, 2),       # no key at all; rows without keys at the start
    ([300, 1], [-299, 0], 28, 4),
    ([200, 333, 5], [500, 0, 64], 28, 4),
    ([700, 3, 129], [0, 10, 70], 40, 8),
    ([1400, 70], [0, 5], 40, 8),
    ([2200, 70], [0, 5], 40, 8),
    ([70, 190, 0, 2, 33], [2000, 31, 300, 900, 1], 40, 8),
    ([3] * 130, [i % 40 for i in range(130)], 4, 4),  # more sequences than lanes
]


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("new,old,heads,kv_heads", CASES)
def test_against_64_bits(ext, new, old, heads, kv_heads, dtype, dim):
    q, k, v = inputs(new, old, heads, kv_heads, dim, dtype, sum(new), behind=5)
    tokens = sum(new)
    out = torch.full((tokens + 5, heads, dim), 9.0, dtype=dtype, device="cuda")
    got = run(q, k, v, new, old, dim ** -0.5, out=out)
    assert_within(got[:tokens], *reference(q, k, v, new, old, dim ** -0.5))
    assert (out[tokens:] == 9).all()  # rows behind the last sequence
    again = run(q, k, v, new, old, dim ** -0.5)
    assert torch.equal(again[:tokens], got[:tokens])


@pytest.mark.parametrize("scale", [1.0, -0.7, 0.0])
@pytest.mark.parametrize("new,old,heads", [([200, 40], [100, 0], 8), ([900], [50], 40), ([1800], [50], 40)])
def test_scores_that_grow_along_the_keys(ext, new, old, heads, scale):
    q, k, v = inputs(new, old, heads, heads, 128, BF16, 3, spread=0.5)
    k = (k.float() * torch.linspace(0.05, 4, k.shape[0], device="cuda")[:, None, None]).to(BF16)
    assert_within(run(q, k, v, new, old, scale), *reference(q, k, v, new, old, scale))


@pytest.mark.parametrize("new,heads,kv_heads", [([64, 10], 8, 8), ([323, 50], 28, 4), ([704], 40, 8), ([1409, 200], 56, 7)])
def test_a_sequence_and_a_query_do_not_reach_the_others(ext, new, heads, kv_heads):
    """Other contents of one sequence, and a query of far larger scores, leave the bits of all other queries."""
    old = [0] * len(new)
    q, k, v = inputs(new, old, heads, kv_heads, 128, BF16, 11)
    want = run(q, k, v, new, old, 0.09)
    loud = 32 * (new[0] // 32) - 1
    q[loud] *= 30
    got = run(q, k, v, new, old, 0.09)
    rows = [t for t in range(sum(new)) if t != loud]
    assert torch.equal(got[rows], want[rows]) and not torch.equal(got[loud], want[loud])
    if len(new) > 1:
        k[:new[0]], v[:new[0]] = float("nan"), float("inf")
        got = run(q, k, v, new, old, 0.09)
        assert torch.equal(got[new[0]:], want[new[0]:]) and torch.isnan(got[:new[0]]).all()


def test_keys_behind_a_query_reach_it_in_no_way(ext):
    """Infinities and NaN in keys, and the largest values, that the mask hides."""
    new, old = [150], [20]
    q, k, v = inputs(new, old, 8, 2, 128, BF16, 5)
    want = run(q, k, v, new, old, 0.09)
    k[120:, 0], k[120:, 1], v[120:] = float("inf"), float("nan"), torch.finfo(BF16).max
    got = run(q, k, v, new, old, 0.09)
    assert torch.equal(got[:100], want[:100])  # query 99 sees the keys up to 119


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (FP16, 64), (FP16, 128), (BF16, 64)])
@pytest.mark.parametrize("new,old,heads,kv_heads", [([150, 9], [20, 3], 8, 2), ([700, 33], [5, 0], 16, 2), ([50] * 40, [i for i in range(40)], 16, 4),
                                                    ([1000, 70], [30, 90], 40, 8), ([1400, 70], [0, 5], 40, 8),
                                                    ([2200, 70], [0, 5], 40, 8)])
def test_values_behind_a_query_reach_it_in_no_way(ext, new, old, heads, kv_heads, dtype, dim):
    """Infinities and NaN among the values: the queries before them, and other columns, are what they were within the bound."""
    q, k, v = inputs(new, old, heads, kv_heads, dim, dtype, 21)
    want, bound = reference(q, k, v, new, old, -dim ** -0.5)
    starts = [sum(new[:s]) + sum(old[:s]) for s in range(len(new))]
    struck = torch.zeros(sum(new), heads, dim, dtype=torch.bool, device="cuda")
    q0 = 0
    for s, (n, o) in enumerate(zip(new, old)):
        for place, value, head, column in ((o + n // 2, float("inf"), 0, 7), (o + n - 1, float("nan"), kv_heads - 1, dim - 1),
                                           (o + n // 3, float("-inf"), kv_heads - 1, 33)):
            v[starts[s] + place, head, column] = value
            group = heads // kv_heads
            struck[q0 + place - o:q0 + n, head * group:(head + 1) * group, column] = True
        q0 += n
    got = run(q, k, v, new, old, -dim ** -0.5)
    assert not torch.isfinite(got[struck]).any()
    assert_within(torch.where(struck, 0, got), want.masked_fill(struck, 0), bound)


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (FP16, 64), (FP16, 128), (BF16, 64)])
@pytest.mark.parametrize("new,old,heads,kv_heads", [([300, 40], [30, 0], 8, 2), ([60, 90], [-20, 10], 8, 2), ([700, 33], [5, 0], 16, 2),
                                                    ([1000, 70], [30, 90], 28, 4), ([1000, 70], [30, 90], 40, 8),
                                                    ([50] * 40, [i for i in range(40)], 16, 4), ([2200, 70], [0, 5], 40, 8)])
def test_scores_of_minus_infinity(ext, new, old, heads, kv_heads, dtype, dim):
    """Two thirds of each sequence's keys score -infinity: a query that sees no others has no softmax and gets NaN, later ones
    are what the other keys make them, and one that sees no key at all still gets zeros."""
    q, k, v = inputs(new, old, heads, kv_heads, dim, dtype, 23)
    scale, group = dim ** -0.5, heads // kv_heads
    q[:, :, 3] = q[:, :, 3].abs() + 0.1
    want, bound = reference(q, k, v, new, old, scale)
    undefined = torch.zeros(sum(new), heads, dtype=torch.bool, device="cuda")
    q0 = k0 = 0
    for n, o in zip(new, old):
        struck = (n + o) * 2 // 3
        k[k0:k0 + struck, 0, 3] = float("-inf")
        first, blind = max(0, struck - o), max(0, -o)  # the first query with a finite score, the queries without a key
        undefined[q0 + blind:q0 + first, :group] = True
        for h in range(group):
            want[q0 + first:q0 + n, h], bound[q0 + first:q0 + n, h] = attention64(
                q[q0 + first:q0 + n, h], k[k0 + struck:k0 + n + o, 0], v[k0 + struck:k0 + n + o, 0], scale, first + o - struck)
        q0, k0 = q0 + n, k0 + n + o
    got = run(q, k, v, new, old, scale)
    assert torch.isnan(got[undefined]).all() and undefined.any()
    assert_within(got.masked_fill(undefined[..., None], 0), want.masked_fill(undefined[..., None], 0), bound)


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (FP16, 64), (FP16, 128), (BF16, 64)])
@pytest.mark.parametrize("new,old,heads,kv_heads", [([300, 40], [30, 0], 8, 2), ([700, 33], [5, 0], 16, 2), ([1000, 70], [30, 90], 28, 4),
                                                    ([1000, 70], [30, 90], 40, 8), ([50] * 40, [i for i in range(40)], 16, 4),
                                                    ([2200, 70], [0, 5], 40, 8), ([100], [9000], 8, 2)])
def test_the_largest_values(ext, new, old, heads, kv_heads, dtype, dim):
    """Values of the type's largest magnitude, all of one sign or of both, give finite averages, also to the queries that are
    computed again because the last key's value is infinite."""
    q, k, v = inputs(new, old, heads, kv_heads, dim, dtype, 29)
    v.copy_(torch.where(v > 0, torch.finfo(dtype).max, -torch.finfo(dtype).max))
    v[..., dim // 2:] = torch.finfo(dtype).max
    want, bound = reference(q, k, v, new, old, dim ** -0.5)
    assert_within(run(q, k, v, new, old, dim ** -0.5), want, bound)
    ends = torch.tensor(new).cumsum(0) - 1
    v[(torch.tensor(new) + torch.tensor(old)).cumsum(0) - 1, 0, 5] = float("inf")
    got = run(q, k, v, new, old, dim ** -0.5)
    group = heads // kv_heads
    assert not torch.isfinite(got[ends, :group, 5]).any()
    got[ends, :group, 5] = want[ends, :group, 5].to(dtype)
    assert_within(got, want, bound)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,old,heads,kv_heads", [([300, 40], [30, 0], 8, 2), ([50] * 40, [i for i in range(40)], 16, 4), ([100], [9000], 8, 2)])
def test_small_values_keep_their_bits(ext, new, old, heads, kv_heads, dim):
    """Values of 2^-100: the power of two that keeps sums of the largest values finite does not cost them any."""
    q, k, v = inputs(new, old, heads, kv_heads, dim, BF16, 31)
    v.mul_(2.0 ** -100)
    assert_within(run(q, k, v, new, old, dim ** -0.5), *reference(q, k, v, new, old, dim ** -0.5))


def test_views_that_agree_with_the_packed_call(ext):
    """The same rows at other strides and offsets, and an output with gaps, give the same bits."""
    new, old = [130, 40], [3, 60]
    q, k, v = inputs(new, old, 6, 2, 64, FP16, 7)
    want = run(q.contiguous(), k.contiguous(), v.contiguous(), new, old, 0.1)
    assert torch.equal(run(q, k, v, new, old, 0.1), want)
    wide = torch.full((170, 6, 80), 9.0, dtype=FP16, device="cuda")
    run(q, k.transpose(0, 1).contiguous().transpose(0, 1), v, new, old, 0.1, out=wide[:, :, 4:68])
    assert torch.equal(wide[:, :, 4:68], want) and (wide[:, :, :4] == 9).all() and (wide[:, :, 68:] == 9).all()


@pytest.mark.parametrize("old", [0, 40])
@pytest.mark.parametrize("heads", [1, 4])
def test_strides_of_dimensions_of_one(ext, heads, old):
    """One query, one head, one key: whatever stride the tensor names there."""
    q, k, v = (t.contiguous() for t in inputs([1], [old], heads, 1, 64, BF16, 19))
    want = run(q, k, v, [1], [old], 0.1)
    odd = [t.as_strided(t.shape, [s if n > 1 else o for n, s, o in zip(t.shape, t.stride(), (3, 5, 1))]) for t in (q, k, v)]
    far = [t.as_strided(t.shape, [s if n > 1 else 1 << 40 for n, s in zip(t.shape, t.stride())]) for t in (q, k, v)]
    for views in (odd, far):
        out = torch.zeros_like(want)
        run(*views, [1], [old], 0.1, out=out.as_strided(out.shape, [views[0].stride(0), views[0].stride(1), 1]))
        assert torch.equal(out, want) and torch.isfinite(want).all() and want.any()


def test_heads_farther_apart_than_rows_may_be(ext):
    """Keys and values with the heads first: 2^24 elements and more between a token's heads."""
    keys = (1 << 24) // 128 + 100
    q, k, v = inputs([40], [keys - 40], 4, 2, 128, BF16, 17)
    k, v = k.contiguous(), v.contiguous()
    want = run(q, k, v, [40], [keys - 40], 0.1)
    first = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (k, v)]
    assert first[0].stride(1) > 1 << 24 and torch.equal(run(q, *first, [40], [keys - 40], 0.1), want)


@pytest.mark.parametrize("tokens", [1, 150])
def test_an_output_among_the_columns_of_its_inputs(ext, tokens):
    """q, k, v and the output side by side in one buffer run as apart; an output that shares a column with them is refused."""
    heads, kv_heads, dim = 6, 2, 64
    wide = torch.randn(tokens, 2 * heads + 2 * kv_heads, dim, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(BF16)
    q, k, v, out = wide.split([heads, kv_heads, kv_heads, heads], dim=1)
    want = run(q.clone(), k.clone(), v.clone(), [tokens], [0], 0.1)
    before = wide.clone()
    run(q, k, v, [tokens], [0], 0.1, out=out)
    assert torch.equal(out, want) and torch.equal(wide[:, :-heads], before[:, :-heads])
    for column in (0, 1, heads - 1, heads, heads + 2 * kv_heads - 1):
        with pytest.raises(_lib.TexelatorError, match="overlap"):
            run(q, k, v, [tokens], [0], 0.1, out=wide[:, column:column + heads])
    assert torch.equal(wide[:, :-heads], before[:, :-heads])


def test_sequence_starts_outside_the_rows(ext):
    """cu is data: starts past the arrays, below zero or falling are cut to them; nothing outside is written."""
    q, k, v = inputs([100], [0], 4, 2, 128, BF16, 9)
    out = torch.full((100, 4, 128), 9.0, dtype=BF16, device="cuda")
    layers.packed_attention(q, k, v, i32([-50, 40, 20, 10 ** 9]), 0.1, cu_k=i32([0, 40, 10 ** 9, -7]), out=out)
    want = run(q[:40], k[:40], v[:40], [40], [0], 0.1)
    assert torch.equal(out[:20], want[:20])  # the third sequence wrote rows 20 .. 99 as well
    assert not torch.isnan(out).any()


def test_a_captured_call_serves_other_lengths(ext):
    heads, kv_heads, dim = 8, 2, 128
    q, k, v = inputs([400], [200], heads, kv_heads, dim, BF16, 13)
    cu_q, cu_k = i32([0, 100, 100, 400]), i32([0, 150, 160, 600])
    out = torch.zeros(400, heads, dim, dtype=BF16, device="cuda")
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        layers.packed_attention(q, k, v, cu_q, 0.09, cu_k=cu_k, out=out)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            layers.packed_attention(q, k, v, cu_q, 0.09, cu_k=cu_k, out=out)
        for new, keys in (([100, 0, 300], [150, 10, 440]), ([1, 2, 3], [1, 2, 3]), ([400, 0, 0], [600, 0, 0]), ([0, 399, 1], [5, 500, 90])):
            cu_q.copy_(cumulative(new))
            cu_k.copy_(cumulative(keys))
            out.fill_(9.0)
            graph.replay()
            stream.synchronize()
            tokens, old = sum(new), [m - n for m, n in zip(keys, new)]
            assert_within(out[:tokens], *reference(q, k, v, new, old, 0.09))
            assert (out[tokens:] == 9).all()


def test_wrong_tensors_are_refused(ext):
    q = torch.zeros(10, 4, 64, dtype=BF16, device="cuda")
    k, cu = torch.zeros(10, 2, 64, dtype=BF16, device="cuda"), i32([0, 4, 10])
    good = (q, k, k, cu, 0.1)
    layers.packed_attention(*good)
    for position, bad in [(0, q.float()), (0, q.cpu()), (0, q[:, :3]), (0, q[0]), (0, q.transpose(1, 2)), (1, k.half()), (1, k[:, :0]), (1, k[:9]),
                          (1, k.cpu()), (2, k[:9]), (2, k[:, :1]), (2, k[:, :, :32]), (3, cu.long()), (3, cu.cpu()), (3, cu[:0]), (3, cu[::2])]:
        with pytest.raises(_lib.TexelatorError):
            layers.packed_attention(*good[:position], bad, *good[position + 1:])
    for more in (dict(cu_k=cu[:2]), dict(cu_k=cu.long()), dict(out=q[:9]), dict(out=q.half())):
        with pytest.raises(_lib.TexelatorError):
            layers.packed_attention(*good, **more)
    off = torch.zeros(10 * 4 * 64 + 4, dtype=BF16, device="cuda")[4:].view(10, 4, 64)
    with pytest.raises(_lib.TexelatorError, match="aligned"):
        layers.packed_attention(off, k, k, cu, 0.1)
    assert layers.packed_attention(q[:0], k[:0], k[:0], i32([0]), 0.1).shape == (0, 4, 64)
    none = layers.packed_attention(q, k[:0], k[:0], cu, 0.1, cu_k=i32([0, 0, 0]))
    assert none.shape == q.shape and not none.any()
