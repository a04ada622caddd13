"""The entry points for several sequences refuse what their kernels cannot run, before any launch (no GPU needed)."""
from __future__ import annotations

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from texelator_amd import _lib, layers

P = 4096  # an address that is never read: every call here is refused


def packed(**change):
    a = dict(q=P, q_token=2048, q_head=128, k=P, k_token=256, k_head=128, v=P, v_token=256, v_head=128, dtype=1, heads=16,
             kv_heads=2, head_dim=128, cu_q=P, cu_k=P, sequences=3, total_q=10, total_k=10, scale=0.1, out=P, out_token=2048,
             out_head=128, device=0, stream=None)
    assert set(change) <= set(a)
    return "tx_packed_attention", {**a, **change}


POOL = dict(pages=P, num_pages=9, kv_heads=2, head_dim=128, page_size=64, block_table=P, table_stride=5, max_pages=5, lengths=P,
            sequences=3)


def rows(name, **change):
    a = dict(k=P, k_token=256, k_head=128, v=P, v_token=256, v_head=128, dtype=1, tokens=7, cu=P, **POOL, device=0, stream=None)
    assert set(change) <= set(a)
    return name, {**a, **change}


def attend(**change):
    a = dict(q=P, q_sequence=2048, q_head=128, dtype=1, heads=16, **POOL, scale=0.1, workspace=P, workspace_bytes=1 << 40, out=P,
             out_sequence=2048, out_head=128, device=0, stream=None)
    assert set(change) <= set(a)
    return "tx_kv4_attention", {**a, **change}


POOL_FAULTS = [dict(pages=None), dict(pages=P + 8), dict(num_pages=0), dict(num_pages=1 << 31), dict(kv_heads=0), dict(head_dim=96),
               dict(head_dim=32), dict(page_size=48), dict(page_size=8), dict(page_size=2048), dict(block_table=None),
               dict(block_table=P + 2), dict(table_stride=-1), dict(max_pages=0), dict(max_pages=1 << 25), dict(lengths=None),
               dict(lengths=P + 1), dict(sequences=-1), dict(sequences=65536)]
REFUSED = [
    *(packed(**c) for c in [
        dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(cu_q=None), dict(cu_k=None), dict(dtype=2), dict(head_dim=96),
        dict(heads=15), dict(heads=0), dict(kv_heads=0), dict(sequences=-1), dict(sequences=65536), dict(total_q=-1), dict(total_k=-1),
        dict(total_q=(1 << 28) + 1), dict(total_q=1 << 28, heads=1024), dict(sequences=65535, heads=512), dict(q=P + 2), dict(k=P + 8), dict(v=P + 4), dict(q_token=2052),
        dict(k_token=260), dict(v_head=4), dict(q_head=-128), dict(k_token=1 << 25), dict(k_token=64), dict(v_token=0), dict(out=P + 4),
        dict(out_token=2049), dict(out_head=2), dict(cu_q=P + 2), dict(cu_k=P + 1)]),
    *(rows(name, **c) for name in ("tx_kv4_append", "tx_kv4_read") for c in [
        *POOL_FAULTS, dict(k=None), dict(v=None), dict(dtype=2), dict(tokens=-1), dict(tokens=1 << 31), dict(cu=None), dict(k=P + 8),
        dict(v=P + 2), dict(k_token=260), dict(v_head=4), dict(cu=P + 2)]),
    *(attend(**c) for c in [
        *POOL_FAULTS, dict(q=None), dict(out=None), dict(workspace=None, max_pages=500), dict(dtype=2), dict(heads=15), dict(heads=0), dict(q=P + 8),
        dict(q_head=60), dict(q_sequence=4), dict(out=P + 4), dict(out_head=2), dict(workspace=P + 8), dict(workspace_bytes=64, max_pages=500),
        dict(max_pages=1 << 24, sequences=4096, kv_heads=16), dict(max_pages=1, sequences=32768, kv_heads=512, heads=512)]),
]


@pytest.mark.parametrize("call", REFUSED, ids=lambda c: c[0])
def test_bad_arguments_are_refused_before_any_launch(call):
    name, arguments = call
    lib = _lib.load()
    assert getattr(lib, name)(*arguments.values()) == _lib.TX_ERR_INVALID, arguments
    assert lib.tx_last_error().startswith(name[3:].encode() + b": ")


def test_empty_calls_launch_nothing():
    lib = _lib.load()
    for name, arguments in [packed(sequences=0), packed(total_q=0), rows("tx_kv4_append", tokens=0),
                            rows("tx_kv4_read", sequences=0), attend(sequences=0)]:
        assert getattr(lib, name)(*arguments.values()) == _lib.TX_OK


def copy(src, dst, **change):
    a = dict(pages=P, layers=2, num_pages=9, page_bytes=544)
    a.update(change)
    ids = ctypes.c_int64 * max(1, len(src))
    return _lib.load().tx_kv4_copy_pages(a["pages"], a["layers"], a["num_pages"], a["page_bytes"], ids(*src), ids(*dst), len(src), 0, None)


@pytest.mark.parametrize("src,dst,change,message", [
    ([0, 1], [2, 2], {}, b"copied to twice"), ([0, 1], [1, 2], {}, b"both"), ([3], [3], {}, b"both"), ([2, 1], [1, 2], {}, b"both"),
    ([0], [9], {}, b"outside"), ([9], [0], {}, b"outside"), ([-1], [0], {}, b"outside"), ([0], [-1], {}, b"outside"),
    ([0], [1], dict(pages=None), b"null"), ([0], [1], dict(pages=P + 8), b"aligned"), ([0], [1], dict(page_bytes=520), b"16 bytes"),
    ([0], [1], dict(layers=0), b"pages"), ([0] * 10, list(range(10)), {}, b"more copies"),
])
def test_copies_that_depend_on_their_order_are_refused(src, dst, change, message):
    assert copy(src, dst, **change) == _lib.TX_ERR_INVALID
    assert message in _lib.load().tx_last_error()


@pytest.mark.parametrize("src,dst,message", [([5, 1], [2 ** 30, 2 ** 30], b"copied to twice"), ([7, 2 ** 30], [2 ** 30, 3], b"both"),
                                             ([0], [2 ** 31 - 2], b"outside")])
def test_the_same_for_a_pool_far_larger_than_the_lists(src, dst, message):
    assert copy(src, dst, num_pages=2 ** 31 - 2) == _lib.TX_ERR_INVALID
    assert message in _lib.load().tx_last_error()


def test_no_copies_launch_nothing():
    assert copy([], []) == _lib.TX_OK


def test_tensors_are_checked():
    pages = layers.kv4_pages(4, 2, 64, 16, device="cpu")
    assert pages.shape == (4, 2, 2, 544) and pages.dtype == torch.uint8
    assert layers.kv4_pages(4, 2, 128, 32, layers=3, device="cpu").shape == (3, 4, 2, 2, 2176)
    for bad in [(0, 2, 64, 16), (4, 0, 64, 16), (4, 2, 96, 16), (4, 2, 64, 24), (4, 2, 64, 8), (4, 2, 64, 2048)]:
        with pytest.raises(_lib.TexelatorError):
            layers.kv4_pages(*bad, device="cpu")
    k = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    table, lengths = torch.zeros(3, 2, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    for call in (lambda: layers.kv4_append(k, k, pages, table, lengths), lambda: layers.kv4_read(pages, table, lengths, 64),
                 lambda: layers.kv4_attention(k, pages, table, lengths, 1.0), lambda: layers.kv4_copy_pages(pages, [0], [1]),
                 lambda: layers.packed_attention(k, k, k, lengths, 1.0)):
        with pytest.raises(_lib.TexelatorError, match="CUDA"):
            call()


@pytest.mark.parametrize("shape", [(4, 2, 1, 544), (3, 4, 2, 1, 544), (4, 2, 3, 544), (2, 2, 544), (1, 3, 4, 2, 2, 544)])
def test_copies_in_pools_of_another_shape_are_refused(shape, monkeypatch):
    """The bytes of a page follow from the shape, so one without keys and values both never reaches the native call."""
    calls = []
    monkeypatch.setattr(_lib, "load", lambda: calls.append(shape))
    with FakeTensorMode():
        pages = torch.empty(shape, dtype=torch.uint8, device="cuda:0")
    with pytest.raises(_lib.TexelatorError, match="kv_heads, 2, page bytes"):
        layers.kv4_copy_pages(pages, [0], [1])
    assert not calls


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("group", range(1, 18))
def test_pieces_of_the_workspace_are_whole_vectors(head_dim, group):
    """Partial results, two for each workgroup, are accessed 16 bytes at a time: each begins on 16 bytes, with room for a query's output,
    maximum and sum."""
    lib, sizes = _lib.load(), []
    for heads in (4, group):  # of groups of four the size is exact: 4 (head_dim + 2) floats a piece
        size = ctypes.c_int64()
        assert lib.tx_kv4_attention_workspace(3, heads, 1, head_dim, 64, 500, 0, size) == _lib.TX_OK
        sizes.append(size.value)
    pieces, rest = divmod(sizes[0], 4 * (head_dim + 2) * 4)
    assert rest == 0 and pieces % 2 == 0 and pieces > 0
    piece, rest = divmod(sizes[1], pieces)
    assert rest == 0 and piece % 16 == 0 and 0 <= piece - group * (head_dim + 2) * 4 < 16


def test_shapes_without_heads_or_of_other_pools_are_refused(monkeypatch):
    """Pools without KV heads, layered ones, and sizes of rows that no pool has: the error of every other bad argument."""
    monkeypatch.setattr(_lib, "load", lambda: pytest.fail("reached the native call"))
    def pool(*shape):
        with FakeTensorMode():
            return torch.empty(shape, dtype=torch.uint8, device="cuda:0")

    with FakeTensorMode():
        table, lengths = (torch.empty(s, dtype=torch.int32, device="cuda:0") for s in ((3, 2), (3,)))
        q = torch.empty(3, 4, 64, dtype=torch.bfloat16, device="cuda:0")
    for pages in (pool(4, 0, 2, 544), pool(2, 4, 2, 2, 544), pool(4, 2, 1, 544), pool(4, 2, 2, 545)):
        with pytest.raises(_lib.TexelatorError, match="pages"):
            layers.kv4_attention(q, pages, table, lengths, 1.0)
        with pytest.raises(_lib.TexelatorError, match="pages"):
            layers.kv4_attention_workspace_bytes(pages, table, 4, 64)
    for head_dim in (0, 32, 96):
        with pytest.raises(_lib.TexelatorError, match="head_dim"):
            layers.kv4_attention_workspace_bytes(pool(4, 2, 2, 544), table, 4, head_dim)
    with pytest.raises(_lib.TexelatorError, match="block_table"):
        layers.kv4_attention_workspace_bytes(pool(4, 2, 2, 544), lengths, 4, 64)


FAR = 1 << 40  # away from everything else
# Rows of 40 heads of 128 of one buffer: q in the first 16, k in the next 2, v in the next 2, 20 heads between the rows' ends.
FUSED = dict(q=P, q_token=5120, k=P + 2 * 2048, k_token=5120, v=P + 2 * 2304, v_token=5120, out_token=5120)


@pytest.mark.parametrize("change", [
    dict(k=FAR, v=FAR, out=P), dict(q=FAR, v=2 * FAR, out=P), dict(q=FAR, k=2 * FAR, out=P),    # the same rows
    dict(k=FAR, v=FAR, out=P + 9 * 4096), dict(k=FAR, v=FAR, out=P + 8, out_head=64),           # the last row of q, the middle of one
    dict(k=FAR, v=FAR, out=P + 2048, out_token=4096),                                           # other strides within q's ends
    dict(FUSED, out=P + 2 * 2044), dict(FUSED, out=P + 2 * 2304), dict(FUSED, out=P + 2 * 5120 * 7),
    dict(FUSED, out=P + 2 * (5120 - 2048 + 128)), dict(FUSED, total_q=1, out=P + 2 * 5120 * 3 + 2 * 2048),
], ids=str)
def test_outputs_that_overlap_inputs_are_refused(change):
    name, arguments = packed(**change)
    lib = _lib.load()
    assert getattr(lib, name)(*arguments.values()) == _lib.TX_ERR_INVALID
    assert b"overlap q, k or v" in lib.tx_last_error()
