"""The entry points of a drafted step refuse what their kernels cannot run, before any launch (no GPU needed)."""
from __future__ import annotations

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from texelator_amd import _lib, layers

P = 1 << 20  # an address that is never read: every call here is refused
FAR = 1 << 40
POOL = dict(pages=P, num_pages=9, kv_heads=2, head_dim=128, page_size=64, block_table=P, table_stride=5, max_pages=5, lengths=P,
            sequences=3)
POOL_FAULTS = [dict(pages=None), dict(pages=P + 8), dict(num_pages=0), dict(num_pages=1 << 31), dict(kv_heads=0), dict(head_dim=96),
               dict(page_size=48), dict(page_size=8), dict(page_size=2048), dict(block_table=None), dict(block_table=P + 2),
               dict(table_stride=-1), dict(max_pages=0), dict(max_pages=1 << 25), dict(lengths=None), dict(lengths=P + 1),
               dict(sequences=-1), dict(sequences=65536)]


def call(name, arguments, change):
    assert set(change) <= set(arguments)
    return name, {**arguments, **change}


def rope(**change):
    return call("tx_kv4_append_rope", dict(
        q=P, q_token=2048, q_head=128, k=2 * P, k_token=256, k_head=128, v=3 * P, v_token=256, v_head=128, dtype=1, tokens=7, heads=16,
        cos=P, cos_row=64, sin=P, sin_row=64, table_rows=100, rotary=128, interleaved=0, positions=P, cu=P, **POOL, q_out=FAR,
        q_out_token=2048, q_out_head=128, k_out=2 * FAR, k_out_token=256, k_out_head=128, device=0, stream=None), change)


def tree(**change):
    return call("tx_kv4_tree_attention", dict(
        q=P, q_token=2048, q_head=128, dtype=1, tokens=20, heads=16, cu=P, parents=P, **POOL, scale=0.1, workspace=P,
        workspace_bytes=1 << 40, out=FAR, out_token=2048, out_head=128, device=0, stream=None), change)


def verify(**change):
    return call("tx_verify_drafts", dict(
        logits=P, logits_row=1000, draft_logits=None, draft_row=1000, dtype=1, tokens=20, vocab=1000, ids=2 * P, uniforms=2 * P, cu=2 * P,
        parents=2 * P, sequences=3, temperatures=2 * P, temperature=1.0, workspace=3 * P, workspace_bytes=1 << 24, accepted=FAR,
        path=2 * FAR, next=3 * FAR, device=0, stream=None), change)


def keep(**change):
    a = dict(pages=P, layers=2, **{k: v for k, v in POOL.items() if k != "pages"}, cu=2 * P, tokens=20, path=3 * P, accepted=4 * P,
             lengths_out=FAR, device=0, stream=None)
    return call("tx_kv4_keep_path", a, change)


REFUSED = [
    *(rope(**c) for c in [
        *POOL_FAULTS, dict(q=None), dict(k=None), dict(v=None), dict(q_out=None), dict(cos=None), dict(sin=None), dict(dtype=2),
        dict(heads=0), dict(heads=40000), dict(tokens=-1), dict(tokens=1 << 31), dict(cu=None), dict(cu=P + 2), dict(q=P + 8),
        dict(k=P + 8), dict(v=P + 2), dict(q_out=FAR + 8), dict(k_out=FAR + 4), dict(q_token=2052), dict(q_head=4), dict(k_token=260),
        dict(v_head=4), dict(q_out_token=2052), dict(q_out_head=132), dict(k_out_token=4), dict(q_head=-128), dict(k_out_head=-128),
        dict(rotary=0), dict(rotary=-16), dict(rotary=144), dict(rotary=24), dict(rotary=128, head_dim=64), dict(cos=P + 2), dict(sin=P + 1),
        dict(positions=P + 2), dict(cos_row=-1), dict(sin_row=-64), dict(table_rows=-1), dict(table_rows=1 << 31),
        dict(q_out=P), dict(q_out=P + 256, q_out_head=256), dict(q_out=2 * P), dict(q_out=3 * P), dict(k_out=P), dict(k_out=2 * P),
        dict(k_out=3 * P), dict(k_out=FAR)]),
    *(tree(**c) for c in [
        *POOL_FAULTS, dict(q=None), dict(out=None), dict(cu=None), dict(cu=P + 2), dict(parents=P + 1), dict(dtype=2), dict(heads=15),
        dict(heads=0), dict(heads=1 << 17), dict(tokens=-1), dict(tokens=(1 << 22) + 1), dict(q=P + 8), dict(q_head=60), dict(q_token=4),
        dict(q_token=-8), dict(out=FAR + 4), dict(out_head=2), dict(out_token=-4), dict(workspace=P + 8), dict(workspace=None, max_pages=500),
        dict(workspace_bytes=64, max_pages=500), dict(out=P), dict(out=P + 4096 * 19), dict(max_pages=1 << 24, sequences=4096),
        dict(max_pages=1, sequences=32768, kv_heads=512, heads=512)]),
    *(verify(**c) for c in [
        dict(logits=None), dict(ids=None), dict(uniforms=None), dict(cu=None), dict(accepted=None), dict(path=None), dict(next=None),
        dict(dtype=3), dict(tokens=-1), dict(tokens=65536), dict(sequences=-1), dict(sequences=65536), dict(vocab=0),
        dict(vocab=(1 << 24) + 1), dict(draft_logits=P), dict(logits=P + 1), dict(dtype=2, logits=P + 2), dict(logits_row=-1),
        dict(draft_row=-1), dict(ids=P + 4), dict(next=FAR + 4), dict(uniforms=P + 2), dict(temperatures=P + 2), dict(cu=P + 2),
        dict(parents=P + 2), dict(accepted=FAR + 2), dict(path=FAR + 1), dict(workspace=P + 8), dict(workspace=None),
        dict(workspace_bytes=64), dict(next=2 * P), dict(path=2 * P), dict(accepted=2 * P + 8), dict(next=P + 2 * 1000 * 19),
        dict(path=3 * P + 16), dict(path=FAR), dict(next=2 * FAR), dict(next=FAR + 8)]),
    *(keep(**c) for c in [
        *POOL_FAULTS, dict(layers=0), dict(layers=65536), dict(cu=None), dict(cu=P + 2), dict(path=None), dict(path=P + 2), dict(accepted=None),
        dict(accepted=P + 1), dict(lengths_out=None), dict(lengths_out=FAR + 2), dict(tokens=-1), dict(tokens=1 << 23), dict(lengths_out=P),
        dict(lengths_out=P + 8), dict(lengths_out=2 * P + 12), dict(lengths_out=3 * P + 76), dict(lengths_out=4 * P)]),
]


@pytest.mark.parametrize("refused", REFUSED, ids=lambda c: c[0])
def test_bad_arguments_are_refused_before_any_launch(refused):
    name, arguments = refused
    lib = _lib.load()
    assert getattr(lib, name)(*arguments.values()) == _lib.TX_ERR_INVALID, arguments
    assert lib.tx_last_error().startswith(name[3:].encode() + b": ")


def test_empty_calls_launch_nothing():
    lib = _lib.load()
    for name, arguments in [rope(tokens=0), rope(sequences=0), tree(tokens=0), tree(sequences=0), keep(sequences=0), verify(sequences=0)]:
        assert getattr(lib, name)(*arguments.values()) == _lib.TX_OK, name


def test_sizes_of_workspaces():
    """They follow the shapes; shapes that the calls refuse have none."""
    lib, out = _lib.load(), ctypes.c_int64()
    # Many sequences of at most 320 positions are not cut.
    assert lib.tx_kv4_tree_attention_workspace(2000, 20, 16, 2, 128, 64, 5, 0, out) == _lib.TX_OK and out.value == 0
    assert lib.tx_kv4_tree_attention_workspace(3, 20, 16, 2, 128, 64, 5, 0, out) == _lib.TX_OK and out.value > 0
    sizes = []
    for tokens in (1, 4, 8, 64, 6000):
        assert lib.tx_kv4_tree_attention_workspace(3, tokens, 16, 2, 128, 64, 500, 0, out) == _lib.TX_OK
        sizes.append(out.value)
    assert sizes == sorted(sizes) and sizes[0] > 0 and all(n % 16 == 0 for n in sizes)
    for bad in ((3, 20, 15, 2, 128, 64, 5), (3, 20, 1 << 14, 2, 128, 64, 5), (3, -1, 16, 2, 128, 64, 5), (3, 20, 16, 2, 96, 64, 5), (-1, 20, 16, 2, 128, 64, 5),
                (4096, 20, 16, 2, 128, 1024, 1 << 20)):
        assert lib.tx_kv4_tree_attention_workspace(*bad, 0, out) == _lib.TX_ERR_INVALID
    assert lib.tx_kv4_tree_attention_workspace(3, 20, 16, 2, 128, 64, 5, 0, None) == _lib.TX_ERR_INVALID
    assert lib.tx_verify_drafts_workspace(1, 20, 1000, 3, 0, 0, out) == _lib.TX_OK
    plain = out.value
    assert lib.tx_verify_drafts_workspace(1, 20, 1000, 3, 1, 0, out) == _lib.TX_OK and out.value > plain > 0
    for bad in ((3, 20, 1000, 3, 0), (1, -1, 1000, 3, 0), (1, 20, 0, 3, 0), (1, 20, 1000, -1, 0)):
        assert lib.tx_verify_drafts_workspace(*bad, 0, out) == _lib.TX_ERR_INVALID
    assert lib.tx_verify_drafts_workspace(1, 20, 1000, 3, 0, 0, None) == _lib.TX_ERR_INVALID


@pytest.mark.parametrize("sequences,tokens,heads,kv_heads,dim,page_size,max_pages", [
    (1024, 6144, 64, 8, 128, 1024, 1024), (4096, 20000, 32, 8, 64, 256, 2048), (6, 157, 128, 2, 128, 1024, 1 << 20), (1, 64, 4096, 1, 128, 1024, 1 << 20)])
def test_tables_with_room_for_long_sequences(sequences, tokens, heads, kv_heads, dim, page_size, max_pages):
    """What single tokens' attention takes, a drafted step takes: how many rows a sequence could have is no reason to refuse the few it has."""
    lib, out = _lib.load(), ctypes.c_int64()
    assert lib.tx_kv4_attention_workspace(sequences, heads, kv_heads, dim, page_size, max_pages, 0, out) == _lib.TX_OK
    assert lib.tx_kv4_tree_attention_workspace(sequences, tokens, heads, kv_heads, dim, page_size, max_pages, 0, out) == _lib.TX_OK
    assert 0 < out.value < 1 << 30


def test_tensors_are_checked(monkeypatch):
    """Wrong types, shapes and strides never reach the native call."""
    monkeypatch.setattr(_lib, "load", lambda: pytest.fail("reached the native call"))
    with FakeTensorMode():
        def new(*shape, dtype=torch.bfloat16, device="cuda:0"):
            return torch.empty(shape, dtype=dtype, device=device)

        def ints(n, dtype=torch.int32, device="cuda:0"):
            return torch.empty(n, dtype=dtype, device=device)

        pages, table, lengths, cu = new(4, 2, 2, 544, dtype=torch.uint8), ints((3, 2)), ints(3), ints(4)
        q, k = new(7, 6, 64), new(7, 2, 64)
        cos = new(9, 32, dtype=torch.float32)
        good = dict(q=q, k=k, v=k, cos=cos, sin=cos, pages=pages, block_table=table, lengths=lengths, cu=cu)
        for change in [dict(q=q[:6]), dict(q=q.float()), dict(q=q.half()), dict(q=new(7, 6, 64, device="cpu")), dict(q=q[0]), dict(q=q[:, :0]),
                       dict(q=new(7, 6, 128)), dict(q=new(7, 64, 6).transpose(1, 2)), dict(k=k[:, :1]), dict(v=k.half()), dict(cu=ints(3)),
                       dict(cu=None), dict(cos=cos.double()), dict(cos=cos[0]), dict(sin=cos[:8]), dict(cos=new(9, 32, dtype=torch.float32, device="cpu")),
                       dict(cos=new(32, 9, dtype=torch.float32).t()), dict(positions=ints(6)), dict(positions=ints(7, torch.int64)),
                       dict(out=q[:6]), dict(out=q.half()), dict(k_out=q), dict(k_out=k[:6]), dict(pages=pages.short()), dict(lengths=lengths.long()),
                       dict(block_table=table[0])]:
            with pytest.raises(_lib.TexelatorError):
                layers.kv4_append_rope(**{**good, **change})
        good = dict(q=q, pages=pages, block_table=table, lengths=lengths, cu=cu, scale=1.0)
        for change in [dict(q=q.float()), dict(q=q[:, :5]), dict(q=q[:, :0]), dict(q=q[0]), dict(cu=ints(3)),
                       dict(cu=ints(4, torch.int64)), dict(parents=ints(6)), dict(parents=ints(7, device="cpu")), dict(out=q[:, :4]),
                       dict(out=q[:5]), dict(workspace=new(100, device="cpu")), dict(workspace=new(100, 2)[:, 0]), dict(pages=pages[0]),
                       dict(lengths=ints(2))]:
            with pytest.raises(_lib.TexelatorError):
                layers.kv4_tree_attention(**{**good, **change})
        logits, ids, uniforms = new(7, 50), ints(7, torch.int64), ints(7, torch.float32)
        good = dict(logits=logits, ids=ids, uniforms=uniforms, cu=cu)
        for change in [dict(logits=logits.double()), dict(logits=logits[0]), dict(logits=new(50, 7).t()), dict(logits=new(7, 50, device="cpu")),
                       dict(ids=ids[:6]), dict(ids=ids.int()), dict(ids=ints(14, torch.int64)[::2]), dict(uniforms=uniforms.double()),
                       dict(uniforms=uniforms[:6]), dict(cu=cu.long()), dict(cu=cu[:0]), dict(parents=ints(6)), dict(parents=ints(7), draft_logits=logits),
                       dict(draft_logits=logits.float()), dict(draft_logits=logits[:6]), dict(temperature=ints(2, torch.float32)),
                       dict(temperature=ints(3, torch.float64)), dict(out=(ints(2), ints(7), ids)), dict(out=(ints(3), ints(6), ids)),
                       dict(out=(ints(3), ints(7), ints(7))), dict(workspace=new(100, device="cpu"))]:
            with pytest.raises(_lib.TexelatorError):
                layers.verify_drafts(**{**good, **change})
        good = dict(pages=pages, block_table=table, lengths=lengths, cu=cu, path=ints(7), accepted=ints(3), head_dim=64)
        for change in [dict(pages=pages.short()), dict(pages=pages[0]), dict(pages=pages[:, :, :1]), dict(pages=new(0, 4, 2, 2, 544, dtype=torch.uint8)),
                       dict(pages=new(1, 3, 4, 2, 2, 544, dtype=torch.uint8)), dict(head_dim=96), dict(head_dim=128, pages=new(4, 2, 2, 545, dtype=torch.uint8)),
                       dict(cu=ints(3)), dict(path=ids), dict(path=ints((7, 1))), dict(accepted=ints(2)), dict(out=ints(2)), dict(out=ints(3, torch.int64))]:
            with pytest.raises(_lib.TexelatorError):
                layers.kv4_keep_path(**{**good, **change})
        for call_bytes in (lambda: layers.kv4_tree_attention_workspace_bytes(pages, lengths, 7, 6, 64),
                           lambda: layers.kv4_tree_attention_workspace_bytes(pages, table, 7, 6, 96),
                           lambda: layers.verify_drafts_workspace_bytes(logits[0], 3), lambda: layers.verify_drafts_workspace_bytes(logits.int(), 3)):
            with pytest.raises(_lib.TexelatorError):
                call_bytes()
