"""Decoder-layer helpers of ``libtexelator_hip.so`` on torch tensors (no reference counterpart:
the reference leaves these layers to Hugging Face modules; see ``include/texelator_hip.h``).

Every function checks shapes, dtypes and devices on the host before the launch, and launches on
the current stream. Nothing here allocates unless an output is not supplied.
"""
from __future__ import annotations

import array
import ctypes
import functools

import torch

from . import _lib
from ._hip import _stream_address
from ._hip import shape as _hip_shape
from ._lib import TexelatorError, check


# Plain integers: the declared argument types make them pointers, and an object per argument cost
# ~0.15 us each of a small call's host time.
def _ptr(t: torch.Tensor | None) -> int | None:
    return t.data_ptr() if t is not None else None


def _stream(t: torch.Tensor) -> int:
    return _stream_address(t.device)


def _expect(condition: bool, message: str) -> None:
    if not condition:
        raise TexelatorError(message)


def add_rmsnorm(residual: torch.Tensor, delta: torch.Tensor | None, weight: torch.Tensor, eps: float,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """``residual += delta`` (in place, fp32) then ``out = bf16(weight * bf16(rmsnorm(residual)))``."""
    _expect(residual.is_cuda and residual.dtype == torch.float32 and residual.is_contiguous() and residual.dim() == 2,
            "residual must be a contiguous CUDA float32 [rows, hidden]")
    rows, hidden = residual.shape
    _expect(weight.dtype == torch.bfloat16 and weight.is_contiguous() and weight.numel() == hidden, "weight must be bf16 [hidden]")
    if delta is not None:
        _expect(delta.dtype == torch.bfloat16 and delta.is_contiguous() and delta.shape == residual.shape,
                "delta must be a contiguous bf16 tensor shaped like the residual")
    if out is None:
        out = torch.empty((rows, hidden), dtype=torch.bfloat16, device=residual.device)
    _expect(out.dtype == torch.bfloat16 and out.is_contiguous() and out.shape == residual.shape, "bad output")
    check(_lib.load().tx_add_rmsnorm(_ptr(residual), _ptr(delta), _ptr(weight), float(eps), _ptr(out), rows, hidden,
                                     _stream(residual)))
    return out


def add_rmsnorm_bf16(residual: torch.Tensor, delta: torch.Tensor | None, weight: torch.Tensor,
                     eps: float) -> tuple[torch.Tensor | None, torch.Tensor]:
    """RMSNorm over a bf16 residual ``[..., hidden]`` kept in bf16: with ``delta``, ``(bf16(residual +
    delta), norm of that sum)`` (torch's bf16 add, then Hugging Face's RMSNorm roundings); without,
    ``(None, norm of residual)``. One launch; outputs shaped like ``residual``."""
    _expect(residual.is_cuda and residual.dtype == torch.bfloat16 and residual.is_contiguous()
            and residual.data_ptr() % 8 == 0, "residual must be a contiguous, 8-byte aligned CUDA bf16 tensor")
    hidden = residual.shape[-1]
    rows = residual.numel() // hidden if hidden else 0
    _expect(weight.is_cuda and weight.dtype == torch.bfloat16 and weight.is_contiguous() and weight.numel() == hidden,
            "weight must be bf16 [hidden]")
    total = None
    if delta is not None:
        _expect(delta.dtype == torch.bfloat16 and delta.is_contiguous() and delta.shape == residual.shape
                and delta.device == residual.device, "delta must be a contiguous bf16 tensor shaped like the residual")
        total = torch.empty_like(residual)
    out = torch.empty_like(residual)
    check(_lib.load().tx_add_rmsnorm_bf16(_ptr(residual), _ptr(delta), _ptr(weight), float(eps), _ptr(total), _ptr(out),
                                          rows, hidden, _stream(residual)))
    return total, out


def rope_kv_cache(qkv: torch.Tensor, positions: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, heads: int,
                  kv_heads: int, head_dim: int, k_cache: torch.Tensor, v_cache: torch.Tensor,
                  q_out: torch.Tensor | None = None) -> torch.Tensor:
    """RoPE on the q and k heads of packed ``[q | k | v]`` rows; k and v go into the caches at
    ``positions``; returns the rotated q ``[tokens, heads * head_dim]``."""
    _expect(qkv.dtype == torch.bfloat16 and qkv.dim() == 2 and qkv.stride(1) == 1, "qkv must be bf16 [tokens, width]")
    tokens = qkv.shape[0]
    _expect(qkv.shape[1] >= (heads + 2 * kv_heads) * head_dim, "qkv row too short for the heads")
    _expect(positions.dtype == torch.int64 and positions.is_contiguous() and positions.numel() == tokens,
            "positions must be int64 [tokens]")
    max_ctx = k_cache.shape[1]
    for cache in (k_cache, v_cache):
        _expect(cache.dtype == torch.bfloat16 and cache.is_contiguous() and tuple(cache.shape) == (kv_heads, max_ctx, head_dim),
                "caches must be contiguous bf16 [kv_heads, max_context, head_dim]")
    for table in (cos, sin):
        _expect(table.dtype == torch.float32 and table.is_contiguous() and tuple(table.shape) == (max_ctx, head_dim),
                "rope tables must be float32 [max_context, head_dim]")
    if q_out is None:
        q_out = torch.empty((tokens, heads * head_dim), dtype=torch.bfloat16, device=qkv.device)
    _expect(q_out.dtype == torch.bfloat16 and q_out.is_contiguous() and q_out.numel() == tokens * heads * head_dim, "bad q_out")
    check(_lib.load().tx_rope_kv_cache(_ptr(qkv), qkv.stride(0), tokens, _ptr(positions), _ptr(cos), _ptr(sin), heads,
                                       kv_heads, head_dim, _ptr(q_out), _ptr(k_cache), _ptr(v_cache), max_ctx,
                                       _stream(qkv)))
    return q_out


def decode_attention_supported(config) -> bool:
    """The fused decode attention handles head_dim 128 and at most 8 query heads per KV head."""
    return config.head_dim == 128 and config.heads % config.kv_heads == 0 and config.heads // config.kv_heads <= 8


def decode_attention_workspace_bytes(heads: int, length: int) -> int:
    out = ctypes.c_int64(0)
    check(_lib.load().tx_decode_attention_workspace(int(heads), int(length), out))
    return out.value


def decode_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, position: torch.Tensor, length: int,
                     heads: int, kv_heads: int, scale: float, workspace: torch.Tensor,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """One-token grouped-query attention over cache positions 0..position (device int64 [1])."""
    head_dim = k_cache.shape[2]
    _expect(q.dtype == torch.bfloat16 and q.is_contiguous() and q.numel() == heads * head_dim, "q must be bf16 [heads*head_dim]")
    _expect(position.dtype == torch.int64 and position.numel() == 1, "position must be int64 [1]")
    for cache in (k_cache, v_cache):
        _expect(cache.dtype == torch.bfloat16 and cache.is_contiguous() and cache.shape[0] == kv_heads, "bad cache")
    need = decode_attention_workspace_bytes(heads, length)
    _expect(workspace.is_cuda and workspace.numel() * workspace.element_size() >= need, "decode attention workspace too small")
    if out is None:
        out = torch.empty((1, heads * head_dim), dtype=torch.bfloat16, device=q.device)
    check(_lib.load().tx_decode_attention(_ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(position), int(length), heads,
                                          kv_heads, head_dim, k_cache.shape[1], float(scale), _ptr(workspace),
                                          workspace.numel() * workspace.element_size(), _ptr(out), _stream(q)))
    return out


def prefill_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, heads: int, kv_heads: int,
                      scale: float, out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal self-attention of a prompt: ``q`` bf16 ``[tokens, heads * head_dim]`` (rows 16-byte
    aligned) at positions 0..tokens-1 against cache rows 0..tokens-1 of ``k_cache``/``v_cache``
    (bf16 ``[kv_heads, max_context, head_dim]``). Returns bf16 ``[tokens, heads * head_dim]``."""
    _expect(q.is_cuda and q.dtype == torch.bfloat16 and q.dim() == 2 and q.stride(1) == 1, "q must be bf16 [tokens, width]")
    head_dim = k_cache.shape[2]
    tokens = q.shape[0]
    _expect(q.shape[1] == heads * head_dim, "q width must be heads * head_dim")
    for cache in (k_cache, v_cache):
        _expect(cache.dtype == torch.bfloat16 and cache.is_contiguous() and cache.shape[0] == kv_heads and
                cache.device == q.device, "bad cache")
    if out is None:
        out = torch.empty((tokens, heads * head_dim), dtype=torch.bfloat16, device=q.device)
    _expect(out.dtype == torch.bfloat16 and out.dim() == 2 and out.stride(1) == 1 and out.shape == (tokens, heads * head_dim),
            "bad output")
    check(_lib.load().tx_prefill_attention(_ptr(q), q.stride(0), _ptr(k_cache), _ptr(v_cache), tokens, heads, kv_heads,
                                           head_dim, k_cache.shape[1], float(scale), _ptr(out), out.stride(0),
                                           _stream(q)))
    return out


def decode_attention_split(qkv_handle: int, positions: torch.Tensor, rope_row: torch.Tensor, heads: int,
                           kv_heads: int, head_dim: int, k_cache: torch.Tensor, v_cache: torch.Tensor, length: int,
                           scale: float, workspace: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`rope_kv_cache_split` then :func:`decode_attention` with one kernel launch fewer
    (bit-identical to the two calls): one token whose ``[q | k | v]`` row is the last
    :func:`linear_split` of ``qkv_handle``; ``rope_row`` holds the RoPE tables' rows at
    ``positions[0]`` (fp32 ``[cos (head_dim) | sin (head_dim)]``). The key and value are written to
    the caches at ``positions[0]``."""
    _expect(positions.dtype == torch.int64 and positions.is_contiguous() and positions.numel() == 1,
            "positions must be int64 [1]")
    _expect(rope_row.dtype == torch.float32 and rope_row.is_contiguous() and rope_row.numel() == 2 * head_dim,
            "rope_row must be float32 [2 * head_dim]")
    max_ctx = k_cache.shape[1]
    for cache in (k_cache, v_cache):
        _expect(cache.dtype == torch.bfloat16 and cache.is_contiguous() and tuple(cache.shape) == (kv_heads, max_ctx, head_dim),
                "caches must be contiguous bf16 [kv_heads, max_context, head_dim]")
    need = decode_attention_workspace_bytes(heads, length)
    _expect(workspace.is_cuda and workspace.numel() * workspace.element_size() >= need, "decode attention workspace too small")
    if out is None:
        out = torch.empty((1, heads * head_dim), dtype=torch.bfloat16, device=k_cache.device)
    _expect(out.dtype == torch.bfloat16 and out.is_contiguous() and out.numel() == heads * head_dim, "bad out")
    check(_lib.load().tx_decode_attention_split(qkv_handle, _ptr(positions), _ptr(rope_row), int(length), heads,
                                                kv_heads, head_dim, _ptr(k_cache), _ptr(v_cache), max_ctx, float(scale),
                                                _ptr(workspace), workspace.numel() * workspace.element_size(),
                                                _ptr(out), _stream(positions)))
    return out


def decode_attention_o_split(qkv_handle: int, o_handle: int, positions: torch.Tensor, rope_row: torch.Tensor,
                             heads: int, kv_heads: int, head_dim: int, k_cache: torch.Tensor, v_cache: torch.Tensor,
                             length: int, scale: float, workspace: torch.Tensor) -> bool:
    """:func:`decode_attention_split` then :func:`linear_split` of ``o_handle`` on its output, with
    the attention's chunk merge done inside the o GEMV (one launch fewer, o's split-K partials
    bitwise the same; read them with :func:`add_rmsnorm_split`). Returns False, with nothing
    launched, where the merge does not fit the o GEMV (more than 16 chunks of 64 positions, too many
    heads per o split, a LUT handle): then make the two calls."""
    _expect(positions.dtype == torch.int64 and positions.is_contiguous() and positions.numel() == 1,
            "positions must be int64 [1]")
    _expect(rope_row.dtype == torch.float32 and rope_row.is_contiguous() and rope_row.numel() == 2 * head_dim,
            "rope_row must be float32 [2 * head_dim]")
    max_ctx = k_cache.shape[1]
    for cache in (k_cache, v_cache):
        _expect(cache.dtype == torch.bfloat16 and cache.is_contiguous() and tuple(cache.shape) == (kv_heads, max_ctx, head_dim),
                "caches must be contiguous bf16 [kv_heads, max_context, head_dim]")
    need = decode_attention_workspace_bytes(heads, length)
    _expect(workspace.is_cuda and workspace.numel() * workspace.element_size() >= need, "decode attention workspace too small")
    status = _lib.load().tx_decode_attention_o_split(qkv_handle, o_handle, _ptr(positions), _ptr(rope_row), int(length),
                                                    heads, kv_heads, head_dim, _ptr(k_cache), _ptr(v_cache), max_ctx,
                                                    float(scale), _ptr(workspace),
                                                    workspace.numel() * workspace.element_size(), _stream(positions))
    if status == _lib.TX_ERR_UNSUPPORTED:
        return False
    check(status)
    return True


def linear_split(handle: int, x: torch.Tensor) -> None:
    """One-token decode GEMV of ``handle`` (``x`` bf16 ``[K]``) whose output stays as split-K
    partials inside the handle, for :func:`add_rmsnorm_split` or :func:`rope_kv_cache_split`."""
    _expect(x.is_cuda and x.dtype == torch.bfloat16 and x.is_contiguous() and x.data_ptr() % 16 == 0,
            "x must be a contiguous, 16-byte aligned CUDA bf16 tensor")
    _expect(x.numel() == _hip_shape(handle)[1], "x has the wrong length for this handle")
    check(_lib.load().tx_linear_split(handle, _ptr(x), _stream(x)))


def linear_swiglu(handle: int, x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """``swiglu(linear(handle, x))`` for one token of a merged ``[gate | up]`` handle, in one kernel
    (bit-identical to the two calls). Raises ``UnsupportedError`` for a handle whose GEMV is split
    or in LUT mode."""
    _expect(x.is_cuda and x.dtype == torch.bfloat16 and x.is_contiguous() and x.data_ptr() % 16 == 0,
            "x must be a contiguous, 16-byte aligned CUDA bf16 tensor")
    m, k = _hip_shape(handle)
    _expect(x.numel() == k, "x has the wrong length for this handle")
    if out is None:
        out = torch.empty((1, m // 2), dtype=torch.bfloat16, device=x.device)
    _expect(out.dtype == torch.bfloat16 and out.is_contiguous() and out.numel() == m // 2, "bad output")
    check(_lib.load().tx_linear_swiglu(handle, _ptr(x), _ptr(out), _stream(x)))
    return out


def linear_add_bias(handle: int, x: torch.Tensor, bias: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """``linear(handle, x) + bias`` for one bf16 token and a separate bf16 bias ``[M]`` (the handle
    has none of its own): the GEMV's bf16 output plus the bias rounded again, bit for bit the two
    operations, in the GEMV's own launches. Returns ``[..., M]`` shaped like ``x``."""
    _expect(x.is_cuda and x.dtype == torch.bfloat16 and x.is_contiguous() and x.data_ptr() % 16 == 0,
            "x must be a contiguous, 16-byte aligned CUDA bf16 tensor")
    m, k = _hip_shape(handle)
    _expect(x.numel() == k and x.shape[-1] == k, "x must be one token of this handle's K")
    _expect(bias.is_cuda and bias.dtype == torch.bfloat16 and bias.is_contiguous() and bias.numel() == m,
            "bias must be a contiguous CUDA bf16 [M]")
    if out is None:
        out = torch.empty((*x.shape[:-1], m), dtype=torch.bfloat16, device=x.device)
    _expect(out.dtype == torch.bfloat16 and out.is_contiguous() and out.numel() == m, "bad output")
    check(_lib.load().tx_linear_add_bias(handle, _ptr(x), _ptr(bias), _ptr(out), _stream(x)))
    return out


def linear_swiglu_pair(gate: int, up: int, x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """``swiglu(linear(gate, x), linear(up, x))`` for one token over two handles of one shape, in one
    kernel: bit for bit :func:`linear_swiglu` of the merged ``[gate | up]`` handle. Raises
    ``UnsupportedError`` for LUT-mode handles or handles with a bias."""
    _expect(x.is_cuda and x.dtype == torch.bfloat16 and x.is_contiguous() and x.data_ptr() % 16 == 0,
            "x must be a contiguous, 16-byte aligned CUDA bf16 tensor")
    m, k = _hip_shape(gate)
    _expect(_hip_shape(up) == (m, k), "gate and up must have the same shape")
    _expect(x.numel() == k, "x has the wrong length for these handles")
    if out is None:
        out = torch.empty((1, m), dtype=torch.bfloat16, device=x.device)
    _expect(out.dtype == torch.bfloat16 and out.is_contiguous() and out.numel() == m, "bad output")
    check(_lib.load().tx_linear_swiglu_pair(gate, up, _ptr(x), _ptr(out), _stream(x)))
    return out


def _norm_args(residual_in: torch.Tensor, residual_out: torch.Tensor, weight: torch.Tensor, k: int) -> None:
    for name, t in (("residual_in", residual_in), ("residual_out", residual_out)):
        _expect(t.is_cuda and t.dtype == torch.float32 and t.is_contiguous() and t.numel() == k and t.data_ptr() % 16 == 0,
                f"{name} must be a contiguous, 16-byte aligned CUDA float32 row of K values")
    _expect(residual_in.data_ptr() != residual_out.data_ptr(), "residual_out must be another buffer than residual_in")
    _expect(weight.dtype == torch.bfloat16 and weight.is_contiguous() and weight.numel() == k and weight.data_ptr() % 16 == 0,
            "weight must be a contiguous, 16-byte aligned bf16 [K]")


def linear_split_norm(handle: int, residual_in: torch.Tensor, residual_out: torch.Tensor, delta_handle: int,
                      weight: torch.Tensor, eps: float) -> bool:
    """:func:`add_rmsnorm_split` of ``residual_in`` and ``delta_handle``'s last :func:`linear_split`,
    then :func:`linear_split` of ``handle`` on the result, in one launch: the GEMV's workgroups
    normalize their x themselves (bitwise the same partials) and the updated residual goes to
    ``residual_out``. Returns False, with nothing launched, where that does not fit the GEMV (K
    above 2048, a delta split more than 8 ways, a LUT handle, or too many workgroups); then make the
    two calls."""
    _norm_args(residual_in, residual_out, weight, _hip_shape(handle)[1])
    status = _lib.load().tx_linear_split_norm(handle, _ptr(residual_in), _ptr(residual_out), delta_handle, _ptr(weight),
                                             float(eps), _stream(residual_in))
    if status == _lib.TX_ERR_UNSUPPORTED:
        return False
    check(status)
    return True


def linear_split_embed_norm(handle: int, embed: torch.Tensor, token: torch.Tensor, residual_out: torch.Tensor,
                            weight: torch.Tensor, eps: float) -> bool:
    """The first layer's :func:`linear_split_norm`: ``residual_out`` = row ``token`` (device int64
    [1], clamped into the table) of the bf16 embedding table ``embed`` [vocab, K] in fp32, then
    :func:`add_rmsnorm` of it (no delta) and :func:`linear_split` of ``handle``, in one launch.
    False, with nothing launched, where that does not fit the GEMV."""
    k = _hip_shape(handle)[1]
    _expect(embed.is_cuda and embed.dtype == torch.bfloat16 and embed.is_contiguous() and embed.dim() == 2 and
            embed.shape[1] == k and embed.data_ptr() % 16 == 0, "embed must be a contiguous CUDA bf16 [vocab, K] table")
    _expect(token.dtype == torch.int64 and token.numel() == 1 and token.is_contiguous(), "token must be int64 [1]")
    _expect(residual_out.is_cuda and residual_out.dtype == torch.float32 and residual_out.is_contiguous() and
            residual_out.numel() == k and residual_out.data_ptr() % 16 == 0, "residual_out must be float32 [K]")
    _expect(weight.dtype == torch.bfloat16 and weight.is_contiguous() and weight.numel() == k and weight.data_ptr() % 16 == 0,
            "weight must be a contiguous, 16-byte aligned bf16 [K]")
    status = _lib.load().tx_linear_split_embed_norm(handle, _ptr(embed), embed.shape[0], _ptr(token), _ptr(residual_out),
                                                   _ptr(weight), float(eps), _stream(residual_out))
    if status == _lib.TX_ERR_UNSUPPORTED:
        return False
    check(status)
    return True


def linear_swiglu_norm(handle: int, residual_in: torch.Tensor, residual_out: torch.Tensor, delta_handle: int,
                       weight: torch.Tensor, eps: float, out: torch.Tensor) -> bool:
    """:func:`linear_split_norm` for :func:`linear_swiglu`: the add+RMSNorm of the residual and
    ``delta_handle``'s partials, then the gate|up GEMV with its SwiGLU epilogue into ``out``, in one
    launch; False, with nothing launched, where that does not fit."""
    m, k = _hip_shape(handle)
    _norm_args(residual_in, residual_out, weight, k)
    _expect(out.dtype == torch.bfloat16 and out.is_contiguous() and out.numel() == m // 2, "bad output")
    status = _lib.load().tx_linear_swiglu_norm(handle, _ptr(residual_in), _ptr(residual_out), delta_handle, _ptr(weight),
                                              float(eps), _ptr(out), _stream(residual_in))
    if status == _lib.TX_ERR_UNSUPPORTED:
        return False
    check(status)
    return True


def linear_swiglu_prefill(handle: int, x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """``swiglu(linear(handle, x))`` for a prefill-sized ``x`` [tokens, K] of a merged ``[gate | up]``
    handle, in one GEMM whose epilogue applies SwiGLU (bit-identical to the two calls). Raises
    ``UnsupportedError`` where the call's prefill would run the pair tile or the dense backend, or
    split K."""
    _expect(x.is_cuda and x.dtype == torch.bfloat16 and x.is_contiguous() and x.dim() == 2 and x.data_ptr() % 16 == 0,
            "x must be a contiguous, 16-byte aligned CUDA bf16 [tokens, K] tensor")
    m, k = _hip_shape(handle)
    _expect(x.shape[1] == k, "x has the wrong width for this handle")
    tokens = x.shape[0]
    if out is None:
        out = torch.empty((tokens, m // 2), dtype=torch.bfloat16, device=x.device)
    _expect(out.dtype == torch.bfloat16 and out.is_contiguous() and out.shape == (tokens, m // 2), "bad output")
    check(_lib.load().tx_linear_swiglu_prefill(handle, _ptr(x), tokens, _ptr(out), _stream(x)))
    return out


def prefill_plan(handle: int, tokens: int) -> int:
    """The faster path for a call of ``tokens`` tokens (``_lib.TX_PREFILL_*``): K whole (``linear``), partials
    (:func:`prefill_split` and a consumer), or split and summed (:func:`linear_into` and the plain helper)."""
    out = ctypes.c_int(0)
    check(_lib.load().tx_prefill_plan(handle, int(tokens), out))
    return out.value


def linear_into(handle: int, x: torch.Tensor, out: torch.Tensor, workspace: torch.Tensor) -> torch.Tensor:
    """``linear(handle, x)`` of a bf16 x [tokens, K] into ``out`` [tokens, M], with a workspace of
    ``workspace_bytes(handle, tokens)`` bytes the caller keeps between calls on one stream."""
    m, k = _hip_shape(handle)
    x_ptr, workspace_ptr = x.data_ptr(), workspace.data_ptr()
    _expect(x.is_cuda and x.dtype == torch.bfloat16 and x.is_contiguous() and x.dim() == 2 and x.shape[1] == k
            and x_ptr % 16 == 0, "x must be a contiguous, 16-byte aligned CUDA bf16 [tokens, K] tensor")
    tokens = x.shape[0]
    _expect(out.is_cuda and out.dtype == torch.bfloat16 and out.is_contiguous() and out.shape == (tokens, m),
            "out must be a contiguous CUDA bf16 [tokens, M]")
    _expect(workspace.is_cuda and workspace.is_contiguous() and workspace_ptr % 16 == 0,
            "workspace must be a contiguous, 16-byte aligned CUDA tensor")
    device = x.device
    check(_lib.load().tx_linear(handle, x_ptr, _lib.TX_DTYPE_BF16, tokens * k, k, device.index, out.data_ptr(), workspace_ptr,
                                workspace.nbytes, _stream_address(device)))
    return out


def prefill_split(handle: int, x: torch.Tensor, workspace: torch.Tensor) -> int:
    """The prefill GEMM of ``x`` [tokens, K] (bf16, at or above the handle's prefill threshold)
    leaving its fp32 K-split partials in ``workspace`` (at least ``workspace_bytes(handle, tokens)``
    bytes) for :func:`add_rmsnorm_prefill_split` or :func:`rope_kv_cache_prefill_split`; returns
    the split count. Raises ``UnsupportedError`` when the call does not split K or runs the dense
    backend (then :func:`linear` is the path)."""
    _expect(x.is_cuda and x.dtype == torch.bfloat16 and x.is_contiguous() and x.dim() == 2 and x.data_ptr() % 16 == 0,
            "x must be a contiguous, 16-byte aligned CUDA bf16 [tokens, K] tensor")
    _expect(x.shape[1] == _hip_shape(handle)[1], "x has the wrong width for this handle")
    _expect(workspace.is_cuda and workspace.is_contiguous() and workspace.data_ptr() % 16 == 0,
            "workspace must be a contiguous, 16-byte aligned CUDA tensor")
    splits = ctypes.c_int(0)
    check(_lib.load().tx_prefill_split(handle, _ptr(x), x.shape[0], _ptr(workspace),
                                       workspace.numel() * workspace.element_size(), ctypes.byref(splits), _stream(x)))
    return splits.value


def add_rmsnorm_prefill_split(residual: torch.Tensor, delta_handle: int, partials: torch.Tensor, weight: torch.Tensor,
                              eps: float, out: torch.Tensor) -> torch.Tensor:
    """:func:`add_rmsnorm` of ``tokens`` rows whose delta is ``linear(delta_handle, x)``, read from
    the partials :func:`prefill_split` left (bit-identical)."""
    _expect(residual.is_cuda and residual.dtype == torch.float32 and residual.is_contiguous() and residual.dim() == 2,
            "residual must be a contiguous CUDA float32 [tokens, hidden]")
    tokens, hidden = residual.shape
    _expect(_hip_shape(delta_handle)[0] == hidden, "the delta handle's output size must equal hidden")
    _expect(weight.dtype == torch.bfloat16 and weight.is_contiguous() and weight.numel() == hidden, "weight must be bf16 [hidden]")
    _expect(out.dtype == torch.bfloat16 and out.is_contiguous() and out.shape == residual.shape, "bad output")
    _expect(partials.is_cuda and partials.is_contiguous(), "partials must be the workspace prefill_split filled")
    check(_lib.load().tx_add_rmsnorm_prefill_split(_ptr(residual), delta_handle, _ptr(partials), tokens, _ptr(weight),
                                                   float(eps), _ptr(out), hidden, _stream(residual)))
    return out


def rope_kv_cache_prefill_split(qkv_handle: int, partials: torch.Tensor, positions: torch.Tensor, cos: torch.Tensor,
                                sin: torch.Tensor, heads: int, kv_heads: int, head_dim: int, k_cache: torch.Tensor,
                                v_cache: torch.Tensor, q_out: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`rope_kv_cache` of ``tokens`` tokens whose ``[q | k | v]`` rows are
    ``linear(qkv_handle, x)``, read from the partials :func:`prefill_split` left (bit-identical);
    returns the rotated q ``[tokens, heads * head_dim]``."""
    _expect(_hip_shape(qkv_handle)[0] >= (heads + 2 * kv_heads) * head_dim, "qkv handle too narrow for the heads")
    _expect(positions.dtype == torch.int64 and positions.is_contiguous() and positions.dim() == 1,
            "positions must be int64 [tokens]")
    tokens = positions.numel()
    max_ctx = k_cache.shape[1]
    for cache in (k_cache, v_cache):
        _expect(cache.dtype == torch.bfloat16 and cache.is_contiguous() and tuple(cache.shape) == (kv_heads, max_ctx, head_dim),
                "caches must be contiguous bf16 [kv_heads, max_context, head_dim]")
    for table in (cos, sin):
        _expect(table.dtype == torch.float32 and table.is_contiguous() and tuple(table.shape) == (max_ctx, head_dim),
                "rope tables must be float32 [max_context, head_dim]")
    _expect(partials.is_cuda and partials.is_contiguous(), "partials must be the workspace prefill_split filled")
    if q_out is None:
        q_out = torch.empty((tokens, heads * head_dim), dtype=torch.bfloat16, device=positions.device)
    _expect(q_out.dtype == torch.bfloat16 and q_out.is_contiguous() and q_out.numel() == tokens * heads * head_dim, "bad q_out")
    check(_lib.load().tx_rope_kv_cache_prefill_split(qkv_handle, _ptr(partials), tokens, _ptr(positions), _ptr(cos),
                                                     _ptr(sin), heads, kv_heads, head_dim, _ptr(q_out), _ptr(k_cache),
                                                     _ptr(v_cache), max_ctx, _stream(positions)))
    return q_out


def add_rmsnorm_split(residual: torch.Tensor, delta_handle: int, weight: torch.Tensor, eps: float,
                      out: torch.Tensor) -> torch.Tensor:
    """:func:`add_rmsnorm` of one row whose delta is the last :func:`linear_split` of ``delta_handle``."""
    _expect(residual.is_cuda and residual.dtype == torch.float32 and residual.is_contiguous() and residual.numel() ==
            weight.numel(), "residual must be a contiguous CUDA float32 row of hidden values")
    hidden = residual.numel()
    _expect(_hip_shape(delta_handle)[0] == hidden, "the delta handle's output size must equal hidden")
    _expect(weight.dtype == torch.bfloat16 and weight.is_contiguous(), "weight must be bf16 [hidden]")
    _expect(out.dtype == torch.bfloat16 and out.is_contiguous() and out.numel() == hidden, "bad output")
    check(_lib.load().tx_add_rmsnorm_split(_ptr(residual), delta_handle, _ptr(weight), float(eps), _ptr(out), hidden,
                                           _stream(residual)))
    return out


def rope_kv_cache_split(qkv_handle: int, positions: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, heads: int,
                        kv_heads: int, head_dim: int, k_cache: torch.Tensor, v_cache: torch.Tensor,
                        q_out: torch.Tensor) -> torch.Tensor:
    """:func:`rope_kv_cache` of one token whose ``[q | k | v]`` row is the last :func:`linear_split`
    of ``qkv_handle``."""
    _expect(_hip_shape(qkv_handle)[0] >= (heads + 2 * kv_heads) * head_dim, "qkv handle too narrow for the heads")
    _expect(positions.dtype == torch.int64 and positions.is_contiguous() and positions.numel() == 1,
            "positions must be int64 [1]")
    max_ctx = k_cache.shape[1]
    for cache in (k_cache, v_cache):
        _expect(cache.dtype == torch.bfloat16 and cache.is_contiguous() and tuple(cache.shape) == (kv_heads, max_ctx, head_dim),
                "caches must be contiguous bf16 [kv_heads, max_context, head_dim]")
    for table in (cos, sin):
        _expect(table.dtype == torch.float32 and table.is_contiguous() and tuple(table.shape) == (max_ctx, head_dim),
                "rope tables must be float32 [max_context, head_dim]")
    _expect(q_out.dtype == torch.bfloat16 and q_out.is_contiguous() and q_out.numel() == heads * head_dim, "bad q_out")
    check(_lib.load().tx_rope_kv_cache_split(qkv_handle, _ptr(positions), _ptr(cos), _ptr(sin), heads, kv_heads,
                                             head_dim, _ptr(q_out), _ptr(k_cache), _ptr(v_cache), max_ctx,
                                             _stream(positions)))
    return q_out


def lm_head_argmax_workspace_bytes() -> int:
    """Device scratch of :func:`lm_head_argmax`."""
    out = ctypes.c_int64(0)
    check(_lib.load().tx_lm_head_argmax_workspace(ctypes.byref(out)))
    return int(out.value)


def lm_head_argmax(weight: torch.Tensor, x: torch.Tensor, workspace: torch.Tensor, out: torch.Tensor | None = None,
                   logits: torch.Tensor | None = None) -> torch.Tensor:
    """Greedy next token ``argmax(bf16(x @ weight^T))`` (the first row among equal maxima) for one
    bf16 hidden state ``x`` [hidden] or [1, hidden], written to ``out`` (int64 [1]); the bf16
    logits [vocab] too when ``logits`` is given."""
    _expect(weight.is_cuda and weight.dtype == torch.bfloat16 and weight.is_contiguous() and weight.dim() == 2,
            "weight must be a contiguous CUDA bf16 [vocab, hidden] tensor")
    vocab, hidden = weight.shape
    _expect(x.dtype == torch.bfloat16 and x.is_contiguous() and x.numel() == hidden and x.data_ptr() % 16 == 0,
            "x must be one contiguous, 16-byte aligned bf16 hidden state")
    _expect(workspace.is_cuda and workspace.is_contiguous(), "workspace must be a contiguous CUDA tensor")
    if out is None:
        out = torch.empty(1, dtype=torch.int64, device=x.device)
    _expect(out.dtype == torch.int64 and out.is_contiguous() and out.numel() == 1, "out must be int64 [1]")
    if logits is not None:
        _expect(logits.dtype == torch.bfloat16 and logits.is_contiguous() and logits.numel() == vocab, "logits must be bf16 [vocab]")
    check(_lib.load().tx_lm_head_argmax(_ptr(weight), vocab, hidden, _ptr(x), _ptr(logits), _ptr(workspace),
                                        workspace.numel() * workspace.element_size(), _ptr(out), _stream(x)))
    return out


def rope_rotate_half(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Hugging Face's ``apply_rotary_pos_emb`` (rotate-half form) on ``q`` ``[..., tokens, heads,
    dim]`` and ``k`` ``[..., tokens, kv_heads, dim]`` (contiguous bf16, the projections' own layout)
    with ``cos``/``sin`` ``[..., tokens, dim]`` bf16, bit for bit, in one kernel; returns new
    ``(q, k)`` of the same shapes."""
    _expect(all(t.is_cuda and t.dtype == torch.bfloat16 and t.is_contiguous() for t in (q, k, cos, sin)),
            "q, k, cos and sin must be contiguous CUDA bf16 tensors")
    dim = q.shape[-1]
    tokens = cos.numel() // dim
    _expect(cos.shape == sin.shape and cos.shape[-1] == dim and k.shape[-1] == dim and q.dim() >= 2 and k.dim() >= 2,
            "cos and sin must be [tokens, dim] rows of the heads' dim")
    _expect(q.numel() % (tokens * dim) == 0 and k.numel() % (tokens * dim) == 0, "q and k must hold whole tokens")
    heads, kv_heads = q.numel() // (tokens * dim), k.numel() // (tokens * dim)
    _expect(q.shape[-2] == heads and k.shape[-2] == kv_heads, "q and k must be [tokens, heads, dim]")
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    check(_lib.load().tx_rope_rotate_half(_ptr(q), _ptr(k), tokens, heads, kv_heads, dim, _ptr(cos), _ptr(sin),
                                          _ptr(q_out), _ptr(k_out), _stream(q)))
    return q_out, k_out


def kv_cache_append(k: torch.Tensor, v: torch.Tensor, keys: torch.Tensor, values: torch.Tensor,
                    length: torch.Tensor) -> None:
    """One token's ``k`` and ``v`` (``kv_heads x dim`` bf16 each, any view of one token) into a static
    cache ``keys``/``values`` ``[1, kv_heads, max_len, dim]`` at row ``length`` (a CUDA int64 scalar
    tensor), then ``length += 1``, in one launch; a full cache is left unchanged."""
    _expect(keys.is_cuda and keys.dtype == values.dtype == torch.bfloat16 and keys.is_contiguous()
            and values.is_contiguous() and keys.dim() == 4 and keys.shape[0] == 1 and keys.shape == values.shape,
            "keys and values must be contiguous CUDA bf16 [1, kv_heads, max_len, dim]")
    _, kv_heads, max_len, dim = keys.shape
    _expect(k.dtype == v.dtype == torch.bfloat16 and k.numel() == v.numel() == kv_heads * dim
            and k.device == v.device == keys.device, "k and v must be one token's bf16 [kv_heads, dim]")
    _expect(length.is_cuda and length.dtype == torch.int64 and length.numel() == 1 and length.device == keys.device,
            "length must be a CUDA int64 scalar")
    k, v = k.reshape(kv_heads, dim).contiguous(), v.reshape(kv_heads, dim).contiguous()
    check(_lib.load().tx_kv_cache_append(_ptr(k), _ptr(v), kv_heads, dim, _ptr(keys), _ptr(values), max_len,
                                         _ptr(length), _stream(keys)))


def swiglu(gate_up: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """``bf16(silu(g) * u)`` for rows ``[g | u]``."""
    _expect(gate_up.dtype == torch.bfloat16 and gate_up.is_contiguous() and gate_up.dim() == 2 and gate_up.shape[1] % 2 == 0,
            "gate_up must be contiguous bf16 [rows, 2 * intermediate]")
    rows, width = gate_up.shape
    if out is None:
        out = torch.empty((rows, width // 2), dtype=torch.bfloat16, device=gate_up.device)
    check(_lib.load().tx_swiglu(_ptr(gate_up), rows, width // 2, _ptr(out), _stream(gate_up)))
    return out


# ---------------------------------------------------------------------------------------------
# Several sequences at once

_ROW_CODE = {torch.float16: _lib.TX_DTYPE_F16, torch.bfloat16: _lib.TX_DTYPE_BF16}


# The messages are put together only for the calls that fail: formatting them took a tenth of a small call's host time.
def _expect_rows(name: str, t: torch.Tensor, like: torch.Tensor, heads: int, head_dim: int) -> None:
    shape = t.shape
    if (len(shape) != 3 or shape[1] != heads or shape[2] != head_dim or t.dtype != like.dtype or t.device != like.device
            or t.stride(2) != 1):
        raise TexelatorError(f"{name} must be {like.dtype} [rows, {heads}, {head_dim}] on one device, the last dimension contiguous")


def _expect_ints(name: str, t: torch.Tensor, count: int, device: torch.device) -> None:
    shape = t.shape
    if len(shape) != 1 or shape[0] != count or t.dtype != torch.int32 or t.device != device or not t.is_contiguous():
        raise TexelatorError(f"{name} must be a contiguous int32 [{count}] on the same device")


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor, scale: float,
                     cu_k: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of several sequences packed one behind the other: ``q`` ``[tokens, heads, dim]`` against
    ``k``/``v`` ``[keys, kv_heads, dim]`` (bf16 or fp16, dim 64 or 128, every row 16-byte aligned: views of one
    ``[q | k | v]`` projection will do). Sequence ``s`` has the queries ``cu_q[s] .. cu_q[s + 1] - 1`` and the keys
    ``cu_k[s] .. cu_k[s + 1] - 1`` (int32 on the device; ``cu_k`` defaults to ``cu_q``); its last query sees its last key,
    so keys of earlier turns come first. A query that sees no key gets zeros; rows of ``out`` that belong to no
    sequence are left as they are (uninitialised where ``out`` is not given); ``out`` shares no element with q, k and v, but
    may be columns of their buffer. Keys that a query does not see, and their values, may hold anything. Scores, softmax statistics
    and sums are fp32; the probabilities are rounded to the rows' type before they meet the values, and the sum that divides is of
    the rounded ones. Returns ``[tokens, heads, dim]``."""
    shape, rows, dtype, device, code = q.shape, k.shape, q.dtype, q.device, _ROW_CODE.get(q.dtype)
    if code is None or len(shape) != 3 or not q.is_cuda or q.stride(2) != 1:
        raise TexelatorError("q must be CUDA bf16 or fp16 [tokens, heads, dim], the last dimension contiguous")
    total, heads, dim = shape
    if (len(rows) != 3 or rows != v.shape or rows[1] == 0 or rows[2] != dim or k.dtype != dtype or v.dtype != dtype
            or k.device != device or v.device != device):
        raise TexelatorError(f"k and v must be {dtype} [keys, kv_heads, {dim}] on q's device")
    q_strides, k_strides, v_strides = q.stride(), k.stride(), v.stride()
    if k_strides[2] != 1 or v_strides[2] != 1:
        raise TexelatorError("the last dimension of k and v must be contiguous")
    sequences = cu_q.numel() - 1
    _expect(sequences >= 0, "cu_q must be int32 [sequences + 1]")
    _expect_ints("cu_q", cu_q, sequences + 1, device)
    if cu_k is None:
        _expect(rows[0] == total, "without cu_k there is a key for each query")
        cu_k = cu_q
    else:
        _expect_ints("cu_k", cu_k, sequences + 1, device)
    if out is None:
        out = q.new_empty(shape)
    else:
        _expect_rows("out", out, q, heads, dim)
        _expect(out.shape[0] == total, "out must be shaped like q")
    if total == 0:
        return out
    out_strides = out.stride()
    check(_lib.load().tx_packed_attention(
        q.data_ptr(), q_strides[0], q_strides[1], k.data_ptr(), k_strides[0], k_strides[1], v.data_ptr(), v_strides[0],
        v_strides[1], code, heads, rows[1], dim, cu_q.data_ptr(), cu_k.data_ptr(), sequences, total, rows[0], float(scale),
        out.data_ptr(), out_strides[0], out_strides[1], device.index, _stream_address(device)))
    return out


def kv4_pages(num_pages: int, kv_heads: int, head_dim: int, page_size: int = 64, layers: int | None = None,
              device: torch.device | str = "cuda") -> torch.Tensor:
    """An empty pool of a paged 4-bit KV cache: uint8 ``[num_pages, kv_heads, 2, page_size * head_dim * 17 / 32]``, behind
    ``layers`` where given (``pages[i]`` is layer i's pool, and one block table serves them all). A key or value takes
    ``head_dim * 17 / 32`` bytes: E2M1 codes and an E8M0 scale for 32 elements. ``page_size``: positions of a page, a
    power of two from 16 to 1024; ``head_dim`` 64 or 128. The calls take ``head_dim`` from the rows they are given: a pool made for
    128 and used with 64 is not told from one of twice the page size."""
    _expect(head_dim in (64, 128), "head_dim must be 64 or 128")
    _expect(16 <= page_size <= 1024 and page_size & (page_size - 1) == 0, "page_size must be a power of two from 16 to 1024")
    _expect(num_pages > 0 and kv_heads > 0 and (layers is None or layers > 0), "bad pool shape")
    shape = (num_pages, kv_heads, 2, page_size * head_dim * 17 // 32)
    return torch.zeros(shape if layers is None else (layers, *shape), dtype=torch.uint8, device=device)


def _kv4_page_size(shape: torch.Size, head_dim: int) -> int:
    """Positions of a page of a pool [num_pages, kv_heads, 2, page bytes]."""
    if len(shape) != 4 or shape[1] == 0 or shape[2] != 2:
        raise TexelatorError("pages must be [num_pages, kv_heads, 2, page bytes]")
    if head_dim not in (64, 128):
        raise TexelatorError("head_dim must be 64 or 128")
    page_size, rest = divmod(shape[3], head_dim * 17 // 32)
    if rest:
        raise TexelatorError("pages were made for another head_dim")
    return page_size


def _kv4_args(pages: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, head_dim: int, device: torch.device) -> tuple:
    """The cache's arguments of a C call, from pages to sequences."""
    shape, table = pages.shape, block_table.shape
    if pages.dtype != torch.uint8 or not pages.is_cuda or pages.device != device or not pages.is_contiguous():
        raise TexelatorError("pages must be contiguous CUDA uint8 [num_pages, kv_heads, 2, page bytes] on the rows' device")
    page_size = _kv4_page_size(shape, head_dim)
    if (len(table) != 2 or block_table.dtype != torch.int32 or block_table.device != device
            or (block_table.stride(1) != 1 and table[1] != 1)):
        raise TexelatorError("block_table must be int32 [sequences, pages] on the same device, rows contiguous")
    _expect_ints("lengths", lengths, table[0], device)
    return (pages.data_ptr(), shape[0], shape[1], head_dim, page_size, block_table.data_ptr(), block_table.stride(0), table[1],
            lengths.data_ptr(), table[0])


def _kv4_rows(k: torch.Tensor, v: torch.Tensor, kv_heads: int, head_dim: int, device: torch.device) -> tuple:
    """The arguments of a C call that k and v [tokens, kv_heads, head_dim] make, to the token count."""
    shape, dtype, k_strides, v_strides = k.shape, k.dtype, k.stride(), v.stride()
    code = _ROW_CODE.get(dtype)
    if (code is None or len(shape) != 3 or shape != v.shape or shape[1] != kv_heads or shape[2] != head_dim or v.dtype != dtype
            or k.device != device or v.device != device or k_strides[2] != 1 or v_strides[2] != 1):
        raise TexelatorError(f"k and v must be CUDA bf16 or fp16 [tokens, {kv_heads}, {head_dim}] on the pages' device, the last "
                             "dimension contiguous")
    return k.data_ptr(), k_strides[0], k_strides[1], v.data_ptr(), v_strides[0], v_strides[1], code, shape[0]


def kv4_append(k: torch.Tensor, v: torch.Tensor, pages: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor,
               cu: torch.Tensor | None = None) -> None:
    """New keys and values into a paged 4-bit cache (:func:`kv4_pages`): ``k``/``v`` ``[tokens, kv_heads, dim]`` bf16 or fp16,
    every row 16-byte aligned. Position p of sequence s lies at offset ``p % page_size`` of page ``block_table[s, p //
    page_size]`` (int32 ``[sequences, pages]``, -1 or any id outside the pool where there is none). ``lengths`` (int32
    ``[sequences]``) counts the new tokens already, so that one update serves all layers: the tokens ``cu[s] .. cu[s + 1] - 1``
    become the last ones of ``lengths[s]`` positions (``cu`` int32 ``[sequences + 1]``; without it, one token for each
    sequence). A page that receives tokens must belong to one sequence alone."""
    device = pages.device
    cache = _kv4_args(pages, block_table, lengths, k.shape[-1] if k.dim() else 0, device)
    rows = _kv4_rows(k, v, cache[2], cache[3], device)
    tokens, sequences = rows[-1], cache[-1]
    if cu is None:
        _expect(tokens == sequences, "without cu there is one token for each sequence")
    else:
        _expect_ints("cu", cu, sequences + 1, device)
    if tokens and sequences:
        check(_lib.load().tx_kv4_append(*rows, None if cu is None else cu.data_ptr(), *cache, device.index, _stream_address(device)))


def kv4_read(pages: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, head_dim: int,
             cu: torch.Tensor | None = None, tokens: int | None = None, dtype: torch.dtype = torch.bfloat16,
             out: tuple[torch.Tensor, torch.Tensor] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows of a paged 4-bit cache as the values they stand for: ``(k, v)``, each ``[tokens, kv_heads, head_dim]`` packed as
    :func:`kv4_append` takes them: the last ``cu[s + 1] - cu[s]`` of ``lengths[s]`` positions of every sequence (all of them
    where ``cu`` is the sums of ``lengths``, as :func:`packed_attention` takes the keys of earlier turns); without ``cu``
    the last one of each. ``tokens``: the rows in all, ``cu[-1]`` (needed with ``cu`` unless ``out`` is given). Rows that name
    no position are left as they are."""
    device = pages.device
    cache = _kv4_args(pages, block_table, lengths, head_dim, device)
    sequences = cache[-1]
    if cu is None:
        _expect(tokens is None or tokens == sequences, "without cu there is one token for each sequence")
        tokens = sequences
    else:
        _expect_ints("cu", cu, sequences + 1, device)
    if out is None:
        _expect(tokens is not None and tokens >= 0 and dtype in _ROW_CODE, "tokens is needed with cu; dtype is bf16 or fp16")
        k, v = torch.empty((2, tokens, cache[2], head_dim), dtype=dtype, device=device).unbind(0)
    else:
        k, v = out
    rows = _kv4_rows(k, v, cache[2], head_dim, device)
    _expect(tokens is None or rows[-1] == tokens, "out must have a row for each token")
    if rows[-1] and sequences:
        check(_lib.load().tx_kv4_read(*rows, None if cu is None else cu.data_ptr(), *cache, device.index, _stream_address(device)))
    return k, v


@functools.lru_cache(maxsize=256)
def _kv4_workspace_bytes(*sizes: int) -> int:
    out = ctypes.c_int64(0)
    check(_lib.load().tx_kv4_attention_workspace(*sizes, out))
    return out.value


def kv4_attention_workspace_bytes(pages: torch.Tensor, block_table: torch.Tensor, heads: int, head_dim: int) -> int:
    """Device scratch of :func:`kv4_attention`: it depends on shapes alone, not on the lengths."""
    _expect(pages.is_cuda and block_table.dim() == 2, "pages must be a CUDA tensor, block_table [sequences, pages]")
    sequences, max_pages = block_table.shape
    page_size = _kv4_page_size(pages.shape, head_dim)
    return _kv4_workspace_bytes(sequences, heads, pages.shape[1], head_dim, page_size, max_pages, pages.device.index)


def kv4_attention(q: torch.Tensor, pages: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, scale: float,
                  workspace: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one query token for each sequence over a paged 4-bit cache: ``q`` ``[sequences, heads, dim]`` bf16 or fp16
    (every query 16-byte aligned) against the ``lengths[s]`` positions that ``block_table[s]`` names (see
    :func:`kv4_append`); heads a multiple of the pages' KV heads. Returns ``[sequences, heads, dim]``, zeros for an empty
    sequence (one without a position in the pool). Scores, statistics and sums are fp32; the probabilities are rounded to q's type, and
    the sum that divides is of the rounded ones. Cached values become q's type: exact in bf16; in fp16 they are rounded where they are
    subnormal and infinite beyond 65504. ``workspace``: :func:`kv4_attention_workspace_bytes` bytes that no call running at the same time uses;
    allocated on the current stream where not given."""
    shape, device, code = q.shape, q.device, _ROW_CODE.get(q.dtype)
    if code is None or len(shape) != 3 or not q.is_cuda or q.stride(2) != 1:
        raise TexelatorError("q must be CUDA bf16 or fp16 [sequences, heads, dim], the last dimension contiguous")
    sequences, heads, dim = shape
    cache = _kv4_args(pages, block_table, lengths, dim, device)
    _expect(cache[-1] == sequences and heads > 0 and heads % cache[2] == 0,
            "q must have a row for each sequence and a multiple of the pages' heads")
    if out is None:
        out = q.new_empty(shape)
    else:
        _expect_rows("out", out, q, heads, dim)
        _expect(out.shape[0] == sequences, "out must be shaped like q")
    if sequences == 0:
        return out
    if workspace is None:
        size = _kv4_workspace_bytes(sequences, heads, cache[2], dim, cache[4], cache[7], device.index)
        workspace = torch.empty(size, dtype=torch.uint8, device=device) if size else None  # short sequences need no scratch
    else:
        _expect(workspace.is_cuda and workspace.is_contiguous() and workspace.device == device,
                "workspace must be a contiguous CUDA tensor on the same device")
        size = workspace.nbytes
    q_strides, out_strides = q.stride(), out.stride()
    check(_lib.load().tx_kv4_attention(q.data_ptr(), q_strides[0], q_strides[1], code, heads, *cache, float(scale), _ptr(workspace),
                                       size, out.data_ptr(), out_strides[0], out_strides[1], device.index, _stream_address(device)))
    return out


def kv4_copy_pages(pages: torch.Tensor, src: list[int], dst: list[int]) -> None:
    """Page ``src[i]`` to page ``dst[i]`` for every i, in one pool (:func:`kv4_pages`) or in all layers' pools
    ``[layers, ...]`` at once: a fork copies the last, partly filled page, a compaction moves pages and frees theirs.
    ``src`` and ``dst`` are host integers (a captured call repeats the copies it was captured with). All copies happen at once:
    a page that is copied to twice, or both copied from and copied to, is refused."""
    # The page's bytes follow from its keys and values both: a pool of one of them would be left past its end.
    _expect(pages.is_cuda and pages.dtype == torch.uint8 and pages.dim() in (4, 5) and pages.shape[-2] == 2 and pages.is_contiguous(),
            "pages must be contiguous CUDA uint8 [num_pages, kv_heads, 2, page bytes], layers before it or not")
    count = len(src)
    _expect(len(dst) == count, "src and dst must have as many pages")
    if count == 0:
        return
    *layers, num_pages, kv_heads, _, half = pages.shape
    try:
        sources, targets = array.array("q", src), array.array("q", dst)
    except (TypeError, OverflowError) as error:
        raise TexelatorError("src and dst must be integers") from error
    _expect(len(sources) == len(targets) == count, "src and dst must be integers")  # bytes make one of eight
    check(_lib.load().tx_kv4_copy_pages(pages.data_ptr(), layers[0] if layers else 1, num_pages, kv_heads * 2 * half,
                                        sources.buffer_info()[0], targets.buffer_info()[0], count, pages.device.index,
                                        _stream(pages)))
