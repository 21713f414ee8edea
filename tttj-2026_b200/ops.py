"""Thin torch-tensor wrappers over the per-kernel C entry points.

Each wrapper checks dtype, shape, contiguity and device (the reference's
TORCH_CHECK conventions, kernels/csrc/case14_softmax.cpp:18-35) and launches on the
current CUDA stream.  They exist for parity tests and for callers composing their
own layer; the forward of ``B200Transformer`` runs the same kernels from C.  The serving
operators at the end (prompts with grouped heads, a paged key/value cache) stand beside it.
"""
from __future__ import annotations

import ctypes
import functools
import struct
from typing import Optional

import torch
from torch.autograd import forward_ad as _forward_ad

from . import _lib


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream(device: torch.device):
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _need(cond: bool, msg: str) -> None:
    if not cond:
        raise ValueError(msg)


def linear(a: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, *, epilogue: str = "bias",
           residual: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
           rows_dev: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out = epi(a @ weight.T + bias) on the tcgen05 GEMM.

    epilogue: "bias", "gelu" (exact erf GELU), "residual" (out = residual + ...;
    ``out`` may be ``residual`` itself; fp16) or "residual_f32" (fp32 residual and
    out, the forward's residual stream).  a [M, K] fp16, weight [N, K] fp16,
    bias [N] fp32.
    """
    epi = {"bias": _lib.EPI_BIAS, "gelu": _lib.EPI_BIAS_GELU, "residual": _lib.EPI_BIAS_RESIDUAL,
           "residual_f32": _lib.EPI_BIAS_RESIDUAL_F32}[epilogue]
    _need(a.dtype == torch.float16 and weight.dtype == torch.float16, "linear: a and weight must be fp16")
    _need(bias.dtype == torch.float32, "linear: bias must be fp32")
    _need(a.dim() == 2 and weight.dim() == 2 and a.shape[1] == weight.shape[1], "linear: shape mismatch")
    _need(a.stride(1) == 1 and weight.stride(1) == 1 and bias.is_contiguous(), "linear: inner dims must be contiguous")
    M, K = a.shape
    N = weight.shape[0]
    out_dtype = torch.float32 if epi == _lib.EPI_BIAS_RESIDUAL_F32 else torch.float16
    if out is None:
        out = torch.empty(M, N, dtype=out_dtype, device=a.device)
    _need(out.dtype == out_dtype and out.stride(1) == 1, f"linear: out must be {out_dtype} [M, N]")
    if epi in (_lib.EPI_BIAS_RESIDUAL, _lib.EPI_BIAS_RESIDUAL_F32):
        _need(residual is not None and residual.shape == (M, N) and residual.dtype == out_dtype,
              f"linear: residual must be {out_dtype} [M, N]")
    rc = _lib.lib().tttj_linear(
        _ptr(a), a.stride(0), _ptr(weight), weight.stride(0), _ptr(bias), _ptr(out), out.stride(0),
        _ptr(residual), residual.stride(0) if residual is not None else 0, M, _ptr(rows_dev), N, K, epi,
        _ptr(status), _stream(a.device))
    _lib.check(rc, "linear")
    return out


def layernorm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, eps: float = 1e-5,
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """nn.LayerNorm over the last dim of a contiguous fp16 [rows, d] tensor."""
    _need(x.dtype == torch.float16 and x.is_contiguous() and x.dim() == 2, "layernorm: x must be contiguous fp16 [rows, d]")
    _need(weight.dtype == torch.float32 and bias.dtype == torch.float32, "layernorm: weight/bias must be fp32")
    if out is None:
        out = torch.empty_like(x)
    rc = _lib.lib().tttj_layernorm(_ptr(x), _ptr(out), x.shape[0], x.shape[1], _ptr(weight), _ptr(bias),
                                   float(eps), _stream(x.device))
    _lib.check(rc, "layernorm")
    return out


def attention_workspace_bytes(batch: int, seq_len: int, num_heads: int) -> int:
    return int(_lib.lib().tttj_attention_workspace_bytes(batch, seq_len, num_heads))


def attention(qkv: torch.Tensor, valid_token_mask: Optional[torch.Tensor], batch: int, seq_len: int,
              num_heads: int, causal: bool, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention over the packed valid-token layout: qkv [Tv, 3D] fp16 -> ctx [Tv, D]."""
    _need(qkv.dtype == torch.float16 and qkv.is_contiguous() and qkv.dim() == 2, "attention: qkv must be contiguous fp16 [Tv, 3D]")
    D = qkv.shape[1] // 3
    ctx = torch.zeros(qkv.shape[0], D, dtype=torch.float16, device=qkv.device)
    nbytes = attention_workspace_bytes(batch, seq_len, num_heads)
    if workspace is None:
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=qkv.device)
    mask = None
    if valid_token_mask is not None:
        mask = valid_token_mask.to(torch.bool).contiguous().view(torch.uint8)
    rc = _lib.lib().tttj_attention(_ptr(qkv), _ptr(ctx), qkv.shape[0], _ptr(mask), batch, seq_len, D, num_heads,
                                   1 if causal else 0, _ptr(workspace), workspace.numel(),
                                   _stream(qkv.device))
    _lib.check(rc, "attention")
    return ctx


def selftest_wait_timeout(status: torch.Tensor, limit_ns: int) -> None:
    """Launch the bounded-wait self test (writes 0x1ff into ``status`` on timeout)."""
    _need(status.dtype == torch.int32 and status.is_cuda, "selftest: status must be a CUDA int32 tensor")
    _lib.check(_lib.lib().tttj_selftest_wait_timeout(_ptr(status), int(limit_ns), _stream(status.device)), "selftest")


# ------------------------------------------------------------------ serving operators
# Prompts with grouped heads, and a paged key/value cache: append, attention of new tokens,
# the attention mass each slot gathers, eviction.  Common to all of them:
#
# * Tokens of all sequences are packed: sequence b owns rows seq_offsets[b] ..
#   seq_offsets[b + 1] (int32 [B + 1] on the device).  Rows behind the last sequence are left
#   as they were, so a batch may be padded.
# * q [T, heads, head_dim], k / v [T, kv_heads, head_dim], fp16 or bf16, head_dim 32, 64, 128
#   or 256, the last dimension contiguous, other strides any positive multiples of 8 (views
#   of one packed projection will do).  Query head h reads key/value head
#   h // (heads // kv_heads).
# * A cache is [pages, page_size, kv_heads, head_dim] for k and for v (any stride order: pass a
#   transposed view for heads-first pages), page_size 16 .. 256; page_table int32 [B, P] holds
#   each sequence's pages in order, cache_lens int32 [B] its tokens, the new ones included.
#   New token i of n is at slot len - n + i.
# * Lengths, offsets and page numbers are read on the device only: calls can be captured into
#   CUDA graphs and replayed with new ones.  They are bounds-checked there; ``status`` (int32
#   [1], zeroed by the caller) records a wrong one (include/tttj_b200.h, TTTJ_DEV_BAD_*).
# * A device wait that gave up (2 s; status TTTJ_DEV_SERVE_TIMEOUT) makes the next call on the device
#   raise RuntimeError, with or without ``status``; ``serve_status`` asks for it.
# * Launches go to the current stream of the tensors' device, whichever device is current.
# * Inference only: tensors that require gradients are refused while gradients are enabled, and
#   tensors that carry a forward-mode tangent.

_SERVE_DTYPES = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}
# tttj_rows, tttj_pages and tttj_seqs of include/tttj_b200.h as bytes in C layout: a decode
# step's host time counts, and packing is several times cheaper than ctypes structures.
_pack_rows = struct.Struct("@Pqq").pack
_pack_pages = struct.Struct("@Pqqq").pack
_pack_seqs = struct.Struct("@PPPq9iP").pack


def _call(device: torch.device, fn, *args) -> int:
    """Run a C entry point with ``device`` current, its current stream as last argument."""
    index = device.index
    if torch._C._cuda_getDevice() == index:
        return fn(*args, torch._C._cuda_getCurrentRawStream(index))
    with torch.cuda.device(device):
        return fn(*args, torch._C._cuda_getCurrentRawStream(index))


def _refuse_tangents(what: str, **tensors: Optional[torch.Tensor]) -> None:
    """Inside a forward-mode level: raise if a tensor carries a tangent, which would be dropped."""
    for name, t in tensors.items():
        if t is not None and _forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError(f"{what}: inference only ({name} carries a forward-mode tangent)")


def _serve_rows(what: str, name: str, t: torch.Tensor, shape: tuple, dtype: torch.dtype, device: torch.device) -> bytes:
    if t.shape != shape or t.dtype != dtype or t.device != device:
        raise ValueError(f"{what}: {name} must be [tokens, heads, head_dim] = {list(shape)}, {dtype} on {device}, "
                         f"got {list(t.shape)}, {t.dtype} on {t.device}")
    tok, head, one = t.stride()
    if one != 1:
        raise ValueError(f"{what}: head_dim of {name} must be contiguous")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what}: inference only ({name} requires a gradient)")
    return _pack_rows(t.data_ptr(), tok, head)


def _serve_ints(what: str, name: str, t: torch.Tensor, n: int, device: torch.device) -> int:
    if t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] != n or t.device != device or (n > 1 and t.stride(0) != 1):
        raise ValueError(f"{what}: {name} must be a contiguous int32 tensor [{n}] on {device}")
    return t.data_ptr()


def _serve_pages(what: str, name: str, t: torch.Tensor, shape: tuple, dtype: torch.dtype, device: torch.device) -> bytes:
    if t.shape != shape or t.dtype != dtype or t.device != device:
        raise ValueError(f"{what}: {name} must be [pages, page_size, kv_heads, head_dim] = {list(shape)}, {dtype} on "
                         f"{device}, got {list(t.shape)}, {t.dtype} on {t.device}")
    page, slot, head, one = t.stride()
    if one != 1:
        raise ValueError(f"{what}: head_dim of {name} must be contiguous")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what}: inference only ({name} requires a gradient)")
    return _pack_pages(t.data_ptr(), page, slot, head)


def _serve_type(what: str, t: torch.Tensor) -> int:
    dtype = _SERVE_DTYPES.get(t.dtype)
    if dtype is None:
        raise ValueError(f"{what}: dtype {t.dtype} unsupported (float16, bfloat16)")
    if not t.is_cuda:
        raise ValueError(f"{what}: tensors must be on a CUDA device")
    return dtype


def _serve_offsets(what: str, seq_offsets: torch.Tensor, device: torch.device) -> tuple:
    batch = seq_offsets.shape[0] - 1 if seq_offsets.dim() == 1 else 0
    if batch < 1:
        raise ValueError(f"{what}: seq_offsets must be [sequences + 1]")
    return batch, _serve_ints(what, "seq_offsets", seq_offsets, batch + 1, device)


def _cache_seqs(what: str, off: Optional[int], batch: int, tokens: int, dtype: int, heads: int, cache: torch.Tensor,
                page_table: torch.Tensor, cache_lens: torch.Tensor, status: Optional[torch.Tensor],
                device: torch.device) -> tuple:
    """(tttj_seqs as bytes, slots per sequence) of a call over a cache."""
    if page_table.dim() != 2 or page_table.dtype != torch.int32 or page_table.device != device or \
            page_table.shape[0] != batch or page_table.stride(1) != 1:
        raise ValueError(f"{what}: page_table must be int32 [{batch}, pages per sequence] on {device}, rows contiguous")
    pages, page, kv_heads, head_dim = cache.shape
    per_seq = page_table.shape[1]
    lens = _serve_ints(what, "cache_lens", cache_lens, batch, device)
    stat = 0 if status is None else _serve_ints(what, "status", status, 1, device)
    return _pack_seqs(off or 0, lens, page_table.data_ptr(), page_table.stride(0) if batch > 1 else per_seq, batch, tokens,
                      per_seq, page, pages, dtype, heads, kv_heads, head_dim, stat), per_seq * page


@functools.lru_cache(maxsize=1024)
def _serve_workspace_bytes(batch: int, tokens: int, dtype: int, heads: int, kv_heads: int, head_dim: int) -> int:
    return int(_lib.lib().tttj_serve_workspace_bytes(
        _pack_seqs(0, 0, 0, 0, batch, tokens, 0, 0, 0, dtype, heads, kv_heads, head_dim, 0)))


def serve_workspace_bytes(batch: int, tokens: int, heads: int, kv_heads: int, head_dim: int) -> int:
    """Workspace of prompt_attention and cache_attention for this many sequences, packed
    tokens and heads; a larger one serves smaller calls too."""
    n = _serve_workspace_bytes(batch, tokens, _lib.DTYPE_F16, heads, kv_heads, head_dim)
    if n == 0:
        _lib.check(_lib.TTTJ_ERR_INVALID, "serve_workspace_bytes")
    return n


def serve_status(device: torch.device) -> int:
    """Synchronise ``device`` and raise RuntimeError if a bounded wait of a serving kernel gave up
    there (returns 0 when healthy).  Without this call the device's next serving call raises
    instead; replayed graphs make none."""
    with torch.cuda.device(device):
        v = ctypes.c_int(0)
        _lib.check(_lib.lib().tttj_serve_status(ctypes.byref(v)), "serve_status")
    return 0


def serve_selftest_timeout(device: torch.device, limit_ns: int = 2_000_000, status: Optional[torch.Tensor] = None) -> None:
    """Failure-detection self test: a bounded device wait on nothing gives up after ``limit_ns`` and
    reports as a serving kernel's would, so that the next serving call on ``device`` raises
    RuntimeError.  No GPU fault is involved."""
    device = torch.device(device)
    stat = None if status is None else _serve_ints("serve_selftest", "status", status, 1, device)
    with torch.cuda.device(device):
        _lib.check(_lib.lib().tttj_serve_selftest_timeout(stat, int(limit_ns), _stream(device)), "serve_selftest")


def _serve_out(what: str, out: Optional[torch.Tensor], q: torch.Tensor) -> tuple:
    """The output [tokens, heads, head_dim], made contiguous if not given, and its tttj_rows."""
    if out is not None:
        return out, _serve_rows(what, "out", out, q.shape, q.dtype, q.device)
    _, heads, d = q.shape
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    return out, _pack_rows(out.data_ptr(), heads * d, d)


def _serve_workspace(what: str, workspace: Optional[torch.Tensor], nbytes: int, device: torch.device) -> torch.Tensor:
    if workspace is None:
        return torch.empty(nbytes, dtype=torch.uint8, device=device)
    if workspace.dtype != torch.uint8 or workspace.device != device or workspace.dim() != 1 or \
            not workspace.is_contiguous():
        raise ValueError(f"{what}: workspace must be a contiguous 1-D uint8 tensor on {device}")
    return workspace


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, seq_offsets: torch.Tensor, *,
                     causal: bool = True, scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                     return_lse: bool = False, workspace: Optional[torch.Tensor] = None,
                     status: Optional[torch.Tensor] = None):
    """Attention inside each packed sequence: out[i] = softmax(scale q[i] k^T) v over the
    tokens j <= i of the same sequence (all of them with ``causal=False``).

    scale defaults to head_dim^-0.5.  Returns out [T, heads, head_dim] in q's dtype (``out``
    may be given; it must not overlap the inputs), with ``return_lse`` also the fp32 [T, heads]
    log-sum-exp of the scaled scores.  ``workspace`` (uint8,
    ``serve_workspace_bytes``) may be kept between calls that do not overlap."""
    what = "prompt_attention"
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError(f"{what}: q and k must be [tokens, heads, head_dim]")
    if _forward_ad._current_level >= 0:
        _refuse_tangents(what, q=q, k=k, v=v, out=out)
    dtype, device, kind = q.dtype, q.device, _serve_type(what, q)
    tokens, heads, d = q.shape
    kv_heads = k.shape[1]
    batch, off = _serve_offsets(what, seq_offsets, device)
    rows, kv_rows = (tokens, heads, d), (tokens, kv_heads, d)
    out, ro = _serve_out(what, out, q)
    s = _pack_seqs(off, 0, 0, 0, batch, tokens, 0, 0, 0, kind, heads, kv_heads, d,
                   0 if status is None else _serve_ints(what, "status", status, 1, device))
    rq, rk = _serve_rows(what, "q", q, rows, dtype, device), _serve_rows(what, "k", k, kv_rows, dtype, device)
    rv = _serve_rows(what, "v", v, kv_rows, dtype, device)
    lse = q.new_empty((tokens, heads), dtype=torch.float32) if return_lse else None
    ws = _serve_workspace(what, workspace, _serve_workspace_bytes(batch, tokens, kind, heads, kv_heads, d), device)
    rc = _call(device, _lib.lib().tttj_prompt_attention, s, rq, rk, rv, ro, lse.data_ptr() if return_lse else None,
               1 if causal else 0, d ** -0.5 if scale is None else scale, ws.data_ptr(), ws.shape[0])
    if rc:
        _lib.check(rc, what)
    return (out, lse) if return_lse else out


def cache_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                    seq_offsets: torch.Tensor, cache_lens: torch.Tensor, *, max_new: Optional[int] = None,
                    scale: Optional[float] = None, out: Optional[torch.Tensor] = None, return_lse: bool = False,
                    workspace: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None):
    """Attention of each sequence's new tokens over its cache (their own keys and values
    appended before): new token i of n sees slots 0 .. len - n + i.

    ``max_new``: the most new tokens a sequence of this call has, if known (1 for a decode
    step); it picks the kernels and need not be exact.  Returns as ``prompt_attention``."""
    what = "cache_attention"
    if q.dim() != 3 or k_cache.dim() != 4:
        raise ValueError(f"{what}: q must be [tokens, heads, head_dim], k_cache [pages, page_size, kv_heads, head_dim]")
    if _forward_ad._current_level >= 0:
        _refuse_tangents(what, q=q, k_cache=k_cache, v_cache=v_cache, out=out)
    dtype, device, kind = q.dtype, q.device, _serve_type(what, q)
    tokens, heads, d = q.shape
    pages = k_cache.shape
    kv_heads = pages[2]
    if pages[3] != d:
        raise ValueError(f"{what}: the cache has head_dim {pages[3]}, q {d}")
    batch, off = _serve_offsets(what, seq_offsets, device)
    s, _ = _cache_seqs(what, off, batch, tokens, kind, heads, k_cache, page_table, cache_lens, status, device)
    out, ro = _serve_out(what, out, q)
    rq = _serve_rows(what, "q", q, (tokens, heads, d), dtype, device)
    ck = _serve_pages(what, "k_cache", k_cache, pages, dtype, device)
    cv = _serve_pages(what, "v_cache", v_cache, pages, dtype, device)
    lse = q.new_empty((tokens, heads), dtype=torch.float32) if return_lse else None
    ws = _serve_workspace(what, workspace, _serve_workspace_bytes(batch, tokens, kind, heads, kv_heads, d), device)
    rc = _call(device, _lib.lib().tttj_cache_attention, s, rq, ck, cv, ro, lse.data_ptr() if return_lse else None,
               min(max_new or 0, tokens), d ** -0.5 if scale is None else scale, ws.data_ptr(), ws.shape[0])
    if rc:
        _lib.check(rc, what)
    return (out, lse) if return_lse else out


def _slot_tensor(what: str, name: str, t: torch.Tensor, dtype: torch.dtype, shape: tuple, device: torch.device) -> int:
    if t.dtype != dtype or t.shape != shape or t.device != device or not t.is_contiguous():
        raise ValueError(f"{what}: {name} must be a contiguous {dtype} tensor {list(shape)} "
                         f"(sequences, kv_heads, slots) on {device}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what}: inference only ({name} requires a gradient)")
    return t.data_ptr()


def cache_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 page_table: torch.Tensor, seq_offsets: torch.Tensor, cache_lens: torch.Tensor, *,
                 positions: Optional[torch.Tensor] = None, mass: Optional[torch.Tensor] = None,
                 seen: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> None:
    """Write the new tokens' keys and values to their slots of the cache.

    With ``positions`` (int32) / ``mass`` (fp32), both [B, kv_heads, P * page_size], a new
    slot's position becomes seen[b] - n + i and its mass 0; ``seen`` int32 [B] counts the tokens
    of each sequence, new ones included (default cache_lens; they differ once tokens were
    evicted).  New tokens whose slot would not be in the table are dropped, and ``status`` says
    so (TTTJ_DEV_BAD_LENS)."""
    what = "cache_append"
    if k.dim() != 3 or k_cache.dim() != 4:
        raise ValueError(f"{what}: k must be [tokens, kv_heads, head_dim], k_cache [pages, page_size, kv_heads, head_dim]")
    if _forward_ad._current_level >= 0:
        _refuse_tangents(what, k=k, v=v, k_cache=k_cache, v_cache=v_cache, mass=mass)
    dtype, device, kind = k.dtype, k.device, _serve_type(what, k)
    tokens, kv_heads, d = rows = k.shape
    pages = k_cache.shape
    if pages[2:] != rows[1:]:
        raise ValueError(f"{what}: the cache has rows {list(pages[2:])}, k {list(rows[1:])}")
    batch, off = _serve_offsets(what, seq_offsets, device)
    s, cap = _cache_seqs(what, off, batch, tokens, kind, kv_heads, k_cache, page_table, cache_lens, status, device)
    rk, rv = _serve_rows(what, "k", k, rows, dtype, device), _serve_rows(what, "v", v, rows, dtype, device)
    ck = _serve_pages(what, "k_cache", k_cache, pages, dtype, device)
    cv = _serve_pages(what, "v_cache", v_cache, pages, dtype, device)
    slots = (batch, kv_heads, cap)
    pos = None if positions is None else _slot_tensor(what, "positions", positions, torch.int32, slots, device)
    ms = None if mass is None else _slot_tensor(what, "mass", mass, torch.float32, slots, device)
    sn = None if seen is None else _serve_ints(what, "seen", seen, batch, device)
    rc = _call(device, _lib.lib().tttj_cache_append, s, rk, rv, ck, cv, pos, ms, sn)
    if rc:
        _lib.check(rc, what)


def cache_evict(mass: torch.Tensor, positions: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                page_table: torch.Tensor, cache_lens: torch.Tensor, keep: int, *, recent: int = 0,
                status: Optional[torch.Tensor] = None):
    """Evict down to ``keep`` slots per sequence and key/value head, those of least mass.

    mass fp32 and positions int32 [B, kv_heads, P * page_size].  The slots of the largest masses
    stay (equal ones: the lower slot; NaN counts as -inf); those whose position is among the
    head's ``recent`` newest count as +inf.  Kept slots behind the budget move into the freed ones in
    front of it, the i-th into the i-th, in both caches (whose pages must be the sequence's own);
    all others keep their place, so the cache is no longer in the tokens' order.  Returns new
    (mass, positions, cache_lens): 0 and -1 behind the new lengths min(len, keep).  A captured call
    reads the tensors that it was captured with: copy the returned ones into them for the next
    replay."""
    what = "cache_evict"
    if k_cache.dim() != 4 or cache_lens.dim() != 1 or cache_lens.shape[0] < 1:
        raise ValueError(f"{what}: k_cache must be [pages, page_size, kv_heads, head_dim], cache_lens [sequences]")
    if _forward_ad._current_level >= 0:
        _refuse_tangents(what, mass=mass, k_cache=k_cache, v_cache=v_cache)
    dtype, device, kind = k_cache.dtype, k_cache.device, _serve_type(what, k_cache)
    pages = k_cache.shape
    batch, kv_heads = cache_lens.shape[0], pages[2]
    s, cap = _cache_seqs(what, None, batch, 0, kind, kv_heads, k_cache, page_table, cache_lens, status, device)
    ck = _serve_pages(what, "k_cache", k_cache, pages, dtype, device)
    cv = _serve_pages(what, "v_cache", v_cache, pages, dtype, device)
    if keep <= 0 or not 0 <= recent <= keep:
        raise ValueError(f"{what}: keep={keep} must be positive, recent={recent} in 0 .. keep")
    keep, recent = min(keep, cap), min(recent, cap)  # (the C arguments have 32 bits)
    slots = (batch, kv_heads, cap)
    ms = _slot_tensor(what, "mass", mass, torch.float32, slots, device)
    pos = _slot_tensor(what, "positions", positions, torch.int32, slots, device)
    L = _lib.lib()
    nbytes = L.tttj_cache_evict_workspace_bytes(s, keep)
    if nbytes == 0:
        _lib.check(_lib.TTTJ_ERR_INVALID, what)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    mass_out, pos_out = torch.empty_like(mass), torch.empty_like(positions)
    lens_out = torch.empty_like(cache_lens)
    rc = _call(device, L.tttj_cache_evict, s, ck, cv, ms, pos, keep, recent, mass_out.data_ptr(), pos_out.data_ptr(),
               lens_out.data_ptr(), ws.data_ptr(), nbytes)
    if rc:
        _lib.check(rc, what)
    return mass_out, pos_out, lens_out


def cache_mass(q: torch.Tensor, lse: torch.Tensor, k_cache: torch.Tensor, page_table: torch.Tensor,
               seq_offsets: torch.Tensor, cache_lens: torch.Tensor, mass: torch.Tensor, *,
               max_new: Optional[int] = None, scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
               status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """mass plus the attention weight that the new tokens give to every slot: for key/value
    head g and slot j, the sum over the tokens that see j and the heads of g of
    exp(scale q k_j - lse), with the ``lse`` that ``cache_attention`` (or
    ``prompt_attention``) returned for the same queries.

    mass fp32 [B, kv_heads, P * page_size]; returns a new tensor, or ``out``, which may be
    ``mass`` itself.  ``max_new`` and ``scale`` as for ``cache_attention``."""
    what = "cache_mass"
    if q.dim() != 3 or k_cache.dim() != 4:
        raise ValueError(f"{what}: q must be [tokens, heads, head_dim], k_cache [pages, page_size, kv_heads, head_dim]")
    if _forward_ad._current_level >= 0:
        _refuse_tangents(what, q=q, lse=lse, k_cache=k_cache, mass=mass, out=out)
    dtype, device, kind = q.dtype, q.device, _serve_type(what, q)
    tokens, heads, d = rows = q.shape
    pages = k_cache.shape
    if pages[3] != d:
        raise ValueError(f"{what}: the cache has head_dim {pages[3]}, q {d}")
    batch, off = _serve_offsets(what, seq_offsets, device)
    s, cap = _cache_seqs(what, off, batch, tokens, kind, heads, k_cache, page_table, cache_lens, status, device)
    if lse.dtype != torch.float32 or lse.shape != rows[:2] or lse.device != device or not lse.is_contiguous():
        raise ValueError(f"{what}: lse must be a contiguous float32 tensor [{tokens}, {heads}] on {device}")
    if lse.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what}: inference only (lse requires a gradient)")
    slots = (batch, pages[2], cap)
    ms = _slot_tensor(what, "mass", mass, torch.float32, slots, device)
    if out is None:
        out = torch.empty_like(mass)
    mo = _slot_tensor(what, "out", out, torch.float32, slots, device)
    rq = _serve_rows(what, "q", q, rows, dtype, device)
    ck = _serve_pages(what, "k_cache", k_cache, pages, dtype, device)
    rc = _call(device, _lib.lib().tttj_cache_mass, s, rq, lse.data_ptr(), ck, ms, mo, min(max_new or 0, tokens),
               d ** -0.5 if scale is None else scale)
    if rc:
        _lib.check(rc, what)
    return out
