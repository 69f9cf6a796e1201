"""Torch-tensor wrappers over the C ABI (device memory and streams come from torch).

Every wrapper validates shapes, dtypes, devices and strides on the host before
it launches, so a kernel never sees an operand that disagrees with its grid.
All outputs and workspaces are caller-provided or allocated here *outside*
any graph capture; the kernels themselves never allocate or synchronise.
"""
from __future__ import annotations

import ctypes
import functools
import math
from dataclasses import dataclass
from typing import Optional, Sequence

import torch

from . import _lib

PAGE_SIZE = 16
HEAD_DIM = 128
_DEFAULT_SCALE = 1.0 / math.sqrt(HEAD_DIM)

_DTYPES = {torch.bfloat16: _lib.DELTA_BF16, torch.float16: _lib.DELTA_FP16}


def _dtype_code(t: torch.Tensor) -> int:
    try:
        return _DTYPES[t.dtype]
    except KeyError:
        raise TypeError(f"unsupported dtype {t.dtype}; expected bfloat16 or float16") from None


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _stream(device: torch.device):
    return torch.cuda.current_stream(device).cuda_stream


def _check_cuda(*tensors, device=None):
    dev = device
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError("delta_amd kernels need GPU tensors")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError(f"tensors on different devices: {t.device} vs {dev}")
    return dev


def _check_i32(name: str, t: torch.Tensor, min_numel: int = 0):
    if t.dtype != torch.int32:
        raise TypeError(f"{name} must be int32, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if t.numel() < min_numel:
        raise ValueError(f"{name} needs >= {min_numel} entries, has {t.numel()}")


def _check_cache(kv_cache: torch.Tensor):
    if kv_cache.dim() != 5 or kv_cache.shape[1] != 2 or kv_cache.shape[2] != PAGE_SIZE \
            or kv_cache.shape[4] != HEAD_DIM:
        raise ValueError(f"kv_cache must be [pages, 2, 16, Hkv, 128], got {tuple(kv_cache.shape)}")
    if not kv_cache.is_contiguous():
        raise ValueError("kv_cache must be contiguous")
    _dtype_code(kv_cache)


def _check_heads(q: torch.Tensor, kv_cache: torch.Tensor):
    if q.dim() != 3 or q.shape[2] != HEAD_DIM:
        raise ValueError(f"q must be [batch, Hq, 128], got {tuple(q.shape)}")
    if q.stride(2) != 1 or q.stride(1) % 8 or q.stride(0) % 8:
        raise ValueError("q needs a unit inner stride and strides in multiples of 8 elements")
    if q.dtype != kv_cache.dtype:
        raise TypeError(f"q dtype {q.dtype} != kv_cache dtype {kv_cache.dtype}")
    hq, hkv = q.shape[1], kv_cache.shape[3]
    if hq % hkv or hq // hkv > 8:
        raise ValueError(f"num_qo_heads={hq} must be a multiple of num_kv_heads={hkv}, group <= 8")
    return hq, hkv


class Workspace:
    """Grow-only device scratch buffer (allocate before any graph capture).  A buffer that a
    larger request replaces is kept alive, not freed: a graph captured earlier still holds its
    address and may be replayed."""

    def __init__(self):
        self._buf: dict = {}
        self._retired: list = []

    def get(self, nbytes: int, device: torch.device) -> torch.Tensor:
        nbytes = max(int(nbytes), 256)
        key = (device.type, device.index)
        buf = self._buf.get(key)
        if buf is None or buf.numel() < nbytes:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("workspace must be sized before graph capture")
            if buf is not None:
                self._retired.append(buf)
            buf = torch.empty(nbytes, dtype=torch.uint8, device=device)
            self._buf[key] = buf
        return buf


_default_ws = Workspace()


def decode_workspace_bytes(batch: int, hq: int, hkv: int, max_pages: int) -> int:
    return int(_lib.query("delta_paged_decode_workspace_bytes", batch, hq, hkv, max_pages))


def decode_num_splits(batch: int, hkv: int, max_pages: int) -> int:
    """Units that ``paged_decode`` cuts a row of ``max_pages`` pages into."""
    return int(_lib.query("delta_decode_num_splits", batch, hkv, max_pages))


@dataclass
class DecodeAppend:
    """The decode token's RoPE and KV append, fused into a ``paged_decode`` launch
    (``delta_decode_append_t``): q is then the un-rotated query, and row b's new token (k, v
    rows b, position ``offsets[b]`` for the rotation) is written at ``kv_len_b - 1`` of the
    cache's full CSR ``(kv_indptr, kv_indices)``, sharing ``kv_last_page_len`` with the
    attention.  Bit-identical to ``rope_append`` followed by the plain attention."""
    k: torch.Tensor
    v: torch.Tensor
    offsets: torch.Tensor
    kv_indptr: torch.Tensor
    kv_indices: torch.Tensor
    rope_scale: float = 1.0
    rope_theta: float = 1e4
    low_freq_factor: Optional[float] = None
    high_freq_factor: Optional[float] = None
    old_context_len: Optional[float] = None


def _append_struct(ap: "DecodeAppend", B: int, hkv: int, kv_cache: torch.Tensor):
    for name, t in (("k", ap.k), ("v", ap.v)):
        if t.dim() != 3 or tuple(t.shape) != (B, hkv, HEAD_DIM) or t.stride(2) != 1 or t.stride(1) != HEAD_DIM \
                or t.stride(0) % 2 or t.dtype != kv_cache.dtype or not t.is_cuda:
            raise ValueError(f"append.{name} must be [{B}, {hkv}, 128] of the cache dtype with contiguous heads")
    _check_i32("append.offsets", ap.offsets, B)
    _check_i32("append.kv_indptr", ap.kv_indptr, B + 1)
    _check_i32("append.kv_indices", ap.kv_indices)
    llama31 = ap.low_freq_factor is not None and ap.high_freq_factor is not None
    return _lib.DecodeAppendC(
        ap.k.data_ptr(), ap.k.stride(0), ap.v.data_ptr(), ap.v.stride(0), ap.offsets.data_ptr(),
        ap.kv_indptr.data_ptr(), ap.kv_indices.data_ptr(), ap.kv_indices.numel(), float(ap.rope_scale),
        float(ap.rope_theta), int(llama31), float(ap.low_freq_factor or 0.0), float(ap.high_freq_factor or 0.0),
        float(ap.old_context_len or 0.0))


def paged_decode(q: torch.Tensor, kv_cache: torch.Tensor, kv_indptr: torch.Tensor,
                 kv_indices: torch.Tensor, kv_last_page_len: torch.Tensor, *,
                 max_pages_per_row: int, sm_scale: Optional[float] = None,
                 out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                 logits_dump: Optional[torch.Tensor] = None,
                 workspace: Optional[torch.Tensor] = None, subset: bool = False,
                 append: Optional[DecodeAppend] = None) -> torch.Tensor:
    """Paged decode attention (``delta_paged_decode``); returns ``out`` [B, Hq, 128].

    ``logits_dump`` (fp32, [B_max, Hq, S] or any view with unit last stride)
    receives the planner-layer logits for ``t < kv_len``.  ``subset=True``
    runs the same attention through ``delta_paged_decode_subset`` (selected
    pages; no dump).  ``append`` fuses the decode token's RoPE and KV append in
    (``delta_paged_decode[_subset]_append``).
    """
    if subset and logits_dump is not None:
        raise ValueError("the subset attention writes no logits dump")
    dev = _check_cuda(q, kv_cache, kv_indptr, kv_indices, kv_last_page_len, out, lse, logits_dump)
    _check_cache(kv_cache)
    hq, hkv = _check_heads(q, kv_cache)
    B = q.shape[0]
    _check_i32("kv_indptr", kv_indptr, B + 1)
    _check_i32("kv_indices", kv_indices)
    _check_i32("kv_last_page_len", kv_last_page_len, B)
    if out is None:
        out = torch.empty_like(q)
    if out.shape != q.shape or out.dtype != q.dtype or out.stride(2) != 1:
        raise ValueError("out must match q's shape/dtype with unit inner stride")
    if lse is not None and (lse.dtype != torch.float32 or lse.shape[0] < B or lse.shape[1] != hq
                            or not lse.is_contiguous()):
        raise ValueError("lse must be contiguous fp32 [>=B, Hq]")
    dsb = dsh = 0
    if logits_dump is not None:
        if logits_dump.dtype != torch.float32 or logits_dump.dim() != 3 or logits_dump.stride(2) != 1:
            raise ValueError("logits_dump must be fp32 [B, Hq, S] with unit last stride")
        if logits_dump.shape[0] < B or logits_dump.shape[1] != hq \
                or logits_dump.shape[2] < max_pages_per_row * PAGE_SIZE:
            raise ValueError(f"logits_dump {tuple(logits_dump.shape)} too small for "
                             f"B={B}, Hq={hq}, {max_pages_per_row} pages")
        dsb, dsh = logits_dump.stride(0), logits_dump.stride(1)
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(HEAD_DIM)
    need = decode_workspace_bytes(B, hq, hkv, max_pages_per_row)
    if workspace is None:
        workspace = _default_ws.get(need, dev)
    elif workspace.numel() * workspace.element_size() < need:
        raise ValueError(f"workspace too small: {need} bytes needed")
    common_head = (q.data_ptr(), q.stride(0), q.stride(1), kv_cache.data_ptr(), kv_cache.shape[0],
                   kv_indptr.data_ptr(), kv_indices.data_ptr(), kv_indices.numel(), kv_last_page_len.data_ptr(),
                   out.data_ptr(), out.stride(0), out.stride(1), _ptr(lse))
    common_tail = (B, hq, hkv, HEAD_DIM, _dtype_code(q), float(sm_scale), int(max_pages_per_row),
                   workspace.data_ptr(), workspace.numel() * workspace.element_size(), _stream(dev))
    if append is not None:
        ap = ctypes.byref(_append_struct(append, B, hkv, kv_cache))
        if subset:
            _lib.call("delta_paged_decode_subset_append", ap, *common_head, *common_tail)
        else:
            _lib.call("delta_paged_decode_append", ap, *common_head, _ptr(logits_dump), dsb, dsh, *common_tail)
    elif subset:
        _lib.call("delta_paged_decode_subset", *common_head, *common_tail)
    else:
        _lib.call("delta_paged_decode", *common_head, _ptr(logits_dump), dsb, dsh, *common_tail)
    return out


def paged_decode_scores_supported(batch: int, num_qo_heads: int, num_kv_heads: int, max_pages_per_row: int,
                                  with_append: bool = False) -> bool:
    """True when ``paged_decode_scores`` applies to this shape (the rows' logits fit on chip)."""
    return bool(_lib.query("delta_paged_decode_scores_supported", int(batch), int(num_qo_heads),
                           int(num_kv_heads), int(max_pages_per_row), int(bool(with_append))))


def paged_decode_scores_workspace_bytes(batch: int, num_kv_heads: int, max_pages_per_row: int) -> int:
    """Workspace bytes of ``paged_decode_scores`` (its per-token maxima)."""
    return int(_lib.query("delta_paged_decode_scores_workspace_bytes", int(batch), int(num_kv_heads),
                          int(max_pages_per_row)))


def paged_decode_scores(q: torch.Tensor, kv_cache: torch.Tensor, kv_indptr: torch.Tensor,
                        kv_indices: torch.Tensor, kv_last_page_len: torch.Tensor, *,
                        max_pages_per_row: int, sm_scale: Optional[float] = None,
                        out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                        scores: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None,
                        append: Optional[DecodeAppend] = None):
    """The planner layer without a logits dump (``delta_paged_decode_scores[_append]``): full
    attention and the del3_legacy_softmax page scores in one pass; returns ``(out, scores)``,
    scores fp32 [B, max_pages_per_row].  Only where ``paged_decode_scores_supported``."""
    dev = _check_cuda(q, kv_cache, kv_indptr, kv_indices, kv_last_page_len, out, lse, scores)
    _check_cache(kv_cache)
    hq, hkv = _check_heads(q, kv_cache)
    B = q.shape[0]
    _check_i32("kv_indptr", kv_indptr, B + 1)
    _check_i32("kv_indices", kv_indices)
    _check_i32("kv_last_page_len", kv_last_page_len, B)
    if out is None:
        out = torch.empty_like(q)
    if out.shape != q.shape or out.dtype != q.dtype or out.stride(2) != 1:
        raise ValueError("out must match q's shape/dtype with unit inner stride")
    if lse is not None and (lse.dtype != torch.float32 or lse.shape[0] < B or lse.shape[1] != hq
                            or not lse.is_contiguous()):
        raise ValueError("lse must be contiguous fp32 [>=B, Hq]")
    if scores is None:
        scores = torch.empty((B, max_pages_per_row), dtype=torch.float32, device=dev)
    if scores.dtype != torch.float32 or scores.stride(1) != 1 or scores.shape[0] < B \
            or scores.shape[1] < max_pages_per_row:
        raise ValueError("scores must be fp32 [>=B, >=max_pages_per_row]")
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(HEAD_DIM)
    need = paged_decode_scores_workspace_bytes(B, hkv, max_pages_per_row)
    if workspace is None:
        workspace = _default_ws.get(need, dev)
    elif workspace.numel() * workspace.element_size() < need:
        raise ValueError(f"workspace too small: {need} bytes needed")
    args = (q.data_ptr(), q.stride(0), q.stride(1), kv_cache.data_ptr(), kv_cache.shape[0],
            kv_indptr.data_ptr(), kv_indices.data_ptr(), kv_indices.numel(), kv_last_page_len.data_ptr(),
            out.data_ptr(), out.stride(0), out.stride(1), _ptr(lse), scores.data_ptr(), scores.stride(0),
            B, hq, hkv, HEAD_DIM, _dtype_code(q), float(sm_scale), int(max_pages_per_row),
            workspace.data_ptr(), workspace.numel() * workspace.element_size(), _stream(dev))
    if append is not None:
        _lib.call("delta_paged_decode_scores_append",
                  ctypes.byref(_append_struct(append, B, hkv, kv_cache)), *args)
    else:
        _lib.call("delta_paged_decode_scores", *args)
    return out, scores


def _split_decode_rows(max_qo_len: int, tokens: int, hq: int, hkv: int, pages: int, longest: int) -> bool:
    """Whether a prompt step's rows of one new token (``pages`` pages, the longest ``longest``) go to split
    decode units.  One prefill block per kv head sweeps such a row alone, 0.33 us a page; the rows launch and
    its merge cost ~11 us (5 without prompts), in front of the prompts, and the rows' bytes.  So the longest
    row has to outlast the longest prompt (0.022 us a token) by that, or, where the prompts alone are more
    blocks than the chip holds and the row starts behind them, to be worth it by itself; and where rows times kv
    heads keep the CUs streaming anyway there is less to gain (us without / with, 8 kv heads of 4 q heads: one row
    of 63 / 126 pages beside 50 tokens 24 / 19, 44 / 20, beside 1000 29 / 41, 47 / 43, beside 2000 55 / 68, 57 /
    68; of 82 / 188 beside 4000 151 / 151, 180 / 152; 30 rows of 126 / 188 beside 300 55 / 63, 79 / 85, 31 of
    64-500 beside 777 180 / 138)."""
    if max_qo_len == 1:
        least = 24.0
    elif tokens * hkv > 512 * 4 * (32 // (hq // hkv)):
        least = 90.0
    else:
        least = 40.0 + 0.065 * max_qo_len
    return longest > least + min(0.0033 * hkv * pages, 160.0)


def _prefill_has_decode_rows(tokens: int, batch: int, max_qo_len: int, pages: int) -> bool:
    """Whether a prompt step whose caller does not say so is likely to hold rows with one new token and a
    long cache: the rows but the longest average under half its tokens (the row lengths themselves are on the
    device), hold 1024 cached tokens or more on average (1344 below 16 rows), and four times their new tokens
    (prompts without a past hold their new ones: 4096 and 1500 tokens, 162 us and 4 for two idle launches)."""
    if batch <= 0 or max_qo_len <= 0:
        return False
    long_pages = 64 if batch >= 16 else 84
    if max_qo_len == 1:
        return pages >= long_pages * batch
    rest, rest_pages = tokens - max_qo_len, pages - (max_qo_len + 15) // 16
    return (batch > 1 and 2 * rest < (batch - 1) * max_qo_len and rest_pages >= long_pages * (batch - 1)
            and PAGE_SIZE * rest_pages >= 4 * rest)


def paged_prefill_workspace_bytes(batch: int, hq: int, hkv: int, pages: int) -> int:
    """Bytes of ``paged_prefill``'s workspace for steps of up to ``batch`` rows and ``pages`` pages."""
    return int(_lib.query("delta_paged_prefill_rows_workspace_bytes", batch, hq, hkv, pages))


def paged_prefill(q: torch.Tensor, kv_cache: torch.Tensor, qo_indptr: torch.Tensor,
                  kv_indptr: torch.Tensor, kv_indices: torch.Tensor, kv_last_page_len: torch.Tensor, *,
                  max_qo_len: int, sm_scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                  lse: Optional[torch.Tensor] = None, single_pages: Optional[Sequence[int]] = None,
                  workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal paged prefill attention (``delta_paged_prefill_rows``); q/out [nnz, Hq, 128].

    ``single_pages``: the pages of each row of exactly one new token, where the caller knows them (they
    choose how those rows run, no result depends on them); without it they are guessed from the totals.
    ``workspace`` (``paged_prefill_workspace_bytes``) holds those rows' partials; without one they are
    allocated for the call, and where that fails the step runs without them."""
    dev = _check_cuda(q, kv_cache, qo_indptr, kv_indptr, kv_indices, kv_last_page_len, out, lse, workspace)
    _check_cache(kv_cache)
    hq, hkv = _check_heads(q, kv_cache)
    B = qo_indptr.numel() - 1
    _check_i32("qo_indptr", qo_indptr, B + 1)
    _check_i32("kv_indptr", kv_indptr, B + 1)
    _check_i32("kv_indices", kv_indices)
    _check_i32("kv_last_page_len", kv_last_page_len, B)
    if out is None:
        out = torch.empty_like(q)
    if out.shape != q.shape or out.dtype != q.dtype or out.stride(2) != 1:
        raise ValueError("out must match q's shape/dtype with unit inner stride")
    if lse is not None and (lse.dtype != torch.float32 or tuple(lse.shape) != (q.shape[0], hq)
                            or not lse.is_contiguous()):
        raise ValueError("lse must be contiguous fp32 [nnz, Hq]")
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(HEAD_DIM)
    pages = kv_indices.numel()
    if single_pages is not None:
        rows, total, longest = len(single_pages), sum(single_pages), max(single_pages, default=0)
        if rows > B or total > pages or min(single_pages, default=0) < 0:
            raise ValueError(f"single_pages names {rows} rows of {total} pages, the step has {B} of {pages}")
        split = _split_decode_rows(int(max_qo_len), q.shape[0], hq, hkv, total, longest)
    else:
        split = _prefill_has_decode_rows(q.shape[0], B, int(max_qo_len), pages)
        rows = total = longest = 0
        if split:
            rows = B if max_qo_len == 1 else B - 1
            total = pages if max_qo_len == 1 else pages - (int(max_qo_len) + 15) // 16
            longest = min(total, 4 * -(-total // rows))
    if split:
        need = paged_prefill_workspace_bytes(B, hq, hkv, pages)
        if workspace is None:
            try:  # of this call: safe on any stream, in any capture
                workspace = torch.empty(need, dtype=torch.uint8, device=dev)
            except torch.OutOfMemoryError:
                split = False
        elif workspace.numel() * workspace.element_size() < need:
            raise ValueError(f"workspace too small: {need} bytes needed")
    _lib.call("delta_paged_prefill_rows", q.data_ptr(), q.stride(0), q.stride(1), kv_cache.data_ptr(), kv_cache.shape[0],
              qo_indptr.data_ptr(), kv_indptr.data_ptr(), kv_indices.data_ptr(), pages, kv_last_page_len.data_ptr(),
              out.data_ptr(), out.stride(0), out.stride(1), _ptr(lse), int(B), hq, hkv, HEAD_DIM, _dtype_code(q),
              float(sm_scale), int(max_qo_len), q.shape[0], rows, total, longest, workspace.data_ptr() if split else None,
              workspace.numel() * workspace.element_size() if split else 0, _stream(dev))
    return out


@functools.lru_cache(maxsize=1024)
def prefix_attention_workspace_bytes(tokens: int, hq: int, hkv: int, max_pages: int) -> int:
    """Bytes of workspace of ``paged_decode_prefix`` (``tokens`` = rows, ``max_pages`` = its ``max_pages_per_row``)
    and ``paged_prefill_prefix`` (``tokens`` = query tokens, ``max_pages`` = entries of ``kv_indices``)."""
    return int(_lib.query("delta_prefix_attention_workspace_bytes", int(tokens), int(hq), int(hkv), int(max_pages)))


def _call_on(dev: torch.device, name: str, *args) -> None:
    """``_lib.call`` with ``dev`` as the current device (the launch's stream is one of its)."""
    if dev.index == torch.cuda.current_device():
        _lib.call(name, *args, torch._C._cuda_getCurrentRawStream(dev.index))
    else:
        with torch.cuda.device(dev):
            _lib.call(name, *args, _stream(dev))


def _prefix_call(name: str, q, kv_cache, B: int, tables: tuple, prefix: tuple, out, lse, workspace, max_pages: int,
                 sm_scale: Optional[float], tail: tuple, alone: Optional[int] = None) -> torch.Tensor:
    """What the two attention calls over shared prefixes have in common: checks, outputs, workspace, the call.
    ``tables`` are the row tables in the entry point's order, the page indices next to last; ``tail`` the arguments
    between the batch and the head counts.  ``alone``: max_qo_len of prompts that the ordinary launch attends faster."""
    indices, row_prefix, p_indptr, p_indices = tables[-2], *prefix
    dev = _check_cuda(q, kv_cache, *tables, *prefix, out, lse, workspace)
    _check_cache(kv_cache)
    hq, hkv = _check_heads(q, kv_cache)
    for what, t, n in (("kv_indptr", tables[-3], B + 1), ("kv_indices", indices, 0), ("kv_last_page_len", tables[-1], B),
                       ("row_prefix", row_prefix, B), ("prefix_indptr", p_indptr, 1), ("prefix_indices", p_indices, 0)):
        _check_i32(what, t, n)
    if out is None:
        out = torch.empty_like(q)
    elif out.shape != q.shape or out.dtype != q.dtype or out.stride(2) != 1:
        raise ValueError("out must match q's shape/dtype with unit inner stride")
    if lse is not None and (lse.dtype != torch.float32 or lse.shape != q.shape[:2] or not lse.is_contiguous()):
        raise ValueError(f"lse must be contiguous fp32 [{q.shape[0]}, {hq}]")
    scale = _DEFAULT_SCALE if sm_scale is None else float(sm_scale)
    if alone is not None and out.data_ptr() % 8 == 0 and out.stride(0) % 4 == 0 and out.stride(1) % 4 == 0:
        _call_on(dev, "delta_paged_prefill_rows", q.data_ptr(), q.stride(0), q.stride(1), kv_cache.data_ptr(),
                 kv_cache.shape[0], *[t.data_ptr() for t in tables[:-1]], indices.numel(), tables[-1].data_ptr(),
                 out.data_ptr(), out.stride(0), out.stride(1), _ptr(lse), B, hq, hkv, HEAD_DIM, _DTYPES[q.dtype], scale,
                 alone, q.shape[0], 0, 0, 0, None, 0)
        return out
    need = prefix_attention_workspace_bytes(q.shape[0], hq, hkv, max_pages)
    if workspace is None:  # of this call: safe on any stream, in any capture
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    elif workspace.numel() * workspace.element_size() < need:
        raise ValueError(f"workspace too small: {need} bytes needed")
    px = _lib.SharedPrefixC(row_prefix.data_ptr(), p_indptr.data_ptr(), p_indices.data_ptr(), p_indices.numel(),
                            p_indptr.numel() - 1)
    _call_on(dev, name, ctypes.byref(px), q.data_ptr(), q.stride(0), q.stride(1), kv_cache.data_ptr(), kv_cache.shape[0],
             *[t.data_ptr() for t in tables[:-1]], indices.numel(), tables[-1].data_ptr(), out.data_ptr(), out.stride(0),
             out.stride(1), _ptr(lse), B, *tail[0], hq, hkv, HEAD_DIM, _DTYPES[q.dtype],
             scale, *tail[1], workspace.data_ptr(), workspace.numel() * workspace.element_size())
    return out


def paged_decode_prefix(q: torch.Tensor, kv_cache: torch.Tensor, kv_indptr: torch.Tensor, kv_indices: torch.Tensor,
                        kv_last_page_len: torch.Tensor, row_prefix: torch.Tensor, prefix_indptr: torch.Tensor,
                        prefix_indices: torch.Tensor, *, max_pages_per_row: int, sm_scale: Optional[float] = None,
                        out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                        workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``paged_decode`` for a batch whose rows share prefixes (``delta_paged_decode_prefix``): each prefix's pages
    are read once for all its rows.

    ``row_prefix`` (int32 [B]) names each row's prefix, -1 for none; prefix p's full pages are
    ``prefix_indices[prefix_indptr[p]:prefix_indptr[p + 1]]``, and the rows' CSR lists them too, first.  A row that
    its prefix does not fit in attends its own CSR alone, and so do all rows of a small batch (``decode_alone`` in
    csrc/prefix_attention.hip).  At most 1024 rows and prefixes.  ``workspace``
    (``prefix_attention_workspace_bytes``) is allocated for the call where none is given."""
    return _prefix_call("delta_paged_decode_prefix", q, kv_cache, q.shape[0], (kv_indptr, kv_indices, kv_last_page_len),
                        (row_prefix, prefix_indptr, prefix_indices), out, lse, workspace, int(max_pages_per_row), sm_scale,
                        ((), (int(max_pages_per_row),)))


def paged_prefill_prefix(q: torch.Tensor, kv_cache: torch.Tensor, qo_indptr: torch.Tensor, kv_indptr: torch.Tensor,
                         kv_indices: torch.Tensor, kv_last_page_len: torch.Tensor, row_prefix: torch.Tensor,
                         prefix_indptr: torch.Tensor, prefix_indices: torch.Tensor, *, max_qo_len: int,
                         max_pages_per_row: Optional[int] = None, sm_scale: Optional[float] = None,
                         out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                         workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``paged_prefill`` for prompts that continue shared prefixes (``delta_paged_prefill_prefix``); q/out
    [nnz, Hq, 128], the prefixes as in ``paged_decode_prefix``.

    A row's prefix applies where it ends before the row's query tokens.  ``max_qo_len`` is at least the longest row's
    count of them, as for ``paged_prefill``, which is as fast or faster where the rows bring several hundred tokens each
    (sharing spares reads, not products).  ``max_pages_per_row``, where the caller knows it, is the most pages of a row: up
    to 40 the ordinary launch attends the rows (32 rows of 20 pages 11 us, shared 31).  ``out`` and ``lse`` of tokens behind
    the last row are left as they were."""
    _check_i32("qo_indptr", qo_indptr, 1)
    return _prefix_call("delta_paged_prefill_prefix", q, kv_cache, qo_indptr.numel() - 1,
                        (qo_indptr, kv_indptr, kv_indices, kv_last_page_len), (row_prefix, prefix_indptr, prefix_indices),
                        out, lse, workspace, kv_indices.numel(), sm_scale, ((q.shape[0], int(max_qo_len)), ()),
                        int(max_qo_len) if max_pages_per_row is not None and max_pages_per_row <= 40 else None)


@dataclass(frozen=True)
class Rotary:
    """A position rotation of each head's first ``rotary_dim`` elements (``delta_rotary_t``), made by ``rotary`` once
    per model and device: ``turns`` (int64 [rotary_dim / 2]) is each pair's turn per position as a fraction of 2^64."""
    turns: torch.Tensor
    rotary_dim: int
    interleaved: bool
    factor: float
    c: _lib.RotaryC


def rotary_frequencies(rotary_dim: int, *, rope_theta: float = 1e4, rope_scale: float = 1.0,
                       low_freq_factor: Optional[float] = None, high_freq_factor: Optional[float] = None,
                       old_context_len: Optional[float] = None, scaling: Optional[str] = None, beta_fast: float = 32.0,
                       beta_slow: float = 1.0, ramp: str = "turns"):
    """(radians per position of each pair, factor on what is rotated) of a scaling, in 64 bits.

    With f_j = rope_theta^(-2j / rotary_dim), s = rope_scale and r_j = old_context_len f_j / (2 pi), the turns over the
    trained context:
      ``linear``  f_j / s
      ``ntk``     f_j of the base rope_theta s^(rotary_dim / (rotary_dim - 2)): the first pair's kept, the last one's / s
      ``llama31`` f_j / s where r_j <= low_freq_factor, f_j where r_j >= high_freq_factor, between them linear in r_j
      ``yarn``    the same between beta_slow and beta_fast turns, and a factor of 0.1 ln(s) + 1 (s > 1) on q and k;
                  with ``ramp="pairs"`` linear in j instead, from the pair of beta_fast turns (rounded down) to that of
                  beta_slow turns (rounded up).  The first is the formula as published; checkpoints whose configuration
                  says "yarn" are trained with the second, whose pairs between the two ends turn faster (s = 4: the
                  first's are up to 42% slower)
    Without ``scaling``: ``llama31`` where both frequency factors are given, as for ``rope``, else ``linear``."""
    if rotary_dim % 2 or not 2 <= rotary_dim <= HEAD_DIM:
        raise ValueError(f"rotary_dim must be even and in [2, {HEAD_DIM}], got {rotary_dim}")
    if not rope_theta > 0 or not rope_scale > 0 or math.isinf(rope_theta) or math.isinf(rope_scale):
        raise ValueError("rope_theta and rope_scale must be positive and finite")
    if ramp not in ("turns", "pairs") or (ramp == "pairs" and scaling != "yarn"):
        raise ValueError(f"ramp must be 'turns', or for yarn 'pairs', got {ramp!r}")
    if scaling is None:
        scaling = "llama31" if low_freq_factor is not None and high_freq_factor is not None else "linear"
    theta, factor = float(rope_theta), 1.0
    if scaling == "ntk":
        if rotary_dim == 2:
            raise ValueError("ntk scaling needs a rotary_dim over 2")
        theta *= rope_scale ** (rotary_dim / (rotary_dim - 2))
    freqs = [theta ** (-2.0 * j / rotary_dim) for j in range(rotary_dim // 2)]
    if scaling == "linear":
        freqs = [f / rope_scale for f in freqs]
    elif scaling in ("llama31", "yarn"):
        lo, hi = (low_freq_factor, high_freq_factor) if scaling == "llama31" else (beta_slow, beta_fast)
        if lo is None or hi is None or not hi > lo > 0 or old_context_len is None or not old_context_len > 0:
            raise ValueError(f"{scaling} scaling needs old_context_len and 0 < low < high turns")
        if ramp == "pairs":  # pair j turns L theta^(-2j / R) / (2 pi) times
            if not theta > 1:
                raise ValueError("a ramp over the pairs needs a rope_theta over 1")
            at = [rotary_dim * math.log(old_context_len / (2 * math.pi * r)) / (2 * math.log(theta)) for r in (hi, lo)]
            first, last = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rotary_dim - 1)
            keep = [1.0 - min(max((j - first) / max(last - first, 1), 0.0), 1.0) for j in range(len(freqs))]
        else:
            keep = [min(max((old_context_len * f / (2 * math.pi) - lo) / (hi - lo), 0.0), 1.0) for f in freqs]
        freqs = [f / rope_scale * (1 - k) + f * k for f, k in zip(freqs, keep)]
        if scaling == "yarn" and rope_scale > 1:
            factor = 0.1 * math.log(rope_scale) + 1.0
    elif scaling != "ntk":
        raise ValueError(f"unknown scaling {scaling!r}")
    return freqs, factor


def rotary(rotary_dim: int = HEAD_DIM, *, interleaved: bool = False, device=None,
           frequencies: Optional[Sequence[float]] = None, factor: Optional[float] = None, **scaling) -> Rotary:
    """The rotation that ``qk_norm_rope`` and ``qk_norm_rope_append`` apply; keep it for all layers and steps.

    Pairs (2j, 2j + 1) where ``interleaved``, else (j, j + rotary_dim / 2).  ``scaling``: the arguments of
    ``rotary_frequencies``; or ``frequencies``, each pair's radians per position, as they are.  ``factor`` replaces the
    scaling's."""
    if frequencies is None:
        freqs, f = rotary_frequencies(rotary_dim, **scaling)
    else:
        freqs, f = [float(x) for x in frequencies], 1.0
        if scaling:
            raise ValueError("frequencies are taken as they are: no scaling beside them")
        if rotary_dim % 2 or not 2 <= rotary_dim <= HEAD_DIM or len(freqs) != rotary_dim // 2:
            raise ValueError(f"{rotary_dim // 2} frequencies for an even rotary_dim in [2, {HEAD_DIM}], got {len(freqs)}")
        if not all(math.isfinite(x) for x in freqs):
            raise ValueError("frequencies must be finite")
    f = f if factor is None else float(factor)
    if not math.isfinite(f):
        raise ValueError("factor must be finite")
    turns = [int(math.ldexp(math.fmod(x / (2 * math.pi), 1.0), 64)) % (1 << 64) for x in freqs]
    t = torch.tensor([v - (1 << 64) if v >> 63 else v for v in turns], dtype=torch.int64, device=device or "cuda")
    return Rotary(t, rotary_dim, bool(interleaved), f, _lib.RotaryC(t.data_ptr(), rotary_dim, int(bool(interleaved)), f))


# The calls below take a few microseconds on the GPU, so what they check on the host they check in as few steps as that
# takes: one condition over all of it, and only where that fails the checks that say what is wrong.
def _launch(index: int, name: str, *args) -> None:
    """``_lib.call`` on GPU ``index``'s current stream."""
    if index == torch._C._cuda_getDevice():
        _lib.call(name, *args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            _lib.call(name, *args, torch._C._cuda_getCurrentRawStream(index))


def _same_gpu(first: torch.Tensor, *tensors) -> int:
    """The GPU that all the tensors (None: left out) are on."""
    index = first.get_device()
    if index < 0:
        _check_cuda(first)
    for t in tensors:
        if t is not None and t.get_device() != index:
            _check_cuda(t, device=first.device)
    return index


def _head_rows(name: str, t: torch.Tensor, dtype: torch.dtype, heads: Optional[int] = None, rows: Optional[int] = None):
    """(rows, heads, row stride) of [rows, heads, 128] with contiguous heads and 16-byte aligned rows."""
    shape, stride = t.shape, t.stride()
    if len(shape) != 3 or shape[2] != HEAD_DIM or stride[2] != 1 or (stride[1] != HEAD_DIM and shape[1] != 1) \
            or stride[0] % 8 or t.data_ptr() % 16 or (heads is not None and shape[1] != heads):
        raise ValueError(f"{name} must be [nnz, {heads or 'heads'}, 128] with contiguous heads and 16-byte aligned rows")
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}, as q, is {t.dtype}")
    if rows is not None and shape[0] != rows:
        raise ValueError(f"{name} holds {shape[0]} tokens, q {rows}")
    return shape[0], shape[1], stride[0]


def _norm_c(dtype, q_weight, k_weight, eps):
    if q_weight is None and k_weight is None:
        return None
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is None or w.dtype is not dtype or w.numel() != HEAD_DIM or not w.is_contiguous() or w.data_ptr() % 16:
            raise ValueError(f"{name} must be a contiguous, 16-byte aligned [128] tensor of q's dtype (both weights or none)")
    return ctypes.byref(_lib.HeadNormC(q_weight.data_ptr(), k_weight.data_ptr(), eps))


def _i32_tables(*named) -> None:
    """``_check_i32`` of (name, tensor, least entries), for each."""
    for name, t, n in named:
        if t.dtype is not torch.int32 or t.numel() < n or not t.is_contiguous():
            _check_i32(name, t, n)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, indptr: torch.Tensor, offsets: torch.Tensor,
                 rotary: Optional[Rotary], *, q_weight: Optional[torch.Tensor] = None,
                 k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, q_out: Optional[torch.Tensor] = None,
                 k_out: Optional[torch.Tensor] = None):
    """RMS norm of each head (with ``q_weight`` and ``k_weight``, [128] each) and rotation by the token's position, in
    fp32, rounded once (``delta_qk_norm_rope``); returns (q_out, k_out), which may be q and k themselves.

    Token i of row b (rows from ``indptr``) is at position ``offsets[b] + i - indptr[b]``; tokens of no row are left
    as they were."""
    gpu = _same_gpu(q, k, indptr, offsets, q_weight, k_weight, q_out, k_out, None if rotary is None else rotary.turns)
    dtype = q.dtype
    code = _dtype_code(q)
    T, hq, qs = _head_rows("q", q, dtype)
    _, hkv, ks = _head_rows("k", k, dtype, None, T)
    B = indptr.numel() - 1
    _i32_tables(("indptr", indptr, 1), ("offsets", offsets, B))
    q_out = torch.empty_like(q) if q_out is None else q_out
    k_out = torch.empty_like(k) if k_out is None else k_out
    qos, kos = _head_rows("q_out", q_out, dtype, hq, T)[2], _head_rows("k_out", k_out, dtype, hkv, T)[2]
    _launch(gpu, "delta_qk_norm_rope", None if rotary is None else rotary.c, _norm_c(dtype, q_weight, k_weight, eps),
            q.data_ptr(), qs, k.data_ptr(), ks, q_out.data_ptr(), qos, k_out.data_ptr(), kos, indptr.data_ptr(),
            offsets.data_ptr(), T, B, hq, hkv, HEAD_DIM, code)
    return q_out, k_out


def qk_norm_rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, kv_append_indptr: torch.Tensor,
                        offsets: torch.Tensor, kv_cache: torch.Tensor, kv_indices: torch.Tensor, kv_indptr: torch.Tensor,
                        kv_last_page_len: torch.Tensor, rotary: Optional[Rotary], *,
                        q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                        eps: float = 1e-6, q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``qk_norm_rope`` then ``append_kv`` of its keys and of ``v`` in one launch (``delta_qk_norm_rope_append``);
    returns the rotated q (``q_out``, which may be q itself)."""
    gpu = _same_gpu(q, k, v, kv_append_indptr, offsets, kv_cache, kv_indices, kv_indptr, kv_last_page_len, q_weight, k_weight,
                    q_out, None if rotary is None else rotary.turns)
    dtype = q.dtype
    code = _dtype_code(q)
    _check_cache(kv_cache)
    if kv_cache.dtype is not dtype:
        raise TypeError(f"kv_cache must be {dtype}, as q, is {kv_cache.dtype}")
    pages, _, _, hkv, _ = kv_cache.shape
    T, hq, qs = _head_rows("q", q, dtype)
    ks, vs = _head_rows("k", k, dtype, hkv, T)[2], _head_rows("v", v, dtype, hkv, T)[2]
    B = kv_append_indptr.numel() - 1
    _i32_tables(("kv_append_indptr", kv_append_indptr, 1), ("offsets", offsets, B), ("kv_indices", kv_indices, 0),
                ("kv_indptr", kv_indptr, B + 1), ("kv_last_page_len", kv_last_page_len, B))
    q_out = torch.empty_like(q) if q_out is None else q_out
    qos = _head_rows("q_out", q_out, dtype, hq, T)[2]
    _launch(gpu, "delta_qk_norm_rope_append", None if rotary is None else rotary.c,
            _norm_c(dtype, q_weight, k_weight, eps), q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs,
            q_out.data_ptr(), qos, kv_append_indptr.data_ptr(), offsets.data_ptr(), kv_cache.data_ptr(), pages,
            kv_indices.data_ptr(), kv_indices.numel(), kv_indptr.data_ptr(), kv_last_page_len.data_ptr(), T, B, hq, hkv,
            HEAD_DIM, code)
    return q_out


@dataclass
class ScoreRule:
    """What attention does to the score ``x = q.k * sm_scale`` of a query token at position ``pos`` and a key
    (``delta_score_rule_t``), in this order:

    * ``softcap`` c > 0: ``c * tanh(x / c)``;
    * ``slopes`` (fp32 [Hq]): ``x - slopes[h] * |pos - key|``;
    * ``window`` w > 0: keys in front of ``pos - w + 1`` are left out;
    * ``kv_begin`` (int32 [tokens]): keys in front of ``kv_begin[token]`` are left out -- for documents packed into a
      row each token's first key of its own document;
    * ``kv_end`` (int32 [tokens]): keys from ``kv_end[token]`` on are left out, instead of those behind ``pos`` -- a prefix
      seen as a whole is ``max(pos + 1, prefix length)``.

    Key positions count from the row's first cached token.  A token that sees no key gets o = 0 and lse = -inf."""
    softcap: float = 0.0
    slopes: Optional[torch.Tensor] = None
    window: int = 0
    kv_begin: Optional[torch.Tensor] = None
    kv_end: Optional[torch.Tensor] = None


def _rule_call(name: str, q, kv_cache, B: int, qo_indptr, kv_indptr, kv_indices, kv_last_page_len, rule: ScoreRule, out,
               lse, workspace, size, sm_scale, longest: int) -> torch.Tensor:
    """What the two attention calls under a score rule have in common: checks, outputs, workspace, the call.  ``size`` is
    the workspace's query of the head counts and the window, ``longest`` the call's maximum over the rows."""
    slopes, begin, end, window = rule.slopes, rule.kv_begin, rule.kv_end, rule.window
    gpu = _same_gpu(q, kv_cache, qo_indptr, kv_indptr, kv_indices, kv_last_page_len, slopes, begin, end, out, lse, workspace)
    _check_cache(kv_cache)
    hq, hkv = _check_heads(q, kv_cache)
    T = q.shape[0]
    _i32_tables(("kv_indptr", kv_indptr, B + 1), ("kv_indices", kv_indices, 0), ("kv_last_page_len", kv_last_page_len, B))
    if slopes is not None and (slopes.dtype is not torch.float32 or slopes.numel() != hq or not slopes.is_contiguous()):
        raise ValueError(f"slopes must be contiguous fp32 [{hq}]")
    if begin is not None:
        _check_i32("kv_begin", begin, T)
    if end is not None:
        _check_i32("kv_end", end, T)
    if not 0 <= window < 1 << 31:
        raise ValueError(f"window must be 0 (none) or a positive int32, got {window}")
    if out is None:
        out = torch.empty_like(q)
    elif out.shape != q.shape or out.dtype is not q.dtype or out.stride(2) != 1:
        raise ValueError("out must match q's shape/dtype with unit inner stride")
    ot, oh, _ = out.stride()
    if lse is not None and (lse.dtype is not torch.float32 or lse.shape != (T, hq) or not lse.is_contiguous()):
        raise ValueError(f"lse must be contiguous fp32 [{T}, {hq}]")
    need = size(hq, hkv, window)
    if workspace is None:  # of this call: safe on any stream, in any capture
        if need:
            workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    else:
        nbytes = workspace.numel() * workspace.element_size()
        if nbytes < need:
            raise ValueError(f"workspace too small: {need} bytes needed")
        need = nbytes
    qt, qh, _ = q.stride()
    args = (_lib.ScoreRuleC(rule.softcap, _ptr(slopes), window, _ptr(begin), _ptr(end)), q.data_ptr(), qt, qh,
            kv_cache.data_ptr(), kv_cache.shape[0])
    tables = (kv_indptr.data_ptr(), kv_indices.data_ptr(), kv_indices.numel(), kv_last_page_len.data_ptr(), out.data_ptr(),
              ot, oh, _ptr(lse), B)
    scale = _DEFAULT_SCALE if sm_scale is None else float(sm_scale)
    ws = _ptr(workspace), need
    if qo_indptr is None:
        _launch(gpu, name, *args, *tables, hq, hkv, HEAD_DIM, _DTYPES[q.dtype], scale, longest, *ws)
    else:
        _launch(gpu, name, *args, qo_indptr.data_ptr(), *tables, T, longest, hq, hkv, HEAD_DIM, _DTYPES[q.dtype], scale, *ws)
    return out


@functools.lru_cache(maxsize=1024)
def decode_rule_workspace_bytes(batch: int, hq: int, hkv: int, max_pages: int, window: int = 0) -> int:
    """Bytes of ``paged_decode_rule``'s workspace."""
    return int(_lib.query("delta_paged_decode_rule_workspace_bytes", batch, hq, hkv, max_pages, window))


@functools.lru_cache(maxsize=1024)
def prefill_rule_workspace_bytes(tokens: int, batch: int, hq: int, hkv: int, max_qo_len: int, pages: int,
                                 window: int = 0) -> int:
    """Bytes of ``paged_prefill_rule``'s workspace (``pages``: entries of its ``kv_indices``)."""
    return int(_lib.query("delta_paged_prefill_rule_workspace_bytes", tokens, batch, hq, hkv, max_qo_len, pages, window))


def paged_decode_rule(q: torch.Tensor, kv_cache: torch.Tensor, kv_indptr: torch.Tensor, kv_indices: torch.Tensor,
                      kv_last_page_len: torch.Tensor, rule: ScoreRule, *, max_pages_per_row: int,
                      sm_scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                      lse: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``paged_decode`` under a score rule (``delta_paged_decode_rule``): one query token per row, the last of its cached
    ones; only the pages of keys that the rule leaves in are read.  At most 16 kv heads, as ``paged_decode``; more of them are
    ``paged_prefill_rule``'s, with ``max_qo_len=1``.

    ``workspace`` (``decode_rule_workspace_bytes``) is allocated for the call where none is given."""
    B, mp = q.shape[0], int(max_pages_per_row)
    return _rule_call("delta_paged_decode_rule", q, kv_cache, B, None, kv_indptr, kv_indices, kv_last_page_len, rule, out,
                      lse, workspace, lambda hq, hkv, w: decode_rule_workspace_bytes(B, hq, hkv, mp, w), sm_scale, mp)


def paged_prefill_rule(q: torch.Tensor, kv_cache: torch.Tensor, qo_indptr: torch.Tensor, kv_indptr: torch.Tensor,
                       kv_indices: torch.Tensor, kv_last_page_len: torch.Tensor, rule: ScoreRule, *, max_qo_len: int,
                       sm_scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                       lse: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``paged_prefill`` under a score rule (``delta_paged_prefill_rule``); q/out [nnz, Hq, 128], row b's last
    ``qo_indptr[b + 1] - qo_indptr[b]`` cached tokens its query tokens, ``max_qo_len`` at least the longest row's count.

    ``out`` and ``lse`` of tokens behind the last row are left as they were.  ``workspace``
    (``prefill_rule_workspace_bytes``) is allocated for the call where none is given."""
    _i32_tables(("qo_indptr", qo_indptr, 1))
    B, T, mq, pages = qo_indptr.numel() - 1, q.shape[0], int(max_qo_len), kv_indices.numel()
    return _rule_call("delta_paged_prefill_rule", q, kv_cache, B, qo_indptr, kv_indptr, kv_indices, kv_last_page_len, rule,
                      out, lse, workspace, lambda hq, hkv, w: prefill_rule_workspace_bytes(T, B, hq, hkv, mq, pages, w),
                      sm_scale, mq)


def copy_pages(caches: Sequence[torch.Tensor], src: torch.Tensor, dst: torch.Tensor, *,
               tokens: Optional[torch.Tensor] = None) -> None:
    """Copy pages in place inside each of ``caches`` (one per layer, one shape) in one launch (``delta_copy_pages``):
    entry i copies the first ``tokens[i]`` tokens (all 16 without ``tokens``) of page ``src[i]`` to page ``dst[i]``.

    Entries run in no order: a ``dst`` may not be listed twice nor be another entry's ``src``; a ``src`` may be listed
    any number of times.  An entry with a page id outside the caches copies nothing."""
    if len(caches) == 0:
        raise ValueError("no caches")
    first = caches[0]
    dev = _check_cuda(first, src, dst, tokens)
    _check_cache(first)
    shape, dtype = first.shape, first.dtype
    for c in caches:  # (a launch of a few microseconds goes over every layer: no more than is needed for each)
        if c.shape != shape or c.dtype is not dtype or c.device != dev or not c.is_contiguous():
            raise ValueError("the caches must be contiguous, on one device, and share a shape and a dtype")
    n = src.numel()
    _check_i32("src", src)
    _check_i32("dst", dst)
    if dst.numel() != n:
        raise ValueError(f"src names {n} pages, dst {dst.numel()}")
    if tokens is not None:
        _check_i32("tokens", tokens)
        if tokens.numel() != n:
            raise ValueError(f"src names {n} pages, tokens {tokens.numel()}")
    ptrs = (ctypes.c_void_p * len(caches))(*[c.data_ptr() for c in caches])
    _call_on(dev, "delta_copy_pages", ptrs, len(caches), shape[0], shape[3], HEAD_DIM, _DTYPES[dtype], src.data_ptr(),
             dst.data_ptr(), _ptr(tokens), n)


def page_scores_from_logits(logits_dump: torch.Tensor, kv_indptr: torch.Tensor,
                            kv_last_page_len: torch.Tensor, max_pages: int, *,
                            lse: Optional[torch.Tensor] = None,
                            scores: Optional[torch.Tensor] = None,
                            batch: Optional[int] = None,
                            workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """del3_legacy_softmax page scores from a logits dump; returns fp32 [B, max_pages]."""
    dev = _check_cuda(logits_dump, kv_indptr, kv_last_page_len, lse, scores)
    if logits_dump.dtype != torch.float32 or logits_dump.dim() != 3 or logits_dump.stride(2) != 1:
        raise ValueError("logits_dump must be fp32 [B, Hq, S] with unit last stride")
    B = int(batch if batch is not None else kv_indptr.numel() - 1)
    hq = logits_dump.shape[1]
    if logits_dump.shape[0] < B or logits_dump.shape[2] < max_pages * PAGE_SIZE:
        raise ValueError("logits_dump too small")
    _check_i32("kv_indptr", kv_indptr, B + 1)
    _check_i32("kv_last_page_len", kv_last_page_len, B)
    if scores is None:
        scores = torch.empty((B, max_pages), dtype=torch.float32, device=dev)
    if scores.dtype != torch.float32 or scores.stride(1) != 1 or scores.shape[0] < B \
            or scores.shape[1] < max_pages:
        raise ValueError("scores must be fp32 [>=B, >=max_pages] with unit inner stride")
    if lse is not None and (lse.dtype != torch.float32 or not lse.is_contiguous()
                            or lse.shape[0] < B or lse.shape[1] != hq):
        raise ValueError("lse must be contiguous fp32 [>=B, Hq]")
    need = int(_lib.query("delta_page_score_workspace_bytes", B, hq))
    if workspace is None:
        workspace = _default_ws.get(need, dev)
    _lib.call("delta_page_scores_from_logits",
              logits_dump.data_ptr(), logits_dump.stride(0), logits_dump.stride(1), _ptr(lse),
              kv_indptr.data_ptr(), kv_last_page_len.data_ptr(), scores.data_ptr(), scores.stride(0),
              B, hq, int(max_pages), workspace.data_ptr(),
              workspace.numel() * workspace.element_size(), _stream(dev))
    return scores


def page_score(q: torch.Tensor, kv_cache: torch.Tensor, kv_indptr: torch.Tensor,
               kv_indices: torch.Tensor, kv_last_page_len: torch.Tensor, max_pages: int, *,
               sm_scale: Optional[float] = None, logits_dump: Optional[torch.Tensor] = None,
               scores: Optional[torch.Tensor] = None,
               workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Standalone scorer (K read once): returns fp32 page scores [B, max_pages].

    Without ``logits_dump`` the scorer keeps each row's logits on chip when the shape allows
    (``delta_page_score_needs_dump`` == 0: no dump written); otherwise a dump buffer is used."""
    dev = _check_cuda(q, kv_cache, kv_indptr, kv_indices, kv_last_page_len, logits_dump, scores)
    _check_cache(kv_cache)
    hq, hkv = _check_heads(q, kv_cache)
    B = q.shape[0]
    _check_i32("kv_indptr", kv_indptr, B + 1)
    _check_i32("kv_indices", kv_indices)
    _check_i32("kv_last_page_len", kv_last_page_len, B)
    if logits_dump is None and int(_lib.query("delta_page_score_needs_dump", B, hq, hkv, max_pages)):
        logits_dump = torch.empty((B, hq, max_pages * PAGE_SIZE), dtype=torch.float32, device=dev)
    if logits_dump is not None and (
            logits_dump.dtype != torch.float32 or logits_dump.dim() != 3 or logits_dump.stride(2) != 1
            or logits_dump.shape[0] < B or logits_dump.shape[1] != hq
            or logits_dump.shape[2] < max_pages * PAGE_SIZE):
        raise ValueError("logits_dump must be fp32 [>=B, Hq, >=max_pages*16] with unit last stride")
    if scores is None:
        scores = torch.empty((B, max_pages), dtype=torch.float32, device=dev)
    if scores.dtype != torch.float32 or scores.stride(1) != 1 or scores.shape[0] < B \
            or scores.shape[1] < max_pages:
        raise ValueError("scores must be fp32 [>=B, >=max_pages]")
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(HEAD_DIM)
    need = int(_lib.query("delta_page_score_kv_workspace_bytes", B, hq, hkv, max_pages))
    if workspace is None:
        workspace = _default_ws.get(need, dev)
    _lib.call("delta_page_score",
              q.data_ptr(), q.stride(0), q.stride(1), kv_cache.data_ptr(), kv_cache.shape[0],
              kv_indptr.data_ptr(), kv_indices.data_ptr(), kv_indices.numel(),
              kv_last_page_len.data_ptr(), _ptr(logits_dump), 0 if logits_dump is None else logits_dump.stride(0),
              0 if logits_dump is None else logits_dump.stride(1), scores.data_ptr(), scores.stride(0),
              B, hq, hkv, HEAD_DIM, _dtype_code(q), float(sm_scale), int(max_pages),
              workspace.data_ptr(), workspace.numel() * workspace.element_size(), _stream(dev))
    return scores


def select_pages(scores: torch.Tensor, kv_indptr: torch.Tensor, block_table: torch.Tensor,
                 k: int, L: int, *, pos_bias_scale: float = 1e-7, fixed_count: bool = False,
                 batch: Optional[int] = None, max_pages: Optional[int] = None,
                 k_per_row: Optional[torch.Tensor] = None,
                 use_subset: Optional[torch.Tensor] = None,
                 out_indices: Optional[torch.Tensor] = None,
                 out_indptr: Optional[torch.Tensor] = None):
    """PageSelectorV2 selection (``delta_select_pages``) -> (indices, indptr) int32.

    ``out_indices`` is returned whole (callers slice with ``indptr[-1]``); when
    allocated here it holds ``batch * k`` entries (or the full page count when
    ``use_subset`` may be 0).
    """
    dev = _check_cuda(scores, kv_indptr, block_table, k_per_row, use_subset, out_indices, out_indptr)
    B = int(batch if batch is not None else kv_indptr.numel() - 1)
    n = int(max_pages if max_pages is not None else scores.shape[1])
    if scores.dtype != torch.float32 or scores.stride(1) != 1 or scores.shape[0] < B or scores.shape[1] < n:
        raise ValueError("scores must be fp32 [>=B, >=max_pages] with unit inner stride")
    _check_i32("kv_indptr", kv_indptr, B + 1)
    if block_table.dtype != torch.int32 or block_table.stride(1) != 1 or block_table.shape[0] < B \
            or block_table.shape[1] < n:
        raise ValueError("block_table must be int32 [>=B, >=max_pages] with unit inner stride")
    if k_per_row is not None:
        _check_i32("k_per_row", k_per_row, B)
    if use_subset is not None:
        _check_i32("use_subset", use_subset, 1)
    if k_per_row is None and k > n:
        raise RuntimeError("selected index k out of range")
    if out_indptr is None:
        out_indptr = torch.empty(B + 1, dtype=torch.int32, device=dev)
    _check_i32("out_indptr", out_indptr, B + 1)
    if out_indices is None:
        cap = B * max(int(k), 1) if k_per_row is None else int(k_per_row.sum())
        if use_subset is not None:
            cap = max(cap, B * n)
        out_indices = torch.empty(max(cap, 1), dtype=torch.int32, device=dev)
    _check_i32("out_indices", out_indices)
    _lib.call("delta_select_pages",
              scores.data_ptr(), scores.stride(0), kv_indptr.data_ptr(), block_table.data_ptr(),
              block_table.stride(0), B, n, int(k), _ptr(k_per_row), int(L), float(pos_bias_scale),
              int(bool(fixed_count)), _ptr(use_subset), out_indices.data_ptr(), out_indices.numel(),
              out_indptr.data_ptr(), _stream(dev))
    return out_indices, out_indptr


def pack_page_indices(slot_block_table: torch.Tensor, active_slots: torch.Tensor,
                      start_cols: torch.Tensor, counts: torch.Tensor, indptr: torch.Tensor,
                      out_indices: torch.Tensor, row_block_table: torch.Tensor, n_rows: int,
                      max_count: int, *, write_row_block: bool) -> None:
    """In-place page-list pack (``delta_pack_page_indices``, page_metadata.py:42-70)."""
    if n_rows <= 0 or max_count <= 0:
        return
    dev = _check_cuda(slot_block_table, active_slots, start_cols, counts, indptr, out_indices,
                      row_block_table)
    for name, t in (("slot_block_table", slot_block_table), ("active_slots", active_slots),
                    ("start_cols", start_cols), ("counts", counts), ("indptr", indptr),
                    ("out_indices", out_indices)):
        _check_i32(name, t)
    if write_row_block:
        _check_i32("row_block_table", row_block_table)
    if write_row_block and row_block_table.numel() < n_rows * slot_block_table.shape[1]:
        raise ValueError("row_block_table too small")
    if active_slots.numel() < n_rows or start_cols.numel() < n_rows or counts.numel() < n_rows \
            or indptr.numel() < n_rows:
        raise ValueError("metadata arrays shorter than n_rows")
    _lib.call("delta_pack_page_indices",
              slot_block_table.data_ptr(), int(slot_block_table.shape[0]), active_slots.data_ptr(),
              start_cols.data_ptr(), counts.data_ptr(), indptr.data_ptr(), out_indices.data_ptr(),
              out_indices.numel(), _ptr(row_block_table) if write_row_block else None, int(n_rows),
              int(slot_block_table.shape[1]), int(max_count), int(bool(write_row_block)),
              _stream(dev))


def decode_page_info(cachelens: torch.Tensor, slot_block_table: torch.Tensor, batch: int, k: int,
                     compression_ratio: float, selective: bool, kv_indptr: torch.Tensor,
                     kv_indices: torch.Tensor, kv_last_page_len: torch.Tensor,
                     row_block_table: Optional[torch.Tensor] = None,
                     subset_indices: Optional[torch.Tensor] = None,
                     subset_indptr: Optional[torch.Tensor] = None,
                     use_subset: Optional[torch.Tensor] = None,
                     active: Optional[torch.Tensor] = None,
                     k_per_row: Optional[torch.Tensor] = None,
                     budget_rule: Optional[tuple] = None) -> None:
    """Device-side decode page info for rows 0..batch-1 (``delta_decode_page_info``).

    ``active`` (int32 [batch], optional) marks the rows the ``use_subset`` gate counts; idle
    rows still get their CSR entries.  ``k_per_row`` (int32 [batch], optional) gives each row
    its own subset budget in place of ``k``.  ``budget_rule`` = ``(min_tokens, divisor, out)``
    derives each row's budget from its length instead, ``max(min_tokens, kv_len // divisor) // 16``
    pages clamped to [1, k], and writes them to ``out`` (int32 [batch]) for ``select_pages``."""
    rule_out = budget_rule[2] if budget_rule is not None else None
    dev = _check_cuda(cachelens, slot_block_table, kv_indptr, kv_indices, kv_last_page_len,
                      row_block_table, subset_indices, subset_indptr, use_subset, active, k_per_row, rule_out)
    pps = slot_block_table.shape[1]
    _check_i32("cachelens", cachelens, batch)
    if active is not None:
        _check_i32("active", active, batch)
    _check_i32("slot_block_table", slot_block_table, batch * pps)
    _check_i32("kv_indptr", kv_indptr, batch + 1)
    _check_i32("kv_indices", kv_indices, batch * pps)
    _check_i32("kv_last_page_len", kv_last_page_len, batch)
    if row_block_table is not None:
        _check_i32("row_block_table", row_block_table, batch * pps)
        if row_block_table.shape[-1] != pps:
            raise ValueError("row_block_table must have pages_per_slot columns")
    if subset_indices is not None:
        _check_i32("subset_indices", subset_indices, batch * pps)
        _check_i32("subset_indptr", subset_indptr, batch + 1)
    if use_subset is not None:
        _check_i32("use_subset", use_subset, 1)
    if k_per_row is not None:
        _check_i32("k_per_row", k_per_row, batch)
    rule = None
    if budget_rule is not None:
        if k_per_row is not None:
            raise ValueError("budget_rule and k_per_row are exclusive")
        min_tokens, divisor, out = budget_rule
        _check_i32("budget_rule out", out, batch)
        rule = ctypes.byref(_lib.BudgetRuleC(int(min_tokens), int(divisor), out.data_ptr()))
    _lib.call("delta_decode_page_info",
              cachelens.data_ptr(), _ptr(active), slot_block_table.data_ptr(), int(batch), int(pps), int(k),
              _ptr(k_per_row), rule, float(compression_ratio), int(bool(selective)), kv_indptr.data_ptr(),
              kv_indices.data_ptr(), kv_last_page_len.data_ptr(), _ptr(row_block_table),
              _ptr(subset_indices), _ptr(subset_indptr), _ptr(use_subset), _stream(dev))


def append_kv(k: torch.Tensor, v: torch.Tensor, kv_append_indptr: torch.Tensor,
              kv_cache: torch.Tensor, kv_indices: torch.Tensor, kv_indptr: torch.Tensor,
              kv_last_page_len: torch.Tensor) -> None:
    """In-place KV append (``delta_append_kv``, utils.py:31-79)."""
    dev = _check_cuda(k, v, kv_append_indptr, kv_cache, kv_indices, kv_indptr, kv_last_page_len)
    _check_cache(kv_cache)
    hkv = kv_cache.shape[3]
    for name, t in (("k", k), ("v", v)):
        if t.dim() != 3 or t.shape[1] != hkv or t.shape[2] != HEAD_DIM or t.stride(2) != 1 \
                or t.stride(1) != HEAD_DIM or t.stride(0) % 8:
            raise ValueError(f"{name} must be [nnz, {hkv}, 128] with contiguous heads")
        if t.dtype != kv_cache.dtype:
            raise TypeError(f"{name} dtype must match kv_cache")
    nnz = k.shape[0]
    if v.shape[0] != nnz:
        raise ValueError("k and v token counts differ")
    B = kv_append_indptr.numel() - 1
    _check_i32("kv_append_indptr", kv_append_indptr)
    _check_i32("kv_indices", kv_indices)
    _check_i32("kv_indptr", kv_indptr, B + 1)
    _check_i32("kv_last_page_len", kv_last_page_len, B)
    _lib.call("delta_append_kv",
              k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), kv_append_indptr.data_ptr(),
              kv_cache.data_ptr(), kv_cache.shape[0], kv_indices.data_ptr(), kv_indices.numel(),
              kv_indptr.data_ptr(), kv_last_page_len.data_ptr(), int(nnz), int(B), int(hkv),
              HEAD_DIM, _dtype_code(kv_cache), _stream(dev))


def rope(q: torch.Tensor, k: torch.Tensor, indptr: torch.Tensor, offsets: torch.Tensor, *,
         rope_scale: float = 1.0, rope_theta: float = 1e4,
         low_freq_factor: Optional[float] = None, high_freq_factor: Optional[float] = None,
         old_context_len: Optional[float] = None,
         q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None):
    """Interleaved RoPE (``delta_rope``); returns (q_rope, k_rope)."""
    dev = _check_cuda(q, k, indptr, offsets, q_out, k_out)
    for name, t in (("q", q), ("k", k)):
        if t.dim() != 3 or t.shape[2] != HEAD_DIM or t.stride(2) != 1 or t.stride(1) != HEAD_DIM:
            raise ValueError(f"{name} must be [nnz, H, 128] with contiguous heads")
    if k.dtype != q.dtype or k.shape[0] != q.shape[0]:
        raise ValueError("q/k mismatch")
    q_out = torch.empty_like(q) if q_out is None else q_out
    k_out = torch.empty_like(k) if k_out is None else k_out
    for name, t, ref in (("q_out", q_out, q), ("k_out", k_out, k)):
        if t.shape != ref.shape or t.dtype != ref.dtype or t.stride(2) != 1 or t.stride(1) != HEAD_DIM:
            raise ValueError(f"{name} must match its input's shape with contiguous heads")
    B = indptr.numel() - 1
    _check_i32("indptr", indptr, B + 1)
    _check_i32("offsets", offsets, B)
    llama31 = low_freq_factor is not None and high_freq_factor is not None
    _lib.call("delta_rope",
              q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0), q_out.data_ptr(),
              q_out.stride(0), k_out.data_ptr(), k_out.stride(0), indptr.data_ptr(),
              offsets.data_ptr(), int(q.shape[0]), int(B), int(q.shape[1]), int(k.shape[1]),
              HEAD_DIM, _dtype_code(q), float(rope_scale), float(rope_theta), int(llama31),
              float(low_freq_factor or 0.0), float(high_freq_factor or 0.0),
              float(old_context_len or 0.0), _stream(dev))
    return q_out, k_out


def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, kv_append_indptr: torch.Tensor,
                offsets: torch.Tensor, kv_cache: torch.Tensor, kv_indices: torch.Tensor,
                kv_indptr: torch.Tensor, kv_last_page_len: torch.Tensor, *, rope_scale: float = 1.0,
                rope_theta: float = 1e4, low_freq_factor: Optional[float] = None,
                high_freq_factor: Optional[float] = None, old_context_len: Optional[float] = None,
                q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``rope`` then ``append_kv`` in one launch (``delta_rope_append``); returns the rotated q."""
    dev = _check_cuda(q, k, v, kv_append_indptr, offsets, kv_cache, kv_indices, kv_indptr, kv_last_page_len, q_out)
    _check_cache(kv_cache)
    hkv = kv_cache.shape[3]
    if q.dim() != 3 or q.shape[2] != HEAD_DIM or q.stride(2) != 1 or q.stride(1) != HEAD_DIM:
        raise ValueError("q must be [nnz, Hq, 128] with contiguous heads")
    for name, t in (("k", k), ("v", v)):
        if t.dim() != 3 or t.shape[1] != hkv or t.shape[2] != HEAD_DIM or t.stride(2) != 1 \
                or t.stride(1) != HEAD_DIM or (name == "v" and t.stride(0) % 8) or t.shape[0] != q.shape[0]:
            raise ValueError(f"{name} must be [nnz, {hkv}, 128] with contiguous heads (v rows 16-byte aligned)")
        if t.dtype != kv_cache.dtype or q.dtype != kv_cache.dtype:
            raise TypeError("q, k, v and kv_cache must share a dtype")
    q_out = torch.empty_like(q) if q_out is None else q_out
    if q_out.shape != q.shape or q_out.dtype != q.dtype or q_out.stride(2) != 1 or q_out.stride(1) != HEAD_DIM:
        raise ValueError("q_out must match q's shape with contiguous heads")
    B = kv_append_indptr.numel() - 1
    _check_i32("kv_append_indptr", kv_append_indptr, B + 1)
    _check_i32("offsets", offsets, B)
    _check_i32("kv_indices", kv_indices)
    _check_i32("kv_indptr", kv_indptr, B + 1)
    _check_i32("kv_last_page_len", kv_last_page_len, B)
    llama31 = low_freq_factor is not None and high_freq_factor is not None
    _lib.call("delta_rope_append",
              q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), q_out.data_ptr(),
              q_out.stride(0), kv_append_indptr.data_ptr(), offsets.data_ptr(), kv_cache.data_ptr(),
              kv_cache.shape[0], kv_indices.data_ptr(), kv_indices.numel(), kv_indptr.data_ptr(),
              kv_last_page_len.data_ptr(), int(q.shape[0]), int(B), int(q.shape[1]), int(hkv), HEAD_DIM,
              _dtype_code(q), float(rope_scale), float(rope_theta), int(llama31), float(low_freq_factor or 0.0),
              float(high_freq_factor or 0.0), float(old_context_len or 0.0), _stream(dev))
    return q_out


def argmax_rows(logits: torch.Tensor, out: Optional[torch.Tensor] = None,
                workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """First index of each row's maximum (``delta_argmax_rows``); logits [rows, cols]."""
    dev = _check_cuda(logits, out, workspace)
    if logits.dim() != 2 or logits.stride(1) != 1:
        raise ValueError("logits must be [rows, cols] with unit inner stride")
    rows, cols = logits.shape
    if out is None:
        out = torch.empty(rows, dtype=torch.int64, device=dev)
    if out.dtype != torch.int64 or out.dim() != 1 or out.shape[0] < rows:
        raise ValueError("out must be int64 [>=rows]")
    need = int(_lib.query("delta_argmax_workspace_bytes", rows))
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    nbytes = workspace.numel() * workspace.element_size()
    _lib.call("delta_argmax_rows", logits.data_ptr(), logits.stride(0), int(rows), int(cols),
              _dtype_code(logits), out.data_ptr(), out.stride(0), workspace.data_ptr(), nbytes, _stream(dev))
    return out


def _rows2d(name: str, t: torch.Tensor, dim: int) -> torch.Tensor:
    t2 = t.reshape(-1, dim)
    if t2.stride(1) != 1 or t2.stride(0) % 8 or t2.data_ptr() % 16:
        raise ValueError(f"{name} must have 16-byte aligned contiguous rows")
    return t2


def add_rmsnorm(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor, eps: float,
                out: Optional[torch.Tensor] = None):
    """(x + residual, RMSNorm(x + residual) * weight) in one kernel (``delta_add_rmsnorm``).

    ``residual`` may also be the fp32 partials ``[S, rows, dim]`` of a split-K
    ``gemm_rows32`` (``delta_add_rmsnorm_partials``: summed and rounded to x's dtype first).
    Returns ``(h, y)``; ``h`` is ``x`` itself when ``residual`` is None."""
    dev = _check_cuda(x, residual, weight, out)
    dim = x.shape[-1]
    _dtype_code(x)
    if weight.dtype != x.dtype or weight.numel() != dim or not weight.is_contiguous():
        raise ValueError("weight must be a contiguous [dim] tensor of x's dtype")
    x2 = _rows2d("x", x, dim)
    rows = x2.shape[0]
    if residual is not None and residual.dtype == torch.float32 and x.dtype != torch.float32:
        if residual.dim() != 3 or tuple(residual.shape[1:]) != (rows, dim) or not residual.is_contiguous():
            raise ValueError(f"partials must be contiguous fp32 [S, {rows}, {dim}]")
        h = torch.empty_like(x)
        h2 = _rows2d("h", h, dim)
        if out is None:
            out = torch.empty_like(x)
        o2 = _rows2d("out", out, dim)
        _lib.call("delta_add_rmsnorm_partials", x2.data_ptr(), x2.stride(0), residual.data_ptr(),
                  int(residual.shape[0]), weight.data_ptr(), float(eps), h2.data_ptr(), h2.stride(0),
                  o2.data_ptr(), o2.stride(0), int(rows), int(dim), _dtype_code(x), _stream(dev))
        return h, out
    h = x if residual is None else torch.empty_like(x)
    r2 = None if residual is None else _rows2d("residual", residual, dim)
    h2 = None if residual is None else _rows2d("h", h, dim)
    if out is None:
        out = torch.empty_like(x)
    o2 = _rows2d("out", out, dim)
    _lib.call("delta_add_rmsnorm", x2.data_ptr(), x2.stride(0), _ptr(r2), 0 if r2 is None else r2.stride(0),
              weight.data_ptr(), float(eps), _ptr(h2), 0 if h2 is None else h2.stride(0), o2.data_ptr(),
              o2.stride(0), int(rows), int(dim), _dtype_code(x), _stream(dev))
    return h, out


def silu_mul(gate_up: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """silu(gate) * up of a ``[..., 2 * inter]`` gate|up tensor (``delta_silu_mul``)."""
    dev = _check_cuda(gate_up, out)
    inter = gate_up.shape[-1] // 2
    g2 = _rows2d("gate_up", gate_up, 2 * inter)
    if out is None:
        out = torch.empty(*gate_up.shape[:-1], inter, dtype=gate_up.dtype, device=dev)
    o2 = _rows2d("out", out, inter)
    _lib.call("delta_silu_mul", g2.data_ptr(), g2.stride(0), o2.data_ptr(), o2.stride(0), int(g2.shape[0]),
              int(inter), _dtype_code(gate_up), _stream(dev))
    return out


def gemm_skinny_ok(x: torch.Tensor, weight: torch.Tensor) -> bool:
    """True when ``delta_gemm_skinny`` takes ``x @ weight.T``: decode-sized rows, K % 64 == 0,
    N % 16 == 0, 16-byte aligned rows of a bf16/fp16 weight of x's dtype."""
    if x.dtype not in _DTYPES or weight.dtype != x.dtype or weight.dim() != 2 or not x.is_cuda:
        return False
    N, Kd = weight.shape
    rows = x.numel() // max(x.shape[-1], 1)
    return (x.shape[-1] == Kd and Kd % 64 == 0 and N % 16 == 0 and 0 < rows <= 32
            and weight.stride(1) == 1 and weight.stride(0) % 8 == 0 and weight.data_ptr() % 16 == 0)


def gemm_rows32_splits(M: int, N: int, K: int) -> int:
    """K splits ``delta_gemm_rows32`` uses for this shape (1: rounded output; > 1: fp32 partials)."""
    return int(_lib.query("delta_gemm_rows32_splits", int(M), int(N), int(K)))


def gemm_rows32(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                out: Optional[torch.Tensor] = None, partials: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x @ weight.T (+ bias)`` for <= 32 token rows on ``delta_gemm_rows32``.

    Returns the rounded output ``[..., N]`` when the shape runs unsplit, else the fp32 partials
    ``[S, M, N]`` whose sum over S is the product (bias included once)."""
    dev = _check_cuda(x, weight, bias, out, partials)
    N, Kd = weight.shape
    if x.shape[-1] != Kd:
        raise ValueError(f"x has {x.shape[-1]} features, weight expects {Kd}")
    if weight.dtype != x.dtype or (bias is not None and (bias.dtype != x.dtype or bias.numel() != N
                                                         or not bias.is_contiguous())):
        raise TypeError("x, weight and bias must share a dtype; bias must be contiguous [N]")
    if weight.stride(1) != 1:
        raise ValueError("weight rows must be contiguous")
    x2 = _rows2d("x", x, Kd)
    M = x2.shape[0]
    S = gemm_rows32_splits(M, N, Kd)
    if S < 1:
        raise ValueError(f"delta_gemm_rows32 does not take [{M}, {Kd}] x [{N}, {Kd}]^T")
    o2 = None
    if S == 1:
        if out is None:
            out = torch.empty(*x.shape[:-1], N, dtype=x.dtype, device=dev)
        o2 = out.reshape(-1, N)
        if o2.stride(1) != 1 or o2.shape[0] != M:
            raise ValueError("out must be [..., N] with contiguous rows")
    else:
        if partials is None:
            partials = torch.empty(S, M, N, dtype=torch.float32, device=dev)
        if partials.dtype != torch.float32 or not partials.is_contiguous() or tuple(partials.shape) != (S, M, N):
            raise ValueError(f"partials must be contiguous fp32 [{S}, {M}, {N}]")
    _lib.call("delta_gemm_rows32", x2.data_ptr(), x2.stride(0), weight.data_ptr(), weight.stride(0), _ptr(bias),
              o2.data_ptr() if o2 is not None else None, o2.stride(0) if o2 is not None else 0,
              partials.data_ptr() if S > 1 else None, int(M), int(N), int(Kd), _dtype_code(x), _stream(dev))
    return out if S == 1 else partials


def gemm_rows32_silu(x: torch.Tensor, w13: torch.Tensor, out: Optional[torch.Tensor] = None,
                     _entry: str = "delta_gemm_rows32_silu") -> torch.Tensor:
    """``silu(x @ w1.T) * (x @ w3.T)`` for <= 32 token rows in one launch (``delta_gemm_rows32_silu``);
    ``w13`` is the row-major merged ``[2 * inter, dim]`` weight (w1 rows, then w3 rows)."""
    dev = _check_cuda(x, w13, out)
    N2, Kd = w13.shape
    inter = N2 // 2
    if x.shape[-1] != Kd or N2 % 2:
        raise ValueError("x must be [..., dim] and w13 [2 * inter, dim]")
    if w13.dtype != x.dtype or w13.stride(1) != 1:
        raise ValueError("w13 must share x's dtype and have contiguous rows")
    x2 = _rows2d("x", x, Kd)
    M = x2.shape[0]
    if out is None:
        out = torch.empty(*x.shape[:-1], inter, dtype=x.dtype, device=dev)
    o2 = out.reshape(-1, inter)
    if o2.stride(1) != 1 or o2.shape[0] != M:
        raise ValueError("out must be [..., inter] with contiguous rows")
    _lib.call(_entry, x2.data_ptr(), x2.stride(0), w13.data_ptr(), w13.stride(0), o2.data_ptr(),
              o2.stride(0), int(M), int(inter), int(Kd), _dtype_code(x), _stream(dev))
    return out


def gemm_rows128_ok(x: torch.Tensor, weight: torch.Tensor) -> bool:
    """True when ``delta_gemm_rows128`` takes ``x @ weight.T`` for an inference call: at most 128
    contiguous, 16-byte aligned rows of a bf16/fp16 weight of x's dtype, K % 64 == 0, N % 16 == 0."""
    if x.dtype not in _DTYPES or weight.dtype != x.dtype or weight.dim() != 2 or not x.is_cuda \
            or weight.device != x.device:
        return False
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        return False
    N, Kd = weight.shape
    rows = x.numel() // max(x.shape[-1], 1)
    return (x.shape[-1] == Kd and Kd % 64 == 0 and N % 16 == 0 and 0 < rows <= 128 and x.is_contiguous()
            and x.data_ptr() % 16 == 0 and Kd <= 1 << 23 and weight.stride(1) == 1 and weight.stride(0) >= Kd
            and weight.stride(0) % 8 == 0 and weight.data_ptr() % 16 == 0 and (N + 192) * weight.stride(0) < 1 << 31)


def gemm_rows128_splits(M: int, N: int, K: int) -> int:
    """K splits ``delta_gemm_rows128`` uses for this shape (1: rounded output; > 1: fp32 partials)."""
    return int(_lib.query("delta_gemm_rows128_splits", int(M), int(N), int(K)))


def gemm_rows128(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                 out: Optional[torch.Tensor] = None, partials: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x @ weight.T (+ bias)`` for <= 128 token rows on ``delta_gemm_rows128``; returns as
    ``gemm_rows32`` does: the rounded output ``[..., N]``, or the fp32 partials ``[S, M, N]``."""
    dev = _check_cuda(x, weight, bias, out, partials)
    N, Kd = weight.shape
    if x.shape[-1] != Kd:
        raise ValueError(f"x has {x.shape[-1]} features, weight expects {Kd}")
    if weight.dtype != x.dtype or (bias is not None and (bias.dtype != x.dtype or bias.numel() != N
                                                         or not bias.is_contiguous())):
        raise TypeError("x, weight and bias must share a dtype; bias must be contiguous [N]")
    if weight.stride(1) != 1:
        raise ValueError("weight rows must be contiguous")
    x2 = _rows2d("x", x, Kd)
    M = x2.shape[0]
    S = gemm_rows128_splits(M, N, Kd)
    if S < 1:
        raise ValueError(f"delta_gemm_rows128 does not take [{M}, {Kd}] x [{N}, {Kd}]^T")
    o2 = None
    if S == 1:
        if out is None:
            out = torch.empty(*x.shape[:-1], N, dtype=x.dtype, device=dev)
        o2 = out.reshape(-1, N)
        if o2.stride(1) != 1 or o2.shape[0] != M or o2.data_ptr() != out.data_ptr() or o2.dtype != x.dtype:
            raise ValueError("out must be [..., N] of x's dtype with contiguous rows")
    else:
        if partials is None:
            partials = torch.empty(S, M, N, dtype=torch.float32, device=dev)
        if partials.dtype != torch.float32 or not partials.is_contiguous() or tuple(partials.shape) != (S, M, N):
            raise ValueError(f"partials must be contiguous fp32 [{S}, {M}, {N}]")
    _lib.call("delta_gemm_rows128", x2.data_ptr(), x2.stride(0), weight.data_ptr(), weight.stride(0), _ptr(bias),
              o2.data_ptr() if o2 is not None else None, o2.stride(0) if o2 is not None else 0,
              partials.data_ptr() if S > 1 else None, int(M), int(N), int(Kd), _dtype_code(x), _stream(dev))
    return out if S == 1 else partials


def gemm_rows128_silu(x: torch.Tensor, w13: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The fused gate/up GEMM + SiLU-mul for <= 128 token rows (``delta_gemm_rows128_silu``)."""
    return gemm_rows32_silu(x, w13, out, _entry="delta_gemm_rows128_silu")


def gemm_skinny_silu(x: torch.Tensor, w13: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The same fused gate/up GEMM + SiLU-mul for <= 8 token rows (``delta_gemm_skinny_silu``)."""
    return gemm_rows32_silu(x, w13, out, _entry="delta_gemm_skinny_silu")


def gemm_skinny(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``F.linear(x, weight, bias)`` for decode-sized x on ``delta_gemm_skinny``."""
    dev = _check_cuda(x, weight, bias, out)
    N, Kd = weight.shape
    if x.shape[-1] != Kd:
        raise ValueError(f"x has {x.shape[-1]} features, weight expects {Kd}")
    if weight.dtype != x.dtype or (bias is not None and (bias.dtype != x.dtype or bias.numel() != N
                                                         or not bias.is_contiguous())):
        raise TypeError("x, weight and bias must share a dtype; bias must be contiguous [N]")
    if weight.stride(1) != 1:
        raise ValueError("weight rows must be contiguous")
    x2 = _rows2d("x", x, Kd)
    M = x2.shape[0]
    if out is None:
        out = torch.empty(*x.shape[:-1], N, dtype=x.dtype, device=dev)
    o2 = out.reshape(-1, N)
    if o2.stride(1) != 1 or o2.shape[0] != M:
        raise ValueError("out must be [..., N] with contiguous rows")
    _lib.call("delta_gemm_skinny", x2.data_ptr(), x2.stride(0), weight.data_ptr(), weight.stride(0),
              _ptr(bias), o2.data_ptr(), o2.stride(0), int(M), int(N), int(Kd), _dtype_code(x), _stream(dev))
    return out
