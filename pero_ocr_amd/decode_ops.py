"""Decoding operators on torch tensors in HBM: a paged cache of attention keys and values in 8 bits or bfloat16, attention of the newest
tokens over it (single tokens, chains, trees of drafted tokens), and the scores of given tokens.

They stand next to the cached attention of the sequence-to-sequence engine (csrc/decoder.hpp, which keeps float32 keys and values of
one launch) and the logit operators `_native.ctc_greedy` / `_native.sparsify`, for a decoding loop of the caller's own; kernels and C entries:
csrc/decode_ops.hip, include/pocr.h "decoding operators".  One step of a loop that drafts a tree of tokens and verifies it:

    pages = kv_pages(num_pages, kv_heads, page_size, head_dim)       # once per layer
    mask = tree_mask(parents, device="cuda")                         # which drafted tokens each of them sees
    kv_write(pages, k, v, slots)                                     # the drafted tokens' keys and values
    x = tree_attention(q, pages, page_table, lengths, q_start, mask=mask)
    ...                                                              # rest of the network -> logits of every drafted token
    logprob, entropy, top_logprob, top_index = token_logprobs(logits, drafted, top=8)
    kv_write(pages, k[accepted], v[accepted], next_slots)            # the accepted path moves together; lengths shrink to it

Every call enqueues on torch's current stream of the tensors' device and returns; tensors made on another stream are the caller's to
order, as for any torch operation.  Results and scratch memory come from torch's allocator, so calls may run on several streams at once
and may be captured into graphs.  Inference only: a tensor that requires a gradient is refused while gradients are recorded.
There is no CPU path.  Importing this module loads torch: it has to happen before the first engine or `_native.load()` of the process,
because torch brings its own HIP runtime and device pointers are only valid inside one (a process that holds two is refused)."""
from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence, Tuple

import numpy as np
import torch

from . import _native

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_FORMATS = {torch.bfloat16: 0, torch.float8_e4m3fn: 1}
MAX_TOP = 64

_checked_lib = None


def _lib():
    """The native library, once it is known that it and torch talk to the same HIP runtime."""
    global _checked_lib
    if _checked_lib is None:
        lib = _native.load()
        with open("/proc/self/maps") as f:
            runtimes = {line.split()[-1] for line in f if "libamdhip64" in line}
        if len(runtimes) > 1:
            raise RuntimeError("two HIP runtimes in this process (" + ", ".join(sorted(runtimes)) + "): import torch, or pero_ocr_amd.decode_ops, "
                               "before the first engine is created")
        _checked_lib = lib
    return _checked_lib


def _fail(what: str):
    raise RuntimeError(what + ": " + (_native.load().pocr_last_error() or b"").decode("utf8", "replace"))


# current_stream(device).cuda_stream without building the stream object (2 us, a third of a small call)
_stream = torch._C._cuda_getCurrentRawStream
_Tensor = torch.Tensor


def _need(t, name: str, device: Optional[torch.device], dtypes, dims: int):
    """The checks that every tensor argument has to pass, one short expression where they do."""
    if type(t) is _Tensor and t.dtype in dtypes and t.dim() == dims and not t.requires_grad and (t.device == device if device is not None else t.is_cuda):
        return
    if not isinstance(t, _Tensor):
        raise TypeError(f"{name}: expected a torch tensor, got {type(t).__name__}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name}: {t.dtype}; expected one of {', '.join(str(d) for d in dtypes)}")
    if t.dim() != dims:
        raise ValueError(f"{name}: expected {dims} dimensions, got shape {tuple(t.shape)}")
    if device is None:
        if not t.is_cuda:
            raise RuntimeError(f"{name} is on {t.device}: pero_ocr_amd has no CPU path")
    elif t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name} requires a gradient: the decoding operators are for inference (use torch.no_grad())")


_IDS = (torch.int64, torch.int32)
_I32 = (torch.int32,)
_I64 = (torch.int64,)
_U8 = (torch.uint8,)


class KVPages:
    """One layer's cache: k, v [pages, kv_heads, page_size, head_dim], bfloat16 or float8_e4m3fn; in 8 bits k_exp, v_exp uint8
    [pages, kv_heads, page_size] hold the power of two of every row: it stands for code * 2 ** (exp - 127).  Slot s is row
    s % page_size of page s // page_size.  The tensors stay the caller's (contiguous, same device); kv_pages() makes them."""
    __slots__ = ("k", "v", "k_exp", "v_exp", "device", "index", "native")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_exp: Optional[torch.Tensor] = None, v_exp: Optional[torch.Tensor] = None):
        _need(k, "k", None, _FORMATS, 4)
        device, dtype, shape = k.device, k.dtype, k.shape
        _need(v, "v", device, (dtype,), 4)
        if v.shape != shape:
            raise ValueError(f"k and v differ in shape: {tuple(shape)}, {tuple(v.shape)}")
        whole = k.is_contiguous() and v.is_contiguous()
        if dtype is torch.float8_e4m3fn:
            _need(k_exp, "k_exp", device, _U8, 3)
            _need(v_exp, "v_exp", device, _U8, 3)
            rows = shape[:3]
            if k_exp.shape != rows or v_exp.shape != rows:
                raise ValueError(f"k_exp, v_exp: expected shape {tuple(rows)}, got {tuple(k_exp.shape)}, {tuple(v_exp.shape)}")
            whole = whole and k_exp.is_contiguous() and v_exp.is_contiguous()
            exps = k_exp.data_ptr(), v_exp.data_ptr()
        elif k_exp is not None or v_exp is not None:
            raise ValueError("a bfloat16 cache has no exponents")
        else:
            exps = None, None
        if not whole:
            raise ValueError("the cache's tensors must be contiguous")
        n, h, p, d = shape
        if d not in (32, 64, 128, 256):
            raise ValueError(f"head_dim {d}: 32, 64, 128 or 256")
        if p < 16 or p & (p - 1):
            raise ValueError(f"page_size {p}: a power of two from 16 on")
        if n < 1 or h < 1:
            raise ValueError(f"an empty cache: {tuple(shape)}")
        self.k, self.v, self.k_exp, self.v_exp, self.device, self.index = k, v, k_exp, v_exp, device, device.index
        self.native = _native.KvPages(k.data_ptr(), v.data_ptr(), exps[0], exps[1], n, h, p, d, _FORMATS[dtype])


def kv_pages(num_pages: int, kv_heads: int, page_size: int, head_dim: int, dtype: str = "fp8", device="cuda") -> KVPages:
    """An empty cache (all rows zero) of `num_pages` pages; dtype "fp8" or "bf16"."""
    if dtype not in ("fp8", "bf16"):
        raise ValueError(f"cache dtype {dtype!r}: 'fp8' or 'bf16'")
    shape = (int(num_pages), int(kv_heads), int(page_size), int(head_dim))
    if dtype == "bf16":
        return KVPages(*(torch.zeros(shape, dtype=torch.bfloat16, device=device) for _ in range(2)))
    k, v = (torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn) for _ in range(2))
    return KVPages(k, v, *(torch.full(shape[:3], 27, dtype=torch.uint8, device=device) for _ in range(2)))


def _check_slots(slots, pages: KVPages) -> int:
    _need(slots, "slots", pages.device, _IDS, 1)
    if not slots.is_contiguous():
        raise ValueError("slots must be contiguous")
    return slots.shape[0]


def kv_write(pages: KVPages, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Rounds k, v [tokens, kv_heads, head_dim] (float32, bfloat16 or float16; any token and head strides, such as slices of a fused
    projection) into the cache's format and stores them at slots [tokens].  A slot outside the cache (-1 for padding) is skipped; the
    slots of one call are distinct."""
    tokens = _check_slots(slots, pages)
    _need(k, "k", pages.device, _DTYPES, 3)
    _need(v, "v", pages.device, (k.dtype,), 3)
    n = pages.native
    shape = (tokens, n.kv_heads, n.head_dim)
    if k.shape != shape or v.shape != shape:
        raise ValueError(f"k, v: expected shape {shape}, got {tuple(k.shape)}, {tuple(v.shape)}")
    kt, kh, k1 = k.stride()
    vt, vh, v1 = v.stride()
    if k1 != 1 or v1 != 1:
        raise ValueError("the last axis of k and v must be contiguous")
    if _lib().pocr_kv_write(pages.index, _stream(pages.index), n, k.data_ptr(), v.data_ptr(), _DTYPES[k.dtype], kt, kh, vt, vh, slots.data_ptr(),
                            slots.dtype is torch.int64, tokens):
        _fail("pocr_kv_write")


def kv_read(pages: KVPages, slots: torch.Tensor, dtype: torch.dtype = torch.float32) -> Tuple[torch.Tensor, torch.Tensor]:
    """The rows at slots [tokens] as two tensors [tokens, kv_heads, head_dim] of `dtype`; a slot outside the cache reads as zeros."""
    tokens = _check_slots(slots, pages)
    if dtype not in _DTYPES:
        raise TypeError(f"dtype {dtype}: float32, bfloat16 or float16")
    n = pages.native
    k = torch.empty((tokens, n.kv_heads, n.head_dim), dtype=dtype, device=pages.device)
    v = torch.empty_like(k)
    if _lib().pocr_kv_read(pages.index, _stream(pages.index), n, slots.data_ptr(), slots.dtype is torch.int64, tokens, k.data_ptr(), v.data_ptr(), _DTYPES[dtype]):
        _fail("pocr_kv_read")
    return k, v


def tree_mask(parents: Sequence[int], device="cuda") -> torch.Tensor:
    """The mask of one tree of drafted tokens: parents[i] < i is the token that i continues, -1 for one that continues the cached
    text.  -> int64 [n, ceil(n / 64)]; bit j of row i (bit j % 64 of word j // 64): token i sees token j, its ancestors and itself."""
    n = len(parents)
    words = -(-n // 64)
    seen = np.zeros((n, words), dtype=np.uint64)
    for i, p in enumerate(parents):
        p = int(p)
        if not -1 <= p < i:
            raise ValueError(f"parents[{i}] = {p}: a token's parent comes before it, or is -1")
        if p >= 0:
            seen[i] = seen[p]
        seen[i, i // 64] |= np.uint64(1 << (i % 64))
    return torch.from_numpy(seen.view(np.int64)).to(device)


def tree_attention(q: torch.Tensor, pages: KVPages, page_table: torch.Tensor, lengths: torch.Tensor, q_start: torch.Tensor,
                   mask: Optional[torch.Tensor] = None, scale: Optional[float] = None, max_queries: int = 0, want_lse: bool = False,
                   out: Optional[torch.Tensor] = None):
    """Attention of the newest tokens of many sequences over their cached keys and values.

    q [tokens, heads, head_dim] (float32, bfloat16 or float16; any token and head strides): the new tokens of all sequences one after
    the other, sequence s owning rows q_start[s] .. q_start[s + 1] - 1.  page_table int32 [seqs, pages of a sequence], lengths int32 [seqs]:
    cached positions, the new tokens (already written by kv_write) being the last ones; q_start int32 [seqs + 1], from 0 on.
    A new token sees every older position and, among the new ones, those up to itself (mask None) or those its mask row names (int64
    [tokens, words], see tree_mask; bits count from the sequence's first new token).  heads is a multiple of the cache's key heads;
    query head h reads key head h // (heads // kv_heads).  A token that sees nothing gets zeros and lse -inf.  Positions whose page id
    lies outside the cache (-1) are absent.  scale: head_dim ** -0.5 unless given.  max_queries: the most new tokens of one sequence,
    if the caller knows it (it shapes the launch, never the answer).

    -> out [tokens, heads, head_dim] in q's type, or (out, lse float32 [tokens, heads]).  Rows behind q_start[-1] (a padded batch) are zeros
    (lse -inf) in a tensor made here and are left alone in an `out` of the caller's (contiguous)."""
    n, device = pages.native, pages.device
    _need(q, "q", device, _DTYPES, 3)
    _need(page_table, "page_table", device, _I32, 2)
    _need(lengths, "lengths", device, _I32, 1)
    _need(q_start, "q_start", device, _I32, 1)
    tokens, heads, dim = q.shape
    seqs, width = page_table.shape
    if dim != n.head_dim or heads < 1 or heads % n.kv_heads:
        raise ValueError(f"q {tuple(q.shape)} does not fit a cache of {n.kv_heads} key heads of {n.head_dim}")
    if lengths.shape[0] != seqs or q_start.shape[0] != seqs + 1:
        raise ValueError(f"page_table {tuple(page_table.shape)} and q_start {tuple(q_start.shape)} do not fit {seqs} sequences")
    qs, ps = q.stride(), page_table.stride()
    if qs[2] != 1 or (width > 1 and ps[1] != 1) or not lengths.is_contiguous() or not q_start.is_contiguous():
        raise ValueError("the last axis of q, page_table, lengths and q_start must be contiguous")
    if mask is not None:
        _need(mask, "mask", device, _I64, 2)
        if mask.shape[0] != tokens or (tokens and mask.shape[1] < 1) or (mask.shape[1] > 1 and mask.stride(1) != 1):
            raise ValueError(f"mask: expected [{tokens}, at least one word] with a contiguous last axis, got {tuple(mask.shape)}")
    fresh = out is None
    if fresh:
        out = torch.empty((tokens, heads, dim), dtype=q.dtype, device=device)
    else:
        _need(out, "out", device, (q.dtype,), 3)
        if out.shape != q.shape or not out.is_contiguous():
            raise ValueError(f"out: expected a contiguous tensor of shape {tuple(q.shape)}")
    lse = torch.empty((tokens, heads), dtype=torch.float32, device=device) if want_lse else None
    if tokens:
        lib = _lib()
        at = q.data_ptr()
        per16 = 16 // q.element_size()
        if at % 16 or qs[0] % per16 or qs[1] % per16:          # (the kernel loads 16 bytes at a time)
            q = q.clone(memory_format=torch.contiguous_format)
            qs, at = q.stride(), q.data_ptr()
        args = _native.TreeAttentionArgs(
            at, out.data_ptr(), lse.data_ptr() if want_lse else None, page_table.data_ptr(), lengths.data_ptr(), q_start.data_ptr(),
            mask.data_ptr() if mask is not None else None, None, 0, qs[0], qs[1], ps[0], mask.stride(0) if mask is not None else 0, tokens, max_queries,
            _DTYPES[q.dtype], seqs, heads, width, mask.shape[1] if mask is not None else 0, fresh, dim ** -0.5 if scale is None else scale)
        need = lib.pocr_tree_attention_workspace(n, args)
        if need:
            if need < 0:
                _fail("pocr_tree_attention")
            scratch = torch.empty((need,), dtype=torch.uint8, device=device)
            args.workspace, args.workspace_bytes = scratch.data_ptr(), need
        if lib.pocr_tree_attention(pages.index, _stream(pages.index), n, args):
            _fail("pocr_tree_attention")
    return (out, lse) if want_lse else out


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Scores of given tokens under logits [rows, classes] (float32, bfloat16 or float16, any row stride).

    tokens: int64 or int32, [rows] or [rows, given].  -> logprob float32 of tokens' shape, log softmax(row)[token] (0 for a negative token:
    padding; NaN for one beyond the classes); entropy float32 [rows] of softmax(row); top_logprob float32 and top_index int32 [rows, top], the
    `top` <= 64 likeliest classes, equally likely ones in the order of their index.  A logit of -inf has probability 0; a row of nothing else
    has log probabilities -inf and entropy 0; a row with NaN or +inf has NaN."""
    _need(logits, "logits", None, _DTYPES, 2)
    device = logits.device
    if not isinstance(tokens, _Tensor) or tokens.dim() not in (1, 2):
        raise ValueError("tokens: expected a tensor [rows] or [rows, given]")
    _need(tokens, "tokens", device, _IDS, tokens.dim())
    rows, classes = logits.shape
    shape = tokens.shape
    if shape[0] != rows or not tokens.is_contiguous():
        raise ValueError(f"tokens: expected a contiguous tensor with {rows} rows, got {tuple(shape)}")
    if classes < 1 or not 0 <= top <= MAX_TOP or top > classes:
        raise ValueError(f"top = {top}: 0 .. {MAX_TOP}, and at most the {classes} classes")
    stride, last = logits.stride()
    if classes > 1 and last != 1:
        raise ValueError("the last axis of logits must be contiguous")
    logprob = torch.empty(shape, dtype=torch.float32, device=device)
    entropy = logprob.new_empty((rows,))
    top_logprob = logprob.new_empty((rows, top))
    top_index = torch.empty((rows, top), dtype=torch.int32, device=device)
    if rows:
        lib = _lib()
        args = _native.TokenLogprobsArgs(
            logits.data_ptr(), tokens.data_ptr(), logprob.data_ptr(), entropy.data_ptr(), top_logprob.data_ptr(), top_index.data_ptr(), None, 0, stride, rows,
            _DTYPES[logits.dtype], classes, shape[1] if len(shape) == 2 else 1, top, tokens.dtype is torch.int64)
        need = lib.pocr_token_logprobs_workspace(args)
        if need:
            if need < 0:
                _fail("pocr_token_logprobs")
            scratch = torch.empty((need,), dtype=torch.uint8, device=device)
            args.workspace, args.workspace_bytes = scratch.data_ptr(), need
        if lib.pocr_token_logprobs(device.index, _stream(device.index), args):
            _fail("pocr_token_logprobs")
    return logprob, entropy, top_logprob, top_index
