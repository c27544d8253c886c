"""Decoding operators on torch tensors in HBM: a paged cache of attention keys and values in 8 bits or bfloat16, attention of the newest
tokens over it (single tokens, chains, trees of drafted tokens), and the scores of given tokens.

They stand next to the cached attention of the sequence-to-sequence engine (csrc/decoder.hpp, which keeps float32 keys and values of
one launch) and the logit operators `_native.ctc_greedy` / `_native.sparsify`, for a decoding loop of the caller's own; kernels and C entries:
csrc/decode_ops.hip, include/pocr.h "decoding operators".  One step of a loop that drafts a tree of tokens and verifies it:

    pages = kv_pages(num_pages, kv_heads, page_size, head_dim)       # once per layer
    mask = tree_mask(parents, device="cuda")                         # which drafted tokens each of them sees (once per form of a tree)
    kv_write(pages, k, v, slots)                                     # the drafted tokens' keys and values
    x = tree_attention(q, pages, page_table, lengths, q_start, mask=mask)
    ...                                                              # rest of the network -> logits of every drafted token
    logprob, entropy, top_logprob, top_index = token_logprobs(logits, drafted, top=8)
    kv_write(pages, k[accepted], v[accepted], next_slots)            # the accepted path moves together; lengths shrink to it

Every call but tree_mask enqueues on torch's current stream of the tensors' device and returns; tensors made on another stream are the caller's to
order, as for any torch operation.  Results and scratch memory come from torch's allocator, so calls may run on several streams at once
and may be captured into graphs.  tree_mask builds a mask on the host and copies it, which waits: trees of a fixed form are made once, before the
loop.  Inference only: a tensor that requires a gradient is refused while gradients are recorded, one that carries a forward-mode
derivative always.
There is no CPU path.  Importing this module loads torch: it has to happen before the first engine or `_native.load()` of the process,
because torch brings its own HIP runtime and device pointers are only valid inside one (a process that holds two is refused)."""
from __future__ import annotations

import ctypes as C
from operator import attrgetter
from typing import Optional, Sequence, Tuple

import numpy as np
import torch
from torch.autograd import forward_ad as _forward

from . import _native

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_FORMATS = {torch.bfloat16: 0, torch.float8_e4m3fn: 1}
_BF16, _FP8, _BYTE, _INT, _LONG = torch.bfloat16, torch.float8_e4m3fn, torch.uint8, torch.int32, torch.int64
_IDS = (_LONG, _INT)
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
    """The checks that every tensor argument has to pass, with the reason where one does not.  (Called where a short expression of the
    caller's says that something is wrong: a call of these operators takes as long on the host as on the GPU.)"""
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


def _no_tangent(**tensors):
    """(called inside a level of forward-mode differentiation, _forward._current_level >= 0; such a tensor is an ordinary one by all other signs)"""
    for name, t in tensors.items():
        if isinstance(t, _Tensor) and _forward.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{name} carries a forward-mode derivative: the decoding operators are for inference")


class KVPages:
    """One layer's cache: k, v [pages, kv_heads, page_size, head_dim], bfloat16 or float8_e4m3fn; in 8 bits k_exp, v_exp uint8
    [pages, kv_heads, page_size] hold the power of two of every row: it stands for code * 2 ** (exp - 127).  Slot s is row
    s % page_size of page s // page_size.  The tensors stay the caller's (contiguous, same device); kv_pages() makes them.  They are read-only
    attributes and have to keep their memory: a call with a cache whose tensors were given other storage is refused."""
    __slots__ = ("_k", "_v", "_k_exp", "_v_exp", "_index", "_native", "_at")
    k, v, k_exp, v_exp = (property(attrgetter(name)) for name in __slots__[:4])
    index, native = property(attrgetter("_index")), property(attrgetter("_native"))

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_exp: Optional[torch.Tensor] = None, v_exp: Optional[torch.Tensor] = None):
        if _forward._current_level >= 0:
            _no_tangent(k=k, v=v)
        fp8 = k_exp is not None
        if not (type(k) is _Tensor and type(v) is _Tensor and k.is_cuda and k.dtype is (_FP8 if fp8 else _BF16) and v.dtype is k.dtype
                and k.dim() == 4 and k.shape == v.shape and v.get_device() == k.get_device() and k.is_contiguous() and v.is_contiguous()
                and not (k.requires_grad or v.requires_grad)
                and (type(k_exp) is _Tensor and type(v_exp) is _Tensor and k_exp.dtype is _BYTE and v_exp.dtype is _BYTE
                     and k_exp.shape == v_exp.shape == k.shape[:3] and k_exp.get_device() == k.get_device() == v_exp.get_device()
                     and k_exp.is_contiguous() and v_exp.is_contiguous() if fp8 else v_exp is None)):
            self._refuse(k, v, k_exp, v_exp)
        n, h, p, d = k.shape
        if d not in (32, 64, 128, 256):
            raise ValueError(f"head_dim {d}: 32, 64, 128 or 256")
        if p < 16 or p & (p - 1):
            raise ValueError(f"page_size {p}: a power of two from 16 on")
        if n < 1 or h < 1:
            raise ValueError(f"an empty cache: {tuple(k.shape)}")
        at = (k.data_ptr(), v.data_ptr(), k_exp.data_ptr() if fp8 else None, v_exp.data_ptr() if fp8 else None)
        self._k, self._v, self._k_exp, self._v_exp, self._index, self._at = k, v, k_exp, v_exp, k.get_device(), at
        self._native = _native.KvPages(*at, n, h, p, d, fp8)

    def plan(self) -> _native.KvPages:
        """The cache as the C entries take it; raises if a tensor is no longer where it was when this object was made, or has come to require a
        gradient."""
        k, v, k_exp, v_exp = self._at
        if self._k.data_ptr() != k or self._v.data_ptr() != v or k_exp is not None and (self._k_exp.data_ptr() != k_exp or self._v_exp.data_ptr() != v_exp):
            raise RuntimeError("the cache's tensors have other memory than when this KVPages was made: make a new one")
        if (self._k.requires_grad or self._v.requires_grad) and torch.is_grad_enabled():
            raise RuntimeError("the cache requires a gradient: the decoding operators are for inference (use torch.no_grad())")
        return self._native

    @property
    def device(self) -> torch.device:
        return self.k.device

    @staticmethod
    def _refuse(k, v, k_exp, v_exp):
        _need(k, "k", None, _FORMATS, 4)
        _need(v, "v", k.device, (k.dtype,), 4)
        if v.shape != k.shape:
            raise ValueError(f"k and v differ in shape: {tuple(k.shape)}, {tuple(v.shape)}")
        if k.dtype is _FP8:
            _need(k_exp, "k_exp", k.device, (_BYTE,), 3)
            _need(v_exp, "v_exp", k.device, (_BYTE,), 3)
            if k_exp.shape != k.shape[:3] or v_exp.shape != k.shape[:3]:
                raise ValueError(f"k_exp, v_exp: expected shape {tuple(k.shape[:3])}, got {tuple(k_exp.shape)}, {tuple(v_exp.shape)}")
        elif k_exp is not None or v_exp is not None:
            raise ValueError("a bfloat16 cache has no exponents")
        if not all(t.is_contiguous() for t in (k, v, k_exp, v_exp) if t is not None):
            raise ValueError("the cache's tensors must be contiguous")


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
    if not (type(slots) is _Tensor and slots.dtype in _IDS and slots.dim() == 1 and slots.get_device() == pages._index):
        _need(slots, "slots", pages.device, _IDS, 1)
    if not slots.is_contiguous():
        raise ValueError("slots must be contiguous")
    return slots.numel()


def kv_write(pages: KVPages, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Rounds k, v [tokens, kv_heads, head_dim] (float32, bfloat16 or float16; any token and head strides, such as slices of a fused
    projection) into the cache's format and stores them at slots [tokens].  A slot outside the cache (-1 for padding) is skipped; the
    slots of one call are distinct."""
    tokens = _check_slots(slots, pages)
    n, index = pages.plan(), pages._index
    if _forward._current_level >= 0:
        _no_tangent(k=k, v=v)
    if not (type(k) is _Tensor and type(v) is _Tensor and k.dtype in _DTYPES and v.dtype is k.dtype and k.dim() == 3 == v.dim()
            and k.get_device() == index == v.get_device() and not (k.requires_grad or v.requires_grad)):
        _need(k, "k", pages.device, _DTYPES, 3)
        _need(v, "v", pages.device, (k.dtype,), 3)
    shape = k.shape
    if shape != v.shape or shape[0] != tokens or shape[1] != n.kv_heads or shape[2] != n.head_dim:
        raise ValueError(f"k, v: expected shape {(tokens, n.kv_heads, n.head_dim)}, got {tuple(shape)}, {tuple(v.shape)}")
    kt, kh, k1 = k.stride()
    vt, vh, v1 = v.stride()
    if k1 != 1 or v1 != 1:
        raise ValueError("the last axis of k and v must be contiguous")
    rows = _native.KvRows(k.data_ptr(), v.data_ptr(), slots.data_ptr(), kt, kh, vt, vh, tokens, _DTYPES[k.dtype], slots.dtype is _LONG)
    if _lib().pocr_kv_write(index, _stream(index), n, rows):
        _fail("pocr_kv_write")


def kv_read(pages: KVPages, slots: torch.Tensor, dtype: torch.dtype = torch.float32) -> Tuple[torch.Tensor, torch.Tensor]:
    """The rows at slots [tokens] as two tensors [tokens, kv_heads, head_dim] of `dtype`; a slot outside the cache reads as zeros."""
    tokens = _check_slots(slots, pages)
    if dtype not in _DTYPES:
        raise TypeError(f"dtype {dtype}: float32, bfloat16 or float16")
    if _forward._current_level >= 0:
        _no_tangent(cache=pages.k, cached_values=pages.v)
    n, index = pages.plan(), pages._index
    k = pages.k.new_empty((tokens, n.kv_heads, n.head_dim), dtype=dtype)
    v = torch.empty_like(k)
    if _lib().pocr_kv_read(index, _stream(index), n, slots.data_ptr(), slots.dtype is _LONG, tokens, k.data_ptr(), v.data_ptr(), _DTYPES[dtype]):
        _fail("pocr_kv_read")
    return k, v


def tree_mask(parents: Sequence[int], device="cuda") -> torch.Tensor:
    """The mask of one tree of drafted tokens: parents[i] < i is the token that i continues, -1 for one that continues the cached
    text.  -> int64 [n, ceil(n / 64)]; bit j of row i (bit j % 64 of word j // 64): token i sees token j, its ancestors and itself.  Made on the
    host, a loop over the tokens and a copy that is waited for: not for a step that is timed or captured into a graph."""
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
    query head h reads key head h // (heads // kv_heads).  A token that sees nothing, or only scores of -inf, gets zeros and lse -inf.
    Positions whose page id lies outside the cache (-1) are absent; a length beyond the table counts as the table's positions.
    scale: head_dim ** -0.5 unless given.  max_queries: the most new tokens of one sequence, if the caller knows it (it shapes the launch;
    the answer differs at most by the order of its sums, and comes later if there are more).  The table's width shapes the launch too:
    pass page_table[:, :n] where the longest sequence is known to have n pages.

    -> out [tokens, heads, head_dim] in q's type, or (out, lse float32 [tokens, heads]).  Rows behind q_start[-1] (a padded batch) are zeros in a
    tensor made here and are left alone in an `out` of the caller's (contiguous); lse, always made here, has -inf there."""
    n, index = pages.plan(), pages._index
    if _forward._current_level >= 0:
        _no_tangent(q=q, out=out, cache=pages.k, cached_values=pages.v)
    if not (type(q) is _Tensor and type(page_table) is _Tensor and type(lengths) is _Tensor and type(q_start) is _Tensor and q.dtype in _DTYPES
            and page_table.dtype is _INT and lengths.dtype is _INT and q_start.dtype is _INT and q.dim() == 3 and page_table.dim() == 2
            and lengths.dim() == 1 and q_start.dim() == 1 and not q.requires_grad
            and q.get_device() == page_table.get_device() == lengths.get_device() == q_start.get_device() == index):
        device = pages.device
        _need(q, "q", device, _DTYPES, 3)
        _need(page_table, "page_table", device, (_INT,), 2)
        _need(lengths, "lengths", device, (_INT,), 1)
        _need(q_start, "q_start", device, (_INT,), 1)
    tokens, heads, dim = q.shape
    seqs, width = page_table.shape
    if dim != n.head_dim or heads < 1 or heads % n.kv_heads:
        raise ValueError(f"q {tuple(q.shape)} does not fit a cache of {n.kv_heads} key heads of {n.head_dim}")
    if lengths.numel() != seqs or q_start.numel() != seqs + 1:
        raise ValueError(f"page_table {tuple(page_table.shape)} and q_start {tuple(q_start.shape)} do not fit {seqs} sequences")
    qs, ps = q.stride(), page_table.stride()
    if qs[2] != 1 or (width > 1 and ps[1] != 1) or not lengths.is_contiguous() or not q_start.is_contiguous():
        raise ValueError("the last axis of q, page_table, lengths and q_start must be contiguous")
    if mask is not None:
        _need(mask, "mask", pages.device, (_LONG,), 2)
        if mask.shape[0] != tokens or (tokens and mask.shape[1] < 1) or (mask.shape[1] > 1 and mask.stride(1) != 1):
            raise ValueError(f"mask: expected [{tokens}, at least one word] with a contiguous last axis, got {tuple(mask.shape)}")
    fresh = out is None
    if fresh:
        out = q.new_empty((tokens, heads, dim))
    else:
        _need(out, "out", pages.device, (q.dtype,), 3)
        if out.shape != q.shape or not out.is_contiguous():
            raise ValueError(f"out: expected a contiguous tensor of shape {tuple(q.shape)}")
    lse = q.new_empty((tokens, heads), dtype=torch.float32) if want_lse else None
    if tokens:
        lib = _lib()
        at = q.data_ptr()
        per16 = 16 // q.element_size()
        if at % 16 or qs[0] % per16 or qs[1] % per16:          # (the kernel loads 16 bytes at a time)
            q = q.clone(memory_format=torch.contiguous_format)
            qs, at = q.stride(), q.data_ptr()
        args = _native.TreeAttentionArgs(
            at, out.data_ptr(), lse.data_ptr() if want_lse else None, page_table.data_ptr(), lengths.data_ptr(), q_start.data_ptr(),
            mask.data_ptr() if mask is not None else None, None, 0, qs[0], qs[1], ps[0], mask.stride(0) if mask is not None else 0, tokens, int(max_queries),
            _DTYPES[q.dtype], seqs, heads, width, mask.shape[1] if mask is not None else 0, 1 if fresh else 2 if want_lse else 0, dim ** -0.5 if scale is None else float(scale))
        need = lib.pocr_tree_attention_workspace(n, args)
        if need:
            if need < 0:
                _fail("pocr_tree_attention")
            scratch = q.new_empty((need,), dtype=_BYTE)
            args.workspace, args.workspace_bytes = scratch.data_ptr(), need
        if lib.pocr_tree_attention(index, _stream(index), n, args):
            _fail("pocr_tree_attention")
    return (out, lse) if want_lse else out


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Scores of given tokens under logits [rows, classes] (float32, bfloat16 or float16, any row stride).

    tokens: int64 or int32, [rows] or [rows, given].  -> logprob float32 of tokens' shape, log softmax(row)[token] (0 for a negative token:
    padding; NaN for one beyond the classes); entropy float32 [rows] of softmax(row); top_logprob float32 and top_index int32 [rows, top], the
    `top` <= 64 likeliest classes, equally likely ones in the order of their index.  A logit of -inf has probability 0; a row of nothing else
    has log probabilities -inf and entropy 0; a row with NaN or +inf has NaN."""
    if _forward._current_level >= 0:
        _no_tangent(logits=logits)
    if not (type(logits) is _Tensor and type(tokens) is _Tensor and logits.is_cuda and logits.dtype in _DTYPES and logits.dim() == 2 and tokens.dtype in _IDS
            and 1 <= tokens.dim() <= 2 and tokens.get_device() == logits.get_device() and not logits.requires_grad):
        _need(logits, "logits", None, _DTYPES, 2)
        _need(tokens, "tokens", logits.device, _IDS, 2 if isinstance(tokens, _Tensor) and tokens.dim() == 2 else 1)
    rows, classes = logits.shape
    shape = tokens.shape
    if shape[0] != rows or not tokens.is_contiguous():
        raise ValueError(f"tokens: expected a contiguous tensor with {rows} rows, got {tuple(shape)}")
    top = int(top)
    if classes < 1 or not 0 <= top <= MAX_TOP or top > classes:
        raise ValueError(f"top = {top}: 0 .. {MAX_TOP}, and at most the {classes} classes")
    stride, last = logits.stride()
    if classes > 1 and last != 1:
        raise ValueError("the last axis of logits must be contiguous")
    logprob = logits.new_empty(shape, dtype=torch.float32)
    entropy = logprob.new_empty((rows,))
    top_logprob = logprob.new_empty((rows, top))
    top_index = logprob.new_empty((rows, top), dtype=_INT)
    if rows:
        lib = _lib()
        args = _native.TokenLogprobsArgs(
            logits.data_ptr(), tokens.data_ptr(), logprob.data_ptr(), entropy.data_ptr(), top_logprob.data_ptr(), top_index.data_ptr(), None, 0, stride, rows,
            _DTYPES[logits.dtype], classes, shape[1] if len(shape) == 2 else 1, top, tokens.dtype is _LONG)
        need = lib.pocr_token_logprobs_workspace(args)
        if need:
            if need < 0:
                _fail("pocr_token_logprobs")
            scratch = logits.new_empty((need,), dtype=_BYTE)
            args.workspace, args.workspace_bytes = scratch.data_ptr(), need
        index = logits.get_device()
        if lib.pocr_token_logprobs(index, _stream(index), args):
            _fail("pocr_token_logprobs")
    return logprob, entropy, top_logprob, top_index
