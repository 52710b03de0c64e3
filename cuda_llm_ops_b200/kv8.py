"""The 8-bit KV cache: append, decode attention, a prompt's attention weights, eviction.

Serving a long context through ``gqa_decode`` reads two bytes per cached value and keeps every token.  The operators here
halve the bytes and bound the tokens:

* ``kv8_cache`` / ``KV8Cache``  codes (e4m3 or int8) with one fp32 scale per (batch, kv head, block of tokens)
* ``kv8_append``                bf16 K/V rows into the cache: whole prompts or one token per sequence
* ``kv8_decode``                one query token per sequence against the cache, optionally accumulating how much weight
                                every cached token received
* ``attention_weight_sums``     the same statistic for a prompt, from the forward's q, k and lse
* ``kv8_evict``                 keeps the tokens with the largest accumulated weight, moved to another cache

Sequence lengths are int32 tensors on the device and are never read by the host, so every call can be captured into a CUDA
graph and follows the lengths at replay.  None of the calls changes a length; ``kv8_evict`` returns the new ones.
(Upstream has no counterpart of these operators.)
"""
import contextlib
import ctypes
import functools
import math
import threading

import torch

from . import _lib
from .flash_gqa import HEAD_DIM, KV_BHSD, KV_BSHD, _counted_workspaces, _require_cuda_bf16

_FORMATS = {torch.float8_e4m3fn: _lib.FMT_E4M3, torch.int8: _lib.FMT_INT8}
BLOCK_TOKENS = (16, 32, 64, 128)
_MAX_POSITIONS = 1 << 30
_FP32, _INT32 = torch.float32, torch.int32

# A decoding step's calls take a few microseconds on the GPU: the device switch and the stream look-up of torch.cuda cost
# as much again per call, so the switch is skipped where the device is current and the stream comes from the raw getter.
_NO_SWITCH = contextlib.nullcontext()


def _on(device):
    return _NO_SWITCH if torch._C._cuda_getDevice() == device.index else torch.cuda.device(device)


def _stream_ptr(device):
    return torch._C._cuda_getCurrentRawStream(device.index)


class KV8Cache:
    """The tensors of an 8-bit KV cache.

    ``k``, ``v``: float8_e4m3fn or int8, [B,S,Hkv,D] (``KV_BSHD``) or [B,Hkv,S,D] (``KV_BHSD``), S = capacity in tokens;
    ``k_scale``, ``v_scale``: fp32 [B,Hkv,ceil(S / block_tokens)].  A value is ``code * scale`` of its block; scales are not
    negative, and 0 goes with codes that are 0.
    """

    __slots__ = ("k", "v", "k_scale", "v_scale", "kv_layout", "block_tokens", "batch", "capacity", "num_kv_heads",
                 "format")

    def __init__(self, k, v, k_scale, v_scale, kv_layout=KV_BHSD, block_tokens=64):
        dtype, shape, device = k.dtype, k.shape, k.device
        fmt = _FORMATS.get(dtype)
        if fmt is None or v.dtype is not dtype:
            raise ValueError("k and v must both be float8_e4m3fn or both int8")
        if block_tokens not in BLOCK_TOKENS:
            raise ValueError("block_tokens must be one of %s" % (BLOCK_TOKENS,))
        if len(shape) != 4 or v.shape != shape or shape[3] != HEAD_DIM:
            raise ValueError("expected k and v of identical 4-D shape with head_dim %d" % HEAD_DIM)
        if kv_layout == KV_BSHD:
            batch, capacity, heads, _ = shape
        elif kv_layout == KV_BHSD:
            batch, heads, capacity, _ = shape
        else:
            raise ValueError("unknown kv_layout")
        if not (batch and capacity and heads):
            raise ValueError("a cache holds at least one sequence, one token and one kv head")
        scales = (batch, heads, -(-capacity // block_tokens))
        if k_scale.dtype is not _FP32 or v_scale.dtype is not _FP32 or k_scale.shape != scales \
                or v_scale.shape != scales:
            raise ValueError("k_scale and v_scale must be fp32 [batch, num_kv_heads, ceil(capacity / block_tokens)]")
        if not (k.is_contiguous() and v.is_contiguous() and k_scale.is_contiguous() and v_scale.is_contiguous()):
            raise ValueError("the cache's tensors must be contiguous")
        if v.device != device or k_scale.device != device or v_scale.device != device:
            raise ValueError("the cache's tensors must be on one device")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.kv_layout, self.block_tokens = kv_layout, block_tokens
        self.batch, self.capacity, self.num_kv_heads, self.format = batch, capacity, heads, fmt


def kv8_cache(batch, capacity, num_kv_heads, dtype=torch.float8_e4m3fn, kv_layout=KV_BHSD, block_tokens=64,
              device="cuda"):
    """A zeroed cache for ``capacity`` tokens per sequence."""
    if kv_layout == KV_BSHD:
        shape = (batch, capacity, num_kv_heads, HEAD_DIM)
    else:
        shape = (batch, num_kv_heads, capacity, HEAD_DIM)
    if block_tokens not in BLOCK_TOKENS:
        raise ValueError("block_tokens must be one of %s" % (BLOCK_TOKENS,))
    k, v = (torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype) for _ in range(2))
    scales = (batch, num_kv_heads, -(-capacity // block_tokens))
    ks, vs = (torch.zeros(scales, dtype=torch.float32, device=device) for _ in range(2))
    return KV8Cache(k, v, ks, vs, kv_layout, block_tokens)


def _check_lens(name, t, batch, device):
    if not isinstance(t, torch.Tensor) or t.dtype is not _INT32 or t.shape != (batch,) or t.device != device \
            or not t.is_contiguous():
        raise ValueError("%s must be a contiguous int32 tensor [batch] on the cache's device" % name)


def _check_fp32(name, t, shape, device):
    if not isinstance(t, torch.Tensor) or t.dtype is not _FP32 or t.shape != shape or t.device != device or not t.is_contiguous():
        raise ValueError("%s must be a contiguous fp32 tensor of shape %s on the same device" % (name, list(shape)))


def _check_workspace(t, device):
    if not isinstance(t, torch.Tensor) or t.device != device or not t.is_contiguous():
        raise ValueError("workspace must be a contiguous tensor on the device of the call")


def _require_cuda(cache):
    if not cache.k.is_cuda:
        raise RuntimeError("the cache must be on a CUDA device: this library has no CPU path")


_Strides = ctypes.c_longlong * 3


@functools.lru_cache(maxsize=1024)
def _row_strides(s, kv_layout):
    """{batch, token, head} of a [B,T,H,D] or [B,H,T,D] tensor's strides; None if its rows are not contiguous and aligned."""
    if s[3] != 1 or (s[0] | s[1] | s[2]) % 8:
        return None
    return _Strides(s[0], s[1], s[2]) if kv_layout == KV_BSHD else _Strides(s[0], s[2], s[1])


def kv8_append(cache, k_new, v_new, seq_lens, new_lens=None):
    """Write K/V rows of up to T tokens per sequence behind the ``seq_lens`` tokens that the cache holds (in place).

    ``k_new``, ``v_new``: bf16, [B,T,Hkv,D] or [B,Hkv,T,D] as the cache's layout; slices of a larger tensor are fine as long
    as rows are contiguous and 16-byte aligned.  ``seq_lens`` int32 [B]: tokens held before the call; ``new_lens`` int32
    [B] (default: T for all): how many of the T rows are real.  Rows beyond the capacity are not stored.  A block that was
    partly filled keeps its scale unless the new rows need a larger one; then its old rows are re-rounded.
    """
    _require_cuda_bf16("k_new", k_new)
    _require_cuda_bf16("v_new", v_new)
    _require_cuda(cache)
    device, layout, shape = cache.k.device, cache.kv_layout, k_new.shape
    if len(shape) != 4 or v_new.shape != shape:
        raise ValueError("k_new and v_new must be of identical 4-D shape")
    if layout == KV_BSHD:
        B, T, H, D = shape
    else:
        B, H, T, D = shape
    if B != cache.batch or H != cache.num_kv_heads or D != HEAD_DIM:
        raise ValueError("k_new and v_new must match the cache's batch, kv heads and head_dim")
    if k_new.device != device or v_new.device != device:
        raise ValueError("k_new and v_new must be on the cache's device")
    k_at, k_strides = k_new.data_ptr(), _row_strides(k_new.stride(), layout)
    v_at, v_strides = v_new.data_ptr(), _row_strides(v_new.stride(), layout)
    if k_strides is None or v_strides is None or k_at % 16 or v_at % 16:
        raise ValueError("k_new and v_new must have contiguous, 16-byte aligned rows")
    _check_lens("seq_lens", seq_lens, B, device)
    if new_lens is not None:
        _check_lens("new_lens", new_lens, B, device)
    if T == 0:
        return
    with _on(device):
        rc = _lib.load().cllo_kv8_append_bf16(
            k_at, k_strides, v_at, v_strides, seq_lens.data_ptr(), None if new_lens is None else new_lens.data_ptr(),
            cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scale.data_ptr(), cache.v_scale.data_ptr(), B, T,
            cache.capacity, H, D, layout, cache.block_tokens, cache.format, _stream_ptr(device))
    _lib.check(rc, "cllo_kv8_append_bf16")


_workspaces = {}
_workspaces_lock = threading.Lock()
_counted_workspaces.append(_workspaces)


def _workspace(kind, device, nbytes):
    """(scratch, flag): scratch whose arrival counters are zero, and the flag that vouches for it.

    Eager calls of one kind share one tensor per (device, stream): launches on one stream do not overlap, and the kernel leaves
    the counters zero.  A call that is being captured gets a tensor of its own from the graph's pool, and the call clears the
    counters at every replay: two graphs may be replayed at the same time.
    """
    if torch._C._cuda_isCurrentStreamCapturing():
        return torch.empty(nbytes, dtype=torch.uint8, device=device), 0
    key = (kind, device.index, _stream_ptr(device))
    ws = _workspaces.get(key)
    if ws is None or ws.numel() < nbytes:
        with _workspaces_lock:
            ws = _workspaces.get(key)
            if ws is None or ws.numel() < nbytes:
                ws = _workspaces[key] = torch.zeros(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
    return ws, _lib.WS_COUNTERS_ZERO


# A decode with weights is two launches, the second of which reads what the first left in the scratch.  No other host thread's
# call on that scratch, with weights or without, may come between them: one thread at a time makes its launches.
_launch_locks = [threading.Lock() for _ in range(61)]


def _launch_lock(workspace):
    return _launch_locks[(workspace.data_ptr() >> 8) % len(_launch_locks)]


def kv8_decode(q, cache, seq_lens, scale=None, out=None, lse=None, weights=None, num_workers=0, workspace=None):
    """Attention of one query token per sequence over an 8-bit cache; returns out [B,Hq,D] bf16.

    ``q`` [B,Hq,D] bf16, ``seq_lens`` int32 [B] tokens per sequence (0 gives zeros), ``lse`` (fp32 [B,Hq], optional) is
    filled with the log-sum-exp of the scores.  ``weights`` (fp32 [B,Hkv,capacity], optional): the step's probabilities,
    summed over the query heads of each group, are added to it -- what ``kv8_evict`` goes by.

    Eager calls keep their scratch per (device, stream) for the life of the process; with ``weights`` it holds 4 bytes per query
    head and token of the capacity.  ``workspace`` (contiguous, on the cache's device, of
    ``cllo_kv8_decode_workspace_bytes`` bytes) takes its place; calls that may overlap on the GPU need one each.
    """
    _require_cuda_bf16("q", q)
    _require_cuda(cache)
    device = cache.k.device
    shape = q.shape
    if len(shape) != 3 or shape[2] != HEAD_DIM or shape[0] != cache.batch:
        raise ValueError("expected q [B,Hq,%d] with the cache's batch" % HEAD_DIM)
    if not q.is_contiguous() or q.device != device:
        raise ValueError("q must be contiguous and on the cache's device")
    B, Hq, D = shape
    H = cache.num_kv_heads
    if Hq == 0 or Hq % H != 0:
        raise ValueError("Query heads must be divisible by KV heads")
    _check_lens("seq_lens", seq_lens, B, device)
    if not 0 <= num_workers <= _MAX_POSITIONS:
        raise ValueError("num_workers must not be negative")
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    if out is None:
        out = torch.empty_like(q)
    elif out.dtype != torch.bfloat16 or out.shape != shape or not out.is_contiguous() or out.device != device:
        raise ValueError("Output tensor must be contiguous bf16 of q's shape")
    if lse is not None:
        _check_fp32("lse", lse, (B, Hq), device)
    if weights is not None:
        _check_fp32("weights", weights, (B, H, cache.capacity), device)
    lib = _lib.load()
    with _on(device):
        nbytes = _decode_workspace_bytes(device, B, cache.capacity, Hq, H, weights is not None, num_workers)
        if workspace is None:
            workspace, flag = _workspace("decode", device, nbytes)
        else:
            _check_workspace(workspace, device)
            nbytes, flag = workspace.numel() * workspace.element_size(), 0
        with _launch_lock(workspace):
            rc = lib.cllo_kv8_decode_bf16(
                q.data_ptr(), cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scale.data_ptr(), cache.v_scale.data_ptr(),
                seq_lens.data_ptr(), scale, out.data_ptr(), None if lse is None else lse.data_ptr(),
                None if weights is None else weights.data_ptr(), workspace.data_ptr(), nbytes, B, cache.capacity, Hq, H, D,
                cache.kv_layout | flag, cache.block_tokens, cache.format, num_workers, _stream_ptr(device))
    _lib.check(rc, "cllo_kv8_decode_bf16")
    return out


_ws_bytes_cache = {}


def _decode_workspace_bytes(device, B, capacity, Hq, Hkv, with_weights, num_workers):
    key = (device.index, B, capacity, Hq, Hkv, with_weights, num_workers)
    n = _ws_bytes_cache.get(key)
    if n is None:
        n = int(_lib.load().cllo_kv8_decode_workspace_bytes(B, capacity, Hq, Hkv, HEAD_DIM, int(with_weights),
                                                            num_workers))
        if len(_ws_bytes_cache) > 4096:
            _ws_bytes_cache.clear()
        _ws_bytes_cache[key] = n
    return n


@functools.lru_cache(maxsize=64)
def _sums_workspace_bytes(device_index):  # asked with that device current
    return int(_lib.load().cllo_attn_weight_sums_workspace_bytes())


def attention_weight_sums(q, k, lse, scale=None, causal=True, q_start=0, seq_lens=None, window=None, out=None,
                          accumulate=False, workspace=None):
    """How much weight a prompt's queries gave to every key: fp32 [B,Hkv,Skv].

    ``out[b,h,t] = sum over the group's heads g and the query rows i of exp(scale * q[b,g,i] . k[b,h,t] - lse[b,g,i])``
    with q [B,Hq,Sq,D], k [B,Hkv,Skv,D] bf16 and the forward's ``lse`` [B,Hq,Sq] fp32; ``causal`` keeps
    t <= q_start + i.  ``seq_lens`` (int32 [B], optional): real lengths of a padded batch -- keys behind them get 0 and,
    under a causal mask, query rows behind them do not count.  ``window``: only the last ``window`` query positions
    of each sequence count (default: all); without lengths or without a causal mask these are the last rows of ``q``.  Rows with
    ``lse`` = -inf add nothing.  ``accumulate=True`` adds to ``out``.  ``q`` and ``k`` are copied where they are not contiguous.
    """
    _require_cuda_bf16("q", q)
    _require_cuda_bf16("k", k)
    q_shape, k_shape = q.shape, k.shape
    if len(q_shape) != 4 or len(k_shape) != 4 or k_shape[0] != q_shape[0] or q_shape[3] != HEAD_DIM \
            or k_shape[3] != HEAD_DIM:
        raise ValueError("expected q [B,Hq,Sq,%d] and k [B,Hkv,Skv,%d]" % (HEAD_DIM, HEAD_DIM))
    B, Hq, Sq, D = q_shape
    _, H, Skv, _ = k_shape
    if not (B and Hq and Sq and H and Skv):
        raise ValueError("q and k must not be empty")
    if Hq % H != 0:
        raise ValueError("Query heads must be divisible by KV heads")
    device = q.device
    if k.device != device:
        raise ValueError("q and k must be on the same device")
    if not (q.is_contiguous() and k.is_contiguous()):
        q, k = q.contiguous(), k.contiguous()
    _check_fp32("lse", lse, (B, Hq, Sq), device)
    if seq_lens is not None:
        _check_lens("seq_lens", seq_lens, B, device)
    if window is not None and window < 1:
        raise ValueError("window must be positive")
    if not 0 <= q_start <= _MAX_POSITIONS // 2:
        raise ValueError("q_start must not be negative or beyond 2^29")
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs out")
        out = torch.empty((B, H, Skv), dtype=torch.float32, device=device)
    else:
        _check_fp32("out", out, (B, H, Skv), device)
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    lib = _lib.load()
    with _on(device):
        flags = _lib.SUMS_ACCUMULATE if accumulate else 0
        if workspace is None:
            nbytes = _sums_workspace_bytes(device.index)
            workspace, zero = _workspace("sums", device, nbytes)
            flags |= zero
        else:
            _check_workspace(workspace, device)
            nbytes = workspace.numel() * workspace.element_size()
        rc = lib.cllo_attn_weight_sums_bf16(
            q.data_ptr(), k.data_ptr(), lse.data_ptr(), None if seq_lens is None else seq_lens.data_ptr(), scale,
            1 if causal else 0, q_start, min(window or 0, _MAX_POSITIONS), flags, out.data_ptr(), workspace.data_ptr(),
            nbytes, B, Sq, Skv, Hq, H, D, _stream_ptr(device))
    _lib.check(rc, "cllo_attn_weight_sums_bf16")
    return out


def kv8_evict(cache, weights, seq_lens, budget, sink=0, recent=0, out=None, out_weights=None):
    """Shrink every sequence to at most ``budget`` tokens per kv head; returns (cache, weights, seq_lens, indices).

    The first ``sink`` and the last ``recent`` tokens stay, and of the others those with the largest ``weights``
    (fp32 [B,Hkv,capacity]; the earlier of equal ones first).  What stays keeps its order and moves to ``out`` (default: a
    new cache of ``budget`` tokens; it must not share memory with ``cache``), the kept weights to ``out_weights``
    (fp32 [B,Hkv,capacity of out]; default: new, zero behind the kept ones).  ``indices`` int32 [B,Hkv,budget] are the
    kept positions, -1 behind them; the returned lengths are ``min(seq_lens, budget)``.

    A sequence that was cut fills the default ``out``, and ``kv8_append`` stores nothing beyond a cache's capacity: where tokens
    are to follow, pass an ``out`` with room for them.  Of a given ``out`` and ``out_weights`` what lies behind the kept tokens is
    left as it was: zero ``out_weights`` before the call where ``kv8_decode`` is to add to it afterwards.
    """
    _require_cuda(cache)
    device = cache.k.device
    B, H = cache.batch, cache.num_kv_heads
    if not 1 <= budget <= _MAX_POSITIONS or sink < 0 or recent < 0 or sink + recent > budget:
        raise ValueError("budget must be positive (at most 2^30) and hold the sink and recent tokens")
    _check_fp32("weights", weights, (B, H, cache.capacity), device)
    _check_lens("seq_lens", seq_lens, B, device)
    if out is None:
        out = kv8_cache(B, min(budget, cache.capacity), H, cache.k.dtype, cache.kv_layout, cache.block_tokens, device)
    if out.batch != B or out.num_kv_heads != H or out.format != cache.format or out.kv_layout != cache.kv_layout \
            or out.block_tokens != cache.block_tokens or out.k.device != device:
        raise ValueError("out must match the cache in batch, kv heads, format, layout, block_tokens and device")
    if out.capacity < min(budget, cache.capacity):
        raise ValueError("out must have room for the budget")
    if out_weights is None:
        out_weights = torch.zeros((B, H, out.capacity), dtype=torch.float32, device=device)
    else:
        _check_fp32("out_weights", out_weights, (B, H, out.capacity), device)
    with _on(device):
        new_lens = torch.empty_like(seq_lens)
        indices = seq_lens.new_empty((B, H, budget))
        rc = _lib.load().cllo_kv8_evict(
            cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scale.data_ptr(), cache.v_scale.data_ptr(),
            weights.data_ptr(), seq_lens.data_ptr(), out.k.data_ptr(), out.v.data_ptr(), out.k_scale.data_ptr(),
            out.v_scale.data_ptr(), out_weights.data_ptr(), new_lens.data_ptr(), indices.data_ptr(), B, cache.capacity,
            out.capacity, H, HEAD_DIM, budget, sink, recent, cache.kv_layout, cache.block_tokens, cache.format,
            _stream_ptr(device))
    _lib.check(rc, "cllo_kv8_evict")
    return out, out_weights, new_lens, indices
