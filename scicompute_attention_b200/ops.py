"""Python harness over the C ABI: the same operators the C++ host layer exposes
(sca::decode_attention, sca::paged_attention, sca::flash_attention, KVCache::Append/Reset/Gather),
taking torch CUDA tensors only as device memory + stream providers.

Argument meaning follows the reference's public API (include/scicompute_attention/*.hpp):
q is [B, H_q, S_q, D] (layout "bhsd") or [B, S_q, H_q, D] ("bshd"); k/v likewise with H_kv;
outputs are always freshly allocated contiguous BHSD tensors, allocated on `stream` where one is given.

A call in its plain form (tensors, the current stream) goes through one C function of _native (csrc/torch/native_ops.cpp),
which answers None where it does not take the call; the code here is the general form, and the one that refuses. A launch that
failed raises its error on either way.
"""
from __future__ import annotations

import ctypes as C
import functools
import math
import struct
import threading
import warnings
from typing import NamedTuple

import torch

from . import _lib
from ._lib import (DTYPE_BF16, DTYPE_F16, DTYPE_F32, DecodeFwdParams, DecodeStrides, FlashFwdParams,
                   KvCacheShape, check, lib)

MAX_SPLITS = 64          # upper bound of the automatic split count on B200

_DTYPE_IDS = {torch.float32: DTYPE_F32, torch.float16: DTYPE_F16, torch.bfloat16: DTYPE_BF16}
MAX_SCRATCH_BUFFERS = 32  # scratch buffers a thread keeps


_native_module = None


def torch_build() -> str:
    """The torch a native module fits: it reads tensors through this build's headers."""
    return f"{torch.__version__} {torch.version.git_version}"


class _GeneralFormOnly:
    def __getattr__(self, name):
        return lambda *args: None  # takes no call


def _native():
    """The native form of the operators. Where it has not been built, or for another torch, the general form serves every call
    (the kernels are the same ones) and a warning says so once."""
    global _native_module
    if _native_module is None:
        try:
            from . import _native as module
            why = None if module.built_with == torch_build() else f"was built for torch {module.built_with}, this is {torch_build()}"
        except ImportError as e:
            why = f"does not load ({e})"
        if why is None:
            module.init(_scratch, acquire_scratch_fp32, check)
        else:
            warnings.warn(f"scicompute_attention_b200._native {why}: calls take 5 to 10 us longer on the host. Build it with "
                          "`python -m scicompute_attention_b200.build`", RuntimeWarning, stacklevel=3)
            module = _GeneralFormOnly()
        _native_module = module
    return _native_module


class _Scratch(threading.local):
    def __init__(self):
        self.pool: dict[tuple[int, int, int], torch.Tensor] = {}


_scratch = _Scratch()
_sm_count: dict[int, int] = {}


def dtype_id(dtype: torch.dtype) -> int:
    try:
        return _DTYPE_IDS[dtype]
    except KeyError:
        raise _lib.ScaError(4, f"dtype={dtype} (supported: float32, float16, bfloat16)")


def _stream_ptr(stream=None) -> int:
    if stream is not None:
        return stream.cuda_stream
    # the handle of torch.cuda.current_stream() without the Stream object around it
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())


def _require_cuda(*tensors: torch.Tensor) -> None:
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise _lib.ScaError(5, "device=cpu (attention kernels run on CUDA devices only; there is no CPU path)")


def _require_packed(what: str, *tensors: torch.Tensor) -> None:
    """The kernels address rows through the strides of a contiguous tensor."""
    for t in tensors:
        if not t.is_contiguous():
            raise _lib.ScaError(4, f"non-contiguous {what} rejected; pass a contiguous tensor")


def _require_ints(what: str, t: torch.Tensor, count: int) -> None:
    """A device list of at least `count` int32 entries."""
    _require_cuda(t)
    if t.dtype != torch.int32 or not t.is_contiguous() or t.numel() < count:
        raise _lib.ScaError(4, f"{what} must be a contiguous int32 tensor of at least {count} entries; got {t.dtype}{list(t.shape)}")


def _require_table(page_table: torch.Tensor, rows: int) -> None:
    if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.shape[0] < rows or not page_table.is_contiguous():
        raise _lib.ScaError(4, "page_table must be int32 [num_seqs, max_blocks_per_seq], contiguous")


def _require_like(q, k, v) -> None:
    if q.dtype != k.dtype or q.dtype != v.dtype:
        raise _lib.ScaError(4, "q/k/v shape or dtype mismatch")


def _same_kind(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether rows of `a` may be stored as rows of `b`: the same type, or raw integers of its width on one side."""
    return a.dtype == b.dtype or (a.element_size() == b.element_size() and not (a.is_floating_point() and b.is_floating_point()))


def _require_pools(layer_k, layer_v) -> None:
    _require_packed("pool", layer_k, layer_v)
    if tuple(layer_k.shape[1:]) != tuple(layer_v.shape[1:]) or layer_v.shape[0] < layer_k.shape[0] or not _same_kind(layer_v, layer_k):
        raise _lib.ScaError(4, "pool geometry mismatch")


def _require_rows(pool, rows: int, *tensors: torch.Tensor) -> None:
    """New K / V rows: at least `rows` of them, each [H_kv, D] of the pool in any shape, of the pool's type."""
    width = pool.shape[2] * pool.shape[3]
    for t in tensors:
        if not t.is_contiguous() or t.dim() < 1 or t.shape[0] < rows or t.numel() != t.shape[0] * width or not _same_kind(t, pool):
            raise _lib.ScaError(4, f"new K / V must be contiguous [{rows}, {pool.shape[2]}, {pool.shape[3]}] of the pool's type {pool.dtype}; "
                                   f"got {t.dtype}{list(t.shape)}")


def sm_count(device: torch.device) -> int:
    idx = device.index if device.index is not None else torch.cuda.current_device()
    if idx not in _sm_count:
        _sm_count[idx] = torch.cuda.get_device_properties(idx).multi_processor_count
    return _sm_count[idx]


def _on(stream):
    """Makes `stream` the current one: what is allocated there is reused in that stream's order."""
    return torch.cuda.stream(stream if isinstance(stream, torch.cuda.Stream) else torch.cuda.ExternalStream(stream.cuda_stream))


def _empty(shape, dtype, device, stream=None) -> torch.Tensor:
    """Device memory for a launch on `stream` (None: the current one)."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    with _on(stream):
        t = torch.empty(shape, dtype=dtype, device=device)
    t.record_stream(torch.cuda.current_stream(device))  # the caller goes on with the result there
    return t


def acquire_scratch_fp32(elements: int, device: torch.device, kind: int = 1, *, stream=None, handle: int | None = None) -> torch.Tensor:
    """Grow-only fp32 scratch of this thread per (device, kind, stream), so that calls that may overlap on the GPU never
    share it; same growth rule as the reference's pool (src/runtime/scratch_pool.cpp:38-60): 1.25 x request + 1024
    elements. A call that is being captured gets memory of the graph's own pool: no graph points into this one.
    `handle` is the launch's stream handle where the caller has it already."""
    if stream is None:
        capturing = torch.cuda.is_current_stream_capturing()
    else:
        with _on(stream):
            capturing = torch.cuda.is_current_stream_capturing()
    if capturing:
        return _empty(elements, torch.float32, device, stream)
    idx = device.index
    key = (idx if idx is not None else torch.cuda.current_device(), kind, _stream_ptr(stream) if handle is None else handle)
    pool = _scratch.pool
    cur = pool.get(key)
    if cur is None or cur.numel() < elements:
        pool.pop(key, None)
        if len(pool) >= MAX_SCRATCH_BUFFERS:
            del pool[next(iter(pool))]  # the oldest; the allocator reuses it in the order of its stream
        cur = pool[key] = _empty(int(elements * 1.25) + 1024, torch.float32, device, stream)
    return cur


DECODE_STEP_TOKENS = 64  # tokens one CTA of the decode kernel consumes per step (4 warps x 16)
FP8_BORDER_STEPS = 2     # what the schedule over an 8-bit cache counts for a border between two sequences
# Upper bound of its slot count. A sequence that has the machine to itself is on 511 CTAs at most, where up to 588 would have a share (D <= 64, one
# column): more parts cost more than they save. With 593 slots for 512, 16 / 1 heads, D=64: 100 thousand tokens 25.0 us for 21.8, 300 thousand 32.0
# for 28.2, 700 thousand 46.4 for 42.5, 1.5 million 67.9 for 67.3.
FP8_MAX_SPLITS = 512


def slots_for_schedule(column_steps: int, longest_steps: int, columns: int, sms: int, ctas_per_sm: int = 2, most: int = MAX_SPLITS,
                       even: bool = False) -> int:
    """Partial slots per row for the decode kernel's schedule: one wave of resident CTAs (2 per SM unless said), the same number
    for every (kv head, head chunk) column; the CTAs of a column split its list of 64-token steps (sequence after
    sequence) into equal contiguous shares, and a sequence cut by share boundaries yields one partial per piece.
    Needed: the pieces of the longest sequence, plus one for a share that starts in its middle. (The reference's rule,
    one CTA per fixed split, is ceil(seq_kv / 512) capped at 16: src/backends/decode/decode_config.hpp:24-31.)"""
    if column_steps <= 0 or longest_steps <= 1:
        return 1
    resident = ctas_per_sm * (sms if sms > 0 else 148)
    sharers = max(1, resident // max(1, columns))
    per_cta = max(1, column_steps // sharers if even else -(-column_steps // sharers))  # `even`: shares of a step more or less
    return max(2, min(-(-longest_steps // per_cta) + 1, most))


def splits_for(seq_kv: int, batch: int, num_kv_heads: int, group: int, sms: int) -> int:
    """Automatic slot count for equally long sequences."""
    if seq_kv <= 0:
        return 1
    steps = -(-seq_kv // DECODE_STEP_TOKENS)
    return slots_for_schedule(max(1, batch) * steps, steps, num_kv_heads * ((group + 15) // 16), sms)


def paged_splits_for(typical_len: int, num_seqs: int, num_kv_heads: int, group: int, sms: int, longest_len: int = 0,
                     step_tokens: int = DECODE_STEP_TOKENS, ctas_per_sm: int = 2, most: int = MAX_SPLITS, border: int = 0) -> int:
    """Slot count for a ragged batch of mean length `typical_len`; the longest sequence is taken as twice the mean
    unless `longest_len` says otherwise."""
    if typical_len <= 0:
        return 1
    steps = -(-typical_len // step_tokens)
    longest = -(-longest_len // step_tokens) if longest_len > 0 else 2 * steps
    if longest > 1:  # what a sequence's border counts for
        steps, longest = steps + border, longest + border
    return slots_for_schedule(max(1, num_seqs) * steps, longest, num_kv_heads * ((group + 15) // 16), sms, ctas_per_sm, most, border > 0)


def _strides(layout: str, seq: int, heads: int, d: int) -> tuple[int, int, int]:
    """(s_b, s_h, s_s) in elements (reference: detail/layout_traits.hpp:32-45)."""
    if layout == "bhsd":
        return heads * seq * d, seq * d, d
    if layout == "bshd":
        return seq * heads * d, d, heads * d
    raise _lib.ScaError(4, f"layout={layout} (supported: bhsd, bshd)")


def _dims(t: torch.Tensor, layout: str):
    if t.dim() != 4:
        raise _lib.ScaError(4, f"tensor ndims={t.dim()} (expected 4)")
    if not t.is_contiguous():
        raise _lib.ScaError(4, "non-contiguous input rejected; pass a contiguous tensor")
    if layout == "bhsd":
        b, h, s, d = t.shape
    else:
        b, s, h, d = t.shape
    return b, h, s, d


def effective_scale(scale, head_dim: int) -> float:
    """cfg.scale > 0 wins, otherwise float(1 / sqrt(double(D))) (reference: api_validate.cpp:31-35)."""
    if scale is not None and scale > 0:
        return float(scale)
    return _default_scale(head_dim)


@functools.lru_cache(maxsize=64)
def _default_scale(head_dim: int) -> float:
    return struct.unpack("f", struct.pack("f", 1.0 / math.sqrt(float(head_dim))))[0]  # rounded to fp32


# ------------------------------------------------------------------------------------------------
# decode / paged
# ------------------------------------------------------------------------------------------------
def decode_attention(q, k, v, *, scale=None, num_splits: int = 0, layout: str = "bhsd",
                     seq_lens=None, stream=None, return_stats: bool = False):
    """Split-K decode over a contiguous KV cache; S_q must be 1 (sca::decode_attention)."""
    if stream is None and num_splits <= 0 and not return_stats and q.is_cuda:
        out = _native().decode(q, k, v, scale, layout, seq_lens)
        if out is not None:
            return out
    _require_cuda(q, k, v)
    b, hq, sq, d = _dims(q, layout)
    bk, hkv, skv, dk = _dims(k, layout)
    if sq != 1:
        raise _lib.ScaError(5, f"decode backend requires seq_q=1; seq_q={sq} belongs to the flash backend")
    if (bk, dk) != (b, d) or tuple(v.shape) != tuple(k.shape) or q.dtype != k.dtype or q.dtype != v.dtype:
        raise _lib.ScaError(4, "q/k/v shape or dtype mismatch")
    _require_packed("v", v)
    if hq % hkv != 0:
        raise _lib.ScaError(4, f"num_heads={hq} % num_kv_heads={hkv} != 0")
    if seq_lens is not None:
        _require_ints("seq_lens", seq_lens, b)
    device, handle = q.device, _stream_ptr(stream)
    splits = min(num_splits, MAX_SPLITS) if num_splits > 0 else splits_for(skv, b, hkv, hq // hkv, sm_count(device))
    base = b * hq * splits
    ws = acquire_scratch_fp32(base * (2 + d), device, stream=stream, handle=handle)
    out = _empty((b, hq, 1, d), q.dtype, device, stream)

    p = DecodeFwdParams()
    p.q, p.k, p.v, p.out = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
    scratch = ws.data_ptr()
    p.partial_m, p.partial_l, p.partial_o = scratch, scratch + 4 * base, scratch + 8 * base
    p.batch, p.num_heads, p.num_kv_heads, p.seq_kv, p.head_dim, p.num_splits = b, hq, hkv, skv, d, splits
    p.q_stride = DecodeStrides(*_strides(layout, 1, hq, d))
    p.k_stride = DecodeStrides(*_strides(layout, skv, hkv, d))
    p.v_stride = p.k_stride
    p.o_stride = DecodeStrides(hq * d, d, d)
    p.scale = effective_scale(scale, d)
    p.dtype = dtype_id(q.dtype)
    p.page_table = None
    p.seq_lens = seq_lens.data_ptr() if seq_lens is not None else None
    return _launch_decode(p, num_splits, handle, out, return_stats)


def _launch_decode(p, num_splits, handle, out, return_stats):
    """An explicit split count asks for that many partials in the scratch; otherwise the size of the call decides."""
    cluster = C.c_int32(0) if return_stats else None
    if num_splits > 0:
        launch = lib().sca_launch_decode_splitk_paged if p.page_table else lib().sca_launch_decode_splitk
        check(launch(C.byref(p), handle))
    else:
        check(lib().sca_launch_decode_auto(C.byref(p), cluster, handle))
    if not return_stats:
        return out
    # num_splits: pieces a sequence is cut into at most; cluster: CTAs per cluster of the one-launch kernel, 0 = two kernels
    return out, {"num_splits": cluster.value or p.num_splits, "cluster": cluster.value,
                 "workspace_bytes": p.batch * p.num_heads * p.num_splits * (2 + p.head_dim) * 4}


def paged_attention(q, k_pool, v_pool, page_table, seq_lens, *, block_size: int, scale=None,
                    num_splits: int = 0, typical_len: int = 0, longest_len: int = 0, stream=None,
                    return_stats: bool = False, seq_order=None):
    """Decode over page-table-indirected K/V (sca::paged_attention).

    q [num_seqs, H_q, 1, D]; pools [num_blocks, block_size, H_kv, D]; page_table int32
    [num_seqs, max_blocks_per_seq] on the device (-1 = unmapped); seq_lens int32 [num_seqs] on the
    device or None (every sequence then scans max_blocks_per_seq * block_size positions).
    `typical_len` / `longest_len` are optional host-side hints (the mean and the maximum sequence length, which a
    cache object tracks anyway) used only to size the partial scratch: enough slots for an even schedule. seq_order
    is accepted for compatibility and ignored: the kernel balances the work itself."""
    if stream is None and num_splits <= 0 and not return_stats and seq_order is None and q.is_cuda:
        out = _native().paged(q, k_pool, v_pool, page_table, seq_lens, block_size, scale, typical_len, longest_len)
        if out is not None:
            return out
    _require_cuda(q, k_pool, v_pool, page_table, seq_lens)
    if q.dim() != 4:
        raise _lib.ScaError(4, f"paged_attention expects q=[num_seqs, H_q, seq_q, D]; got ndims={q.dim()}")
    s, hq, sq, d = q.shape
    if sq != 1:
        raise _lib.ScaError(5, f"paged attention implements the decode form only (seq_q=1); got seq_q={sq}")
    nblk, bs, hkv, dk = k_pool.shape
    if bs != block_size or dk != d or tuple(v_pool.shape) != tuple(k_pool.shape):
        raise _lib.ScaError(4, "pool geometry mismatch")
    _require_like(q, k_pool, v_pool)
    _require_packed("q or pool", q, k_pool, v_pool)
    _require_table(page_table, s)
    if seq_lens is not None:
        _require_ints("seq_lens", seq_lens, s)
    max_blocks = page_table.shape[1]
    upper = nblk * bs
    device, handle = q.device, _stream_ptr(stream)
    if num_splits > 0:
        splits = min(num_splits, MAX_SPLITS)
    else:
        splits = paged_splits_for(typical_len if typical_len > 0 else min(upper, max_blocks * bs), s, hkv,
                                  hq // hkv, sm_count(device), longest_len)
    base = s * hq * splits
    ws = acquire_scratch_fp32(base * (2 + d), device, stream=stream, handle=handle)
    out = _empty((s, hq, 1, d), q.dtype, device, stream)

    p = DecodeFwdParams()
    p.q, p.k, p.v, p.out = q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), out.data_ptr()
    scratch = ws.data_ptr()
    p.partial_m, p.partial_l, p.partial_o = scratch, scratch + 4 * base, scratch + 8 * base
    p.batch, p.num_heads, p.num_kv_heads, p.seq_kv, p.head_dim, p.num_splits = s, hq, hkv, upper, d, splits
    p.q_stride = DecodeStrides(hq * d, d, d)
    p.o_stride = DecodeStrides(hq * d, d, d)
    p.k_stride = DecodeStrides(0, d, hkv * d)   # row = one token of the pool (reference: paged_backend.cpp:131-134)
    p.v_stride = p.k_stride
    p.scale = effective_scale(scale, d)
    p.dtype = dtype_id(q.dtype)
    p.seq_lens = seq_lens.data_ptr() if seq_lens is not None else None
    if seq_order is not None and (seq_order.dtype != torch.int32 or seq_order.numel() != s or not seq_order.is_cuda):
        raise _lib.ScaError(4, "seq_order must be a device int32 permutation of the sequences")
    p.page_table = page_table.data_ptr()
    if not p.page_table:
        raise _lib.ScaError(4, "paged attention: null page table")
    p.block_size, p.max_blocks_per_seq, p.num_kv_blocks = bs, max_blocks, nblk
    return _launch_decode(p, num_splits, handle, out, return_stats)


def _shard_dims(q, k, v):
    b, hq, sq, d = _dims(q, "bhsd")
    bk, hkv, skv, dk = _dims(k, "bhsd")
    if sq != 1 or (bk, dk) != (b, d) or tuple(v.shape) != tuple(k.shape):
        raise _lib.ScaError(4, "q/k/v shape or dtype mismatch")
    _require_like(q, k, v)
    _require_packed("v", v)
    return b, hq, hkv, skv, d


def decode_triples(q, k, v, *, scale=None, num_splits: int = 0, stream=None):
    """This rank's share of a sequence-split decode: merged but unnormalised {m, l, O[D]} per
    (batch, head), fp32 [B*H_q, 2 + D]."""
    _require_cuda(q, k, v)
    b, hq, hkv, skv, d = _shard_dims(q, k, v)
    splits = min(num_splits, MAX_SPLITS) if num_splits > 0 else splits_for(skv, b, hkv, hq // hkv, sm_count(q.device))
    base = b * hq * splits
    ws = acquire_scratch_fp32(base * (2 + d), q.device, stream=stream)
    triples = _empty((b * hq, 2 + d), torch.float32, q.device, stream)
    p = DecodeFwdParams()
    p.q, p.k, p.v, p.out = q.data_ptr(), k.data_ptr(), v.data_ptr(), None
    scratch = ws.data_ptr()
    p.partial_m, p.partial_l, p.partial_o = scratch, scratch + 4 * base, scratch + 8 * base
    p.batch, p.num_heads, p.num_kv_heads, p.seq_kv, p.head_dim, p.num_splits = b, hq, hkv, skv, d, splits
    p.q_stride = DecodeStrides(*_strides("bhsd", 1, hq, d))
    p.k_stride = DecodeStrides(*_strides("bhsd", skv, hkv, d))
    p.v_stride = p.k_stride
    p.o_stride = DecodeStrides(*_strides("bhsd", 1, hq, d))
    p.scale = effective_scale(scale, d)
    p.dtype = dtype_id(q.dtype)
    check(lib().sca_launch_decode_triples(C.byref(p), triples.data_ptr(), _stream_ptr(stream)))
    return triples


def decode_partials(q, k, v, *, scale=None, num_splits: int = 0, stream=None):
    """The split-K partial kernel alone. Returns (m [rows, splits], l [rows, splits], O [rows, splits, D],
    splits) as fp32 views of the scratch pool (valid until this thread's next decode call on the stream)."""
    _require_cuda(q, k, v)
    b, hq, hkv, skv, d = _shard_dims(q, k, v)
    splits = min(num_splits, MAX_SPLITS) if num_splits > 0 else splits_for(skv, b, hkv, hq // hkv, sm_count(q.device))
    base = b * hq * splits
    ws = acquire_scratch_fp32(base * (2 + d), q.device, stream=stream)
    p = DecodeFwdParams()
    p.q, p.k, p.v, p.out = q.data_ptr(), k.data_ptr(), v.data_ptr(), None
    scratch = ws.data_ptr()
    p.partial_m, p.partial_l, p.partial_o = scratch, scratch + 4 * base, scratch + 8 * base
    p.batch, p.num_heads, p.num_kv_heads, p.seq_kv, p.head_dim, p.num_splits = b, hq, hkv, skv, d, splits
    p.q_stride = DecodeStrides(*_strides("bhsd", 1, hq, d))
    p.k_stride = DecodeStrides(*_strides("bhsd", skv, hkv, d))
    p.v_stride = p.k_stride
    p.o_stride = DecodeStrides(*_strides("bhsd", 1, hq, d))
    p.scale = effective_scale(scale, d)
    p.dtype = dtype_id(q.dtype)
    check(lib().sca_launch_decode_partials(C.byref(p), _stream_ptr(stream)))
    return ws[:base], ws[base: 2 * base], ws[2 * base: base * (2 + d)], splits


def merge_triples(gathered, out_dtype, *, stream=None):
    """gathered fp32 [ranks, rows, 2 + D] -> normalised output [rows, D] of `out_dtype`."""
    _require_cuda(gathered)
    _require_packed("triples", gathered)
    if gathered.dtype != torch.float32:
        raise _lib.ScaError(4, f"triples must be float32; got {gathered.dtype}")
    ranks, rows, width = gathered.shape
    d = width - 2
    out = _empty((rows, d), out_dtype, gathered.device, stream)
    check(lib().sca_launch_merge_triples(gathered.data_ptr(), ranks, rows, d, out.data_ptr(),
                                         dtype_id(out_dtype), _stream_ptr(stream)))
    return out


# ------------------------------------------------------------------------------------------------
# prefill
# ------------------------------------------------------------------------------------------------
def _fwd_params(q, k, v, out, lse, causal, scale, layout):
    b, hq, sq, d = _dims(q, layout)
    bk, hkv, skv, dk = _dims(k, layout)
    if (bk, dk) != (b, d) or tuple(v.shape) != tuple(k.shape) or q.dtype != k.dtype or q.dtype != v.dtype:
        raise _lib.ScaError(4, "q/k/v shape or dtype mismatch")
    _require_packed("v", v)
    if not out.is_contiguous() or out.dtype != q.dtype or out.numel() < q.numel() or (
            lse is not None and (not lse.is_contiguous() or lse.dtype != torch.float32 or lse.numel() < b * hq * sq)):
        raise _lib.ScaError(4, "out must be a contiguous tensor of q's type and size, lse of float32 and one entry per row")
    if causal and skv < sq:
        raise _lib.ScaError(4, f"causal=true but seq_kv({skv}) < seq_q({sq})")
    p = FlashFwdParams()
    p.q, p.k, p.v, p.out = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
    p.lse = lse.data_ptr() if lse is not None else None
    p.batch, p.num_heads, p.num_kv_heads, p.seq_q, p.seq_kv, p.head_dim = b, hq, hkv, sq, skv, d
    p.q_sb, p.q_sh, p.q_ss = _strides(layout, sq, hq, d)
    p.k_sb, p.k_sh, p.k_ss = _strides(layout, skv, hkv, d)
    p.v_sb, p.v_sh, p.v_ss = p.k_sb, p.k_sh, p.k_ss
    p.o_sb, p.o_sh, p.o_ss = _strides("bhsd", sq, hq, d)
    p.scale = effective_scale(scale, d)
    p.causal = int(bool(causal))
    p.return_lse = int(lse is not None)
    p.diagonal = (skv - sq) if causal else 0
    p.dtype_id = dtype_id(q.dtype)
    return p


def _alloc_out(q, layout, return_lse, stream):
    b, hq, sq, d = _dims(q, layout)
    out = _empty((b, hq, sq, d), q.dtype, q.device, stream)
    lse = _empty((b, hq, sq), torch.float32, q.device, stream) if return_lse else None
    return out, lse


def flash_status(device=None) -> int:
    """0 when every flash launch on `device` so far ran to completion, otherwise 1 + the warp whose bounded wait ran
    out (that launch's output is invalid). Synchronise the stream first; reading clears the record."""
    index = torch.cuda.current_device() if device is None else torch.device(device).index
    code = C.c_int32(0)
    check(lib().sca_flash_status(int(index or 0), C.byref(code)))
    return int(code.value)


def flash_attention(q, k, v, *, causal=False, scale=None, return_lse=False, layout="bhsd", stream=None,
                    out=None, lse=None):
    """tcgen05 flash prefill (sca::flash_attention); fp16 / bf16 only."""
    if stream is None and out is None and q.is_cuda:
        res = _native().flash(q, k, v, causal, scale, return_lse, layout, False)
        if res is not None:
            return res
    _require_cuda(q, k, v)
    if q.dtype == torch.float32:
        raise _lib.ScaError(4, "flash backend computes in fp16/bf16; dtype=float32 is served by the naive "
                               "(reference) or tiled backend")
    if out is None:
        out, lse = _alloc_out(q, layout, return_lse, stream)
    else:
        _require_cuda(out, lse)
    p = _fwd_params(q, k, v, out, lse, causal, scale, layout)
    check(lib().sca_launch_flash_fwd(C.byref(p), _stream_ptr(stream)))
    return (out, lse) if return_lse else out


def flash_attention_varlen(q, k, v, cu_seqlens_q, cu_seqlens_kv, *, causal=False, scale=None, stream=None):
    """Packed variable-length prefill in one launch. q [T_q, H_q, D], k / v [T_kv, H_kv, D] on the device;
    cu_seqlens_* are HOST int32 offsets (num_seqs + 1 entries, as in the reference API). Returns [T_q, H_q, D]."""
    if stream is None and q.is_cuda:
        out = _native().varlen(q, k, v, cu_seqlens_q, cu_seqlens_kv, causal, scale)
        if out is not None:
            return out
    import numpy as np
    _require_cuda(q, k, v)
    if q.dim() != 3 or k.dim() != 3 or tuple(k.shape) != tuple(v.shape) or not (q.is_contiguous() and k.is_contiguous() and v.is_contiguous()):
        raise _lib.ScaError(4, "varlen expects contiguous packed [T, H, D] tensors")
    _require_like(q, k, v)
    if k.shape[2] != q.shape[2]:
        raise _lib.ScaError(4, "q/k/v shape or dtype mismatch")
    cu_q = np.ascontiguousarray(cu_seqlens_q, dtype=np.int32)
    cu_kv = np.ascontiguousarray(cu_seqlens_kv, dtype=np.int32)
    if cu_q.ndim != 1 or cu_q.shape != cu_kv.shape or cu_q.shape[0] < 2:
        raise _lib.ScaError(4, "cu_seqlens_q / cu_seqlens_kv must be host int32 arrays of num_seqs + 1 entries")
    tq, hq, d = q.shape
    tkv, hkv, _ = k.shape
    n = cu_q.shape[0] - 1
    out = _empty(q.shape, q.dtype, q.device, stream)
    ws_bytes = lib().sca_flash_varlen_workspace_bytes(n, tq)
    ws = _empty(max(int(ws_bytes), 16), torch.uint8, q.device, stream)
    p = _lib.FlashVarlenParams()
    p.q, p.k, p.v, p.out = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
    p.total_q, p.total_kv, p.num_heads, p.num_kv_heads, p.head_dim, p.num_seqs = tq, tkv, hq, hkv, d, n
    p.cu_seqlens_q, p.cu_seqlens_kv = cu_q.ctypes.data, cu_kv.ctypes.data
    p.scale = effective_scale(scale, d)
    p.causal = 1 if causal else 0
    p.dtype_id = dtype_id(q.dtype)
    p.workspace, p.workspace_bytes = ws.data_ptr(), ws.numel()
    check(lib().sca_launch_flash_varlen(C.byref(p), _stream_ptr(stream)))
    return out


def flash_attention_paged(q, k_pool, v_pool, page_table, cu_seqlens_q, seq_lens_kv, *, causal=True, scale=None, stream=None):
    """Chunked prefill over a paged KV cache in one launch: q packed [T_q, H_q, D] (the new tokens of every
    sequence), pools [num_blocks, block_size, H_kv, D], page_table int32 [num_seqs, max_blocks_per_seq] on the device,
    cu_seqlens_q (num_seqs + 1) and seq_lens_kv (num_seqs: tokens of each sequence in the cache, the new ones
    included) on the HOST. Returns [T_q, H_q, D]."""
    if stream is None and q.is_cuda:
        out = _native().chunk(q, k_pool, v_pool, page_table, cu_seqlens_q, seq_lens_kv, causal, scale)
        if out is not None:
            return out
    import numpy as np
    _require_cuda(q, k_pool, v_pool, page_table)
    if q.dim() != 3 or k_pool.dim() != 4 or tuple(k_pool.shape) != tuple(v_pool.shape) or not (
            q.is_contiguous() and k_pool.is_contiguous() and v_pool.is_contiguous() and page_table.is_contiguous()):
        raise _lib.ScaError(4, "paged prefill expects packed q [T, H, D] and contiguous pools [blocks, block_size, H_kv, D]")
    _require_like(q, k_pool, v_pool)
    if page_table.dtype != torch.int32 or page_table.dim() != 2:
        raise _lib.ScaError(4, "page_table must be int32 [num_seqs, max_blocks_per_seq]")
    cu_q = np.ascontiguousarray(cu_seqlens_q, dtype=np.int32)
    lens = np.ascontiguousarray(seq_lens_kv, dtype=np.int32)
    n = lens.shape[0]
    if cu_q.ndim != 1 or cu_q.shape[0] != n + 1 or page_table.shape[0] < n:
        raise _lib.ScaError(4, "cu_seqlens_q needs num_seqs + 1 entries, seq_lens_kv and the page table num_seqs")
    tq, hq, d = q.shape
    nblk, bs, hkv, dk = k_pool.shape
    if dk != d:
        raise _lib.ScaError(4, "pool head_dim differs from q")
    out = _empty(q.shape, q.dtype, q.device, stream)
    ws_bytes = lib().sca_flash_varlen_workspace_bytes(n, tq)
    ws = _empty(max(int(ws_bytes), 16), torch.uint8, q.device, stream)
    p = _lib.FlashPagedParams()
    p.q, p.out, p.k_pool, p.v_pool, p.page_table = q.data_ptr(), out.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), page_table.data_ptr()
    p.total_q, p.num_heads, p.num_kv_heads, p.head_dim, p.num_seqs = tq, hq, hkv, d, n
    p.num_blocks, p.block_size, p.max_blocks_per_seq = nblk, bs, page_table.shape[1]
    p.cu_seqlens_q, p.seq_lens_kv = cu_q.ctypes.data, lens.ctypes.data
    p.scale = effective_scale(scale, d)
    p.causal = 1 if causal else 0
    p.dtype_id = dtype_id(q.dtype)
    p.workspace, p.workspace_bytes = ws.data_ptr(), ws.numel()
    check(lib().sca_launch_flash_paged(C.byref(p), _stream_ptr(stream)))
    return out


def simt_attention(q, k, v, *, causal=False, scale=None, return_lse=False, layout="bhsd", stream=None):
    """Functional SIMT attention behind the naive / tiled backends (any compute dtype)."""
    if stream is None and q.is_cuda:
        res = _native().flash(q, k, v, causal, scale, return_lse, layout, True)
        if res is not None:
            return res
    _require_cuda(q, k, v)
    out, lse = _alloc_out(q, layout, return_lse, stream)
    p = _fwd_params(q, k, v, out, lse, causal, scale, layout)
    check(lib().sca_launch_simt_forward(C.byref(p), _stream_ptr(stream)))
    return (out, lse) if return_lse else out


def naive_attention(q, k, v, *, causal=False, scale=None, return_lse=False, layout="bhsd", stream=None):
    """Level-1 attention with the fp32 score matrix materialised in scratch (sca::naive_attention)."""
    _require_cuda(q, k, v)
    out, lse = _alloc_out(q, layout, return_lse, stream)
    p = _fwd_params(q, k, v, out, lse, causal, scale, layout)
    need = lib().sca_naive_score_bytes(p.batch, p.num_heads, p.seq_q, p.seq_kv)
    if need <= 0:
        raise _lib.ScaError(4, "naive attention: invalid geometry")
    scores = _empty(need // 4, torch.float32, q.device, stream)
    check(lib().sca_launch_naive_forward(C.byref(p), scores.data_ptr(), _stream_ptr(stream)))
    return (out, lse) if return_lse else out


# ------------------------------------------------------------------------------------------------
# KV cache data movement (pools are [num_blocks, block_size, H_kv, D])
# ------------------------------------------------------------------------------------------------
def _kv_shape(pool: torch.Tensor) -> KvCacheShape:
    nblk, bs, hkv, d = pool.shape
    return KvCacheShape(nblk, bs, hkv, d)


def kv_append(layer_k, layer_v, k_new, v_new, slot_mapping, *, stream=None) -> None:
    """k_new/v_new [num_tokens, H_kv, D]; slot_mapping int32 [num_tokens] on the device."""
    if stream is None and layer_k.is_cuda and _native().append(layer_k, layer_v, k_new, v_new, slot_mapping):
        return
    _require_cuda(layer_k, layer_v, k_new, v_new, slot_mapping)
    shape = _kv_shape(layer_k)
    _require_pools(layer_k, layer_v)
    _require_rows(layer_k, k_new.shape[0], k_new, v_new)
    _require_ints("slot_mapping", slot_mapping, k_new.shape[0])
    check(lib().sca_launch_kv_append(layer_k.data_ptr(), layer_v.data_ptr(), k_new.data_ptr(),
                                     v_new.data_ptr(), slot_mapping.data_ptr(), k_new.shape[0],
                                     C.byref(shape), layer_k.element_size(), _stream_ptr(stream)))


def kv_append_batched(layer_k, layer_v, k_new, v_new, page_table, seq_lens, *, stream=None) -> None:
    """One new token per sequence; the slot comes from the page table at position seq_lens[s] - 1."""
    if stream is None and layer_k.is_cuda and _native().append_batched(layer_k, layer_v, k_new, v_new, page_table, seq_lens):
        return
    _require_cuda(layer_k, layer_v, k_new, v_new, page_table, seq_lens)
    shape = _kv_shape(layer_k)
    _require_pools(layer_k, layer_v)
    _require_rows(layer_k, k_new.shape[0], k_new, v_new)
    _require_table(page_table, k_new.shape[0])
    _require_ints("seq_lens", seq_lens, k_new.shape[0])
    check(lib().sca_launch_kv_append_batched(layer_k.data_ptr(), layer_v.data_ptr(), k_new.data_ptr(),
                                             v_new.data_ptr(), page_table.data_ptr(), seq_lens.data_ptr(),
                                             k_new.shape[0], page_table.shape[1], C.byref(shape),
                                             layer_k.element_size(), _stream_ptr(stream)))


def kv_reset(layer_k, layer_v, block_ids, *, stream=None) -> None:
    if stream is None and layer_k.is_cuda and _native().reset(layer_k, layer_v, block_ids):
        return
    _require_cuda(layer_k, layer_v, block_ids)
    shape = _kv_shape(layer_k)
    _require_pools(layer_k, layer_v)
    _require_ints("block_ids", block_ids, 0)
    check(lib().sca_launch_kv_reset_block(layer_k.data_ptr(), layer_v.data_ptr(), block_ids.data_ptr(),
                                          block_ids.numel(), C.byref(shape), layer_k.element_size(),
                                          _stream_ptr(stream)))


def kv_gather(layer, block_ids, *, stream=None) -> torch.Tensor:
    if stream is None and layer.is_cuda:
        out = _native().gather(layer, block_ids)
        if out is not None:
            return out
    _require_cuda(layer, block_ids)
    shape = _kv_shape(layer)
    _require_packed("pool", layer)
    _require_ints("block_ids", block_ids, 0)
    out = _empty((block_ids.numel(),) + tuple(layer.shape[1:]), layer.dtype, layer.device, stream)
    check(lib().sca_launch_kv_gather(layer.data_ptr(), block_ids.data_ptr(), block_ids.numel(),
                                     out.data_ptr(), C.byref(shape), layer.element_size(),
                                     _stream_ptr(stream)))
    return out


# ------------------------------------------------------------------------------------------------
# 8-bit KV cache
# ------------------------------------------------------------------------------------------------
class Fp8Pool(NamedTuple):
    """K or V of one layer in 8 bits. A row - one token of one kv head - is D codes of type e4m3 and one scale 2^e with e in [-14, 7], the
    smallest one with min(max |x|, 57344) <= 448 * 2^e; value = code * 2^e, exact in fp16 and bf16. Numbers beyond +-57344 (bf16, fp32)
    are kept as +-57344, NaN stays NaN.

    codes   float8_e4m3fn (or uint8) [num_blocks, block_size, H_kv, D], D a multiple of 16 up to 256
    scales  uint8 [num_blocks, H_kv, block_size rounded up to 16]: e + 15

    Append and read-back take any such pair. Attention takes D = 32, 64, 96, 128, 160, 192 and 256: a token per sequence (paged_attention_fp8) a
    block_size that is a multiple of 4, chunks (flash_attention_paged_fp8) one of 8, 16, 32 or 64. Other pools are for storage alone.
    Blocks are freed by kv_reset on the codes: a code of 0 is 0 under every scale."""
    codes: torch.Tensor
    scales: torch.Tensor


def fp8_scale_row(block_size: int) -> int:
    """Bytes of scales per block and kv head."""
    return -(-block_size // 16) * 16


def fp8_pool(num_blocks: int, block_size: int, num_kv_heads: int, head_dim: int, *, device="cuda") -> Fp8Pool:
    """An empty pool: every value 0."""
    return Fp8Pool(torch.zeros((num_blocks, block_size, num_kv_heads, head_dim), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn),
                   torch.full((num_blocks, num_kv_heads, fp8_scale_row(block_size)), 15, dtype=torch.uint8, device=device))


def fp8_ctas_per_sm(head_dim: int, group: int) -> int:
    """CTAs of the 8-bit decode kernel that stay on an SM."""
    return 4 if head_dim <= 64 else 2 if group > 8 and head_dim > 96 else 3


def fp8_step_tokens(head_dim: int) -> int:
    """The unit of its schedule."""
    return 64 if head_dim > 128 else 128


def _require_one_device(first: torch.Tensor, *others: torch.Tensor) -> None:
    for t in others:
        if t.device != first.device:
            raise _lib.ScaError(4, f"tensors on {first.device} and {t.device}: a call's tensors are on one device")


def _require_fp8_pool(pool) -> None:
    codes, scales = pool
    _require_cuda(codes, scales)
    if codes.dim() != 4 or codes.dtype not in (torch.float8_e4m3fn, torch.uint8) or not codes.is_contiguous():
        raise _lib.ScaError(4, f"codes must be contiguous float8_e4m3fn [num_blocks, block_size, H_kv, D]; got {codes.dtype}{list(codes.shape)}")
    nblk, bs, hkv, _ = codes.shape
    if scales.dtype != torch.uint8 or tuple(scales.shape) != (nblk, hkv, fp8_scale_row(bs)) or not scales.is_contiguous():
        raise _lib.ScaError(4, f"scales must be contiguous uint8 {[nblk, hkv, fp8_scale_row(bs)]}; got {scales.dtype}{list(scales.shape)}")


def _require_fp8_pools(layer_k, layer_v) -> None:
    _require_fp8_pool(layer_k)
    _require_fp8_pool(layer_v)
    if layer_k[0].shape != layer_v[0].shape:
        raise _lib.ScaError(4, "pool geometry mismatch")


def _require_fp8_rows(codes, rows: int, k_new, v_new) -> None:
    _require_cuda(k_new, v_new)
    dtype_id(k_new.dtype)  # one that can be quantised
    if k_new.dtype != v_new.dtype:
        raise _lib.ScaError(4, "k_new/v_new shape or dtype mismatch")
    width = codes.shape[2] * codes.shape[3]
    for t in (k_new, v_new):
        if not t.is_contiguous() or t.dim() < 1 or t.shape[0] < rows or t.numel() != t.shape[0] * width:
            raise _lib.ScaError(4, f"new K / V must be contiguous [{rows}, {codes.shape[2]}, {codes.shape[3]}]; got {t.dtype}{list(t.shape)}")


def _fp8_layer(layer_k, layer_v):
    return _lib.Fp8Layer(layer_k[0].data_ptr(), layer_v[0].data_ptr(), layer_k[1].data_ptr(), layer_v[1].data_ptr())


def _elsewhere(t: torch.Tensor, stream) -> bool:
    """Whether a launch without a stream of its own has to make the tensors' device the current one."""
    return stream is None and t.device.index != torch.cuda.current_device()


def kv_append_fp8(layer_k, layer_v, k_new, v_new, slot_mapping, *, stream=None) -> None:
    """kv_append into an 8-bit layer (two Fp8Pool): k_new/v_new [num_tokens, H_kv, D] of float32, float16 or bfloat16 are quantised as they
    are written; slot_mapping int32 [num_tokens] on the device, slots < 0 or beyond the pool are skipped. The slots of a call are distinct:
    one that is named twice is left with pieces of both rows."""
    if stream is None and _native().append_fp8(*layer_k, *layer_v, k_new, v_new, slot_mapping):
        return
    _require_fp8_pools(layer_k, layer_v)
    _require_fp8_rows(layer_k[0], k_new.shape[0], k_new, v_new)
    _require_ints("slot_mapping", slot_mapping, k_new.shape[0])
    _require_one_device(k_new, v_new, slot_mapping, *layer_k, *layer_v)
    if k_new.shape[0] == 0:
        return
    if _elsewhere(k_new, stream):
        with torch.cuda.device(k_new.device):
            return kv_append_fp8(layer_k, layer_v, k_new, v_new, slot_mapping)
    shape = _kv_shape(layer_k[0])
    check(lib().sca_launch_kv_append_fp8(C.byref(_fp8_layer(layer_k, layer_v)), k_new.data_ptr(), v_new.data_ptr(), slot_mapping.data_ptr(),
                                         k_new.shape[0], C.byref(shape), dtype_id(k_new.dtype), _stream_ptr(stream)))


def kv_append_batched_fp8(layer_k, layer_v, k_new, v_new, page_table, seq_lens, *, stream=None) -> None:
    """kv_append_batched into an 8-bit layer: one new token per sequence, at position seq_lens[s] - 1 of its pages; no two at the same place."""
    if stream is None and _native().append_batched_fp8(*layer_k, *layer_v, k_new, v_new, page_table, seq_lens):
        return
    _require_fp8_pools(layer_k, layer_v)
    _require_fp8_rows(layer_k[0], k_new.shape[0], k_new, v_new)
    _require_cuda(page_table)
    _require_table(page_table, k_new.shape[0])
    _require_ints("seq_lens", seq_lens, k_new.shape[0])
    _require_one_device(k_new, v_new, page_table, seq_lens, *layer_k, *layer_v)
    if k_new.shape[0] == 0:
        return
    if _elsewhere(k_new, stream):
        with torch.cuda.device(k_new.device):
            return kv_append_batched_fp8(layer_k, layer_v, k_new, v_new, page_table, seq_lens)
    shape = _kv_shape(layer_k[0])
    check(lib().sca_launch_kv_append_batched_fp8(C.byref(_fp8_layer(layer_k, layer_v)), k_new.data_ptr(), v_new.data_ptr(), page_table.data_ptr(),
                                                 seq_lens.data_ptr(), k_new.shape[0], page_table.shape[1], C.byref(shape),
                                                 dtype_id(k_new.dtype), _stream_ptr(stream)))


def kv_gather_fp8(layer, block_ids, dtype, *, stream=None) -> torch.Tensor:
    """Reads blocks of an 8-bit pool back: [len(block_ids), block_size, H_kv, D] of `dtype` (float32, float16 or bfloat16). Ids outside the
    pool read as zeros."""
    if stream is None:
        out = _native().gather_fp8(*layer, block_ids, dtype)
        if out is not None:
            return out
    _require_fp8_pool(layer)
    _require_ints("block_ids", block_ids, 0)
    codes, scales = layer
    _require_one_device(codes, scales, block_ids)
    kind = dtype_id(dtype)
    if _elsewhere(codes, stream):
        with torch.cuda.device(codes.device):
            return kv_gather_fp8(layer, block_ids, dtype)
    shape = _kv_shape(codes)
    out = _empty((block_ids.numel(),) + tuple(codes.shape[1:]), dtype, codes.device, stream)
    if out.numel() > 0:
        check(lib().sca_launch_kv_gather_fp8(codes.data_ptr(), scales.data_ptr(), block_ids.data_ptr(), block_ids.numel(), out.data_ptr(),
                                             C.byref(shape), kind, _stream_ptr(stream)))
    return out


def paged_attention_fp8(q, k_pool, v_pool, page_table, seq_lens, *, block_size: int, scale=None, typical_len: int = 0, longest_len: int = 0,
                        stream=None, return_stats: bool = False):
    """paged_attention over an 8-bit cache: q [num_seqs, H_q, 1, D] of float16 or bfloat16, pools as Fp8Pool with a block_size that is a
    multiple of 4; table, lengths and hints as there. The new tokens' K / V are in the cache (kv_append_batched_fp8)."""
    if stream is None and not return_stats:
        out = _native().paged_fp8(*k_pool, *v_pool, q, page_table, seq_lens, block_size, scale, typical_len, longest_len)
        if out is not None:
            return out
    _require_cuda(q, page_table, seq_lens)
    _require_fp8_pools(k_pool, v_pool)
    if q.dim() != 4:
        raise _lib.ScaError(4, f"paged_attention expects q=[num_seqs, H_q, seq_q, D]; got ndims={q.dim()}")
    s, hq, sq, d = q.shape
    if sq != 1:
        raise _lib.ScaError(5, f"paged attention implements the decode form only (seq_q=1); got seq_q={sq}")
    codes = k_pool[0]
    nblk, bs, hkv, dk = codes.shape
    if bs != block_size or dk != d:
        raise _lib.ScaError(4, "pool geometry mismatch")
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise _lib.ScaError(4, f"attention over an 8-bit cache takes float16 or bfloat16 queries; got {q.dtype}")
    if hkv < 1 or hq % hkv != 0:
        raise _lib.ScaError(4, f"num_heads={hq} % num_kv_heads={hkv} != 0")
    _require_packed("q", q)
    _require_table(page_table, s)
    if seq_lens is not None:
        _require_ints("seq_lens", seq_lens, s)
    _require_one_device(q, page_table, *k_pool, *v_pool, *(() if seq_lens is None else (seq_lens,)))
    if _elsewhere(q, stream):
        with torch.cuda.device(q.device):
            return paged_attention_fp8(q, k_pool, v_pool, page_table, seq_lens, block_size=block_size, scale=scale, typical_len=typical_len,
                                       longest_len=longest_len, return_stats=return_stats)
    max_blocks, upper = page_table.shape[1], nblk * bs
    device, handle = q.device, _stream_ptr(stream)
    splits = paged_splits_for(typical_len if typical_len > 0 else min(upper, max_blocks * bs), s, hkv, hq // hkv, sm_count(device), longest_len,
                              fp8_step_tokens(d), fp8_ctas_per_sm(d, hq // hkv), FP8_MAX_SPLITS, FP8_BORDER_STEPS)
    base = s * hq * splits
    o_at = -(-2 * base // 4) * 4  # the O of a part starts on 16 bytes
    ws = acquire_scratch_fp32(o_at + base * d, device, stream=stream, handle=handle)
    out = _empty((s, hq, 1, d), q.dtype, device, stream)
    p = DecodeFwdParams()
    p.q, p.k, p.v, p.out = q.data_ptr(), codes.data_ptr(), v_pool[0].data_ptr(), out.data_ptr()
    scratch = ws.data_ptr()
    p.partial_m, p.partial_l, p.partial_o = scratch, scratch + 4 * base, scratch + 4 * o_at
    p.batch, p.num_heads, p.num_kv_heads, p.seq_kv, p.head_dim, p.num_splits = s, hq, hkv, min(upper, longest_len) if longest_len > 0 and seq_lens is not None else upper, d, splits
    p.q_stride = DecodeStrides(hq * d, d, d)
    p.o_stride = DecodeStrides(hq * d, d, d)
    p.scale = effective_scale(scale, d)
    p.dtype = dtype_id(q.dtype)
    p.seq_lens = seq_lens.data_ptr() if seq_lens is not None else None
    p.page_table = page_table.data_ptr()
    p.block_size, p.max_blocks_per_seq, p.num_kv_blocks = bs, max_blocks, nblk
    cluster = C.c_int32(0)
    check(lib().sca_launch_paged_attention_fp8(C.byref(p), k_pool[1].data_ptr(), v_pool[1].data_ptr(), C.byref(cluster), handle))
    if not return_stats:
        return out
    return out, {"num_splits": cluster.value or splits, "cluster": cluster.value, "workspace_bytes": base * (2 + d) * 4}


def flash_attention_paged_fp8(q, k_pool, v_pool, page_table, cu_seqlens_q, seq_lens_kv, *, causal=True, scale=None, stream=None):
    """flash_attention_paged over an 8-bit cache: q packed [T_q, H_q, D] of float16 or bfloat16, pools as Fp8Pool; the rest as there. The
    new tokens' K / V are in the cache (kv_append_fp8)."""
    if stream is None:
        out = _native().chunk_fp8(*k_pool, *v_pool, q, page_table, cu_seqlens_q, seq_lens_kv, causal, scale)
        if out is not None:
            return out
    import numpy as np
    _require_cuda(q, page_table)
    _require_fp8_pools(k_pool, v_pool)
    codes = k_pool[0]
    if q.dim() != 3 or not q.is_contiguous():
        raise _lib.ScaError(4, "paged prefill expects packed q [T, H, D]")
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise _lib.ScaError(4, f"attention over an 8-bit cache takes float16 or bfloat16 queries; got {q.dtype}")
    cu_q = np.ascontiguousarray(cu_seqlens_q, dtype=np.int32)
    lens = np.ascontiguousarray(seq_lens_kv, dtype=np.int32)
    if lens.ndim != 1 or cu_q.ndim != 1 or cu_q.shape[0] != lens.shape[0] + 1:
        raise _lib.ScaError(4, "cu_seqlens_q needs num_seqs + 1 entries, seq_lens_kv and the page table num_seqs")
    n = lens.shape[0]
    _require_table(page_table, n)
    tq, hq, d = q.shape
    nblk, bs, hkv, dk = codes.shape
    if dk != d:
        raise _lib.ScaError(4, "pool head_dim differs from q")
    _require_one_device(q, page_table, *k_pool, *v_pool)
    if _elsewhere(q, stream):
        with torch.cuda.device(q.device):
            return flash_attention_paged_fp8(q, k_pool, v_pool, page_table, cu_q, lens, causal=causal, scale=scale)
    out = _empty(q.shape, q.dtype, q.device, stream)
    ws_bytes = lib().sca_flash_varlen_workspace_bytes(n, tq)
    ws = _empty(max(int(ws_bytes), 16), torch.uint8, q.device, stream)
    p = _lib.FlashPagedParams()
    p.q, p.out, p.k_pool, p.v_pool, p.page_table = q.data_ptr(), out.data_ptr(), codes.data_ptr(), v_pool[0].data_ptr(), page_table.data_ptr()
    p.total_q, p.num_heads, p.num_kv_heads, p.head_dim, p.num_seqs = tq, hq, hkv, d, n
    p.num_blocks, p.block_size, p.max_blocks_per_seq = nblk, bs, page_table.shape[1]
    p.cu_seqlens_q, p.seq_lens_kv = cu_q.ctypes.data, lens.ctypes.data
    p.scale = effective_scale(scale, d)
    p.causal = 1 if causal else 0
    p.dtype_id = dtype_id(q.dtype)
    p.workspace, p.workspace_bytes = ws.data_ptr(), ws.numel()
    check(lib().sca_launch_flash_paged_fp8(C.byref(p), k_pool[1].data_ptr(), v_pool[1].data_ptr(), _stream_ptr(stream)))
    return out


# ------------------------------------------------------------------------------------------------
# a paged cache that stays small: what each cached token weighs, shared prefixes, eviction
# ------------------------------------------------------------------------------------------------
def _require_weights(weights, rows: int, kv_heads: int, tokens: int) -> None:
    _require_cuda(weights)
    if weights.dtype != torch.float32 or weights.dim() != 3 or weights.shape[0] < rows or weights.shape[1] != kv_heads or weights.shape[2] < tokens or \
            not weights.is_contiguous():
        raise _lib.ScaError(4, f"weights must be contiguous float32 [{rows}, {kv_heads}, {tokens}] or more rows and columns; got {weights.dtype}{list(weights.shape)}")


def _host_ints(what: str, values):
    """A host list as a contiguous int32 array of one dimension."""
    import numpy as np
    given = np.asarray(values)
    if given.ndim != 1 or given.dtype.kind not in "iu":
        raise _lib.ScaError(4, f"{what} must be a list of whole numbers on the host; got {given.dtype}{list(given.shape)}")
    out = np.ascontiguousarray(given, dtype=np.int32)
    if not np.array_equal(out, given):
        raise _lib.ScaError(4, f"{what} must fit 32 bits")
    return out


def _paged_step(q, k_pool, v_pool, page_table, seq_lens, cu_groups, prefix_lens, weights, block_size, scale, typical_len, longest_len, stream):
    if stream is None:
        out = _native().paged_step(q, k_pool, v_pool, page_table, seq_lens, cu_groups, prefix_lens, weights, block_size, scale, typical_len, longest_len)
        if out is not None:
            return out
    _require_cuda(q, k_pool, v_pool, page_table, seq_lens)
    if q.dim() != 4:
        raise _lib.ScaError(4, f"paged_attention expects q=[num_seqs, H_q, seq_q, D]; got ndims={q.dim()}")
    s, hq, sq, d = q.shape
    if sq != 1:
        raise _lib.ScaError(5, f"paged attention implements the decode form only (seq_q=1); got seq_q={sq}")
    if k_pool.dim() != 4:
        raise _lib.ScaError(4, "pool geometry mismatch")
    nblk, bs, hkv, dk = k_pool.shape
    if bs != block_size or dk != d or tuple(v_pool.shape) != tuple(k_pool.shape):
        raise _lib.ScaError(4, "pool geometry mismatch")
    _require_like(q, k_pool, v_pool)
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise _lib.ScaError(4, f"weights and shared prefixes are for float16 or bfloat16; got {q.dtype}")
    if hkv < 1 or hq < 1 or hq % hkv != 0:
        raise _lib.ScaError(4, f"num_heads={hq} % num_kv_heads={hkv} != 0")
    _require_packed("q or pool", q, k_pool, v_pool)
    _require_table(page_table, s)
    if seq_lens is not None:
        _require_ints("seq_lens", seq_lens, s)
    if cu_groups is not None and (cu_groups[0] != 0 or cu_groups[-1] != s):
        raise _lib.ScaError(4, f"cu_groups must go from 0 to num_seqs={s}")
    max_blocks = page_table.shape[1]
    tensors = [k_pool, v_pool, page_table] + ([seq_lens] if seq_lens is not None else [])
    if weights is not None:
        _require_weights(weights, s, hkv, max_blocks * bs)
        tensors.append(weights)
    _require_one_device(q, *tensors)
    if _elsewhere(q, stream):
        with torch.cuda.device(q.device):
            return _paged_step(q, k_pool, v_pool, page_table, seq_lens, cu_groups, prefix_lens, weights, block_size, scale, typical_len, longest_len, None)
    handle = _stream_ptr(stream)
    out = _empty((s, hq, 1, d), q.dtype, q.device, stream)
    if s == 0:
        return out
    p = DecodeFwdParams()
    p.q, p.k, p.v, p.out = q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), out.data_ptr()
    p.batch, p.num_heads, p.num_kv_heads, p.head_dim = s, hq, hkv, d
    p.q_stride = DecodeStrides(hq * d, d, d)
    p.o_stride = DecodeStrides(hq * d, d, d)
    p.scale = effective_scale(scale, d)
    p.dtype = dtype_id(q.dtype)
    p.page_table = page_table.data_ptr()
    p.seq_lens = seq_lens.data_ptr() if seq_lens is not None else None
    p.block_size, p.max_blocks_per_seq, p.num_kv_blocks = bs, max_blocks, nblk
    x = _lib.PagedStep()
    if prefix_lens is not None:
        x.cu_groups, x.prefix_lens, x.num_groups = cu_groups.ctypes.data, prefix_lens.ctypes.data, prefix_lens.shape[0]
    if weights is not None:
        x.weights, x.weights_row = weights.data_ptr(), weights.shape[2]
    x.typical_len, x.longest_len = max(0, int(typical_len)), max(0, int(longest_len))
    need = lib().sca_paged_step_scratch_floats(C.byref(p), C.byref(x))
    if need < 0:
        check(4)
    ws = acquire_scratch_fp32(need, q.device, stream=stream, handle=handle)
    x.scratch, x.scratch_floats = ws.data_ptr(), ws.numel()
    check(lib().sca_launch_paged_step(C.byref(p), C.byref(x), handle))
    return out


def paged_attention_weights(q, k_pool, v_pool, page_table, seq_lens, weights, *, block_size: int, scale=None, typical_len: int = 0, longest_len: int = 0,
                            stream=None):
    """paged_attention that adds up what each cached token weighs: weights[s, g, j] += the sum over the query heads h of kv head g of
    softmax_j(scale q[s, h] . k[j]), in float32, for every token j of sequence s; what lies behind its last token is left as it is. The order of
    the sum is fixed: the same call gives the same bits.

    q, pools, table, lengths as paged_attention takes them, of float16 or bfloat16; weights float32 [num_seqs, H_kv, max_blocks_per_seq *
    block_size] or more rows and columns, on the device. A query of NaN makes the weights of its kv head NaN. `typical_len` sizes the launch;
    `longest_len` does too and bounds the lengths: no sequence is longer, and a token behind it would count for nothing. The scratch of a call with weights has a
    score for every query head and token up to `longest_len`, or up to the end of the table's rows without it (2 GB at most, or one sequence's: what needs more
    runs in slices of sequences); it is kept as paged_attention's is. Give it where the table is wide."""
    if weights is None:
        raise _lib.ScaError(4, "weights must be a tensor")
    return _paged_step(q, k_pool, v_pool, page_table, seq_lens, None, None, weights, block_size, scale, typical_len, longest_len, stream)


def paged_attention_shared(q, k_pool, v_pool, page_table, seq_lens, cu_groups, prefix_lens, *, block_size: int, weights=None, scale=None, typical_len: int = 0,
                           longest_len: int = 0, stream=None):
    """paged_attention over sequences that have the pages of a prefix in common, which are read once for all of them.

    Group i is the sequences cu_groups[i] .. cu_groups[i + 1] - 1 (neighbours; cu_groups has num_groups + 1 entries from 0 to num_seqs), and all of
    them begin with the same prefix_lens[i] tokens: the table's entries of the whole pages of those tokens are the same in all rows of the group
    and are taken from its first row; tokens of a page that the prefix does not fill are each sequence's own, as are the ones behind. Both lists
    are on the HOST. At most 128 groups of two or more sequences that share a page; pages of 8, 16, 32 or 64 tokens.
    Where the shared pages are read once, their V of bfloat16 and the softmax weights become float16 numbers, as in the prefill: values beyond +-65504
    count as +-65504, those below 2^-14 as multiples of 2^-24, and a weight has 11 bits. A call that does not fill the machine may read shared pages once
    per sequence, without either: outputs of the two differ by roundings.
    With `weights` (see paged_attention_weights) the weights of each sequence's own tokens are added up; those of shared pages are left alone.
    The rest is as paged_attention_weights has it."""
    if stream is None and cu_groups is not None:
        out = _native().paged_step(q, k_pool, v_pool, page_table, seq_lens, cu_groups, prefix_lens, weights, block_size, scale, typical_len, longest_len)
        if out is not None:
            return out
    cu, lens = _host_ints("cu_groups", cu_groups), _host_ints("prefix_lens", prefix_lens)
    if cu.shape[0] < 1 or cu.shape[0] != lens.shape[0] + 1:
        raise _lib.ScaError(4, "cu_groups needs num_groups + 1 entries, prefix_lens num_groups")
    return _paged_step(q, k_pool, v_pool, page_table, seq_lens, cu, lens, weights, block_size, scale, typical_len, longest_len, stream)


def flash_attention_paged_weights(q, k_pool, v_pool, page_table, cu_seqlens_q, seq_lens_kv, weights, *, causal=True, scale=None, last: int = 0, stream=None):
    """flash_attention_paged that adds up what each cached token weighs: weights[s, g, j] += the sum over the new tokens i of sequence s and the query
    heads h of kv head g of softmax_j(scale q[i, h] . k[j]), in float32; what lies behind a sequence's last token is left as it is. The order of
    the sum is fixed: the same call gives the same bits. With `last` > 0 the last so many new tokens of each sequence count, with 0 all of them.

    q, pools, table and the lists on the host as flash_attention_paged takes them, of float16 or bfloat16; weights float32 [num_seqs, H_kv,
    max_blocks_per_seq * block_size] or more rows and columns, on the device. A query of NaN makes the weights it counts for NaN. As there, a sequence's last page is
    read whole: what it holds behind the last token counts for nothing, but must be finite in V."""
    if stream is None:
        out = _native().chunk_weights(q, k_pool, v_pool, page_table, cu_seqlens_q, seq_lens_kv, weights, causal, scale, last)
        if out is not None:
            return out
    _require_cuda(q, k_pool, v_pool, page_table)
    if q.dim() != 3 or k_pool.dim() != 4 or tuple(k_pool.shape) != tuple(v_pool.shape):
        raise _lib.ScaError(4, "paged prefill expects packed q [T, H, D] and contiguous pools [blocks, block_size, H_kv, D]")
    _require_packed("q or pool", q, k_pool, v_pool)
    _require_like(q, k_pool, v_pool)
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise _lib.ScaError(4, f"weights and shared prefixes are for float16 or bfloat16; got {q.dtype}")
    cu_q, lens = _host_ints("cu_seqlens_q", cu_seqlens_q), _host_ints("seq_lens_kv", seq_lens_kv)
    n = lens.shape[0]
    if cu_q.shape[0] != n + 1:
        raise _lib.ScaError(4, "cu_seqlens_q needs num_seqs + 1 entries, seq_lens_kv and the page table num_seqs")
    _require_table(page_table, n)
    tq, hq, d = q.shape
    nblk, bs, hkv, dk = k_pool.shape
    if dk != d:
        raise _lib.ScaError(4, "pool head_dim differs from q")
    if hkv < 1 or hq < 1 or hq % hkv != 0:
        raise _lib.ScaError(4, f"num_heads={hq} % num_kv_heads={hkv} != 0")
    if last < 0:
        raise _lib.ScaError(4, f"last={last} must not be negative")
    _require_weights(weights, n, hkv, page_table.shape[1] * bs)
    _require_one_device(q, k_pool, v_pool, page_table, weights)
    if _elsewhere(q, stream):
        with torch.cuda.device(q.device):
            return flash_attention_paged_weights(q, k_pool, v_pool, page_table, cu_q, lens, weights, causal=causal, scale=scale, last=last)
    out = _empty(q.shape, q.dtype, q.device, stream)
    ws_bytes = max(int(lib().sca_flash_varlen_workspace_bytes(n, tq)), 16)
    ws = _empty(ws_bytes, torch.uint8, q.device, stream)
    lse = _empty((hq, tq), torch.float32, q.device, stream)
    p = _lib.FlashPagedParams()
    p.q, p.out, p.k_pool, p.v_pool, p.page_table = q.data_ptr(), out.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), page_table.data_ptr()
    p.total_q, p.num_heads, p.num_kv_heads, p.head_dim, p.num_seqs = tq, hq, hkv, d, n
    p.num_blocks, p.block_size, p.max_blocks_per_seq = nblk, bs, page_table.shape[1]
    p.cu_seqlens_q, p.seq_lens_kv = cu_q.ctypes.data, lens.ctypes.data
    p.scale = effective_scale(scale, d)
    p.causal = 1 if causal else 0
    p.dtype_id = dtype_id(q.dtype)
    p.workspace, p.workspace_bytes = ws.data_ptr(), ws.numel()
    w = _lib.ChunkWeights(lse.data_ptr(), weights.data_ptr(), weights.shape[2], int(last))
    check(lib().sca_launch_flash_paged_weights(C.byref(p), C.byref(w), _stream_ptr(stream)))
    return out


def kv_evict(layer_k, layer_v, weights, page_table, seq_lens, *, keep: int, recent: int = 0, first=0, stream=None) -> torch.Tensor:
    """Brings every sequence down to m = max(keep, first + recent) tokens, each kv head on its own: of n > m tokens the first `first` are kept, the
    last `recent`, and of those in between the m - first - recent of the largest weights (equal ones: the lower place; NaN counts as the
    largest). Returns the new lengths, int32 [num_seqs]: min(n, m). The pages behind them may be freed.

    In place, and a row moves once at most: afterwards [0, first) and [m - recent, m) hold the first and the last tokens in order; in
    [first, m - recent) those kept stay where they are, and the i-th place that comes free takes the i-th of those kept behind m - recent, both
    counted upwards. weights (float32, as paged_attention_weights takes them) go along and become 0 in places [m, n). Sequences of up to m tokens
    are left alone.
    `first`: a number, or int32 [num_seqs] on the device - the tokens of a shared prefix, say, whose pages belong to others too: a page that
    holds any other token belongs to one sequence only. Pools as kv_append takes them, of any type, but not the codes of an 8-bit layer, whose
    scales would stay where they are; rows on unmapped pages are not copied. The launch is sized by the width of the table: one that fits its sequences is
    the faster one."""
    if stream is None:
        new_lens = _native().evict(layer_k, layer_v, weights, page_table, seq_lens, keep, recent, first)
        if new_lens is not None:
            return new_lens
    _require_cuda(layer_k, layer_v, weights, page_table, seq_lens)
    if layer_k.dim() != 4 or layer_v.dim() != 4:
        raise _lib.ScaError(4, "pool geometry mismatch")
    _require_pools(layer_k, layer_v)
    if page_table.dim() != 2:
        raise _lib.ScaError(4, "page_table must be int32 [num_seqs, max_blocks_per_seq], contiguous")
    n = seq_lens.numel()
    _require_ints("seq_lens", seq_lens, 0)
    _require_table(page_table, n)
    shape, max_blocks = _kv_shape(layer_k), page_table.shape[1]
    _require_weights(weights, n, shape.num_kv_heads, max_blocks * shape.block_size)
    tensors = [layer_v, weights, page_table, seq_lens]
    by_sequence = isinstance(first, torch.Tensor)
    if by_sequence:
        _require_ints("first", first, n)
        tensors.append(first)
    keep, recent, first = int(keep), int(recent), first if by_sequence else int(first)
    if keep < 0 or recent < 0 or (not by_sequence and first < 0):
        raise _lib.ScaError(4, f"keep={keep}, recent={recent} and first must not be negative")
    _require_one_device(layer_k, *tensors)
    if _elsewhere(layer_k, stream):
        with torch.cuda.device(layer_k.device):
            return kv_evict(layer_k, layer_v, weights, page_table, seq_lens, keep=keep, recent=recent, first=first)
    new_lens = _empty((n,), torch.int32, layer_k.device, stream)
    if n == 0:
        return new_lens
    x = _lib.KvEvict()
    x.layer_k, x.layer_v, x.weights, x.weights_row = layer_k.data_ptr(), layer_v.data_ptr(), weights.data_ptr(), weights.shape[2]
    x.page_table, x.seq_lens, x.new_lens = page_table.data_ptr(), seq_lens.data_ptr(), new_lens.data_ptr()
    x.first_lens, x.first = (first.data_ptr(), 0) if by_sequence else (None, first)
    x.num_seqs, x.max_blocks_per_seq, x.keep, x.recent = n, max_blocks, keep, recent
    need = lib().sca_kv_evict_scratch_ints(n, shape.num_kv_heads, keep, max_blocks * shape.block_size)
    if need < 0:
        raise _lib.ScaError(4, "kv evict: sizes must be positive")
    handle = _stream_ptr(stream)
    ws = acquire_scratch_fp32(need, layer_k.device, stream=stream, handle=handle)
    x.scratch, x.scratch_ints = ws.data_ptr(), ws.numel()
    check(lib().sca_launch_kv_evict(C.byref(x), C.byref(shape), layer_k.element_size(), handle))
    return new_lens
