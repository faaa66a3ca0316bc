"""The reference's per-operator host wrappers (src/kernels.cuh:24-36) over the C ABI, for torch CUDA tensors.

Same names and argument meaning as the reference; tensors stand in for raw device pointers.  Work is
queued on torch's current stream; nothing here synchronises.  There is no CPU path.
"""
from __future__ import annotations

import ctypes as C
import functools
import struct

import torch

from .engine import LPP_BF16, LPP_F16, LPP_F32, _check, load_library

WEIGHT_FP32, WEIGHT_FP16 = 0, 1  # src/model.h:8-12


def _p(t: torch.Tensor) -> C.c_void_p:
    if not t.is_cuda or not t.is_contiguous():
        raise ValueError("expected a contiguous CUDA tensor")
    return C.c_void_p(t.data_ptr())


def _s() -> C.c_void_p:
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


_bound = None


def _lib():
    return _bound or _bind()


def _bind():
    global _bound
    lib = load_library()
    if not getattr(lib, "_ops_bound", False):
        vp, i, f, i64 = C.c_void_p, C.c_int, C.c_float, C.c_int64
        lib.lpp_op_convert_f32_to_f16.argtypes = [vp, vp, i64, vp]
        lib.lpp_op_gemv.argtypes = [vp, vp, vp, i, i, i, vp]
        lib.lpp_op_rmsnorm.argtypes = [vp, vp, vp, i, vp]
        lib.lpp_op_rope.argtypes = [vp, vp, i, i, i, i, f, vp]
        lib.lpp_op_swiglu.argtypes = [vp, vp, vp, i, vp]
        lib.lpp_op_softmax_multihead.argtypes = [vp, vp, i, i, i, vp]
        lib.lpp_op_scale_multihead.argtypes = [vp, f, i, i, i, vp]
        lib.lpp_op_aggregation_multihead.argtypes = [vp, vp, vp, i, i, i, i, i, vp]
        lib.lpp_op_residual_add.argtypes = [vp, vp, vp, i, vp]
        lib.lpp_op_scatter_kv.argtypes = [vp, vp, vp, vp, i, i, i, i, i, vp]
        lib.lpp_op_multihead_gemv.argtypes = [vp, vp, vp, i, i, i, i, i, i, vp]
        lib.lpp_op_rope_scatter.argtypes = [vp, vp, vp, vp, vp, i, i, i, i, i, i, f, vp]
        lib.lpp_op_sample.argtypes = [vp, i, f, f, vp, i, f, vp, vp]
        lib.lpp_op_sample_on.argtypes = [vp, i64, vp, i, f, f, vp, i, f, vp, vp]
        lib.lpp_op_sample_scratch_bytes.argtypes = [i]
        lib.lpp_op_sample_scratch_bytes.restype = i64
        lib.lpp_op_prompt_attention.argtypes = [vp, vp, vp, vp, vp, i, i, i, i, i, i64, i64, i64, i64, f, i, vp]
        lib.lpp_op_kv4_row_bytes.argtypes = [i]
        lib.lpp_op_kv4_row_bytes.restype = i64
        lib.lpp_op_kv4_write.argtypes = [vp, vp, vp, vp, vp, i, i, i, i64, i, i64, i64, i, vp]
        lib.lpp_op_kv4_read.argtypes = [vp, vp, vp, vp, vp, i, i, i, i64, i, i64, i64, i, vp]
        lib.lpp_op_kv4_attention_scratch_bytes.argtypes = [i, i, i, i64, i, i]
        lib.lpp_op_kv4_attention_scratch_bytes.restype = i64
        lib.lpp_op_kv4_attention.argtypes = [vp, i64, vp, vp, vp, vp, vp, vp, vp, f, i, i, i, i64, i, i64, i64, i, vp]
        lib.lpp_op_call.argtypes = [i, C.c_char_p, i, vp]
        lib.lpp_op_kv4_evict.argtypes = [vp, vp, vp, vp, vp, vp, vp, vp, vp, i, i, i64, i64, i, i, i, vp]
        lib._ops_bound = True
    _bound = lib
    return lib


def cuda_convert_f32_to_f16(dst, src, n):
    _check(_lib().lpp_op_convert_f32_to_f16(_p(dst), _p(src), int(n), _s()), "cuda_convert_f32_to_f16")


def cuda_gemv(d_out, d_x, d_w, n, d, precision):
    """out[n] = w[n,d] . x[d]; ``precision`` is WEIGHT_FP32 / WEIGHT_FP16.  No workspace argument: x is never
    rounded to FP16 (the reference needs one for that, src/matmul.cu:136-141)."""
    _check(_lib().lpp_op_gemv(_p(d_out), _p(d_x), _p(d_w), int(n), int(d), LPP_F16 if precision == WEIGHT_FP16 else LPP_F32,
                              _s()), "cuda_gemv")


def cuda_rmsnorm(d_out, d_x, d_w, n):
    _check(_lib().lpp_op_rmsnorm(_p(d_out), _p(d_x), _p(d_w), int(n), _s()), "cuda_rmsnorm")


def cuda_rope(d_q, d_k, pos, dim, kv_dim, head_size, rope_base):
    _check(_lib().lpp_op_rope(_p(d_q), _p(d_k), int(pos), int(dim), int(kv_dim), int(head_size), float(rope_base), _s()),
           "cuda_rope")


def cuda_swiglu(d_hb, d_h1, d_h3, size):
    _check(_lib().lpp_op_swiglu(_p(d_hb), _p(d_h1), _p(d_h3), int(size), _s()), "cuda_swiglu")


def cuda_softmax_multihead(d_out, d_x, n_heads, seq_len, att_stride):
    _check(_lib().lpp_op_softmax_multihead(_p(d_out), _p(d_x), int(n_heads), int(seq_len), int(att_stride), _s()),
           "cuda_softmax_multihead")


def cuda_scale_multihead(d_att, scale, n_heads, seq_len, att_stride):
    _check(_lib().lpp_op_scale_multihead(_p(d_att), float(scale), int(n_heads), int(seq_len), int(att_stride), _s()),
           "cuda_scale_multihead")


def cuda_aggregation_multihead(d_out, d_v, d_att, n_heads, seq_len, head_size, gqa_factor, att_stride):
    _check(_lib().lpp_op_aggregation_multihead(_p(d_out), _p(d_v), _p(d_att), int(n_heads), int(seq_len), int(head_size),
                                               int(gqa_factor), int(att_stride), _s()), "cuda_aggregation_multihead")


def cuda_residual_add(d_out, d_a, d_b, n):
    _check(_lib().lpp_op_residual_add(_p(d_out), _p(d_a), _p(d_b), int(n), _s()), "cuda_residual_add")


def cuda_scatter_kv(d_key_cache, d_value_cache, d_k, d_v, layer, pos, n_kv_heads, head_size, seq_len):
    _check(_lib().lpp_op_scatter_kv(_p(d_key_cache), _p(d_value_cache), _p(d_k), _p(d_v), int(layer), int(pos),
                                    int(n_kv_heads), int(head_size), int(seq_len), _s()), "cuda_scatter_kv")


def cuda_multihead_gemv(d_out, d_q, d_k_cache, layer, pos, n_heads, n_kv_heads, head_size, seq_len):
    _check(_lib().lpp_op_multihead_gemv(_p(d_out), _p(d_q), _p(d_k_cache), int(layer), int(pos), int(n_heads),
                                        int(n_kv_heads), int(head_size), int(seq_len), _s()), "cuda_multihead_gemv")


def cuda_rope_scatter(d_q, d_k, d_v, d_key_cache, d_value_cache, layer, pos, dim, n_kv_heads, head_size, seq_len,
                      rope_base):
    _check(_lib().lpp_op_rope_scatter(_p(d_q), _p(d_k), _p(d_v), _p(d_key_cache), _p(d_value_cache), int(layer),
                                      int(pos), int(dim), int(n_kv_heads), int(head_size), int(seq_len),
                                      float(rope_base), _s()), "cuda_rope_scatter")


def cuda_sample(d_logits, vocab_size, temperature, penalty, d_history, history_len, r, d_sampled_token):
    """``r`` is passed in (the reference wrapper draws it from rand(), src/sample.cu:211)."""
    lib = _lib()
    hp = _p(d_history) if d_history is not None and history_len > 0 else C.c_void_p(None)
    logits, token = _p(d_logits), _p(d_sampled_token)
    n = lib.lpp_op_sample_scratch_bytes(int(vocab_size))
    # torch's allocator hands blocks on in stream order, so the scratch may be let go as soon as the work is queued
    scratch = torch.empty(max(n, 1), dtype=torch.uint8, device=d_logits.device)
    _check(lib.lpp_op_sample_on(_p(scratch), n, logits, int(vocab_size), float(temperature), float(penalty), hp, int(history_len),
                                float(r), token, _s()), "cuda_sample")


# ---- operators beyond the reference's: sizes come from the tensors, work is queued on the current stream of their device.  One
# sequence's (or token's) heads lie behind one another; from one to the next there may be a gap (a view of a wider tensor).
#
# A small call takes the GPU less time than the host: checks look at every tensor once, and arguments travel as one block.  (With a device
# guard around every call, sizes asked of the library each time, shapes compared as tuples and 18 arguments through ctypes a call took 22 -
# 26 us of host time; now 7.5 - 11.5.)

_DTYPES = {torch.float32: LPP_F32, torch.float16: LPP_F16, torch.bfloat16: LPP_BF16}
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda device: torch.cuda.current_stream(device).cuda_stream)


# (number of the operator, its arguments as 64-bit words: pointers, integers, a factor) as lpp_op_call takes them
_PROMPT_ATTENTION, _KV4_WRITE, _KV4_READ, _KV4_ATTENTION, _KV4_EVICT = ((i, struct.Struct(f)) for i, f in enumerate(("=5Q9qdq", "=5Q8q", "=5Q8q", "=Qq7Qd8q", "=9Q7q")))


def _call(what, entry, device, *args):
    """Queues the call on the current stream of ``device``."""
    op, words = entry
    lib = _bound or _bind()
    if torch.cuda.current_device() == device:
        st = lib.lpp_op_call(op, words.pack(*args), words.size >> 3, _raw_stream(device))
    else:
        with torch.cuda.device(device):
            st = lib.lpp_op_call(op, words.pack(*args), words.size >> 3, _raw_stream(device))
    if st:
        _check(st, what)


def _no_device(what):
    raise ValueError(f"{what}: expected CUDA tensors on one device")


def _want(what, t, dtype, *shape):
    if t.dtype is not dtype or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{what}: expected a contiguous {dtype} tensor of shape {shape}, got {t.dtype} {tuple(t.shape)}")


def _heads(what, t, dtype, shape):
    """Elements from one token of ``t`` [tokens, heads, head_size] to the next."""
    if t.dtype is dtype and t.shape == shape and t.is_contiguous() and len(shape) == 3:
        return shape[1] * shape[2]
    if t.dtype is not dtype or t.shape != shape or len(shape) != 3:
        raise ValueError(f"{what}: got {t.dtype} {tuple(t.shape)}, expected {dtype} [tokens, heads, head_size]" + (f" = {tuple(shape)}" if t.shape != shape else ""))
    tokens, heads, size = shape
    if (size > 1 and t.stride(2) != 1) or (heads > 1 and t.stride(1) != size):
        raise ValueError(f"{what}: the heads of a token lie behind one another")
    return t.stride(0) if tokens > 1 else heads * size


def _type(what, t):
    dtype = _DTYPES.get(t.dtype)
    if dtype is None:
        raise ValueError(f"{what}: {t.dtype} is none of F32, F16 and BF16")
    return dtype


def _ptr(t):
    return t.data_ptr() if t is not None else 0


def _cache(what, k, v, head_size):
    """(batch, kv heads, capacity) of a 4-bit cache."""
    shape = k.shape
    row = kv4_row_bytes(head_size)
    if len(shape) != 4 or shape[3] != row or v.shape != shape or k.dtype is not torch.uint8 or v.dtype is not torch.uint8 or not k.is_contiguous() or not v.is_contiguous():
        raise ValueError(f"{what}: a 4-bit cache is two contiguous [batch, kv heads, capacity, {row}] tensors of bytes, got {tuple(shape)} and {tuple(v.shape)}")
    return shape[:3]


def cuda_prompt_attention(d_out, d_q, d_k, d_v, d_offsets, scale):
    """Causal attention of packed prompts: ``d_q``, ``d_out`` [tokens, heads, head_size], ``d_k``, ``d_v`` [tokens, kv heads, head_size] (F16
    or BF16); ``d_offsets`` (int32, prompts + 1) has the first token of each prompt and the end of the last.  Tokens behind are left as they were."""
    what = "cuda_prompt_attention"
    device = d_q.get_device()
    if not 0 <= device == d_out.get_device() == d_k.get_device() == d_v.get_device() == d_offsets.get_device():
        _no_device(what)
    dtype, shape, kv_shape = d_q.dtype, d_q.shape, d_k.shape
    qs, outs = _heads(what, d_q, dtype, shape), _heads(what, d_out, dtype, shape)
    ks, vs = _heads(what, d_k, dtype, kv_shape), _heads(what, d_v, dtype, kv_shape)
    n, heads, size = shape
    if kv_shape[0] != n or kv_shape[2] != size or d_offsets.dim() != 1 or d_offsets.shape[0] < 1:
        raise ValueError(f"{what}: as many keys as queries, of one head size, and offsets of prompts + 1")
    prompts = d_offsets.shape[0] - 1
    _want(what, d_offsets, torch.int32, prompts + 1)
    _call(what, _PROMPT_ATTENTION, device, d_out.data_ptr(), d_q.data_ptr(), d_k.data_ptr(), d_v.data_ptr(), d_offsets.data_ptr(), prompts, n, heads, kv_shape[1],
          size, outs, qs, ks, vs, float(scale), _type(what, d_q))


@functools.lru_cache(maxsize=None)
def kv4_row_bytes(head_size):
    """Bytes of a row of the 4-bit cache: ``torch.zeros(batch, kv_heads, capacity, kv4_row_bytes(head_size), dtype=torch.uint8)`` is one."""
    n = _lib().lpp_op_kv4_row_bytes(int(head_size))
    if n < 0:
        raise ValueError("head sizes are 1 to 256")
    return n


def _kv4_rows(what, entry, first, second, k, v, caches, slots):
    device = k.get_device()
    if not 0 <= device == v.get_device() == slots.get_device() == caches[0].get_device() == caches[1].get_device():
        _no_device(what)
    shape = k.shape
    ks, vs = _heads(what, k, k.dtype, shape), _heads(what, v, k.dtype, shape)
    n, heads, size = shape
    batch, kv, capacity = _cache(what, *caches, size)
    _want(what, slots, torch.int64, n)
    if heads != kv:
        raise ValueError(f"{what}: the cache has another number of heads")
    _call(what, entry, device, first[0].data_ptr(), first[1].data_ptr(), second[0].data_ptr(), second[1].data_ptr(), slots.data_ptr(), n, batch, kv, capacity, size, ks, vs,
          _type(what, k))


def cuda_kv4_write(d_k_cache, d_v_cache, d_k, d_v, d_slots):
    """Rows ``d_k``, ``d_v`` [tokens, kv heads, head_size] into the 4-bit cache at ``d_slots`` (int64; sequence * capacity + position,
    all different; a token whose slot is negative, or beyond the cache, is left out)."""
    caches, rows = (d_k_cache, d_v_cache), (d_k, d_v)
    _kv4_rows("cuda_kv4_write", _KV4_WRITE, caches, rows, d_k, d_v, caches, d_slots)


def cuda_kv4_read(d_k, d_v, d_k_cache, d_v_cache, d_slots):
    """The values that the cache holds at ``d_slots``, rounded to the type of ``d_k`` (F16 has infinities from 65520 on, which rows written from
    numbers near 65504 may reach); a token whose slot is negative, or beyond the cache, is left as it was."""
    caches, rows = (d_k_cache, d_v_cache), (d_k, d_v)
    _kv4_rows("cuda_kv4_read", _KV4_READ, rows, caches, d_k, d_v, caches, d_slots)


@functools.lru_cache(maxsize=256)  # (a host whose capacities keep changing does not gather them all)
def _kv4_scratch_bytes(device, *sizes):
    with torch.cuda.device(device):
        return _lib().lpp_op_kv4_attention_scratch_bytes(*sizes)


def cuda_kv4_attention(d_out, d_q, d_k_cache, d_v_cache, d_lens, scale, d_sums_in=None, d_sums_out=None):
    """Attention of one token per sequence, ``d_q`` [batch, heads, head_size], over the first ``d_lens`` (int32) positions of the 4-bit
    cache.  ``d_sums_out`` [batch, kv heads, capacity] (FP32) = ``d_sums_in`` (None: zeros) + the softmax summed over a key/value head's queries."""
    what = "cuda_kv4_attention"
    device = d_q.get_device()
    if not 0 <= device == d_out.get_device() == d_k_cache.get_device() == d_v_cache.get_device() == d_lens.get_device():
        _no_device(what)
    dtype, shape = d_q.dtype, d_q.shape
    qs, outs = _heads(what, d_q, dtype, shape), _heads(what, d_out, dtype, shape)
    n, heads, size = shape
    batch, kv, capacity = _cache(what, d_k_cache, d_v_cache, size)
    _want(what, d_lens, torch.int32, n)
    if batch != n:
        raise ValueError(f"{what}: one query token per sequence of the cache")
    for sums in (d_sums_in, d_sums_out):
        if sums is not None:
            if sums.get_device() != device:
                _no_device(what)
            _want(what, sums, torch.float32, batch, kv, capacity)
    room = _kv4_scratch_bytes(device, batch, heads, kv, capacity, size, d_sums_out is not None)
    # torch's allocator hands blocks on in stream order, so the scratch may be let go as soon as the work is queued
    scratch = torch.empty(room, dtype=torch.uint8, device=d_q.device) if room > 0 else None
    _call(what, _KV4_ATTENTION, device, _ptr(scratch), room, d_out.data_ptr(), d_q.data_ptr(), d_k_cache.data_ptr(), d_v_cache.data_ptr(), d_lens.data_ptr(),
          _ptr(d_sums_in), _ptr(d_sums_out), float(scale), batch, heads, kv, capacity, size, outs, qs, _type(what, d_q))


_KV4_SIZES = {}  # row bytes -> a head size that has them


def cuda_kv4_evict(d_k_out, d_v_out, d_sums_out, d_kept, d_lens_out, d_k_cache, d_v_cache, d_sums, d_lens, keep, recent):
    """Moves ``keep`` rows of every head into a shorter cache: the ``recent`` last ones and those with the largest ``d_sums``.  ``d_kept``
    [batch, kv heads, keep] (int32) gets their old positions, ``d_lens_out`` (int32) the new lengths."""
    what, keep, recent = "cuda_kv4_evict", int(keep), int(recent)
    device = d_k_cache.get_device()
    if not 0 <= device == d_v_cache.get_device() == d_k_out.get_device() == d_v_out.get_device() == d_sums_out.get_device() == d_kept.get_device() \
            == d_lens_out.get_device() == d_sums.get_device() == d_lens.get_device():
        _no_device(what)
    if not _KV4_SIZES:
        _KV4_SIZES.update((kv4_row_bytes(s), s) for s in (32, 64, 96, 128, 256))
    size = _KV4_SIZES.get(d_k_cache.shape[-1], 0)  # (rows are moved whole)
    if not size:
        raise ValueError(f"{what}: no head has rows of {d_k_cache.shape[-1]} bytes")
    batch, kv, capacity = _cache(what, d_k_cache, d_v_cache, size)
    batch_out, kv_out, capacity_out = _cache(what, d_k_out, d_v_out, size)
    if batch_out != batch or kv_out != kv:
        raise ValueError(f"{what}: the new cache has other sequences or heads")
    _want(what, d_sums, torch.float32, batch, kv, capacity)
    _want(what, d_sums_out, torch.float32, batch, kv, capacity_out)
    _want(what, d_kept, torch.int32, batch, kv, keep)
    _want(what, d_lens, torch.int32, batch)
    _want(what, d_lens_out, torch.int32, batch)
    _call(what, _KV4_EVICT, device, d_k_out.data_ptr(), d_v_out.data_ptr(), d_sums_out.data_ptr(), d_kept.data_ptr(), d_lens_out.data_ptr(), d_k_cache.data_ptr(),
          d_v_cache.data_ptr(), d_sums.data_ptr(), d_lens.data_ptr(), batch, kv, capacity, capacity_out, size, keep, recent)
