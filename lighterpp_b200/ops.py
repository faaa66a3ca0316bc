"""The reference's per-operator host wrappers (src/kernels.cuh:24-36) over the C ABI, for torch CUDA tensors.

Same names and argument meaning as the reference; tensors stand in for raw device pointers.  Work is
queued on torch's current stream; nothing here synchronises.  There is no CPU path.
"""
from __future__ import annotations

import ctypes as C

import torch

from .engine import LPP_BF16, LPP_F16, LPP_F32, _check, load_library

WEIGHT_FP32, WEIGHT_FP16 = 0, 1  # src/model.h:8-12


def _p(t: torch.Tensor) -> C.c_void_p:
    if not t.is_cuda or not t.is_contiguous():
        raise ValueError("expected a contiguous CUDA tensor")
    return C.c_void_p(t.data_ptr())


def _s() -> C.c_void_p:
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _lib():
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
        lib.lpp_op_kv4_evict.argtypes = [vp, vp, vp, vp, vp, vp, vp, vp, vp, i, i, i64, i64, i, i, i, vp]
        lib._ops_bound = True
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

_DTYPES = {torch.float32: LPP_F32, torch.float16: LPP_F16, torch.bfloat16: LPP_BF16}


def _same_device(*tensors):
    first = tensors[0]
    for t in tensors:
        if t is not None and (not t.is_cuda or t.device != first.device):
            raise ValueError("expected CUDA tensors on one device")
    return torch.cuda.device(first.device)


def _want(what, t, dtype, shape):
    if t.dtype != dtype or tuple(t.shape) != tuple(shape) or not t.is_contiguous():
        raise ValueError(f"{what}: expected a contiguous {dtype} tensor of shape {tuple(shape)}, got {t.dtype} {tuple(t.shape)}")


def _heads(what, t, dtype=None, shape=None):
    """Elements from one token of ``t`` [tokens, heads, head_size] to the next."""
    if t.dim() != 3 or t.dtype not in _DTYPES or (dtype is not None and t.dtype != dtype) or (shape is not None and tuple(t.shape) != tuple(shape)):
        raise ValueError(f"{what}: got {t.dtype} {tuple(t.shape)}" + (f", expected {dtype} {tuple(shape)}" if shape is not None else ""))
    if t.numel() and ((t.shape[2] > 1 and t.stride(2) != 1) or (t.shape[1] > 1 and t.stride(1) != t.shape[2])):
        raise ValueError(f"{what}: the heads of a token lie behind one another")
    dense = t.shape[1] * t.shape[2]
    return t.stride(0) if t.shape[0] > 1 else dense


def _raw(t):
    return C.c_void_p(t.data_ptr() if t is not None else None)


def _cache(what, k, v, head_size):
    """(batch, kv heads, capacity) of a 4-bit cache."""
    row = kv4_row_bytes(head_size)
    if k.dim() != 4:
        raise ValueError(f"{what}: a 4-bit cache is [batch, kv heads, capacity, {row}] bytes")
    _want(what, k, torch.uint8, tuple(k.shape[:3]) + (row,))
    _want(what, v, torch.uint8, k.shape)
    return k.shape[:3]


def cuda_prompt_attention(d_out, d_q, d_k, d_v, d_offsets, scale):
    """Causal attention of packed prompts: ``d_q``, ``d_out`` [tokens, heads, head_size], ``d_k``, ``d_v`` [tokens, kv heads, head_size] (F16
    or BF16); ``d_offsets`` (int32, prompts + 1) has the first token of each prompt and the end of the last.  Tokens behind are left as they were."""
    with _same_device(d_q, d_out, d_k, d_v, d_offsets):
        qs = _heads("cuda_prompt_attention", d_q)
        outs = _heads("cuda_prompt_attention", d_out, d_q.dtype, d_q.shape)
        ks = _heads("cuda_prompt_attention", d_k, d_q.dtype)
        vs = _heads("cuda_prompt_attention", d_v, d_q.dtype, d_k.shape)
        if d_k.shape[0] != d_q.shape[0] or d_k.shape[2] != d_q.shape[2] or d_offsets.dim() != 1 or d_offsets.shape[0] < 1:
            raise ValueError("cuda_prompt_attention: as many keys as queries, of one head size, and offsets of prompts + 1")
        _want("cuda_prompt_attention", d_offsets, torch.int32, d_offsets.shape)
        _check(_lib().lpp_op_prompt_attention(_raw(d_out), _raw(d_q), _raw(d_k), _raw(d_v), _raw(d_offsets), d_offsets.shape[0] - 1, d_q.shape[0], d_q.shape[1], d_k.shape[1],
                                              d_q.shape[2], outs, qs, ks, vs, float(scale), _DTYPES[d_q.dtype], _s()), "cuda_prompt_attention")


def kv4_row_bytes(head_size):
    """Bytes of a row of the 4-bit cache: ``torch.zeros(batch, kv_heads, capacity, kv4_row_bytes(head_size), dtype=torch.uint8)`` is one."""
    n = _lib().lpp_op_kv4_row_bytes(int(head_size))
    if n < 0:
        raise ValueError("head sizes are 1 to 256")
    return n


def cuda_kv4_write(d_k_cache, d_v_cache, d_k, d_v, d_slots):
    """Rows ``d_k``, ``d_v`` [tokens, kv heads, head_size] into the 4-bit cache at ``d_slots`` (int64; sequence * capacity + position,
    all different; a token whose slot is negative, or beyond the cache, is left out)."""
    with _same_device(d_k_cache, d_v_cache, d_k, d_v, d_slots):
        ks = _heads("cuda_kv4_write", d_k)
        vs = _heads("cuda_kv4_write", d_v, d_k.dtype, d_k.shape)
        b, kv, cap = _cache("cuda_kv4_write", d_k_cache, d_v_cache, d_k.shape[2])
        _want("cuda_kv4_write", d_slots, torch.int64, d_k.shape[:1])
        if d_k.shape[1] != kv:
            raise ValueError("cuda_kv4_write: the cache has another number of heads")
        _check(_lib().lpp_op_kv4_write(_raw(d_k_cache), _raw(d_v_cache), _raw(d_k), _raw(d_v), _raw(d_slots), d_k.shape[0], b, kv, cap, d_k.shape[2], ks, vs,
                                       _DTYPES[d_k.dtype], _s()), "cuda_kv4_write")


def cuda_kv4_read(d_k, d_v, d_k_cache, d_v_cache, d_slots):
    """The values that the cache holds at ``d_slots``; a token whose slot is negative, or beyond the cache, is left as it was."""
    with _same_device(d_k_cache, d_v_cache, d_k, d_v, d_slots):
        ks = _heads("cuda_kv4_read", d_k)
        vs = _heads("cuda_kv4_read", d_v, d_k.dtype, d_k.shape)
        b, kv, cap = _cache("cuda_kv4_read", d_k_cache, d_v_cache, d_k.shape[2])
        _want("cuda_kv4_read", d_slots, torch.int64, d_k.shape[:1])
        if d_k.shape[1] != kv:
            raise ValueError("cuda_kv4_read: the cache has another number of heads")
        _check(_lib().lpp_op_kv4_read(_raw(d_k), _raw(d_v), _raw(d_k_cache), _raw(d_v_cache), _raw(d_slots), d_k.shape[0], b, kv, cap, d_k.shape[2], ks, vs,
                                      _DTYPES[d_k.dtype], _s()), "cuda_kv4_read")


def cuda_kv4_attention(d_out, d_q, d_k_cache, d_v_cache, d_lens, scale, d_sums_in=None, d_sums_out=None):
    """Attention of one token per sequence, ``d_q`` [batch, heads, head_size], over the first ``d_lens`` (int32) positions of the 4-bit
    cache.  ``d_sums_out`` [batch, kv heads, capacity] (FP32) = ``d_sums_in`` (None: zeros) + the softmax summed over a key/value head's queries."""
    with _same_device(d_q, d_out, d_k_cache, d_v_cache, d_lens, d_sums_in, d_sums_out):
        qs = _heads("cuda_kv4_attention", d_q)
        outs = _heads("cuda_kv4_attention", d_out, d_q.dtype, d_q.shape)
        n, heads, size = d_q.shape
        b, kv, cap = _cache("cuda_kv4_attention", d_k_cache, d_v_cache, size)
        _want("cuda_kv4_attention", d_lens, torch.int32, (n,))
        if b != n:
            raise ValueError("cuda_kv4_attention: one query token per sequence of the cache")
        for t in (d_sums_in, d_sums_out):
            if t is not None:
                _want("cuda_kv4_attention", t, torch.float32, (b, kv, cap))
        lib = _lib()
        bytes_ = lib.lpp_op_kv4_attention_scratch_bytes(b, heads, kv, cap, size, d_sums_out is not None)
        # torch's allocator hands blocks on in stream order, so the scratch may be let go as soon as the work is queued
        scratch = torch.empty(max(bytes_, 1), dtype=torch.uint8, device=d_q.device)
        _check(lib.lpp_op_kv4_attention(_raw(scratch), bytes_, _raw(d_out), _raw(d_q), _raw(d_k_cache), _raw(d_v_cache), _raw(d_lens), _raw(d_sums_in), _raw(d_sums_out),
                                        float(scale), b, heads, kv, cap, size, outs, qs, _DTYPES[d_q.dtype], _s()), "cuda_kv4_attention")


def cuda_kv4_evict(d_k_out, d_v_out, d_sums_out, d_kept, d_lens_out, d_k_cache, d_v_cache, d_sums, d_lens, keep, recent):
    """Moves ``keep`` rows of every head into a shorter cache: the ``recent`` last ones and those with the largest ``d_sums``.  ``d_kept``
    [batch, kv heads, keep] (int32) gets their old positions, ``d_lens_out`` (int32) the new lengths."""
    with _same_device(d_k_cache, d_v_cache, d_k_out, d_v_out, d_sums_out, d_kept, d_lens_out, d_sums, d_lens):
        lib = _lib()
        if d_k_cache.dim() != 4 or d_k_out.dim() != 4:
            raise ValueError("cuda_kv4_evict: a 4-bit cache is [batch, kv heads, capacity, row] bytes")
        b, kv, cap, row = d_k_cache.shape
        size = next((s for s in (32, 64, 96, 128, 256) if lib.lpp_op_kv4_row_bytes(s) == row), 0)  # (rows are moved whole)
        cap_out = d_k_out.shape[2]
        for t, shape in ((d_k_cache, (b, kv, cap, row)), (d_v_cache, (b, kv, cap, row)), (d_k_out, (b, kv, cap_out, row)), (d_v_out, (b, kv, cap_out, row))):
            _want("cuda_kv4_evict", t, torch.uint8, shape)
        _want("cuda_kv4_evict", d_sums, torch.float32, (b, kv, cap))
        _want("cuda_kv4_evict", d_sums_out, torch.float32, (b, kv, cap_out))
        _want("cuda_kv4_evict", d_kept, torch.int32, (b, kv, int(keep)))
        _want("cuda_kv4_evict", d_lens, torch.int32, (b,))
        _want("cuda_kv4_evict", d_lens_out, torch.int32, (b,))
        _check(lib.lpp_op_kv4_evict(_raw(d_k_out), _raw(d_v_out), _raw(d_sums_out), _raw(d_kept), _raw(d_lens_out), _raw(d_k_cache), _raw(d_v_cache), _raw(d_sums),
                                    _raw(d_lens), b, kv, cap, cap_out, size, int(keep), int(recent), _s()), "cuda_kv4_evict")
