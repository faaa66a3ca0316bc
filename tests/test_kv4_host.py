"""The 4-bit cache's entry points without a GPU: sizes, and arguments that are refused before anything is launched."""
import ctypes as C

import numpy as np
import pytest

import kv4_util as U
from lighterpp_b200 import engine as E, ops

P = 1 << 20  # stands for a pointer: never followed by a call that is refused
OK = dict(kc=P, vc=2 * P, k=3 * P, v=4 * P, slots=5 * P, n=2, batch=2, kv=2, cap=64, size=64, ks=128, vs=128, dtype=1)


def rows(fn, **kw):
    a = {**OK, **kw}
    if fn == "write":
        return ops._lib().lpp_op_kv4_write(a["kc"], a["vc"], a["k"], a["v"], a["slots"], a["n"], a["batch"], a["kv"], a["cap"], a["size"], a["ks"], a["vs"], a["dtype"], None)
    return ops._lib().lpp_op_kv4_read(a["k"], a["v"], a["kc"], a["vc"], a["slots"], a["n"], a["batch"], a["kv"], a["cap"], a["size"], a["ks"], a["vs"], a["dtype"], None)


@pytest.mark.parametrize("size", [1, 31, 32, 33, 48, 64, 96, 100, 128, 129, 224, 256])
def test_row_bytes(size):
    assert ops.kv4_row_bytes(size) == U.row_bytes(size)


@pytest.mark.parametrize("size", [0, -1, 257])
def test_row_bytes_of_no_head(size):
    with pytest.raises(ValueError):
        ops.kv4_row_bytes(size)


@pytest.mark.parametrize("fn", ["write", "read"])
@pytest.mark.parametrize("wrong", [dict(kc=0), dict(vc=0), dict(k=0), dict(v=0), dict(slots=0), dict(kc=P + 8), dict(vc=P + 4), dict(k=P + 1), dict(slots=P + 4), dict(n=-1),
                                   dict(batch=0), dict(kv=0), dict(cap=0), dict(cap=66), dict(cap=1 << 31), dict(size=0), dict(size=257), dict(ks=127), dict(vs=0),
                                   dict(dtype=3), dict(dtype=-1), dict(k=P + 2, dtype=0), dict(n=1 << 30, kv=4, ks=256, vs=256)])
def test_rows_refused(fn, wrong):
    assert rows(fn, **wrong) == 1
    assert E.load_library().lpp_last_error()


@pytest.mark.parametrize("fn", ["write", "read"])
def test_no_rows_is_no_work(fn):
    assert rows(fn, n=0, k=0, v=0, slots=0) == 0


ATT = dict(scratch=P, bytes=1 << 40, out=2 * P, q=3 * P, kc=4 * P, vc=5 * P, lens=6 * P, si=0, so=0, scale=0.1, batch=2, heads=8, kv=2, cap=64, size=64, os=512, qs=512, dtype=1)


def attention(**kw):
    a = {**ATT, **kw}
    return ops._lib().lpp_op_kv4_attention(*(a[x] for x in ("scratch", "bytes", "out", "q", "kc", "vc", "lens", "si", "so", "scale", "batch", "heads", "kv", "cap", "size", "os",
                                                             "qs", "dtype")), None)


@pytest.mark.parametrize("wrong", [dict(scratch=P + 128), dict(out=0), dict(q=0), dict(kc=0), dict(vc=0), dict(lens=0), dict(lens=P + 2), dict(so=P + 1),
                                   dict(si=P), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(heads=7), dict(heads=0), dict(kv=0),
                                   dict(batch=0), dict(cap=62), dict(size=300), dict(os=511), dict(qs=0), dict(dtype=7), dict(q=P + 1), dict(q=P + 2, dtype=0),
                                   dict(heads=4096, kv=2, size=1, os=4096, qs=4096)])
def test_attention_refused(wrong):
    assert attention(**wrong) == 1


def test_scratch_of_no_shape():
    f = ops._lib().lpp_op_kv4_attention_scratch_bytes
    assert f(0, 8, 2, 64, 64, 0) == -1 and f(1, 7, 2, 64, 64, 0) == -1 and f(1, 8, 2, 63, 64, 0) == -1 and f(1, 8, 2, 64, 0, 0) == -1


EV = dict(ko=P, vo=2 * P, so=3 * P, kept=4 * P, lo=5 * P, kc=6 * P, vc=7 * P, sums=8 * P, lens=9 * P, batch=1, kv=2, cap=64, capo=32, size=64, keep=20, recent=5)


def evict(**kw):
    a = {**EV, **kw}
    return ops._lib().lpp_op_kv4_evict(*(a[x] for x in ("ko", "vo", "so", "kept", "lo", "kc", "vc", "sums", "lens", "batch", "kv", "cap", "capo", "size", "keep", "recent")), None)


@pytest.mark.parametrize("wrong", [dict(ko=0), dict(vo=0), dict(so=0), dict(kept=0), dict(lo=0), dict(kc=0), dict(vc=0), dict(sums=0), dict(lens=0), dict(keep=0), dict(keep=33),
                                   dict(recent=-1), dict(recent=21), dict(capo=30), dict(cap=0), dict(size=0), dict(ko=6 * P), dict(vo=6 * P + 1600), dict(ko=7 * P), dict(vo=P),
                                   dict(so=8 * P), dict(lo=9 * P), dict(kept=P + 2), dict(ko=P + 8)])
def test_evict_refused(wrong):
    assert evict(**wrong) == 1


def test_arguments_as_words_are_the_same_call():
    """The block of words reaches the same refusals; a wrong number of words, or a number beyond 32 bits, is one."""
    lib = ops._lib()

    def words(entry, *args, n=None):
        op, fmt = entry
        return lib.lpp_op_call(op, fmt.pack(*args), fmt.size // 8 if n is None else n, None)

    rows_ok = (P, 2 * P, 3 * P, 4 * P, 5 * P, 2, 2, 2, 64, 64, 128, 128, 1)
    for i, bad in ((0, 0), (2, P + 1), (4, P + 4), (5, -1), (6, 0), (7, 0), (8, 66), (9, 257), (10, 127), (11, 0), (12, 3)):
        args = list(rows_ok)
        args[i] = bad
        assert words(ops._KV4_WRITE, *args) == 1
    assert words(ops._KV4_READ, P, 2 * P, 3 * P, 4 * P, 5 * P, 0, 2, 2, 64, 64, 128, 128, 1) == 0  # no rows
    assert words(ops._KV4_READ, P, 2 * P, 3 * P, 4 * P, 5 * P, 1 << 32, 2, 2, 64, 64, 128, 128, 1) == 1
    assert words(ops._KV4_WRITE, *rows_ok, n=12) == 1 and lib.lpp_op_call(5, b"", 0, None) == 1 and lib.lpp_op_call(-1, b"", 0, None) == 1
    attn = [P, 1 << 40, 2 * P, 3 * P, 4 * P, 5 * P, 6 * P, 0, 0, 0.1, 2, 8, 2, 64, 64, 512, 512, 1]
    for i, bad in ((0, P + 128), (2, 0), (6, P + 2), (7, P), (9, -1.0), (9, float("nan")), (11, 7), (13, 62), (14, 300), (15, 511), (17, 7), (17, 1 << 33)):
        args = list(attn)
        args[i] = bad
        assert words(ops._KV4_ATTENTION, *args) == 1
    ev = [P, 2 * P, 3 * P, 4 * P, 5 * P, 6 * P, 7 * P, 8 * P, 9 * P, 1, 2, 64, 32, 64, 20, 5]
    for i, bad in ((0, 6 * P), (3, 0), (11, 66), (12, 18), (13, 0), (14, 33), (15, 21)):
        args = list(ev)
        args[i] = bad
        assert words(ops._KV4_EVICT, *args) == 1
    prompt = [P, 2 * P, 3 * P, 4 * P, 5 * P, 2, 10, 4, 2, 64, 256, 256, 128, 128, 0.1, 1]
    for i, bad in ((0, 0), (5, -1), (7, 5), (9, 12), (10, 255), (13, 0), (14, 0.0), (15, 0)):
        args = list(prompt)
        args[i] = bad
        assert words(ops._PROMPT_ATTENTION, *args) == 1


def test_tensors_of_the_host_are_refused():
    import torch
    z = torch.zeros(1, 2, 64, 40, dtype=torch.uint8)
    with pytest.raises(ValueError):
        ops.cuda_kv4_write(z, z.clone(), torch.zeros(2, 2, 64), torch.zeros(2, 2, 64), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError):
        ops.cuda_kv4_attention(torch.zeros(1, 4, 64), torch.zeros(1, 4, 64), z, z.clone(), torch.zeros(1, dtype=torch.int32), 0.1)


def test_plain_rows_hold_what_the_text_says():
    """The statement itself: a group's ends and zero are held to half a step and the roundings of scale and zero."""
    rng = np.random.default_rng(2)
    x = rng.standard_normal((50, 48)) * rng.choice([1e-3, 1.0, 300.0], (50, 1))
    y, s, z = U.unpack(U.pack(x), 48)
    # half a step, or what lies beyond the last code: 7.5 steps of scale's rounding (2^-11) and zero's rounding
    assert np.all(np.abs(y - x) <= s * (0.5 + 16 * 2.0 ** -11) + np.abs(z) * 2.0 ** -11 + 2.0 ** -24)
    const = U.unpack(U.pack(np.full((1, 40), 0.25)), 40)[0]
    assert np.all(const == 0.25)


@pytest.mark.parametrize("scale", [3e38, 2.4e38])
def test_a_scale_beyond_fp32_in_base_2_is_refused(scale):
    """scale * log2(e) would be infinite, and the scores of zeros no numbers."""
    assert attention(scale=scale) == 1
    assert b"scale" in E.load_library().lpp_last_error()


@pytest.mark.parametrize("wrong", [dict(kept=8 * P), dict(kept=8 * P + 2 * 64 * 4 - 4), dict(kept=9 * P), dict(kept=6 * P), dict(kept=P + 4), dict(so=4 * P), dict(so=7 * P), dict(so=9 * P),
                                   dict(so=2 * P), dict(lo=4 * P + 8), dict(lo=8 * P), dict(lo=7 * P + 40), dict(lo=3 * P), dict(ko=8 * P), dict(vo=9 * P)])
def test_evict_into_what_it_reads_or_writes_elsewhere_is_refused(wrong):
    """Kept positions over the sums that are still being looked at would be counted one way and written another."""
    assert evict(**wrong) == 1


def test_evict_of_arrays_side_by_side_is_not_refused():
    """Arrays that touch do not overlap (the call gets as far as the device)."""
    if __import__("torch").cuda.is_available():
        pytest.skip("addresses that stand for pointers are not followed")
    assert evict(kept=8 * P + 2 * 64 * 4, lo=4 * P - 4, so=9 * P + 4) == 7  # no device here


def test_sizes_asked_for_are_not_gathered_without_end():
    assert 0 < ops._kv4_scratch_bytes.cache_info().maxsize < 10000
