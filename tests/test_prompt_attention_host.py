"""Attention of packed prompts without a GPU: arguments that are refused before anything is launched."""
import pytest

from lighterpp_b200 import engine as E, ops

P = 1 << 20  # stands for a pointer: never followed by a call that is refused
OK = dict(out=P, q=2 * P, k=3 * P, v=4 * P, off=5 * P, seqs=2, tokens=10, heads=4, kv=2, size=64, os=256, qs=256, ks=128, vs=128, scale=0.1, dtype=1)


def call(**kw):
    a = {**OK, **kw}
    return ops._lib().lpp_op_prompt_attention(*(a[x] for x in OK), None)


@pytest.mark.parametrize("wrong", [dict(out=0), dict(q=0), dict(k=0), dict(v=0), dict(off=0), dict(out=P + 8), dict(q=P + 2), dict(k=P + 4), dict(v=P + 1), dict(off=P + 2),
                                   dict(seqs=-1), dict(tokens=-1), dict(tokens=(1 << 30) + 1), dict(heads=0), dict(heads=5), dict(kv=0), dict(kv=3), dict(size=0), dict(size=12),
                                   dict(size=136, os=1 << 12, qs=1 << 12, ks=1 << 12, vs=1 << 12), dict(os=255), dict(qs=260), dict(ks=120), dict(vs=0), dict(scale=0.0), dict(scale=-0.5),
                                   dict(scale=float("nan")), dict(scale=float("inf")), dict(dtype=0), dict(dtype=3), dict(ks=1 << 33)])
def test_refused(wrong):
    assert call(**wrong) == 1
    assert E.load_library().lpp_last_error()


def test_nothing_to_do():
    assert call(seqs=0) == 0 and call(tokens=0, q=0, k=0, v=0, out=0) == 0


def test_tensors_that_do_not_fit_are_refused():
    import torch
    q = torch.zeros(4, 4, 64, dtype=torch.float16)
    with pytest.raises(ValueError):  # of the host
        ops.cuda_prompt_attention(torch.zeros_like(q), q, q, q, torch.zeros(2, dtype=torch.int32), 0.1)


@pytest.mark.parametrize("scale", [3e38, 2.4e38])
def test_a_scale_beyond_fp32_in_base_2_is_refused(scale):
    """scale * log2(e) would be infinite, and masked scores no numbers."""
    assert call(scale=scale) == 1
    assert b"scale" in E.load_library().lpp_last_error()
