"""Attention of packed prompts on the GPU against the formula in 64 bits, within bounds counted from the roundings: probabilities
and results are rounded to the type, scores and sums are FP32 sums of exact products."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def T():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch


def dtype(T, name):
    return {"f16": T.float16, "bf16": T.bfloat16}[name]


def reference(T, q, k, v, lengths, scale):
    """Results and error bounds of the tokens of all prompts (on the GPU, 64 bits).

    Half a step of the type for a probability and for the result (2^-11, 2^-8); a score of `size` products: (size + 8) 2^-23 of the sum
    of magnitudes, tensor cores truncating; twice that and 2^-21 for a probability; sums over n positions: n / 16 steps of 2^-23 in tensor
    memory and n / 2 of 2^-24 for the denominator; FP16 probabilities below the normal range are off by 2^-31 of the largest one."""
    heads, kv, size = q.shape[1], k.shape[1], q.shape[2]
    half = 2.0 ** (-11 if q.dtype == T.float16 else -8)
    n_all = sum(lengths)
    out, bound = (T.zeros((n_all, heads, size), dtype=T.float64, device="cuda") for _ in range(2))
    at = 0
    for n in lengths:
        for h in range(heads if n else 0):
            Q, K, V = (x[at:at + n, i].double() for x, i in ((q, h), (k, h // (heads // kv)), (v, h // (heads // kv))))
            x = Q @ K.T * scale
            hidden = T.full_like(x, float("-inf")).triu(1)
            dx = (size + 8) * 2.0 ** -23 * (Q.abs() @ K.T.abs()) * scale + x.abs() * 2.0 ** -22
            x = x + hidden
            p = T.softmax(x, -1)
            dx = dx + 2.0 ** -21
            dp = T.expm1(dx + (dx * p).sum(-1, keepdim=True)) + (n / 16 + 8) * 2.0 ** -23 + (n / 2 + 8) * 2.0 ** -24 + half
            out[at:at + n, h] = p @ V
            bound[at:at + n, h] = (p * dp) @ V.abs() + n * 2.0 ** -31 * V.abs().amax()
        at += n
    return out, bound + half * (out.abs() + bound) + 2.0 ** -25


def inputs(T, tokens, heads, kv, size, name, seed, keys=1.0, vals=1.0):
    g = T.Generator(device="cuda").manual_seed(seed)
    dt = dtype(T, name)
    return ((T.randn((tokens, heads, size), device="cuda", generator=g) * keys).to(dt), T.randn((tokens, kv, size), device="cuda", generator=g).to(dt),
            (T.randn((tokens, kv, size), device="cuda", generator=g) * vals).to(dt))


def offsets(T, lengths):
    return T.tensor([0] + list(np.cumsum(lengths)), dtype=T.int32, device="cuda")


def close(T, got, want, bound):
    off = (got.double() - want).abs() - bound
    assert bool((off <= 0).all()), (float(off.max()), (off > 0).nonzero()[:4].tolist(), int((off > 0).sum()))


@pytest.mark.parametrize("name", ["f16", "bf16"])
@pytest.mark.parametrize("lengths,heads,kv,size,behind", [
    ((1,), 2, 2, 64, 0), ((1,), 4, 1, 128, 3), ((201,), 6, 6, 48, 0), ((127, 1, 128, 0, 129), 8, 2, 64, 5), ((255, 256, 257), 4, 2, 128, 0), ((1000,), 8, 1, 128, 0),
    ((3, 0, 0, 5, 1, 1, 2), 4, 2, 64, 200), ((640,), 3, 1, 72, 0), ((300, 77), 9, 3, 8, 1), ((50,) * 30, 4, 4, 96, 0), ((384,), 2, 1, 128, 0), ((2000, 33), 2, 1, 64, 7),
    ((0, 0), 2, 1, 64, 4), ((1,) * 300, 2, 1, 16, 0), ((4100,), 2, 1, 128, 0)])
def test_prompts(T, name, lengths, heads, kv, size, behind):
    from lighterpp_b200 import ops
    n = sum(lengths)
    q, k, v = inputs(T, n + behind, heads, kv, size, name, n + size)
    q[n:], k[n:], v[n:] = float("nan"), float("inf"), float("nan")  # not looked at
    out = T.full_like(q, 9.0)
    ops.cuda_prompt_attention(out, q, k, v, offsets(T, lengths), size ** -0.5)
    want, bound = reference(T, q[:n], k[:n], v[:n], lengths, size ** -0.5)
    close(T, out[:n], want, bound)
    assert bool((out[n:] == 9.0).all())


def test_more_prompts_than_shared_memory_holds_offsets(T):
    from lighterpp_b200 import ops
    rng = np.random.default_rng(0)
    lengths = tuple(int(x) for x in rng.integers(0, 4, 1500)) + (300, 0, 5)
    n = sum(lengths)
    q, k, v = inputs(T, n + 3, 2, 1, 64, "f16", 2)
    out = T.full_like(q, 9.0)
    ops.cuda_prompt_attention(out, q, k, v, offsets(T, lengths), 0.125)
    want, bound = reference(T, q[:n], k[:n], v[:n], lengths, 0.125)
    close(T, out[:n], want, bound)
    assert bool((out[n:] == 9.0).all())


@pytest.mark.parametrize("name", ["f16", "bf16"])
def test_views_of_wider_tensors(T, name):
    """Queries, keys and values as one projection leaves them, results between other columns."""
    from lighterpp_b200 import ops
    heads, kv, size, n = 8, 2, 64, 333
    wide = T.randn((n, (heads + 2 * kv) * size + 8), device="cuda").to(dtype(T, name))
    q, k, v = (wide[:, a * size:b * size].unflatten(1, (-1, size)) for a, b in ((0, heads), (heads, heads + kv), (heads + kv, heads + 2 * kv)))
    room = T.full((n, heads * size + 24), 5.0, device="cuda", dtype=wide.dtype)
    out = room[:, 8:8 + heads * size].unflatten(1, (heads, size))
    ops.cuda_prompt_attention(out, q, k, v, offsets(T, (100, 233)), 0.125)
    want, bound = reference(T, q, k, v, (100, 233), 0.125)
    close(T, out, want, bound)
    assert bool((room[:, :8] == 5.0).all()) and bool((room[:, 8 + heads * size:] == 5.0).all())


@pytest.mark.parametrize("name", ["f16", "bf16"])
@pytest.mark.parametrize("keys,vals", [(30.0, 1.0), (0.0, 1.0), (1e-3, 100.0), (200.0, 0.01)])
def test_scores_of_odd_sizes(T, name, keys, vals):
    """One key that wins, all alike, maxima that keep growing along the sequence."""
    from lighterpp_b200 import ops
    q, k, v = inputs(T, 700, 4, 2, 64, name, 3, keys, vals)
    k[:, :, 0] += T.linspace(0, 8, 700, device="cuda")[:, None].to(k.dtype)
    q[:, :, 0] = q[:, :, 0].abs()
    out = T.zeros_like(q)
    ops.cuda_prompt_attention(out, q, k, v, offsets(T, (700,)), 0.125)
    want, bound = reference(T, q, k, v, (700,), 0.125)
    close(T, out, want, bound)


def test_a_sum_of_equal_values_is_that_value(T):
    """No drift along a long row: every result is the one value that all positions have."""
    from lighterpp_b200 import ops
    q, k, v = inputs(T, 5000, 2, 1, 128, "f16", 1)
    v[:] = 1.5
    out = T.zeros_like(q)
    ops.cuda_prompt_attention(out, q, k, v, offsets(T, (5000,)), 0.09)
    # truncating sums: n / 16 steps of 2^-23 and the probabilities' roundings, which do not add up to more than half a step
    assert float((out.float() - 1.5).abs().max()) <= 1.5 * (2.0 ** -11 + 5000 / 16 * 2.0 ** -23 + 2.0 ** -11)


@pytest.mark.parametrize("name", ["f16", "bf16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("heads,kv,size", [(4, 2, 64), (3, 3, 128)])
def test_what_is_not_finite_reaches_those_that_see_it_and_nobody_else(T, name, bad, heads, kv, size):
    from lighterpp_b200 import ops
    lengths = (150, 200, 130)
    q, k, v = inputs(T, 480, heads, kv, size, name, 5)
    clean = T.zeros_like(q)
    ops.cuda_prompt_attention(clean, q, k, v, offsets(T, lengths), 0.1)
    seen = T.zeros((480, heads), dtype=T.bool, device="cuda")
    vb, kb = v.clone(), k.clone()
    for token in (40, 149, 160, 349, 479):
        end = 150 if token < 150 else 350 if token < 350 else 480
        seen[token:end, 0:heads // kv] = True  # key/value head 0
        vb[token, 0, 3] = bad
    out = T.zeros_like(q)
    ops.cuda_prompt_attention(out, q, k, vb, offsets(T, lengths), 0.1)
    assert bool((~T.isfinite(out[..., 3]) == seen).all())
    if bad != bad or bad > 0:
        assert bool((T.isnan(out[..., 3]) == (seen if bad != bad else T.zeros_like(seen))).all())
    keep = T.ones(size, dtype=T.bool, device="cuda")
    keep[3] = False
    assert T.equal(out[:, :, keep], clean[:, :, keep])
    assert T.equal(out[..., 3][~seen], clean[..., 3][~seen])
    if bad != bad:  # a key that is not a number: every row that sees it
        for token in (40, 349):
            kb[token, 0, 0] = bad
        out = T.zeros_like(q)
        ops.cuda_prompt_attention(out, q, kb, v, offsets(T, lengths), 0.1)
        seen = T.zeros((480, heads), dtype=T.bool, device="cuda")
        seen[40:150, 0:heads // kv] = True
        seen[349:350, 0:heads // kv] = True
        assert bool((T.isnan(out).all(-1) == seen).all()) and T.equal(out[~seen], clean[~seen])


def test_the_same_bits_whatever_lies_around(T):
    """A prompt's results do not depend on its neighbours beyond how key tiles are cut; the same call gives the same bits."""
    from lighterpp_b200 import ops
    q, k, v = inputs(T, 900, 8, 2, 128, "bf16", 8)
    outs = []
    for _ in range(3):
        out = T.zeros_like(q)
        ops.cuda_prompt_attention(out, q, k, v, offsets(T, (450, 450)), 0.09)
        outs.append(out)
    assert all(T.equal(outs[0], o) for o in outs[1:])
    alone = T.zeros_like(q[:450])
    ops.cuda_prompt_attention(alone, q[:450], k[:450], v[:450], offsets(T, (450,)), 0.09)
    assert T.equal(alone, outs[0][:450])


def test_captured_and_replayed_with_other_offsets(T):
    from lighterpp_b200 import ops
    q, k, v = inputs(T, 600, 4, 2, 64, "f16", 4)
    off, out = offsets(T, (600, 0, 0)), T.zeros_like(q)
    side = T.cuda.Stream()
    side.wait_stream(T.cuda.current_stream())
    with T.cuda.stream(side):
        ops.cuda_prompt_attention(out, q, k, v, off, 0.125)
    T.cuda.current_stream().wait_stream(side)
    graph = T.cuda.CUDAGraph()
    with T.cuda.graph(graph):
        ops.cuda_prompt_attention(out, q, k, v, off, 0.125)
    for lengths in ((600, 0, 0), (1, 300, 299), (10, 20, 30), (0, 0, 0)):
        off.copy_(offsets(T, lengths))
        out.fill_(3.0)
        graph.replay()
        n = sum(lengths)
        want, bound = reference(T, q[:n], k[:n], v[:n], lengths, 0.125)
        close(T, out[:n], want, bound)
        assert bool((out[n:] == 3.0).all())


def test_prompts_into_the_cache_and_on(T):
    """Prompts, their rows into the 4-bit cache, and a decoded token behind each: the step over the cache is near the same attention over
    the rows that the cache was given (as near as 4 bits are), and the prompts' own results do not come from the cache."""
    from lighterpp_b200 import ops
    lengths, heads, kv, size, cap = (150, 33, 260), 8, 2, 64, 264
    n = sum(lengths)
    q, k, v = inputs(T, n, heads, kv, size, "f16", 12)
    out = T.zeros_like(q)
    ops.cuda_prompt_attention(out, q, k, v, offsets(T, lengths), 0.125)
    want, bound = reference(T, q, k, v, lengths, 0.125)
    close(T, out, want, bound)
    kc, vc = (T.zeros((3, kv, cap, ops.kv4_row_bytes(size)), dtype=T.uint8, device="cuda") for _ in range(2))
    slots = T.cat([b * cap + T.arange(m, device="cuda") for b, m in enumerate(lengths)])
    ops.cuda_kv4_write(kc, vc, k, v, slots)
    kb, vb = T.zeros_like(k), T.zeros_like(v)
    ops.cuda_kv4_read(kb, vb, kc, vc, slots)
    last = [sum(lengths[:b + 1]) - 1 for b in range(3)]
    got = T.zeros((3, heads, size), device="cuda", dtype=T.float16)
    ops.cuda_kv4_attention(got, q[last].contiguous(), kc, vc, T.tensor(lengths, dtype=T.int32, device="cuda"), 0.125)
    # the prompt's last row over the cache's own values (rounded to FP16 once more on the way out: half a step of a key and of a value)
    want, bound = reference(T, q, kb, vb, lengths, 0.125)
    for b, i in enumerate(last):
        for h in range(heads):
            first = i + 1 - lengths[b]
            K, V = kb[first:i + 1, h // 4].double(), vb[first:i + 1, h // 4].double()
            dx = 2.0 ** -11 * (q[i, h].double().abs() @ K.T.abs()) * 0.125
            p = T.softmax(q[i, h].double() @ K.T * 0.125, -1)
            more = (p * T.expm1(2 * dx)) @ V.abs() + 2.0 ** -11 * (p @ V.abs())
            assert bool(((got[b, h].double() - want[i, h]).abs() <= bound[i, h] + 2 * more + 2.0 ** -10 * (p @ V.abs())).all())


def test_strides_beyond_32_bits(T):
    """Tokens 64 MB apart: the same bits as from tensors without gaps, a value that is not a number among them."""
    from lighterpp_b200 import ops
    if T.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("needs 30 GB")
    n, heads, kv, size, apart = 130, 4, 2, 64, 1 << 25
    q, k, v = inputs(T, n, heads, kv, size, "f16", 5)
    v[100, 1, 7] = float("nan")
    want = T.zeros_like(q)
    ops.cuda_prompt_attention(want, q, k, v, offsets(T, (129, 1)), 0.125)
    room = T.empty(n * apart, dtype=T.float16, device="cuda")

    def place(at, x):
        view = room.as_strided(x.shape, (apart, size, 1), at)
        return view.copy_(x)

    views = [place(0, T.zeros_like(q)), place(256, q), place(512, k), place(640, v)]
    ops.cuda_prompt_attention(*views, offsets(T, (129, 1)), 0.125)
    assert T.equal(views[0].contiguous().view(T.int16), want.view(T.int16))
    assert bool(want[100:129, 2:, 7].isnan().all()) and int(want.isnan().sum()) == 29 * 2


@pytest.mark.parametrize("name", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv,size", [(4, 2, 64), (3, 3, 128), (4, 2, 128), (2, 1, 40)])
@pytest.mark.parametrize("before", [0, 1, 77, 128])
def test_values_that_are_infinite_whatever_their_weight(T, name, heads, kv, size, before):
    """An infinite value whose weight has become 0 in the type, and what becomes of it, do not go by where key tiles are cut: results are
    infinite wherever the prompt lies, not numbers where both signs are seen, and those of other dimensions as without."""
    from lighterpp_b200 import ops
    n = 700
    q, k, v = inputs(T, before + n, heads, kv, size, name, 9)
    weak = [before + i for i in (0, 5, 126, 200, 399)]
    q[:, :, 0], k[:, :, 0] = 40.0, 0.0
    k[weak, :, 0] = -40.0  # their scores lie 288 powers of two below the others
    lengths = ((before, n) if before else (n,))
    clean = T.zeros_like(q)
    ops.cuda_prompt_attention(clean, q, k, v, offsets(T, lengths), 0.125)
    v[weak[1], 0, 3] = float("inf")
    v[weak[2], 0, 5] = float("-inf")
    v[weak[3], 0, 3] = float("-inf")
    v[weak[4], 0, 7] = float("nan")
    out = T.zeros_like(q)
    ops.cuda_prompt_attention(out, q, k, v, offsets(T, lengths), 0.125)
    want = clean.clone()
    g = heads // kv
    want[weak[1]:, :g, 3] = float("inf")
    want[weak[3]:, :g, 3] = float("nan")
    want[weak[2]:, :g, 5] = float("-inf")
    want[weak[4]:, :g, 7] = float("nan")
    same = (out == want) | (out.isnan() & want.isnan())
    assert bool(same.all()), (~same).nonzero()[:5].tolist()


@pytest.mark.parametrize("name", ["f16", "bf16"])
def test_values_near_the_largest(T, name):
    """Finite values near the type's largest: results are their weighted means, which no part on the way takes beyond FP32."""
    from lighterpp_b200 import ops
    q, k, v = inputs(T, 300, 2, 1, 64, name, 10)
    v[:] = 60000.0 if name == "f16" else 1e33
    out = T.zeros_like(q)
    ops.cuda_prompt_attention(out, q, k, v, offsets(T, (300,)), 0.125)
    want, bound = reference(T, q, k, v, (300,), 0.125)
    close(T, out, want, bound)
