"""FP32 steps over a 4-bit cache whose groups of 32 dimensions differ in size: every group is as exact as FP32 has it, not only the row's
largest one.  Bounds go group by group, with no term of another group's size."""
import numpy as np
import pytest

import kv4_util as U

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def T():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch


def attention(q, k_rows, v_rows, n, scale):
    """Results [heads, size] of one sequence, the sums of the softmax, and bounds of the error of either, in 64 bits.

    u = 2^-24.  A score is a sum of `size` products with codes, scales and zeros, off by at most (size + 16) u of the sum of the magnitudes (a
    query as two FP16 numbers is off by 4 u of itself, or 2^-31 of the largest one of its group, whose magnitude counts 16 times a scale).  A
    probability is off by that twice, by the exponent's rounding and the exponential; it meets a scale in FP32 (u) and a zero in FP32 (u).
    Sums over positions: 2 u for each tile of 16 positions behind another in a warp (one in 128 positions), 64 for warps and runs."""
    heads, size = q.shape
    kv = k_rows.shape[0]
    gqa, u = heads // kv, 2.0 ** -24
    out, bound = np.zeros((heads, size)), np.zeros((heads, size))
    sums, sums_bound = np.zeros((kv, n)), np.zeros((kv, n))
    for h in range(kv):
        k, ks, kz = U.unpack(k_rows[h, :n], size)
        v, _, vz = U.unpack(v_rows[h, :n], size)
        qh = q[h * gqa:(h + 1) * gqa]
        x = qh @ k.T * scale
        dx = (size + 16) * u * (np.abs(qh) @ (16 * ks + np.abs(kz)).T) * scale
        p = np.exp(x - x.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        dp = dx + (np.abs(x) + np.abs(x).max(-1, keepdims=True) + 8) * 2 * u
        dp = np.expm1(dp + (dp * p).sum(-1, keepdims=True)) + (2 * (n / 128) + 64) * 2 * u
        out[h * gqa:(h + 1) * gqa] = p @ v
        bound[h * gqa:(h + 1) * gqa] = (p * (dp + 2 * u)) @ (np.abs(v - vz) + np.abs(vz))
        sums[h], sums_bound[h] = p.sum(0), (p * dp).sum(0)
    return out, bound + u * (np.abs(out) + bound), sums, sums_bound + u * sums


def run(T, q, k, v, n, scale):
    from lighterpp_b200 import ops
    heads, size = q.shape
    kv, cap = k.shape[:2]
    out, sums = T.zeros((1, heads, size), device="cuda"), T.zeros((1, kv, cap), device="cuda")
    ops.cuda_kv4_attention(out, T.from_numpy(q.astype(np.float32))[None].cuda(), T.from_numpy(k)[None].cuda(), T.from_numpy(v)[None].cuda(),
                           T.tensor([n], dtype=T.int32, device="cuda"), scale, None, sums)
    want, bound, want_sums, sums_bound = attention(q, k, v, n, scale)
    off = np.abs(out[0].double().cpu().numpy() - want) / bound
    assert np.all(off <= 1), [float(off[:, g * 32:(g + 1) * 32].max()) for g in range(-(-size // 32))]
    off = np.abs(sums[0, :, :n].double().cpu().numpy() - want_sums) / sums_bound
    assert np.all(off <= 1), float(off.max())


def sizes_of(groups, size, first, last):
    """A factor for every dimension: powers of two from one group to the next, 2^first at one end and 2^last at the other."""
    return np.exp2(np.rint(np.linspace(first, last, groups)))[np.arange(size) // 32]


# either side of what counts as a short cache, every number of groups that is held
SHAPES = [(8, 2, 128, 900, 1000), (8, 2, 128, 3000, 4000), (4, 4, 64, 640, 700), (4, 1, 64, 5000, 5000), (3, 3, 96, 500, 520), (9, 1, 96, 3000, 3000), (4, 2, 256, 700, 704),
          (2, 1, 160, 2700, 2720)]


@pytest.mark.parametrize("heads,kv,size,n,cap", SHAPES)
@pytest.mark.parametrize("first,last", [(12, 2), (-8, 6), (13, -7), (-11, 13)])
def test_values_of_different_size(T, heads, kv, size, n, cap, first, last):
    rng = np.random.default_rng(size + n)
    groups = -(-size // 32)
    k = U.pack(rng.standard_normal((kv, cap, size)).astype(np.float32).astype(np.float64))
    v = U.pack((rng.standard_normal((kv, cap, size)) * sizes_of(groups, size, first, last)).astype(np.float32).astype(np.float64))
    q = rng.standard_normal((heads, size)).astype(np.float32).astype(np.float64)
    run(T, q, k, v, n, size ** -0.5)


@pytest.mark.parametrize("heads,kv,size,n,cap", SHAPES)
@pytest.mark.parametrize("first,last", [(8, -8), (-10, 12)])
def test_keys_of_different_size(T, heads, kv, size, n, cap, first, last):
    """Queries make up for it: all groups have a part in the scores."""
    rng = np.random.default_rng(size + n + 1)
    each = sizes_of(-(-size // 32), size, first, last)
    k = U.pack((rng.standard_normal((kv, cap, size)) * each).astype(np.float32).astype(np.float64))
    v = U.pack(rng.standard_normal((kv, cap, size)).astype(np.float32).astype(np.float64))
    q = (rng.standard_normal((heads, size)) / each).astype(np.float32).astype(np.float64)
    run(T, q, k, v, n, size ** -0.5)


def test_groups_without_a_part(T):
    """Groups of queries that are 0, keys that are alike, values that are 0, in every place."""
    rng = np.random.default_rng(5)
    for none in range(4):
        gone = np.where(np.arange(128) // 32 == none, 0.0, 1.0)
        k = U.pack((rng.standard_normal((2, 700, 128)) * np.roll(gone, 32) + 0.5).astype(np.float32).astype(np.float64))
        v = U.pack((rng.standard_normal((2, 700, 128)) * np.roll(gone, 64)).astype(np.float32).astype(np.float64))
        q = (rng.standard_normal((8, 128)) * gone).astype(np.float32).astype(np.float64)
        run_zero(T, q, k, v, 700, 0.09, np.roll(gone, 64) == 0)


def run_zero(T, q, k, v, n, scale, zero):
    from lighterpp_b200 import ops
    out = T.zeros((1,) + q.shape, device="cuda")
    ops.cuda_kv4_attention(out, T.from_numpy(q.astype(np.float32))[None].cuda(), T.from_numpy(k)[None].cuda(), T.from_numpy(v)[None].cuda(),
                           T.tensor([n], dtype=T.int32, device="cuda"), scale)
    want, bound, _, _ = attention(q, k, v, n, scale)
    got = out[0].double().cpu().numpy()
    assert np.all(np.abs(got - want) <= bound) and not got[:, zero].any()


@pytest.mark.parametrize("factor,first,last", [(1e30, 4, -4), (1e-30, 4, -4), (1e37, 0, 0), (1e-36, -3, 3)])
def test_queries_of_any_size_over_groups(T, factor, first, last):
    """As far as FP32 goes at either end, the scale undoing it."""
    rng = np.random.default_rng(6)
    each = sizes_of(2, 64, first, last)
    k = U.pack((rng.standard_normal((1, 336, 64)) * each).astype(np.float32).astype(np.float64))
    v = U.pack(rng.standard_normal((1, 336, 64)).astype(np.float32).astype(np.float64))
    q = (rng.uniform(-1, 1, (4, 64)) / each * (factor / 16)).astype(np.float32).astype(np.float64)
    scale = float(np.float32(1 / factor))
    run(T, q, k, v, 333, scale)
