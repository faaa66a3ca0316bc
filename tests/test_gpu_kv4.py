"""The cache held in 4 bits on the GPU against its statement in 64 bits (kv4_util): rows written are the statement's bytes, rows read
its values, attention within bounds counted from the roundings, eviction keeps the statement's rows."""
import numpy as np
import pytest

import kv4_util as U

pytestmark = pytest.mark.gpu
TYPES = ["f32", "f16", "bf16"]


@pytest.fixture(scope="module")
def T():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch


def dtype(T, name):
    return {"f32": T.float32, "f16": T.float16, "bf16": T.bfloat16}[name]


def half_step(name):
    return {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[name]


def values(T, shape, name, seed, kind="normal"):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal(shape).astype(np.float32)
    if kind == "wild":  # sizes of every kind, groups of one value, what has no place in the format
        x *= np.exp(rng.uniform(-18, 12, shape[:-1] + (1,))).astype(np.float32)
        x[::7] = x[::7, :, :1]
        x[3, 0, 0], x[4, 0, -1], x[5 % len(x), 0, 0] = np.inf, -np.inf, np.nan
        x[6 % len(x)] = 0.0
    return T.from_numpy(x).cuda().to(dtype(T, name))


def wide(T, x, gap):
    """The same values as a view of a wider tensor."""
    n, h, d = x.shape
    w = T.full((n, h * d + gap), 7.0, device="cuda", dtype=x.dtype)
    w[:, :h * d] = x.view(n, h * d)
    return w[:, :h * d].unflatten(1, (h, d))


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("size,kv,gap,kind", [(64, 2, 0, "normal"), (128, 8, 0, "wild"), (48, 6, 8, "normal"), (96, 1, 0, "wild"), (33, 3, 0, "normal"), (1, 2, 1, "normal"),
                                              (100, 2, 4, "wild"), (160, 1, 0, "normal"), (256, 2, 16, "wild"), (32, 5, 3, "normal")])
def test_rows(T, name, size, kv, gap, kind):
    from lighterpp_b200 import ops
    batch, cap, n = 3, 20, 37
    k, v = values(T, (n, kv, size), name, size, kind), values(T, (n, kv, size), name, size + 1)
    rng = np.random.default_rng(size)
    slots = rng.permutation(batch * cap)[:n].astype(np.int64)
    slots[[2, 9]] = [-1, batch * cap]  # left out
    shape = (batch, kv, cap, U.row_bytes(size))
    kc, vc = (T.full(shape, 0xa5, dtype=T.uint8, device="cuda") for _ in range(2))
    ds = T.from_numpy(slots).cuda()
    ops.cuda_kv4_write(kc, vc, wide(T, k, gap), v, ds)
    back = [wide(T, T.full_like(k, 3.0), gap), T.full_like(v, 3.0)]
    ops.cuda_kv4_read(back[0], back[1], kc, vc, ds)
    for cache, x, y in ((kc, k, back[0]), (vc, v, back[1])):
        want = np.full(shape, 0xa5, dtype=np.uint8)
        rows = U.pack(x.double().cpu().numpy())
        held = T.from_numpy(U.unpack(rows, size)[0]).float().to(x.dtype)
        for i, s in enumerate(slots):
            if 0 <= s < batch * cap:
                want[s // cap, :, s % cap] = rows[i]
            else:
                held[i] = 3.0
        got = cache.cpu().numpy()
        assert np.array_equal(got, want), np.argwhere(got != want)[:5]
        assert T.equal(y.cpu(), held)


def test_codes_next_to_a_border(T):
    """Values that lie on, just below and just above the middle between two codes."""
    from lighterpp_b200 import ops
    x = np.zeros((64, 1, 32), dtype=np.float32)
    rng = np.random.default_rng(0)
    for i in range(64):
        scale = np.float32(np.float16(rng.uniform(0.01, 3)))
        lo = np.float32(np.float16(rng.uniform(-5, 5)))
        mids = lo + scale * (np.arange(15, dtype=np.float32) + np.float32(0.5))
        x[i, 0, :15] = np.nextafter(mids, np.float32(rng.choice([-100, 100]))) if i % 3 else mids
        x[i, 0, 15:30] = np.nextafter(np.nextafter(mids, np.float32(-100)), np.float32(-100))
        x[i, 0, 30], x[i, 0, 31] = lo, lo + 15 * scale
    k = T.from_numpy(x).cuda()
    kc, vc = (T.zeros((1, 1, 64, 20), dtype=T.uint8, device="cuda") for _ in range(2))
    ops.cuda_kv4_write(kc, vc, k, k, T.arange(64, device="cuda"))
    assert np.array_equal(kc.cpu().numpy()[0, 0], U.pack(x.astype(np.float64))[:, 0])
    assert T.equal(kc, vc)


def setup(T, heads, kv, size, name, lens, cap, seed, keys=1.0, vals=0.5, garbage=True):
    rng = np.random.default_rng(seed)
    batch = len(lens)
    k = U.pack((rng.standard_normal((batch, kv, cap, size)) * keys).astype(np.float16).astype(np.float64))
    v = U.pack((rng.standard_normal((batch, kv, cap, size)) * vals).astype(np.float16).astype(np.float64))
    if garbage:  # rows behind the sequences: scales and zeros that are NaN
        for b, n in enumerate(lens):
            k[b, :, n:], v[b, :, n:] = 0xff, 0xff
    q = T.from_numpy(rng.standard_normal((batch, heads, size)).astype(np.float32)).cuda().to(dtype(T, name))
    return q, k, v


def check(T, q, k, v, lens, scale, name, with_sums=True, gap=0, call=None):
    from lighterpp_b200 import ops
    batch, heads, size = q.shape
    kv, cap = k.shape[1:3]
    out = T.full((batch, heads * size + gap), 9.0, device="cuda", dtype=q.dtype)
    o = out[:, :heads * size].unflatten(1, (heads, size))
    ref, bound, sums, sums_bound = U.attention(q.double().cpu().numpy(), k, v, lens, scale, name != "f32")
    s_in = T.rand((batch, kv, cap), device="cuda") if with_sums else None
    s_out = T.full((batch, kv, cap), -5.0, device="cuda") if with_sums else None
    args = (o, wide(T, q, gap) if gap else q, T.from_numpy(k).cuda(), T.from_numpy(v).cuda(), T.tensor(list(lens), dtype=T.int32, device="cuda"), scale, s_in, s_out)
    (call or ops.cuda_kv4_attention)(*args)
    got = o.double().cpu().numpy()
    bound = bound + half_step(name) * (np.abs(ref) + bound) + 2.0 ** -25
    assert np.all(np.abs(got - ref) <= bound), (np.abs(got - ref) - bound).max()
    assert np.all(out[:, heads * size:].float().cpu().numpy() == 9.0)
    if with_sums:
        got, want = s_out.double().cpu().numpy(), s_in.double().cpu().numpy() + sums
        for b, n in enumerate(lens):
            assert np.all(got[b, :, n:] == -5.0)
            assert np.all(np.abs(got[b, :, :n] - want[b, :, :n]) <= sums_bound[b, :, :n] + 2.0 ** -24 * want[b, :, :n])
    return o


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("heads,kv,size,lens,cap", [
    (8, 2, 64, (1, 0, 17, 128), 128), (32, 8, 128, (129, 1000), 1024), (6, 6, 48, (200,), 200), (3, 1, 32, (15, 16, 31), 32), (9, 1, 64, (300, 5), 300),
    (40, 2, 128, (257,), 260), (8, 8, 96, (127, 640, 64), 640), (4, 2, 33, (77,), 80), (2, 1, 256, (333, 2), 336), (12, 3, 160, (140,), 140), (1, 1, 1, (9,), 12),
    # caches that are not short: heads dealt out in runs
    (8, 2, 64, (2500, 0, 17, 1), 2600), (32, 8, 128, (4000,), 4096), (6, 6, 48, (2300, 100), 2304), (9, 1, 64, (2500, 5), 2560), (40, 2, 128, (2570,), 2600),
    (2, 1, 256, (2700,), 2720), (8, 4, 160, (2200, 2305), 2400), (1, 1, 1, (2100,), 2100), (16, 16, 96, (700, 1024, 3, 129), 2500)])
def test_attention(T, name, heads, kv, size, lens, cap):
    q, k, v = setup(T, heads, kv, size, name, lens, cap, heads + size)
    check(T, q, k, v, lens, size ** -0.5, name, with_sums=True, gap=5 if size == 48 else 0)


@pytest.mark.parametrize("name", TYPES)
def test_attention_without_sums(T, name):
    lens = (513, 4, 0, 2000, 1)
    q, k, v = setup(T, 16, 2, 128, name, lens, 2048, 5)
    check(T, q, k, v, lens, 0.09, name, with_sums=False)


@pytest.mark.parametrize("name", ["f32", "f16"])
def test_attention_over_many_sequences(T, name):
    """More sequences than lanes of a warp; most of the runs hold several heads."""
    rng = np.random.default_rng(1)
    for most in (200, 400):  # either side of what counts as short
        lens = tuple(int(x) for x in rng.integers(0, most, 75))
        q, k, v = setup(T, 8, 2, 64, name, lens, most, 6)
        check(T, q, k, v, lens, 0.125, name)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("keys,vals", [(40.0, 1.0), (1e-4, 1e-5), (1.0, 6e3), (300.0, 1e-6), (0.0, 1.0), (1.0, 0.0)])
def test_attention_of_odd_sizes_of_values(T, name, keys, vals):
    """Scores that let one position win, or all alike; values near either end of the FP16 range, or all the same."""
    lens = (700,)
    q, k, v = setup(T, 8, 2, 64, name, lens, 700, 8, keys, vals)
    check(T, q, k, v, lens, 0.125, name)


def test_probabilities_grow_along_the_sequence(T):
    """Every position weighs more than all before it, and its values are larger: the reference has to move again and again."""
    rng = np.random.default_rng(3)
    n, size = 1500, 32
    k = np.zeros((1, 1, 1500, size))
    k[0, 0, :, 0] = np.linspace(0, 60, n)
    v = rng.standard_normal((1, 1, n, size)) * np.exp(np.linspace(-10, 9, n))[None, None, :, None]
    q = T.zeros((1, 4, size), device="cuda")
    q[:, :, 0] = T.tensor([5.0, -5.0, 1.0, 0.01], device="cuda")
    check(T, q, U.pack(k), U.pack(v), (n,), 1.0, "f32")


@pytest.mark.parametrize("name,factor", [("f32", 1e30), ("f32", 1e-30), ("bf16", 1e30), ("f16", 6e4)])
def test_queries_of_any_size(T, name, factor):
    lens = (333,)
    q, k, v = setup(T, 4, 1, 64, name, lens, 336, 4)
    q = (q.float() / q.float().abs().max() * factor).to(q.dtype)
    check(T, q, k, v, lens, 1.0 / factor, name)


def test_queries_near_the_largest_value(T):
    """The factor that goes back from the operands to scores is beyond FP32 there."""
    lens = (333,)
    q, k, v = setup(T, 4, 1, 64, "bf16", lens, 336, 4)
    big = (q.float() / q.float().abs().max() * 3e38).to(q.dtype)
    check(T, big, k, v, lens, 1e-37, "bf16")
    k[0, :, :333] = U.pack(np.zeros((333, 64)))  # keys of 0: all positions alike
    check(T, big, k, v, lens, 0.125, "bf16")


def test_lengths_beyond_the_capacity_are_cut(T):
    q, k, v = setup(T, 4, 2, 64, "f16", (64, 64), 64, 1)
    from lighterpp_b200 import ops
    a, b = T.zeros_like(q), T.zeros_like(q)
    kc, vc = T.from_numpy(k).cuda(), T.from_numpy(v).cuda()
    ops.cuda_kv4_attention(a, q, kc, vc, T.tensor([64, 0], dtype=T.int32, device="cuda"), 0.1)
    ops.cuda_kv4_attention(b, q, kc, vc, T.tensor([1000, -3], dtype=T.int32, device="cuda"), 0.1)
    assert T.equal(a, b) and not b[1].any()


def test_sums_in_place_and_from_nothing(T):
    from lighterpp_b200 import ops
    lens = (900, 33)
    q, k, v = setup(T, 8, 2, 64, "f16", lens, 900, 2)
    kc, vc, dl = T.from_numpy(k).cuda(), T.from_numpy(v).cuda(), T.tensor(lens, dtype=T.int32, device="cuda")
    out, fresh = T.zeros_like(q), T.zeros((2, 2, 900), device="cuda")
    ops.cuda_kv4_attention(out, q, kc, vc, dl, 0.125, None, fresh)
    total = fresh.clone()
    ops.cuda_kv4_attention(out, q, kc, vc, dl, 0.125, total, total)
    assert T.equal(total, fresh + fresh)
    # a head's probabilities add up to 1 each: four query heads
    assert np.allclose(fresh[0].sum(-1).cpu(), 4.0, atol=900 * 2.0 ** -20)


def test_the_same_call_gives_the_same_bits(T):
    from lighterpp_b200 import ops
    lens = (5000, 1, 777)
    q, k, v = setup(T, 16, 2, 128, "f32", lens, 5000, 3)
    kc, vc, dl = T.from_numpy(k).cuda(), T.from_numpy(v).cuda(), T.tensor(lens, dtype=T.int32, device="cuda")
    got = []
    for _ in range(3):
        out, sums = T.zeros_like(q), T.zeros((3, 2, 5000), device="cuda")
        ops.cuda_kv4_attention(out, q, kc, vc, dl, 0.09, None, sums)
        got.append((out, sums))
    assert all(T.equal(got[0][0], o) and T.equal(got[0][1], s) for o, s in got[1:])


@pytest.mark.parametrize("cap", [640, 4000])
@pytest.mark.parametrize("scratch_fill", [0, 255])
def test_captured_replayed_and_on_another_stream(T, scratch_fill, cap):
    """One captured graph follows what lies in its inputs; scratch may hold anything."""
    from lighterpp_b200 import ops
    lib = ops._lib()
    q, k, v = setup(T, 8, 2, 64, "f16", (cap, cap), cap, 9, garbage=False)
    kc, vc, dl = T.from_numpy(k).cuda(), T.from_numpy(v).cuda(), T.tensor([cap, 0], dtype=T.int32, device="cuda")
    out, sums = T.zeros_like(q), T.zeros((2, 2, cap), device="cuda")
    n = lib.lpp_op_kv4_attention_scratch_bytes(2, 8, 2, cap, 64, 1)
    scratch = T.full((n,), scratch_fill, dtype=T.uint8, device="cuda")

    def call():
        st = lib.lpp_op_kv4_attention(ops._ptr(scratch), n, ops._ptr(out), ops._ptr(q), ops._ptr(kc), ops._ptr(vc), ops._ptr(dl), None, ops._ptr(sums), 0.125, 2, 8, 2, cap, 64,
                                      512, 512, 1, ops._s())
        assert st == 0

    T.cuda.synchronize()
    side = T.cuda.Stream()
    with T.cuda.stream(side):
        call()
    side.synchronize()
    graph = T.cuda.CUDAGraph()
    with T.cuda.graph(graph):
        call()
    for lens in ((3, cap), (cap, 129), (0, 0)):
        dl.copy_(T.tensor(lens, dtype=T.int32))
        q.copy_(T.randn_like(q))
        out.fill_(9.0)
        graph.replay()
        T.cuda.synchronize()
        got, got_sums = out.clone(), sums.clone()
        out.fill_(9.0)
        call()
        assert T.equal(out, got) and T.equal(sums, got_sums)
        ref, bound, _, _ = U.attention(q.double().cpu().numpy(), k, v, lens, 0.125, True)
        assert np.all(np.abs(got.double().cpu().numpy() - ref) <= bound + 2.0 ** -11 * (np.abs(ref) + bound) + 2.0 ** -25)


def test_scratch_that_is_too_small_is_refused(T):
    from lighterpp_b200 import ops
    lib = ops._lib()
    x = T.zeros(1 << 20, dtype=T.uint8, device="cuda")
    p = ops._ptr(x)

    def call(scratch, n, cap, sums):
        return lib.lpp_op_kv4_attention(scratch, n, p, p, p, p, p, None, p if sums else None, 0.1, 1, 8, 2, cap, 64, 512, 512, 1, ops._s())

    short, long = (lib.lpp_op_kv4_attention_scratch_bytes(1, 8, 2, cap, 64, 0) for cap in (640, 6400))
    assert short == 0 < long < lib.lpp_op_kv4_attention_scratch_bytes(1, 8, 2, 6400, 64, 1)
    assert call(p, long - 1, 6400, False) == 1 and call(p, long, 6400, True) == 1 and call(None, long, 6400, False) == 1
    n = lib.lpp_op_kv4_attention_scratch_bytes(1, 8, 2, 640, 64, 1)
    assert n >= 640 * 8 * 4 and call(p, n - 1, 640, True) == 1 and call(None, n, 640, True) == 1


def evict(T, size, kv, lens, cap, keep, recent, sums, cap_out=None, seed=0):
    from lighterpp_b200 import ops
    rng = np.random.default_rng(seed)
    batch, row = len(lens), U.row_bytes(size)
    cap_out = cap_out or -(-keep // 4) * 4
    k, v = (rng.integers(0, 256, (batch, kv, cap, row), dtype=np.uint8) for _ in range(2))
    ko, vo = (T.full((batch, kv, cap_out, row), 0x5a, dtype=T.uint8, device="cuda") for _ in range(2))
    so, kept = T.full((batch, kv, cap_out), -3.0, device="cuda"), T.full((batch, kv, keep), -7, dtype=T.int32, device="cuda")
    lo = T.full((batch,), -1, dtype=T.int32, device="cuda")
    ops.cuda_kv4_evict(ko, vo, so, kept, lo, T.from_numpy(k).cuda(), T.from_numpy(v).cuda(), T.from_numpy(sums).cuda(), T.tensor(list(lens), dtype=T.int32, device="cuda"), keep,
                       recent)
    ko, vo, so, kept, lo = (x.cpu().numpy() for x in (ko, vo, so, kept, lo))
    for b, n in enumerate(lens):
        assert lo[b] == min(n, keep)
        for h in range(kv):
            rows = U.keep_rows(sums[b, h], n, keep, recent)
            m = len(rows)
            assert list(kept[b, h, :m]) == rows, (b, h)
            assert np.all(kept[b, h, m:] == -7)
            assert np.array_equal(ko[b, h, :m], k[b, h, rows]) and np.all(ko[b, h, m:] == 0x5a)
            assert np.array_equal(vo[b, h, :m], v[b, h, rows]) and np.all(vo[b, h, m:] == 0x5a)
            assert np.array_equal(so[b, h, :m], sums[b, h, rows], equal_nan=True) and np.all(so[b, h, m:] == -3.0)


@pytest.mark.parametrize("size,kv,lens,cap,keep,recent", [
    (64, 2, (100, 40, 0, 1), 100, 40, 8), (128, 3, (2500,), 2500, 1000, 100), (48, 1, (1025, 1024, 1023), 1028, 1, 0), (96, 2, (333,), 336, 200, 200), (32, 2, (50, 9), 52, 8, 1),
    (256, 1, (700,), 700, 699, 1), (64, 1, (5000, 4999, 7), 5000, 4096, 0), (128, 1, (9,), 12, 9, 3)])
def test_evict(T, size, kv, lens, cap, keep, recent):
    sums = np.exp(2 * np.random.default_rng(cap).standard_normal((len(lens), kv, cap))).astype(np.float32)
    evict(T, size, kv, lens, cap, keep, recent, sums)


@pytest.mark.parametrize("size", [20, 64, 96, 128, 200])
@pytest.mark.parametrize("cap,keep,recent", [(600, 256, 20), (600, 257, 20), (2052, 1024, 0), (2052, 1025, 30)])
def test_evict_of_few_and_of_many_rows(T, size, cap, keep, recent):
    """Either side of what one kernel moves; sums that leave most of the rows to one end of the cache."""
    rng = np.random.default_rng(size + keep)
    sums = rng.random((1, 3, cap)).astype(np.float32)
    sums[0, 1] *= np.linspace(0, 1, cap) ** 4
    sums[0, 2] *= np.linspace(1, 0, cap) ** 4
    evict(T, size, 3, (cap - 1,), cap, keep, recent, sums)


@pytest.mark.parametrize("kind", ["equal", "few", "wild", "close"])
def test_evict_of_equal_and_odd_sums(T, kind):
    rng = np.random.default_rng(4)
    n, cap = 3001, 3004
    if kind == "equal":
        sums = np.full((1, 2, cap), 0.25, np.float32)
    elif kind == "few":
        sums = rng.choice(np.float32([0.0, -0.0, 0.5, 1.0]), (1, 2, cap))
    elif kind == "close":  # that differ in the last bits
        sums = (np.float32(1.0) + rng.integers(0, 9, (1, 2, cap)).astype(np.float32) * np.float32(2.0 ** -23)).astype(np.float32)
    else:
        sums = rng.choice(np.float32([np.inf, -np.inf, np.nan, 1e-45, -1e-45, 3e38, -1.0, 0.0, -0.0]), (1, 2, cap))
    for keep, recent in ((1500, 0), (1500, 700), (3000, 1), (1, 1)):
        evict(T, 64, 2, (n,), cap, keep, recent, sums, seed=keep)


def test_evict_captured_and_replayed(T):
    """The second kernel starts behind the first in a graph too, with other lengths and sums at every replay."""
    from lighterpp_b200 import ops
    rng = np.random.default_rng(7)
    cap, keep, recent, row = 3000, 700, 50, U.row_bytes(128)
    k = rng.integers(0, 256, (1, 4, cap, row), dtype=np.uint8)
    kc, sums, lens = T.from_numpy(k).cuda(), T.zeros((1, 4, cap), device="cuda"), T.zeros(1, dtype=T.int32, device="cuda")
    vc = kc.flip(-1).contiguous()
    ko, vo, so = T.zeros((1, 4, keep, row), dtype=T.uint8, device="cuda"), T.zeros((1, 4, keep, row), dtype=T.uint8, device="cuda"), T.zeros((1, 4, keep), device="cuda")
    kept, lo = T.zeros((1, 4, keep), dtype=T.int32, device="cuda"), T.zeros(1, dtype=T.int32, device="cuda")

    def call():
        ops.cuda_kv4_evict(ko, vo, so, kept, lo, kc, vc, sums, lens, keep, recent)

    side = T.cuda.Stream()
    side.wait_stream(T.cuda.current_stream())
    with T.cuda.stream(side):
        call()
    T.cuda.current_stream().wait_stream(side)
    graph = T.cuda.CUDAGraph()
    with T.cuda.graph(graph):
        call()
    for n in (3000, 701, 12, 2999):
        w = rng.random((1, 4, cap)).astype(np.float32)
        sums.copy_(T.from_numpy(w))
        lens.fill_(n)
        graph.replay()
        for h in range(4):
            rows = U.keep_rows(w[0, h], n, keep, recent)
            assert int(lo) == len(rows) and list(kept[0, h, :len(rows)].cpu().numpy()) == rows
            assert np.array_equal(ko[0, h, :len(rows)].cpu().numpy(), k[0, h, rows]) and np.array_equal(vo[0, h, :len(rows)].cpu().numpy(), k[0, h, rows][:, ::-1])


def test_evict_of_many_rows_captured_and_replayed(T):
    from lighterpp_b200 import ops
    rng = np.random.default_rng(8)
    cap, keep, row = 4096, 2100, U.row_bytes(64)
    k = rng.integers(0, 256, (1, 2, cap, row), dtype=np.uint8)
    kc, sums, lens = T.from_numpy(k).cuda(), T.zeros((1, 2, cap), device="cuda"), T.full((1,), cap, dtype=T.int32, device="cuda")
    ko, vo, so = T.zeros((1, 2, keep, row), dtype=T.uint8, device="cuda"), T.zeros((1, 2, keep, row), dtype=T.uint8, device="cuda"), T.zeros((1, 2, keep), device="cuda")
    kept, lo = T.zeros((1, 2, keep), dtype=T.int32, device="cuda"), T.zeros(1, dtype=T.int32, device="cuda")
    graph = T.cuda.CUDAGraph()
    ops.cuda_kv4_evict(ko, vo, so, kept, lo, kc, kc, sums, lens, keep, 3)
    with T.cuda.graph(graph):
        ops.cuda_kv4_evict(ko, vo, so, kept, lo, kc, kc, sums, lens, keep, 3)
    for n in (4096, 2101, 5):
        w = rng.random((1, 2, cap)).astype(np.float32)
        sums.copy_(T.from_numpy(w))
        lens.fill_(n)
        graph.replay()
        for h in range(2):
            rows = U.keep_rows(w[0, h], n, keep, 3)
            assert int(lo) == len(rows) and list(kept[0, h, :len(rows)].cpu().numpy()) == rows
            assert np.array_equal(ko[0, h, :len(rows)].cpu().numpy(), k[0, h, rows]) and T.equal(ko[0, h, :len(rows)], vo[0, h, :len(rows)])


def test_a_longer_cache_takes_everything(T):
    sums = np.random.default_rng(1).random((2, 2, 64)).astype(np.float32)
    evict(T, 64, 2, (64, 10), 64, 64, 10, sums, cap_out=128)


def test_prompt_steps_eviction_and_steps_behind_one_another(T):
    """As a host uses them: rows of a prompt and of every decoded token go in, steps add to the sums, the cache is cut, decoding goes on."""
    from lighterpp_b200 import ops
    rng = np.random.default_rng(11)
    batch, heads, kv, size, cap, keep, recent = 2, 8, 2, 64, 96, 40, 8
    lens = np.array([70, 33])
    row = U.row_bytes(size)
    kc, vc = (T.zeros((batch, kv, cap, row), dtype=T.uint8, device="cuda") for _ in range(2))
    ref = [np.zeros((batch, kv, cap, row), dtype=np.uint8) for _ in range(2)]
    sums, ref_sums, ref_bound = T.zeros((batch, kv, cap), device="cuda"), np.zeros((batch, kv, cap)), np.zeros((batch, kv, cap))

    def write(tokens, slots, cap):
        k, v = (T.from_numpy(rng.standard_normal((tokens, kv, size)).astype(np.float32)).cuda() for _ in range(2))
        ops.cuda_kv4_write(kc, vc, k, v, T.tensor(slots, device="cuda"))
        for r, x in zip(ref, (k, v)):
            rows = U.pack(x.double().cpu().numpy())
            for i, s in enumerate(slots):
                r[s // cap, :, s % cap] = rows[i]

    def step(cap):
        nonlocal lens, ref_sums, ref_bound
        write(batch, [int(b * cap + lens[b]) for b in range(batch)], cap)
        lens = lens + 1
        q = T.from_numpy(rng.standard_normal((batch, heads, size)).astype(np.float32)).cuda()
        out = T.zeros_like(q)
        ops.cuda_kv4_attention(out, q, kc, vc, T.tensor(lens, dtype=T.int32, device="cuda"), 0.125, sums, sums)
        want, bound, s, sb = U.attention(q.double().cpu().numpy(), ref[0], ref[1], lens, 0.125, False)
        assert np.all(np.abs(out.double().cpu().numpy() - want) <= bound + 2.0 ** -24 * (np.abs(want) + bound))
        ref_sums = ref_sums + s
        ref_bound = ref_bound + sb + 2.0 ** -24 * ref_sums

    write(103, [int(p) for p in range(70)] + [cap + p for p in range(33)], cap)
    for _ in range(12):
        step(cap)
    assert np.all(np.abs(sums.double().cpu().numpy() - ref_sums) <= ref_bound)
    ko, vo = (T.zeros((batch, kv, 64, row), dtype=T.uint8, device="cuda") for _ in range(2))
    so, kept, lo = T.zeros((batch, kv, 64), device="cuda"), T.zeros((batch, kv, keep), dtype=T.int32, device="cuda"), T.zeros(batch, dtype=T.int32, device="cuda")
    ops.cuda_kv4_evict(ko, vo, so, kept, lo, kc, vc, sums, T.tensor(lens, dtype=T.int32, device="cuda"), keep, recent)
    had = sums.cpu().numpy()
    new = [np.zeros((batch, kv, 64, row), dtype=np.uint8) for _ in range(2)]
    new_sums, new_bound = np.zeros((batch, kv, 64)), np.zeros((batch, kv, 64))
    for b in range(batch):
        for h in range(kv):
            rows = U.keep_rows(had[b, h], int(lens[b]), keep, recent)
            assert list(kept[b, h, :len(rows)].cpu().numpy()) == rows
            for r, x in zip(new, ref):
                r[b, h, :len(rows)] = x[b, h, rows]
            new_sums[b, h, :len(rows)], new_bound[b, h, :len(rows)] = ref_sums[b, h, rows], ref_bound[b, h, rows]
    kc, vc, sums, ref, ref_sums, ref_bound = ko, vo, so, new, new_sums, new_bound
    lens = np.minimum(lens, keep)
    assert np.array_equal(lo.cpu().numpy(), lens)
    for _ in range(5):
        step(64)
    assert np.all(np.abs(sums.double().cpu().numpy() - ref_sums) <= ref_bound)


def test_a_cache_beyond_32_bits(T):
    """A head's rows, scores and slots far behind the first 2^32 bytes, and more positions than an FP32 sum counts.  All rows are 0 but a few."""
    from lighterpp_b200 import ops
    if T.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB")
    rng = np.random.default_rng(12)
    heads, kv, size, cap, keep, scale = 8, 2, 128, 1 << 26, 64, 0.125
    n, some = cap - 4, np.array([0, 5, (1 << 25) + 1, cap - 100, cap - 5])
    kc, vc = (T.zeros((1, kv, cap, U.row_bytes(size)), dtype=T.uint8, device="cuda") for _ in range(2))
    q = T.from_numpy(rng.standard_normal((1, heads, size)).astype(np.float32)).cuda().half()
    q64 = q.double().cpu().numpy()[0].reshape(kv, heads // kv, size)
    k = q64.mean(1)[None] * rng.uniform(4, 6, (len(some), kv, 1))  # keys along a head's queries: scores that some 10^7 others do not hide
    k, v = (T.from_numpy(x.astype(np.float32)).cuda().half() for x in (k, rng.standard_normal((len(some), kv, size))))
    slots = T.from_numpy(some).cuda()
    ops.cuda_kv4_write(kc, vc, k, v, slots)
    k_rows, v_rows = (U.pack(x.double().cpu().numpy()) for x in (k, v))
    assert np.array_equal(kc[0][:, slots].transpose(0, 1).cpu().numpy(), k_rows) and np.array_equal(vc[0][:, slots].transpose(0, 1).cpu().numpy(), v_rows)
    assert T.count_nonzero(kc[0, 1, 1 << 25:]) <= 3 * U.row_bytes(size)
    back = T.zeros_like(k), T.zeros_like(v)
    ops.cuda_kv4_read(*back, kc, vc, slots)
    for x, rows in zip(back, (k_rows, v_rows)):
        assert np.array_equal(x.cpu().numpy(), U.unpack(rows, size)[0].astype(np.float16))
    out, sums = T.zeros_like(q), T.zeros((1, kv, cap), device="cuda")
    ops.cuda_kv4_attention(out, q, kc, vc, T.tensor([n], dtype=T.int32, device="cuda"), scale, sums, sums)
    u = 2.0 ** -24
    for h in range(kv):
        (kh, ks, kz), (vh, _, vz) = U.unpack(k_rows[:, h], size), U.unpack(v_rows[:, h], size)
        x = q64[h] @ kh.T * scale
        total = (n - len(some)) + np.exp(x).sum(-1, keepdims=True)
        p = np.exp(x) / total
        # a score's rounding as in kv4_util, that of its exponential and of the sum's members; sums of 3542 tiles in a lane (148 SMs, two CTAs each),
        # five lanes' steps, eight warps and at most 300 parts behind one another
        dp = 2 * ((size + 16) * u * (np.abs(q64[h]) @ (16 * ks + np.abs(kz)).T) * scale + (np.abs(x).max() + 8) * 2 * u) + 4000 * u
        want = p @ vh
        bound = (p * dp) @ (np.abs(vh - vz) + np.abs(vz)) + 2.0 ** -11 * (p @ np.abs(vh - vz))
        got = out[0, h * 4:h * 4 + 4].double().cpu().numpy()
        assert np.all(np.abs(got - want) <= bound + 2.0 ** -11 * (np.abs(want) + bound) + 2.0 ** -25)
        assert np.all(np.abs(sums[0, h, slots].double().cpu().numpy() - p.sum(0)) <= (p * dp).sum(0) + 8 * u * p.sum(0))
        other = (1 / total).sum()
        assert abs(float(sums[0, h, cap - 50]) - other) <= (dp.max() + 8 * u) * other
        assert not sums[0, h, n:].any()
    ko, vo = (T.zeros((1, kv, keep, U.row_bytes(size)), dtype=T.uint8, device="cuda") for _ in range(2))
    so, kept, lo = T.zeros((1, kv, keep), device="cuda"), T.zeros((1, kv, keep), dtype=T.int32, device="cuda"), T.zeros(1, dtype=T.int32, device="cuda")
    ops.cuda_kv4_evict(ko, vo, so, kept, lo, kc, vc, sums, T.tensor([n], dtype=T.int32, device="cuda"), keep, 1)
    first = sorted(set(range(62)) | {int(s) for s in some})  # all others weigh the same: the lowest positions stay
    first = [r for r in first if r in some or first.index(r) < 61][:61] + [int(s) for s in some[2:]]
    for h in range(kv):
        assert list(kept[0, h].cpu().numpy()) == first
        at = [first.index(int(s)) for s in some]
        assert np.array_equal(ko[0, h, at].cpu().numpy(), k_rows[:, h]) and np.array_equal(vo[0, h, at].cpu().numpy(), v_rows[:, h])


def test_two_streams_at_once(T):
    """Calls of either stream have scratch of their own."""
    from lighterpp_b200 import ops
    sets = []
    for seed, lens in ((1, (5000, 9, 2000)), (2, (17, 4097, 4999))):
        q, k, v = setup(T, 16, 2, 128, "f16", lens, 5000, seed)
        kc, vc, dl = T.from_numpy(k).cuda(), T.from_numpy(v).cuda(), T.tensor(lens, dtype=T.int32, device="cuda")
        out, sums = T.zeros_like(q), T.zeros((3, 2, 5000), device="cuda")
        ops.cuda_kv4_attention(out, q, kc, vc, dl, 0.09, None, sums)
        sets.append((q, kc, vc, dl, out, sums, T.cuda.Stream()))
    T.cuda.synchronize()
    got = []
    for _ in range(20):
        for q, kc, vc, dl, _, _, stream in sets:
            with T.cuda.stream(stream):
                out, sums = T.zeros_like(q), T.zeros((3, 2, 5000), device="cuda")
                ops.cuda_kv4_attention(out, q, kc, vc, dl, 0.09, None, sums)
                got.append((out, sums))
    T.cuda.synchronize()
    for i, (out, sums) in enumerate(got):
        assert T.equal(out, sets[i % 2][4]) and T.equal(sums, sets[i % 2][5])


def test_scale_and_zero_by_way_of_fp32(T):
    """Groups whose scale, or zero, is another FP16 number when the exact one is rounded without the step over FP32."""
    from lighterpp_b200 import ops
    rng = np.random.default_rng(1)
    lo, hi = -np.abs(rng.standard_normal(400000)).astype(np.float32) * 3, np.abs(rng.standard_normal(400000)).astype(np.float32) * 3
    lo[0], hi[0] = float.fromhex("-0x1.750b5ap+1"), float.fromhex("0x1.42314ap+0")
    exact = (hi.astype(np.float64) - lo.astype(np.float64)) / 15
    by_way = exact.astype(np.float32).astype(np.float16)
    zero = lo.astype(np.float64) + 8 * by_way.astype(np.float64)
    some = np.flatnonzero((exact.astype(np.float16) != by_way) | (zero.astype(np.float16) != zero.astype(np.float32).astype(np.float16)))
    assert 0 in some and len(some) > 10
    x = np.linspace(lo[some], hi[some], 32, axis=-1).astype(np.float32)
    x[:, 0], x[:, -1] = lo[some], hi[some]
    x = np.ascontiguousarray(np.clip(x, lo[some][:, None], hi[some][:, None])[:, None])
    n = len(some)
    cap = -(-n // 4) * 4
    kc, vc = (T.zeros((1, 1, cap, 20), dtype=T.uint8, device="cuda") for _ in range(2))
    xs = T.from_numpy(x).cuda()
    ops.cuda_kv4_write(kc, vc, xs, xs, T.arange(n, device="cuda"))
    assert np.array_equal(kc.cpu().numpy()[0, 0, :n], U.pack(x.astype(np.float64))[:, 0])


def test_held_values_beyond_fp16(T):
    """scale and zero are rounded, so a group that reaches +-65504 may stand for a little more: FP32 and BF16 get it as it is, FP16 rounded
    to what it has, an infinity from 65520 on."""
    from lighterpp_b200 import ops
    x = np.zeros((4, 1, 32), dtype=np.float32)
    x[0, 0, 0] = 65504
    x[1, 0, :2] = 65504, -65504
    x[2, 0, :2] = np.inf, -1
    x[3, 0, :2] = -np.inf, 60000
    rows = U.pack(x.astype(np.float64))
    held = U.unpack(rows, 32)[0]
    assert held[0, 0, 0] == 65520 and held[1, 0, 0] == 65536
    kc, vc = (T.zeros((1, 1, 4, 20), dtype=T.uint8, device="cuda") for _ in range(2))
    slots = T.arange(4, device="cuda")
    xs = T.from_numpy(x).cuda()
    ops.cuda_kv4_write(kc, vc, xs, xs, slots)
    assert np.array_equal(kc.cpu().numpy()[0, 0], rows[:, 0])
    for name in TYPES:
        k, v = (T.zeros((4, 1, 32), dtype=dtype(T, name), device="cuda") for _ in range(2))
        ops.cuda_kv4_read(k, v, kc, vc, slots)
        assert T.equal(k.cpu(), T.from_numpy(held.astype(np.float32)).to(k.dtype)) and T.equal(k, v)
        assert bool(k.isfinite().all()) == (name != "f16")
        out = T.zeros((1, 1, 32), dtype=dtype(T, name), device="cuda")
        ops.cuda_kv4_attention(out, T.zeros_like(out), kc, vc, T.tensor([1], dtype=T.int32, device="cuda"), 1.0)  # one position: its values
        assert T.equal(out[0, 0].cpu(), T.from_numpy(held[0, 0].astype(np.float32)).to(out.dtype))


@pytest.mark.parametrize("kind", ["random", "few"])
@pytest.mark.parametrize("batch,kv,n,cap,keeps", [(1, 1, 39999, 40000, (1, 2048, 2049, 20000)), (1, 2, 70001, 70004, (2000, 50000)), (10, 8, 5000, 5000, (256, 257, 4500)),
                                                  (40, 4, 4700, 4800, (100, 3000))])
def test_evict_of_more_rows_than_a_thread_holds(T, kind, batch, kv, n, cap, keeps):
    """More than 4096 rows a CTA: a cluster over one long head, and heads that get a CTA each."""
    rng = np.random.default_rng(cap + batch)
    if kind == "random":
        sums = rng.random((batch, kv, cap)).astype(np.float32)
        sums[..., ::3] *= np.linspace(0, 1, cap, dtype=np.float32)[::3]
    else:  # equals among what is kept and what goes, before and behind the rows that a thread holds
        sums = rng.choice(np.float32([0.25, 0.5, 0.5 + 2.0 ** -24, 1.0]), (batch, kv, cap))
    for keep in keeps:
        evict(T, 32, kv, (n,) + tuple(int(x) for x in rng.integers(0, n + 1, batch - 1)), cap, keep, min(keep, 33), sums, seed=keep)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("heads,kv,lens,cap", [(16, 2, (3000, 511), 3000), (24, 2, (2600,), 2600), (32, 2, (513, 2300), 2400), (12, 2, (2500,), 2500), (3, 1, (5000,), 5000)])
def test_sums_of_groups_of_any_size(T, name, heads, kv, lens, cap):
    """Heads that lie in several runs, with groups of 8, 12, 16, 6 and 3 query heads: scores are taken up in fours, or one by one."""
    q, k, v = setup(T, heads, kv, 64, name, lens, cap, heads)
    check(T, q, k, v, lens, 0.125, name)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("n,cap", [(600, 600), (4000, 4000)])
def test_queries_that_are_not_finite_spoil_their_own_head_only(T, name, bad, n, cap):
    from lighterpp_b200 import ops
    q, k, v = setup(T, 8, 2, 64, name, (n, n), cap, 13, garbage=False)
    q[0, 2, 5] = bad
    kc, vc = T.from_numpy(k).cuda(), T.from_numpy(v).cuda()
    out, sums = T.zeros_like(q), T.zeros((2, 2, cap), device="cuda")
    ops.cuda_kv4_attention(out, q, kc, vc, T.tensor([n, n], dtype=T.int32, device="cuda"), 0.125, None, sums)
    q[0, 2, 5] = 0.0
    ref, bound, want_sums, sums_bound = U.attention(q.double().cpu().numpy(), k, v, (n, n), 0.125, name != "f32")
    got, got_sums = out.double().cpu().numpy(), sums.double().cpu().numpy()
    assert np.isnan(got[0, 2]).all() and np.isnan(got_sums[0, 0]).all()
    ok = np.ones((2, 8), dtype=bool)
    ok[0, 2] = False
    bound = bound + half_step(name) * (np.abs(ref) + bound) + 2.0 ** -25
    assert np.all(np.abs(got - ref)[ok] <= bound[ok])
    for b, h in ((0, 1), (1, 0), (1, 1)):
        assert np.all(np.abs(got_sums - want_sums)[b, h] <= (sums_bound + 2.0 ** -24 * want_sums)[b, h])
