"""Low-rank adapters of many requests beside a projection (llattn_adapters_w4a8) against the formula in 64 bits.

Where everything is a small whole number nothing is rounded, and the results have to be equal. Elsewhere the bound is the sum of the
roundings: a group's 128 exact products are added in eight instructions of sixteen (four roundings of 2^-23 each allowed, the tensor core
truncates), then a multiply-add for each group and three more operations; H in parts (two of tf32 or fp16, three of bf16) keeps 2^-22 of it at
least; the second product is one instruction for eight ranks and each part at most, four roundings of 2^-23 each again; the addition into Y is one rounding. Each is
relative to the sum of the absolute values of what is added."""
import importlib
import os
import subprocess
import sys

import numpy as np
import pytest

torch = pytest.importorskip("torch")
F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def api(pkg):
    m = importlib.import_module(pkg.__name__ + ".api")
    m.lib()
    return m


def _frag(orc, K):
    return np.array([orc.frag_pos(c) for c in range(K)])


def _case(T, K, rank, n, parts, dtype, seed, whole=False):
    """q (logical order), s, Y and per part (row0, A, B); whole: small whole numbers, scales powers of two."""
    g = np.random.default_rng(seed)
    q = g.integers(-128 if not whole else -3, 128 if not whole else 4, (T, K)).astype(np.int8)
    if whole:
        s = 2.0 ** g.integers(-1, 2, (T, K // 128))
        ab = [(g.integers(-2, 3, (n, rank, K)) * (g.random((n, rank, K)) < 0.2), g.integers(-3, 4, (n, rows, rank))) for _, rows in parts]
    else:
        s = 0.02 * np.exp(0.5 * g.standard_normal((T, K // 128)))
        ab = [(g.standard_normal((n, rank, K)) / np.sqrt(K), g.standard_normal((n, rows, rank)) / np.sqrt(rank)) for _, rows in parts]
    ab = [tuple(torch.from_numpy(np.asarray(x, np.float32)).to(dtype) for x in p) for p in ab]
    width = max(r0 + rows for r0, rows in parts) + 8
    Y = (g.integers(-9, 10, (T, width)) if whole else g.standard_normal((T, width))).astype(np.float32)
    return q, s.astype(np.float32), Y, ab


def _plain(q, s, Y, ab, parts, segs, scale, ranks):
    """(Y, bound) in 64 bits. segs: (first token, end, adapter)."""
    K = q.shape[1]
    want, bound = Y.astype(np.float64), np.zeros(Y.shape)
    x = q.astype(np.float64) * np.repeat(s.astype(np.float64), 128, 1)
    for t0, t1, a in segs:
        n = ab[0][0].shape[0]
        if t1 <= t0 or not 0 <= a < n:
            continue
        r = ab[0][0].shape[1] if ranks is None else int(ranks[a])
        c = 1.0 if scale is None else float(scale[a])
        for (row0, rows), (A, B) in zip(parts, ab):
            A64, B64 = A[a, :r].double().numpy(), B[a, :, :r].double().numpy()
            H, mag = x[t0:t1] @ A64.T, np.abs(x[t0:t1]) @ np.abs(A64).T
            off = (8 * 4 + K // 128 + 3) * 2.0 ** -23 * mag + 2.0 ** -22 * np.abs(H)
            d, big = c * (H @ B64.T), abs(c) * ((np.abs(H) + off) @ np.abs(B64).T)
            want[t0:t1, row0:row0 + rows] += d
            bound[t0:t1, row0:row0 + rows] = abs(c) * (off @ np.abs(B64).T) + (-(-r // 8) * 2 * 4 + 1) * 2.0 ** -23 * big + 2.0 ** -24 * np.abs(want[t0:t1, row0:row0 + rows])
    return want, bound


def _run(api, orc, q, s, Y, ab, parts, first, adapter, scale=None, ranks=None, stream=None):
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
    qf = np.zeros_like(q)
    qf[:, _frag(orc, q.shape[1])] = q
    sc = None if scale is None else dev(np.asarray(scale, np.float32))
    rk = None if ranks is None else dev(np.asarray(ranks, np.int32))
    pools = api.adapter_pools([api.AdapterPool(A.cuda(), B.cuda(), row0=row0, scale=sc, ranks=rk) for (row0, _), (A, B) in zip(parts, ab)])
    dY = dev(Y)
    api.adapters_w4a8(pools, dev(qf), dev(s), dY, dev(np.asarray(first, np.int32)), dev(np.asarray(adapter, np.int32)))
    torch.cuda.synchronize()
    return dY.cpu().numpy()


def _segs(first, adapter):
    return list(zip(first[:-1], first[1:], adapter))


def _random_segments(T, nseg, n, seed):
    g = np.random.default_rng(seed)
    first = [0] + sorted(int(v) for v in g.integers(0, T + 1, nseg))
    return first, [int(v) for v in g.integers(-1, n, nseg)]


# (tokens, segments, K, rank, adapters, parts)
CASES = [(1, 1, 2048, 8, 3, [(0, 2048)]), (1, 1, 128, 8, 1, [(0, 4)]), (7, 7, 256, 16, 9, [(4, 36)]), (32, 1, 2048, 16, 2, [(0, 2048)]), (33, 1, 1152, 24, 2, [(0, 512)]),
         (31, 2, 128, 128, 2, [(0, 132)]), (100, 5, 384, 40, 4, [(8, 260)]), (64, 64, 512, 32, 5, [(0, 512)]), (257, 3, 2176, 64, 3, [(0, 1024), (1280, 256)]),
         (300, 300, 256, 8, 7, [(0, 64), (64, 128), (192, 32), (240, 4)]), (515, 20, 2048, 72, 6, [(0, 256)]), (90, 700, 128, 8, 4, [(0, 96)]), (40, 2, 4224, 128, 2, [(0, 2048)]),
         # many tiles: clusters of four, two and one for each of the kernels
         (1700, 3, 256, 16, 2, [(0, 96)]), (3001, 40, 384, 16, 3, [(0, 64)]), (9600, 5, 128, 8, 2, [(0, 36)]), (1300, 3, 384, 24, 2, [(0, 68)]), (4900, 7, 128, 32, 2, [(0, 32)]),
         (10000, 2, 128, 32, 2, [(0, 32)]), (900, 9, 384, 48, 3, [(0, 300)]), (2500, 1, 256, 40, 1, [(0, 132)]), (4800, 3, 128, 64, 2, [(0, 260)]), (1000, 2, 256, 96, 2, [(0, 140)]),
         (1500, 1, 128, 128, 1, [(0, 132)]), (5000, 2, 128, 72, 2, [(0, 132)])]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("T,nseg,K,rank,n,parts", CASES)
def test_adapters_whole_numbers(api, orc, T, nseg, K, rank, n, parts, dtype):
    q, s, Y, ab = _case(T, K, rank, n, parts, dtype, T + K, whole=True)
    first, adapter = ([0, T], [n - 1]) if nseg == 1 else _random_segments(T, nseg, n, T)
    scale = 2.0 ** (np.arange(n) % 3 - 1)
    ranks = [(rank - 3 * i) % (rank + 1) for i in range(n)] if n > 1 else None
    want, _ = _plain(q, s, Y, ab, parts, _segs(first, adapter), scale, ranks)
    assert np.abs(want).max() < 2 ** 21                           # quarters and halves: all sums are exact in 24 bits
    got = _run(api, orc, q, s, Y, ab, parts, first, adapter, scale, ranks)
    assert np.array_equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("T,nseg,K,rank,n,parts", CASES)
def test_adapters(api, orc, T, nseg, K, rank, n, parts, dtype):
    q, s, Y, ab = _case(T, K, rank, n, parts, dtype, T + rank)
    first, adapter = ([0, T], [0]) if nseg == 1 else _random_segments(T, nseg, n, T + 1)
    scale = None if rank == 16 else np.random.default_rng(1).uniform(-2, 2, n).astype(np.float32)
    want, bound = _plain(q, s, Y, ab, parts, _segs(first, adapter), scale, None)
    got = _run(api, orc, q, s, Y, ab, parts, first, adapter, scale)
    assert (np.abs(got - want) <= bound).all(), float((np.abs(got - want) - bound).max())
    assert np.array_equal(got[bound == 0], Y[bound == 0])
    again = _run(api, orc, q, s, Y, ab, parts, first, adapter, scale)
    assert np.array_equal(got.view(np.uint32), again.view(np.uint32))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_adapters_leave_alone_what_is_not_theirs(api, orc, dtype):
    """Tokens in front of the first segment and behind the last, segments without an adapter or with one that the pool does not have, empty ones, bounds
    that go back or beyond the tokens, ranks of 0, NaN in unused adapters and behind the ranks: nothing of it is touched or counts."""
    T, K, rank, n, parts = 200, 256, 24, 6, [(4, 100)]
    q, s, Y, ab = _case(T, K, rank, n, parts, dtype, 1)
    ranks = [24, 5, 0, 17, 8, 24]
    A, B = ab[0]
    for a, r in enumerate(ranks):
        A[a, r:] = float("nan")
        B[a, :, r:] = float("inf")
    A[5] = B[5] = float("nan")
    first = [10, 20, 20, 55, 90, 91, 130, 150, 500]
    adapter = [0, 3, -1, 1, 2, 3, n, 4]
    want, bound = _plain(q, s, Y, ab, parts, [(t0, min(t1, T), a) for t0, t1, a in _segs(first, adapter)], None, ranks)
    got = _run(api, orc, q, s, Y, ab, parts, first, adapter, None, ranks)
    assert np.isfinite(got).all() and (np.abs(got - want) <= bound).all()
    assert np.array_equal(got[bound == 0], Y[bound == 0])
    for first, adapter in [([150, 40, 40, -7], [0, 0, 0]), ([T, T + 50], [0]), ([0, 0], [0]), ([-9, 0], [1]), ([0, T], [-2 ** 31]), ([0, T], [2 ** 31 - 1])]:
        assert np.array_equal(_run(api, orc, q, s, Y, ab, parts, first, adapter, None, ranks), Y)
    got = _run(api, orc, q, s, Y, ab, parts, [0, T], [0], None, [2 ** 31 - 1] * n)             # a rank beyond the pool's is the pool's
    want, bound = _plain(q, s, Y, ab, parts, [(0, T, 0)], None, None)
    assert (np.abs(got - want) <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rank", [16, 32, 64])
def test_adapters_of_any_magnitude(api, orc, rank, dtype):
    """Ranks whose parts of H differ by many powers of two, tokens of all sizes and zeros: each within its own bound."""
    T, K, n, parts = 48, 256, 2, [(0, 64)]
    q, s, Y, ab = _case(T, K, rank, n, parts, dtype, 7)
    s *= (2.0 ** np.linspace(-40, 40, T))[:, None].astype(np.float32)
    q[5] = 0
    s[6] = 0
    A, B = ab[0]
    A *= (2.0 ** torch.linspace(-8, 8, rank))[None, :, None].to(dtype)
    want, bound = _plain(q, s, Y, ab, parts, [(0, T, 1)], None, None)
    got = _run(api, orc, q, s, Y, ab, parts, [0, T], [1])
    assert (np.abs(got - want) <= bound).all() and np.array_equal(got[5:7], Y[5:7])


@pytest.mark.gpu
def test_adapters_far_into_the_memory(api, orc):
    """Elements of Y, and of a pool's A, whose index does not fit 31 bits."""
    g = torch.Generator(device="cuda"); g.manual_seed(3)
    T, K, rows, rank = 2_200_000, 128, 1024, 8
    Y = torch.zeros((T, rows), device="cuda")
    q = torch.randint(-9, 10, (T, K), generator=g, device="cuda", dtype=torch.int8)
    s = torch.ones((T, 1), device="cuda")
    A, B = torch.randint(-2, 3, (2, rank, K), generator=g, device="cuda").half(), torch.randint(-2, 3, (2, rows, rank), generator=g, device="cuda").half()
    first = torch.tensor([0, T - 40, T - 3], dtype=torch.int32, device="cuda")
    api.adapters_w4a8(api.adapter_pools([api.AdapterPool(A, B)]), q, s, Y, first, torch.tensor([-1, 1], dtype=torch.int32, device="cuda"))
    x = q[T - 40:].float()[:, torch.from_numpy(_frag(orc, K)).cuda()]
    want = x @ A[1].float().t() @ B[1].float().t()
    want[-3:] = 0
    assert torch.equal(Y[T - 40:], want) and not bool(Y[T - 80:T - 40].any()) and not bool(Y[:1000].any())
    del Y, q
    n, K, rank = 1100, 16384, 128
    A = torch.zeros((n, rank, K), dtype=torch.half, device="cuda")
    A[n - 1] = torch.randint(-1, 2, (rank, K), generator=g, device="cuda").half()
    B = torch.ones((n, 8, rank), dtype=torch.half, device="cuda")
    q, s, Y = torch.randint(-1, 2, (3, K), generator=g, device="cuda", dtype=torch.int8), torch.ones((3, K // 128), device="cuda"), torch.zeros((3, 8), device="cuda")
    api.adapters_w4a8(api.adapter_pools([api.AdapterPool(A, B)]), q, s, Y, torch.tensor([0, 3], dtype=torch.int32, device="cuda"), torch.tensor([n - 1], dtype=torch.int32, device="cuda"))
    want = (q.float()[:, torch.from_numpy(_frag(orc, K)).cuda()] @ A[n - 1].float().t()).sum(1, keepdim=True).expand(3, 8)
    assert torch.equal(Y, want) and bool(Y.any())


@pytest.mark.gpu
def test_adapters_of_nan_activations_are_nan(api, orc):
    T, K, rank, n, parts = 40, 256, 8, 2, [(0, 64)]
    q, s, Y, ab = _case(T, K, rank, n, parts, F16, 2)
    s[3, 1] = np.nan
    got = _run(api, orc, q, s, Y, ab, parts, [0, T], [1])
    assert np.isnan(got[3, :64]).all() and np.isfinite(np.delete(got, 3, 0)).all() and np.array_equal(got[3, 64:], Y[3, 64:])


@pytest.mark.gpu
def test_adapters_first_call_under_capture(pkg):
    """A process whose first call of a kernel is captured: nothing that a call sets up once may disturb the capture."""
    code = f"""
import importlib, torch
api = importlib.import_module({pkg.__name__!r} + ".api")
z = lambda *s, dtype=torch.float32: torch.zeros(s, dtype=dtype, device="cuda")
T = 40
q, s, Y, first, adapter = torch.ones((T, 256), dtype=torch.int8, device="cuda"), torch.ones((T, 2), device="cuda"), z(T, 64), torch.tensor([0, T], dtype=torch.int32, device="cuda"), z(1, dtype=torch.int32)
for dtype in (torch.half, torch.bfloat16):
    for rank in (8, 32, 64, 128):
        pools = api.adapter_pools([api.AdapterPool(torch.ones((1, rank, 256), dtype=dtype, device="cuda"), torch.ones((1, 64, rank), dtype=dtype, device="cuda"))])
        x, n8, ns, nsum = z(T, 256), z(T, 256, dtype=torch.int8), z(T, 2), z(T, 2, dtype=torch.int32)
        graph = torch.cuda.CUDAGraph()
        Y.zero_()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            api.adapters_w4a8(pools, q, s, Y, first, adapter)
            api.add_norm_q8(x, torch.ones(256, device="cuda"), 1e-6, n8, ns, nsum)
        assert not bool(Y.any())
        graph.replay()
        torch.cuda.synchronize()
        assert bool((Y == 256 * rank).all()), (dtype, rank)
assert api.dense_status() == 0
print("done")
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))), capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "done" in r.stdout, r.stderr[-1500:]


@pytest.mark.gpu
def test_nothing_to_do(api):
    z = lambda *s, dtype=torch.float32: torch.zeros(s, dtype=dtype, device="cuda")
    i32, pools = torch.int32, api.adapter_pools([api.AdapterPool(z(1, 8, 128, dtype=F16), z(1, 4, 8, dtype=F16))])
    api.adapters_w4a8(pools, z(0, 128, dtype=torch.int8), z(0, 1), z(0, 4), z(2, dtype=i32), z(1, dtype=i32))
    api.adapters_w4a8(pools, z(3, 128, dtype=torch.int8), z(3, 1), z(3, 4), z(1, dtype=i32), z(0, dtype=i32))
    api.add_norm_q8(z(0, 128), z(128), 1e-6, z(0, 128, dtype=torch.int8), z(0, 1), z(0, 1, dtype=i32))
    freq, axes = torch.from_numpy(api.inv_freq()).cuda(), api.rope_axes([16, 16])
    out = [z(0, n, 128, dtype=F16) for n in (16, 4, 4)]
    api.qk_norm_rope_axes(z(0, 3072), z(2, 0, dtype=i32), axes, z(128), z(128), 1e-6, freq, *out)
    api.qkv_prepare_commit_axes(z(0, 3072), z(2, 0, dtype=i32), axes, z(128), z(128), 1e-6, freq, *out, z(4, 1, 4736, dtype=torch.uint8), max_blocks=1)


@pytest.mark.gpu
def test_adapters_on_two_streams_at_once(api, orc, pkg):
    """Calls of every kernel that overlap on the device, a tcgen05 projection between them, give the bits of calls one at a time."""
    T, K, n, parts = 700, 512, 3, [(0, 512)]
    strips = torch.from_numpy(pkg.workload.dense_weights(512, K, 1)[0]).cuda()
    jobs = []
    for k, (rank, dtype) in enumerate([(16, F16), (64, BF16), (128, F16), (32, BF16), (64, F16), (8, BF16)]):
        q, s, Y, ab = _case(T, K, rank, n, parts, dtype, k)
        first, adapter = _random_segments(T, 9, n, k)
        dev = lambda a, t=None: torch.from_numpy(np.ascontiguousarray(a)).cuda()
        qsum = dev(q.reshape(T, K // 128, 128).sum(2, dtype=np.int32))
        pools = api.adapter_pools([api.AdapterPool(*[x.cuda() for x in ab[0]])])
        jobs.append((pools, dev(q), dev(s), qsum, dev(Y[:, :512]), dev(np.asarray(first, np.int32)), dev(np.asarray(adapter, np.int32))))
    torch.cuda.synchronize()

    def run(streams):
        outs = []
        for i, (pools, q, s, qsum, Y, first, adapter) in enumerate(jobs):
            with torch.cuda.stream(streams[i % len(streams)]):
                y = Y.clone()
                for _ in range(3):
                    api.adapters_w4a8(pools, q, s, y, first, adapter)
                    api.dense_w4a8(strips, q, s, qsum, y)
                outs.append(y)
            if len(streams) == 1:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        return outs

    want = run([torch.cuda.current_stream()])
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(4):
        assert all(torch.equal(a, b) for a, b in zip(want, run(streams)))
    assert api.dense_status() == 0 and all(bool(torch.isfinite(a).all()) for a in want)


def _args(api, **changed):
    """A call of the C entry point with addresses that no check refuses, but for what is changed. Nothing is launched: a call that passes has no tokens."""
    pool = dict(A=0x100000, B=0x200000, scale=0x300000, ranks=0x310000, n=4, rank=16, rows=64, row0=0, type=api.F16)
    a = dict(npools=1, q=0x400000, s=0x500000, Y=0x600000, ldy=256, T=0, K=256, first=0x700000, adapter=0x710000, nseg=2)
    more = changed.pop("pools", None)
    pool.update({k: v for k, v in changed.items() if k in pool})
    a.update({k: v for k, v in changed.items() if k in a})
    assert set(changed) <= set(pool) | set(a) | {"none"}
    arr = (api._AdapterPool * 4)(*[api._AdapterPool(**{**pool, **p}) for p in (more or [{}])])
    return api.lib().llattn_adapters_w4a8(None if "none" in changed else arr, a["npools"], a["q"], a["s"], a["Y"], a["ldy"], a["T"], a["K"], a["first"], a["adapter"], a["nseg"], None)


@pytest.mark.parametrize("bad", [
    dict(none=True), dict(npools=0), dict(npools=5), dict(q=None), dict(s=None), dict(Y=None), dict(first=None), dict(adapter=None), dict(A=None), dict(B=None), dict(T=-1), dict(T=(1 << 22) + 1),
    dict(K=0), dict(K=200), dict(K=(1 << 20) + 128), dict(nseg=-1), dict(nseg=(1 << 16) + 1), dict(ldy=0), dict(ldy=66), dict(ldy=60), dict(q=0x400008), dict(Y=0x600004), dict(s=0x500002), dict(first=0x700001),
    dict(type=0), dict(type=3), dict(n=0), dict(rank=0), dict(rank=12), dict(rank=136), dict(rows=0), dict(rows=6), dict(rows=260), dict(row0=-4), dict(row0=2), dict(row0=196), dict(row0=2 ** 31 - 4),
    dict(A=0x100008), dict(B=0x200004), dict(scale=0x300002), dict(ranks=0x310001),
    dict(npools=2, pools=[{}, {}]), dict(npools=2, pools=[{}, dict(row0=60)]), dict(npools=2, pools=[{}, dict(row0=64, type=2)]), dict(npools=3, pools=[{}, dict(row0=128), dict(row0=100)]),
    # Y over an input
    dict(T=8, Y=0x400010), dict(T=8, Y=0x500000), dict(T=8, Y=0x100000), dict(T=8, Y=0x200000), dict(T=8, Y=0x300000), dict(T=8, Y=0x310000), dict(T=8, Y=0x6ffff0), dict(T=8, Y=0x70fff0)])
def test_adapter_refusals(api, bad):
    assert _args(api, **bad) == api.EINVAL and b"adapters_w4a8" in api.lib().llattn_last_error()


def test_adapters_of_nothing_are_nothing(api):
    assert _args(api) == api.OK and _args(api, T=8, nseg=0) == api.OK and _args(api, scale=None, ranks=None) == api.OK
    assert _args(api, npools=3, pools=[{}, dict(row0=128), dict(row0=64)]) == api.OK and _args(api, row0=192) == api.OK


@pytest.mark.gpu
def test_adapter_binding_refusals(api):
    z = lambda *s, dtype=torch.float32: torch.zeros(s, dtype=dtype, device="cuda")
    A, B = z(3, 16, 256, dtype=F16), z(3, 64, 16, dtype=F16)
    for kw in [dict(A=A.float(), B=B.float()), dict(A=A, B=B[:2]), dict(A=A, B=B.bfloat16()), dict(A=A, B=B, scale=z(2)), dict(A=A, B=B, ranks=z(3)), dict(A=A[:, :8], B=B), dict(A=A.cpu(), B=B)]:
        with pytest.raises((ValueError, api.LlattnError)):
            p = api.adapter_pools([api.AdapterPool(**kw)])
            api.adapters_w4a8(p, z(4, 256, dtype=torch.int8), z(4, 2), z(4, 64), z(2, dtype=torch.int32), z(1, dtype=torch.int32))
    with pytest.raises(ValueError):
        api.adapter_pools([])
    pools = api.adapter_pools([api.AdapterPool(A, B)])
    good = [z(4, 256, dtype=torch.int8), z(4, 2), z(4, 64), z(2, dtype=torch.int32), z(1, dtype=torch.int32)]
    api.adapters_w4a8(pools, *good)
    for i, t in [(0, z(4, 128, dtype=torch.int8)), (0, z(4, 256)), (1, z(4, 3)), (2, z(4, 60)), (2, z(3, 64)), (2, z(4, 64, dtype=F16)), (2, z(64, 4).t()), (3, z(3, dtype=torch.int32)), (3, z(2)),
                 (4, z(1)), (0, good[0].cpu()), (3, good[3].cpu())]:
        with pytest.raises(ValueError):
            api.adapters_w4a8(pools, *[t if k == i else v for k, v in enumerate(good)])
