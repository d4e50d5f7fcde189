"""Residual addition, RMS norm and int8 activations (llattn_add_norm_q8) against a plain form in numpy.

The codes, their sums and the residual are fixed by single IEEE operations in fp32 and have to be the same bits. The scale is e * r: e is one of
those values, r = 1 / sqrt(mean + eps) comes from a sum of K squares in fp32. A thread folds at most 4 K / 128 of them one after the other, a
butterfly (5) and the warps' results (up to 16) follow, so the sum is off by at most (4 K / 128 + 22) 2^-24 of itself, r by half of that and by
the mean's division and addition and rsqrtf (2 ulp): (2 K / 128 + 16) 2^-24 covers it with the product. y is rounded once more, by
half a step of its type, and behind fp16's smallest normal by half of its smallest number."""
import importlib

import numpy as np
import pytest

torch = pytest.importorskip("torch")
F = np.float32


@pytest.fixture(scope="module")
def api(pkg):
    m = importlib.import_module(pkg.__name__ + ".api")
    m.lib()
    return m


def _plain(x, d, gain, eps, frag):
    """(v, codes in fragment order, s, sum, y) with numpy: fp32 where a single operation defines the value, else 64 bits."""
    T, K = x.shape
    v = x if d is None else (x + d.astype(F)).astype(F)
    with np.errstate(all="ignore"):
        t = (v * gain).astype(F).reshape(T, K // 128, 128)
        a = np.abs(t).max(2)                                  # NaN where there is one
        e = np.where(np.isfinite(a), np.maximum(a / F(127), F(1e-30)), np.nan).astype(F)
        codes = np.where(np.isfinite(e)[..., None], np.rint((t / e[..., None]).astype(F)), 0).astype(np.int8)
        r = 1.0 / np.sqrt((v.astype(np.float64) ** 2).mean(1) + eps)
        s = e.astype(np.float64) * r[:, None]
        y = t.astype(np.float64).reshape(T, K) * r[:, None]
    q = np.zeros((T, K), np.int8)
    q[:, frag] = codes.reshape(T, K)
    return v, q, s, codes.sum(2, dtype=np.int64).astype(np.int32), y


def _frag(orc, K):
    return np.array([orc.frag_pos(c) for c in range(K)])


def _inputs(T, K, delta, seed):
    g = np.random.default_rng(seed)
    x = (g.standard_normal((T, K)) * np.exp(g.standard_normal((T, 1)))).astype(F)
    x[:, g.integers(0, K, max(1, K // 300))] *= F(50)
    d = None if delta is None else torch.from_numpy(g.standard_normal((T, K)).astype(F)).to(delta)
    return x, d, (1 + 0.2 * g.standard_normal(K)).astype(F)


def _as_np(d):
    return None if d is None else d.float().numpy()


def _run(api, x, d, gain, eps, y_type=None, q=True, pad=0):
    T, K = x.shape
    wide = torch.full((T, K + pad), 7.0, device="cuda")
    wide[:, :K] = torch.from_numpy(x)
    dx = wide[:, :K]
    dd = None
    if d is not None:
        dd = torch.full((T, K + 2 * pad), 9.0, device="cuda", dtype=d.dtype)[:, :K]
        dd.copy_(d)
    out = dict(q=torch.full((T, K), 99, dtype=torch.int8, device="cuda"), s=torch.full((T, K // 128), -1.0, device="cuda"),
               qsum=torch.full((T, K // 128), -1, dtype=torch.int32, device="cuda")) if q else {}
    y = None if y_type is None else torch.full((T, K), 3.0, dtype=y_type, device="cuda")
    api.add_norm_q8(dx, torch.from_numpy(gain).cuda(), eps, delta=dd, y=y, **out)
    torch.cuda.synchronize()
    assert pad == 0 or bool((wide[:, K:] == 7).all())
    return dx.cpu().numpy(), {k: t.cpu().numpy() for k, t in out.items()}, None if y is None else y.double().cpu().numpy()


def _check(orc, x, d, gain, eps, got, y_type=None):
    T, K = x.shape
    v, q, s, qsum, y = _plain(x, _as_np(d), gain, eps, _frag(orc, K))
    gx, out, gy = got
    assert np.array_equal(gx.view(np.uint32), v.view(np.uint32))
    tol = (2 * K / 128 + 16) * 2.0 ** -24
    if out:
        assert np.array_equal(out["q"], q) and np.array_equal(out["qsum"], qsum)
        assert np.array_equal(np.isnan(out["s"]), np.isnan(s))
        fine = ~np.isnan(s)
        assert (np.abs(out["s"].astype(np.float64) - s)[fine] <= tol * np.abs(s)[fine] + 2.0 ** -149).all()
    if y_type is not None:
        half = torch.finfo(y_type).eps / 2
        assert (np.abs(gy - y) <= (half + tol * 1.01) * np.abs(y) + (2.0 ** -25 if y_type == torch.float16 else 0)).all()


SIZES = [(1, 128), (1, 2048), (3, 384), (32, 2048), (5, 32768), (147, 640), (148, 2048), (149, 2048), (150, 128), (301, 2176), (515, 5120), (200, 32768), (1000, 256), (296, 384), (297, 384), (592, 1024), (593, 1024), (593, 896),
         (700, 4096), (592, 8192), (593, 8192), (4736, 1024), (4737, 1024)]


@pytest.mark.gpu
@pytest.mark.parametrize("delta", [None, torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,K", SIZES)
def test_norm_q8(api, orc, T, K, delta):
    x, d, gain = _inputs(T, K, delta, T + K)
    _check(orc, x, d, gain, 1e-6, _run(api, x, d, gain, 1e-6))


@pytest.mark.gpu
@pytest.mark.parametrize("y_type", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,K,delta,q,pad", [(1, 2048, None, True, 0), (33, 2048, torch.bfloat16, True, 8), (33, 2048, None, False, 4), (300, 640, torch.float32, True, 128),
                                             (300, 8192, torch.float16, False, 0), (149, 128, torch.float16, True, 4), (2, 32768, torch.float32, True, 16)])
def test_norm_16_bits_and_strides(api, orc, T, K, delta, q, pad, y_type):
    x, d, gain = _inputs(T, K, delta, T + K + pad)
    _check(orc, x, d, gain, 1e-5, _run(api, x, d, gain, 1e-5, y_type, q, pad), y_type)


@pytest.mark.gpu
@pytest.mark.parametrize("T,K", [(4, 512), (160, 512)])
def test_norm_of_hard_rows(api, orc, T, K):
    """Rows of zeros, of the smallest numbers, of one value, of ties (t / e half-way between two codes), with an infinity, with NaN, with a group of zeros."""
    x, _, gain = _inputs(T, K, None, 5)
    gain[:] = 1
    x[0] = 0
    x[1] = F(2.0 ** -140)
    x[2] = F(-3.25)
    x[3] = (np.arange(K) % 128 * 2 + 1).astype(F) / 2         # 0.5, 1.5, ..., 127.5: the largest becomes 127
    x[3, ::128] = F(127)
    if T > 4:
        x[4:8, 200] = [np.inf, -np.inf, np.nan, F(3e38)]
        x[8, 128:256] = 0
        x[9] = (np.arange(K) % 2 * 126 + 0.5).astype(F)
        x[9, ::128] = F(127)                                  # e = 1: 0.5 and 126.5 are ties
    want_nan = {4, 5, 6} if T > 4 else set()
    got = _run(api, x, None, gain, 0.0 if T == 4 else 1e-6)
    if T == 4:
        got[1]["s"][0] = 0                                    # zeros and eps 0: 0 / 0, whatever that gives
        v, q, s, qsum, _ = _plain(x, None, gain, 0.0, _frag(orc, K))
        assert np.array_equal(got[1]["q"], q) and np.array_equal(got[1]["qsum"], qsum) and not q[0].any()
        return
    rows = [i for i in range(T) if i not in want_nan and i != 7]
    _check(orc, x[rows], None, gain, 1e-6, (got[0][rows], {k: a[rows] for k, a in got[1].items()}, None))
    s = got[1]["s"]
    assert np.isnan(s[4, 1]) and np.isnan(s[5, 1]) and np.isnan(s[6]).all() and not s[4, [0, 2, 3]].any()
    assert not got[1]["q"][4:7, 128:256].any() and not got[1]["qsum"][4:7, 1].any()
    assert not s[7].any()                                     # the squares pass fp32: r = 0


@pytest.mark.gpu
def test_norm_does_not_depend_on_the_batch(api):
    """A row has the same bits in a call of one and of many: codes, sums; and the scales of calls that take the same launch shape."""
    x, d, gain = _inputs(400, 2048, torch.bfloat16, 9)
    many = _run(api, x, d, gain, 1e-6)[1]
    for i in (0, 7, 399):
        one = _run(api, x[i:i + 1], d[i:i + 1], gain, 1e-6)[1]
        assert np.array_equal(one["q"][0], many["q"][i]) and np.array_equal(one["qsum"][0], many["qsum"][i])
        assert np.allclose(one["s"][0], many["s"][i], rtol=1e-6, atol=0)
    assert all(np.array_equal(a, b) for a, b in zip(_run(api, x, d, gain, 1e-6)[1].values(), many.values()))


@pytest.mark.gpu
def test_norm_takes_columns_of_one_matrix(api, orc):
    """x and delta side by side in one matrix."""
    x, d, gain = _inputs(40, 256, torch.float32, 3)
    both = torch.cat([torch.from_numpy(x), d], 1).cuda()
    q, s, qsum = torch.zeros((40, 256), dtype=torch.int8, device="cuda"), torch.zeros((40, 2), device="cuda"), torch.zeros((40, 2), dtype=torch.int32, device="cuda")
    api.add_norm_q8(both[:, :256], torch.from_numpy(gain).cuda(), 1e-6, q, s, qsum, delta=both[:, 256:])
    out = {"q": q.cpu().numpy(), "s": s.cpu().numpy(), "qsum": qsum.cpu().numpy()}
    _check(orc, x, d, gain, 1e-6, (both[:, :256].cpu().numpy(), out, None))
    assert torch.equal(both[:, 256:].cpu(), d)


@pytest.mark.gpu
def test_norm_far_into_the_memory(api):
    """Rows whose values lie beyond 31 bits of index, in the residual, the codes and the 16-bit copy: what a call on these rows alone gives."""
    T, K = 1_060_000, 2048
    x = torch.full((T, K), 0.5, device="cuda")
    x[-50:] = torch.randn((50, K), device="cuda")
    d, gain = torch.ones((T, K), dtype=torch.half, device="cuda"), torch.ones(K, device="cuda")
    new = lambda n: (torch.zeros((n, K), dtype=torch.int8, device="cuda"), torch.zeros((n, K // 128), device="cuda"), torch.zeros((n, K // 128), dtype=torch.int32, device="cuda"))
    tail, outs, y = x[-50:].clone(), new(T), torch.zeros((T, K), dtype=torch.half, device="cuda")
    api.add_norm_q8(x, gain, 1e-6, *outs, delta=d, y=y)
    few, yf = new(50), torch.zeros((50, K), dtype=torch.half, device="cuda")
    api.add_norm_q8(tail, gain, 1e-6, *few, delta=d[:50], y=yf)
    assert torch.equal(x[-50:], tail) and torch.equal(outs[0][-50:], few[0]) and torch.equal(outs[2][-50:], few[2])
    assert torch.allclose(outs[1][-50:], few[1], rtol=1e-6, atol=0) and torch.allclose(y[-50:].float(), yf.float(), rtol=2.0 ** -10, atol=0)
    assert bool((x[:100] == 1.5).all()) and bool((outs[0][:100] == 127).all()) and bool((y[:100] == 1).all())


@pytest.mark.gpu
def test_norm_feeds_the_projection(api, orc, pkg):
    x, d, gain = _inputs(70, 2048, torch.float16, 31)
    got = _run(api, x, d, gain, 1e-6)[1]
    strips, _, _, _ = pkg.workload.dense_weights(256, 2048, 32)
    Y = torch.zeros((70, 256), device="cuda")
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
    api.dense_w4a8(dev(strips), dev(got["q"]), dev(got["s"]), dev(got["qsum"]), Y)
    want = np.zeros((70, 256), F)
    orc.dense_w4a8(strips, got["q"], got["s"], got["qsum"], want)
    assert np.array_equal(Y.cpu().numpy().view(np.uint32), want.view(np.uint32))


def _call(api, **changed):
    """The C entry point with host addresses that no check refuses, but for what is changed. Nothing is launched: a call that passes has T = 0."""
    a = dict(x=0x10000, ldx=256, delta=None, delta_type=0, ldd=0, gain=0x20000, eps=1e-6, q=0x30000, s=0x40000, sum=0x50000, y=None, y_type=1, T=0, K=256)
    a.update(changed)
    return api.lib().llattn_add_norm_q8(a["x"], a["ldx"], a["delta"], a["delta_type"], a["ldd"], a["gain"], a["eps"], a["q"], a["s"], a["sum"], a["y"], a["y_type"],
                                        a["T"], a["K"], None)


@pytest.mark.parametrize("bad", [
    dict(x=None), dict(gain=None), dict(q=None, s=None, sum=None), dict(s=None), dict(sum=None), dict(q=None, y=0x60000), dict(T=-1), dict(T=(1 << 24) + 1), dict(K=0), dict(K=100),
    dict(K=32896, ldx=32896), dict(ldx=128), dict(ldx=258), dict(delta=0x70000, ldd=128), dict(delta=0x70000, ldd=257), dict(delta=0x70000, ldd=256, delta_type=3),
    dict(delta=0x70000, ldd=256, delta_type=-1), dict(y=0x60000, y_type=0), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(x=0x10004), dict(q=0x30008), dict(gain=0x20004),
    dict(s=0x40002), dict(y=0x60002), dict(delta=0x70008, ldd=256),
    # an output over another argument
    dict(T=4, q=0x10000), dict(T=4, s=0x20000), dict(T=4, sum=0x40000), dict(T=4, y=0x30000), dict(T=4, delta=0x10000 + 512, ldd=256), dict(T=4, delta=0x30000, ldd=256)])
def test_norm_refusals(api, bad):
    assert _call(api, **bad) == api.EINVAL and b"add_norm_q8" in api.lib().llattn_last_error()


def test_norm_of_nothing_is_nothing(api):
    assert _call(api) == api.OK and _call(api, delta=0x70000, ldd=256, delta_type=2) == api.OK and _call(api, q=None, s=None, sum=None, y=0x60000) == api.OK


@pytest.mark.gpu
def test_norm_binding_refusals(api):
    z = lambda *s, dtype=torch.float32: torch.zeros(s, dtype=dtype, device="cuda")
    x, gain, q, s, qsum = z(4, 256), z(256), z(4, 256, dtype=torch.int8), z(4, 2), z(4, 2, dtype=torch.int32)
    api.add_norm_q8(x, gain, 1e-6, q, s, qsum)
    for a in [(x.half(), gain, q, s, qsum), (x, gain[:128], q, s, qsum), (x, gain, q[:3], s, qsum), (x, gain, q, s[:, :1], qsum), (x, gain, q, s, qsum.float()),
              (x, gain, q, s, None), (x.t(), gain, q, s, qsum), (x.cpu(), gain, q, s, qsum), (x, gain.cpu(), q, s, qsum)]:
        with pytest.raises(ValueError):
            api.add_norm_q8(a[0], a[1], 1e-6, *a[2:])
    for kw in [dict(delta=z(3, 256)), dict(y=z(4, 128, dtype=torch.half))]:
        with pytest.raises(ValueError):
            api.add_norm_q8(x, gain, 1e-6, q, s, qsum, **kw)
    for kw in [dict(delta=z(4, 256, dtype=torch.float64)), dict(y=z(4, 256))]:
        with pytest.raises(api.LlattnError):
            api.add_norm_q8(x, gain, 1e-6, q, s, qsum, **kw)
