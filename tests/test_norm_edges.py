"""Arguments of llattn_add_norm_q8 that share memory: columns of one matrix may stand for the residual and its addend, columns that
overlap may not (warps would read what others write). Rows that are hard to norm or to quantise, in every way of sharing a row among warps."""
import importlib

import numpy as np
import pytest
from test_norm_q8 import _as_np, _frag, _inputs, _plain, _run

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def api(pkg):
    m = importlib.import_module(pkg.__name__ + ".api")
    m.lib()
    return m


X = 0x100000


# Rows of 256 values; byte distances from the residual's first row to the addend's. (first byte of delta - X, ldx, ldd, type of delta, rows)
@pytest.mark.parametrize("off,ldx,ldd,dtype,T", [
    (256, 512, 512, 0, 4),                          # columns 64 .. 319 next to columns 0 .. 255
    (-256, 512, 512, 0, 4), (1008, 512, 512, 0, 4), (-1008, 512, 512, 0, 4), (0, 512, 512, 0, 4), (0, 260, 260, 0, 1),
    (2048 - 1008, 512, 512, 0, 2),                  # the addend's columns reach into the next row's of the residual
    (2048 * 3 - 16, 512, 512, 0, 4), (-2048 * 3 + 16, 512, 512, 0, 4),
    (512, 512, 1024, 1, 9), (1552, 512, 1024, 2, 9),    # 16-bit columns of the same rows
    (1024, 512, 768, 0, 3),                         # other distances: rows 2 and 1 meet
    (1024, 512, 388, 0, 9), (-1000 * 1024, 260, 516, 0, 1000)])
def test_columns_that_overlap_are_refused(api, off, ldx, ldd, dtype, T):
    rc = api.lib().llattn_add_norm_q8(X, ldx, X + off, dtype, ldd, 0x8000000, 1e-6, 0x9000000, 0xA000000, 0xB000000, None, 0, T, 256, None)
    assert rc == api.EINVAL and b"overlaps" in api.lib().llattn_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("off,ldx,ldd,T", [(256, 512, 512, 5), (-256, 512, 512, 5), (260, 520, 520, 1), (256, 512, 1024, 2), (256, 512, 512, 1), (256, 1024, 512, 2)])
def test_columns_side_by_side_are_taken(api, off, ldx, ldd, T):
    """Distances in values, the addend's to the residual's first row: equal row distances, and others whose rows lie in one another's gaps."""
    g = torch.Generator(device="cuda"); g.manual_seed(off + T)
    m, K = torch.randn(16 * 1024, generator=g, device="cuda"), 256
    x, d = m.as_strided((T, K), (ldx, 1), 4096), m.as_strided((T, K), (ldd, 1), 4096 + off)
    want, kept, before = x + d, d.clone(), m.clone()
    gain, q, s, qsum = torch.ones(K, device="cuda"), torch.zeros((T, K), dtype=torch.int8, device="cuda"), torch.zeros((T, 2), device="cuda"), torch.zeros((T, 2), dtype=torch.int32, device="cuda")
    api.add_norm_q8(x, gain, 1e-6, q, s, qsum, delta=d)
    assert torch.equal(x, want) and torch.equal(d, kept)
    x.copy_(before.as_strided((T, K), (ldx, 1), 4096))
    assert torch.equal(m, before)


def _shapes():
    """(rows, K) for each way of sharing a row among warps (16, 16, 8, 8, 4, 2 of them), on a device with n SMs."""
    n = torch.cuda.get_device_properties(0).multi_processor_count if torch.cuda.is_available() else 148
    return [(n + 12, 512), (4 * n + 8, 8192), (2 * n + 104, 512), (4 * n + 8, 4096), (4 * n + 108, 1024), (4 * n + 109, 512)]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", range(6))
@pytest.mark.parametrize("eps", [0.0, 1e-6])
@pytest.mark.parametrize("delta", [False, True])
@pytest.mark.parametrize("copy", [None, torch.float16, torch.bfloat16])
def test_hard_rows_in_every_launch_shape(api, orc, shape, eps, delta, copy):
    """Rows of zeros, of the smallest numbers, of one value, of ties, with infinities, NaN, squares beyond fp32, a group of zeros; at the beginning, in the middle and
    at the end of a launch. Codes, sums and the residual to the bit, scales and copies within the plain test's bounds, and NaN where the formula says so."""
    T, K = _shapes()[shape]
    x, d, gain = _inputs(T, K, torch.bfloat16 if delta else None, shape)
    gain[:] = 1
    ties = (np.arange(K) % 128 + 0.5).astype(np.float32)
    ties = np.minimum(ties, np.float32(126.5)) * np.where(np.arange(K) % 3 == 0, -1, 1).astype(np.float32)
    ties[::128] = 127                                           # e = 1: every other value is a tie
    assert (np.abs(ties).max() == 127) and (np.abs(ties) % 1 == 0.5).sum() == K - K // 128
    hard = np.zeros((11, K), np.float32)
    hard[1], hard[2], hard[3], hard[4] = 2.0 ** -140, -3.25, ties, 2 * ties
    hard[5:9] = x[:4]
    hard[5:9, 200] = [np.inf, -np.inf, np.nan, 3e38]
    hard[9] = x[4]
    hard[9, 128:256] = 0
    hard[10] = 2.0 ** 40 * x[5]
    at = np.concatenate([np.arange(11), T // 2 + np.arange(11), T - 11 + np.arange(11)])
    x[at] = np.tile(hard, (3, 1))
    if d is not None:
        d[at] = 0
    gx, out, y = _run(api, x, d, gain, eps, copy)
    with np.errstate(all="ignore"):
        v, q, s, qsum, wy = _plain(x, _as_np(d), gain, eps, _frag(orc, K))
    nan = np.isnan(v)                                           # (whose bits an addition chooses)
    assert np.array_equal(gx.view(np.uint32)[~nan], v.view(np.uint32)[~nan]) and np.isnan(gx[nan]).all()
    assert np.array_equal(out["q"], q) and np.array_equal(out["qsum"], qsum)
    assert (q[at[3]] % 2 == 0).sum() == K - K // 128 and not q[at[0]].any()      # ties go to even codes
    # In fp32 the squares of row 8 are infinite (r = 0), of row 1 zero: r is that of eps alone, without one infinite (1e-30 of it too, and zeros times it are NaN).
    # Infinities make r = 0 too, but for their own group's scale.
    tol = (2 * K / 128 + 16) * 2.0 ** -24
    for rows in at.reshape(3, 11):
        s[rows[8]], wy[rows[8]] = 0, 0
        for i in (5, 6):
            s[rows[i]] = np.where(np.arange(K // 128) == 1, np.nan, 0)
            wy[rows[i]] = np.where(np.isinf(x[rows[i]]), np.nan, 0)
        if eps == 0:
            s[rows[:2]], wy[rows[0]], wy[rows[1]] = np.inf, np.nan, np.inf

    def close(got, want, half, least):
        assert np.array_equal(np.isnan(got), np.isnan(want))
        inf = np.isinf(want)
        assert np.array_equal(got[inf], want[inf])
        fine = np.isfinite(want)
        assert (np.abs(got[fine] - want[fine]) <= (half + tol * 1.01) * np.abs(want[fine]) + least).all()

    close(out["s"].astype(np.float64), s, 0, 2.0 ** -149)
    if copy is not None:
        close(y, wy, torch.finfo(copy).eps / 2, 2.0 ** -25 if copy == torch.float16 else 2.0 ** -134)
