"""Arguments of llattn_add_norm_q8 that share memory: columns of one matrix may stand for the residual and its addend, columns that
overlap may not (warps would read what others write)."""
import importlib

import pytest

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
