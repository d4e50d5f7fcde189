"""Segments whose bounds go back (llattn_adapters_w4a8): a bound below an earlier one counts as that one, so a token belongs to the first segment that
reaches it and no tile is lost. Small whole numbers and powers of two: nothing is rounded, and the results have to be equal."""
import importlib

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
K, RANK, N, ROWS = 256, 8, 5, 36


@pytest.fixture(scope="module")
def api(pkg):
    m = importlib.import_module(pkg.__name__ + ".api")
    m.lib()
    return m


def _call(api, orc, T, first, adapter, rank=RANK):
    g = torch.Generator(device="cuda"); g.manual_seed(T + len(adapter))
    small = lambda lo, hi, *s: torch.randint(lo, hi, s, generator=g, device="cuda")
    q, s, Y = small(-3, 4, T, K).to(torch.int8), 2.0 ** small(-1, 2, T, K // 128), small(-9, 10, T, ROWS).float()
    A, B = small(-2, 3, N, rank, K).half(), small(-3, 4, N, ROWS, rank).half()
    at = torch.tensor([orc.frag_pos(c) for c in range(K)], device="cuda")
    x = q[:, at].double() * s.double().repeat_interleave(128, 1)
    want = Y.double()
    ends = np.maximum.accumulate(np.clip(np.asarray(first), 0, T))
    whose = np.full(T, -1)
    for t0, t1, a in zip(ends[:-1], ends[1:], adapter):
        whose[t0:t1] = a
    for a in range(N):
        mine = torch.from_numpy(np.flatnonzero(whose == a)).cuda()
        want[mine] += x[mine] @ A[a].double().t() @ B[a].double().t()
    assert float(want.abs().max()) < 2 ** 21
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    api.adapters_w4a8(api.adapter_pools([api.AdapterPool(A, B)]), q, s, Y, i32(first), i32(adapter))
    return Y, want


@pytest.mark.parametrize("T,first,adapter", [
    (150, [0, 100, 50, 150], [0, 1, 2]), (150, [0, 100, 50, 40, 120, 150], [0, 1, 2, 3, 4]), (150, [40, 10, 60, 60, 20, 90, 0, 150], [0, 1, 2, 3, 4, 0, 1]), (64, [0, 64, 0, 64, 0, 64], [0, 1, 2, 3, 4]),
    (32, [500, 0, 32], [0, 1]), (32, [0, 500, 0, 32], [3, 1, 2]), (90, [0, 31, -2 ** 31, 33, 2 ** 31 - 1, 7], [0, 1, 2, 3, 4]), (1, [1, 0, 1], [0, 1])])
def test_bounds_that_go_back(api, orc, T, first, adapter):
    got, want = _call(api, orc, T, first, adapter)
    assert torch.equal(got.double(), want)


@pytest.mark.parametrize("T,nseg,rank", [(700, 31, 8), (700, 32, 8), (700, 33, 64), (500, 64, 24), (3000, 700, 8), (97, 1500, 64)])
@pytest.mark.parametrize("kind", ["any", "one", "runs"])
def test_many_bounds_that_go_back(api, orc, T, nseg, rank, kind):
    """Bounds in any order; in order but for one; runs that each begin again."""
    r = np.random.default_rng(nseg)
    first = r.integers(-T // 4, T + T // 4, nseg + 1)
    if kind != "any":
        first = np.sort(first)
        if kind == "one":
            first[nseg // 2] = 0
        else:
            first = np.concatenate([first[::3], first[1::3], first[2::3]])
    got, want = _call(api, orc, T, [int(v) for v in first], [int(v) for v in r.integers(-1, N, nseg)], rank)
    assert torch.equal(got.double(), want)


@pytest.mark.parametrize("rank", [8, 64])
def test_the_most_segments(api, orc, rank):
    """65,536 segments of one token, a few of them empty and one bound far back."""
    T = nseg = 1 << 16
    first = list(range(nseg + 1))
    first[7] = first[9] = 9
    first[40000] = 3
    got, want = _call(api, orc, T, first, [i % (N + 1) - 1 for i in range(nseg)], rank)
    assert torch.equal(got.double(), want)
