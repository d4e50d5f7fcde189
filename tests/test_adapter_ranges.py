"""The inner sums of a token's ranks keep their 24 bits on the way into the second product, however far the ranks are from one another, and fp16
and bf16 weights are multiplied as they are (llattn_adapters_w4a8).

Far ranks: the ranks of group g read only the activations of group g, whose scale is 2^-spread g / 3, and row i of B takes the ranks of one group only. So a row's
result is that group's alone, and its bound has nothing of the larger ones. An inner sum: a group's 128 exact products in eight instructions of
sixteen, four roundings of 2^-23 each, a multiply-add for each group and three more operations, relative to the sum of absolute values. The second product:
H in two
parts of tf32 is off by 2^-23 at most (11 bits each, rounded to nearest), in three of bf16 by less; sixteen ranks are four instructions at most, two eights for each of two parts,
of four roundings of 2^-23 each; one addition of parts, and one of 2^-24 into Y."""
import importlib

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
GROUPS = 4
K = 128 * GROUPS


@pytest.fixture(scope="module")
def api(pkg):
    m = importlib.import_module(pkg.__name__ + ".api")
    m.lib()
    return m


def _run(api, orc, q, s, A, B, rows, scale=None):
    """Y of zeros behind one segment of all tokens; q in logical order."""
    at = [orc.frag_pos(c) for c in range(q.shape[1])]
    qf = np.zeros_like(q)
    qf[:, at] = q
    T = q.shape[0]
    Y = torch.zeros((T, rows), device="cuda")
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    api.adapters_w4a8(api.adapter_pools([api.AdapterPool(A[None].cuda(), B[None].cuda(), scale=scale)]), torch.from_numpy(qf).cuda(), torch.from_numpy(s).cuda(), Y, i32([0, T]), i32([0]))
    return Y.double().cpu().numpy()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rank", [8, 16, 32, 64, 128])
@pytest.mark.parametrize("T", [1, 45, 5000])
@pytest.mark.parametrize("spread", [0, 24, 48, 84, 144])
def test_ranks_far_apart(api, orc, T, rank, dtype, spread):
    g, rows = np.random.default_rng(spread + rank + T), 68
    q = g.integers(-127, 128, (T, K)).astype(np.int8)
    s = (2.0 ** (spread // 2 - spread // 3 * np.arange(GROUPS)) * np.exp(0.3 * g.standard_normal((T, GROUPS)))).astype(np.float32)
    mine = np.arange(rank) % GROUPS
    A = g.standard_normal((rank, K)) / 16 * (mine[:, None] == np.arange(K) // 128)
    B = g.standard_normal((rows, rank)) * (mine == np.arange(rows)[:, None] % GROUPS)
    A, B = torch.from_numpy(A).to(dtype), torch.from_numpy(B).to(dtype)
    got = _run(api, orc, q, s, A, B, rows)
    x, A64, B64 = q.astype(np.float64) * np.repeat(s.astype(np.float64), 128, 1), A.double().numpy(), B.double().numpy()
    H, mag = x @ A64.T, np.abs(x) @ np.abs(A64).T
    off = (8 * 4 + GROUPS + 3) * 2.0 ** -23 * mag + 2.0 ** -23 * np.abs(H)
    want, big = H @ B64.T, (np.abs(H) + off) @ np.abs(B64).T
    bound = off @ np.abs(B64).T + (-(-rank // 16) * 4 * 4 + 2) * 2.0 ** -23 * big + 2.0 ** -24 * np.abs(want)
    assert (np.abs(got - want) <= bound).all(), [float((np.abs(got - want) / np.maximum(bound, 1e-300))[:, i::GROUPS].max()) for i in range(GROUPS)]
    # The bound says something: a group that is lost is off by its own size. Of 128 ranks 32 are a group's, with sums of 128 terms whose absolute values add up to
    # some 14 times the sum, so about (39 * 14 + 131) 2^-23 * 8 = 6e-4 of a row's size.
    assert np.median(bound / np.maximum(np.abs(want), 1e-300)) < 2.0 ** -8


@pytest.mark.parametrize("dtype,bits,low", [(F16, 11, 0), (F16, 10, -24), (BF16, 8, 0), (BF16, 8, -60), (BF16, 8, 40)])
@pytest.mark.parametrize("rank", [8, 32, 40, 64, 128])
def test_every_bit_of_the_weights(api, orc, rank, dtype, bits, low):
    """B of all numbers of its bits, of fp16 the smallest ones too (subnormal), inner sums of small whole numbers: nothing is rounded."""
    T, rows = 70, 132
    g = np.random.default_rng(rank + bits)
    q = g.integers(-2, 3, (T, K)).astype(np.int8)
    A = (g.integers(-1, 2, (rank, K)) * (g.random((rank, K)) < 0.02)).astype(np.float64)
    B = g.integers(-2 ** bits + 1, 2 ** bits, (rows, rank)) * 2.0 ** low
    B[0], B[1] = (2 ** bits - 1) * 2.0 ** low, -2.0 ** low
    A, B = torch.from_numpy(A).to(dtype), torch.from_numpy(B).to(dtype)
    assert torch.equal(B.double() * 2.0 ** -low, (B.double() * 2.0 ** -low).round())
    got = _run(api, orc, q, np.ones((T, GROUPS), np.float32), A, B, rows)
    want = q.astype(np.float64) @ A.double().numpy().T @ B.double().numpy().T
    assert np.abs(want).max() * 2.0 ** -low < 2 ** 23
    assert np.array_equal(got, want)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rank", [16, 64])
def test_infinite_weights_stay_in_their_rows(api, orc, rank, dtype):
    """An infinity or NaN in B makes its row not finite and leaves the other rows alone."""
    T, rows = 33, 64
    g = np.random.default_rng(3)
    q, s = g.integers(1, 100, (T, K)).astype(np.int8), np.ones((T, GROUPS), np.float32)
    A, B = torch.from_numpy(g.random((rank, K)) + 0.1).to(dtype), torch.from_numpy(g.standard_normal((rows, rank))).to(dtype)
    want = _run(api, orc, q, s, A, B, rows)
    B[5, 3], B[9, rank - 1], B[20, 0] = float("inf"), float("-inf"), float("nan")
    got = _run(api, orc, q, s, A, B, rows)
    bad = [5, 9, 20]
    assert not np.isfinite(got[:, bad]).any() and np.array_equal(np.delete(got, bad, 1), np.delete(want, bad, 1))
