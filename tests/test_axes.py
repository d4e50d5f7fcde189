"""The producer with several position axes (llattn_qk_norm_rope_axes, llattn_qkv_prepare_commit_axes).

A frequency turns by the position on its axis and every other operation is the one-axis producer's, so the outputs are put together from
that one's, run once for each axis: the same bits. That a wrong axis would show is checked on the inputs. Against the oracle in 64 bits the
tolerance is the one-axis test's: an fp16 ulp for 99.5 % of the values, 2^-7 of a rotated pair where the last bit of a sine crosses a bf16 border."""
import importlib

import numpy as np
import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def api(pkg):
    m = importlib.import_module(pkg.__name__ + ".api")
    m.lib()
    return m


def _inputs(api, T, naxes, seed):
    g = np.random.default_rng(seed)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
    qkv = (g.standard_normal((T, 3072)) * g.uniform(0.2, 3.0, (T, 1))).astype(np.float32)
    pos = g.integers(0, 40000, (naxes, T)).astype(np.int32)
    return dict(qkv=dev(qkv), pos=dev(pos), gq=dev(g.uniform(0.5, 1.5, 128).astype(np.float32)), gk=dev(g.uniform(0.5, 1.5, 128).astype(np.float32)), freq=dev(api.inv_freq()))


def _outputs(T):
    return [torch.full((T, n, 128), 7.0, dtype=torch.half, device="cuda") for n in (16, 4, 4)]


def _same(a, b):
    return torch.equal(a.view(torch.int16), b.view(torch.int16))


def _from_one_axis(api, i, axis_of):
    T = i["qkv"].shape[0]
    want = _outputs(T)
    for a in range(i["pos"].shape[0]):
        one = _outputs(T)
        api.qk_norm_rope(i["qkv"], i["pos"][a].contiguous(), i["gq"], i["gk"], 1e-6, i["freq"], *one)
        at = [f for f in range(32) if axis_of[f] == a]
        dims = torch.tensor(at + [f + 32 for f in at] + (list(range(64, 128)) if a == 0 else []), dtype=torch.long, device="cuda")
        for w, o in zip(want[:2], one[:2]):
            w[:, :, dims] = o[:, :, dims]
        want[2].copy_(one[2])
    return want


def test_rope_axes(api):
    assert api.rope_axes([32]) == bytes(32) and api.rope_axes([8, 12, 12]) == bytes([0] * 8 + [1] * 12 + [2] * 12)
    assert api.rope_axes([3, 1, 28], interleaved=True)[:8] == bytes([0, 1, 2, 0, 2, 0, 2, 2]) and api.rope_axes([0, 32]) == bytes([1] * 32)
    for bad in ([], [31], [33], [16, 17, -1], [8, 8, 8, 4, 4]):
        with pytest.raises(ValueError):
            api.rope_axes(bad)


@pytest.mark.gpu
@pytest.mark.parametrize("T,sections,interleaved", [(1, [8, 12, 12], False), (32, [16, 16], False), (33, [12, 10, 10], True), (7, [32], False), (300, [1, 2, 3, 26], False), (1153, [8, 8, 8, 8], True),
                                                    (9, [0, 32], False)])
def test_axes_are_the_one_axis_form_frequency_by_frequency(api, T, sections, interleaved):
    axis_of, i = api.rope_axes(sections, interleaved), _inputs(api, T, len(sections), T)
    want, got = _from_one_axis(api, i, axis_of), _outputs(T)
    api.qk_norm_rope_axes(i["qkv"], i["pos"], axis_of, i["gq"], i["gk"], 1e-6, i["freq"], *got)
    assert all(_same(a, b) for a, b in zip(got, want))
    if len(sections) > 1 and T > 8:                             # another assignment gives other values
        other = _outputs(T)
        api.qk_norm_rope_axes(i["qkv"], i["pos"], bytes((a + 1) % len(sections) for a in axis_of), i["gq"], i["gk"], 1e-6, i["freq"], *other)
        assert not _same(other[0], got[0]) and not _same(other[1], got[1]) and _same(other[2], got[2])


@pytest.mark.gpu
def test_axes_that_agree_are_the_one_axis_form(api):
    i = _inputs(api, 77, 1, 3)
    i["pos"] = i["pos"].expand(3, 77).contiguous()
    got, want = _outputs(77), _outputs(77)
    api.qk_norm_rope_axes(i["qkv"], i["pos"], api.rope_axes([8, 12, 12], True), i["gq"], i["gk"], 1e-6, i["freq"], *got)
    api.qk_norm_rope(i["qkv"], i["pos"][0].contiguous(), i["gq"], i["gk"], 1e-6, i["freq"], *want)
    assert all(_same(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_axes_against_the_oracle(api, orc):
    T, axis_of = 200, api.rope_axes([8, 12, 12])
    i = _inputs(api, T, 3, 4)
    got = _outputs(T)
    api.qk_norm_rope_axes(i["qkv"], i["pos"], axis_of, i["gq"], i["gk"], 1e-6, i["freq"], *got)
    x, pos = i["qkv"].double().cpu().numpy().reshape(T, 24, 128), i["pos"].cpu().numpy()
    n = x[:, :20] / np.sqrt((x[:, :20] ** 2).mean(-1, keepdims=True) + 1e-6) * np.concatenate([np.tile(i["gq"].cpu().numpy(), (16, 1)), np.tile(i["gk"].cpu().numpy(), (4, 1))])
    angle = (pos[list(axis_of)].T.astype(np.float32) * api.inv_freq()).astype(np.float32).astype(np.float64)
    bf = lambda a: torch.from_numpy(a).float().bfloat16().double().numpy()[:, None]
    cs, sn = bf(np.cos(angle)), bf(np.sin(angle))
    want = n.copy()
    want[..., :32], want[..., 32:64] = n[..., :32] * cs - n[..., 32:64] * sn, n[..., 32:64] * cs + n[..., :32] * sn
    for g, w in ((got[0], want[:, :16]), (got[1], want[:, 16:])):
        g = g.double().cpu().numpy()
        ulp = np.spacing(np.abs(w).astype(np.float16)).astype(np.float64)
        pair = np.abs(w[..., :32]) + np.abs(w[..., 32:64])
        bound = np.concatenate([pair, pair, np.zeros_like(pair), np.zeros_like(pair)], -1) * 2.0 ** -7 + 2 * ulp
        assert (np.abs(g - w) <= ulp).mean() >= 0.995 and (np.abs(g - w) <= bound).all()
    assert np.array_equal(got[2].cpu().numpy(), x[:, 20:].astype(np.float32).astype(np.float16))


@pytest.mark.gpu
@pytest.mark.parametrize("nb,paged", [(1, False), (5, True), (65, False), (66, True)])
def test_axes_with_the_commit(api, nb, paged):
    T, axis_of = 32 * nb, api.rope_axes([12, 10, 10], True)
    i = _inputs(api, T, 3, nb)
    want, got = _outputs(T), _outputs(T)
    caches = [torch.full((4, nb + 2, 4736), 9, dtype=torch.uint8, device="cuda") for _ in range(2)]
    args = (i["qkv"], i["pos"], axis_of, i["gq"], i["gk"], 1e-6, i["freq"])
    api.qk_norm_rope_axes(*args, *want)
    K, V = want[1].view(nb, 32, 4, 128), want[2].view(nb, 32, 4, 128)
    if paged:
        pages = torch.from_numpy(np.random.default_rng(nb).permutation(4 * (nb + 2))[:4 * nb].astype(np.int32).reshape(nb, 4)).cuda()
        api.kv_commit_paged(K, V, caches[0], pages)
        api.qkv_prepare_commit_axes(*args, *got, caches[1], pages=pages)
    else:
        api.kv_commit(K, V, caches[0], nb + 2, 1)
        api.qkv_prepare_commit_axes(*args, *got, caches[1], max_blocks=nb + 2, blk=1)
    assert all(_same(a, b) for a, b in zip(got, want)) and torch.equal(*caches)


def test_axes_refusals(api):
    L, ok = api.lib(), bytes([0] * 16 + [2] * 16)
    call = lambda naxes=3, axes=ok, pos=0x2000, k=0x8000, T=0: L.llattn_qk_norm_rope_axes(0x1000, pos, naxes, axes, 0x3000, 0x4000, 1e-6, 0x5000, 0x6000, k, 0x9000, T, None)
    fused = lambda naxes=3, axes=ok, nb=0, cache=0xA000, max_blocks=4, blk=0: L.llattn_qkv_prepare_commit_axes(
        0x1000, 0x2000, naxes, axes, 0x3000, 0x4000, 1e-6, 0x5000, 0x6000, 0x8000, 0x9000, nb, cache, None, max_blocks, blk, None)
    assert call() == fused() == api.OK
    for bad in (dict(naxes=0), dict(naxes=5), dict(naxes=2), dict(axes=None), dict(axes=bytes([0] * 31 + [3])), dict(axes=bytes([255] * 32))):
        assert call(**bad) == fused(**bad) == api.EINVAL
    assert call(pos=None) == call(T=-1) == call(k=0x8008) == api.EINVAL
    assert fused(cache=None) == fused(nb=-1) == fused(nb=5) == fused(nb=2, blk=3) == fused(cache=0xA004) == api.EINVAL


@pytest.mark.gpu
def test_axes_binding_refusals(api):
    i, ok = _inputs(api, 32, 3, 1), api.rope_axes([8, 12, 12])
    out = _outputs(32)
    args = dict(qkv=i["qkv"], pos=i["pos"], axis_of=ok, gq=i["gq"], gk=i["gk"], freq=i["freq"], q=out[0], k=out[1], v=out[2])
    call = lambda a: api.qk_norm_rope_axes(a["qkv"], a["pos"], a["axis_of"], a["gq"], a["gk"], 1e-6, a["freq"], a["q"], a["k"], a["v"])
    call(args)
    for bad in (dict(pos=i["pos"][:, :31]), dict(pos=i["pos"][0]), dict(pos=i["pos"].long()), dict(axis_of=ok[:31]), dict(qkv=i["qkv"].half()), dict(qkv=i["qkv"][:, :2048]), dict(gq=i["gq"][:64]),
                dict(freq=i["freq"].double()), dict(q=out[1]), dict(v=out[2].float()), dict(pos=i["pos"].cpu()), dict(pos=i["pos"].t().contiguous().t())):
        with pytest.raises(ValueError):
            call({**args, **bad})
    with pytest.raises(api.LlattnError):
        call({**args, "pos": i["pos"][:2].contiguous()})
    cache = torch.zeros((4, 1, 4736), dtype=torch.uint8, device="cuda")
    with pytest.raises(ValueError):
        api.qkv_prepare_commit_axes(*[args[k][:31] if k in ("qkv",) else i["pos"][:, :31].contiguous() if k == "pos" else args[k] for k in ("qkv", "pos", "axis_of", "gq", "gk")], 1e-6,
                                    i["freq"], *[o[:31] for o in out], cache, max_blocks=1)
