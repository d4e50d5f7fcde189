"""What the binding of the newer operators hands to the C entry points, with CPU tensors and a recording library in the place of the real one: no
launch, so calls whose arguments are wrong can be made."""
import gc
import importlib

import numpy as np
import pytest

torch = pytest.importorskip("torch")


class Recorder:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *args: self.calls.append((name, args)) or 0


@pytest.fixture
def api(pkg, monkeypatch):
    m = importlib.import_module(pkg.__name__ + ".api")
    types = {torch.float32: m.F32, torch.float16: m.F16, torch.bfloat16: m.BF16}
    rec = Recorder()
    monkeypatch.setattr(m, "_torch_of", (torch.float32, torch.float16, torch.int8, torch.int32, types, lambda: -1, lambda dev: 0))      # -1: the CPU's index
    monkeypatch.setattr(m, "_lib", rec)
    m.recorder = rec
    return m


def _producer(axes=3, T=32):
    z = lambda *s, dtype=torch.float32: torch.zeros(s, dtype=dtype)
    return dict(qkv=z(T, 6 * 512), pos=z(axes, T, dtype=torch.int32), axis_of=bytes([0] * 8 + [1] * 12 + [2] * 12), gq=z(128), gk=z(128), eps=1e-6, inv_freq_t=z(32),
                q=z(T, 16, 128, dtype=torch.half), k=z(T, 4, 128, dtype=torch.half), v=z(T, 4, 128, dtype=torch.half))


@pytest.mark.parametrize("dtype", [torch.float32, torch.uint32, torch.int64, torch.int16])
def test_pages_of_another_type_are_refused(api, dtype):
    """Page indices are read as int32: the bits of floats would be indices far outside the pool."""
    args, cache = _producer(), torch.zeros((4, 4736), dtype=torch.uint8)
    pages = torch.arange(4).reshape(1, 4)
    api.qkv_prepare_commit_axes(**args, cache=cache, pages=pages.to(torch.int32))
    assert [name for name, _ in api.recorder.calls] == ["llattn_qkv_prepare_commit_axes"]
    with pytest.raises(ValueError):
        api.qkv_prepare_commit_axes(**args, cache=cache, pages=pages.to(dtype))
    assert len(api.recorder.calls) == 1


@pytest.mark.parametrize("as_given", [bytes, bytearray, list, tuple, np.array, lambda a: np.array(a, np.int32), lambda a: np.array(a, np.uint8), torch.tensor])
def test_axes_may_come_as_any_sequence(api, as_given):
    """The axis of a frequency is what the sequence has there, not what the memory behind it has: arrays of wider numbers too."""
    axes = [0, 2, 1, 1] * 8
    args = dict(_producer(), axis_of=as_given(axes))
    api.qk_norm_rope_axes(**args)
    api.qkv_prepare_commit_axes(**args, cache=torch.zeros((4, 4736), dtype=torch.uint8), max_blocks=1)
    assert [a[3] for _, a in api.recorder.calls] == [bytes(axes)] * 2


@pytest.mark.parametrize("bad", [np.arange(32) - 1, [256] * 32, np.full(32, 0.5), list(range(31))])
def test_axes_that_are_no_axes_are_refused(api, bad):
    with pytest.raises((ValueError, TypeError)):
        api.qk_norm_rope_axes(**dict(_producer(), axis_of=bad))
    assert api.recorder.calls == []


@pytest.mark.parametrize("name", ["A", "B", "scale", "ranks"])
@pytest.mark.parametrize("how", ["attribute", "data", "pool"])
def test_pools_keep_the_memory_they_call_with(api, name, how):
    """The addresses of a call are those of the tensors at the check. A pool's field, a tensor's memory or the list of pools may change behind it: what
    the addresses stand for lives as long as the pools, and takes the pools' next calls."""
    def tensors():
        return dict(A=torch.ones((3, 8, 128), dtype=torch.half), B=torch.ones((3, 4, 8), dtype=torch.half), scale=torch.ones(3), ranks=torch.ones(3, dtype=torch.int32))
    first = tensors()
    at = first[name].data_ptr()
    pools = api.adapter_pools([api.AdapterPool(**first)])
    pool = pools.pools[0]
    if how == "attribute":
        setattr(pool, name, tensors()[name])
    elif how == "data":
        first[name].data = tensors()[name]
    else:
        pools.pools.clear()
    del first, pool
    gc.collect()
    assert getattr(pools._c[0], name) == at
    assert any(t.data_ptr() == at for t in _held(pools)), "the memory behind a call's address is not held"
    z = lambda *s, dtype=torch.float32: torch.zeros(s, dtype=dtype)
    api.adapters_w4a8(pools, z(4, 128, dtype=torch.int8), z(4, 1), z(4, 4), z(2, dtype=torch.int32), z(1, dtype=torch.int32))
    assert [n for n, _ in api.recorder.calls] == ["llattn_adapters_w4a8"]


def _held(pools):
    """The tensors that can be reached from the pools."""
    seen, todo, found = set(), [vars(pools)], []
    while todo:
        x = todo.pop()
        if id(x) in seen:
            continue
        seen.add(id(x))
        if torch.is_tensor(x):
            found.append(x)
        elif isinstance(x, dict):
            todo += x.values()
        elif isinstance(x, (list, tuple)):
            todo += x
        elif hasattr(x, "A"):
            todo.append(vars(x))
    return found
