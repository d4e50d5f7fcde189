"""The attention sub-layer of a batch of requests with adapters, as a serving program runs it: norm with int8 output, joint q|k|v projection and the
adapters of its q and v parts, producer with three position axes fused with the block commit, attention, output projection and its
adapters into the residual, and the next layer's norm with a 16-bit copy. Calls in a row, in a captured graph and on a stream of their own give
the bits of the calls one at a time; a captured step follows what its device arrays say when it is replayed."""
import importlib

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

NB, CTXB, LAYERS, RANK, NAD = 9, 3, 3, 24, 5
T = 32 * NB


@pytest.fixture(scope="module")
def api(pkg):
    return importlib.import_module(pkg.__name__ + ".api")


@pytest.fixture(scope="module")
def model(api, pkg):
    g = torch.Generator(device="cuda"); g.manual_seed(5)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")
    m = dict(h=rand(T, 2048), gain=1 + 0.1 * rand(2048), Wqkv=torch.from_numpy(pkg.workload.dense_weights(3072, 2048, 1)[0]).cuda(),
             Wo=torch.from_numpy(pkg.workload.dense_weights(2048, 2048, 2)[0]).cuda(), pos=torch.randint(0, 5000, (3, T), generator=g, device="cuda", dtype=torch.int32),
             hg=torch.ones(128, device="cuda"), freq=torch.from_numpy(api.inv_freq()).cuda(), axis_of=api.rope_axes([8, 12, 12]),
             caches=torch.zeros((NB, 4, CTXB + 1, 4736), dtype=torch.uint8, device="cuda"),
             A=[(rand(NAD, RANK, 2048) / 45).to(torch.bfloat16) for _ in range(3)], B=[(rand(NAD, rows, RANK) / 5).to(torch.bfloat16) for rows in (2048, 512, 2048)],
             ranks=torch.tensor([24, 8, 3, 17, 0], dtype=torch.int32, device="cuda"), scale=1 + 0.2 * rand(NAD))
    for i in range(NB):
        api.kv_commit(rand(CTXB, 32, 4, 128).half(), rand(CTXB, 32, 4, 128).half(), m["caches"][i], CTXB + 1, 0)
    m["pages"] = ((torch.arange(NB, device="cuda")[:, None] * 4 + torch.arange(4, device="cuda")) * (CTXB + 1) + CTXB).to(torch.int32).contiguous()
    return m


def _state(api, model):
    z = lambda *s, dtype=torch.float32: torch.zeros(s, dtype=dtype, device="cuda")
    st = dict(h=model["h"].clone(), caches=model["caches"].clone(), q8=z(T, 2048, dtype=torch.int8), s8=z(T, 16), sum8=z(T, 16, dtype=torch.int32), a8=z(T, 2048, dtype=torch.int8), as8=z(T, 16),
              asum8=z(T, 16, dtype=torch.int32), qkv=z(T, 3072), q=z(T, 16, 128, dtype=torch.half), k=z(T, 4, 128, dtype=torch.half), v=z(T, 4, 128, dtype=torch.half),
              y=z(T, 2048, dtype=torch.bfloat16), first=torch.tensor([0, 64, 64, 160, 224, 256], dtype=torch.int32, device="cuda"), adapter=torch.tensor([3, 1, 0, -1, 2], dtype=torch.int32, device="cuda"),
              A=[a.clone() for a in model["A"]], ctx=api.Context(0))
    pool = lambda i, row0: api.AdapterPool(st["A"][i], model["B"][i], row0=row0, scale=model["scale"], ranks=model["ranks"])
    st["qv"], st["o"] = api.adapter_pools([pool(0, 0), pool(1, 2560)]), api.adapter_pools([pool(2, 0)])
    st["plan"] = st["ctx"].plan([api.Seq(cache=st["caches"][i], nblocks=CTXB + 1, nq=1, q_first=i) for i in range(NB)])
    torch.cuda.synchronize()
    return st


def _step(api, m, st, between):
    delta = None
    for _ in range(LAYERS):
        api.add_norm_q8(st["h"], m["gain"], 1e-6, st["q8"], st["s8"], st["sum8"], delta=delta, y=st["y"]); between()
        st["qkv"].zero_(); between()
        api.dense_w4a8(m["Wqkv"], st["q8"], st["s8"], st["sum8"], st["qkv"]); between()
        api.adapters_w4a8(st["qv"], st["q8"], st["s8"], st["qkv"], st["first"], st["adapter"]); between()
        api.qkv_prepare_commit_axes(st["qkv"], m["pos"], m["axis_of"], m["hg"], m["hg"], 1e-6, m["freq"], st["q"], st["k"], st["v"], st["caches"], pages=m["pages"]); between()
        st["ctx"].attention(st["plan"], st["q"].view(NB, 32, 16, 128), st["k"].view(NB, 32, 4, 128), st["v"].view(NB, 32, 4, 128), q8=st["a8"], s8=st["as8"], sum8=st["asum8"]); between()
        api.dense_w4a8(m["Wo"], st["a8"], st["as8"], st["asum8"], st["h"]); between()
        api.adapters_w4a8(st["o"], st["a8"], st["as8"], st["h"], st["first"], st["adapter"]); between()
        delta = st["q"].view(T, 2048)            # in the place of an expert layer's fp16 output
    return [st[k].clone() for k in ("h", "q8", "s8", "sum8", "qkv", "q", "k", "v", "caches", "y")]


def _same(a, b):
    return all(torch.equal(x, y) and bool(torch.isfinite(x.float()).all()) for x, y in zip(a, b))


def test_steps_in_a_row_on_a_stream_and_in_a_graph(api, model):
    want = _step(api, model, _state(api, model), torch.cuda.synchronize)
    bare = _state(api, model)
    bare["adapter"].fill_(-1)
    assert not torch.equal(_step(api, model, bare, torch.cuda.synchronize)[0], want[0])
    for side in (False, True):
        st = _state(api, model)
        stream = torch.cuda.Stream() if side else torch.cuda.current_stream()
        with torch.cuda.stream(stream):
            torch.cuda._sleep(40_000_000)                      # everything is in the queue before its first kernel runs
            got = _step(api, model, st, lambda: None)
        torch.cuda.synchronize()
        assert _same(want, got)
    st, graph = _state(api, model), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _step(api, model, st, lambda: None)
    for _ in range(2):
        st["h"].copy_(model["h"]); st["caches"].copy_(model["caches"])
        graph.replay()
        torch.cuda.synchronize()
        assert _same(want, got)
    # the captured step reads its segments, adapters and weights when it runs
    other = _state(api, model)
    for s in (st, other):
        s["first"].copy_(torch.tensor([0, 32, 128, 128, 250, 288], dtype=torch.int32)); s["adapter"].copy_(torch.tensor([1, 4, 2, 3, 3], dtype=torch.int32))
        s["A"][2].mul_(2)
    st["h"].copy_(model["h"]); st["caches"].copy_(model["caches"])
    graph.replay()
    torch.cuda.synchronize()
    again = _step(api, model, other, torch.cuda.synchronize)
    assert _same(again, got) and not torch.equal(again[0], want[0])
    assert st["ctx"].device_status() == 0 and api.dense_status() == 0


def test_two_graphs_on_two_streams(api, model):
    """Nothing of these operators is shared between calls: two captured steps that run at once give their own results."""
    states, graphs, outs = [], [], []
    for k in range(2):
        st = _state(api, model)
        st["adapter"].copy_(torch.tensor([k, 2, 1 - k, 3, -k], dtype=torch.int32))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(4):
                api.add_norm_q8(st["h"], model["gain"], 1e-6, st["q8"], st["s8"], st["sum8"], y=st["y"])
                api.adapters_w4a8(st["qv"], st["q8"], st["s8"], st["qkv"], st["first"], st["adapter"])
                api.adapters_w4a8(st["o"], st["q8"], st["s8"], st["h"], st["first"], st["adapter"])
                api.qk_norm_rope_axes(st["qkv"], model["pos"], model["axis_of"], model["hg"], model["hg"], 1e-6, model["freq"], st["q"], st["k"], st["v"])
        states.append(st); graphs.append(graph)
    def run(apart):
        for st in states:
            st["h"].copy_(model["h"]); st["qkv"].zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
            if apart:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        return [st[k].clone() for st in states for k in ("h", "q8", "qkv", "q", "y")]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    want = run(True)
    for _ in range(5):
        assert _same(want, run(False))
    assert not torch.equal(want[0], want[5])
