"""Operators around the projection and the producer, measured through the public Python binding:

  norm      `add_norm_q8`: the residual takes a sub-layer's output, is normalised (root mean square, learned gain) and leaves as the
            int8 activations that the W4.A8 projection reads: codes, a scale and a code sum for each group of 128; for a second reader
            (a router, say) in 16 bits too
  adapters  `adapters_w4a8`: low-rank adapters of many requests, added to a shared projection's output from the same int8 activations
  axes      `qk_norm_rope_axes`: the producer of the attention inputs with several position axes (time, height, width)

With `own` false the same outputs come from elementary torch operations in 32 bits, rounded once at the end.

The int8 codes and their sums are compared as the whole numbers they are: a code is rint(t / e) of two numbers that single IEEE
operations fix (t = (x + d) * gain, e = max|t| / 127 of the group), so both sides have the same ones to the last bit.
"""
import importlib
import math
import random

import torch

own = False

HEADS, KV_HEADS, D = 16, 4, 128          # query and kv heads of the model, head dim; its hidden size is 2048
QKV = (HEADS + 2 * KV_HEADS) * D
EPS = 1e-6
THETA = 3e6
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "none": None}


# ---------------------------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # one token behind a sub-layer: the smallest call, all latency
        dict(name="norm 1 x 2048", op="norm", tokens=1, K=2048, delta="f16", y="none"),
        # one query block at the model's width; the projection has added into the residual already, so nothing is added here
        dict(name="norm 32 x 2048", op="norm", tokens=32, K=2048, delta="none", y="none"),
        # an odd batch at a wider model, the expert layer's bf16 output added, the router's 16-bit copy written
        dict(name="norm 515 x 5120", op="norm", tokens=515, K=5120, delta="bf16", y="bf16"),
        # a prefill pass over several prompts, the last block not full: fp32 sub-layer output
        dict(name="norm 8191 x 2048", op="norm", tokens=8191, K=2048, delta="f32", y="none"),
        # a single token of one request with a small adapter
        dict(name="adapters 1", op="adapters", tokens=1, segs=1, n=4, rank=8, mixed=False, bare=False, ragged=False, dtype="f16", K=2048, rows=2048, slices=1),
        # one user's query block
        dict(name="adapters 32", op="adapters", tokens=32, segs=1, n=16, rank=16, mixed=False, bare=False, ragged=False, dtype="bf16", K=2048, rows=2048, slices=1),
        # a full serving batch: 64 requests of a 32-token block, each with an adapter of its own
        dict(name="adapters 64 x 32", op="adapters", tokens=2048, segs=64, n=64, rank=16, mixed=False, bare=False, ragged=False, dtype="bf16", K=2048, rows=2048, slices=1),
        # requests of any length, some without an adapter, ranks of all sizes; q and v of the joint q|k|v projection have adapters
        dict(name="adapters 777 ragged q+v", op="adapters", tokens=777, segs=23, n=9, rank=64, mixed=True, bare=True, ragged=True, dtype="f16", K=2048, rows=2048, slices=2),
        # one long prompt under a large adapter
        dict(name="adapters 4096 r64", op="adapters", tokens=4096, segs=1, n=2, rank=64, mixed=False, bare=False, ragged=False, dtype="bf16", K=2048, rows=2048, slices=1),
        # one query block of text behind images
        dict(name="axes 32", op="axes", tokens=32, axes=3, split="8,12,12", interleaved=False),
        # an image's patches in a prompt, an odd number of them
        dict(name="axes 1153", op="axes", tokens=1153, axes=3, split="8,12,12", interleaved=False),
        # a video's, frequencies dealt to the axes in turn
        dict(name="axes 8192 interleaved", op="axes", tokens=8192, axes=3, split="12,10,10", interleaved=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng: random.Random):
    op = rng.choice(["norm", "adapters", "adapters", "axes"])
    if op == "norm":
        K = 128 * _log_int(rng, 1, 64)
        return dict(op=op, tokens=_log_int(rng, 1, min(8191, (8191 * 2048) // K)), K=K, delta=rng.choice(["none", "f32", "f16", "bf16"]), y=rng.choice(["none", "none", "f16", "bf16"]))
    if op == "axes":
        axes = rng.randint(2, 4)
        cuts = sorted(rng.sample(range(1, 32), axes - 1))
        split = ",".join(str(b - a) for a, b in zip([0] + cuts, cuts + [32]))
        return dict(op=op, tokens=_log_int(rng, 1, 8191), axes=axes, split=split, interleaved=rng.random() < 0.5)
    tokens = _log_int(rng, 1, 4095)
    return dict(op=op, tokens=tokens, segs=_log_int(rng, 1, min(128, tokens)), n=_log_int(rng, 1, 64), rank=8 * _log_int(rng, 1, 8), mixed=rng.random() < 0.5,
                bare=rng.random() < 0.3, ragged=rng.random() < 0.6, dtype=rng.choice(["f16", "bf16"]), K=128 * rng.randint(4, 16), rows=512 * rng.randint(1, 4),
                slices=rng.choice([1, 2]))


# --------------------------------------------------------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _logical(K):
    """Where each of a row's K values is in the fragment order that the int8 activations have inside every group of 128."""
    r = torch.arange(K, device="cuda")
    c = r % 128
    return r - c + 32 * (c // 4 % 4) + 8 * (c // 32) + 4 * (c // 16 % 2) + c % 4


def _axis_of(case):
    """The axis of each of the 32 frequencies: a run of them for each axis, or dealt in turn while an axis has some left."""
    left = [int(x) for x in case["split"].split(",")]
    if not case["interleaved"]:
        return [a for a, n in enumerate(left) for _ in range(n)]
    got = []
    while len(got) < 32:
        for a in range(len(left)):
            if left[a]:
                left[a] -= 1
                got.append(a)
    return got


def _slices(case):
    """(first row, rows) of each adapted part of the output, and the output's width: all of it, or q and v of a q|k|v output whose k and
    v are a quarter of q."""
    rows = case["rows"]
    return ([(0, rows)], rows) if case["slices"] == 1 else ([(0, rows), (rows + rows // 4, rows // 4)], rows + rows // 2)


def _segments(case, seed):
    """First tokens of the segments and where the last ends. Ragged: any lengths, empty ones among them, tokens left over behind the last."""
    T, n = case["tokens"], case["segs"]
    if not case["ragged"]:
        return [i * T // n for i in range(n)] + [T]
    rng = random.Random(seed)
    return [0] + sorted(rng.randint(0, T) for _ in range(n))


def _adapter_of(case, i):
    return -1 if case["bare"] and i % 4 == 3 else i * 7 % case["n"]


def _rank_of(case, i):
    return case["rank"] - 5 * i % case["rank"] if case["mixed"] else case["rank"]


def prepare(case, seed):
    g = _gen(seed)
    rand = lambda *shape: torch.randn(shape, generator=g, device="cuda")
    st = dict(case=dict(case))
    T = case["tokens"]
    if case["op"] == "norm":
        K = case["K"]
        x = rand(T, K) * torch.exp(0.5 * rand(T, 1))
        x[:, torch.randint(0, K, (max(1, K // 512),), generator=g, device="cuda")] *= 30.0      # a residual stream has a few large channels
        st.update(x=x, gain=1.0 + 0.1 * rand(K), delta=None if case["delta"] == "none" else rand(T, K).to(TYPES[case["delta"]]), step=torch.tensor(127.0, device="cuda"),
                  q=torch.zeros((T, K), dtype=torch.int8, device="cuda"), s=torch.zeros((T, K // 128), device="cuda"),
                  qsum=torch.zeros((T, K // 128), dtype=torch.int32, device="cuda"), at=_logical(K),
                  y=None if case["y"] == "none" else torch.zeros((T, K), dtype=TYPES[case["y"]], device="cuda"))
    elif case["op"] == "adapters":
        K, n, rank = case["K"], case["n"], case["rank"]
        parts, width = _slices(case)
        first = _segments(case, seed)
        st.update(q=torch.randint(-127, 128, (T, K), generator=g, device="cuda", dtype=torch.int8), s=0.02 * torch.exp(0.5 * rand(T, K // 128)), Y=rand(T, width), at=_logical(K),
                  first=torch.tensor(first, dtype=torch.int32, device="cuda"),
                  adapter=torch.tensor([_adapter_of(case, i) for i in range(case["segs"])], dtype=torch.int32, device="cuda"),
                  ranks=torch.tensor([_rank_of(case, i) for i in range(n)], dtype=torch.int32, device="cuda"),
                  scale=0.5 + torch.rand((n,), generator=g, device="cuda"),
                  A=[(rand(n, rank, K) / math.sqrt(K)).to(TYPES[case["dtype"]]) for _ in parts],
                  B=[(rand(n, rows, rank) / math.sqrt(rank)).to(TYPES[case["dtype"]]) for _, rows in parts])
        if own:                              # what a serving program makes once, when it loads its adapters
            api = importlib.import_module("llada2-orin-cuda_b200.api")
            st["pools"] = api.adapter_pools([api.AdapterPool(A, B, row0=row0, scale=st["scale"], ranks=st["ranks"]) for A, B, (row0, _) in zip(st["A"], st["B"], parts)])
    else:
        # a prompt as a model with images has it: text tokens have one position on all axes, a picture's patches a time, a row and a column
        rng = random.Random(seed)
        t, pos = rng.randint(0, 16384), []
        while len(pos) < T:
            if rng.random() < 0.5:
                n = rng.randint(1, 64)
                pos += [(t + i,) * case["axes"] for i in range(n)]
                t += n
            else:
                h, w = rng.randint(4, 32), rng.randint(4, 32)
                pos += [(t, t + i, t + j, t + (i + j) // 2)[:case["axes"]] for i in range(h) for j in range(w)]
                t += max(h, w)
        st.update(qkv=rand(T, QKV) * torch.exp(0.5 * rand(T, 1)), pos=torch.tensor(pos[:T], dtype=torch.int32).t().contiguous().cuda(),
                  gq=1.0 + 0.1 * rand(D), gk=1.0 + 0.1 * rand(D), freq=torch.tensor([THETA ** (-i / 32) for i in range(32)], device="cuda"),
                  q=torch.zeros((T, HEADS, D), dtype=torch.half, device="cuda"), k=torch.zeros((T, KV_HEADS, D), dtype=torch.half, device="cuda"),
                  v=torch.zeros((T, KV_HEADS, D), dtype=torch.half, device="cuda"), axis=torch.tensor(_axis_of(case), device="cuda"), axis_of=bytes(_axis_of(case)))
    torch.cuda.synchronize()
    return st


# ----------------------------------------------------------------------------------------------------------------- pass

def _norm_outputs(st, q, s, qsum, y):
    """What a pass writes: the residual where something was added to it, the activations, the 16-bit copy where one is asked for."""
    out = {"q": q, "s": s, "sum": qsum}
    if st["delta"] is not None:
        out["x"] = st["x"]
    if y is not None:
        out["y"] = y
    return out


def _plain_norm(st):
    x, K = st["x"], st["case"]["K"]
    v = x if st["delta"] is None else x.add_(st["delta"].float())
    r = torch.rsqrt((v * v).mean(1, keepdim=True) + EPS)
    t = v * st["gain"]
    step = (t.abs().view(-1, K // 128, 128).amax(2) / st["step"]).clamp(min=1e-30)          # by a tensor: a number would be multiplied by its reciprocal
    codes = torch.round(t.view(-1, K // 128, 128) / step[..., None]).clamp(-127, 127)
    q = torch.empty_like(st["q"])
    q[:, st["at"]] = codes.view(-1, K).to(torch.int8)
    return _norm_outputs(st, q, step * r, codes.sum(2).to(torch.int32), None if st["y"] is None else (t * r).to(st["y"].dtype))


def _plain_adapters(st):
    case = st["case"]
    T, K, n, rank = case["tokens"], case["K"], case["n"], case["rank"]
    x = (st["q"][:, st["at"]].float().view(T, K // 128, 128) * st["s"][..., None]).view(T, K)
    token = torch.arange(T, device="cuda", dtype=torch.int32)
    seg = torch.searchsorted(st["first"][1:].contiguous(), token, right=True)
    whose = torch.where(seg < case["segs"], st["adapter"][seg.clamp(max=case["segs"] - 1)], -1)
    # the products with all adapters at once, of which a token keeps its own
    mine = (whose[:, None] == torch.arange(n, device="cuda"))[..., None] & (torch.arange(rank, device="cuda") < st["ranks"][:, None])
    for A, B, (row0, rows) in zip(st["A"], st["B"], _slices(case)[0]):
        H = (x @ A.float().view(n * rank, K).t()).view(T, n, rank) * st["scale"][:, None]
        H = torch.where(mine, H, 0.0).view(T, n * rank)
        st["Y"][:, row0:row0 + rows] += H @ B.float().transpose(1, 2).reshape(n * rank, rows)
    return {"Y": st["Y"]}


def _plain_axes(st):
    T = st["case"]["tokens"]
    x = st["qkv"].view(T, HEADS + 2 * KV_HEADS, D)
    n = x[:, :HEADS + KV_HEADS]
    gain = torch.cat([st["gq"].expand(HEADS, D), st["gk"].expand(KV_HEADS, D)])
    n = n * torch.rsqrt((n * n).mean(2, keepdim=True) + EPS) * gain
    # the angle is a 32-bit product, as models compute it; its cosine and sine are rounded to bf16
    angle = (st["pos"][st["axis"]].t().float() * st["freq"]).double()
    cs, sn = angle.cos().float().bfloat16().float()[:, None], angle.sin().float().bfloat16().float()[:, None]
    a, b = n[..., :32], n[..., 32:64]
    n = torch.cat([a * cs - b * sn, b * cs + a * sn, n[..., 64:]], 2)
    return {"q": n[:, :HEADS].half(), "k": n[:, HEADS:].half(), "v": x[:, HEADS + KV_HEADS:].half()}


def run(st):
    op = st["case"]["op"]
    if own:
        api = importlib.import_module("llada2-orin-cuda_b200.api")
        if op == "norm":
            api.add_norm_q8(st["x"], st["gain"], EPS, st["q"], st["s"], st["qsum"], delta=st["delta"], y=st["y"])
            return _norm_outputs(st, st["q"], st["s"], st["qsum"], st["y"])
        if op == "adapters":
            api.adapters_w4a8(st["pools"], st["q"], st["s"], st["Y"], st["first"], st["adapter"])
            return {"Y": st["Y"]}
        api.qk_norm_rope_axes(st["qkv"], st["pos"], st["axis_of"], st["gq"], st["gk"], EPS, st["freq"], st["q"], st["k"], st["v"])
        return {"q": st["q"], "k": st["k"], "v": st["v"]}
    return _plain_norm(st) if op == "norm" else _plain_adapters(st) if op == "adapters" else _plain_axes(st)


# ------------------------------------------------------------------------------------------------------- work, exact values

def work(case):
    T = case["tokens"]
    if case["op"] == "norm":
        K = case["K"]
        size = {"none": 0, "f16": 2, "bf16": 2, "f32": 4}
        a_value = 4 + 1 + size[case["y"]] + (4 + size[case["delta"]] if case["delta"] != "none" else 0)      # x is written where something is added
        return {"bytes": T * K * a_value + 8 * T * (K // 128) + 4 * K, "flops": 6 * T * K}
    if case["op"] == "axes":
        return {"bytes": T * (6 * QKV + 4 * case["axes"]), "flops": 8 * T * (HEADS + KV_HEADS) * D}
    K, segs = case["K"], case["segs"]
    cols = sum(rows for _, rows in _slices(case)[0])
    used = [_adapter_of(case, i) for i in range(segs)]
    share = sum(a >= 0 for a in used) / segs                                    # of the tokens: segments are alike in the mean
    if case["ragged"]:
        share *= segs / (segs + 1)                                              # and as much is left over behind the last
    read = 2 * len(_slices(case)[0]) * K * sum(_rank_of(case, a) for a in set(used) if a >= 0) + 2 * cols * sum(_rank_of(case, a) for a in set(used) if a >= 0)
    rank = sum(_rank_of(case, a) for a in used if a >= 0) / max(1, sum(a >= 0 for a in used))
    return {"bytes": share * T * (K + K // 32 + 8 * cols) + read, "flops": 2 * share * T * rank * (len(_slices(case)[0]) * K + cols)}


def exact(case, seed):
    """The formulas in 64 bits. The int8 codes have no such value: they are whole numbers."""
    st = prepare(case, seed)
    T = case["tokens"]
    if case["op"] == "norm":
        v = st["x"].double()
        if st["delta"] is not None:
            v = v + st["delta"].double()
        inv = 1.0 / torch.sqrt(v.pow(2).sum(1) / case["K"] + EPS)
        u = v * st["gain"].double()
        s = torch.stack([g.abs().max(1).values for g in u.split(128, 1)], 1) / 127.0 * inv[:, None]
        return {"x": None if st["delta"] is None else v, "q": None, "s": s, "sum": None, "y": None if st["y"] is None else u * inv[:, None]}
    if case["op"] == "adapters":
        Y = st["Y"].double()
        x = torch.zeros((T, case["K"]), dtype=torch.float64, device="cuda")
        for i in range(case["K"]):
            c = i % 128
            x[:, i] = st["q"][:, i - c + 32 * (c // 4 % 4) + 8 * (c // 32) + 4 * (c // 16 % 2) + c % 4].double() * st["s"][:, i // 128].double()
        first = _segments(case, seed)
        for i in range(case["segs"]):
            a, t0, t1 = _adapter_of(case, i), first[i], first[i + 1]
            if a >= 0 and t1 > t0:
                r = _rank_of(case, a)
                for A, B, (row0, rows) in zip(st["A"], st["B"], _slices(case)[0]):
                    Y[t0:t1, row0:row0 + rows] += float(st["scale"][a]) * ((x[t0:t1] @ A[a, :r].double().t()) @ B[a, :, :r].double().t())
        return {"Y": Y}
    x = st["qkv"].double().view(T, -1, D)
    cos, sin = [], []
    for i, a in enumerate(_axis_of(case)):
        angle = (st["pos"][a].float() * st["freq"][i]).double()
        cos.append(torch.cos(angle).bfloat16().double())
        sin.append(torch.sin(angle).bfloat16().double())
    cos, sin = torch.stack(cos, 1)[:, None], torch.stack(sin, 1)[:, None]

    def head(z, gain):
        z = z / torch.sqrt(z.pow(2).sum(2, keepdim=True) / D + EPS) * gain.double()
        out = z.clone()
        out[..., :32] = z[..., :32] * cos - z[..., 32:64] * sin
        out[..., 32:64] = z[..., 32:64] * cos + z[..., :32] * sin
        return out

    return {"q": head(x[:, :HEADS], st["gq"]), "k": head(x[:, HEADS:HEADS + KV_HEADS], st["gk"]), "v": x[:, HEADS + KV_HEADS:]}
