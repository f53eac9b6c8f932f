"""The ragged products of this package, measured: linears grouped by expert, the gated pair of
them with its activation, and low-rank adapters of many requests beside a shared projection.

`run` is one call. With `own` false it computes the operator from elementary torch operations in
32 bits; with `own` true it makes the package's call.
"""
import math

import torch

own = False

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # One decoded token: the down projections of its 8 experts out of 256 (weights streamed, latency counts).
        _linear("linear_decode_1", tokens=1, topk=8, E=256, K=2048, N=6144, dtype="bf16", out="fp32"),
        # A decode batch of 64 requests: almost every expert is in use, with two rows each.
        _linear("linear_decode_64", tokens=64, topk=8, E=256, K=2048, N=6144, dtype="bf16", out="fp32"),
        # A prompt of 2048 tokens on 16 large experts: about 1000 rows each, bound by the matrix cores.
        _linear("linear_prefill_2048", tokens=2048, topk=8, E=16, K=6144, N=2048, dtype="bf16", out="bf16", gather=True),
        # A small layer of odd sizes with a skewed router: rows and weights not aligned to anything.
        _linear("linear_odd", tokens=333, topk=4, E=13, K=1031, N=515, dtype="fp16", out="fp16", gather=True, zipf=1.0),
        # The gate and up projections of one decoded token.
        _gate_up("gate_up_decode_1", tokens=1, topk=8, E=256, K=6144, N=2048, dtype="bf16"),
        # The same for a decode batch of 64 requests.
        _gate_up("gate_up_decode_64", tokens=64, topk=8, E=256, K=6144, N=2048, dtype="bf16"),
        # One rank's share of the experts (an eighth of the features) on a chunk of 1024 tokens, skewed.
        _gate_up("gate_up_shard_1024", tokens=1024, topk=8, E=256, K=6144, N=256, dtype="fp16", zipf=1.0),
        # A prefill chunk of 4096 tokens through all 256 experts: the largest.
        _gate_up("gate_up_prefill_4096", tokens=4096, topk=8, E=256, K=6144, N=2048, dtype="bf16"),
        # One decoded token with an adapter of rank 16 beside a shared expert's gate projection, fp32 rows.
        _lora("lora_decode_1", tokens=1, L=8, r=16, K=6144, N=2048, x="fp32", w="bf16"),
        # 64 requests decoding together, 32 adapters of ranks up to 64 and some requests without one.
        _lora("lora_decode_64", tokens=64, L=32, r=64, K=6144, N=6144, x="bf16", w="bf16", mixed=True),
        # Prompts of eight requests, one adapter each, 4096 tokens in one batch, fp32 rows as the quantized linears have them.
        _lora("lora_prefill_4096", tokens=4096, L=8, r=64, K=6144, N=2048, x="fp32", w="bf16", prompts=8),
        # Prompts and decoding requests in one batch, odd sizes and rank.
        _lora("lora_odd", tokens=700, L=20, r=12, K=1000, N=2050, x="fp16", w="fp16", prompts=3, mixed=True),
    ]


def _linear(name=None, gather=False, zipf=0.0, **c):
    return _named(name, dict(op="linear", gather=gather, zipf=zipf, **c))


def _gate_up(name=None, zipf=0.0, **c):
    return _named(name, dict(op="gate_up", gather=True, zipf=zipf, out=c["dtype"], **c))


def _lora(name=None, prompts=0, mixed=False, **c):
    return _named(name, dict(op="lora", prompts=prompts, mixed=mixed, **c))


def _named(name, c):
    return dict(name=name, **c) if name else c


def draw(rng):
    def size(lo, hi):
        v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        step = rng.choice([1, 8, 64])
        return max(lo, min(hi, v // step * step))

    op = rng.choice(["linear", "gate_up", "lora"])
    tokens = size(1, 4096)
    if op == "lora":
        x = rng.choice(["fp32", "bf16", "fp16"])
        w = rng.choice(["bf16", "fp16"]) if x == "fp32" else x
        return _lora(tokens=tokens, L=size(1, 64), r=rng.choice([4, 8, 12, 16, 32, 64]), K=size(128, 6144),
                     N=size(128, 6144), x=x, w=w, prompts=rng.randint(1, 8) if tokens >= 256 else 0,
                     mixed=rng.random() < 0.5)
    c = dict(tokens=tokens, topk=rng.randint(1, 8), E=size(8, 256), K=size(128, 6144), N=size(128, 6144),
             dtype=rng.choice(["bf16", "fp16"]), zipf=rng.choice([0.0, 1.0]))
    if op == "linear":
        d = _linear(gather=rng.random() < 0.5, out=rng.choice(["fp32", c["dtype"]]), **c)
    else:
        d = _gate_up(**c)
    most = work(listed()[7])
    while 2 * _weights(d) > most["bytes"] or work(d)["flops"] > most["flops"]:
        d["N"] = d["N"] * 3 // 4
    return d


def _weights(c):
    return c["E"] * c["N"] * c["K"] * (2 if c["op"] == "gate_up" else 1)


def _in_use(c):
    """Experts that get a row, on average."""
    p = [(e + 1.0) ** -c["zipf"] for e in range(c["E"])]
    s = sum(p)
    return sum(1.0 - (1.0 - min(1.0, c["topk"] * v / s)) ** c["tokens"] for v in p)


def work(case):
    c = case
    n, K, N = c["tokens"], c["K"], c["N"]
    if c["op"] == "lora":
        used = min(c["L"], c["prompts"] or n)
        r = c["r"] * (0.6 if c["mixed"] else 1.0)
        b = n * (K + 2 * N) * SIZE[c["x"]] + used * r * (K + N) * SIZE[c["w"]]
        return {"bytes": b, "flops": 2.0 * n * r * (K + N)}
    m = 2 if c["op"] == "gate_up" else 1
    rows = n * c["topk"]
    b = _in_use(c) * m * N * K * 2 + (n if c["gather"] else rows) * K * 2 + rows * N * SIZE[c["out"]]
    return {"bytes": b, "flops": 2.0 * m * rows * N * K}


def _gen(seed, k):
    return torch.Generator(device="cuda").manual_seed((int(seed) * 1000003 + k) % (1 << 62))


def _randn(g, shape, dtype, scale):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype).mul_(scale)


def _padded(groups, n_groups):
    """For rows in order of their group: the groups in use, the rows of each as a padded table, and where each row stands in it."""
    counts = torch.bincount(groups, minlength=n_groups)
    active = torch.nonzero(counts).flatten()
    start = torch.cumsum(counts, 0) - counts
    within = torch.arange(groups.numel(), device="cuda") - start[groups]
    place = torch.cumsum((counts > 0).long(), 0) - 1
    most = int(counts.max()) if groups.numel() else 0
    table = start[active][:, None] + torch.arange(most, device="cuda")[None, :]
    return {"active": active, "table": table.clamp_(max=max(0, groups.numel() - 1)), "group": place[groups], "within": within,
            "counts": counts}


def prepare(case, seed):
    c = case
    return _prepare_lora(c, seed) if c["op"] == "lora" else _prepare_experts(c, seed)


def _prepare_experts(c, seed):
    n, k, E, K, N, dt = c["tokens"], c["topk"], c["E"], c["K"], c["N"], DT[c["dtype"]]
    g = _gen(seed, 1)
    # A router's choice: k different experts for each token, the skew on experts of its own.
    rank = torch.randperm(E, generator=g, device="cuda").float()
    noise = -torch.log(-torch.log(torch.rand(n, E, generator=g, device="cuda").clamp_(1e-9, 1 - 1e-6)))
    ids = torch.topk(noise - c["zipf"] * torch.log(rank + 1.0), k, dim=1).indices.flatten()
    groups, order = torch.sort(ids, stable=True)
    st = {"case": c, "pad": _padded(groups, E)}
    st["offsets"] = torch.cat([torch.zeros(1, device="cuda"), torch.cumsum(st["pad"]["counts"], 0)]).int()
    st["rows"] = (order // k).int() if c["gather"] else None
    st["x"] = _randn(_gen(seed, 2), (n if c["gather"] else n * k, K), dt, 1.0)
    st["w"] = _randn(_gen(seed, 3), (E, N, K), dt, 0.02)
    if c["op"] == "gate_up":
        st["up"] = _randn(_gen(seed, 4), (E, N, K), dt, 0.02)
    st["y"] = torch.empty(n * k, N, dtype=DT[c["out"]], device="cuda")
    return st


def _prepare_lora(c, seed):
    n, L, r, K, N = c["tokens"], c["L"], c["r"], c["K"], c["N"]
    g = _gen(seed, 1)
    if c["prompts"]:
        # Requests one after the other, each with its adapter; the last tokens are decoding requests of their own.
        cuts = torch.sort(torch.randint(0, n, (c["prompts"] - 1,), generator=g, device="cuda")).values
        of = torch.randint(0, L, (c["prompts"],), generator=g, device="cuda")
        ids = of[torch.searchsorted(cuts, torch.arange(n, device="cuda"), right=True)]
        tail = min(32, n // 8)
        ids[n - tail:] = torch.randint(-1, L, (tail,), generator=g, device="cuda")
    else:
        ids = torch.randint(-1 if n > 1 else 0, L, (n,), generator=g, device="cuda")
    st = {"case": c, "ids": ids.int()}
    st["ranks"] = None
    if c["mixed"]:
        choice = torch.tensor([max(1, r // 4), max(1, r // 2), r, r], device="cuda")
        st["ranks"] = choice[torch.randint(0, 4, (L,), generator=g, device="cuda")].int()
    groups, order = torch.sort(ids, stable=True)
    used = groups >= 0
    st["tokens"] = order[used]
    st["pad"] = _padded(groups[used], L)
    st["scale"] = 0.5 + torch.rand(L, generator=g, device="cuda")
    st["x"] = _randn(_gen(seed, 2), (n, K), DT[c["x"]], 1.0)
    st["A"] = _randn(_gen(seed, 3), (L, r, K), DT[c["w"]], K ** -0.5)
    st["B"] = _randn(_gen(seed, 4), (L, N, r), DT[c["w"]], 0.1)
    st["base"] = _randn(_gen(seed, 5), (n, N), DT[c["x"]], 1.0)
    st["y"] = torch.empty_like(st["base"])
    return st


def run(state):
    op = state["case"]["op"]
    if own:
        import glmserve_amd as G
        if op == "linear":
            G.grouped_linear(state["x"], state["w"], state["offsets"], state["y"], state["rows"])
        elif op == "gate_up":
            G.grouped_gate_up(state["x"], state["w"], state["up"], state["offsets"], state["y"], state["rows"])
        else:
            # fp32 rows are added to in place, as the plain form does; 16-bit ones go to a buffer of their own.
            base = state["base"]
            y = base if base.dtype == torch.float32 else state["y"]
            G.lora_add(state["x"], state["ids"], state["A"], state["B"], state["scale"], base, y, ranks=state["ranks"])
            return y
        return state["y"]
    if op == "lora":
        return _plain_lora(state)
    x = state["x"].float()
    if state["rows"] is not None:
        x = x[state["rows"].long()]
    y = _products(x, state["w"], state["pad"])
    if op == "gate_up":
        u = _products(x, state["up"], state["pad"])
        y = y / (1.0 + torch.exp(-y)) * u
    return y.to(DT[state["case"]["out"]])


def _products(x, w, pad):
    """x in order of the groups times each group's weights, in 32 bits."""
    if not x.shape[0]:
        return x.new_zeros(0, w.shape[1])
    y = torch.bmm(x[pad["table"]], w[pad["active"]].float().transpose(1, 2))
    return y[pad["group"], pad["within"]]


def _plain_lora(st):
    pad = st["pad"]
    y = st["base"].float()
    if not st["tokens"].numel():
        return y.to(st["base"].dtype)
    t = _products(st["x"].float()[st["tokens"]], st["A"], pad)
    adapter = pad["active"][pad["group"]]
    if st["ranks"] is not None:
        live = torch.arange(t.shape[1], device=t.device)[None, :] < st["ranks"].long()[adapter][:, None]
        t = torch.where(live, t, torch.zeros_like(t))
    y[st["tokens"]] += st["scale"][adapter][:, None] * _products(t, st["B"], pad)
    return y.to(st["base"].dtype)


def exact(case, seed):
    st = prepare(case, seed)
    x = st["x"].double()
    if case["op"] == "lora":
        y = st["base"].double()
        ids = st["ids"].tolist()
        for a in sorted(set(ids) - {-1}):
            rank = case["r"] if st["ranks"] is None else int(st["ranks"][a])
            at = torch.tensor([i for i, v in enumerate(ids) if v == a], device="cuda")
            low = x[at] @ st["A"][a, :rank].double().T
            y[at] += st["scale"][a].double() * (low @ st["B"][a, :, :rank].double().T)
        return y
    off = st["offsets"].tolist()
    y = torch.zeros(st["y"].shape, dtype=torch.float64, device="cuda")
    for e in range(case["E"]):
        lo, hi = off[e], off[e + 1]
        if lo == hi:
            continue
        rows = x[lo:hi] if st["rows"] is None else x[st["rows"][lo:hi].long()]
        v = rows @ st["w"][e].double().T
        if case["op"] == "gate_up":
            v = v * torch.sigmoid(v) * (rows @ st["up"][e].double().T)
        y[lo:hi] = v
    return y
