"""GPU parity of the low-rank adapters against 64 bits."""
import pytest
import torch

import glmserve_amd as G
from ragged_cases import check, gen, lora_ref, randn

pytestmark = pytest.mark.gpu
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
TYPES = [(F32, BF, F32), (F32, FP, F32), (BF, BF, BF), (FP, FP, FP), (BF, BF, F32), (F32, FP, FP)]


def _case(n, L, r, K, N, types, seed=1, ids=None, ranks=None, scale=True):
    xt, wt, yt = types
    x = randn((n, K), xt, seed)
    A, B = randn((L, r, K), wt, seed + 1, K ** -0.5), randn((L, N, r), wt, seed + 2, 0.3)
    if ids is None:
        ids = torch.randint(-1, L, (n,), generator=gen(seed + 3), device="cuda").int()
    s = 0.5 + torch.rand(L, generator=gen(seed + 4), device="cuda") if scale else None
    base = randn((n, N), yt, seed + 5)
    return x, ids, A, B, s, base, ranks


def _check(x, ids, A, B, s, base, ranks, y):
    live = torch.ones(x.shape[0], dtype=torch.bool, device="cuda")
    check(y, *lora_ref(x, ids, A, B, s, base, ranks), live)
    none = (ids < 0) | (ids >= A.shape[0])
    assert torch.equal(y[none], base[none]), "tokens without an adapter keep the base"


def _run(*args, **kw):
    c = _case(*args, **kw)
    x, ids, A, B, s, base, ranks = c
    y = torch.full_like(base, 7.0)
    G.lora_add(x, ids, A, B, s, base, y, ranks=ranks)
    _check(*c, y)
    z = base.clone()
    G.lora_add(x, ids, A, B, s, z, z, ranks=ranks)
    assert torch.equal(z, y), "in place: the same bits"
    return y


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("n", [1, 16, 37, 300, 1100])
def test_types_and_tokens(types, n):
    _run(n, 5, 16, 512, 320, types)


@pytest.mark.parametrize("r", [1, 3, 8, 12, 31, 32, 48, 64, 65, 100, 256])
@pytest.mark.parametrize("n", [5, 1030])
def test_ranks(r, n):
    _run(n, 3, r, 256, 136, (F32, BF, F32))
    _run(n, 3, r, 200, 130, (FP, FP, FP))


@pytest.mark.parametrize("K,N", [(1, 1), (7, 5), (129, 257), (1000, 2050), (2048, 64), (6144, 96)])
@pytest.mark.parametrize("n", [2, 70])
def test_sizes(K, N, n):
    _run(n, 4, 16, K, N, (F32, BF, F32))
    _run(n, 4, 10, K, N, (BF, BF, BF))


@pytest.mark.parametrize("K", [2, 4, 5, 6, 9, 10, 11, 12, 13, 14, 15, 66, 68, 69, 70, 255])
def test_every_row_end(K):
    _run(21, 4, K % 9 + 1, K, K, (BF, BF, BF))
    _run(21, 4, 16 + K % 8, 530 + K, 64 + K, (F32, FP, F32))


@pytest.mark.parametrize("n", [64, 600, 1500])
def test_adapter_patterns(n):
    t = (F32, BF, F32)
    ar = torch.arange(n, device="cuda")
    _run(n, 64, 16, 256, 128, t, ids=(ar % 64).int())                       # every block all different
    _run(n, 64, 16, 256, 128, t, ids=(ar * 5 // n).int())                   # prompts one after the other
    _run(n, 1, 16, 256, 128, t, ids=torch.zeros(n, device="cuda").int())
    _run(n, 2, 16, 256, 128, t, ids=torch.full((n,), -1, device="cuda").int())   # nobody has one
    wild = torch.randint(-2 ** 31, 2 ** 31 - 1, (n,), generator=gen(9), device="cuda").int()
    wild[::3] = 1
    _run(n, 2, 16, 256, 128, t, ids=wild)


def test_ranks_in_use_and_what_lies_beyond():
    n, L, r, K, N = 90, 6, 20, 264, 100
    ranks = torch.tensor([0, 1, 8, 20, 25, -3], dtype=torch.int32, device="cuda")
    for types in TYPES:
        x, ids, A, B, s, base, _ = _case(n, L, r, K, N, types)
        for a, rk in enumerate((0, 1, 8, 20, 20, 0)):
            A[a, rk:] = float("nan")
            B[a, :, rk:] = float("inf")
        y = torch.empty_like(base)
        G.lora_add(x, ids, A, B, s, base, y, ranks=ranks)
        _check(x, ids, A, B, s, base, ranks, y)


def test_not_finite_stays_with_its_tokens():
    n, L, r, K, N = 40, 4, 16, 200, 80
    for types in TYPES:
        x, ids, A, B, s, base, _ = _case(n, L, r, K, N, types)
        ids = (torch.arange(n, device="cuda") % 4 - 1).int()     # -1, 0, 1, 2, ...
        A[1, 3, 5] = float("nan")
        B[1] = float("inf")
        x[1, 7] = float("inf")                                   # a token of adapter 0
        y = torch.empty_like(base)
        G.lora_add(x, ids, A, B, s, base, y)
        assert not torch.isfinite(y[ids == 1]).any()
        assert not torch.isfinite(y[1]).any()
        keep = (ids != 1) & (torch.arange(n, device="cuda") != 1)
        ref, err = lora_ref(x, ids, A, B, s, base)
        check(y, ref, err, keep)


def test_infinite_products_of_fp32_rows_keep_their_sign():
    # One term of an infinite or huge value must not turn into inf - inf.
    x = torch.zeros(3, 64, device="cuda")
    x[0, 5], x[1, 5], x[2, 5] = float("inf"), -float("inf"), 3.4028234e38
    A = torch.full((1, 1, 64), 0.5, dtype=BF, device="cuda")
    B = torch.ones(1, 16, 1, dtype=BF, device="cuda")
    y = torch.empty(3, 16, device="cuda")
    G.lora_add(x, torch.zeros(3, dtype=torch.int32, device="cuda"), A, B, None, torch.zeros(3, 16, device="cuda"), y)
    # 0 * 0.5 everywhere else: inf * 0.5 = inf, then 1 * inf in the second product.
    assert torch.all(y[0] == float("inf")) and torch.all(y[1] == -float("inf"))
    assert torch.all((y[2] / 3.4028234e38 - 0.5).abs() < 1e-6)


@pytest.mark.parametrize("n", [40, 1100])
def test_strides(n):
    L, r, K, N = 3, 16, 264, 100
    x, ids, A, B, s, base, _ = _case(n, L, r, K, N, (F32, BF, F32))
    xs = randn((n, K + 12), F32, 5)
    for lo in (4, 1):                          # aligned rows, and rows at odd addresses
        xv = xs[:, lo:lo + K]
        out = torch.full((n, 2 * N + 8), 7.0, device="cuda")
        out[:, 4:4 + N] = base
        yv = out[:, 4:4 + N]
        G.lora_add(xv, ids, A, B, s, yv, yv)   # a slice of a wider projection, in place
        live = torch.ones(n, dtype=torch.bool, device="cuda")
        check(yv, *lora_ref(xv, ids, A, B, s, base), live)
        assert torch.all(out[:, :4] == 7.0) and torch.all(out[:, 4 + N:] == 7.0)


def test_streams_graphs_and_repeats():
    n, L, r, K, N = 50, 4, 16, 512, 200
    c = _case(n, L, r, K, N, (F32, BF, F32))
    x, ids, A, B, s, base, _ = c
    want = torch.empty_like(base)
    G.lora_add(x, ids, A, B, s, base, want)
    streams, outs = [torch.cuda.Stream(), torch.cuda.Stream()], [torch.empty_like(base) for _ in range(2)]
    torch.cuda.synchronize()
    for st, o in zip(streams, outs):
        for _ in range(3):
            G.lora_add(x, ids, A, B, s, base, o, stream=st)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
    ws = torch.empty(G.lora_workspace_bytes(n, L, K, r), dtype=torch.uint8, device="cuda")
    xs, idv, y, y2 = x.clone(), ids.clone(), torch.empty_like(base), torch.empty_like(base)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        G.lora_add(xs, idv, A, B, s, base, y, ws=ws)
        G.lora_add(xs, idv, A, B, s, base, y2)       # its workspace from the graph's pool
    for k in range(3):
        xs.copy_(randn((n, K), F32, 70 + k))
        idv.copy_(torch.randint(-1, L, (n,), generator=gen(80 + k), device="cuda").int())
        graph.replay()
        torch.cuda.synchronize()
        _check(xs, idv, A, B, s, base, None, y)
        assert torch.equal(y, y2)


def test_a_workspace_for_more_tokens():
    # 8192 tokens take one pass over K, 8176 two: the workspace of the former serves both, to its end.
    L, r, K, N = 3, 16, 1024, 64
    x, ids, A, B, s, base, _ = _case(8192, L, r, K, N, (BF, BF, BF))
    nb = G.lora_workspace_bytes(8192, L, K, r)
    ws = torch.full((nb + 4096,), 7, dtype=torch.uint8, device="cuda")
    for n in (8176, 8192, 4097, 300, 1):
        y = torch.empty_like(base[:n])
        G.lora_add(x[:n], ids[:n], A, B, s, base[:n], y, ws=ws[:nb])
        _check(x[:n], ids[:n], A, B, s, base[:n], None, y)
        assert torch.all(ws[nb:] == 7)


def test_x_may_be_the_output():
    n, L, r, K = 70, 3, 16, 264
    x, ids, A, B, s, base, _ = _case(n, L, r, K, K, (F32, BF, F32))
    want, z = torch.empty_like(x), x.clone()
    G.lora_add(x, ids, A, B, s, x, want)
    G.lora_add(z, ids, A, B, s, z, z)
    assert torch.equal(z, want)
    _check(x, ids, A, B, s, x, None, want)


@pytest.mark.parametrize("n", [3, 1200])
def test_adapters_beyond_32_bit_offsets(n):
    # More than 2^31 elements of A before the last adapter's.
    L, r, K, N = 8200, 128, 2048, 16
    A = torch.empty(L, r, K, dtype=BF, device="cuda")
    B = torch.empty(L, N, r, dtype=BF, device="cuda")
    last = L - 1
    A[last], B[last] = randn((r, K), BF, 1, K ** -0.5), randn((N, r), BF, 2, 0.3)
    x, base = randn((n, K), F32, 3), randn((n, N), F32, 4)
    ids = torch.full((n,), last, dtype=torch.int32, device="cuda")
    ids[n // 2] = L                                   # one past the last: none
    y = torch.empty_like(base)
    G.lora_add(x, ids, A, B, None, base, y)
    here = torch.where(ids == last, 0, -1).int()
    _check(x, here, A[last:], B[last:], None, base, None, y)


def test_python_refusals():
    x, ids, A, B, s, base, _ = _case(4, 2, 8, 64, 32, (F32, BF, F32))
    y = torch.empty_like(base)
    ok = dict(x=x, adapter_ids=ids, A=A, B=B, scale=s, base=base, y=y)
    for k, v in dict(x=x.half(), adapter_ids=ids.long(), A=A.float(), B=B[:, :, :4], scale=s.double(),
                     base=base[:3], y=y.bfloat16()).items():
        with pytest.raises(G.GlmMoeError):
            G.lora_add(**{**ok, k: v})
    with pytest.raises(G.GlmMoeError):
        G.lora_add(**ok, ranks=torch.zeros(1, dtype=torch.int32, device="cuda"))
    with pytest.raises(G.GlmMoeError):
        G.lora_add(**ok, ws=torch.empty(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(G.GlmMoeError):           # y over base, one row on
        z = torch.empty(5, 32, device="cuda")
        G.lora_add(**{**ok, "base": z[:4], "y": z[1:]})
    e = torch.empty(0, 64, device="cuda")
    G.lora_add(e, ids[:0], A, B, s, base[:0], y[:0])


def test_beside_quantized_linears():
    """A shared expert in int4 with adapters on its three linears, as a server runs it."""
    n, H, I, L, r = 33, 512, 256, 4, 8
    x = randn((n, H), F32, 3)
    ids = torch.randint(-1, L, (n,), generator=gen(4), device="cuda").int()
    s = torch.full((L,), 2.0, device="cuda")

    def linear(rows, K, seed):
        q, sc = G.quantize_w4(randn((rows, K), F32, seed, K ** -0.5))
        from glmserve_amd.checkpoint import dequant_w4
        return (q, sc, dequant_w4(q, sc), randn((L, r, K), BF, seed + 1, K ** -0.5),
                randn((L, rows, r), BF, seed + 2, 0.3))

    def run(lin, v):
        q, sc, w, A, B = lin
        y = torch.empty(n, q.shape[0], device="cuda")
        G.ops.ref_gemm_w4a16(v, q, sc, None, y)
        G.lora_add(v, ids, A, B, s, y, y)
        return y

    def ref(lin, v):
        q, sc, w, A, B = lin
        y = v @ w.double().T
        for a in range(L):
            at = ids == a
            y[at] += 2.0 * (v[at] @ A[a].double().T) @ B[a].double().T
        return y
    gate, up, down = linear(I, H, 10), linear(I, H, 20), linear(H, I, 30)
    g, u = run(gate, x), run(up, x)
    h = torch.empty_like(g)
    G.ops.ref_silu_mul(g, u, h)
    y = run(down, h)
    gd, ud = ref(gate, x.double()), ref(up, x.double())
    want = ref(down, gd * torch.sigmoid(gd) * ud)
    # fp32 throughout: three products of at most 512 terms, each (K / 32 + 4) steps in the norm, the
    # errors of the first two doubled by the product of gate and up.
    assert float((y.double() - want).norm() / want.norm()) < 5 * (512 / 32 + 4) * 2.0 ** -23
