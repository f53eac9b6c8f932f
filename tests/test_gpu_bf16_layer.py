"""GPU parity of the MoE layer with bf16 experts: routing bit-exact against the router's own
entry points, the output against 64 bits with h's rounding to bf16 in the bound."""
import pytest
import torch

import glmserve_amd as G
from ragged_cases import gen, randn

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _layer(H, I, E, k, seed=1, shared=True):
    m = lambda e, r, K, s: randn((e, r, K) if e else (r, K), BF, seed + s, K ** -0.5)
    sh = (m(0, I, H, 5), m(0, I, H, 6), m(0, H, I, 7)) if shared else None
    return G.BF16MoELayer(H, I, E, k, randn((E, H), BF, seed, 0.02), randn((E,), F32, seed + 1, 0.05),
                          m(E, I, H, 2), m(E, I, H, 3), m(E, H, I, 4), sh)


def _ffn(x, g, u, d):
    """(y, bound) of one expert in 64 bits; h is rounded to bf16 between the products."""
    g, u, d = g.double(), u.double(), d.double()
    e1, e2 = (g.shape[1] + 16) * 2.0 ** -23, (d.shape[1] + 16) * 2.0 ** -23
    a, b = x @ g.T, x @ u.T
    da, db = x.abs() @ g.abs().T * e1, x.abs() @ u.abs().T * e1
    s = a * torch.sigmoid(a)
    h = s * b
    dh = 1.1 * da * (b.abs() + db) + s.abs() * db + h.abs() * (8 + a.abs()) * 2.0 ** -23
    dh = dh + 2.0 ** -8 * (h.abs() + dh)
    return h @ d.T, dh @ d.abs().T + (h.abs() + dh) @ d.abs().T * e2


def _expect(L, x, ids, w):
    rw, eb, gate, up, down, sh = L.keep
    xd = x.double()
    out = torch.zeros(x.shape[0], L.hidden, dtype=torch.float64, device="cuda")
    err = torch.zeros_like(out)
    for e in range(L.n_experts):
        t, s = (ids == e).nonzero(as_tuple=True)
        if t.numel():
            y, dy = _ffn(xd[t], gate[e], up[e], down[e])
            ws = w[t, s].double()[:, None]
            out.index_add_(0, t, ws * y)
            err.index_add_(0, t, ws.abs() * dy)
    if sh is not None:
        y, dy = _ffn(xd, *sh)
        out, err = out + y, err + dy
    return out, err + (out.abs() + err) * 2.0 ** -20      # 9 fp32 terms added


def _check(out, want):
    ref, err = want
    assert torch.isfinite(out).all()
    assert torch.all((out.double() - ref).abs() <= err)
    # in the norm: h's half step 2^-9 to 2^-8 of each value, spread evenly
    assert float((out.double() - ref).norm() / ref.norm()) < 2.0 ** -8


@pytest.mark.parametrize("H,I,E,k,shared", [(256, 128, 16, 4, True), (512, 200, 40, 8, False),
                                            (768, 256, 300, 8, True), (256, 64, 512, 8, True)])
@pytest.mark.parametrize("n", [1, 7, 64, 300, 1200])
def test_layer(H, I, E, k, shared, n):
    L = _layer(H, I, E, k, shared=shared)
    x = randn((n, H), BF, 9)
    ws = L.alloc_workspace(n)
    out = torch.full((n, H), float("nan"), device="cuda")
    L.forward(x, out, ws)
    v = L.workspace_view(n, ws)
    ids = G.ops.ws_tensor(None, v.topk_ids, ws, torch.int32, n * k).view(n, k)
    w = G.ops.ws_tensor(None, v.topk_w, ws, F32, n * k).view(n, k)
    logits = torch.empty(n, E, device="cuda")
    G.router_logits(x, L.keep[0], logits)
    rid, rw = torch.empty_like(ids), torch.empty_like(w)
    G.moe_router(logits, L.keep[1], n, E, k, True, 2.5, rid, rw)
    assert torch.equal(ids, rid) and torch.equal(w.view(torch.int32), rw.view(torch.int32))
    _check(out, _expect(L, x, ids.long(), w))
    # the expert stage alone gives the same bits from the same routing
    alone = torch.empty_like(out)
    L.expert_ffn(x, rid, rw, alone, L.alloc_workspace(n))
    assert torch.equal(alone, out)


@pytest.mark.parametrize("n", [3, 400])
def test_caller_routing_with_ids_out_of_range(n):
    L = _layer(256, 128, 16, 4)
    x = randn((n, 256), BF, 11)
    ids = torch.randint(0, 16, (n, 4), generator=gen(12), device="cuda").int()
    ids[0, 1], ids[n - 1, 3], ids[1, 0] = -1, 16, 2 ** 31 - 1
    w = torch.rand(n, 4, generator=gen(13), device="cuda")
    w[0, 1] = float("nan")                   # a slot that counts nothing
    out = torch.empty(n, 256, device="cuda")
    L.expert_ffn(x, ids, w, out, L.alloc_workspace(n))
    _check(out, _expect(L, x, ids.long(), w))


def test_same_expert_for_every_token():
    # One expert with every row, twice the same id in a token.
    L = _layer(256, 128, 16, 4)
    n = 700
    x = randn((n, 256), BF, 14)
    ids = torch.tensor([3, 3, 0, 15], device="cuda").int().repeat(n, 1)
    w = torch.rand(n, 4, generator=gen(15), device="cuda")
    out = torch.empty(n, 256, device="cuda")
    L.expert_ffn(x, ids, w, out, L.alloc_workspace(n))
    _check(out, _expect(L, x, ids.long(), w))


@pytest.mark.parametrize("n", [4, 200])
def test_graph(n):
    L = _layer(256, 128, 16, 4)
    x, ws = randn((n, 256), BF, 21), L.alloc_workspace(n)
    out, eager = torch.empty(n, 256, device="cuda"), torch.empty(n, 256, device="cuda")
    L.forward(x, out, ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        L.forward(x, out, ws)
    for k in range(3):
        x.copy_(randn((n, 256), BF, 30 + k))
        graph.replay()
        torch.cuda.synchronize()
        L.forward(x, eager, L.alloc_workspace(n))
        assert torch.equal(out, eager)


def test_from_a_checkpoint(tmp_path):
    from safetensors.torch import save_file
    H, I, E, k = 256, 128, 4, 2
    g = torch.Generator().manual_seed(5)
    p = "model.layers.3.mlp."
    t = {p + "gate.weight": torch.randn(E, H, generator=g) * 0.05}
    for pre in [f"experts.{e}." for e in range(E)] + ["shared_experts."]:
        for name, r, K in (("gate_proj", I, H), ("up_proj", I, H), ("down_proj", H, I)):
            t[p + pre + name + ".weight"] = (torch.randn(r, K, generator=g) * K ** -0.5).to(BF)
    f = str(tmp_path / "m.safetensors")
    save_file(t, f)
    L = G.load_layer(f, 3, topk=k, experts="bf16")
    assert isinstance(L, G.BF16MoELayer) and (L.hidden, L.moe_inter, L.n_experts) == (H, I, E)
    assert torch.equal(L.keep[4][2].cpu(), t[p + "experts.2.down_proj.weight"])
    n = 21
    x, ws = randn((n, H), BF, 6), L.alloc_workspace(n)
    out = torch.empty(n, H, device="cuda")
    L.forward(x, out, ws)
    v = L.workspace_view(n, ws)
    ids = G.ops.ws_tensor(None, v.topk_ids, ws, torch.int32, n * k).view(n, k).long()
    w = G.ops.ws_tensor(None, v.topk_w, ws, F32, n * k).view(n, k)
    _check(out, _expect(L, x, ids, w))


def test_empty_and_short_workspace():
    L = _layer(256, 128, 16, 4)
    e = torch.empty(0, 256, dtype=BF, device="cuda")
    L.forward(e, torch.empty(0, 256, device="cuda"), torch.empty(0, dtype=torch.uint8, device="cuda"))
    with pytest.raises(G.GlmMoeError):
        L.forward(randn((8, 256), BF, 1), torch.empty(8, 256, device="cuda"), L.alloc_workspace(7)[:4096])
    with pytest.raises(G.GlmMoeError):
        G.BF16MoELayer(256, 128, 16, 4, None, None, L.keep[2].float(), L.keep[3], L.keep[4])
