"""The ragged products' refusals and sizes without a GPU: every check happens on the host before
any HIP call, so pointers are placeholders."""
import ctypes as C

import pytest
import torch

import glmserve_amd as G
from glmserve_amd import _lib
from glmserve_amd.checkpoint import read_layer

P, Q = C.c_void_p(1 << 20), C.c_void_p(1 << 40)
ARG, SHAPE, WORKSPACE = -1, -2, -3


def _grouped(dual=False, **over):
    a = dict(dtype=1, x=P, ldx=64, x_rows=8, ids=None, w=Q, wu=Q, ws=64 * 32, off=P, E=4, rows=8, N=32, K=64,
             ydt=1, y=Q, ldy=32)
    a.update(over)
    L = _lib.lib()
    ws = [a["w"], a["wu"]] if dual else [a["w"]]
    fn = L.glmmoe_grouped_gate_up if dual else L.glmmoe_grouped_linear
    return fn(a["dtype"], a["x"], a["ldx"], a["x_rows"], a["ids"], *ws, a["ws"], a["off"], a["E"], a["rows"],
              a["N"], a["K"], a["ydt"], a["y"], a["ldy"], None)


@pytest.mark.parametrize("dual", [False, True])
@pytest.mark.parametrize("over,rc", [
    (dict(dtype=0), ARG), (dict(dtype=3), ARG), (dict(ydt=2), ARG), (dict(ydt=-1), ARG),
    (dict(x=None), ARG), (dict(w=None), ARG), (dict(off=None), ARG), (dict(y=None), ARG),
    (dict(E=0), ARG), (dict(N=0), ARG), (dict(K=0), ARG), (dict(rows=-1), ARG), (dict(x_rows=0), ARG),
    (dict(E=4097), SHAPE), (dict(N=1 << 24, ldy=1 << 25, ws=1 << 40), SHAPE), (dict(K=1 << 24, ldx=1 << 25), SHAPE),
    (dict(rows=1 << 30, x_rows=1 << 29), SHAPE), (dict(x_rows=7), SHAPE),
    (dict(ldx=63), SHAPE), (dict(ldy=31), SHAPE), (dict(ws=64 * 32 - 1), SHAPE), (dict(ws=-1), SHAPE),
    (dict(x=C.c_void_p(4097)), ARG), (dict(y=C.c_void_p(4097)), ARG), (dict(ydt=0, y=C.c_void_p(4098)), ARG),
    (dict(y=P), ARG), (dict(y=C.c_void_p((1 << 20) + 7 * 64 * 2)), ARG),
    (dict(rows=0), 0), (dict(rows=0, x=None, off=None, y=None, x_rows=0), 0)])
def test_grouped_refusals(dual, over, rc):
    assert _grouped(dual, **over) == rc
    if dual:
        assert _grouped(True, wu=None) == ARG


def _lora(**over):
    a = dict(xdt=0, x=P, ldx=64, ids=P, n=5, wdt=1, A=P, B=P, ranks=None, scale=None, L=3, r=8, K=64, N=32, ydt=0,
             base=P, ldb=32, y=P, ldy=32, ws=Q, wb=1 << 30)
    a.update(over)
    return _lib.lib().glmmoe_lora_add(*[a[k] for k in ("xdt", "x", "ldx", "ids", "n", "wdt", "A", "B", "ranks",
                                                       "scale", "L", "r", "K", "N", "ydt", "base", "ldb", "y", "ldy",
                                                       "ws", "wb")], None)


@pytest.mark.parametrize("over,rc", [
    (dict(wdt=0), ARG), (dict(xdt=2), ARG), (dict(ydt=2), ARG), (dict(xdt=1, wdt=2), ARG),
    (dict(x=None), ARG), (dict(ids=None), ARG), (dict(A=None), ARG), (dict(B=None), ARG), (dict(base=None), ARG),
    (dict(y=None), ARG), (dict(n=-1), ARG), (dict(L=0), ARG), (dict(r=0), ARG), (dict(K=0), ARG), (dict(N=0), ARG),
    (dict(r=257), SHAPE), (dict(n=1 << 24), SHAPE), (dict(K=1 << 24, ldx=1 << 24), SHAPE),
    (dict(N=1 << 24, ldb=1 << 24, ldy=1 << 24), SHAPE), (dict(ldx=63), SHAPE), (dict(ldb=31), SHAPE),
    (dict(ldy=31), SHAPE), (dict(x=C.c_void_p(4098)), ARG), (dict(A=C.c_void_p(4097)), ARG),
    (dict(y=C.c_void_p((1 << 20) + 64)), ARG), (dict(ldy=40), ARG),
    (dict(ws=None), WORKSPACE), (dict(wb=63), WORKSPACE), (dict(ws=C.c_void_p(4104)), WORKSPACE),
    (dict(n=0), 0), (dict(n=0, x=None, base=None, y=None, ws=None), 0)])
def test_lora_refusals(over, rc):
    assert _lora(**over) == rc


def test_lora_workspace():
    f = _lib.lib().glmmoe_lora_workspace_bytes
    assert f(0, 3, 64, 8) == 0 and f(5, 3, 64, 257) == 0 and f(5, 0, 64, 8) == 0
    # whole rows of fp32 sums for every token and split; more K is never less
    for n in (1, 15, 64, 513, 4096):
        for r in (1, 16, 40, 256):
            rp = (r + 15) // 16 * 16
            sizes = [f(n, 8, K, r) for K in (64, 512, 2048, 6144)]
            assert all(s % (n * rp * 4) == 0 and s > 0 for s in sizes) and sizes == sorted(sizes)
            assert sizes[0] == n * rp * 4


def _bf16(**over):
    L = _lib.Bf16Layer()
    L.hidden, L.moe_inter, L.n_experts, L.topk, L.norm_topk, L.routed_scale = 256, 128, 16, 4, 1, 2.5
    for f in ("router_w", "gate", "up", "down", "sh_gate", "sh_up", "sh_down"):
        setattr(L, f, 4096)
    for k, v in over.items():
        setattr(L, k, v)
    return L


@pytest.mark.parametrize("over,rc", [
    (dict(hidden=0), ARG), (dict(hidden=100), SHAPE), (dict(hidden=8448), SHAPE), (dict(moe_inter=100), SHAPE),
    (dict(n_experts=513), SHAPE), (dict(topk=9), SHAPE), (dict(topk=17), SHAPE), (dict(gate=None), ARG),
    (dict(sh_up=None), ARG), (dict(down=4098), ARG)])
def test_bf16_layer_refusals(over, rc):
    L = _bf16(**over)
    lib = _lib.lib()
    assert lib.glmmoe_moe_layer_bf16(C.byref(L), P, 4, P, P, 1 << 30, None) == rc
    assert lib.glmmoe_expert_ffn_bf16(C.byref(L), P, 4, P, P, P, P, 1 << 30, None) == rc
    assert lib.glmmoe_bf16_layer_workspace_bytes(C.byref(L), 4) == 0


def test_bf16_layer_arguments_and_workspace():
    lib, L = _lib.lib(), _bf16()
    call = lambda x=P, n=4, out=P, ws=P, wb=1 << 30: lib.glmmoe_moe_layer_bf16(C.byref(L), x, n, out, ws, wb, None)
    assert call(n=0, x=None, out=None, ws=None, wb=0) == 0
    assert call(x=None) == ARG and call(out=None) == ARG and call(ws=None) == ARG and call(n=-1) == ARG
    assert call(wb=100) == WORKSPACE and call(x=C.c_void_p(4098)) == ARG and call(n=1 << 23) == SHAPE
    L.router_w = None
    assert call() == ARG
    need = lib.glmmoe_bf16_layer_workspace_bytes(C.byref(_bf16()), 64)
    v = _lib.Bf16Ws()
    assert lib.glmmoe_bf16_layer_workspace_view(C.byref(_bf16()), 64, C.c_void_p(1 << 20), C.byref(v)) == 0
    assert v.bytes == need
    fields = [getattr(v, f) for f, _ in _lib.Bf16Ws._fields_[:-1]]
    assert fields == sorted(fields) and fields[-1] + 64 * 5 * 256 * 4 <= (1 << 20) + need
    assert v.dpart - v.h >= 64 * 5 * 128 * 2


def test_python_wrappers_refuse_host_tensors():
    x, w, off = torch.zeros(4, 32).bfloat16(), torch.zeros(2, 16, 32).bfloat16(), torch.zeros(3).int()
    with pytest.raises(G.GlmMoeError):
        G.grouped_linear(x, w, off, torch.zeros(4, 16).bfloat16())
    with pytest.raises(G.GlmMoeError):
        G.grouped_gate_up(x, w, w, off, torch.zeros(4, 16).bfloat16())
    with pytest.raises(G.GlmMoeError):
        G.lora_add(torch.zeros(4, 32), torch.zeros(4).int(), torch.zeros(2, 8, 32).bfloat16(),
                   torch.zeros(2, 16, 8).bfloat16(), None, torch.zeros(4, 16), torch.zeros(4, 16))


def test_checkpoint_in_bf16(tmp_path):
    from safetensors.torch import save_file
    H, I, E = 256, 64, 3
    g = torch.Generator().manual_seed(1)
    p = "model.layers.0.mlp."
    t = {p + "router.weight": torch.randn(E, H, generator=g)}
    kinds = [torch.bfloat16, torch.float16, torch.float32]
    for e in range(E):
        for name, r, K in (("gate_proj", I, H), ("up_proj", I, H), ("down_proj", H, I)):
            t[p + f"experts.{e}.{name}.weight"] = torch.randn(r, K, generator=g).to(kinds[e])
    f = str(tmp_path / "m.safetensors")
    save_file(t, f)
    d = read_layer(f, 0, experts="bf16")
    assert d["shared"] is None and d["gate"].dtype == torch.bfloat16 and tuple(d["down"].shape) == (E, H, I)
    assert torch.equal(d["up"][2], t[p + "experts.2.up_proj.weight"].bfloat16())
    with pytest.raises(G.GlmMoeError):
        read_layer(f, 0, experts="fp8")
    q, s = G.quantize_w4(torch.randn(I, H, generator=g))
    del t[p + "experts.1.gate_proj.weight"]
    t[p + "experts.1.gate_proj.qweight"], t[p + "experts.1.gate_proj.scales"] = q, s
    save_file(t, f)
    with pytest.raises(G.GlmMoeError):
        read_layer(f, 0, experts="bf16")


@pytest.mark.parametrize("K,r", [(1000, 12), (6144, 64), (6144, 256)])
def test_lora_workspace_of_more_tokens_is_enough_for_fewer(K, r):
    f, last = _lib.lib().glmmoe_lora_workspace_bytes, 0
    for n in range(1, 20001):
        need = f(n, 32, K, r)
        assert need >= last, n
        last = need
    for n in (1, 64, 1000, 8176):
        assert f(n, 4, K, r) == f(n, 32, K, r) >= f(n, 32, K - 500, r) and f(n, 32, K, r) >= f(n, 32, K, r - 5)
