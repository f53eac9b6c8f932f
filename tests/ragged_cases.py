"""Inputs and 64-bit references of the ragged products on 16-bit weights, shared by their tests.

Bounds. A matrix-core sum of K products in fp32, in any order, is off by at most
(K + 16) * 2^-23 * sum |x w| (one step of the accumulator per addition, however it rounds),
and in the norm by (K / 32 + 4) * 2^-23 of the result where the addends are random (32 products
per addition into a sum whose mean square grows to the result's). A stored value adds half a
step of its type.
"""
import torch

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# Below the smallest normal number of fp16 a step is 2^-24 whatever the value.
SUB = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(shape, dtype, seed, scale=1.0):
    return (torch.randn(*shape, generator=gen(seed), device="cuda") * scale).to(dtype)


def offsets(counts, first=0):
    o = [first]
    for c in counts:
        o.append(o[-1] + c)
    return torch.tensor(o, dtype=torch.int32, device="cuda")


def groups(off, rows):
    """(expert, first row, last row + 1) of every expert with rows, offsets clamped."""
    o = [min(max(int(v), 0), rows) for v in off.tolist()]
    return [(e, o[e], o[e + 1]) for e in range(len(o) - 1) if o[e] < o[e + 1]]


def linear_ref(x, w, off, rows, row_ids=None):
    """(y, bound on a sum's error, rows written) in 64 bits; a row id out of range gives zeros."""
    y = torch.zeros(rows, w.shape[1], dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(y)
    live = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for e, a, b in groups(off, rows):
        if row_ids is None:
            xs = x[a:b].double()
        else:
            ids = row_ids[a:b].long()
            ok = (ids >= 0) & (ids < x.shape[0])
            xs = torch.where(ok[:, None], x[ids.clamp(0, x.shape[0] - 1)].double(),
                             torch.zeros((), dtype=torch.float64, device="cuda"))
        we = w[e].double()
        y[a:b] = xs @ we.T
        mag[a:b] = xs.abs() @ we.abs().T
        live[a:b] = True
    return y, mag * ((x.shape[1] + 16) * 2.0 ** -23), live


def gate_up_ref(x, wg, wu, off, rows, row_ids=None):
    g, dg, live = linear_ref(x, wg, off, rows, row_ids)
    u, du, _ = linear_ref(x, wu, off, rows, row_ids)
    s = g * torch.sigmoid(g)
    # |silu'| <= 1.1; exp2, reciprocal and two products: 8 steps of the value at most, and
    # exp's argument is off by up to |g| / 2 steps.
    err = 1.1 * dg * (u.abs() + du) + s.abs() * du + (s * u).abs() * (8 + g.abs()) * 2.0 ** -23
    return s * u, err, live


def check(got, ref, err, live, K=None):
    """got within err plus its type's half step of ref on the live rows."""
    t = got.dtype
    got = got.double()[live]
    ref, err = ref[live], err[live]
    assert torch.isfinite(got).all()
    bound = err + HALF[t] * (ref.abs() + err) + SUB[t] + 1e-37
    bad = ((got - ref).abs() > bound).nonzero()
    assert bad.numel() == 0, (bad[0].tolist(), got[tuple(bad[0])].item(), ref[tuple(bad[0])].item())
    if K is not None and ref.numel() >= 4096:
        rel = float((got - ref).norm() / ref.norm())
        assert rel <= (K / 32 + 4) * 2.0 ** -23 + HALF[t], rel


def lora_ref(x, ids, A, B, scale, base, ranks=None):
    """(y, bound) in 64 bits."""
    L, r, K = A.shape
    y = base.double().clone()
    err = torch.zeros_like(y)
    for a in range(L):
        at = (ids == a).nonzero().flatten()
        if at.numel() == 0:
            continue
        rk = r if ranks is None else min(max(int(ranks[a]), 0), r)
        Aa, Ba, xs = A[a, :rk].double(), B[a, :, :rk].double(), x[at].double()
        t, mag = xs @ Aa.T, xs.abs() @ Aa.abs().T
        s = 1.0 if scale is None else float(scale[a])
        y[at] += s * (t @ Ba.T)
        # Each of the three terms of an fp32 factor adds products (or six, with fp16 adapters): 6 x.
        dt = mag * ((6 * K + 64) * 2.0 ** -23)
        err[at] = abs(s) * (dt @ Ba.abs().T + (t.abs() + dt) @ Ba.abs().T * ((6 * rk + 64) * 2.0 ** -23))
    return y, err + y.abs() * 2.0 ** -23
