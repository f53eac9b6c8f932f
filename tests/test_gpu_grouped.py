"""GPU parity of the linears grouped by expert and of the gated pair, against 64 bits."""
import pytest
import torch

import glmserve_amd as G
from ragged_cases import check, gate_up_ref, gen, linear_ref, offsets, randn

pytestmark = pytest.mark.gpu
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32

# Groups around the 16-, 32-, 64-, 128- and 256-row tiles, empty ones first, last and between.
FEW = [0, 1, 0, 3, 16, 17, 0]
MID = [5, 0, 31, 33, 64, 65, 1, 20]
MANY = [300, 0, 129, 1, 255, 257, 513, 64, 190]


def _linear(counts, N, K, dtype, out, seed, gather=False, first=0, after=0):
    rows = first + sum(counts) + after
    E = len(counts)
    xr = max(1, rows // 3) if gather else rows
    x, w = randn((xr, K), dtype, seed), randn((E, N, K), dtype, seed + 1, K ** -0.5)
    ids = torch.randint(0, xr, (rows,), generator=gen(seed + 2), device="cuda").int() if gather else None
    off = offsets(counts, first)
    y = torch.full((rows, N), 7.0, dtype=out, device="cuda")
    G.grouped_linear(x, w, off, y, ids)
    ref, err, live = linear_ref(x, w, off, rows, ids)
    check(y, ref, err, live, K)
    assert torch.all(y[~live] == 7.0), "rows outside the offsets stay"
    return y


@pytest.mark.parametrize("dtype,out", [(BF, BF), (BF, F32), (FP, FP), (FP, F32)])
@pytest.mark.parametrize("counts", [FEW, MID, MANY], ids=["few", "mid", "many"])
@pytest.mark.parametrize("N,K", [(128, 256), (96, 1064), (515, 1031)])
def test_linear(counts, N, K, dtype, out):
    _linear(counts, N, K, dtype, out, 1, gather=N != 128, first=3, after=5)


@pytest.mark.parametrize("N,K", [(1, 1), (3, 7), (16, 8), (17, 31), (33, 32), (5, 129), (300, 72), (256, 64),
                                 (257, 520), (640, 2048)])
@pytest.mark.parametrize("counts", [[1], [0, 2, 70], [300, 1]], ids=["one", "mixed", "large"])
def test_linear_odd_sizes(counts, N, K):
    _linear(counts, N, K, BF, BF, N + K)
    _linear(counts, N, K, FP, F32, N + K, gather=True)


@pytest.mark.parametrize("K", [2, 4, 5, 6, 9, 10, 11, 12, 13, 14, 15, 66, 67, 68, 69, 70, 71, 127])
def test_linear_every_row_end(K):
    _linear([3, 0, 70], 37, K, BF, F32, K)


@pytest.mark.parametrize("dtype,out", [(BF, BF), (FP, FP), (BF, F32)])
@pytest.mark.parametrize("counts", [[1], FEW, MID, MANY], ids=["one", "few", "mid", "many"])
@pytest.mark.parametrize("N,K", [(128, 256), (260, 1064), (67, 131)])
def test_gate_up(counts, N, K, dtype, out):
    rows, E = sum(counts), len(counts)
    xr = max(1, rows // 2)
    x = randn((xr, K), dtype, 5)
    wg, wu = randn((E, N, K), dtype, 6, 2 * K ** -0.5), randn((E, N, K), dtype, 7, K ** -0.5)
    ids = torch.randint(0, xr, (rows,), generator=gen(8), device="cuda").int()
    h = torch.empty(rows, N, dtype=out, device="cuda")
    G.grouped_gate_up(x, wg, wu, offsets(counts), h, ids)
    check(h, *gate_up_ref(x, wg, wu, offsets(counts), rows, ids))


# So many columns that the large tiles fill the GPU: W read once, and shared by an expert's tiles, the last ones in
# halves of the columns.
WIDE = [MANY, [600, 0, 900, 257]]


@pytest.mark.parametrize("dtype,out", [(BF, BF), (FP, F32)])
@pytest.mark.parametrize("counts", WIDE, ids=["once", "shared"])
@pytest.mark.parametrize("K", [72, 264])
def test_large_tiles(counts, K, dtype, out):
    _linear(counts, 5300, K, dtype, out, 91, gather=K == 72, first=3, after=5)


@pytest.mark.parametrize("dtype,out", [(FP, FP), (BF, F32)])
@pytest.mark.parametrize("counts", WIDE, ids=["once", "shared"])
def test_large_tiles_gate_up(counts, dtype, out):
    rows, E, K, N = sum(counts), len(counts), 136, 2700
    x = randn((rows, K), dtype, 92)
    wg, wu = randn((E, N, K), dtype, 93, 2 * K ** -0.5), randn((E, N, K), dtype, 94, K ** -0.5)
    h = torch.empty(rows, N, dtype=out, device="cuda")
    G.grouped_gate_up(x, wg, wu, offsets(counts), h)
    check(h, *gate_up_ref(x, wg, wu, offsets(counts), rows))


@pytest.mark.parametrize("counts", WIDE, ids=["once", "shared"])
def test_large_tiles_bad_ids_not_finite_and_bits(counts):
    rows, K, N = sum(counts), 128, 5300
    x, w, off = randn((50, K), BF, 95), randn((len(counts), N, K), BF, 96, 0.1), offsets(counts)
    ids = torch.randint(0, 49, (rows,), generator=gen(97), device="cuda").int()
    ids[0], ids[299], ids[rows - 1], ids[5] = -1, 50, 2 ** 31 - 1, 49
    x[49, 7] = float("nan")
    y = torch.full((rows, N), 7.0, dtype=F32, device="cuda")
    G.grouped_linear(x, w, off, y, ids)
    assert torch.isnan(y[5]).all()
    for r in (0, 299, rows - 1):
        assert torch.all(y[r] == 0)
    ref, err, live = linear_ref(x, w, off, rows, ids)
    live[5] = False
    check(y, ref, err, live)
    again = torch.empty_like(y)
    G.grouped_linear(x, w, off, again, ids)
    part = torch.empty(rows, 64, dtype=F32, device="cuda")       # few columns: the small tiles
    G.grouped_linear(x, w[:, :64].contiguous(), off, part, ids)
    live[5] = False
    assert torch.equal(again[live], y[live]) and torch.equal(part[live], y[live][:, :64])


def test_many_experts():
    # More experts than lanes, most of them empty, groups far apart.
    counts = [0] * 700
    for i, e in enumerate((0, 63, 64, 255, 511, 512, 698, 699)):
        counts[e] = 1 + 9 * i
    _linear(counts, 64, 128, BF, F32, 21)


def test_strides_and_halves():
    rows, K, N, E = 90, 264, 72, 3
    big = randn((rows, K + 40), BF, 31)
    x = big[:, 8:8 + K]                       # 16-byte aligned rows
    both = randn((E, 2 * N, K), BF, 32, K ** -0.5)
    off = offsets([30, 0, 60])
    out = torch.full((rows, N + 9), 7.0, dtype=BF, device="cuda")
    h = out[:, 4:4 + N]
    G.grouped_gate_up(x, both[:, :N], both[:, N:], off, h)
    check(h, *gate_up_ref(x, both[:, :N], both[:, N:], off, rows))
    assert torch.all(out[:, :4] == 7.0) and torch.all(out[:, 4 + N:] == 7.0)
    odd = big[:, 3:3 + K]                     # rows at odd addresses
    y = torch.empty(rows, N, dtype=F32, device="cuda")
    G.grouped_linear(odd, both[:, N:], off, y)
    check(y, *linear_ref(odd, both[:, N:], off, rows))
    flat = randn((E * N * K + 1,), BF, 33, K ** -0.5)[1:].view(E, N, K)   # weights at an odd address
    G.grouped_linear(x, flat, off, y)
    check(y, *linear_ref(x, flat, off, rows))


@pytest.mark.parametrize("counts", [[2, 3], [40, 90], [300, 20]], ids=["few", "mid", "large"])
def test_bad_row_ids_and_offsets(counts):
    rows, K, N = sum(counts), 192, 80
    x, w = randn((9, K), FP, 41), randn((2, N, K), FP, 42, 0.1)
    ids = torch.randint(0, 9, (rows,), generator=gen(43), device="cuda").int()
    ids[0], ids[rows - 1], ids[1] = -1, 9, 2 ** 31 - 1
    off = offsets(counts)
    y = torch.full((rows, N), 7.0, dtype=FP, device="cuda")
    G.grouped_linear(x, w, off, y, ids)
    check(y, *linear_ref(x, w, off, rows, ids))
    assert torch.all(y[0] == 0) and torch.all(y[rows - 1] == 0)
    wild = torch.tensor([-5, 2, 2 ** 31 - 1], dtype=torch.int32, device="cuda")   # taken as 0, 2, rows
    y.fill_(7.0)
    G.grouped_linear(x, w, wild, y, ids)
    check(y, *linear_ref(x, w, wild, rows, ids))
    back = torch.tensor([rows, 1, 0], dtype=torch.int32, device="cuda")           # descending: no rows
    y.fill_(7.0)
    G.grouped_linear(x, w, back, y, ids)
    assert torch.all(y == 7.0)


@pytest.mark.parametrize("counts", [[3, 5], [50, 70], [200, 290]], ids=["few", "mid", "large"])
@pytest.mark.parametrize("K", [256, 203])
def test_not_finite_stays_in_its_row_and_expert(counts, K):
    rows, N = sum(counts), 144
    x, w = randn((rows, K), BF, 51), randn((3, N, K), BF, 52, 0.1)
    w[2] = float("nan")                        # an expert without rows
    x[1, K - 1] = float("inf")
    x[counts[0], 0] = float("nan")
    w[0, 5, 3] = float("inf")
    off = offsets(counts + [0])
    y = torch.empty(rows, N, dtype=F32, device="cuda")
    G.grouped_linear(x, w, off, y)
    ref, err, live = linear_ref(x, w, off, rows)
    assert torch.equal(torch.isnan(y), torch.isnan(ref)) and torch.equal(torch.isinf(y), torch.isinf(ref))
    inf = torch.isinf(ref)
    assert torch.equal(y[inf].double(), ref[inf])
    fine = torch.isfinite(ref) & torch.isfinite(err)
    assert torch.all((y.double() - ref)[fine].abs() <= (err + 2.0 ** -23 * ref.abs())[fine])


def test_fp16_subnormals_count():
    # Values below 2^-14 are kept by the products: K times 2^-16 * 2^8.
    x = torch.full((3, 512), 2.0 ** 8, dtype=FP, device="cuda")
    w = torch.full((1, 32, 512), 2.0 ** -16, dtype=FP, device="cuda")
    y = torch.empty(3, 32, dtype=F32, device="cuda")
    G.grouped_linear(x, w, offsets([3]), y)
    assert torch.all(y == 2.0)


def test_large_strides_pass_32_bits():
    # Three experts' matrices 2^31 + 8 elements apart, the last beyond 8 GiB.
    N, K, step = 48, 128, 2 ** 31 + 8
    store = torch.empty(2 * step + N * K, dtype=BF, device="cuda")
    w = store.as_strided((3, N, K), (step, K, 1))
    for e in range(3):
        w[e] = randn((N, K), BF, 60 + e, 0.1)
    for counts in ([1, 2, 3], [70, 0, 200]):
        rows = sum(counts)
        x = randn((rows, K), BF, 63)
        y = torch.empty(rows, N, dtype=F32, device="cuda")
        G.grouped_linear(x, w, offsets(counts), y)
        check(y, *linear_ref(x, w, offsets(counts), rows))


@pytest.mark.parametrize("counts", [[4, 2, 0, 1], [300, 40, 0, 129]], ids=["few", "large"])
def test_streams_graphs_and_repeats(counts):
    rows, K, N, E = sum(counts), 320, 200, len(counts)
    x, w, u = randn((rows, K), BF, 71), randn((E, N, K), BF, 72, 0.1), randn((E, N, K), BF, 73, 0.1)
    off = offsets(counts)
    want = torch.empty(rows, N, dtype=BF, device="cuda")
    G.grouped_gate_up(x, w, u, off, want)
    # the same bits again, on a stream of its own, and from two streams at once
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    outs = [torch.empty_like(want) for _ in range(2)]
    torch.cuda.synchronize()
    for s, o in zip((side, other), outs):
        G.grouped_gate_up(x, w, u, off, o, stream=s)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
    # captured, with inputs and offsets that change between replays
    h, y = torch.empty_like(want), torch.empty(rows, N, dtype=F32, device="cuda")
    xs, offs = x.clone(), off.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        G.grouped_gate_up(xs, w, u, offs, h)
        G.grouped_linear(xs, w, offs, y)
    for k in range(3):
        xs.copy_(randn((rows, K), BF, 80 + k))
        offs.copy_(offsets(counts if k != 1 else counts[::-1]))
        graph.replay()
        torch.cuda.synchronize()
        check(h, *gate_up_ref(xs, w, u, offs, rows))
        check(y, *linear_ref(xs, w, offs, rows))


@pytest.mark.parametrize("dtype", [BF, FP])
def test_a_row_has_the_same_bits_in_any_batch(dtype):
    # Decode, verify and prefill of a token agree bit for bit: K in ascending pieces of 32, whatever
    # the tile, the batch or the alignment.
    K, N, E = 520, 200, 3
    x, w = randn((700, K), dtype, 101), randn((E, N, K), dtype, 102, 0.1)
    u = randn((E, N, K), dtype, 103, 0.1)
    off = offsets([50, 640, 10])
    y, h = torch.empty(700, N, dtype=F32, device="cuda"), torch.empty(700, N, dtype=F32, device="cuda")
    G.grouped_linear(x, w, off, y)
    G.grouped_gate_up(x, w, u, off, h)
    wide = torch.zeros(700, K + 1, dtype=dtype, device="cuda")
    wide[:, 1:] = x
    odd = torch.empty_like(y)
    G.grouped_linear(wide[:, 1:], w, off, odd)
    assert torch.equal(odd, y)
    for r, e in ((0, 0), (49, 0), (50, 1), (333, 1), (689, 1), (690, 2), (699, 2)):
        one = torch.empty(1, N, dtype=F32, device="cuda")
        at = torch.tensor([r], dtype=torch.int32, device="cuda")
        alone = offsets([1 if k == e else 0 for k in range(E)])
        G.grouped_linear(x, w, alone, one, at)
        assert torch.equal(one[0], y[r])
        G.grouped_gate_up(x, w, u, alone, one, at)
        assert torch.equal(one[0], h[r])


def test_no_rows():
    w = randn((2, 16, 32), BF, 90)
    y = torch.empty(0, 16, dtype=BF, device="cuda")
    G.grouped_linear(torch.empty(0, 32, dtype=BF, device="cuda"), w, offsets([0, 0]), y)
    y = torch.full((4, 16), 7.0, dtype=BF, device="cuda")
    G.grouped_linear(randn((4, 32), BF, 91), w, offsets([0, 0]), y)
    assert torch.all(y == 7.0)


def test_python_refusals():
    x, w, off = randn((4, 32), BF, 1), randn((2, 16, 32), BF, 2), offsets([2, 2])
    y = torch.empty(4, 16, dtype=BF, device="cuda")
    bad = [(x.float(), w, off, y), (x, w.half(), off, y), (x, w, off.long(), y), (x, w, off[:2], y),
           (x, w, off, y.half()), (x, w, off, y[:, :8]), (x[:2], w, off, y), (x.cpu(), w, off, y),
           (x, w.transpose(1, 2), off, y), (x.t(), w, off, y)]
    for args in bad:
        with pytest.raises(G.GlmMoeError):
            G.grouped_linear(*args)
    with pytest.raises(G.GlmMoeError):
        G.grouped_linear(x, w, off, y, torch.zeros(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(G.GlmMoeError):       # the output over the input
        z = torch.empty(4, 48, dtype=BF, device="cuda")
        G.grouped_linear(z[:, :32], w, off, z[:, 24:40])
