"""bf16 products grouped by expert against fp64: integer-valued inputs bit for bit, real ones within the derived error."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF = torch.bfloat16

# (sizes of the groups, rows behind the last, n, k)
CASES = [
    ([1], 0, 8, 8),
    ([5], 3, 16, 64),
    ([0, 1, 0, 2, 0], 0, 128, 64),
    ([17, 0, 64, 15, 33], 5, 136, 72),
    ([63, 64, 65, 1], 0, 256, 128),
    ([128, 0, 127, 129], 9, 200, 320),
    ([300, 2, 511], 40, 264, 1000),
    ([256, 512, 255, 257], 0, 384, 256),
    ([1000], 0, 1032, 136),
    ([0, 0, 0], 4, 64, 64),
    ([3] * 70, 1, 96, 200),
    ([2600, 40, 0, 700], 0, 128, 64),
]
IDS = [f"{len(g)}groups_{sum(g)}rows_{n}x{k}" for g, _, n, k in CASES]


def borders(sizes):
    return torch.tensor([0] + sizes, device=DEV).cumsum(0).to(torch.int32)


def ints(shape, seed, top=3):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randint(-top, top + 1, shape, device=DEV, generator=g).to(BF)


def reals(shape, seed):
    return torch.randn(shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed)).to(BF)


def plain(side, sizes, a, b, out):
    """a, b in fp64 by groups into `out` (fp64)."""
    at = 0
    for e, s in enumerate(sizes):
        rows = slice(at, at + s)
        if side == "fwd":
            out[rows] = a[rows].double() @ b[e].double().t()
        elif side == "dgrad":
            out[rows] = a[rows].double() @ b[e].double()
        else:
            out[e] = a[rows].double().t() @ b[rows].double()
        at += s
    return out


def run(pb, side, sizes, spare, n, k, make, dtype=BF):
    """(got, want in fp64, sum of |products| in fp64, length of the sums)"""
    rows, E, offsets = sum(sizes) + spare, len(sizes), borders(sizes)
    w, x, dy = make((E, n, k), 1), make((rows, k), 2), make((rows, n), 3)
    end = sum(sizes)
    x[end:], dy[end:] = float("nan"), float("nan")   # behind the last group: never used
    if side == "wgrad":
        got = pb.grouped_gemm_bf16_wgrad(dy, x, offsets, dtype=dtype)
        want = plain(side, sizes, dy, x, torch.zeros((E, n, k), dtype=torch.float64, device=DEV))
        size = plain(side, sizes, dy.abs(), x.abs(), torch.zeros((E, n, k), dtype=torch.float64, device=DEV))
        return got, want, size, max(sizes)
    a, width = (x, n) if side == "fwd" else (dy, k)
    out = torch.full((rows, width), 7.0, dtype=BF, device=DEV)
    got = (pb.grouped_gemm_bf16 if side == "fwd" else pb.grouped_gemm_bf16_dgrad)(a, w, offsets, out=out)
    want = plain(side, sizes, a, w, torch.full((rows, width), 7.0, dtype=torch.float64, device=DEV))   # rows of no group stay
    size = plain(side, sizes, a.abs(), w.abs(), torch.zeros((rows, width), dtype=torch.float64, device=DEV))
    return got, want, size, k if side == "fwd" else n


@pytest.mark.parametrize("side,dtype", [("fwd", BF), ("dgrad", BF), ("wgrad", BF), ("wgrad", torch.float32)])
@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_integers_bit_for_bit(pb, case, side, dtype):
    """Products of integers up to 3: every partial sum is below 2^24, so the fp32 sums are exact in any order."""
    got, want, size, _ = run(pb, side, *case, ints, dtype)
    assert size.max() < 2 ** 24
    assert torch.equal(got, want.to(dtype))


@pytest.mark.parametrize("side,dtype", [("fwd", BF), ("dgrad", BF), ("wgrad", BF), ("wgrad", torch.float32)])
@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_reals(pb, case, side, dtype):
    got, want, size, length = run(pb, side, *case, reals, dtype)
    fp32 = (length + 1) * 2.0 ** -23 * size          # each addition off by less than one step of a partial sum
    half_step = 2.0 ** -8 if dtype == BF else 0.0
    assert ((got.double() - want).abs() <= fp32 + half_step * (want.abs() + fp32)).all()


@pytest.mark.parametrize("side", ["fwd", "dgrad", "wgrad"])
def test_many_shapes(pb, side):
    """Seeded shapes over the tile widths: groups of mixed sizes, n and k any multiple of 8."""
    import random
    rng = random.Random(side)
    for i in range(14):
        E = rng.choice([1, 2, 5, 16, 40])
        sizes = [rng.choice([0, 1, rng.randint(0, 40), rng.randint(0, 400)]) for _ in range(E)]
        if not sum(sizes):
            sizes[0] = 3
        n, k = 8 * rng.randint(1, 90), 8 * rng.randint(1, 90)
        got, want, size, _ = run(pb, side, sizes, rng.choice([0, 5]), n, k, ints)
        assert size.max() < 2 ** 24 and torch.equal(got, want.to(BF)), (sizes, n, k)


def test_sums_past_the_tiles_of_all_sms(pb):
    """Several tiles per CTA in each mode, both accumulators in turn."""
    sizes = [700, 0, 1300, 2100, 60]
    for side in ("fwd", "dgrad", "wgrad"):
        got, want, size, _ = run(pb, side, sizes, 0, 2048, 1536, lambda shape, seed: ints(shape, seed, 2))
        assert size.max() < 2 ** 24 and torch.equal(got, want.to(BF)), side


def test_strided_rows(pb):
    sizes, n, k = [30, 0, 99], 72, 136
    offsets, rows = borders(sizes), sum(sizes)
    both = ints((rows, 304), 5)
    x, dy, w = both[:, 8:8 + k], both[:, 160:160 + n], ints((3, n, k), 6)
    out = torch.zeros((rows, 200), dtype=BF, device=DEV)
    got = pb.grouped_gemm_bf16(x, w, offsets, out=out[:, 16:16 + n])
    assert torch.equal(got, pb.grouped_gemm_bf16(x.contiguous(), w, offsets))
    assert (out[:, :16] == 0).all() and (out[:, 16 + n:] == 0).all()
    assert torch.equal(pb.grouped_gemm_bf16_dgrad(dy, w, offsets), pb.grouped_gemm_bf16_dgrad(dy.contiguous(), w, offsets))
    assert torch.equal(pb.grouped_gemm_bf16_wgrad(dy, x, offsets), pb.grouped_gemm_bf16_wgrad(dy.contiguous(), x.contiguous(), offsets))
    # interleaved columns of one buffer: input and output do not overlap
    buf = torch.zeros((rows, 256), dtype=BF, device=DEV)
    buf[:, :k] = x
    assert torch.equal(pb.grouped_gemm_bf16(buf[:, :k], w, offsets, out=buf[:, 144:144 + n]), got)


def test_infinities_stay_in_their_group(pb):
    sizes, n, k = [20, 13, 40], 64, 128
    offsets = borders(sizes)
    x, dy, w = ints((73, k), 1), ints((73, n), 2), ints((3, n, k), 3)
    clean = [pb.grouped_gemm_bf16(x, w, offsets), pb.grouped_gemm_bf16_dgrad(dy, w, offsets), pb.grouped_gemm_bf16_wgrad(dy, x, offsets)]
    x[20:33], dy[20:33], w[1] = float("inf"), float("nan"), float("nan")
    dirty = [pb.grouped_gemm_bf16(x, w, offsets), pb.grouped_gemm_bf16_dgrad(dy, w, offsets), pb.grouped_gemm_bf16_wgrad(dy, x, offsets)]
    for a, b in zip(clean[:2], dirty[:2]):
        assert torch.equal(a[:20], b[:20]) and torch.equal(a[33:], b[33:]) and not torch.isfinite(b[20:33]).any()
    assert torch.equal(clean[2][0], dirty[2][0]) and torch.equal(clean[2][2], dirty[2][2]) and not torch.isfinite(dirty[2][1]).any()


def test_wrong_borders_stay_inside_the_matrices(pb):
    """Borders are clamped to the rows and to each other: groups in order are still right, others are empty or cut."""
    x, w = ints((50, 64), 1), ints((4, 64, 64), 2)
    guard = torch.full((52, 64), 7.0, dtype=BF, device=DEV)
    offsets = torch.tensor([-5, 20, 10, 1 << 30, 40], dtype=torch.int32, device=DEV)
    got = pb.grouped_gemm_bf16(x, w, offsets, out=guard[1:51])
    assert torch.equal(got[:10].double(), x[:10].double() @ w[0].double().t())
    assert (guard[0] == 7).all() and (guard[51] == 7).all()
    dw = pb.grouped_gemm_bf16_wgrad(x, x, offsets, dtype=torch.float32)
    assert torch.equal(dw[0].double(), x[:20].double().t() @ x[:20].double()) and (dw[1] == 0).all() and (dw[3] == 0).all()


def test_no_rows(pb):
    offsets = torch.zeros(4, dtype=torch.int32, device=DEV)
    x, w = torch.empty((0, 64), dtype=BF, device=DEV), ints((3, 32, 64), 1)
    assert pb.grouped_gemm_bf16(x, w, offsets).shape == (0, 32)
    out = torch.full((3, 32, 64), 7.0, device=DEV)
    assert (pb.grouped_gemm_bf16_wgrad(x[:, :32], x, offsets, out=out) == 0).all()


def test_graph_with_changing_borders(pb):
    """One captured graph, replayed for other groups and other rows."""
    E, n, k, rows = 6, 128, 192, 500
    x, dy, w, offsets = ints((rows, k), 1), ints((rows, n), 2), ints((E, n, k), 3), borders([10, 20, 30, 40, 50, 60])
    out, dx, dw = (torch.zeros(s, dtype=BF, device=DEV) for s in ((rows, n), (rows, k), (E, n, k)))

    def call():
        pb.grouped_gemm_bf16(x, w, offsets, out=out)
        pb.grouped_gemm_bf16_dgrad(dy, w, offsets, out=dx)
        pb.grouped_gemm_bf16_wgrad(dy, x, offsets, out=dw)

    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for i, sizes in enumerate(([0, 500, 0, 0, 0, 0], [100, 1, 99, 200, 0, 30])):
        x.copy_(ints((rows, k), 10 + i))
        offsets.copy_(borders(sizes))
        graph.replay()
        torch.cuda.synchronize()
        end = sum(sizes)
        for got, side, a, b in ((out[:end], "fwd", x, w), (dx[:end], "dgrad", dy, w), (dw, "wgrad", dy, x)):
            assert torch.equal(got, plain(side, sizes, a, b, torch.zeros(got.shape, dtype=torch.float64, device=DEV)).to(BF))


def test_two_streams_at_once(pb):
    sizes = [100, 0, 300, 57]
    offsets, x, w = borders(sizes), ints((457, 256), 1), ints((4, 512, 256), 2)
    want = pb.grouped_gemm_bf16(x, w, offsets)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            got.append(pb.grouped_gemm_bf16(x, w, offsets))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_refusals(pb):
    offsets = borders([4, 4])
    x, w = ints((8, 64), 1), ints((2, 32, 64), 2)
    for bad, error in ((lambda: pb.grouped_gemm_bf16(x.float(), w, offsets), TypeError),
                       (lambda: pb.grouped_gemm_bf16(x, w[0], offsets), ValueError),
                       (lambda: pb.grouped_gemm_bf16(x, w, offsets[:2]), ValueError),
                       (lambda: pb.grouped_gemm_bf16(x, w, offsets.long()), TypeError),
                       (lambda: pb.grouped_gemm_bf16(x[:, :56], w, offsets), ValueError),
                       (lambda: pb.grouped_gemm_bf16(x.cpu(), w, offsets), TypeError),
                       (lambda: pb.grouped_gemm_bf16(x, w.transpose(1, 2), offsets), ValueError),
                       (lambda: pb.grouped_gemm_bf16(x[:, :60], ints((2, 32, 60), 3), offsets), pb.PrismB200Error),
                       (lambda: pb.grouped_gemm_bf16(ints((8, 68), 4)[:, :64], w, offsets), pb.PrismB200Error),
                       (lambda: pb.grouped_gemm_bf16(ints((8, 72), 4)[:, 1:65], w, offsets), pb.PrismB200Error),
                       (lambda: pb.grouped_gemm_bf16_wgrad(x, x, offsets, dtype=torch.float16), TypeError),
                       (lambda: pb.grouped_gemm_bf16_wgrad(x, x[:7], offsets), ValueError),
                       (lambda: pb.grouped_gemm_bf16_dgrad(x, w, offsets), ValueError),
                       (lambda: pb.grouped_gemm_bf16(x, ints((2, 64, 64), 2), offsets, out=x), pb.PrismB200Error)):
        with pytest.raises(error):
            bad()
