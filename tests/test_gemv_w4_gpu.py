"""Products with 4-bit weights against fp64."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, HF = torch.bfloat16, torch.float16


def borders(sizes):
    return torch.tensor([0] + sizes, device=DEV).cumsum(0).to(torch.int32)


def weights(lead, n, k, group, dtype, zeros, seed, exact=False):
    g = torch.Generator(device=DEV).manual_seed(seed)
    q = torch.randint(0, 256, (*lead, n, k // 2), dtype=torch.uint8, device=DEV, generator=g)
    if exact:
        scales = 2.0 ** torch.randint(-2, 2, (*lead, n, k // group), device=DEV, generator=g)
    else:
        scales = 0.01 + torch.rand((*lead, n, k // group), device=DEV, generator=g) / 10
    z = torch.randint(0, 16, (*lead, n, k // group), dtype=torch.uint8, device=DEV, generator=g) if zeros else None
    return q, scales.to(dtype), z


def dense(q, scales, z, group):
    """scales * (q - z) in fp64, the group's scale and zero point repeated."""
    v = torch.stack([q & 15, q >> 4], dim=-1).flatten(-2).double()
    s = scales.double().repeat_interleave(group, -1)
    zz = torch.full_like(s, 8.0) if z is None else z.double().repeat_interleave(group, -1)
    return s * (v - zz)


def check(pb, sizes, spare, n, k, group, dtype, zeros, seed=0, exact=False, grouped=True):
    E, rows = len(sizes), sum(sizes) + spare
    lead = (E,) if grouped else ()
    q, scales, z = weights(lead, n, k, group, dtype, zeros, seed, exact)
    g = torch.Generator(device=DEV).manual_seed(seed + 1)
    x = (torch.randint(-2, 3, (rows, k), device=DEV, generator=g) if exact else torch.randn((rows, k), device=DEV, generator=g)).to(dtype)
    out = torch.full((rows, n), 7.0, dtype=dtype, device=DEV)
    got = pb.gemv_w4(x, q, scales, zeros=z, offsets=borders(sizes) if grouped else None, out=out)
    w = dense(q, scales, z, group)
    want = torch.full((rows, n), 7.0, dtype=torch.float64, device=DEV)
    terms = torch.zeros_like(want)
    at = 0
    for e, s in enumerate(sizes):
        r = slice(at, at + s)
        we = w[e] if grouped else w
        want[r], terms[r] = x[r].double() @ we.t(), x[r].double().abs() @ we.abs().t()
        at += s
    if exact:   # integers times powers of two: all fp32 sums are exact
        assert torch.equal(got, want.to(dtype)), (sizes, n, k, group)
        return
    # the products are exact; one step of a partial sum per addition inside a group, half a step for the groups' additions
    fp32 = ((group + 2) * 2.0 ** -23 + (k // group + 20) * 2.0 ** -24) * terms
    half_step, least = (2.0 ** -8, 0.0) if dtype == BF else (2.0 ** -11, 2.0 ** -25)
    assert ((got.double() - want).abs() <= fp32 + half_step * (want.abs() + fp32) + least).all(), (sizes, n, k, group)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_one_matrix(pb, dtype, zeros, group):
    for rows, n, slices in ((1, 1, 1), (1, 33, 2), (2, 64, 3), (7, 100, 9), (8, 32, 17), (9, 31, 8), (24, 257, 5), (3, 1000, 40)):
        for exact in (True, False):
            check(pb, [rows], 0, n, 128 * slices, group, dtype, zeros, rows + n, exact, grouped=False)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("zeros", [False, True])
def test_k_that_ends_inside_a_slice(pb, dtype, zeros):
    for group, k in ((32, 32), (32, 160), (32, 1120), (64, 64), (64, 320), (64, 1088), (32, 4064)):
        for exact in (True, False):
            check(pb, [3], 0, 70, k, group, dtype, zeros, k, exact, grouped=False)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_one_or_two_rows_of_long_k(pb, dtype, zeros, group):
    """Slices of 256 k: ends inside one, with and without whole blocks of eight scales, one matrix or several."""
    for n, k in ((70, 4096), (33, 4096 + group), (200, 4096 + 3 * group), (5000, 4224), (8, 12288)):
        for rows in (1, 2):
            check(pb, [rows], 0, n, k, group, dtype, zeros, seed=k, exact=True, grouped=False)
            check(pb, [rows], 0, n, k, group, dtype, zeros, seed=n, grouped=False)
    check(pb, [0, 1, 0, 1], 0, 96, 4096, group, dtype, zeros, seed=5, exact=True)
    check(pb, [0, 1], 1, 96, 4352, group, dtype, zeros, seed=6)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("group", [32, 128])
def test_groups_of_rows(pb, dtype, group):
    for sizes, spare in (([1], 0), ([0, 3, 0], 2), ([8, 9, 1, 0, 16, 17], 0), ([1] * 40, 5), ([0, 0], 1), ([60, 0, 4], 0)):
        for exact in (True, False):
            check(pb, sizes, spare, 97, 512, group, dtype, group == 32, len(sizes), exact)


def test_many_items_per_block(pb):
    """More work items than resident blocks: the rings run on across items."""
    check(pb, [2, 0, 11, 5] * 12, 3, 512, 1152, 128, BF, True, 3, True)
    check(pb, [1], 0, 20000, 256, 64, HF, False, 4, True, grouped=False)
    check(pb, [4], 0, 20000, 2048, 32, BF, True, 5, False, grouped=False)


def test_unaligned_scales_and_zeros(pb):
    n, k, group = 40, 1024, 32
    q, scales, z = weights((), n, k, group, BF, True, 7)
    x = torch.randn((5, k), device=DEV).to(BF)
    want = pb.gemv_w4(x, q, scales, zeros=z)
    s2 = torch.empty(scales.numel() + 1, dtype=BF, device=DEV)[1:].view_as(scales).copy_(scales)
    z2 = torch.empty(z.numel() + 3, dtype=torch.uint8, device=DEV)[3:].view_as(z).copy_(z)
    assert torch.equal(pb.gemv_w4(x, q, s2, zeros=z2), want)


def test_strided_rows(pb):
    q, scales, _ = weights((), 64, 256, 64, HF, False, 8)
    wide = torch.randn((6, 512), device=DEV).to(HF)
    out = torch.zeros((6, 100), dtype=HF, device=DEV)
    got = pb.gemv_w4(wide[:, 8:264], q, scales, out=out[:, 3:67])
    assert torch.equal(got, pb.gemv_w4(wide[:, 8:264].contiguous(), q, scales))
    assert (out[:, :3] == 0).all() and (out[:, 67:] == 0).all()


def test_a_nan_stays_in_its_row(pb):
    q, scales, _ = weights((2,), 64, 256, 64, BF, False, 9)
    x, offsets = torch.randn((12, 256), device=DEV).to(BF), borders([9, 3])
    clean = pb.gemv_w4(x, q, scales, offsets=offsets)
    x[4, 17] = float("nan")
    x[10, 3] = float("inf")
    dirty = pb.gemv_w4(x, q, scales, offsets=offsets)
    keep = [i for i in range(12) if i not in (4, 10)]
    assert torch.equal(clean[keep], dirty[keep]) and not torch.isfinite(dirty[[4, 10]]).any()


@pytest.mark.parametrize("dtype,exponents", [(BF, (120, 100, -100, -119, -120, -126, -130, -133)), (HF, (10, -14, -20, -24))])
def test_the_smallest_and_largest_values(pb, dtype, exponents):
    """x near the ends of its type, subnormals included: products and sums of equal powers of two are exact."""
    k, n = 4096, 40
    q = torch.full((n, k // 2), 0x99, dtype=torch.uint8, device=DEV)   # 9 - 8
    for e in exponents:
        scale = 100 if e < -60 else 8 if e < 0 else -30 if e > 60 else -14
        x = torch.full((2, k), 2.0 ** e, dtype=torch.float64, device=DEV).to(dtype)
        x[1, 1::2] = 0
        scales = torch.full((n, k // 128), 2.0 ** scale, dtype=torch.float64, device=DEV).to(dtype)
        for rows in (x, x.repeat(4, 1)):
            got = pb.gemv_w4(rows, q, scales)[:2].double()
            assert bool((got[0] == k * 2.0 ** (e + scale)).all() and (got[1] == k * 2.0 ** (e + scale - 1)).all()), e


def test_graph_and_streams(pb):
    q, scales, z = weights((3,), 96, 384, 128, BF, True, 10)
    x, offsets = torch.randn((10, 384), device=DEV).to(BF), borders([4, 0, 6])
    out = torch.empty((10, 96), dtype=BF, device=DEV)
    pb.gemv_w4(x, q, scales, z, offsets, out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pb.gemv_w4(x, q, scales, z, offsets, out)
    x.copy_(torch.randn((10, 384), device=DEV).to(BF))
    offsets.copy_(borders([1, 9, 0]))
    graph.replay()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        want = pb.gemv_w4(x, q, scales, z, offsets)
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_empty(pb):
    q, scales, _ = weights((), 64, 256, 64, HF, False, 8)
    assert pb.gemv_w4(torch.empty((0, 256), dtype=HF, device=DEV), q, scales).shape == (0, 64)


def test_refusals(pb):
    q, scales, z = weights((2,), 64, 256, 64, HF, True, 8)
    x, offsets = torch.zeros((4, 256), dtype=HF, device=DEV), borders([2, 2])
    for bad, error in ((lambda: pb.gemv_w4(x.float(), q, scales, z, offsets), TypeError),
                       (lambda: pb.gemv_w4(x, q, scales.to(BF), z, offsets), TypeError),
                       (lambda: pb.gemv_w4(x, q, scales), ValueError),
                       (lambda: pb.gemv_w4(x[:, :128], q, scales, z, offsets), ValueError),
                       (lambda: pb.gemv_w4(x, q, scales, z[:, :, :3], offsets), ValueError),
                       (lambda: pb.gemv_w4(x, q, scales, z, offsets[:2]), ValueError),
                       (lambda: pb.gemv_w4(x, q.to(torch.int8), scales, z, offsets), TypeError),
                       (lambda: pb.gemv_w4(x, q, scales[:, :, :1].contiguous(), None, offsets), pb.PrismB200Error),   # a group of 256
                       (lambda: pb.gemv_w4(torch.zeros((4, 260), dtype=HF, device=DEV)[:, 1:257], q, scales, z, offsets), pb.PrismB200Error)):
        with pytest.raises(error):
            bad()
