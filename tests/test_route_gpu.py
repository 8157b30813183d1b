"""Routing of rows to experts: choices, order, gather, combine and their gradients against plain NumPy / fp64 forms."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
INF = float("inf")


def plain_route(logits, k, renorm):
    """Choices by a stable sort in fp64, order by a stable sort of the experts."""
    l = logits.double().cpu().numpy()
    l = np.where(np.isnan(l), -np.inf, l)
    T, E = l.shape
    ids = np.argsort(-l, axis=1, kind="stable")[:, :k].astype(np.int32)
    top = np.take_along_axis(l, ids.astype(np.int64), 1)
    ids = np.where(top > -np.inf, ids, -1)
    m = np.where(top[:, :1] > -np.inf, top[:, :1], 0.0)
    e = np.where(ids >= 0, np.exp(np.where(ids >= 0, top, 0.0) - m), 0.0)
    total = e.sum(1, keepdims=True) if renorm else np.exp(l - m).sum(1, keepdims=True)
    weights = e / np.where(total > 0, total, 1.0)
    flat = ids.reshape(-1)
    rows = np.argsort(np.where(flat < 0, E, flat), kind="stable")
    n = int((flat >= 0).sum())
    order = np.full(T * k, -1, np.int32)
    order[:n] = rows[:n]
    pos = np.full(T * k, -1, np.int32)
    pos[rows[:n]] = np.arange(n)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat[flat >= 0], minlength=E))]).astype(np.int32)
    return ids, weights, pos.reshape(T, k), order, offsets


def check_route(pb, logits, k, renorm, **kw):
    r = pb.route_topk(logits, k, renormalize=renorm, **kw)
    ids, weights, pos, order, offsets = plain_route(logits, k, renorm)
    for name, want in (("ids", ids), ("pos", pos), ("order", order), ("offsets", offsets)):
        assert np.array_equal(getattr(r, name).cpu().numpy(), want), name
    # exp: 2 ulp, its argument rounded once (|l - m| <= 64 here: 2^-24 * 64), up to 37 additions, one division
    tol = weights * (2.0 ** -22 + 2.0 ** -18 + 40 * 2.0 ** -24) + 1e-37
    assert (np.abs(r.weights.cpu().numpy().astype(np.float64) - weights) <= tol).all()
    return r


def make_logits(T, E, dtype, seed, masked=0.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    l = 3 * torch.randn((T, E), device=DEV, generator=g)
    if masked:
        l[torch.rand((T, E), device=DEV, generator=g) < masked] = -INF
        l[torch.rand((T,), device=DEV, generator=g) < masked] = -INF
    return l.to(dtype)


@pytest.mark.parametrize("T", [1, 3, 32, 63, 64, 65, 127, 129, 500, 4736, 4737, 20001])
@pytest.mark.parametrize("E,k", [(8, 2), (64, 8)])
def test_token_counts(pb, T, E, k):
    check_route(pb, make_logits(T, E, torch.float32, T + E, 0.1), k, True)


@pytest.mark.parametrize("E,k", [(1, 1), (2, 2), (31, 7), (32, 32), (33, 3), (65, 1), (128, 8), (200, 9), (256, 16), (300, 5), (512, 8),
                                 (513, 32), (1000, 4), (1024, 32)])
@pytest.mark.parametrize("renorm", [True, False])
def test_expert_counts(pb, E, k, renorm):
    for T in (5, 700):
        check_route(pb, make_logits(T, E, torch.float32, 7 * E + k, 0.2), k, renorm)


@pytest.mark.parametrize("dtype", DTYPES)
def test_types_and_ties(pb, dtype):
    check_route(pb, make_logits(777, 96, DTYPES[dtype], 5), 6, False)
    coarse = (make_logits(300, 100, torch.float32, 6) / 2).round().to(DTYPES[dtype])   # many equal logits, both zeros
    coarse = torch.where((coarse == 0) & (torch.rand_like(coarse, dtype=torch.float32) < 0.5), -coarse, coarse)
    check_route(pb, coarse, 8, True)
    check_route(pb, torch.zeros((130, 40), dtype=DTYPES[dtype], device=DEV), 5, True)


def test_masks(pb):
    l = make_logits(260, 33, torch.float32, 9)
    l[::3] = -INF                                        # rows that choose nothing
    l[1::3, 2:] = -INF                                   # fewer open experts than choices
    check_route(pb, l, 4, True)
    check_route(pb, l, 4, False)
    r = check_route(pb, torch.full((200, 16), -INF, device=DEV), 3, True)
    assert int(r.offsets[-1]) == 0 and int((r.order != -1).sum()) == 0
    lowest = torch.finfo(torch.float32).min              # a mask of the type's lowest value is a number like others
    l = torch.full((140, 20), lowest, device=DEV)
    l[:, 7] = 1.0
    r = check_route(pb, l, 2, True)
    assert (r.ids[:, 0] == 7).all() and (r.ids[:, 1] == 0).all()
    check_route(pb, torch.full((3, 20), lowest, device=DEV), 4, False)
    for dtype in DTYPES.values():                        # NaN is passed over
        for experts in (24, 100, 300):
            l = make_logits(150, experts, torch.float32, 10, 0.1)
            l[torch.rand_like(l) < 0.3] = float("nan")
            check_route(pb, l.to(dtype), 5, True)
            check_route(pb, l.to(dtype), 5, False)
        low = torch.full((90, 40), torch.finfo(dtype).min, dtype=dtype, device=DEV)
        low[:, 30] = torch.finfo(dtype).max
        r = check_route(pb, low, 2, True) if dtype != torch.float32 else pb.route_topk(low, 2)   # max - min overflows fp32: weights 1, 0
        assert (r.ids[:, 0] == 30).all() and (r.ids[:, 1] == 0).all() and (r.weights[:, 0] == 1).all()


def test_strided_logits_given_outputs_and_workspace(pb):
    wide = make_logits(900, 160, torch.bfloat16, 11)
    logits = wide[:, 40:131]
    ws = torch.full((pb.route_workspace_size(900, 91, 6),), 255, dtype=torch.uint8, device=DEV)
    first = check_route(pb, logits, 6, True, workspace=ws)
    again = check_route(pb, make_logits(900, 91, torch.bfloat16, 12), 6, True, out=first, workspace=ws)
    assert all(a.data_ptr() == b.data_ptr() for a, b in zip(first, again))


def test_no_tokens(pb):
    r = pb.route_topk(torch.empty((0, 12), device=DEV), 3)
    assert r.ids.shape == (0, 3) and r.offsets.tolist() == [0] * 13


def test_other_stream_and_graph(pb):
    logits = make_logits(1000, 64, torch.float32, 13)
    want = check_route(pb, logits, 4, True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = pb.route_topk(logits, 4)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    into = pb.Routing(*(torch.empty_like(t) for t in want))
    ws = torch.empty(pb.route_workspace_size(1000, 64, 4), dtype=torch.uint8, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pb.route_topk(logits, 4, out=into, workspace=ws)
    fresh = make_logits(1000, 64, torch.float32, 14)
    logits.copy_(fresh)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    want = check_route(pb, fresh, 4, True)
    assert all(torch.equal(a, b) for a, b in zip(want, into))


# ---- the weights' gradient ------------------------------------------------------------------------------------
def plain_grad(logits, ids, g, renorm):
    l = logits.double()
    l = torch.where(torch.isnan(l), -INF, l)
    chosen = ids >= 0
    at = torch.where(chosen, ids, 0).long()
    G = torch.zeros_like(l).scatter_add_(1, at, torch.where(chosen, g.double(), 0.0))
    if renorm:
        member = torch.zeros_like(l).scatter_add_(1, at, chosen.double()) > 0
        l = torch.where(member, l, -INF)
    m = l.amax(1, keepdim=True)
    p = torch.where(l > -INF, torch.exp(l - torch.where(m > -INF, m, 0.0)), 0.0)
    p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
    return p * (G - (p * G).sum(1, keepdim=True))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("T,E,k", [(1, 8, 2), (77, 33, 5), (300, 128, 8), (41, 200, 3), (9, 1000, 32), (64, 40, 1)])
def test_route_grad(pb, dtype, renorm, T, E, k):
    logits = make_logits(T, E, DTYPES[dtype], T + E + k, 0.15)
    r = pb.route_topk(logits, k, renormalize=renorm)
    g = torch.randn((T, k), device=DEV, generator=torch.Generator(device=DEV).manual_seed(3))
    got = pb.route_topk_grad(logits, r.ids, r.weights, g, renormalize=renorm)
    want = plain_grad(logits, r.ids, g, renorm)
    assert got.dtype == logits.dtype and torch.isfinite(got).all()
    # p to 5e-6 of itself (see check_route), the mean of up to 32 terms g * w to 40 * 2^-24 * max|g| + the weights' share;
    # then the type's rounding (fp16: below 2^-14 its step is 2^-24)
    big = g.abs().amax(1, keepdim=True).double()
    fp32 = 5e-6 * (want.abs() + 2 * big)
    half_step = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}[dtype]
    tol = fp32 + half_step * (want.abs() + fp32) + (2.0 ** -25 if dtype == "f16" else 0.0)
    assert ((got.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("renorm", [True, False])
def test_route_grad_against_differences(pb, renorm):
    """The gradient of sum(c * weights), in fp64 differences of the plain form around the same choice."""
    logits = make_logits(6, 12, torch.float32, 21)
    r = pb.route_topk(logits, 3, renormalize=renorm)
    c = torch.randn((6, 3), device=DEV, generator=torch.Generator(device=DEV).manual_seed(4))
    got = pb.route_topk_grad(logits, r.ids, r.weights, c, renormalize=renorm).double()
    l, ids = logits.double(), r.ids.long()

    def loss(l):
        over = l.gather(1, ids) if renorm else l
        return (c.double() * torch.exp(l.gather(1, ids) - torch.logsumexp(over, 1, keepdim=True))).sum(1)

    h = 1e-5
    for e in range(12):
        d = torch.zeros_like(l)
        d[:, e] = h
        diff = (loss(l + d) - loss(l - d)) / (2 * h)
        assert ((diff - got[:, e]).abs() <= 1e-5 * (1 + c.abs().amax(1).double())).all()   # h^2 and fp32, both below 1e-5


# ---- rows between token order and expert order -------------------------------------------------------------------
def make_pos(T, k, E, seed, dropped=0.2):
    logits = make_logits(T, E, torch.float32, seed, dropped)
    import prism_b200
    return prism_b200.route_topk(logits, k)


WIDTHS = [1, 2, 7, 8, 36, 64, 250, 256, 1000, 2047, 2048, 4104, 40000]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H", WIDTHS)
def test_gather_and_combine(pb, dtype, H):
    dt = DTYPES[dtype]
    T, k, E = (37, 3, 8) if H < 40000 else (5, 2, 4)
    r = make_pos(T, k, E, H)
    gen = torch.Generator(device=DEV).manual_seed(H)
    x = torch.randn((T, H), device=DEV, generator=gen).to(dt)
    out = torch.full((T * k + 3, H), 7.0, dtype=dt, device=DEV)
    got = pb.route_gather(x, r.pos, out=out)
    want = torch.full_like(out, 7.0)                      # rows behind the last keep what they held
    live = r.pos >= 0
    want[r.pos[live].long()] = x[torch.arange(T, device=DEV)[:, None].expand(T, k)[live]]
    assert torch.equal(got, want)

    y = torch.randn((T * k, H), device=DEV, generator=gen).to(dt)
    y[int(r.offsets[-1]):] = float("nan")                 # never read
    for weights in (r.weights, None):
        w = torch.where(live, torch.ones_like(r.weights) if weights is None else weights, 0.0).double()
        terms = w[..., None] * torch.where(live[..., None], y[r.pos.clamp(min=0).long()].double(), 0.0)
        want = terms.sum(1)
        got = pb.route_combine(y, r.pos, weights)
        fp32 = (k + 1) * 2.0 ** -24 * terms.abs().sum(1)  # one rounding per fused multiply-add
        half_step = {"f32": 0.0, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}[dtype]
        assert ((got.double() - want).abs() <= fp32 + half_step * (want.abs() + fp32) + 2.0 ** -25 * (dtype == "f16")).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,k,H", [(37, 3, 1), (37, 1, 7), (20, 4, 64), (9, 2, 250), (300, 8, 1000), (11, 5, 2047), (6, 16, 2048), (3, 32, 4104),
                                   (2, 9, 40000)])
def test_combine_grad(pb, dtype, T, k, H):
    dt = DTYPES[dtype]
    r = make_pos(T, k, 40, H + k)
    gen = torch.Generator(device=DEV).manual_seed(H + 1)
    dout = torch.randn((T, H), device=DEV, generator=gen).to(dt)
    y = torch.randn((T * k, H), device=DEV, generator=gen).to(dt)
    y[int(r.offsets[-1]):] = float("nan")
    dy = torch.full((T * k, H), 7.0, dtype=dt, device=DEV)
    got, dw = pb.route_combine_grad(dout, y, r.pos, r.weights, dy=dy)
    live = r.pos >= 0
    token = torch.arange(T, device=DEV)[:, None].expand(T, k)[live]
    want = torch.full_like(dy, 7.0)
    want[r.pos[live].long()] = (r.weights[live][:, None] * dout[token].float()).to(dt)   # one fp32 product, rounded once
    assert torch.equal(got, want)
    prod = dout[token].double() * y[r.pos[live].long()].double()
    # a thread adds at most H / 32 + 8 terms, then 5 + 8 additions
    tol = (H / 32 + 24) * 2.0 ** -24 * prod.abs().sum(1)
    assert ((dw[live].double() - prod.sum(1)).abs() <= tol).all()
    assert (dw[~live] == 0).all()


def test_rows_with_strides_and_offsets(pb):
    """Views into wider buffers, at addresses that allow only narrow accesses."""
    r = make_pos(50, 2, 8, 3)
    gen = torch.Generator(device=DEV).manual_seed(9)
    for shift, width in ((8, 64), (4, 60), (2, 62), (1, 63)):
        x = torch.randn((50, 200), device=DEV, generator=gen).to(torch.bfloat16)[:, shift:shift + width]
        buf = torch.zeros((100, 136), dtype=torch.bfloat16, device=DEV)
        got = pb.route_gather(x, r.pos, out=buf[:, 3:3 + width])
        assert torch.equal(got, pb.route_gather(x.contiguous(), r.pos, out=torch.zeros((100, width), dtype=torch.bfloat16, device=DEV)))
        assert (buf[:, :3] == 0).all() and (buf[:, 3 + width:] == 0).all()
        assert torch.equal(pb.route_combine(got, r.pos, r.weights), pb.route_combine(got.contiguous(), r.pos, r.weights))
        a, b = pb.route_combine_grad(x, got, r.pos, r.weights, dy=torch.zeros_like(got))
        c, d = pb.route_combine_grad(x.contiguous(), got.contiguous(), r.pos, r.weights, dy=torch.zeros_like(got))
        assert torch.equal(a, c) and torch.allclose(b, d, rtol=0, atol=64 * 2.0 ** -22 * 100)


def test_gather_and_combine_are_adjoint(pb):
    """<gather(x), y> = <x, combine(y)>, exactly in integers."""
    r = make_pos(300, 4, 16, 5)
    gen = torch.Generator(device=DEV).manual_seed(2)
    x = torch.randint(-3, 4, (300, 96), device=DEV, generator=gen).float()
    y = torch.randint(-3, 4, (1200, 96), device=DEV, generator=gen).float()
    xs = pb.route_gather(x, r.pos, out=torch.zeros_like(y))
    assert (xs * y).sum().item() == (x * pb.route_combine(y, r.pos)).sum().item()


def test_positions_outside_the_rows_are_passed_over(pb):
    x = torch.ones((4, 16), device=DEV)
    pos = torch.tensor([[0, 9], [1, -1], [100000, 2], [-7, 3]], dtype=torch.int32, device=DEV)
    out = pb.route_gather(x, pos, out=torch.zeros((4, 16), device=DEV))
    assert (out == 1).all()
    assert pb.route_combine(out, pos).sum(1).tolist() == [16.0] * 4
    dy, dw = pb.route_combine_grad(x, out, pos, torch.ones((4, 2), device=DEV))
    assert dw.tolist() == [[16.0, 0.0], [16.0, 0.0], [0.0, 16.0], [0.0, 16.0]] and (dy == 1).all()


def test_refusals(pb):
    logits = torch.zeros((4, 8), device=DEV)
    for bad, error in ((lambda: pb.route_topk(logits, 9), ValueError), (lambda: pb.route_topk(logits, 0), ValueError),
                       (lambda: pb.route_topk(logits.double(), 2), TypeError), (lambda: pb.route_topk(logits.t(), 2), ValueError),
                       (lambda: pb.route_topk(logits[0], 2), ValueError), (lambda: pb.route_topk(torch.zeros((2, 1025), device=DEV), 2), pb.PrismB200Error),
                       (lambda: pb.route_topk(torch.zeros((2, 64), device=DEV), 33), pb.PrismB200Error),
                       (lambda: pb.route_topk(torch.zeros((500, 8), device=DEV), 2, workspace=torch.empty(8, dtype=torch.uint8, device=DEV)), ValueError)):
        with pytest.raises(error):
            bad()
    r = pb.route_topk(logits, 2)
    x = torch.zeros((4, 32), device=DEV)
    with pytest.raises(TypeError):
        pb.route_gather(x, r.pos.long())
    with pytest.raises(ValueError):
        pb.route_gather(x[:3], r.pos)
    with pytest.raises(pb.PrismB200Error):
        pb.route_gather(x, r.pos, out=x)
    with pytest.raises(TypeError):
        pb.route_combine(x, r.pos, r.weights.double())
    with pytest.raises(pb.PrismB200Error):
        pb.route_combine(x, r.pos, out=x)
    y = torch.zeros((8, 32), device=DEV)
    with pytest.raises(pb.PrismB200Error):
        pb.route_combine_grad(x, y, r.pos, r.weights, dy=y)
    with pytest.raises(ValueError):
        pb.route_topk_grad(logits, r.ids, r.weights[:3], r.weights)
    with pytest.raises(pb.PrismB200Error):
        pb.route_topk_grad(logits, r.ids, r.weights, r.weights, out=logits)


def test_own_scratch_lives_until_the_call_is_queued(pb, monkeypatch):
    """Memory that another thread allocates while the launches are queued is not the call's own scratch."""
    from prism_b200 import experts
    inner, seen = experts._run, []

    def run(device, fn, *args):
        other = torch.empty(pb.route_workspace_size(500, 64, 4), dtype=torch.uint8, device=device)
        seen.append((args[-1], other.data_ptr()))
        inner(device, fn, *args)

    logits = make_logits(500, 64, torch.float32, 3)
    pb.route_topk(logits, 4)   # leaves a block of that size with the allocator
    monkeypatch.setattr(experts, "_run", run)
    pb.route_topk(logits, 4)
    (scratch, other), = seen
    assert scratch and scratch != other


@pytest.mark.parametrize("E,k", [(8, 8), (64, 8), (256, 3)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_every_16_bit_pattern(pb, dtype, E, k):
    """All 65536 patterns, several times among others: both zeros, subnormals, infinities and NaNs."""
    g = torch.Generator(device=DEV).manual_seed(E)
    bits = torch.cat([torch.randperm(1 << 16, device=DEV, generator=g) for _ in range(4)])
    logits = bits.to(torch.int32).sub(1 << 15).to(torch.int16).view(DTYPES[dtype]).view(-1, E)
    ids, _, pos, order, offsets = plain_route(logits, k, True)
    r = pb.route_topk(logits, k)
    for name, want in (("ids", ids), ("pos", pos), ("order", order), ("offsets", offsets)):
        assert np.array_equal(getattr(r, name).cpu().numpy(), want), name


@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("T,E,k", [(3, 8, 1), (64, 40, 8), (70, 64, 4), (999, 128, 8), (4801, 504, 7), (300, 1024, 8)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_16_bit_logits_in_vectors_or_not(pb, dtype, T, E, k, renorm):
    """Whole 16-byte vectors take another way than rows at odd strides; both make the same choice."""
    logits = make_logits(T, E, DTYPES[dtype], T, 0.2)
    logits[::7] = logits[::7].round()   # ties
    check_route(pb, logits, k, renorm)
    odd = torch.zeros((T, E + 3), dtype=DTYPES[dtype], device=DEV)[:, 1:E + 1]
    odd.copy_(logits)
    a, b = pb.route_topk(logits, k, renormalize=renorm), pb.route_topk(odd, k, renormalize=renorm)
    for name in ("ids", "pos", "order", "offsets"):
        assert torch.equal(getattr(a, name), getattr(b, name)), name


def test_blocks_of_more_tokens_than_16_bits_count(pb):
    """65537 tokens per block: the counts between the launches are 32 bits wide."""
    T, E = 148 * 65536 + 5, 3
    logits = torch.randn((T, E), device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    logits[:, 2] -= 30.0   # so that a block has more than 65535 rows of one expert
    logits[: 3 * 65536, 0] += 60.0
    r = pb.route_topk(logits, 1)
    ids = logits.argmax(1)
    assert torch.equal(r.ids[:, 0].long(), ids) and bool((r.weights == 1).all())
    counts = torch.bincount(ids, minlength=E)
    assert torch.equal(r.offsets.long(), torch.cat([counts.new_zeros(1), counts.cumsum(0)]))
    rows = torch.sort(ids, stable=True).indices
    assert torch.equal(r.order.long(), rows)
    want = torch.empty_like(rows)
    want[rows] = torch.arange(T, device=DEV)
    assert torch.equal(r.pos[:, 0].long(), want)
