"""The operators of a mixture-of-experts layer as they are used together: forward, backward and the 4-bit form."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF = torch.bfloat16


def make(T, E, k, H, F, seed=0, masked=0.1):
    g = torch.Generator(device=DEV).manual_seed(seed)
    randn = lambda *s: torch.randn(s, device=DEV, generator=g)  # noqa: E731
    logits = randn(T, E)
    if masked:
        logits[torch.rand((T,), device=DEV, generator=g) < masked] = float("-inf")
    return logits, randn(T, H).to(BF), (randn(E, F, H) / H ** 0.5).to(BF), (randn(E, H, F) / F ** 0.5).to(BF), randn(T, H).to(BF)


def layer(pb, logits, x, w1, w2, dout, k):
    """Forward and backward of y = sum of weights * relu(x w1') w2' over the chosen experts."""
    r = pb.route_topk(logits, k)
    xs = pb.route_gather(x, r.pos)
    h = pb.grouped_gemm_bf16(xs, w1, r.offsets)
    act = torch.relu(h)
    ys = pb.grouped_gemm_bf16(act, w2, r.offsets)
    y = pb.route_combine(ys, r.pos, r.weights)
    dys, dweights = pb.route_combine_grad(dout, ys, r.pos, r.weights)
    dact = pb.grouped_gemm_bf16_dgrad(dys, w2, r.offsets)
    dw2 = pb.grouped_gemm_bf16_wgrad(dys, act, r.offsets, dtype=torch.float32)
    dh = torch.where(h > 0, dact, torch.zeros_like(dact))
    dxs = pb.grouped_gemm_bf16_dgrad(dh, w1, r.offsets)
    dw1 = pb.grouped_gemm_bf16_wgrad(dh, xs, r.offsets, dtype=torch.float32)
    dx = pb.route_combine(dxs, r.pos)
    dlogits = pb.route_topk_grad(logits, r.ids, r.weights, dweights)
    return {"y": y, "dx": dx, "dw1": dw1, "dw2": dw2, "dlogits": dlogits}, r


def plain(logits, x, w1, w2, dout, ids):
    """The same in fp64 with autograd, a token at a time over its experts by one-hot sums."""
    E = w1.shape[0]
    args = [t.double().requires_grad_() for t in (logits, x, w1, w2)]
    l, x, w1, w2 = args
    chosen = torch.zeros(l.shape, dtype=torch.bool, device=DEV)
    t, j = (ids >= 0).nonzero(as_tuple=True)
    chosen[t, ids[t, j].long()] = True
    kept = torch.where(chosen, l, torch.full_like(l, -1e30))
    gate = torch.where(chosen, torch.softmax(kept, 1), torch.zeros_like(l))
    y = 0
    for e in range(E):
        y = y + gate[:, e:e + 1] * (torch.relu(x @ w1[e].t()) @ w2[e].t())
    grads = torch.autograd.grad(y, args, dout.double())
    return {"y": y.detach(), "dlogits": torch.where(chosen, grads[0], 0.0), "dx": grads[1], "dw1": grads[2], "dw2": grads[3]}


@pytest.mark.parametrize("T,E,k,H,F", [(1, 4, 2, 64, 128), (50, 8, 2, 128, 192), (700, 16, 4, 256, 320)])
def test_layer_and_its_gradients(pb, T, E, k, H, F):
    inputs = make(T, E, k, H, F, seed=T, masked=0.0 if T == 1 else 0.1)
    got, r = layer(pb, *inputs, k)
    want = plain(*inputs, r.ids)
    # Up to four values in a row are rounded to bf16 on the way (h, ys or dys, dact, the output): 2^-8 of each at most,
    # and the relu's border moves by h's rounding.  Over a whole tensor the roundings are independent and half that on
    # average, so 4 * 2^-8 bounds the norm of the difference.
    for name, value in got.items():
        off = (value.double() - want[name]).norm() / want[name].norm().clamp(min=1e-30)
        assert off <= 4 * 2.0 ** -8, (name, float(off))


def test_captured_layer_with_other_tokens(pb):
    """Forward and backward in one graph; replayed for tokens that choose other experts."""
    T, E, k, H, F = 300, 8, 2, 128, 256
    inputs = make(T, E, k, H, F, seed=1)
    layer(pb, *inputs, k)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, r = layer(pb, *inputs, k)
    fresh = make(T, E, k, H, F, seed=2)
    for a, b in zip(inputs, fresh):
        a.copy_(b)
    graph.replay()
    torch.cuda.synchronize()
    want, r2 = layer(pb, *fresh, k)
    assert torch.equal(r.ids, r2.ids) and torch.equal(r.offsets, r2.offsets)
    for name in got:
        assert torch.equal(got[name], want[name]), name


def test_decoding_with_4_bit_experts(pb):
    """The layer's forward with 4-bit matrices is the one with the matrices they stand for."""
    T, E, k, H, F, G = 5, 16, 4, 256, 512, 64
    logits, x, _, _, _ = make(T, E, k, H, F, seed=3, masked=0.0)
    g = torch.Generator(device=DEV).manual_seed(4)

    def quantised(n, kk):
        q = torch.randint(0, 256, (E, n, kk // 2), dtype=torch.uint8, device=DEV, generator=g)
        s = 2.0 ** torch.randint(-7, -4, (E, n, kk // G), device=DEV, generator=g).to(BF)   # scale * (q - 8) is a bf16 number
        v = torch.stack([q & 15, q >> 4], dim=-1).flatten(-2).float() - 8
        return q, s, (v * s.float().repeat_interleave(G, -1)).to(BF)

    q1, s1, w1 = quantised(F, H)
    q2, s2, w2 = quantised(H, F)
    r = pb.route_topk(logits, k)
    xs = pb.route_gather(x, r.pos)
    a = torch.relu(pb.gemv_w4(xs, q1, s1, offsets=r.offsets))
    b = torch.relu(pb.grouped_gemm_bf16(xs, w1, r.offsets))
    # the same products added up in fp32 in another order: the bf16 results are equal or neighbours
    assert ((a.float() - b.float()).abs() <= 2.0 ** -7 * b.float().abs() + 1e-4).all()
    ya = pb.route_combine(pb.gemv_w4(b, q2, s2, offsets=r.offsets), r.pos, r.weights)
    yb = pb.route_combine(pb.grouped_gemm_bf16(b, w2, r.offsets), r.pos, r.weights)
    assert ((ya.float() - yb.float()).abs() <= 3 * 2.0 ** -7 * yb.float().abs().amax()).all()


def test_results_repeat(pb):
    inputs = make(900, 32, 4, 128, 256, seed=7)
    first, _ = layer(pb, *inputs, 4)
    for _ in range(3):
        again, _ = layer(pb, *inputs, 4)
        assert all(torch.equal(first[n], again[n]) for n in first)


def test_wrong_device_is_refused(pb):
    logits, x, w1, _, _ = make(10, 4, 2, 64, 64)
    r = pb.route_topk(logits, 2)
    with pytest.raises(TypeError):
        pb.route_gather(x.cpu(), r.pos)
    with pytest.raises(TypeError):
        pb.grouped_gemm_bf16(x, w1, r.offsets.cpu())


def ints(shape, seed, dtype=BF):
    return torch.randint(-3, 4, shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed)).to(dtype)


def test_matrices_past_32_bits(pb):
    """150 matrices of 4096 x 4096 (2.5 G elements, 5 GB); the first, one past 2^31 elements and the last have rows."""
    E, n = 150, 4096
    used, sizes = (0, 129, E - 1), [0] * E
    for e, s in zip(used, (3, 40, 5)):
        sizes[e] = s
    offsets = torch.tensor([0] + sizes, device=DEV).cumsum(0).to(torch.int32)
    x, dy = ints((48, n), 1), ints((48, n), 2)
    w = torch.empty((E, n, n), dtype=BF, device=DEV)
    for e in used:
        w[e] = ints((n, n), 10 + e)
    groups = [(e, slice(int(offsets[e]), int(offsets[e + 1]))) for e in used]
    out, dx = pb.grouped_gemm_bf16(x, w, offsets), pb.grouped_gemm_bf16_dgrad(dy, w, offsets)
    for e, r in groups:   # integers below 2^24: fp32 sums are exact, one rounding
        assert torch.equal(out[r], (x[r].double() @ w[e].double().t()).to(BF)) and torch.equal(dx[r], (dy[r].double() @ w[e].double()).to(BF))
    for dtype in (BF, torch.float32):
        dw = torch.full((E, n, n), 7.0, dtype=dtype, device=DEV)
        pb.grouped_gemm_bf16_wgrad(dy, x, offsets, out=dw)
        for e, r in groups:
            assert torch.equal(dw[e], (dy[r].double().t() @ x[r].double()).to(dtype))
        assert not dw[130:E - 1].any() and not dw[1:129].any()


def test_4_bit_matrices_past_32_bits(pb):
    """1024 matrices of 4104 x 2048 (4.3 GB of weights, offsets past 2^32 bytes)."""
    E, n, k, group = 1024, 4104, 2048, 128
    sizes = [0] * E
    sizes[1], sizes[700], sizes[E - 1] = 2, 9, 1
    offsets = torch.tensor([0] + sizes, device=DEV).cumsum(0).to(torch.int32)
    q = torch.empty((E, n, k // 2), dtype=torch.uint8, device=DEV)
    scales = torch.ones((E, n, k // group), dtype=BF, device=DEV)
    x = ints((12, k), 3)
    for e in (1, 700, E - 1):
        q[e] = torch.randint(0, 256, (n, k // 2), device=DEV, generator=torch.Generator(device=DEV).manual_seed(e)).to(torch.uint8)
        scales[e, :, ::2] = 0.5
    got = pb.gemv_w4(x, q, scales, offsets=offsets)
    for e in (1, 700, E - 1):
        r = slice(int(offsets[e]), int(offsets[e + 1]))
        v = torch.stack([q[e] & 15, q[e] >> 4], -1).flatten(-2).double() - 8
        assert torch.equal(got[r], (x[r].double() @ (v * scales[e].double().repeat_interleave(group, -1)).t()).to(BF))


def test_rows_past_32_bits(pb):
    """Buffers of 2.4 G elements: rows at both ends."""
    T, k, H, rows = 37, 3, 4096, 590_000
    x, weights = ints((T, H), 4), (ints((T, k), 5, torch.float32) / 4)
    pos = torch.randperm(T * k, device=DEV, generator=torch.Generator(device=DEV).manual_seed(6)).to(torch.int32).view(T, k)
    pos = torch.where(pos < 50, pos, rows - T * k + pos).contiguous()
    at = pos.long()
    y = torch.full((rows, H), 7.0, dtype=BF, device=DEV)
    pb.route_gather(x, pos, out=y)
    assert torch.equal(y[at], x[:, None].expand(T, k, H)) and bool((y[50:rows - T * k + 50] == 7.0).all())
    y[at] = ints((T, k, H), 7)
    assert torch.equal(pb.route_combine(y, pos, weights), (weights[:, :, None].double() * y[at].double()).sum(1).to(BF))
    dy = torch.full((rows, H), 7.0, dtype=BF, device=DEV)
    _, dweights = pb.route_combine_grad(x, y, pos, weights, dy=dy)
    assert torch.equal(dy[at], (weights[:, :, None] * x[:, None].float()).to(BF))
    assert torch.equal(dweights, (y[at].double() * x[:, None].double()).sum(2).float())
    assert bool((dy[50:rows - T * k + 50] == 7.0).all())


def test_threads_on_streams_of_their_own(pb):
    """Four host threads at once: each one's results repeat bit for bit and no call fails."""
    import threading
    wrong = []

    def work(seed):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for T in (1, 60, 130, 900):
                    logits, x, w1, w2, dout = make(T, 16, 3, 128, 192, seed=seed + T)
                    a, r = layer(pb, logits, x, w1, w2, dout, 3)
                    b, _ = layer(pb, logits, x, w1, w2, dout, 3)
                    wrong.extend((seed, T, name) for name in a if not torch.equal(a[name], b[name]))
            stream.synchronize()
        except Exception as e:  # noqa: BLE001 -- reported by the test's own thread
            wrong.append((seed, repr(e)))

    threads = [threading.Thread(target=work, args=(100 * i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and pb.last_error()[0] == 0
