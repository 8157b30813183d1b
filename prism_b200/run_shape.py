"""Run one kernel family on one shape and print its time: `python -m prism_b200.run_shape gemm_bf16 4096 8192 8192`.

For looking at a shape that the benchmark does not time by itself (a shard of the multi-GPU run on one GPU, a block of
a host plan) with CUDA events or under a profiler.  Inputs are seeded; every launch is timed on its own.

    gemm_bf16 M N K     D = A * B^T, bf16 in and out, C column-major     (prism_b200.runmyh100)
    sgemm M N K         C = 1.5 * A * B + 0.5 * C in fp32, kernel 5       (prism_b200.run_my_kernel)
    scan N              inclusive scan of N uint32 values in place        (prism_b200.launch_scan)
    route T E C         the C of E experts of T tokens, bf16 logits       (prism_b200.route_topk)
    combine T C H       C rows of H bf16 values added up per token        (prism_b200.route_combine)
    combine_grad T C H  its gradient                                      (prism_b200.route_combine_grad)
    grouped R E N K     R rows in E equal groups times N x K matrices     (prism_b200.grouped_gemm_bf16)
    grouped_wgrad R E N K   the matrices' gradients in bf16               (prism_b200.grouped_gemm_bf16_wgrad)
    gemv_w4 R N K       R rows times one N x K matrix of 4-bit weights in groups of 128 (prism_b200.gemv_w4)
"""
from __future__ import annotations

import argparse

import torch

import prism_b200 as pb


EXPERTS = ("route", "combine", "combine_grad", "grouped", "grouped_wgrad", "gemv_w4")


def expert_case(family, dims, dev, g):
    """The call, its work per launch and the unit of the rate for the operators of an expert layer."""
    bf = torch.bfloat16
    rand = lambda *s: (torch.randn(s, device=dev, generator=g) * 0.1).to(bf)  # noqa: E731
    if family == "route":
        T, E, C = dims
        logits = rand(T, E)
        out, ws = pb.route_topk(logits, C), torch.empty(pb.route_workspace_size(T, E, C), dtype=torch.uint8, device=dev)
        return (lambda: pb.route_topk(logits, C, out=out, workspace=ws)), T * (2.0 * E + 16 * C) + 4 * (E + 1), "GB/s"
    if family in ("combine", "combine_grad"):
        T, C, H = dims
        r = pb.route_topk(rand(T, 8 * C), C)
        y, d = rand(T * C, H), rand(T, H)
        if family == "combine":
            return (lambda: pb.route_combine(y, r.pos, r.weights, out=d)), T * (2.0 * H * (C + 1) + 8 * C), "GB/s"
        dy, dw = torch.empty_like(y), torch.empty_like(r.weights)
        return (lambda: pb.route_combine_grad(d, y, r.pos, r.weights, dy, dw)), T * (2.0 * H * (2 * C + 1) + 12 * C), "GB/s"
    if family == "gemv_w4":
        R, N, K = dims
        q = torch.randint(0, 256, (N, K // 2), dtype=torch.uint8, device=dev, generator=g)
        x, scales = rand(R, K), rand(N, K // 128)
        out = torch.empty((R, N), dtype=bf, device=dev)
        return (lambda: pb.gemv_w4(x, q, scales, out=out)), N * K / 2 + 2.0 * scales.numel() + 2.0 * R * (N + K), "GB/s"
    R, E, N, K = dims
    offsets = torch.tensor([R * e // E for e in range(E + 1)], dtype=torch.int32, device=dev)
    x = rand(R, K)
    if family == "grouped":
        w, out = rand(E, N, K), torch.empty((R, N), dtype=bf, device=dev)
        return (lambda: pb.grouped_gemm_bf16(x, w, offsets, out=out)), 2.0 * R * N * K, "GFLOP/s"
    dy, dw = rand(R, N), torch.empty((E, N, K), dtype=bf, device=dev)
    return (lambda: pb.grouped_gemm_bf16_wgrad(dy, x, offsets, out=dw)), 2.0 * R * N * K, "GFLOP/s"


def main() -> int:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("family", choices=["gemm_bf16", "sgemm", "scan", *EXPERTS])
    ap.add_argument("dims", type=int, nargs="+")
    ap.add_argument("--launches", type=int, default=10)
    ap.add_argument("--device", default="cuda:0")
    a = ap.parse_args()
    dev = torch.device(a.device)
    torch.cuda.set_device(dev)
    g = torch.Generator(device=dev).manual_seed(1234)
    if a.family == "scan":
        (n,) = a.dims
        x0 = torch.randint(0, 2, (n,), dtype=torch.int32, device=dev, generator=g)
        x = x0.clone()
        ws = pb.scan_workspace(n, dev)
        restore, run = (lambda: x.copy_(x0)), (lambda: pb.launch_scan(n, x, ws))
        work, unit = 8.0 * n, "GB/s"
    elif a.family in EXPERTS:
        restore = lambda: None  # noqa: E731
        run, work, unit = expert_case(a.family, a.dims, dev, g)
    else:
        M, N, K = a.dims
        if a.family == "gemm_bf16":
            A = (torch.randn((M, K), device=dev, generator=g) * 0.1).to(torch.bfloat16)
            B = (torch.randn((N, K), device=dev, generator=g) * 0.1).to(torch.bfloat16)
            C = torch.empty((N, M), dtype=torch.bfloat16, device=dev)
            restore, run = (lambda: None), (lambda: pb.runmyh100(M, N, K, A, B, C))
        else:
            A = torch.rand((M, K), device=dev, generator=g) * 2 - 1
            B = torch.rand((K, N), device=dev, generator=g) * 2 - 1
            C0 = torch.rand((M, N), device=dev, generator=g) * 2 - 1
            C = C0.clone()
            restore, run = (lambda: C.copy_(C0)), (lambda: pb.run_my_kernel(5, M, N, K, 1.5, A, B, 0.5, C))
        work, unit = 2.0 * M * N * K, "GFLOP/s"
    times = []
    for _ in range(a.launches):
        restore()
        start, stop = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        run()
        stop.record()
        stop.synchronize()
        times.append(start.elapsed_time(stop))
    code, msg = pb.last_error()
    if code:
        raise SystemExit(f"prism_b200: {msg}")
    best, med = min(times), sorted(times)[len(times) // 2]
    print(f"{a.family} {' x '.join(map(str, a.dims))}: median {med:.4f} ms ({work / med / 1e6:.1f} {unit}), "
          f"best {best:.4f} ms ({work / best / 1e6:.1f} {unit}) of {a.launches} launches")
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
