// Products of a few rows with matrices of 4-bit weights:
//   y[r, n] = sum over groups g of s[n, g] * sum over k in g of (q[n, k] - z[n, g]) * x[r, k]
// with one matrix for all rows or one per expert (rows grouped by offsets, as in grouped_gemm.cu).
//
// What bounds it: the weights, half a byte each, are read once; a row of x adds 2 flop per weight, so for up to about
// eight rows the kernel has to stream.  The hard part is turning nibbles into operands fast enough: an SM has to take
// 23 bytes (46 weights) per clock to keep up with HBM.
//   * Products and sums are mma.sync m16n8k16 with fp32 accumulators: 16 weight rows x 16 k against up to 8 rows of x.
//     tcgen05 would want the converted weights in shared memory, a round trip of four times the bytes read here.
//   * A nibble becomes an operand by one shift and one LOP3: put into the four top bits of the mantissa of 16.0 it
//     makes 16 + q, exactly, in bf16 and fp16 alike.  The 16 + z is taken off afterwards, once per group, in fp32:
//     sum (q - z) x = sum (16 + q) x - (16 + z) * sum x, with sum x from one more MMA whose weight operand is all ones.
//     The larger terms cost at most 3 bits of the fp32 accumulator's 24, far below the rounding of y to 16 bits.
//   * A 32-bit word holds 8 consecutive k; the MMA's order of k is free as long as both operands follow it, so the
//     pairs are (k, k + 4) as the masks deliver them, and x is brought into that order by four PRMTs per 8 values.
//   * The four lanes of a quad take the four words of 32 consecutive k, so a group of 32, 64 or 128 is 1, 2 or 4 steps
//     and its sum is complete in the accumulator when its scale is applied (fp32).
//   * A warp owns 32 weight rows and every 8th slice of 128 k; slices (and the rows of x that go with them) arrive by
//     cp.async in a ring of the warp's own, which runs on across work items: no block barrier is between a load and
//     its use.  The eight warps' sums meet in shared memory once per item, added in warp order.
#include "common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace prism_b200 {
namespace {

namespace w4 {
constexpr int WARPS = 8;
constexpr int THREADS = 32 * WARPS;
constexpr int ROWS = 32;                 // weight rows per item
constexpr int SLICE = 128;               // k per stage
constexpr int W_BYTES = ROWS * SLICE / 2;
constexpr int X_PITCH = SLICE * 2;
constexpr int COLS = 8;                  // rows of x per item: the columns of one MMA
constexpr int RED_PITCH = 36;            // a fragment's 8 x 4 places lie in 32 banks
constexpr int RED_FLOATS = WARPS * COLS * RED_PITCH;
constexpr int MAX_EXPERTS = 1024;

// A stage: 32 weight rows of 64 bytes, then the rows of x of 256 bytes, in 16-byte pieces.  The pieces of a row are
// permuted so that a step's reads lie in 32 different banks: 8 weight rows' words of one piece, and a quarter warp's two
// rows of x with four pieces each.
__device__ __forceinline__ int w_piece(int row, int piece) { return row * (SLICE / 2) + ((piece ^ ((row >> 1) & 3)) << 4); }
__device__ __forceinline__ int x_piece(int row, int piece) { return W_BYTES + row * X_PITCH + ((piece ^ ((row & 1) << 2)) << 4); }

struct Smem {
    int stage, ring, bytes;              // ring: all warps' stages
    __host__ __device__ Smem(int stages, int rows, int experts)
        : stage(W_BYTES + (rows < COLS ? rows : COLS) * X_PITCH), ring(WARPS * stages * stage),
          bytes(ring + RED_FLOATS * 4 + (3 * experts + 1) * 4) {}
};
}  // namespace w4

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <typename T> struct W4Type;
template <> struct W4Type<__nv_bfloat16> {
    static constexpr uint32_t ONES = 0x3F803F80u;
    // nibble i of the word's two halves -> (16 + q) twice; 16.0 is 0x4180, the mantissa's top four bits are bits 3-6
    template <int I> static __device__ __forceinline__ uint32_t pair(uint32_t w) {
        const uint32_t s = I == 0 ? w << 3 : w >> (4 * I - 3);
        return (s & 0x00780078u) | 0x41804180u;
    }
    static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
    static __device__ __forceinline__ float to_f32(uint16_t v) { return __uint_as_float(static_cast<uint32_t>(v) << 16); }
    static __device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }
};
template <> struct W4Type<__half> {
    static constexpr uint32_t ONES = 0x3C003C00u;
    // 16.0 is 0x4C00, the mantissa's top four bits are bits 6-9
    template <int I> static __device__ __forceinline__ uint32_t pair(uint32_t w) {
        const uint32_t s = I < 2 ? w << (6 - 4 * I) : w >> (4 * I - 6);
        return (s & 0x03C003C0u) | 0x4C004C00u;
    }
    static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
    static __device__ __forceinline__ float to_f32(uint16_t v) { return __half2float(__ushort_as_half(v)); }
    static __device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }
};

struct W4Args {
    const void* x;
    long long ldx;
    const uint8_t* q;
    const uint16_t* scales;
    const uint8_t* zeros;     // null: 8 everywhere
    const int* offsets;       // null: one matrix, all rows
    void* out;
    long long ldo;
    int rows, experts, n, k;
    int aligned;              // a slice's scales (zeros) of a row can be read as one vector
};

struct Item {
    int e, n0, r0, cols;
};

// A warp's place in the sequence of (item, slice) pairs that its CTA works through; moves forward only.
struct Cursor {
    int t, s, e = 0;
    Item item;
    __device__ __forceinline__ void decode(const W4Args& a, const int* first, const int* last, const int* items, int n_tiles) {
        while (items[e + 1] <= t) ++e;
        const int in = t - items[e];
        const int chunks = (last[e] - first[e] + w4::COLS - 1) / w4::COLS;   // chunks of one weight tile follow one another: L2
        const int tile = in / chunks, chunk = in - tile * chunks;
        item.e = e;
        item.n0 = tile * w4::ROWS;
        item.r0 = first[e] + chunk * w4::COLS;
        item.cols = min(w4::COLS, last[e] - item.r0);
    }
};

template <typename T, int G, bool Z, int STAGES>
__global__ void __launch_bounds__(w4::THREADS, 2) gemv_w4_kernel(const W4Args a) {
    using namespace w4;
    using M = W4Type<T>;
    constexpr int PER = SLICE / G;          // groups per slice: 4, 2, 1
    constexpr int STEPS = G / 32;           // steps per group
    extern __shared__ __align__(16) unsigned char smem[];
    const Smem layout(STAGES, a.rows, a.experts);
    float* red = reinterpret_cast<float*>(smem + layout.ring);
    int* first = reinterpret_cast<int*>(red + RED_FLOATS);
    int* last = first + a.experts;
    int* items = last + a.experts;          // [experts + 1]: first item of each expert
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, c = lane & 3;
    const int n_tiles = (a.n + ROWS - 1) / ROWS;
    const int slices = (a.k + SLICE - 1) / SLICE;
    const int groups_row = a.k / G;

    for (int e = threadIdx.x; e < a.experts; e += THREADS) {
        const int lo = a.offsets ? min(max(a.offsets[e], 0), a.rows) : 0;
        first[e] = lo;
        last[e] = a.offsets ? min(max(a.offsets[e + 1], lo), a.rows) : a.rows;
    }
    __syncthreads();
    if (warp == 0) {
        int carry = 0;
        for (int e0 = 0; e0 < a.experts; e0 += 32) {
            const int e = e0 + lane;
            const int n = e < a.experts ? (last[e] - first[e] + w4::COLS - 1) / w4::COLS * n_tiles : 0;
            int incl = n;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, incl, d);
                if (lane >= d) incl += up;
            }
            if (e < a.experts) items[e] = carry + incl - n;
            carry += __shfl_sync(0xffffffffu, incl, 31);
        }
        if (lane == 0) items[a.experts] = carry;
    }
    __syncthreads();
    const int total = items[a.experts];

    unsigned char* ring = smem + warp * STAGES * layout.stage;
    const uint32_t ring_addr = smem_u32(ring);

    // ---- loads: one slice per call, in the order in which they are used ----
    Cursor load;
    load.t = blockIdx.x;
    load.s = warp;
    if (load.t < total) load.decode(a, first, last, items, n_tiles);
    int load_slot = 0;
    auto issue = [&] {
        if (load.t < total && load.s < slices) {
            const uint32_t dst = ring_addr + load_slot * layout.stage;
            const int k0 = load.s * SLICE;
            const int piece = lane & 3;                       // 16 bytes = 32 k
            if (k0 + piece * 32 < a.k) {
                const uint8_t* src = a.q + ((static_cast<size_t>(load.item.e) * a.n + load.item.n0 + g) * a.k + k0) / 2 + piece * 16;
#pragma unroll
                for (int i = 0; i < ROWS / 8; ++i)
                    if (load.item.n0 + g + 8 * i < a.n)
                        cp_async16(dst + w_piece(g + 8 * i, piece), src + static_cast<size_t>(i) * 4 * a.k);
            }
            const int xpiece = lane & 15;                     // 16 bytes = 8 k
            if (k0 + xpiece * 8 < a.k) {
                const T* src = static_cast<const T*>(a.x) + static_cast<size_t>(load.item.r0) * a.ldx + k0 + xpiece * 8;
                for (int r = lane >> 4; r < load.item.cols; r += 2)
                    cp_async16(dst + x_piece(r, xpiece), src + static_cast<size_t>(r) * a.ldx);
            }
            load.s += WARPS;
            if (load.s >= slices) {
                load.s = warp;
                load.t += gridDim.x;
                if (load.t < total) load.decode(a, first, last, items, n_tiles);
            }
        }
        cp_async_commit();
        load_slot = load_slot + 1 == STAGES ? 0 : load_slot + 1;
    };
    for (int i = 0; i < STAGES - 1; ++i) issue();

    // ---- scales and zeros of the next slice, in registers: rows g + 8 h, h = 0..3, PER groups each ----
    Cursor ahead;
    ahead.t = blockIdx.x;
    ahead.s = warp;
    if (ahead.t < total) ahead.decode(a, first, last, items, n_tiles);
    uint16_t sc_next[4][PER];
    uint8_t zr_next[4][PER];
    auto fetch = [&] {
        if (ahead.t < total && ahead.s < slices) {
            const int g0 = ahead.s * PER;
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                const int row = min(ahead.item.n0 + g + 8 * h, a.n - 1);
                const size_t at = (static_cast<size_t>(ahead.item.e) * a.n + row) * groups_row + g0;
                if (PER == 1 || a.aligned) {
                    struct alignas(2 * PER) S { uint16_t v[PER]; };
                    struct alignas(PER) B { uint8_t v[PER]; };
                    const S s = *reinterpret_cast<const S*>(a.scales + at);
#pragma unroll
                    for (int p = 0; p < PER; ++p) sc_next[h][p] = s.v[p];
                    if (Z) {
                        const B z = *reinterpret_cast<const B*>(a.zeros + at);
#pragma unroll
                        for (int p = 0; p < PER; ++p) zr_next[h][p] = z.v[p];
                    }
                } else {
#pragma unroll
                    for (int p = 0; p < PER; ++p) {
                        if (g0 + p < groups_row) {
                            sc_next[h][p] = a.scales[at + p];
                            if (Z) zr_next[h][p] = a.zeros[at + p];
                        }
                    }
                }
            }
            ahead.s += WARPS;
            if (ahead.s >= slices) {
                ahead.s = warp;
                ahead.t += gridDim.x;
                if (ahead.t < total) ahead.decode(a, first, last, items, n_tiles);
            }
        }
    };
    fetch();

    Cursor at;
    int slot = 0;
    for (at.t = blockIdx.x; at.t < total; at.t += gridDim.x) {
        at.decode(a, first, last, items, n_tiles);
        const int cols = at.item.cols;
        float sum[2][4];   // [16 weight rows][C fragment]
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[0][i] = sum[1][i] = 0.f;

        for (int s = warp; s < slices; s += WARPS) {
            cp_async_wait<STAGES - 2>();
            __syncwarp();
            issue();   // into the slot consumed one iteration ago
            float sc[4][PER], zr[4][PER];
#pragma unroll
            for (int h = 0; h < 4; ++h)
#pragma unroll
                for (int p = 0; p < PER; ++p) {
                    sc[h][p] = M::to_f32(sc_next[h][p]);
                    zr[h][p] = Z ? 16.f + static_cast<float>(zr_next[h][p]) : 24.f;
                }
            fetch();
            const unsigned char* here = ring + slot * layout.stage;
            slot = slot + 1 == STAGES ? 0 : slot + 1;
            const int groups_here = min(PER, (a.k - s * SLICE) / G);
#pragma unroll
            for (int p = 0; p < PER; ++p) {
                if (p >= groups_here) break;
                float acc[2][4], ones[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[0][i] = acc[1][i] = ones[i] = 0.f;
#pragma unroll
                for (int st = 0; st < STEPS; ++st) {
                    const int step = p * STEPS + st;
                    uint32_t w[4];
#pragma unroll
                    for (int h = 0; h < 4; ++h)
                        w[h] = *reinterpret_cast<const uint32_t*>(here + w_piece(g + 8 * h, step) + c * 4);
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (g < cols) v = *reinterpret_cast<const uint4*>(here + x_piece(g, step * 4 + c));
                    const uint32_t b0 = __byte_perm(v.x, v.z, 0x5410), b1 = __byte_perm(v.x, v.z, 0x7632);
                    const uint32_t b2 = __byte_perm(v.y, v.w, 0x5410), b3 = __byte_perm(v.y, v.w, 0x7632);
                    M::mma(ones, M::ONES, M::ONES, M::ONES, M::ONES, b0, b1);
                    M::mma(ones, M::ONES, M::ONES, M::ONES, M::ONES, b2, b3);
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
                        const uint32_t lo = w[2 * m], hi = w[2 * m + 1];
                        M::mma(acc[m], M::template pair<0>(lo), M::template pair<0>(hi), M::template pair<1>(lo), M::template pair<1>(hi), b0, b1);
                        M::mma(acc[m], M::template pair<2>(lo), M::template pair<2>(hi), M::template pair<3>(lo), M::template pair<3>(hi), b2, b3);
                    }
                }
                // C fragment: [0], [1] row g, columns 2c, 2c + 1; [2], [3] row g + 8.
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int h = 2 * m + (i >> 1);
                        sum[m][i] = fmaf(sc[h][p], fmaf(-zr[h][p], ones[i & 1], acc[m][i]), sum[m][i]);
                    }
            }
        }

        float* part = red + warp * COLS * RED_PITCH;
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int col = 2 * c + (i & 1);
                if (col < cols) part[col * RED_PITCH + m * 16 + (i >> 1) * 8 + g] = sum[m][i];
            }
        __syncthreads();
        for (int i = threadIdx.x; i < cols * ROWS; i += THREADS) {
            const int col = i / ROWS, row = i % ROWS;
            if (at.item.n0 + row >= a.n) continue;
            const float* p = red + col * RED_PITCH + row;
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) v += p[w * COLS * RED_PITCH];
            static_cast<T*>(a.out)[static_cast<size_t>(at.item.r0 + col) * a.ldo + at.item.n0 + row] = M::from_f32(v);
        }
        __syncthreads();   // the next item's sums go to the same place
    }
    cp_async_wait<0>();
}

template <typename T, int G, bool Z, int STAGES>
int launch_w4(const W4Args& a, long long most_items, cudaStream_t s) {
    auto kern = gemv_w4_kernel<T, G, Z, STAGES>;
    static std::mutex mu;
    static int sm_count[64] = {};
    int dev = 0, sms = 0;
    PRISM_CUDA_TRY(cudaGetDevice(&dev));
    {
        std::lock_guard<std::mutex> lk(mu);
        const bool cacheable = dev >= 0 && dev < 64;
        if (!cacheable || !sm_count[dev]) {
            PRISM_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                w4::Smem(STAGES, w4::COLS, w4::MAX_EXPERTS).bytes));
            PRISM_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
            if (cacheable) sm_count[dev] = sms;
        } else {
            sms = sm_count[dev];
        }
    }
    const long long cap = 2LL * sms;   // resident CTAs, by registers and shared memory
    const int grid = static_cast<int>(most_items < cap ? most_items : cap);
    kern<<<grid, w4::THREADS, w4::Smem(STAGES, a.rows, a.experts).bytes, s>>>(a);
    PRISM_CUDA_TRY(cudaGetLastError());
    count_launch();
    return PRISM_B200_OK;
}

// Stages of a warp's ring: four with up to four rows of x, three with more, so that two CTAs fit an SM.
template <typename T, int G, bool Z>
int launch_w4_stages(const W4Args& a, cudaStream_t s) {
    const long long tiles = (a.n + w4::ROWS - 1) / w4::ROWS;
    const long long groups = a.offsets ? (a.experts < a.rows ? a.experts : a.rows) : 1;
    const long long most = tiles * (a.rows / w4::COLS + groups);
    return a.rows <= 4 ? launch_w4<T, G, Z, 4>(a, most, s) : launch_w4<T, G, Z, 3>(a, most, s);
}

template <typename T, int G>
int launch_w4_zeros(const W4Args& a, cudaStream_t s) {
    return a.zeros ? launch_w4_stages<T, G, true>(a, s) : launch_w4_stages<T, G, false>(a, s);
}

template <typename T>
int launch_w4_group(const W4Args& a, int group, cudaStream_t s) {
    if (group == 32) return launch_w4_zeros<T, 32>(a, s);
    if (group == 64) return launch_w4_zeros<T, 64>(a, s);
    return launch_w4_zeros<T, 128>(a, s);
}

}  // namespace
}  // namespace prism_b200

using namespace prism_b200;

extern "C" int prism_b200_gemv_w4(int dtype, int rows, int experts, int n, int k, int group, const void* x, long long ldx,
                                  const uint8_t* q, const void* scales, const uint8_t* zeros, const int* offsets, void* out,
                                  long long ldo, void* stream) {
    if (rows < 0 || experts < 0 || n < 0 || k < 0) return set_error(PRISM_B200_ERR_INVALID_ARGUMENT, "gemv_w4: negative size");
    if (dtype != PRISM_B200_BF16 && dtype != PRISM_B200_F16)
        return set_error(PRISM_B200_ERR_INVALID_ARGUMENT, "gemv_w4: x, scales and out are bf16 or fp16");
    if (group != 32 && group != 64 && group != 128)
        return set_error(PRISM_B200_ERR_UNSUPPORTED_SHAPE, "gemv_w4: groups of 32, 64 or 128 weights (got %d)", group);
    if (k % group) return set_error(PRISM_B200_ERR_UNSUPPORTED_SHAPE, "gemv_w4: k must be a multiple of the group (got %d, %d)", k, group);
    if (experts > w4::MAX_EXPERTS)
        return set_error(PRISM_B200_ERR_UNSUPPORTED_SHAPE, "gemv_w4: at most %d experts (got %d)", w4::MAX_EXPERTS, experts);
    if (!offsets && experts > 1) return set_error(PRISM_B200_ERR_INVALID_ARGUMENT, "gemv_w4: several matrices need offsets");
    if (rows == 0 || n == 0 || experts == 0) return PRISM_B200_OK;
    if (k == 0) return set_error(PRISM_B200_ERR_UNSUPPORTED_SHAPE, "gemv_w4: nothing to add up (k is 0)");
    if (!x || !q || !scales || !out) return set_error(PRISM_B200_ERR_INVALID_ARGUMENT, "gemv_w4: null pointer");
    if ((n + 31LL) / 32 * (rows + static_cast<long long>(experts)) > 0x3fffffffLL)
        return set_error(PRISM_B200_ERR_TOO_LARGE, "gemv_w4: too many tiles");
    if (ldx < k || ldo < n) return set_error(PRISM_B200_ERR_INVALID_ARGUMENT, "gemv_w4: a row stride below the row's width");
    if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(q)) & 15u || ldx % 8)
        return set_error(PRISM_B200_ERR_MISALIGNED, "gemv_w4: x and q must be 16-byte aligned, x's row stride a multiple of 8");
    if ((reinterpret_cast<uintptr_t>(scales) | reinterpret_cast<uintptr_t>(out)) & 1u)
        return set_error(PRISM_B200_ERR_MISALIGNED, "gemv_w4: scales and out must be 2-byte aligned");
    const int per = 128 / group;
    const bool aligned = k % 128 == 0 && reinterpret_cast<uintptr_t>(scales) % (2 * per) == 0 && reinterpret_cast<uintptr_t>(zeros) % per == 0;
    const W4Args a{x, ldx, q, static_cast<const uint16_t*>(scales), zeros, offsets, out, ldo, rows, experts, n, k, aligned ? 1 : 0};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return dtype == PRISM_B200_BF16 ? launch_w4_group<__nv_bfloat16>(a, group, s) : launch_w4_group<__half>(a, group, s);
}
