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
//   * A warp takes 32 weight rows and a share of k in slices of 128; `split` warps share the same rows, so that long rows
//     are split and short ones are not (four slices per warp where there are enough).  A slice (2 KB of weights, and its
//     256 bytes of each row of x) is two TMA copies into a ring of the warp's own, issued by one lane; the ring runs on
//     across work items, so no block barrier is between a copy and its use.  The copies' 64-byte swizzle keeps a step's
//     reads free of bank conflicts, and what lies outside the matrices arrives as zeros.
//   * The warps' sums meet in shared memory once per item, added in warp order.
// Integer instructions (ALU pipe, half rate) are the next bound: 7 per word of 8 weights, about 40 per 512 bytes in all.
// The first form, with 16-byte cp.async copies by all lanes, spent 72 there and took 20.8 us at 8192 x 8192.
#include "common.cuh"
#include "tcgen05.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace prism_b200 {
namespace {

namespace w4 {
constexpr int WARPS = 16;
constexpr int THREADS = 32 * WARPS;
constexpr int ROWS = 32;                 // weight rows per warp
constexpr int SLICE = 128;               // k per stage
constexpr int COLS = 8;                  // rows of x per item: the columns of one MMA
constexpr int W_BYTES = ROWS * SLICE / 2;
constexpr int X_PITCH = SLICE * 2;
constexpr int RED_PITCH = 36;            // a fragment's 8 x 4 places lie in 32 banks
constexpr int MAX_STAGES = 6;
constexpr int MAX_EXPERTS = 1024;
constexpr int RING_BYTES = 196608;

// Shared memory: rings (512-byte aligned), sums of the warps, barriers, flags, tables.
struct Layout {
    int xrows, stage, stages, red, bars, bytes;
    __host__ __device__ Layout(int rows, int experts) {
        xrows = rows < COLS ? rows : COLS;
        stage = W_BYTES + (xrows * X_PITCH + 511) / 512 * 512;
        stages = RING_BYTES / (WARPS * stage);
        if (stages > MAX_STAGES) stages = MAX_STAGES;
        red = WARPS * stages * stage;
        bars = red + WARPS * xrows * RED_PITCH * 4;
        bytes = 1024 + bars + WARPS * MAX_STAGES * 8 + 16 + (3 * experts + 1) * 4;
    }
};
}  // namespace w4

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
    const uint16_t* scales;
    const uint8_t* zeros;     // null: 8 everywhere
    const int* offsets;       // null: one matrix, all rows
    void* out;
    long long ldo;
    int rows, experts, n, k;
    int split;                // warps that share 32 weight rows along k (a power of two)
    int aligned;              // a slice's scales (zeros) of a row can be read as one vector
};

__device__ __forceinline__ void tma_load_w4(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tma_load_x(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
}

// A warp's place in the sequence of (item, slice) pairs that it works through; moves forward only.  An item is
// 32 * (WARPS / split) weight rows of one expert and up to 8 of its rows of x; the items of one weight tile follow one
// another, so that more than 8 rows find the weights in L2.
struct Cursor {
    int t, s, e = 0;
    int n0, r0, cols;
    __device__ __forceinline__ void decode(const W4Args& a, const int* first, const int* last, const int* items, int warp_row) {
        const int tile_rows = w4::ROWS * (w4::WARPS / a.split);
        int in = t, lo = 0, hi = a.rows;
        if (a.offsets) {
            while (items[e + 1] <= t) ++e;
            in = t - items[e];
            lo = first[e];
            hi = last[e];
        }
        const int chunks = (hi - lo + w4::COLS - 1) / w4::COLS;
        const int tile = chunks == 1 ? in : in / chunks, chunk = in - tile * chunks;
        n0 = tile * tile_rows + warp_row * w4::ROWS;
        r0 = lo + chunk * w4::COLS;
        cols = min(w4::COLS, hi - r0);
    }
};

template <typename T, int G, bool Z>
__global__ void __launch_bounds__(w4::THREADS, 1)
gemv_w4_kernel(const W4Args a, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x) {
    using namespace w4;
    using M = W4Type<T>;
    constexpr int PER = SLICE / G;          // groups per slice: 4, 2, 1
    constexpr int STEPS = G / 32;           // steps per group
    extern __shared__ __align__(16) unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const Layout layout(a.rows, a.experts);
    float* red = reinterpret_cast<float*>(smem + layout.red);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + layout.bars);
    uint32_t* flags = reinterpret_cast<uint32_t*>(bars + WARPS * MAX_STAGES);
    volatile uint32_t* abort_flag = flags;
    volatile uint32_t* never_flag = flags + 1;
    int* first = reinterpret_cast<int*>(flags + 4);
    int* last = first + a.experts;
    int* items = last + a.experts;          // [experts + 1]: first item of each expert
    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int g = lane >> 2, c = lane & 3;
    const int warp_row = warp / a.split, warp_k = warp % a.split;
    const int tile_rows = ROWS * (WARPS / a.split);
    const int n_tiles = (a.n + tile_rows - 1) / tile_rows;
    const int slices = (a.k + SLICE - 1) / SLICE;
    const int groups_row = a.k / G;
    const int stages = layout.stages;

    uint64_t* full = bars + warp * MAX_STAGES;
    if (lane == 0) {
        for (int i = 0; i < stages; ++i) mbar_init(&full[i], 1);
        if (warp == 0) *abort_flag = *never_flag = 0;
        fence_barrier_init();
    }
    int total;
    if (a.offsets) {
        for (int e = threadIdx.x; e < a.experts; e += THREADS) {
            const int lo = min(max(a.offsets[e], 0), a.rows);
            first[e] = lo;
            last[e] = min(max(a.offsets[e + 1], lo), a.rows);
        }
        __syncthreads();
        if (warp == 0) {
            int carry = 0;
            for (int e0 = 0; e0 < a.experts; e0 += 32) {
                const int e = e0 + lane;
                const int n = e < a.experts ? (last[e] - first[e] + COLS - 1) / COLS * n_tiles : 0;
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
        total = items[a.experts];
    } else {
        __syncthreads();
        total = (a.rows + COLS - 1) / COLS * n_tiles;
    }

    unsigned char* ring = smem + warp * stages * layout.stage;
    const uint32_t ring_addr = smem_u32(ring), full_addr = smem_u32(full);
    const uint32_t stage_bytes = W_BYTES + layout.xrows * X_PITCH;

    // ---- copies: one slice per call, in the order in which they are used ----
    Cursor load;
    load.t = blockIdx.x;
    load.s = warp_k;
    if (load.t < total) load.decode(a, first, last, items, warp_row);
    int load_slot = 0, armed = 0;
    auto issue = [&] {
        if (load.t >= total) return;
        if (lane == 0) {
            const uint32_t dst = ring_addr + load_slot * layout.stage, bar = full_addr + load_slot * 8;
            mbar_arrive_expect_tx(&full[load_slot], stage_bytes);
            tma_load_w4(dst, &map_w, load.s * (SLICE / 2), load.n0, load.e, bar);
            tma_load_x(dst + W_BYTES, &map_x, load.s * SLICE, load.r0, bar);
        }
        ++armed;
        load_slot = load_slot + 1 == stages ? 0 : load_slot + 1;
        load.s += a.split;
        if (load.s >= slices) {
            load.s = warp_k;
            load.t += gridDim.x;
            if (load.t < total) load.decode(a, first, last, items, warp_row);
        }
    };
    for (int i = 0; i < stages - 1; ++i) issue();

    // ---- scales and zeros of the next slice, in registers: rows g + 8 h, h = 0..3, PER groups each ----
    Cursor ahead;
    ahead.t = blockIdx.x;
    ahead.s = warp_k;
    const uint16_t* sc_row[4];
    const uint8_t* zr_row[4];
    auto rows_of = [&] {
        ahead.decode(a, first, last, items, warp_row);
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            const size_t at = (static_cast<size_t>(ahead.e) * a.n + min(ahead.n0 + g + 8 * h, a.n - 1)) * groups_row;
            sc_row[h] = a.scales + at;
            if (Z) zr_row[h] = a.zeros + at;
        }
    };
    if (ahead.t < total) rows_of();
    struct alignas(2 * PER) Scales { uint16_t v[PER]; };
    struct alignas(PER) Zeros { uint8_t v[PER]; };
    Scales sc_next[4];
    Zeros zr_next[4];
    auto fetch = [&] {
        if (ahead.t >= total) return;
        const int g0 = ahead.s * PER;
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            if (PER == 1 || a.aligned) {
                sc_next[h] = *reinterpret_cast<const Scales*>(sc_row[h] + g0);
                if (Z) zr_next[h] = *reinterpret_cast<const Zeros*>(zr_row[h] + g0);
            } else {
#pragma unroll
                for (int p = 0; p < PER; ++p) {   // no scale behind the row's last group: its products are zeros
                    const bool there = g0 + p < groups_row;
                    sc_next[h].v[p] = there ? sc_row[h][g0 + p] : 0;
                    if (Z) zr_next[h].v[p] = there ? zr_row[h][g0 + p] : 0;
                }
            }
        }
        ahead.s += a.split;
        if (ahead.s >= slices) {
            ahead.s = warp_k;
            ahead.t += gridDim.x;
            if (ahead.t < total) rows_of();
        }
    };
    fetch();

    Cursor at;
    int slot = 0;
    uint32_t phase = 0;
    bool timed_out = false;
    // Offsets inside a stage that do not change: a lane's words of step 0 in rows g + 8 h (the swizzle of rows 8 apart is
    // the same), and its piece of x.
    const int w_at = g * (SLICE / 2) + c * 4, w_swizzle = ((g >> 1) & 3) << 4;
    const int x_at = W_BYTES + g * X_PITCH + c * 16;
    for (at.t = blockIdx.x; at.t < total; at.t += gridDim.x) {
        at.decode(a, first, last, items, warp_row);
        const int cols = at.cols;
        float sum[2][4];   // [16 weight rows][C fragment]
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[0][i] = sum[1][i] = 0.f;

        for (int s = warp_k; s < slices; s += a.split) {
            if (!timed_out && !__all_sync(0xffffffffu, mbar_wait_bounded(&full[slot], phase, abort_flag))) {
                timed_out = true;   // go on to the block's barriers without waiting for copies again
                *abort_flag = 1;
                if (lane == 0) raise_device_status(DEV_GEMV_PIPE_TIMEOUT);
            }
            __syncwarp();
            if (!timed_out) issue();   // into the slot consumed one iteration ago
            float sc[4][PER], zr[4][PER];
#pragma unroll
            for (int h = 0; h < 4; ++h)
#pragma unroll
                for (int p = 0; p < PER; ++p) {
                    sc[h][p] = M::to_f32(sc_next[h].v[p]);
                    zr[h][p] = Z ? -16.f - static_cast<float>(zr_next[h].v[p]) : -24.f;
                }
            fetch();
            const unsigned char* here = ring + slot * layout.stage;
            if (++slot == stages) {
                slot = 0;
                phase ^= 1u;
            }
#pragma unroll
            for (int p = 0; p < PER; ++p) {
                float acc[2][4], ones[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[0][i] = acc[1][i] = ones[i] = 0.f;
#pragma unroll
                for (int st = 0; st < STEPS; ++st) {
                    const int step = p * STEPS + st;
                    const unsigned char* words = here + w_at + ((step << 4) ^ w_swizzle);
                    uint32_t w[4];
#pragma unroll
                    for (int h = 0; h < 4; ++h) w[h] = *reinterpret_cast<const uint32_t*>(words + 8 * h * (SLICE / 2));
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (g < cols) v = *reinterpret_cast<const uint4*>(here + x_at + step * 64);
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
                        sum[m][i] = fmaf(sc[h][p], fmaf(zr[h][p], ones[i & 1], acc[m][i]), sum[m][i]);
                    }
            }
        }

        float* part = red + warp * layout.xrows * RED_PITCH;
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int col = 2 * c + (i & 1);
                if (col < cols) part[col * RED_PITCH + m * 16 + (i >> 1) * 8 + g] = sum[m][i];
            }
        __syncthreads();
        const int n_first = at.n0 - warp_row * ROWS;
        for (int i = threadIdx.x; i < cols * tile_rows; i += THREADS) {
            const int col = i / tile_rows, row = i - col * tile_rows;
            if (n_first + row >= a.n) continue;
            const float* p = red + ((row / ROWS) * a.split * layout.xrows + col) * RED_PITCH + row % ROWS;
            float v = 0.f;
            for (int w = 0; w < a.split; ++w) v += p[w * layout.xrows * RED_PITCH];
            static_cast<T*>(a.out)[static_cast<size_t>(at.r0 + col) * a.ldo + n_first + row] = M::from_f32(v);
        }
        __syncthreads();   // the next item's sums go to the same place
    }
    if (timed_out && lane == 0) {
        // Unwind: let copies already in flight land before shared memory is released.
        for (int i = 0; i < stages && i < armed; ++i) {
            const int behind = armed - 1 - i;   // the behind-th copy went to slot behind % stages, phase behind / stages
            mbar_wait_bounded(&full[behind % stages], (behind / stages) & 1, never_flag, 2000000ull);
        }
    }
}

// ---- host side ---------------------------------------------------------------------------------------------------

// Weights as bytes [experts][n][k / 2], boxes of 64 bytes x 32 rows; x as rows of 16-bit elements, boxes of 128 x xrows.
int w4_maps(CUtensorMap* map_w, CUtensorMap* map_x, const W4Args& a, const uint8_t* q, const void* x, long long ldx, int xrows) {
    const cuuint64_t wdims[3] = {static_cast<cuuint64_t>(a.k) / 2, static_cast<cuuint64_t>(a.n), static_cast<cuuint64_t>(a.experts)};
    const cuuint64_t wstrides[2] = {static_cast<cuuint64_t>(a.k) / 2, static_cast<cuuint64_t>(a.n) * a.k / 2};
    const cuuint32_t wbox[3] = {w4::SLICE / 2, w4::ROWS, 1};
    if (int rc = encode_tensor_map(map_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, q, wdims, wstrides, wbox, CU_TENSOR_MAP_SWIZZLE_64B)) return rc;
    const cuuint64_t xdims[2] = {static_cast<cuuint64_t>(a.k), static_cast<cuuint64_t>(a.rows)};
    const cuuint64_t xstrides[1] = {static_cast<cuuint64_t>(ldx) * 2};
    const cuuint32_t xbox[2] = {w4::SLICE, static_cast<cuuint32_t>(xrows)};
    return encode_tensor_map(map_x, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, x, xdims, xstrides, xbox, CU_TENSOR_MAP_SWIZZLE_NONE);
}

template <typename T, int G, bool Z>
int launch_w4(W4Args a, const uint8_t* q, const void* x, long long ldx, cudaStream_t s) {
    auto kern = gemv_w4_kernel<T, G, Z>;
    static std::mutex mu;
    static int sm_count[64] = {};
    int dev = 0, sms = 0;
    PRISM_CUDA_TRY(cudaGetDevice(&dev));
    {
        std::lock_guard<std::mutex> lk(mu);
        const bool cacheable = dev >= 0 && dev < 64;
        if (!cacheable || !sm_count[dev]) {
            PRISM_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448));
            PRISM_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
            if (cacheable) sm_count[dev] = sms;
        } else {
            sms = sm_count[dev];
        }
    }
    // Warps per 32 weight rows: as many as leave each four slices of k, more where the rows alone do not fill the SMs.
    const int slices = (a.k + w4::SLICE - 1) / w4::SLICE;
    const long long groups = a.offsets ? (a.experts < a.rows ? a.experts : a.rows) : 1;
    auto most = [&](int split) {
        const int tile_rows = w4::ROWS * (w4::WARPS / split);
        return (a.n + tile_rows - 1LL) / tile_rows * (a.rows / w4::COLS + groups);
    };
    int split = 1;
    while (split < w4::WARPS && slices >= 8 * split) split *= 2;
    while (split < w4::WARPS && slices >= 2 * split && most(split) < sms) split *= 2;
    a.split = split;
    const w4::Layout layout(a.rows, a.experts);
    CUtensorMap map_w, map_x;
    if (int rc = w4_maps(&map_w, &map_x, a, q, x, ldx, layout.xrows)) return rc;
    const int grid = static_cast<int>(most(split) < sms ? most(split) : sms);
    kern<<<grid, w4::THREADS, layout.bytes, s>>>(a, map_w, map_x);
    PRISM_CUDA_TRY(cudaGetLastError());
    count_launch();
    return PRISM_B200_OK;
}

template <typename T, int G>
int launch_w4_zeros(const W4Args& a, const uint8_t* q, const void* x, long long ldx, cudaStream_t s) {
    return a.zeros ? launch_w4<T, G, true>(a, q, x, ldx, s) : launch_w4<T, G, false>(a, q, x, ldx, s);
}

template <typename T>
int launch_w4_group(const W4Args& a, int group, const uint8_t* q, const void* x, long long ldx, cudaStream_t s) {
    if (group == 32) return launch_w4_zeros<T, 32>(a, q, x, ldx, s);
    if (group == 64) return launch_w4_zeros<T, 64>(a, q, x, ldx, s);
    return launch_w4_zeros<T, 128>(a, q, x, ldx, s);
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
    if (int rc = bind_status_word()) return rc;
    const W4Args a{static_cast<const uint16_t*>(scales), zeros, offsets, out, ldo, rows, experts, n, k, 1, aligned ? 1 : 0};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return dtype == PRISM_B200_BF16 ? launch_w4_group<__nv_bfloat16>(a, group, q, x, ldx, s) : launch_w4_group<__half>(a, group, q, x, ldx, s);
}
