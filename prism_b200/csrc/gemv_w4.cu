// Products of a few rows with matrices of 4-bit weights:
//   y[r, n] = sum over groups g of s[n, g] * sum over k in g of (q[n, k] - z[n, g]) * x[r, k]
// with one matrix for all rows or one per expert (rows grouped by offsets, as in grouped_gemm.cu).
//
// What bounds it: the weights, half a byte each, are read once; a row of x adds 2 flop per weight, so for up to about
// eight rows the kernel has to stream.  The hard part is turning nibbles into operands fast enough: an SM has to take
// 23 bytes (46 weights) per clock to keep up with HBM.
//   * Products and sums are mma.sync m16n8k16 with fp32 accumulators: 16 weight rows x 16 k against up to 8 rows of x.
//     tcgen05 would want the converted weights in shared memory, a round trip of four times the bytes read here.
//   * Nibbles become operands where they lie in a byte, two bytes at a time: by one AND or LOP3 and one packed FMA or
//     subtraction that leaves q - z (bf16: times 2^-7), exactly; a word needs one shift.  So the products are exact and
//     only the sums round, in fp32.  (One base for all nibbles takes three shifts and a multiplication, bf16, or one and
//     two, fp16: with slices of 128, 39 us at 16384 x 16384 against 36; shifts as high halves of products 42 to 44; base and
//     z taken off afterwards with sum x from one more MMA no less than 39, and it costs bits.)
//   * A 32-bit word holds 8 consecutive k; the MMA's order of k is free as long as both operands follow it, so the
//     pairs are (k, k + 4) as the masks deliver them, and x is brought into that order by four PRMTs per 8 values.
//   * The four lanes of a quad take one, two or four consecutive words each, 32, 64 or 128 k together: a group, whose sum is
//     then complete in the accumulator when its scale is applied (fp32).  A group of 128 is one 16-byte read per row.
//   * A team of 1 to 16 warps takes 32 weight rows, each warp a range of k in slices of 128 or 256.  A slice (64 or 128
//     bytes of each weight row, four times that of each row of x) is two TMA copies into a ring of the warp's own, issued
//     by one lane; the ring runs on across work items, so no barrier is between a copy and its use.  What lies outside the
//     matrices arrives as zeros.  The copies' swizzle and the order of the fragments' rows keep the reads free of bank
//     conflicts.  Scales and zero points come in blocks of eight groups (16 and 8 bytes per row, cp.async) one block ahead.
//   * The team's sums meet in shared memory once per item, added in warp order.
// Where the time goes: 16384 x 16384, one row, takes 32.5 us; the copies alone take 25.  On the SMs at work the schedulers
// issue in 69% of the cycles and the ALU pipe is 64% busy; the tensor pipe, an mma.sync taking it 8 cycles per scheduler,
// is at 33%.  512 tiles in teams of four warps use 128 of the 148 SMs: 18944 rows, which use all, take 33.2 us (4.8 TB/s).
#include "common.cuh"
#include "tcgen05.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace prism_b200 {
namespace {

namespace w4 {
constexpr int WARPS = 16;
constexpr int ROWS = 32;                 // weight rows per item
constexpr int THREADS = 32 * WARPS;
constexpr int COLS = 8;                  // rows of x per item: the columns of one MMA
constexpr int RED_PITCH = ROWS + 4;      // a fragment's 8 x 4 places lie in 32 banks
constexpr int BLOCK = 8;                 // groups whose scales are copied at a time
constexpr int SC_BYTES = ROWS * BLOCK * 3;   // a block: 16 bytes of scales per row, then 8 bytes of zero points per row
constexpr int MAX_EXPERTS = 1024;
constexpr int SMEM_BYTES = 232448;

// SLICE: k per stage.  256 halves what a slice costs besides its products; where one or two rows of x leave room for two
// such stages per warp and k is long (launch_w4), 16384 x 16384 takes 33.4 us against 36.2, groups of 32 42.9 against 46.7.
template <int SLICE>
struct Cut {
    static constexpr int X_PITCH = SLICE * 2;
    static constexpr int W_BYTES = ROWS * SLICE / 2;
    static constexpr int ALIGN = SLICE == 128 ? 512 : 1024;   // of a stage: the swizzle's period
    static constexpr int MAX_STAGES = SLICE == 128 ? 3 : 2;   // more only crowd the memory: copies alone of 16384 x 16384 take
                                                              // 25 us with three of 128, 37 with six
};

// Shared memory: rings, scales (two blocks per warp), sums of the warps (two sets), barriers, flags, tables.
template <int SLICE>
struct Layout {
    int xrows, stage, stages, red_floats, scales, red, bars, bytes;
    __host__ __device__ constexpr Layout(int rows, int experts)
        : xrows(0), stage(0), stages(0), red_floats(0), scales(0), red(0), bars(0), bytes(0) {
        xrows = rows < COLS ? rows : COLS;
        using C = Cut<SLICE>;
        stage = C::W_BYTES + (xrows * C::X_PITCH + C::ALIGN - 1) / C::ALIGN * C::ALIGN;
        red_floats = xrows * RED_PITCH;
        const int rest = 1024 + WARPS * (2 * SC_BYTES + 2 * red_floats * 4 + C::MAX_STAGES * 8) + 16 + (experts > 1 ? (3 * experts + 1) * 4 : 16);
        stages = (SMEM_BYTES - rest) / (WARPS * stage);
        if (stages > C::MAX_STAGES) stages = C::MAX_STAGES;
        scales = WARPS * stages * stage;
        red = scales + WARPS * 2 * SC_BYTES;
        bars = red + WARPS * 2 * red_floats * 4;
        bytes = rest + scales;
    }
};
static_assert(Layout<128>(COLS, MAX_EXPERTS).stages >= 2 && Layout<256>(2, MAX_EXPERTS).stages >= 2,
              "a copy is in flight while a slice is used, at the largest sizes too");
}  // namespace w4

// (a & b) | c in one instruction.
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}

template <typename T> struct W4Type;
template <> struct W4Type<__nv_bfloat16> {
    static constexpr float UNIT = 128.f;   // operands are (q - z) / 128
    // An integer in the lowest eight bits of a bf16 is itself times 2^-133, through the subnormals and the first normal
    // numbers; so both nibbles of a byte serve where they lie, and one FMA scales them and takes z off, exactly.
    // (Products with subnormal x stay exact too: 2^-133 / 128 is 2^-140, and fp32 goes down to 2^-149.)
    template <int ODD> static __device__ __forceinline__ uint32_t zero(uint32_t z) { return ODD ? 0u : fma(z * 0x10001u, 0xFE80FE80u, 0u); }
    template <int I> static __device__ __forceinline__ uint32_t operand(uint32_t w, uint32_t even, uint32_t odd) {
        const uint32_t s = I < 2 ? w : w >> 8;
        return I & 1 ? fma(s & 0x00F000F0u, 0x7C807C80u, even) : fma(s & 0x000F000Fu, 0x7E807E80u, even);   // 2^122, 2^126
    }
    static __device__ __forceinline__ uint32_t fma(uint32_t a, uint32_t b, uint32_t c) {
        uint32_t d;
        asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
        return d;
    }
    // d = a * b + d, or a * b where FIRST (no registers to clear before a group's first step)
    template <bool FIRST>
    static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
        if constexpr (FIRST) {
            asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                         : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                         : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
        } else {
            asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                         : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                         : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
        }
    }
    static __device__ __forceinline__ float to_f32(uint16_t v) { return __uint_as_float(static_cast<uint32_t>(v) << 16); }
    static __device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }
};
template <> struct W4Type<__half> {
    static constexpr float UNIT = 1.f;
    // 1024.0 is 0x6400 and counts bits 0-3 of its mantissa in ones, 64.0 is 0x5400 and counts bits 4-7: both nibbles of a
    // byte become 1024 + q or 64 + q where they lie, and 1024 + z or 64 + z is taken off.
    template <int ODD> static __device__ __forceinline__ uint32_t zero(uint32_t z) {
        return ODD ? (z << 4) * 0x10001u | 0x54005400u : z * 0x10001u | 0x64006400u;
    }
    template <int I> static __device__ __forceinline__ uint32_t operand(uint32_t w, uint32_t even, uint32_t odd) {
        const uint32_t s = I < 2 ? w : w >> 8;
        return I & 1 ? sub(and_or(s, 0x00F000F0u, 0x54005400u), odd) : sub(and_or(s, 0x000F000Fu, 0x64006400u), even);
    }
    static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
        const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
        return *reinterpret_cast<const uint32_t*>(&d);
    }
    // d = a * b + d, or a * b where FIRST (no registers to clear before a group's first step)
    template <bool FIRST>
    static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
        if constexpr (FIRST) {
            asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                         : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                         : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
        } else {
            asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                         : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                         : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
        }
    }
    static __device__ __forceinline__ float to_f32(uint16_t v) { return __half2float(__ushort_as_half(v)); }
    static __device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }
};

// cp.async of 16 bytes past L1, of 8 bytes, and the wait for all of a thread's copies.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async8(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

struct W4Args {
    const uint16_t* scales;
    const uint8_t* zeros;     // null: 8 everywhere
    const int* offsets;       // null: one matrix, all rows
    void* out;
    long long ldo;
    int rows, experts, n, k;
    int split;                // warps of a team (a power of two)
    int aligned;              // blocks of eight scales (zeros) can be copied as 16 (8) bytes
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

// An item: 32 weight rows of one expert and up to 8 of its rows of x.  The items of one weight tile follow one another, so
// that more than 8 rows find the weights in L2.  The walk over the experts only moves forward.
struct Item {
    int t, e = 0;
    int n0, r0, cols;
    __device__ __forceinline__ void decode(const W4Args& a, const int* first, const int* last, const int* items) {
        int in = t, lo = 0, hi = a.rows;
        if (a.offsets) {
            while (items[e + 1] <= t) ++e;
            in = t - items[e];
            lo = first[e];
            hi = last[e];
        }
        const int chunks = (hi - lo + w4::COLS - 1) / w4::COLS;
        const int tile = chunks == 1 ? in : in / chunks, chunk = in - tile * chunks;
        n0 = tile * w4::ROWS;
        r0 = lo + chunk * w4::COLS;
        cols = min(w4::COLS, hi - r0);
    }
};

// The weight row (of eight) that takes place g of the MMA's fragments: the order in which lanes that read together find
// their pieces in different banks.  A slice's rows lie 64 or 128 bytes apart, 16-byte pieces XORed by the row.
template <int SLICE, int G>
__device__ __forceinline__ int fragment_row(int g) {
    if (SLICE == 256 && G == 128) return g >> 1 | (g & 1) << 2;
    if (SLICE == 256 && G == 64) return (g & 3) << 1 | g >> 2;
    if (SLICE == 128 && G == 64) return (g & 1) | (g & 2) << 1 | (g & 4) >> 1;
    return g;
}

// Barrier of the warps of team `team` (named barrier team + 1).
__device__ __forceinline__ void team_sync(int team, int threads) {
    __syncwarp();
    if (threads > 32) asm volatile("barrier.cta.sync.aligned %0, %1;" ::"r"(team + 1), "r"(threads) : "memory");
}

template <typename T, int G, bool Z, int SLICE>
__global__ void __launch_bounds__(w4::THREADS, 1)
gemv_w4_kernel(const W4Args a, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x) {
    using namespace w4;
    using M = W4Type<T>;
    constexpr int X_PITCH = Cut<SLICE>::X_PITCH, W_BYTES = Cut<SLICE>::W_BYTES, MAX_STAGES = Cut<SLICE>::MAX_STAGES;
    constexpr int PER = SLICE / G;          // groups per slice
    constexpr int STEPS = G / 32;           // steps per group, and consecutive words per lane
    constexpr int RUN = BLOCK / PER;        // slices per block of scales
    extern __shared__ __align__(16) unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const Layout<SLICE> layout(a.rows, a.experts);
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
    const int team = warp / a.split, warp_k = warp % a.split, teams = WARPS / a.split, team_threads = 32 * a.split;
    const int n_tiles = (a.n + ROWS - 1) / ROWS;
    const int slices = (a.k + SLICE - 1) / SLICE;
    const int per_warp = (slices + a.split - 1) / a.split;
    const int s_first = warp_k * per_warp, s_last = min(slices, s_first + per_warp);   // may be empty
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
    const int t_first = blockIdx.x * teams + team, t_step = gridDim.x * teams;
    const int t_end = s_first < s_last ? total : 0;   // for the copies: a warp without slices has none

    unsigned char* ring = smem + warp * stages * layout.stage;
    const uint32_t ring_addr = smem_u32(ring), full_addr = smem_u32(full);
    const uint32_t stage_bytes = W_BYTES + layout.xrows * X_PITCH;

    // ---- copies: one slice per call, in the order in which they are used ----
    Item load;
    load.t = t_first;
    int load_s = s_first;
    if (load.t < t_end) load.decode(a, first, last, items);
    int load_slot = 0, armed = 0;
    auto issue = [&] {
        if (load.t >= t_end) return;
        if (lane == 0) {
            const uint32_t dst = ring_addr + load_slot * layout.stage, bar = full_addr + load_slot * 8;
            mbar_arrive_expect_tx(&full[load_slot], stage_bytes);
            tma_load_w4(dst, &map_w, load_s * (SLICE / 2), load.n0, load.e, bar);
            tma_load_x(dst + W_BYTES, &map_x, load_s * SLICE, load.r0, bar);
        }
        ++armed;
        load_slot = load_slot + 1 == stages ? 0 : load_slot + 1;
        if (++load_s == s_last) {
            load_s = s_first;
            load.t += t_step;
            if (load.t < t_end) load.decode(a, first, last, items);
        }
    };
    for (int i = 0; i < stages - 1; ++i) issue();

    // ---- scales and zeros, a block of eight groups per call: lane l copies row l ----
    unsigned char* blocks = smem + layout.scales + warp * 2 * SC_BYTES;
    const uint32_t blocks_addr = smem_u32(blocks);
    Item ahead;
    ahead.t = t_first;
    int ahead_s = s_first;      // first slice of the block to be copied
    int copies = 0;
    if (ahead.t < t_end) ahead.decode(a, first, last, items);
    auto copy_scales = [&] {
        if (ahead.t >= t_end) return;
        const int g0 = ahead_s * PER / BLOCK * BLOCK;
        const size_t at = (static_cast<size_t>(ahead.e) * a.n + min(ahead.n0 + lane, a.n - 1)) * groups_row + g0;
        const int into = (copies & 1) * SC_BYTES;
        if (a.aligned) {
            cp_async16(blocks_addr + into + lane * 16, a.scales + at);
            if (Z) cp_async8(blocks_addr + into + ROWS * 16 + lane * 8, a.zeros + at);
        } else {
            uint16_t* sc = reinterpret_cast<uint16_t*>(blocks + into) + lane * BLOCK;
            uint8_t* zr = blocks + into + ROWS * 16 + lane * BLOCK;
            for (int i = 0; i < BLOCK; ++i) {   // no scale behind the row's last group: its products are zeros
                const bool there = g0 + i < groups_row;
                sc[i] = there ? a.scales[at + i] : 0;
                if (Z) zr[i] = there ? a.zeros[at + i] : 0;
            }
        }
        ++copies;
        ahead_s = (ahead_s / RUN + 1) * RUN;
        if (ahead_s >= s_last) {
            ahead_s = s_first;
            ahead.t += t_step;
            if (ahead.t < t_end) ahead.decode(a, first, last, items);
        }
    };
    copy_scales();

    Item at;
    int slot = 0, set = 0, block = 0;
    uint32_t phase = 0;
    bool timed_out = false;
    // Where a lane reads in a stage: its words of row wr (rows 8 apart have the same swizzle), its pieces of x.
    const int wr = fragment_row<SLICE, G>(g);
    const int w_row = wr * (SLICE / 2), w_swizzle = SLICE == 128 ? (wr >> 1) & 3 : wr;   // of 64 or 128 bytes
    const int x_row = W_BYTES + min(g, layout.xrows - 1) * X_PITCH;   // columns without a row of x repeat one; they are not stored
    for (at.t = t_first; at.t < total; at.t += t_step) {
        at.decode(a, first, last, items);
        const int cols = at.cols;
        float sum[2][4];   // [16 weight rows][C fragment]
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[0][i] = sum[1][i] = 0.f;

        for (int s = s_first; s < s_last;) {
            // A block of scales: the copy made one block ago has landed, the next one starts.
            cp_async_wait_all();
            __syncwarp();
            const unsigned char* sc_block = blocks + (block & 1) * SC_BYTES;
            ++block;
            copy_scales();
            const int run_last = min(s_last, (s / RUN + 1) * RUN);
            for (; s < run_last; ++s) {
                if (!timed_out && !__all_sync(0xffffffffu, mbar_wait_bounded(&full[slot], phase, abort_flag))) {
                    timed_out = true;   // go on to the team's barriers without waiting for copies again
                    *abort_flag = 1;
                    if (lane == 0) raise_device_status(DEV_GEMV_PIPE_TIMEOUT);
                }
                __syncwarp();
                if (!timed_out) issue();   // into the slot consumed one iteration ago
                const unsigned char* here = ring + slot * layout.stage;
                if (++slot == stages) {
                    slot = 0;
                    phase ^= 1u;
                }
                const unsigned char* sc_slice = sc_block + wr * 16 + (s % RUN) * (PER * 2);
                const unsigned char* zr_slice = sc_block + ROWS * 16 + wr * 8 + (s % RUN) * PER;
#pragma unroll
                for (int p = 0; p < PER; ++p) {
                    // A lane's STEPS consecutive words in rows wr, wr + 8, wr + 16, wr + 24.
                    struct alignas(4 * STEPS) Words { uint32_t v[STEPS]; };
                    Words w[4];
                    const int byte = p * (G / 2) + c * (4 * STEPS);   // in the row's 64
                    const unsigned char* words = here + w_row + ((((byte >> 4) ^ w_swizzle) << 4) | (byte & 15));
#pragma unroll
                    for (int h = 0; h < 4; ++h) w[h] = *reinterpret_cast<const Words*>(words + 8 * h * (SLICE / 2));
                    float acc[2][4];
                    uint32_t even[4], odd[4];   // base + z of the four rows
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
                        const uint32_t z = Z ? zr_slice[h * 8 * 8 + p] : 8u;
                        even[h] = M::template zero<0>(z);
                        odd[h] = M::template zero<1>(z);
                    }
#pragma unroll
                    for (int st = 0; st < STEPS; ++st) {
                        const uint4 v = *reinterpret_cast<const uint4*>(here + x_row + (p * G + (c * STEPS + st) * 8) * 2);
                        const uint32_t b0 = __byte_perm(v.x, v.z, 0x5410), b1 = __byte_perm(v.x, v.z, 0x7632);
                        const uint32_t b2 = __byte_perm(v.y, v.w, 0x5410), b3 = __byte_perm(v.y, v.w, 0x7632);
#pragma unroll
                        for (int m = 0; m < 2; ++m) {
                            const uint32_t lo = w[2 * m].v[st], hi = w[2 * m + 1].v[st];
                            const uint32_t el = even[2 * m], eh = even[2 * m + 1], ol = odd[2 * m], oh = odd[2 * m + 1];
                            const uint32_t a0 = M::template operand<0>(lo, el, ol), a1 = M::template operand<0>(hi, eh, oh);
                            const uint32_t a2 = M::template operand<1>(lo, el, ol), a3 = M::template operand<1>(hi, eh, oh);
                            if (st == 0) M::template mma<true>(acc[m], a0, a1, a2, a3, b0, b1);
                            else M::template mma<false>(acc[m], a0, a1, a2, a3, b0, b1);
                            M::template mma<false>(acc[m], M::template operand<2>(lo, el, ol), M::template operand<2>(hi, eh, oh),
                                                   M::template operand<3>(lo, el, ol), M::template operand<3>(hi, eh, oh), b2, b3);
                        }
                    }
                    // C fragment: [0], [1] row wr, columns 2c, 2c + 1; [2], [3] row wr + 8.
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
                        const float sc = M::to_f32(*reinterpret_cast<const uint16_t*>(sc_slice + h * 8 * 16 + p * 2));
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            float& to = sum[h >> 1][2 * (h & 1) + i];
                            to = fmaf(sc, acc[h >> 1][2 * (h & 1) + i], to);
                        }
                    }
                }
            }
        }

        // Two sets of sums: the next item's go to the other one, so one barrier per item is enough.
        float* sums = red + (set * WARPS + team * a.split) * layout.red_floats;
        set ^= 1;
        float* part = sums + warp_k * layout.red_floats;
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int col = 2 * c + (i & 1);
                if (col < cols) part[col * RED_PITCH + m * 16 + (i >> 1) * 8 + wr] = sum[m][i];
            }
        team_sync(team, team_threads);
        for (int i = warp_k * 32 + lane; i < cols * ROWS; i += team_threads) {
            const int col = i / ROWS, row = i % ROWS;
            if (at.n0 + row >= a.n) continue;
            const float* p = sums + col * RED_PITCH + row;
            float v = 0.f;
            for (int w = 0; w < a.split; ++w) v += p[w * layout.red_floats];
            static_cast<T*>(a.out)[static_cast<size_t>(at.r0 + col) * a.ldo + at.n0 + row] = M::from_f32(v * M::UNIT);
        }
    }
    cp_async_wait_all();
    if (timed_out && lane == 0) {
        // Unwind: let copies already in flight land before shared memory is released.
        for (int i = 0; i < stages && i < armed; ++i) {
            const int behind = armed - 1 - i;   // copy number `behind` went to slot behind % stages in phase behind / stages
            mbar_wait_bounded(&full[behind % stages], (behind / stages) & 1, never_flag, 2000000ull);
        }
    }
}

// ---- host side ---------------------------------------------------------------------------------------------------

// Weights as bytes [experts][n][k / 2], boxes of a slice of 32 rows; x as rows of 16-bit elements, boxes of a slice of xrows.
int w4_maps(CUtensorMap* map_w, CUtensorMap* map_x, const W4Args& a, const uint8_t* q, const void* x, long long ldx, int xrows, int slice) {
    const cuuint64_t wdims[3] = {static_cast<cuuint64_t>(a.k) / 2, static_cast<cuuint64_t>(a.n), static_cast<cuuint64_t>(a.experts)};
    const cuuint64_t wstrides[2] = {static_cast<cuuint64_t>(a.k) / 2, static_cast<cuuint64_t>(a.n) * a.k / 2};
    const cuuint32_t wbox[3] = {static_cast<cuuint32_t>(slice) / 2, w4::ROWS, 1};
    if (int rc = encode_tensor_map(map_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, q, wdims, wstrides, wbox,
                                    slice == 128 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
    const cuuint64_t xdims[2] = {static_cast<cuuint64_t>(a.k), static_cast<cuuint64_t>(a.rows)};
    const cuuint64_t xstrides[1] = {static_cast<cuuint64_t>(ldx) * 2};
    const cuuint32_t xbox[2] = {static_cast<cuuint32_t>(slice), static_cast<cuuint32_t>(xrows)};
    return encode_tensor_map(map_x, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, x, xdims, xstrides, xbox, CU_TENSOR_MAP_SWIZZLE_NONE);
}

// Items of a call at most: every group may end in an item of its own.
long long most_items(const W4Args& a) {
    const long long tiles = (a.n + w4::ROWS - 1LL) / w4::ROWS;
    if (!a.offsets) return tiles * ((a.rows + w4::COLS - 1) / w4::COLS);
    return tiles * (a.rows / w4::COLS + (a.experts < a.rows ? a.experts : a.rows));
}

// Warps per team: the fewest rounds of (slices per warp + the item's own cost, about one slice) over all teams.
int w4_split(const W4Args& a, int sms, int slice) {
    const int slices = (a.k + slice - 1) / slice;
    long long least = 0;
    int best = 1;
    for (int split = 1; split <= w4::WARPS && (split == 1 || split <= slices); split *= 2) {
        const long long teams = static_cast<long long>(sms) * (w4::WARPS / split);
        const long long cost = (most_items(a) + teams - 1) / teams * ((slices + split - 1) / split + 1);
        if (least == 0 || cost < least) {
            least = cost;
            best = split;
        }
    }
    return best;
}

template <typename T, int G, bool Z, int SLICE>
int launch_w4(W4Args a, const uint8_t* q, const void* x, long long ldx, cudaStream_t s) {
    auto kern = gemv_w4_kernel<T, G, Z, SLICE>;
    static std::mutex mu;
    static int sm_count[64] = {};
    int dev = 0, sms = 0;
    PRISM_CUDA_TRY(cudaGetDevice(&dev));
    {
        std::lock_guard<std::mutex> lk(mu);
        const bool cacheable = dev >= 0 && dev < 64;
        if (!cacheable || !sm_count[dev]) {
            PRISM_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, w4::SMEM_BYTES));
            PRISM_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
            if (cacheable) sm_count[dev] = sms;
        } else {
            sms = sm_count[dev];
        }
    }
    a.split = w4_split(a, sms, SLICE);
    const w4::Layout<SLICE> layout(a.rows, a.experts);
    CUtensorMap map_w, map_x;
    if (int rc = w4_maps(&map_w, &map_x, a, q, x, ldx, layout.xrows, SLICE)) return rc;
    const int teams = w4::WARPS / a.split;
    const long long blocks = (most_items(a) + teams - 1) / teams;
    kern<<<static_cast<int>(blocks < sms ? blocks : sms), w4::THREADS, layout.bytes, s>>>(a, map_w, map_x);
    PRISM_CUDA_TRY(cudaGetLastError());
    count_launch();
    return PRISM_B200_OK;
}

template <typename T, int G, bool Z>
int launch_w4_slice(const W4Args& a, const uint8_t* q, const void* x, long long ldx, cudaStream_t s) {
    // Below 4096 the longer slices are too few to go round (2048 x 1024: 4.8 us against 4.2; 4096 x 4096: 5.2 against 5.3).
    return a.rows <= 2 && a.k >= 4096 ? launch_w4<T, G, Z, 256>(a, q, x, ldx, s) : launch_w4<T, G, Z, 128>(a, q, x, ldx, s);
}

template <typename T, int G>
int launch_w4_zeros(const W4Args& a, const uint8_t* q, const void* x, long long ldx, cudaStream_t s) {
    return a.zeros ? launch_w4_slice<T, G, true>(a, q, x, ldx, s) : launch_w4_slice<T, G, false>(a, q, x, ldx, s);
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
    if (rows > 1 << 30 || n > 1 << 30 || k > 1 << 30 || (n + 31LL) / 32 * (rows + static_cast<long long>(experts)) > 0x3fffffffLL)
        return set_error(PRISM_B200_ERR_TOO_LARGE, "gemv_w4: a size above 2^30 or too many tiles");
    if (ldx < k || ldo < n) return set_error(PRISM_B200_ERR_INVALID_ARGUMENT, "gemv_w4: a row stride below the row's width");
    if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(q)) & 15u || ldx % 8)
        return set_error(PRISM_B200_ERR_MISALIGNED, "gemv_w4: x and q must be 16-byte aligned, x's row stride a multiple of 8");
    if ((reinterpret_cast<uintptr_t>(scales) | reinterpret_cast<uintptr_t>(out)) & 1u)
        return set_error(PRISM_B200_ERR_MISALIGNED, "gemv_w4: scales and out must be 2-byte aligned");
    if (rows_overlap(out, rows, n, ldo, x, rows, k, ldx, 2))
        return set_error(PRISM_B200_ERR_INVALID_ARGUMENT, "gemv_w4: out overlaps x");
    const bool aligned = k / group % w4::BLOCK == 0 && reinterpret_cast<uintptr_t>(scales) % 16 == 0 && reinterpret_cast<uintptr_t>(zeros) % 8 == 0;
    if (int rc = bind_status_word()) return rc;
    const W4Args a{static_cast<const uint16_t*>(scales), zeros, offsets, out, ldo, rows, experts, n, k, 1, aligned ? 1 : 0};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return dtype == PRISM_B200_BF16 ? launch_w4_group<__nv_bfloat16>(a, group, q, x, ldx, s) : launch_w4_group<__half>(a, group, q, x, ldx, s);
}
