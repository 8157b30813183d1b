// bf16 matrix products grouped by expert, with group borders on the device: expert e owns the rows
// offsets[e] <= r < offsets[e + 1] of the activations.
//
//   fwd    out[r, n] = sum_k x[r, k] * W[e][n, k]        (a row of out per row of x)
//   dgrad  dx[r, k]  = sum_n dy[r, n] * W[e][n, k]       (the gradient of the rows)
//   wgrad  dW[e][n, k] = sum over the expert's rows of dy[r, n] * x[r, k]
//
// One kernel in three modes on tcgen05.mma with fp32 accumulators in tensor memory:
//   * The weights' dimension (n, k, n) indexes the 128 tensor-memory lanes of a tile.  In fwd and dgrad the rows index
//     its columns, so a tile of few rows is an MMA of few columns (a multiple of 16, chosen per tile): a group costs
//     what its rows cost, rounded up to 16, and a group of one row still streams its matrix at full width.
//   * Operands lie in shared memory as TMA writes them, in 128-byte swizzle spans: K-major where the contraction is
//     contiguous in memory (x, W in fwd; dy in dgrad), MN-major where the other dimension is (W in dgrad, both in
//     wgrad); the MMA takes either, so nothing is transposed.
//   * fwd and dgrad read past a group's last row into the next group's: those columns are computed and not stored.
//     wgrad contracts over rows, so there the rows behind the group's last are overwritten with zeros in shared memory
//     before the tile's last MMAs (both operands: a NaN there must not meet a zero).
//   * Warp 0 loads, warp 1 issues the MMAs, warps 2-5 store; two accumulators alternate.  Every wait is bounded as in
//     gemm_bf16.cu.  Tiles are dealt round-robin to persistent CTAs; every CTA works out the groups' tiles from the
//     offsets by itself (no launch before this one, no host copy of the offsets).
// Offsets are read with care: each border is clamped to the rows that exist and to the border before it, so a wrong
// array gives wrong products but no access outside the matrices.
#include "common.cuh"
#include "tcgen05.cuh"

#include <mutex>

namespace prism_b200 {
namespace {

namespace gg {
constexpr int FWD = 0, DGRAD = 1, WGRAD = 2;
constexpr int BLOCK_P = 128;       // lanes: n (fwd, wgrad) or k (dgrad)
constexpr int BLOCK_C = 64;        // contraction per stage: one 128-byte span, or 64 rows of it
constexpr int UMMA_K = 16;
constexpr int THREADS = 192;
constexpr int EPI_WARPS = 4;
constexpr int TMEM_COLS = 512;
constexpr int MAX_EXPERTS = 1024;
constexpr int GROUP_Q = 8;         // row tiles walked for each lane tile (L2 reuse), as in gemm_bf16.cu
constexpr uint32_t CHUNK_BYTES = 64 * 64 * 2;   // one 64 x 64 box

template <int BQ>
struct Cfg {
    static constexpr int STAGES = BQ == 256 ? 4 : BQ == 128 ? 6 : 8;
    static constexpr uint32_t P_BYTES = BLOCK_P * BLOCK_C * 2;
    static constexpr uint32_t Q_BYTES = BQ * BLOCK_C * 2;
    static constexpr uint32_t STAGE_BYTES = P_BYTES + Q_BYTES;
    static constexpr uint32_t BAR_BYTES = 256;
    static constexpr uint32_t EPI_WARP_BYTES = 4096;
    static constexpr uint32_t TABLE_BYTES = (3 * MAX_EXPERTS + 4) * 4;
    static constexpr size_t SMEM_BYTES =
        1024 + static_cast<size_t>(STAGES) * STAGE_BYTES + EPI_WARPS * EPI_WARP_BYTES + BAR_BYTES + TABLE_BYTES;
    static_assert(SMEM_BYTES <= 232448, "shared memory of one CTA");
};

// kind::f16, D fp32, A and B bf16; bits 15 / 16: A / B is MN-major.
__host__ __device__ constexpr uint32_t instr_desc(bool a_mn, bool b_mn, int m, int n) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) |
           (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
}  // namespace gg

// MN-major operand, 128-byte swizzle: 64 elements contiguous, the next contraction index 128 bytes on (8 of them make a
// 1024-byte swizzle atom: stride byte offset), the next 64 elements one 64 x 64 box on (leading byte offset).
__device__ __forceinline__ uint64_t smem_desc_mn_sw128(uint32_t smem_addr) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
    d |= static_cast<uint64_t>(gg::CHUNK_BYTES >> 4) << 16;
    d |= static_cast<uint64_t>(1024 >> 4) << 32;
    d |= static_cast<uint64_t>(1) << 46;
    d |= static_cast<uint64_t>(2) << 61;
    return d;
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}

struct GroupedArgs {
    const int* offsets;
    int experts;
    int rows;         // rows of the activations
    int p_dim;        // extent of the lane dimension
    int q_dim;        // wgrad: extent of the column dimension (k)
    int c_dim;        // fwd, dgrad: extent of the contraction
    void* out;
    long long ldo;    // fwd, dgrad: row stride of out; wgrad: q_dim
};

struct Tile {
    int e, p0, q0;    // expert, first lane index, first row (fwd, dgrad) or column (wgrad)
    int cols;         // rows (columns) of the tile that exist
    int first, blocks, tail;   // wgrad: first row; contraction blocks; rows of the last block (0: all 64)
};

// Walks a CTA's tiles in order; the cursor over the experts only moves forward.
template <int MODE, int BQ>
struct TileWalk {
    const int *row_first, *row_last, *tile_first;
    int p_tiles, q_tiles, e = 0;
    __device__ __forceinline__ TileWalk(const GroupedArgs& a, const int* table)
        : row_first(table), row_last(table + gg::MAX_EXPERTS), tile_first(table + 2 * gg::MAX_EXPERTS),
          p_tiles((a.p_dim + gg::BLOCK_P - 1) / gg::BLOCK_P), q_tiles(MODE == gg::WGRAD ? (a.q_dim + BQ - 1) / BQ : 0) {}
    __device__ __forceinline__ Tile at(int t, const GroupedArgs& a) {
        Tile r;
        int in, qt;
        if (MODE == gg::WGRAD) {
            const int per = p_tiles * q_tiles;
            r.e = t / per;
            in = t - r.e * per;
            qt = q_tiles;
        } else {
            while (tile_first[e + 1] <= t) ++e;   // t < tile_first[experts]
            r.e = e;
            in = t - tile_first[e];
            qt = (row_last[e] - row_first[e] + BQ - 1) / BQ;
        }
        const int per_band = gg::GROUP_Q * p_tiles;
        const int band = in / per_band, q_first = band * gg::GROUP_Q;
        const int in_band = in - band * per_band, height = min(gg::GROUP_Q, qt - q_first);
        const int q = q_first + in_band % height;
        r.p0 = (in_band / height) * gg::BLOCK_P;
        if (MODE == gg::WGRAD) {
            r.q0 = q * BQ;
            r.cols = min(BQ, a.q_dim - r.q0);
            r.first = row_first[r.e];
            const int rows = row_last[r.e] - r.first;
            r.blocks = (rows + gg::BLOCK_C - 1) / gg::BLOCK_C;
            r.tail = rows % gg::BLOCK_C;
        } else {
            r.q0 = row_first[e] + q * BQ;
            r.cols = min(BQ, row_last[e] - r.q0);
            r.first = 0;
            r.blocks = (a.c_dim + gg::BLOCK_C - 1) / gg::BLOCK_C;
            r.tail = 0;
        }
        return r;
    }
};

// Zeros the contraction rows [tail, next multiple of 16) of `boxes` MN-major 64 x 64 boxes: row c of a box is its 128
// bytes at c * 128 (the swizzle permutes 16-byte pieces within a row only).  One warp.
__device__ __forceinline__ void zero_tail_rows(unsigned char* stage, int boxes, int tail, int lane) {
    const int end = (tail + gg::UMMA_K - 1) / gg::UMMA_K * gg::UMMA_K;
    const int per_box = (end - tail) * 8;   // 16-byte pieces
    for (int i = lane; i < boxes * per_box; i += 32) {
        const int box = i / per_box, piece = i - box * per_box;
        *reinterpret_cast<uint4*>(stage + box * gg::CHUNK_BYTES + tail * 128 + piece * 16) = make_uint4(0, 0, 0, 0);
    }
    fence_proxy_async_smem();
}

template <int MODE, int BQ, typename Out>
__global__ void __launch_bounds__(gg::THREADS, 1)
grouped_gemm_kernel(const GroupedArgs a, const __grid_constant__ CUtensorMap map_p, const __grid_constant__ CUtensorMap map_q) {
    using namespace gg;
    using C_ = Cfg<BQ>;
    constexpr int STAGES = C_::STAGES;
    constexpr bool P_MN = MODE != FWD, Q_MN = MODE == WGRAD;

    extern __shared__ unsigned char smem_raw[];
    const uint32_t raw_addr = smem_u32(smem_raw);
    unsigned char* ring = smem_raw + ((1024u - (raw_addr & 1023u)) & 1023u);
    unsigned char* epi_smem = ring + STAGES * C_::STAGE_BYTES;
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(epi_smem + EPI_WARPS * C_::EPI_WARP_BYTES);
    uint64_t* empty_bar = full_bar + STAGES;
    uint64_t* acc_full_bar = empty_bar + STAGES;   // [2]
    uint64_t* acc_empty_bar = acc_full_bar + 2;    // [2]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty_bar + 2);
    volatile uint32_t* abort_flag = tmem_slot + 1;
    volatile uint32_t* never_flag = tmem_slot + 2;
    int* table = reinterpret_cast<int*>(reinterpret_cast<unsigned char*>(full_bar) + C_::BAR_BYTES);
    int* row_first = table;
    int* row_last = table + MAX_EXPERTS;
    int* tile_first = table + 2 * MAX_EXPERTS;     // [experts + 1]

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int p_tiles = (a.p_dim + BLOCK_P - 1) / BLOCK_P;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full_bar[b], 1);
            mbar_init(&acc_empty_bar[b], EPI_WARPS);
        }
        *abort_flag = 0;
        *never_flag = 0;
        fence_barrier_init();
    }
    if (warp == 1) {
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(static_cast<uint32_t>(TMEM_COLS))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    for (int e = threadIdx.x; e < a.experts; e += THREADS) {
        const int first = min(max(a.offsets[e], 0), a.rows);
        row_first[e] = first;
        row_last[e] = min(max(a.offsets[e + 1], first), a.rows);
    }
    __syncthreads();
    if (MODE != WGRAD && warp == 2) {
        int carry = 0;
        for (int e0 = 0; e0 < a.experts; e0 += 32) {
            const int e = e0 + lane;
            const int n = e < a.experts ? (row_last[e] - row_first[e] + BQ - 1) / BQ * p_tiles : 0;
            int incl = n;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, incl, d);
                if (lane >= d) incl += up;
            }
            if (e < a.experts) tile_first[e] = carry + incl - n;
            carry += __shfl_sync(0xffffffffu, incl, 31);
        }
        if (lane == 0) tile_first[a.experts] = carry;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int total_tiles = MODE == WGRAD ? a.experts * p_tiles * ((a.q_dim + BQ - 1) / BQ) : tile_first[a.experts];

    bool timed_out = false;

    if (warp == 0) {
        // ------------------------- TMA producer -------------------------
        if (lane == 0) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_p)) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_q)) : "memory");
            TileWalk<MODE, BQ> walk(a, table);
            int stage = 0;
            uint32_t phase = 0;
            int armed = 0;
            for (int t = blockIdx.x; t < total_tiles && !timed_out; t += gridDim.x) {
                const Tile tile = walk.at(t, a);
                const int boxes = (tile.cols + 63) / 64;
                for (int cb = 0; cb < tile.blocks; ++cb) {
                    if (!mbar_wait_bounded_sleepy(&empty_bar[stage], phase ^ 1u, abort_flag, 40)) {
                        timed_out = true;
                        break;
                    }
                    unsigned char* p_dst = ring + stage * C_::STAGE_BYTES;
                    unsigned char* q_dst = p_dst + C_::P_BYTES;
                    uint64_t* bar = &full_bar[stage];
                    const int c0 = tile.first + cb * BLOCK_C;
                    mbar_arrive_expect_tx(bar, C_::P_BYTES + boxes * CHUNK_BYTES);
                    if (MODE == FWD) {
                        tma_load_3d(p_dst, &map_p, c0, tile.p0, tile.e, bar);
                    } else if (MODE == DGRAD) {
                        tma_load_3d(p_dst, &map_p, tile.p0, c0, tile.e, bar);
                        tma_load_3d(p_dst + CHUNK_BYTES, &map_p, tile.p0 + 64, c0, tile.e, bar);
                    } else {
                        tma_load_2d(p_dst, &map_p, tile.p0, c0, bar);
                        tma_load_2d(p_dst + CHUNK_BYTES, &map_p, tile.p0 + 64, c0, bar);
                    }
                    for (int b = 0; b < boxes; ++b) {
                        if (MODE == WGRAD) tma_load_2d(q_dst + b * CHUNK_BYTES, &map_q, tile.q0 + 64 * b, c0, bar);
                        else tma_load_2d(q_dst + b * CHUNK_BYTES, &map_q, c0, tile.q0 + 64 * b, bar);
                    }
                    armed = armed < STAGES ? armed + 1 : STAGES;
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            if (timed_out || *abort_flag) {
                // Unwind: let loads already in flight land before shared memory is released.
                int s = stage;
                uint32_t ph = phase;
                for (int i = 0; i < armed; ++i) {
                    if (--s < 0) {
                        s = STAGES - 1;
                        ph ^= 1u;
                    }
                    mbar_wait_bounded(&full_bar[s], ph, never_flag, 2000000ull);
                }
            }
        }
    } else if (warp == 1) {
        // ------------------------- MMA issuer -------------------------
        // Lane 0 waits and issues; the whole warp walks along because all of it zeros a wgrad tile's tail rows.
        TileWalk<MODE, BQ> walk(a, table);
        int stage = 0;
        uint32_t phase = 0;
        int acc = 0;
        uint32_t acc_phase = 0;
        for (int t = blockIdx.x; t < total_tiles && !timed_out; t += gridDim.x) {
            const Tile tile = walk.at(t, a);
            if (tile.blocks == 0) continue;   // an empty group's weights: the epilogue stores zeros
            bool ready = lane != 0 || mbar_wait_bounded(&acc_empty_bar[acc], acc_phase ^ 1u, abort_flag);
            if (!__all_sync(0xffffffffu, ready)) {
                timed_out = true;
                break;
            }
            tc_fence_after();
            const uint32_t idesc = instr_desc(P_MN, Q_MN, BLOCK_P, (tile.cols + 15) & ~15);
            const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * BQ);
            for (int cb = 0; cb < tile.blocks; ++cb) {
                ready = lane != 0 || mbar_wait_bounded(&full_bar[stage], phase, abort_flag);
                if (!__all_sync(0xffffffffu, ready)) {
                    timed_out = true;
                    break;
                }
                unsigned char* p_src = ring + stage * C_::STAGE_BYTES;
                int steps = BLOCK_C / UMMA_K;
                if (MODE == WGRAD && tile.tail && cb == tile.blocks - 1) {
                    __syncwarp();
                    zero_tail_rows(p_src, 2 + (tile.cols + 63) / 64, tile.tail, lane);
                    __syncwarp();
                    steps = (tile.tail + UMMA_K - 1) / UMMA_K;
                }
                if (lane == 0) {
                    tc_fence_after();
                    const uint32_t p_addr = smem_u32(p_src), q_addr = p_addr + C_::P_BYTES;
                    const uint64_t p_desc = P_MN ? smem_desc_mn_sw128(p_addr) : smem_desc_k_sw128(p_addr);
                    const uint64_t q_desc = Q_MN ? smem_desc_mn_sw128(q_addr) : smem_desc_k_sw128(q_addr);
                    // 16 contraction indices on: 32 bytes inside the span (K-major), 16 rows of 128 bytes (MN-major).
                    constexpr uint64_t P_STEP = P_MN ? 128 : 2, Q_STEP = Q_MN ? 128 : 2;
                    for (int k = 0; k < steps; ++k)
                        umma_bf16(d_tmem, p_desc + P_STEP * k, q_desc + Q_STEP * k, idesc, (cb | k) != 0 ? 1u : 0u);
                    umma_commit(&empty_bar[stage]);
                }
                if (++stage == STAGES) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
            if (timed_out) break;
            if (lane == 0) umma_commit(&acc_full_bar[acc]);
            if (++acc == 2) {
                acc = 0;
                acc_phase ^= 1u;
            }
        }
    } else {
        // ------------------------- epilogue warps -------------------------
        const int quarter = warp & 3;
        unsigned char* stage_buf = epi_smem + (warp - 2) * C_::EPI_WARP_BYTES;
        Out* out = static_cast<Out*>(a.out);
        TileWalk<MODE, BQ> walk(a, table);
        int acc = 0;
        uint32_t acc_phase = 0;
        for (int t = blockIdx.x; t < total_tiles; t += gridDim.x) {
            const Tile tile = walk.at(t, a);
            const bool zeros = tile.blocks == 0;
            if (!zeros) {
                const bool ready = lane != 0 || mbar_wait_bounded_sleepy(&acc_full_bar[acc], acc_phase, abort_flag, 200);
                if (!__all_sync(0xffffffffu, ready)) {
                    timed_out = true;
                    break;
                }
                tc_fence_after();
            }
            const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(acc * BQ);
            const int p_warp = tile.p0 + quarter * 32;   // this warp's first lane index
            if (MODE == WGRAD) {
                // A lane holds consecutive columns of one row of dW.  32 rows x 128 bytes at a time pass through shared
                // memory (16-byte pieces XOR-swizzled by row), so that a store instruction writes whole lines.
                constexpr int COLS = 128 / sizeof(Out);   // columns per pass
                constexpr int PIECE = 16 / sizeof(Out);
                Out* dst = out + (static_cast<size_t>(tile.e) * a.p_dim + p_warp) * a.ldo + tile.q0;
                for (int c0 = 0; c0 < tile.cols; c0 += COLS) {
                    uint32_t r[COLS / 32][32];
#pragma unroll
                    for (int h = 0; h < COLS / 32; ++h) {
                        if (zeros) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) r[h][i] = 0;
                        } else {
                            tmem_ld_32cols(t_row + c0 + 32 * h, r[h]);
                        }
                    }
                    if (!zeros) tmem_ld_wait();
#pragma unroll
                    for (int ch = 0; ch < 8; ++ch) {
                        const uint32_t* v = &r[ch * PIECE / 32][ch * PIECE % 32];
                        uint4 o;
                        if constexpr (sizeof(Out) == 2) {
                            o = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
                        } else {
                            o = make_uint4(v[0], v[1], v[2], v[3]);
                        }
                        *reinterpret_cast<uint4*>(stage_buf + lane * 128 + ((ch ^ (lane & 7)) << 4)) = o;
                    }
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int row = 4 * j + (lane >> 3), ch = lane & 7;
                        const uint4 v = *reinterpret_cast<const uint4*>(stage_buf + row * 128 + ((ch ^ (row & 7)) << 4));
                        if (p_warp + row < a.p_dim && c0 + ch * PIECE < tile.cols)
                            *reinterpret_cast<uint4*>(dst + static_cast<size_t>(row) * a.ldo + c0 + ch * PIECE) = v;
                    }
                    __syncwarp();
                }
            } else {
                // A lane holds one weight row's products with consecutive activation rows; out has the weight dimension
                // contiguous.  32 activation rows at a time are transposed through shared memory.
                __nv_bfloat16* buf = reinterpret_cast<__nv_bfloat16*>(stage_buf);
                Out* dst = out + static_cast<size_t>(tile.q0) * a.ldo + p_warp;
                for (int c0 = 0; c0 < tile.cols; c0 += 32) {
                    uint32_t r[32];
                    tmem_ld_32cols(t_row + c0, r);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 32; ++i) buf[i * 32 + lane] = __float2bfloat16_rn(__uint_as_float(r[i]));
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int row = 8 * j + (lane >> 2), col = (lane & 3) * 8;
                        const uint4 v = *reinterpret_cast<const uint4*>(buf + row * 32 + col);
                        if (c0 + row < tile.cols && p_warp + col < a.p_dim)
                            *reinterpret_cast<uint4*>(dst + static_cast<size_t>(c0 + row) * a.ldo + col) = v;
                    }
                    __syncwarp();
                }
            }
            if (zeros) continue;
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty_bar[acc]);
            if (++acc == 2) {
                acc = 0;
                acc_phase ^= 1u;
            }
        }
    }

    if (timed_out) {
        *abort_flag = 1;
        raise_device_status(DEV_GROUPED_PIPE_TIMEOUT);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base),
                     "r"(static_cast<uint32_t>(TMEM_COLS))
                     : "memory");
    }
}

// ---- host side ---------------------------------------------------------------------------------------------------

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                   const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

int encode(CUtensorMap* out, int rank, const void* ptr, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
    static std::mutex mu;
    static EncodeTiledFn fn = nullptr;
    {
        std::lock_guard<std::mutex> lk(mu);
        if (!fn) {
            void* p = nullptr;
            cudaDriverEntryPointQueryResult q;
            cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q);
            if (e != cudaSuccess || !p || q != cudaDriverEntryPointSuccess)
                return set_error(PRISM_B200_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
            fn = reinterpret_cast<EncodeTiledFn>(p);
        }
    }
    const cuuint32_t estr[3] = {1, 1, 1};
    const CUresult r = fn(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(ptr), dims, strides, box, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(PRISM_B200_ERR_CUDA, "cuTensorMapEncodeTiled failed with %d", static_cast<int>(r));
    return PRISM_B200_OK;
}

// Rows of activations: width contiguous, 64 x 64 boxes.
int rows_map(CUtensorMap* out, const void* ptr, long long rows, int width, long long ld) {
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(width), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld) * 2};
    const cuuint32_t box[2] = {64, 64};
    return encode(out, 2, ptr, dims, strides, box);
}

// Weights [experts][n][k]: boxes of 64 k and box_n rows of one expert.
int weights_map(CUtensorMap* out, const void* ptr, int experts, int n, int k, int box_n) {
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(k), static_cast<cuuint64_t>(n), static_cast<cuuint64_t>(experts)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(k) * 2, static_cast<cuuint64_t>(n) * k * 2};
    const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_n), 1};
    return encode(out, 3, ptr, dims, strides, box);
}

template <int MODE, int BQ, typename Out>
int launch_grouped(const GroupedArgs& a, long long most_tiles, const CUtensorMap& map_p, const CUtensorMap& map_q, cudaStream_t s) {
    auto kern = grouped_gemm_kernel<MODE, BQ, Out>;
    constexpr size_t smem = gg::Cfg<BQ>::SMEM_BYTES;
    static std::mutex mu;
    static int sm_count[64] = {};
    int dev = 0, sms = 0;
    PRISM_CUDA_TRY(cudaGetDevice(&dev));
    {
        std::lock_guard<std::mutex> lk(mu);
        const bool cacheable = dev >= 0 && dev < 64;
        if (!cacheable || !sm_count[dev]) {
            PRISM_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
            PRISM_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
            if (cacheable) sm_count[dev] = sms;
        } else {
            sms = sm_count[dev];
        }
    }
    const int grid = most_tiles < sms ? static_cast<int>(most_tiles) : sms;
    kern<<<grid, gg::THREADS, smem, s>>>(a, map_p, map_q);
    PRISM_CUDA_TRY(cudaGetLastError());
    count_launch();
    return PRISM_B200_OK;
}

// Checks that the three entry points share.  Returns a status; *done: nothing to compute.
int check_grouped(const char* fn, int experts, int rows, int n, int k, bool* done) {
    *done = false;
    if (experts < 0 || rows < 0 || n < 0 || k < 0) return set_error(PRISM_B200_ERR_INVALID_ARGUMENT, "%s: negative size", fn);
    if (experts > gg::MAX_EXPERTS)
        return set_error(PRISM_B200_ERR_UNSUPPORTED_SHAPE, "%s: at most %d experts (got %d)", fn, gg::MAX_EXPERTS, experts);
    if (n % 8 || k % 8)
        return set_error(PRISM_B200_ERR_UNSUPPORTED_SHAPE, "%s: need n %% 8 == 0 and k %% 8 == 0 (got %d, %d)", fn, n, k);
    if (experts == 0) *done = true;
    const long long tiles = ((n > k ? n : k) / 64LL + 1) * (rows / 64LL + experts) , wtiles = (n / 128LL + 1) * (k / 128LL + 1) * experts;
    if (rows > 1 << 30 || tiles > 0x3fffffffLL || wtiles > 0x3fffffffLL) return set_error(PRISM_B200_ERR_TOO_LARGE, "%s: too many tiles", fn);
    return PRISM_B200_OK;
}

int check_matrix(const char* fn, const char* name, const void* ptr, long long ld, int width, int multiple) {
    if (!ptr) return set_error(PRISM_B200_ERR_INVALID_ARGUMENT, "%s: null pointer (%s)", fn, name);
    if (reinterpret_cast<uintptr_t>(ptr) & 15u) return set_error(PRISM_B200_ERR_MISALIGNED, "%s: %s must be 16-byte aligned", fn, name);
    if (ld < width) return set_error(PRISM_B200_ERR_INVALID_ARGUMENT, "%s: row stride of %s below its width", fn, name);
    if (ld % multiple)
        return set_error(PRISM_B200_ERR_MISALIGNED, "%s: row stride of %s must be a multiple of %d", fn, name, multiple);
    return PRISM_B200_OK;
}

// fwd (lanes n, contraction k) and dgrad (lanes k, contraction n).
template <int MODE>
int grouped_rows(const char* fn, int experts, int rows, int n, int k, const uint16_t* in, long long ld_in, const uint16_t* w,
                 const int* offsets, uint16_t* out, long long ld_out, void* stream) {
    bool done;
    if (int rc = check_grouped(fn, experts, rows, n, k, &done)) return rc;
    const int p_dim = MODE == gg::FWD ? n : k, c_dim = MODE == gg::FWD ? k : n;
    if (done || rows == 0 || p_dim == 0) return PRISM_B200_OK;
    if (c_dim == 0) return set_error(PRISM_B200_ERR_UNSUPPORTED_SHAPE, "%s: nothing to add up (%s is 0)", fn, MODE == gg::FWD ? "k" : "n");
    if (!offsets) return set_error(PRISM_B200_ERR_INVALID_ARGUMENT, "%s: null pointer (offsets)", fn);
    if (int rc = check_matrix(fn, "the input", in, ld_in, c_dim, 8)) return rc;
    if (int rc = check_matrix(fn, "the weights", w, k, k, 8)) return rc;
    if (int rc = check_matrix(fn, "the output", out, ld_out, p_dim, 8)) return rc;
    if (rows_overlap(out, rows, p_dim, ld_out, in, rows, c_dim, ld_in, 2) ||
        rows_overlap(out, rows, p_dim, ld_out, w, static_cast<long long>(experts) * n, k, k, 2))
        return set_error(PRISM_B200_ERR_INVALID_ARGUMENT, "%s: the output overlaps an input", fn);
    if (int rc = bind_status_word()) return rc;
    CUtensorMap map_p, map_q;
    if (int rc = weights_map(&map_p, w, experts, n, k, MODE == gg::FWD ? gg::BLOCK_P : 64)) return rc;
    if (int rc = rows_map(&map_q, in, rows, c_dim, ld_in)) return rc;
    const GroupedArgs a{offsets, experts, rows, p_dim, 0, c_dim, out, ld_out};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const long long p_tiles = (p_dim + gg::BLOCK_P - 1) / gg::BLOCK_P;
    const int groups = experts < rows ? experts : rows;
    auto most = [&](int bq) { return (rows / bq + static_cast<long long>(groups)) * p_tiles; };
    // Rows per tile by the mean group: a tile of few rows leaves its ring to the weights (64: eight stages of 24 KB).
    if (rows <= 64LL * experts) return launch_grouped<MODE, 64, __nv_bfloat16>(a, most(64), map_p, map_q, s);
    if (rows <= 128LL * experts) return launch_grouped<MODE, 128, __nv_bfloat16>(a, most(128), map_p, map_q, s);
    return launch_grouped<MODE, 256, __nv_bfloat16>(a, most(256), map_p, map_q, s);
}

}  // namespace
}  // namespace prism_b200

using namespace prism_b200;

extern "C" int prism_b200_grouped_gemm_bf16(int experts, int rows, int n, int k, const uint16_t* x, long long ldx, const uint16_t* w,
                                            const int* offsets, uint16_t* out, long long ldo, void* stream) {
    return grouped_rows<gg::FWD>("grouped_gemm_bf16", experts, rows, n, k, x, ldx, w, offsets, out, ldo, stream);
}

extern "C" int prism_b200_grouped_gemm_bf16_dgrad(int experts, int rows, int n, int k, const uint16_t* dy, long long lddy,
                                                  const uint16_t* w, const int* offsets, uint16_t* dx, long long lddx, void* stream) {
    return grouped_rows<gg::DGRAD>("grouped_gemm_bf16_dgrad", experts, rows, n, k, dy, lddy, w, offsets, dx, lddx, stream);
}

extern "C" int prism_b200_grouped_gemm_bf16_wgrad(int experts, int rows, int n, int k, const uint16_t* dy, long long lddy,
                                                  const uint16_t* x, long long ldx, const int* offsets, int out_dtype, void* dw,
                                                  void* stream) {
    const char* fn = "grouped_gemm_bf16_wgrad";
    bool done;
    if (int rc = check_grouped(fn, experts, rows, n, k, &done)) return rc;
    if (out_dtype != PRISM_B200_F32 && out_dtype != PRISM_B200_BF16)
        return set_error(PRISM_B200_ERR_INVALID_ARGUMENT, "%s: dw is fp32 or bf16", fn);
    if (done || n == 0 || k == 0) return PRISM_B200_OK;
    if (int rc = check_matrix(fn, "dw", dw, k, k, 8)) return rc;
    const size_t dw_bytes = static_cast<size_t>(experts) * n * k * (out_dtype == PRISM_B200_F32 ? 4 : 2);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (rows == 0) {
        PRISM_CUDA_TRY(cudaMemsetAsync(dw, 0, dw_bytes, s));
        return PRISM_B200_OK;
    }
    if (!offsets) return set_error(PRISM_B200_ERR_INVALID_ARGUMENT, "%s: null pointer (offsets)", fn);
    if (int rc = check_matrix(fn, "dy", dy, lddy, n, 8)) return rc;
    if (int rc = check_matrix(fn, "x", x, ldx, k, 8)) return rc;
    const long long dw_halves = static_cast<long long>(dw_bytes / 2);
    if (rows_overlap(dw, 1, dw_halves, dw_halves, dy, rows, n, lddy, 2) || rows_overlap(dw, 1, dw_halves, dw_halves, x, rows, k, ldx, 2))
        return set_error(PRISM_B200_ERR_INVALID_ARGUMENT, "%s: dw overlaps an input", fn);
    if (int rc = bind_status_word()) return rc;
    CUtensorMap map_p, map_q;
    if (int rc = rows_map(&map_p, dy, rows, n, lddy)) return rc;
    if (int rc = rows_map(&map_q, x, rows, k, ldx)) return rc;
    const GroupedArgs a{offsets, experts, rows, n, k, 0, dw, k};
    const long long tiles = static_cast<long long>(experts) * ((n + gg::BLOCK_P - 1) / gg::BLOCK_P) * ((k + 255) / 256);
    return out_dtype == PRISM_B200_F32 ? launch_grouped<gg::WGRAD, 256, float>(a, tiles, map_p, map_q, s)
                                       : launch_grouped<gg::WGRAD, 256, __nv_bfloat16>(a, tiles, map_p, map_q, s);
}
