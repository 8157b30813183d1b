// bf16 matrix products grouped by expert, with group borders on the device: expert e owns the rows
// offsets[e] <= r < offsets[e + 1] of the activations.
//
//   fwd    out[r, n] = sum_k x[r, k] * W[e][n, k]        (a row of out per row of x)
//   dgrad  dx[r, k]  = sum_n dy[r, n] * W[e][n, k]       (the gradient of the rows)
//   wgrad  dW[e][n, k] = sum over the expert's rows of dy[r, n] * x[r, k]
//
// One kernel in three modes on tcgen05.mma with fp32 accumulators in tensor memory, two CTAs to a tile (cta_group::2):
//   * The weights' dimension (n, k, n) indexes tensor-memory lanes, in blocks of 256 (128 in each CTA), one or two to a
//     tile.  In fwd and dgrad the rows index the columns, so a tile of few rows is an MMA of few columns (a multiple of 32,
//     chosen per tile): a group costs what its rows cost, and a group of one row still streams its matrix at full width.
//   * Operands lie in shared memory as TMA writes them, in 128-byte swizzle spans: K-major where the contraction is
//     contiguous in memory (x, W in fwd; dy in dgrad), MN-major where the other dimension is (W in dgrad, both in
//     wgrad); the MMA takes either, so nothing is transposed.
//   * A tile of two lane blocks (512 x 256, four 48 KB stages) reads a quarter less per MMA than a tile of one (six 32 KB
//     stages) and gives each load more MMA time to hide in: at the sizes below fwd 795 us against 989, dgrad 754 against
//     1024, wgrad 879 against 1139.  One block serves where there are too few tiles, for groups of few rows (which stream
//     their matrices and have no use for more MMA: 64 rows over 32 experts of 2048 x 4096 94 us against 109), and for fp32
//     results, whose promotion below takes the registers.
//   * The MMAs are issued by one elected lane of a warp that stays together, from descriptors kept as words: the issue
//     must not take longer than the MMAs.
//   * The epilogue moves an accumulator into registers, hands it back by an arrival that orders nothing else, and then
//     stores.  (An arrival with .release also waits for the stores of the tile before: wgrad 879 -> 940 us.)
//   * fwd and dgrad read past a group's last row into the next group's: those columns are computed and not stored.
//     wgrad contracts over rows, so there the rows behind the group's last are overwritten with zeros in shared memory
//     before the tile's last MMAs (both operands: a NaN there must not meet a zero).  Each CTA does so for its own
//     stage, in warp 1; the second CTA's loads of such a stage complete on a barrier of its own, and its warp tells the
//     first CTA, whose warp 1 issues all MMAs, when the zeros are in place.
//   * wgrad to fp32: the tensor core adds with truncation, so a long sum drifts (by up to 2^-23 of a partial sum per step;
//     4.4e-6 of the result's norm at 4096 rows).  Every 512 rows the accumulator is added to fp32 registers by the epilogue
//     warps instead (4.8e-7), while the MMAs go on into the other accumulator.
//   * Warp 0 loads, warp 1 issues the MMAs, warps 2-17 store.  Every wait is bounded as in gemm_bf16.cu.  Tiles are dealt
//     round-robin to persistent CTA pairs; every CTA works out the groups' tiles from the offsets by itself (no launch
//     before this one, no host copy of the offsets).
// Measured (CUDA events, cold L2, median of 40; the card is at its power limit, quartiles within 8%): 32768 rows,
// 32 equal groups, 4096 x 4096: fwd 795 us (1384 TFLOP/s), dgrad 754, wgrad to bf16 879, to fp32 1200; uneven groups
// (183 to 2237 rows) 884, 883, 951, 1262.  The dense kernel of gemm_bf16.cu takes 724 warm
// on the first of these sizes, this one 742.
// Offsets are read with care: each border is clamped to the rows that exist and to the border before it, so a wrong
// array gives wrong products but no access outside the matrices.
#include "common.cuh"
#include "tcgen05.cuh"

#include <mutex>

namespace prism_b200 {
namespace {

namespace gg {
constexpr int FWD = 0, DGRAD = 1, WGRAD = 2;
constexpr int HALF_P = 128;        // lanes of one CTA and block; a block of a tile has 256: n (fwd, wgrad) or k (dgrad)
constexpr int BLOCK_P = 256;
constexpr int BLOCK_Q = 256;       // columns of a tile: rows (fwd, dgrad) or k (wgrad)
constexpr int BLOCK_C = 64;        // contraction per stage: one 128-byte span, or 64 rows of it
constexpr int UMMA_K = 16;
constexpr int EPI_WARPS = 16;
constexpr int THREADS = 64 + 32 * EPI_WARPS;
constexpr int TMEM_COLS = 512;
constexpr int MAX_EXPERTS = 1024;
constexpr int GROUP_Q = 16;        // column tiles walked for each lane tile (L2 reuse); 4, 8 and 32 measure the same
constexpr int PROMOTE_BLOCKS = 8;  // contraction blocks per accumulator of an fp32 wgrad
constexpr uint32_t CHUNK_BYTES = 64 * 64 * 2;   // one 64 x 64 box
constexpr uint32_t P_BYTES = HALF_P * BLOCK_C * 2;
constexpr uint32_t Q_BYTES = BLOCK_Q / 2 * BLOCK_C * 2;
constexpr uint32_t RING_BYTES = 196608;
constexpr uint32_t BAR_BYTES = 256;
constexpr int SKEW = 3;            // stages whose MMAs are ordered by lane block at a tile's ends
// Epilogue staging: per warp 16 rows of 128 bytes (wgrad); per four warps 16 rows of 256 bytes, and the tile table (fwd, dgrad).
__host__ __device__ constexpr uint32_t epi_bytes(int mode) { return EPI_WARPS * (mode == WGRAD ? 2048 : 1024); }
constexpr int smem_bytes(int mode, int experts) {
    return 1024 + RING_BYTES + epi_bytes(mode) + BAR_BYTES + (mode == WGRAD ? 0 : (experts + 1) * 4);
}
static_assert(smem_bytes(FWD, MAX_EXPERTS) <= 232448 && smem_bytes(WGRAD, MAX_EXPERTS) <= 232448, "shared memory of one CTA");

// NB: lane blocks of a tile.
template <int NB>
struct Cfg {
    static constexpr int STAGES = NB == 1 ? 6 : 4;
    static constexpr uint32_t STAGE_BYTES = NB * P_BYTES + Q_BYTES;
    static constexpr int SIDES = NB == 1 ? 4 : 2;    // epilogue warps that share a lane quarter of a block
    static constexpr int HELD = 8 / SIDES;           // column blocks of 32 per epilogue warp
    static_assert(STAGES * STAGE_BYTES == RING_BYTES, "both cuts fill the ring");
};

// kind::f16, D fp32, A and B bf16; bits 15 / 16: A / B is MN-major.
__host__ __device__ constexpr uint32_t instr_desc(bool a_mn, bool b_mn, int m, int n) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) |
           (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
}  // namespace gg

// Shared-memory matrix descriptors, 128-byte swizzle, as two words: the low one holds the address (>> 4) and the leading
// byte offset, the high one is constant (stride byte offset 1024, version 1, swizzle mode 2).
//   K-major:  8 rows of one 128-byte span make a 1024-byte atom, 8 more rows 1024 bytes on (the stride offset).
//   MN-major: 64 elements contiguous, the next contraction index 128 bytes on, 8 of them an atom (the stride offset); the
//             next 64 elements one 64 x 64 box on (the leading offset).
constexpr uint32_t DESC_HIGH = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_low(bool mn_major, uint32_t smem_addr) {
    return ((smem_addr & 0x3FFFFu) >> 4) | ((mn_major ? gg::CHUNK_BYTES >> 4 : 1u) << 16);
}

// One MMA of both CTAs.  Descriptors arrive as words so that a step along the contraction is one 32-bit addition: the
// issuing thread has 128 cycles per MMA of 256 x 256 x 16.
__device__ __forceinline__ void umma_pair(uint32_t tmem_d, uint32_t a_low, uint32_t b_low, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        ".reg .b64 da, db;\n\t"
        "mov.b64 da, {%1, %5};\n\t"
        "mov.b64 db, {%2, %5};\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], da, db, %3, p;\n\t"
        "}\n" ::"r"(tmem_d),
        "r"(a_low), "r"(b_low), "r"(idesc), "r"(accumulate), "r"(DESC_HIGH)
        : "memory");
}
// Arrives on the barrier at this offset in both CTAs once every MMA issued so far has finished.
__device__ __forceinline__ void umma_commit_both(uint64_t* bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
        "h"(static_cast<uint16_t>(3))
        : "memory");
}

__device__ __forceinline__ void tma_load_3d_pair(void* dst, const CUtensorMap* map, int x, int y, int z, uint32_t cluster_bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(cluster_bar)
        : "memory");
}

// An arrival in another CTA that orders nothing but the tensor-memory reads before it (tcgen05.wait::ld and the fence have
// done that).  With .release the epilogue warps wait here until their stores of the tile before have reached L2.
__device__ __forceinline__ void mbar_arrive_cluster_relaxed(uint32_t cluster_bar_addr) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar_addr) : "memory");
}

// Bounded wait for an arrival from the other CTA, with acquire semantics for what that CTA wrote before it.
__device__ __forceinline__ bool mbar_wait_cluster_bounded(uint64_t* bar, uint32_t parity, volatile uint32_t* abort_flag) {
    const unsigned long long t0 = global_timer_ns();
    for (uint32_t i = 1;; ++i) {
        uint32_t ok;
        asm volatile(
            "{\n\t"
            ".reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t"
            "}\n"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity)
            : "memory");
        if (ok) return true;
        if ((i & 63u) == 0u && (*abort_flag || global_timer_ns() - t0 > kWaitLimitNs)) return false;
    }
}

// 16 consecutive fp32 columns of this thread's tensor-memory lane.
__device__ __forceinline__ void tmem_ld_16cols(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
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
    int nb;           // lane blocks that exist
    int first, blocks, tail;   // wgrad: first row; contraction blocks; rows of the last block (0: all 64)
    __device__ __forceinline__ int half() const { return ((cols + 31) & ~31) >> 1; }   // columns staged by each CTA
    __device__ __forceinline__ int boxes() const { return (half() + 63) >> 6; }
};

// Rows of expert e, clamped to the rows that exist and to a first row not behind the last.
__device__ __forceinline__ int2 group_rows(const GroupedArgs& a, int e) {
    const int first = min(max(__ldg(a.offsets + e), 0), a.rows);
    return make_int2(first, min(max(__ldg(a.offsets + e + 1), first), a.rows));
}

// Walks a CTA pair's tiles in order; the cursor over the experts only moves forward.
template <int MODE, int NB>
struct TileWalk {
    const int* tile_first;      // fwd, dgrad: first tile of each expert
    int p_tiles, q_tiles, e = 0;
    __device__ __forceinline__ TileWalk(const GroupedArgs& a, const int* table)
        : tile_first(table), p_tiles((a.p_dim + NB * gg::BLOCK_P - 1) / (NB * gg::BLOCK_P)),
          q_tiles(MODE == gg::WGRAD ? (a.q_dim + gg::BLOCK_Q - 1) / gg::BLOCK_Q : 0) {}
    __device__ __forceinline__ Tile at(int t, const GroupedArgs& a) {
        using namespace gg;
        Tile r;
        int in, qt;
        int2 rows;
        if (MODE == WGRAD) {
            const int per = p_tiles * q_tiles;
            r.e = t / per;
            in = t - r.e * per;
            rows = group_rows(a, r.e);
            qt = q_tiles;
        } else {
            while (tile_first[e + 1] <= t) ++e;   // t < tile_first[experts]
            r.e = e;
            in = t - tile_first[e];
            rows = group_rows(a, e);
            qt = (rows.y - rows.x + BLOCK_Q - 1) / BLOCK_Q;
        }
        const int per_band = GROUP_Q * p_tiles;
        const int band = in / per_band, q_first = band * GROUP_Q;
        const int in_band = in - band * per_band, height = min(GROUP_Q, qt - q_first);
        const int q = q_first + in_band % height;
        r.p0 = (in_band / height) * (NB * BLOCK_P);
        r.nb = NB == 1 || r.p0 + BLOCK_P < a.p_dim ? NB : 1;
        if (MODE == WGRAD) {
            r.q0 = q * BLOCK_Q;
            r.cols = min(BLOCK_Q, a.q_dim - r.q0);
            r.first = rows.x;
            r.blocks = (rows.y - rows.x + BLOCK_C - 1) / BLOCK_C;
            r.tail = (rows.y - rows.x) % BLOCK_C;
        } else {
            // A group's rows in equal shares (multiples of 32 but for the last), not 256 at a time and a rest: the tiles'
            // costs differ less (30000 x 2048 x 2048 over 60 uneven experts 227 -> 224 us, 32768 x 4096 x 4096 over 32 893 -> 884).
            const int share = ((rows.y - rows.x + qt - 1) / qt + 31) & ~31;
            r.q0 = rows.x + q * share;
            r.cols = min(share, rows.y - r.q0);
            r.first = 0;
            r.blocks = (a.c_dim + BLOCK_C - 1) / BLOCK_C;
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
}

// The same for a whole stage: the lane blocks' boxes, then the columns'; visible to the MMA afterwards.
template <int NB>
__device__ __forceinline__ void zero_tail(unsigned char* stage, const Tile& tile, int lane) {
    zero_tail_rows(stage, 2 * tile.nb, tile.tail, lane);
    zero_tail_rows(stage + NB * gg::P_BYTES, tile.boxes(), tile.tail, lane);
    fence_proxy_async_smem();
    __syncwarp();
}

// Barriers of the four epilogue warps `four` (named barrier four + 1): plain, and with the conjunction of `ready`.  Every
// thread of the four takes part each time, so none can be left waiting by another's timeout.
__device__ __forceinline__ void four_warps_sync(int four) {
    __syncwarp();
    asm volatile("barrier.cta.sync.aligned %0, 128;" ::"r"(four + 1) : "memory");
}
__device__ __forceinline__ bool four_warps_all(int four, bool ready) {
    uint32_t all;
    __syncwarp();
    asm volatile(
        "{\n\t"
        ".reg .pred p, q;\n\t"
        "setp.ne.b32 p, %2, 0;\n\t"
        "barrier.cta.red.and.pred.aligned q, %1, 128, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t"
        "}\n"
        : "=r"(all)
        : "r"(four + 1), "r"(static_cast<uint32_t>(ready))
        : "memory");
    return all != 0;
}

template <int MODE, typename Out, int NB>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(gg::THREADS, 1)
grouped_gemm_kernel(const GroupedArgs a, const __grid_constant__ CUtensorMap map_p, const __grid_constant__ CUtensorMap map_q) {
    using namespace gg;
    constexpr bool P_MN = MODE != FWD, Q_MN = MODE == WGRAD;
    constexpr bool PROMOTE = MODE == WGRAD && sizeof(Out) == 4;
    static_assert(!PROMOTE || NB == 1, "fp32 sums of two lane blocks do not fit the epilogue's registers");
    using C_ = Cfg<NB>;
    constexpr int STAGES = C_::STAGES;
    constexpr uint32_t STAGE_BYTES = C_::STAGE_BYTES;

    extern __shared__ unsigned char smem_raw[];
    const uint32_t raw_addr = smem_u32(smem_raw);
    unsigned char* ring = smem_raw + ((1024u - (raw_addr & 1023u)) & 1023u);   // same offset in both CTAs
    unsigned char* epi_smem = ring + RING_BYTES;
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(epi_smem + epi_bytes(MODE));   // the leader's are used
    uint64_t* empty_bar = full_bar + STAGES;
    uint64_t* tail_bar = empty_bar + STAGES;       // second CTA: a tail stage has landed; leader: its zeros are in place
    uint64_t* acc_full_bar = tail_bar + STAGES;    // [2]: the accumulators that alternate, or one per lane block
    uint64_t* acc_empty_bar = acc_full_bar + 2;    // [2], the leader's are used
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty_bar + 2);
    volatile uint32_t* abort_flag = tmem_slot + 1;
    volatile uint32_t* never_flag = tmem_slot + 2;
    int* tile_first = reinterpret_cast<int*>(reinterpret_cast<unsigned char*>(full_bar) + BAR_BYTES);   // [experts + 1], not in wgrad
    static_assert((3 * STAGES + 4) * 8 + 12 <= BAR_BYTES, "barriers, TMEM slot, flags");

    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);   // known to be the same in a warp
    const int lane = threadIdx.x & 31;
    const uint32_t rank = cluster_cta_rank();
    const bool leader = rank == 0;
    const int pair = blockIdx.x >> 1;
    const int pairs = gridDim.x >> 1;
    const int p_tiles = (a.p_dim + NB * BLOCK_P - 1) / (NB * BLOCK_P);

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
            mbar_init(&tail_bar[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full_bar[b], 1);
            mbar_init(&acc_empty_bar[b], 2 * EPI_WARPS / NB);
        }
        *abort_flag = 0;
        *never_flag = 0;
        fence_barrier_init();
    }
    if (warp == 1) {
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(static_cast<uint32_t>(TMEM_COLS))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    if (MODE != WGRAD && warp == 2) {
        int carry = 0;
        for (int e0 = 0; e0 < a.experts; e0 += 32) {
            const int e = e0 + lane;
            const int2 rows = e < a.experts ? group_rows(a, e) : make_int2(0, 0);
            const int n = (rows.y - rows.x + BLOCK_Q - 1) / BLOCK_Q * p_tiles;
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
    cluster_sync_all();   // barriers of both CTAs are initialised, tensor memory is allocated
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int total_tiles = MODE == WGRAD ? a.experts * p_tiles * ((a.q_dim + BLOCK_Q - 1) / BLOCK_Q) : tile_first[a.experts];

    bool timed_out = false;

    if (warp == 0) {
        // ------------------------- TMA producer (both CTAs) -------------------------
        if (lane == 0) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_p)) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_q)) : "memory");
            TileWalk<MODE, NB> walk(a, tile_first);
            int stage = 0;
            uint32_t phase = 0;
            int armed = 0;   // stages loaded and not known to be consumed (for the unwind path)
            for (int t = pair; t < total_tiles && !timed_out; t += pairs) {
                const Tile tile = walk.at(t, a);
                const int boxes = tile.boxes();
                const int p0 = tile.p0 + static_cast<int>(rank) * HALF_P;
                const int q0 = tile.q0 + static_cast<int>(rank) * tile.half();
                const uint32_t bytes = tile.nb * P_BYTES + boxes * CHUNK_BYTES;
                for (int cb = 0; cb < tile.blocks; ++cb) {
                    if (!mbar_wait_bounded_sleepy(&empty_bar[stage], phase ^ 1u, abort_flag, 40)) {
                        timed_out = true;
                        break;
                    }
                    unsigned char* p_dst = ring + stage * STAGE_BYTES;
                    unsigned char* q_dst = p_dst + NB * P_BYTES;
                    const int c0 = tile.first + cb * BLOCK_C;
                    const bool tail = MODE == WGRAD && tile.tail && cb == tile.blocks - 1;
                    uint32_t bar = cluster_addr(&full_bar[stage], 0);
                    if (leader) {
                        mbar_arrive_expect_tx(&full_bar[stage], tail ? bytes : 2 * bytes);   // both CTAs' bytes, or its own
                    } else if (tail) {
                        mbar_arrive_expect_tx(&tail_bar[stage], bytes);
                        bar = cluster_addr(&tail_bar[stage], 1);
                    }
#pragma unroll
                    for (int n = 0; n < NB; ++n) {
                        if (n >= tile.nb) break;
                        const int p = p0 + n * BLOCK_P;
                        unsigned char* dst = p_dst + n * P_BYTES;
                        if (MODE == FWD) {
                            tma_load_3d_pair(dst, &map_p, c0, p, tile.e, bar);
                        } else if (MODE == DGRAD) {
                            tma_load_3d_pair(dst, &map_p, p, c0, tile.e, bar);
                            tma_load_3d_pair(dst + CHUNK_BYTES, &map_p, p + 64, c0, tile.e, bar);
                        } else {
                            tma_load_2d_pair(dst, &map_p, p, c0, bar);
                            tma_load_2d_pair(dst + CHUNK_BYTES, &map_p, p + 64, c0, bar);
                        }
                    }
                    for (int b = 0; b < boxes; ++b) {
                        if (MODE == WGRAD) tma_load_2d_pair(q_dst + b * CHUNK_BYTES, &map_q, q0 + 64 * b, c0, bar);
                        else tma_load_2d_pair(q_dst + b * CHUNK_BYTES, &map_q, c0, q0 + 64 * b, bar);
                    }
                    armed = armed < STAGES ? armed + 1 : STAGES;
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            if (timed_out || *abort_flag) drain_pair_loads(full_bar, stage, phase, armed, STAGES, leader, never_flag);
        }
    } else if (warp == 1 && leader) {
        // ------------------------- MMA issuer -------------------------
        // The warp walks along as one (all of it zeros a wgrad tile's tail rows); one elected lane issues.
        TileWalk<MODE, NB> walk(a, tile_first);
        const uint32_t p_ring = desc_low(P_MN, smem_u32(ring)), q_ring = desc_low(Q_MN, smem_u32(ring) + NB * P_BYTES);
        int stage = 0;
        uint32_t phase = 0, tail_phase = 0;   // tail_phase: a bit per stage
        int acc = 0;                          // NB == 1: the accumulator in turn
        uint32_t acc_phase = 0;               // a bit per accumulator
        auto wait = [&](uint64_t* bar, uint32_t parity) {
            if (!__all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, abort_flag))) timed_out = true;
            return !timed_out;
        };
        Tile next{};
        if (pair < total_tiles) next = walk.at(pair, a);
        for (int t = pair; t < total_tiles && !timed_out; t += pairs) {
            const Tile tile = next;
            const uint32_t idesc = instr_desc(P_MN, Q_MN, BLOCK_P, 2 * tile.half());
            // Runs of contraction blocks.  Two lane blocks fill tensor memory, so the next tile can only start where the
            // epilogue has emptied it; therefore a tile's first and last SKEW stages go through the MMAs by lane block:
            // block 0 starts while block 1 of the previous tile is still being read, and is done while block 1 computes.
            for (int done = 0; done < tile.blocks && !timed_out;) {   // an empty group's weights have no blocks
                const int left = tile.blocks - done;
                const int chunk = NB == 2 ? tile.blocks : PROMOTE ? PROMOTE_BLOCKS : tile.blocks;
                const bool begin = done % chunk == 0;
                const int run = NB == 2 ? (begin || left <= SKEW ? min(SKEW, left) : 1) : 1;
                const bool end = run == left || (done + run) % chunk == 0;
                for (int n = 0; n < tile.nb && !timed_out; ++n) {
                    const int slot = NB == 2 ? n : acc;
                    if (begin) {
                        if (!wait(&acc_empty_bar[slot], ((acc_phase >> slot) & 1u) ^ 1u)) break;
                        acc_phase ^= 1u << slot;
                    }
                    const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(slot * BLOCK_Q);
                    for (int i = 0; i < run; ++i) {
                        const bool wraps = stage + i >= STAGES;
                        const int st = wraps ? stage + i - STAGES : stage + i;
                        const bool tail = MODE == WGRAD && tile.tail && done + i == tile.blocks - 1;
                        if (n == 0) {
                            if (!wait(&full_bar[st], wraps ? phase ^ 1u : phase)) break;
                            if (tail) {
                                zero_tail<NB>(ring + st * STAGE_BYTES, tile, lane);
                                if (!__all_sync(0xffffffffu, mbar_wait_cluster_bounded(&tail_bar[st], (tail_phase >> st) & 1u, abort_flag))) {
                                    timed_out = true;
                                    break;
                                }
                                tail_phase ^= 1u << st;
                            }
                        }
                        const int steps = tail ? (tile.tail + UMMA_K - 1) / UMMA_K : BLOCK_C / UMMA_K;
                        tc_fence_after();
                        const uint32_t p_low = p_ring + st * (STAGE_BYTES >> 4) + n * (P_BYTES >> 4);
                        const uint32_t q_low = q_ring + st * (STAGE_BYTES >> 4);
                        if (elect_one()) {
                            // 16 contraction indices on: 32 bytes inside the span (K-major), 16 rows of 128 bytes (MN-major).
                            constexpr uint32_t P_STEP = P_MN ? 128 : 2, Q_STEP = Q_MN ? 128 : 2;
                            umma_pair(d_tmem, p_low, q_low, idesc, begin && i == 0 ? 0u : 1u);
#pragma unroll
                            for (int k = 1; k < BLOCK_C / UMMA_K; ++k)
                                if (MODE != WGRAD || k < steps) umma_pair(d_tmem, p_low + P_STEP * k, q_low + Q_STEP * k, idesc, 1u);
                            if (n == tile.nb - 1) umma_commit_both(&empty_bar[st]);   // frees the stage in both CTAs
                        }
                        __syncwarp();
                    }
                    if (timed_out) break;
                    if (end) {
                        if (elect_one()) umma_commit_both(&acc_full_bar[slot]);
                        __syncwarp();
                        acc ^= 1;
                    }
                }
                stage += run;
                if (stage >= STAGES) {
                    stage -= STAGES;
                    phase ^= 1u;
                }
                if (done == 0 && t + pairs < total_tiles) next = walk.at(t + pairs, a);   // while the MMAs issued so far run
                done += run;
            }
            if (tile.blocks == 0 && t + pairs < total_tiles) next = walk.at(t + pairs, a);
        }
    } else if (warp == 1) {
        // ------------------------- the second CTA's tail stages -------------------------
        if (MODE == WGRAD) {
            TileWalk<MODE, NB> walk(a, tile_first);
            int stage = 0;
            uint32_t tail_phase = 0;
            for (int t = pair; t < total_tiles; t += pairs) {
                const Tile tile = walk.at(t, a);
                if (tile.blocks == 0) continue;
                const int at = (stage + tile.blocks - 1) % STAGES;   // stage of the last block
                stage = (stage + tile.blocks) % STAGES;
                if (!tile.tail) continue;
                if (!__all_sync(0xffffffffu, mbar_wait_bounded(&tail_bar[at], (tail_phase >> at) & 1u, abort_flag))) {
                    timed_out = true;
                    break;
                }
                __syncwarp();
                tail_phase ^= 1u << at;
                zero_tail<NB>(ring + at * STAGE_BYTES, tile, lane);
                if (lane == 0) mbar_arrive_cluster(cluster_addr(&tail_bar[at], 0));
            }
        }
    } else {
        // ------------------------- epilogue warps (both CTAs) -------------------------
        // A warp has a lane quarter of one lane block and some of its columns; four neighbours have the same columns of the
        // four quarters and move together (their waits have one outcome: barrier.red below).
        const int quarter = warp & 3, four = (warp - 2) >> 2;
        const int block = NB == 1 ? 0 : four & 1;
        const int side = NB == 1 ? four : four >> 1;
        Out* out = static_cast<Out*>(a.out);
        TileWalk<MODE, NB> walk(a, tile_first);
        int acc = 0;               // NB == 1: the accumulator in turn
        uint32_t acc_phase = 0;    // a bit per accumulator
        Tile next{};
        if (pair < total_tiles) next = walk.at(pair, a);
        for (int t = pair; t < total_tiles; t += pairs) {
            const Tile tile = next;
            if (t + pairs < total_tiles) next = walk.at(t + pairs, a);   // before the wait, not after it
            if (block >= tile.nb) continue;
            const int p_block = tile.p0 + block * BLOCK_P + static_cast<int>(rank) * HALF_P;
            const int p_warp = p_block + quarter * 32;   // first lane index
            constexpr int HELD = C_::HELD;
            constexpr int REGS = PROMOTE ? 32 : 16;   // registers per column block: fp32, or packed bf16
            // Column blocks of 32: in wgrad to bf16 a warp's come in neighbouring pairs, 128 bytes of a row.
            auto column = [&](int i) {
                return MODE == WGRAD && !PROMOTE ? 64 * (C_::SIDES * (i >> 1) + side) + 32 * (i & 1) : 32 * (C_::SIDES * i + side);
            };
            uint32_t held[HELD][REGS];
            if (MODE == WGRAD) {
#pragma unroll
                for (int i = 0; i < HELD; ++i)
#pragma unroll
                    for (int j = 0; j < REGS; ++j) held[i][j] = 0;
            }
            for (int c0 = 0; c0 < tile.blocks; c0 += PROMOTE ? PROMOTE_BLOCKS : tile.blocks) {
                const int slot = NB == 2 ? block : acc;
                const bool ready = lane != 0 || mbar_wait_bounded_sleepy(&acc_full_bar[slot], (acc_phase >> slot) & 1u, abort_flag, 40);
                if (!four_warps_all(four, ready)) {
                    timed_out = true;
                    break;
                }
                acc_phase ^= 1u << slot;
                acc ^= 1;
                tc_fence_after();
                const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(slot * BLOCK_Q);
                // The accumulator goes into registers first and is handed back before anything is stored.
#pragma unroll
                for (int i = 0; i < HELD; ++i) {
                    if (column(i) >= tile.cols) break;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {   // 16 at a time: with 32 the registers spill
                        uint32_t r[16];
                        tmem_ld_16cols(t_row + column(i) + 16 * h, r);
                        tmem_ld_wait();
                        if constexpr (PROMOTE) {
#pragma unroll
                            for (int j = 0; j < 16; ++j)
                                held[i][16 * h + j] = __float_as_uint(__uint_as_float(held[i][16 * h + j]) + __uint_as_float(r[j]));
                        } else {
#pragma unroll
                            for (int j = 0; j < 8; ++j) held[i][8 * h + j] = pack_bf16(r[2 * j], r[2 * j + 1]);
                        }
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster_relaxed(cluster_addr(&acc_empty_bar[slot], 0));
            }
            if (timed_out) break;
            if (MODE == WGRAD) {
                // A lane holds consecutive columns of one row of dW.  16 rows x 128 bytes at a time pass through the warp's
                // 2 KB of shared memory (16-byte pieces XOR-swizzled by row), so that stores write whole lines.
                constexpr int PIECE = 16 / sizeof(Out);
                unsigned char* buf = epi_smem + (warp - 2) * 2048;
#pragma unroll
                for (int i = 0; i < HELD * REGS / 32; ++i) {
                    const int col0 = column(PROMOTE ? i : 2 * i);
                    if (col0 >= tile.cols) break;
                    Out* dst = out + (static_cast<size_t>(tile.e) * a.p_dim + p_warp) * a.ldo + tile.q0 + col0;
#pragma unroll
                    for (int rows = 0; rows < 32; rows += 16) {
                        if ((lane & 16) == rows) {
#pragma unroll
                            for (int ch = 0; ch < 8; ++ch) {
                                const int i2 = PROMOTE ? i : 2 * i + (ch >> 2), j = PROMOTE ? 4 * ch : 4 * (ch & 3);
                                *reinterpret_cast<uint4*>(buf + (lane & 15) * 128 + ((ch ^ (lane & 7)) << 4)) =
                                    make_uint4(held[i2][j], held[i2][j + 1], held[i2][j + 2], held[i2][j + 3]);
                            }
                        }
                        __syncwarp();
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int at = 4 * j + (lane >> 3), ch = lane & 7, row = rows + at;
                            const uint4 v = *reinterpret_cast<const uint4*>(buf + at * 128 + ((ch ^ (at & 7)) << 4));
                            if (p_warp + row < a.p_dim && col0 + ch * PIECE < tile.cols)
                                *reinterpret_cast<uint4*>(dst + static_cast<size_t>(row) * a.ldo + ch * PIECE) = v;
                        }
                        __syncwarp();
                    }
                }
            } else {
                // A lane holds one weight row's products with consecutive activation rows; out has the weight dimension
                // contiguous.  16 activation rows of the four warps' 128 lanes at a time are transposed through their 4 KB
                // of shared memory and stored as rows of 256 bytes.
                uint16_t* buf = reinterpret_cast<uint16_t*>(epi_smem + four * 4096);
                const int thread = quarter * 32 + lane;
#pragma unroll
                for (int i = 0; i < HELD; ++i) {
                    const int col0 = column(i);
                    if (col0 >= tile.cols) break;
                    Out* dst = out + static_cast<size_t>(tile.q0 + col0) * a.ldo + p_block;
#pragma unroll
                    for (int rows = 0; rows < 32; rows += 16) {
                        if (col0 + rows >= tile.cols) break;
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            buf[(2 * j) * 128 + thread] = static_cast<uint16_t>(held[i][rows / 2 + j]);
                            buf[(2 * j + 1) * 128 + thread] = static_cast<uint16_t>(held[i][rows / 2 + j] >> 16);
                        }
                        four_warps_sync(four);
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const int at = 8 * j + (thread >> 4), col = (thread & 15) * 8;
                            const uint4 v = *reinterpret_cast<const uint4*>(buf + at * 128 + col);
                            if (col0 + rows + at < tile.cols && p_block + col < a.p_dim)
                                *reinterpret_cast<uint4*>(dst + static_cast<size_t>(rows + at) * a.ldo + col) = v;
                        }
                        four_warps_sync(four);
                    }
                }
            }
        }
    }

    if (timed_out) {
        *abort_flag = 1;
        raise_device_status(DEV_GROUPED_PIPE_TIMEOUT);
    }
    __syncwarp();
    tc_fence_before();
    cluster_sync_all();   // nobody leaves while the other CTA may still read its operands or signal its barriers
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base),
                     "r"(static_cast<uint32_t>(TMEM_COLS))
                     : "memory");
    }
}

// ---- host side ---------------------------------------------------------------------------------------------------

// Rows of activations: width contiguous, 64 x 64 boxes.
int rows_map(CUtensorMap* out, const void* ptr, long long rows, int width, long long ld) {
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(width), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld) * 2};
    const cuuint32_t box[2] = {64, 64};
    return encode_tensor_map(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, ptr, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Weights [experts][n][k]: boxes of 64 k and box_n rows of one expert.
int weights_map(CUtensorMap* out, const void* ptr, int experts, int n, int k, int box_n) {
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(k), static_cast<cuuint64_t>(n), static_cast<cuuint64_t>(experts)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(k) * 2, static_cast<cuuint64_t>(n) * k * 2};
    const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_n), 1};
    return encode_tensor_map(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, ptr, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int MODE, typename Out, int NB>
int launch_grouped(const GroupedArgs& a, long long most_tiles, const CUtensorMap& map_p, const CUtensorMap& map_q, cudaStream_t s) {
    auto kern = grouped_gemm_kernel<MODE, Out, NB>;
    static std::mutex mu;
    static int pair_count[64] = {};
    int dev = 0, capacity = 0;
    PRISM_CUDA_TRY(cudaGetDevice(&dev));
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.blockDim = dim3(gg::THREADS);
    cfg.dynamicSmemBytes = gg::smem_bytes(MODE, gg::MAX_EXPERTS);
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    {
        std::lock_guard<std::mutex> lk(mu);
        const bool cacheable = dev >= 0 && dev < 64;
        if (!cacheable || !pair_count[dev]) {
            int sms = 0;
            PRISM_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, gg::smem_bytes(MODE, gg::MAX_EXPERTS)));
            PRISM_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
            cfg.gridDim = dim3(static_cast<unsigned>(sms / 2 * 2));
            PRISM_CUDA_TRY(cudaOccupancyMaxActiveClusters(&capacity, kern, &cfg));
            if (capacity < 1) return set_error(PRISM_B200_ERR_CUDA, "grouped_gemm_bf16: no 2-CTA cluster fits on this device");
            if (cacheable) pair_count[dev] = capacity;
        } else {
            capacity = pair_count[dev];
        }
    }
    const int pairs = most_tiles < capacity ? static_cast<int>(most_tiles) : capacity;
    cfg.gridDim = dim3(static_cast<unsigned>(2 * pairs));
    cfg.dynamicSmemBytes = gg::smem_bytes(MODE, a.experts);
    cfg.stream = s;
    PRISM_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, a, map_p, map_q));
    count_launch();
    return PRISM_B200_OK;
}

long long tiles_of(int p_dim, int blocks) { return (p_dim + blocks * gg::BLOCK_P - 1) / (blocks * gg::BLOCK_P); }

// One or two lane blocks per tile, by the rounds of tiles that the 74 CTA pairs make, with a tile of two at 1.55 of a tile
// of one (2 x 754/1024 to 2 x 795/989 at the sizes above).  Over 36 drawn problems (1500 to 30000 rows, 4 to 60 experts,
// matrices of 400 to 5600) the choice is 1.3% behind the better of the two on average and 25% at worst (2637 rows, 9
// experts, 1224 x 1560: 30.7 us with two, 24.6 with one); always one would be 8% behind, always two 4%.
bool two_blocks(int p_dim, long long q_tiles) {
    constexpr long long PAIRS = 74;
    const long long t1 = tiles_of(p_dim, 1) * q_tiles, t2 = tiles_of(p_dim, 2) * q_tiles;
    return (t2 + PAIRS - 1) / PAIRS * 1.55 <= static_cast<double>((t1 + PAIRS - 1) / PAIRS);
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
    if (rows > 1 << 30 || n > 1 << 30 || k > 1 << 30 || tiles > 0x3fffffffLL || wtiles > 0x3fffffffLL) return set_error(PRISM_B200_ERR_TOO_LARGE, "%s: a size above 2^30 or too many tiles", fn);
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
    if (int rc = weights_map(&map_p, w, experts, n, k, MODE == gg::FWD ? gg::HALF_P : 64)) return rc;
    if (int rc = rows_map(&map_q, in, rows, c_dim, ld_in)) return rc;
    const GroupedArgs a{offsets, experts, rows, p_dim, 0, c_dim, out, ld_out};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const long long groups = experts < rows ? experts : rows, q_most = rows / gg::BLOCK_Q + groups;
    const long long q_tiles = (rows + gg::BLOCK_Q / 2 * groups + gg::BLOCK_Q - 1) / gg::BLOCK_Q;   // half a tile per group is empty
    // Groups of few rows only stream their matrices: one block, with twice as many tiles to spread over the SMs.
    if (rows >= 128LL * experts && two_blocks(p_dim, q_tiles))
        return launch_grouped<MODE, __nv_bfloat16, 2>(a, q_most * tiles_of(p_dim, 2), map_p, map_q, s);
    return launch_grouped<MODE, __nv_bfloat16, 1>(a, q_most * tiles_of(p_dim, 1), map_p, map_q, s);
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
    const long long q_tiles = static_cast<long long>(experts) * ((k + gg::BLOCK_Q - 1) / gg::BLOCK_Q);
    if (out_dtype == PRISM_B200_F32) return launch_grouped<gg::WGRAD, float, 1>(a, q_tiles * tiles_of(n, 1), map_p, map_q, s);
    if (two_blocks(n, q_tiles)) return launch_grouped<gg::WGRAD, __nv_bfloat16, 2>(a, q_tiles * tiles_of(n, 2), map_p, map_q, s);
    return launch_grouped<gg::WGRAD, __nv_bfloat16, 1>(a, q_tiles * tiles_of(n, 1), map_p, map_q, s);
}
