// Routing of rows to experts: the choice of k experts for each token and the order of the rows that it makes
// (prism_b200_route_topk), its gradient, and the copies between token order and expert order (gather, combine and
// combine's gradient).  The grouped products (grouped_gemm.cu, gemv_w4.cu) work on rows in this order.
//
// Expert order: row r of expert e lies in [offsets[e], offsets[e + 1]), and within an expert the rows follow their
// tokens' order, so nothing depends on which block or warp came first.  No kernel here waits for another block: the
// order is made in two launches (counts per block, then positions) and nothing is added up by floating-point atomics.
#include "common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

namespace prism_b200 {
namespace {

namespace rt {
constexpr int MAX_EXPERTS = 1024;
constexpr int MAX_CHOICES = 32;    // lane j of a token's warp holds its choice j
constexpr int CHUNK = 128;         // tokens whose choices a block ranks at a time
constexpr int WORDS = CHUNK / 32;
constexpr int ONE_BLOCK = 64;      // tokens up to which one block makes the whole order: 128 (of 128 experts, 8 choices) take 12.8 us, 7.3 in two launches
constexpr int MAX_BLOCKS = 148;    // one block of 32 warps per SM
constexpr unsigned FULL = 0xffffffffu;
}  // namespace rt

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// Unsigned integers in the order of the floats.  0 stands for "not to be chosen": -inf, NaN, or no such expert.
// The two zeros compare equal as floats and so get one key.
__device__ __forceinline__ uint32_t order_key(float v) {
    if (!(v > -INFINITY)) return 0u;
    const uint32_t b = v == 0.f ? 0u : __float_as_uint(v);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t key) {
    return __uint_as_float((key & 0x80000000u) ? (key ^ 0x80000000u) : ~key);
}

// The same for 16-bit types, from the bits: the order in the upper half, the lowest expert first among equals in the lower
// half, so that all keys of a token differ and one maximum decides.
template <typename T> __device__ __forceinline__ uint32_t packed_key(T v, int expert) {
    const uint32_t b = *reinterpret_cast<const uint16_t*>(&v);
    constexpr uint32_t INF = sizeof(T) == 2 && std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
    if ((b & 0x7FFFu) > INF || b == (0x8000u | INF)) return 0u;
    const uint32_t order = b == 0x8000u ? 0x8000u : (b & 0x8000u) ? (~b & 0xFFFFu) : (b | 0x8000u);
    return (order << 16) | (0xFFFFu ^ static_cast<uint32_t>(expert));
}
template <typename T> __device__ __forceinline__ float packed_value(uint32_t key) {
    const uint32_t order = key >> 16;
    const uint16_t b = static_cast<uint16_t>((order & 0x8000u) ? (order ^ 0x8000u) : ~order);
    return to_f32(*reinterpret_cast<const T*>(&b));
}

// The k choices of one token by one warp (row: its logits of experts lane, lane + 32, ...): lane j < k returns its
// choice's expert (-1: none) and logit, every lane the largest logit and, with `all`, this lane's share of the sum of
// exp(logit - largest) over all experts.
// A round takes the largest key of the lanes' best (redux.sync); the lane that has it goes on to its next.  Lanes with up
// to eight keys sort them first, so that this is a shift; others look through their keys again.
template <typename T, int EPL>
__device__ __forceinline__ void choose(const T (&row)[EPL], int experts, int k, bool all, int lane, int& id, float& logit, float& largest,
                                       float& sum) {
    constexpr bool SORTED = EPL <= 8;
    uint32_t key[EPL];
    int index[EPL];   // 32-bit types only
    id = -1;
    logit = largest = sum = 0.f;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < EPL; ++i) {
            const int e = i * 32 + lane;
            key[i] = e < experts ? packed_key(row[i], e) : 0u;
        }
        if constexpr (SORTED) {
#pragma unroll
            for (int n = EPL - 1; n > 0; --n)
#pragma unroll
                for (int i = 0; i < n; ++i) {
                    const uint32_t hi = max(key[i], key[i + 1]), lo = min(key[i], key[i + 1]);
                    key[i] = hi;
                    key[i + 1] = lo;
                }
        }
        uint32_t best = key[0];
#pragma unroll
        for (int i = 1; i < EPL; ++i) best = max(best, key[i]);
        uint32_t top = __reduce_max_sync(rt::FULL, best), mine = 0;
        if (!top) return;
        largest = packed_value<T>(top);
        if (all) {
#pragma unroll
            for (int i = 0; i < EPL; ++i) sum += key[i] ? expf(packed_value<T>(key[i]) - largest) : 0.f;
        }
        for (int j = 0;; ) {
            if (lane == j) mine = top;
            if (++j == k) break;
            if constexpr (SORTED) {
                if (key[0] == top) {
#pragma unroll
                    for (int i = 0; i + 1 < EPL; ++i) key[i] = key[i + 1];
                    key[EPL - 1] = 0;
                }
                best = key[0];
            } else if (best == top) {
                best = 0;
#pragma unroll
                for (int i = 0; i < EPL; ++i) best = max(best, key[i] < top ? key[i] : 0u);
            }
            top = __reduce_max_sync(rt::FULL, best);
            if (!top) break;
        }
        if (mine) {
            id = static_cast<int>(0xFFFFu ^ (mine & 0xFFFFu));
            logit = packed_value<T>(mine);
        }
    } else {
#pragma unroll
        for (int i = 0; i < EPL; ++i) {
            const int e = i * 32 + lane;
            key[i] = e < experts ? order_key(to_f32(row[i])) : 0u;
            index[i] = e;
        }
        if constexpr (SORTED) {   // stable: a lane's experts ascend, equal keys stay in that order
#pragma unroll
            for (int n = EPL - 1; n > 0; --n)
#pragma unroll
                for (int i = 0; i < n; ++i) {
                    const bool swap = key[i + 1] > key[i];
                    const uint32_t a = key[i], b = key[i + 1];
                    const int x = index[i], y = index[i + 1];
                    key[i] = swap ? b : a;
                    key[i + 1] = swap ? a : b;
                    index[i] = swap ? y : x;
                    index[i + 1] = swap ? x : y;
                }
        }
        uint32_t best = key[0];
        int at = index[0];
#pragma unroll
        for (int i = 1; i < EPL; ++i)
            if (key[i] > best) best = key[i], at = index[i];
        uint32_t top = __reduce_max_sync(rt::FULL, best), mine = 0;
        if (!top) return;
        largest = key_value(top);
        if (all) {
#pragma unroll
            for (int i = 0; i < EPL; ++i) sum += key[i] ? expf(key_value(key[i]) - largest) : 0.f;
        }
        for (int j = 0;; ) {
            const int win = __reduce_min_sync(rt::FULL, best == top ? at : 0x7fffffff);
            if (lane == j) id = win, mine = top;
            if (++j == k) break;
            if ((win & 31) == lane) {
                if constexpr (SORTED) {
#pragma unroll
                    for (int i = 0; i + 1 < EPL; ++i) key[i] = key[i + 1], index[i] = index[i + 1];
                    key[EPL - 1] = 0;
                    best = key[0];
                    at = index[0];
                } else {
                    best = 0;
#pragma unroll
                    for (int i = 0; i < EPL; ++i) {
                        if (i * 32 + lane == win) key[i] = 0;
                        if (key[i] > best) best = key[i], at = i * 32 + lane;
                    }
                }
            }
            top = __reduce_max_sync(rt::FULL, best);
            if (!top) break;
        }
        if (mine) logit = key_value(mine);
    }
}

// ---- k <= 8 choices by eight lanes per token (16-bit types, rows of whole 16-byte vectors) ----
// A lane sorts the eight keys of a vector by a network of 19 exchanges and merges them into its best eight (8 maxima, 12
// exchanges), and three exchanges between lanes leave the token's best eight in all of them.  What bounds both this and
// the rounds of choose() is issue slots, and this takes fewer: both launches of 16384 tokens x 128 experts 9.7 us against
// 14.1 for 8 choices, 8.8 against 11.4 for 2; 65536 x 256, 8 choices 32 against 55; 64 x 128 4.5 against 6.7.  (32-bit
// logits would need keys of 64 bits, whose exchange is six instructions instead of two; choose() serves them.)

__device__ __forceinline__ void exchange(uint32_t& a, uint32_t& b) {
    const uint32_t hi = max(a, b), lo = min(a, b);
    a = hi;
    b = lo;
}
__device__ __forceinline__ void sort8(uint32_t (&v)[8]) {   // descending
    exchange(v[0], v[2]); exchange(v[1], v[3]); exchange(v[4], v[6]); exchange(v[5], v[7]);
    exchange(v[0], v[4]); exchange(v[1], v[5]); exchange(v[2], v[6]); exchange(v[3], v[7]);
    exchange(v[0], v[1]); exchange(v[2], v[3]); exchange(v[4], v[5]); exchange(v[6], v[7]);
    exchange(v[2], v[4]); exchange(v[3], v[5]);
    exchange(v[1], v[4]); exchange(v[3], v[6]);
    exchange(v[1], v[2]); exchange(v[3], v[4]); exchange(v[5], v[6]);
}
// The eight largest of two descending lists, descending: the maxima of one list and the other reversed are those eight, and
// rise at most once after falling, which three rounds of exchanges sort.
__device__ __forceinline__ void best8(uint32_t (&a)[8], const uint32_t (&b)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = max(a[i], b[7 - i]);
#pragma unroll
    for (int d = 4; d; d >>= 1)
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (!(i & d)) exchange(a[i], a[i + d]);
}

template <typename T> struct Pair16;
template <> struct Pair16<__nv_bfloat16> {
    static constexpr uint32_t LOWEST = 0xFF80FF80u;   // -inf, twice
    static __device__ __forceinline__ uint32_t plain(uint32_t w) {
        const __nv_bfloat162 v = *reinterpret_cast<const __nv_bfloat162*>(&w);
        const uint32_t low = LOWEST, zero = 0u;
        const __nv_bfloat162 r = __hmax2(__hadd2(v, *reinterpret_cast<const __nv_bfloat162*>(&zero)), *reinterpret_cast<const __nv_bfloat162*>(&low));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
};
template <> struct Pair16<__half> {
    static constexpr uint32_t LOWEST = 0xFC00FC00u;
    static __device__ __forceinline__ uint32_t plain(uint32_t w) {
        const __half2 v = *reinterpret_cast<const __half2*>(&w);
        const uint32_t low = LOWEST, zero = 0u;
        const __half2 r = __hmax2(__hadd2(v, *reinterpret_cast<const __half2*>(&zero)), *reinterpret_cast<const __half2*>(&low));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
};

// Lane `sub` of a token's eight returns choice `sub` (-1: none, or sub >= k), every lane the largest logit and the sum of
// exp(logit - largest) over the chosen, or over all with `all`.  Plain values: -0 became 0 (x + 0) and NaN -inf (maximum).
// A key is the value's order (bits flipped so that unsigned integers compare alike) over 0xFFFF - expert.
template <typename T, int EPL>
__device__ __forceinline__ void choose8(const T* row, int experts, int k, bool all, int sub, int& id, float& mine, float& sum) {
    constexpr int VECTORS = (EPL + 1) / 2;
    constexpr uint32_t NONE = (Pair16<T>::LOWEST & 0xFFFFu) ^ 0xFFFFu;   // the order of -inf
    uint32_t best[8];
    auto load = [&](int v) {
        const int at = (v * 8 + sub) * 8;
        uint4 w = make_uint4(Pair16<T>::LOWEST, Pair16<T>::LOWEST, Pair16<T>::LOWEST, Pair16<T>::LOWEST);
        if (at < experts) w = *reinterpret_cast<const uint4*>(row + at);
        return w;
    };
#pragma unroll(VECTORS < 4 ? VECTORS : 4)
    for (int v = 0; v < VECTORS; ++v) {
        const uint4 raw = load(v);
        const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
        uint32_t key[8];
        const uint32_t low = 0xFFFFu - (v * 8 + sub) * 8;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = Pair16<T>::plain(words[i]);
            uint32_t sign;   // 0xFFFF for each negative half
            asm("prmt.b32 %0, %1, 0, 0xBB99;" : "=r"(sign) : "r"(w));
            const uint32_t order = w ^ (sign | 0x80008000u);
            key[2 * i] = __byte_perm(low - 2 * i, order, 0x5410);
            key[2 * i + 1] = __byte_perm(low - 2 * i - 1, order, 0x7610);
        }
        sort8(key);
        if (v == 0) {
#pragma unroll
            for (int i = 0; i < 8; ++i) best[i] = key[i];
        } else {
            best8(best, key);
        }
    }
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) {
        uint32_t other[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) other[i] = __shfl_xor_sync(rt::FULL, best[i], d);
        best8(best, other);
    }
    uint32_t key = best[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) key = sub == i ? best[i] : key;
    const float largest = packed_value<T>(best[0]);
    id = sub < k && (key >> 16) > NONE ? static_cast<int>(0xFFFFu - (key & 0xFFFFu)) : -1;
    mine = id >= 0 ? expf(packed_value<T>(key) - largest) : 0.f;
    sum = mine;
    if (all) {
        sum = 0.f;
#pragma unroll 1
        for (int v = 0; v < VECTORS; ++v) {
            const uint4 raw = load(v);
            const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
            float part[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t w = Pair16<T>::plain(words[i]);
                const T* pair = reinterpret_cast<const T*>(&w);
                part[i] = expf(to_f32(pair[0]) - largest) + expf(to_f32(pair[1]) - largest);
            }
            sum += (part[0] + part[1]) + (part[2] + part[3]);   // 22 additions deep at 1024 experts
        }
    }
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) sum += __shfl_xor_sync(rt::FULL, sum, d);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(rt::FULL, v, d);
    return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v = fmaxf(v, __shfl_xor_sync(rt::FULL, v, d));
    return v;
}

struct RouteArgs {
    const void* logits;
    long long ld;
    int tokens, experts, k, renorm, tokens_per_block;
    int* ids;
    float* weights;
    int* pos;
    int* order;
    int* offsets;
    void* counts;   // [experts][blocks], only with more than one block: 16 bits each (rows of an even number) while that holds
                    // a block's tokens, else 32
    int narrow;
    int eights;     // choose8 instead of choose
};

// Exclusive prefix sums of EPL * 32 counts by one warp: base[e] = first + sum of count[e'], e' < e; returns the total.
template <int EPL>
__device__ __forceinline__ int warp_exclusive_scan(const int* count, int* base, int lane) {
    int v[EPL], carry = 0;
#pragma unroll
    for (int i = 0; i < EPL; ++i) v[i] = count[i * 32 + lane];
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
        int incl = v[i];
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int up = __shfl_up_sync(rt::FULL, incl, d);
            if (lane >= d) incl += up;
        }
        base[i * 32 + lane] = carry + incl - v[i];
        carry += __shfl_sync(rt::FULL, incl, 31);
    }
    return carry;
}

// One warp per token (choose).  Then the block ranks its choices: a token chooses an expert at most once, so a bit per
// (expert, token) says everything, and the rank of a choice is a popcount of the bits of earlier tokens.  With one block
// (grid 1, tokens <= ONE_BLOCK) the order is complete here; otherwise the ranks are relative to the block and
// route_place_kernel adds the rest.
template <typename T, int EPL>
__global__ void __launch_bounds__(1024, 1) route_choose_kernel(RouteArgs a) {
    using namespace rt;
    __shared__ uint32_t mask[EPL * 32][WORDS];
    __shared__ int running[EPL * 32], base[EPL * 32];
    __shared__ int16_t chosen[CHUNK * MAX_CHOICES];
    __shared__ int total;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int k = a.k;
    const bool single = gridDim.x == 1;
    const int first = blockIdx.x * a.tokens_per_block;
    const int last = min(a.tokens, first + a.tokens_per_block);
    for (int e = threadIdx.x; e < EPL * 32; e += blockDim.x) {
        running[e] = 0;
#pragma unroll
        for (int w = 0; w < WORDS; ++w) mask[e][w] = 0;
    }
    __syncthreads();
    for (int c0 = first; c0 < last; c0 += CHUNK) {
        const int n = min(CHUNK, last - c0);
        auto keep = [&](int tt, int j, int id, float weight) {
            const size_t at = (static_cast<size_t>(c0) + tt) * k + j;
            a.ids[at] = id;
            a.weights[at] = weight;
            chosen[tt * MAX_CHOICES + j] = static_cast<int16_t>(id);
            if (id >= 0) atomicOr(&mask[id][tt >> 5], 1u << (tt & 31));
        };
        if (sizeof(T) == 2 && a.eights) {
            if constexpr (sizeof(T) == 2) {
                const int sub = lane & 7;
                for (int t4 = warp * 4; t4 < n; t4 += warps * 4) {   // four tokens a warp
                    const int tt = t4 + (lane >> 3);
                    int id;
                    float mine, sum;
                    choose8<T, EPL>(static_cast<const T*>(a.logits) + (static_cast<size_t>(c0) + min(tt, n - 1)) * a.ld, a.experts, k,
                                    !a.renorm, sub, id, mine, sum);
                    if (tt < n && sub < k) keep(tt, sub, id, id >= 0 ? mine / sum : 0.f);
                }
            }
        } else {
            T row[EPL], next[EPL];   // the next token's logits are on their way while this one's choices are made
            auto load = [&](int tt) {
                const T* from = static_cast<const T*>(a.logits) + (static_cast<size_t>(c0) + tt) * a.ld;
#pragma unroll
                for (int i = 0; i < EPL; ++i)
                    if (i * 32 + lane < a.experts) next[i] = from[i * 32 + lane];
            };
            if (warp < n) load(warp);
            for (int tt = warp; tt < n; tt += warps) {
#pragma unroll
                for (int i = 0; i < EPL; ++i) row[i] = next[i];
                if (tt + warps < n) load(tt + warps);
                int id;
                float logit, largest, sum;
                choose<T, EPL>(row, a.experts, k, !a.renorm, lane, id, logit, largest, sum);
                const float mine = id >= 0 ? expf(logit - largest) : 0.f;
                sum = warp_sum(a.renorm ? mine : sum);
                if (lane < k) keep(tt, lane, id, id >= 0 ? mine / sum : 0.f);
            }
        }
        __syncthreads();
        for (int e = threadIdx.x; e < EPL * 32; e += blockDim.x) {
            int c = 0;
#pragma unroll
            for (int w = 0; w < WORDS; ++w) c += __popc(mask[e][w]);
            base[e] = running[e];
            running[e] += c;
        }
        __syncthreads();
        if (single) {
            if (warp == 0) {
                const int sum = warp_exclusive_scan<EPL>(running, base, lane);
                for (int e = lane; e < a.experts; e += 32) a.offsets[e] = base[e];
                if (lane == 0) total = a.offsets[a.experts] = sum;
            }
            __syncthreads();
        }
        for (int i = threadIdx.x; i < n * k; i += blockDim.x) {
            const int tt = i / k, j = i - tt * k;
            const int id = chosen[tt * MAX_CHOICES + j];
            int p = -1;
            if (id >= 0) {
                p = base[id] + __popc(mask[id][tt >> 5] & ((1u << (tt & 31)) - 1u));
                for (int w = 0; w < (tt >> 5); ++w) p += __popc(mask[id][w]);
            }
            const size_t at = static_cast<size_t>(c0) * k + i;
            a.pos[at] = p;
            if (single) {
                if (id >= 0) a.order[p] = static_cast<int>(at);
                if (static_cast<int>(at) >= total) a.order[at] = -1;
            }
        }
        __syncthreads();
        for (int e = threadIdx.x; e < EPL * 32; e += blockDim.x) {
#pragma unroll
            for (int w = 0; w < WORDS; ++w) mask[e][w] = 0;
        }
        __syncthreads();
    }
    if (!single)
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (!single) {
        const int pitch = (gridDim.x + 1) & ~1;
        for (int e = threadIdx.x; e < a.experts; e += blockDim.x) {
            if (a.narrow) static_cast<uint16_t*>(a.counts)[e * pitch + blockIdx.x] = static_cast<uint16_t>(running[e]);
            else static_cast<int*>(a.counts)[e * gridDim.x + blockIdx.x] = running[e];
        }
    }
}

// Second launch with the first one's grid: every block adds up the counts of all blocks (offsets) and of the blocks
// before it (where its own rows begin), then turns its ranks into positions.  The counts are read once per block from
// L2 (148 x experts x 2 bytes), which costs less than a third launch.  They lie by expert, so that a warp reads and adds up
// a row: with rows by block, as they are made, the sums take atomics in shared memory (both launches 14.7 us for 16384
// tokens x 128 experts, 14.2 so).
template <int EPL>
__global__ void __launch_bounds__(1024, 1) route_place_kernel(RouteArgs a) {
    constexpr int EP = EPL * 32;
    __shared__ int all[EP], before[EP], base[EP];
    __shared__ int total;
    const int lane = threadIdx.x & 31;
    asm volatile("griddepcontrol.wait;" ::: "memory");   // launched while the first kernel still runs
    const int first = blockIdx.x * a.tokens_per_block;
    const int last = min(a.tokens, first + a.tokens_per_block);
    const int begin = first * a.k + threadIdx.x, end = last * a.k;
    int id = begin < end ? a.ids[begin] : -1, rank = begin < end ? a.pos[begin] : 0;   // before the counts: one latency for both
    // A warp adds up an expert's counts, up to eight experts in flight.
    const int blocks = gridDim.x, here = blockIdx.x, warp = threadIdx.x >> 5;
    constexpr int AT_ONCE = EPL < 8 ? EPL : 8;
#pragma unroll 1
    for (int e0 = warp; e0 < EP; e0 += AT_ONCE * 32) {
        int sum[AT_ONCE], pre[AT_ONCE];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            const int e = e0 + i * 32;
            sum[i] = pre[i] = 0;
            if (e >= a.experts) continue;
            if (a.narrow) {
                const int words = (blocks + 1) / 2;
                const uint32_t* row = static_cast<const uint32_t*>(a.counts) + e * words;
#pragma unroll
                for (int n = 0; n < (rt::MAX_BLOCKS / 2 + 31) / 32; ++n) {
                    const int w = n * 32 + lane, b = 2 * w;
                    const uint32_t v = w < words ? row[w] : 0u;
                    const int lo = v & 0xFFFFu, hi = b + 1 < blocks ? v >> 16 : 0u;   // an odd row's last half is not written
                    sum[i] += lo + hi;
                    pre[i] += (b < here ? lo : 0) + (b + 1 < here ? hi : 0);
                }
            } else {
                const int* row = static_cast<const int*>(a.counts) + e * blocks;
                for (int b = lane; b < blocks; b += 32) {
                    const int v = row[b];
                    sum[i] += v;
                    pre[i] += b < here ? v : 0;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            const int s = __reduce_add_sync(rt::FULL, sum[i]), p = __reduce_add_sync(rt::FULL, pre[i]);
            if (lane == 0) all[e0 + i * 32] = s, before[e0 + i * 32] = p;
        }
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        const int sum = warp_exclusive_scan<EPL>(all, base, lane);
        if (blockIdx.x == 0) {
            for (int e = lane; e < a.experts; e += 32) a.offsets[e] = base[e];
            if (lane == 0) a.offsets[a.experts] = sum;
        }
        if (lane == 0) total = sum;
    }
    __syncthreads();
    for (int i = begin; i < end;) {
        if (id >= 0) {
            const int p = base[id] + before[id] + rank;
            a.pos[i] = p;
            a.order[p] = i;
        }
        if (i >= total) a.order[i] = -1;
        i += blockDim.x;
        if (i < end) id = a.ids[i], rank = a.pos[i];
    }
}

// dl = p * (g - mean) with mean = sum of g * w over the chosen.  renorm: p is w on the chosen and 0 elsewhere, and the
// logits are not read.  Otherwise p is the softmax over all logits, computed again here (its sum was not kept).
// One warp per token; the row is first written as if nothing was chosen, then the chosen places are written over.
template <typename T, int EPL>
__global__ void __launch_bounds__(256) route_grad_kernel(const T* logits, long long ld, int tokens, int experts, int k,
                                                         int renorm, const int* ids, const float* weights,
                                                         const float* dweights, T* out) {
    const int lane = threadIdx.x & 31;
    const size_t t = static_cast<size_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    if (t >= static_cast<size_t>(tokens)) return;
    int id = -1;
    float w = 0.f, g = 0.f;
    if (lane < k) {
        id = ids[t * k + lane];
        if (id >= experts) id = -1;
        if (id >= 0) w = weights[t * k + lane], g = dweights[t * k + lane];
    }
    const float mean = warp_sum(id >= 0 ? g * w : 0.f);
    T* row = out + t * experts;
    float p = w;
    if (renorm) {
        for (int e = lane; e < experts; e += 32) row[e] = from_f32<T>(0.f);
    } else {
        const T* in = logits + t * ld;
        float v[EPL];
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < EPL; ++i) {
            const int e = i * 32 + lane;
            v[i] = e < experts ? to_f32(in[e]) : -INFINITY;
            top = fmaxf(top, v[i]);   // a NaN (never chosen) does not enter
        }
        top = warp_max(top);
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < EPL; ++i) {
            v[i] = v[i] > -INFINITY ? expf(v[i] - top) : 0.f;
            sum += v[i];
        }
        const float scale = 1.f / warp_sum(sum);
        const bool some = top > -INFINITY;   // a row without an open expert has no gradient
#pragma unroll
        for (int i = 0; i < EPL; ++i) {
            const int e = i * 32 + lane;
            if (e < experts) row[e] = from_f32<T>(v[i] != 0.f ? v[i] * scale * -mean : 0.f);
        }
        p = id >= 0 && some ? expf(to_f32(in[id]) - top) * scale : 0.f;
    }
    __syncwarp();
    if (id >= 0) row[id] = from_f32<T>(p * (g - mean));
}

// ---- copies between token order and expert order --------------------------------------------------------------
// Memory-bound: every source row is read once and every destination row written once.  threadIdx.x walks a row in
// vectors, threadIdx.y the tokens of a block, blockIdx.y the pieces of a long row.

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
    T v[V];
};

template <int BYTES> struct RawOf;
template <> struct RawOf<16> { using type = uint4; };
template <> struct RawOf<8> { using type = uint2; };
template <> struct RawOf<4> { using type = unsigned; };
template <> struct RawOf<2> { using type = unsigned short; };

// Rows pass through once: loads and stores that leave the caches to others.
template <typename W> __device__ __forceinline__ W load_once(const void* p) {
    using Raw = typename RawOf<sizeof(W)>::type;
    const Raw r = sizeof(W) < 8 ? __ldca(static_cast<const Raw*>(p)) : __ldcs(static_cast<const Raw*>(p));   // small pieces share sectors
    return *reinterpret_cast<const W*>(&r);
}
template <typename W> __device__ __forceinline__ void store_once(void* p, const W& v) {
    using Raw = typename RawOf<sizeof(W)>::type;
    if (sizeof(W) < 8) *static_cast<Raw*>(p) = *reinterpret_cast<const Raw*>(&v);
    else __stcs(static_cast<Raw*>(p), *reinterpret_cast<const Raw*>(&v));
}

// out[pos[t, j]] = x[t]; U: raw unit of the copy.
template <typename U>
__global__ void __launch_bounds__(256) route_gather_kernel(const U* __restrict__ x, long long ldx, int tokens, int k, int units,
                                                           const int* __restrict__ pos, long long rows, U* __restrict__ out,
                                                           long long ldo) {
    const size_t t = static_cast<size_t>(blockIdx.x) * blockDim.y + threadIdx.y;
    if (t >= static_cast<size_t>(tokens)) return;
    const U* src = x + t * ldx;
    const int* p = pos + t * k;
    for (int c = blockIdx.y * blockDim.x * 2 + threadIdx.x; c < units; c += gridDim.y * blockDim.x * 2) {
        const int c2 = c + blockDim.x;
        const U v = __ldcs(src + c);
        const U v2 = c2 < units ? __ldcs(src + c2) : v;
        for (int j = 0; j < k; ++j) {
            const int r = p[j];
            if (r < 0 || r >= rows) continue;
            U* dst = out + static_cast<size_t>(r) * ldo;
            __stcs(dst + c, v);
            if (c2 < units) __stcs(dst + c2, v2);
        }
    }
}

// out[t] = sum over j of w[t, j] * y[pos[t, j]], added up in fp32 in the order of j and rounded once.  KB rows in flight.
template <typename T, int V, int KB>
__global__ void __launch_bounds__(256, 4) route_combine_kernel(const T* __restrict__ y, long long ldy, long long rows, int tokens, int k,
                                                               int units, const int* __restrict__ pos,
                                                               const float* __restrict__ weights, T* __restrict__ out, long long ldo) {
    using W = Vec<T, V>;
    const size_t t = static_cast<size_t>(blockIdx.x) * blockDim.y + threadIdx.y;
    if (t >= static_cast<size_t>(tokens)) return;
    const int* p = pos + t * k;
    const float* wt = weights ? weights + t * k : nullptr;
    constexpr int U = V >= 4 ? 1 : 4;   // vectors of a row per thread: narrow ones share the reading of positions and weights
    const int step = blockDim.x;
    for (int c = blockIdx.y * step * U + threadIdx.x; c < units; c += gridDim.y * step * U) {
        float acc[U][V];
#pragma unroll
        for (int n = 0; n < U; ++n)
#pragma unroll
            for (int i = 0; i < V; ++i) acc[n][i] = 0.f;
        for (int j0 = 0; j0 < k; j0 += KB) {
            int r[KB];
            W v[KB][U];
#pragma unroll
            for (int u = 0; u < KB; ++u) {
                r[u] = j0 + u < k ? p[j0 + u] : -1;
                if (r[u] >= rows) r[u] = -1;
            }
#pragma unroll
            for (int u = 0; u < KB; ++u)
#pragma unroll
                for (int n = 0; n < U; ++n)
                    if (r[u] >= 0 && c + n * step < units)
                        v[u][n] = load_once<W>(y + static_cast<size_t>(r[u]) * ldy + static_cast<size_t>(c + n * step) * V);
#pragma unroll
            for (int u = 0; u < KB; ++u) {
                if (r[u] < 0) continue;
                const float w = wt ? wt[j0 + u] : 1.f;
#pragma unroll
                for (int n = 0; n < U; ++n)
#pragma unroll
                    for (int i = 0; i < V; ++i) acc[n][i] = fmaf(w, to_f32(v[u][n].v[i]), acc[n][i]);
            }
        }
#pragma unroll
        for (int n = 0; n < U; ++n) {
            if (c + n * step >= units) break;
            W o;
#pragma unroll
            for (int i = 0; i < V; ++i) o.v[i] = from_f32<T>(acc[n][i]);
            store_once(out + t * ldo + static_cast<size_t>(c + n * step) * V, o);
        }
    }
}

// dy[pos[t, j]] = w[t, j] * dout[t] and dw[t, j] = dot(dout[t], y[pos[t, j]]): one pass over the rows, KB of them in flight;
// the dot products (KT of them) in fp32 in registers, added up over the token's threads by shuffles and then in warp order.
template <typename T, int V, int KT>
__global__ void __launch_bounds__(256) route_combine_grad_kernel(const T* __restrict__ dout, long long ldd, const T* __restrict__ y,
                                                                 long long ldy, long long rows, int tokens, int k, int units,
                                                                 const int* __restrict__ pos, const float* __restrict__ weights,
                                                                 T* __restrict__ dy, long long lddy, float* __restrict__ dw) {
    using W = Vec<T, V>;
    constexpr int KB = KT < 8 ? KT : 8;
    __shared__ float part[8][KT];
    const size_t t = static_cast<size_t>(blockIdx.x) * blockDim.y + threadIdx.y;
    const bool here = t < static_cast<size_t>(tokens);   // blockDim.x is a multiple of 32: whole warps
    const int warps_x = blockDim.x >> 5, warp_x = threadIdx.x >> 5;
    float acc[KT];
#pragma unroll
    for (int j = 0; j < KT; ++j) acc[j] = 0.f;
    if (here) {
        const int* p = pos + t * k;
        int r[KT];
        float w[KT];
#pragma unroll
        for (int j = 0; j < KT; ++j) {
            r[j] = j < k ? p[j] : -1;
            if (r[j] >= rows) r[j] = -1;
            w[j] = r[j] >= 0 ? weights[t * k + j] : 0.f;
        }
        for (int c = threadIdx.x; c < units; c += blockDim.x) {
            const size_t at = static_cast<size_t>(c) * V;
            const W d = load_once<W>(dout + t * ldd + at);
#pragma unroll
            for (int j0 = 0; j0 < KT; j0 += KB) {
                W a[KB];
#pragma unroll
                for (int u = 0; u < KB; ++u)
                    if (r[j0 + u] >= 0) a[u] = load_once<W>(y + static_cast<size_t>(r[j0 + u]) * ldy + at);
#pragma unroll
                for (int u = 0; u < KB; ++u) {
                    const int j = j0 + u;
                    if (r[j] < 0) continue;
                    W o;
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const float df = to_f32(d.v[i]);
                        acc[j] = fmaf(df, to_f32(a[u].v[i]), acc[j]);
                        o.v[i] = from_f32<T>(w[j] * df);
                    }
                    store_once(dy + static_cast<size_t>(r[j]) * lddy + at, o);
                }
            }
        }
    }
#pragma unroll
    for (int j = 0; j < KT; ++j) acc[j] = warp_sum(acc[j]);
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
        for (int j = 0; j < KT; ++j) part[threadIdx.y * warps_x + warp_x][j] = acc[j];
    }
    __syncthreads();
    if (here && threadIdx.x < static_cast<unsigned>(k)) {
        float s = 0.f;
        for (int i = 0; i < warps_x; ++i) s += part[threadIdx.y * warps_x + i][threadIdx.x];
        dw[t * k + threadIdx.x] = s;
    }
}

int blocks_for(int tokens) {
    if (tokens <= rt::ONE_BLOCK) return 1;
    const int by_warp = (tokens + 31) / 32;   // a token per warp while that leaves SMs without a block
    return by_warp < rt::MAX_BLOCKS ? by_warp : rt::MAX_BLOCKS;
}

int check_choice(const char* fn, int tokens, int experts, int k) {
    if (tokens < 0 || experts < 0 || k < 0) return set_error(PRISM_B200_ERR_INVALID_ARGUMENT, "%s: negative size", fn);
    if (experts < 1 || experts > rt::MAX_EXPERTS)
        return set_error(PRISM_B200_ERR_UNSUPPORTED_SHAPE, "%s: 1 to %d experts (got %d)", fn, rt::MAX_EXPERTS, experts);
    if (k < 1 || k > experts || k > rt::MAX_CHOICES)
        return set_error(PRISM_B200_ERR_UNSUPPORTED_SHAPE, "%s: 1 to min(experts, %d) choices (got %d)", fn, rt::MAX_CHOICES, k);
    if (static_cast<long long>(tokens) * k > 1LL << 30)
        return set_error(PRISM_B200_ERR_TOO_LARGE, "%s: tokens x k at most 2^30", fn);
    return PRISM_B200_OK;
}

int check_rows(const char* fn, long long ld, long long width) {
    if (ld < width) return set_error(PRISM_B200_ERR_INVALID_ARGUMENT, "%s: a row stride below the row's width", fn);
    return PRISM_B200_OK;
}

int elem_size(int dtype) { return dtype == PRISM_B200_F32 ? 4 : (dtype == PRISM_B200_BF16 || dtype == PRISM_B200_F16) ? 2 : 0; }

// Largest vector, in elements, that divides the width, the strides and the addresses (at most 16 bytes).
int vector_elems(int size, long long width, long long ld_a, const void* a, long long ld_b, const void* b, long long ld_c = 0,
                 const void* c = nullptr) {
    int v = 16 / size;
    const uintptr_t addr = reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(c);
    while (v > 1 && (width % v || ld_a % v || ld_b % v || ld_c % v || addr % (static_cast<uintptr_t>(v) * size))) v >>= 1;
    return v;
}

template <typename T>
int launch_choose(const RouteArgs& a, int blocks, int threads, cudaStream_t s) {
    const int per_lane = (a.experts + 31) / 32;
    if (per_lane <= 1) route_choose_kernel<T, 1><<<blocks, threads, 0, s>>>(a);
    else if (per_lane <= 2) route_choose_kernel<T, 2><<<blocks, threads, 0, s>>>(a);
    else if (per_lane <= 4) route_choose_kernel<T, 4><<<blocks, threads, 0, s>>>(a);
    else if (per_lane <= 8) route_choose_kernel<T, 8><<<blocks, threads, 0, s>>>(a);
    else if (per_lane <= 16) route_choose_kernel<T, 16><<<blocks, threads, 0, s>>>(a);
    else route_choose_kernel<T, 32><<<blocks, threads, 0, s>>>(a);
    PRISM_CUDA_TRY(cudaGetLastError());
    count_launch();
    return PRISM_B200_OK;
}

int launch_place(const RouteArgs& a, int blocks, cudaStream_t s) {
    const int per_lane = (a.experts + 31) / 32;
    void (*kern)(RouteArgs) = per_lane <= 1    ? route_place_kernel<1>
                              : per_lane <= 2  ? route_place_kernel<2>
                              : per_lane <= 4  ? route_place_kernel<4>
                              : per_lane <= 8  ? route_place_kernel<8>
                              : per_lane <= 16 ? route_place_kernel<16>
                                               : route_place_kernel<32>;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;   // its launch overlaps the first kernel's end
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(blocks));
    cfg.blockDim = dim3(1024);
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    PRISM_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, a));
    count_launch();
    return PRISM_B200_OK;
}

template <typename T>
int launch_grad(const void* logits, long long ld, int tokens, int experts, int k, int renorm, const int* ids, const float* weights,
                const float* dweights, void* out, cudaStream_t s) {
    const int blocks = (tokens + 7) / 8;
    const int per_lane = (experts + 31) / 32;
    const T* l = static_cast<const T*>(logits);
    T* o = static_cast<T*>(out);
    auto kern = renorm || per_lane <= 1 ? route_grad_kernel<T, 1>
                : per_lane <= 2         ? route_grad_kernel<T, 2>
                : per_lane <= 4         ? route_grad_kernel<T, 4>
                : per_lane <= 8         ? route_grad_kernel<T, 8>
                : per_lane <= 16        ? route_grad_kernel<T, 16>
                                        : route_grad_kernel<T, 32>;
    kern<<<blocks, 256, 0, s>>>(l, ld, tokens, experts, k, renorm, ids, weights, dweights, o);
    PRISM_CUDA_TRY(cudaGetLastError());
    count_launch();
    return PRISM_B200_OK;
}

// Threads along a row (a power of two, at least `least`) and tokens per block of 256 threads.
dim3 row_block(int units, int least) {
    int x = least;
    while (x < 256 && x < units) x <<= 1;
    return dim3(static_cast<unsigned>(x), static_cast<unsigned>(256 / x));
}

template <typename U>
int launch_gather(const void* x, long long ldx, int tokens, int k, int units, const int* pos, long long rows, void* out, long long ldo,
                  cudaStream_t s) {
    const dim3 block = row_block(units, 16);
    const int pieces = (units + 511) / 512;
    const dim3 grid((tokens + block.y - 1) / block.y, pieces < 64 ? pieces : 64);
    route_gather_kernel<U><<<grid, block, 0, s>>>(static_cast<const U*>(x), ldx, tokens, k, units, pos, rows, static_cast<U*>(out), ldo);
    PRISM_CUDA_TRY(cudaGetLastError());
    count_launch();
    return PRISM_B200_OK;
}

template <typename T, int V>
int launch_combine(const void* y, long long ldy, long long rows, int tokens, int k, int width, const int* pos, const float* weights,
                   void* out, long long ldo, cudaStream_t s) {
    const int units = width / V;
    const dim3 block = row_block(units, 16);
    const int per_block = V >= 4 ? 256 : 1024;
    const int pieces = (units + per_block - 1) / per_block;
    const dim3 grid((tokens + block.y - 1) / block.y, pieces < 64 ? pieces : 64);
    auto kern = k <= 2 ? route_combine_kernel<T, V, 2> : k <= 4 ? route_combine_kernel<T, V, 4> : route_combine_kernel<T, V, 8>;
    kern<<<grid, block, 0, s>>>(static_cast<const T*>(y), ldy, rows, tokens, k, units, pos, weights, static_cast<T*>(out), ldo);
    PRISM_CUDA_TRY(cudaGetLastError());
    count_launch();
    return PRISM_B200_OK;
}

struct CombineGrad {
    const void *dout, *y;
    void* dy;
    long long ldd, ldy, lddy, rows;
    int tokens, k, width;
    const int* pos;
    const float* weights;
    float* dw;
};

template <typename T, int V, int KT>
int launch_combine_grad_k(const CombineGrad& a, cudaStream_t s) {
    const int units = a.width / V;
    const dim3 block = row_block(units, 32);
    const unsigned grid = (a.tokens + block.y - 1) / block.y;
    route_combine_grad_kernel<T, V, KT><<<grid, block, 0, s>>>(static_cast<const T*>(a.dout), a.ldd, static_cast<const T*>(a.y), a.ldy,
                                                               a.rows, a.tokens, a.k, units, a.pos, a.weights, static_cast<T*>(a.dy),
                                                               a.lddy, a.dw);
    PRISM_CUDA_TRY(cudaGetLastError());
    count_launch();
    return PRISM_B200_OK;
}

template <typename T, int V>
int launch_combine_grad(const CombineGrad& a, cudaStream_t s) {
    if (a.k <= 2) return launch_combine_grad_k<T, V, 2>(a, s);
    if (a.k <= 4) return launch_combine_grad_k<T, V, 4>(a, s);
    if (a.k <= 8) return launch_combine_grad_k<T, V, 8>(a, s);
    return launch_combine_grad_k<T, V, 32>(a, s);
}

}  // namespace
}  // namespace prism_b200

using namespace prism_b200;

extern "C" int prism_b200_route_workspace_size(int tokens, int experts, int k, size_t* bytes) {
    if (!bytes) return set_error(PRISM_B200_ERR_INVALID_ARGUMENT, "route_workspace_size: null pointer");
    if (int rc = check_choice("route_workspace_size", tokens, experts, k)) return rc;
    const int blocks = blocks_for(tokens);
    *bytes = blocks == 1 ? 0 : static_cast<size_t>(blocks) * experts * sizeof(int);
    return PRISM_B200_OK;
}

extern "C" int prism_b200_route_topk(int tokens, int experts, int k, int dtype, const void* logits, long long ld, int renormalize,
                                     int* ids, float* weights, int* pos, int* order, int* offsets, void* workspace, void* stream) {
    if (int rc = check_choice("route_topk", tokens, experts, k)) return rc;
    if (!elem_size(dtype)) return set_error(PRISM_B200_ERR_INVALID_ARGUMENT, "route_topk: unknown element type %d", dtype);
    const int blocks = blocks_for(tokens);
    if (!offsets || (tokens > 0 && (!logits || !ids || !weights || !pos || !order)) || (blocks > 1 && !workspace))
        return set_error(PRISM_B200_ERR_INVALID_ARGUMENT, "route_topk: null pointer");
    if (int rc = check_rows("route_topk", ld, experts)) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (tokens == 0) {
        PRISM_CUDA_TRY(cudaMemsetAsync(offsets, 0, (static_cast<size_t>(experts) + 1) * sizeof(int), s));
        return PRISM_B200_OK;
    }
    RouteArgs a{logits, ld, tokens, experts, k, renormalize ? 1 : 0, (tokens + blocks - 1) / blocks, ids, weights, pos, order, offsets,
                workspace, 0, 0};
    a.narrow = a.tokens_per_block <= 0xFFFF;
    a.eights = dtype != PRISM_B200_F32 && k <= 8 && experts % 8 == 0 && ld % 8 == 0 && reinterpret_cast<uintptr_t>(logits) % 16 == 0;
    // a warp per token, up to 32 of them; at least four so that the ranking of many experts is not left to one warp
    int threads = 32 * a.tokens_per_block;
    threads = threads < 128 ? 128 : threads > 1024 ? 1024 : threads;
    int rc = dtype == PRISM_B200_F32    ? launch_choose<float>(a, blocks, threads, s)
             : dtype == PRISM_B200_BF16 ? launch_choose<__nv_bfloat16>(a, blocks, threads, s)
                                        : launch_choose<__half>(a, blocks, threads, s);
    if (rc || blocks == 1) return rc;
    return launch_place(a, blocks, s);
}

extern "C" int prism_b200_route_topk_grad(int tokens, int experts, int k, int dtype, const void* logits, long long ld, int renormalize,
                                          const int* ids, const float* weights, const float* dweights, void* dlogits, void* stream) {
    if (int rc = check_choice("route_topk_grad", tokens, experts, k)) return rc;
    if (!elem_size(dtype)) return set_error(PRISM_B200_ERR_INVALID_ARGUMENT, "route_topk_grad: unknown element type %d", dtype);
    if (tokens == 0) return PRISM_B200_OK;
    if (!logits || !ids || !weights || !dweights || !dlogits)
        return set_error(PRISM_B200_ERR_INVALID_ARGUMENT, "route_topk_grad: null pointer");
    if (int rc = check_rows("route_topk_grad", ld, experts)) return rc;
    if (rows_overlap(dlogits, tokens, experts, experts, logits, tokens, experts, ld, elem_size(dtype)))
        return set_error(PRISM_B200_ERR_INVALID_ARGUMENT, "route_topk_grad: dlogits and logits overlap");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == PRISM_B200_F32) return launch_grad<float>(logits, ld, tokens, experts, k, renormalize, ids, weights, dweights, dlogits, s);
    if (dtype == PRISM_B200_BF16)
        return launch_grad<__nv_bfloat16>(logits, ld, tokens, experts, k, renormalize, ids, weights, dweights, dlogits, s);
    return launch_grad<__half>(logits, ld, tokens, experts, k, renormalize, ids, weights, dweights, dlogits, s);
}

namespace prism_b200 {
namespace {
int check_copy(const char* fn, int dtype, int tokens, int k, int width, long long rows, long long ld_a, long long ld_b) {
    if (!elem_size(dtype)) return set_error(PRISM_B200_ERR_INVALID_ARGUMENT, "%s: unknown element type %d", fn, dtype);
    if (tokens < 0 || k < 0 || width < 0 || rows < 0) return set_error(PRISM_B200_ERR_INVALID_ARGUMENT, "%s: negative size", fn);
    if (k < 1 || k > rt::MAX_CHOICES)
        return set_error(PRISM_B200_ERR_UNSUPPORTED_SHAPE, "%s: 1 to %d choices (got %d)", fn, rt::MAX_CHOICES, k);
    if (static_cast<long long>(tokens) * k > 1LL << 30)
        return set_error(PRISM_B200_ERR_TOO_LARGE, "%s: tokens x k at most 2^30", fn);
    if (width > 1 << 30) return set_error(PRISM_B200_ERR_TOO_LARGE, "%s: rows of at most 2^30 elements", fn);
    if (int rc = check_rows(fn, ld_a, width)) return rc;
    return check_rows(fn, ld_b, width);
}
}  // namespace
}  // namespace prism_b200

extern "C" int prism_b200_route_gather(int dtype, int tokens, int k, int width, const void* x, long long ldx, const int* pos,
                                       long long rows, void* out, long long ldo, void* stream) {
    if (int rc = check_copy("route_gather", dtype, tokens, k, width, rows, ldx, ldo)) return rc;
    if (tokens == 0 || width == 0 || rows == 0) return PRISM_B200_OK;
    if (!x || !pos || !out) return set_error(PRISM_B200_ERR_INVALID_ARGUMENT, "route_gather: null pointer");
    const int size = elem_size(dtype);
    if (rows_overlap(x, tokens, width, ldx, out, rows, width, ldo, size))
        return set_error(PRISM_B200_ERR_INVALID_ARGUMENT, "route_gather: x and out overlap");
    const int v = vector_elems(size, width, ldx, x, ldo, out), unit = v * size;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (unit == 16) return launch_gather<uint4>(x, ldx / v, tokens, k, width / v, pos, rows, out, ldo / v, s);
    if (unit == 8) return launch_gather<uint2>(x, ldx / v, tokens, k, width / v, pos, rows, out, ldo / v, s);
    if (unit == 4) return launch_gather<uint32_t>(x, ldx / v, tokens, k, width / v, pos, rows, out, ldo / v, s);
    return launch_gather<uint16_t>(x, ldx / v, tokens, k, width / v, pos, rows, out, ldo / v, s);
}

extern "C" int prism_b200_route_combine(int dtype, int tokens, int k, int width, const void* y, long long ldy, long long rows,
                                        const int* pos, const float* weights, void* out, long long ldo, void* stream) {
    if (int rc = check_copy("route_combine", dtype, tokens, k, width, rows, ldy, ldo)) return rc;
    if (tokens == 0 || width == 0) return PRISM_B200_OK;
    if ((!y && rows > 0) || !pos || !out) return set_error(PRISM_B200_ERR_INVALID_ARGUMENT, "route_combine: null pointer");
    const int size = elem_size(dtype);
    if (rows_overlap(y, rows, width, ldy, out, tokens, width, ldo, size))
        return set_error(PRISM_B200_ERR_INVALID_ARGUMENT, "route_combine: y and out overlap");
    const int v = vector_elems(size, width, ldy, y, ldo, out);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
#define COMBINE(T, V) return launch_combine<T, V>(y, ldy, rows, tokens, k, width, pos, weights, out, ldo, s)
    if (dtype == PRISM_B200_F32) {
        if (v == 4) COMBINE(float, 4);
        if (v == 2) COMBINE(float, 2);
        COMBINE(float, 1);
    }
    if (dtype == PRISM_B200_BF16) {
        if (v == 8) COMBINE(__nv_bfloat16, 8);
        if (v >= 2) COMBINE(__nv_bfloat16, 2);
        COMBINE(__nv_bfloat16, 1);
    }
    if (v == 8) COMBINE(__half, 8);
    if (v >= 2) COMBINE(__half, 2);
    COMBINE(__half, 1);
#undef COMBINE
}

extern "C" int prism_b200_route_combine_grad(int dtype, int tokens, int k, int width, const void* dout, long long ldd, const void* y,
                                             long long ldy, long long rows, const int* pos, const float* weights, void* dy,
                                             long long lddy, float* dweights, void* stream) {
    if (int rc = check_copy("route_combine_grad", dtype, tokens, k, width, rows, ldd, ldy)) return rc;
    if (int rc = check_rows("route_combine_grad", lddy, width)) return rc;
    if (tokens == 0) return PRISM_B200_OK;
    if (((!y || !dy) && rows > 0 && width > 0) || (!dout && width > 0) || !pos || !weights || !dweights)
        return set_error(PRISM_B200_ERR_INVALID_ARGUMENT, "route_combine_grad: null pointer");
    const int size = elem_size(dtype);
    if (rows_overlap(dy, rows, width, lddy, y, rows, width, ldy, size) || rows_overlap(dy, rows, width, lddy, dout, tokens, width, ldd, size))
        return set_error(PRISM_B200_ERR_INVALID_ARGUMENT, "route_combine_grad: dy overlaps y or dout");
    const CombineGrad a{dout, y, dy, ldd, ldy, lddy, rows, tokens, k, width, pos, weights, dweights};
    const int v = vector_elems(size, width, ldd, dout, ldy, y, lddy, dy);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == PRISM_B200_F32) {
        if (v == 4) return launch_combine_grad<float, 4>(a, s);
        return v == 2 ? launch_combine_grad<float, 2>(a, s) : launch_combine_grad<float, 1>(a, s);
    }
    if (dtype == PRISM_B200_BF16) {
        if (v == 8) return launch_combine_grad<__nv_bfloat16, 8>(a, s);
        return v >= 2 ? launch_combine_grad<__nv_bfloat16, 2>(a, s) : launch_combine_grad<__nv_bfloat16, 1>(a, s);
    }
    if (v == 8) return launch_combine_grad<__half, 8>(a, s);
    return v >= 2 ? launch_combine_grad<__half, 2>(a, s) : launch_combine_grad<__half, 1>(a, s);
}
