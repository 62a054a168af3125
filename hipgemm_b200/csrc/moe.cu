// A mixture-of-experts layer for a few tokens: the router, and the experts' gated products over
// 4-bit weights.
//
//   route:   logits = x . R^T, p = softmax(logits) over all E experts, the top_k largest
//   experts: out[t] = sum_j weight[t][j] * down_e( silu(gate_e x[t]) * (up_e x[t]) ),  e = ids[t][j]
//
// Both products of the experts read each reached expert's codes once for all the tokens that are
// sent to it: (token, expert) pairs are grouped by expert into segments of up to 8 NT columns.
// A third, small kernel adds up a token's experts, in the order of its ids.
#include <cooperative_groups.h>

#include <atomic>

#include "hipgemm_b200.h"
#include "w4.cuh"

namespace cg = cooperative_groups;

namespace hgw {

constexpr int kMoeWarps = 8;
constexpr int kMoeThreads = kMoeWarps * 32;
constexpr int kMaxExperts = 1024;
constexpr int kMaxTopK = 16;
constexpr int kMaxPairs = 512;   // (token, expert) pairs of one launch
constexpr int kMaxTokens = 64;   // tokens of one launch
constexpr int kMaxSegments = kMaxPairs;

// ---- router -----------------------------------------------------------------------------
//
// A cluster of 8 CTAs takes TT tokens; its warps, in pairs that take half of D each, split the
// experts, EW at a time, so that a load of x serves EW experts and one of the router TT tokens.
// Sixteen products a lane are summed in fp32 and then added in 64 bits: a logit is off by 16 roundings at
// most, 16 * 2^-24 of the sum of |x r|, and experts whose logits are nearer than twice that may change
// places (equal rows of the router never do: their sums have the same bits).  64 bits throughout took 50.8
// us where this takes 32.5, and 7.1 where this takes 5.8; telling the close ones by a bound of |x| |r| and
// summing those again 45 and 8.3.  The logits go to the CTA that selects the
// token's experts over distributed shared memory.  Bound by the latency of the router's loads, all of
// which each cluster reads from L2: hence two loads of each row at a time, in a branch without other
// conditions (64 tokens, 7168 x 256 fp32: 32.5 us, 48 with a condition a load), and two CTAs an SM.
// One token, 2048 x 128 bf16: 5.8 us.

constexpr int kRouteCluster = 8;
constexpr int kRouteWarps = 8;

struct RouteParams {
    const void* x;
    const void* router;
    long long ldx;
    int T, D, E, top_k;
    bool renormalize, vec;
    int* ids;
    float* weights;
};

// A lane's 16 bytes of a row: 4 fp32 or 8 bf16 from `at` on; zeros at and past `len`.
template <typename T>
struct RouteLoad {
    static constexpr int kElements = 16 / sizeof(T);
    uint4 v;
    // Volatile, so that loads of whole chunks are not merged with those below (36.1 instead of 32.5 us).
    __device__ __forceinline__ void load_full(const T* row, int at) {
        asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(row + at));
    }
    __device__ __forceinline__ void load(const T* row, int at, int len, bool vec) {
        v = make_uint4(0u, 0u, 0u, 0u);
        if (vec) {
            if (at < len) load_full(row, at);
        } else {
            uint32_t e[kElements];
#pragma unroll
            for (int i = 0; i < kElements; ++i) {
                if constexpr (sizeof(T) == 4) e[i] = at + i < len ? __float_as_uint(row[at + i]) : 0u;
                else e[i] = at + i < len ? *reinterpret_cast<const unsigned short*>(row + at + i) : 0u;
            }
            if constexpr (sizeof(T) == 4) v = make_uint4(e[0], e[1], e[2], e[3]);
            else v = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
        }
    }
    __device__ __forceinline__ float element(int i) const {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
        else return i & 1 ? bf16_hi(w[i / 2]) : bf16_lo(w[i / 2]);
    }
};

// A key that orders as the numbers do, NaN below everything.
__device__ __forceinline__ unsigned long long order_key(double v) {
    if (v != v) return 0ull;
    const unsigned long long b = static_cast<unsigned long long>(__double_as_longlong(v));
    return b >> 63 ? ~b : b | 0x8000000000000000ull;
}

// Sums v[i], i < N, over the lanes: afterwards v[0] of lane l is the sum of v[l / (32 / N)].  (A recursion over
// N, so that every index is known and v stays in registers.)
template <int N, int O = 16, int M>
__device__ __forceinline__ void reduce_lanes(double (&v)[M], int lane) {
    if constexpr (O > 0) {
        if constexpr (N > 1) {
            const bool upper = (lane & O) != 0;
#pragma unroll
            for (int i = 0; i < N / 2; ++i) {
                const double keep = upper ? v[N / 2 + i] : v[i], give = upper ? v[i] : v[N / 2 + i];
                v[i] = keep + __shfl_xor_sync(0xffffffffu, give, O);
            }
            reduce_lanes<N / 2, O / 2>(v, lane);
        } else {
            v[0] += __shfl_xor_sync(0xffffffffu, v[0], O);
            reduce_lanes<1, O / 2>(v, lane);
        }
    }
}

template <typename T, int EW, int TT>
__global__ void __launch_bounds__(kRouteWarps * 32, 2) __cluster_dims__(kRouteCluster, 1, 1) moe_route_kernel(const RouteParams p) {
    __shared__ double halves[2][kMaxExperts];  // logits of the token that this CTA selects for, by half of D
    double* logits = halves[0];
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = static_cast<int>(cluster.block_rank());
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    const int t0 = static_cast<int>(blockIdx.x) / kRouteCluster * TT;
    pdl_trigger();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    pdl_wait();

    const T* x[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) x[t] = static_cast<const T*>(p.x) + min(t0 + t, p.T - 1) * p.ldx;
    constexpr int kChunk = 32 * RouteLoad<T>::kElements, kFlush = 16 / RouteLoad<T>::kElements;  // chunks between additions in 64 bits
    const int half = warp & 1, middle = ceil_div(p.D, 2 * kChunk) * kChunk, d1 = half ? p.D : min(middle, p.D);
    bool started = false;
    for (int e0 = (rank * kRouteWarps + warp) / 2 * EW; e0 < p.E; e0 += kRouteCluster * kRouteWarps / 2 * EW) {
        const T* r[EW];
#pragma unroll
        for (int e = 0; e < EW; ++e) r[e] = static_cast<const T*>(p.router) + static_cast<size_t>(min(e0 + e, p.E - 1)) * p.D;
        double sum[EW * TT] = {};
        for (int d = half * middle; d < d1; d += kFlush * kChunk) {
            float part[EW * TT] = {};
#pragma unroll
            for (int c = 0; c < kFlush; c += 2) {
                RouteLoad<T> w[2][EW], v[2][TT];
                const int at = d + c * kChunk + lane * RouteLoad<T>::kElements;
                if (p.vec && d + (c + 2) * kChunk <= d1) {  // a branch for all loads together, so that they are in flight together
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
#pragma unroll
                        for (int e = 0; e < EW; ++e) w[u][e].load_full(r[e], at + u * kChunk);
#pragma unroll
                        for (int t = 0; t < TT; ++t) v[u][t].load_full(x[t], at + u * kChunk);
                    }
                } else {
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
#pragma unroll
                        for (int e = 0; e < EW; ++e) w[u][e].load(r[e], at + u * kChunk, d1, p.vec);
#pragma unroll
                        for (int t = 0; t < TT; ++t) v[u][t].load(x[t], at + u * kChunk, d1, p.vec);
                    }
                }
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int i = 0; i < RouteLoad<T>::kElements; ++i)
#pragma unroll
                        for (int e = 0; e < EW; ++e)
#pragma unroll
                            for (int t = 0; t < TT; ++t)
                                part[e * TT + t] = fmaf(w[u][e].element(i), v[u][t].element(i), part[e * TT + t]);
            }
#pragma unroll
            for (int i = 0; i < EW * TT; ++i) sum[i] += static_cast<double>(part[i]);
        }
        reduce_lanes<EW * TT>(sum, lane);
        if (!started) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // every CTA of the cluster runs
        started = true;
        // Token t of the cluster is selected by CTA t.
        constexpr int kLanes = 32 / (EW * TT);
        const int i = lane / kLanes, e = e0 + i / TT;
        if (lane % kLanes == 0 && e < p.E) *cluster.map_shared_rank(&halves[half][e], i % TT) = sum[0];
    }
    if (!started) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    cluster.sync();
    // One warp per token: softmax sums, then top_k rounds of a maximum over the keys.
    const int t = t0 + rank;
    if (rank >= TT || t >= p.T || warp != 0) return;
    double top = -INFINITY;
    for (int e = lane; e < p.E; e += 32) {
        logits[e] += halves[1][e];
        top = fmax(top, logits[e]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
    unsigned long long taken = 0, best = 0;  // this lane's chosen experts by e / 32; the largest key of the others
    int at = p.E;                            // its expert, E if there is none
    auto scan = [&]() {
        best = 0;
        at = p.E;
        for (int e = lane, i = 0; e < p.E; e += 32, ++i) {
            const unsigned long long key = order_key(logits[e]);
            if (!(taken >> i & 1) && (at == p.E || key > best)) best = key, at = e;
        }
    };
    scan();
    float total = 0.0f;
    for (int e = lane; e < p.E; e += 32) total += expf(static_cast<float>(logits[e] - top));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    __syncwarp();
    int my_id = 0;
    for (int k = 0; k < p.top_k; ++k) {
        // The largest upper half, the largest lower half among those, the lowest expert among those.
        const bool any = at < p.E;
        const unsigned hi = any ? static_cast<unsigned>(best >> 32) : 0u;
        const unsigned high = __reduce_max_sync(0xffffffffu, hi);
        const unsigned lo = any && hi == high ? static_cast<unsigned>(best) : 0u;
        const unsigned low = __reduce_max_sync(0xffffffffu, lo);
        const int from = __reduce_min_sync(0xffffffffu, any && hi == high && lo == low ? at : p.E);
        if (lane == k) my_id = from;
        if (any && at == from) {
            taken |= 1ull << (at / 32);
            scan();
        }
    }
    const float mine = lane < p.top_k ? expf(static_cast<float>(logits[my_id] - top)) / total : 0.0f;
    float chosen = mine;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) chosen += __shfl_xor_sync(0xffffffffu, chosen, o);
    if (lane < p.top_k) {
        const size_t to = static_cast<size_t>(t) * p.top_k + lane;
        p.ids[to] = my_id;
        p.weights[to] = p.renormalize ? mine / chosen : mine;
    }
}

template <typename T, int EW, int TT>
int launch_route(const RouteParams& p, cudaStream_t stream) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(ceil_div(p.T, TT)) * kRouteCluster, 1, 1);
    cfg.blockDim = dim3(kRouteWarps * 32, 1, 1);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, moe_route_kernel<T, EW, TT>, p) == cudaSuccess) return HGEMM_OK;
    cudaGetLastError();
    return HGEMM_ERR_CUDA;
}

// Few tokens: a cluster each (18 clusters fit the GPU at most), 2 experts a warp at a time.  More: 4 tokens a cluster, 4 experts.
template <typename T>
int run_route(const RouteParams& p, cudaStream_t stream) {
    return p.T <= 16 ? launch_route<T, 2, 1>(p, stream) : launch_route<T, 4, 4>(p, stream);
}

// ---- grouping pairs by expert ------------------------------------------------------------

struct Segment {
    short expert, first, columns, unused;  // pairs order[first .. first + columns)
};

struct PairLists {
    int count[kMaxExperts];      // pairs of an expert, then its first place in `order`
    short rank[kMaxPairs];       // a pair's place among its expert's, -1 if it does not count
    short order[kMaxPairs];      // pairs by expert
    Segment segments[kMaxSegments];
    int n_segments;
};

// Whether pair p counts: its id is in [0, E) and its token does not have the same id at an earlier place (the
// weights of such pairs are added to the first one's).  The id, or -1.
__device__ __forceinline__ int counted_id(const int* ids, int p, int top_k, int E) {
    int id = ids[p];
    if (id < 0 || id >= E) return -1;
    for (int q = p / top_k * top_k; q < p; ++q)
        if (ids[q] == id) return -1;
    return id;
}

// Fills the lists from `given` (T x top_k ids), T * top_k <= kMaxPairs.  Within an expert pairs keep their order, and
// so do the segments: the result's bits depend on the inputs alone.  All threads call it.  `ids`: shared memory
// for kMaxPairs numbers, free again afterwards.
__device__ void build_lists(PairLists& s, int* ids, const int* given, int T, int top_k, int E, int columns) {
    const int pairs = T * top_k, lane = threadIdx.x & 31;
    __shared__ int done;
    for (int p = threadIdx.x; p < pairs; p += kMoeThreads) ids[p] = __ldcg(given + p);
    __syncthreads();
    if (threadIdx.x < 32) {
        // Up to 32 pairs, and no expert with more than a segment: all in one warp's registers.
        bool ok = false;
        if (pairs <= 32) {
            const int id = lane < pairs ? counted_id(ids, lane, top_k, E) : -1;
            const unsigned same = __match_any_sync(0xffffffffu, id), below = (1u << lane) - 1u;
            const int count = id >= 0 ? __popc(same) : 0, rank = __popc(same & below);
            ok = __all_sync(0xffffffffu, count <= columns);
            if (ok) {
                const bool leads = id >= 0 && rank == 0;
                const unsigned leaders = __ballot_sync(0xffffffffu, leads);
                int first = leads ? count : 0;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int up = __shfl_up_sync(0xffffffffu, first, o);
                    if (lane >= o) first += up;
                }
                first -= leads ? count : 0;
                if (leads)
                    s.segments[__popc(leaders & below)] = {static_cast<short>(id), static_cast<short>(first), static_cast<short>(count), 0};
                first = __shfl_sync(0xffffffffu, first, __ffs(same) - 1);
                if (id >= 0) s.order[first + rank] = static_cast<short>(lane);
                if (lane == 0) s.n_segments = __popc(leaders);
            }
        }
        if (lane == 0) done = ok;
    }
    __syncthreads();
    if (done) return;
    for (int e = threadIdx.x; e < E; e += kMoeThreads) s.count[e] = 0;
    __syncthreads();
    if (threadIdx.x < 32) {
        for (int p0 = 0; p0 < pairs; p0 += 32) {
            const int p = p0 + lane, id = p < pairs ? counted_id(ids, p, top_k, E) : -1;
            const unsigned same = __match_any_sync(0xffffffffu, id);
            const int before = __popc(same & ((1u << lane) - 1u)), base = id >= 0 ? s.count[id] : 0;
            __syncwarp();
            if (p < pairs) s.rank[p] = static_cast<short>(id >= 0 ? base + before : -1);
            if (id >= 0 && before == 0) s.count[id] = base + __popc(same);
            __syncwarp();
        }
        // First places and segments, by a scan over the experts.
        int pair_at = 0, seg_at = 0;
        for (int e0 = 0; e0 < E; e0 += 32) {
            const int e = e0 + lane, n = e < E ? s.count[e] : 0, segs = (n + columns - 1) / columns;
            int a = n, b = segs;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int ua = __shfl_up_sync(0xffffffffu, a, o), ub = __shfl_up_sync(0xffffffffu, b, o);
                if (lane >= o) a += ua, b += ub;
            }
            const int first = pair_at + a - n;
            if (e < E) s.count[e] = first;
            for (int i = 0; i < segs; ++i)
                s.segments[seg_at + b - segs + i] = {static_cast<short>(e), static_cast<short>(first + i * columns),
                                                     static_cast<short>(min(columns, n - i * columns)), 0};
            pair_at += __shfl_sync(0xffffffffu, a, 31);
            seg_at += __shfl_sync(0xffffffffu, b, 31);
        }
        if (lane == 0) s.n_segments = seg_at;
    }
    __syncthreads();
    for (int p = threadIdx.x; p < pairs; p += kMoeThreads)
        if (s.rank[p] >= 0) s.order[s.count[ids[p]] + s.rank[p]] = static_cast<short>(p);
    __syncthreads();
}

// ---- the experts' products ----------------------------------------------------------------------
//
// A persistent grid over units: a segment's columns times 8 / WK groups of rows.  A group is RH row
// blocks (of gate and of up, or of down); WK warps split its K, and their sums are joined in shared
// memory in a fixed order.
//
// h = silu(gate x) * (up x) is kept in fp32 and enters the product with down as three bf16 terms, whose sum it
// is: nothing between the two products is rounded to fewer bits.  As two bf16 (16 bits) it cost bf16 outputs
// their last place more often than the order of summation does (2-norm of the difference to fp32's outputs
// 1.3e-4 to 1.6e-4, now 2e-5 to 9e-5), and took 240 us instead of 285 (32 tokens), 16.3 instead of 18.1 (one).

struct ExpertParams {
    const void* x;
    long long ldx;
    const int* ids;
    const float* weights;
    int T, top_k, E, D, F;
    Weight gate, up, down;
    bool vec;
    float* h;               // rows of h_stride by pair
    int h_stride;           // F rounded up to whole row blocks
    float* y;               // rows of y_stride by pair: down's products
    int y_stride;           // D rounded up to whole row blocks
    void* out;
};

// MATS = 2: gate and up, from x to h.  MATS = 1: down, from h to y.
template <typename T, int MATS, int RH, int NT, int STAGES, int WK, int GROUP, bool ZERO>
struct ExpertShape {
    using Source = std::conditional_t<MATS == 2, RowSource<T>, RowSource<float>>;
    using Product = WarpProduct<MATS * RH, NT, STAGES, GROUP, ZERO, MATS == 2, Source>;
    static constexpr int kGroups = kMoeWarps / WK;      // row groups of a unit
    static constexpr int kOut = MATS * RH * NT * 128;   // a warp's sums
    static constexpr int kRings = kMoeWarps * Product::kWarpBytes, kSmem = kRings + kMoeWarps * kOut * 4;
};

template <typename T, int MATS, int RH, int NT, int STAGES, int WK, int GROUP, bool ZERO>
__global__ void __launch_bounds__(kMoeThreads) moe_expert_kernel(const ExpertParams p) {
    using Shape = ExpertShape<T, MATS, RH, NT, STAGES, WK, GROUP, ZERO>;
    constexpr int kOut = Shape::kOut;
    extern __shared__ __align__(16) uint8_t smem[];  // the warps' rings, then their sums
    __shared__ PairLists lists;
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, group = warp / WK, part = warp % WK;
    const Weight& first = MATS == 2 ? p.gate : p.down;
    // The next kernels look at ids (and weights) before they wait for this one.  They start when every CTA of the product
    // with gate and up has come to its trigger, which is after its wait: whatever made ids is complete by then, and
    // in L2, where they load it from (an SM's L1 is only sure to be up to date after the kernel's own wait).
    if (MATS == 2) pdl_wait();
    pdl_trigger();
    build_lists(lists, reinterpret_cast<int*>(smem), p.ids, p.T, p.top_k, p.E, 8 * NT);
    if (MATS == 1) pdl_wait();
    const int row_blocks = first.row_blocks, chunks = ceil_div(row_blocks, RH * Shape::kGroups), units = lists.n_segments * chunks;
    const int steps = ceil_div(first.k_blocks, 2), s0 = steps * part / WK, s1 = steps * (part + 1) / WK;
    for (int u = blockIdx.x; u < units; u += gridDim.x) {
        const int seg = u / chunks, group0 = (u - seg * chunks) * Shape::kGroups, block0 = (group0 + group) * RH;
        const Segment sg = lists.segments[seg];
        typename Shape::Product product;
#pragma unroll
        for (int r = 0; r < RH; ++r) {
            const int block = min(block0 + r, row_blocks - 1);
            product.set_rows(r, first, sg.expert, block, lane);
            if (MATS == 2) product.set_rows(RH + r, p.up, sg.expert, block, lane);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int pair = lists.order[sg.first + min(8 * n + lane / 4, sg.columns - 1)], k = 8 * (lane & 3);
            if constexpr (MATS == 2) {
                product.x[n] = {static_cast<const T*>(p.x) + static_cast<long long>(pair / p.top_k) * p.ldx + k, p.D - k, p.vec};
            } else {
                product.x[n] = {p.h + static_cast<size_t>(pair) * p.h_stride + k, p.h_stride - k, true};
            }
        }
        product.set_columns(MATS == 2 ? (p.vec ? p.D : 0) : p.h_stride);
        float acc[MATS * RH][NT][4] = {};
        if (block0 < row_blocks) product.run(smem + warp * Shape::Product::kWarpBytes, s0, s1, lane, acc);
        float* partial = reinterpret_cast<float*>(smem + Shape::kRings);
#pragma unroll
        for (int r = 0; r < MATS * RH; ++r)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) partial[warp * kOut + ((r * NT + n) * 4 + i) * 32 + lane] = acc[r][n][i];
        __syncthreads();
        constexpr int kEach = RH * NT * 128;
        for (int i = threadIdx.x; i < Shape::kGroups * kEach; i += kMoeThreads) {
            const int gr = i / kEach, j = i - gr * kEach;
            const float* from = partial + gr * WK * kOut + j;
            float a = 0.0f, b = 0.0f;
#pragma unroll
            for (int w = 0; w < WK; ++w) {
                a += from[w * kOut];
                if (MATS == 2) b += from[w * kOut + kEach];
            }
            const int l = j & 31, f = (j >> 5) & 3, n = (j >> 7) % NT, r = (j >> 7) / NT;
            const int row = ((group0 + gr) * RH + r) * 16 + l / 4 + 8 * (f >> 1), col = 8 * n + 2 * (l & 3) + (f & 1);
            if (row >= row_blocks * 16 || col >= sg.columns) continue;
            const size_t pair = static_cast<size_t>(lists.order[sg.first + col]);
            if constexpr (MATS == 1) {
                p.y[pair * p.y_stride + row] = a;
            } else {
                // Rows past F (up to the row block's end) are zeros, which the next product may read.
                p.h[pair * p.h_stride + row] = row < p.F ? a / (1.0f + expf(-a)) * b : 0.0f;
            }
        }
        __syncthreads();
    }
}

// out[t] = sum over a token's counted pairs, in their order, of the weight times y.  4 elements a thread.
constexpr int kCombineThreads = 128;

template <typename T>
__global__ void __launch_bounds__(kCombineThreads) moe_combine_kernel(const ExpertParams p) {
    __shared__ float given[kMaxTopK], weight[kMaxTopK];  // 0: not counted
    __shared__ int ids[kMaxTopK];
    __shared__ bool counts[kMaxTopK];
    const int t = blockIdx.y, d = (blockIdx.x * kCombineThreads + threadIdx.x) * 4, slot = threadIdx.x;
    pdl_trigger();
    if (slot < p.top_k) {  // from L2, as above
        ids[slot] = __ldcg(p.ids + t * p.top_k + slot);
        given[slot] = __ldcg(p.weights + t * p.top_k + slot);
    }
    __syncthreads();
    if (slot < p.top_k) {
        const int id = counted_id(ids, slot, p.top_k, p.E);
        float w = 0.0f;
        for (int q = slot; q < p.top_k; ++q)
            if (q == slot || ids[q] == id) w += given[q];
        weight[slot] = w;
        counts[slot] = id >= 0;
    }
    __syncthreads();
    pdl_wait();
    if (d >= p.D) return;
    float v[4] = {};
    for (int j = 0; j < p.top_k; ++j) {
        if (!counts[j]) continue;
        const float4 y = *reinterpret_cast<const float4*>(p.y + static_cast<size_t>(t * p.top_k + j) * p.y_stride + d);
        v[0] = fmaf(weight[j], y.x, v[0]);
        v[1] = fmaf(weight[j], y.y, v[1]);
        v[2] = fmaf(weight[j], y.z, v[2]);
        v[3] = fmaf(weight[j], y.w, v[3]);
    }
    T* to = static_cast<T*>(p.out) + static_cast<size_t>(t) * p.D + d;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (d + i >= p.D) break;
        if constexpr (sizeof(T) == 4) to[i] = v[i];
        else to[i] = __float2bfloat16_rn(v[i]);
    }
}

// ---- host -----------------------------------------------------------------------------------

inline int tokens_per_launch(int top_k) {
    const int t = kMaxPairs / top_k;
    return t < kMaxTokens ? t : kMaxTokens;
}

template <typename T, int MATS, int RH, int NT, int STAGES, int WK, int GROUP, bool ZERO>
int launch_experts(const ExpertParams& p, int sms, int dev, cudaStream_t stream) {
    using Shape = ExpertShape<T, MATS, RH, NT, STAGES, WK, GROUP, ZERO>;
    constexpr auto kernel = moe_expert_kernel<T, MATS, RH, NT, STAGES, WK, GROUP, ZERO>;
    static_assert(Shape::kSmem <= 200 * 1024, "shared memory of a CTA");
    const int per_sm = resident_ctas<kernel>(dev, kMoeThreads, Shape::kSmem);
    if (per_sm < 1) return HGEMM_ERR_CUDA;
    const int pairs = p.T * p.top_k, experts = pairs < p.E ? pairs : p.E;
    const Weight& w = MATS == 2 ? p.gate : p.down;
    const long long most = static_cast<long long>(experts + pairs / (8 * NT)) * ceil_div(w.row_blocks, RH * Shape::kGroups);
    const long long wave = static_cast<long long>(sms) * per_sm;
    return launch<kernel>(dim3(static_cast<unsigned>(most < wave ? most : wave)), kMoeThreads, 1, Shape::kSmem, stream, p);
}

// WK: 2 where that gives units enough, else 4.  Measured (bf16, groups of 128; WK = 2, 4, 8): gate and up of 32 tokens
// through 6 of 64 experts of 4096 x 2048 145, 148, 156 us, of 4 tokens through 8 of 64 of 2048 x 1024 19.0,
// 20.9, 21.9, of one token 10.2, 10.5, 9.6; the three kernels together, by down's WK, 289, 297, 302, then 49.3,
// 46.2, 47.4, then 22.2, 18.0, 18.2.  Two row blocks of down a warp: 347 instead of 289 with one.  But one of gate
// and one of up: 177 instead of 145 with two, whose CTAs then fit an SM once instead of three times.
template <typename T, int MATS, int NT, int GROUP, bool ZERO>
int run_experts(const ExpertParams& p, int sms, int dev, cudaStream_t stream) {
    constexpr int RH = MATS == 2 ? 1 : 2;
    const int pairs = p.T * p.top_k, experts = pairs < p.E ? pairs : p.E;
    const int units = experts * ceil_div((MATS == 2 ? p.gate : p.down).row_blocks, RH * 4);
    using Of = std::conditional_t<MATS == 2, T, float>;  // down reads h, fp32 for either type of x
    if (units >= (MATS == 2 ? 2 : 4) * sms) return launch_experts<Of, MATS, RH, NT, 3, 2, GROUP, ZERO>(p, sms, dev, stream);
    return launch_experts<Of, MATS, RH, NT, 3, 4, GROUP, ZERO>(p, sms, dev, stream);
}

// Columns of a segment: 8, or 16 where an expert has more than 8 tokens on average (bf16 only: fp32's three terms
// and two tiles of columns do not fit the registers).
template <typename T, int MATS, int GROUP, bool ZERO>
int run_expert_product(const ExpertParams& p, int sms, int dev, cudaStream_t stream) {
    if constexpr (sizeof(T) == 2) {
        if (p.T * p.top_k > 8 * p.E) return run_experts<T, MATS, 2, GROUP, ZERO>(p, sms, dev, stream);
    }
    return run_experts<T, MATS, 1, GROUP, ZERO>(p, sms, dev, stream);
}

inline size_t padded_rows(int n) { return static_cast<size_t>(ceil_div(n, kTileRows)) * kTileRows; }

}  // namespace hgw

extern "C" {

int hgemm_moe_route(const void* x, int x_dtype, long long ldx, const void* router, int T, int D, int E, int top_k,
                    int renormalize, int* ids, float* weights, hgemm_stream_t stream) {
    if (T < 0 || D < 0 || E < 1 || top_k < 1 || top_k > E) return HGEMM_ERR_INVALID_VALUE;
    if (x_dtype != HGEMM_DTYPE_F32 && x_dtype != HGEMM_DTYPE_BF16) return HGEMM_ERR_INVALID_VALUE;
    if (E > hgw::kMaxExperts || top_k > hgw::kMaxTopK) return HGEMM_ERR_UNSUPPORTED;
    if (T > 1 && ldx < D) return HGEMM_ERR_INVALID_VALUE;
    if (T == 0) return HGEMM_OK;
    if (!ids || !weights || (D > 0 && (!x || !router))) return HGEMM_ERR_INVALID_VALUE;
    const unsigned size = x_dtype == HGEMM_DTYPE_F32 ? 4 : 2;
    if (hgw::misaligned(x, size) || hgw::misaligned(router, size) || hgw::misaligned(ids, 4) || hgw::misaligned(weights, 4))
        return HGEMM_ERR_ALIGNMENT;
    int sms = 0, dev = 0;
    if (int rc = hgw::current_device(&sms, &dev)) return rc;
    hgw::RouteParams p{x, router, T > 1 ? ldx : 0, T, D, E, top_k, renormalize != 0, false, ids, weights};
    p.vec = !hgw::misaligned(x, 16) && !hgw::misaligned(router, 16) && D % 8 == 0 && p.ldx % (16 / size) == 0;
    const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    return x_dtype == HGEMM_DTYPE_F32 ? hgw::run_route<float>(p, s) : hgw::run_route<__nv_bfloat16>(p, s);
}

size_t hgemm_w4_moe_workspace_bytes(int T, int top_k, int D, int F) {
    if (T <= 0 || top_k <= 0 || top_k > hgw::kMaxTopK || D <= 0 || F <= 0) return 0;
    const int most = hgw::tokens_per_launch(top_k), tokens = T < most ? T : most;
    return static_cast<size_t>(tokens) * top_k * (hgw::padded_rows(F) + hgw::padded_rows(D)) * 4;  // h and y
}

int hgemm_w4_moe(const void* x, int x_dtype, long long ldx, const int* ids, const float* weights, int T, int top_k, int E,
                 int D, int F, const hgemm_w4_weight* gate, const hgemm_w4_weight* up, const hgemm_w4_weight* down,
                 void* out, void* workspace, size_t workspace_bytes, hgemm_stream_t stream) {
    if (T < 0 || D < 0 || F < 0 || E < 1 || top_k < 1 || !gate || !up || !down) return HGEMM_ERR_INVALID_VALUE;
    if (x_dtype != HGEMM_DTYPE_F32 && x_dtype != HGEMM_DTYPE_BF16) return HGEMM_ERR_INVALID_VALUE;
    if (!hgw::valid_group(gate->group) || !hgw::valid_group(up->group) || !hgw::valid_group(down->group))
        return HGEMM_ERR_INVALID_VALUE;
    if (E > hgw::kMaxExperts || top_k > hgw::kMaxTopK) return HGEMM_ERR_UNSUPPORTED;
    if (gate->group != up->group || !gate->zeros != !up->zeros) return HGEMM_ERR_UNSUPPORTED;
    if (T > 1 && ldx < D) return HGEMM_ERR_INVALID_VALUE;
    if (T == 0 || D == 0) return HGEMM_OK;
    if (!x || !ids || !weights || !out) return HGEMM_ERR_INVALID_VALUE;
    const unsigned size = x_dtype == HGEMM_DTYPE_F32 ? 4 : 2;
    if (hgw::misaligned(x, size) || hgw::misaligned(out, size) || hgw::misaligned(ids, 4) || hgw::misaligned(weights, 4))
        return HGEMM_ERR_ALIGNMENT;
    const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    int sms = 0, dev = 0;
    if (F == 0) {
        if (int rc = hgw::current_device(&sms, &dev)) return rc;
        return cudaMemsetAsync(out, 0, static_cast<size_t>(T) * D * size, s) == cudaSuccess ? HGEMM_OK : HGEMM_ERR_CUDA;
    }
    for (const hgemm_w4_weight* w : {gate, up, down}) {
        if (!w->q || !w->scales) return HGEMM_ERR_INVALID_VALUE;
        if (hgw::misaligned(w->q, 16) || hgw::misaligned(w->scales, 16) || hgw::misaligned(w->zeros, 16))
            return HGEMM_ERR_ALIGNMENT;
    }
    if (!workspace || workspace_bytes < hgemm_w4_moe_workspace_bytes(T, top_k, D, F)) return HGEMM_ERR_INVALID_VALUE;
    if (hgw::misaligned(workspace, 16)) return HGEMM_ERR_ALIGNMENT;
    // A launch's out is written when its x has been read, but before the next launch's x is: out may be x itself, whose
    // rows end before those of the next launch's begin.
    if (T > hgw::tokens_per_launch(top_k) && out != x && hgw::meets_rows(out, static_cast<size_t>(T) * D * size, x, T, ldx, D, size))
        return HGEMM_ERR_INVALID_VALUE;
    if (int rc = hgw::current_device(&sms, &dev)) return rc;

    const int most = hgw::tokens_per_launch(top_k);
    hgw::ExpertParams p{};
    p.ldx = T > 1 ? ldx : 0;
    p.top_k = top_k;
    p.E = E;
    p.D = D;
    p.F = F;
    p.gate = hgw::make_weight(gate->q, gate->scales, gate->zeros, F, D, gate->group);
    p.up = hgw::make_weight(up->q, up->scales, up->zeros, F, D, up->group);
    p.down = hgw::make_weight(down->q, down->scales, down->zeros, D, F, down->group);
    p.vec = !hgw::misaligned(x, 16) && D % 8 == 0 && p.ldx % (16 / size) == 0;
    const int held = (T < most ? T : most) * top_k;  // pairs of a launch
    p.h = static_cast<float*>(workspace);
    p.h_stride = static_cast<int>(hgw::padded_rows(F));
    p.y = p.h + static_cast<size_t>(held) * p.h_stride;
    p.y_stride = static_cast<int>(hgw::padded_rows(D));
    // Launches of up to kMaxTokens tokens; they share the workspace, in stream order.
    for (int t0 = 0; t0 < T; t0 += most) {
        p.T = T - t0 < most ? T - t0 : most;
        p.x = static_cast<const char*>(x) + static_cast<size_t>(t0) * ldx * size;
        p.ids = ids + static_cast<size_t>(t0) * top_k;
        p.weights = weights + static_cast<size_t>(t0) * top_k;
        p.out = static_cast<char*>(out) + static_cast<size_t>(t0) * D * size;
        int rc = hgw::with_format(gate->group, gate->zeros != nullptr, [&](auto g, auto z) {
            constexpr int G = decltype(g)::value;
            constexpr bool Z = decltype(z)::value;
            return x_dtype == HGEMM_DTYPE_F32 ? hgw::run_expert_product<float, 2, G, Z>(p, sms, dev, s)
                                              : hgw::run_expert_product<__nv_bfloat16, 2, G, Z>(p, sms, dev, s);
        });
        if (rc) return rc;
        rc = hgw::with_format(down->group, down->zeros != nullptr, [&](auto g, auto z) {
            constexpr int G = decltype(g)::value;
            constexpr bool Z = decltype(z)::value;
            return x_dtype == HGEMM_DTYPE_F32 ? hgw::run_expert_product<float, 1, G, Z>(p, sms, dev, s)
                                              : hgw::run_expert_product<__nv_bfloat16, 1, G, Z>(p, sms, dev, s);
        });
        if (rc) return rc;
        const dim3 grid(static_cast<unsigned>(hgw::ceil_div(D, 4 * hgw::kCombineThreads)), static_cast<unsigned>(p.T), 1);
        rc = x_dtype == HGEMM_DTYPE_F32
                 ? hgw::launch<hgw::moe_combine_kernel<float>>(grid, hgw::kCombineThreads, 1, 0, s, p)
                 : hgw::launch<hgw::moe_combine_kernel<__nv_bfloat16>>(grid, hgw::kCombineThreads, 1, 0, s, p);
        if (rc) return rc;
    }
    return HGEMM_OK;
}

}  // extern "C"
