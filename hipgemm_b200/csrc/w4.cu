// 4-bit weights with group scales: quantiser, its inverse, and the product of a few rows of
// activations with such a weight.  Layout and inner product: w4.cuh.
#include <cooperative_groups.h>

#include <atomic>

#include "hipgemm_b200.h"
#include "w4.cuh"

namespace cg = cooperative_groups;

namespace hgw {

int current_device(int* sms, int* dev) {
    static std::atomic<int> known[kMaxDevices];  // SM count, or -1 for a device of another architecture
    if (cudaGetDevice(dev) != cudaSuccess || *dev < 0 || *dev >= kMaxDevices) {
        cudaGetLastError();
        return HGEMM_ERR_NO_DEVICE;
    }
    int v = known[*dev].load(std::memory_order_relaxed);
    if (v == 0) {
        int major = 0, minor = 0, n = 0;
        if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, *dev) != cudaSuccess ||
            cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, *dev) != cudaSuccess ||
            cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, *dev) != cudaSuccess) {
            cudaGetLastError();
            return HGEMM_ERR_NO_DEVICE;
        }
        v = major == 10 && minor == 0 ? n : -1;
        known[*dev].store(v, std::memory_order_relaxed);
    }
    if (v < 0) return HGEMM_ERR_NO_DEVICE;
    *sms = v;
    return HGEMM_OK;
}

// ---- quantiser --------------------------------------------------------------------------
//
// Per group, exactly what 64-bit arithmetic would give:
//   symmetric:  scale = bf16(fp32(amax / 7)),          code = clamp(rint(w / scale), -8, 7) + 8
//   asymmetric: scale = bf16(fp32((max - min) / 15)),  zero = clamp(rint(-min / scale), 0, 15),
//               code = clamp(rint(w / scale) + zero, 0, 15)       with min <= 0 <= max
// scale is 1 where that is 0 and at most the largest bf16; NaN does not count toward the
// extremes and takes the code of 0.

constexpr float kMaxBf16 = 3.3895313892515355e38f;

// rint(w / s) for s > 0, limited to +-17, without a division: a product with the reciprocal is
// off by at most one, and w - q s (one rounding, monotonic) tells on which side of the half-step
// border, which is representable, w lies.  Ties go to the even code.
__device__ __forceinline__ float rint_quotient(float w, float s, float inv) {
    float q = rintf(fminf(fmaxf(w * inv, -17.0f), 17.0f));
    const float e2 = 2.0f * fmaf(-q, s, w);
    const bool odd = (static_cast<int>(q) & 1) != 0;
    if (e2 > s || (e2 == s && odd)) q += 1.0f;
    if (e2 < -s || (e2 == -s && odd)) q -= 1.0f;
    return w == w ? q : 0.0f;
}

struct GroupScale {
    float scale, inv, boost;  // w and scale are taken times boost (a power of two) where scale is tiny
    float zero;               // 8 for symmetric
};

__device__ __forceinline__ float bf16_scale(float v) {
    float s = fminf(__bfloat162float(__float2bfloat16_rn(v)), kMaxBf16);
    return s == 0.0f ? 1.0f : s;
}

template <bool ZERO>
__device__ __forceinline__ GroupScale group_scale(float lo, float hi) {
    GroupScale g;
    if (ZERO) {
        g.scale = bf16_scale(static_cast<float>((static_cast<double>(hi) - static_cast<double>(lo)) / 15.0));
    } else {
        g.scale = bf16_scale(__fdiv_rn(fmaxf(hi, -lo), 7.0f));
    }
    g.boost = g.scale < 0x1p-60f ? 0x1p80f : 1.0f;
    g.inv = __frcp_rn(g.scale * g.boost);
    g.zero = ZERO ? fminf(fmaxf(rint_quotient(-lo * g.boost, g.scale * g.boost, g.inv), 0.0f), 15.0f) : 8.0f;
    return g;
}

template <bool ZERO>
__device__ __forceinline__ uint32_t encode(float w, const GroupScale& g) {
    const float q = rint_quotient(w * g.boost, g.scale * g.boost, g.inv);
    // Symmetric: amax / scale < 7.03, so -8 is only reached by an infinity.
    const float c = fminf(fmaxf(q + g.zero, 0.0f), 15.0f);
    return static_cast<uint32_t>(c);
}

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

// 8 consecutive elements from `at` on; zeros at and past `len`.
template <typename T>
__device__ __forceinline__ void load8(const T* row, int at, int len, bool vec, float (&v)[8]) {
    if (vec && at < len) {
        if constexpr (sizeof(T) == 4) {
            const float4 a = __ldg(reinterpret_cast<const float4*>(row + at));
            const float4 b = __ldg(reinterpret_cast<const float4*>(row + at) + 1);
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else {
            const uint4 u = __ldg(reinterpret_cast<const uint4*>(row + at));
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = bf16_lo(w[i]);
                v[2 * i + 1] = bf16_hi(w[i]);
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = at + i < len ? to_float<T>(row[at + i]) : 0.0f;
}

constexpr int kQuantThreads = 256;

// A warp takes 16 rows x 128 K at a time: two tiles, and whole groups of any size.  Lane 4 g + t
// reads rows g and g + 8, K 8 t .. 8 t + 7 of each 32: exactly the codes of its own 16 bytes, so
// nothing is exchanged but the extremes (two shuffles over t).  HBM-bound: w read once.
template <typename T, bool ZERO>
__global__ void __launch_bounds__(kQuantThreads) quantize_w4_kernel(const T* __restrict__ w, int N, int K, int row_blocks,
                                                                    int k_blocks, int groups, int group, bool vec,
                                                                    size_t items, uint8_t* __restrict__ q,
                                                                    uint32_t* __restrict__ scales,
                                                                    uint16_t* __restrict__ zeros) {
    const int lane = threadIdx.x & 31, g = lane / 4, t = lane & 3;
    const int k_pairs = (k_blocks + 1) / 2;
    const size_t warps = static_cast<size_t>(gridDim.x) * (kQuantThreads / 32);
    for (size_t item = static_cast<size_t>(blockIdx.x) * (kQuantThreads / 32) + threadIdx.x / 32; item < items;
         item += warps) {
        const size_t block = item / k_pairs;  // row block of the whole stack
        const int kp = static_cast<int>(item - block * k_pairs);
        const size_t matrix = block / row_blocks;
        const int row0 = static_cast<int>(block - matrix * row_blocks) * kTileRows + g;
        float v[2][4][8];  // [row g, g + 8][32 K][element]
#pragma unroll
        for (int rr = 0; rr < 2; ++rr) {
            const int row = row0 + 8 * rr;
            const T* src = w + (matrix * N + (row < N ? row : 0)) * K;
#pragma unroll
            for (int c = 0; c < 4; ++c) load8<T>(src, kp * 128 + 32 * c + 8 * t, row < N ? K : 0, vec, v[rr][c]);
        }
        float lo[2][4], hi[2][4];
#pragma unroll
        for (int rr = 0; rr < 2; ++rr) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                float l = 0.0f, h = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    l = fminf(l, v[rr][c][i]);
                    h = fmaxf(h, v[rr][c][i]);
                }
#pragma unroll
                for (int o = 1; o < 4; o <<= 1) {
                    l = fminf(l, __shfl_xor_sync(0xffffffffu, l, o));
                    h = fmaxf(h, __shfl_xor_sync(0xffffffffu, h, o));
                }
                lo[rr][c] = l;
                hi[rr][c] = h;
            }
        }
        const int per = group / 32;  // 32-K parts in a group: 1, 2 or 4
        uint32_t out[2][4] = {};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            GroupScale gs[2];
#pragma unroll
            for (int rr = 0; rr < 2; ++rr) {
                float l = lo[rr][c], h = hi[rr][c];
                if (per >= 2) l = fminf(l, lo[rr][c ^ 1]), h = fmaxf(h, hi[rr][c ^ 1]);
                if (per == 4) {
                    l = fminf(l, fminf(lo[rr][c ^ 2], lo[rr][c ^ 3]));
                    h = fmaxf(h, fmaxf(hi[rr][c ^ 2], hi[rr][c ^ 3]));
                }
                gs[rr] = group_scale<ZERO>(l, h);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    // element i: word 2 (c % 2) + i / 4, nibble 4 (i % 2) + 2 ((i % 4) / 2) + rr
                    const uint32_t code = encode<ZERO>(v[rr][c][i], gs[rr]);
                    out[c / 2][2 * (c & 1) + i / 4] |= code << (16 * (i & 1) + 8 * ((i & 3) / 2) + 4 * rr);
                }
            }
            const int k0 = kp * 128 + 32 * c;
            if (t == 0 && k0 % group == 0 && k0 < K) {
                const size_t at = (block * groups + k0 / group) * 8 + g;
                scales[at] = __float_as_uint(gs[0].scale) >> 16 | (__float_as_uint(gs[1].scale) & 0xFFFF0000u);
                if (ZERO) zeros[at] = static_cast<uint16_t>(static_cast<uint32_t>(gs[0].zero) | static_cast<uint32_t>(gs[1].zero) << 8);
            }
        }
#pragma unroll
        for (int tile = 0; tile < 2; ++tile) {
            const int kb = 2 * kp + tile;
            if (kb < k_blocks) {
                uint4* dst = reinterpret_cast<uint4*>(q + (block * k_blocks + kb) * kTileBytes) + lane;
                *dst = make_uint4(out[tile][0], out[tile][1], out[tile][2], out[tile][3]);
            }
        }
    }
}

// The inverse: (code - zero) * scale, exact in fp32, rounded once to T.  A warp takes one tile.
template <typename T, bool ZERO>
__global__ void __launch_bounds__(kQuantThreads) dequantize_w4_kernel(const uint8_t* __restrict__ q,
                                                                      const uint32_t* __restrict__ scales,
                                                                      const uint16_t* __restrict__ zeros, int N, int K,
                                                                      int row_blocks, int k_blocks, int groups,
                                                                      int group_shift, bool vec, size_t items,
                                                                      T* __restrict__ w) {
    const int lane = threadIdx.x & 31, g = lane / 4, t = lane & 3;
    const size_t warps = static_cast<size_t>(gridDim.x) * (kQuantThreads / 32);
    for (size_t item = static_cast<size_t>(blockIdx.x) * (kQuantThreads / 32) + threadIdx.x / 32; item < items;
         item += warps) {
        const size_t block = item / k_blocks;
        const int kb = static_cast<int>(item - block * k_blocks);
        const size_t matrix = block / row_blocks;
        const int row0 = static_cast<int>(block - matrix * row_blocks) * kTileRows + g;
        const uint4 u = load_stream(q + item * kTileBytes + lane * 16);
        const uint32_t words[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int k0 = kb * kTileK + 32 * c + 8 * t;
            if (k0 >= K) continue;
            const size_t at = (block * groups + (k0 >> group_shift)) * 8 + g;
            const uint32_t sc = __ldg(scales + at);
            const uint32_t z = ZERO ? __ldg(zeros + at) : 0x0808u;
#pragma unroll
            for (int rr = 0; rr < 2; ++rr) {
                const int row = row0 + 8 * rr;
                if (row >= N) continue;
                const float s = rr ? bf16_hi(sc) : bf16_lo(sc);
                const int zero = static_cast<int>(rr ? z >> 8 : z & 0xFFu);
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int code = (words[2 * c + i / 4] >> (16 * (i & 1) + 8 * ((i & 3) / 2) + 4 * rr)) & 15;
                    v[i] = static_cast<float>(code - zero) * s;
                }
                T* dst = w + (matrix * N + row) * K + k0;
                if (vec) {
                    if constexpr (sizeof(T) == 4) {
                        reinterpret_cast<float4*>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
                        reinterpret_cast<float4*>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
                    } else {
                        __nv_bfloat162 p[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) p[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                        *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<uint4*>(p);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        if (k0 + i >= K) break;
                        if constexpr (sizeof(T) == 4) dst[i] = v[i];
                        else dst[i] = __float2bfloat16_rn(v[i]);
                    }
                }
            }
        }
    }
}

// One wave of resident blocks at most.
template <auto KERNEL>
unsigned one_wave(size_t items, int sms, int dev) {
    const int per_sm = resident_ctas<KERNEL>(dev, kQuantThreads, 0);
    const size_t blocks = (items + kQuantThreads / 32 - 1) / (kQuantThreads / 32);
    const size_t cap = static_cast<size_t>(sms) * (per_sm > 0 ? per_sm : 1);
    return static_cast<unsigned>(blocks < cap ? blocks : cap);
}

template <typename T, bool ZERO>
int run_quantize(const T* w, int count, int N, int K, int group, bool vec, uint8_t* q, uint32_t* scales, uint16_t* zeros,
                 int sms, int dev, cudaStream_t stream) {
    const int rb = ceil_div(N, kTileRows), kb = ceil_div(K, kTileK);
    const size_t items = static_cast<size_t>(count) * rb * ceil_div(kb, 2);
    quantize_w4_kernel<T, ZERO><<<one_wave<quantize_w4_kernel<T, ZERO>>(items, sms, dev), kQuantThreads, 0, stream>>>(
        w, N, K, rb, kb, ceil_div(K, group), group, vec, items, q, scales, zeros);
    return cudaGetLastError() == cudaSuccess ? HGEMM_OK : HGEMM_ERR_CUDA;
}

template <typename T, bool ZERO>
int run_dequantize(const uint8_t* q, const uint32_t* scales, const uint16_t* zeros, int count, int N, int K, int group,
                   bool vec, T* w, int sms, int dev, cudaStream_t stream) {
    const Weight v = make_weight(q, scales, zeros, N, K, group);
    const size_t items = static_cast<size_t>(count) * v.row_blocks * v.k_blocks;
    dequantize_w4_kernel<T, ZERO><<<one_wave<dequantize_w4_kernel<T, ZERO>>(items, sms, dev), kQuantThreads, 0, stream>>>(
        q, scales, zeros, N, K, v.row_blocks, v.k_blocks, v.groups, v.group_shift, vec, items, w);
    return cudaGetLastError() == cudaSuccess ? HGEMM_OK : HGEMM_ERR_CUDA;
}

// ---- y[M, N] = x[M, K] . W[N, K]^T for few rows -----------------------------------------------
//
// The weights are the A operand (16 rows of W a tile), up to 8 NT rows of x the columns.  A CTA
// takes R row blocks; its 8 warps split K, and a cluster of `split` CTAs splits it again where
// there are too few row blocks for the GPU.  The partial sums are joined in a fixed order, over
// shared memory and then distributed shared memory: the bits do not depend on timing.

constexpr int kWarps = 8;

struct LinearParams {
    const void* x;
    long long ldx;
    void* y;
    int M, N, K;
    Weight w;
    bool vec;
};

template <typename T>
__device__ __forceinline__ void store(T* p, float v);
template <>
__device__ __forceinline__ void store<float>(float* p, float v) { *p = v; }
template <>
__device__ __forceinline__ void store<__nv_bfloat16>(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// Shared memory: the warps' rings, and over them, once the products are done, their sums.
template <typename T, int R, int NT, int STAGES, int GROUP, bool ZERO>
struct LinearShape {
    using Product = WarpProduct<R, NT, STAGES, GROUP, ZERO, RowSource<T>>;
    static constexpr int kOut = R * NT * 128;  // a CTA's outputs: 16 R rows x 8 NT columns, in fragment order
    static constexpr int kRings = kWarps * Product::kWarpBytes, kSums = kWarps * kOut * 4;
    static constexpr int kSmem = kRings > kSums ? kRings : kSums;
};

template <typename T, int R, int NT, int STAGES, int GROUP, bool ZERO>
__global__ void __launch_bounds__(kWarps * 32) w4_linear_kernel(const LinearParams p) {
    using Shape = LinearShape<T, R, NT, STAGES, GROUP, ZERO>;
    constexpr int kOut = Shape::kOut;
    extern __shared__ __align__(16) uint8_t smem[];
    float* partial = reinterpret_cast<float*>(smem);  // [warp][kOut]
    cg::cluster_group cluster = cg::this_cluster();
    const int split = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    const int block0 = static_cast<int>(blockIdx.x) / split * R, col0 = static_cast<int>(blockIdx.y) * 8 * NT;

    typename Shape::Product product;
#pragma unroll
    for (int r = 0; r < R; ++r) product.set_rows(r, p.w, 0, min(block0 + r, p.w.row_blocks - 1), lane);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        // Columns past M repeat the last row; their sums are not stored.
        const int col = min(col0 + 8 * n + lane / 4, p.M - 1);
        product.x[n] = {static_cast<const T*>(p.x) + col * p.ldx + 8 * (lane & 3), p.K - 8 * (lane & 3), p.vec};
    }
    product.set_columns(p.vec ? p.K : 0);
    const int steps = ceil_div(p.w.k_blocks, 2), parts = split * kWarps, part = rank * kWarps + warp;
    const int s0 = static_cast<int>(static_cast<long long>(steps) * part / parts);
    const int s1 = static_cast<int>(static_cast<long long>(steps) * (part + 1) / parts);
    float acc[R][NT][4] = {};
    pdl_trigger();
    pdl_wait();
    product.run(smem + warp * Shape::Product::kWarpBytes, s0, s1, lane, acc);

    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) partial[warp * kOut + ((r * NT + n) * 4 + i) * 32 + lane] = acc[r][n][i];
    __syncthreads();
    auto finish = [&](int i, float v) {
        const int l = i & 31, f = (i >> 5) & 3, n = (i >> 7) % NT, r = (i >> 7) / NT;
        const int row = (block0 + r) * 16 + l / 4 + 8 * (f >> 1), col = col0 + 8 * n + 2 * (l & 3) + (f & 1);
        if (row < p.N && col < p.M) store<T>(static_cast<T*>(p.y) + static_cast<size_t>(col) * p.N + row, v);
    };
    for (int i = threadIdx.x; i < kOut; i += kWarps * 32) {
        float v = partial[i];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) v += partial[w * kOut + i];
        if (split == 1) finish(i, v);
        else partial[i] = v;
    }
    if (split > 1) {
        cluster.sync();
        for (int i = rank * kWarps * 32 + threadIdx.x; i < kOut; i += split * kWarps * 32) {
            float v = 0.0f;
            for (int s = 0; s < split; ++s) v += cluster.map_shared_rank(partial, s)[i];
            finish(i, v);
        }
        cluster.sync();  // no CTA leaves while another reads its sums
    }
}

// CTAs of a cluster that share the K of a row group, for `groups` groups of rows: enough CTAs
// for two on every SM, as long as a warp keeps two steps.
inline int choose_split(int groups, int steps, int sms) {
    int split = 1;
    while (split < 8 && groups * split < 2 * sms && steps >= 2 * split * kWarps * 2) split *= 2;
    return split;
}

template <typename T, int R, int NT, int STAGES, int GROUP, bool ZERO>
int launch_linear(const LinearParams& p, int sms, int dev, cudaStream_t stream) {
    using Shape = LinearShape<T, R, NT, STAGES, GROUP, ZERO>;
    constexpr auto kernel = w4_linear_kernel<T, R, NT, STAGES, GROUP, ZERO>;
    if (resident_ctas<kernel>(dev, kWarps * 32, Shape::kSmem) < 1) return HGEMM_ERR_CUDA;
    const int groups = ceil_div(p.w.row_blocks, R), columns = ceil_div(p.M, 8 * NT);
    const int split = choose_split(groups * columns, ceil_div(p.w.k_blocks, 2), sms);
    return launch<kernel>(dim3(static_cast<unsigned>(groups) * split, static_cast<unsigned>(columns), 1), kWarps * 32, split,
                          Shape::kSmem, stream, p);
}

template <typename T, int GROUP, bool ZERO>
int run_linear(const LinearParams& p, int sms, int dev, cudaStream_t stream) {
    if constexpr (sizeof(T) == 4) {
        return launch_linear<T, 2, 1, 4, GROUP, ZERO>(p, sms, dev, stream);
    } else {
        if (p.M <= 8) return launch_linear<T, 2, 1, 4, GROUP, ZERO>(p, sms, dev, stream);
        if (p.M <= 16) return launch_linear<T, 2, 2, 4, GROUP, ZERO>(p, sms, dev, stream);
        return launch_linear<T, 2, 4, 4, GROUP, ZERO>(p, sms, dev, stream);
    }
}

// The checks that every entry point makes of a blocked weight.  The products copy zero points 4 bytes at a time.
inline int check_weight(const void* q, const void* scales, const void* zeros, unsigned zeros_align) {
    if (!q || !scales) return HGEMM_ERR_INVALID_VALUE;
    if (misaligned(q, 16) || misaligned(scales, 4) || misaligned(zeros, zeros_align)) return HGEMM_ERR_ALIGNMENT;
    return HGEMM_OK;
}

}  // namespace hgw

extern "C" {

size_t hgemm_w4_q_bytes(int N, int K) {
    if (N <= 0 || K <= 0) return 0;
    return static_cast<size_t>(hgw::ceil_div(N, hgw::kTileRows)) * hgw::ceil_div(K, hgw::kTileK) * hgw::kTileBytes;
}

size_t hgemm_w4_scales(int N, int K, int group) {
    if (N <= 0 || K <= 0 || !hgw::valid_group(group)) return 0;
    return static_cast<size_t>(hgw::ceil_div(N, hgw::kTileRows)) * hgw::ceil_div(K, group) * hgw::kTileRows;
}

int hgemm_quantize_w4(const void* w, int w_dtype, int count, int N, int K, int group, void* q, void* scales, void* zeros,
                      hgemm_stream_t stream) {
    if (count < 0 || N < 0 || K < 0 || !hgw::valid_group(group)) return HGEMM_ERR_INVALID_VALUE;
    if (w_dtype != HGEMM_DTYPE_F32 && w_dtype != HGEMM_DTYPE_BF16) return HGEMM_ERR_INVALID_VALUE;
    if (count == 0 || N == 0 || K == 0) return HGEMM_OK;
    if (!w) return HGEMM_ERR_INVALID_VALUE;
    if (int rc = hgw::check_weight(q, scales, zeros, 2)) return rc;
    const unsigned size = w_dtype == HGEMM_DTYPE_F32 ? 4 : 2;
    if (hgw::misaligned(w, size)) return HGEMM_ERR_ALIGNMENT;
    int sms = 0, dev = 0;
    if (int rc = hgw::current_device(&sms, &dev)) return rc;
    const bool vec = !hgw::misaligned(w, 16) && K % 8 == 0;
    const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    uint8_t* const qb = static_cast<uint8_t*>(q);
    uint32_t* const sc = static_cast<uint32_t*>(scales);
    uint16_t* const z = static_cast<uint16_t*>(zeros);
    auto go = [&](auto* typed) {
        return z ? hgw::run_quantize<std::remove_const_t<std::remove_pointer_t<decltype(typed)>>, true>(
                       typed, count, N, K, group, vec, qb, sc, z, sms, dev, s)
                 : hgw::run_quantize<std::remove_const_t<std::remove_pointer_t<decltype(typed)>>, false>(
                       typed, count, N, K, group, vec, qb, sc, z, sms, dev, s);
    };
    if (w_dtype == HGEMM_DTYPE_F32) return go(static_cast<const float*>(w));
    return go(static_cast<const __nv_bfloat16*>(w));
}

int hgemm_dequantize_w4(const void* q, const void* scales, const void* zeros, int count, int N, int K, int group, void* w,
                        int w_dtype, hgemm_stream_t stream) {
    if (count < 0 || N < 0 || K < 0 || !hgw::valid_group(group)) return HGEMM_ERR_INVALID_VALUE;
    if (w_dtype != HGEMM_DTYPE_F32 && w_dtype != HGEMM_DTYPE_BF16) return HGEMM_ERR_INVALID_VALUE;
    if (count == 0 || N == 0 || K == 0) return HGEMM_OK;
    if (!w) return HGEMM_ERR_INVALID_VALUE;
    if (int rc = hgw::check_weight(q, scales, zeros, 2)) return rc;
    const unsigned size = w_dtype == HGEMM_DTYPE_F32 ? 4 : 2;
    if (hgw::misaligned(w, size)) return HGEMM_ERR_ALIGNMENT;
    int sms = 0, dev = 0;
    if (int rc = hgw::current_device(&sms, &dev)) return rc;
    const bool vec = !hgw::misaligned(w, 16) && K % 8 == 0;
    const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const uint8_t* const qb = static_cast<const uint8_t*>(q);
    const uint32_t* const sc = static_cast<const uint32_t*>(scales);
    const uint16_t* const z = static_cast<const uint16_t*>(zeros);
    auto go = [&](auto* typed) {
        using T = std::remove_pointer_t<decltype(typed)>;
        return z ? hgw::run_dequantize<T, true>(qb, sc, z, count, N, K, group, vec, typed, sms, dev, s)
                 : hgw::run_dequantize<T, false>(qb, sc, z, count, N, K, group, vec, typed, sms, dev, s);
    };
    if (w_dtype == HGEMM_DTYPE_F32) return go(static_cast<float*>(w));
    return go(static_cast<__nv_bfloat16*>(w));
}

int hgemm_w4_gemm_tn(const void* x, int x_dtype, long long ldx, const void* q, const void* scales, const void* zeros,
                     void* y, int M, int N, int K, int group, hgemm_stream_t stream) {
    if (M < 0 || N < 0 || K < 0 || !hgw::valid_group(group)) return HGEMM_ERR_INVALID_VALUE;
    if (x_dtype != HGEMM_DTYPE_F32 && x_dtype != HGEMM_DTYPE_BF16) return HGEMM_ERR_INVALID_VALUE;
    if (M > 1 && ldx < K) return HGEMM_ERR_INVALID_VALUE;
    if (M == 0 || N == 0) return HGEMM_OK;
    if (!y) return HGEMM_ERR_INVALID_VALUE;
    const unsigned size = x_dtype == HGEMM_DTYPE_F32 ? 4 : 2;
    if (hgw::misaligned(y, size)) return HGEMM_ERR_ALIGNMENT;
    const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    int sms = 0, dev = 0;
    if (K == 0) {
        if (int rc = hgw::current_device(&sms, &dev)) return rc;
        const size_t bytes = static_cast<size_t>(M) * N * size;
        return cudaMemsetAsync(y, 0, bytes, s) == cudaSuccess ? HGEMM_OK : HGEMM_ERR_CUDA;
    }
    if (!x) return HGEMM_ERR_INVALID_VALUE;
    if (int rc = hgw::check_weight(q, scales, zeros, 4)) return rc;
    if (hgw::misaligned(x, size)) return HGEMM_ERR_ALIGNMENT;
    if (int rc = hgw::current_device(&sms, &dev)) return rc;
    if (M > 65535 * 8) return HGEMM_ERR_UNSUPPORTED;  // grid.y
    hgw::LinearParams p{x, M > 1 ? ldx : 0, y, M, N, K, hgw::make_weight(q, scales, zeros, N, K, group),
                        !hgw::misaligned(x, 16) && K % 8 == 0 && (M == 1 || ldx % (16 / size) == 0)};
    return hgw::with_format(group, zeros != nullptr, [&](auto g, auto z) {
        constexpr int G = decltype(g)::value;
        constexpr bool Z = decltype(z)::value;
        return x_dtype == HGEMM_DTYPE_F32 ? hgw::run_linear<float, G, Z>(p, sms, dev, s)
                                          : hgw::run_linear<__nv_bfloat16, G, Z>(p, sms, dev, s);
    });
}

}  // extern "C"
