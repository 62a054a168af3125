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

// rint(w / s) for s > 0, limited to +-17, for any w: a product with the reciprocal is off by at
// most one, and w - q s (one rounding, monotonic) tells on which side of the half-step border,
// which is representable, w lies.  Ties go to the even code.
__device__ __forceinline__ float rint_quotient(float w, float s, float inv) {
    float q = rintf(fminf(fmaxf(w * inv, -17.0f), 17.0f));
    const float e2 = 2.0f * fmaf(-q, s, w);
    const bool odd = (static_cast<int>(q) & 1) != 0;
    if (e2 > s || (e2 == s && odd)) q += 1.0f;
    if (e2 < -s || (e2 == -s && odd)) q -= 1.0f;
    return w == w ? q : 0.0f;
}

struct GroupScale {
    float scale, inv, zero;  // inv = 1 / (scale * boost()); zero is 8 for symmetric
    // w and scale are taken times this power of two where scale is tiny.
    __device__ __forceinline__ float boost() const { return scale < 0x1p-60f ? 0x1p80f : 1.0f; }
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
    g.inv = __frcp_rn(g.scale * g.boost());
    g.zero = ZERO ? fminf(fmaxf(rint_quotient(-lo * g.boost(), g.scale * g.boost(), g.inv), 0.0f), 15.0f) : 8.0f;
    return g;
}

// 8 consecutive elements from `at` on; zeros at and past `len`.
template <typename T>
__device__ __forceinline__ void load8(const T* row, int at, int len, float (&v)[8]) {
    if (at >= len) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    } else if constexpr (sizeof(T) == 4) {
        const float4 a = *reinterpret_cast<const float4*>(row + at);
        const float4 b = reinterpret_cast<const float4*>(row + at)[1];
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
        const uint4 u = *reinterpret_cast<const uint4*>(row + at);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = bf16_lo(w[i]);
            v[2 * i + 1] = bf16_hi(w[i]);
        }
    }
}

constexpr int kQuantThreads = 256;
constexpr int kQuantWarps = kQuantThreads / 32;
// Rows that are not 16-byte aligned go through shared memory: 16 rows x 64 K a warp, padded to 65 elements a row
// (68 would be aligned for wide accesses, but its 8-element accesses of 8 rows meet in the same banks).
constexpr int kPitch = 65;

template <typename T, bool VEC>
struct QuantSmem {
    static constexpr int kElements = VEC ? 1 : kQuantWarps * 16 * kPitch;
};

// The codes of 8 elements of two rows (g and g + 8): two words.  In the common case a quotient is the product with
// the reciprocal and one correction, which is the correctly rounded one (and exact where it is a tie), so that
// adding 1.5 * 2^23 rounds it as exact arithmetic would: always for bf16 (no other quotient of two bf16 is
// nearer than 2^-11 to a border), and for fp32 unless w - q s says otherwise.  The codes are put together as
// numbers, byte by byte, by FMAs.
template <typename T, bool ZERO>
__device__ __forceinline__ void encode8(const float (&w0)[8], const float (&w1)[8], const GroupScale& s0, const GroupScale& s1,
                                        bool regular, uint32_t (&out)[2]) {
    float c[2][8];
    if (regular) {
        float worst = 0.0f;
#pragma unroll
        for (int rr = 0; rr < 2; ++rr) {
            const GroupScale& g = rr ? s1 : s0;
            float far = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float w = rr ? w1[i] : w0[i];
                float q = w * g.inv;
                q = fmaf(fmaf(-q, g.scale, w), g.inv, q);
                q = (q + kMagic) - kMagic;
                if (sizeof(T) == 4) far = fmaxf(far, fabsf(fmaf(-q, g.scale, w)));
                c[rr][i] = ZERO ? fminf(fmaxf(q + g.zero, 0.0f), 15.0f) : q;
            }
            worst = fmaxf(worst, far - 0.5f * g.scale);
        }
        if (sizeof(T) == 4) regular = worst <= 0.0f;
    }
    if (!regular) {
#pragma unroll
        for (int rr = 0; rr < 2; ++rr) {
            const GroupScale& g = rr ? s1 : s0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float q = rint_quotient((rr ? w1[i] : w0[i]) * g.boost(), g.scale * g.boost(), g.inv);
                // Symmetric: amax / scale < 7.03, so -8 is only reached by an infinity.
                c[rr][i] = fminf(fmaxf(q + g.zero, 0.0f), 15.0f) - (ZERO ? 0.0f : 8.0f);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        float byte[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) byte[i] = fmaf(c[1][4 * j + i], 16.0f, c[0][4 * j + i]);
        // 2^23, and for symmetric codes 8 in each of the four places.
        constexpr float kBias = 8388608.0f + (ZERO ? 0.0f : 34952.0f);
        const uint32_t lo = __float_as_uint(fmaf(byte[2], 256.0f, byte[0]) + kBias);
        const uint32_t hi = __float_as_uint(fmaf(byte[3], 256.0f, byte[1]) + kBias);
        out[j] = __byte_perm(lo, hi, 0x5410);
    }
}

// A warp takes 16 rows x 128 K at a time: two tiles, and whole groups of any size.  Lane 4 g + t
// has rows g and g + 8, K 8 t .. 8 t + 7 of each 32: exactly the codes of its own 16 bytes, so
// nothing is exchanged but the extremes (two shuffles over t) and the scales, of which lane t
// works out those of group t.  HBM-bound in the main: w is read once; about 8 instructions an element.
// 28672 x 8192 bf16 to codes and back takes 241 us, 4.9 TB/s of the two kernels' traffic (a division an
// element made it 697); 4999 x 5115 fp32, whose rows go through shared memory, 72 us (scalar loads 211).
template <typename T, bool ZERO, int GROUP, bool VEC>
__global__ void __launch_bounds__(kQuantThreads) quantize_w4_kernel(const T* w, int N, int K, int row_blocks, int k_blocks,
                                                                    int groups, unsigned items, uint8_t* q,
                                                                    uint32_t* scales, uint16_t* zeros) {
    __shared__ T staged[QuantSmem<T, VEC>::kElements];
    constexpr int kGroups = 128 / GROUP, kParts = GROUP / 32;
    const int lane = threadIdx.x & 31, g = lane / 4, t = lane & 3;
    const unsigned k_pairs = (k_blocks + 1) / 2, warps = gridDim.x * kQuantWarps;
    pdl_trigger();
    pdl_wait();
    for (unsigned item = blockIdx.x * kQuantWarps + threadIdx.x / 32; item < items; item += warps) {
        const unsigned block = item / k_pairs;  // row block of the whole stack
        const int kp = static_cast<int>(item - block * k_pairs);
        const unsigned matrix = block / row_blocks;
        const int row0 = static_cast<int>(block - matrix * row_blocks) * kTileRows;
        const T* from = w + (static_cast<size_t>(matrix) * N + row0) * K + kp * 128;
        float v[2][4][8];  // [row g, g + 8][32 K][element]
        if constexpr (VEC) {
#pragma unroll
            for (int rr = 0; rr < 2; ++rr) {
                const int r = g + 8 * rr;
                const T* src = from + static_cast<size_t>(row0 + r < N ? r : 0) * K;
#pragma unroll
                for (int c = 0; c < 4; ++c) load8<T>(src, 32 * c + 8 * t, row0 + r < N ? K - kp * 128 : 0, v[rr][c]);
            }
        } else {
            T* tile = staged + threadIdx.x / 32 * (16 * kPitch);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int left = K - kp * 128 - 64 * half;
                T e[16][2];
#pragma unroll
                for (int r = 0; r < 16; ++r)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        e[r][i] = row0 + r < N && lane + 32 * i < left ? from[static_cast<size_t>(r) * K + 64 * half + lane + 32 * i] : T(0.0f);
                __syncwarp();
#pragma unroll
                for (int r = 0; r < 16; ++r)
#pragma unroll
                    for (int i = 0; i < 2; ++i) tile[r * kPitch + lane + 32 * i] = e[r][i];
                __syncwarp();
#pragma unroll
                for (int rr = 0; rr < 2; ++rr)
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            v[rr][2 * half + c][i] = static_cast<float>(tile[(g + 8 * rr) * kPitch + 32 * c + 8 * t + i]);
            }
        }
        // Extremes of the groups; with a NaN among them, fmax and fmin leave it out and `nan` is not 0.
        float lo[2][kGroups], hi[2][kGroups], nan = 0.0f;
#pragma unroll
        for (int rr = 0; rr < 2; ++rr) {
#pragma unroll
            for (int j = 0; j < kGroups; ++j) {
                float l = 0.0f, h = 0.0f;
#pragma unroll
                for (int c = j * kParts; c < (j + 1) * kParts; ++c)
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float e = v[rr][c][i];
                        if (ZERO) {
                            l = fminf(l, e);
                            h = fmaxf(h, e);
                        } else {
                            h = fmaxf(h, fabsf(e));
                        }
                        nan = fmaf(e, 0.0f, nan);  // an infinity or a NaN makes it NaN
                    }
#pragma unroll
                for (int o = 1; o < 4; o <<= 1) {
                    if (ZERO) l = fminf(l, __shfl_xor_sync(0xffffffffu, l, o));
                    h = fmaxf(h, __shfl_xor_sync(0xffffffffu, h, o));
                }
                lo[rr][j] = l;
                hi[rr][j] = h;
            }
        }
        GroupScale mine[2];
#pragma unroll
        for (int rr = 0; rr < 2; ++rr) {
            float l = lo[rr][0], h = hi[rr][0];
#pragma unroll
            for (int j = 1; j < kGroups; ++j)
                if (t % kGroups == j) l = lo[rr][j], h = hi[rr][j];
            mine[rr] = group_scale<ZERO>(l, h);
        }
        if (t < kGroups && kp * 128 + t * GROUP < K) {
            const size_t at = (static_cast<size_t>(block) * groups + kp * kGroups + t) * 8 + g;
            scales[at] = __float_as_uint(mine[0].scale) >> 16 | (__float_as_uint(mine[1].scale) & 0xFFFF0000u);
            if (ZERO) zeros[at] = static_cast<uint16_t>(static_cast<uint32_t>(mine[0].zero) | static_cast<uint32_t>(mine[1].zero) << 8);
        }
        uint32_t out[2][4];
#pragma unroll
        for (int j = 0; j < kGroups; ++j) {
            GroupScale gs[2];
#pragma unroll
            for (int rr = 0; rr < 2; ++rr) {
                const int from_lane = (lane & ~3) + j;
                gs[rr].scale = kGroups == 1 ? mine[rr].scale : __shfl_sync(0xffffffffu, mine[rr].scale, from_lane);
                gs[rr].inv = kGroups == 1 ? mine[rr].inv : __shfl_sync(0xffffffffu, mine[rr].inv, from_lane);
                gs[rr].zero = !ZERO ? 8.0f : kGroups == 1 ? mine[rr].zero : __shfl_sync(0xffffffffu, mine[rr].zero, from_lane);
            }
            // Beyond 2^100 the correction's products could overflow.
            const bool regular = nan == 0.0f && fminf(gs[0].scale, gs[1].scale) >= 0x1p-60f && fmaxf(gs[0].scale, gs[1].scale) <= 0x1p100f;
#pragma unroll
            for (int c = j * kParts; c < (j + 1) * kParts; ++c) {
                uint32_t words[2];
                encode8<T, ZERO>(v[0][c], v[1][c], gs[0], gs[1], regular, words);
                out[c / 2][2 * (c & 1)] = words[0];
                out[c / 2][2 * (c & 1) + 1] = words[1];
            }
        }
#pragma unroll
        for (int tile = 0; tile < 2; ++tile) {
            const int kb = 2 * kp + tile;
            if (kb < k_blocks) {
                uint4* dst = reinterpret_cast<uint4*>(q + (static_cast<size_t>(block) * k_blocks + kb) * kTileBytes) + lane;
                *dst = make_uint4(out[tile][0], out[tile][1], out[tile][2], out[tile][3]);
            }
        }
    }
}

// The inverse: (code - zero) * scale, exact in fp32, rounded once to T.  A warp takes one tile.
// For bf16 the codes are unpacked as the products do it, two at a time, and multiplied by the
// scale in bf16, which rounds the exact product once: the same value.
template <typename T, bool ZERO, bool VEC>
__global__ void __launch_bounds__(kQuantThreads) dequantize_w4_kernel(const uint8_t* q, const uint32_t* scales,
                                                                      const uint16_t* zeros, int N, int K,
                                                                      int row_blocks, int k_blocks, int groups,
                                                                      int group_shift, unsigned items, T* w) {
    __shared__ T staged[QuantSmem<T, VEC>::kElements];
    const int lane = threadIdx.x & 31, g = lane / 4, t = lane & 3;
    const unsigned warps = gridDim.x * kQuantWarps;
    const UnpackConstants constants;
    pdl_trigger();
    pdl_wait();
    for (unsigned item = blockIdx.x * kQuantWarps + threadIdx.x / 32; item < items; item += warps) {
        const unsigned block = item / k_blocks;
        const int kb = static_cast<int>(item - block * k_blocks);
        const unsigned matrix = block / row_blocks;
        const int row0 = static_cast<int>(block - matrix * row_blocks) * kTileRows;
        const uint4 u = load_stream(q + static_cast<size_t>(item) * kTileBytes + lane * 16);
        const uint32_t words[4] = {u.x, u.y, u.z, u.w};
        T* to = w + (static_cast<size_t>(matrix) * N + row0) * K + kb * kTileK;
        const int left = K - kb * kTileK;
        T* tile = staged + threadIdx.x / 32 * (VEC ? 0 : 16 * kPitch);
        if (!VEC) __syncwarp();
        uint32_t half_scales[2], half_zeros[2];  // of both halves before the first store
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            int group = (kb * kTileK + 32 * c) >> group_shift;
            group = group < groups ? group : groups - 1;
            const size_t at = (static_cast<size_t>(block) * groups + group) * 8 + g;
            half_scales[c] = scales[at];
            half_zeros[c] = ZERO ? zeros[at] : 0x0808u;
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int k0 = 32 * c + 8 * t;
            const uint32_t sc = half_scales[c], z = half_zeros[c];
            uint32_t a[2][4];
#pragma unroll
            for (int j = 0; j < 2; ++j)
                unpack(words[2 * c + j], constants, __byte_perm(z, 0x43u, 0x4040), __byte_perm(z, 0x43u, 0x4141), a[j]);
#pragma unroll
            for (int rr = 0; rr < 2; ++rr) {
                const uint32_t pairs[4] = {a[0][rr], a[0][2 + rr], a[1][rr], a[1][2 + rr]};
                __align__(16) T v[8];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (sizeof(T) == 4) {
                        const float s = rr ? bf16_hi(sc) : bf16_lo(sc);
                        v[2 * i] = bf16_lo(pairs[i]) * s;
                        v[2 * i + 1] = bf16_hi(pairs[i]) * s;
                    } else {
                        const uint32_t s = __byte_perm(sc, 0u, rr ? 0x3232 : 0x1010);
                        asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(reinterpret_cast<uint32_t*>(v)[i]) : "r"(pairs[i]), "r"(s));
                    }
                }
                const int r = g + 8 * rr;
                if constexpr (VEC) {
                    if (row0 + r < N && k0 < left) {
                        uint4* dst = reinterpret_cast<uint4*>(to + static_cast<size_t>(r) * K + k0);
#pragma unroll
                        for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) dst[i] = reinterpret_cast<uint4*>(v)[i];
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) tile[r * kPitch + k0 + i] = v[i];
                }
            }
        }
        if constexpr (!VEC) {
            __syncwarp();
#pragma unroll
            for (int r = 0; r < 16; ++r)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    if (row0 + r < N && lane + 32 * i < left) to[static_cast<size_t>(r) * K + lane + 32 * i] = tile[r * kPitch + lane + 32 * i];
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

template <typename T, bool ZERO, int GROUP, bool VEC>
int launch_quantize(const T* w, int count, int N, int K, uint8_t* q, uint32_t* scales, uint16_t* zeros, int sms, int dev,
                    cudaStream_t stream) {
    const int rb = ceil_div(N, kTileRows), kb = ceil_div(K, kTileK);
    const size_t items = static_cast<size_t>(count) * rb * ceil_div(kb, 2);
    if (items > 0x7FFFFFFFu) return HGEMM_ERR_UNSUPPORTED;  // 2^31 x 2048 elements
    constexpr auto kernel = quantize_w4_kernel<T, ZERO, GROUP, VEC>;
    return launch<kernel>(dim3(one_wave<kernel>(items, sms, dev)), kQuantThreads, 1, 0, stream, w, N, K, rb, kb, ceil_div(K, GROUP),
                          static_cast<unsigned>(items), q, scales, zeros);
}

template <typename T>
int run_quantize(const T* w, int count, int N, int K, int group, uint8_t* q, uint32_t* scales, uint16_t* zeros, int sms,
                 int dev, cudaStream_t stream) {
    const bool vec = !misaligned(w, 16) && K % 8 == 0;
    return with_format(group, zeros != nullptr, [&](auto g, auto z) {
        constexpr int G = decltype(g)::value;
        constexpr bool Z = decltype(z)::value;
        return vec ? launch_quantize<T, Z, G, true>(w, count, N, K, q, scales, zeros, sms, dev, stream)
                   : launch_quantize<T, Z, G, false>(w, count, N, K, q, scales, zeros, sms, dev, stream);
    });
}

template <typename T, bool ZERO, bool VEC>
int launch_dequantize(const Weight& v, int count, int N, int K, T* w, int sms, int dev, cudaStream_t stream) {
    const size_t items = static_cast<size_t>(count) * v.row_blocks * v.k_blocks;
    if (items > 0x7FFFFFFFu) return HGEMM_ERR_UNSUPPORTED;
    constexpr auto kernel = dequantize_w4_kernel<T, ZERO, VEC>;
    return launch<kernel>(dim3(one_wave<kernel>(items, sms, dev)), kQuantThreads, 1, 0, stream, v.q, v.scales, v.zeros, N, K,
                          v.row_blocks, v.k_blocks, v.groups, v.group_shift, static_cast<unsigned>(items), w);
}

template <typename T>
int run_dequantize(const Weight& v, int count, int N, int K, T* w, int sms, int dev, cudaStream_t stream) {
    if (!misaligned(w, 16) && K % 8 == 0) {
        return v.zeros ? launch_dequantize<T, true, true>(v, count, N, K, w, sms, dev, stream)
                       : launch_dequantize<T, false, true>(v, count, N, K, w, sms, dev, stream);
    }
    return v.zeros ? launch_dequantize<T, true, false>(v, count, N, K, w, sms, dev, stream)
                   : launch_dequantize<T, false, false>(v, count, N, K, w, sms, dev, stream);
}

// ---- y[M, N] = x[M, K] . W[N, K]^T for few rows -----------------------------------------------
//
// The weights are the A operand (16 rows of W a tile), up to 8 NT rows of x the columns.  A CTA
// takes R row blocks; its warps split K, and a cluster of `split` CTAs splits it again where
// there are too few row blocks for the GPU.  The partial sums are joined in a fixed order, over
// shared memory and then distributed shared memory: the bits do not depend on timing.
// Two row blocks a warp and 3 stages were the best of 1, 2 and 4 by 3 and 4 (28672 x 8192 by one
// row: 34, against 36 with one block and 38 with four; by 16 rows 46, 58 and 58 us).

struct LinearParams {
    const void* x;
    long long ldx;
    void* y;
    int M, N, K;
    Weight w;
    bool vec;
    bool stall;  // hgemm_debug_stalled_w4
};

template <typename T>
__device__ __forceinline__ void store(T* p, float v);
template <>
__device__ __forceinline__ void store<float>(float* p, float v) { *p = v; }
template <>
__device__ __forceinline__ void store<__nv_bfloat16>(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// Shared memory: the warps' rings, and over them, once the products are done, their sums.
template <typename T, int R, int NT, int STAGES, int GROUP, bool ZERO, int WARPS>
struct LinearShape {
    using Product = WarpProduct<R, NT, STAGES, GROUP, ZERO, false, RowSource<T>>;
    static constexpr int kOut = R * NT * 128;  // a CTA's outputs: 16 R rows x 8 NT columns, in fragment order
    static constexpr int kRings = WARPS * Product::kWarpBytes, kSums = WARPS * kOut * 4;
    static constexpr int kSmem = kRings > kSums ? kRings : kSums;
};

template <typename T, int R, int NT, int STAGES, int GROUP, bool ZERO, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) w4_linear_kernel(const LinearParams p) {
    using Shape = LinearShape<T, R, NT, STAGES, GROUP, ZERO, WARPS>;
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
    const int steps = ceil_div(p.w.k_blocks, 2), parts = split * WARPS, part = rank * WARPS + warp;
    const int s0 = static_cast<int>(static_cast<unsigned>(steps) * part / parts);  // steps < 2^24, parts <= 64
    const int s1 = static_cast<int>(static_cast<unsigned>(steps) * (part + 1) / parts);
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
    for (int i = threadIdx.x; i < kOut; i += WARPS * 32) {
        float v = partial[i];
#pragma unroll
        for (int w = 1; w < WARPS; ++w) v += partial[w * kOut + i];
        if (split == 1) finish(i, v);
        else partial[i] = v;
    }
    if (split > 1) {
        cluster.sync();
        for (int i = rank * WARPS * 32 + threadIdx.x; i < kOut; i += split * WARPS * 32) {
            float v = 0.0f;
            for (int s = 0; s < split; ++s) v += cluster.map_shared_rank(partial, s)[i];
            finish(i, v);
        }
        cluster.sync();  // no CTA leaves while another reads its sums
    }
}

// CTAs of a cluster that share the K of a row group, for `groups` groups of rows: enough CTAs for two on every SM, as
// long as a warp keeps a step.  (With two steps at least, 8 rows of 4096 x 4096 took 7.0 us instead of 5.3, of
// 1024 x 8192 6.3 instead of 4.8; 16 of 1024 x 1024 2.6 instead of 3.2.)
inline int choose_split(int groups, int steps, int sms, int warps) {
    int split = 1;
    while (split < 8 && groups * split < 2 * sms && steps >= 2 * split * warps) split *= 2;
    return split;
}

template <typename T, int R, int NT, int STAGES, int GROUP, bool ZERO, int WARPS>
int launch_linear(const LinearParams& p, int sms, int dev, cudaStream_t stream) {
    using Shape = LinearShape<T, R, NT, STAGES, GROUP, ZERO, WARPS>;
    constexpr auto kernel = w4_linear_kernel<T, R, NT, STAGES, GROUP, ZERO, WARPS>;
    if (resident_ctas<kernel>(dev, WARPS * 32, Shape::kSmem) < 1) return HGEMM_ERR_CUDA;
    const int groups = ceil_div(p.w.row_blocks, R), columns = ceil_div(p.M, 8 * NT);
    const int split = choose_split(groups * columns, ceil_div(p.w.k_blocks, 2), sms, WARPS);
    return launch<kernel>(dim3(static_cast<unsigned>(groups) * split, static_cast<unsigned>(columns), 1), WARPS * 32, split,
                          Shape::kSmem, stream, p);
}

// ---- the same for one or two rows, or rows of fp32, x held in registers ---------------------------
//
// A persistent grid, one CTA an SM: a cluster of `split` CTAs takes a range of row blocks, its warps
// a slice of K each for all of them, so that x is read and turned into whole numbers once per warp
// and codes are all that streams: 62 instructions a tile instead of 88.  28672 x 8192 by one row takes
// 24.8 us (4.9 TB/s) instead of 34; what is left is start and end (4.5 us for 7168 x 2048, most of it
// launch, the planes and the first bytes' latency).  W is read once per two rows, or 8 of fp32.  After
// every kBatch row blocks the warps' sums are added up in shared memory, then the CTAs' in distributed
// shared memory, in a fixed order.

constexpr int kRowsWarps = 16;

template <typename T, int MT, int XS, int GROUP, bool ZERO>
struct RowsShape {
    using One = WarpStationary<T, MT, XS, 1, GROUP, ZERO>;
    static constexpr int kBatch = MT == 0 ? 8 : 2;
    static constexpr int kBatchFloats = kBatch * kRowsWarps * One::kResult;  // [row block][warp][kResult]
    static constexpr int kExchange = kBatch * 16 * One::kColumns;       // a CTA's sums: [column][row block][row]
    static constexpr int kSums = 2 * (kBatchFloats + kExchange) * 4;
    // 10 KB of codes and scales a warp are in flight or in use, 160 KB an SM; less where x takes the room.
    static constexpr int kRoom = (227 * 1024 - kSums) / kRowsWarps - (One::kWarpBytes - One::kStageBytes);
    static constexpr int kStages = (kRoom < 10240 ? kRoom : 10240) / One::kStageBytes;
    static_assert(kStages >= 2, "a stage ahead");
    using Product = WarpStationary<T, MT, XS, kStages, GROUP, ZERO>;
    static constexpr int kRings = kRowsWarps * Product::kWarpBytes;
    static constexpr int kSmem = kRings + kSums;
};

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

template <typename T, int MT, int XS, int GROUP, bool ZERO>
__global__ void __launch_bounds__(kRowsWarps * 32, 1) w4_rows_kernel(const LinearParams p) {
    using Shape = RowsShape<T, MT, XS, GROUP, ZERO>;
    using Product = typename Shape::Product;
    constexpr int kStages = Shape::kStages, kBatch = Shape::kBatch, kThreads = kRowsWarps * 32;
    extern __shared__ __align__(16) uint8_t smem[];
    float* partial = reinterpret_cast<float*>(smem + Shape::kRings);
    float* exchange = partial + 2 * Shape::kBatchFloats;
    cg::cluster_group cluster = cg::this_cluster();
    const int split = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
    const int clusters = static_cast<int>(gridDim.x) / split, id = static_cast<int>(blockIdx.x) / split;
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    const int col0 = static_cast<int>(blockIdx.y) * Product::kColumns, columns = min(Product::kColumns, p.M - col0);
    const int begin = static_cast<int>(static_cast<long long>(p.w.row_blocks) * id / clusters);
    const int end = static_cast<int>(static_cast<long long>(p.w.row_blocks) * (id + 1) / clusters);

    Product product;
    product.set_slice(smem + warp * Product::kWarpBytes, (rank * kRowsWarps + warp) * 2 * XS, p.w.k_blocks, lane);
#pragma unroll
    for (int m = 0; m < Product::kRowTiles; ++m) {
        // Columns past M repeat the last row; their sums are not stored.
        const int row = min(col0 + (Product::kPacked ? lane / 16 : 8 * m + lane / 4), p.M - 1), k = 8 * (lane & 3);
        product.x.tile[m] = {static_cast<const T*>(p.x) + row * p.ldx + k, p.K - k, p.vec};
    }
    auto copy = [&](int block, int stage) {
        const size_t groups_at = p.w.group_base(0, block);
        product.copy(stage, p.w.q + p.w.tile_base(0, block) + lane * 16,
                     reinterpret_cast<const uint8_t*>(p.w.scales + groups_at),
                     reinterpret_cast<const uint8_t*>(p.w.zeros + groups_at), p.w.groups, lane);
    };
    uint32_t flip, high;  // in registers, as UnpackConstants
    asm volatile("mov.b32 %0, 0x88888888;\n\tmov.b32 %1, 0xF0F0F0F0;" : "=r"(flip), "=r"(high));
    pdl_trigger();
    pdl_wait();
#pragma unroll
    for (int d = 0; d < kStages - 1; ++d) {
        if (begin + d < end) copy(begin + d, d);
        copy_commit();
    }
    product.convert(p.vec ? p.K / kTileK : 0, lane);

    auto finish = [&](int base, int column, int r, float v) {
        const int row = base * 16 + r;
        if (row < p.N) store<T>(static_cast<T*>(p.y) + static_cast<size_t>(col0 + column) * p.N + row, v);
    };
    auto gather = [&](float* sums, int base, int batch) {
        for (int i = rank * kThreads + threadIdx.x; i < columns * batch * 16; i += split * kThreads) {
            float v = 0.0f;
            for (int s = 0; s < split; ++s) v += cluster.map_shared_rank(sums, s)[i];
            finish(base, i / (batch * 16), i % (batch * 16), v);
        }
    };
    int stage = 0, buffer = 0;
    for (int base = begin; base < end; base += kBatch, buffer ^= 1) {
        const int batch = min(kBatch, end - base);
        float* sums = partial + buffer * Shape::kBatchFloats;
        for (int i = 0; i < batch; ++i) {
            const int ahead = base + i + kStages - 1;
            __syncwarp();  // all lanes are done with the stage that is filled next
            if (ahead < end) copy(ahead, stage == 0 ? kStages - 1 : stage - 1);
            copy_commit();
            copy_wait<kStages - 1>();
            __syncwarp();
            product.compute(stage, flip, high, sums + (i * kRowsWarps + warp) * Product::kResult, lane);
            stage = stage == kStages - 1 ? 0 : stage + 1;
        }
        __syncthreads();
        // Between CTAs one batch late, so that no CTA waits for another's sums: what the cluster wrote for the last
        // batch is added up after this batch's products.  A buffer's readers are done before they arrive for the
        // next batch, which is waited for before the buffer is written again.
        if (split > 1 && base > begin) {
            cluster_wait();
            gather(exchange + (buffer ^ 1) * Shape::kExchange, base - kBatch, kBatch);
        }
        float* out = exchange + buffer * Shape::kExchange;
        for (int i = threadIdx.x; i < columns * batch * 16; i += kThreads) {
            const int column = i / (batch * 16), r = i - column * (batch * 16);
            const float* from = sums + r / 16 * (kRowsWarps * Product::kResult) + column * Product::kSumStride + r % 16;
            float v = from[0];
#pragma unroll
            for (int w = 1; w < kRowsWarps; ++w) v += from[w * Product::kResult];
            if (split == 1) finish(base, column, r, v);
            else out[i] = v;
        }
        if (split > 1) cluster_arrive();
    }
    copy_wait<0>();
    if (split > 1 && begin < end) {
        cluster_wait();
        const int last = (end - begin - 1) / kBatch * kBatch;
        gather(exchange + (buffer ^ 1) * Shape::kExchange, begin + last, end - begin - last);
    }
    if (split > 1) cluster.sync();  // no CTA leaves while another reads its sums
}

// How the kernel above is laid over the GPU: CTAs of a cluster, steps of 128 K a warp holds.
struct RowsPlan {
    int split = 0, steps = 0, clusters = 0;
    long long cost = 0;
};

// Clusters of `split` CTAs, one an SM, that the device keeps resident: a cluster lies in one GPC, so that fewer
// than SMs / split fit (B200: 74 of 2, 33 of 4).  Every instance of the kernel fills an SM alike.
int resident_clusters(int split, int sms, int dev) {
    static std::atomic<int> known[kMaxDevices][4];
    if (split == 1) return sms;
    std::atomic<int>& slot = known[dev][split / 2];
    int n = slot.load(std::memory_order_relaxed);
    if (n == 0) {
        constexpr auto kernel = w4_rows_kernel<__nv_bfloat16, 0, 1, 128, false>;
        constexpr int smem = RowsShape<__nv_bfloat16, 0, 1, 128, false>::kSmem;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(static_cast<unsigned>(sms / split * split), 1, 1);
        cfg.blockDim = dim3(512, 1, 1);
        cfg.dynamicSmemBytes = smem;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = static_cast<unsigned>(split);
        attr.val.clusterDim.y = 1;
        attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        if (resident_ctas<kernel>(dev, 512, smem) < 1 || cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1) {
            cudaGetLastError();
            return 0;
        }
        slot.store(n, std::memory_order_relaxed);
    }
    return n;
}

// Candidate `split`, for warps that may hold up to `most` steps.  The cost is a warp's steps from begin to end, two
// for each step of x that it turns into planes, and one for the exchange between CTAs (8192 x 8192 by one row: 13.0
// us for 1 CTA, 10.8 for 2 and 12.9 for 4; 28672 x 8192: 25.3, 24.8, 33).
inline RowsPlan rows_plan(int row_blocks, int steps, int split, int clusters, int warps, int most) {
    RowsPlan plan;
    int held = ceil_div(steps, split * warps);
    held = held == 3 ? 4 : held;  // built for 1, 2 and 4
    if (held > most || clusters < 1) return plan;
    plan.split = split;
    plan.steps = held;
    plan.clusters = clusters < row_blocks ? clusters : row_blocks;
    plan.cost = static_cast<long long>(ceil_div(row_blocks, plan.clusters) + 2) * held + (split > 1 ? 1 : 0);
    return plan;
}

template <typename T, int MT, int XS, int GROUP, bool ZERO>
int launch_rows(const LinearParams& p, const RowsPlan& plan, int dev, cudaStream_t stream) {
    using Shape = RowsShape<T, MT, XS, GROUP, ZERO>;
    constexpr auto kernel = w4_rows_kernel<T, MT, XS, GROUP, ZERO>;
    static_assert(Shape::kSmem <= 227 * 1024, "shared memory of a CTA");
    if (resident_ctas<kernel>(dev, kRowsWarps * 32, Shape::kSmem) < 1) return HGEMM_ERR_CUDA;
    const unsigned columns = static_cast<unsigned>(ceil_div(p.M, Shape::Product::kColumns));
    return launch<kernel>(dim3(static_cast<unsigned>(plan.clusters * plan.split), columns, 1), kRowsWarps * 32, plan.split,
                          Shape::kSmem, stream, p);
}

// Most steps that a warp's registers take: 8 registers a step and tile of planes.
template <int MT>
struct RowsLimits {
    static_assert(MT <= 1, "16 warps leave 128 registers a thread");
    static constexpr int kSteps = MT == 0 ? 4 : 2;
};

// False where the plan costs less than `least` (too little work to hold x for) or K is too long for the warps' registers.
template <typename T, int MT, int GROUP, bool ZERO>
bool run_rows(const LinearParams& p, int least, int sms, int dev, cudaStream_t stream, int* rc) {
    using Limits = RowsLimits<MT>;
    RowsPlan best;
    for (int split = 1; split <= 4; split *= 2) {
        const RowsPlan plan = rows_plan(p.w.row_blocks, ceil_div(p.w.k_blocks, 2), split, resident_clusters(split, sms, dev),
                                        kRowsWarps, Limits::kSteps);
        if (plan.split && (!best.split || plan.cost < best.cost)) best = plan;
    }
    if (!best.split || best.cost < least) return false;
    if (best.steps == 1) *rc = launch_rows<T, MT, 1, GROUP, ZERO>(p, best, dev, stream);
    else if (best.steps == 2) *rc = launch_rows<T, MT, 2, GROUP, ZERO>(p, best, dev, stream);
    else if constexpr (Limits::kSteps >= 4) *rc = launch_rows<T, MT, 4, GROUP, ZERO>(p, best, dev, stream);
    return true;
}

// w4_tc.cu
int run_tc(const void* x, long long ldx, void* y, int M, int N, int K, const Weight& w, int group, bool stall, int sms,
           int dev, cudaStream_t stream);

template <typename T, int GROUP, bool ZERO>
int run_linear(const LinearParams& p, int sms, int dev, cudaStream_t stream) {
    int rc = 0;
    if constexpr (sizeof(T) == 4) {
        // Three matrix instructions for the three terms of x, and making the terms: x held in registers is faster nearly
        // throughout (us here and there: 8192 x 8192 by 1 row 12.6 and 30.7, by 3 rows 19.6 and 31.2, by 16 45 and
        // 57; 4096 x 1024 by 3 4.7 and 6.7), but for the least work (1024 x 1024 by 1: 3.6 and 3.1).
        if (p.M <= 2 ? run_rows<T, 0, GROUP, ZERO>(p, 4, sms, dev, stream, &rc) : run_rows<T, 1, GROUP, ZERO>(p, 4, sms, dev, stream, &rc))
            return rc;
        return launch_linear<T, 2, 1, 3, GROUP, ZERO, 4>(p, sms, dev, stream);
    } else {
        // One or two rows: x held in registers pays where there is work enough (us here and there: 28672 x 8192 24.8 and
        // 34.3, 7168 x 2048 4.5 and 5.6, 4096 x 1024 3.9 and 2.8).  Three to eight rows take three times the integer
        // instructions: 8192 x 8192 16.5 and 12.7.
        if (p.M <= 2 && run_rows<T, 0, GROUP, ZERO>(p, 6, sms, dev, stream, &rc)) return rc;
        // The tensor cores from 17 rows on (us below and there, groups of 128, at 4096 x 4096, 8192 x 8192 and 28672 x 8192):
        // 9 rows 5.6 and 7.6, 15.1 and 16.6, 45.5 and 51.3; 16 rows 5.8 and 7.7, 15.4 and 16.9, 47.0 and 52.3 (8192 x
        // 8192 in groups of 64 20.0 and 18.0, of 32 with zero points 23.6 and 25.5); 17 rows, of the last two, 28.5 and
        // 16.9, 86.4 and 51.7; 64 rows 44.3 and 22.1, 153 and 68.2.
        if (p.M > 16 && p.vec) return run_tc(p.x, p.ldx, p.y, p.M, p.N, p.K, p.w, GROUP, p.stall, sms, dev, stream);
        if (p.M <= 8) return launch_linear<T, 2, 1, 3, GROUP, ZERO, 8>(p, sms, dev, stream);
        if (p.M <= 16) return launch_linear<T, 2, 2, 3, GROUP, ZERO, 4>(p, sms, dev, stream);
        return launch_linear<T, 2, 4, 3, GROUP, ZERO, 4>(p, sms, dev, stream);
    }
}

// The checks that every entry point makes of a blocked weight.  The products copy 16 bytes of scales
// and zero points at a time.
inline int check_weight(const void* q, const void* scales, const void* zeros, unsigned scales_align) {
    if (!q || !scales) return HGEMM_ERR_INVALID_VALUE;
    if (misaligned(q, 16) || misaligned(scales, scales_align) || misaligned(zeros, scales_align == 16 ? 16 : 2)) return HGEMM_ERR_ALIGNMENT;
    return HGEMM_OK;
}

}  // namespace hgw

namespace {

int gemm_w4(const void* x, int x_dtype, long long ldx, const void* q, const void* scales, const void* zeros, void* y, int M,
            int N, int K, int group, bool stall, hgemm_stream_t stream) {
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
    if (int rc = hgw::check_weight(q, scales, zeros, 16)) return rc;
    if (hgw::misaligned(x, size)) return HGEMM_ERR_ALIGNMENT;
    // CTAs read x while others write y.
    if (hgw::meets_rows(y, static_cast<size_t>(M) * N * size, x, M, ldx, K, size)) return HGEMM_ERR_INVALID_VALUE;
    if (int rc = hgw::current_device(&sms, &dev)) return rc;
    if (M > 65535 * 8) return HGEMM_ERR_UNSUPPORTED;  // grid.y
    hgw::LinearParams p{x, M > 1 ? ldx : 0, y, M, N, K, hgw::make_weight(q, scales, zeros, N, K, group),
                        !hgw::misaligned(x, 16) && K % 8 == 0 && (M == 1 || ldx % (16 / size) == 0), stall};
    return hgw::with_format(group, zeros != nullptr, [&](auto g, auto z) {
        constexpr int G = decltype(g)::value;
        constexpr bool Z = decltype(z)::value;
        return x_dtype == HGEMM_DTYPE_F32 ? hgw::run_linear<float, G, Z>(p, sms, dev, s)
                                          : hgw::run_linear<__nv_bfloat16, G, Z>(p, sms, dev, s);
    });
}

}  // namespace

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
    if (int rc = hgw::check_weight(q, scales, zeros, 4)) return rc;
    const unsigned size = w_dtype == HGEMM_DTYPE_F32 ? 4 : 2;
    if (hgw::misaligned(w, size)) return HGEMM_ERR_ALIGNMENT;
    int sms = 0, dev = 0;
    if (int rc = hgw::current_device(&sms, &dev)) return rc;
    const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    uint8_t* const qb = static_cast<uint8_t*>(q);
    uint32_t* const sc = static_cast<uint32_t*>(scales);
    uint16_t* const z = static_cast<uint16_t*>(zeros);
    if (w_dtype == HGEMM_DTYPE_F32) return hgw::run_quantize(static_cast<const float*>(w), count, N, K, group, qb, sc, z, sms, dev, s);
    return hgw::run_quantize(static_cast<const __nv_bfloat16*>(w), count, N, K, group, qb, sc, z, sms, dev, s);
}

int hgemm_dequantize_w4(const void* q, const void* scales, const void* zeros, int count, int N, int K, int group, void* w,
                        int w_dtype, hgemm_stream_t stream) {
    if (count < 0 || N < 0 || K < 0 || !hgw::valid_group(group)) return HGEMM_ERR_INVALID_VALUE;
    if (w_dtype != HGEMM_DTYPE_F32 && w_dtype != HGEMM_DTYPE_BF16) return HGEMM_ERR_INVALID_VALUE;
    if (count == 0 || N == 0 || K == 0) return HGEMM_OK;
    if (!w) return HGEMM_ERR_INVALID_VALUE;
    if (int rc = hgw::check_weight(q, scales, zeros, 4)) return rc;
    const unsigned size = w_dtype == HGEMM_DTYPE_F32 ? 4 : 2;
    if (hgw::misaligned(w, size)) return HGEMM_ERR_ALIGNMENT;
    int sms = 0, dev = 0;
    if (int rc = hgw::current_device(&sms, &dev)) return rc;
    const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const hgw::Weight v = hgw::make_weight(q, scales, zeros, N, K, group);
    if (w_dtype == HGEMM_DTYPE_F32) return hgw::run_dequantize(v, count, N, K, static_cast<float*>(w), sms, dev, s);
    return hgw::run_dequantize(v, count, N, K, static_cast<__nv_bfloat16*>(w), sms, dev, s);
}

int hgemm_w4_gemm_tn(const void* x, int x_dtype, long long ldx, const void* q, const void* scales, const void* zeros,
                     void* y, int M, int N, int K, int group, hgemm_stream_t stream) {
    return gemm_w4(x, x_dtype, ldx, q, scales, zeros, y, M, N, K, group, false, stream);
}

int hgemm_debug_stalled_w4(const void* x, long long ldx, const void* q, const void* scales, const void* zeros, void* y,
                           int M, int N, int K, int group, hgemm_stream_t stream) {
    // The kernel with bounded waits takes more than 16 rows of aligned bf16 x.
    if (M <= 16 || K <= 0 || K % 8 || ldx % 8 || hgw::misaligned(x, 16)) return HGEMM_ERR_INVALID_VALUE;
    return gemm_w4(x, HGEMM_DTYPE_BF16, ldx, q, scales, zeros, y, M, N, K, group, true, stream);
}

}  // extern "C"
