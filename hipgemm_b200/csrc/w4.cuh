// 4-bit weights with group scales: the blocked layout, and the warp-level product that the
// linear and mixture-of-experts kernels share.
//
// A weight is W[n][k] = (code[n][k] - zero) * scale with one bf16 scale (and, if asymmetric,
// one zero point 0..15; else 8) per row and group of 32, 64 or 128 K.  Codes are stored in
// tiles of 16 rows x 64 K, 512 bytes, so that a warp's 16-byte loads are one contiguous
// stretch and each 32-bit word is one A fragment of mma.m16n8k16 with nothing to permute:
// lane 4 g + t holds words j = 0..3 at byte 16 * lane + 4 j; nibble 4 half + 2 rk + rr of word
// j is row g + 8 rr, k = 32 (j / 2) + 8 t + 4 (j % 2) + 2 rk + half.  The sum over K does not
// care about its order, so K is permuted inside each 32 such that a lane's B fragments are 8
// consecutive elements of x: one 16-byte load of bf16 from where x lies, no staging.
// Scales and zero points: [row block][group][g][rr].
//
// Numerics: 128 + code is exact in bf16 (0x4300 | code), and so is its difference to 128 + zero.
// Products of two bf16 are exact, the tensor core sums a 32- or 64-deep part of a group in
// fp32, and the scale multiplies that sum in fp32: nothing is rounded to 16 bits on the way.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace hgw {

constexpr int kTileRows = 16;
constexpr int kTileK = 64;
constexpr int kTileBytes = 512;

__host__ __device__ constexpr int ceil_div(int a, int b) { return a / b + (a % b != 0); }

// One matrix, or a stack of `count` equal ones back to back.
struct Weight {
    const uint8_t* q;
    const uint32_t* scales;   // pairs of bf16: rows g and g + 8
    const uint16_t* zeros;    // pairs of bytes, or null
    int row_blocks, k_blocks, groups, group_shift;
    __device__ size_t tile_base(int index, int row_block) const {
        return (static_cast<size_t>(index) * row_blocks + row_block) * k_blocks * kTileBytes;
    }
    __device__ size_t group_base(int index, int row_block) const {
        return (static_cast<size_t>(index) * row_blocks + row_block) * groups * 8;
    }
};

inline Weight make_weight(const void* q, const void* scales, const void* zeros, int N, int K, int group) {
    const int shift = group == 32 ? 5 : group == 64 ? 6 : 7;
    return {static_cast<const uint8_t*>(q), static_cast<const uint32_t*>(scales), static_cast<const uint16_t*>(zeros),
            ceil_div(N, kTileRows), ceil_div(K, kTileK), ceil_div(K, group), shift};
}

inline bool valid_group(int group) { return group == 32 || group == 64 || group == 128; }

__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
        "%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t sub_bf16x2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

__device__ __forceinline__ float bf16_lo(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t v) { return __uint_as_float(v & 0xFFFF0000u); }

// Word j of a tile -> the A fragment of its 16 K: code - zero, exact.  z0 and z1 are 128 + zero
// as two equal bf16, for rows g and g + 8.
__device__ __forceinline__ void unpack(uint32_t w, uint32_t z0, uint32_t z1, uint32_t (&a)[4]) {
#pragma unroll
    for (int r = 0; r < 4; ++r) a[r] = sub_bf16x2(((w >> (4 * r)) & 0x000F000Fu) | 0x43004300u, r & 1 ? z1 : z0);
}

// A streaming 16-byte load: each weight byte is used once per call.
__device__ __forceinline__ uint4 load_stream(const uint8_t* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}

// ---- the activations' side -----------------------------------------------------------------
//
// A source gives a lane its B fragments of one 64-K block: kTerms bf16 terms whose sum is x
// (exactly, for fp32: three truncations of 8 bits each).  Raw is what is kept in registers
// while a block is in flight.

// Rows of bf16 or fp32 in memory.  `row` points to the lane's column's row; elements at and past
// `len` are zero (a stored pad would do for the codes, but x may hold infinities there).
template <typename T>
struct RowSource;

template <>
struct RowSource<__nv_bfloat16> {
    static constexpr int kTerms = 1;
    struct Raw {
        uint4 v[2];
    };
    const __nv_bfloat16* row;
    int len;
    bool vec;  // rows 16-byte aligned and len % 8 == 0
    __device__ __forceinline__ void load(Raw& raw, int k) const {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int at = k + 32 * h;
            raw.v[h] = make_uint4(0u, 0u, 0u, 0u);
            if (vec) {
                if (at < len) raw.v[h] = __ldg(reinterpret_cast<const uint4*>(row + at));
            } else {
                uint32_t e[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    e[i] = at + i < len ? __ldg(reinterpret_cast<const unsigned short*>(row + at + i)) : 0u;
                raw.v[h] = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
            }
        }
    }
    __device__ __forceinline__ static void terms(const Raw& raw, uint32_t (&b)[1][8]) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            b[0][4 * h] = raw.v[h].x;
            b[0][4 * h + 1] = raw.v[h].y;
            b[0][4 * h + 2] = raw.v[h].z;
            b[0][4 * h + 3] = raw.v[h].w;
        }
    }
};

// What is left of x after its upper 16 bits (a bf16 by truncation): exact.  An infinity leaves 0.
__device__ __forceinline__ float after_bf16(float x) {
    const float hi = __uint_as_float(__float_as_uint(x) & 0xFFFF0000u);
    return fabsf(x) == __int_as_float(0x7F800000) ? 0.0f : x - hi;
}
__device__ __forceinline__ uint32_t upper_halves(float lo, float hi) {
    return __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x7632);
}

template <>
struct RowSource<float> {
    static constexpr int kTerms = 3;
    struct Raw {
        float v[16];
    };
    const float* row;
    int len;
    bool vec;
    __device__ __forceinline__ void load(Raw& raw, int k) const {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int at = k + 32 * h;
            if (vec) {
                float4 f0 = make_float4(0.f, 0.f, 0.f, 0.f), f1 = f0;
                if (at < len) {
                    f0 = __ldg(reinterpret_cast<const float4*>(row + at));
                    f1 = __ldg(reinterpret_cast<const float4*>(row + at) + 1);
                }
                float* v = raw.v + 8 * h;
                v[0] = f0.x, v[1] = f0.y, v[2] = f0.z, v[3] = f0.w;
                v[4] = f1.x, v[5] = f1.y, v[6] = f1.z, v[7] = f1.w;
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) raw.v[8 * h + i] = at + i < len ? __ldg(row + at + i) : 0.0f;
            }
        }
    }
    // x = three bf16 by truncation, 8 significant bits each: 24 bits, so nothing is lost.
    __device__ __forceinline__ static void terms(const Raw& raw, uint32_t (&b)[3][8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float x0 = raw.v[2 * i], x1 = raw.v[2 * i + 1];
#pragma unroll
            for (int s = 0; s < 3; ++s) {
                b[s][i] = upper_halves(x0, x1);
                x0 = after_bf16(x0);
                x1 = after_bf16(x1);
            }
        }
    }
};

// ---- a warp's product ------------------------------------------------------------------------
//
// acc[r][n][.] += sum over K blocks [kb0, kb1) of rows (row block r) x columns (tile n of 8).
// Fragment element i of lane 4 g + t is row g + 8 (i / 2), column 2 t + i % 2.
// Per K block and row block a lane loads 16 bytes of codes and its scales; DEPTH blocks are in
// flight.  The group's sum is scaled once per 64 K (per 32 K for groups of 32): 4 FMAs for 4
// (2) matrix instructions.
template <int R, int NT, int DEPTH, bool G32, bool ZERO, typename Source>
struct WarpProduct {
    static constexpr int kScales = G32 ? 2 : 1;  // groups that start in a 64-K block
    struct Stage {
        uint4 q[R];
        uint32_t scale[R][kScales];
        uint16_t zero[R][kScales];
        typename Source::Raw x[NT];
    };

    const uint8_t* q[R];         // this lane's 16 bytes of the row blocks' first tiles
    const uint32_t* scales[R];   // this lane's pair of the row blocks' first groups
    const uint16_t* zeros[R];
    Source x[NT];
    int group_shift, groups;

    __device__ __forceinline__ void set_rows(int r, const Weight& w, int index, int row_block, int lane) {
        q[r] = w.q + w.tile_base(index, row_block) + lane * 16;
        const size_t base = w.group_base(index, row_block) + lane / 4;
        scales[r] = w.scales + base;
        if (ZERO) zeros[r] = w.zeros + base;
        group_shift = w.group_shift;
        groups = w.groups;
    }

    __device__ __forceinline__ void load(Stage& s, int kb, int lane) const {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            s.q[r] = load_stream(q[r] + static_cast<size_t>(kb) * kTileBytes);
#pragma unroll
            for (int i = 0; i < kScales; ++i) {
                // The last block's second group of 32 may not exist: its codes are padding and x is 0 there.
                int group = (kb * kTileK + 32 * i) >> group_shift;
                if (G32 && i) group = group < groups ? group : groups - 1;
                s.scale[r][i] = __ldg(scales[r] + static_cast<size_t>(group) * 8);
                if (ZERO) s.zero[r][i] = __ldg(zeros[r] + static_cast<size_t>(group) * 8);
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) x[n].load(s.x[n], kb * kTileK + 8 * (lane & 3));
    }

    __device__ __forceinline__ static void compute(const Stage& s, float (&acc)[R][NT][4]) {
        uint32_t b[NT][Source::kTerms][8];
#pragma unroll
        for (int n = 0; n < NT; ++n) Source::terms(s.x[n], b[n]);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const uint32_t words[4] = {s.q[r].x, s.q[r].y, s.q[r].z, s.q[r].w};
            float sum[NT][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int i = G32 ? j / 2 : 0;
                uint32_t z0 = 0x43084308u, z1 = 0x43084308u;  // 128 + 8
                if (ZERO) {
                    z0 = 0x43004300u | (s.zero[r][i] & 0xFFu) * 0x10001u;
                    z1 = 0x43004300u | (s.zero[r][i] >> 8) * 0x10001u;
                }
                uint32_t a[4];
                unpack(words[j], z0, z1, a);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    if (j == 0 || (G32 && j == 2)) sum[n][0] = sum[n][1] = sum[n][2] = sum[n][3] = 0.0f;
#pragma unroll
                    for (int t = Source::kTerms - 1; t >= 0; --t)
                        mma_bf16(sum[n], a, b[n][t][2 * j], b[n][t][2 * j + 1]);
                }
                if (j == 3 || (G32 && j == 1)) {
                    const float s0 = bf16_lo(s.scale[r][i]), s1 = bf16_hi(s.scale[r][i]);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        acc[r][n][0] = fmaf(s0, sum[n][0], acc[r][n][0]);
                        acc[r][n][1] = fmaf(s0, sum[n][1], acc[r][n][1]);
                        acc[r][n][2] = fmaf(s1, sum[n][2], acc[r][n][2]);
                        acc[r][n][3] = fmaf(s1, sum[n][3], acc[r][n][3]);
                    }
                }
            }
        }
    }

    __device__ __forceinline__ void run(int kb0, int kb1, int lane, float (&acc)[R][NT][4]) const {
        Stage s[DEPTH];
#pragma unroll
        for (int d = 0; d < DEPTH; ++d)
            if (kb0 + d < kb1) load(s[d], kb0 + d, lane);
        for (int kb = kb0; kb < kb1; kb += DEPTH) {
#pragma unroll
            for (int d = 0; d < DEPTH; ++d) {
                if (kb + d < kb1) {
                    compute(s[d], acc);
                    if (kb + d + DEPTH < kb1) load(s[d], kb + d + DEPTH, lane);
                }
            }
        }
    }
};

// ---- host side ---------------------------------------------------------------------------

// SM count of the current device; a negative HGEMM_ERR_* code when there is none or it is not
// an sm_100.  Defined in w4.cu.
int current_sms(int* sms);

}  // namespace hgw
