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
// Products of two bf16 are exact, the tensor core sums a whole group (32, 64 or 128 K) in fp32, and
// the scale multiplies that sum in fp32: nothing is rounded to 16 bits on the way.  A group's sum
// has no scale in it yet: 128 products of 15 x leave fp32's range from |x| = 2^117 on.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstddef>
#include <cstdint>
#include <type_traits>

namespace hgw {

constexpr int kTileRows = 16;
constexpr int kTileK = 64;
constexpr int kTileBytes = 512;
constexpr int kMaxDevices = 64;

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

__device__ __forceinline__ void pdl_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ float bf16_lo(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t v) { return __uint_as_float(v & 0xFFFF0000u); }

// The unpacking's constants, in registers that the compiler cannot see through: a logic instruction
// takes one immediate operand, so that with both constants known it would take two of them.
struct UnpackConstants {
    uint32_t mask, magic;
    __device__ __forceinline__ UnpackConstants() {
        asm volatile("mov.b32 %0, 0x000F000F;\n\tmov.b32 %1, 0x43004300;" : "=r"(mask), "=r"(magic));
    }
};

// Word j of a tile -> the A fragment of its 16 K: code - zero, exact.  z0 and z1 are 128 + zero
// as two equal bf16, for rows g and g + 8.  3 shifts, 4 logic instructions, 4 subtractions.
__device__ __forceinline__ void unpack(uint32_t w, const UnpackConstants& c, uint32_t z0, uint32_t z1, uint32_t (&a)[4]) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        uint32_t v;
        asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(v) : "r"(w >> (4 * r)), "r"(c.mask), "r"(c.magic));  // (a & b) | c
        a[r] = sub_bf16x2(v, r & 1 ? z1 : z0);
    }
}

// Loads: these kernels may start while the one before them on the stream still runs (see launch()), which may be what
// writes their operands.  So they use ordinary loads after griddepcontrol.wait and none of the non-coherent path
// (ld.global.nc, __ldg, const __restrict__), whose data has to be unchanged for the whole kernel.

// A streaming 16-byte load: each weight byte is used once per call.
__device__ __forceinline__ uint4 load_stream(const uint8_t* p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}

// ---- the activations' side -----------------------------------------------------------------
//
// A source gives a lane its B fragments of 64 K: kTerms bf16 terms whose sum is x (exactly, for
// fp32: three truncations of 8 bits each).  Raw is what is kept in registers while it is in flight.

// Rows of bf16 or fp32 in memory.  `row` points to the lane's column's row, 8 (lane % 4) elements
// in; `len` is what is left of the row there.  Elements at and past it are zero: the codes there
// are padding that stands for anything, and what follows a row may be an infinity.
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
    bool vec;  // rows 16-byte aligned and of a multiple of 8 elements
    __device__ __forceinline__ void load_full(Raw& raw, int k) const {
#pragma unroll
        for (int h = 0; h < 2; ++h) raw.v[h] = reinterpret_cast<const uint4*>(row + k)[4 * h];
    }
    __device__ __forceinline__ void load(Raw& raw, int k) const {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int at = k + 32 * h;
            raw.v[h] = make_uint4(0u, 0u, 0u, 0u);
            if (vec) {
                if (at < len) raw.v[h] = *reinterpret_cast<const uint4*>(row + at);
            } else {
                uint32_t e[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    e[i] = at + i < len ? *reinterpret_cast<const unsigned short*>(row + at + i) : 0u;
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
    __device__ __forceinline__ void load_full(Raw& raw, int k) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 f = reinterpret_cast<const float4*>(row + k)[(i & 1) + 8 * (i / 2)];
            raw.v[4 * i] = f.x, raw.v[4 * i + 1] = f.y, raw.v[4 * i + 2] = f.z, raw.v[4 * i + 3] = f.w;
        }
    }
    __device__ __forceinline__ void load(Raw& raw, int k) const {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int at = k + 32 * h;
            if (vec) {
                float4 f0 = make_float4(0.f, 0.f, 0.f, 0.f), f1 = f0;
                if (at < len) {
                    f0 = reinterpret_cast<const float4*>(row + at)[0];
                    f1 = reinterpret_cast<const float4*>(row + at)[1];
                }
                float* v = raw.v + 8 * h;
                v[0] = f0.x, v[1] = f0.y, v[2] = f0.z, v[3] = f0.w;
                v[4] = f1.x, v[5] = f1.y, v[6] = f1.z, v[7] = f1.w;
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) raw.v[8 * h + i] = at + i < len ? row[at + i] : 0.0f;
            }
        }
    }
    // x = three bf16 by truncation, 8 significant bits each: 24 bits, so nothing is lost (of |x| below 2^-110 what lies
    // under bf16's smallest number, 2^-133).
    __device__ __forceinline__ static void terms(const Raw& raw, uint32_t (&b)[3][8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float x0 = raw.v[2 * i], x1 = raw.v[2 * i + 1], y0 = after_bf16(x0), y1 = after_bf16(x1);
            b[0][i] = upper_halves(x0, x1);
            b[1][i] = upper_halves(y0, y1);
            b[2][i] = upper_halves(y0 - bf16_hi(__float_as_uint(y0)), y1 - bf16_hi(__float_as_uint(y1)));  // y is no infinity
        }
    }
};

// ---- a warp's product ------------------------------------------------------------------------
//
// acc[r][n][.] += sum over steps [s0, s1) of 128 K of (row block r) x (columns: tile n of 8).
// Fragment element i of lane 4 g + t is row g + 8 (i / 2), column 2 t + i % 2.
//
// The first term's products with the codes have 13 significant bits, so that a group's sum of them is nearly exact in
// fp32; the other terms have a sum of their own, 2^-8 of it.  (In one sum every addition of the small terms cost the
// large ones a truncation: fp32 experts 1.0e-6 from 64 bits in the 2-norm, 1.7e-7 now, in the same time.)
//
// Codes and scales come through a ring of STAGES steps in shared memory that each lane fills with
// asynchronous copies of its own 16 (4) bytes and reads back itself: enough bytes in flight for
// HBM without registers for them, and no barrier.  The activations, which are in L1 or L2, are
// loaded one tile ahead.  Per tile (512 bytes of codes) a warp issues about 60 instructions in the
// loop, 28 of them logic at 2 cycles each, and some 25 more are its share of what comes before and
// after; at HBM speed a scheduler has 86 cycles for a tile, and takes 160 (28672 x 8192 by 8 rows:
// 34 us, 3.6 TB/s).  No one part bounds it: without the copies it would take 33 us, without the
// loads of x 30, without the unpacking 34, without those three 21.

__device__ __forceinline__ void copy16(uint32_t smem, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem), "l"(src) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t smem, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

constexpr int kStepK = 128;

// DEEP loads x two tiles ahead instead of one: registers for latency.  For the experts' gate and up, whose units are
// short, 15.7 us instead of 17.5 (one token) and 239 instead of 246 (32); for kernels that then fit an SM less often
// it costs: the experts' down (three terms of fp32 a column) 19.4 instead of 18.0 and 314 instead of 289, the linear
// kernel 38 instead of 34 (28672 x 8192 by 8 rows) and 54 instead of 47 (by 16).
template <int R, int NT, int STAGES, int GROUP, bool ZERO, bool DEEP, typename Source>
struct WarpProduct {
    static constexpr int kGroups = kStepK / GROUP;  // groups of a step
    static constexpr int kCodes = R * 2 * kTileBytes;
    static constexpr int kScales = R * kGroups * 32 * 4;
    static constexpr int kStageBytes = kCodes + kScales * (ZERO ? 2 : 1);
    static constexpr int kWarpBytes = kStageBytes * STAGES;

    const uint8_t* q[R];         // this lane's 16 bytes of the row blocks' first tiles
    const uint32_t* scales[R];   // this lane's pair of the row blocks' first groups
    const uint8_t* zeros[R];     // the 4 bytes that this lane's pair is in
    Source x[NT];
    int k_blocks, groups;
    int full_blocks;             // K blocks whose x is loaded without a look at the row's end

    // `columns`: elements of a row of x, or 0 where its rows are not aligned.
    __device__ __forceinline__ void set_columns(int columns) { full_blocks = columns / kTileK; }

    __device__ __forceinline__ void set_rows(int r, const Weight& w, int index, int row_block, int lane) {
        q[r] = w.q + w.tile_base(index, row_block) + lane * 16;
        const size_t base = w.group_base(index, row_block);
        scales[r] = w.scales + base + lane / 4;
        if (ZERO) zeros[r] = reinterpret_cast<const uint8_t*>(w.zeros + base) + (lane / 8) * 4;
        k_blocks = w.k_blocks;
        groups = w.groups;
    }

    // What is past the end of a row is not copied (a tile's second group of 32 among it): its x is 0,
    // its scale is taken for 0 where it is used.
    __device__ __forceinline__ void copy(uint32_t stage, int step, int lane) const {
        const bool whole = 2 * step + 1 < k_blocks;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const uint8_t* from = q[r] + static_cast<size_t>(step) * (2 * kTileBytes);
            const uint32_t to = stage + r * (2 * kTileBytes) + lane * 16;
            copy16(to, from);
            if (whole) copy16(to + kTileBytes, from + kTileBytes);
            const uint32_t* scale = scales[r] + static_cast<size_t>(step) * (kGroups * 8);
            const uint8_t* zero = ZERO ? zeros[r] + static_cast<size_t>(step) * (kGroups * 16) : nullptr;
#pragma unroll
            for (int i = 0; i < kGroups; ++i) {
                if (i > 0 && step * kGroups + i >= groups) continue;
                const uint32_t at = stage + kCodes + ((r * kGroups + i) * 32 + lane) * 4;
                copy4(at, scale + 8 * i);
                if (ZERO) copy4(at + kScales, zero + 16 * i);
            }
        }
    }
    __device__ __forceinline__ void load_x(typename Source::Raw (&raw)[NT], int block) const {
        if (block < full_blocks) {
#pragma unroll
            for (int n = 0; n < NT; ++n) x[n].load_full(raw[n], block * kTileK);
        } else {
#pragma unroll
            for (int n = 0; n < NT; ++n) x[n].load(raw[n], block * kTileK);
        }
    }

    // One tile of 64 K (half h of a step) of all row blocks.
    template <int H>
    __device__ __forceinline__ void tile(const UnpackConstants& c, const uint8_t* stage, int step, int lane, const typename Source::Raw (&raw)[NT],
                                         float (&sum)[R][NT][4], float (&low)[R][NT][4], float (&acc)[R][NT][4]) const {
        constexpr int kTerms = Source::kTerms;
        uint32_t b[NT][Source::kTerms][8];
#pragma unroll
        for (int n = 0; n < NT; ++n) Source::terms(raw[n], b[n]);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const uint4 codes = *reinterpret_cast<const uint4*>(stage + (2 * r + H) * kTileBytes + lane * 16);
            const uint32_t words[4] = {codes.x, codes.y, codes.z, codes.w};
            uint32_t z0 = 0x43084308u, z1 = 0x43084308u;  // 128 + 8
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int i = (64 * H + 16 * j) / GROUP;  // the group, of the step's
                const uint8_t* at = stage + kCodes + ((r * kGroups + i) * 32 + lane) * 4;
                const bool first = (64 * H + 16 * j) % GROUP == 0, last = (64 * H + 16 * j + 16) % GROUP == 0;
                if (ZERO && (j == 0 || first)) {
                    const uint32_t pair = *reinterpret_cast<const uint32_t*>(at + kScales) >> (lane & 4 ? 16 : 0);
                    z0 = __byte_perm(pair, 0x43u, 0x4040);
                    z1 = __byte_perm(pair, 0x43u, 0x4141);
                }
                uint32_t a[4];
                unpack(words[j], c, z0, z1, a);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    if (first) {
                        sum[r][n][0] = sum[r][n][1] = sum[r][n][2] = sum[r][n][3] = 0.0f;
                        if (kTerms > 1) low[r][n][0] = low[r][n][1] = low[r][n][2] = low[r][n][3] = 0.0f;
                    }
#pragma unroll
                    for (int t = Source::kTerms - 1; t > 0; --t) mma_bf16(low[r][n], a, b[n][t][2 * j], b[n][t][2 * j + 1]);
                    mma_bf16(sum[r][n], a, b[n][0][2 * j], b[n][0][2 * j + 1]);
                }
                if (last) flush(i, step, *reinterpret_cast<const uint32_t*>(at), sum[r], low[r], acc[r]);
            }
        }
    }
    __device__ __forceinline__ void flush(int i, int step, uint32_t pair, const float (&sum)[NT][4], const float (&low)[NT][4], float (&acc)[NT][4]) const {
        if (GROUP == 32 && i > 0) pair = step * kGroups + i < groups ? pair : 0u;
        const float s0 = bf16_lo(pair), s1 = bf16_hi(pair);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            acc[n][0] = fmaf(s0, Source::kTerms > 1 ? sum[n][0] + low[n][0] : sum[n][0], acc[n][0]);
            acc[n][1] = fmaf(s0, Source::kTerms > 1 ? sum[n][1] + low[n][1] : sum[n][1], acc[n][1]);
            acc[n][2] = fmaf(s1, Source::kTerms > 1 ? sum[n][2] + low[n][2] : sum[n][2], acc[n][2]);
            acc[n][3] = fmaf(s1, Source::kTerms > 1 ? sum[n][3] + low[n][3] : sum[n][3], acc[n][3]);
        }
    }

    // `ring`: this warp's kWarpBytes of shared memory, 16-byte aligned.
    __device__ __forceinline__ void run(uint8_t* ring, int s0, int s1, int lane, float (&acc)[R][NT][4]) const {
        const uint32_t base = static_cast<uint32_t>(__cvta_generic_to_shared(ring));
#pragma unroll
        for (int d = 0; d < STAGES - 1; ++d) {
            if (s0 + d < s1) copy(base + d * kStageBytes, s0 + d, lane);
            copy_commit();
        }
        // x is loaded a tile ahead, or (DEEP) a step of two.
        constexpr int kAhead = DEEP ? 2 : 1;
        typename Source::Raw even[2][NT], odd[kAhead][NT];
        if (s0 < s1) {
            load_x(even[0], 2 * s0);
            if (DEEP) load_x(even[1], 2 * s0 + 1);
        }
        const UnpackConstants c;
        int at = 0;  // the stage's place in the ring
        // One step with x in `raw`; `next` takes the next step's (DEEP).
        auto one = [&](int step, typename Source::Raw (&raw)[2][NT], auto& next) {
            const int ahead = step + STAGES - 1;
            const int into = at == 0 ? STAGES - 1 : at - 1;
            if (ahead < s1) copy(base + into * kStageBytes, ahead, lane);
            copy_commit();
            if constexpr (DEEP) {
                if (step + 1 < s1) {
                    load_x(next[0], 2 * step + 2);
                    load_x(next[1], 2 * step + 3);
                }
            } else {
                load_x(raw[1], 2 * step + 1);
            }
            copy_wait<STAGES - 1>();
            const uint8_t* stage = ring + at * kStageBytes;
            float sum[R][NT][4], low[R][NT][4];
            tile<0>(c, stage, step, lane, raw[0], sum, low, acc);
            if (!DEEP && step + 1 < s1) load_x(raw[0], 2 * step + 2);
            if (2 * step + 1 < k_blocks) {
                tile<1>(c, stage, step, lane, raw[1], sum, low, acc);
            } else if (GROUP == 128) {
                // The row ends with half a group.
#pragma unroll
                for (int r = 0; r < R; ++r)
                    flush(0, step, *reinterpret_cast<const uint32_t*>(stage + kCodes + (r * 32 + lane) * 4), sum[r], low[r], acc[r]);
            }
            at = at == STAGES - 1 ? 0 : at + 1;
        };
        if constexpr (DEEP) {
            for (int step = s0; step < s1; step += 2) {
                one(step, even, odd);
                if (step + 1 < s1) one(step + 1, odd, even);
            }
        } else {
            for (int step = s0; step < s1; ++step) one(step, even, odd);
        }
        copy_wait<0>();
    }
};

// ---- a warp's product with the activations held as whole numbers ---------------------------------
//
// For few rows of x the products above are bound by instructions: 28 logic instructions and 16
// subtractions per 512 bytes of codes to make bf16 of them.  As bytes the codes need 12: (w ^ 0x88..)
// & 0xF0.. is 16 (code - 8) of the four high nibbles as signed bytes, and the same of w << 4 that of
// the low ones; with integer tensor instructions the sums are exact as well.  So x is turned into
// whole numbers, once: a warp keeps its K slice of x (XS steps of 128) in registers for all the row
// blocks it goes through.  With 2^e just above the largest element of a row's slice, x = 2^(e - 31) n and the
// bytes of n, each in -128..127, are four planes:
//     n = 2^24 i0 + 2^16 i1 + 2^8 i2 + i3        (n + 0x808080, then the lower three bytes less 128).
// Every element keeps its value whatever the largest is, since a row of W may have only zeros there:
//   bf16: a slice with an element that is no multiple of the unit 2^(e - 31), for which it has to be below 2^(e - 24),
//         is computed from x itself (direct());
//   fp32: where an element is off by more than 2^-20 of itself, 2^8 (x / unit - n) is a fifth plane, kept in shared
//         memory (of normally distributed x one slice of 512 elements in five has such an element); where that is
//         not enough, direct().
// direct() also takes slices with an infinity, a NaN or an extreme exponent.  A warp with the fifth plane issues a
// quarter more matrix instructions (8192 x 8192 by 3 rows of fp32, every warp: 25.3 us instead of 19.6; that is why
// not for 2^-24), one that takes direct() has twice the work (by 3 rows with nine elements of 1e5: 32 us;
// 28672 x 8192 by one row of bf16 24.8 and 44).
//
// Columns: up to two rows of x take one tile, column 4 m + plane; else (fp32) plane p of 8 rows is
// tile p, and the planes are put together in the same lane.

__device__ __forceinline__ void mma_s8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const int (&c)[4]) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, "
        "%13};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(c[0]), "r"(c[1]), "r"(c[2]), "r"(c[3]));
}

// 1.5 * 2^23: its bits plus a whole number n, |n| < 2^22, are the bits of 1.5 * 2^23 + n.
constexpr int kMagicBits = 0x4B400000;
constexpr float kMagic = 12582912.0f;

template <typename T>
__device__ __forceinline__ float raw_element(const typename RowSource<T>::Raw& raw, int i);
template <>
__device__ __forceinline__ float raw_element<float>(const RowSource<float>::Raw& raw, int i) {
    return raw.v[i];
}
template <>
__device__ __forceinline__ float raw_element<__nv_bfloat16>(const RowSource<__nv_bfloat16>::Raw& raw, int i) {
    const uint4 v = raw.v[i / 8];
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    return i & 1 ? bf16_hi(w[i % 8 / 2]) : bf16_lo(w[i % 8 / 2]);
}

// MT = 0: up to two rows of x in one tile; MT = 1: 8 rows, a tile a plane.
template <typename T, int MT, int XS, int STAGES, int GROUP, bool ZERO>
struct WarpStationary {
    static constexpr bool kPacked = MT == 0, kFifth = sizeof(T) == 4;
    static constexpr int kRowTiles = kPacked ? 1 : MT;
    static constexpr int kPlanes = 4;
    static constexpr int kTiles = kPacked ? 1 : MT * kPlanes;        // tiles of plane columns in registers
    static constexpr int kAllTiles = kTiles + (kFifth ? kRowTiles : 0);  // and in shared memory
    static constexpr int kColumns = kPacked ? 2 : 8 * MT;
    static constexpr int kGroups = kStepK / GROUP;
    static constexpr int kCodes = XS * 2 * kTileBytes;
    static constexpr int kScales = XS * kGroups * 32;  // a group: 8 pairs of bf16, then (ZERO) 8 pairs of bytes
    static constexpr int kStageBytes = kCodes + (ZERO ? kScales * 3 / 2 : kScales);
    static constexpr int kSumBytes = ZERO ? XS * kGroups * kAllTiles * 8 * 4 : 0;  // sums of x by group and column
    // The fifth plane: B fragments, 8 bytes a lane, by 32 K; packed, of the 8 lanes that have columns 0 and 4.
    static constexpr int kFifthWords = kPacked ? 16 : 64;
    static constexpr int kFifthBytes = kFifth ? kRowTiles * XS * 4 * kFifthWords * 4 : 0;
    static constexpr int kWarpBytes = kStageBytes * STAGES + kSumBytes + kFifthBytes;
    static constexpr int kSumStride = 20;  // floats from column to column of a warp's result: no bank conflicts
    static constexpr int kResult = kColumns * kSumStride;
    // An element of fp32 x is off by no more than this part of itself.
    static constexpr float kHeld = 0x1p-20f;

    struct Rows {
        RowSource<T> tile[kRowTiles];  // rows of x by B fragment column
    };
    Rows x;
    uint32_t b[XS][4][kTiles][2];
    float factor[kRowTiles][2];      // 2^(e - 11) of columns 2 t, 2 t + 1 (of a plane's, if packed)
    bool special, fifth;             // computed from x itself; with the fifth plane
    int block0, blocks;              // K blocks of the slice
    uint8_t* ring;
    float* x_sums;
    uint32_t* fifth_words;           // this lane's two of each 32 K, null if it has none

    // K blocks [first, first + 2 XS); those past `k_blocks` do not exist.
    __device__ __forceinline__ void set_slice(uint8_t* warp_smem, int first, int k_blocks, int lane) {
        ring = warp_smem;
        x_sums = reinterpret_cast<float*>(warp_smem + kStageBytes * STAGES);
        fifth_words = reinterpret_cast<uint32_t*>(warp_smem + kStageBytes * STAGES + kSumBytes);
        if (!kPacked) fifth_words += 2 * lane;
        else fifth_words = lane / 4 % 4 == 0 ? fifth_words + 2 * (lane / 16 * 4 + lane % 4) : nullptr;
        block0 = first;
        blocks = min(2 * XS, max(0, k_blocks - first));
        // Scales that are never copied stand for groups past the end of a row.
        for (int s = 0; s < STAGES; ++s)
            for (int i = lane * 4; i < kStageBytes - kCodes; i += 128)
                *reinterpret_cast<uint32_t*>(ring + s * kStageBytes + kCodes + i) = 0u;
        __syncwarp();
    }

    // Four bytes, one of each y, in the codes' order in a word: k, k + 2, k + 1, k + 3.  `pick`: the byte as __byte_perm
    // selects it from its first operand, and 16 times (4 more) for the second.
    __device__ __forceinline__ static uint32_t gather(const uint32_t (&y)[4], uint32_t pick) {
        return __byte_perm(__byte_perm(y[0], y[2], pick), __byte_perm(y[1], y[3], pick), 0x5410);
    }

    // Turns the slice of x into planes.  `full_blocks`: K blocks loaded without a look at the row's end.
    __device__ __forceinline__ void convert(int full_blocks, int lane) {
        special = fifth = false;
        auto load = [&](typename RowSource<T>::Raw& raw, int m, int i) {
            if (block0 + i < full_blocks) x.tile[m].load_full(raw, (block0 + i) * kTileK);
            else x.tile[m].load(raw, (block0 + i) * kTileK);
        };
        typename RowSource<T>::Raw raw;
        uint32_t lost = 0u;  // bf16: bits of what the planes do not hold
        // Packed, lane 4 g + t has plane g % 4 of row g / 4.
        const int plane = lane / 4 % 4;
        const uint32_t pick = 0x73u - 0x11u * static_cast<uint32_t>(plane);
#pragma unroll
        for (int m = 0; m < kRowTiles; ++m) {
            // Once for the largest element, once more (from L1) for the planes: the slice does not fit the registers.
            float top = 0.0f;
#pragma unroll
            for (int i = 0; i < 2 * XS; ++i) {
                load(raw, m, i);
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(fabsf(raw_element<T>(raw, j))));
            }
#pragma unroll
            for (int o = 1; o < 4; o <<= 1) {
                const float other = __shfl_xor_sync(0xffffffffu, top, o);
                asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(other));
            }
            // e = exponent - 126, with top below 2^e (1 - 2^-7): then n + 0x808080 does not overflow.  e <= 31, so that
            // x * 2^(31 - e) is exact.
            const uint32_t bits = __float_as_uint(top);
            special |= bits != 0u && (bits < 50u << 23 || bits >= 157u << 23);
            const int exponent = min(max(static_cast<int>((bits + 0x20000u) >> 23), 50), 157);
            const float up = __uint_as_float(static_cast<uint32_t>(284 - exponent) << 23);     // 2^(31 - e)
            float down = __uint_as_float(static_cast<uint32_t>(exponent - 10) << 23);          // 2^(e - 7), and 16 less
            if (kPacked) down *= __uint_as_float(static_cast<uint32_t>(127 - 8 * plane) << 23);
#pragma unroll
            for (int i = 0; i < 2; ++i) factor[m][i] = __shfl_sync(0xffffffffu, down, 4 * (2 * (lane & 3) + i));
#pragma unroll
            for (int i = 0; i < 2 * XS; ++i) {
                load(raw, m, i);
#pragma unroll
                for (int j = 0; j < 4; ++j) {  // 4 elements: one register of each plane
                    uint32_t y[4], z[4];
#pragma unroll
                    for (int l = 0; l < 4; ++l) {
                        const float r = raw_element<T>(raw, 4 * j + l) * up;
                        const int n = __float2int_rn(r);
                        y[l] = (static_cast<uint32_t>(n) + 0x00808080u) ^ 0x00808080u;
                        const float rest = r - __int2float_rn(n);  // exact: 0 from 2^23 on
                        if constexpr (kFifth) {
                            // 128 does not fit: 127, and what that leaves.
                            const float whole = fminf(fmaf(rest, 256.0f, kMagic), kMagic + 127.0f);
                            z[l] = __float_as_uint(whole);
                            const float held = kHeld * fabsf(r);
                            fifth |= fabsf(rest) > held;
                            special |= fabsf(fmaf(whole - kMagic, -0x1p-8f, rest)) > held;
                        } else {
                            lost |= __float_as_uint(rest);
                        }
                    }
                    if constexpr (kPacked) {
                        b[i / 2][i % 2 * 2 + j / 2][0][j % 2] = gather(y, pick);
                    } else {
#pragma unroll
                        for (int p = 0; p < kPlanes; ++p) b[i / 2][i % 2 * 2 + j / 2][m * kPlanes + p][j % 2] = gather(y, 0x73u - 0x11u * p);
                    }
                    if constexpr (kFifth) {
                        const uint32_t word = gather(z, 0x40u);
                        if (!kPacked || plane == 0) fifth_words[(m * XS * 4 + 2 * i + j / 2) * kFifthWords + j % 2] = word;
                    }
                }
            }
        }
        special = __any_sync(0xffffffffu, special || lost != 0u);
        fifth = __any_sync(0xffffffffu, fifth);
        if (ZERO) {
            const uint32_t ones[4] = {0x10101010u, 0x10101010u, 0x10101010u, 0x10101010u};
#pragma unroll
            for (int g = 0; g < XS * kGroups; ++g)
#pragma unroll
                for (int n = 0; n < kAllTiles; ++n) {
                    int sum[4] = {0, 0, 0, 0};
#pragma unroll
                    for (int c = 0; c < GROUP / 32; ++c) {
                        const int at = g * (GROUP / 32) + c;
                        if (n < kTiles) {
                            mma_s8(sum, ones, b[at / 4][at % 4][n][0], b[at / 4][at % 4][n][1], sum);
                        } else {
                            const uint2 w = fifth_at(n - kTiles, at);
                            mma_s8(sum, ones, w.x, w.y, sum);
                        }
                    }
                    if (lane < 4)
                        *reinterpret_cast<float2*>(x_sums + (g * kAllTiles + n) * 8 + 2 * lane) =
                            make_float2(static_cast<float>(sum[0]), static_cast<float>(sum[1]));
                }
            __syncwarp();
        }
    }

    // This lane's B fragment of the fifth plane, 32 K `k32` of the slice.
    __device__ __forceinline__ uint2 fifth_at(int m, int k32) const {
        if (kPacked && !fifth_words) return make_uint2(0u, 0u);
        return *reinterpret_cast<const uint2*>(fifth_words + (m * XS * 4 + k32) * kFifthWords);
    }

    // Starts the copies of the slice of one row block.  q: this lane's 16 bytes of the row block's first tile; scales,
    // zeros: the row block's first group.  A lane copies 16 bytes of the scales, and of the zero points, for all.
    __device__ __forceinline__ void copy(int stage, const uint8_t* q, const uint8_t* scales, const uint8_t* zeros, int groups,
                                         int lane) const {
        static_assert(XS * kGroups <= 16, "one copy a lane");
        const uint32_t base = static_cast<uint32_t>(__cvta_generic_to_shared(ring)) + stage * kStageBytes;
        q += static_cast<size_t>(block0) * kTileBytes;
#pragma unroll
        for (int i = 0; i < 2 * XS; ++i)
            if (i < blocks) copy16(base + i * kTileBytes + lane * 16, q + i * kTileBytes);
        const int group0 = block0 / 2 * kGroups;
        if (lane < XS * kGroups * 2 && group0 + lane / 2 < groups)
            copy16(base + kCodes + lane * 16, scales + static_cast<size_t>(group0) * 32 + lane * 16);
        if (ZERO && lane < XS * kGroups && group0 + lane < groups)
            copy16(base + kCodes + kScales + lane * 16, zeros + static_cast<size_t>(group0) * 16 + lane * 16);
    }

    // The row block in `stage`: 16 rows x kColumns sums, written to result[column * kSumStride + row].
    __device__ __forceinline__ void compute(int stage, uint32_t flip, uint32_t high, float* result, int lane) const {
        const uint8_t* in = ring + stage * kStageBytes;
        if (special) {
            direct(in, x, block0, blocks, result, lane);
        } else if (kFifth && fifth) {
            products<kFifth>(in, flip, high, result, lane);
        } else {
            products<false>(in, flip, high, result, lane);
        }
    }

private:
    template <bool FIFTH>
    __device__ __forceinline__ void products(const uint8_t* in, uint32_t flip, uint32_t high, float* result, int lane) const {
        float acc[kRowTiles][4];
#pragma unroll
        for (int m = 0; m < kRowTiles; ++m) acc[m][0] = acc[m][1] = acc[m][2] = acc[m][3] = 0.0f;
        const int magic[4] = {kMagicBits, kMagicBits, kMagicBits, kMagicBits};
        constexpr int kUsed = FIFTH ? kAllTiles : kTiles;
        int sum[kUsed][4];
#pragma unroll
        for (int i = 0; i < 2 * XS; ++i) {
            const uint4 codes = *reinterpret_cast<const uint4*>(in + i * kTileBytes + lane * 16);
            const uint32_t words[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t a[4];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t w = words[2 * h + j];
                    asm("lop3.b32 %0, %1, %2, %3, 0x28;" : "=r"(a[2 * j]) : "r"(w << 4), "r"(flip), "r"(high));  // (a ^ b) & c
                    asm("lop3.b32 %0, %1, %2, %3, 0x28;" : "=r"(a[2 * j + 1]) : "r"(w), "r"(flip), "r"(high));
                }
                const int k32 = 2 * i + h;  // of the slice
                const bool first = k32 * 32 % GROUP == 0, last = (k32 + 1) * 32 % GROUP == 0;
#pragma unroll
                for (int n = 0; n < kUsed; ++n) {
                    uint32_t b0, b1;
                    if (n < kTiles) {
                        b0 = b[i / 2][k32 % 4][n][0];
                        b1 = b[i / 2][k32 % 4][n][1];
                    } else {
                        const uint2 w = fifth_at(n - kTiles, k32);
                        b0 = w.x;
                        b1 = w.y;
                    }
                    if (first) mma_s8(sum[n], a, b0, b1, magic);
                    else mma_s8(sum[n], a, b0, b1, sum[n]);
                }
                if (last) flush<FIFTH>(in, k32 * 32 / GROUP, sum, acc, lane);
            }
        }
        if (kPacked) {
            // Columns 4 m + plane: lanes 2 m and 2 m + 1 of four have two planes each.
            float v0 = acc[0][0] + acc[0][1], v1 = acc[0][2] + acc[0][3];
            v0 += __shfl_xor_sync(0xffffffffu, v0, 1);
            v1 += __shfl_xor_sync(0xffffffffu, v1, 1);
            if ((lane & 1) == 0) {
                float* at = result + (lane & 3) / 2 * kSumStride + lane / 4;
                at[0] = v0;
                at[8] = v1;
            }
        } else {
            write(result, acc, lane);
        }
    }

    // acc += scale * 2^(e - 7) * sum over the group of (code - zero) * (the planes).
    template <bool FIFTH, int USED>
    __device__ __forceinline__ void flush(const uint8_t* in, int group, const int (&sum)[USED][4], float (&acc)[kRowTiles][4],
                                          int lane) const {
        const uint32_t pair = *reinterpret_cast<const uint32_t*>(in + kCodes + group * 32 + lane / 4 * 4);
        const float scale[2] = {bf16_lo(pair), bf16_hi(pair)};
        float shift[2] = {0.0f, 0.0f};  // 8 - zero
        if (ZERO) {
            const uint32_t z = *reinterpret_cast<const uint16_t*>(in + kCodes + kScales + group * 16 + lane / 4 * 2);
            // 2^23 + 0..255 as bits.
            shift[0] = (8388608.0f + 8.0f) - __uint_as_float(__byte_perm(z, 0x4B000000u, 0x7550));
            shift[1] = (8388608.0f + 8.0f) - __uint_as_float(__byte_perm(z, 0x4B000000u, 0x7551));
        }
        // A plane's sums, whole numbers below 2^23.
        auto whole = [&](int n, int i) {
            float u = __int_as_float(sum[n][i]) - kMagic;
            if (ZERO) {
                const float2 sums = *reinterpret_cast<const float2*>(x_sums + (group * kAllTiles + n) * 8 + 2 * (lane & 3));
                u = fmaf(shift[i / 2], i % 2 ? sums.y : sums.x, u);
            }
            return u;
        };
#pragma unroll
        for (int m = 0; m < kRowTiles; ++m) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                // Packed, the fifth plane lies in the first one's column, and the others add up across lanes.
                float v = 0.0f;
                if (FIFTH) v = kPacked ? whole(kTiles + m, i) * 0x1p-24f : whole(kTiles + m, i);
#pragma unroll
                for (int p = kPacked ? 0 : kPlanes - 1; p >= 0; --p) {
                    const float u = whole(kPacked ? 0 : m * kPlanes + p, i);
                    v = FIFTH || (!kPacked && p < kPlanes - 1) ? fmaf(v, 0x1p-8f, u) : u;
                }
                acc[m][i] = fmaf(scale[i / 2], v * factor[m][i % 2], acc[m][i]);
            }
        }
    }

    __device__ __forceinline__ static void write(float* result, const float (&acc)[kRowTiles][4], int lane) {
#pragma unroll
        for (int m = 0; m < kRowTiles; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                int column = 8 * m + 2 * (lane & 3) + i % 2;
                if (kPacked) {  // row of x: column / 4
                    if (column % 4 != 0) continue;
                    column /= 4;
                }
                result[column * kSumStride + lane / 4 + 8 * (i / 2)] = acc[m][i];
            }
    }

    // The same from x as it is: bf16 (or three bf16 of fp32) products as WarpProduct's.  Not inlined, and not a
    // member that would want the planes in memory.
    __device__ __noinline__ static void direct(const uint8_t* in, Rows x, int block0, int blocks, float* result, int lane) {
        constexpr int kTerms = RowSource<T>::kTerms;
        const UnpackConstants c;
        float acc[kRowTiles][4] = {};
        for (int i = 0; i < blocks; ++i) {
            uint32_t terms[kRowTiles][kTerms][8];
#pragma unroll
            for (int m = 0; m < kRowTiles; ++m) {
                typename RowSource<T>::Raw raw;
                x.tile[m].load(raw, (block0 + i) * kTileK);
                RowSource<T>::terms(raw, terms[m]);
            }
            const uint4 codes = *reinterpret_cast<const uint4*>(in + i * kTileBytes + lane * 16);
            const uint32_t words[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int group = (i * kTileK + 32 * h) / GROUP;
                const uint32_t pair = *reinterpret_cast<const uint32_t*>(in + kCodes + group * 32 + lane / 4 * 4);
                uint32_t z0 = 0x43084308u, z1 = 0x43084308u;
                if (ZERO) {
                    const uint32_t z = *reinterpret_cast<const uint16_t*>(in + kCodes + kScales + group * 16 + lane / 4 * 2);
                    z0 = __byte_perm(z, 0x43u, 0x4040);
                    z1 = __byte_perm(z, 0x43u, 0x4141);
                }
                float sum[kRowTiles][4] = {};
#pragma unroll
                for (int j = 2 * h; j < 2 * h + 2; ++j) {
                    uint32_t a[4];
                    unpack(words[j], c, z0, z1, a);
#pragma unroll
                    for (int m = 0; m < kRowTiles; ++m)
#pragma unroll
                        for (int t = kTerms - 1; t >= 0; --t) mma_bf16(sum[m], a, terms[m][t][2 * j], terms[m][t][2 * j + 1]);
                }
#pragma unroll
                for (int m = 0; m < kRowTiles; ++m)
#pragma unroll
                    for (int k = 0; k < 4; ++k) acc[m][k] = fmaf(k < 2 ? bf16_lo(pair) : bf16_hi(pair), sum[m][k], acc[m][k]);
            }
        }
        write(result, acc, lane);
    }
};

// ---- host side ---------------------------------------------------------------------------

// SM count of the current device and its number; a negative HGEMM_ERR_* code when there is none
// or it is not an sm_100.  Defined in w4.cu.
int current_device(int* sms, int* dev);

// Lets KERNEL have `bytes` of dynamic shared memory on device `dev` (once per device), and gives the
// CTAs of `threads` that an SM keeps resident.  0 on failure.
template <auto KERNEL>
int resident_ctas(int dev, int threads, size_t bytes) {
    static std::atomic<int> known[kMaxDevices];
    int n = known[dev].load(std::memory_order_relaxed);
    if (n == 0) {
        if (cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)) != cudaSuccess ||
            cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, KERNEL, threads, bytes) != cudaSuccess) {
            cudaGetLastError();
            return 0;
        }
        known[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}

// Launches KERNEL with a cluster of `cluster` CTAs.  Programmatic dependent launch: the CTAs may start while the
// stream's previous kernel ends; they touch global memory only after griddepcontrol.wait, but for ids and weights of
// the experts, which their second and third kernel read before it: the first waits before it triggers, so that
// whatever wrote those has ended when the others start.
template <auto KERNEL, typename... Args>
int launch(dim3 grid, int threads, int cluster, size_t smem, cudaStream_t stream, const Args&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    if (cudaLaunchKernelEx(&cfg, KERNEL, args...) == cudaSuccess) return 0;
    cudaGetLastError();
    return -4;  // HGEMM_ERR_CUDA
}

inline bool misaligned(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1u)) != 0; }

// Whether `y_bytes` from y on meet one of `rows` rows of x, `ld` apart, of `columns` elements of `size` bytes.
inline bool meets_rows(const void* y, size_t y_bytes, const void* x, int rows, long long ld, int columns, unsigned size) {
    const uintptr_t x0 = reinterpret_cast<uintptr_t>(x), y0 = reinterpret_cast<uintptr_t>(y);
    const size_t row = static_cast<size_t>(columns) * size, step = rows > 1 ? static_cast<size_t>(ld) * size : row;
    if (rows < 1 || row == 0 || y_bytes == 0 || y0 >= x0 + (rows - 1) * step + row) return false;
    if (y0 < x0) return x0 - y0 < y_bytes;
    const size_t r = (y0 - x0) / step, at = (y0 - x0) % step;  // y starts in row r, or behind it
    return at < row || (r + 1 < static_cast<size_t>(rows) && at + y_bytes > step);
}

// Calls go(std::integral_constant<int, GROUP>, std::bool_constant<ZERO>) for a weight's group size and kind.
template <typename Go>
int with_format(int group, bool zeros, Go go) {
    using std::integral_constant;
    if (group == 32) return zeros ? go(integral_constant<int, 32>{}, std::true_type{}) : go(integral_constant<int, 32>{}, std::false_type{});
    if (group == 64) return zeros ? go(integral_constant<int, 64>{}, std::true_type{}) : go(integral_constant<int, 64>{}, std::false_type{});
    return zeros ? go(integral_constant<int, 128>{}, std::true_type{}) : go(integral_constant<int, 128>{}, std::false_type{});
}

}  // namespace hgw
