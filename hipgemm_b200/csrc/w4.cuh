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
        for (int h = 0; h < 2; ++h) raw.v[h] = __ldg(reinterpret_cast<const uint4*>(row + k) + 4 * h);
    }
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
    __device__ __forceinline__ void load_full(Raw& raw, int k) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 f = __ldg(reinterpret_cast<const float4*>(row + k) + (i & 1) + 8 * (i / 2));
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
// acc[r][n][.] += sum over steps [s0, s1) of 128 K of (row block r) x (columns: tile n of 8).
// Fragment element i of lane 4 g + t is row g + 8 (i / 2), column 2 t + i % 2.
//
// Codes and scales come through a ring of STAGES steps in shared memory that each lane fills with
// asynchronous copies of its own 16 (4) bytes and reads back itself: enough bytes in flight for
// HBM without registers for them, and no barrier.  The activations, which are in L1 or L2, are
// loaded one tile ahead.  Per tile (512 bytes of codes) a warp issues about 60 instructions, 28
// of them logic at 2 cycles each; at HBM speed a scheduler has 86 cycles for a tile.

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

template <int R, int NT, int STAGES, int GROUP, bool ZERO, typename Source>
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
                                         float (&sum)[R][NT][4], float (&acc)[R][NT][4]) const {
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
                    if (first) sum[r][n][0] = sum[r][n][1] = sum[r][n][2] = sum[r][n][3] = 0.0f;
#pragma unroll
                    for (int t = Source::kTerms - 1; t >= 0; --t) mma_bf16(sum[r][n], a, b[n][t][2 * j], b[n][t][2 * j + 1]);
                }
                if (last) flush(i, step, *reinterpret_cast<const uint32_t*>(at), sum[r], acc[r]);
            }
        }
    }
    __device__ __forceinline__ void flush(int i, int step, uint32_t pair, const float (&sum)[NT][4], float (&acc)[NT][4]) const {
        if (GROUP == 32 && i > 0) pair = step * kGroups + i < groups ? pair : 0u;
        const float s0 = bf16_lo(pair), s1 = bf16_hi(pair);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            acc[n][0] = fmaf(s0, sum[n][0], acc[n][0]);
            acc[n][1] = fmaf(s0, sum[n][1], acc[n][1]);
            acc[n][2] = fmaf(s1, sum[n][2], acc[n][2]);
            acc[n][3] = fmaf(s1, sum[n][3], acc[n][3]);
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
        typename Source::Raw raw[2][NT];
        if (s0 < s1) load_x(raw[0], 2 * s0);
        const UnpackConstants c;
        int at = 0;  // the stage's place in the ring
        for (int step = s0; step < s1; ++step) {
            const int ahead = step + STAGES - 1;
            const int into = at == 0 ? STAGES - 1 : at - 1;
            if (ahead < s1) copy(base + into * kStageBytes, ahead, lane);
            copy_commit();
            copy_wait<STAGES - 1>();
            const uint8_t* stage = ring + at * kStageBytes;
            float sum[R][NT][4];
            load_x(raw[1], 2 * step + 1);
            tile<0>(c, stage, step, lane, raw[0], sum, acc);
            const bool more = 2 * step + 1 < k_blocks;
            if (step + 1 < s1) load_x(raw[0], 2 * step + 2);
            if (more) {
                tile<1>(c, stage, step, lane, raw[1], sum, acc);
            } else if (GROUP == 128) {
                // The row ends with half a group.
#pragma unroll
                for (int r = 0; r < R; ++r)
                    flush(0, step, *reinterpret_cast<const uint32_t*>(stage + kCodes + (r * 32 + lane) * 4), sum[r], acc[r]);
            }
            at = at == STAGES - 1 ? 0 : at + 1;
        }
        copy_wait<0>();
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
// stream's previous kernel ends; they touch global memory only after griddepcontrol.wait.
template <auto KERNEL, typename Params>
int launch(dim3 grid, int threads, int cluster, size_t smem, cudaStream_t stream, const Params& p) {
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
    if (cudaLaunchKernelEx(&cfg, KERNEL, p) == cudaSuccess) return 0;
    cudaGetLastError();
    return -4;  // HGEMM_ERR_CUDA
}

inline bool misaligned(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1u)) != 0; }

// Calls go(std::integral_constant<int, GROUP>, std::bool_constant<ZERO>) for a weight's group size and kind.
template <typename Go>
int with_format(int group, bool zeros, Go go) {
    using std::integral_constant;
    if (group == 32) return zeros ? go(integral_constant<int, 32>{}, std::true_type{}) : go(integral_constant<int, 32>{}, std::false_type{});
    if (group == 64) return zeros ? go(integral_constant<int, 64>{}, std::true_type{}) : go(integral_constant<int, 64>{}, std::false_type{});
    return zeros ? go(integral_constant<int, 128>{}, std::true_type{}) : go(integral_constant<int, 128>{}, std::false_type{});
}

}  // namespace hgw
