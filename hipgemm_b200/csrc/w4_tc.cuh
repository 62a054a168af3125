// y[M, N] = x[M, K] . W[N, K]^T over 4-bit weights on the 5th-generation tensor cores, for more than 16
// rows of bf16 x.
//
// The A operand is made, not loaded: warps turn codes into bf16 (code - zero, exact) in registers and
// store them to tensor memory, whose fragment-shaped store (16x256b) takes a 16 x 64 tile of the
// blocked layout in one instruction: a tile's word j of lane 4 g + t is rows g and g + 8, columns 2 t
// and 2 t + 1 of the 8 32-bit columns that one 16-deep tcgen05.mma reads.  128 rows of W are the
// MMA's M; the rows of x are its N, so the cost of unpacking does not depend on how many there are
// (with mma.sync each 8 rows cost another 32 cycles a tile, of the 86 that HBM speed allows).
// The group's sum is read back from tensor memory (two accumulators take turns) and added to
// registers times its scale, in fp32.
//
// Roles of a CTA: 8 flush warps, a thread a row of W; unpacking warps in teams of 4 that take a
// step of 128 K each in turn, 4 tiles a warp; 3 warps that copy x to shared memory, a step each in
// turn; and one that issues the MMAs.  (A step a team, not a tile a warp: every step costs a role
// some 500 cycles of latency - store, wait, signal - whatever it does in it.)  Codes come by
// asynchronous copies, 8 steps ahead, private to the lane that unpacks them.  x is copied by 8 bytes:
// the MMA's 16 K are, as the codes' words have them, 4 of each of four 8-element stretches.
//
// What bounds it: latencies and instructions of the roles (28672 x 8192 by 32 rows: 52.6 us, 2.2 TB/s of
// codes; 8192 x 8192 by 64: 21.7 us, where copying x takes a warp 1500 cycles a step), far from the
// tensor cores' rate; mma.sync takes 88.5 and 44.3 us.
#pragma once

#define HG_PTX_WITHOUT_STATUS
#include <cooperative_groups.h>

#include "ptx.cuh"
#include "w4.cuh"

namespace hgw {

struct TcParams {
    const __nv_bfloat16* x;
    long long ldx;
    __nv_bfloat16* y;
    int M, N, K;
    Weight w;
    uint32_t* status;
    bool stall;  // test hook (hgemm_debug_stalled_w4 only): the first step's x is never reported as copied
};

constexpr int kCopyWarps = 3;

template <int NC>
struct TcShape {
    static_assert(NC == 32 || NC == 64, "columns");
    // 8 flush warps: two halves of the columns, or two teams that take groups in turn (a group costs a flush
    // warp some 500 cycles of latency, a step's codes at HBM speed 350).
    static constexpr int kFlushWarps = 8, kFlushTeams = NC == 64 ? 1 : 2;
    static constexpr int kColumns = NC == 64 ? 32 : NC;  // columns of a flush warp
    // 20 warps leave 96 registers a thread.  (With 29 warps, at 64 registers, a few spills made every step 1500 cycles
    // longer: nearly all of L1 is shared memory here.)
    static constexpr int kUnpackWarps = 8;
    static constexpr int kWarps = kFlushWarps + kUnpackWarps + kCopyWarps + 1;
    static constexpr int kAStages = NC == 32 ? 6 : 4, kTeams = kUnpackWarps / 4;
    // Turns that copies run ahead: 8 steps for codes, 3 or 9 for x, whose stages are those, and kAStages more that
    // MMAs may still read.
    static constexpr int kAhead = 8 / kTeams, kXAhead = NC == 64 ? 1 : 3;
    static constexpr int kXStages = kCopyWarps * kXAhead + kAStages;
    static constexpr int kBuffers = 4;  // accumulators
    static constexpr int kTmemColumns = 512, kAColumns = kStepK / 2, kA = kBuffers * NC;  // accumulators, then A's stages
    static_assert(kA + kAStages * kAColumns <= kTmemColumns, "tensor memory");
    static constexpr int kTurnBytes = 4 * kTileBytes;
    static constexpr int kCodeBytes = kUnpackWarps * (kAhead + 1) * kTurnBytes;
    static constexpr int kXBytes = NC * kStepK * 2;
    static constexpr int kSums = NC * 128 * 4;
    static_assert(kSums <= kXStages * kXBytes, "the sums lie over x");
    static constexpr int kSmem = kXStages * kXBytes + kCodeBytes;
};

struct TcBarriers {
    uint64_t full[8], a_empty[8], d_full[4], d_empty[4];  // full: a step's A and x
    uint32_t tmem;
    volatile uint32_t abort;
};

// A wait that ends: after HG_WAIT_LIMIT_NS the code is recorded and every role of the CTA gives up.
__device__ __forceinline__ bool tc_wait(uint32_t bar, uint32_t parity, TcBarriers& b, uint32_t* status, uint32_t code) {
    if (hg::mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = hg::globaltimer_ns();
    for (uint32_t n = 1;; ++n) {
        if (hg::mbar_try_wait(bar, parity)) return true;
        if ((n & 15u) == 0) {
            if (b.abort) return false;
            if (hg::globaltimer_ns() - t0 > HG_WAIT_LIMIT_NS) {
                b.abort = 1u;
                atomicCAS(status, 0u, code);
                return false;
            }
        }
    }
}

// The same for a whole warp, whose lanes go on together or not at all (what follows is warp-wide).
__device__ __forceinline__ bool tc_wait_warp(uint32_t bar, uint32_t parity, TcBarriers& b, uint32_t* status, uint32_t code) {
    return __all_sync(0xffffffffu, tc_wait(bar, parity, b, status, code)) != 0;
}

// D[tmem] (+)= A[tmem] * B[smem]^T, bf16 x bf16 -> f32, and a commit: called by a whole warp, issued by the
// lane with `elected`.  (In a branch of one lane every operand would have to be moved to uniform registers
// first: 66 cycles an MMA were measured that way, and there are 8 a step.)
__device__ __forceinline__ void mma_f16_tmem_a(uint32_t d, uint32_t a, uint64_t b_desc, uint32_t idesc, uint32_t accumulate,
                                               uint32_t elected) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
        "r"(a), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(elected)
        : "memory");
}
__device__ __forceinline__ void commit_by(uint32_t bar, uint32_t elected) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(bar),
        "r"(elected)
        : "memory");
}
__device__ __forceinline__ uint32_t elect() {
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(e));
    return e;
}

// 16 lanes x 32 columns: lane 4 g + t has, of each 8 columns, 2 t and 2 t + 1 of rows g and g + 8.
__device__ __forceinline__ void tmem_st_16x256b_x4(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// 8 bytes, or zeros where !valid (nothing is read then).
__device__ __forceinline__ void copy8(uint32_t smem, const void* src, bool valid) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(smem), "l"(src), "r"(valid ? 8 : 0) : "memory");
}

template <int NC, int GROUP, bool ZERO>
__global__ void __launch_bounds__(TcShape<NC>::kWarps * 32, 1) w4_tc_kernel(const TcParams p) {
    using S = TcShape<NC>;
    constexpr int kGroups = kStepK / GROUP;
    extern __shared__ __align__(1024) uint8_t smem[];  // x's stages, then the unpacking warps' codes
    __shared__ TcBarriers bars;
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    const int split = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    const int block0 = static_cast<int>(blockIdx.x) / split * 8, col0 = static_cast<int>(blockIdx.y) * NC;
    const int all_steps = ceil_div(p.w.k_blocks, 2);
    const int first = static_cast<int>(static_cast<unsigned>(all_steps) * rank / split);
    const int steps = static_cast<int>(static_cast<unsigned>(all_steps) * (rank + 1) / split) - first;
    auto bar = [](uint64_t& b) { return hg::smem_u32(&b); };

    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(hg::smem_u32(&bars.tmem)),
                     "r"(S::kTmemColumns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    } else if (warp == 1 && lane == 0) {
        for (int i = 0; i < S::kAStages; ++i) {
            hg::mbar_init(bar(bars.full[i]), 5);  // 4 unpacking warps, 1 that copies x
            hg::mbar_init(bar(bars.a_empty[i]), 1);
        }
        for (int i = 0; i < S::kBuffers; ++i) {
            hg::mbar_init(bar(bars.d_full[i]), 1);
            hg::mbar_init(bar(bars.d_empty[i]), S::kFlushWarps / S::kFlushTeams);
        }
        bars.abort = 0u;
        hg::fence_mbarrier_init();
    }
    hg::tc_fence_before();
    __syncthreads();
    hg::tc_fence_after();
    const uint32_t tmem = bars.tmem;
    pdl_trigger();
    pdl_wait();

    float acc[S::kColumns];
    if (warp < S::kFlushWarps) {
        // ---- flush: acc += scale * (the group's sums) --------------------------------------------
        const int sub = warp & 3, team = S::kFlushTeams == 2 ? warp / 4 : 0, c0 = S::kFlushTeams == 2 ? 0 : warp / 4 * S::kColumns;
        // This thread's row: its row block, and its place among the block's scales.
        const int block = min(block0 + 2 * sub + lane / 16, p.w.row_blocks - 1), r = lane & 15;
        const unsigned short* scales = reinterpret_cast<const unsigned short*>(p.w.scales + p.w.group_base(0, block)) + (r & 7) * 2 + r / 8;
#pragma unroll
        for (int i = 0; i < S::kColumns; ++i) acc[i] = 0.0f;
        // The scales of a turn of 4 steps are loaded a turn ahead: they come from HBM like the codes.
        constexpr int kMine = 4 * kGroups / S::kFlushTeams;  // this team's groups of a turn
        uint32_t next[kMine], now[kMine / 2];
        auto load_scales = [&](int s) {
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
                const int group = (first + s) * kGroups + S::kFlushTeams * i + team;
                next[i] = group < p.w.groups ? scales[static_cast<size_t>(group) * 16] : 0u;
            }
        };
        load_scales(0);
        bool alive = true;
        for (int s0 = 0; s0 < steps && alive; s0 += 4) {
#pragma unroll
            for (int i = 0; i < kMine / 2; ++i) now[i] = next[2 * i] | next[2 * i + 1] << 16;
            load_scales(s0 + 4);
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
                const uint32_t use = static_cast<uint32_t>(s0 * kGroups + S::kFlushTeams * i + team), buffer = use % S::kBuffers;
                if (use >= static_cast<uint32_t>(steps * kGroups)) break;
                if (!alive || !tc_wait_warp(bar(bars.d_full[buffer]), use / S::kBuffers & 1u, bars, p.status, 0x0401u)) {
                    alive = false;
                    break;
                }
                hg::tc_fence_after();
                const uint32_t from = tmem + (static_cast<uint32_t>(32 * sub) << 16) + buffer * NC + c0;
                uint32_t v[S::kColumns / 16][16];
#pragma unroll
                for (int c = 0; c < S::kColumns / 16; ++c) hg::tmem_ld_32x32b_x16(from + 16 * c, v[c]);
#pragma unroll
                for (int c = 0; c < S::kColumns / 16; ++c) hg::tmem_ld_wait(v[c]);
                hg::tc_fence_before();
                __syncwarp();
                if (lane == 0) hg::mbar_arrive(bar(bars.d_empty[buffer]));
                const float scale = i & 1 ? bf16_hi(now[i / 2]) : bf16_lo(now[i / 2]);
#pragma unroll
                for (int c = 0; c < S::kColumns; ++c) acc[c] = fmaf(scale, __uint_as_float(v[c / 16][c % 16]), acc[c]);
            }
        }
    } else if (warp < S::kFlushWarps + S::kUnpackWarps) {
        // ---- unpack: codes -> bf16 in tensor memory ------------------------------------------------
        const int u = warp - S::kFlushWarps, sub = warp & 3, team = u / 4;
        const uint8_t* q[2];
        const uint16_t* zeros[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int block = min(block0 + 2 * sub + half, p.w.row_blocks - 1);
            q[half] = p.w.q + p.w.tile_base(0, block) + lane * 16;
            zeros[half] = p.w.zeros + p.w.group_base(0, block) + lane / 4;
        }
        uint8_t* ring = smem + S::kXStages * S::kXBytes + u * ((S::kAhead + 1) * S::kTurnBytes) + lane * 16;
        const uint32_t ring_at = hg::smem_u32(ring);
        const UnpackConstants constants;
        // Tile 2 half + kh of a turn: row block `half` of the warp's two, K block kh of the step's two.
        auto copy = [&](int s, int slot) {
#pragma unroll
            for (int kh = 0; kh < 2; ++kh) {
                const int kb = 2 * (first + s) + kh;
                if (s < steps && kb < p.w.k_blocks) {
#pragma unroll
                    for (int half = 0; half < 2; ++half)
                        copy16(ring_at + slot * S::kTurnBytes + (2 * half + kh) * kTileBytes, q[half] + static_cast<size_t>(kb) * kTileBytes);
                }
            }
            copy_commit();
        };
        uint32_t next[2][kGroups], zero[2][kGroups];
        auto load_zeros = [&](int s) {
            if (!ZERO) return;
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int i = 0; i < kGroups; ++i)
                    next[half][i] = zeros[half][static_cast<size_t>(min((first + s) * kGroups + i, p.w.groups - 1)) * 8];
        };
#pragma unroll
        for (int v = 0; v < S::kAhead; ++v) copy(team + S::kTeams * v, v);
        load_zeros(team);
        int slot = 0;
        for (int s = team; s < steps; s += S::kTeams) {
            copy(s + S::kTeams * S::kAhead, slot == 0 ? S::kAhead : slot - 1);
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int i = 0; i < kGroups; ++i) zero[half][i] = next[half][i];
            load_zeros(s + S::kTeams);
            const uint32_t stage = static_cast<uint32_t>(s) % S::kAStages, round = static_cast<uint32_t>(s) / S::kAStages;
            if (!tc_wait_warp(bar(bars.a_empty[stage]), (round & 1u) ^ 1u, bars, p.status, 0x0501u)) break;
            hg::tc_fence_after();
            copy_wait<S::kAhead>();
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int kh = 0; kh < 2; ++kh) {
                    // A tile past the end of K: whatever lies in the ring, finite as bf16, against zeros of x.
                    const uint4 codes = *reinterpret_cast<const uint4*>(ring + slot * S::kTurnBytes + (2 * half + kh) * kTileBytes);
                    const uint32_t words[4] = {codes.x, codes.y, codes.z, codes.w};
                    uint32_t r[16];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint32_t z0 = 0x43084308u, z1 = 0x43084308u;  // 128 + 8
                        if (ZERO) {
                            z0 = __byte_perm(zero[half][(64 * kh + 16 * j) / GROUP], 0x43u, 0x4040);
                            z1 = __byte_perm(zero[half][(64 * kh + 16 * j) / GROUP], 0x43u, 0x4141);
                        }
                        uint32_t a[4];
                        unpack(words[j], constants, z0, z1, a);
                        r[4 * j] = a[0];
                        r[4 * j + 1] = a[2];
                        r[4 * j + 2] = a[1];
                        r[4 * j + 3] = a[3];
                    }
                    tmem_st_16x256b_x4(tmem + (static_cast<uint32_t>(32 * sub + 16 * half) << 16) + S::kA + stage * S::kAColumns + 32 * kh, r);
                }
            slot = slot == S::kAhead ? 0 : slot + 1;
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            hg::tc_fence_before();
            __syncwarp();
            if (lane == 0) hg::mbar_arrive(bar(bars.full[stage]));
        }
        copy_wait<0>();
    } else if (warp < S::kFlushWarps + S::kUnpackWarps + kCopyWarps) {
        // ---- x to shared memory: K-major core matrices (8 rows x 16 bytes), no swizzle ---------------
        const int c = warp - S::kFlushWarps - S::kUnpackWarps, n8 = lane / 4, t = lane & 3;
        const uint32_t base = hg::smem_u32(smem);
        // Row group i of 8 rows and 32-K part f: this lane has 8 elements of one row, two pieces of 8 bytes.
        // Piece jk of part f goes to MMA 2 f + jk, slots 4 t .. 4 t + 3.
        auto copy = [&](int s) {
            if (s < steps) {
                const uint32_t stage = base + static_cast<uint32_t>(s) % S::kXStages * S::kXBytes + t / 2 * (NC * 16) + n8 * 16 + (t & 1) * 8;
#pragma unroll
                for (int f = 0; f < 4; ++f) {
                    const int k = (first + s) * kStepK + 32 * f + 8 * t;
                    const bool valid = k < p.K;  // K is a multiple of 8
#pragma unroll
                    for (int i = 0; i < NC / 8; ++i) {
                        const int row = min(col0 + 8 * i + n8, p.M - 1);  // columns past M repeat the last row, unused
                        const __nv_bfloat16* src = p.x + row * p.ldx + (valid ? k : 0);
#pragma unroll
                        for (int jk = 0; jk < 2; ++jk) copy8(stage + (2 * f + jk) * (NC * 32) + i * 128, src + 4 * jk, valid);
                    }
                }
            }
            copy_commit();
        };
#pragma unroll
        for (int v = 0; v < S::kXAhead; ++v) copy(c + kCopyWarps * v);
        for (int s = c; s < steps; s += kCopyWarps) {
            // The stage that is filled next was read by the MMAs of step s - kAStages.
            const uint32_t round = static_cast<uint32_t>(s) / S::kAStages;
            if (!tc_wait_warp(bar(bars.a_empty[static_cast<uint32_t>(s) % S::kAStages]), (round & 1u) ^ 1u, bars, p.status, 0x0601u)) break;
            copy(s + kCopyWarps * S::kXAhead);
            copy_wait<S::kXAhead>();
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the MMA reads through the async proxy
            __syncwarp();
            if (lane == 0 && !(p.stall && s == 0)) hg::mbar_arrive(bar(bars.full[static_cast<uint32_t>(s) % S::kAStages]));
        }
        copy_wait<0>();
    } else {
        // ---- MMA ------------------------------------------------------------------------------
        // D f32, A and B bf16, both K-major: N / 8 at bit 17, M / 16 at bit 24.
        constexpr uint32_t kIdesc = (1u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(NC / 8) << 17) | (8u << 24);
        // No swizzle: core matrices NC * 16 bytes apart along K, 128 along N.
        const uint64_t desc = (static_cast<uint64_t>(NC) << 16 | static_cast<uint64_t>(128 >> 4) << 32 | 1ull << 46) +
                              ((hg::smem_u32(smem) & 0x3FFFFu) >> 4);
        const uint32_t columns = __shfl_sync(0xffffffffu, tmem, 0), elected = elect();
        // Two groups at a time, with all their waits under way together: a wait costs 130 cycles even where there is
        // nothing to wait for.
        const int groups = steps * kGroups;
        uint32_t xs = 0;  // the x stage of the step
        bool alive = true;
        for (int g = 0; g < groups; g += 2) {
            const uint32_t s = static_cast<uint32_t>(g) / kGroups, b0 = static_cast<uint32_t>(g) % S::kBuffers;
            const uint32_t empty = (static_cast<uint32_t>(g) / S::kBuffers & 1u) ^ 1u;
            const bool two = g + 1 < groups, new_step = g % kGroups == 0, next_step = kGroups == 1 && two;
            const uint32_t f0 = bar(bars.full[s % S::kAStages]), f1 = bar(bars.full[(s + 1) % S::kAStages]);
            const uint32_t p0 = s / S::kAStages & 1u, p1 = (s + 1) / S::kAStages & 1u;
            bool ready = hg::mbar_try_wait(bar(bars.d_empty[b0]), empty);
            if (two) ready &= hg::mbar_try_wait(bar(bars.d_empty[b0 + 1]), empty);
            if (new_step) ready &= hg::mbar_try_wait(f0, p0);
            if (next_step) ready &= hg::mbar_try_wait(f1, p1);
            if (!__all_sync(0xffffffffu, ready)) {
                alive = tc_wait_warp(bar(bars.d_empty[b0]), empty, bars, p.status, 0x0703u) &&
                        (!two || tc_wait_warp(bar(bars.d_empty[b0 + 1]), empty, bars, p.status, 0x0703u)) &&
                        (!new_step || tc_wait_warp(f0, p0, bars, p.status, 0x0701u)) &&
                        (!next_step || tc_wait_warp(f1, p1, bars, p.status, 0x0701u));
                if (!alive) break;
            }
            hg::tc_fence_after();
#pragma unroll
            for (uint32_t j = 0; j < 2; ++j) {
                if (j == 1 && !two) break;
                const uint32_t step = (static_cast<uint32_t>(g) + j) / kGroups, in_step = (static_cast<uint32_t>(g) + j) % kGroups;
                const uint32_t a = step % S::kAStages;
#pragma unroll
                for (uint32_t k = 0; k < GROUP / 16; ++k) {
                    const uint32_t at = in_step * (GROUP / 16) + k;
                    mma_f16_tmem_a(columns + (b0 + j) * NC, columns + S::kA + a * S::kAColumns + at * 8,
                                   desc + (xs * (S::kXBytes / 16) + at * (NC * 2)), kIdesc, k > 0, elected);
                }
                commit_by(bar(bars.d_full[b0 + j]), elected);
                if (in_step == kGroups - 1) {
                    commit_by(bar(bars.a_empty[a]), elected);
                    xs = xs == S::kXStages - 1 ? 0 : xs + 1;
                }
            }
        }
        // The last commit has arrived before this CTA's shared memory is another's.
        const uint32_t last = static_cast<uint32_t>(steps - 1);
        if (alive && steps > 0)
            tc_wait_warp(bar(bars.a_empty[last % S::kAStages]), last / S::kAStages & 1u, bars, p.status, 0x0704u);
    }

    // All MMAs' sums have been read, so that no MMA is running, unless a wait expired: then what is in flight
    // gets time to land before its memory is freed.
    hg::tc_fence_before();
    __syncthreads();
    hg::tc_fence_after();
    if (bars.abort) hg::sleep_ns_bounded(100000);
    if (warp == 0) hg::tmem_dealloc<1>(tmem, S::kTmemColumns);

    const int columns = min(NC, p.M - col0);
    float* sums = reinterpret_cast<float*>(smem);  // [column][row]
    const int c0 = S::kFlushTeams == 2 ? 0 : warp / 4 * S::kColumns, in_tile = 32 * (warp & 3) + lane;
    if (S::kFlushTeams == 2) {
        // The second team's sums to the first.
        if (warp >= 4 && warp < 8) {
#pragma unroll
            for (int c = 0; c < S::kColumns; ++c) sums[c * 128 + in_tile] = acc[c];
        }
        __syncthreads();
        if (warp < 4) {
#pragma unroll
            for (int c = 0; c < S::kColumns; ++c) acc[c] += sums[c * 128 + in_tile];
        }
    }
    const bool holds = warp < (S::kFlushTeams == 2 ? 4 : 8);
    if (split == 1) {
        const int row = block0 * 16 + in_tile;
        if (holds && row < p.N) {
#pragma unroll
            for (int c = 0; c < S::kColumns; ++c)
                if (c0 + c < columns) p.y[static_cast<size_t>(col0 + c0 + c) * p.N + row] = __float2bfloat16_rn(acc[c]);
        }
        return;
    }
    if (holds) {
#pragma unroll
        for (int c = 0; c < S::kColumns; ++c) sums[(c0 + c) * 128 + in_tile] = acc[c];
    }
    cluster.sync();
    for (int i = rank * (S::kWarps * 32) + threadIdx.x; i < columns * 128; i += split * (S::kWarps * 32)) {
        float v = 0.0f;
        for (int s = 0; s < split; ++s) v += cluster.map_shared_rank(sums, s)[i];
        const int row = block0 * 16 + (i & 127);
        if (row < p.N) p.y[static_cast<size_t>(col0 + (i >> 7)) * p.N + row] = __float2bfloat16_rn(v);
    }
    cluster.sync();  // no CTA leaves while another reads its sums
}

}  // namespace hgw
