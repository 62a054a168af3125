// Host side of the tensor-core product over 4-bit weights (w4_tc.cuh).
#include "w4_tc.cuh"

#include "hipgemm_b200.h"

namespace hg {
uint32_t* status_word(int dev);  // hipgemm_b200.cu
}

namespace hgw {

// Clusters of `split` CTAs, one an SM, that fit the device (defined in w4.cu).
int resident_clusters(int split, int sms, int dev);

// CTAs that share a row group's K, by the time of the waves: a wave takes a CTA's steps, about 8 more to begin and
// end, and 4 for the exchange between CTAs.
static int choose_tc_split(int tiles, int steps, int sms, int dev) {
    int best = 1;
    long long least = 0;
    for (int split = 1; split <= 4; split *= 2) {
        const int fit = resident_clusters(split, sms, dev);
        if (fit < 1 || (split > 1 && steps < 4 * split)) continue;
        const long long cost = static_cast<long long>(ceil_div(tiles, fit)) * (ceil_div(steps, split) + 8 + (split > 1 ? 4 : 0));
        if (split == 1 || cost < least) best = split, least = cost;
    }
    return best;
}

template <int NC, int GROUP, bool ZERO>
static int launch_tc(const TcParams& p, int sms, int dev, cudaStream_t stream) {
    using S = TcShape<NC>;
    constexpr auto kernel = w4_tc_kernel<NC, GROUP, ZERO>;
    if (resident_ctas<kernel>(dev, S::kWarps * 32, S::kSmem) < 1) return HGEMM_ERR_CUDA;
    const int groups = ceil_div(p.w.row_blocks, 8), columns = ceil_div(p.M, NC);
    const int split = choose_tc_split(groups * columns, ceil_div(p.w.k_blocks, 2), sms, dev);
    return launch<kernel>(dim3(static_cast<unsigned>(groups) * split, static_cast<unsigned>(columns), 1), S::kWarps * 32, split,
                          S::kSmem, stream, p);
}

// x: rows 16-byte aligned, K a multiple of 8.
int run_tc(const void* x, long long ldx, void* y, int M, int N, int K, const Weight& w, int group, bool stall, int sms,
           int dev, cudaStream_t stream) {
    TcParams p{static_cast<const __nv_bfloat16*>(x), ldx, static_cast<__nv_bfloat16*>(y), M, N, K, w, hg::status_word(dev), stall};
    if (!p.status) return HGEMM_ERR_CUDA;
    return with_format(group, w.zeros != nullptr, [&](auto g, auto z) {
        constexpr int G = decltype(g)::value;
        constexpr bool Z = decltype(z)::value;
        if (M <= 32) return launch_tc<32, G, Z>(p, sms, dev, stream);
        return launch_tc<64, G, Z>(p, sms, dev, stream);
    });
}

}  // namespace hgw
