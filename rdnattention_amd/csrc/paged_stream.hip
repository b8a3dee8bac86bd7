// Paged attention of few rows: the kernels of calls whose keys are in one part.
#include "paged_stream.hpp"

namespace rdna_amd {

int64_t paged_stream_cost(const PagedAttnArgs&, const PagedWork& w) {
    return paged_max_cost<kRows, kTile, 0>(w);
}

int paged_stream_attention(const PagedAttnArgs& a, PagedJoinParams& p, const PagedLaunch& l, hipStream_t stream,
                           std::string& err) {
    return p.join.any() ? paged_out_stream_attention(a, p, l, stream, err)
                        : paged_stream_launch<false>(a, p, l, stream, err);
}

} // namespace rdna_amd
