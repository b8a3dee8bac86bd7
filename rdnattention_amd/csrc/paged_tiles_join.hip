// Paged attention of many rows whose keys are in two parts, or with the log-sum-exp.
#include "paged_tiles.hpp"

namespace rdna_amd {

int paged_join_tile_attention(const PagedAttnArgs& a, PagedJoinParams& p, const PagedLaunch& l, hipStream_t stream,
                              std::string& err) {
    return paged_tile_launch<true>(a, p, l, stream, err);
}

} // namespace rdna_amd
