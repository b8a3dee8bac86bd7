// Paged attention of many rows: the kernels of calls whose keys are in one part.
#include "paged_tiles.hpp"

namespace rdna_amd {

int64_t paged_tile_cost(const PagedAttnArgs& a, const PagedWork& w) {
    return a.D <= 128 ? paged_max_cost<TileCfg<128, false>::ROWS, kBN, kItemCost>(w)
                      : paged_max_cost<TileCfg<256, false>::ROWS, kBN, kItemCost>(w);
}

int paged_tile_attention(const PagedAttnArgs& a, PagedJoinParams& p, const PagedLaunch& l, hipStream_t stream,
                         std::string& err) {
    return p.join.any() ? paged_join_tile_attention(a, p, l, stream, err)
                        : paged_tile_launch<false>(a, p, l, stream, err);
}

} // namespace rdna_amd
