// Paged attention of few rows whose keys are in two parts, or with the log-sum-exp.
#include "paged_stream.hpp"

namespace rdna_amd {

int paged_out_stream_attention(const PagedAttnArgs& a, PagedJoinParams& p, const PagedLaunch& l, hipStream_t stream,
                               std::string& err) {
    return paged_stream_launch<true>(a, p, l, stream, err);
}

} // namespace rdna_amd
