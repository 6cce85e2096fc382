// cc1d_attn_fp16.hip -- linear attention's kernels for fp16.
#include "cc1d_attn_kernels.hpp"

namespace cc1d {

template <> int launch_attn_jobs<f16>(const AttnArgs& a, int da, int dc, bool states, hipStream_t stream) {
    return states ? launch_attn_sizes<f16, true>(a, da, dc, stream) : launch_attn_sizes<f16, false>(a, da, dc, stream);
}

}  // namespace cc1d
