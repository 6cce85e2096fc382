// cc1d_attn_fp32.hip -- linear attention's kernels for fp32.
#include "cc1d_attn_kernels.hpp"

namespace cc1d {

template <> int launch_attn_jobs<float>(const AttnArgs& a, int da, int dc, bool states, hipStream_t stream) {
    return launch_attn_modes<float>(a, da, dc, states, stream);
}

}  // namespace cc1d
