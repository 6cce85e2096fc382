// cc1d_attn_fp32.hip -- linear attention's kernels for fp32, of whole vectors.
#include "cc1d_attn_kernels.hpp"

namespace cc1d {

template <> int launch_attn_modes<float, true>(const AttnArgs& a, int da, int dc, bool states, hipStream_t stream) {
    return launch_attn_modes_impl<float, true>(a, da, dc, states, stream);
}

}  // namespace cc1d
