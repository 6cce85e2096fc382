// cc1d_attn_fp32_any.hip -- linear attention's kernels for fp32, element by element.
#include "cc1d_attn_kernels.hpp"

namespace cc1d {

template <> int launch_attn_modes<float, false>(const AttnArgs& a, int da, int dc, bool states, hipStream_t stream) {
    return launch_attn_modes_impl<float, false>(a, da, dc, states, stream);
}

}  // namespace cc1d
