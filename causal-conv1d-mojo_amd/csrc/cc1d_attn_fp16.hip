// cc1d_attn_fp16.hip -- linear attention's kernels for fp16, of whole vectors.
#include "cc1d_attn_kernels.hpp"

namespace cc1d {

template <> int launch_attn_modes<f16, true>(const AttnArgs& a, int da, int dc, bool states, hipStream_t stream) {
    return launch_attn_modes_impl<f16, true>(a, da, dc, states, stream);
}

}  // namespace cc1d
