// cc1d_attn_bf16_any.hip -- linear attention's kernels for bf16, element by element.
#include "cc1d_attn_kernels.hpp"

namespace cc1d {

template <> int launch_attn_modes<bf16, false>(const AttnArgs& a, int da, int dc, bool states, hipStream_t stream) {
    return launch_attn_modes_impl<bf16, false>(a, da, dc, states, stream);
}

}  // namespace cc1d
