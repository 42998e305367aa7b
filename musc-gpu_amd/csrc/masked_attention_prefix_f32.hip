// Masked attention after a shared prefix on fp32 storage; the kernels are in masked_attention_kernel.hpp.
#include "masked_attention_kernel.hpp"

void musc::mattn::launch_prefix_f32(const Args& a, const Args* more, int waves, hipStream_t stream) {
  launch_prefixed<MUSC_DTYPE_F32>(a, more, waves, stream);
}
