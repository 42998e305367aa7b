// Masked attention after a shared prefix on bf16 storage; the kernels are in masked_attention_kernel.hpp.
#include "masked_attention_kernel.hpp"

void musc::mattn::launch_prefix_bf16(const Args& a, const Args* more, int waves, hipStream_t stream) {
  launch_prefixed<MUSC_DTYPE_BF16>(a, more, waves, stream);
}
