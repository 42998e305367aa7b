// Masked attention after a shared prefix on fp16 storage (its matrix instructions, __builtin_amdgcn_mfma_*, are in
// masked_attention_kernel.hpp).
#include "masked_attention_kernel.hpp"

void musc::mattn::launch_prefix_f16(const Args& a, int waves, const Args* more, int more_waves, hipStream_t stream) {
  launch_prefixed<MUSC_DTYPE_F16>(a, waves, more, more_waves, stream);
}
