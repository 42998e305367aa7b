// Masked attention on fp32 storage (its matrix instructions, __builtin_amdgcn_mfma_*, are in
// masked_attention_kernel.hpp).
#include "masked_attention_kernel.hpp"

void musc::mattn::launch_f32(const Args& a, int waves, hipStream_t stream) {
  launch_all<MUSC_DTYPE_F32>(a, waves, stream);
}
