// Masked attention with a window and sinks on fp32 storage; the kernels are in masked_attention_kernel.hpp.
#include "masked_attention_kernel.hpp"

void musc::mattn::launch_window_f32(const Args& a, int waves, hipStream_t stream) {
  launch_windowed<MUSC_DTYPE_F32>(a, waves, stream);
}
