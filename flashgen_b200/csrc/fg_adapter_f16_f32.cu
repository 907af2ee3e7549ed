// fg_adapter_f16_f32.cu — the LM-head kernels with f16 operands and f32 logits.
#include "fg_adapter_launch.cuh"

template int fg::adapt::launch<FG_DTYPE_F16, FG_DTYPE_F32>(const fg::adapt::Params&, const CUtensorMap&,
                                                          const CUtensorMap&, bool, fg::host::DevInfo*, cudaStream_t);
