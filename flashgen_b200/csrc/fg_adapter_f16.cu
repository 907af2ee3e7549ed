// fg_adapter_f16.cu — the LM-head kernels with f16 operands and f16 logits.
#include "fg_adapter_launch.cuh"

template int fg::adapt::launch<FG_DTYPE_F16, FG_DTYPE_F16>(const fg::adapt::Params&, const CUtensorMap&,
                                                          const CUtensorMap&, bool, fg::host::DevInfo*, cudaStream_t);
