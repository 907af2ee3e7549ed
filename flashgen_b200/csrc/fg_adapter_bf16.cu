// fg_adapter_bf16.cu — the LM-head kernels with bf16 operands and bf16 logits.
#include "fg_adapter_launch.cuh"

template int fg::adapt::launch<FG_DTYPE_BF16, FG_DTYPE_BF16>(const fg::adapt::Params&, const CUtensorMap&,
                                                          const CUtensorMap&, bool, fg::host::DevInfo*, cudaStream_t);
