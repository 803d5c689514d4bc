// Loss-head products on 16-bit operands (bf16, fp16).
#include "common.cuh"
#include "head_gemm.cuh"

namespace po {
template int dispatch_head<KIND_BF16>(int, const HeadParams&, int, cudaStream_t);
}
