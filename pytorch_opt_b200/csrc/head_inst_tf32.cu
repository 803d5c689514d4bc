// Loss-head products on fp32 operands held as tf32 (hi, lo) pairs.
#include "common.cuh"
#include "head_gemm.cuh"

namespace po {
template int dispatch_head<KIND_TF32>(int, const HeadParams&, int, cudaStream_t);
}
