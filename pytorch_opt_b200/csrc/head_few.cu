// Logits of a few rows with their softmax statistics: what the tensor-core
// kernel of head_gemm.cuh computes for the LOGITS product, on the CUDA cores.
//
// With 1 or 2 rows (8 in fp32) the product is a read of W (2 V D bytes) with 2
// T operations an element; a 256-row tensor-core tile would spend 256 / T times
// the multiplications, and its ring and accumulators take longer to fill than
// the tile to compute. Sums are plain fp32 FMA chains over D / 16 terms and
// three shuffles, so a single token's loss carries no accumulator truncation.
// Bound by memory: 50257 x 768 bf16 for one row 15.2 us, 5.1 TB/s. (Eight fp32
// rows are bound by their loads of H and the FMAs: 32000 x 4096 in 170 us, 3.1
// TB/s, with registers held to 128 for four blocks on an SM; 410 us without.)
//
// A block takes 64 rows of W: a warp 16, in four groups of 8 lanes; a lane
// holds 4 of its group's rows in registers while it walks T rows of H (in L1),
// so a value of H is converted once for 4 products. The 64 logits of each row
// then leave the statistics, the target's logits and the scaled exponentials
// in the formats of the tensor-core kernel, per 64 columns instead of 256.
#include "head_gemm.cuh"

namespace po {
namespace {

constexpr int kFewCols = 64;
constexpr int kFewThreads = 128;
constexpr int R = 4;  // rows of W a lane works on

// 16 bytes at p, of which `left` elements belong to the row, as pairs of floats.
template <int DT>
__device__ __forceinline__ void load_pairs(const typename ElemOf<DT>::T* p, int left, uint64_t (&x)[DT == PO_F32 ? 2 : 4]) {
  constexpr int VEC = DT == PO_F32 ? 4 : 8;
  float f[VEC];
  if (left >= VEC) {
    unpack16<DT>(__ldg(reinterpret_cast<const uint4*>(p)), f);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = i < left ? to_f32(p[i]) : 0.0f;
  }
#pragma unroll
  for (int i = 0; i < VEC / 2; ++i) x[i] = pack2(f[2 * i], f[2 * i + 1]);
}

template <int DT, int TT>
__global__ void __launch_bounds__(kFewThreads, TT == 8 ? 4 : 0) few_rows_kernel(FewParams P) {
  using T = typename ElemOf<DT>::T;
  constexpr int VEC = DT == PO_F32 ? 4 : 8;
  __shared__ float s_z[TT][kFewCols];
  __shared__ double dbuf[32];
  __shared__ int s_last;
  const FinishArgs& F = P.finish;
  grid_launch_next();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = lane & 7;
  const int n0 = blockIdx.x * kFewCols;
  const int r0 = n0 + warp * 16 + (lane >> 3) * R;  // first of the lane's rows of W
  const T* w[R];
#pragma unroll
  for (int i = 0; i < R; ++i)
    w[i] = static_cast<const T*>(P.w) + static_cast<long long>(min(r0 + i, P.V - 1)) * P.w_ld;  // (repeats the last row)
  // The products need the call's own inputs alone, so they run beside the
  // launches before; which rows count is asked for afterwards.
  const T* h[TT];
#pragma unroll
  for (int t = 0; t < TT; ++t) h[t] = static_cast<const T*>(P.h) + (t < F.T ? t * P.h_ld : 0);
  // Even and odd terms of each sum in the halves of a register pair.
  uint64_t acc[R][TT];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int t = 0; t < TT; ++t) acc[i][t] = 0;
  const auto step = [&](int d, int left) {
    uint64_t x[R][VEC / 2];
#pragma unroll
    for (int i = 0; i < R; ++i) load_pairs<DT>(w[i] + d, left, x[i]);
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      uint64_t y[VEC / 2];
      load_pairs<DT>(h[t] + d, left, y);
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int e = 0; e < VEC / 2; ++e) acc[i][t] = fma2(x[i][e], y[e], acc[i][t]);
    }
  };
  int d = sub * VEC;
#pragma unroll (TT == 8 ? 1 : 2)
  for (; d + VEC <= P.D; d += 8 * VEC) step(d, VEC);
  if (d < P.D) step(d, P.D - d);
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      const float2 a = unpack2(acc[i][t]);
      float v = a.x + a.y;
      v += __shfl_xor_sync(0xffffffffu, v, 4);
      v += __shfl_xor_sync(0xffffffffu, v, 2);
      v += __shfl_xor_sync(0xffffffffu, v, 1);
      if (sub == 0) s_z[t][warp * 16 + (lane >> 3) * R + i] = v;
    }
  grid_wait();
  __syncthreads();
  const int count = F.st->count;
  // A warp a counted row, two columns a lane.
  for (int r = warp; r < count; r += kFewThreads / 32) {
    const int c = 2 * lane, t = F.rowmap[r];
    const float z0 = n0 + c < P.V ? s_z[t][c] : -INFINITY, z1 = n0 + c + 1 < P.V ? s_z[t][c + 1] : -INFINITY;
    const float m = warp_max(fmaxf(z0, z1));
    const float off = m == -INFINITY ? 0.0f : -m;
    const float e0 = ex2((z0 + off) * P.scale2), e1 = ex2((z1 + off) * P.scale2);
    const float s = warp_sum(e0 + e1);
    const long long at = static_cast<long long>(r) * F.nparts + blockIdx.x;
    if (lane == 0) P.part[at] = make_float2(m, s);
    if (P.zsum != nullptr) {
      const float zs = warp_sum((n0 + c < P.V ? z0 : 0.0f) + (n0 + c + 1 < P.V ? z1 : 0.0f));
      if (lane == 0) P.zsum[at] = zs;
    }
    if (P.e != nullptr) {
      const long long to = static_cast<long long>(r) * P.e_ld + n0 + c;  // e_ld: a multiple of 256
      if (DT == PO_F32) *reinterpret_cast<float2*>(static_cast<float*>(P.e) + to) = make_float2(e0, e1);
      else *reinterpret_cast<uint32_t*>(static_cast<__half*>(P.e) + to) = pack_f16x2(e0, e1);
    }
    const long long tk = static_cast<long long>(t) * F.top;
    for (int k = lane; k < F.top; k += 32) {
      const int col = F.ent[tk + k] - n0;
      if (col >= 0 && col < kFewCols) P.zpick[tk + k] = s_z[t][col];
    }
  }
  if (count > 0)  // the rows that complete dW's K block
    for (int r = count + blockIdx.x * (kFewThreads / 32) + warp; r < kRowPad; r += gridDim.x * (kFewThreads / 32))
      zero_row(F, r, lane);
  // The last block joins the statistics of all and writes the losses.
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) s_last = atomicAdd(&F.st->done, 1) == static_cast<int>(gridDim.x) - 1;
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  for (int r = warp; r < count; r += kFewThreads / 32) finish_row(F, r, lane);
  if (F.loss == nullptr) return;
  __threadfence();
  __syncthreads();
  finish_total(F, dbuf);
}

template <int DT>
int launch_few_typed(const FewParams& P, int rows, cudaStream_t s) {
  auto kern = rows == 1 ? few_rows_kernel<DT, 1> : few_rows_kernel<DT, 2>;
  if constexpr (DT == PO_F32)
    if (rows > 2) kern = rows <= 4 ? few_rows_kernel<DT, 4> : few_rows_kernel<DT, 8>;
  return launch_next(false, kern, P.finish.nparts, kFewThreads, 0, s, "linear_loss few rows", P);
}

}  // namespace

static_assert(kFewPartCols == kFewCols, "columns a partial statistic covers");

int launch_few_rows(const FewParams& P, int dtype, int rows, cudaStream_t s) {
  if (dtype == PO_F32) return launch_few_typed<PO_F32>(P, rows, s);
  if (dtype == PO_BF16) return launch_few_typed<PO_BF16>(P, rows, s);
  return launch_few_typed<PO_F16>(P, rows, s);
}

}  // namespace po
