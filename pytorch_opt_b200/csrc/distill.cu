// Divergence of student logits from a teacher's top logits, with its gradient
// (po_distill_logits), and the scaling of gradients by a device scalar.
//
//   q = softmax(teacher / a),  l = a^2 sum_k q_k (log q_k + lse(z/a) - z_k/a),
//   dz = a (softmax(z / a) - q scattered)
//
// Bound by memory: each logit is read once and each gradient written once (4
// bytes a logit in 16-bit types). A row's sum has to be known before its first
// gradient is written, so a row is read twice, the second time from L2: one CTA
// a row keeps about 300 rows in work, 76 MB at 128 thousand 16-bit columns.
// Where there are too few rows for that, a cluster of up to 8 CTAs shares one
// and exchanges (max, sum) through distributed shared memory.
#include <climits>
#include <cmath>

#include "losses.cuh"
#include "ptx.cuh"

namespace po {
namespace {

struct DistillState {
  int count;  // rows that the mean divides by
  unsigned int done;
};

struct DistillArgs {
  const void* z;
  long long ld;
  void* dz;  // nullable
  long long dz_ld;
  long long T;
  int V;
  const long long* index;
  long long index_ld;
  const void* teacher;
  long long teacher_ld;
  int teacher_dtype;
  int top;
  float temperature;
  int mean;
  const float* row_grad;
  float* loss_rows;
  float* loss;
  DistillState* st;
  float* unscale;  // nullable: 1 / store_scale
  int by_powers;   // gradients are stored by powers of two: fp16 ones beside an `unscale`
  int seg;  // elements a CTA takes
};

// Whether the row has an entry with mass; bad indices are found here too.
__device__ __forceinline__ int entry_status(const DistillArgs& a, long long t, int k, long long& x, float& l) {
  x = a.index[t * a.index_ld + k];
  l = -INFINITY;
  if (x >= a.V) return ROW_BAD;
  if (x < 0) return ROW_IGNORED;
  l = load_as_f32(a.teacher, a.teacher_dtype, t * a.teacher_ld + k);
  return l > -INFINITY || isnan(l) ? ROW_COUNTED : ROW_IGNORED;
}

// The power of two that fp16 gradients of a scalar are stored by, so that the
// rounding here comes above fp16's smallest values and the caller's loss scale
// not too late: |dz| <= 2 a / n, times n 2^14 / max(a, 1) at most, n = 1 for a sum.
__device__ __forceinline__ float store_scale(const DistillArgs& a) {
  if (!a.by_powers) return 1.0f;
  const float n = a.mean ? static_cast<float>(a.st->count) : 1.0f;
  return exp2f(floorf(log2f(n / fmaxf(a.temperature, 1.0f))) + 14.0f);
}

// Rows that the mean divides by (counted ones and those with a bad index).
__global__ void __launch_bounds__(256) count_rows_kernel(DistillArgs a) {
  grid_launch_next();
  const int lane = threadIdx.x & 31;
  const long long warps = static_cast<long long>(gridDim.x) * (blockDim.x >> 5);
  int n = 0;
  for (long long t = static_cast<long long>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5); t < a.T; t += warps) {
    bool any = false;
    for (int k = lane; k < a.top; k += 32) {
      long long x;
      float l;
      any |= entry_status(a, t, k, x, l) != ROW_IGNORED;
    }
    n += __any_sync(0xffffffffu, any) ? 1 : 0;
  }
  if (lane == 0 && n > 0) atomicAdd(&a.st->count, n);
}

__device__ __forceinline__ uint32_t cluster_nctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void st_cluster_f2(const float2* p, uint32_t rank, float x, float y) {
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(mapa_shared(smem_u32(p), rank)), "f"(x), "f"(y)
               : "memory");
}

// The warp's (m, s) joined: sums of 2^(scale2 z) relative to their maxima. An
// empty one holds (-inf, 0), or a NaN sum, which is kept.
__device__ __forceinline__ void warp_join(float scale2, float& m, float& s) {
  const float top = warp_max(m);
  s = warp_sum(m == -INFINITY ? s : s * ex2((m - top) * scale2));
  m = top;
}

// Largest of a vector's values: the 16-bit types compare two at a time.
template <int DT>
__device__ __forceinline__ float max16(const uint4& v) {
  if constexpr (DT == PO_F32) {
    return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
  } else if constexpr (DT == PO_BF16) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
    const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
  } else {
    const __half2* h = reinterpret_cast<const __half2*>(&v);
    const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
  }
}

// (m, s) <- (m, s) joined with a vector of logits.
template <int DT>
__device__ __forceinline__ void online_add(const uint4& raw, float scale2, float& m, float& s) {
  constexpr int N = DT == PO_F32 ? 4 : 8;
  const float c = max16<DT>(raw);
  if (c > m) {
    s *= ex2((m - c) * scale2);
    m = c;
  }
  // The maximum is subtracted before the scaling: exact where it matters, and a
  // row of the type's lowest value does not overflow.
  const float off = m == -INFINITY ? 0.0f : -m;
  const uint64_t off2 = pack2(off, off), sc2 = pack2(scale2, scale2);
  float x[N];
  unpack16<DT>(raw, x);
  uint64_t add = 0;
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const float2 e = unpack2(mul2(add2(pack2(x[i], x[i + 1]), off2), sc2));
    add = add2(add, pack2(ex2(e.x), ex2(e.y)));
  }
  const float2 a = unpack2(add);
  s += a.x + a.y;
}

// Threads a CTA has at most (and one warp more), and CTAs an SM should hold.
// With gradients 512 and 2: the rows in work (256 KB each at 128 thousand
// 16-bit columns) stay in L2 between their two reads; 2048 such rows 224 us,
// with 256 threads 257 us. Without: 256 and 5, 94 us against 107 us.
constexpr int kGradThreads = 512, kEvalThreads = 256;
constexpr int kMaxPairs = 8 * kGradThreads / 32;

// A CTA's part of one row: the vectors of its segment lie on 16-byte
// boundaries of the logits; the first holds `mis` elements that belong to
// someone else, and so may the last. Whole vectors j0 .. j1 - 1 go to the
// threads in turn, the up to two others (read and written element by element)
// to threads 0 and 1.
template <typename T>
struct Segment {
  static constexpr int VEC = 16 / sizeof(T);
  const T* z0;
  int mis, end, j0, j1, edge;
  __device__ __forceinline__ Segment(const T* row, int s0, int s1) {
    mis = static_cast<int>((reinterpret_cast<uintptr_t>(row + s0) / sizeof(T)) % VEC);
    z0 = row + s0 - mis;
    end = s1 - s0 + mis;
    j0 = mis > 0 ? 1 : 0;
    j1 = end / VEC;
    const int nvec = (end + VEC - 1) / VEC;
    edge = -1;
    if (threadIdx.x == 0 && j0 > 0 && nvec > 0) edge = 0;
    if (threadIdx.x == 1 && j1 < nvec && j1 >= j0) edge = j1;
  }
  __device__ __forceinline__ uint4 load_edge() const {  // others' elements read as -inf
    uint4 raw;
    T* o = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int c = edge * VEC + i;
      from_f32(-INFINITY, o[i]);
      if (c >= mis && c < end) o[i] = z0[c];
    }
    return raw;
  }
  __device__ __forceinline__ void put(T* out0, int j, const uint4& v) const {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int c = j * VEC + i;
      if (c >= mis && c < end) out0[c] = reinterpret_cast<const T*>(&v)[i];
    }
  }
};

// In each of a row's CTAs
//   the last warp takes the teacher's entries, their distribution and the
//   logits there (three dependent loads, which would hold up the row if a
//   warp with a share of the segment made them); whether the row has mass goes
//   by the entries as they are, as in the counting kernel, and their maximum
//   is subtracted before the scaling, as the student's is;
//   the others run over their vectors of the segment (each thread its own)
//   and hand each warp's (max, sum) to every CTA of the row;
//   after one barrier of the row's CTAs every thread joins the row's pairs in
//   the same order and writes its own vectors' gradients, while the last warp
//   of the first CTA writes the loss.
template <int DT, bool GRAD>
__global__ void __launch_bounds__((GRAD ? kGradThreads : kEvalThreads) + 32, GRAD ? 2 : 5)
    distill_kernel(DistillArgs a) {
  using T = typename ElemOf<DT>::T;
  constexpr int VEC = 16 / sizeof(T);
  extern __shared__ __align__(16) uint8_t sm[];
  __shared__ float2 s_pairs[kMaxPairs];  // (max, sum) of every warp of the row's CTAs
  __shared__ double dbuf[32];
  __shared__ float s_qlogq;
  __shared__ int s_status, s_last;
  const uint32_t cs = cluster_nctarank(), rank = cluster_ctarank();
  const long long t = blockIdx.x / cs;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int nthreads = blockDim.x - 32, nwarps = nthreads >> 5;
  const bool teacher_warp = warp == nwarps;
  int* si = reinterpret_cast<int*>(sm);              // entries' indices (-1: none)
  float* sq = reinterpret_cast<float*>(si + a.top);  // q
  float* sz = sq + a.top;                            // logits at the entries
  const float scale2 = kLog2e / a.temperature;
  const T* z = static_cast<const T*>(a.z) + t * a.ld;
  const int s0 = min(static_cast<long long>(rank) * a.seg, static_cast<long long>(a.V));
  const int s1 = min(static_cast<long long>(s0) + a.seg, static_cast<long long>(a.V));
  const Segment<T> g(z, s0, s1);
  const uint4* src = reinterpret_cast<const uint4*>(g.z0);
  grid_wait();  // (behind the counting kernel, where there is one)
  if (cs > 1) cluster_arrive_relaxed();  // this CTA runs: its shared memory may be written

  float m = -INFINITY, s = 0.0f;
  if (teacher_warp) {
    const float inv_temp = 1.0f / a.temperature;
    float tm = -INFINITY;
    int bad = 0, mass = 0;
#pragma unroll 4
    for (int k = lane; k < a.top; k += 32) {
      const long long x = a.index[t * a.index_ld + k];
      const float l = load_as_f32(a.teacher, a.teacher_dtype, t * a.teacher_ld + k);
      const bool there = x >= 0 && x < a.V;
      bad |= x >= a.V;
      mass |= there && !(l == -INFINITY);
      si[k] = there ? static_cast<int>(x) : -1;
      sq[k] = there ? l : -INFINITY;
      sz[k] = there ? to_f32(z[x]) : 0.0f;
      if (there) tm = fmaxf(tm, l);
    }
    bad = __any_sync(0xffffffffu, bad);
    mass = __any_sync(0xffffffffu, mass);
    tm = warp_max(tm);
    float sum = 0.0f;
    for (int k = lane; k < a.top; k += 32) {
      const float e = si[k] >= 0 ? expf((sq[k] - tm) * inv_temp) : 0.0f;
      sum += e;
    }
    sum = warp_sum(sum);
    const float logsum = logf(sum), inv_sum = 1.0f / sum;
    float c = 0.0f;
    for (int k = lane; k < a.top; k += 32) {
      float q = 0.0f;
      if (si[k] >= 0) {
        const float d = (sq[k] - tm) * inv_temp;
        q = expf(d) * inv_sum;
        if (q != 0.0f) c += q * (d - logsum);
      }
      sq[k] = q;
    }
    c = warp_sum(c);
    if (lane == 0) {
      s_qlogq = c;
      s_status = bad ? ROW_BAD : (mass ? ROW_COUNTED : ROW_IGNORED);
    }
  } else {
    for (int j = g.j0 + threadIdx.x; j < g.j1; j += 4 * nthreads) {  // four loads in flight
      uint4 raw[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (j + u * nthreads < g.j1) raw[u] = GRAD ? __ldcg(src + j + u * nthreads) : __ldcs(src + j + u * nthreads);
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (j + u * nthreads < g.j1) online_add<DT>(raw[u], scale2, m, s);
    }
    if (g.edge >= 0) online_add<DT>(g.load_edge(), scale2, m, s);
    warp_join(scale2, m, s);
  }
  // Every warp's pair to every CTA of the row; one barrier for the row (and
  // for what the teacher's warp left in shared memory).
  if (cs > 1) {
    cluster_wait();
    if (lane < cs && !teacher_warp) st_cluster_f2(s_pairs + rank * nwarps + warp, lane, m, s);
    cluster_arrive();
    cluster_wait();
  } else {
    if (lane == 0 && !teacher_warp) s_pairs[warp] = make_float2(m, s);
    __syncthreads();
  }
  {
    const int npairs = static_cast<int>(cs) * nwarps;
    float2 p[kMaxPairs / 32];
    m = -INFINITY;
    s = 0.0f;
#pragma unroll
    for (int u = 0; u < kMaxPairs / 32; ++u) {
      p[u] = lane + 32 * u < npairs ? s_pairs[lane + 32 * u] : make_float2(-INFINITY, 0.0f);
      m = fmaxf(m, p[u].x);
    }
#pragma unroll
    for (int u = 0; u < kMaxPairs / 32; ++u) s += p[u].x == -INFINITY ? p[u].y : p[u].y * ex2((p[u].x - m) * scale2);
    warp_join(scale2, m, s);
  }
  const int status = s_status;
  const bool live = status == ROW_COUNTED;

  if (teacher_warp) {
    if (rank == 0) {
      float c = 0.0f;
      const float logs = logf(s);  // log sum exp(z / a) = m / a + logs
      for (int k = lane; k < a.top; k += 32)
        if (sq[k] != 0.0f) c += sq[k] * ((m - sz[k]) / a.temperature + logs);
      c = warp_sum(c);
      if (lane == 0) {
        a.loss_rows[t] = live ? a.temperature * a.temperature * (s_qlogq + c) : (status == ROW_BAD ? NAN : 0.0f);
        if (a.unscale != nullptr && t == 0) *a.unscale = !a.mean || a.st->count > 0 ? 1.0f / store_scale(a) : 1.0f;
        if (a.loss != nullptr) {
          __threadfence();
          s_last = atomicAdd(&a.st->done, 1u) == static_cast<unsigned int>(a.T) - 1;
        }
      }
    }
  } else if (GRAD) {
    T* out = static_cast<T*>(a.dz) + t * a.dz_ld;
    T* out0 = out + s0 - g.mis;
    uint4* dst = reinterpret_cast<uint4*>(out0);
    const bool vec = reinterpret_cast<uintptr_t>(out0) % 16 == 0;
    float w = 0.0f;
    if (live) {
      w = a.temperature * store_scale(a);
      if (a.mean) w /= static_cast<float>(a.st->count);
      if (a.row_grad != nullptr) w *= a.row_grad[t];
    }
    const float ws = w / s;
    const auto grad = [&](const uint4& raw) {
      const uint64_t off2 = pack2(-m, -m), sc2 = pack2(scale2, scale2), w2 = pack2(ws, ws);
      float x[VEC];
      unpack16<DT>(raw, x);
#pragma unroll
      for (int i = 0; i < VEC; i += 2) {
        const float2 e = unpack2(mul2(add2(pack2(x[i], x[i + 1]), off2), sc2));
        const float2 p = unpack2(mul2(pack2(ex2(e.x), ex2(e.y)), w2));
        x[i] = p.x;
        x[i + 1] = p.y;
      }
      return pack16<DT>(x);
    };
    const uint4 none = make_uint4(0, 0, 0, 0);
    // The second read of the segment comes from L2: the rows that are being
    // worked on fit there.
    if (!vec) {
      for (int j = g.j0 + threadIdx.x; j < g.j1; j += nthreads) g.put(out0, j, live ? grad(src[j]) : none);
    } else if (!live) {
      for (int j = g.j0 + threadIdx.x; j < g.j1; j += nthreads) __stcs(dst + j, none);
    } else {
      for (int j = g.j0 + threadIdx.x; j < g.j1; j += 4 * nthreads) {
        uint4 raw[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (j + u * nthreads < g.j1) raw[u] = __ldcs(src + j + u * nthreads);
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (j + u * nthreads < g.j1) __stcs(dst + j + u * nthreads, grad(raw[u]));
      }
    }
    if (g.edge >= 0) g.put(out0, g.edge, live ? grad(g.load_edge()) : none);
    // The entries' places again, with q taken off before the one rounding.
    asm volatile("bar.sync 1, %0;" ::"r"(nthreads) : "memory");
    if (live) {
      for (int k = threadIdx.x; k < a.top; k += nthreads) {
        const int c = si[k];
        if (c < s0 || c >= s1) continue;
        float goal = 0.0f;
        bool first = true;
        for (int j = 0; j < a.top; ++j) {
          if (si[j] != c) continue;
          first = first && j >= k;
          goal += sq[j];
        }
        if (first) from_f32(ws * ex2((sz[k] - m) * scale2) - w * goal, out[c]);
      }
    }
  }

  // The last row to finish sums the losses of all rows in a fixed order.
  if (a.loss == nullptr || rank != 0) return;
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  double sum = 0.0;
  for (long long r = threadIdx.x; r < a.T; r += blockDim.x) sum += static_cast<double>(__ldcg(a.loss_rows + r));
  sum = block_sum(sum, dbuf);
  if (threadIdx.x == 0) {
    if (a.mean) sum /= static_cast<double>(a.st->count > 0 ? a.st->count : 1);
    *a.loss = static_cast<float>(sum);
  }
}

template <int DT, bool GRAD>
int launch_distill(const DistillArgs& a, int cs, int threads, cudaStream_t s) {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[2];
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // see launch_next
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cs;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(a.T * cs), 1, 1);
  cfg.blockDim = dim3(threads + 32, 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(a.top) * 12;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = a.mean ? 2 : 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, distill_kernel<DT, GRAD>, a), "distill launch");
}

template <int DT>
__device__ __forceinline__ void scale_range(void* x, long long n, float f, long long first, long long step) {
  using T = typename ElemOf<DT>::T;
  constexpr int N = DT == PO_F32 ? 4 : 8;
  T* p = static_cast<T*>(x);
  const long long nv = reinterpret_cast<uintptr_t>(x) % 16 == 0 ? n / N : 0;
  for (long long i = first; i < nv; i += step) {
    float v[N];
    unpack16<DT>(reinterpret_cast<const uint4*>(x)[i], v);
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] *= f;
    reinterpret_cast<uint4*>(x)[i] = pack16<DT>(v);
  }
  for (long long i = nv * N + first; i < n; i += step) from_f32(to_f32(p[i]) * f, p[i]);
}

template <int DT>
__global__ void __launch_bounds__(256) scale_kernel(void* x, long long n, void* y, long long ny, const float* factor) {
  const float f = *factor;
  if (f == 1.0f) return;
  const long long first = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  const long long step = static_cast<long long>(gridDim.x) * blockDim.x;
  scale_range<DT>(x, n, f, first, step);
  scale_range<DT>(y, ny, f, first, step);
}

}  // namespace
}  // namespace po

using namespace po;

extern "C" size_t po_distill_logits_workspace_bytes(long long tokens) { return tokens > 0 ? sizeof(DistillState) : 0; }

extern "C" int po_distill_logits(const void* logits, long long ld, int dtype, long long tokens, long long vocab,
                                 const long long* index, long long index_ld, const void* teacher, long long teacher_ld,
                                 int teacher_dtype, long long top, float temperature, int mean, const float* row_grad,
                                 float* loss_rows, float* loss, void* dlogits, long long dl_ld, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  if (dtype != PO_F32 && dtype != PO_BF16 && dtype != PO_F16)
    return set_error(PO_ERR_ARG, "distill_logits: dtype must be fp32, bf16 or fp16");
  if (teacher_dtype != PO_F32 && teacher_dtype != PO_BF16 && teacher_dtype != PO_F16)
    return set_error(PO_ERR_ARG, "distill_logits: teacher dtype must be fp32, bf16 or fp16");
  if (tokens < 0 || tokens > (1 << 26) || vocab <= 0 || vocab > (1 << 28))
    return set_error(PO_ERR_ARG, "distill_logits: bad size");
  if (top < 1 || top > kMaxTop) return set_error(PO_ERR_ARG, "distill_logits: top must be 1 to 1024");
  if (!temperature_ok(temperature))
    return set_error(PO_ERR_ARG, "distill_logits: temperature must be 2^-60 to 2^60");
  if (row_grad != nullptr && (mean || dlogits == nullptr))
    return set_error(PO_ERR_ARG, "distill_logits: row_grad goes with gradients of the sum");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (tokens == 0) return loss == nullptr ? PO_OK : check_cuda(cudaMemsetAsync(loss, 0, 4, s), "distill_logits");
  if (tokens > 1 && (ld < vocab || index_ld < top || teacher_ld < top || (dlogits != nullptr && dl_ld < vocab)))
    return set_error(PO_ERR_ARG, "distill_logits: a pitch is smaller than its row");
  if (logits == nullptr || index == nullptr || teacher == nullptr || loss_rows == nullptr)
    return set_error(PO_ERR_ARG, "distill_logits: null operand");
  DistillArgs a{};
  a.z = logits, a.ld = ld, a.dz = dlogits, a.dz_ld = dl_ld, a.T = tokens, a.V = static_cast<int>(vocab);
  a.index = index, a.index_ld = index_ld, a.teacher = teacher, a.teacher_ld = teacher_ld;
  const bool scaled = mean == PO_MEAN_SCALED || mean == PO_SUM_SCALED;
  if (mean == PO_SUM_SCALED) mean = 0;
  a.teacher_dtype = teacher_dtype, a.top = static_cast<int>(top), a.temperature = temperature, a.mean = mean;
  a.row_grad = row_grad, a.loss_rows = loss_rows, a.loss = loss;
  if (scaled && dlogits != nullptr) a.unscale = loss_rows + tokens, a.by_powers = dtype == PO_F16;
  if (loss != nullptr || mean) {
    if (workspace == nullptr || workspace_bytes < sizeof(DistillState))
      return set_error(PO_ERR_WORKSPACE, "distill_logits: workspace too small");
    a.st = static_cast<DistillState*>(workspace);
    if (int r = check_cuda(cudaMemsetAsync(a.st, 0, sizeof(DistillState), s), "distill_logits")) return r;
  }
  if (mean) {
    const int blocks = cdiv(tokens, 8) < 2 * sm_count() ? cdiv(tokens, 8) : 2 * sm_count();
    count_rows_kernel<<<blocks, 256, 0, s>>>(a);
    if (int r = check_cuda(cudaGetLastError(), "distill_logits count")) return r;
  }
  // CTAs a row: one, unless there are too few rows to fill the SMs.
  const int es = dtype_size(dtype);
  int cs = 1;
  while (cs < 8 && tokens * cs < 2 * sm_count() && vocab > cs * 2048LL) cs *= 2;
  const int vec = 16 / es;
  a.seg = static_cast<int>(round_up((vocab + cs - 1) / cs, vec));
  // About sixteen vectors a thread.
  const long long nvec = (a.seg + vec - 1) / vec + 1;
  int threads = static_cast<int>(round_up((nvec + 15) / 16, 32));
  const bool g = dlogits != nullptr;
  const int most = g ? kGradThreads : kEvalThreads;
  threads = threads < 64 ? 64 : (threads > most ? most : threads);
  if (dtype == PO_F32) return g ? launch_distill<PO_F32, true>(a, cs, threads, s) : launch_distill<PO_F32, false>(a, cs, threads, s);
  if (dtype == PO_BF16)
    return g ? launch_distill<PO_BF16, true>(a, cs, threads, s) : launch_distill<PO_BF16, false>(a, cs, threads, s);
  return g ? launch_distill<PO_F16, true>(a, cs, threads, s) : launch_distill<PO_F16, false>(a, cs, threads, s);
}

extern "C" int po_scale_inplace(void* x, long long n, void* y, long long ny, int dtype, const float* factor,
                                void* stream) {
  if (dtype != PO_F32 && dtype != PO_BF16 && dtype != PO_F16)
    return set_error(PO_ERR_ARG, "scale_inplace: dtype must be fp32, bf16 or fp16");
  if (y == nullptr) ny = 0;
  if (n < 0 || ny < 0) return set_error(PO_ERR_ARG, "scale_inplace: negative size");
  if (n + ny == 0) return PO_OK;
  if ((n > 0 && x == nullptr) || factor == nullptr) return set_error(PO_ERR_ARG, "scale_inplace: null operand");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const long long want = (n + ny + 2047) / 2048;
  const int blocks = static_cast<int>(want < 8LL * sm_count() ? want : 8LL * sm_count());
  const auto kern = dtype == PO_F32 ? scale_kernel<PO_F32> : dtype == PO_BF16 ? scale_kernel<PO_BF16> : scale_kernel<PO_F16>;
  kern<<<blocks, 256, 0, s>>>(x, n, y, ny, factor);
  return check_cuda(cudaGetLastError(), "scale_inplace");
}
