// The three products of a linear loss head on two-SM tcgen05 tiles: logits
// H W^T with their softmax statistics taken in the epilogue, dH = dZ W and
// dW = dZ^T H.
//
// Mainloop as in gemm_pair.cuh (cluster of two CTAs, 256 x 256 tile, 64 KB
// stages, dynamic tile queue), with four differences:
//  * The extent that counts rows of H is read on the device (rows that count
//    for nothing are packed away before, and their number never reaches the
//    host), so tiles beyond it are not computed.
//  * K may be split over tiles (few rows of H, a long vocabulary): each split
//    stores its fp32 partial tile, a later kernel joins them in order.
//  * fp32 operands are read once for their three products (HeadCfg).
//  * The accumulator is drained into registers every `chunk` K blocks and
//    summed there (fp32, round to nearest): the tensor core's own accumulator
//    truncates, by -1.1e-5 of the sum at K = 4096, which the loss (a difference
//    of two nearby logits) would show. A drain is 64 columns loaded and added
//    by each thread, hidden behind the other accumulator's MMAs.
//
// Epilogue of the logits: each thread holds 64 columns of one row, so the
// row's maximum and sum of exponentials over the tile's 256 columns take two
// exchanges between four threads. It leaves (max, sum) per row and tile, the logits at the row's target indices, and, when
// gradients are wanted, exp(z - max) in 16 bits (fp16: the values are in
// (0, 1], so its 11 bits cost less than the one rounding to the products' type
// that follows; 32 bits for fp32 operands). Storing that costs 2 bytes a logit
// once against 2 D operations a logit for computing it again.
#pragma once

#include "common.cuh"
#include "gemm_pair.cuh"
#include "head_finish.cuh"
#include "losses.cuh"

namespace po {

// A stage of the ring (64 KB a CTA, three of them): 16-bit operands, two
// 128-byte atoms of K of A and of B; fp32 operands, one atom of each one's high
// and low halves, from which the three products hi*hi, hi*lo and lo*hi are
// issued: operands are read from L2 once, where a pass over K for each product
// would read the high halves twice (L2 at about 10 TB/s is what bounds these
// tiles: 500 x 50257 x 768 175 us a product in three passes).
template <int KIND>
struct HeadCfg {
  static constexpr int TM = 256;  // rows of a pair's tile
  static constexpr int BN = 256;  // columns
  static constexpr int ES = KIND == KIND_BF16 ? 2 : 4;
  static constexpr int HALVES = KIND == KIND_BF16 ? 1 : 2;
  static constexpr int ATOMS = KIND == KIND_BF16 ? 2 : 1;
  static constexpr int AK = 128 / ES;       // K elements an atom
  static constexpr int BK = ATOMS * AK;     // a stage
  static constexpr int PART = 128 * 128 * ATOMS;  // bytes: 128 rows of one half of one operand
  static constexpr int A_BYTES = HALVES * PART;
  static constexpr int STAGE_BYTES = 2 * A_BYTES;
  static constexpr int STAGES = 3;
  static constexpr int MMA_K = KIND == KIND_BF16 ? 16 : 8;
  static constexpr int KSTEPS = BK / MMA_K;
  static constexpr uint32_t TMEM_COLS = 2 * BN;
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 1024 + 512;
};

enum HeadEpi : int { HEAD_STATS = 0, HEAD_STORE = 1 };
enum HeadLimit : int { LIMIT_M = 0, LIMIT_K = 1 };  // which extent `count` bounds

struct alignas(64) HeadParams {
  CUtensorMap mapA[2];  // [0] = plain / hi, [1] = lo (fp32 operands)
  CUtensorMap mapB[2];
  int M, N, K;
  int limit;         // HeadLimit
  const int* count;  // device: counted rows of the whole call
  int row0;          // first packed row of this launch
  int tiles_n, splits, band;
  const int* splits_at;  // nullable: the number of splits stands there
  int chunk;         // K blocks summed inside the accumulator
  uint32_t fmt;      // operand format of the instruction descriptor
  unsigned int* sched;
  int* err;
  // HEAD_STATS
  float scale2;       // log2(e) / temperature
  float2* part;       // [row][nparts] (max, sum of 2^(scale2 (z - max))) over 256 columns, z the logits
  int nparts;
  float* zsum;        // [row][nparts] sum of the logits (nullable)
  void* e;            // [row][e_ld] 2^(scale2 (z - max)) (nullable)
  long long e_ld;
  const int* rowmap;  // packed row -> row of the call
  const int* ent;     // [row of the call][top] ascending target indices
  int top;
  float* zpick;       // [row of the call][top] logits at those indices
  // HEAD_STORE
  const float* alpha;  // device scalar
  const float* cin;    // fp32, added to row r (nullable)
  long long cin_ld;
  const float* cin_scale;  // device scalar that cin is multiplied by (nullable)
  void* out;           // row r of the product goes to out row (rows ? rows[row0 + r] : r)
  long long out_ld;
  int out_dtype;       // PO_F32 / PO_BF16 / PO_F16
  int vec;             // 32-byte vector access legal
  const int* out_rows;
  float* partial;      // splits > 1: [split][rows][part_ld] fp32, instead of out
  long long part_ld;
};

// Arrival on a barrier of either CTA of the pair that orders what the barrier
// guards (a tile index read from shared memory, TMEM reads behind their tcgen05
// fence) but not this thread's global stores: at cluster scope a release would
// wait for the tile's stores to reach L2 (a third of the epilogue's stalls).
__device__ __forceinline__ void mbar_arrive_pair(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ void head_sched_release(uint64_t* sempty, int j) {
  mbar_arrive_pair(mapa_shared(smem_u32(sempty + j % kSchedSlots), 0));
}

__device__ __forceinline__ void st_global_32B(void* p, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

__device__ __forceinline__ uint32_t pack_f16x2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_bf16x2(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Sixteen epilogue warps a CTA, four to each TMEM lane quarter: four warps a
// scheduler hide the latencies of TMEM loads, ex2 and stores where two (with
// 128 columns a thread) did not.
constexpr int kHeadEpiWarps = 16;
constexpr int HC = 64;  // columns of a tile one epilogue thread holds
// The bounded waits of ptx.cuh read the clock on the first miss; most waits
// here end within a try_wait or two (which suspend the thread by themselves).
__device__ __forceinline__ bool head_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err, int code) {
#pragma unroll 1
  for (int i = 0; i < 4; ++i)
    if (mbar_try_wait(bar, parity)) return true;
  return mbar_wait_bounded(bar, parity, abort_flag, err, code);
}
__device__ __forceinline__ bool head_wait_sleep(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err,
                                                int code) {
#pragma unroll 1
  for (int i = 0; i < 4; ++i)
    if (mbar_try_wait(bar, parity)) return true;
  return mbar_wait_bounded_sleep(bar, parity, abort_flag, err, code);
}

constexpr int kShareFloats = 3 * 128 + 4;  // a lane quarter's maxima, sums, logit sums and flags
constexpr int kStageWords = 256;              // a warp's eight rows on their way to unaligned ones
constexpr int kHeadSmemExtra = kHeadEpiWarps * kStageWords * 4;  // (products that store exchange no statistics)
static_assert(4 * kShareFloats * 4 <= kHeadSmemExtra, "shared memory");
constexpr int kHeadThreads = 64 + 32 * kHeadEpiWarps;
// Readers of a slot of the tile queue: leader MMA issuer and epilogue warps, peer producer and epilogue warps.
constexpr int kHeadReaders = 2 + 2 * kHeadEpiWarps;

struct HeadTile {
  int mt, nt, split, kb0, kb1;
};

// Extents of this launch after the device-side count.
struct HeadExtent {
  int m, tiles_m, nkb, splits, total;
};

template <class C>
__device__ __forceinline__ HeadExtent head_extent(const HeadParams& P) {
  HeadExtent x;
  const int left = max(0, *P.count - P.row0);
  x.m = P.limit == LIMIT_M ? min(P.M, left) : P.M;
  const int k = P.limit == LIMIT_K ? min(P.K, left) : P.K;
  x.tiles_m = (x.m + C::TM - 1) / C::TM;
  x.nkb = (k + C::BK - 1) / C::BK;
  x.splits = P.splits_at != nullptr ? *P.splits_at : P.splits;
  x.total = x.tiles_m * P.tiles_n * x.splits;
  return x;
}

// Splits outermost; in a split, bands of `band` row tiles, walked row tiles
// first, so that tiles in flight share both operands' panels in L2.
__device__ __forceinline__ HeadTile head_tile(const HeadParams& P, const HeadExtent& x, int t) {
  HeadTile h;
  const int per = x.tiles_m * P.tiles_n;
  h.split = x.splits > 1 ? t / per : 0;
  const int r = t - h.split * per;
  const int b = x.tiles_m <= P.band ? 0 : r / (P.band * P.tiles_n);
  const int first = b * P.band;
  const int rows = min(x.tiles_m - first, P.band);
  const int in_band = r - b * P.band * P.tiles_n;
  h.mt = first + in_band % rows;
  h.nt = in_band / rows;
  h.kb0 = 0;
  h.kb1 = x.nkb;
  if (x.splits > 1) {
    h.kb0 = static_cast<int>(static_cast<long long>(x.nkb) * h.split / x.splits);
    h.kb1 = static_cast<int>(static_cast<long long>(x.nkb) * (h.split + 1) / x.splits);
  }
  return h;
}

__device__ __forceinline__ void bar_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// v: 128 bytes of this thread's row, as four blocks of 32 bytes. Four lanes
// exchange blocks (two butterfly rounds): afterwards block i is block lane % 4
// of row 4 (lane / 4) + i of the warp.
__device__ __forceinline__ void quad_exchange(uint32_t (&v)[32], int lane) {
#pragma unroll
  for (int round = 0; round < 2; ++round) {
    const int x = 1 << round;
    const bool hi = (lane & x) != 0;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int a = round == 0 ? 2 * p : p, b = a + x;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t got = __shfl_xor_sync(0xffffffffu, hi ? v[8 * a + i] : v[8 * b + i], x);
        if (hi) v[8 * a + i] = got;
        else v[8 * b + i] = got;
      }
    }
  }
}

// Stores 128 bytes of each of the warp's 32 rows, whole 128-byte lines of eight
// rows an instruction instead of 32-byte pieces of 32 rows. row_ptr(r): where
// row r of the warp goes (on a 32-byte boundary), null where it does not.
template <class RowPtr>
__device__ __forceinline__ void store_lines(uint32_t (&v)[32], int lane, RowPtr row_ptr) {
  quad_exchange(v, lane);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t w[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) w[k] = v[8 * i + k];
    char* at = row_ptr((lane & ~3) + i);
    if (at != nullptr) st_global_32B(at + (lane & 3) * 32, w);
  }
}

// The same for rows on any boundary of ES bytes, of which `n` elements exist:
// eight rows at a time through 1 KB of the warp's shared memory, then a row an
// instruction, by words where they are aligned. (Element stores straight from
// the registers touch a sector each: dW of 1024 x 50257 x 1001 took 460 us, and
// takes 119 this way; 90 with 1024 features.)
template <int ES, class RowPtr>
__device__ __forceinline__ void store_any(uint32_t (&v)[32], int lane, uint32_t* stage, int n, bool words,
                                          RowPtr row_ptr) {
  quad_exchange(v, lane);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    __syncwarp();
    uint4* to = reinterpret_cast<uint4*>(stage + (lane >> 2) * 32 + (lane & 3) * 8);
    to[0] = make_uint4(v[8 * i], v[8 * i + 1], v[8 * i + 2], v[8 * i + 3]);
    to[1] = make_uint4(v[8 * i + 4], v[8 * i + 5], v[8 * i + 6], v[8 * i + 7]);
    __syncwarp();
#pragma unroll 1
    for (int r = 0; r < 8; ++r) {
      char* at = row_ptr(4 * r + i);
      if (at == nullptr) continue;
      const uint32_t* from = stage + r * 32;
      if (ES == 4) {
        if (lane < n) reinterpret_cast<uint32_t*>(at)[lane] = from[lane];
      } else if (words && 2 * lane + 1 < n) {
        reinterpret_cast<uint32_t*>(at)[lane] = from[lane];
      } else if (words) {
        if (2 * lane < n) reinterpret_cast<uint16_t*>(at)[2 * lane] = static_cast<uint16_t>(from[lane]);
      } else {
        const uint16_t* h = reinterpret_cast<const uint16_t*>(from);
        if (lane < n) reinterpret_cast<uint16_t*>(at)[lane] = h[lane];
        if (lane + 32 < n) reinterpret_cast<uint16_t*>(at)[lane + 32] = h[lane + 32];
      }
    }
  }
}

// Whether all four warps of a lane quarter may go on: a wait that gave up in one
// of them must not leave the others at a barrier. (The flags are read before
// the next barrier and written after the one that follows it.)
__device__ __forceinline__ bool quarter_agrees(int* flags, int group, int q, int lane, bool go) {
  if (lane == 0) flags[group] = go ? 1 : 0;
  bar_sync(1 + q, 128);
  const volatile int* f = flags;
  return (f[0] & f[1] & f[2] & f[3]) != 0;
}

// ------------------------------------------------------------- epilogues
// x: accumulators of columns n0 .. n0 + HC - 1 of packed row `row` (of this launch).
// `share`: this lane quarter's rows of shared memory, [column group][row].
template <bool F32E>
__device__ __forceinline__ void stats_epilogue(const HeadParams& P, float (&x)[HC], bool live, int row, int n0,
                                               int nt, long long tk, int lo, int c, float* share, int group, int q,
                                               int lane, int m_rows) {
  const int ncols = P.N - n0;
  // Logits at the targets: c is the next target's column in this tile. One
  // vote per 16 columns; a row has few targets, so most groups have none.
#pragma unroll
  for (int g = 0; g < HC / 16; ++g) {
    while (__any_sync(0xffffffffu, c < 16 * g + 16)) {
      if (c < 16 * g + 16) {
        float v = 0.0f;
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (c == 16 * g + j) v = x[16 * g + j];
        P.zpick[tk + lo] = v;
        ++lo;
        c = lo < P.top ? P.ent[tk + lo] - n0 : 0x7fffffff;
      }
    }
  }
  const long long at = static_cast<long long>(row) * P.nparts + nt;
  float zs = 0.0f;
  if (P.zsum != nullptr) {
    // Columns past the vocabulary come from zero-filled rows of W: they add 0.
    float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
    for (int j = 0; j < HC; j += 2) {
      s0 += x[j];
      s1 += x[j + 1];
    }
    zs = s0 + s1;
  }
  if (ncols < HC) {
#pragma unroll
    for (int j = 0; j < HC; ++j)
      if (j >= ncols) x[j] = -INFINITY;
  }
  float m0 = x[0], m1 = x[1], m2 = x[2], m3 = x[3];
#pragma unroll
  for (int j = 4; j < HC; j += 4) {
    m0 = fmaxf(m0, x[j]);
    m1 = fmaxf(m1, x[j + 1]);
    m2 = fmaxf(m2, x[j + 2]);
    m3 = fmaxf(m3, x[j + 3]);
  }
  // The four warps of this lane quarter share the row's maximum over the tile.
  share[group * 32 + lane] = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3));
  bar_sync(1 + q, 128);
  const float m = fmaxf(fmaxf(share[lane], share[32 + lane]), fmaxf(share[64 + lane], share[96 + lane]));
  // The maximum is subtracted before the scaling: exact where it matters, and
  // neither logits near the type's limit nor low temperatures overflow.
  const float off = m == -INFINITY ? 0.0f : -m;
  uint64_t sum2[2] = {0, 0};
  const uint64_t scale2 = pack2(P.scale2, P.scale2), off2 = pack2(off, off);
#pragma unroll
  for (int j = 0; j < HC; j += 2) {
    const float2 a = unpack2(mul2(add2(pack2(x[j], x[j + 1]), off2), scale2));
    x[j] = ex2(a.x);
    x[j + 1] = ex2(a.y);
    sum2[(j / 2) & 1] = add2(sum2[(j / 2) & 1], pack2(x[j], x[j + 1]));
  }
  const float2 sums = unpack2(add2(sum2[0], sum2[1]));
  share[128 + group * 32 + lane] = sums.x + sums.y;
  share[256 + group * 32 + lane] = zs;
  bar_sync(1 + q, 128);
  if (group == 0 && live) {
    const float* g = share + 128 + lane;
    P.part[at] = make_float2(m, (g[0] + g[32]) + (g[64] + g[96]));
    if (P.zsum != nullptr) P.zsum[at] = (g[128] + g[160]) + (g[192] + g[224]);
  }
  if (P.e == nullptr || ncols <= 0) return;
  // e_ld is a multiple of 256: whole lines, on 128-byte boundaries.
  const int row_w = row - lane;
  constexpr int ES = F32E ? 4 : 2;
  char* base = static_cast<char*>(P.e) + (static_cast<long long>(row_w) * P.e_ld + n0) * ES;
#pragma unroll
  for (int part = 0; part < ES / 2; ++part) {
    uint32_t v[32];
#pragma unroll
    for (int i = 0; i < 32; ++i)
      v[i] = F32E ? __float_as_uint(x[32 * part + i]) : pack_f16x2(x[2 * i], x[2 * i + 1]);
    store_lines(v, lane, [&](int r) { return row_w + r < m_rows ? base + r * P.e_ld * ES + part * 128 : nullptr; });
  }
}

__device__ __forceinline__ void store_epilogue(const HeadParams& P, float (&x)[HC], int row, int n0, int split,
                                               int splits, int lane, int m_rows, uint32_t* stage) {
  const int ncols = min(HC, P.N - n0);
  const int row_w = row - lane;
  if (splits > 1) {
    // part_ld is a multiple of 256: whole lines, on 128-byte boundaries.
    char* base =
        reinterpret_cast<char*>(P.partial + (static_cast<long long>(split) * m_rows + row_w) * P.part_ld + n0);
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      uint32_t v[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(x[32 * part + i]);
      store_lines(v, lane, [&](int r) { return row_w + r < m_rows ? base + r * P.part_ld * 4 + part * 128 : nullptr; });
    }
    return;
  }
  const bool live = row < m_rows;
  const float alpha = *P.alpha;
  const uint64_t alpha2 = pack2(alpha, alpha);
#pragma unroll
  for (int j = 0; j < HC; j += 2) {
    const float2 f = unpack2(mul2(pack2(x[j], x[j + 1]), alpha2));
    x[j] = f.x;
    x[j + 1] = f.y;
  }
  if (P.cin != nullptr && live) {
    const float* ci = P.cin + static_cast<long long>(row) * P.cin_ld + n0;
    const float cs = P.cin_scale != nullptr ? *P.cin_scale : 1.0f;
    if (P.vec && ncols == HC) {
#pragma unroll
      for (int j = 0; j < HC; j += 4) {
        const float4 f = *reinterpret_cast<const float4*>(ci + j);
        x[j] = fmaf(f.x, cs, x[j]);
        x[j + 1] = fmaf(f.y, cs, x[j + 1]);
        x[j + 2] = fmaf(f.z, cs, x[j + 2]);
        x[j + 3] = fmaf(f.w, cs, x[j + 3]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < HC; ++j)
        if (j < ncols) x[j] = fmaf(ci[j], cs, x[j]);
    }
  }
  const bool bf = P.out_dtype == PO_BF16;
  const int es = P.out_dtype == PO_F32 ? 4 : 2;
  char* base = static_cast<char*>(P.out) + static_cast<long long>(n0) * es;
  const auto row_ptr = [&](int r) -> char* {
    if (row_w + r >= m_rows) return nullptr;
    const long long o = P.out_rows != nullptr ? P.out_rows[P.row0 + row_w + r] : row_w + r;
    return base + o * P.out_ld * es;
  };
  const bool lines = P.vec && ncols == HC;
  uint32_t v[32];
  if (P.out_dtype == PO_F32) {
#pragma unroll
    for (int part = 0; part < 2; ++part) {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(x[32 * part + i]);
      if (lines) store_lines(v, lane, row_ptr);
      else store_any<4>(v, lane, stage, ncols - 32 * part, true, row_ptr);
      base += 128;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = bf ? pack_bf16x2(x[2 * i], x[2 * i + 1]) : pack_f16x2(x[2 * i], x[2 * i + 1]);
    if (lines) store_lines(v, lane, row_ptr);
    else store_any<2>(v, lane, stage, ncols, (reinterpret_cast<uintptr_t>(P.out) | static_cast<uintptr_t>(2 * P.out_ld)) % 4 == 0, row_ptr);
  }
}

// ---------------------------------------------------------------- kernel
template <int KIND, bool A_MN, bool B_MN, int EPI>
__global__ void __launch_bounds__(kHeadThreads, 1) head_gemm_kernel(const __grid_constant__ HeadParams P) {
  using C = HeadCfg<KIND>;
  constexpr int BN = C::BN;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* tiles = smem;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::STAGES * C::STAGE_BYTES);
  uint64_t* empty = full + C::STAGES;
  uint64_t* tfull = empty + C::STAGES;
  uint64_t* tempty = tfull + 2;
  uint64_t* drain = tempty + 2;
  uint64_t* sfull = drain + 1;
  uint64_t* sempty = sfull + kSchedSlots;
  int* stile = reinterpret_cast<int*>(sempty + kSchedSlots);
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(stile + kSchedSlots);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  float* shares = reinterpret_cast<float*>(smem + C::STAGES * C::STAGE_BYTES + 512);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull + a, 1);
      mbar_init(tempty + a, 2 * kHeadEpiWarps);
    }
    mbar_init(drain, 1);
    for (int i = 0; i < kSchedSlots; ++i) {
      mbar_init(sfull + i, 1);
      mbar_init(sempty + i, kHeadReaders);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tensormap(&P.mapA[0]);
    prefetch_tensormap(&P.mapB[0]);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_holder, C::TMEM_COLS);
    tmem_relinquish_pair();
  }
  tc_fence_before_sync();
  cluster_sync();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_holder;
  grid_launch_next();
  grid_wait();  // operands and the count come from the kernel before
  const HeadExtent X = head_extent<C>(P);

  if (warp == 0) {
    if (lane == 0) {
      // ------------------------------------------------ TMA producer (both CTAs)
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      uint32_t armed = 0;
      for (int j = 0; ok; ++j) {
        int t;
        if (leader) {
          const int slot = j % kSchedSlots;
          if (!mbar_wait_bounded_cluster(sempty + slot, ((j / kSchedSlots) & 1u) ^ 1u, abort_flag, P.err,
                                         kErrTimeoutProducer))
            break;
          t = static_cast<int>(atomicAdd(P.sched, 1u));
          stile[slot] = t;
          st_shared_cluster_u32(mapa_shared(smem_u32(stile + slot), 1), static_cast<uint32_t>(t));
          mbar_arrive(sfull + slot);
          mbar_arrive_cluster(mapa_shared(smem_u32(sfull + slot), 1));
        } else {
          if (!sched_read(sfull, stile, j, abort_flag, P.err, kErrTimeoutProducer, t)) break;
          head_sched_release(sempty, j);
        }
        if (t >= X.total) break;
        const HeadTile h = head_tile(P, X, t);
        const int arow = h.mt * C::TM + static_cast<int>(rank) * 128;
        const int brow = h.nt * BN + static_cast<int>(rank) * (BN / 2);
        for (int v = h.kb0; v < h.kb1; ++v) {
          const int k0 = v * C::BK;
          if (!head_wait(empty + stage, phase ^ 1u, abort_flag, P.err, kErrTimeoutProducer)) {
            ok = false;
            break;
          }
          if (leader) {
            mbar_arrive_expect_tx(full + stage, 2 * C::STAGE_BYTES);
            armed = (armed & ~(0x101u << stage)) | (1u << stage) | (phase << (8 + stage));
          }
          const uint32_t bar = mapa_shared(smem_u32(full + stage), 0);
#pragma unroll
          for (int half = 0; half < C::HALVES; ++half) {
            const CUtensorMap* ma = &P.mapA[half];
            const CUtensorMap* mb = &P.mapB[half];
            uint8_t* sa = tiles + stage * C::STAGE_BYTES + half * C::PART;
            uint8_t* sb = sa + C::A_BYTES;
            if (!A_MN) {
#pragma unroll
              for (int a = 0; a < C::ATOMS; ++a)
                tma_load_3d_pair(sa + a * 128 * 128, ma, bar, k0 + a * C::AK, arow, 0);
            } else {
#pragma unroll
              for (int i = 0; i < C::ES; ++i)
                tma_load_3d_pair(sa + i * C::BK * 128, ma, bar, arow + i * (128 / C::ES), k0, 0);
            }
            if (!B_MN) {
#pragma unroll
              for (int a = 0; a < C::ATOMS; ++a)
                tma_load_3d_pair(sb + a * 128 * 128, mb, bar, k0 + a * C::AK, brow, 0);
            } else {
#pragma unroll
              for (int i = 0; i < C::ES; ++i)
                tma_load_3d_pair(sb + i * C::BK * 128, mb, bar, brow + i * (128 / C::ES), k0, 0);
            }
          }
          if (++stage == C::STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (!ok && leader) {
        // Once the last arming of each stage completes, no load of either CTA is in flight.
        for (int s = 0; s < C::STAGES; ++s) {
          if (!(armed & (1u << s))) continue;
          const uint32_t par = (armed >> (8 + s)) & 1u;
          const unsigned long long t0 = global_timer_ns();
          while (!mbar_try_wait(full + s, par)) {
            if (global_timer_ns() - t0 > kWaitTimeoutNs) {
              atomicCAS(P.err, 0, kErrTimeoutDrain);
              break;
            }
          }
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && leader) {
      // ------------------------------------------------ MMA issuer (leader CTA)
      const uint32_t idesc = make_idesc(0, C::TM, BN, A_MN ? 1u : 0u, B_MN ? 1u : 0u) | (P.fmt << 7) | (P.fmt << 10);
      constexpr uint32_t A_STEP = A_MN ? C::MMA_K * 128 : 32;
      constexpr uint32_t B_STEP = B_MN ? C::MMA_K * 128 : 32;
      constexpr uint32_t A_LBO = A_MN ? C::BK * 128 : 16;
      constexpr uint32_t B_LBO = B_MN ? C::BK * 128 : 16;
      constexpr bool MN32 = (KIND == KIND_TF32);
      constexpr uint32_t A_LAY = (A_MN && MN32) ? kSwizzle128BAtom32B : kSwizzle128B;
      constexpr uint32_t B_LAY = (B_MN && MN32) ? kSwizzle128BAtom32B : kSwizzle128B;
      constexpr uint32_t A_SBO = (A_MN && MN32) ? 512 : 1024;
      constexpr uint32_t B_SBO = (B_MN && MN32) ? 512 : 1024;
      int stage = 0;
      uint32_t phase = 0;
      int ucount = 0;  // accumulators filled
      bool ok = true;
      for (int j = 0; ok; ++j) {
        int t;
        if (!sched_read(sfull, stile, j, abort_flag, P.err, kErrTimeoutMma, t)) break;
        head_sched_release(sempty, j);
        if (t >= X.total) break;
        const HeadTile h = head_tile(P, X, t);
        const int nv = h.kb1 - h.kb0;
        for (int v0 = 0; v0 < nv && ok; v0 += P.chunk, ++ucount) {
          const int acc = ucount & 1;
          if (!mbar_wait_bounded_cluster(tempty + acc, ((ucount >> 1) & 1u) ^ 1u, abort_flag, P.err,
                                         kErrTimeoutMma)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t dtmem = tmem_base + static_cast<uint32_t>(acc * BN);
          const int v1 = min(nv, v0 + P.chunk);
          for (int v = v0; v < v1; ++v) {
            if (!head_wait(full + stage, phase, abort_flag, P.err, kErrTimeoutMma)) {
              ok = false;
              break;
            }
            const uint32_t sa = smem_u32(tiles + stage * C::STAGE_BYTES);
            const uint32_t sb = sa + C::A_BYTES;
            // lo*hi, hi*lo, hi*hi: the small products meet a small sum, which
            // truncates less (a mean fp32 loss off by 3e-7 for 5e-7).
#pragma unroll
            for (int pass = C::HALVES == 2 ? 2 : 0; pass >= 0; --pass) {
#pragma unroll
              for (int ks = 0; ks < C::KSTEPS; ++ks) {
                constexpr int PER = C::KSTEPS / C::ATOMS;
                const uint32_t aoff = (pass == 2 ? C::PART : 0) +
                                      (A_MN ? ks * A_STEP : (ks / PER) * (128 * 128) + (ks % PER) * 32);
                const uint32_t boff = (pass == 1 ? C::PART : 0) +
                                      (B_MN ? ks * B_STEP : (ks / PER) * (128 * 128) + (ks % PER) * 32);
                const uint64_t ad = make_sw128_desc(sa + aoff, A_LBO, A_SBO, A_LAY);
                const uint64_t bd = make_sw128_desc(sb + boff, B_LBO, B_SBO, B_LAY);
                const uint32_t accumulate = (v > v0 || pass < C::HALVES * 2 - 2 || ks > 0) ? 1u : 0u;
                if (KIND == KIND_BF16) mma_f16_pair(dtmem, ad, bd, idesc, accumulate);
                else mma_tf32_pair(dtmem, ad, bd, idesc, accumulate);
              }
            }
            mma_commit_pair_mc(empty + stage, 0x3);
            if (++stage == C::STAGES) {
              stage = 0;
              phase ^= 1u;
            }
          }
          if (ok) mma_commit_pair_mc(tfull + acc, 0x3);
        }
      }
      mma_commit_pair(drain);
      const unsigned long long t0 = global_timer_ns();
      while (!mbar_try_wait(drain, 0)) {
        if (global_timer_ns() - t0 > kWaitTimeoutNs) {
          atomicCAS(P.err, 0, kErrTimeoutDrain);
          break;
        }
      }
    }
  } else {
    // ------------------------------------------------------ epilogue (both CTAs)
    const int q = warp & 3;
    const int group = (warp - 2) >> 2;
    float* share = shares + q * kShareFloats;
    const uint32_t tcol = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(group * HC);
    int ucount = 0;
    for (int j = 0;; ++j) {
      int t = 0;
      bool go = sched_read(sfull, stile, j, abort_flag, P.err, kErrTimeoutEpilogue, t);
      go = __all_sync(0xffffffffu, go);
      __syncwarp();
      if (go && lane == 0) head_sched_release(sempty, j);
      go = go && t < X.total;
      HeadTile h{0, 0, 0, 0, 0};
      if (go) h = head_tile(P, X, t);
      const int nv = h.kb1 - h.kb0;
      const int row = h.mt * C::TM + static_cast<int>(rank) * 128 + q * 32 + lane;
      const int n0 = h.nt * BN + group * HC;
      const bool live = go && row < X.m;
      long long tk = 0;
      int lo = 0, c = 0x7fffffff;
      if (EPI == HEAD_STATS && live) {
        // First target of this row at or after column n0.
        tk = static_cast<long long>(P.rowmap[P.row0 + row]) * P.top;
        int hi = P.top;
        while (lo < hi) {
          const int mid = (lo + hi) >> 1;
          if (P.ent[tk + mid] < n0) lo = mid + 1;
          else hi = mid;
        }
        if (lo < P.top) c = P.ent[tk + lo] - n0;
      }
      uint64_t acc2[HC / 2];  // two columns a register pair
#pragma unroll
      for (int i = 0; i < HC / 2; ++i) acc2[i] = 0;
      for (int v0 = 0; v0 < nv; v0 += P.chunk, ++ucount) {
        const int acc = ucount & 1;
        const bool ready =
            head_wait_sleep(tfull + acc, (ucount >> 1) & 1u, abort_flag, P.err, kErrTimeoutEpilogue);
        if (!__all_sync(0xffffffffu, ready)) {
          go = false;
          break;
        }
        tc_fence_after_sync();
#pragma unroll
        for (int i = 0; i < HC / 16; ++i) {
          uint32_t r[16];
          tmem_ld_32x16(tcol + static_cast<uint32_t>(acc * BN + i * 16), r);
          tmem_ld_wait();
#pragma unroll
          for (int k = 0; k < 8; ++k)
            acc2[8 * i + k] = add2(acc2[8 * i + k], pack2(__uint_as_float(r[2 * k]), __uint_as_float(r[2 * k + 1])));
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_pair(mapa_shared(smem_u32(tempty + acc), 0));
      }
      // The warps that exchange statistics go on or leave together.
      if (EPI == HEAD_STATS) go = quarter_agrees(reinterpret_cast<int*>(share + 3 * 128), group, q, lane, go);
      if (!go) break;
      float x[HC];
#pragma unroll
      for (int i = 0; i < HC / 2; ++i) {
        const float2 f = unpack2(acc2[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
      if (EPI == HEAD_STATS) {
        stats_epilogue<KIND == KIND_TF32>(P, x, live, row, n0, h.nt, tk, lo, c, share, group, q, lane, X.m);
        __syncwarp();
      } else if (n0 < P.N) {
        store_epilogue(P, x, row, n0, h.split, X.splits, lane, X.m,
                       reinterpret_cast<uint32_t*>(shares) + (warp - 2) * kStageWords);
      }
    }
  }

  __syncwarp();
  tc_fence_before_sync();
  cluster_sync();  // every MMA drained and every TMEM read done in both CTAs
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, C::TMEM_COLS);
  }
  if (threadIdx.x == 0) {
    // The last CTA to finish re-arms the queue for the next launch.
    __threadfence();
    if (atomicAdd(P.sched + 1, 1u) == gridDim.x - 1) {
      atomicExch(P.sched, 0u);
      atomicExch(P.sched + 1, 0u);
    }
  }
}

// `max_tiles` is an upper bound of tiles times splits: the kernel reads the real extent.
template <int KIND, bool A_MN, bool B_MN, int EPI>
int launch_head(const HeadParams& P, int max_tiles, cudaStream_t stream) {
  using C = HeadCfg<KIND>;
  auto kern = head_gemm_kernel<KIND, A_MN, B_MN, EPI>;
  static int max_pairs[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return set_error(PO_ERR_CUDA, "device ordinal out of range");
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[2];
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // see launch_next
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.blockDim = dim3(kHeadThreads, 1, 1);
  cfg.dynamicSmemBytes = C::SMEM_BYTES + kHeadSmemExtra;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (max_pairs[dev] == 0) {
    int r = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                            C::SMEM_BYTES + kHeadSmemExtra),
                       "cudaFuncSetAttribute");
    if (r) return r;
    cfg.gridDim = dim3(2 * (sm_count() / 2), 1, 1);
    int n = 0;
    r = check_cuda(cudaOccupancyMaxActiveClusters(&n, kern, &cfg), "cudaOccupancyMaxActiveClusters");
    if (r) return r;
    if (n <= 0) return set_error(PO_ERR_CUDA, "loss head: no cluster of two CTAs fits on this device");
    max_pairs[dev] = n;
  }
  const int pairs = max_tiles < max_pairs[dev] ? max_tiles : max_pairs[dev];
  cfg.numAttrs = 2;
  cfg.gridDim = dim3(2 * pairs, 1, 1);
  return check_cuda(cudaLaunchKernelEx(&cfg, kern, P), "loss head launch");
}

// logits + statistics (both operands K-major); dH = dZ W (W MN-major); dW = dZ^T H (both MN-major).
enum HeadProduct : int { HEAD_LOGITS = 0, HEAD_DHIDDEN = 1, HEAD_DWEIGHT = 2 };
template <int KIND>
int dispatch_head(int product, const HeadParams& P, int max_tiles, cudaStream_t s) {
  if (product == HEAD_LOGITS) return launch_head<KIND, false, false, HEAD_STATS>(P, max_tiles, s);
  if (product == HEAD_DHIDDEN) return launch_head<KIND, false, true, HEAD_STORE>(P, max_tiles, s);
  return launch_head<KIND, true, true, HEAD_STORE>(P, max_tiles, s);
}

// The logits product for up to kFewRows rows (head_few.cu): the same outputs
// from the call's own hidden rows and weights, statistics per kFewPartCols columns.
constexpr int kFewRows = 8;
constexpr int kFewPartCols = 64, kPartCols = 256;
struct FewParams {
  const void* h;  // [row of the call][h_ld]; rows of both on 16-byte boundaries
  long long h_ld;
  const void* w;
  long long w_ld;
  int D, V;
  float scale2;
  float2* part;
  float* zsum;
  void* e;
  long long e_ld;
  float* zpick;
  FinishArgs finish;  // the last block finishes the rows
};
int launch_few_rows(const FewParams& P, int dtype, int rows, cudaStream_t s);

extern template int dispatch_head<KIND_BF16>(int, const HeadParams&, int, cudaStream_t);
extern template int dispatch_head<KIND_TF32>(int, const HeadParams&, int, cudaStream_t);

}  // namespace po
