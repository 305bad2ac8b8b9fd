// class_loss.cu -- softmax cross entropy of a feature map through a linear
// classifier, without the logits ever in memory, and its gradients.
//
//   z[n,v] = <x_n, w_v> + b_v          lse_n = log sum_v exp z[n,v]
//   loss_n = lse_n - z[n,y_n]          P[n,v] = u_n (exp(z[n,v] - lse_n) - [v = y_n])
//   dX = P W        dW = P^T X         db = sum_n P[n,:]
//
// All three passes stream tiles of one operand past a resident tile of the
// other, recompute the tile of z, and use it at once:
//   forward  rows of X resident, W streams: running maximum and sum per row;
//   dX       rows of X resident, W streams: accumulates P W;
//   dW       rows of W resident, X streams: accumulates P^T X (and db).
// Everything is held in base 2: t = z * log2(e), lse2 = log2 sum 2^t.
//
// Operands are packed once per forward into tiles of 128 rows by 16-column
// multiples, split into bf16 planes whose sum is the value: one for bf16, two
// for fp16 (exact), three for fp32 (exact to 2^-24 of the value).  Packing
// takes care of every stride, tail and ignored row, so the passes see whole
// tiles: rows past the end and ignored rows are zero, classes past the end
// have the bias -inf.
//
// What bounds it: an exponential per row and class in each pass (16 a clock
// and SM) while channels are few, the matrix products from about 256 channels
// (16 bits) or 64 (fp32, six products), and below both the issue of the
// instructions around the exponential.  On a B200, forward / dX / dW:
//   2,073,600 x 256 classes x 16 channels fp32    245 / 378 / 312 us
//     640,000 x 1,000 x 32 bf16                   229 / 229 / 209 us
//      16,384 x 32,768 x 256 bf16                 286 / 406 / 430 us
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "gsb_common.cuh"
#include "gsb_tcgen05.cuh"

namespace gsb {
namespace {

constexpr int THREADS = launch::CLASS_LOSS;
constexpr int TILE = 128;
constexpr float LOG2E = 1.4426950408889634f;
constexpr double LN2 = 0.6931471805599453;

// A forward alone takes fp16 features as they are; gradients multiply them with
// P, which needs bf16's range (upstream factors have any size).
inline int planes_of(const gsb_class_loss_args* a) {
  return a->dtype == GSB_TYPE_FP32 ? 3 : a->dtype == GSB_TYPE_FP16 && a->train ? 2 : 1;
}
inline int pad_c(int C) { return (C + 15) & ~15; }
inline long long tiles_of(long long n) { return (n + TILE - 1) / TILE; }
inline size_t align256(size_t b) { return (b + 255) & ~(size_t)255; }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }

template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

// The features' type behind a number of planes.
template <int NP>
struct PlanesType;
template <>
struct PlanesType<1> {
  using type = __nv_bfloat16;
};
template <>
struct PlanesType<2> {
  using type = __half;
};
template <>
struct PlanesType<3> {
  using type = float;
};

// What forward leaves for backward.
struct Kept {
  uint4 *packed_x, *packed_w;
  float *class_bias2, *row_lse2;  // base 2; classes and rows rounded up to whole tiles
  float* row_exact;               // 2^(row_lse2 - the row's log-sum before it was rounded to fp32)
  int* row_y;                     // labels, -1 where a row has no gradient
  float* inv_count;
};

// ---------------------------------------------------------------------------
// Packing.  Layout: [row / 8][plane][column / 8][row % 8][8 columns] of bf16,
// so that any eight or more rows are one contiguous copy, and 8 x 8 core
// matrices are 128 contiguous bytes with uniform strides in both directions.
// ---------------------------------------------------------------------------
template <int PLANES>
__device__ __forceinline__ void store_planes(uint4* tile, int D8, int d8, int row, const float (&x)[8]) {
  float rest[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) rest[i] = x[i];
#pragma unroll
  for (int p = 0; p < PLANES; ++p) {
    __nv_bfloat162 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      h[i] = __floats2bfloat162_rn(rest[2 * i], rest[2 * i + 1]);
      // an infinity's remainder would be NaN; its first plane says it all
      const float2 f = __bfloat1622float2(h[i]);
      rest[2 * i] = isinf(f.x) ? 0.f : rest[2 * i] - f.x;
      rest[2 * i + 1] = isinf(f.y) ? 0.f : rest[2 * i + 1] - f.y;
    }
    tile[((size_t)(row / 8 * PLANES + p) * D8 + d8) * 8 + row % 8] = *reinterpret_cast<uint4*>(h);
  }
}

// One plane: 16-bit elements as they are.
template <typename T>
__device__ __forceinline__ void store_row(uint4* tile, int D8, int d8, int row, const float (&x)[8]) {
  uint4 raw;
  T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = from_float<T>(x[i]);
  tile[((size_t)(row / 8) * D8 + d8) * 8 + row % 8] = raw;
}

// Eight neighbouring elements of a row, from column c on; zero past C.
template <typename T>
__device__ __forceinline__ void load8(const T* at, long long stride, int c, int C, bool wide, float (&x)[8]) {
  if (wide) {  // contiguous, aligned and whole
    if constexpr (sizeof(T) == 4) {
      const float4 lo = *reinterpret_cast<const float4*>(at + c), hi = *reinterpret_cast<const float4*>(at + c + 4);
      x[0] = lo.x, x[1] = lo.y, x[2] = lo.z, x[3] = lo.w, x[4] = hi.x, x[5] = hi.y, x[6] = hi.z, x[7] = hi.w;
    } else {
      const uint4 raw = *reinterpret_cast<const uint4*>(at + c);
      const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = to_float(e[k]);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = c + k < C ? to_float(at[(c + k) * stride]) : 0.f;
  }
}

// A CTA packs one tile: the classifier's tiles first (with the bias in base
// 2), then the rows' (with their labels).  Ignored rows, rows past the end and
// classes that take no part are zero and their elements are not read; finite
// biases stay finite.
template <typename T, int PLANES>
__global__ void __launch_bounds__(THREADS) pack_kernel(const gsb_class_loss_args a, const Kept kept, int D8, int w_tiles,
                                                       int* __restrict__ ticket) {
  const int row = threadIdx.x % TILE;
  const bool classes = (int)blockIdx.x < w_tiles;
  const long long tile = classes ? blockIdx.x : blockIdx.x - w_tiles;
  const long long n = tile * TILE + row;
  bool used;
  const T* at;
  long long stride;
  if (classes) {
    float bias = -INFINITY;
    if (n < a.V) {
      bias = a.bias ? a.bias[n] : 0.f;
      if (isfinite(bias)) bias = fminf(fmaxf(bias, -2e38f), 2e38f) * LOG2E;
    }
    used = bias != -INFINITY;
    at = (const T*)a.weight + n * a.C;
    stride = 1;
    if (threadIdx.x < TILE) kept.class_bias2[n] = bias;
    if (blockIdx.x == 0 && threadIdx.x == 0) *ticket = 0;
  } else {
    int y = -1;
    if (n < a.B * a.S) {
      const long long l = a.labels64 ? ((const long long*)a.labels)[n] : (long long)((const int*)a.labels)[n];
      if (l != a.ignore_index) {
        if (l >= 0 && l < a.V) y = (int)l;
        else atomicOr((unsigned long long*)a.error_word, (unsigned long long)ERR_BAD_LABEL);
      }
    }
    if (threadIdx.x < TILE) kept.row_y[n] = y;
    used = y >= 0;
    const unsigned b = a.B > 1 ? (unsigned)n / (unsigned)max(a.S, 1ll) : 0u;
    at = (const T*)a.features + b * a.stride_b + (n - b * a.S) * a.stride_s;
    stride = a.stride_c;
  }
  const bool contiguous = stride == 1 && (uintptr_t)at % 16 == 0;
  uint4* const out = (classes ? kept.packed_w : kept.packed_x) + (size_t)tile * PLANES * D8 * TILE;
#pragma unroll(PLANES == 1 ? 4 : 1)
  for (int d8 = threadIdx.x / TILE; d8 < D8; d8 += THREADS / TILE) {
    float x[8];
    if (used) {
      load8(at, stride, d8 * 8, a.C, contiguous && d8 * 8 + 8 <= a.C, x);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = 0.f;
    }
    if constexpr (PLANES == 1) {
      store_row<T>(out, D8, d8, row, x);
    } else {
      store_planes<PLANES>(out, D8, d8, row, x);
    }
  }
}

// ---------------------------------------------------------------------------
// The streaming pass: one persistent CTA per SM.  A work unit is a resident
// tile of 128 rows and a range of the streamed operand's tiles of TN rows
// (columns of z).  One warp loads, two issue the matrix instructions, four
// groups of four warps take the tiles of z in turn, and in the gradient
// passes four more warps store finished accumulators while the next unit
// runs.  A thread owns one row of z (a lane of tensor memory):
//   z tile (TMEM) -> registers -> P, rounded to bf16 planes -> TMEM, over z
//   accumulator (TMEM) += P (TMEM) x streamed tile (shared, as K x channels).
// The streamed tile is read twice, K-major for z and MN-major for the second
// product, from one copy: without a swizzle, its 8 x 8 core matrices serve
// both.
// ---------------------------------------------------------------------------
enum { FWD = 0, DX = 1, DW = 2 };

constexpr int MAX_STAGES = 16, MAX_A_SLOTS = 4;
constexpr int TMEM_COLUMNS = 512;
constexpr int GROUPS = 4;                      // consumer groups of four warps, one z buffer each
constexpr int LOADER = GROUPS * 4, ISSUER = LOADER + 1, ISSUER2 = LOADER + 2;  // warps

// Where and how a gradient is written: element (n, c), times the loss's
// upstream gradient (of the row, or over the count of rows).
struct GradOut {
  void* out;
  const float* upstream;
  const float* inv_count;  // null: upstream has one factor per row
  const int* y;            // rows without a gradient are zero (null: every row has one)
  const float* row_exact;  // dX: what P was computed too small by (null: nothing)
  long long rows, S;       // S > 0: n = b * S + s, written as (b, c, s); S = 0: (n, c)
  int C;
};
__device__ __forceinline__ float grad_scale(const GradOut& o, long long n) {
  const int y = o.y ? o.y[n] : 0;  // loads side by side
  const float u = o.inv_count ? o.upstream[0] * o.inv_count[0] : o.upstream ? o.upstream[n] : 1.f;
  const float e = o.row_exact ? o.row_exact[n] : 1.f;
  return y < 0 ? 0.f : u * e;
}
// Columns c .. c + COUNT - 1 of row n; u from grad_scale.
template <typename T, int COUNT>
__device__ __forceinline__ void write_grad(const GradOut& o, long long n, int c, float (&v)[COUNT], float u) {
#pragma unroll
  for (int i = 0; i < COUNT; ++i) v[i] = u == 0.f ? 0.f : v[i] * u;
  if (o.S > 0) {
    const unsigned b = (unsigned)n / (unsigned)o.S;
    T* at = (T*)o.out + ((long long)b * o.C + c) * o.S + (n - b * o.S);
#pragma unroll
    for (int i = 0; i < COUNT; ++i, at += o.S)
      if (c + i < o.C) *at = from_float<T>(v[i]);
  } else {
    T* at = (T*)o.out + n * o.C + c;
    constexpr int PER = 16 / (int)sizeof(T);
    if (COUNT % PER == 0 && c + COUNT <= o.C && (uintptr_t)at % 16 == 0) {
#pragma unroll
      for (int i = 0; i < COUNT / PER; ++i) {
        uint4 raw;
        T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
        for (int k = 0; k < PER; ++k) e[k] = from_float<T>(v[i * PER + k]);
        reinterpret_cast<uint4*>(at)[i] = raw;
      }
    } else {
#pragma unroll
      for (int i = 0; i < COUNT; ++i)
        if (c + i < o.C) at[i] = from_float<T>(v[i]);
    }
  }
}

struct StreamArgs {
  const uint4* a;          // resident operand, packed
  const uint4* b;          // streamed operand, packed
  const float* b2;         // bias of the classes, base 2
  const float* lse2;       // rows (DX, DW)
  const float* row_exact;  // rows (DX)
  const int* y;            // rows
  const float* row_u;      // per-row upstream (DW, reduction none) or NULL
  int a_tiles, b_tiles, splits, D8;
  int a_slots, stages, acc_slots;
  int slots;               // partial results a unit leaves: its groups that had a tile
  int flush;               // tiles per accumulator
  float* part_m;           // FWD: [split][slot][row]
  float* part_s;
  float* t_label;          // FWD: [row]
  float* part_acc;         // DX, DW: [split][tile][column / 4][row][4 columns]
  float* part_bias;        // DW: [split][slot][row]
  GradOut grad;            // DX, DW with one split: written by the pass itself
  long long* error_word;
};

struct Barriers {
  uint64_t a_full[MAX_A_SLOTS], a_empty[MAX_A_SLOTS], b_full[MAX_STAGES], b_empty[MAX_STAGES];
  uint64_t s_full[GROUPS], s_free[GROUPS], p_full[GROUPS], acc_full[2], acc_empty[2], drained[2];
  uint32_t tmem;
  int stop;
};

// Tensor memory: a buffer of z for each group, over which P is written (two planes fit
// its 32-bit columns, the third has its own), then the accumulators.
template <int MODE>
__host__ __device__ constexpr int z_columns(int np, int tn) {
  return MODE == FWD ? tn : tn * (np == 3 ? 3 : 2) / 2;
}

// The matrix instructions truncate when they add to an accumulator, half an
// ulp of the running sum on average, always towards zero, so a long chain is
// off by its length times 2^-25 (measured: 6.5e-5 of dW after 10,000
// additions).  Accumulators are therefore taken out after a bounded number of
// additions and added up with rounding.  fp32 features: 16 additions of the
// leading planes' product; the other five products, 2^-8 of it and less, have
// columns of their own, so that they do not lengthen the chain (5e-7).
// fp16 (four products): 256 additions, 8e-6; bf16: 512, 1.5e-5 (1,024 and 3e-5
// where P has two planes); all far below the half step of the gradients' type.
__host__ __device__ constexpr int accumulators(int np) { return np == 3 ? 2 : 1; }
__host__ __device__ constexpr int chain_products(int np) { return np == 3 ? 16 : np == 2 ? 64 : 512; }

template <int MODE>
__host__ __device__ constexpr int meta_floats(int tn) { return MODE == DW ? 3 * tn : tn; }
template <int MODE>
__host__ __device__ constexpr int stream_threads() { return (MODE == FWD ? GROUPS * 4 + 2 : GROUPS * 4 + 7) * 32; }

// A position in a ring of buffers and the parity of its current round.
struct Ring {
  int i = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int n) {
    if (++i == n) {
      i = 0;
      phase ^= 1;
    }
  }
};

struct Range {
  int tile, split, lo, hi;
};
__device__ __forceinline__ Range unit_range(const StreamArgs& g, int unit) {
  Range r;
  r.split = unit / g.a_tiles;
  r.tile = unit - r.split * g.a_tiles;
  r.lo = (int)((long long)g.b_tiles * r.split / g.splits);
  r.hi = (int)((long long)g.b_tiles * (r.split + 1) / g.splits);
  return r;
}

// Walks a CTA's units tile by tile, with the rings that go along.
struct Cursor {
  int unit, bt, step;
  Range r;
  Ring as, bs, acc;
  uint32_t t = 0;
  __device__ __forceinline__ Cursor(const StreamArgs& g, int cta, int ctas) : unit(cta), step(ctas) {
    if (unit < g.a_tiles * g.splits) {
      r = unit_range(g, unit);
      bt = r.lo;
    }
  }
  __device__ __forceinline__ void next(const StreamArgs& g) {
    ++t;
    bs.next(g.stages);
    if (++bt < r.hi) return;
    as.next(g.a_slots);
    unit += step;
    if (unit < g.a_tiles * g.splits) {
      r = unit_range(g, unit);
      bt = r.lo;
    }
  }
};

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Packed pairs of fp32 (sm_100a issues both halves at once).
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }

// Products of planes whose sum is the fp32 (fp16) product: from the smallest
// up; what is left out is below 2^-25 of the product.
// One hex digit per product, the first one lowest.
__host__ __device__ constexpr int plane_products(int np) { return np == 3 ? 6 : np == 2 ? 4 : 1; }
__host__ __device__ constexpr int plane_of_a(int np, int q) {
  return (np == 3 ? 0x001102 : np == 2 ? 0x0011 : 0) >> (4 * q) & 15;
}
__host__ __device__ constexpr int plane_of_b(int np, int q) {
  return (np == 3 ? 0x010120 : np == 2 ? 0x0101 : 0) >> (4 * q) & 15;
}

// Splits 16 values into bf16 planes and stores them over z's columns they
// come from: the K = 16 step at column c is 8 words of plane 0 and 8 of plane
// 1 there, and 8 of plane 2 behind the buffer's z.
__device__ __forceinline__ constexpr int p_column(int tn, int c, int plane) {
  return plane < 2 ? c + 8 * plane : tn + c / 2;
}
template <int NP, int TN>
__device__ __forceinline__ void store_p(uint32_t buffer, int c, const float2 (&p)[8]) {
  float2 rest[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) rest[i] = p[i];
#pragma unroll
  for (int k = 0; k < NP; ++k) {
    uint32_t h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const __nv_bfloat162 v = __floats2bfloat162_rn(rest[i].x, rest[i].y);
      h[i] = *reinterpret_cast<const uint32_t*>(&v);
      if (k + 1 < NP) {
        const float2 f = make_float2(__uint_as_float(h[i] << 16), __uint_as_float(h[i] & 0xffff0000u));
        rest[i] = fma2(f, make_float2(-1.f, -1.f), rest[i]);  // exact
      }
    }
    tc::tmem_store(buffer + p_column(TN, c, k), h);
  }
}

// PP: planes of P in the gradients, NP or (for NP = 1) 2.
template <int MODE, int NP, int TN, int PP = NP, bool FP16 = false>
__device__ __forceinline__ void stream_pass(const StreamArgs& g, uint8_t* smem, const int cta, const int ctas) {
  using namespace tc;
  const int D8 = g.D8, D = D8 * 8;
  const uint32_t a_bytes = (uint32_t)NP * D8 * 2048, b_bytes = (uint32_t)NP * D8 * TN * 16;
  constexpr uint32_t META = (uint32_t)meta_floats<MODE>(TN);
  uint8_t* const sA = smem;
  uint8_t* const sB = sA + (size_t)g.a_slots * a_bytes;
  float* const sMeta = reinterpret_cast<float*>(sB + (size_t)g.stages * b_bytes);
  Barriers* const bar = reinterpret_cast<Barriers*>(sMeta + (size_t)g.stages * META);
  volatile int* const stop = &bar->stop;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int units = g.a_tiles * g.splits;
  constexpr int SBUF = z_columns<MODE>(NP, TN);
  constexpr int ACCS = accumulators(NP);
  constexpr uint32_t ACC0 = GROUPS * SBUF;          // first accumulator column

  if (threadIdx.x == 0) {
    bar->stop = 0;
    for (int i = 0; i < MAX_A_SLOTS; ++i) {
      mbar_init(&bar->a_full[i], 1);
      mbar_init(&bar->a_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar->acc_full[i], 1);
      mbar_init(&bar->acc_empty[i], 4);
    }
    for (int i = 0; i < GROUPS; ++i) {
      mbar_init(&bar->s_full[i], 1);
      mbar_init(&bar->s_free[i], MODE == FWD ? 4 : 1);
      mbar_init(&bar->p_full[i], 4);
    }
    for (int i = 0; i < MAX_STAGES; ++i) {
      mbar_init(&bar->b_full[i], 1);
      mbar_init(&bar->b_empty[i], 1 + 4);  // the last product, and the group's warps (bias, sums, labels)
    }
    for (int i = 0; i < 2; ++i) mbar_init(&bar->drained[i], 1);
    mbar_init_fence();
  }
  if (warp == ISSUER) tmem_alloc(&bar->tmem, TMEM_COLUMNS);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = bar->tmem;
  const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // this warp's quarter of the 128 lanes

  if (warp == LOADER) {
    // ---- loads ----
    Ring as, bs;
    bool ok = true;
    for (int u = cta; u < units && ok; u += ctas) {
      const Range r = unit_range(g, u);
      ok = warp_wait(&bar->a_empty[as.i], as.phase ^ 1, stop);
      if (!ok) break;
      if (lane == 0) {
        mbar_expect(&bar->a_full[as.i], a_bytes);
        bulk_load(sA + (size_t)as.i * a_bytes, reinterpret_cast<const uint8_t*>(g.a) + (size_t)r.tile * a_bytes, a_bytes,
                  &bar->a_full[as.i]);
      }
      __syncwarp();
      as.next(g.a_slots);
      for (int bt = r.lo; bt < r.hi; ++bt) {
        ok = warp_wait(&bar->b_empty[bs.i], bs.phase ^ 1, stop);
        if (!ok) break;
        uint64_t* full = &bar->b_full[bs.i];
        const bool with_u = MODE == DW && g.row_u;
        const uint32_t metas = MODE == DW ? (with_u ? 3 : 2) : 1;
        if (lane == 0) {
          const long long col0 = (long long)bt * TN;
          float* meta = sMeta + bs.i * META;
          mbar_expect(full, b_bytes + metas * TN * 4);
          bulk_load(sB + (size_t)bs.i * b_bytes, reinterpret_cast<const uint8_t*>(g.b) + (size_t)bt * b_bytes, b_bytes,
                    full);
          bulk_load(meta, (MODE == DW ? g.lse2 : g.b2) + col0, TN * 4, full);
          if (MODE == DW) bulk_load(meta + TN, g.y + col0, TN * 4, full);
          if (with_u) bulk_load(meta + 2 * TN, g.row_u + col0, TN * 4, full);
        }
        __syncwarp();
        bs.next(g.stages);
      }
    }
    if (!ok) {
      // copies still in flight end before the CTA does
      int never = 0;
      for (int i = 0; i < g.stages; ++i)
        mbar_wait(&bar->b_full[i], i < bs.i ? bs.phase : bs.phase ^ 1, &never);
      for (int i = 0; i < g.a_slots; ++i)
        mbar_wait(&bar->a_full[i], i < as.i ? as.phase : as.phase ^ 1, &never);
    }
  } else if (warp == ISSUER) {
    // ---- first products: z ----
    const uint32_t leader = elect_leader();
    const uint32_t idesc = instr_desc(TN, false, FP16), hi = desc_hi(NP * D8 * 128);
    const uint32_t a0 = smem_u32(sA), b0 = smem_u32(sB);
    bool ok = true;
    for (Cursor c(g, cta, ctas); c.unit < units; c.next(g)) {
      const uint32_t b = c.t % GROUPS;
      ok = (c.bt > c.r.lo || warp_wait(&bar->a_full[c.as.i], c.as.phase, stop)) &&
           warp_wait(&bar->b_full[c.bs.i], c.bs.phase, stop) &&
           warp_wait(&bar->s_free[b], ((c.t / GROUPS) & 1) ^ 1, stop);
      if (!ok) break;
      fence_after();
      const uint32_t a_lo = desc_lo(a0 + c.as.i * a_bytes, 128), b_lo = desc_lo(b0 + c.bs.i * b_bytes, 128);
      const uint32_t z = tmem + b * SBUF;
#pragma unroll
      for (int q = 0; q < plane_products(NP); ++q) {
        const uint32_t aq = a_lo + plane_of_a(NP, q) * D8 * 8, bq = b_lo + plane_of_b(NP, q) * D8 * 8;
        mma_ss(leader, z, aq, hi, bq, hi, idesc, q > 0);
#pragma unroll 1  // the CTA's roles share the instruction cache: unrolled by 4, dX of 1080p fp32 takes 430 us, not 393
        for (int k = 2; k < D8; k += 2) mma_ss(leader, z, aq + k * 8, hi, bq + k * 8, hi, idesc, true);
      }
      mma_commit(leader, &bar->s_full[b]);
      if (c.bt + 1 == c.r.hi) mma_commit(leader, &bar->a_empty[c.as.i]);
      if (MODE == FWD) mma_commit(leader, &bar->b_empty[c.bs.i]);
    }
    if (!ok) {
      // what was issued ends before the tensor memory is freed
      int never = 0;
      mma_commit(leader, &bar->drained[0]);
      mbar_wait(&bar->drained[0], 0, &never);
    }
  } else if (MODE != FWD && warp == ISSUER2) {
    // ---- second products: the accumulators.  A warp of its own, so that waiting for one group's P does not
    // hold up the next group's z ----
    const uint32_t leader = elect_leader();
    const uint32_t idesc = instr_desc(D, true), hi = desc_hi(128), step = NP * D8 * 16;
    const uint32_t b0 = smem_u32(sB);
    bool ok = true;
    for (Cursor c(g, cta, ctas); c.unit < units; c.next(g)) {
      const uint32_t b = c.t % GROUPS;
      const int in_acc = (c.bt - c.r.lo) % g.flush;
      const bool first = in_acc == 0, last = in_acc + 1 == g.flush || c.bt + 1 == c.r.hi;
      ok = (!first || warp_wait(&bar->acc_empty[c.acc.i], c.acc.phase ^ 1, stop)) &&
           warp_wait(&bar->p_full[b], (c.t / GROUPS) & 1, stop);
      if (!ok) break;
      fence_after();
      const uint32_t dst = tmem + ACC0 + c.acc.i * ACCS * D, p = tmem + b * SBUF;
      const uint32_t b_lo = desc_lo(b0 + c.bs.i * b_bytes, NP * D8 * 128);
#pragma unroll
      for (int q = 0; q < (NP == 1 ? PP : plane_products(NP)); ++q) {
        const int pa = NP == 1 ? PP - 1 - q : plane_of_a(NP, q);
        const bool main = q + 1 == plane_products(NP);
        const uint32_t to = NP == 3 && !main ? dst + D : dst;
        const uint32_t bq = b_lo + (NP == 1 ? 0 : plane_of_b(NP, q)) * D8 * 8;
#pragma unroll
        for (int k = 0; k < TN / 16; ++k)
          mma_ts(leader, to, p + p_column(TN, 16 * k, pa), bq + k * step, hi, idesc,
                 k > 0 || (q > 0 && !(NP == 3 && main)) || !first);
      }
      mma_commit(leader, &bar->b_empty[c.bs.i]);
      mma_commit(leader, &bar->s_free[b]);
      if (last) {
        mma_commit(leader, &bar->acc_full[c.acc.i]);
        c.acc.next(g.acc_slots);
      }
    }
    if (!ok) {
      int never = 0;
      mma_commit(leader, &bar->drained[1]);
      mbar_wait(&bar->drained[1], 0, &never);
    }
  } else if (warp < LOADER) {
    // ---- z -> row statistics, or P ----
    constexpr int CH = MODE != FWD && NP == 3 ? 16 : 32;  // columns in registers at a time
    constexpr bool AHEAD = MODE == FWD || CH == 16;       // the next ones are loaded meanwhile, registers permitting
    const int group = warp / 4;
    const uint32_t buffer = tmem + lanes + group * SBUF;
    const int step = ctas;
    Ring bs;
    uint32_t t = 0;
    bool ok = true;
    int y_next = 0;
    float c_next = 0.f, e_next = 1.f;
    auto fetch = [&](int u) {  // the row's constants, one unit ahead
      if (u >= units) return;
      const int row = unit_range(g, u).tile * TILE + (warp & 3) * 32 + lane;
      if (MODE != DW) y_next = g.y[row];
      if (MODE == DX) c_next = -g.lse2[row], e_next = g.row_exact[row];
      if (MODE == DW) c_next = g.b2[row];
    };
    fetch(cta);
    for (int u = cta; u < units && ok; u += step) {
      const Range r = unit_range(g, u);
      const int row = r.tile * TILE + (warp & 3) * 32 + lane;
      const int y = y_next;
      const float row_c = c_next;  // -lse2 (DX) or the class's bias (DW)
      // dX: the row is scaled by row_exact at its end, which makes up for the rounding of lse2 to fp32 (at 2^17
      // classes 6e-7 of every p of the row, which shows where P W cancels); the label's 1 is scaled back
      const float one = MODE == DX ? 1.f / e_next : 1.f;
      fetch(u + step);
      const int slot = (int)((group - t) % GROUPS);  // this group's first tile in the unit
      float m = -INFINITY, s = 0.f;
      float2 bias_sum = make_float2(0.f, 0.f);
      for (int bt = r.lo; bt < r.hi; ++bt, ++t, bs.next(g.stages)) {
        if ((int)(t % GROUPS) != group) continue;
        // the meta data comes with the tile that z is made of
        ok = warp_wait(&bar->b_full[bs.i], bs.phase, stop) && warp_wait(&bar->s_full[group], (t / GROUPS) & 1, stop);
        if (!ok) break;
        fence_after();
        const float* meta = sMeta + bs.i * META;
        const int col0 = bt * TN;
        // whether a label of this warp's rows is among the tile's classes
        bool labelled;
        if (MODE == DW) {
          const int* ym = reinterpret_cast<const int*>(meta + TN);
          const unsigned wrow = row - lane;
          labelled = false;
#pragma unroll
          for (int k = 0; k < TN / 32; ++k) labelled |= (unsigned)ym[32 * k + lane] - wrow < 32u;
        } else {
          labelled = y >= 0 && (unsigned)(y - col0) < (unsigned)TN;
        }
        labelled = __any_sync(0xffffffffu, labelled);
        uint32_t z[CH];
        float2 tile_s[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        if (AHEAD) tmem_load(buffer, z);
#pragma unroll 1
        for (int c = 0; c < TN; c += CH) {
          if (!AHEAD) tmem_load(buffer + c, z);
          tmem_load_wait(z);
          if (MODE == FWD && c + CH == TN) {
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar->s_free[group]);
          }
          // t of the columns: z log2(e) + bias, less the row's or the column's log-sum in the gradients
          float2 x[CH / 2];
          const float2 l2e = make_float2(LOG2E, LOG2E), cst = make_float2(row_c, row_c), neg = make_float2(-1.f, -1.f);
#pragma unroll
          for (int i = 0; i < CH / 2; i += 2) {
            const float4 w = *reinterpret_cast<const float4*>(meta + c + 2 * i);
            const float2 z0 = make_float2(__uint_as_float(z[2 * i]), __uint_as_float(z[2 * i + 1]));
            const float2 z1 = make_float2(__uint_as_float(z[2 * i + 2]), __uint_as_float(z[2 * i + 3]));
            if (MODE == DW) {
              x[i] = fma2(make_float2(w.x, w.y), neg, fma2(z0, l2e, cst));
              x[i + 1] = fma2(make_float2(w.z, w.w), neg, fma2(z1, l2e, cst));
            } else {
              x[i] = fma2(z0, l2e, make_float2(w.x, w.y));
              x[i + 1] = fma2(z1, l2e, make_float2(w.z, w.w));
              if (MODE == DX) {
                x[i] = add2(x[i], cst);
                x[i + 1] = add2(x[i + 1], cst);
              }
            }
          }
          if (AHEAD && c + CH < TN) tmem_load(buffer + c + CH, z);
          if (MODE == FWD) {
            const int rel = y - (col0 + c);
            if (labelled && __any_sync(0xffffffffu, y >= 0 && (unsigned)rel < (unsigned)CH)) {
              float tl = 0.f;
#pragma unroll
              for (int i = 0; i < CH / 2; ++i) {
                if (rel == 2 * i) tl = x[i].x;
                if (rel == 2 * i + 1) tl = x[i].y;
              }
              if (y >= 0 && rel >= 0 && rel < CH) g.t_label[row] = tl;
            }
            float top = x[0].x;
#pragma unroll
            for (int i = 0; i < CH / 2; ++i) top = max3(top, x[i].x, x[i].y);
            // The sums' base follows the maximum only when it is left behind by 2^8: fp32 has the range,
            // and the rescaling is rare.
            if (top > m + 8.f) {
              const float f = ex2(m - top);
              s *= f;
              tile_s[0].x *= f;
              tile_s[0].y *= f;
              tile_s[1].x *= f;
              tile_s[1].y *= f;
              m = top;
            }
            const float nb = m == -INFINITY ? 0.f : -m;
            const float2 base = make_float2(nb, nb);
#pragma unroll
            for (int i = 0; i < CH / 2; ++i) {
              const float2 d = add2(x[i], base);
              tile_s[i & 1] = add2(tile_s[i & 1], make_float2(ex2(d.x), ex2(d.y)));
            }
          } else {
#pragma unroll
            for (int i = 0; i < CH / 2; ++i) x[i] = make_float2(ex2(x[i].x), ex2(x[i].y));
            if (labelled) {
              if (MODE == DX) {
                const int rel = y >= 0 ? y - (col0 + c) : -1;
                if (__any_sync(0xffffffffu, (unsigned)rel < (unsigned)CH))
#pragma unroll
                for (int i = 0; i < CH / 2; ++i) {
                  if (rel == 2 * i) x[i].x -= one;
                  if (rel == 2 * i + 1) x[i].y -= one;
                }
              } else {
                const int4* ym = reinterpret_cast<const int4*>(meta + TN + c);
#pragma unroll
                for (int i = 0; i < CH / 2; i += 2) {
                  const int4 l = ym[i / 2];
                  if (l.x == row) x[i].x -= 1.f;
                  if (l.y == row) x[i].y -= 1.f;
                  if (l.z == row) x[i + 1].x -= 1.f;
                  if (l.w == row) x[i + 1].y -= 1.f;
                }
              }
            }
            if (MODE == DW && g.row_u) {
#pragma unroll
              for (int i = 0; i < CH / 2; i += 2) {
                const float4 w = *reinterpret_cast<const float4*>(meta + 2 * TN + c + 2 * i);
                x[i] = make_float2(x[i].x * w.x, x[i].y * w.y);
                x[i + 1] = make_float2(x[i + 1].x * w.z, x[i + 1].y * w.w);
              }
            }
            if (MODE == DW && g.part_bias) {
#pragma unroll
              for (int i = 0; i < CH / 2; ++i) tile_s[i & 1] = add2(tile_s[i & 1], x[i]);
            }
            if constexpr (MODE != FWD) {
#pragma unroll
              for (int h = 0; h < CH / 16; ++h) {
                float2 half[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) half[i] = x[8 * h + i];
                store_p<PP, TN>(buffer, c + 16 * h, half);
              }
            }
          }
        }
        if (MODE != FWD) {
          tmem_store_wait();
          fence_before();
        }
        __syncwarp();
        if (lane == 0) {
          if (MODE != FWD) mbar_arrive(&bar->p_full[group]);
          mbar_arrive(&bar->b_empty[bs.i]);
        }
        const float2 ts = add2(tile_s[0], tile_s[1]);
        if (MODE == FWD) s += ts.x + ts.y;
        if (MODE == DW) bias_sum = add2(bias_sum, ts);
      }
      if (!ok) break;
      if (slot < g.slots) {
        const size_t at = ((size_t)r.split * g.slots + slot) * ((size_t)g.a_tiles * TILE) + row;
        if (MODE == FWD) {
          g.part_m[at] = m;
          g.part_s[at] = s;
        }
        if (MODE == DW && g.part_bias) g.part_bias[at] = bias_sum.x + bias_sum.y;
      }
    }
  } else if (MODE != FWD) {
    // ---- finished accumulators: added up in fp32 in the unit's partial rows, the last one (where the unit has
    // all of the streamed axis) straight into the gradient ----
    Ring acc;
    bool ok = true;
    const int row = (warp & 3) * 32 + lane;
    float scale_next = 0.f;
    auto fetch = [&](int u) {  // the row's factor, one unit ahead: its loads would hold up every unit
      if (u >= units || !g.grad.out) return;
      const long long n = (long long)unit_range(g, u).tile * TILE + row;
      scale_next = n < g.grad.rows ? grad_scale(g.grad, n) : 0.f;
    };
    fetch(cta);
    for (int u = cta; u < units && ok; u += ctas) {
      const Range r = unit_range(g, u);
      const size_t tile = (size_t)r.split * g.a_tiles + r.tile;
      const float scale = scale_next;
      fetch(u + ctas);
      const long long n = (long long)r.tile * TILE + row;
      float4* const dst = reinterpret_cast<float4*>(g.part_acc) + tile * (D / 4) * TILE + row;
      const bool direct = g.grad.out != nullptr, inside = direct && n < g.grad.rows;
      for (int bt = r.lo; bt < r.hi; bt += g.flush) {
        ok = warp_wait(&bar->acc_full[acc.i], acc.phase, stop);
        if (!ok) break;
        fence_after();
        const uint32_t src = tmem + lanes + ACC0 + acc.i * ACCS * D;
        if (!direct && !g.part_acc) {  // only the bias is wanted
          fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar->acc_empty[acc.i]);
          acc.next(g.acc_slots);
          continue;
        }
#pragma unroll 1
        for (int c = 0; c < D; c += 16) {
          float4* at = dst + (size_t)(c / 4) * TILE;
          float4 old[4];
          if (bt > r.lo) {
#pragma unroll
            for (int i = 0; i < 4; ++i) old[i] = at[i * TILE];
          }
          // the smallest group first
          uint32_t part[16];
          float v[16];
#pragma unroll
          for (int k = ACCS - 1; k >= 0; --k) {
            tmem_load(src + k * D + c, part);
            tmem_load_wait(part);
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(part[i]) + (k == ACCS - 1 ? 0.f : v[i]);
          }
          if (c + 16 >= D) {
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar->acc_empty[acc.i]);
          }
          if (bt > r.lo) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              v[4 * i] += old[i].x;
              v[4 * i + 1] += old[i].y;
              v[4 * i + 2] += old[i].z;
              v[4 * i + 3] += old[i].w;
            }
          }
          if (direct && bt + g.flush >= r.hi) {
            if (inside) write_grad<typename PlanesType<NP>::type>(g.grad, n, c, v, scale);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) at[i * TILE] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
          }
        }
        acc.next(g.acc_slots);
      }
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == ISSUER) tmem_free(tmem, TMEM_COLUMNS);
  if (threadIdx.x == 0 && *stop)
    atomicOr((unsigned long long*)g.error_word, (unsigned long long)ERR_LOOKBACK_TIMEOUT);
}

template <int NP, int TN, bool FP16>
__global__ void __launch_bounds__(stream_threads<FWD>(), 1) forward_kernel(const StreamArgs g) {
  extern __shared__ __align__(1024) uint8_t smem[];
  stream_pass<FWD, NP, TN, NP, FP16>(g, smem, blockIdx.x, gridDim.x);
}

template <int MODE, int NP, int TN, int PP>
__global__ void __launch_bounds__(stream_threads<MODE>(), 1) gradient_kernel(const StreamArgs g) {
  extern __shared__ __align__(1024) uint8_t smem[];
  stream_pass<MODE, NP, TN, PP>(g, smem, blockIdx.x, gridDim.x);
}

// Both gradients in one launch, for calls whose CTAs have one unit each: dW's
// CTAs then start on the SMs that dX leaves idle (8191 x 8200 x 65 fp32 313 ->
// 269 us).  With more units the two kernels are faster apart (1080p, 256
// classes, 16 channels: 708 us, together 785).
template <int NP, int TN, int PP>
__global__ void __launch_bounds__(stream_threads<DX>(), 1)
    gradients_kernel(const StreamArgs gx, const StreamArgs gw, const int x_ctas) {
  extern __shared__ __align__(1024) uint8_t smem[];
  if ((int)blockIdx.x < x_ctas) stream_pass<DX, NP, TN, PP>(gx, smem, blockIdx.x, x_ctas);
  else stream_pass<DW, NP, TN, PP>(gw, smem, blockIdx.x - x_ctas, gridDim.x - x_ctas);
}

// ---------------------------------------------------------------------------
// Joins.
// ---------------------------------------------------------------------------
__device__ __forceinline__ double block_sum(double v) {
  __shared__ double s_part[THREADS / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) s_part[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = 0.0;
  if (threadIdx.x == 0)
    for (int w = 0; w < THREADS / 32; ++w) t += s_part[w];
  __syncthreads();
  return t;
}

// Joins the slots' (maximum, sum) pairs of every row: LANES threads per row
// take every LANES-th slot and are joined in a fixed order (8 where a few rows
// have hundreds of slots: 37 rows of 50,001 classes 63 -> 11 us).  A label whose
// class takes no part (bias -inf) has the loss +inf and no gradient; one whose
// logit overflowed to -inf has its gradient, with the probability 0.  The last
// CTA to finish adds up the CTAs' sums in their order.
template <int LANES>
__global__ void __launch_bounds__(THREADS) join_rows_kernel(const gsb_class_loss_args a, const Kept kept, const float* __restrict__ part_m,
                                                            const float* __restrict__ part_s,
                                                            const float* __restrict__ t_label, int slots,
                                                            long long rows, double* __restrict__ block_loss,
                                                            double* __restrict__ block_count, int* __restrict__ ticket) {
  const long long N = a.B * a.S;
  double loss = 0.0, count = 0.0;
  const int sub = threadIdx.x % LANES;
  for (long long n0 = (long long)blockIdx.x * (THREADS / LANES); n0 < rows;
       n0 += (long long)gridDim.x * (THREADS / LANES)) {
    const long long n = n0 + threadIdx.x / LANES;
    const bool inside = n < rows;
    const int y = inside ? kept.row_y[n] : -1;
    float m = -INFINITY, s = 0.f;
    if (y >= 0)
#pragma unroll 4  // loads in flight (37 rows of 50,001 classes: 22 -> 11 us)
      for (int k = sub; k < slots; k += LANES) {
        const float pm = part_m[k * rows + n], ps = part_s[k * rows + n];
        const float top = fmaxf(m, pm), base = top == -INFINITY ? 0.f : top;
        s = s * ex2(m - base) + ps * ex2(pm - base);
        m = top;
      }
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) {
      const float pm = __shfl_xor_sync(0xffffffffu, m, o), ps = __shfl_xor_sync(0xffffffffu, s, o);
      const float top = fmaxf(m, pm), base = top == -INFINITY ? 0.f : top;
      s = s * ex2(m - base) + ps * ex2(pm - base);
      m = top;
    }
    if (sub == 0 && inside) {
      float l2 = INFINITY, l = 0.f, exact = 1.f;
      if (y >= 0) {
        const float t = t_label[n];
        count += 1.0;
        if (t == -INFINITY && kept.class_bias2[y] == -INFINITY) {
          l = INFINITY;
          kept.row_y[n] = -1;
        } else {
          // (maximum - t) + log2(sum) instead of lse2 - t: the maximum and t often agree in most digits
          const float ls = log2f(s);
          l = (float)(((double)(m - t) + (double)ls) * LN2);
          l2 = m + ls;
          exact = exp2f((l2 - m) - ls);  // l2 - m is exact or nearly so: the part of ls that l2 holds
        }
        loss += l;
      }
      kept.row_lse2[n] = l2;
      kept.row_exact[n] = exact;
      if (a.reduction == GSB_REDUCE_NONE && n < N) a.loss[n] = l;
    }
  }
  loss = block_sum(loss);
  count = block_sum(count);
  __shared__ bool s_last;
  if (threadIdx.x == 0) {
    block_loss[blockIdx.x] = loss;
    block_count[blockIdx.x] = count;
    __threadfence();
    s_last = atomicAdd(ticket, 1) == (int)gridDim.x - 1;
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  loss = count = 0.0;
  for (int i = threadIdx.x; i < (int)gridDim.x; i += THREADS) {
    loss += __ldcg(block_loss + i);
    count += __ldcg(block_count + i);
  }
  loss = block_sum(loss);
  count = block_sum(count);
  if (threadIdx.x == 0) {
    const double inv = a.reduction == GSB_REDUCE_MEAN ? 1.0 / fmax(count, 1.0) : 1.0;
    *kept.inv_count = (float)inv;  // what a mean divides by
    if (a.reduction != GSB_REDUCE_NONE) *a.loss = (float)(loss * inv);
  }
}

// The rows' upstream factors, zero where a row has no gradient (whatever
// upstream holds there).
__global__ void __launch_bounds__(THREADS) row_upstream_kernel(const float* __restrict__ up,
                                                               const int* __restrict__ row_y, long long rows,
                                                               float* __restrict__ out) {
  const long long n = (long long)blockIdx.x * THREADS + threadIdx.x;
  if (n < rows) out[n] = row_y[n] >= 0 ? up[n] : 0.f;
}

// What the passes left in pieces: dX's and dW's partial rows (entries are
// quads of columns, [tile][column / 4][row]) and the bias's partial sums.  A
// CTA takes 32 entries, eight threads each, which take every eighth piece and
// are added in order.  Counts are multiples of 128.
struct Join {
  GradOut out;
  const float* part;
  long long count;
  int splits;
};
struct Joins {
  Join x, w, bias;
};

template <typename T>
__global__ void __launch_bounds__(THREADS) join_grads_kernel(const Joins j, int D) {
  __shared__ float4 s_part[8][32];
  const int lane = threadIdx.x % 32, sub = threadIdx.x / 32;
  long long q = (long long)blockIdx.x * 32 + lane;
  const bool is_x = q < j.x.count;
  if (!is_x) q -= j.x.count;
  const bool is_bias = !is_x && q >= j.w.count;
  if (is_bias) q -= j.w.count;
  const Join& in = is_x ? j.x : is_bias ? j.bias : j.w;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k = sub; k < in.splits; k += 8) {
    if (is_bias) {
      sum.x += in.part[k * in.count + q];
    } else {
      const float4 v = reinterpret_cast<const float4*>(in.part)[k * in.count + q];
      sum = make_float4(sum.x + v.x, sum.y + v.y, sum.z + v.z, sum.w + v.w);
    }
  }
  s_part[sub][lane] = sum;
  __syncthreads();
  if (sub != 0) return;
  for (int k = 1; k < 8; ++k) {
    const float4 v = s_part[k][lane];
    sum = make_float4(sum.x + v.x, sum.y + v.y, sum.z + v.z, sum.w + v.w);
  }
  if (is_bias) {
    if (q < in.out.rows) ((float*)in.out.out)[q] = sum.x * grad_scale(in.out, q);
    return;
  }
  const long long strip = q / TILE;
  const long long n = strip / (D / 4) * TILE + q % TILE;
  if (n >= in.out.rows) return;
  float v[4] = {sum.x, sum.y, sum.z, sum.w};
  write_grad<T>(in.out, n, (int)(strip % (D / 4)) * 4, v, grad_scale(in.out, n));
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------
constexpr int SMS = 148;
constexpr int FEW_CLASSES = 128, FEW_CHANNELS = 8;
constexpr int JOIN_BLOCKS = SMS * 8;

// Pieces of the streamed axis: the number for which the waves of work units
// over the SMs take the least time, in tiles.  A unit costs `unit` tiles
// beside its own, and `split` more when its axis is cut (partial results are
// written and joined).  128 tiles of rows, 512 of classes (256 channels):
// forward in 8 pieces 285 us, in one 321; the gradients stay whole.
inline int split_count(long long a_tiles, long long b_tiles, double unit, double split) {
  int best = 1;
  double least = 0.0;
  const long long most = std::min(b_tiles, std::max(16ll, SMS / a_tiles));
  for (int n = 1; n <= most; ++n) {
    const long long waves = (a_tiles * n + SMS - 1) / SMS;
    const double t = waves * ((b_tiles + n - 1) / n + unit + (n > 1 ? split : 0.0));
    if (n == 1 || t < 0.97 * least) {
      best = n;
      least = t;
    }
  }
  return best;
}

// Shared memory of a pass.  Above half of an SM's, so that a CTA that holds
// all tensor memory columns never shares an SM with another one.
constexpr size_t SMEM_MIN = 118 * 1024, SMEM_MAX = 227 * 1024;

// Columns of a streamed tile: the most of 128 (64 in the gradient passes,
// whose tensor memory then has room for four z buffers), 64 and 32 with which
// the resident tile and four stages fit (three stages of 32 columns for fp16
// in training with more than 224 channels).  Three planes of P take half as
// much tensor memory again.
template <int MODE>
inline int tile_columns(int planes, int D8) {
  int tn = MODE == FWD ? 128 : 64;
  while (tn > 32 && GROUPS * z_columns<MODE>(planes, tn) + (MODE == FWD ? 0 : accumulators(planes) * D8 * 8) >
                        TMEM_COLUMNS)
    tn /= 2;
  while (tn > 32 && (size_t)planes * D8 * (2048 + 4 * tn * 16) + 4 * meta_floats<MODE>(tn) * 4 + sizeof(Barriers) + 128 >
                        SMEM_MAX)
    tn /= 2;
  return tn;
}

struct Dims {
  long long N, x_tiles, w_tiles;  // tiles of 128 rows, as packed
  int D, D8, planes;
  int fwd_tn, grad_tn;            // rows of a streamed tile
  int fwd_cols, dx_cols, dw_cols;  // streamed tiles
  int fwd_splits, dx_splits, dw_splits;
  int fwd_slots, dw_slots;        // partial results per split
};
inline Dims dims_of(const gsb_class_loss_args* a) {
  Dims d;
  d.N = a->B * a->S;
  d.x_tiles = tiles_of(d.N);
  d.w_tiles = tiles_of(a->V);
  d.D = pad_c(a->C);
  d.D8 = d.D / 8;
  d.planes = planes_of(a);
  d.fwd_tn = tile_columns<FWD>(d.planes, d.D8);
  d.grad_tn = tile_columns<DW>(d.planes, d.D8);
  d.fwd_cols = div_up(a->V, d.fwd_tn);
  d.dx_cols = div_up(a->V, d.grad_tn);
  d.dw_cols = div_up(d.N, d.grad_tn);
  d.fwd_splits = d.x_tiles > 0 ? split_count(d.x_tiles, d.fwd_cols, 1.5, 0.0) : 1;
  d.dx_splits = d.x_tiles > 0 ? split_count(d.x_tiles, d.dx_cols, 2.0, d.D / 24.0) : 1;
  d.dw_splits = split_count(d.w_tiles, std::max(d.dw_cols, 1), 2.0, d.D / 24.0);
  d.fwd_slots = std::min(GROUPS, div_up(d.fwd_cols, d.fwd_splits));
  d.dw_slots = std::min(GROUPS, std::max(1, div_up(d.dw_cols, d.dw_splits)));
  return d;
}

struct Carver {
  char* base;
  size_t off = 0;
  template <typename T>
  T* take(size_t n) {
    T* p = (T*)(base + off);
    off += align256(n * sizeof(T));
    return p;
  }
};

inline size_t carve_kept(void* base, const Dims& d, Kept* k) {
  Carver c{(char*)base};
  k->packed_x = c.take<uint4>((size_t)d.x_tiles * TILE * d.planes * d.D8);
  k->packed_w = c.take<uint4>((size_t)d.w_tiles * TILE * d.planes * d.D8);
  k->class_bias2 = c.take<float>((size_t)d.w_tiles * TILE);
  k->row_lse2 = c.take<float>((size_t)d.x_tiles * TILE);
  k->row_exact = c.take<float>((size_t)d.x_tiles * TILE);
  k->row_y = c.take<int>((size_t)d.x_tiles * TILE);
  k->inv_count = c.take<float>(1);
  return c.off;
}

struct FwdWs {
  float *part_m, *part_s, *t_label;
  double *block_loss, *block_count;
  int* ticket;
};
inline size_t carve_fwd(void* base, const Dims& d, FwdWs* w) {
  Carver c{(char*)base};
  const size_t rows = (size_t)d.x_tiles * TILE;
  w->part_m = c.take<float>(rows * d.fwd_splits * d.fwd_slots);
  w->part_s = c.take<float>(rows * d.fwd_splits * d.fwd_slots);
  w->t_label = c.take<float>(rows);
  w->block_loss = c.take<double>(JOIN_BLOCKS);
  w->block_count = c.take<double>(JOIN_BLOCKS);
  w->ticket = c.take<int>(1);
  return c.off;
}

struct BwdWs {
  float *part_x, *part_w, *part_bias, *row_u;
};
// Partial rows are needed by units that have a part of the streamed axis, or
// more of it than one accumulator takes.
inline bool needs_partials(int splits, int cols, int tn, int planes) {
  return splits > 1 || cols > chain_products(planes) / (tn / 16);
}
inline size_t carve_bwd(void* base, const Dims& d, BwdWs* w) {
  Carver c{(char*)base};
  const size_t x = (size_t)d.x_tiles * TILE, v = (size_t)d.w_tiles * TILE;
  w->part_x = c.take<float>(needs_partials(d.dx_splits, d.dx_cols, d.grad_tn, d.planes) ? x * d.dx_splits * d.D : 0);
  w->part_w = c.take<float>(needs_partials(d.dw_splits, d.dw_cols, d.grad_tn, d.planes) ? v * d.dw_splits * d.D : 0);
  w->part_bias = c.take<float>(v * d.dw_splits * d.dw_slots);
  w->row_u = c.take<float>(x);
  return c.off;
}

int check_sizes(const gsb_class_loss_args* a, const char* what) {
  if (!a) {
    set_error("%s: null arguments", what);
    return GSB_ERR_INVALID;
  }
  const int max_c = a->dtype == GSB_TYPE_FP32 ? GSB_CLASS_LOSS_MAX_C_FP32 : GSB_CLASS_LOSS_MAX_C;
  if (a->dtype < GSB_TYPE_FP32 || a->dtype > GSB_TYPE_FP16 || a->reduction < GSB_REDUCE_NONE ||
      a->reduction > GSB_REDUCE_MEAN) {
    set_error("%s: unknown dtype %d or reduction %d", what, a->dtype, a->reduction);
    return GSB_ERR_INVALID;
  }
  if (a->B < 0 || a->S < 0 || a->B >= (1ll << 31) || a->S >= (1ll << 31) || a->B * a->S >= (1ll << 31) - TILE ||
      a->V < 1 || a->V >= (1ll << 31) - TILE || a->C < 1 || a->C > max_c) {
    set_error("%s: sizes out of range (B %lld, S %lld, C %d, V %lld)", what, a->B, a->S, a->C, a->V);
    return GSB_ERR_INVALID;
  }
  return GSB_OK;
}

int check_args(const gsb_class_loss_args* a, const char* what) {
  const int st = check_sizes(a, what);
  if (st != GSB_OK) return st;
  if (!a->kept || !a->error_word || !a->workspace || (uintptr_t)a->kept % 256 || (uintptr_t)a->workspace % 256) {
    set_error("%s: null or unaligned buffer", what);
    return GSB_ERR_INVALID;
  }
  return GSB_OK;
}

// Fills in what a pass's CTAs have room for; returns its shared memory.
template <int MODE, int NP, int TN>
size_t plan_pass(StreamArgs* g) {
  const size_t a_bytes = (size_t)NP * g->D8 * 2048;
  const size_t stage = (size_t)NP * g->D8 * TN * 16 + meta_floats<MODE>(TN) * 4;
  const size_t fixed = sizeof(Barriers) + 128;
  constexpr int SBUF = z_columns<MODE>(NP, TN);
  static_assert(GROUPS * SBUF <= TMEM_COLUMNS, "z buffers");

  g->flush = chain_products(NP) / (TN / 16);
  for (g->a_slots = MAX_A_SLOTS; g->a_slots > 1; --g->a_slots)
    if (g->a_slots * a_bytes + 6 * stage + fixed <= SMEM_MAX) break;
  g->stages = (int)std::min<size_t>(MAX_STAGES, (SMEM_MAX - fixed - g->a_slots * a_bytes) / stage);
  const int acc = MODE == FWD ? 0 : accumulators(NP) * g->D8 * 8;
  g->acc_slots = GROUPS * SBUF + 2 * acc <= TMEM_COLUMNS ? 2 : 1;
  return std::max(SMEM_MIN, g->a_slots * a_bytes + g->stages * stage + fixed);
}
inline int pass_ctas(const StreamArgs& g) { return std::min(g.a_tiles * g.splits, SMS); }

// A kernel's limit of shared memory belongs to the kernel, whose launches need different sizes, and host threads
// launch side by side: every launch sets the same limit.
template <typename... Args>
void launch_pass(void (*kernel)(Args...), int ctas, int threads, size_t smem, cudaStream_t s, const Args&... args) {
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM_MAX) == cudaSuccess)
    kernel<<<ctas, threads, smem, s>>>(args...);
}

template <int NP, int TN, bool FP16 = false>
int launch_forward(StreamArgs g, cudaStream_t s) {
  const size_t smem = plan_pass<FWD, NP, TN>(&g);
  launch_pass(forward_kernel<NP, TN, FP16>, pass_ctas(g), stream_threads<FWD>(), smem, s, g);
  return check_launch("class loss forward");
}
template <int NP, int TN, int PP = NP>
int launch_backward(StreamArgs gx, StreamArgs gw, cudaStream_t s) {
  const size_t x_smem = plan_pass<DX, NP, TN>(&gx), w_smem = plan_pass<DW, NP, TN>(&gw);
  const int x_units = gx.a_tiles * gx.splits, w_units = gw.a_tiles * gw.splits;
  if (x_units && w_units && x_units <= SMS && w_units <= SMS) {
    launch_pass(gradients_kernel<NP, TN, PP>, x_units + w_units, stream_threads<DX>(), std::max(x_smem, w_smem), s, gx,
                gw, x_units);
    return check_launch("class loss backward");
  }
  if (x_units) launch_pass(gradient_kernel<DX, NP, TN, PP>, pass_ctas(gx), stream_threads<DX>(), x_smem, s, gx);
  if (w_units) launch_pass(gradient_kernel<DW, NP, TN, PP>, pass_ctas(gw), stream_threads<DW>(), w_smem, s, gw);
  return check_launch("class loss backward");
}

}  // namespace
}  // namespace gsb

GSB_EXPORT int gsb_class_loss_sizes(const gsb_class_loss_args* a, size_t sizes[3]) {
  using namespace gsb;
  const int st = check_sizes(a, "gsb_class_loss_sizes");
  if (st != GSB_OK) return st;
  const Dims d = dims_of(a);
  Kept k;
  FwdWs f;
  BwdWs b;
  sizes[0] = carve_kept(nullptr, d, &k);
  sizes[1] = carve_fwd(nullptr, d, &f);
  sizes[2] = carve_bwd(nullptr, d, &b);
  return GSB_OK;
}

GSB_EXPORT int gsb_class_loss_fwd(const gsb_class_loss_args* a, void* stream) {
  using namespace gsb;
  const int st = check_args(a, "gsb_class_loss_fwd");
  if (st != GSB_OK) return st;
  const Dims d = dims_of(a);
  if (!a->weight || !a->loss || (d.N > 0 && (!a->features || !a->labels))) {
    set_error("gsb_class_loss_fwd: null pointer");
    return GSB_ERR_INVALID;
  }
  FwdWs w;
  if (a->workspace_bytes < carve_fwd(a->workspace, d, &w)) {
    set_error("gsb_class_loss_fwd: workspace too small");
    return GSB_ERR_INVALID;
  }
  cudaStream_t s = (cudaStream_t)stream;
  Kept kept;
  carve_kept(a->kept, d, &kept);
  StreamArgs g{};
  g.a = kept.packed_x;
  g.b = kept.packed_w;
  g.b2 = kept.class_bias2;
  g.y = kept.row_y;
  g.a_tiles = (int)d.x_tiles;
  g.b_tiles = d.fwd_cols;
  g.splits = d.fwd_splits;
  g.slots = d.fwd_slots;
  g.error_word = a->error_word;
  g.D8 = d.D8;
  g.part_m = w.part_m;
  g.part_s = w.part_s;
  g.t_label = w.t_label;
  const int tiles = (int)(d.w_tiles + d.x_tiles);
  const bool fp16 = a->dtype == GSB_TYPE_FP16 && d.planes == 1;
  if (fp16) pack_kernel<__half, 1><<<tiles, THREADS, 0, s>>>(*a, kept, d.D8, (int)d.w_tiles, w.ticket);
  else if (d.planes == 1) pack_kernel<__nv_bfloat16, 1><<<tiles, THREADS, 0, s>>>(*a, kept, d.D8, (int)d.w_tiles, w.ticket);
  else if (d.planes == 2) pack_kernel<__half, 2><<<tiles, THREADS, 0, s>>>(*a, kept, d.D8, (int)d.w_tiles, w.ticket);
  else pack_kernel<float, 3><<<tiles, THREADS, 0, s>>>(*a, kept, d.D8, (int)d.w_tiles, w.ticket);
  if (d.N > 0) {
    int r = GSB_ERR_INVALID;
    switch (d.planes * 1000 + d.fwd_tn) {
      case 1128: r = fp16 ? launch_forward<1, 128, true>(g, s) : launch_forward<1, 128>(g, s); break;
      case 1064: r = fp16 ? launch_forward<1, 64, true>(g, s) : launch_forward<1, 64>(g, s); break;
      case 2128: r = launch_forward<2, 128>(g, s); break;
      case 2064: r = launch_forward<2, 64>(g, s); break;
      case 2032: r = launch_forward<2, 32>(g, s); break;
      case 3128: r = launch_forward<3, 128>(g, s); break;
      case 3064: r = launch_forward<3, 64>(g, s); break;
      case 3032: r = launch_forward<3, 32>(g, s); break;
      default: set_error("gsb_class_loss_fwd: no pass for %d planes and tiles of %d", d.planes, d.fwd_tn);
    }
    if (r != GSB_OK) return r;
  }
  const int slots = d.fwd_splits * d.fwd_slots;
  const long long rows = d.x_tiles * TILE;
  const int per_cta = slots > 8 ? THREADS / 8 : THREADS;
  const int blocks = (int)std::max(1ll, std::min<long long>(JOIN_BLOCKS, (rows + per_cta - 1) / per_cta));
  if (slots > 8)
    join_rows_kernel<8><<<blocks, THREADS, 0, s>>>(*a, kept, w.part_m, w.part_s, w.t_label, slots, rows, w.block_loss,
                                                   w.block_count, w.ticket);
  else
    join_rows_kernel<1><<<blocks, THREADS, 0, s>>>(*a, kept, w.part_m, w.part_s, w.t_label, slots, rows, w.block_loss,
                                                   w.block_count, w.ticket);
  return check_launch("gsb_class_loss_fwd");
}

GSB_EXPORT int gsb_class_loss_bwd(const gsb_class_loss_args* a, void* stream) {
  using namespace gsb;
  const int st = check_args(a, "gsb_class_loss_bwd");
  if (st != GSB_OK) return st;
  const Dims d = dims_of(a);
  if (!a->train) {
    set_error("gsb_class_loss_bwd: the forward was not a training one");
    return GSB_ERR_INVALID;
  }
  if (!a->upstream && d.N > 0) {
    set_error("gsb_class_loss_bwd: null pointer");
    return GSB_ERR_INVALID;
  }
  BwdWs w;
  if (a->workspace_bytes < carve_bwd(a->workspace, d, &w)) {
    set_error("gsb_class_loss_bwd: workspace too small");
    return GSB_ERR_INVALID;
  }
  cudaStream_t s = (cudaStream_t)stream;
  if (d.N == 0) {
    if (a->grad_weight) cudaMemsetAsync(a->grad_weight, 0, (size_t)a->V * a->C * (a->dtype == GSB_TYPE_FP32 ? 4 : 2), s);
    if (a->grad_bias) cudaMemsetAsync(a->grad_bias, 0, (size_t)a->V * 4, s);
    return check_launch("gsb_class_loss_bwd");
  }
  Kept kept;
  carve_kept(a->kept, d, &kept);
  StreamArgs g{};
  g.b2 = kept.class_bias2;
  g.lse2 = kept.row_lse2;
  g.row_exact = kept.row_exact;
  g.y = kept.row_y;
  g.error_word = a->error_word;
  g.D8 = d.D8;
  const bool per_row = a->reduction == GSB_REDUCE_NONE, want_w = a->grad_weight || a->grad_bias;
  if (!a->grad_features && !want_w) return GSB_OK;
  StreamArgs gx = g, gw = g;  // no units unless wanted
  Joins joins{};
  if (a->grad_features) {
    GradOut& o = joins.x.out;
    o.out = a->grad_features;
    o.upstream = a->upstream;
    o.inv_count = per_row ? nullptr : kept.inv_count;
    o.y = kept.row_y;
    o.row_exact = kept.row_exact;
    o.rows = d.N;
    o.S = a->stride_c == 1 ? 0 : a->S;
    o.C = a->C;
    gx.a = kept.packed_x;
    gx.b = kept.packed_w;
    gx.a_tiles = (int)d.x_tiles;
    gx.b_tiles = d.dx_cols;
    gx.splits = d.dx_splits;
    gx.part_acc = w.part_x;
    if (d.dx_splits == 1) {
      gx.grad = o;
    } else {
      joins.x.part = w.part_x;
      joins.x.splits = d.dx_splits;
      joins.x.count = d.x_tiles * TILE * (d.D / 4);
    }
  }
  if (want_w) {
    GradOut& o = joins.w.out;
    o.out = a->grad_weight;
    o.upstream = per_row ? nullptr : a->upstream;  // a row's factor is already in P
    o.inv_count = per_row ? nullptr : kept.inv_count;
    o.rows = a->V;
    o.C = a->C;
    joins.bias.out = o;
    gw.a = kept.packed_w;
    gw.b = kept.packed_x;
    gw.a_tiles = (int)d.w_tiles;
    gw.b_tiles = d.dw_cols;
    gw.splits = d.dw_splits;
    gw.slots = d.dw_slots;
    gw.part_acc = a->grad_weight ? w.part_w : nullptr;
    gw.part_bias = a->grad_bias ? w.part_bias : nullptr;
    if (d.dw_splits == 1) {
      gw.grad = o;
    } else if (a->grad_weight) {
      joins.w.part = w.part_w;
      joins.w.splits = d.dw_splits;
      joins.w.count = d.w_tiles * TILE * (d.D / 4);
    }
    if (a->grad_bias) {
      joins.bias.out.out = a->grad_bias;
      joins.bias.part = w.part_bias;
      joins.bias.splits = d.dw_splits * d.dw_slots;
      joins.bias.count = d.w_tiles * TILE;
    }
    if (per_row) {
      row_upstream_kernel<<<div_up(d.x_tiles * TILE, THREADS), THREADS, 0, s>>>(a->upstream, kept.row_y,
                                                                               d.x_tiles * TILE, w.row_u);
      gw.row_u = w.row_u;
    }
  }
  int r = GSB_ERR_INVALID;
  switch (d.planes * 1000 + d.grad_tn) {
    case 1064:
      // P's rounding to bf16 averages out over classes and channels. With few of either it does not, and a second
      // plane of P costs little there (the passes are bound by the map's rows). Error of dX in units of that of
      // its own rounding to bf16, one plane: 831,000 x 15 classes x 5 channels 1.65, 788,000 x 149 x 2 1.69,
      // 239,000 x 627 x 9 1.35, 640,000 x 1000 x 32 1.25; two planes 1.0 everywhere, but 26% longer passes in
      // the last, so one stays there.
      r = a->V <= FEW_CLASSES || a->C <= FEW_CHANNELS ? launch_backward<1, 64, 2>(gx, gw, s) : launch_backward<1, 64>(gx, gw, s);
      break;
    case 2064: r = launch_backward<2, 64>(gx, gw, s); break;
    case 2032: r = launch_backward<2, 32>(gx, gw, s); break;
    case 3064: r = launch_backward<3, 64>(gx, gw, s); break;
    case 3032: r = launch_backward<3, 32>(gx, gw, s); break;
    default: set_error("gsb_class_loss_bwd: no pass for %d planes and tiles of %d", d.planes, d.grad_tn);
  }
  if (r != GSB_OK) return r;
  const long long blocks = (joins.x.count + joins.w.count + joins.bias.count) / 32;
  if (blocks > 0) {
    switch (a->dtype) {
      case GSB_TYPE_BF16: join_grads_kernel<__nv_bfloat16><<<(unsigned)blocks, THREADS, 0, s>>>(joins, d.D); break;
      case GSB_TYPE_FP16: join_grads_kernel<__half><<<(unsigned)blocks, THREADS, 0, s>>>(joins, d.D); break;
      default: join_grads_kernel<float><<<(unsigned)blocks, THREADS, 0, s>>>(joins, d.D); break;
    }
  }
  return check_launch("gsb_class_loss_bwd");
}
