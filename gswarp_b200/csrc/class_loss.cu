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
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "gsb_common.cuh"

namespace gsb {
namespace {

constexpr int THREADS = launch::CLASS_LOSS;
constexpr int TILE = 128;
constexpr float LOG2E = 1.4426950408889634f;
constexpr double LN2 = 0.6931471805599453;

__host__ __device__ inline int planes_of(int dtype) { return dtype == GSB_TYPE_FP32 ? 3 : dtype == GSB_TYPE_FP16 ? 2 : 1; }
inline int pad_c(int C) { return (C + 15) & ~15; }
inline long long tiles_of(long long n) { return (n + TILE - 1) / TILE; }
inline size_t tile_bytes(int dtype, int C) { return (size_t)planes_of(dtype) * pad_c(C) * TILE * 2; }
inline size_t align256(size_t b) { return (b + 255) & ~(size_t)255; }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float load_elem(const void* p, long long i, int dtype) {
  if (dtype == GSB_TYPE_FP32) return ((const float*)p)[i];
  if (dtype == GSB_TYPE_BF16) return __bfloat162float(((const __nv_bfloat16*)p)[i]);
  return __half2float(((const __half*)p)[i]);
}
__device__ __forceinline__ void store_elem(void* p, long long i, int dtype, float v) {
  if (dtype == GSB_TYPE_FP32) ((float*)p)[i] = v;
  else if (dtype == GSB_TYPE_BF16) ((__nv_bfloat16*)p)[i] = __float2bfloat16_rn(v);
  else ((__half*)p)[i] = __float2half_rn(v);
}

// ---------------------------------------------------------------------------
// Packing.  Tile layout: [plane][column / 8][row][8 columns] of bf16.
// ---------------------------------------------------------------------------
__device__ __forceinline__ void store_planes(uint4* tile, int D8, int d8, int row, const float (&x)[8], int planes) {
  float rest[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) rest[i] = x[i];
  for (int p = 0; p < planes; ++p) {
    __nv_bfloat162 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      h[i] = __floats2bfloat162_rn(rest[2 * i], rest[2 * i + 1]);
      // an infinity's remainder would be NaN; its first plane says it all
      const float2 f = __bfloat1622float2(h[i]);
      rest[2 * i] = isinf(f.x) ? 0.f : rest[2 * i] - f.x;
      rest[2 * i + 1] = isinf(f.y) ? 0.f : rest[2 * i + 1] - f.y;
    }
    tile[((size_t)p * D8 + d8) * TILE + row] = *reinterpret_cast<uint4*>(h);
  }
}

// One thread per (tile, 8 columns, row); rows without a label are zero.
__global__ void __launch_bounds__(THREADS) pack_rows_kernel(const gsb_class_loss_args a, int D8, long long total,
                                                            uint4* __restrict__ packed, int* __restrict__ row_y) {
  const int planes = planes_of(a.dtype);
  const long long N = a.B * a.S;
  for (long long i = (long long)blockIdx.x * THREADS + threadIdx.x; i < total; i += (long long)gridDim.x * THREADS) {
    const int row = (int)(i % TILE);
    const int d8 = (int)(i / TILE % D8);
    const long long tile = i / TILE / D8;
    const long long n = tile * TILE + row;
    int y = -1;
    if (n < N) {
      const long long l = a.labels64 ? ((const long long*)a.labels)[n] : (long long)((const int*)a.labels)[n];
      if (l != a.ignore_index) {
        if (l >= 0 && l < a.V) y = (int)l;
        else if (d8 == 0) atomicOr((unsigned long long*)a.error_word, (unsigned long long)ERR_BAD_LABEL);
      }
    }
    if (d8 == 0) row_y[n] = y;
    float x[8];
    const long long b = y >= 0 ? n / a.S : 0;
    const long long at = b * a.stride_b + (n - b * a.S) * a.stride_s;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int c = d8 * 8 + k;
      x[k] = y >= 0 && c < a.C ? load_elem(a.features, at + c * a.stride_c, a.dtype) : 0.f;
    }
    store_planes(packed + (size_t)tile * planes * D8 * TILE, D8, d8, row, x, planes);
  }
}

// The classifier's rows and its bias in base 2.  A class with the bias -inf
// takes no part and its row is not read; finite biases stay finite.
__global__ void __launch_bounds__(THREADS) pack_classes_kernel(const gsb_class_loss_args a, int D8, long long total,
                                                               uint4* __restrict__ packed, float* __restrict__ b2) {
  const int planes = planes_of(a.dtype);
  for (long long i = (long long)blockIdx.x * THREADS + threadIdx.x; i < total; i += (long long)gridDim.x * THREADS) {
    const int row = (int)(i % TILE);
    const int d8 = (int)(i / TILE % D8);
    const long long tile = i / TILE / D8;
    const long long v = tile * TILE + row;
    float bias = -INFINITY;
    if (v < a.V) {
      bias = a.bias ? a.bias[v] : 0.f;
      if (isfinite(bias)) bias = fminf(fmaxf(bias, -2e38f), 2e38f) * LOG2E;
    }
    if (d8 == 0) b2[v] = bias;
    float x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int c = d8 * 8 + k;
      x[k] = bias != -INFINITY && c < a.C ? load_elem(a.weight, v * a.C + c, a.dtype) : 0.f;
    }
    store_planes(packed + (size_t)tile * planes * D8 * TILE, D8, d8, row, x, planes);
  }
}

// ---------------------------------------------------------------------------
// The streaming pass: a CTA holds 128 rows and walks its range of the other
// operand's tiles on the fp32 pipes.
// ---------------------------------------------------------------------------
enum { FWD = 0, DX = 1, DW = 2 };

struct StreamArgs {
  const uint4* a;          // resident operand, packed
  const uint4* b;          // streamed operand, packed
  const float* b2;         // bias of the classes, base 2
  const float* lse2;       // rows (DX, DW)
  const int* y;            // rows
  const float* row_u;      // per-row upstream (DW, reduction none) or NULL
  int a_tiles, b_tiles, splits, planes, D8;
  float* part_m;           // FWD: [split][row]
  float* part_s;
  float* t_label;          // FWD: [row]
  float* part_acc;         // DX, DW: [split][row][D8 * 8]
  float* part_bias;        // DW: [split][row]
};

__device__ __forceinline__ float plane_sum(const uint4* tile, int planes, int D8, int d8, int row, int k) {
  float x = 0.f;
  for (int p = planes - 1; p >= 0; --p) {
    const __nv_bfloat16* e = reinterpret_cast<const __nv_bfloat16*>(tile + ((size_t)p * D8 + d8) * TILE + row);
    x += __bfloat162float(e[k]);
  }
  return x;
}

template <int MODE>
__global__ void __launch_bounds__(THREADS) stream_kernel(const StreamArgs g) {
  extern __shared__ float smem[];
  float* sA = smem;                       // [8][TILE]
  float* sB = sA + 8 * TILE;              // [8][TILE]
  float* sS = sB + 8 * TILE;              // [TILE][TILE + 1]
  float* sAcc = sS + TILE * (TILE + 1);   // [TILE][D + 1] (DX, DW)
  const int D = g.D8 * 8;
  const int tid = threadIdx.x;
  const int tile = blockIdx.x, split = blockIdx.y;
  const size_t tile_u4 = (size_t)g.planes * g.D8 * TILE;
  const uint4* A = g.a + (size_t)tile * tile_u4;
  const long long row0 = (long long)tile * TILE;
  const int lo = (int)((long long)g.b_tiles * split / g.splits), hi = (int)((long long)g.b_tiles * (split + 1) / g.splits);
  float m = -INFINITY, s = 0.f, bias_sum = 0.f;
  if (MODE != FWD)
    for (int i = tid; i < TILE * (D + 1); i += THREADS) sAcc[i] = 0.f;

  const int ty = tid / 16, tx = tid % 16;
  for (int bt = lo; bt < hi; ++bt) {
    const uint4* Bt = g.b + (size_t)bt * tile_u4;
    const long long col0 = (long long)bt * TILE;
    float acc[8][8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[i][j] = 0.f;
    for (int d8 = 0; d8 < g.D8; ++d8) {
      __syncthreads();
      for (int i = tid; i < 8 * TILE; i += THREADS) {
        sA[i] = plane_sum(A, g.planes, g.D8, d8, i % TILE, i / TILE);
        sB[i] = plane_sum(Bt, g.planes, g.D8, d8, i % TILE, i / TILE);
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        float x[8], w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = sA[k * TILE + ty * 8 + i];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = sB[k * TILE + tx + 16 * j];
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int j = 0; j < 8; ++j) acc[i][j] += x[i] * w[j];
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) sS[(ty * 8 + i) * (TILE + 1) + tx + 16 * j] = acc[i][j];
    __syncthreads();
    if (tid < TILE) {
      float* srow = sS + tid * (TILE + 1);
      const long long r = row0 + tid;
      if (MODE == FWD) {
        const int y = g.y[r];
        float mx = m;
        for (int c = 0; c < TILE; ++c) {
          const float t = fmaf(srow[c], LOG2E, g.b2[col0 + c]);
          srow[c] = t;
          mx = fmaxf(mx, t);
          if (y == col0 + c) g.t_label[r] = t;
        }
        const float base = mx == -INFINITY ? 0.f : mx;
        float sum = s * ex2(m - base);
        for (int c = 0; c < TILE; ++c) sum += ex2(srow[c] - base);
        m = mx;
        s = sum;
      } else if (MODE == DX) {
        const int y = g.y[r];
        const float l = g.lse2[r];
        for (int c = 0; c < TILE; ++c) {
          const float t = fmaf(srow[c], LOG2E, g.b2[col0 + c]);
          srow[c] = ex2(t - l) - (y == col0 + c ? 1.f : 0.f);
        }
      } else {
        const float b = g.b2[r];
        for (int c = 0; c < TILE; ++c) {
          const float t = fmaf(srow[c], LOG2E, b);
          float p = ex2(t - g.lse2[col0 + c]) - (g.y[col0 + c] == r ? 1.f : 0.f);
          if (g.row_u) p *= g.row_u[col0 + c];
          srow[c] = p;
          bias_sum += p;
        }
      }
    }
    __syncthreads();
    if (MODE != FWD) {
      const int row = tid % TILE;
      for (int d8 = 0; d8 < g.D8; ++d8)
        for (int k = tid / TILE; k < 8; k += THREADS / TILE) {
          float sum = 0.f;
          for (int c = 0; c < TILE; ++c) sum += sS[row * (TILE + 1) + c] * plane_sum(Bt, g.planes, g.D8, d8, c, k);
          sAcc[row * (D + 1) + d8 * 8 + k] += sum;
        }
    }
  }
  __syncthreads();
  const long long rows = (long long)g.a_tiles * TILE;
  if (MODE == FWD) {
    if (tid < TILE) {
      g.part_m[split * rows + row0 + tid] = m;
      g.part_s[split * rows + row0 + tid] = s;
    }
  } else {
    float* dst = g.part_acc + ((size_t)split * rows + row0) * D;
    for (int i = tid; i < TILE * D; i += THREADS) dst[i] = sAcc[i / D * (D + 1) + i % D];
    if (MODE == DW && tid < TILE) g.part_bias[split * rows + row0 + tid] = bias_sum;
  }
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

// Joins the slots' (maximum, sum) pairs of every row, in slot order.  A label
// whose class takes no part (bias -inf) has the loss +inf and no gradient.
__global__ void __launch_bounds__(THREADS) join_rows_kernel(const StreamArgs g, int slots, long long N,
                                                            float* __restrict__ lse2, int* __restrict__ row_y,
                                                            float* __restrict__ row_loss,
                                                            double* __restrict__ block_loss,
                                                            double* __restrict__ block_count) {
  const long long rows = (long long)g.a_tiles * TILE;
  double loss = 0.0, count = 0.0;
  for (long long n = (long long)blockIdx.x * THREADS + threadIdx.x; n < rows; n += (long long)gridDim.x * THREADS) {
    const int y = g.y[n];
    float l2 = INFINITY, l = 0.f;
    if (y >= 0) {
      float m = -INFINITY, s = 0.f;
      for (int k = 0; k < slots; ++k) m = fmaxf(m, g.part_m[k * rows + n]);
      const float base = m == -INFINITY ? 0.f : m;
      for (int k = 0; k < slots; ++k) s += g.part_s[k * rows + n] * ex2(g.part_m[k * rows + n] - base);
      const float t = g.t_label[n];
      count += 1.0;
      if (t == -INFINITY) {
        l = INFINITY;
        row_y[n] = -1;
      } else {
        // two addends instead of lse2 - t: the maximum and t often agree in most of their digits
        const float ls = log2f(s);
        l = (float)(((double)(base - t) + (double)ls) * LN2);
        l2 = base + ls;
      }
      loss += l;
    }
    lse2[n] = l2;
    if (row_loss && n < N) row_loss[n] = l;
  }
  loss = block_sum(loss);
  count = block_sum(count);
  if (threadIdx.x == 0) {
    block_loss[blockIdx.x] = loss;
    block_count[blockIdx.x] = count;
  }
}

// The blocks' sums in one fixed order; *inv_count is what a mean divides by.
__global__ void __launch_bounds__(THREADS) finish_loss_kernel(const double* __restrict__ block_loss,
                                                              const double* __restrict__ block_count, int blocks,
                                                              int reduction, float* __restrict__ loss,
                                                              float* __restrict__ inv_count) {
  double l = 0.0, c = 0.0;
  for (int i = threadIdx.x; i < blocks; i += THREADS) {
    l += block_loss[i];
    c += block_count[i];
  }
  l = block_sum(l);
  c = block_sum(c);
  if (threadIdx.x == 0) {
    const double inv = reduction == GSB_REDUCE_MEAN ? 1.0 / fmax(c, 1.0) : 1.0;
    *inv_count = (float)inv;
    if (reduction != GSB_REDUCE_NONE) *loss = (float)(l * inv);
  }
}

// The rows' upstream factors, zero where a row has no gradient (whatever
// upstream holds there).
__global__ void __launch_bounds__(THREADS) row_upstream_kernel(const float* __restrict__ up,
                                                               const int* __restrict__ row_y, long long rows,
                                                               float* __restrict__ out) {
  for (long long n = (long long)blockIdx.x * THREADS + threadIdx.x; n < rows; n += (long long)gridDim.x * THREADS)
    out[n] = row_y[n] >= 0 ? up[n] : 0.f;
}

// Sums the splits of dX in order, scales, and writes the features' layout.
__global__ void __launch_bounds__(THREADS) join_dx_kernel(const gsb_class_loss_args a, const float* __restrict__ part,
                                                          int splits, int D, long long rows) {
  const long long N = a.B * a.S;
  const long long total = N * a.C;
  for (long long i = (long long)blockIdx.x * THREADS + threadIdx.x; i < total; i += (long long)gridDim.x * THREADS) {
    // consecutive threads along the layout's contiguous direction
    long long n;
    int c;
    if (a.stride_c == 1) {
      n = i / a.C;
      c = (int)(i - n * a.C);
    } else {
      const long long b = i / (a.C * a.S), r = i - b * a.C * a.S;
      c = (int)(r / a.S);
      n = b * a.S + (r - c * a.S);
    }
    float v = 0.f;
    for (int k = 0; k < splits; ++k) v += part[((size_t)k * rows + n) * D + c];
    const float u = a.reduction == GSB_REDUCE_NONE ? a.upstream[n] : a.upstream[0] * a.inv_count[0];
    const long long b = n / a.S;
    // rows without a gradient stay exactly zero whatever upstream holds
    const bool used = a.row_y[n] >= 0;
    store_elem(a.grad_features, b * a.C * a.S + (a.stride_c == 1 ? (n - b * a.S) * a.C + c : c * a.S + (n - b * a.S)),
               a.dtype, used ? v * u : 0.f);
  }
}

__global__ void __launch_bounds__(THREADS) join_dw_kernel(const gsb_class_loss_args a, const float* __restrict__ part,
                                                          const float* __restrict__ part_bias, int splits, int slots,
                                                          int D, long long rows) {
  const float u = a.reduction == GSB_REDUCE_NONE ? 1.f : a.upstream[0] * a.inv_count[0];
  const long long total = a.V * (a.C + 1ll);
  for (long long i = (long long)blockIdx.x * THREADS + threadIdx.x; i < total; i += (long long)gridDim.x * THREADS) {
    const long long v = i / (a.C + 1);
    const int c = (int)(i - v * (a.C + 1));
    float sum = 0.f;
    if (c < a.C) {
      if (!a.grad_weight) continue;
      for (int k = 0; k < splits; ++k) sum += part[((size_t)k * rows + v) * D + c];
      store_elem(a.grad_weight, v * a.C + c, a.dtype, sum * u);
    } else if (a.grad_bias) {
      for (int k = 0; k < slots; ++k) sum += part_bias[k * rows + v];
      a.grad_bias[v] = sum * u;
    }
  }
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------
constexpr int SMS = 148;
constexpr int JOIN_BLOCKS = SMS * 4;

inline int split_count(long long a_tiles, long long b_tiles) {
  const long long want = (SMS + a_tiles - 1) / a_tiles;
  return (int)std::max(1ll, std::min(want, b_tiles));
}

struct Dims {
  long long N, x_tiles, w_tiles;
  int D, D8, planes, v_splits, n_splits;
};
inline Dims dims_of(const gsb_class_loss_args* a) {
  Dims d;
  d.N = a->B * a->S;
  d.x_tiles = tiles_of(d.N);
  d.w_tiles = tiles_of(a->V);
  d.D = pad_c(a->C);
  d.D8 = d.D / 8;
  d.planes = planes_of(a->dtype);
  d.v_splits = d.x_tiles > 0 ? split_count(d.x_tiles, d.w_tiles) : 1;
  d.n_splits = split_count(d.w_tiles, std::max(d.x_tiles, 1ll));
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

struct FwdWs {
  float *part_m, *part_s, *t_label;
  double *block_loss, *block_count;
};
inline size_t carve_fwd(void* base, const Dims& d, FwdWs* w) {
  Carver c{(char*)base};
  const size_t rows = (size_t)d.x_tiles * TILE;
  w->part_m = c.take<float>(rows * d.v_splits);
  w->part_s = c.take<float>(rows * d.v_splits);
  w->t_label = c.take<float>(rows);
  w->block_loss = c.take<double>(JOIN_BLOCKS);
  w->block_count = c.take<double>(JOIN_BLOCKS);
  return c.off;
}

struct BwdWs {
  float *part_x, *part_w, *part_bias, *row_u;
};
inline size_t carve_bwd(void* base, const Dims& d, BwdWs* w) {
  Carver c{(char*)base};
  w->part_x = c.take<float>((size_t)d.x_tiles * TILE * d.v_splits * d.D);
  w->part_w = c.take<float>((size_t)d.w_tiles * TILE * d.n_splits * d.D);
  w->part_bias = c.take<float>((size_t)d.w_tiles * TILE * d.n_splits);
  w->row_u = c.take<float>((size_t)d.x_tiles * TILE);
  return c.off;
}

int check_args(const gsb_class_loss_args* a, const char* what) {
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
  if ((uintptr_t)a->packed_x % 16 || (uintptr_t)a->packed_w % 16) {
    set_error("%s: packed buffers must be 16-byte aligned", what);
    return GSB_ERR_INVALID;
  }
  if (!a->packed_x || !a->packed_w || !a->class_bias2 || !a->row_lse2 || !a->row_y || !a->inv_count ||
      !a->error_word || !a->workspace) {
    set_error("%s: null pointer", what);
    return GSB_ERR_INVALID;
  }
  return GSB_OK;
}

template <int MODE>
int launch_stream(const StreamArgs& g, cudaStream_t s) {
  const size_t smem = (size_t)(16 * TILE + TILE * (TILE + 1) + (MODE == FWD ? 0 : TILE * (g.D8 * 8 + 1))) * 4;
  cudaFuncSetAttribute(stream_kernel<MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  stream_kernel<MODE><<<dim3(g.a_tiles, g.splits), THREADS, smem, s>>>(g);
  return check_launch("class loss pass");
}

inline int blocks_for(long long n) { return (int)std::max(1ll, std::min((n + THREADS - 1) / THREADS, (long long)SMS * 16)); }

}  // namespace
}  // namespace gsb

GSB_EXPORT size_t gsb_class_loss_packed_bytes(long long rows, int C, int dtype) {
  using namespace gsb;
  if (rows < 0 || C < 1 || dtype < GSB_TYPE_FP32 || dtype > GSB_TYPE_FP16) return 0;
  return (size_t)std::max(tiles_of(rows), 1ll) * tile_bytes(dtype, C);
}

GSB_EXPORT size_t gsb_class_loss_workspace_bytes(const gsb_class_loss_args* a, int backward) {
  using namespace gsb;
  if (!a || a->B < 0 || a->S < 0 || a->V < 1 || a->C < 1) return 0;
  const Dims d = dims_of(a);
  FwdWs f;
  BwdWs b;
  return (backward ? carve_bwd(nullptr, d, &b) : carve_fwd(nullptr, d, &f)) + 256;
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
  if (a->workspace_bytes < gsb_class_loss_workspace_bytes(a, 0)) {
    set_error("gsb_class_loss_fwd: workspace too small");
    return GSB_ERR_INVALID;
  }
  cudaStream_t s = (cudaStream_t)stream;
  FwdWs w;
  carve_fwd((void*)(((uintptr_t)a->workspace + 255) & ~(uintptr_t)255), d, &w);
  StreamArgs g{};
  g.a = (const uint4*)a->packed_x;
  g.b = (const uint4*)a->packed_w;
  g.b2 = a->class_bias2;
  g.y = a->row_y;
  g.a_tiles = (int)d.x_tiles;
  g.b_tiles = (int)d.w_tiles;
  g.splits = d.v_splits;
  g.planes = d.planes;
  g.D8 = d.D8;
  g.part_m = w.part_m;
  g.part_s = w.part_s;
  g.t_label = w.t_label;
  const long long x_total = d.x_tiles * d.D8 * TILE, w_total = d.w_tiles * d.D8 * TILE;
  pack_classes_kernel<<<blocks_for(w_total), THREADS, 0, s>>>(*a, d.D8, w_total, (uint4*)a->packed_w, a->class_bias2);
  if (d.N > 0) {
    pack_rows_kernel<<<blocks_for(x_total), THREADS, 0, s>>>(*a, d.D8, x_total, (uint4*)a->packed_x, a->row_y);
    const int r = launch_stream<FWD>(g, s);
    if (r != GSB_OK) return r;
  }
  const int blocks = (int)std::max(1ll, std::min<long long>(JOIN_BLOCKS, (d.x_tiles * TILE + THREADS - 1) / THREADS));
  join_rows_kernel<<<blocks, THREADS, 0, s>>>(g, d.v_splits, d.N, a->row_lse2, a->row_y,
                                              a->reduction == GSB_REDUCE_NONE ? a->loss : nullptr, w.block_loss,
                                              w.block_count);
  finish_loss_kernel<<<1, THREADS, 0, s>>>(w.block_loss, w.block_count, blocks, a->reduction, a->loss, a->inv_count);
  return check_launch("gsb_class_loss_fwd");
}

GSB_EXPORT int gsb_class_loss_bwd(const gsb_class_loss_args* a, void* stream) {
  using namespace gsb;
  const int st = check_args(a, "gsb_class_loss_bwd");
  if (st != GSB_OK) return st;
  const Dims d = dims_of(a);
  if (!a->upstream && d.N > 0) {
    set_error("gsb_class_loss_bwd: null pointer");
    return GSB_ERR_INVALID;
  }
  if (a->workspace_bytes < gsb_class_loss_workspace_bytes(a, 1)) {
    set_error("gsb_class_loss_bwd: workspace too small");
    return GSB_ERR_INVALID;
  }
  cudaStream_t s = (cudaStream_t)stream;
  if (d.N == 0) {
    if (a->grad_weight) cudaMemsetAsync(a->grad_weight, 0, (size_t)a->V * a->C * (a->dtype == GSB_TYPE_FP32 ? 4 : 2), s);
    if (a->grad_bias) cudaMemsetAsync(a->grad_bias, 0, (size_t)a->V * 4, s);
    return check_launch("gsb_class_loss_bwd");
  }
  BwdWs w;
  carve_bwd((void*)(((uintptr_t)a->workspace + 255) & ~(uintptr_t)255), d, &w);
  StreamArgs g{};
  g.b2 = a->class_bias2;
  g.lse2 = a->row_lse2;
  g.y = a->row_y;
  g.planes = d.planes;
  g.D8 = d.D8;
  if (a->grad_features) {
    g.a = (const uint4*)a->packed_x;
    g.b = (const uint4*)a->packed_w;
    g.a_tiles = (int)d.x_tiles;
    g.b_tiles = (int)d.w_tiles;
    g.splits = d.v_splits;
    g.part_acc = w.part_x;
    const int r = launch_stream<DX>(g, s);
    if (r != GSB_OK) return r;
    join_dx_kernel<<<blocks_for(d.N * a->C), THREADS, 0, s>>>(*a, w.part_x, d.v_splits, d.D, d.x_tiles * TILE);
  }
  if (a->grad_weight || a->grad_bias) {
    g.a = (const uint4*)a->packed_w;
    g.b = (const uint4*)a->packed_x;
    g.a_tiles = (int)d.w_tiles;
    g.b_tiles = (int)d.x_tiles;
    g.splits = d.n_splits;
    g.part_acc = w.part_w;
    g.part_bias = w.part_bias;
    if (a->reduction == GSB_REDUCE_NONE) {
      row_upstream_kernel<<<blocks_for(d.x_tiles * TILE), THREADS, 0, s>>>(a->upstream, a->row_y, d.x_tiles * TILE, w.row_u);
      g.row_u = w.row_u;
    }
    const int r = launch_stream<DW>(g, s);
    if (r != GSB_OK) return r;
    join_dw_kernel<<<blocks_for(a->V * (a->C + 1ll)), THREADS, 0, s>>>(*a, w.part_w, w.part_bias, d.n_splits,
                                                                      d.n_splits, d.D, d.w_tiles * TILE);
  }
  return check_launch("gsb_class_loss_bwd");
}
