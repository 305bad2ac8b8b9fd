// codebook.cu -- rows of a shared attribute codebook, and their gradients.
//
// A compressed scene stores one code per Gaussian and a table T of K rows
// (SH rows, DC colours, feature rows); the rasterizer's input row is
//
//   out[p,:] = s_p * T[c_p,:]        s_p = scale * gain[p],  c_p = -1: zero row
//
// and training needs
//
//   dT[k,:] = sum over {p : c_p = k} of s_p * g[p,:]
//   dgain[p] = scale * <g[p,:], T[c_p,:]>.
//
// Forward moves P rows and is bound by that write.  Backward is bound by the
// one read of g; the sums go by sorted code instead of atomics, so that they
// have one order (the same bits on every call) and no hot row serializes:
// the codes are sorted (radix_sort.cuh, only the key bits of K), the sorted
// positions are cut into chunks of equal length, and one group of lanes sums
// each chunk's runs in registers in fp32.  A run that lies inside its chunk
// is stored at once; the at most two that cross a chunk's ends become rows of
// a next level (key, fp32 sum), summed by the same kernel, until one chunk is
// left.  Sums are therefore trees of short sequential sums.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "gsb_common.cuh"
#include "radix_sort.cuh"

namespace gsb {
namespace {

constexpr int THREADS = launch::CODEBOOK;
constexpr int SEG_UNROLL = 4;       // rows in flight per group of lanes
constexpr int FWD_CTA_ROWS = 64;    // rows per CTA of the gather; a multiple of 16 keeps CTAs 16-byte aligned
constexpr long long MAX_ROWS = (1ll << 31) - 4096;

template <typename T>
struct Vec16 {
  static constexpr int N = 16 / (int)sizeof(T);
};

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }

// VW elements in one access (VW * sizeof(T) is 16, or VW is 1).
template <typename T, int VW>
__device__ __forceinline__ void load_vec(const T* p, float (&v)[VW]) {
  if constexpr (VW == 1) {
    v[0] = to_f(*p);
  } else {
    const uint4 raw = *reinterpret_cast<const uint4*>(p);
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < VW; ++i) v[i] = to_f(e[i]);
  }
}
template <typename T, int VW>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[VW]) {
  if constexpr (VW == 1) {
    *p = from_f<T>(v[0]);
  } else {
    uint4 raw;
    T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int i = 0; i < VW; ++i) e[i] = from_f<T>(v[i]);
    *reinterpret_cast<uint4*>(p) = raw;
  }
}

__device__ __forceinline__ long long read_code(const void* codes, int codes64, long long p) {
  return codes64 ? ((const long long*)codes)[p] : (long long)((const int*)codes)[p];
}

// ---------------------------------------------------------------------------
// Forward.  A CTA owns FWD_CTA_ROWS consecutive rows; their codes and factors
// go through shared memory, and the threads walk the CTA's flat output in
// 16-byte pieces.  ALIGNED: rows are whole 16-byte pieces and both pointers
// are aligned, so a piece is one load; otherwise a piece may cross rows and
// is gathered element by element (the rows come from L1/L2), while its store
// still is one when the output is aligned.
// ---------------------------------------------------------------------------
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(THREADS) codebook_gather_kernel(const gsb_codebook_args a, int out_aligned) {
  constexpr int VW = Vec16<T>::N;
  __shared__ int s_code[FWD_CTA_ROWS];
  __shared__ float s_scale[FWD_CTA_ROWS];
  const long long base = (long long)blockIdx.x * FWD_CTA_ROWS;
  const int rows = (int)min((long long)FWD_CTA_ROWS, a.P - base);
  const int tid = threadIdx.x;
  if (tid < rows) {
    const long long c = read_code(a.codes, a.codes64, base + tid);
    const bool ok = c >= 0 && c < a.K;
    if (c < -1 || c >= a.K) atomicOr((unsigned long long*)a.error_word, (unsigned long long)ERR_BAD_CODE);
    s_code[tid] = ok ? (int)c : -1;
    s_scale[tid] = a.gain ? a.scale * a.gain[base + tid] : a.scale;
  }
  __syncthreads();
  const T* table = (const T*)a.table;
  T* out = (T*)a.out + base * a.D;
  const unsigned D = (unsigned)a.D;
  const unsigned total = (unsigned)rows * D;
  for (unsigned e = (unsigned)tid * VW; e < total; e += THREADS * VW) {
    unsigned r = e / D, col = e - r * D;
    float v[VW];
    if constexpr (ALIGNED) {
      const int c = s_code[r];
      if (c >= 0) {
        load_vec<T, VW>(table + (long long)c * D + col, v);
        const float s = s_scale[r];
#pragma unroll
        for (int i = 0; i < VW; ++i) v[i] *= s;
      } else {
#pragma unroll
        for (int i = 0; i < VW; ++i) v[i] = 0.f;
      }
      store_vec<T, VW>(out + e, v);
    } else {
#pragma unroll
      for (int i = 0; i < VW; ++i) {
        v[i] = 0.f;
        if (e + i < total) {
          const int c = s_code[r];
          if (c >= 0) v[i] = s_scale[r] * to_f(table[(long long)c * D + col]);
        }
        if (++col == D) {
          col = 0;
          ++r;
          if (r >= (unsigned)rows) r = rows - 1;
        }
      }
      if (out_aligned && e + VW <= total) {
        store_vec<T, VW>(out + e, v);
      } else {
#pragma unroll
        for (int i = 0; i < VW; ++i)
          if (e + i < total) out[e + i] = from_f<T>(v[i]);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Backward, step 1: sort keys.  Rows without a code get key K, behind every
// code.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(THREADS) code_keys_kernel(const void* codes, int codes64, int P, unsigned K,
                                                            unsigned* __restrict__ keys,
                                                            unsigned* __restrict__ ids) {
  const int p = blockIdx.x * THREADS + threadIdx.x;
  if (p >= P) return;
  const long long c = read_code(codes, codes64, p);
  keys[p] = c >= 0 && c < (long long)K ? (unsigned)c : K;
  ids[p] = (unsigned)p;
}

// ---------------------------------------------------------------------------
// Backward, step 2: sums of runs of equal keys.  A group of `1 << gshift`
// lanes covers a row (or a column block of it, blockIdx.y) in NV pieces of VW
// elements per lane and owns `len` consecutive sorted positions.
//   level 0: position i is the row ids[i] of grad_out, times its factor;
//   above:   position i is row i of the fp32 partial sums below.
// Partial rows of a chunk: 2c is the run that enters from the left, 2c + 1
// the one that leaves to the right; a run that does both is (sum, zero) with
// both keys set, so equal keys stay neighbours.
// ---------------------------------------------------------------------------
struct SegArgs {
  const unsigned* keys;
  const unsigned* ids;     // level 0
  const void* rows;        // grad_out (level 0) or fp32 partial rows
  const float* gain;       // level 0, optional
  float scale;
  const void* table;       // with grad_gain
  float* grad_gain;        // level 0, optional
  void* grad_table;
  unsigned* out_keys;      // 2 per chunk
  float* out_rows;         // 2 per chunk, D floats each
  int n, len, chunks, D, gshift;
  unsigned K;
};

template <typename T, typename R, int VW, int NV, bool LEVEL0, bool DGAIN>
__global__ void __launch_bounds__(THREADS) segment_sum_kernel(const SegArgs a) {
  const int G = 1 << a.gshift;
  const int lane = threadIdx.x & (G - 1);
  const long long chunk = ((long long)blockIdx.x * THREADS + threadIdx.x) >> a.gshift;
  const int col0 = blockIdx.y * (G * NV * VW);
  const bool live = chunk < a.chunks;
  const long long start = live ? chunk * a.len : 0;
  const long long end = live ? min(start + (long long)a.len, (long long)a.n) : 0;
  const R* rows = (const R*)a.rows;
  const T* table = (const T*)a.table;
  T* grad_table = (T*)a.grad_table;
  const unsigned K = a.K;
  const unsigned before = live && start > 0 ? a.keys[start - 1] : K;
  const unsigned after = live && end < a.n ? a.keys[end] : K;

  int col[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    col[j] = col0 + (j * G + lane) * VW;
    if (col[j] >= a.D) col[j] = -1;
  }
  float acc[NV][VW], trow[NV][VW];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < VW; ++i) acc[j][i] = trow[j][i] = 0.f;
  unsigned cur = K;
  bool first_run = true;  // the run that began at `start`
  unsigned left_key = K, right_key = K;

  auto put_partial = [&](int side, bool zero) {
    float* dst = a.out_rows + (2 * chunk + side) * a.D;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (col[j] >= 0) {
        float v[VW];
#pragma unroll
        for (int i = 0; i < VW; ++i) v[i] = zero ? 0.f : acc[j][i];
#pragma unroll
        for (int i = 0; i < VW; ++i) dst[col[j] + i] = v[i];
      }
  };
  auto flush = [&](bool at_end) {
    if (cur == K) return;
    const bool from_left = first_run && before == cur;
    const bool to_right = at_end && after == cur;
    if (from_left) {
      put_partial(0, false);
      left_key = cur;
      if (to_right) {
        put_partial(1, true);
        right_key = cur;
      }
    } else if (to_right) {
      put_partial(1, false);
      right_key = cur;
    } else {
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (col[j] >= 0) store_vec<T, VW>(grad_table + (long long)cur * a.D + col[j], acc[j]);
    }
  };

  for (int off = 0; off < a.len; off += SEG_UNROLL) {
    unsigned key[SEG_UNROLL], id[SEG_UNROLL];
    float s[SEG_UNROLL], v[SEG_UNROLL][NV][VW];
#pragma unroll
    for (int u = 0; u < SEG_UNROLL; ++u) {
      const long long pos = start + off + u;
      key[u] = pos < end ? a.keys[pos] : K;
      id[u] = LEVEL0 ? (pos < end ? a.ids[pos] : 0u) : (unsigned)pos;
    }
#pragma unroll
    for (int u = 0; u < SEG_UNROLL; ++u) {
      s[u] = 1.f;
      if (LEVEL0) s[u] = a.gain && key[u] != K ? a.scale * a.gain[id[u]] : a.scale;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
#pragma unroll
        for (int i = 0; i < VW; ++i) v[u][j][i] = 0.f;
        if (key[u] != K && col[j] >= 0) load_vec<R, VW>(rows + (long long)id[u] * a.D + col[j], v[u][j]);
      }
    }
#pragma unroll
    for (int u = 0; u < SEG_UNROLL; ++u) {
      const bool valid = start + off + u < end;
      if (valid && key[u] != cur) {
        flush(false);
        if (off + u > 0) first_run = false;
        cur = key[u];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
#pragma unroll
          for (int i = 0; i < VW; ++i) acc[j][i] = trow[j][i] = 0.f;
          if (DGAIN && cur != K && col[j] >= 0) load_vec<T, VW>(table + (long long)cur * a.D + col[j], trow[j]);
        }
      }
      if (DGAIN) {
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < VW; ++i) dot += v[u][j][i] * trow[j][i];
        __syncwarp();
        for (int o = G >> 1; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
        if (valid && lane == 0) a.grad_gain[id[u]] = key[u] != K ? a.scale * dot : 0.f;
      }
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < VW; ++i) acc[j][i] += s[u] * v[u][j][i];
    }
  }
  flush(true);
  if (live && a.out_keys && lane == 0 && blockIdx.y == 0) {
    a.out_keys[2 * chunk] = left_key;
    a.out_keys[2 * chunk + 1] = right_key;
  }
}

// dgain alone, or for rows wider than one group covers: a warp per row.
template <typename T>
__global__ void __launch_bounds__(THREADS) gain_dot_kernel(const gsb_codebook_args a) {
  const long long p = ((long long)blockIdx.x * THREADS + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (p >= a.P) return;
  const long long c = read_code(a.codes, a.codes64, p);
  float dot = 0.f;
  if (c >= 0 && c < a.K) {
    const T* g = (const T*)a.grad_out + p * a.D;
    const T* t = (const T*)a.table + c * a.D;
    for (int d = lane; d < a.D; d += 32) dot += to_f(g[d]) * to_f(t[d]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
  if (lane == 0) a.grad_gain[p] = a.scale * dot;
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------
// Chunk length of level 0: long chunks leave few partial rows to write and
// read again, short ones keep enough groups in flight when there are few rows.
inline int level0_len(long long P) { return P >= (1 << 20) ? 128 : 32; }
constexpr int UPPER_LEN = 32;

inline long long chunks_of(long long n, int len) { return (n + len - 1) / len; }

inline int bits_for(long long max_key) {
  int b = 1;
  while ((max_key >> b) != 0) ++b;
  return b;
}

struct Shape {
  int vw, nv, gshift, col_blocks;
};

// Lanes and pieces that cover a row with the least waste.
inline Shape pick_shape(int D, int vw) {
  const int pieces = (D + vw - 1) / vw;
  Shape best{vw, 4, 5, 0};
  int best_slots = 1 << 30;
  for (int g = 0; g <= 5; ++g)
    for (int nv = 1; nv <= 4; ++nv) {
      const int slots = nv << g;
      if (slots >= pieces && slots <= best_slots) {  // ties: more lanes, fewer pieces
        best = Shape{vw, nv, g, 1};
        best_slots = slots;
      }
    }
  if (best.col_blocks == 0) best.col_blocks = (pieces + 127) / 128;
  return best;
}

template <typename T, typename R, int VW, bool LEVEL0, bool DGAIN>
void launch_seg(const SegArgs& a, const Shape& sh, cudaStream_t s) {
  const long long threads = (long long)a.chunks << sh.gshift;
  const dim3 grid((unsigned)((threads + THREADS - 1) / THREADS), sh.col_blocks);
  switch (sh.nv) {
    case 1: segment_sum_kernel<T, R, VW, 1, LEVEL0, DGAIN><<<grid, THREADS, 0, s>>>(a); break;
    case 2: segment_sum_kernel<T, R, VW, 2, LEVEL0, DGAIN><<<grid, THREADS, 0, s>>>(a); break;
    case 3: segment_sum_kernel<T, R, VW, 3, LEVEL0, DGAIN><<<grid, THREADS, 0, s>>>(a); break;
    default: segment_sum_kernel<T, R, VW, 4, LEVEL0, DGAIN><<<grid, THREADS, 0, s>>>(a); break;
  }
}

struct Workspace {
  unsigned* keys[2];
  unsigned* ids[2];
  void* sort;
  unsigned* part_keys[2];
  float* part_rows[2];
  size_t bytes;
};

inline Workspace carve(void* base, long long P, long long K, int D) {
  Workspace w;
  char* p = (char*)(((uintptr_t)base + 255) & ~(uintptr_t)255);
  char* start = p;
  auto take = [&](size_t b) {
    char* q = p;
    p += (b + 255) & ~(size_t)255;
    return (void*)q;
  };
  for (int i = 0; i < 2; ++i) w.keys[i] = (unsigned*)take((size_t)P * 4);
  for (int i = 0; i < 2; ++i) w.ids[i] = (unsigned*)take((size_t)P * 4);
  w.sort = take(radix::scratch_bytes(P, radix::passes_for_bits(bits_for(K))));
  long long n = 2 * chunks_of(P, level0_len(P));
  for (int i = 0; i < 2; ++i) {
    w.part_keys[i] = (unsigned*)take((size_t)n * 4);
    w.part_rows[i] = (float*)take((size_t)n * D * 4);
    n = 2 * chunks_of(n, UPPER_LEN);
  }
  w.bytes = (size_t)(p - start) + 256;
  return w;
}

template <typename T>
int run_bwd(const gsb_codebook_args* a, cudaStream_t s) {
  constexpr int VW = Vec16<T>::N;
  const long long P = a->P;
  const bool aligned = (long long)a->D * sizeof(T) % 16 == 0 && (uintptr_t)a->grad_out % 16 == 0 &&
                       (uintptr_t)a->table % 16 == 0 && (uintptr_t)a->grad_table % 16 == 0;
  const Shape sh = pick_shape(a->D, aligned ? VW : 1);
  const bool fused_gain = a->grad_gain && a->grad_table && sh.col_blocks == 1;
  if (a->grad_gain && !fused_gain && P > 0)
    gain_dot_kernel<T><<<div_up(P * 32, THREADS), THREADS, 0, s>>>(*a);
  if (!a->grad_table) return check_launch("gsb_codebook_bwd");
  cudaMemsetAsync(a->grad_table, 0, (size_t)a->K * a->D * sizeof(T), s);
  if (P == 0) return check_launch("gsb_codebook_bwd");

  Workspace w = carve(a->workspace, P, a->K, a->D);
  code_keys_kernel<<<div_up(P, THREADS), THREADS, 0, s>>>(a->codes, a->codes64, (int)P, (unsigned)a->K, w.keys[0],
                                                          w.ids[0]);
  const int where = radix::sort_pairs(w.keys, w.ids, P, nullptr, bits_for(a->K), w.sort, a->error_word, s, nullptr,
                                      0, true);
  SegArgs g{};
  g.keys = w.keys[where];
  g.ids = w.ids[where];
  g.rows = a->grad_out;
  g.gain = a->gain;
  g.scale = a->scale;
  g.table = a->table;
  g.grad_gain = fused_gain ? a->grad_gain : nullptr;
  g.grad_table = a->grad_table;
  g.n = (int)P;
  g.len = level0_len(P);
  g.chunks = (int)chunks_of(P, g.len);
  g.D = a->D;
  g.gshift = sh.gshift;
  g.K = (unsigned)a->K;
  for (int level = 0;; ++level) {
    const bool more = g.chunks > 1;
    g.out_keys = more ? w.part_keys[level & 1] : nullptr;
    g.out_rows = more ? w.part_rows[level & 1] : nullptr;
    if (level == 0) {
      if (aligned) {
        if (fused_gain) launch_seg<T, T, VW, true, true>(g, sh, s);
        else launch_seg<T, T, VW, true, false>(g, sh, s);
      } else {
        if (fused_gain) launch_seg<T, T, 1, true, true>(g, sh, s);
        else launch_seg<T, T, 1, true, false>(g, sh, s);
      }
    } else {
      const Shape up = pick_shape(a->D, 1);
      g.gshift = up.gshift;
      launch_seg<T, float, 1, false, false>(g, up, s);
    }
    if (!more) break;
    g.keys = g.out_keys;
    g.rows = g.out_rows;
    g.grad_gain = nullptr;
    g.gain = nullptr;
    g.n = 2 * g.chunks;
    g.len = UPPER_LEN;
    g.chunks = (int)chunks_of(g.n, g.len);
  }
  return check_launch("gsb_codebook_bwd");
}

template <typename T>
int run_fwd(const gsb_codebook_args* a, cudaStream_t s) {
  const bool out_aligned = (uintptr_t)a->out % 16 == 0;
  const bool aligned = out_aligned && (long long)a->D * sizeof(T) % 16 == 0 && (uintptr_t)a->table % 16 == 0;
  const int blocks = div_up(a->P, FWD_CTA_ROWS);
  if (aligned) codebook_gather_kernel<T, true><<<blocks, THREADS, 0, s>>>(*a, 1);
  else codebook_gather_kernel<T, false><<<blocks, THREADS, 0, s>>>(*a, out_aligned);
  return check_launch("gsb_codebook_fwd");
}

int check_args(const gsb_codebook_args* a, const char* what) {
  if (!a) {
    set_error("%s: null arguments", what);
    return GSB_ERR_INVALID;
  }
  if (a->P < 0 || a->P >= MAX_ROWS || a->K < 0 || a->K >= (1ll << 31) - 1 || a->D < 1 || a->D > (1 << 24)) {
    set_error("%s: sizes out of range (P %lld, K %lld, D %d)", what, a->P, a->K, a->D);
    return GSB_ERR_INVALID;
  }
  if (a->dtype < GSB_TYPE_FP32 || a->dtype > GSB_TYPE_FP16) {
    set_error("%s: unknown dtype %d", what, a->dtype);
    return GSB_ERR_INVALID;
  }
  if (a->P > 0 && (!a->codes || !a->error_word || (a->K > 0 && !a->table))) {
    set_error("%s: null pointer", what);
    return GSB_ERR_INVALID;
  }
  return GSB_OK;
}

}  // namespace
}  // namespace gsb

GSB_EXPORT int gsb_codebook_fwd(const gsb_codebook_args* a, void* stream) {
  using namespace gsb;
  const int st = check_args(a, "gsb_codebook_fwd");
  if (st != GSB_OK) return st;
  if (a->P == 0) return GSB_OK;
  if (!a->out) {
    set_error("gsb_codebook_fwd: null pointer");
    return GSB_ERR_INVALID;
  }
  cudaStream_t s = (cudaStream_t)stream;
  switch (a->dtype) {
    case GSB_TYPE_BF16: return run_fwd<__nv_bfloat16>(a, s);
    case GSB_TYPE_FP16: return run_fwd<__half>(a, s);
    default: return run_fwd<float>(a, s);
  }
}

GSB_EXPORT size_t gsb_codebook_bwd_workspace_bytes(long long P, long long K, int D) {
  if (P <= 0 || P >= gsb::MAX_ROWS || K < 0 || D < 1) return 256;
  return gsb::carve(nullptr, P, K, D).bytes;
}

GSB_EXPORT int gsb_codebook_bwd(const gsb_codebook_args* a, void* stream) {
  using namespace gsb;
  const int st = check_args(a, "gsb_codebook_bwd");
  if (st != GSB_OK) return st;
  if (a->P > 0 && !a->grad_out) {
    set_error("gsb_codebook_bwd: null pointer");
    return GSB_ERR_INVALID;
  }
  if (a->grad_gain && !a->gain) {
    set_error("gsb_codebook_bwd: grad_gain without gain");
    return GSB_ERR_INVALID;
  }
  if (a->grad_table && a->P > 0 &&
      (!a->workspace || a->workspace_bytes < gsb_codebook_bwd_workspace_bytes(a->P, a->K, a->D))) {
    set_error("gsb_codebook_bwd: workspace too small");
    return GSB_ERR_INVALID;
  }
  cudaStream_t s = (cudaStream_t)stream;
  switch (a->dtype) {
    case GSB_TYPE_BF16: return run_bwd<__nv_bfloat16>(a, s);
    case GSB_TYPE_FP16: return run_bwd<__half>(a, s);
    default: return run_bwd<float>(a, s);
  }
}
