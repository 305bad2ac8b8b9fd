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
// one read of g; the sums go by code instead of atomics, so that they have one
// order (the same bits on every call) and no hot row serializes.
//
// Many rows: the codes are sorted (radix_sort.cuh's passes over the key bits
// of K), the sorted positions are cut into chunks of equal length, and one
// group of lanes sums each chunk's runs in registers in fp32.  A run that lies
// inside its chunk is stored at once; the at most two that cross a chunk's
// ends leave fp32 partial rows.  A CTA whose chunks all lie in one run adds
// theirs up at its end; a second kernel adds up the rest, a warp for each run
// that crosses chunks (a CTA for the longest), so that one code may have most
// of the rows (6M x 48 fp32, 16,384 codes, times of the gradient: codes spread
// 442 us, 60% in one 446, all in two 395).  Few rows or codes: teams of warps
// scan all the codes for the ones they own, in one launch.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "gsb_common.cuh"
#include "radix_sort.cuh"

namespace gsb {
namespace {

constexpr int THREADS = launch::CODEBOOK;
constexpr long long MAX_ROWS = (1ll << 31) - 4096;
constexpr int MAX_COLS = 1 << 22;   // 65,535 column blocks of 128 or more

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

// The same, held as it is read.
template <typename T, int VW>
struct Piece {
  uint4 raw;
  __device__ __forceinline__ void load(const T* p) { raw = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void zero() { raw = make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ float operator[](int i) const { return to_f(reinterpret_cast<const T*>(&raw)[i]); }
};
template <typename T>
struct Piece<T, 1> {
  float x;
  __device__ __forceinline__ void load(const T* p) { x = to_f(*p); }
  __device__ __forceinline__ void zero() { x = 0.f; }
  __device__ __forceinline__ float operator[](int) const { return x; }
};

__device__ __forceinline__ long long read_code(const void* codes, int codes64, long long p) {
  return codes64 ? ((const long long*)codes)[p] : (long long)((const int*)codes)[p];
}

// ---------------------------------------------------------------------------
// Forward.  A CTA owns ROWS consecutive rows (a multiple of 16, which keeps
// CTAs 16-byte aligned); their codes and factors go through shared memory, and
// the threads walk the CTA's flat output in 16-byte pieces.
// ALIGNED: rows are whole 16-byte pieces and both pointers are aligned, so a
// piece is one load; otherwise a piece may cross rows and is gathered element
// by element (the rows come from L1/L2), while its store still is one when the
// output is aligned.
// ---------------------------------------------------------------------------
template <typename T, bool ALIGNED, int ROWS>
__global__ void __launch_bounds__(THREADS) codebook_gather_kernel(const gsb_codebook_args a, int out_aligned,
                                                                  unsigned magic) {
  constexpr int VW = Vec16<T>::N;
  constexpr int UNROLL = ALIGNED ? 1 : 2;
  __shared__ int s_code[ROWS];
  __shared__ float s_scale[ROWS];
  const long long base = (long long)blockIdx.x * ROWS;
  const int rows = (int)min((long long)ROWS, a.P - base);
  const int tid = threadIdx.x;
  for (int i = tid; i < rows; i += THREADS) {
    const long long c = read_code(a.codes, a.codes64, base + i);
    const bool ok = c >= 0 && c < a.K;
    if (c < -1 || c >= a.K) atomicOr((unsigned long long*)a.error_word, (unsigned long long)ERR_BAD_CODE);
    s_code[i] = ok ? (int)c : -1;
    // a row without a code is zero, whatever its gain holds
    s_scale[i] = !ok ? 0.f : a.gain ? a.scale * a.gain[base + i] : a.scale;
  }
  __syncthreads();
  const T* table = (const T*)a.table;
  T* out = (T*)a.out + base * a.D;
  const unsigned D = (unsigned)a.D;
  const unsigned total = (unsigned)rows * D;
  for (unsigned e0 = (unsigned)tid * VW; e0 < total; e0 += THREADS * VW * UNROLL) {
    float v[UNROLL][VW], s[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const unsigned e = e0 + u * (THREADS * VW);
      s[u] = 1.f;
#pragma unroll
      for (int i = 0; i < VW; ++i) v[u][i] = 0.f;
      if (e >= total) continue;
      unsigned r = magic ? __umulhi(e, magic) : e / D, col = e - r * D;
      if constexpr (ALIGNED) {
        const int c = s_code[r];
        s[u] = s_scale[r];
        if (c >= 0) load_vec<T, VW>(table + (long long)c * D + col, v[u]);
      } else if (D >= VW) {
        // at most one row ends inside the piece
        const unsigned r1 = min(r + 1, (unsigned)rows - 1);
        const int c0 = s_code[r], c1 = s_code[r1];
        const float f0 = s_scale[r], f1 = s_scale[r1];
        const T* p0 = table + (long long)c0 * D + col;
        const T* p1 = table + (long long)c1 * D + col - D;
#pragma unroll
        for (int i = 0; i < VW; ++i) {
          const bool next = col + i >= D;
          if ((next ? c1 : c0) >= 0 && e + i < total) v[u][i] = (next ? f1 : f0) * to_f((next ? p1 : p0)[i]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < VW; ++i) {
          if (e + i < total) {
            const int c = s_code[r];
            if (c >= 0) v[u][i] = s_scale[r] * to_f(table[(long long)c * D + col]);
          }
          if (++col == D) {
            col = 0;
            r = min(r + 1, (unsigned)rows - 1);
          }
        }
      }
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const unsigned e = e0 + u * (THREADS * VW);
      if (e >= total) continue;
      if constexpr (ALIGNED) {
#pragma unroll
        for (int i = 0; i < VW; ++i) v[u][i] *= s[u];
      }
      if (ALIGNED || (out_aligned && e + VW <= total)) {
        store_vec<T, VW>(out + e, v[u]);
      } else {
#pragma unroll
        for (int i = 0; i < VW; ++i)
          if (e + i < total) out[e + i] = from_f<T>(v[u][i]);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Backward of few rows, in one scan of all the codes.
// A team of `wpc` warps of a CTA takes a code; each warp scans its part of the
// codes, keeps the rows it finds in a queue and adds them up from there in
// order, a batch at a time: 32 >> gshift rows side by side in groups of lanes,
// UNROLL of them in flight per group, so that a code that most rows have is
// bound by loads in flight and not by one latency per row.  The groups' and
// then the warps' sums are added in a fixed order.
// BY_ROW false (few codes): one team per code.  One more "code" takes the rows
// without one (their gains' gradient is zero).
// BY_ROW true (very few rows): a team takes the code of one row and gives up if
// an earlier row has the same one; the first row's team adds them all.
// ---------------------------------------------------------------------------
constexpr int SCAN_COLS = 128;    // columns that a CTA sums
constexpr int SCAN_QUEUE = 256;   // below a batch (at most 128 rows), and 128 rows more
__host__ __device__ constexpr int scan_unroll(int vw, int nv) { return vw == 1 && nv == 1 ? 8 : 4; }
constexpr size_t scan_smem(int warps) { return (size_t)warps * (SCAN_COLS * 4 + SCAN_QUEUE * 2); }

// A lane's pieces of a row: NV of VW elements.
template <typename T, int VW, int NV, bool BY_ROW, bool DGAIN>
__global__ void __launch_bounds__(1024) code_scan_kernel(const gsb_codebook_args a, int wpc, int gshift) {
  constexpr int UNROLL = scan_unroll(VW, NV);
  extern __shared__ __align__(16) uint8_t scan_shared[];
  __shared__ int s_earlier[32];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, warps = blockDim.x / 32;
  float* const sums = reinterpret_cast<float*>(scan_shared) + warp * SCAN_COLS;
  // rows are below 2^14
  unsigned short* const queue =
      reinterpret_cast<unsigned short*>(scan_shared + (size_t)warps * SCAN_COLS * 4) + warp * SCAN_QUEUE;
  const int team = warp / wpc, part = warp % wpc;
  const int G = 1 << gshift, groups = 32 >> gshift, sub = lane >> gshift;
  const int P = (int)a.P, K = (int)a.K;
  const long long index = (long long)blockIdx.x * (warps / wpc) + team;  // a code, or a row
  auto code_of = [&](int p) {
    const long long c = read_code(a.codes, a.codes64, p);
    return c < 0 || c >= K ? K : (int)c;
  };
  int code = -1;  // none: nothing to do
  if (BY_ROW) {
    if (threadIdx.x < 32) s_earlier[threadIdx.x] = 0;
    __syncthreads();
    if (index < P) code = code_of((int)index);
    if (code == K) {
      if (DGAIN && blockIdx.y == 0 && part == 0 && lane == 0) a.grad_gain[index] = 0.f;
      code = -1;
    }
    if (code >= 0) {
      for (int p0 = part * 128; p0 < index; p0 += wpc * 128) {
        bool same = false;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int p = p0 + 32 * u + lane;
          same |= p < index && code_of(p) == code;
        }
        if (same) s_earlier[team] = 1;
        if (__any_sync(0xffffffffu, same || *(volatile int*)&s_earlier[team])) break;
      }
    }
    __syncthreads();
    if (s_earlier[team]) code = -1;
  } else if (index <= K) {
    code = (int)index;
  }

  const int first = BY_ROW ? (int)index : 0;  // no row before it has the code
  const int lo = first + (int)((long long)(P - first) * part / wpc);
  const int hi = code < 0 ? lo : first + (int)((long long)(P - first) * (part + 1) / wpc);
  const int c0 = blockIdx.y * SCAN_COLS + (lane & (G - 1)) * VW;  // and 32 further on, where NV is not 1 (G is 32)
  const T* const grad = (const T*)a.grad_out + c0;
  float acc[NV][VW], trow[NV][VW];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
#pragma unroll
    for (int i = 0; i < VW; ++i) acc[j][i] = trow[j][i] = 0.f;
    if (DGAIN && code >= 0 && code < K && c0 + 32 * j < a.D)
      load_vec<T, VW>((const T*)a.table + (long long)code * a.D + c0 + 32 * j, trow[j]);
  }
  const int batch = groups * UNROLL;
  // rows queue[from .. from + n - 1], n at most a batch
  auto drain = [&](int from, int n) {
    int r[UNROLL];
    float s[UNROLL], sum[NV][VW];  // a batch's sum of its own: shorter chains of additions
    Piece<T, VW> v[UNROLL][NV];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int i = u * groups + sub;
      r[u] = i < n ? queue[from + i] : -1;
      s[u] = r[u] < 0 ? 0.f : a.gain ? a.scale * a.gain[r[u]] : a.scale;
      const T* const row = grad + (long long)r[u] * a.D;
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (r[u] >= 0 && c0 + 32 * j < a.D) v[u][j].load(row + 32 * j);
        else v[u][j].zero();
    }
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < VW; ++i) sum[j][i] = 0.f;
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      float dot = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < VW; ++i) {
          const float x = v[u][j][i];
          sum[j][i] += s[u] * x;
          if (DGAIN) dot += x * trow[j][i];
        }
      if (DGAIN) {
        for (int o = G >> 1; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
        if (r[u] >= 0 && (lane & (G - 1)) == 0) a.grad_gain[r[u]] = a.scale * dot;
      }
    }
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < VW; ++i) acc[j][i] += sum[j][i];
  };
  // four codes per lane, read a round ahead: the words as they are, so that nothing waits for them yet
  int next_lo[4], next_hi[4];
  auto fetch = [&](int p0) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int p = p0 + 32 * u + lane;
      next_lo[u] = -1, next_hi[u] = -1;
      if (p < hi) {
        if (a.codes64) {
          const int2 w = ((const int2*)a.codes)[p];
          next_lo[u] = w.x, next_hi[u] = w.y;
        } else {
          next_lo[u] = ((const int*)a.codes)[p], next_hi[u] = 0;
        }
      }
    }
  };
  fetch(lo);
  int queued = 0;
  for (int p0 = lo;; p0 += 32 * 4) {
    const bool end = p0 >= hi;
    if (!end) {
      int c[4], high[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) c[u] = next_lo[u], high[u] = next_hi[u];
      fetch(p0 + 32 * 4);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int p = p0 + 32 * u + lane;
        if (code == K) {
          if (DGAIN && blockIdx.y == 0 && p < hi && (high[u] != 0 || (unsigned)c[u] >= (unsigned)K)) a.grad_gain[p] = 0.f;
          continue;
        }
        const bool mine = c[u] == code && high[u] == 0;
        const unsigned hits = __ballot_sync(0xffffffffu, mine);
        if (!hits) continue;
        if (mine) queue[queued + __popc(hits & ((1u << lane) - 1u))] = (unsigned short)p;
        queued += __popc(hits);
      }
      if (queued < batch) continue;
    }
    __syncwarp();
    int from = 0;
    for (; queued - from >= (end ? 1 : batch); from += batch) drain(from, min(batch, queued - from));
    if (end) break;
    // what is left, less than a batch, goes to the front
    queued -= from;
    unsigned short left[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) left[u] = lane + 32 * u < queued ? queue[from + lane + 32 * u] : 0;
    __syncwarp();
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (lane + 32 * u < queued) queue[lane + 32 * u] = left[u];
  }
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < VW; ++i) {
      for (int o = G; o < 32; o <<= 1) acc[j][i] += __shfl_xor_sync(0xffffffffu, acc[j][i], o);
      if (sub == 0) sums[(lane & (G - 1)) * VW + i + 32 * j] = acc[j][i];
    }
  __syncthreads();
  if (part != 0 || code < 0 || code >= K) return;
  for (int c = lane; c < SCAN_COLS && blockIdx.y * SCAN_COLS + c < a.D; c += 32) {
    float sum = sums[c];
    for (int w = 1; w < wpc; ++w) sum += sums[w * SCAN_COLS + c];
    ((T*)a.grad_table)[(long long)code * a.D + blockIdx.y * SCAN_COLS + c] = from_f<T>(sum);
  }
}

// ---------------------------------------------------------------------------
// Backward of many rows, step 1: sort keys, the histograms of their digits,
// and a zero gradient (codes that no row has keep it).  Rows without a code
// take some key and are marked in their id, so that K codes need no more key
// bits.
// ---------------------------------------------------------------------------
constexpr unsigned SKIP = 1u << 31;

__global__ void __launch_bounds__(THREADS) code_keys_kernel(const void* codes, int codes64, int P, unsigned K,
                                                            int passes, unsigned last_mask,
                                                            unsigned* __restrict__ keys, unsigned* __restrict__ ids,
                                                            unsigned* __restrict__ hist, uint4* __restrict__ zero,
                                                            long long zero_vecs, uint8_t* __restrict__ zero_tail,
                                                            int zero_bytes) {
  __shared__ unsigned s_hist[radix::MAX_PASSES][radix::RADIX];
  for (int i = threadIdx.x; i < passes * radix::RADIX; i += THREADS) (&s_hist[0][0])[i] = 0u;
  __syncthreads();
  const int stride = gridDim.x * THREADS, first = blockIdx.x * THREADS + threadIdx.x;
  for (long long i = first; i < zero_vecs; i += stride) zero[i] = make_uint4(0u, 0u, 0u, 0u);
  if (first < zero_bytes) zero_tail[first] = 0;
  for (long long p = first; p < P; p += stride) {
    const long long c = read_code(codes, codes64, p);
    const bool ok = c >= 0 && c < (long long)K;
    // rows without a code are spread over the keys: one long run would be summed for nothing
    const unsigned key = ok ? (unsigned)c : (unsigned)p % K;
    keys[p] = key;
    ids[p] = ok ? (unsigned)p : (unsigned)p | SKIP;
    for (int q = 0; q < passes; ++q)
      atomicAdd(&s_hist[q][(key >> (q * radix::RADIX_BITS)) & (q == passes - 1 ? last_mask : radix::RADIX - 1)], 1u);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < passes * radix::RADIX; i += THREADS) {
    const unsigned c = (&s_hist[0][0])[i];
    if (c) atomicAdd(&hist[i], c);
  }
}

// ---------------------------------------------------------------------------
// Step 2: sums of runs of equal keys.  A group of `1 << gshift` lanes covers a
// row (or a column block of it, blockIdx.y) in NV pieces of VW elements per
// lane and owns `len` consecutive sorted positions.  The run that enters a
// chunk from the left leaves its partial row at 2c, the one that leaves to the
// right at 2c + 1 (a run that does both: its sum at 2c, both keys set).
// ---------------------------------------------------------------------------
constexpr unsigned NONE = 0xffffffffu;
constexpr int LONG_RUN = 8;  // chunks

struct SegArgs {
  const unsigned* keys;
  const unsigned* ids;
  const void* rows;        // grad_out
  const float* gain;       // optional
  float scale;
  const void* table;       // with grad_gain
  float* grad_gain;        // optional
  void* grad_table;
  unsigned* part_keys;     // 2 per chunk
  float* part_rows;        // 2 per chunk, D floats each
  int n, len, chunks, D, gshift;
};

template <typename T, int VW, int NV, bool DGAIN>
__global__ void __launch_bounds__(THREADS) segment_sum_kernel(const SegArgs a) {
  // Rows in flight: registers against occupancy (300,000 x 77 fp16 40 us with 2, 52 with 4; 1M x 48 bf16 56 and 65;
  // 300,000 x 77 fp32 37 and 33; 6M x 48 fp32 with gains 433 and 411, 577 with 8).
  constexpr int SEG_UNROLL = sizeof(T) == 2 ? 2 : 4;
  const int G = 1 << a.gshift;
  const int lane = threadIdx.x & (G - 1);
  const long long chunk = ((long long)blockIdx.x * THREADS + threadIdx.x) >> a.gshift;
  const int col0 = blockIdx.y * (G * NV * VW);
  const bool live = chunk < a.chunks;
  const long long start = live ? chunk * a.len : 0;
  const long long end = live ? min(start + (long long)a.len, (long long)a.n) : 0;
  const T* rows = (const T*)a.rows;
  const T* table = (const T*)a.table;
  T* grad_table = (T*)a.grad_table;
  const unsigned before = live && start > 0 ? a.keys[start - 1] : NONE;
  const unsigned after = live && end < a.n ? a.keys[end] : NONE;

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
  unsigned cur = NONE;
  bool first_run = true;  // the run that began at `start`
  unsigned left_key = NONE, right_key = NONE;

  auto flush = [&](bool at_end) {
    if (cur == NONE) return;
    const bool from_left = first_run && before == cur, to_right = at_end && after == cur;
    if (from_left) left_key = cur;
    if (to_right) right_key = cur;
    if (from_left || to_right) {
      float* dst = a.part_rows + (2 * chunk + (from_left ? 0 : 1)) * a.D;
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (col[j] >= 0) {
#pragma unroll
          for (int i = 0; i < VW; ++i) dst[col[j] + i] = acc[j][i];
        }
    } else {
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (col[j] >= 0) store_vec<T, VW>(grad_table + (long long)cur * a.D + col[j], acc[j]);
    }
  };
  // keys and ids are read one round ahead of the rows that they name
  unsigned next_key[SEG_UNROLL], next_id[SEG_UNROLL];
  auto fetch = [&](long long pos) {
#pragma unroll
    for (int u = 0; u < SEG_UNROLL; ++u) {
      next_key[u] = pos + u < end ? a.keys[pos + u] : NONE;
      next_id[u] = pos + u < end ? a.ids[pos + u] : SKIP;
    }
  };
  fetch(start);
  for (int off = 0; off < a.len; off += SEG_UNROLL) {
    unsigned key[SEG_UNROLL], id[SEG_UNROLL];
    float s[SEG_UNROLL], v[SEG_UNROLL][NV][VW];
#pragma unroll
    for (int u = 0; u < SEG_UNROLL; ++u) {
      key[u] = next_key[u];
      id[u] = next_id[u];
      // rows without a code and positions past the end add 0, not scale * 0
      s[u] = id[u] & SKIP ? 0.f : a.gain ? a.scale * a.gain[id[u]] : a.scale;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
#pragma unroll
        for (int i = 0; i < VW; ++i) v[u][j][i] = 0.f;
        if (!(id[u] & SKIP) && col[j] >= 0) load_vec<T, VW>(rows + (long long)id[u] * a.D + col[j], v[u][j]);
      }
    }
    if (off + SEG_UNROLL < a.len) fetch(start + off + SEG_UNROLL);
#pragma unroll
    for (int u = 0; u < SEG_UNROLL; ++u) {
      if (key[u] != NONE && key[u] != cur) {
        flush(false);
        if (off + u > 0) first_run = false;
        cur = key[u];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
#pragma unroll
          for (int i = 0; i < VW; ++i) acc[j][i] = 0.f;
          if (DGAIN && col[j] >= 0) load_vec<T, VW>(table + (long long)cur * a.D + col[j], trow[j]);
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
        if (key[u] != NONE && lane == 0) a.grad_gain[id[u] & ~SKIP] = id[u] & SKIP ? 0.f : a.scale * dot;
      }
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < VW; ++i) acc[j][i] += s[u] * v[u][j][i];
    }
  }
  flush(true);
  if (live && a.chunks > 1 && lane == 0 && blockIdx.y == 0) {
    a.part_keys[2 * chunk] = left_key;
    a.part_keys[2 * chunk + 1] = right_key;
  }
  // A CTA whose chunks all lie inside one run adds their sums up, into row 2c + 1 of its first chunk, so that a run of
  // most rows is not one CTA's to join.
  if (a.chunks <= LONG_RUN) return;
  __shared__ unsigned s_key;
  const unsigned inside = left_key == right_key ? left_key : NONE;
  if (threadIdx.x == 0) s_key = inside;
  __syncthreads();
  if (!__syncthreads_and(inside != NONE && inside == s_key)) return;
  const int block = THREADS >> a.gshift, c = col0 + threadIdx.x;
  float* const rows0 = a.part_rows + 2ll * blockIdx.x * block * a.D;
  for (int cc = c; cc < min(a.D, col0 + G * NV * VW); cc += THREADS) {
    float sum = 0.f;
#pragma unroll 8
    for (int k = 0; k < block; ++k) sum += rows0[2ll * k * a.D + cc];
    rows0[a.D + cc] = sum;
  }
}

// Step 3: the runs that cross chunks.  A warp looks at one chunk; if a run
// starts there and leaves to the right, it adds up that run's partial rows, or
// the sums of whole blocks of them.  Runs of more than LONG_RUN chunks are left
// to the whole CTA, whose warps take every eighth partial row.
template <typename T>
__global__ void __launch_bounds__(THREADS, 8) run_join_kernel(const SegArgs a) {
  constexpr int WARPS = THREADS / 32;
  __shared__ int s_last[WARPS];
  __shared__ float s_sum[WARPS][128];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int first = blockIdx.x * WARPS;
  const int mine = first + warp;
  int last = -1;  // the run's last chunk
  if (mine < a.chunks) {
    const unsigned key = a.part_keys[2 * mine + 1];
    if (key != NONE && a.part_keys[2 * mine] != key) {
      // the first chunk that the run does not leave: among the next 32, then by 32 probes a round (keys are sorted, and
      // no run leaves the last chunk)
      int from = mine, step = 1;
      last = a.chunks - 1;
      while (last - from > 1) {
        const unsigned stop =
            __ballot_sync(0xffffffffu, a.part_keys[2 * min(from + (lane + 1) * step, last) + 1] != key);
        const int f = stop ? __ffs(stop) - 1 : 32;
        if (stop) last = min(last, from + (f + 1) * step);
        from += f * step;
        step = (last - from + 31) / 32;
      }
    }
  }
  // column c of the partial rows row, row + stride, ..., n of them; every step-th from the from-th on
  auto sum_rows = [&](long long row, int stride, int n, int c, int from, int step) {
    float sum = 0.f;
    if (c < a.D) {
      for (int k = from; k < n; k += 8 * step) {
        float v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int i = k + u * step;
          v[u] = i < n ? a.part_rows[(row + (long long)i * stride) * a.D + c] : 0.f;
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) sum += v[u];
      }
    }
    return sum;
  };
  // a run's rows in chunk order: 2 * start + 1, 2 * (start + 1), 2 * (start + 2), ...
  const bool is_long = last - mine > LONG_RUN && last >= 0;
  if (last >= 0 && !is_long) {
    T* dst = (T*)a.grad_table + (long long)a.part_keys[2 * mine + 1] * a.D;
    for (int c = lane; c < a.D; c += 32)
      dst[c] = from_f<T>(a.part_rows[(2ll * mine + 1) * a.D + c] + sum_rows(2ll * mine + 2, 2, last - mine, c, 0, 1));
  }
  if (lane == 0) s_last[warp] = is_long ? last : -1;
  __syncthreads();
  for (int w = 0; w < WARPS; ++w) {
    const int end = s_last[w];
    if (end < 0) continue;
    T* dst = (T*)a.grad_table + (long long)a.part_keys[2 * (first + w) + 1] * a.D;
    // whole CTAs of the sums after start and before end, and the chunks around them
    const int start = first + w, block = THREADS >> a.gshift;
    const int b0 = start / block + 1, b1 = max(end / block, b0);
    const int head = b1 > b0 ? b0 * block - start - 1 : end - start, tail = b1 > b0 ? end + 1 - b1 * block : 0;
    for (int c0 = 0; c0 < a.D; c0 += 128) {
#pragma unroll 1
      for (int c = lane; c < 128; c += 32) {
        float sum = sum_rows(2ll * start + 1, 1, 1, c0 + c, warp, WARPS);
        sum += sum_rows(2ll * start + 2, 2, head, c0 + c, warp, WARPS);
        sum += sum_rows(2ll * block * b0 + 1, 2 * block, b1 - b0, c0 + c, warp, WARPS);
        sum += sum_rows(2ll * block * b1, 2, tail, c0 + c, warp, WARPS);
        s_sum[warp][c] = sum;
      }
      __syncthreads();
      const int c = threadIdx.x;
      if (c < 128 && c0 + c < a.D) {
        float sum = 0.f;
        for (int k = 0; k < WARPS; ++k) sum += s_sum[k][c];
        dst[c0 + c] = from_f<T>(sum);
      }
      __syncthreads();
    }
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
// Chunk length: long chunks leave few partial rows to write and read again,
// short ones keep enough groups in flight when there are few rows.
inline int chunk_len(long long P) { return P >= (1 << 20) ? 128 : P >= (1 << 19) ? 64 : P >= (1 << 17) ? 32 : 16; }

inline long long chunks_of(long long n, int len) { return (n + len - 1) / len; }

// Bits of the keys 0 .. K - 1.
inline int key_bits(long long K) {
  int b = 1;
  while (((K - 1) >> b) > 0) ++b;
  return b;
}

// The scans.  By code: every code is read K times (from L2), so it stops
// paying once that is tens of microseconds (16,384 x 512 codes x 48 fp32:
// 18 us; the sort's eight launches take 45 and more).  By row: P * P reads at most, whatever
// K is, and a fill of the table's gradient.
// Warps of a team: more while they fit the SMs twice over, for the sake of codes
// that most rows have (16,384 x 48 fp32, 512 codes, 60% in one: 8 warps 111 us,
// 16 63; spread 16 and 18; a single code, 32 warps: 57).
inline int scan_warps(long long P, long long teams) {
  int w = P > 4096 ? 8 : P > 2048 ? 4 : P > 1024 ? 2 : 1;
  while (w < 32 && P > 256 * w && teams * 2 * w <= 148 * 64) w *= 2;
  return w;
}
inline bool scan_by_code(long long P, long long K) { return P <= (1 << 14) && P * K <= (1 << 23); }
inline bool small_case(long long P, long long K) { return P <= (1 << 12) || scan_by_code(P, K); }

struct Shape {
  int vw, nv, gshift, col_blocks;
};

// Lanes and pieces that cover a row with the least waste, of those that hold at
// most 12 elements of a row per lane if there are any.
inline Shape pick_shape(int D, int vw) {
  const int pieces = (D + vw - 1) / vw;
  Shape best{vw, 4, 5, 0};
  int best_slots = 1 << 30;
  for (int g = 0; g <= 5; ++g)
    for (int nv = 1; nv <= 4; ++nv) {
      const int slots = (nv << g) + (nv * vw > 12 ? 1 << 20 : 0);
      if (nv << g >= pieces && slots <= best_slots) {  // ties: more lanes, fewer pieces
        best = Shape{vw, nv, g, 1};
        best_slots = slots;
      }
    }
  if (best.col_blocks == 0) best.col_blocks = (pieces + 127) / 128;
  return best;
}

template <typename T, int VW, bool DGAIN>
void launch_seg(const SegArgs& a, const Shape& sh, cudaStream_t s) {
  const long long threads = (long long)a.chunks << sh.gshift;
  const dim3 grid((unsigned)((threads + THREADS - 1) / THREADS), sh.col_blocks);
  switch (sh.nv) {
    case 1: segment_sum_kernel<T, VW, 1, DGAIN><<<grid, THREADS, 0, s>>>(a); break;
    case 2: segment_sum_kernel<T, VW, 2, DGAIN><<<grid, THREADS, 0, s>>>(a); break;
    case 3: segment_sum_kernel<T, VW, 3, DGAIN><<<grid, THREADS, 0, s>>>(a); break;
    default: segment_sum_kernel<T, VW, 4, DGAIN><<<grid, THREADS, 0, s>>>(a); break;
  }
}

template <typename T, int VW, int NV, bool BY_ROW>
void launch_scan(const gsb_codebook_args& a, long long teams, cudaStream_t s) {
  // lanes that cover a row (of at most SCAN_COLS columns), and few enough rows side by side for the queue
  const int pieces = (std::min(a.D, SCAN_COLS) + VW - 1) / VW;
  int gshift = 0;
  while ((1 << gshift < pieces && gshift < 5) || (32 >> gshift) * scan_unroll(VW, NV) > SCAN_QUEUE / 2) ++gshift;
  const int wpc = scan_warps(a.P, teams), warps = std::max(wpc, 8);
  const dim3 grid(div_up(teams * wpc, warps), div_up(a.D, SCAN_COLS));
  if (a.grad_gain) code_scan_kernel<T, VW, NV, BY_ROW, true><<<grid, warps * 32, scan_smem(warps), s>>>(a, wpc, gshift);
  else code_scan_kernel<T, VW, NV, BY_ROW, false><<<grid, warps * 32, scan_smem(warps), s>>>(a, wpc, gshift);
}
template <typename T, bool BY_ROW>
void launch_scan(const gsb_codebook_args& a, long long teams, bool aligned, cudaStream_t s) {
  if (aligned) launch_scan<T, Vec16<T>::N, 1, BY_ROW>(a, teams, s);
  else if (a.D <= 32) launch_scan<T, 1, 1, BY_ROW>(a, teams, s);
  else launch_scan<T, 1, 4, BY_ROW>(a, teams, s);
}

struct Workspace {
  unsigned* keys[2];
  unsigned* ids[2];
  void* sort;
  unsigned* part_keys;
  float* part_rows;
  size_t bytes;
};

inline Workspace carve(void* base, long long P, long long K, int D) {
  Workspace w{};
  if (small_case(P, K) || K == 0) {
    w.bytes = 0;
    return w;
  }
  char* p = (char*)(((uintptr_t)base + 255) & ~(uintptr_t)255);
  char* start = p;
  auto take = [&](size_t b) {
    char* q = p;
    p += (b + 255) & ~(size_t)255;
    return (void*)q;
  };
  for (int i = 0; i < 2; ++i) w.keys[i] = (unsigned*)take((size_t)P * 4);
  for (int i = 0; i < 2; ++i) w.ids[i] = (unsigned*)take((size_t)P * 4);
  w.sort = take(radix::scratch_bytes(P, radix::passes_for_bits(key_bits(K))));
  const long long n = 2 * chunks_of(P, chunk_len(P));
  w.part_keys = (unsigned*)take((size_t)n * 4);
  w.part_rows = (float*)take((size_t)n * D * 4);
  w.bytes = (size_t)(p - start) + 256;
  return w;
}

template <typename T>
int run_bwd(const gsb_codebook_args* a, cudaStream_t s) {
  constexpr int VW = Vec16<T>::N;
  const long long P = a->P, K = a->K;
  if (P == 0) {
    if (a->grad_table) cudaMemsetAsync(a->grad_table, 0, (size_t)K * a->D * sizeof(T), s);
    return check_launch("gsb_codebook_bwd");
  }
  const bool aligned = (long long)a->D * sizeof(T) % 16 == 0 && (uintptr_t)a->grad_out % 16 == 0 &&
                       (uintptr_t)a->table % 16 == 0 && (uintptr_t)a->grad_table % 16 == 0;
  const Shape sh = pick_shape(a->D, aligned ? VW : 1);
  const bool scan = a->grad_table && K > 0 && small_case(P, K);
  const bool fused_gain = a->grad_gain && a->grad_table && K > 0 && (scan ? a->D <= SCAN_COLS : sh.col_blocks == 1);
  if (a->grad_gain && !fused_gain)
    gain_dot_kernel<T><<<div_up(P * 32, THREADS), THREADS, 0, s>>>(*a);
  if (!a->grad_table || K == 0) return check_launch("gsb_codebook_bwd");
  if (scan) {
    gsb_codebook_args b = *a;
    if (!fused_gain) b.grad_gain = nullptr;
    if (scan_by_code(P, K)) {
      launch_scan<T, false>(b, K + 1, aligned, s);
    } else {
      cudaMemsetAsync(a->grad_table, 0, (size_t)K * a->D * sizeof(T), s);
      launch_scan<T, true>(b, P, aligned, s);
    }
    return check_launch("gsb_codebook_bwd");
  }

  const Workspace w = carve(a->workspace, P, K, a->D);
  const int bits = key_bits(K), passes = radix::passes_for_bits(bits);
  const radix::SortScratch scratch = radix::carve_scratch(w.sort, P, passes);
  cudaMemsetAsync(scratch.hist, 0, scratch.zero_bytes, s);
  const size_t grad_bytes = (size_t)K * a->D * sizeof(T);
  // 16-byte stores where the table's gradient is aligned, bytes at its end (or a fill of its own)
  const bool fill = (uintptr_t)a->grad_table % 16 == 0;
  if (!fill) cudaMemsetAsync(a->grad_table, 0, grad_bytes, s);
  const long long vecs = fill ? (long long)(grad_bytes / 16) : 0;
  const int tail = fill ? (int)(grad_bytes % 16) : 0;
  code_keys_kernel<<<(int)std::min<long long>(148 * 8, (P + THREADS - 1) / THREADS), THREADS, 0, s>>>(
      a->codes, a->codes64, (int)P, (unsigned)K, passes, (1u << (bits - radix::RADIX_BITS * (passes - 1))) - 1u,
      w.keys[0], w.ids[0], scratch.hist, (uint4*)a->grad_table, vecs, (uint8_t*)a->grad_table + vecs * 16, tail);
  unsigned *k[2] = {w.keys[0], w.keys[1]}, *v[2] = {w.ids[0], w.ids[1]};
  const int where = radix::sort_passes(k, v, P, nullptr, bits, scratch, a->error_word, s, nullptr, 0, true);
  SegArgs g{};
  g.keys = w.keys[where];
  g.ids = w.ids[where];
  g.rows = a->grad_out;
  g.gain = a->gain;
  g.scale = a->scale;
  g.table = a->table;
  g.grad_gain = fused_gain ? a->grad_gain : nullptr;
  g.grad_table = a->grad_table;
  g.part_keys = w.part_keys;
  g.part_rows = w.part_rows;
  g.n = (int)P;
  g.len = chunk_len(P);
  g.chunks = (int)chunks_of(P, g.len);
  g.D = a->D;
  g.gshift = sh.gshift;
  if (aligned) {
    if (fused_gain) launch_seg<T, VW, true>(g, sh, s);
    else launch_seg<T, VW, false>(g, sh, s);
  } else {
    if (fused_gain) launch_seg<T, 1, true>(g, sh, s);
    else launch_seg<T, 1, false>(g, sh, s);
  }
  if (g.chunks > 1) run_join_kernel<T><<<div_up(g.chunks, THREADS / 32), THREADS, 0, s>>>(g);
  return check_launch("gsb_codebook_bwd");
}

template <typename T, int ROWS>
void launch_gather(const gsb_codebook_args* a, cudaStream_t s) {
  const bool out_aligned = (uintptr_t)a->out % 16 == 0;
  const bool aligned = out_aligned && (long long)a->D * sizeof(T) % 16 == 0 && (uintptr_t)a->table % 16 == 0;
  const int blocks = div_up(a->P, ROWS);
  // e / D is the high word of e * ceil(2^32 / D) while e * D < 2^32 (the excess of the factor, below D, then adds
  // less than 1 / D): e < ROWS * D
  const unsigned long long D = (unsigned long long)a->D;
  const unsigned magic = D > 1 && ROWS * D * D < (1ull << 32) ? (unsigned)(((1ull << 32) + D - 1) / D) : 0u;
  if (aligned) codebook_gather_kernel<T, true, ROWS><<<blocks, THREADS, 0, s>>>(*a, 1, magic);
  else codebook_gather_kernel<T, false, ROWS><<<blocks, THREADS, 0, s>>>(*a, out_aligned, magic);
}

template <typename T>
int run_fwd(const gsb_codebook_args* a, cudaStream_t s) {
  // Longer CTAs spend less of their time on reading codes, few rows need
  // shorter ones to fill the SMs (6M x 48 fp32: 64 rows 280 us, 128 217,
  // 256 192, 512 201).
  if (a->P >= 148 * 8 * 256) launch_gather<T, 256>(a, s);
  else if (a->P >= 148 * 8 * 128) launch_gather<T, 128>(a, s);
  else launch_gather<T, 32>(a, s);
  return check_launch("gsb_codebook_fwd");
}

int check_args(const gsb_codebook_args* a, const char* what) {
  if (!a) {
    set_error("%s: null arguments", what);
    return GSB_ERR_INVALID;
  }
  if (a->P < 0 || a->P >= MAX_ROWS || a->K < 0 || a->K >= (1ll << 31) - 1 || a->D < 1 || a->D > MAX_COLS) {
    set_error("%s: sizes out of range (P %lld, K %lld, D %d)", what, a->P, a->K, a->D);
    return GSB_ERR_INVALID;
  }
  if (a->dtype < GSB_TYPE_FP32 || a->dtype > GSB_TYPE_FP16) {
    set_error("%s: unknown dtype %d", what, a->dtype);
    return GSB_ERR_INVALID;
  }
  if (a->P > 0 && (!a->codes || !a->error_word)) {
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
  if (!a->out || (a->K > 0 && !a->table)) {
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
  if (P <= 0 || P >= gsb::MAX_ROWS || K < 0 || D < 1) return 0;
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
  if (a->grad_gain && (!a->gain || (a->K > 0 && !a->table))) {
    set_error("gsb_codebook_bwd: grad_gain without gain or table");
    return GSB_ERR_INVALID;
  }
  const size_t need = a->grad_table ? gsb_codebook_bwd_workspace_bytes(a->P, a->K, a->D) : 0;
  if (need > 0 && (!a->workspace || a->workspace_bytes < need)) {
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
