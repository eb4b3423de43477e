// Block bounds and block selection of the sparse decode attention.
//
// bounds[page][j][0/1][d]: least and greatest key, per channel, of the j-th
// 64-token block of a page (of the tokens its row holds).  A query row's dot
// product with any key of the block is at most sum_d max(q_d lo_d, q_d hi_d);
// a block's score for a KV head is the largest of its query heads' bounds.
// Of a row's blocks the first `sink`, the last `recent` and the best others
// are listed, n_select in all, in ascending order; equal scores go to the
// lowest block.  Scores are sums in 64 bits: which block is in must not hang
// on the order of a 32-bit sum, and the products of 16-bit values and their
// sums are then exact for all but extreme exponents.  A score that is not a
// number counts as the highest, so that NaN keys are attended to, not hidden.
#include "hc_host.cuh"
#include "hc_params.cuh"

namespace hc {

constexpr int kBlkPerPage = kPage / HC_SPARSE_BLOCK;
constexpr int kBbThreads = 128;

__device__ __forceinline__ float bb_min(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float bb_max(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// ---------------------------------------------------------------------------
// Bounds of the blocks of some rows from their pages: one CTA per block, a
// thread per channel (one coalesced row of 128 channels per token).
template <typename T>
__global__ void __launch_bounds__(kBbThreads) block_bounds_kernel(const BBParams p) {
  pdl_wait();
  pdl_trigger();
  const int r = p.rows ? p.rows[blockIdx.y] : (int)blockIdx.y;
  if (r < 0 || r >= p.R) {
    if (threadIdx.x == 0) set_err(p.err, HC_ERR_RANGE);
    return;
  }
  const int len = p.heads_len[r];
  const int first = p.last > 0 ? max(0, len - p.last) / HC_SPARSE_BLOCK : 0;
  const int blk = first + (int)blockIdx.x;
  const int t0 = blk * HC_SPARSE_BLOCK;
  if (t0 >= len) return;
  const int page = t0 >> 8;
  const int phys = page < p.max_blocks ? p.bt[(int64_t)r * p.max_blocks + page] : -1;
  if (phys < 0 || phys >= p.n_blocks) {
    if (threadIdx.x == 0) set_err(p.err, HC_ERR_RANGE);
    return;
  }
  const int n = min(HC_SPARSE_BLOCK, len - t0);
  const int d = threadIdx.x;
  const T* k = reinterpret_cast<const T*>(p.kp) + ((int64_t)phys * kPage + (t0 & (kPage - 1))) * kD + d;
  float lo = INFINITY, hi = -INFINITY;
#pragma unroll 8
  for (int i = 0; i < n; ++i) {
    const float x = Elem<T>::to_f(k[(int64_t)i * kD]);
    lo = bb_min(lo, x);
    hi = bb_max(hi, x);
  }
  T* out = reinterpret_cast<T*>(p.bounds) + ((int64_t)phys * kBlkPerPage + (blk & (kBlkPerPage - 1))) * 2 * kD + d;
  out[0] = Elem<T>::from_f(lo);
  out[kD] = Elem<T>::from_f(hi);
}

template <typename T>
static int bb_launch(const BBParams& p, cudaStream_t st) {
  const int64_t blocks = p.last > 0 ? (int64_t)(p.last + HC_SPARSE_BLOCK - 2) / HC_SPARSE_BLOCK + 1
                                    : (int64_t)p.max_blocks * kBlkPerPage;
  const int64_t cap = (int64_t)p.max_blocks * kBlkPerPage;
  const int rows = p.rows ? p.n_rows : p.R;
  if (rows > 65535) return HC_ERR_UNSUPPORTED;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned int)(blocks < cap ? blocks : cap), (unsigned int)rows);
  cfg.blockDim = dim3(kBbThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, block_bounds_kernel<T>, p) == cudaSuccess ? HC_OK : HC_ERR_CUDA;
}

int block_bounds_dispatch(int dtype, const BBParams& p, cudaStream_t st) {
  switch (dtype) {
    case HC_F32: return bb_launch<float>(p, st);
    case HC_BF16: return bb_launch<__nv_bfloat16>(p, st);
    case HC_F16: return bb_launch<__half>(p, st);
    default: return HC_ERR_DTYPE;
  }
}

// ---------------------------------------------------------------------------
// Scores: one warp per (row, block), 4 channels a lane.
constexpr int kBsThreads = 256;
constexpr int kBsWarps = kBsThreads / 32;

template <typename T>
__device__ __forceinline__ void load4(const T* p, float (&f)[4]) {
  if constexpr (sizeof(T) == 4) {
    const float4 w = *reinterpret_cast<const float4*>(p);
    f[0] = w.x; f[1] = w.y; f[2] = w.z; f[3] = w.w;
  } else {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    const float2 a = unpack2<T>(w.x), b = unpack2<T>(w.y);
    f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
  }
}

// Blocks of a row, its length clamped to the page table.
__device__ __forceinline__ int bs_blocks(const BSParams& p, int r) {
  const int len = min(max(p.heads_len[r], 0), p.max_blocks * kPage);
  return (len + HC_SPARSE_BLOCK - 1) / HC_SPARSE_BLOCK;
}

template <typename T>
__global__ void __launch_bounds__(kBsThreads) block_score_kernel(const BSParams p) {
  pdl_wait();
  pdl_trigger();
  const int r = blockIdx.y;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n = bs_blocks(p, r);
  if (n <= p.n_select) return;  // every block is listed
  const int blk = blockIdx.x * kBsWarps + warp;
  if (blk >= n) return;
  const int b = r / p.KV, h = r % p.KV;
  const int phys = p.bt[(int64_t)r * p.max_blocks + blk / kBlkPerPage];
  double* out = p.scores + (int64_t)r * p.max_blocks * kBlkPerPage + blk;
  if (phys < 0 || phys >= p.n_blocks) {
    if (lane == 0) {
      set_err(p.err, HC_ERR_RANGE);
      *out = -INFINITY;
    }
    return;
  }
  const T* lim = reinterpret_cast<const T*>(p.bounds) +
                 ((int64_t)phys * kBlkPerPage + (blk & (kBlkPerPage - 1))) * 2 * kD + 4 * lane;
  float lo[4], hi[4];
  load4<T>(lim, lo);
  load4<T>(lim + kD, hi);
  double best = -INFINITY;
  for (int g = 0; g < p.G; ++g) {
    float q[4];
    load4<T>(reinterpret_cast<const T*>(p.q) + b * p.qsb + (int64_t)(h * p.G + g) * p.qsh + 4 * lane, q);
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // (a product of two 32-bit values is exact in 64 bits)
      const double x = (double)q[i] * (double)lo[i], y = (double)q[i] * (double)hi[i];
      s += x > y || isnan(x) ? x : y;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (isnan(s)) s = INFINITY;
    best = fmax(best, s);
  }
  if (lane == 0) *out = best;
}

// Order-preserving 64-bit key of a score (-0 as +0).
__device__ __forceinline__ unsigned long long score_key(double s) {
  const unsigned long long u = (unsigned long long)__double_as_longlong(s + 0.0);
  return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}

// ---------------------------------------------------------------------------
// Selection: one CTA per row.  Radix select of the n_select-th greatest key,
// 8 bits a round from the top, then one pass in block order.
template <int kThreads>
__global__ void __launch_bounds__(kThreads) block_select_kernel(const BSParams p) {
  __shared__ unsigned int s_hist[256];
  __shared__ int s_warp[32];
  __shared__ int s_digit, s_left;
  pdl_wait();
  pdl_trigger();
  const int r = blockIdx.x;
  const int n = bs_blocks(p, r);
  int32_t* list = p.blocks + (int64_t)r * p.n_select;
  const int count = min(n, p.n_select);
  if (threadIdx.x == 0) {
    p.counts[r] = count;
    const int len = p.heads_len[r];
    if (len < 0 || len > p.max_blocks * kPage) set_err(p.err, HC_ERR_RANGE);
  }
  for (int i = count + threadIdx.x; i < p.n_select; i += kThreads) list[i] = -1;
  if (n <= p.n_select) {
    for (int i = threadIdx.x; i < n; i += kThreads) list[i] = i;
    return;
  }
  const double* sc = p.scores + (int64_t)r * p.max_blocks * kBlkPerPage;
  auto key = [&](int j) -> unsigned long long {
    return (j < p.sink || j >= n - p.recent) ? ~0ull : score_key(sc[j]);
  };
  unsigned long long prefix = 0, mask = 0;
  int left = count;  // how many of the keys that match the prefix are taken
  for (int shift = 56; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += kThreads) s_hist[i] = 0;
    __syncthreads();
    for (int j = threadIdx.x; j < n; j += kThreads) {
      const unsigned long long k = key(j);
      if ((k & mask) == prefix) atomicAdd(&s_hist[(k >> shift) & 255], 1u);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      int run = 0, d = 255;
      while (d > 0 && run + (int)s_hist[d] < left) run += (int)s_hist[d--];
      s_digit = d;
      s_left = left - run;
    }
    __syncthreads();
    left = s_left;
    prefix |= (unsigned long long)s_digit << shift;
    mask |= 255ull << shift;
    __syncthreads();
  }
  // prefix is the n_select-th greatest key; `left` of the blocks that have it are in
  int taken = 0, ties = 0;
  for (int j0 = 0; j0 < n; j0 += kThreads) {
    const int j = j0 + threadIdx.x;
    const unsigned long long k = j < n ? key(j) : 0ull;
    const int eq = j < n && k == prefix;
    int tot;
    const int rank = ties + block_exclusive_scan(eq, s_warp, tot);
    ties += tot;
    const int in = j < n && (k > prefix || (eq && rank < left));
    const int at = taken + block_exclusive_scan(in, s_warp, tot);
    taken += tot;
    if (in) list[at] = j;
  }
}

size_t block_select_ws_bytes(int R, int max_blocks) {
  return (size_t)R * max_blocks * kBlkPerPage * sizeof(double) + 256;
}

template <typename T>
static int bs_launch(BSParams& p, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned int)((p.max_blocks * kBlkPerPage + kBsWarps - 1) / kBsWarps), (unsigned int)p.R);
  cfg.blockDim = dim3(kBsThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, block_score_kernel<T>, (const BSParams)p) != cudaSuccess) return HC_ERR_CUDA;
  cfg.gridDim = dim3((unsigned int)p.R);
  cfg.blockDim = dim3(512);
  return cudaLaunchKernelEx(&cfg, block_select_kernel<512>, (const BSParams)p) == cudaSuccess ? HC_OK : HC_ERR_CUDA;
}

int block_select_dispatch(int dtype, BSParams& p, void* ws, size_t ws_bytes, cudaStream_t st) {
  if (p.R <= 0 || p.R > kMaxRowsFD || p.G <= 0 || p.G > kGMax) return HC_ERR_UNSUPPORTED;
  if ((int64_t)p.max_blocks * kPage > 0x7fffffffLL) return HC_ERR_UNSUPPORTED;
  if (!ws || ws_bytes < block_select_ws_bytes(p.R, p.max_blocks)) return HC_ERR_WORKSPACE;
  p.scores = reinterpret_cast<double*>(ws);
  switch (dtype) {
    case HC_F32: return bs_launch<float>(p, st);
    case HC_BF16: return bs_launch<__nv_bfloat16>(p, st);
    case HC_F16: return bs_launch<__half>(p, st);
    default: return HC_ERR_DTYPE;
  }
}

}  // namespace hc
