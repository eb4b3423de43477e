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
#include <algorithm>

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
  const int64_t blocks = p.last > 0 ? ((int64_t)p.last + HC_SPARSE_BLOCK - 2) / HC_SPARSE_BLOCK + 1
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
// Scores.  A warp takes 8 kHand blocks, kHand for each 4 lanes: lane p of them
// holds the 16-byte chunks p, p + 4, .. of the blocks' least and greatest
// keys (a load of the warp is eight 64-byte pieces), as 64-bit values, and
// multiplies them with the query heads, which lie in shared memory split into
// their positive and negative parts:
//   max(q lo, q hi) = max(q, 0) hi + min(q, 0) lo   for lo <= hi,
// one of the two products being zero.  Bounds the wrong way round are swapped
// first.  A sum that is not finite (an infinite or NaN bound or query) is
// taken again from the formula as it stands.
// The queries' layout puts the four lanes' values side by side: with [dim]
// rows the four read the same banks, which took 130 us at 128 rows x 820
// blocks (80% of the shared-memory pipe, the 64-bit units at 6%).
constexpr int kBsThreads = 128;
constexpr int kBsWarps = kBsThreads / 32;
// Blocks of a CTA whose lanes have kHand of them in hand.
__host__ __device__ constexpr int bs_cta(int hand) { return kBsWarps * 8 * hand; }

// Blocks of a row, its length clamped to the page table.
__device__ __forceinline__ int bs_blocks(const BSParams& p, int r) {
  const int len = min(max(p.heads_len[r], 0), p.max_blocks * kPage);
  return (len + HC_SPARSE_BLOCK - 1) / HC_SPARSE_BLOCK;
}

// E elements of 16 bytes as fp32.
template <typename T, int E>
__device__ __forceinline__ void bs_unpack(const uint4& w, float (&f)[E]) {
  if constexpr (sizeof(T) == 4) {
    f[0] = __uint_as_float(w.x);
    f[1] = __uint_as_float(w.y);
    f[2] = __uint_as_float(w.z);
    f[3] = __uint_as_float(w.w);
  } else {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = unpack2<T>(u[i]);
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  }
}

// The score's definition, for one lane: sums of max(q lo, q hi), NaN as the
// highest, the greatest over the heads.
template <typename T>
__device__ __noinline__ double bs_plain_score(const BSParams& p, int r, const T* lim) {
  const int b = r / p.KV, h = r % p.KV;
  double best = -INFINITY;
#pragma unroll 1
  for (int g = 0; g < p.G; ++g) {
    const T* q = reinterpret_cast<const T*>(p.q) + b * p.qsb + (int64_t)(h * p.G + g) * p.qsh;
    double s = 0.0;
#pragma unroll 1
    for (int d = 0; d < kD; ++d) {
      const double x = (double)Elem<T>::to_f(q[d]) * (double)Elem<T>::to_f(lim[d]);
      const double y = (double)Elem<T>::to_f(q[d]) * (double)Elem<T>::to_f(lim[kD + d]);
      s += x > y || isnan(x) ? x : y;
    }
    best = fmax(best, isnan(s) ? (double)INFINITY : s);
  }
  return best;
}

template <typename T, int kG, int kHand>
__global__ void __launch_bounds__(kBsThreads, 4) block_score_kernel(const BSParams p) {
  constexpr int kBsCta = bs_cta(kHand);
  constexpr int E = 16 / (int)sizeof(T), CH = kD / E, MINE = CH / 4;  // chunks of a row, of a lane
  constexpr int STEP = 8 / kHand;                                     // chunks loaded at a time
  constexpr int GP = (kG + 1) / 2;                                    // pairs of heads
  // [lane's chunk][element][sign][head pair][lane of the four] of two heads
  extern __shared__ __align__(16) double2 s_q[];
  pdl_wait();
  pdl_trigger();
  const int r = blockIdx.y;
  const int n = bs_blocks(p, r);
  if (n <= p.n_select || (int)blockIdx.x * kBsCta >= n) return;  // (n <= n_select: every block is listed)
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int b = r / p.KV, h = r % p.KV;
  for (int i = threadIdx.x; i < 2 * GP * kD; i += kBsThreads) {
    const int g = i / kD, d = i % kD, chunk = d / E;
    const double q = g < p.G ? (double)Elem<T>::to_f(reinterpret_cast<const T*>(
                                   p.q)[b * p.qsb + (int64_t)(h * p.G + g) * p.qsh + d])
                             : 0.0;
    double* at = reinterpret_cast<double*>(
        s_q + ((((chunk >> 2) * E + d % E) * 2) * GP + (g >> 1)) * 4 + (chunk & 3)) + (g & 1);
    at[0] = q < 0.0 ? 0.0 : q;  // (a NaN stays one)
    at[GP * 4 * 2] = q < 0.0 ? q : 0.0;
  }
  __syncthreads();
  const int part = lane & 3;
  double* scores = p.scores + (int64_t)r * p.max_blocks * kBlkPerPage;
#pragma unroll 1
  for (int first = blockIdx.x * kBsCta; first < n; first += gridDim.x * kBsCta) {
    if (first + warp * kHand * 8 >= n) break;
    const T* lim[kHand];
    int blk[kHand];
    bool ok[kHand];
#pragma unroll
    for (int t = 0; t < kHand; ++t) {
      blk[t] = first + (warp * kHand + t) * 8 + (lane >> 2);
      int phys = blk[t] < n ? p.bt[(int64_t)r * p.max_blocks + blk[t] / kBlkPerPage] : -1;
      ok[t] = phys >= 0 && phys < p.n_blocks;
      if (blk[t] < n && !ok[t] && part == 0) set_err(p.err, HC_ERR_RANGE);
      if (!ok[t]) phys = 0;
      lim[t] = reinterpret_cast<const T*>(p.bounds) +
               ((int64_t)phys * kBlkPerPage + (blk[t] & (kBlkPerPage - 1))) * 2 * kD;
    }
    double acc[kHand][2 * GP];
#pragma unroll
    for (int t = 0; t < kHand; ++t)
#pragma unroll
      for (int g = 0; g < 2 * GP; ++g) acc[t][g] = 0.0;
#pragma unroll
    for (int c0 = 0; c0 < MINE; c0 += STEP) {
      uint4 wl[kHand][STEP], wh[kHand][STEP];
#pragma unroll
      for (int t = 0; t < kHand; ++t)
#pragma unroll
        for (int c = 0; c < STEP; ++c) {
          wl[t][c] = wh[t][c] = make_uint4(0u, 0u, 0u, 0u);
          if (ok[t]) {
            wl[t][c] = ld_stream128(lim[t] + (4 * (c0 + c) + part) * E);
            wh[t][c] = ld_stream128(lim[t] + kD + (4 * (c0 + c) + part) * E);
          }
        }
#pragma unroll
      for (int c = 0; c < STEP; ++c) {
        float lo[kHand][E], hi[kHand][E];
#pragma unroll
        for (int t = 0; t < kHand; ++t) {
          bs_unpack<T, E>(wl[t][c], lo[t]);
          bs_unpack<T, E>(wh[t][c], hi[t]);
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
          double x[kHand], y[kHand];
#pragma unroll
          for (int t = 0; t < kHand; ++t) {
            x[t] = bb_max(lo[t][e], hi[t][e]);
            y[t] = bb_min(lo[t][e], hi[t][e]);
          }
          const double2* q = s_q + (((c0 + c) * E + e) * 2) * GP * 4 + part;
#pragma unroll
          for (int g = 0; g < GP; ++g) {
            const double2 up = q[g * 4], down = q[(GP + g) * 4];
#pragma unroll
            for (int t = 0; t < kHand; ++t) {
              acc[t][2 * g] = fma(down.x, y[t], fma(up.x, x[t], acc[t][2 * g]));
              acc[t][2 * g + 1] = fma(down.y, y[t], fma(up.y, x[t], acc[t][2 * g + 1]));
            }
          }
        }
      }
    }
#pragma unroll
    for (int t = 0; t < kHand; ++t) {
      double best = -INFINITY;
      bool odd = false;
#pragma unroll
      for (int g = 0; g < 2 * GP; ++g) {
        acc[t][g] += __shfl_xor_sync(0xffffffffu, acc[t][g], 1);
        acc[t][g] += __shfl_xor_sync(0xffffffffu, acc[t][g], 2);
        if (g < p.G) {
          odd |= !isfinite(acc[t][g]);
          best = fmax(best, acc[t][g]);
        }
      }
      if (part == 0 && blk[t] < n) {
        if (!ok[t]) best = -INFINITY;
        else if (odd) best = bs_plain_score<T>(p, r, lim[t]);
        scores[blk[t]] = best;
      }
    }
  }
}

// Order-preserving 64-bit key of a score (-0 as +0).
__device__ __forceinline__ unsigned long long score_key(double s) {
  const unsigned long long u = (unsigned long long)__double_as_longlong(s + 0.0);
  return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}

// ---------------------------------------------------------------------------
// Selection: one CTA per row.  The sink and recent blocks are in; of the rest
// a radix select finds the key of the last that is, 8 bits a round from the
// highest bit in which the row's keys differ, until a digit's keys are all in
// (three rounds or so).  Then one scan in block order lists them.
constexpr int kSelThreads = 512;
constexpr int kSelKeys = 4096;  // keys held in shared memory (rows of up to 262144 tokens)

__global__ void __launch_bounds__(kSelThreads) block_select_kernel(const BSParams p) {
  __shared__ unsigned long long s_key[kSelKeys];
  __shared__ unsigned int s_hist[256];
  __shared__ unsigned long long s_min[kSelThreads / 32], s_max[kSelThreads / 32];
  __shared__ int s_warp[32];
  __shared__ int s_digit, s_left, s_all;
  pdl_wait();
  pdl_trigger();
  const int r = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n = bs_blocks(p, r);
  int32_t* list = p.blocks + (int64_t)r * p.n_select;
  const int count = min(n, p.n_select);
  if (threadIdx.x == 0) {
    p.counts[r] = count;
    const int len = p.heads_len[r];
    if (len < 0 || len > p.max_blocks * kPage) set_err(p.err, HC_ERR_RANGE);
  }
  for (int i = count + threadIdx.x; i < p.n_select; i += kSelThreads) list[i] = -1;
  if (n <= p.n_select) {
    for (int i = threadIdx.x; i < n; i += kSelThreads) list[i] = i;
    return;
  }
  // blocks lo .. hi - 1 compete for `left` places (sink + recent <= n_select < n)
  const int lo = p.sink, hi = n - p.recent;
  const double* sc = p.scores + (int64_t)r * p.max_blocks * kBlkPerPage;
  const bool held = n <= kSelKeys;
  auto key = [&](int j) -> unsigned long long { return held ? s_key[j] : score_key(sc[j]); };
  unsigned long long kmin = ~0ull, kmax = 0ull;
  for (int j = lo + threadIdx.x; j < hi; j += kSelThreads) {
    const unsigned long long k = score_key(sc[j]);
    if (held) s_key[j] = k;
    kmin = min(kmin, k);
    kmax = max(kmax, k);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    kmin = min(kmin, __shfl_xor_sync(0xffffffffu, kmin, o));
    kmax = max(kmax, __shfl_xor_sync(0xffffffffu, kmax, o));
  }
  if (lane == 0) {
    s_min[warp] = kmin;
    s_max[warp] = kmax;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSelThreads / 32; ++w) {
    kmin = min(kmin, s_min[w]);
    kmax = max(kmax, s_max[w]);
  }
  int left = count - lo - (n - hi);  // places among the keys that match the prefix
  int top = kmin == kmax ? 0 : 64 - __clzll((long long)(kmin ^ kmax));  // bits still open
  unsigned long long prefix = top < 64 ? kmax >> top << top : 0ull;
  unsigned long long mask = top < 64 ? ~0ull >> top << top : 0ull;
  bool all = left == 0;  // every key that matches the prefix is in (or none: left == 0)
  while (top > 0 && !all) {
    const int shift = max(top - 8, 0), bits = top - shift;
    for (int i = threadIdx.x; i < 256; i += kSelThreads) s_hist[i] = 0;
    __syncthreads();
    for (int j = lo + threadIdx.x; j < hi; j += kSelThreads) {
      const unsigned long long k = key(j);
      if ((k & mask) == prefix) atomicAdd(&s_hist[(k >> shift) & ((1u << bits) - 1u)], 1u);
    }
    __syncthreads();
    if (warp == 0) {
      // lane i holds digits 255 - 8 i .. 248 - 8 i: the greatest first
      int c[8], sum = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += c[i] = (int)s_hist[255 - 8 * lane - i];
      int run = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += y;
      }
      run -= sum;  // keys of greater digits
      if (run < left && run + sum >= left) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (run < left && run + c[i] >= left) {
            s_digit = 255 - 8 * lane - i;
            s_left = left - run;
            s_all = left - run == c[i];
          }
          run += c[i];
        }
      }
    }
    __syncthreads();
    prefix |= (unsigned long long)s_digit << shift;
    mask |= ((1ull << bits) - 1ull) << shift;
    left = s_left;
    all = s_all;
    top = shift;
    __syncthreads();
  }
  // keys above the prefix are in, and the first `left` that match it; each
  // thread lists a run of blocks
  const int per = (n + kSelThreads - 1) / kSelThreads;
  const int j0 = min(threadIdx.x * per, n), j1 = min(j0 + per, n);
  int above = 0, equal = 0;
  for (int j = j0; j < j1; ++j) {
    const bool must = j < lo || j >= hi;
    const unsigned long long k = must ? 0ull : key(j) & mask;
    above += must || k > prefix;
    equal += !must && k == prefix;
  }
  int tot;
  int a = block_exclusive_scan(above, s_warp, tot);
  int e = block_exclusive_scan(equal, s_warp, tot);
  for (int j = j0; j < j1; ++j) {
    const bool must = j < lo || j >= hi;
    const unsigned long long k = must ? 0ull : key(j) & mask;
    const bool in = must || k > prefix, eq = !must && k == prefix;
    if (in || (eq && e < left)) list[a + min(e, left)] = j;
    a += in;
    e += eq;
  }
}

size_t block_select_ws_bytes(int R, int max_blocks) {
  return (size_t)R * max_blocks * kBlkPerPage * sizeof(double) + 256;
}

template <typename T, int kG, int kHand>
static cudaError_t bs_launch_scores(const BSParams& p, cudaLaunchConfig_t& cfg, int sms) {
  // CTAs of a row: no more than fit on the SMs at a time (4 each), so that
  // none waits for a second turn
  const int tiles = (p.max_blocks * kBlkPerPage + bs_cta(kHand) - 1) / bs_cta(kHand);
  cfg.gridDim = dim3((unsigned int)std::min(tiles, std::max(1, 4 * sms / p.R)), (unsigned int)p.R);
  cfg.dynamicSmemBytes = (size_t)kD * 2 * ((kG + 1) / 2) * sizeof(double2);
  return cudaLaunchKernelEx(&cfg, block_score_kernel<T, kG, kHand>, p);
}

template <typename T>
static int bs_launch(BSParams& p, cudaStream_t st) {
  const int sms = device_sms(current_device());
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kBsThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  // Four blocks a lane read the queries from shared memory half as often as
  // two; two make twice the CTAs, for few rows.  (Bounds of 128 rows x 820
  // blocks: 28 us with four, 37 with two; 8 rows x 1640: 11 and 9.)  More
  // than four heads leave registers for two.
  const bool four = (int64_t)p.R * p.max_blocks * kBlkPerPage >= (int64_t)2 * sms * bs_cta(4);
  cudaError_t e;
  if (p.G > 4) e = bs_launch_scores<T, 8, 2>(p, cfg, sms);
  else if (p.G > 2) e = four ? bs_launch_scores<T, 4, 4>(p, cfg, sms) : bs_launch_scores<T, 4, 2>(p, cfg, sms);
  else if (p.G > 1) e = four ? bs_launch_scores<T, 2, 4>(p, cfg, sms) : bs_launch_scores<T, 2, 2>(p, cfg, sms);
  else e = four ? bs_launch_scores<T, 1, 4>(p, cfg, sms) : bs_launch_scores<T, 1, 2>(p, cfg, sms);
  if (e != cudaSuccess) return HC_ERR_CUDA;
  cfg.gridDim = dim3((unsigned int)p.R);
  cfg.blockDim = dim3(kSelThreads);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, block_select_kernel, (const BSParams)p) == cudaSuccess ? HC_OK : HC_ERR_CUDA;
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
