// Decode attention of a batch over a prefix that all its sequences share: the
// prefix part.  Every sequence's query heads of one KV head attend to the
// same tokens, so B * G query rows are multiplied with each key and value
// while it is on chip, and the pages are read from HBM once for the batch.
// The tails (each row's own tokens) run through the split decode kernel
// (decode_attn.cu, FD_TAIL), whose combine joins both parts' partials.
#include <algorithm>

#include "hc_host.cuh"
#include "hc_params.cuh"

namespace hc {

constexpr int kSpThreads = 256;
constexpr int kSpTok = 32;   // tokens of a tile
// row pitch of queries and keys in shared memory (elements): 16 bytes more
// than a row, so that rows start on 16-byte boundaries in different banks
template <typename T> constexpr int kSpPad = kD + 16 / (int)sizeof(T);
constexpr int kSpPP = 36;    // row pitch of the probabilities

__device__ __forceinline__ int sp_len(const SPParams& p, int h) {
  return min(max(p.shared_len[h], 0), p.max_blocks * kPage);
}

// Tiles before each head's segments and their total.  (KV heads are few: one
// thread's loop.)
__device__ __forceinline__ int sp_total(const SPParams& p) {
  int n = 0;
  for (int h = 0; h < p.KV; ++h) n += (sp_len(p, h) + p.plan.gran - 1) / p.plan.gran;
  return n * p.plan.n_groups;
}

template <typename T> constexpr size_t sp_smem(int RT) {
  return (size_t)RT * kSpPad<T> * sizeof(T) + 2 * (size_t)kSpTok * kSpPad<T> * sizeof(T) +
         2 * (size_t)kSpTok * kD * sizeof(T) + (size_t)RT * kSpPP * sizeof(float);
}

// 16 bytes to shared memory; nothing is read and zeros are written if !ok.
__device__ __forceinline__ void cp_async16(void* dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(smem_u32(dst)), "l"(src), "r"(ok ? 16 : 0)
               : "memory");
}
template <typename T>
__device__ __forceinline__ float4 lds4(const T* p) {
  if constexpr (sizeof(T) == 4) {
    return *reinterpret_cast<const float4*>(p);
  } else {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    const float2 a = unpack2<T>(w.x), b = unpack2<T>(w.y);
    return make_float4(a.x, a.y, b.x, b.y);
  }
}

// CUDA-core form: RPT query rows a thread (16 * RPT a CTA), tiles of 32
// tokens, two of them in shared memory by cp.async.  Thread (ty, tx) of the
// 16 x 16 holds rows ty * RPT + i, scores of tokens tx and tx + 16, outputs
// of dims 4 tx .. and 64 + 4 tx ...
template <typename T, int RPT>
__global__ void __launch_bounds__(kSpThreads, 2) shared_prefix_kernel(const SPParams p) {
  constexpr int RT = 16 * RPT;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  T* sq = reinterpret_cast<T*>(smem_raw);
  T* sk = sq + RT * kSpPad<T>;
  T* sv = sk + 2 * kSpTok * kSpPad<T>;
  float* sp = reinterpret_cast<float*>(sv + 2 * kSpTok * kD);
  pdl_wait();
  pdl_trigger();
  const int total = sp_total(p);
  const int span = (total + gridDim.x - 1) / (int)gridDim.x;
  const int beg = blockIdx.x * span, end = min(total, beg + span);
  if (beg >= end) return;
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  const int NG = p.plan.n_groups;
  int start = 0;  // first tile of the head's segments
  for (int h = 0; h < p.KV; ++h) {
    const int len = sp_len(p, h);
    const int tiles = (len + kSpTok - 1) / kSpTok;
    for (int ng = 0; ng < NG; ++ng, start += tiles) {
      const int t0 = max(beg, start) - start, t1 = min(end, start + tiles) - start;
      if (t0 >= t1) continue;
      __syncthreads();
      constexpr int CH = kD * sizeof(T) / 16, CE = 16 / (int)sizeof(T);
      for (int i = threadIdx.x; i < RT * CH; i += kSpThreads) {
        const int row = ng * RT + i / CH, c = i % CH;
        const bool ok = row < p.B * p.G;
        const int b = ok ? row / p.G : 0, g = ok ? row % p.G : 0;
        const T* src = reinterpret_cast<const T*>(p.q) + b * p.qsb + (int64_t)(h * p.G + g) * p.qsh + c * CE;
        cp_async16(sq + (i / CH) * kSpPad<T> + c * CE, src, ok);
      }
      auto load = [&](int t, int s) {
        const int pos = t * kSpTok, page = pos >> 8;
        const int blk = p.bt[(int64_t)h * p.max_blocks + page];
        const bool in = blk >= 0 && blk < p.n_blocks;
        if (!in && threadIdx.x == 0) set_err(p.err, HC_ERR_RANGE);
        const int64_t off = ((int64_t)(in ? blk : 0) * kPage + (pos & (kPage - 1))) * kD;
        for (int i = threadIdx.x; i < kSpTok * CH; i += kSpThreads) {
          const int row = i / CH, c = i % CH;
          const bool ok = in && pos + row < len;
          cp_async16(sk + (s * kSpTok + row) * kSpPad<T> + c * CE, reinterpret_cast<const T*>(p.kp) + off + row * kD + c * CE, ok);
          cp_async16(sv + (s * kSpTok + row) * kD + c * CE, reinterpret_cast<const T*>(p.vp) + off + row * kD + c * CE, ok);
        }
        asm volatile("cp.async.commit_group;\n" ::: "memory");
        return in ? min(kSpTok, len - pos) : 0;
      };
      float m[RPT], l[RPT], o[RPT][8];
#pragma unroll
      for (int i = 0; i < RPT; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int d = 0; d < 8; ++d) o[i][d] = 0.f;
      }
      int valid = load(t0, 0);
      for (int t = t0; t < t1; ++t) {
        const int s = (t - t0) & 1;
        int next = 0;
        if (t + 1 < t1) {
          next = load(t + 1, s ^ 1);
          asm volatile("cp.async.wait_group 1;\n" ::: "memory");
        } else {
          asm volatile("cp.async.wait_group 0;\n" ::: "memory");
        }
        __syncthreads();
        const T* kt = sk + s * kSpTok * kSpPad<T>;
        const T* vt = sv + s * kSpTok * kD;
        float a[RPT][2];
#pragma unroll
        for (int i = 0; i < RPT; ++i) a[i][0] = a[i][1] = 0.f;
#pragma unroll 4
        for (int d = 0; d < kD; d += 4) {
          const float4 k0 = lds4<T>(kt + tx * kSpPad<T> + d), k1 = lds4<T>(kt + (tx + 16) * kSpPad<T> + d);
#pragma unroll
          for (int i = 0; i < RPT; ++i) {
            const float4 q = lds4<T>(sq + (ty * RPT + i) * kSpPad<T> + d);
            a[i][0] = fmaf(q.x, k0.x, fmaf(q.y, k0.y, fmaf(q.z, k0.z, fmaf(q.w, k0.w, a[i][0]))));
            a[i][1] = fmaf(q.x, k1.x, fmaf(q.y, k1.y, fmaf(q.z, k1.z, fmaf(q.w, k1.w, a[i][1]))));
          }
        }
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
          const float s0 = tx < valid ? a[i][0] * p.scale_log2 : -INFINITY;
          const float s1 = tx + 16 < valid ? a[i][1] * p.scale_log2 : -INFINITY;
          float mx = fmaxf(s0, s1);
#pragma unroll
          for (int x = 8; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
          const float mn = fmaxf(m[i], mx);
          const float ref = mn == -INFINITY ? 0.f : mn;
          const float corr = exp2f(m[i] - ref);
          const float p0 = exp2f(s0 - ref), p1 = exp2f(s1 - ref);
          m[i] = mn;
          l[i] = l[i] * corr + p0 + p1;  // this thread's tokens; summed over tx at the end
#pragma unroll
          for (int d = 0; d < 8; ++d) o[i][d] *= corr;
          sp[(ty * RPT + i) * kSpPP + tx] = p0;
          sp[(ty * RPT + i) * kSpPP + tx + 16] = p1;
        }
        __syncwarp();  // a row's 16 threads are lanes of one warp
#pragma unroll 2
        for (int j = 0; j < kSpTok; j += 4) {
          float4 pr[RPT];
#pragma unroll
          for (int i = 0; i < RPT; ++i) pr[i] = *reinterpret_cast<const float4*>(sp + (ty * RPT + i) * kSpPP + j);
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const float4 v0 = lds4<T>(vt + (j + u) * kD + 4 * tx), v1 = lds4<T>(vt + (j + u) * kD + 64 + 4 * tx);
#pragma unroll
            for (int i = 0; i < RPT; ++i) {
              const float w = u == 0 ? pr[i].x : u == 1 ? pr[i].y : u == 2 ? pr[i].z : pr[i].w;
              o[i][0] = fmaf(w, v0.x, o[i][0]);
              o[i][1] = fmaf(w, v0.y, o[i][1]);
              o[i][2] = fmaf(w, v0.z, o[i][2]);
              o[i][3] = fmaf(w, v0.w, o[i][3]);
              o[i][4] = fmaf(w, v1.x, o[i][4]);
              o[i][5] = fmaf(w, v1.y, o[i][5]);
              o[i][6] = fmaf(w, v1.z, o[i][6]);
              o[i][7] = fmaf(w, v1.w, o[i][7]);
            }
          }
        }
        __syncthreads();  // the stage is free
        valid = next;
      }
      const int64_t slot = (int64_t)blockIdx.x + h * NG + ng;
#pragma unroll
      for (int i = 0; i < RPT; ++i) {
        float s = l[i];
#pragma unroll
        for (int x = 8; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        const int row = ty * RPT + i;
        if (ng * RT + row >= p.B * p.G) continue;
        const int64_t at = slot * RT + row;
        if (tx == 0) p.plan.part_ml[at] = make_float2(m[i], s);
        *reinterpret_cast<float4*>(p.plan.part_o + at * kD + 4 * tx) = make_float4(o[i][0], o[i][1], o[i][2], o[i][3]);
        *reinterpret_cast<float4*>(p.plan.part_o + at * kD + 64 + 4 * tx) =
            make_float4(o[i][4], o[i][5], o[i][6], o[i][7]);
      }
    }
  }
}

// Rows a CTA of the CUDA-core form: the fewest of 16, 32, 64 that hold the
// batch's (a tile's work is the same for the rows it does not fill).
static int sp_rows(int rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : 64; }

static PrefixPlan sp_plan(int B, int KV, int G, int sms) {
  PrefixPlan pl = {};
  pl.rows_per = sp_rows(B * G);
  pl.n_groups = (B * G + pl.rows_per - 1) / pl.rows_per;
  pl.gran = kSpTok;
  pl.streams = 1;
  pl.stream_rows = pl.rows_per;
  pl.n_ctas = 2 * sms;
  return pl;
}

static size_t sp_bytes(const PrefixPlan& pl, int KV, size_t* ml_at) {
  const size_t rows = ((size_t)pl.n_ctas + (size_t)KV * pl.n_groups) * pl.streams * pl.stream_rows;
  if (ml_at) *ml_at = rows * kD * sizeof(float);
  return (rows * (kD * sizeof(float) + sizeof(float2)) + 255) & ~(size_t)255;
}

size_t shared_prefix_ws_bytes(int dtype, int B, int KV, int G) {
  (void)dtype;
  return sp_bytes(sp_plan(B, KV, G, device_sms(current_device())), KV, nullptr);
}

template <typename T, int RPT>
static int sp_launch(SPParams& p, cudaStream_t st) {
  auto kern = shared_prefix_kernel<T, RPT>;
  constexpr size_t smem = sp_smem<T>(16 * RPT);
  static bool attr_set[kMaxDevices];
  const int dev = current_device();
  if (dev < 0) return HC_ERR_CUDA;
  {
    std::lock_guard<std::mutex> g(host_lock());
    if (!attr_set[dev]) {
      if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
        return HC_ERR_CUDA;
      attr_set[dev] = true;
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned int)p.plan.n_ctas);
  cfg.blockDim = dim3(kSpThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, (const SPParams)p) == cudaSuccess ? HC_OK : HC_ERR_CUDA;
}

template <typename T>
static int sp_launch_rows(SPParams& p, cudaStream_t st) {
  switch (p.plan.rows_per) {
    case 16: return sp_launch<T, 1>(p, st);
    case 32: return sp_launch<T, 2>(p, st);
    default: return sp_launch<T, 4>(p, st);
  }
}

int shared_prefix_dispatch(int dtype, SPParams& p, void* ws, size_t ws_bytes, cudaStream_t st) {
  const int dev = current_device();
  if (dev < 0) return HC_ERR_CUDA;
  p.plan = sp_plan(p.B, p.KV, p.G, device_sms(dev));
  size_t ml_at;
  if (!ws || ws_bytes < sp_bytes(p.plan, p.KV, &ml_at)) return HC_ERR_WORKSPACE;
  p.plan.part_o = reinterpret_cast<float*>(ws);
  p.plan.part_ml = reinterpret_cast<float2*>(reinterpret_cast<unsigned char*>(ws) + ml_at);
  p.wait_ns = wait_limit_ns(kMbarTimeoutNs);
  switch (dtype) {
    case HC_F32: return sp_launch_rows<float>(p, st);
    case HC_BF16: return sp_launch_rows<__nv_bfloat16>(p, st);
    case HC_F16: return sp_launch_rows<__half>(p, st);
    default: return HC_ERR_DTYPE;
  }
}

}  // namespace hc
