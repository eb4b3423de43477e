// Appending new tokens to the paged cache, with the position rotation applied
// on the way.
//
// For every new token t of sequence b (t < counts[b]) and every head, with
// the two halves of a row x = (x1, x2) of 64 dims each:
//   y1 = x1 * cos1 - x2 * sin1,   y2 = x2 * cos2 + x1 * sin2
// (fp32, one rounding to the cache type).  Rotated queries go to q_out;
// rotated keys and the values go to token heads_len[r] + t of row r = b*KV+h,
// through the page table.  Pages a row reaches that are not mapped (-1) are
// taken from the free list in (row, page) order, as the one-token append
// (kv_copy.cu) takes them.  With `bounds`, the least and greatest key of each
// 64-token block, per channel, follow: [page][4 blocks][min, max][128].
//
// Bandwidth bound (each element is read once and written once); one launch.
// Work is split into units of one aligned 64-token block of one row (so a
// block's bounds are reduced inside one CTA, without atomics) and into query
// units of 32 tokens x up to 4 heads (the cosines and sines are loaded once
// for the 4 heads).  Every key/value CTA derives the page allocation for
// itself from the state the call found; the last of them to finish (a
// counter in the workspace) writes the page table, the lengths and the
// free-list pointer, so nothing is written while another CTA still reads.
#include "hc_host.cuh"
#include "hc_params.cuh"

namespace hc {

constexpr int kRaThreads = 256;
constexpr int kRaWarps = kRaThreads / 32;
constexpr int kRaHeads = 4;  // query heads of one query unit

template <typename T> struct RaRow {
  static constexpr int E = 16 / (int)sizeof(T);     // elements of a 16-byte chunk
  static constexpr int CH2 = kD / 2 / E;            // chunks of half a row
};

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <typename T, int E>
__device__ __forceinline__ void unpack_chunk(const uint4& w, float (&f)[E]) {
  if constexpr (sizeof(T) == 4) {
    f[0] = __uint_as_float(w.x);
    f[1] = __uint_as_float(w.y);
    f[2] = __uint_as_float(w.z);
    f[3] = __uint_as_float(w.w);
  } else {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = unpack2<T>(u[i]);
      f[2 * i] = p.x;
      f[2 * i + 1] = p.y;
    }
  }
}
template <typename T, int E>
__device__ __forceinline__ uint4 pack_chunk(const float (&f)[E]) {
  if constexpr (sizeof(T) == 4) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  } else {
    return make_uint4(Elem<T>::cvt2(f[0], f[1]), Elem<T>::cvt2(f[2], f[3]), Elem<T>::cvt2(f[4], f[5]),
                      Elem<T>::cvt2(f[6], f[7]));
  }
}
// E elements of a cosine / sine row: in the cache type or in fp32
template <typename T, int E>
__device__ __forceinline__ void load_trig(const void* base, int64_t off, bool f32, float (&f)[E]) {
  if (sizeof(T) != 4 && f32) {
    const float* p = reinterpret_cast<const float*>(base) + off;
#pragma unroll
    for (int i = 0; i < E; i += 4) {
      const uint4 w = ldg128(p + i);
      f[i] = __uint_as_float(w.x);
      f[i + 1] = __uint_as_float(w.y);
      f[i + 2] = __uint_as_float(w.z);
      f[i + 3] = __uint_as_float(w.w);
    }
  } else {
    unpack_chunk<T, E>(ldg128(reinterpret_cast<const T*>(base) + off), f);
  }
}

// The rotation's factors for one chunk of each half.
template <int E> struct Trig {
  float c1[E], s1[E], c2[E], s2[E];
};
template <typename T, int E>
__device__ __forceinline__ void load_rotation(const RAParams& p, int b, int t, int d0, Trig<E>& g) {
  const int64_t c = b * p.csb + t * p.cst + d0, s = b * p.ssb + t * p.sst + d0;
  load_trig<T, E>(p.cos, c, p.trig_f32, g.c1);
  load_trig<T, E>(p.cos, c + kD / 2, p.trig_f32, g.c2);
  load_trig<T, E>(p.sin, s, p.trig_f32, g.s1);
  load_trig<T, E>(p.sin, s + kD / 2, p.trig_f32, g.s2);
}
template <int E>
__device__ __forceinline__ void rotate(const Trig<E>& g, float (&x1)[E], float (&x2)[E]) {
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const float a = x1[i], z = x2[i];
    x1[i] = fmaf(a, g.c1[i], -(z * g.s1[i]));
    x2[i] = fmaf(z, g.c2[i], a * g.s2[i]);
  }
}

__device__ __forceinline__ int ra_count(const RAParams& p, int b) {
  return p.counts ? min(max(p.counts[b], 0), p.T) : p.T;
}

// Pages that row r's append needs from the free list; bad: the row cannot be
// appended to (a length, count or page id out of range).
__device__ __forceinline__ int ra_need(const RAParams& p, int r, bool& bad) {
  const int b = r / p.KV;
  const int len = p.heads_len[r];
  const int cnt = p.counts ? p.counts[b] : p.T;
  if (len < 0 || cnt < 0 || cnt > p.T || (int64_t)len + cnt > (int64_t)p.max_blocks * kPage) {
    bad = true;
    return 0;
  }
  int need = 0;
  if (cnt > 0) {
    const int last = (len + cnt - 1) >> 8;
    for (int pg = len >> 8; pg <= last; ++pg) {
      const int phys = p.bt[(int64_t)r * p.max_blocks + pg];
      need += phys == -1;
      if (phys < -1 || phys >= p.n_blocks) bad = true;
    }
  }
  return need;
}

// A sum and an "any" over the block.
__device__ __forceinline__ int2 block_sum2(int a, int b, int2* s_red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  if (lane == 0) s_red[warp] = make_int2(a, b);
  __syncthreads();
  int2 t = make_int2(0, 0);
#pragma unroll
  for (int w = 0; w < kRaWarps; ++w) {
    t.x += s_red[w].x;
    t.y += s_red[w].y;
  }
  __syncthreads();
  return t;
}

// Status of the whole append (0, or the error code) and the free pages that
// rows before `row` take.
__device__ __forceinline__ int ra_plan(const RAParams& p, int row, int base, int2* s_red, int& before, int& total) {
  int mine = 0, all = 0, bad = 0;
  const int R = p.B * p.KV;
  for (int r = threadIdx.x; r < R; r += kRaThreads) {
    bool b = false;
    const int n = ra_need(p, r, b);
    bad |= b;
    all += n;
    if (r < row) mine += n;
  }
  const int2 s = block_sum2(all, mine, s_red);
  total = s.x;
  before = s.y;
  int oom = base < 0 || (int64_t)base + total > p.n_free;
  if (!oom)
    for (int i = threadIdx.x; i < total; i += kRaThreads) {
      const int f = p.free_blocks[base + i];
      if (f < 0 || f >= p.n_blocks) bad = 1;
    }
  const int any = __syncthreads_or(bad);
  return any ? HC_ERR_RANGE : (oom ? HC_ERR_OOM : 0);
}

// Physical page of row r's page pg: mapped already, or the row's next page
// of the free list (`take`: the list's index of the row's first free page).
__device__ __forceinline__ int ra_page(const RAParams& p, int r, int len, int pg, int take) {
  const int32_t* row = p.bt + (int64_t)r * p.max_blocks;
  const int phys = row[pg];
  if (phys != -1) return phys;
  for (int i = len >> 8; i < pg; ++i) take += row[i] == -1;
  return p.free_blocks[take];
}

// The last key/value CTA to get here: page table, lengths, free-list pointer.
__device__ __forceinline__ void ra_finish(const RAParams& p, int status, int base, int total, int* s_warp) {
  __shared__ int s_last;
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    const unsigned int n = atomicAdd(p.done, 1u);
    s_last = n == (unsigned int)p.kv_ctas - 1;
    if (s_last) *p.done = 0u;
    __threadfence();
  }
  __syncthreads();
  if (!s_last) return;
  if (status) {
    if (threadIdx.x == 0) set_err(p.err, status);
    return;
  }
  const int R = p.B * p.KV;
  int carry = base;
  for (int r0 = 0; r0 < R; r0 += kRaThreads) {
    const int r = r0 + threadIdx.x;
    bool bad = false;
    const int need = r < R ? ra_need(p, r, bad) : 0;
    int tot;
    const int ex = block_exclusive_scan(need, s_warp, tot);
    if (r < R) {
      const int len = p.heads_len[r];
      const int cnt = ra_count(p, r / p.KV);
      if (need > 0) {
        int take = carry + ex;
        const int last = (len + cnt - 1) >> 8;
        for (int pg = len >> 8; pg <= last; ++pg) {
          int32_t* e = p.bt + (int64_t)r * p.max_blocks + pg;
          if (*e == -1) *e = p.free_blocks[take++];
        }
      }
      p.heads_len_out[r] = len + cnt;
    }
    carry += tot;
    __syncthreads();
  }
  if (threadIdx.x == 0) *p.free_ptr = base + total;
}

// Rotated queries: 32 tokens (of all sequences, end to end) x kRaHeads heads.
template <typename T>
__device__ __forceinline__ void ra_query_unit(const RAParams& p, int unit) {
  constexpr int E = RaRow<T>::E, CH2 = RaRow<T>::CH2, TOK = kRaThreads / CH2;
  const int nh = (p.H + kRaHeads - 1) / kRaHeads;
  const int h0 = (unit % nh) * kRaHeads;
  const int64_t n = (int64_t)(unit / nh) * TOK + threadIdx.x / CH2;
  if (n >= (int64_t)p.B * p.T) return;
  const int b = (int)(n / p.T), t = (int)(n % p.T);
  if (t >= ra_count(p, b)) return;
  const int d0 = (threadIdx.x % CH2) * E;
  const T* src = reinterpret_cast<const T*>(p.q) + b * p.qsb + t * p.qst + d0;
  T* dst = reinterpret_cast<T*>(p.q_out) + b * p.osb + t * p.ost + d0;
  uint4 w1[kRaHeads], w2[kRaHeads];
#pragma unroll
  for (int i = 0; i < kRaHeads; ++i)
    if (h0 + i < p.H) {
      // plain loads: q_out may be q itself
      w1[i] = *reinterpret_cast<const uint4*>(src + (h0 + i) * p.qsh);
      w2[i] = *reinterpret_cast<const uint4*>(src + (h0 + i) * p.qsh + kD / 2);
    }
  Trig<E> g;
  load_rotation<T, E>(p, b, t, d0, g);
#pragma unroll
  for (int i = 0; i < kRaHeads; ++i)
    if (h0 + i < p.H) {
      float x1[E], x2[E];
      unpack_chunk<T, E>(w1[i], x1);
      unpack_chunk<T, E>(w2[i], x2);
      rotate<E>(g, x1, x2);
      *reinterpret_cast<uint4*>(dst + (h0 + i) * p.osh) = pack_chunk<T, E>(x1);
      *reinterpret_cast<uint4*>(dst + (h0 + i) * p.osh + kD / 2) = pack_chunk<T, E>(x2);
    }
}

// One aligned 64-token block of one row: threads c < CH2 of a token take
// chunk c of both halves of the key, the other CH2 those of the value.
template <typename T>
__device__ __forceinline__ void ra_block(const RAParams& p, int r, int len, int cnt, int blk, int take, float* s_mm) {
  constexpr int E = RaRow<T>::E, CH2 = RaRow<T>::CH2, PER = 2 * CH2, TOK = kRaThreads / PER;
  const int b = r / p.KV, h = r % p.KV;
  const int beg = max(blk * HC_SPARSE_BLOCK, len), end = min((blk + 1) * HC_SPARSE_BLOCK, len + cnt);
  const int phys = ra_page(p, r, len, beg >> 8, take);
  const int c = threadIdx.x % PER;
  const bool key = c < CH2;
  const int d0 = (key ? c : c - CH2) * E;
  const T* src = key ? reinterpret_cast<const T*>(p.k) + b * p.ksb + h * p.ksh + d0
                     : reinterpret_cast<const T*>(p.v) + b * p.vsb + h * p.vsh + d0;
  const int64_t sst = key ? p.kst : p.vst;
  T* pool = reinterpret_cast<T*>(key ? p.kp : p.vp) + (int64_t)phys * kPage * kD + d0;
  float mn1[E], mn2[E], mx1[E], mx2[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    mn1[i] = mn2[i] = INFINITY;
    mx1[i] = mx2[i] = -INFINITY;
  }
  for (int pos = beg + (int)threadIdx.x / PER; pos < end; pos += TOK) {
    const int t = pos - len;
    uint4 w1 = ldg128(src + t * sst), w2 = ldg128(src + t * sst + kD / 2);
    if (key) {
      Trig<E> g;
      load_rotation<T, E>(p, b, t, d0, g);
      float x1[E], x2[E];
      unpack_chunk<T, E>(w1, x1);
      unpack_chunk<T, E>(w2, x2);
      rotate<E>(g, x1, x2);
      w1 = pack_chunk<T, E>(x1);
      w2 = pack_chunk<T, E>(x2);
      if (p.bounds) {  // of the rounded keys: what the pages hold
        unpack_chunk<T, E>(w1, x1);
        unpack_chunk<T, E>(w2, x2);
#pragma unroll
        for (int i = 0; i < E; ++i) {
          mn1[i] = min_nan(mn1[i], x1[i]);
          mn2[i] = min_nan(mn2[i], x2[i]);
          mx1[i] = max_nan(mx1[i], x1[i]);
          mx2[i] = max_nan(mx2[i], x2[i]);
        }
      }
    }
    T* dst = pool + (int64_t)(pos & (kPage - 1)) * kD;
    *reinterpret_cast<uint4*>(dst) = w1;
    *reinterpret_cast<uint4*>(dst + kD / 2) = w2;
  }
  if (!p.bounds) return;
  // over the tokens of a warp (lanes PER apart), then over the warps
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = PER; o < 32; o <<= 1)
#pragma unroll
    for (int i = 0; i < E; ++i) {
      mn1[i] = min_nan(mn1[i], __shfl_xor_sync(0xffffffffu, mn1[i], o));
      mn2[i] = min_nan(mn2[i], __shfl_xor_sync(0xffffffffu, mn2[i], o));
      mx1[i] = max_nan(mx1[i], __shfl_xor_sync(0xffffffffu, mx1[i], o));
      mx2[i] = max_nan(mx2[i], __shfl_xor_sync(0xffffffffu, mx2[i], o));
    }
  __syncthreads();
  if (lane < CH2) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      s_mm[(warp * 2) * kD + d0 + i] = mn1[i];
      s_mm[(warp * 2) * kD + kD / 2 + d0 + i] = mn2[i];
      s_mm[(warp * 2 + 1) * kD + d0 + i] = mx1[i];
      s_mm[(warp * 2 + 1) * kD + kD / 2 + d0 + i] = mx2[i];
    }
  }
  __syncthreads();
  const int which = threadIdx.x / kD, d = threadIdx.x % kD;  // 0: min, 1: max
  T* out = reinterpret_cast<T*>(p.bounds) + (((int64_t)phys * (kPage / HC_SPARSE_BLOCK) + (blk & 3)) * 2 + which) * kD + d;
  float x = s_mm[which * kD + d];
#pragma unroll
  for (int w = 1; w < kRaWarps; ++w) {
    const float y = s_mm[(w * 2 + which) * kD + d];
    x = which ? max_nan(x, y) : min_nan(x, y);
  }
  if (blk * HC_SPARSE_BLOCK < len) {  // the block held tokens before
    const float y = Elem<T>::to_f(*out);
    x = which ? max_nan(x, y) : min_nan(x, y);
  }
  *out = Elem<T>::from_f(x);
}

template <typename T>
__global__ void __launch_bounds__(kRaThreads) rope_append_kernel(const RAParams p) {
  __shared__ int2 s_red[kRaWarps];
  __shared__ int s_warp[32];
  __shared__ float s_mm[kRaWarps * 2 * kD];
  pdl_wait();
  pdl_trigger();
  if ((int)blockIdx.x >= p.kv_ctas) {
    ra_query_unit<T>(p, (int)blockIdx.x - p.kv_ctas);
    return;
  }
  const int r = blockIdx.x / p.units, u = blockIdx.x % p.units;
  const int base = *p.free_ptr;
  int before, total;
  const int status = ra_plan(p, r, base, s_red, before, total);
  if (!status) {
    const int len = p.heads_len[r], cnt = ra_count(p, r / p.KV);
    const int blk = len / HC_SPARSE_BLOCK + u;
    if (cnt > 0 && blk * HC_SPARSE_BLOCK < len + cnt) ra_block<T>(p, r, len, cnt, blk, base + before, s_mm);
  }
  ra_finish(p, status, base, total, s_warp);
}

template <typename T>
static int ra_launch(RAParams& p, cudaStream_t st) {
  constexpr int TOK = kRaThreads / RaRow<T>::CH2;
  const int64_t R = (int64_t)p.B * p.KV;
  p.units = (p.T + HC_SPARSE_BLOCK - 2) / HC_SPARSE_BLOCK + 1;  // blocks that T tokens can touch
  const int64_t kv = R * p.units;
  const int64_t q = (((int64_t)p.B * p.T + TOK - 1) / TOK) * ((p.H + kRaHeads - 1) / kRaHeads);
  if (kv + q > 0x7fffffffLL) return HC_ERR_UNSUPPORTED;
  p.kv_ctas = (int)kv;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned int)(kv + q));
  cfg.blockDim = dim3(kRaThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, rope_append_kernel<T>, (const RAParams)p) == cudaSuccess ? HC_OK : HC_ERR_CUDA;
}

int rope_append_dispatch(int dtype, RAParams& p, cudaStream_t st) {
  switch (dtype) {
    case HC_F32: return ra_launch<float>(p, st);
    case HC_BF16: return ra_launch<__nv_bfloat16>(p, st);
    case HC_F16: return ra_launch<__half>(p, st);
    default: return HC_ERR_DTYPE;
  }
}

}  // namespace hc
