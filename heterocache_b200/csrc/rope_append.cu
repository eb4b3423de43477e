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
// 64-token block, per channel, follow: [page][4 blocks][min, max][128].  In the
// block that held tokens before, they are taken over those tokens' keys in the
// page as well, not from its old bounds: these may hold tokens that were
// appended as drafts and dropped since.
//
// Bandwidth bound (each element is read once and written once); one launch.
// Work is split into units of one aligned 64-token block of one row (so a
// block's bounds are reduced inside one CTA, without atomics) and into query
// units of 32 tokens x up to 4 heads (the cosines and sines are loaded once
// for the 4 heads).  Registers are kept to three CTAs an SM, two tokens (four
// heads) of a thread in flight: 16 x 4096 tokens of 32 + 8 heads, 1.36 GB,
// take 236 to 245 us (86 to 89% of the copy rate; with fp32 minima and one
// token in flight at 111 registers, 441 us).  Every key/value CTA derives the
// page allocation for itself from the state the call found; the last of them to have read it (a
// counter) writes the page table, the lengths and the free-list pointer, so
// nothing is written while another CTA still reads.
#include "hc_host.cuh"
#include "hc_params.cuh"

namespace hc {

constexpr int kRaThreads = 256;
constexpr int kRaWarps = kRaThreads / 32;
constexpr int kRaHeads = 4;  // query heads of one query unit
constexpr int kRaRun = 4;    // most blocks of a key/value CTA
constexpr int kRaCtas = 3;   // CTAs an SM

template <typename T> struct RaRow {
  static constexpr int E = 16 / (int)sizeof(T);     // elements of a 16-byte chunk
  static constexpr int CH2 = kD / 2 / E;            // chunks of half a row
};

// Least / greatest of two values, or of two 16-bit pairs at a time; NaN if
// either is.
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
template <typename T> struct Word;  // 32 bits of T
template <> struct Word<float> {
  __device__ __forceinline__ static uint32_t min(uint32_t a, uint32_t b) {
    return __float_as_uint(min_nan(__uint_as_float(a), __uint_as_float(b)));
  }
  __device__ __forceinline__ static uint32_t max(uint32_t a, uint32_t b) {
    return __float_as_uint(max_nan(__uint_as_float(a), __uint_as_float(b)));
  }
  static constexpr uint32_t kInf = 0x7f800000u, kNegInf = 0xff800000u;
};
template <> struct Word<__nv_bfloat16> {
  __device__ __forceinline__ static uint32_t min(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("min.NaN.bf16x2 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  __device__ __forceinline__ static uint32_t max(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static constexpr uint32_t kInf = 0x7f807f80u, kNegInf = 0xff80ff80u;
};
template <> struct Word<__half> {
  __device__ __forceinline__ static uint32_t min(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("min.NaN.f16x2 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  __device__ __forceinline__ static uint32_t max(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.f16x2 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static constexpr uint32_t kInf = 0x7c007c00u, kNegInf = 0xfc00fc00u;
};

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
// The rotation's factors for one chunk of each half, as loaded: of type TT,
// the cache's or fp32.
template <typename TT, int E> struct Trig {
  static constexpr int N = E * (int)sizeof(TT) / 16;
  uint4 c1[N], s1[N], c2[N], s2[N];
};
template <typename TT, int E>
__device__ __forceinline__ void load_rotation(const RAParams& p, int b, int t, int d0, Trig<TT, E>& g) {
  const TT* c = reinterpret_cast<const TT*>(p.cos) + b * p.csb + t * p.cst + d0;
  const TT* s = reinterpret_cast<const TT*>(p.sin) + b * p.ssb + t * p.sst + d0;
#pragma unroll
  for (int i = 0; i < Trig<TT, E>::N; ++i) {
    g.c1[i] = ldg128(reinterpret_cast<const uint4*>(c) + i);
    g.s1[i] = ldg128(reinterpret_cast<const uint4*>(s) + i);
    g.c2[i] = ldg128(reinterpret_cast<const uint4*>(c + kD / 2) + i);
    g.s2[i] = ldg128(reinterpret_cast<const uint4*>(s + kD / 2) + i);
  }
}
template <typename TT, int E>
__device__ __forceinline__ void unpack_trig(const uint4 (&w)[Trig<TT, E>::N], float (&f)[E]) {
  constexpr int PER = 16 / (int)sizeof(TT);
#pragma unroll
  for (int i = 0; i < Trig<TT, E>::N; ++i) {
    float part[PER];
    unpack_chunk<TT, PER>(w[i], part);
#pragma unroll
    for (int j = 0; j < PER; ++j) f[i * PER + j] = part[j];
  }
}
// y1 = x1 c1 - x2 s1, y2 = x2 c2 + x1 s2: two roundings in fp32, then one to T.
template <typename T, typename TT, int E>
__device__ __forceinline__ void rotate(const Trig<TT, E>& g, uint4& w1, uint4& w2) {
  float x1[E], x2[E], c[E], s[E], y[E];
  unpack_chunk<T, E>(w1, x1);
  unpack_chunk<T, E>(w2, x2);
  unpack_trig<TT, E>(g.c1, c);
  unpack_trig<TT, E>(g.s1, s);
#pragma unroll
  for (int i = 0; i < E; ++i) y[i] = fmaf(x1[i], c[i], -(x2[i] * s[i]));
  w1 = pack_chunk<T, E>(y);
  unpack_trig<TT, E>(g.c2, c);
  unpack_trig<TT, E>(g.s2, s);
#pragma unroll
  for (int i = 0; i < E; ++i) y[i] = fmaf(x2[i], c[i], x1[i] * s[i]);
  w2 = pack_chunk<T, E>(y);
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

// Called by all threads of a key/value CTA once each has read what it needs of
// the lengths, the page table and the free list, and before any of its stores
// (so the fence finds none in flight).  *last: the CTA is the last of the launch
// to get here, known after the next barrier.
__device__ __forceinline__ void ra_arrive(const RAParams& p, int* last) {
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    const unsigned int n = atomicAdd(p.done, 1u);
    *last = n == (unsigned int)p.kv_ctas - 1;
    if (*last) *p.done = 0u;
    __threadfence();
  }
}

// The last CTA to arrive: page table, lengths, free-list pointer.
__device__ __forceinline__ void ra_finish(const RAParams& p, int status, int base, int total, int* s_warp) {
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
template <typename T, typename TT>
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
  Trig<TT, E> g;
  load_rotation<TT, E>(p, b, t, d0, g);
#pragma unroll
  for (int i = 0; i < kRaHeads; ++i)
    if (h0 + i < p.H) {
      rotate<T, TT, E>(g, w1[i], w2[i]);
      *reinterpret_cast<uint4*>(dst + (h0 + i) * p.osh) = w1[i];
      *reinterpret_cast<uint4*>(dst + (h0 + i) * p.osh + kD / 2) = w2[i];
    }
}

// One aligned 64-token block of one row: threads c < CH2 of a token take
// chunk c of both halves of the key, the other CH2 those of the value; two
// tokens a thread are in flight.  With bounds the key threads start at the
// block's first token, whose key is in the page if the row held it before.
template <typename T, typename TT>
__device__ __forceinline__ void ra_block(const RAParams& p, int r, int len, int cnt, int blk, int phys,
                                         uint32_t* s_mm) {
  constexpr int E = RaRow<T>::E, CH2 = RaRow<T>::CH2, PER = 2 * CH2, TOK = kRaThreads / PER;
  constexpr int RW = kD * (int)sizeof(T) / 4;  // 32-bit words of a row
  const int b = r / p.KV, h = r % p.KV;
  const int beg = max(blk * HC_SPARSE_BLOCK, len), end = min((blk + 1) * HC_SPARSE_BLOCK, len + cnt);
  const int c = threadIdx.x % PER;
  const bool key = c < CH2;
  const int d0 = (key ? c : c - CH2) * E;
  const T* src = key ? reinterpret_cast<const T*>(p.k) + b * p.ksb + h * p.ksh + d0
                     : reinterpret_cast<const T*>(p.v) + b * p.vsb + h * p.vsh + d0;
  const int64_t sst = key ? p.kst : p.vst;
  T* pool = reinterpret_cast<T*>(key ? p.kp : p.vp) + (int64_t)phys * kPage * kD + d0;
  uint32_t mn[8], mx[8];  // of the two chunks
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    mn[i] = Word<T>::kInf;
    mx[i] = Word<T>::kNegInf;
  }
  const int from = p.bounds ? blk * HC_SPARSE_BLOCK : beg;
  for (int pos0 = from + (int)threadIdx.x / PER; pos0 < end; pos0 += 2 * TOK) {
    uint4 w1[2], w2[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int pos = pos0 + u * TOK;
      if (pos < end && (pos >= len || key)) {
        const T* x = pos >= len ? src + (pos - len) * sst : pool + (int64_t)(pos & (kPage - 1)) * kD;
        w1[u] = *reinterpret_cast<const uint4*>(x);
        w2[u] = *reinterpret_cast<const uint4*>(x + kD / 2);
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int pos = pos0 + u * TOK;
      if (pos >= end || (pos < len && !key)) continue;
      if (key) {
        if (pos >= len) {
          Trig<TT, E> g;
          load_rotation<TT, E>(p, b, pos - len, d0, g);
          rotate<T, TT, E>(g, w1[u], w2[u]);
        }
        if (p.bounds) {  // of the rounded keys: what the pages hold
          const uint32_t x[8] = {w1[u].x, w1[u].y, w1[u].z, w1[u].w, w2[u].x, w2[u].y, w2[u].z, w2[u].w};
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            mn[i] = Word<T>::min(mn[i], x[i]);
            mx[i] = Word<T>::max(mx[i], x[i]);
          }
        }
      }
      if (pos < len) continue;
      T* dst = pool + (int64_t)(pos & (kPage - 1)) * kD;
      *reinterpret_cast<uint4*>(dst) = w1[u];
      *reinterpret_cast<uint4*>(dst + kD / 2) = w2[u];
    }
  }
  if (!p.bounds) return;
  // over the tokens of a warp (lanes PER apart), then over the warps
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = PER; o < 32; o <<= 1)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      mn[i] = Word<T>::min(mn[i], __shfl_xor_sync(0xffffffffu, mn[i], o));
      mx[i] = Word<T>::max(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], o));
    }
  __syncthreads();
  if (lane < CH2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s_mm[(warp * 2) * RW + lane * 4 + i] = mn[i];
      s_mm[(warp * 2) * RW + RW / 2 + lane * 4 + i] = mn[4 + i];
      s_mm[(warp * 2 + 1) * RW + lane * 4 + i] = mx[i];
      s_mm[(warp * 2 + 1) * RW + RW / 2 + lane * 4 + i] = mx[4 + i];
    }
  }
  __syncthreads();
  const int which = threadIdx.x / RW, d = threadIdx.x % RW;  // 0: least, 1: greatest
  if (which > 1) return;
  uint32_t* out = reinterpret_cast<uint32_t*>(p.bounds) +
                  (((int64_t)phys * (kPage / HC_SPARSE_BLOCK) + (blk & (kPage / HC_SPARSE_BLOCK - 1))) * 2 + which) * RW +
                  d;
  uint32_t x = s_mm[which * RW + d];
#pragma unroll
  for (int w = 1; w < kRaWarps; ++w) {
    const uint32_t y = s_mm[(w * 2 + which) * RW + d];
    x = which ? Word<T>::max(x, y) : Word<T>::min(x, y);
  }
  *out = x;
}

// One token a sequence: a row's token takes as many threads as a token of
// ra_block, and a CTA a run of rows from r0 on (16 of a 16-bit cache), so
// that few CTAs go through all rows for the allocation.  What is appended does
// not hang on the allocation: it is loaded first.  With bounds a CTA has an
// eighth or a quarter of the rows where all CTAs are resident at once all the
// same: its warps then read a row's earlier keys eight or four at a time.  (Of
// 64 sequences of 8 rows: 6.9 us without bounds, 8.4 with an eighth of the rows
// a CTA, 8.9 with a quarter; of 512 sequences 27 without, 32 with all rows, 53
// with a quarter.)
template <typename T>
__host__ __device__ constexpr int ra_rows() {
  return kRaThreads / (2 * RaRow<T>::CH2);
}
// Warps of a row's earlier keys: those of a CTA of `rows` rows, one if it has more rows than warps.
__host__ __device__ constexpr int ra_row_warps(int rows) { return rows < kRaWarps ? kRaWarps / rows : 1; }

// Least and greatest key, per channel, of the tokens before the new one in its
// block, of the CTA's `rows` rows: row r0 + i's partials at s_mm[i * WPR ..][least,
// greatest].  What ra_plan will find bad is not read.
template <typename T, int ROWS>
__device__ __forceinline__ void ra_past(const RAParams& p, int r0, uint32_t* s_mm) {
  constexpr int WPR = ra_row_warps(ROWS);
  constexpr int RW = kD * (int)sizeof(T) / 4, CH = RW / 4, TW = 32 / CH;  // a row's words, chunks; tokens of a warp
  constexpr int STEP = WPR * TW, U = 8;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll 1
  for (int slot = warp; slot < ROWS * WPR; slot += kRaWarps) {
    const int r = r0 + slot / WPR;
    int n = 0;
    const uint4* x = nullptr;
    if (r < p.B * p.KV && ra_count(p, r / p.KV) > 0) {
      const int len = p.heads_len[r];
      if (len > 0 && (len >> 8) < p.max_blocks) n = len & (HC_SPARSE_BLOCK - 1);
      if (n > 0) {
        const int phys = p.bt[(int64_t)r * p.max_blocks + (len >> 8)];
        if (phys < 0 || phys >= p.n_blocks) n = 0;
        else x = reinterpret_cast<const uint4*>(p.kp) + ((int64_t)phys * kPage + (len & (kPage - 1)) - n) * CH + lane % CH;
      }
    }
    uint32_t mn[4], mx[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      mn[i] = Word<T>::kInf;
      mx[i] = Word<T>::kNegInf;
    }
    for (int t0 = (slot % WPR) * TW + lane / CH; t0 < n; t0 += U * STEP) {
      uint4 w[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (t0 + u * STEP < n) w[u] = x[(t0 + u * STEP) * CH];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (t0 + u * STEP < n) {
          const uint32_t y[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            mn[i] = Word<T>::min(mn[i], y[i]);
            mx[i] = Word<T>::max(mx[i], y[i]);
          }
        }
    }
#pragma unroll
    for (int o = CH; o < 32; o <<= 1)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        mn[i] = Word<T>::min(mn[i], __shfl_xor_sync(0xffffffffu, mn[i], o));
        mx[i] = Word<T>::max(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], o));
      }
    if (lane < CH) {
      uint4* out = reinterpret_cast<uint4*>(s_mm) + slot * 2 * CH + lane;
      out[0] = make_uint4(mn[0], mn[1], mn[2], mn[3]);
      out[CH] = make_uint4(mx[0], mx[1], mx[2], mx[3]);
    }
  }
}

template <typename T, typename TT> struct RaToken {
  static constexpr int E = RaRow<T>::E, CH2 = RaRow<T>::CH2, PER = 2 * CH2;
  int r, b, c, pos, phys;
  bool ok, key;
  uint4 w1, w2;
  Trig<TT, E> g;

  __device__ __forceinline__ void load(const RAParams& p, int r0) {
    r = r0 + (int)threadIdx.x / PER;
    c = threadIdx.x % PER;
    key = c < CH2;
    ok = r < p.B * p.KV && r - r0 < p.rows;
    if (!ok) return;
    b = r / p.KV;
    const int h = r % p.KV;
    const int d0 = (key ? c : c - CH2) * E;
    const T* src = key ? reinterpret_cast<const T*>(p.k) + b * p.ksb + h * p.ksh + d0
                       : reinterpret_cast<const T*>(p.v) + b * p.vsb + h * p.vsh + d0;
    w1 = ldg128(src);
    w2 = ldg128(src + kD / 2);
    if (key) load_rotation<TT, E>(p, b, 0, d0, g);
    ok = ra_count(p, b) > 0;
  }
  // Where the token goes; `take`: the free list's index of row r0's first free page.
  __device__ __forceinline__ void place(const RAParams& p, int r0, int take) {
    if (!ok) return;
    pos = p.heads_len[r];
    phys = p.bt[(int64_t)r * p.max_blocks + (pos >> 8)];
    if (phys != -1) return;
    bool bad = false;
    for (int k = r0; k < r; ++k) take += ra_need(p, k, bad);
    phys = p.free_blocks[take];
  }
  __device__ __forceinline__ void store(const RAParams& p, int r0, const uint32_t* s_mm) {
    if (!ok) return;
    const int d0 = (key ? c : c - CH2) * E;
    if (key) rotate<T, TT, E>(g, w1, w2);
    T* dst = reinterpret_cast<T*>(key ? p.kp : p.vp) + ((int64_t)phys * kPage + (pos & (kPage - 1))) * kD + d0;
    *reinterpret_cast<uint4*>(dst) = w1;
    *reinterpret_cast<uint4*>(dst + kD / 2) = w2;
    if (!key || !p.bounds) return;
    uint4* lim = reinterpret_cast<uint4*>(p.bounds) +
                 ((int64_t)phys * (kPage / HC_SPARSE_BLOCK) + ((pos & (kPage - 1)) / HC_SPARSE_BLOCK)) * 4 * CH2 + c;
    const int n = ra_row_warps(p.rows);
    const uint4* past = reinterpret_cast<const uint4*>(s_mm) + (r - r0) * n * 4 * CH2 + c;
    merge(lim, past, n, w1);
    merge(lim + CH2, past + CH2, n, w2);
  }
  // The bounds of a chunk: of the new key and the partials of ra_past.
  __device__ __forceinline__ void merge(uint4* at, const uint4* past, int n, const uint4& w) {
    uint4 lo = w, hi = w;
    for (int i = 0; i < n; ++i) {
      const uint4 a = past[i * 4 * CH2], z = past[i * 4 * CH2 + 2 * CH2];
      lo = make_uint4(Word<T>::min(a.x, lo.x), Word<T>::min(a.y, lo.y), Word<T>::min(a.z, lo.z), Word<T>::min(a.w, lo.w));
      hi = make_uint4(Word<T>::max(z.x, hi.x), Word<T>::max(z.y, hi.y), Word<T>::max(z.z, hi.z), Word<T>::max(z.w, hi.w));
    }
    at[0] = lo;
    at[2 * CH2] = hi;
  }
};

template <typename T, typename TT>
__global__ void __launch_bounds__(kRaThreads, kRaCtas) rope_append_kernel(const RAParams p) {
  __shared__ int2 s_red[kRaWarps];
  __shared__ int s_warp[32];
  __shared__ __align__(16) uint32_t s_mm[(ra_rows<T>() > kRaWarps ? ra_rows<T>() : kRaWarps) * 2 * kD * sizeof(T) / 4];
  __shared__ int s_phys[kRaRun], s_last;
  pdl_wait();
  pdl_trigger();
  if ((int)blockIdx.x >= p.kv_ctas) {
    ra_query_unit<T, TT>(p, (int)blockIdx.x - p.kv_ctas);
    return;
  }
  const int per_row = (p.units + p.run - 1) / p.run;
  const bool single = p.T == 1;
  const int r = single ? (int)blockIdx.x * p.rows : (int)blockIdx.x / per_row;
  const int u0 = (blockIdx.x % per_row) * p.run;
  RaToken<T, TT> tok;
  if (single && p.bounds) {
    if (p.rows == ra_rows<T>() / 8) ra_past<T, ra_rows<T>() / 8>(p, r, s_mm);
    else if (p.rows == ra_rows<T>() / 4) ra_past<T, ra_rows<T>() / 4>(p, r, s_mm);
    else ra_past<T, ra_rows<T>()>(p, r, s_mm);
  }
  if (single) tok.load(p, r);
  const int base = *p.free_ptr;
  int before, total;
  const int status = ra_plan(p, r, base, s_red, before, total);
  int len = 0, cnt = 0;
  if (!status && single) {
    tok.place(p, r, base + before);
  } else if (!status) {
    len = p.heads_len[r], cnt = ra_count(p, r / p.KV);
    const int blk = len / HC_SPARSE_BLOCK + u0 + (int)threadIdx.x;
    if (threadIdx.x < p.run && cnt > 0 && blk * HC_SPARSE_BLOCK < len + cnt)
      s_phys[threadIdx.x] = ra_page(p, r, len, max(blk * HC_SPARSE_BLOCK, len) >> 8, base + before);
  }
  ra_arrive(p, &s_last);
  if (!status && single) {
    tok.store(p, r, s_mm);
  } else if (!status) {
    for (int u = u0; u < min(u0 + p.run, p.units); ++u) {
      const int blk = len / HC_SPARSE_BLOCK + u;
      if (cnt > 0 && blk * HC_SPARSE_BLOCK < len + cnt) ra_block<T, TT>(p, r, len, cnt, blk, s_phys[u - u0], s_mm);
    }
  }
  __syncthreads();
  if (s_last) ra_finish(p, status, base, total, s_warp);
}

template <typename T, typename TT>
static int ra_launch(RAParams& p, cudaStream_t st) {
  constexpr int TOK = kRaThreads / RaRow<T>::CH2;
  const int64_t R = (int64_t)p.B * p.KV;
  p.units = (p.T + HC_SPARSE_BLOCK - 2) / HC_SPARSE_BLOCK + 1;  // blocks that T tokens can touch
  // a CTA finds the allocation once for a run of 4 blocks, where there are
  // still CTAs enough to fill the GPU
  p.run = R * p.units >= kRaRun * 8 * (int64_t)device_sms(current_device()) ? kRaRun : 1;
  p.rows = ra_rows<T>();
  if (p.bounds)
    for (const int part : {8, 4})
      if (p.rows == ra_rows<T>() && R * part / p.rows < kRaCtas * (int64_t)device_sms(current_device())) p.rows /= part;
  const int64_t kv = p.T == 1 ? (R + p.rows - 1) / p.rows : R * ((p.units + p.run - 1) / p.run);
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
  return cudaLaunchKernelEx(&cfg, rope_append_kernel<T, TT>, (const RAParams)p) == cudaSuccess ? HC_OK : HC_ERR_CUDA;
}

int rope_append_dispatch(int dtype, RAParams& p, cudaStream_t st) {
  switch (dtype) {
    case HC_F32: return ra_launch<float, float>(p, st);
    case HC_BF16:
      return p.trig_f32 ? ra_launch<__nv_bfloat16, float>(p, st) : ra_launch<__nv_bfloat16, __nv_bfloat16>(p, st);
    case HC_F16: return p.trig_f32 ? ra_launch<__half, float>(p, st) : ra_launch<__half, __half>(p, st);
    default: return HC_ERR_DTYPE;
  }
}

}  // namespace hc
