// Decode attention of a batch over a prefix that all its sequences share: the
// prefix part.  Every sequence's query heads of one KV head attend to the
// same tokens, so B * G query rows are multiplied with each key and value
// while it is on chip, and the pages are read from HBM once for the batch.
// The tails (each row's own tokens) run through the split decode kernel
// (decode_attn.cu, FD_TAIL), and a join there merges both parts' partials.
#include <type_traits>

#include "hc_host.cuh"
#include "hc_params.cuh"
#include "umma.cuh"

namespace hc {

constexpr int kSpTok = 32;   // tokens of a tile
// row pitch of queries and keys in shared memory (elements): 16 bytes more
// than a row, so that rows start on 16-byte boundaries in different banks
constexpr int kSpPad = kD + 4;
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

constexpr size_t sp_smem(int RT) {
  return ((size_t)RT * kSpPad + 2 * (size_t)kSpTok * kSpPad + 2 * (size_t)kSpTok * kD + (size_t)RT * kSpPP) *
         sizeof(float);
}

// 16 bytes to shared memory; nothing is read and zeros are written if !ok.
__device__ __forceinline__ void cp_async16(void* dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(smem_u32(dst)), "l"(src), "r"(ok ? 16 : 0)
               : "memory");
}
// Two fp32 values in one 64-bit register: a * b + c, a + b and a * b of both.
__device__ __forceinline__ uint64_t pack_f2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack_f2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;\n" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma_f2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add_f2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

__device__ __forceinline__ uint64_t mul_f2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// Four floats of shared memory as two pairs.
__device__ __forceinline__ ulonglong2 lds4(const float* p) { return *reinterpret_cast<const ulonglong2*>(p); }

// CUDA-core form, for fp32: RT query rows a CTA, a warp for 4 RPT of them,
// tiles of 32 tokens, two of them in shared memory by cp.async.  Thread
// (ty, tx) of a warp's 4 x 8 holds rows RPT ty + i: scores of tokens tx + 8 u,
// then outputs of dims 4 tx + 32 c ..  Bound by what comes out of shared memory
// (a 16-byte load of a warp takes 4 clocks, broadcast or not), so a thread's
// tile is large: 4 x 4 scores for 8 loads, 4 x 16 outputs for 20 loads of 4
// tokens.  With 16 rows two a thread, for twice the warps.  20000 tokens x 8
// heads take 68 us for up to 16 rows (102 with one row a thread and 16 x 16
// threads), 145 for 64 (161; 179 with eight a thread, too few warps); 3000
// tokens x 8 heads for 24 rows 28 (31).
template <int RT, int RPT>
__global__ void __launch_bounds__(8 * RT / RPT, 2) shared_prefix_kernel(const SPParams p) {
  constexpr int kThreads = 8 * RT / RPT;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  float* sq = reinterpret_cast<float*>(smem_raw);
  float* sk = sq + RT * kSpPad;
  float* sv = sk + 2 * kSpTok * kSpPad;
  float* sp = sv + 2 * kSpTok * kD;
  // in this order: the tails' kernel starts at the trigger and relies on what
  // came before this kernel being complete (decode_attn.cu, pdl_launch)
  pdl_wait();
  pdl_trigger();
  const int total = sp_total(p);
  const int span = (total + gridDim.x - 1) / (int)gridDim.x;
  const int beg = blockIdx.x * span, end = min(total, beg + span);
  if (beg >= end) return;
  const int tx = threadIdx.x & 7;
  const int row0 = RPT * (threadIdx.x >> 3);  // the thread's first row
  const int NG = p.plan.n_groups;
  int start = 0;  // first tile of the head's segments
  for (int h = 0; h < p.KV; ++h) {
    const int len = sp_len(p, h);
    const int tiles = (len + kSpTok - 1) / kSpTok;
    for (int ng = 0; ng < NG; ++ng, start += tiles) {
      const int t0 = max(beg, start) - start, t1 = min(end, start + tiles) - start;
      if (t0 >= t1) continue;
      __syncthreads();
      constexpr int CH = kD / 4, CE = 4;
      for (int i = threadIdx.x; i < RT * CH; i += kThreads) {
        const int row = ng * RT + i / CH, c = i % CH;
        const bool ok = row < p.B * p.G;
        const int b = ok ? row / p.G : 0, g = ok ? row % p.G : 0;
        const float* src = reinterpret_cast<const float*>(p.q) + b * p.qsb + (int64_t)(h * p.G + g) * p.qsh + c * CE;
        cp_async16(sq + (i / CH) * kSpPad + c * CE, src, ok);
      }
      auto load = [&](int t, int s) {
        const int pos = t * kSpTok, page = pos >> 8;
        const int blk = p.bt[(int64_t)h * p.max_blocks + page];
        const bool in = blk >= 0 && blk < p.n_blocks;
        if (!in && threadIdx.x == 0) set_err(p.err, HC_ERR_RANGE);
        const int64_t off = ((int64_t)(in ? blk : 0) * kPage + (pos & (kPage - 1))) * kD;
#pragma unroll 4
        for (int i = threadIdx.x; i < kSpTok * CH; i += kThreads) {
          const int row = i / CH, c = i % CH;
          const bool ok = in && pos + row < len;
          cp_async16(sk + (s * kSpTok + row) * kSpPad + c * CE, reinterpret_cast<const float*>(p.kp) + off + row * kD + c * CE, ok);
          cp_async16(sv + (s * kSpTok + row) * kD + c * CE, reinterpret_cast<const float*>(p.vp) + off + row * kD + c * CE, ok);
        }
        asm volatile("cp.async.commit_group;\n" ::: "memory");
        return in ? min(kSpTok, len - pos) : 0;
      };
      float m[RPT], l[RPT];
      uint64_t o[RPT][8];  // pairs of dims
#pragma unroll
      for (int i = 0; i < RPT; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int d = 0; d < 8; ++d) o[i][d] = 0ull;
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
        const float* kt = sk + s * kSpTok * kSpPad;
        const float* vt = sv + s * kSpTok * kD;
        uint64_t a[RPT][4];  // sums over even and odd dims
#pragma unroll
        for (int i = 0; i < RPT; ++i)
#pragma unroll
          for (int u = 0; u < 4; ++u) a[i][u] = 0ull;
#pragma unroll 4
        for (int d = 0; d < kD; d += 4) {
          ulonglong2 k[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) k[u] = lds4(kt + (tx + 8 * u) * kSpPad + d);
#pragma unroll
          for (int i = 0; i < RPT; ++i) {
            const ulonglong2 q = lds4(sq + (row0 + i) * kSpPad + d);
#pragma unroll
            for (int u = 0; u < 4; ++u) a[i][u] = fma_f2(q.y, k[u].y, fma_f2(q.x, k[u].x, a[i][u]));
          }
        }
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
          float x[4], mx = -INFINITY;
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const float2 v = unpack_f2(a[i][u]);
            x[u] = tx + 8 * u < valid ? (v.x + v.y) * p.scale_log2 : -INFINITY;
            mx = fmaxf(mx, x[u]);
          }
#pragma unroll
          for (int y = 4; y > 0; y >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, y));
          const float mn = fmaxf(m[i], mx);
          const float ref = mn == -INFINITY ? 0.f : mn;
          const float corr = exp2f(m[i] - ref);
          m[i] = mn;
          l[i] *= corr;  // this thread's tokens; summed over tx at the end
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const float e = exp2f(x[u] - ref);
            l[i] += e;
            sp[(row0 + i) * kSpPP + tx + 8 * u] = e;
          }
#pragma unroll
          for (int d = 0; d < 8; ++d) o[i][d] = mul_f2(o[i][d], pack_f2(corr, corr));
        }
        __syncwarp();  // a row's threads are lanes of one warp
#pragma unroll 2
        for (int j = 0; j < kSpTok; j += 4) {
          float pr[RPT][4];
#pragma unroll
          for (int i = 0; i < RPT; ++i)
            *reinterpret_cast<float4*>(pr[i]) = *reinterpret_cast<const float4*>(sp + (row0 + i) * kSpPP + j);
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            ulonglong2 v[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) v[c] = lds4(vt + (j + u) * kD + 32 * c + 4 * tx);
#pragma unroll
            for (int i = 0; i < RPT; ++i) {
              const uint64_t w = pack_f2(pr[i][u], pr[i][u]);
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                o[i][2 * c] = fma_f2(w, v[c].x, o[i][2 * c]);
                o[i][2 * c + 1] = fma_f2(w, v[c].y, o[i][2 * c + 1]);
              }
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
        for (int y = 4; y > 0; y >>= 1) s += __shfl_xor_sync(0xffffffffu, s, y);
        const int row = row0 + i;
        if (ng * RT + row >= p.B * p.G) continue;
        if (tx == 0) p.plan.part_ml[slot * RT + row] = make_float2(m[i], s);
        // dims 4 tx + 32 c ..: half an 8-dim group of the layout
        float* dst = p.plan.part_o + slot * RT * kD + ((int64_t)(tx >> 1) * RT + row) * 8 + (tx & 1) * 4;
#pragma unroll
        for (int c = 0; c < 4; ++c)
          *reinterpret_cast<ulonglong2*>(dst + (int64_t)4 * c * RT * 8) = make_ulonglong2(o[i][2 * c], o[i][2 * c + 1]);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Tensor-core form (16-bit types): one CTA per SM, tiles of 128 tokens.
//   S = Q K^T  (M = 128 query rows on the TMEM lanes, N = 128 tokens)
//   O += P V   (A = P from tensor memory, B = V as loaded, MN-major)
// Two streams X = 0, 1, each with its own S (P is written over its first 64
// columns) and O accumulators, so that the tensor core works on one while
// the softmax warps work on the other.  With at most 128 query rows a group
// both streams hold the same rows and take the tiles in turn (X takes tiles
// X, X + 2, ...): two independent splits of the tokens.  With up to 256 the
// streams hold 128 rows each and every tile serves both.
// Measured: 64 rows x 8 heads of 6554 to 32768 tokens (96 MB), 26 to 31 us,
// the steady part near the reading of the pages; 256 rows x 8 heads of up to
// 131072 tokens (376 MB, 97 GFLOP), 123 us, 0.47 of the measured bf16 rate.
// There the chain of a stream (S, softmax, O) sets the pace: a step of both
// takes some 4300 clocks (the difference between calls of 8 and 16 tiles a
// CTA; 4900 to 5400 in long ones, under the power limit), of which the tensor
// core works 2048; its 8 MMAs take 512 clocks alone and 600 to 1000 beside the
// softmax warps' loads of tensor memory, whose exponentials are 2048 clocks of
// their unit a step.
// Warps: 0 key producer, 2 value producer (TMA), 1 MMA issuer, 4-7 and 8-11
// softmax of stream 0 and 1 (one query row a thread); 3 has no role.  The
// CTA's span may cover several segments (KV head, row group); between them
// the softmax warps store the partials and put the next queries into shared
// memory, while the producers run ahead.
// Tokens behind the shared ones in the last tile (and a bad page's) are
// masked, and their values zeroed in shared memory before the MMA, whatever
// the page holds there.
// Every wait is bounded; a role whose wait gives up marks the launch failed
// (HC_ERR_TIMEOUT) and waits no more; copies and MMAs in flight are waited
// for (bounded) before tensor memory is released.
constexpr int kTcThreads = 12 * 32;
constexpr int kTcTile = 128;
constexpr int kTcBox = 128 * 128;        // bytes: 128 rows x 64 16-bit elements
constexpr int kTcTileBytes = 2 * kTcBox;
constexpr int kTcTiles = 7;              // tile buffers: queries, keys, values
constexpr size_t kTcSmem = 1024 + (size_t)kTcTiles * kTcTileBytes;
constexpr int kTcK = 3;                  // key stages; values have the rest
constexpr int kTcValidRing = 8;          // tiles whose valid counts are kept
// tensor-memory columns: S of stream X at 128 X (P in its first 64), O at 256 + 128 X
constexpr uint32_t kTcColS = 0, kTcColO = 256;

// The same answer for the whole warp (each lane polls for itself).
__device__ __forceinline__ bool mbar_wait_warp(uint64_t* bar, uint32_t parity, uint64_t limit_ns) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, limit_ns));
}

__device__ __forceinline__ void named_bar_arrive(int id, int nthreads) {
  asm volatile("bar.arrive %0, %1;\n" ::"r"(id), "r"(nthreads) : "memory");
}

// One lane of the (converged) warp.  A branch on it tells the compiler that
// one thread is active, so that it need not serialise the instructions whose
// operands are uniform registers (MMAs, commits).
__device__ __forceinline__ bool elect_one() {
  uint32_t is;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.b32 %0, 1, 0, p;\n}\n" : "=r"(is));
  return is != 0;
}

// One CTA's part of one segment: tiles t0 .. t1 - 1 of head h's `len` tokens.
struct TcPiece {
  int h, ng, t0, t1, len;
};
// Walks the CTA's pieces in order; called by whole warps (lane i holds the
// shared length of the i-th of 32 heads).
struct TcWalk {
  int beg, end, start, h, ng, lens;
  __device__ __forceinline__ void init(const SPParams& p) {
    const int lane = threadIdx.x & 31;
    int n = 0;
    for (int k = lane; k < p.KV; k += 32) n += (sp_len(p, k) + kTcTile - 1) / kTcTile;
    lens = lane < p.KV ? sp_len(p, lane) : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    n *= p.plan.n_groups;
    const int span = (n + (int)gridDim.x - 1) / (int)gridDim.x;
    beg = (int)blockIdx.x * span;
    end = min(n, beg + span);
    start = h = ng = 0;
  }
  __device__ __forceinline__ bool next(const SPParams& p, TcPiece& out) {
    while (h < p.KV && start < end) {
      const int len = __shfl_sync(0xffffffffu, lens, h & 31);
      const int tiles = (len + kTcTile - 1) / kTcTile;
      const int t0 = max(beg, start) - start, t1 = min(end, start + tiles) - start;
      out.h = h;
      out.ng = ng;
      out.t0 = t0;
      out.t1 = t1;
      out.len = len;
      start += tiles;
      if (++ng == p.plan.n_groups) {
        ng = 0;
        if ((++h & 31) == 0) {
          const int k = h + (int)(threadIdx.x & 31);
          lens = k < p.KV ? sp_len(p, k) : 0;
        }
      }
      if (t0 < t1) return true;
    }
    return false;
  }
};

// What the MMA issuer needs of the CTA's shared memory.
struct TcSmem {
  unsigned char* tiles;  // buffers 0 .. kTcK - 1 keys, then values, the last one or two queries
  int vst;
  uint64_t *q_full, *k_full, *k_empty, *v_empty;
  uint64_t *s_full, *p_ready, *o_done;
};

// The MMAs of both streams in turn, called by a whole warp: all lanes wait,
// one issues (the same one throughout: MMAs of one thread execute in order,
// so a tile's S may follow the O step that reads the P it overwrites).  What
// this warp does between two MMAs the tensor core waits for, so it does
// little: the softmax warps have waited for a step's values before they
// report its P.
template <typename T>
__device__ __forceinline__ bool tc_issue(const SPParams& p, const TcSmem& sm, TcWalk& walk, bool wide) {
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  const uint32_t id_s = idesc_f16_m128(kBf16, 128);
  const uint32_t id_o = idesc_f16_m128(kBf16, 128) | kIdescBMajorMN;
  const uint32_t tiles = smem_u32(sm.tiles);
  const uint64_t dq1 = smem_desc_sw128(tiles + (kTcTiles - 1) * kTcTileBytes);
  const uint64_t dq0 = wide ? smem_desc_sw128(tiles + (kTcTiles - 2) * kTcTileBytes) : dq1;
  int kbase = 0, piece = 0;   // the piece's first tile, pieces
  int done0 = 0, done1 = 0;   // steps of earlier pieces per stream
  TcPiece pc;
  auto wait_k = [&](int n) {
    if (!mbar_wait_warp(&sm.k_full[n % kTcK], (n / kTcK) & 1, p.wait_ns)) return false;
    tc_fence_after();
    return true;
  };
  // S of tile n for stream x; free_k: no other stream reads the tile later
  auto issue_s = [&](int x, int n, bool free_k) {
    const int st = n % kTcK;
    if (elect_one()) {
      const uint64_t dq = x ? dq1 : dq0, dk = smem_desc_sw128(tiles + st * kTcTileBytes);
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) {
        const uint64_t off = (uint64_t)(((kk >> 2) * kTcBox + (kk & 3) * 32) >> 4);
        umma_f16(kTcColS + 128u * x, dq + off, dk + off, id_s, kk > 0 ? 1u : 0u);
      }
      umma_commit(&sm.s_full[x]);
      if (free_k) umma_commit(&sm.k_empty[st]);
    }
    __syncwarp();
  };
  auto issue_pv = [&](int x, int n, bool first, bool free_v) {
    const int st = n % sm.vst;
    if (elect_one()) {
      const uint64_t dv = smem_desc_sw128_mn(tiles + (kTcK + st) * kTcTileBytes, kTcBox);
      const uint32_t d = kTcColO + 128u * x, pa = kTcColS + 128u * x;
#pragma unroll
      for (int kk = 0; kk < 8; ++kk)
        umma_f16_ts(d, pa + (uint32_t)(8 * kk), dv + (uint64_t)((kk * 16 * 128) >> 4), id_o,
                    (!first || kk > 0) ? 1u : 0u);
      umma_commit(&sm.o_done[x]);
      if (free_v) umma_commit(&sm.v_empty[st]);
    }
    __syncwarp();
  };
  while (walk.next(p, pc)) {
    const int nt = pc.t1 - pc.t0;
    // each stream's tiles: first, first + step, ..
    const int step = wide ? 1 : 2;
    const bool both = !wide || p.B * p.G - pc.ng * 256 > 128;  // (wide: stream 1 has rows)
    const int n0 = wide ? nt : (nt + 1) >> 1, n1 = !both ? 0 : wide ? nt : nt >> 1;
    const int f0 = kbase, f1 = kbase + (wide ? 0 : 1);
    // wide: a tile's stage is free once stream 1, which comes second, has read it
    const bool free0 = !wide || !both;
    kbase += nt;
    if (!mbar_wait_warp(sm.q_full, piece++ & 1, p.wait_ns) || !wait_k(f0)) return false;
    issue_s(0, f0, free0);
    if (n1 > 0) {
      if (!wide && !wait_k(f1)) return false;
      issue_s(1, f1, true);
    }
    for (int i = 0; i < n0; ++i) {
      const int t0 = f0 + i * step, t1 = f1 + i * step;
      if (!mbar_wait_warp(&sm.p_ready[0], (done0 + i) & 1, p.wait_ns)) return false;
      tc_fence_after();
      issue_pv(0, t0, i == 0, free0);
      if (i + 1 < n0) {
        if (!wait_k(t0 + step)) return false;
        issue_s(0, t0 + step, free0);
      }
      if (i < n1) {
        if (!mbar_wait_warp(&sm.p_ready[1], (done1 + i) & 1, p.wait_ns)) return false;
        tc_fence_after();
        issue_pv(1, t1, i == 0, true);
        if (i + 1 < n1) {
          if (!wide && !wait_k(t1 + step)) return false;
          issue_s(1, t1 + step, true);
        }
      }
    }
    done0 += n0;
    done1 += n1;
  }
  return true;
}

template <typename T>
__global__ void __launch_bounds__(kTcThreads, 1)
    shared_prefix_tc_kernel(const SPParams p, const __grid_constant__ CUtensorMap tmk,
                            const __grid_constant__ CUtensorMap tmv) {
  extern __shared__ __align__(16) unsigned char smem_dyn[];
  const bool wide = p.plan.rows_per > 128;  // the streams hold different rows
  const int nq = wide ? 2 : 1;
  const int vst = kTcTiles - kTcK - nq;
  // tile buffers: keys, values, queries
  unsigned char* sk = smem_dyn + ((1024 - (smem_u32(smem_dyn) & 1023)) & 1023);
  unsigned char* sv = sk + kTcK * kTcTileBytes;
  unsigned char* sq = sk + (kTcTiles - nq) * kTcTileBytes;
  __shared__ __align__(8) uint64_t q_full, k_full[kTcK], k_empty[kTcK], v_full[kTcTiles - kTcK],
      v_empty[kTcTiles - kTcK], s_full[2], p_ready[2], o_done[2], all_done;
  __shared__ uint32_t s_tmem;
  __shared__ int s_fail, s_kissued, s_vissued;
  __shared__ int s_valid[kTcValidRing];  // tokens of the tile that count, by the CTA's tile number
  __shared__ float s_m[2][128], s_l1[128];  // the streams' maxima, stream 1's sums (streams of the same rows)

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(&q_full, 8);
    for (int i = 0; i < kTcK; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < vst; ++i) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&s_full[x], 1);
      mbar_init(&p_ready[x], 4);
      mbar_init(&o_done[x], 1);
    }
    mbar_init(&all_done, 1);
    s_fail = 0;
    s_kissued = s_vissued = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&s_tmem, 512u);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;  // all 512 columns: column 0 on
  // in this order, by every CTA, as in the CUDA-core form
  pdl_wait();
  pdl_trigger();
  TcWalk walk;
  walk.init(p);
  TcPiece pc;

  if (warp == 0 || warp == 2) {
    // ---- producers (lane 0 issues).  The first queries are asked for before
    // the tiles: behind those, at the memory's full rate, they came 1.5 to 2
    // us later.
    named_bar_sync(2, 256 + 64);
    const bool keys = warp == 0;
    const int NS = keys ? kTcK : vst;
    uint64_t* full = keys ? k_full : v_full;
    uint64_t* empty = keys ? k_empty : v_empty;
    unsigned char* ring = keys ? sk : sv;
    const CUtensorMap* map = keys ? &tmk : &tmv;
    const uint64_t pol = l2_evict_first_policy();
    int n = 0;
    bool ok = true;
    while (ok && walk.next(p, pc)) {
      const int32_t* bt = p.bt + (int64_t)pc.h * p.max_blocks;
      // an injected stall (hc_set_wait_limits) loads no key tile: every wait
      // on one runs out, for tests of the timeout path
      if (keys && p.stall) continue;
      // lane i holds the page of the i-th of 32 pages
      int page0 = pc.t0 >> 1;
      int pages = page0 + lane < p.max_blocks ? bt[page0 + lane] : -1;
      for (int t = pc.t0; t < pc.t1; ++t, ++n) {
        if ((t >> 1) - page0 == 32) {
          page0 += 32;
          pages = page0 + lane < p.max_blocks ? bt[page0 + lane] : -1;
        }
        const int blk = __shfl_sync(0xffffffffu, pages, (t >> 1) - page0);
        if (lane == 0) {
          const int pos = t * kTcTile;
          const bool in = blk >= 0 && blk < p.n_blocks;
          const int s = n % NS;
          if (!mbar_wait_sleep(&empty[s], ((n / NS) & 1) ^ 1, p.wait_ns)) {
            atomicExch(&s_fail, 1);
            ok = false;
          } else {
            if (keys) {
              if (!in) set_err(p.err, HC_ERR_RANGE);
              s_valid[n % kTcValidRing] = in ? min(kTcTile, pc.len - pos) : 0;
            }
            unsigned char* dst = ring + (size_t)s * kTcTileBytes;
            const int y = (in ? blk : 0) * kPage + (pos & (kPage - 1));
            mbar_arrive_expect_tx(&full[s], (uint32_t)kTcTileBytes);
            tma_load_2d(dst, map, 0, y, &full[s], pol);
            tma_load_2d(dst + kTcBox, map, 64, y, &full[s], pol);
            if (keys) s_kissued = n + 1;
            else s_vissued = n + 1;
          }
        }
        ok = __shfl_sync(0xffffffffu, (int)ok, 0);
        if (!ok) break;
      }
    }
    // the last stages' releases (asynchronous arrivals) have landed before
    // the CTA gives up its shared memory
    for (int i = max(0, n - NS); ok && i < n; ++i)
      if (!mbar_wait_warp(&empty[i % NS], (i / NS) & 1, p.wait_ns)) {
        if (lane == 0) atomicExch(&s_fail, 1);
        ok = false;
      }
  } else if (warp == 1) {
    // ---- MMA issuer
    const TcSmem sm = {sk, vst, &q_full, k_full, k_empty, v_empty, s_full, p_ready, o_done};
    const bool ok = tc_issue<T>(p, sm, walk, wide);
    if (!ok && lane == 0) atomicExch(&s_fail, 1);
    // every MMA issued has completed before the tensor memory is released
    if (elect_one()) umma_commit(&all_done);
    __syncwarp();
    (void)mbar_wait_warp(&all_done, 0, p.wait_ns);
    __syncwarp();
  } else if (warp >= 4) {
    // ---- softmax: one query row per thread (TMEM lane)
    const int x = (warp - 4) >> 2;
    const int row = 32 * (warp & 3) + lane;
    const uint32_t lane_off = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t cs = tmem + lane_off + kTcColS + (uint32_t)(128 * x);
    const uint32_t co = tmem + lane_off + kTcColO + (uint32_t)(128 * x);
    const float sl2 = p.scale_log2;
    const int tid = threadIdx.x - 128;  // of 256
    const int gq = 16 % p.G, gb = 16 / p.G;
    int kbase = 0, steps = 0;
    bool dead = false, started = false;
    while (walk.next(p, pc)) {
      const int nt = pc.t1 - pc.t0;
      const int g0 = pc.ng * p.plan.rows_per;                       // the group's first query row
      const int grows = min(p.plan.rows_per, p.B * p.G - g0);       // its rows
      const int srows = min(128, grows - (wide ? 128 * x : 0));     // this stream's rows (may be <= 0)
      const int n = wide ? (srows > 0 ? nt : 0) : (nt + 1 - x) >> 1;  // steps: the stream's tiles
      // the queries, 128-byte swizzled; the MMAs that read the old ones, and
      // the loads of the old accumulators, have completed
      named_bar_sync(1, 256);
      {
        const int c = tid & 15;
        int b = (g0 + (tid >> 4)) / p.G, g = (g0 + (tid >> 4)) % p.G;
        const T* q = reinterpret_cast<const T*>(p.q) + (int64_t)pc.h * p.G * p.qsh + c * 8;
        unsigned char* dst = sq + (c >> 3) * kTcBox;
#pragma unroll 4
        for (int r = tid >> 4; r < nq * 128; r += 16) {
          const bool ok = r < grows;
          cp_async16(dst + (r >> 7) * kTcTileBytes + swz128(r & 127, c & 7), ok ? q + b * p.qsb + g * p.qsh : q, ok);
          g += gq;
          b += gb;
          if (g >= p.G) {
            g -= p.G;
            ++b;
          }
        }
      }
      if (!started) {
        named_bar_arrive(2, 256 + 64);
        started = true;
      }
      asm volatile("cp.async.wait_all;\n" ::: "memory");
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full);
      const bool active = 32 * (warp & 3) < srows;  // the warp's lanes hold query rows
      float m_used = -INFINITY, l = 0.f;
      for (int j = 0; j < n && !dead; ++j) {
        if (!mbar_wait_warp(&s_full[x], (steps + j) & 1, p.wait_ns)) {
          dead = true;
          break;
        }
        tc_fence_after();
        if (active) {
          const int valid = s_valid[(kbase + (wide ? j : 2 * j + x)) % kTcValidRing];
          // the maximum over the tile; the first 64 scores stay in registers,
          // the others are loaded again for P
          uint32_t v[64];
          tmem_ld32(cs + 64u, v);
          tmem_ld32(cs + 96u, v + 32);
          tmem_ld_wait();
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
          if (valid < kTcTile) {
#pragma unroll
            for (int k = 0; k < 64; ++k) mx[k & 3] = fmaxf(mx[k & 3], 64 + k < valid ? __uint_as_float(v[k]) : -INFINITY);
          } else {
#pragma unroll
            for (int k = 0; k < 64; ++k) mx[k & 3] = fmaxf(mx[k & 3], __uint_as_float(v[k]));
          }
          tmem_ld32(cs, v);
          tmem_ld32(cs + 32u, v + 32);
          tmem_ld_wait();
          if (valid < 64) {
#pragma unroll
            for (int k = 0; k < 64; ++k)
              if (k >= valid) v[k] = 0xff800000u;  // -infinity
          }
#pragma unroll
          for (int k = 0; k < 64; ++k) mx[k & 3] = fmaxf(mx[k & 3], __uint_as_float(v[k]));
          // log2 domain (scale > 0)
          const float m_new = fmaxf(m_used, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sl2);
          const bool resc = j > 0 && m_new > m_used + 8.f;
          if (j == 0) m_used = m_new;
          if (__any_sync(0xffffffffu, resc)) {
            // P stays below 2^8: O and l are rescaled only when the maximum
            // has grown by more since they last were
            if (!mbar_wait_warp(&o_done[x], (steps + j - 1) & 1, p.wait_ns)) {
              dead = true;
              break;
            }
            tc_fence_after();
            const float alpha = resc ? exp2_approx(m_used - m_new) : 1.f;
#pragma unroll 1
            for (int c = 0; c < 8; ++c) {
              uint32_t o[16];
              tmem_ld16(co + (uint32_t)(16 * c), o);
              tmem_ld_wait();
#pragma unroll
              for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
              tmem_st16(co + (uint32_t)(16 * c), o);
            }
            if (resc) {
              l *= alpha;
              m_used = m_new;
            }
          }
          const float nm = m_used == -INFINITY ? 0.f : -m_used;  // (no token so far: every P is 0)
          const uint64_t sl22 = pack_f2(sl2, sl2), nm2 = pack_f2(nm, nm);
          uint64_t ps[2] = {0ull, 0ull};
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            if (c == 2) {
              tmem_ld32(cs + 64u, v);
              tmem_ld32(cs + 96u, v + 32);
              tmem_ld_wait();
              if (valid < kTcTile) {
#pragma unroll
                for (int k = 0; k < 64; ++k)
                  if (64 + k >= valid) v[k] = 0xff800000u;
              }
            }
            uint32_t w[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              const int at = 32 * (c & 1) + 2 * k;
              const float2 t =
                  unpack_f2(fma_f2(pack_f2(__uint_as_float(v[at]), __uint_as_float(v[at + 1])), sl22, nm2));
              const float e0 = exp2_approx(t.x), e1 = exp2_approx(t.y);
              ps[k & 1] = add_f2(ps[k & 1], pack_f2(e0, e1));
              // one rounding to 16 bits, what the product takes; l is of the
              // unrounded ones (64 rows x 32768: 0.0023 from 64 bits, relative,
              // where probabilities in 32 bits give 0.0017, the output's own)
              w[k] = Elem<T>::cvt2(e0, e1);
            }
            tmem_st16(cs + (uint32_t)(16 * c), w);
          }
          const float2 sum = unpack_f2(add_f2(ps[0], ps[1]));
          l += sum.x + sum.y;
          tmem_st_wait();
        }
        // the step's values are there before P is reported; those of tokens
        // that do not count are zeroed (by both streams alike, where both
        // read the tile)
        const int tile = kbase + (wide ? j : 2 * j + x);
        const int valid_v = s_valid[tile % kTcValidRing];
        if ((warp & 3) == 0 || valid_v < kTcTile) {
          if (!mbar_wait_warp(&v_full[tile % vst], (tile / vst) & 1, p.wait_ns)) {
            dead = true;
            break;
          }
          if (valid_v < kTcTile && row >= valid_v) {
            unsigned char* vt = sv + (size_t)(tile % vst) * kTcTileBytes + row * 128;
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              *reinterpret_cast<uint4*>(vt + c * 16) = make_uint4(0u, 0u, 0u, 0u);
              *reinterpret_cast<uint4*>(vt + kTcBox + c * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
            fence_proxy_async_smem();
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[x]);
      }
      // the piece's partials: O relative to the maximum, not divided by the sum
      if (n > 0 && !dead && !mbar_wait_warp(&o_done[x], (steps + n - 1) & 1, p.wait_ns)) dead = true;
      const int64_t slot = (int64_t)blockIdx.x + pc.h * p.plan.n_groups + pc.ng;
      float f0 = 1.f, f1 = 0.f;
      if (!wide) {
        // both streams hold the row: joined here, each warp half of the dims
        // (either stream's accumulator is in the warp's own lanes)
        s_m[x][row] = m_used;
        if (x == 1) s_l1[row] = l;
        tc_fence_after();
        tc_fence_before();
        named_bar_sync(1, 256);
        const float m0 = s_m[0][row], m1 = s_m[1][row];
        m_used = fmaxf(m0, m1);
        const float ref = m_used == -INFINITY ? 0.f : m_used;
        f0 = exp2_approx(m0 - ref);
        f1 = exp2_approx(m1 - ref);
        l = f0 * l + f1 * s_l1[row];  // (stream 0 stores it)
      }
      if (active && !dead) {
        tc_fence_after();
        const int64_t set = wide ? (slot * 2 + x) * 128 : slot * 128;
        // 8 dims of all rows, then the next 8: a warp's stores are 1 KB in a piece
        float* dst = p.plan.part_o + set * kD + row * 8;
        if (row < srows && (wide || x == 0)) p.plan.part_ml[set + row] = make_float2(m_used, l);
        const bool both = !wide && nt > 1;  // (one tile: stream 1 has no accumulator)
        const uint32_t ca = tmem + lane_off + kTcColO + (wide ? (uint32_t)(128 * x) : 0u);
        const int c0 = wide ? 0 : 4 * x, c1 = wide ? 8 : 4 * x + 4;
#pragma unroll 1
        for (int c = c0; c < c1; ++c) {
          uint32_t v[16], u[16];
          tmem_ld16(ca + (uint32_t)(16 * c), v);
          if (both) tmem_ld16(ca + (uint32_t)(128 + 16 * c), u);
          tmem_ld_wait();
          if (!wide) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
              v[i] = __float_as_uint(__uint_as_float(v[i]) * f0 + (both ? __uint_as_float(u[i]) * f1 : 0.f));
          }
          if (row < srows)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              *reinterpret_cast<uint4*>(dst + (2 * c + (i >> 1)) * 128 * 8 + (i & 1) * 4) =
                  make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        }
        tc_fence_before();
      }
      steps += n;
      kbase += nt;
    }
    if (!started) named_bar_arrive(2, 256 + 64);  // (no piece)
    if (dead && lane == 0) atomicExch(&s_fail, 1);
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && s_fail) {
    set_err(p.err, HC_ERR_TIMEOUT);
    // the copies still in flight land before the CTA's shared memory is released
    for (int j = max(0, s_kissued - kTcK); j < s_kissued; ++j)
      (void)mbar_wait_sleep(&k_full[j % kTcK], (j / kTcK) & 1, p.wait_ns);
    for (int j = max(0, s_vissued - vst); j < s_vissued; ++j)
      (void)mbar_wait_sleep(&v_full[j % vst], (j / vst) & 1, p.wait_ns);
  }
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512u);
  }
}

// Rows a CTA of the CUDA-core form: the fewest of 16, 32, 64 that hold the
// batch's (a tile's work is the same for the rows it does not fill).
static int sp_rows(int rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : 64; }

static PrefixPlan sp_plan(int dtype, int B, int G, int sms) {
  PrefixPlan pl = {};
  const int rows = B * G;
  if (dtype == HC_F32) {
    pl.rows_per = pl.stream_rows = sp_rows(rows);
    pl.gran = kSpTok;
    pl.streams = 1;
    pl.n_ctas = 2 * sms;
  } else {
    pl.rows_per = rows > 128 ? 256 : 128;
    pl.stream_rows = 128;
    pl.gran = kTcTile;
    pl.streams = pl.rows_per / 128;
    pl.n_ctas = sms;
  }
  pl.n_groups = (rows + pl.rows_per - 1) / pl.rows_per;
  return pl;
}

static size_t sp_bytes(const PrefixPlan& pl, int KV, size_t* ml_at) {
  const size_t rows = ((size_t)pl.n_ctas + (size_t)KV * pl.n_groups) * pl.streams * pl.stream_rows;
  if (ml_at) *ml_at = rows * kD * sizeof(float);
  return (rows * (kD * sizeof(float) + sizeof(float2)) + 255) & ~(size_t)255;
}

size_t shared_prefix_ws_bytes(int dtype, int B, int KV, int G) {
  return sp_bytes(sp_plan(dtype, B, G, device_sms(current_device())), KV, nullptr);
}

// Raises a kernel's dynamic shared-memory limit once per device.
template <typename K>
static bool sp_allow_smem(K kern, size_t bytes, bool (&done)[kMaxDevices], int dev) {
  std::lock_guard<std::mutex> g(host_lock());
  if (done[dev]) return true;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != cudaSuccess) return false;
  done[dev] = true;
  return true;
}

template <typename K, typename... Args>
static int sp_pdl_launch(K kern, int grid, int threads, size_t smem, cudaStream_t st, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned int)grid);
  cfg.blockDim = dim3((unsigned int)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, args...) == cudaSuccess ? HC_OK : HC_ERR_CUDA;
}

template <int RT, int RPT>
static int sp_launch_f32(const SPParams& p, int dev, cudaStream_t st) {
  static bool done[kMaxDevices];
  constexpr size_t smem = sp_smem(RT);
  if (!sp_allow_smem(shared_prefix_kernel<RT, RPT>, smem, done, dev)) return HC_ERR_CUDA;
  return sp_pdl_launch(shared_prefix_kernel<RT, RPT>, p.plan.n_ctas, 8 * RT / RPT, smem, st, p);
}

template <typename T>
static int sp_launch_tc(const SPParams& p, int dtype, int dev, cudaStream_t st) {
  static bool done[kMaxDevices];
  CUtensorMap tmk, tmv;
  const long long rows = (long long)p.n_blocks * kPage;
  if (!pool_tensor_map(&tmk, p.kp, rows, dtype, kTcTile)) return HC_ERR_CUDA;
  if (!pool_tensor_map(&tmv, p.vp, rows, dtype, kTcTile)) return HC_ERR_CUDA;
  if (!sp_allow_smem(shared_prefix_tc_kernel<T>, kTcSmem, done, dev)) return HC_ERR_CUDA;
  return sp_pdl_launch(shared_prefix_tc_kernel<T>, p.plan.n_ctas, kTcThreads, kTcSmem, st, p, tmk, tmv);
}

int shared_prefix_dispatch(int dtype, SPParams& p, void* ws, size_t ws_bytes, cudaStream_t st) {
  const int dev = current_device();
  if (dev < 0) return HC_ERR_CUDA;
  p.plan = sp_plan(dtype, p.B, p.G, device_sms(dev));
  size_t ml_at;
  if (!ws || ws_bytes < sp_bytes(p.plan, p.KV, &ml_at)) return HC_ERR_WORKSPACE;
  p.plan.part_o = reinterpret_cast<float*>(ws);
  p.plan.part_ml = reinterpret_cast<float2*>(reinterpret_cast<unsigned char*>(ws) + ml_at);
  p.wait_ns = wait_limit_ns(kMbarTimeoutNs);
  p.stall = injected_stall();
  switch (dtype) {
    case HC_F32:
      switch (p.plan.rows_per) {
        case 16: return sp_launch_f32<16, 2>(p, dev, st);
        case 32: return sp_launch_f32<32, 4>(p, dev, st);
        default: return sp_launch_f32<64, 4>(p, dev, st);
      }
    case HC_BF16: return sp_launch_tc<__nv_bfloat16>(p, dtype, dev, st);
    case HC_F16: return sp_launch_tc<__half>(p, dtype, dev, st);
    default: return HC_ERR_DTYPE;
  }
}

}  // namespace hc
