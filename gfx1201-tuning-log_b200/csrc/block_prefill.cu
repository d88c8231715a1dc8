// Attention of many query tokens a sequence over a block-scaled fp8 paged cache
// (sm_100a): prompts and chunks of prompts, more than kMaxRows (query token, head)
// rows per kv head.
//
// A CTA holds two 128-row query tiles (tokens x the heads of one kv head) and walks
// 128-key tiles, each read once for both:
//   S = Q K^T   kind::f8f6f4, Q as two e4m3 terms (8 significant bits), K as stored;
//   O += P V    kind::f16, P from tensor memory, V converted to f16 in shared memory.
// Splitting P into two e4m3 terms instead keeps V as stored but costs the softmax
// threads five operations a score; converting V costs four warps four operations a
// code, a quarter as many codes as scores, and P keeps f16's 11 bits.  An e4m3 code's
// bits shifted by one are the f16 of 2^-8 its value, subnormals included (codes of
// NaN become 480: no non-finite value enters the product).
//
// Block scales ks, vs as in block_decode.cu: x = sm_scale log2(e) ks (q . k) + log2(vs),
// P = 2^(x - m), and the softmax sum adds P / vs.  A softmax thread is a query row:
// it finds the tile's maximum of x (the block's raw maximum, then the scale), moves m
// when it is passed by 2^4, and then forms P in f16 pairs.  P <= 2^4.  The sum of a
// block is taken in f16 pairs and joined in fp32; where a block's scale is below
// 2^-10 of the largest seen, whose P may underflow though its weight P / vs does
// not, the sum is formed from fp32 exponentials.
//
// Shares of the batch's tiles as in block_decode.cu, an item being the two query
// tiles of a kv head; what a cut item's shares leave is joined by a second kernel.
//
// Roles: 8 softmax warps (four a query tile), 4 that convert V, an MMA warp a query
// tile (each waits for its own P V before its next Q K^T, which overwrites P: the
// other tile's products fill the gap), a TMA warp, a warp for the blocks' scales.

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "b200kv.h"
#include "b200kv_common.cuh"
#include "block_attn.cuh"
#include "fp8_terms.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"

namespace b200kv {
namespace {

constexpr int kHead = 128;
constexpr int kTile = 128;               // keys of a tile, rows of a query tile
constexpr int kBytes8 = kTile * kHead;   // an 8-bit operand
constexpr int kKStages = 3, kVStages = 2, kScStages = 4;
constexpr int kMaxPages = 8;
constexpr int kSoftWarps = 8, kConvWarp = 8, kConvWarps = 4, kMmaWarp = 12, kTmaWarp = 14, kScaleWarp = 15;
constexpr int kThreads = 512;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLazy = 4.f;
constexpr float kFar = 10.f;             // log2 of how far apart blocks' scales may be for f16 sums
constexpr float kMinScale = 8.2718061e-25f, kMaxScale = 1.2089258e24f;  // 2^-80, 2^80
constexpr float kNone = -1e30f;          // the reference of a row that has seen no key
constexpr float kTiny = 1e-37f;          // a factor of zero becomes it, so that a hidden key stays -inf

// shared memory
constexpr int kOffQ = 0;                          // [query tile][hi, lo]
constexpr int kOffK = kOffQ + 4 * kBytes8;
constexpr int kOffV8 = kOffK + kKStages * kBytes8;
constexpr int kOffV16 = kOffV8 + kVStages * kBytes8;  // [stage][dims 0-63, 64-127][key][128 B]
constexpr int kSmem = kOffV16 + kVStages * 2 * kBytes8;

struct Shared {
  uint64_t k_full[kKStages], k_empty[kKStages];
  uint64_t v8_full[kVStages], v8_empty[kVStages], v16_full[kVStages], v16_empty[kVStages];
  uint64_t sc_full[kScStages], sc_empty[kScStages];
  uint64_t q_full[2], q_free[2], s_full[2], p_full[2], pv_done[2];
  uint32_t tmem;
  alignas(16) float4 scale[kScStages][kMaxPages];  // ks, log2 vs, 1 / vs, the tile's largest log2 vs
  int first[4];                                    // of this share: sequence, head of the CTA's, pair, tile
  int warp_sum[kThreads / 32];
};

// Two query tiles of a sequence and the key tiles they see.
struct Pair {
  int row0, qlen, q0, kv_end;  // of the sequence
  int tokens;                  // of a query tile
  int t0;                      // first token of tile 0
  KeyTiles keys;
  // positions of the first and last query of tile X; last < first where it is empty
  __device__ __forceinline__ int first(int X) const { return q0 + t0 + X * tokens; }
  __device__ __forceinline__ int last(int X) const { return q0 + min(qlen, t0 + (X + 1) * tokens) - 1; }
};
struct Seq {
  int row0, qlen, q0, kv_end, pairs;
};
__device__ __forceinline__ Seq seq_of(const BlockAttnParams& p, int seq) {
  Seq s;
  s.row0 = p.cu[seq];
  s.qlen = p.cu[seq + 1] - s.row0;
  const int total = p.lens[seq];
  s.q0 = total - s.qlen;
  s.kv_end = min(total, p.max_blocks << p.shift);
  const int tokens = kTile / p.group;
  const bool many = s.qlen > kMaxRows || s.qlen * p.group > kMaxRows;
  s.pairs = many ? (s.qlen - 1) / (2 * tokens) + 1 : 0;
  return s;
}
__device__ __forceinline__ Pair pair_of(const BlockAttnParams& p, const Seq& s, int pair) {
  Pair r;
  r.row0 = s.row0;
  r.qlen = s.qlen;
  r.q0 = s.q0;
  r.kv_end = s.kv_end;
  r.tokens = kTile / p.group;
  r.t0 = pair * 2 * r.tokens;
  r.keys = key_tiles(p, s.q0 + r.t0, min(s.kv_end, s.q0 + min(s.qlen, r.t0 + 2 * r.tokens)));
  return r;
}
// whether no query of tile X sees key tile t
__device__ __forceinline__ bool skips(const BlockAttnParams& p, const Pair& r, int X, int t) {
  const int lo = t * kTile, first = r.first(X), last = r.last(X);
  return last < first || lo > last || lo >= r.kv_end ||
         (p.window > 0 && lo + kTile - 1 <= first - p.window && lo >= p.sinks);
}

// A CTA's share, segment by segment.
struct Walk {
  const BlockAttnParams& p;
  Seq s;
  Pair r;
  int seq, sub, pair, off;
  int left;
  int64_t item;
  __device__ Walk(const BlockAttnParams& p_, const Shared& S, int64_t begin, int count) : p(p_), left(count) {
    seq = S.first[0];
    sub = S.first[1];
    pair = S.first[2];
    off = S.first[3];
    item = begin - off;
    s = seq_of(p, seq);
    r = pair_of(p, s, pair);
  }
  __device__ __forceinline__ int count() const { return min(r.keys.count - off, left); }
  __device__ __forceinline__ int kh() const { return blockIdx.x % p.slots * p.heads + sub; }
  __device__ __forceinline__ void next() {
    left -= count();
    if (left <= 0) return;
    item += r.keys.count;
    off = 0;
    do {
      if (++pair >= s.pairs) {
        pair = 0;
        if (s.pairs == 0 || ++sub == p.heads) {
          sub = 0;
          if (++seq >= p.num_seqs) {  // not reached while tiles are left
            left = 0;
            return;
          }
          s = seq_of(p, seq);
          if (s.pairs == 0) continue;
        }
      }
      r = pair_of(p, s, pair);
    } while (s.pairs == 0 || r.keys.count == 0);
  }
};

__device__ __forceinline__ uint32_t pack_h2(float a, float b) {  // a in the low half
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %2, %1;" : "=r"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint32_t ex2_h2(uint32_t x) {
  uint32_t y;
  asm("ex2.approx.f16x2 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t add_h2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ float sum_h2(uint32_t x) {
  float a, b;
  asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n cvt.f32.f16 %0, l;\n cvt.f32.f16 %1, h;\n}"
      : "=f"(a), "=f"(b)
      : "r"(x));
  return a + b;
}
// two e4m3 codes (bytes 2 s, 2 s + 1 of w) -> f16x2 of 2^-8 their values
template <int S>
__device__ __forceinline__ uint32_t half2_of(uint32_t w) {
  const uint32_t t = __byte_perm(w, 0u, S ? 0x3424 : 0x1404);  // codes in the high bytes
  return (t & 0x80008000u) | ((t & 0x7F007F00u) >> 1);
}

__global__ void __launch_bounds__(kThreads, 1)
    block_prefill_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                         const BlockAttnParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ Shared S;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  if (tid == 0) {
    griddep_launch_dependents();
    for (int s = 0; s < kKStages; ++s) {
      mbar_init(&S.k_full[s], 1);
      mbar_init(&S.k_empty[s], 2);  // one arrival a query tile
    }
    for (int s = 0; s < kVStages; ++s) {
      mbar_init(&S.v8_full[s], 1);
      mbar_init(&S.v8_empty[s], kConvWarps);
      mbar_init(&S.v16_full[s], kConvWarps);
      mbar_init(&S.v16_empty[s], 2);
    }
    for (int s = 0; s < kScStages; ++s) {
      mbar_init(&S.sc_full[s], 1);
      mbar_init(&S.sc_empty[s], kSoftWarps);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&S.q_full[b], 4);
      mbar_init(&S.q_free[b], 1);
      mbar_init(&S.s_full[b], 1);
      mbar_init(&S.p_full[b], 4);
      mbar_init(&S.pv_done[b], 1);
    }
    fence_mbar_init();
  }
  if (warp == kMmaWarp) tc::tmem_alloc(&S.tmem, 512);
  griddep_wait();  // lengths, tables and q may be the previous kernel's

  // ---- this CTA's share ----------------------------------------------------------------
  const int per = (p.num_seqs + kThreads - 1) / kThreads;
  const int s_lo = min(p.num_seqs, tid * per), s_hi = min(p.num_seqs, s_lo + per);
  auto seq_tiles = [&](int seq) {
    const Seq s = seq_of(p, seq);
    int n = 0;
    for (int i = 0; i < s.pairs; ++i) n += pair_of(p, s, i).keys.count;
    return n;
  };
  int mine = 0;
  for (int s = s_lo; s < s_hi; ++s) mine += seq_tiles(s);
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) S.warp_sum[warp] = incl;
  if (tid == 0) p.records[blockIdx.x * 8] = 0;
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  int before = 0, tiles = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += S.warp_sum[w];
    tiles += S.warp_sum[w];
  }
  const int64_t total = (int64_t)tiles * p.heads;
  const int share = blockIdx.x / p.slots;
  const int64_t shares = min((int64_t)(gridDim.x / p.slots), total);
  const bool busy = share < shares;
  const int64_t begin = busy ? share_begin(share, total, shares) : 0;
  const int count = busy ? (int)(share_begin(share + 1, total, shares) - begin) : 0;
  if (busy) {
    int at = before + incl - mine;
    if (begin >= (int64_t)at * p.heads && begin < (int64_t)(at + mine) * p.heads)
      for (int s = s_lo; s < s_hi; ++s) {
        const int n = seq_tiles(s);
        if (begin < (int64_t)(at + n) * p.heads) {
          int rel = (int)(begin - (int64_t)at * p.heads);
          const Seq q = seq_of(p, s);
          S.first[0] = s;
          S.first[1] = rel / n;
          rel %= n;
          int pair = 0;
          for (int m; rel >= (m = pair_of(p, q, pair).keys.count); ++pair) rel -= m;
          S.first[2] = pair;
          S.first[3] = rel;
          break;
        }
        at += n;
      }
  }
  __syncthreads();
  const uint32_t tbase = S.tmem;  // S (then P) of tile 0, 1, O of tile 0, 1: 128 columns each

  if (warp == kScaleWarp) {
    // queries that see no key and whose pair has none: zeros
    for (int s = blockIdx.x; s < p.num_seqs; s += gridDim.x) {
      const Seq q = seq_of(p, s);
      if (q.pairs == 0 || (q.q0 >= 0 && q.kv_end > 0)) continue;
      for (int i = 0; i < q.pairs; ++i) {
        const Pair r = pair_of(p, q, i);
        if (r.keys.count) continue;
        const int n = min(q.qlen - r.t0, 2 * r.tokens), width = p.hkv * p.group * kHead;
        for (int64_t e = lane; e < (int64_t)n * width; e += 32)
          p.out[(int64_t)(q.row0 + r.t0 + e / width) * p.o_st + e % width / kHead * p.o_sh + e % kHead] =
              __float2bfloat16_rn(0.f);
      }
    }
  }
  if (!busy) {
  } else if (warp == kTmaWarp) {
    // ---------------- TMA producer ------------------------------------------------------
    const int ppt = kTile >> p.shift, bs = 1 << p.shift, tpw = 32 / ppt;
    if (lane == 0) {
      tma_prefetch_desc(&kmap);
      tma_prefetch_desc(&vmap);
    }
    int i = 0;
    bool ok = true;
    for (Walk w(p, S, begin, count); w.left > 0 && ok; w.next()) {
      const int n = w.count(), kh = w.kh();
      const int32_t* row = p.bt + (int64_t)w.seq * p.bt_stride;
      auto entry = [&](int j0) {
        const int j = j0 + lane / ppt;
        if (j >= n) return -1;
        const int page = w.r.keys.tile(w.off + j) * ppt + lane % ppt;
        return page << p.shift < w.r.kv_end ? __ldg(row + page) : -1;
      };
      int cur = entry(0), nxt = entry(tpw);
      for (int j = 0; j < n; ++j, ++i) {
        const int ks = i % kKStages, vs = i % kVStages, j0 = j % tpw;
        if (j > 0 && j0 == 0) {
          cur = nxt;
          nxt = entry(j + tpw);
        }
        const int keys = min(kTile, w.r.kv_end - w.r.keys.tile(w.off + j) * kTile);
        const int pages = (keys + bs - 1) >> p.shift;
        const int pg = lane - j0 * ppt;
        const bool mine = pg >= 0 && pg < pages;
        int free = 1;
        if (lane == 0 && i >= kKStages) free = mbar_wait_bounded(&S.k_empty[ks], (i / kKStages - 1) & 1);
        if (!__shfl_sync(0xffffffffu, free, 0)) {
          ok = false;
          break;
        }
        if (lane == 0) mbar_arrive_expect_tx(&S.k_full[ks], (uint32_t)(pages * bs * kHead));
        __syncwarp();
        if (mine) tma_load_4d(smem + kOffK + ks * kBytes8 + pg * bs * kHead, &kmap, 0, kh, 0, cur, &S.k_full[ks]);
        if (lane == 0 && i >= kVStages) free = mbar_wait_bounded(&S.v8_empty[vs], (i / kVStages - 1) & 1);
        if (!__shfl_sync(0xffffffffu, free, 0)) {
          // K of this tile is in flight, V is not: the consumers' waits give up too
          if (lane == 0) mbar_wait_bounded(&S.k_full[ks], (i / kKStages) & 1);
          ok = false;
          break;
        }
        if (lane == 0) mbar_arrive_expect_tx(&S.v8_full[vs], (uint32_t)(pages * bs * kHead));
        __syncwarp();
        if (mine) tma_load_4d(smem + kOffV8 + vs * kBytes8 + pg * bs * kHead, &vmap, 0, kh, 0, cur, &S.v8_full[vs]);
      }
    }
    if (lane == 0) {  // every copy issued has landed before the CTA may exit
      for (int j = max(0, i - kKStages); j < i; ++j) mbar_wait_bounded(&S.k_full[j % kKStages], (j / kKStages) & 1);
      for (int j = max(0, i - kVStages); j < i; ++j) mbar_wait_bounded(&S.v8_full[j % kVStages], (j / kVStages) & 1);
    }
    __syncwarp();
  } else if (warp == kScaleWarp) {
    // ---------------- the blocks' scales ------------------------------------------------
    const int ppt = kTile >> p.shift;
    int i = 0;
    bool failed = false;
    for (Walk w(p, S, begin, count); w.left > 0; w.next()) {
      const int n = w.count(), kh = w.kh();
      const int32_t* row = p.bt + (int64_t)w.seq * p.bt_stride;
      auto load = [&](int j) {  // this lane's page of tile j
        float2 v = make_float2(0.f, 0.f);
        const int page = j < n ? w.r.keys.tile(w.off + j) * ppt + lane : 0;
        if (j < n && lane < ppt && page << p.shift < w.r.kv_end) {
          const int blk = __ldg(row + page);
          if (blk >= 0 && blk < p.num_blocks)  // else the block reads as zeros
            v = make_float2(p.ks[(int64_t)blk * p.ks0 + (int64_t)kh * p.ks1], p.vs[(int64_t)blk * p.vs0 + (int64_t)kh * p.vs1]);
        }
        return v;
      };
      float2 nxt = load(0);
      for (int j = 0; j < n; ++j, ++i) {
        const int st = i % kScStages;
        const float2 v = nxt;
        nxt = load(j + 1);
        const float vs = fminf(fmaxf(v.y, kMinScale), kMaxScale);
        const float lvs = __log2f(vs);
        const bool real = lane < ppt && (w.r.keys.tile(w.off + j) * ppt + lane) << p.shift < w.r.kv_end;
        float top = real ? lvs : -100.f;
#pragma unroll
        for (int o = 1; o < kMaxPages; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (i >= kScStages && !failed) failed = !mbar_wait_bounded(&S.sc_empty[st], (i / kScStages - 1) & 1);
        if (lane < ppt) S.scale[st][lane] = make_float4(v.x, lvs, __frcp_rn(vs), top);
        __syncwarp();
        if (lane == 0) mbar_arrive(&S.sc_full[st]);
      }
    }
  } else if (warp >= kMmaWarp && warp < kMmaWarp + 2) {
    // ---------------- the products of one query tile --------------------------------------
    if (lane == 0) {
      constexpr uint32_t kIdescQK = tc::idesc_f16_f32(kTile, kTile, false);
      constexpr uint32_t kIdescPV = tc::idesc_f16_f32(kTile, kHead, true);
      const int X = warp - kMmaWarp;
      const uint32_t a_q = smem_u32(smem + kOffQ + 2 * X * kBytes8), a_k = smem_u32(smem + kOffK);
      const uint32_t a_v = smem_u32(smem + kOffV16), t_s = tbase + X * kTile, t_o = tbase + 2 * kTile + X * kTile;
      bool failed = false;
      int i = 0, done = 0, seg = 0;  // done: tiles of this query tile
      for (Walk w(p, S, begin, count); w.left > 0; w.next(), ++seg) {
        const int n = w.count();
        if (!failed) failed = !mbar_wait_bounded(&S.q_full[X], seg & 1);
        bool first = true;
        for (int j = 0; j < n; ++j, ++i) {
          const int ks = i % kKStages, vs = i % kVStages;
          if (skips(p, w.r, X, w.r.keys.tile(w.off + j))) {
            // the tile's buffers are released once they have been filled, so that no
            // arrival runs ahead of its phase
            if (!failed) failed = !mbar_wait_bounded(&S.k_full[ks], (i / kKStages) & 1);
            mbar_arrive(&S.k_empty[ks]);
            if (!failed) failed = !mbar_wait_bounded(&S.v16_full[vs], (i / kVStages) & 1);
            mbar_arrive(&S.v16_empty[vs]);
            continue;
          }
          if (!failed) failed = !mbar_wait_bounded(&S.k_full[ks], (i / kKStages) & 1);
          if (!failed) {
            tc::fence_after_sync();
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
              for (int d = 0; d < 4; ++d)
                tc::mma_f8(t_s, tc::sdesc_sw128(a_q + t * kBytes8 + d * 32, 16, 1024),
                           tc::sdesc_sw128(a_k + ks * kBytes8 + d * 32, 16, 1024), kIdescQK, (t | d) != 0);
          }
          tc::commit(&S.s_full[X]);
          tc::commit(&S.k_empty[ks]);
          if (!failed) failed = !mbar_wait_bounded(&S.p_full[X], done & 1);
          if (!failed) failed = !mbar_wait_bounded(&S.v16_full[vs], (i / kVStages) & 1);
          if (!failed) {
            tc::fence_after_sync();
#pragma unroll
            for (int c = 0; c < 8; ++c)
              tc::mma_f16_ts(t_o, t_s + 8 * c, tc::sdesc_sw128(a_v + vs * 2 * kBytes8 + c * 16 * 128, kBytes8, 1024),
                             kIdescPV, !first || c != 0);
          }
          tc::commit(&S.pv_done[X]);
          tc::commit(&S.v16_empty[vs]);
          // the next Q K^T overwrites P
          if (!failed) failed = !mbar_wait_bounded(&S.pv_done[X], done & 1);
          first = false;
          ++done;
        }
        mbar_arrive(&S.q_free[X]);
      }
    }
    __syncwarp();
  } else if (warp >= kConvWarp && warp < kConvWarp + kConvWarps) {
    // ---------------- V codes to f16 ----------------------------------------------------
    const int ct = tid - kConvWarp * 32, c = ct & 7;  // 16 codes, dims 16 c .., of keys ct / 8 + 16 e
    bool failed = false;
    for (int i = 0; i < count; ++i) {
      const int st = i % kVStages;
      if (!failed) failed = !mbar_wait_bounded(&S.v8_full[st], (i / kVStages) & 1);
      if (i >= kVStages && !failed) failed = !mbar_wait_bounded(&S.v16_empty[st], (i / kVStages - 1) & 1);
      const uint8_t* src = smem + kOffV8 + st * kBytes8;
      uint8_t* dst = smem + kOffV16 + st * 2 * kBytes8 + (c >> 2) * kBytes8;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int key = ct / 8 + 16 * e;
        const uint4 v = *reinterpret_cast<const uint4*>(src + swz(key, c));
        const uint4 a = make_uint4(half2_of<0>(v.x), half2_of<1>(v.x), half2_of<0>(v.y), half2_of<1>(v.y));
        const uint4 b = make_uint4(half2_of<0>(v.z), half2_of<1>(v.z), half2_of<0>(v.w), half2_of<1>(v.w));
        // the two halves' chunks lie in the same banks: lanes of the second store b first
        const int odd = c >> 2;
        *reinterpret_cast<uint4*>(dst + swz(key, 2 * (c & 3) + odd)) = odd ? b : a;
        *reinterpret_cast<uint4*>(dst + swz(key, 2 * (c & 3) + (odd ^ 1))) = odd ? a : b;
      }
      tc::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&S.v8_empty[st]);
        mbar_arrive(&S.v16_full[st]);
      }
    }
  } else if (warp < kSoftWarps) {
    // ---------------- softmax: a thread is a query row ------------------------------------
    const int X = warp >> 2, row = tid & 127;
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t t_s = tbase + X * kTile + lane_off, t_o = tbase + 2 * kTile + X * kTile + lane_off;
    bool failed = false;
    int i = 0, done = 0, seg = 0;
    for (Walk w(p, S, begin, count); w.left > 0; w.next(), ++seg) {
      const int n = w.count(), kh = w.kh();
      const Pair& r = w.r;
      const int t = r.t0 + X * r.tokens + row / p.group;
      const bool valid = row < r.tokens * p.group && t < r.qlen;
      const int pos = valid ? r.q0 + t : r.last(X);
      const int64_t q_row = r.row0 + (valid ? t : 0);
      const int head = kh * p.group + row % p.group;
      float coef;
      // the issuer is through with the segment before (one whose tiles this query tile
      // skips would else let these warps run ahead of its barriers)
      if (seg > 0 && !failed) failed = !mbar_wait_bounded(&S.q_free[X], (seg - 1) & 1);
      {
        // Q: a power-of-two prescale (maximum in [2^7, 2^8)) with the sign of sm_scale, two
        // terms; the row is read twice, the second time from L1
        const uint4* src = reinterpret_cast<const uint4*>(p.q + q_row * p.q_st + (int64_t)head * p.q_sh);
        const uint4 zero = make_uint4(0, 0, 0, 0);
        float mx = 0.f;
#pragma unroll 4
        for (int c = 0; c < 16; ++c) {
          const uint4 w4 = valid ? __ldg(src + c) : zero;
          const uint32_t u[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mx = fmaxf(mx, fmaxf(fabsf(__uint_as_float(u[k] << 16)), fabsf(__uint_as_float(u[k] & 0xFFFF0000u))));
        }
        const int E = (int)((__float_as_uint(mx) >> 23) & 0xFF);
        int sh = (E == 0xFF || mx == 0.f) ? 0 : 134 - E;
        sh = max(-126, min(126, sh));
        float up = __uint_as_float((uint32_t)(sh + 127) << 23);
        if (p.sm_scale < 0.f) up = -up;
        uint8_t* q = smem + kOffQ + 2 * X * kBytes8;
#pragma unroll 1
        for (int c = 0; c < 8; ++c) {
          float v[16];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint4 w4 = valid ? __ldg(src + 2 * c + h) : zero;
            const uint32_t u[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              v[8 * h + 2 * k] = __uint_as_float(u[k] << 16) * up;
              v[8 * h + 2 * k + 1] = __uint_as_float(u[k] & 0xFFFF0000u) * up;
            }
          }
          uint4 hi, lo;
          pack16<1>(v, hi, lo);
          *reinterpret_cast<uint4*>(q + swz(row, c)) = hi;
          *reinterpret_cast<uint4*>(q + kBytes8 + swz(row, c)) = lo;
        }
        coef = fabsf(p.sm_scale) * kLog2e * __uint_as_float((uint32_t)(127 - sh) << 23);
      }
      tc::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&S.q_full[X]);

      float ref = kNone, l = 0.f, lvs_top = -100.f;
      bool first = true;
      for (int j = 0; j < n; ++j, ++i) {
        const int st = i % kScStages, tile = r.keys.tile(w.off + j), key0 = tile * kTile;
        if (!failed) failed = !mbar_wait_bounded(&S.sc_full[st], (i / kScStages) & 1);
        if (skips(p, r, X, tile)) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&S.sc_empty[st]);
          continue;
        }
        if (!failed) failed = !mbar_wait_bounded(&S.s_full[X], done & 1);
        tc::fence_after_sync();
        const bool open = key0 + kTile - 1 <= r.first(X) && key0 + kTile <= r.kv_end &&
                          (p.window == 0 || key0 > r.last(X) - p.window || key0 + kTile <= p.sinks);
        // which of 32 keys the row sees, one bit a key
        auto visible = [&](int key) {
          auto below = [&](int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; };  // keys before key + n
          uint32_t m = below(min(pos + 1, r.kv_end) - key);
          if (p.window > 0) m &= ~below(pos - p.window + 1 - key) | below(p.sinks - key);
          return m;
        };
        const float4* sc = S.scale[st];
        lvs_top = fmaxf(lvs_top, sc[0].w);
        // the tile's maximum (loops kept short: the softmax warps' code has to stay in the
        // instruction caches beside the other roles')
        float top = kNone;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          float s[32];
          tc::ld32_wait(t_s + 32 * c, s);
          if (!open) {
            const uint32_t m = visible(key0 + 32 * c);
#pragma unroll
            for (int k = 0; k < 32; ++k) s[k] = m >> k & 1 ? s[k] : -INFINITY;
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float m = s[16 * h];
#pragma unroll
            for (int k = 1; k < 15; k += 2) m = fmaxf(m, fmaxf(s[16 * h + k], s[16 * h + k + 1]));
            m = fmaxf(m, s[16 * h + 15]);
            const float4 f = sc[(32 * c + 16 * h) >> p.shift];
            if (m != -INFINITY) top = fmaxf(top, fmaf(m, coef * f.x, f.y));
          }
        }
        const bool moves = top > ref + kLazy;
        if (__any_sync(0xffffffffu, moves)) {
          const float now = moves ? top : ref, alpha = ex2(ref - now);
          ref = now;
          l *= alpha;
          if (!first) {  // the product before this tile's is done: its issuer waited for it
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              float o[32];
              tc::ld32_wait(t_o + 32 * c, o);
#pragma unroll
              for (int k = 0; k < 32; ++k) o[k] *= alpha;
              tc::st32(t_o + 32 * c, o);
            }
            tc::wait_st();
          }
        }
        first = false;
        // P, 32 keys at a time, over the scores already read
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          float s[32], pk[16];
          tc::ld32_wait(t_s + 32 * c, s);
          if (!open) {
            const uint32_t m = visible(key0 + 32 * c);
#pragma unroll
            for (int k = 0; k < 32; ++k) s[k] = m >> k & 1 ? s[k] : -INFINITY;
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float4 f = sc[(32 * c + 16 * h) >> p.shift];
            const float mul = fmaxf(coef * f.x, kTiny), add = f.y - ref;
            float* y = s + 16 * h;
            uint32_t e[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              y[2 * k] = fmaf(y[2 * k], mul, add);
              y[2 * k + 1] = fmaf(y[2 * k + 1], mul, add);
              e[k] = ex2_h2(pack_h2(y[2 * k], y[2 * k + 1]));
              pk[8 * h + k] = __uint_as_float(e[k]);
            }
            if (f.y > lvs_top - kFar) {  // uniform over the CTA
#pragma unroll
              for (int o = 4; o > 0; o >>= 1)
#pragma unroll
                for (int k = 0; k < o; ++k) e[k] = add_h2(e[k], e[k + o]);
              l = fmaf(sum_h2(e[0]), f.z, l);
            } else {
              float sum = 0.f;
#pragma unroll
              for (int k = 0; k < 16; ++k) sum += ex2(y[k]);
              l = fmaf(sum, f.z, l);
            }
          }
          tc::st(t_s + 16 * c, pk);
        }
        tc::wait_st();
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&S.sc_empty[st]);
          mbar_arrive(&S.p_full[X]);
        }
        ++done;
      }

      // ---- the segment's end ----------------------------------------------------------------
      const bool whole = n == r.keys.count;
      float* part = p.partials + (int64_t)(2 * blockIdx.x + (w.item >= begin ? 1 : 0)) * kPartialFloats;
      if (!first && !failed) failed = !mbar_wait_bounded(&S.pv_done[X], (done - 1) & 1);
      tc::fence_after_sync();
      const float f = whole ? (l > 0.f ? __fdividef(256.f, l) : 0.f) : 256.f;  // V entered as 2^-8 V
      __nv_bfloat16* dst = p.out + q_row * p.o_st + (int64_t)head * p.o_sh;
      float* pdst = part + (X * kTile + row) * kHead;
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        float o[32];
        if (!first) {
          tc::ld32_wait(t_o + 32 * c, o);
        } else {
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = 0.f;
        }
#pragma unroll
        for (int k = 0; k < 32; ++k) o[k] *= f;
        if (valid && whole) {
#pragma unroll
          for (int k = 0; k < 32; k += 8) {
            uint32_t u[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const __nv_bfloat162 b = __floats2bfloat162_rn(o[k + 2 * e], o[k + 2 * e + 1]);
              u[e] = *reinterpret_cast<const uint32_t*>(&b);
            }
            *reinterpret_cast<uint4*>(dst + 32 * c + k) = make_uint4(u[0], u[1], u[2], u[3]);
          }
        } else if (valid) {
#pragma unroll
          for (int k = 0; k < 32; k += 4)
            *reinterpret_cast<float4*>(pdst + 32 * c + k) = make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
        }
      }
      if (!whole && valid)
        *reinterpret_cast<float2*>(part + kPairRows * kHead + 2 * (X * kTile + row)) = make_float2(ref, l);
      if (!whole && w.item >= begin && tid == 0) {  // the item begins here and is cut: what its join needs
        int* rec = p.records + blockIdx.x * 8;
        rec[1] = r.row0;
        rec[2] = r.qlen;
        rec[3] = r.t0;
        rec[4] = kh;
        rec[5] = share_owner(w.item + r.keys.count - 1, total, shares);
        rec[0] = 1;
      }
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (warp == kMmaWarp) tc::tmem_dealloc(tbase, 512);
}

// Joins what the shares left of the item cut at the end of CTA blockIdx.x's share, in
// their order: 16 rows a block.
constexpr int kJoinRows = 16;
__global__ void __launch_bounds__(128) block_prefill_join_kernel(const BlockAttnParams p) {
  if (threadIdx.x == 0) griddep_launch_dependents();
  griddep_wait();
  const int* rec = p.records + blockIdx.x * 8;
  if (!rec[0]) return;
  const int row0 = rec[1], qlen = rec[2], t0 = rec[3], kh = rec[4], c_hi = rec[5];
  const int slot = blockIdx.x % p.slots, c_lo = blockIdx.x / p.slots, tokens = kTile / p.group;
  for (int e = threadIdx.x; e < kJoinRows * (kHead / 4); e += 128) {
    const int a = blockIdx.y * kJoinRows + e / (kHead / 4), c = e % (kHead / 4);
    const int X = a / kTile, row = a % kTile, t = t0 + X * tokens + row / p.group;
    if (row >= tokens * p.group || t >= qlen) continue;
    float top = kNone, sum = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    constexpr int kFlight = 8;
    for (int c0 = c_lo; c0 <= c_hi; c0 += kFlight) {
      float2 ml[kFlight];
      float4 v[kFlight];
      float nt = top;
#pragma unroll
      for (int u = 0; u < kFlight; ++u) {
        ml[u] = make_float2(kNone, 0.f);
        v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (c0 + u <= c_hi) {
          const int64_t cta = (int64_t)(c0 + u) * p.slots + slot;
          const float* q = p.partials + (2 * cta + (c0 + u == c_lo ? 1 : 0)) * kPartialFloats;
          ml[u] = __ldcg(reinterpret_cast<const float2*>(q + kPairRows * kHead + 2 * a));
          v[u] = __ldcg(reinterpret_cast<const float4*>(q + a * kHead + 4 * c));
        }
      }
#pragma unroll
      for (int u = 0; u < kFlight; ++u) nt = fmaxf(nt, ml[u].x);
      const float f = ex2(top - nt);
      sum *= f;
      o.x *= f; o.y *= f; o.z *= f; o.w *= f;
#pragma unroll
      for (int u = 0; u < kFlight; ++u) {
        const float g = ex2(ml[u].x - nt);
        sum = fmaf(g, ml[u].y, sum);
        o.x = fmaf(g, v[u].x, o.x); o.y = fmaf(g, v[u].y, o.y);
        o.z = fmaf(g, v[u].z, o.z); o.w = fmaf(g, v[u].w, o.w);
      }
      top = nt;
    }
    const float f = sum > 0.f ? __fdividef(1.f, sum) : 0.f;
    const __nv_bfloat162 x = __floats2bfloat162_rn(o.x * f, o.y * f), y = __floats2bfloat162_rn(o.z * f, o.w * f);
    *reinterpret_cast<uint2*>(p.out + (int64_t)(row0 + t) * p.o_st +
                              (int64_t)(kh * p.group + row % p.group) * p.o_sh + 4 * c) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
  }
}

}  // namespace

cudaError_t block_prefill_launch(const CUtensorMap& km, const CUtensorMap& vm, BlockAttnParams p, cudaStream_t st) {
  const int smem = kSmem + 1024;
  static PerDevice sized;
  if (!sized.done()) {
    const cudaError_t e =
        cudaFuncSetAttribute(block_prefill_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    sized.set();
  }
  const int ctas = block_attn_shares(&p);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t lc = {};
  lc.gridDim = dim3(ctas, 1, 1);
  lc.blockDim = dim3(kThreads, 1, 1);
  lc.dynamicSmemBytes = smem;
  lc.stream = st;
  lc.attrs = attr;
  lc.numAttrs = pdl_enabled() ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&lc, block_prefill_kernel, km, vm, p);
  if (e != cudaSuccess) return e;
  lc.gridDim = dim3(ctas, kPairRows / kJoinRows, 1);
  lc.blockDim = dim3(128, 1, 1);
  lc.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&lc, block_prefill_join_kernel, p);
}

}  // namespace b200kv
