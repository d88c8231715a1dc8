// Verification of drafted tokens against the target's probabilities (sm_100a).
//
// p = softmax(logits / temperature) per row.  Row r takes its draft d while
// u q(d) < p(d); the row that stops emits argmax_v w(v) / e(v) with w = max(p - q, 0)
// (p after the last draft) and e ~ Exp(1): the race that v wins with probability
// w(v) / sum w, with no prefix sum over the vocabulary.
//
// One cluster of kCs CTAs per sequence, a contiguous chunk of the vocabulary each.
// Per row every CTA reduces its chunk to (max, sum of exponentials, lowest index of
// the maximum) with an online softmax per thread; the ranks read each other's
// through distributed shared memory, so every CTA knows which row stops, and races
// its chunk of that row.  Statistics are fp32, the temperature divides as a
// multiplication by its reciprocal.

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

#include "b200kv.h"
#include "b200kv_common.cuh"

namespace cg = cooperative_groups;

namespace b200kv {
namespace {

constexpr int kCs = 8;
constexpr int kThr = 512;
constexpr int kBatch = 8;  // rows whose statistics are exchanged together

struct VerifyParams {
  const void* logits;
  int64_t ld;
  const int64_t* tokens;
  const int32_t* cu;
  const float* uniforms;
  const float* noise;
  int64_t noise_ld;
  const float* temperature;
  const float* draft;
  int64_t draft_ld;
  int64_t* out;
  int32_t* accepted;
  int vocab;
};

struct Stat {
  float m, z;
  int best;
};

// NaN counts as -inf, +inf as the largest finite value (so that inf - inf never occurs)
__device__ __forceinline__ float clean(float x) { return x == x ? fminf(x, FLT_MAX) : -INFINITY; }
template <bool HALF>
__device__ __forceinline__ float logit(const void* row, int i) {
  if constexpr (HALF) return clean(__bfloat162float(static_cast<const __nv_bfloat16*>(row)[i]));
  else return clean(static_cast<const float*>(row)[i]);
}
// (m, z): the sum of exp((x - m) / T); -inf is the empty sum
__device__ __forceinline__ Stat join(Stat a, Stat b, float inv_t) {
  if (b.m > a.m || (b.m == a.m && b.best < a.best)) {
    const Stat t = a;
    a = b;
    b = t;
  }
  if (b.m != -INFINITY) a.z += b.z * __expf((b.m - a.m) * inv_t);
  return a;
}

struct Race {
  float w;   // residual / noise
  int i;
  float wp;  // p / noise
  int ip;
};
__device__ __forceinline__ Race win(Race a, const Race& b) {
  if (b.w > a.w || (b.w == a.w && b.i < a.i)) { a.w = b.w; a.i = b.i; }
  if (b.wp > a.wp || (b.wp == a.wp && b.ip < a.ip)) { a.wp = b.wp; a.ip = b.ip; }
  return a;
}

template <bool HALF>
__global__ void __cluster_dims__(kCs, 1, 1) __launch_bounds__(kThr) spec_verify_kernel(const VerifyParams p) {
  __shared__ Stat s_warp[kThr / 32][kBatch];
  __shared__ Stat s_mine[kBatch];
  __shared__ Race s_race[kThr / 32];
  __shared__ Race s_won;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), seq = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) griddep_launch_dependents();
  griddep_wait();
  const int r0 = p.cu[seq], n = p.cu[seq + 1] - r0;
  if (n <= 0) {  // no rows: nothing to verify (the whole cluster leaves)
    if (rank == 0 && tid == 0) p.accepted[seq] = 0;
    return;
  }
  const float temp = p.temperature ? p.temperature[seq] : 1.f;
  const bool greedy = !(temp > 0.f);
  const float inv_t = greedy ? 1.f : __fdiv_rn(1.f, temp);
  const int chunk = (p.vocab + kCs - 1) / kCs;
  const int lo = min(p.vocab, rank * chunk), hi = min(p.vocab, lo + chunk);
  const int esz = HALF ? 2 : 4;
  auto row_of = [&](int i) { return static_cast<const char*>(p.logits) + (int64_t)(r0 + i) * p.ld * esz; };

  int stop = n - 1;
  Stat at = {-INFINITY, 0.f, 0};
  for (int b0 = 0; b0 < n; b0 += kBatch) {
    const int nb = min(kBatch, n - b0);
    for (int b = 0; b < nb; ++b) {
      const char* row = row_of(b0 + b);
      Stat st = {-INFINITY, 0.f, INT32_MAX};
      for (int i = lo + tid; i < hi; i += kThr) {
        const float x = logit<HALF>(row, i);
        if (x > st.m) {
          st.z = st.z * __expf((st.m - x) * inv_t) + 1.f;  // exp(-inf) = 0 at the first
          st.m = x;
          st.best = i;
        } else if (x != -INFINITY) {
          st.z += __expf((x - st.m) * inv_t);
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        Stat ot;
        ot.m = __shfl_xor_sync(0xffffffffu, st.m, o);
        ot.z = __shfl_xor_sync(0xffffffffu, st.z, o);
        ot.best = __shfl_xor_sync(0xffffffffu, st.best, o);
        st = join(st, ot, inv_t);
      }
      if (lane == 0) s_warp[warp][b] = st;
    }
    __syncthreads();
    if (tid < nb) {
      Stat st = s_warp[0][tid];
      for (int w = 1; w < kThr / 32; ++w) st = join(st, s_warp[w][tid], inv_t);
      s_mine[tid] = st;
    }
    cluster.sync();
    bool done = false;
    for (int b = 0; b < nb && !done; ++b) {  // every thread of every rank finds the same answer
      Stat st = {-INFINITY, 0.f, INT32_MAX};
      for (int r = 0; r < kCs; ++r) st = join(st, *cluster.map_shared_rank(&s_mine[b], r), inv_t);
      if (st.best == INT32_MAX) st.best = 0;
      at = st;
      stop = b0 + b;
      if (stop == n - 1) break;
      const int64_t d = p.tokens[r0 + stop + 1];
      bool take = false;
      if (d >= 0 && d < p.vocab) {
        const float x = logit<HALF>(row_of(stop), (int)d);
        const float pd = greedy ? (d == st.best && st.m != -INFINITY ? 1.f : 0.f)
                                : (x == -INFINITY ? 0.f : __expf((x - st.m) * inv_t) / st.z);
        const float qd = p.draft ? p.draft[(int64_t)(r0 + stop) * p.draft_ld + d] : 1.f;
        take = p.uniforms[r0 + stop] * qd < pd;
      }
      done = !take;
    }
    cluster.sync();  // the ranks have read each other's statistics
    if (done) break;
  }

  // ---- the race over row `stop` ------------------------------------------------------
  const bool last = stop == n - 1;
  int token = at.best;
  if (!greedy && at.m != -INFINITY) {  // a greedy row, or one of -inf, emits its argmax
    const int64_t d = last ? -1 : p.tokens[r0 + stop + 1];
    const float* q = !last && p.draft ? p.draft + (int64_t)(r0 + stop) * p.draft_ld : nullptr;
    const float* e = p.noise + (int64_t)seq * p.noise_ld;
    const char* row = row_of(stop);
    const float inv_z = 1.f / at.z;
    Race rc = {-1.f, INT32_MAX, -1.f, INT32_MAX};
    for (int i = lo + tid; i < hi; i += kThr) {
      const float x = logit<HALF>(row, i);
      const float pv = x == -INFINITY ? 0.f : __expf((x - at.m) * inv_t) * inv_z;
      const float qv = q ? q[i] : (i == d ? 1.f : 0.f);
      const float ie = 1.f / fmaxf(e[i], FLT_MIN);
      const float w = fmaxf(pv - qv, 0.f) * ie, wp = pv * ie;
      if (w > rc.w) { rc.w = w; rc.i = i; }
      if (wp > rc.wp) { rc.wp = wp; rc.ip = i; }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      Race ot;
      ot.w = __shfl_xor_sync(0xffffffffu, rc.w, o);
      ot.i = __shfl_xor_sync(0xffffffffu, rc.i, o);
      ot.wp = __shfl_xor_sync(0xffffffffu, rc.wp, o);
      ot.ip = __shfl_xor_sync(0xffffffffu, rc.ip, o);
      rc = win(rc, ot);
    }
    if (lane == 0) s_race[warp] = rc;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < kThr / 32; ++w) rc = win(rc, s_race[w]);
      s_won = rc;
    }
    cluster.sync();
    if (rank == 0 && tid == 0) {
      for (int r = 1; r < kCs; ++r) rc = win(rc, *cluster.map_shared_rank(&s_won, r));
      token = rc.w > 0.f ? rc.i : rc.ip;
    }
    cluster.sync();  // peers keep their shared memory until rank 0 has read it
  }
  if (rank == 0) {
    for (int i = tid; i < n; i += kThr)
      if (i != stop) p.out[r0 + i] = i < stop ? p.tokens[r0 + i + 1] : -1;
    if (tid == 0) {
      p.out[r0 + stop] = token;
      p.accepted[seq] = stop;
    }
  }
}

}  // namespace

int spec_verify_launch(const void* logits, int64_t ld, int half, const int64_t* tokens, const int32_t* cu,
                       const float* uniforms, const float* noise, int64_t noise_ld, const float* temperature,
                       const float* draft, int64_t draft_ld, int64_t* out, int32_t* accepted, int num_seqs,
                       int num_rows, int vocab, void* stream) {
  if (!logits || !tokens || !cu || !uniforms || !noise || !out || !accepted) return B200KV_ERR_INVALID_ARG;
  if (num_seqs < 0 || num_rows < 0 || vocab <= 0 || ld < vocab || noise_ld < vocab || (draft && draft_ld < vocab))
    return B200KV_ERR_INVALID_ARG;
  if (num_seqs > 65535) return B200KV_ERR_UNSUPPORTED;
  if (sm_major_current_device() < 10) return B200KV_ERR_NO_DEVICE;
  if (num_seqs == 0) return B200KV_OK;
  VerifyParams p;
  p.logits = logits;
  p.ld = ld;
  p.tokens = tokens;
  p.cu = cu;
  p.uniforms = uniforms;
  p.noise = noise;
  p.noise_ld = noise_ld;
  p.temperature = temperature;
  p.draft = draft;
  p.draft_ld = draft_ld;
  p.out = out;
  p.accepted = accepted;
  p.vocab = vocab;
  cudaLaunchConfig_t lc = {};
  lc.gridDim = dim3(kCs, num_seqs, 1);
  lc.blockDim = dim3(kThr, 1, 1);
  lc.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  lc.attrs = attr;
  lc.numAttrs = pdl_enabled() ? 1 : 0;
  const cudaError_t e = half ? cudaLaunchKernelEx(&lc, spec_verify_kernel<true>, p)
                             : cudaLaunchKernelEx(&lc, spec_verify_kernel<false>, p);
  return e == cudaSuccess ? B200KV_OK : B200KV_ERR_LAUNCH;
}

}  // namespace b200kv
