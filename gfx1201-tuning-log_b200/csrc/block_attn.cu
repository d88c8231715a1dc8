// Causal attention over a block-scaled fp8 paged cache (sm_100a).
//
// The plain kernel: one CTA per (query token, kv head), one thread per key for
// the scores and one per dimension for the output, fp32 throughout, an online
// softmax over chunks of 128 keys.

#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <stdint.h>

#include "b200kv.h"
#include "b200kv_common.cuh"
#include "block_attn.cuh"
#include "tma.cuh"

namespace b200kv {

int block_cache_check(const b200kv_block_cache* c);

namespace {

constexpr int kHead = 128;

__device__ __forceinline__ float e4m3(uint8_t b) {
  const __half_raw h = __nv_cvt_fp8_to_halfraw(b, __NV_E4M3);
  return __half2float(*reinterpret_cast<const __half*>(&h));
}

__global__ void __launch_bounds__(kHead) block_attn_plain_kernel(const BlockAttnParams p) {
  __shared__ float s_q[kMaxGroup][kHead], s_p[kMaxGroup][kHead], s_red[kHead / 32][kMaxGroup];
  __shared__ float s_vs[kHead];
  __shared__ int64_t s_v[kHead];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x, kh = blockIdx.y, G = p.group;
  griddep_wait();
  int seq = 0;
  while (seq + 1 < p.num_seqs && p.cu[seq + 1] <= row) ++seq;
  if (row < p.cu[seq] || row >= p.cu[seq + 1]) return;
  if ((p.cu[seq + 1] - p.cu[seq]) * G <= kMaxRows) return;  // the few-query kernel's
  const int pos = p.lens[seq] - (p.cu[seq + 1] - row);
  for (int g = 0; g < G; ++g)
    s_q[g][tid] = __bfloat162float(p.q[(int64_t)row * p.q_st + (int64_t)(kh * G + g) * p.q_sh + tid]);
  __syncthreads();
  float m[kMaxGroup], l[kMaxGroup], o[kMaxGroup];
#pragma unroll
  for (int g = 0; g < kMaxGroup; ++g) { m[g] = -INFINITY; l[g] = 0.f; o[g] = 0.f; }
  for (int base = 0; base <= pos; base += kHead) {
    const int j = base + tid;
    const int page = j >> p.shift;
    const bool sees = j <= pos && page < p.max_blocks && (p.window == 0 || j > pos - p.window || j < p.sinks);
    if (!__syncthreads_or(sees)) continue;
    float sc[kMaxGroup];
#pragma unroll
    for (int g = 0; g < kMaxGroup; ++g) sc[g] = -INFINITY;
    s_vs[tid] = 0.f;
    s_v[tid] = -1;
    if (sees) {
      const int blk = p.bt[(int64_t)seq * p.bt_stride + page], slot = j & ((1 << p.shift) - 1);
      const bool ok = blk >= 0 && blk < p.num_blocks;
#pragma unroll
      for (int g = 0; g < kMaxGroup; ++g) sc[g] = 0.f;
      if (ok) {
        const uint8_t* kp = p.kc + (int64_t)blk * p.sk0 + (int64_t)slot * p.sk1 + (int64_t)kh * p.sk2;
        for (int d = 0; d < kHead; ++d) {
          const float kv = e4m3(kp[d]);
#pragma unroll
          for (int g = 0; g < kMaxGroup; ++g)
            if (g < G) sc[g] += s_q[g][d] * kv;
        }
        const float f = p.sm_scale * p.ks[(int64_t)blk * p.ks0 + kh * p.ks1];
#pragma unroll
        for (int g = 0; g < kMaxGroup; ++g) sc[g] *= f;
        s_vs[tid] = p.vs[(int64_t)blk * p.vs0 + kh * p.vs1];
        s_v[tid] = (int64_t)blk * p.sv0 + (int64_t)slot * p.sv1 + (int64_t)kh * p.sv2;
      }
    }
#pragma unroll
    for (int g = 0; g < kMaxGroup; ++g) {
      if (g >= G) break;
      float v = sc[g];
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, x));
      if (lane == 0) s_red[warp][g] = v;
    }
    __syncthreads();
#pragma unroll
    for (int g = 0; g < kMaxGroup; ++g) {
      if (g >= G) break;
      float v = m[g];
#pragma unroll
      for (int w = 0; w < kHead / 32; ++w) v = fmaxf(v, s_red[w][g]);
      const float a = m[g] == v ? 1.f : __expf(m[g] - v);
      m[g] = v;
      l[g] *= a;
      o[g] *= a;
      s_p[g][tid] = sees ? __expf(sc[g] - v) : 0.f;
    }
    __syncthreads();
    for (int t = 0; t < kHead; ++t) {
      const float x = s_v[t] >= 0 ? e4m3(p.vc[s_v[t] + tid]) * s_vs[t] : 0.f;
#pragma unroll
      for (int g = 0; g < kMaxGroup; ++g)
        if (g < G) {
          l[g] += s_p[g][t];
          o[g] += s_p[g][t] * x;
        }
    }
    __syncthreads();
  }
#pragma unroll
  for (int g = 0; g < kMaxGroup; ++g)
    if (g < G)
      p.out[(int64_t)row * p.o_st + (int64_t)(kh * G + g) * p.o_sh + tid] =
          __float2bfloat16_rn(l[g] > 0.f ? o[g] / l[g] : 0.f);
}

}  // namespace

// counters, then the partials
size_t block_attn_workspace_bytes(int num_seqs, int num_kv_heads) {
  if (num_seqs <= 0 || num_kv_heads <= 0) return 0;
  return align_up((size_t)num_seqs * num_kv_heads * sizeof(int), 256) +
         (size_t)2 * kMaxCtas * kMaxRows * (kHead + 2) * sizeof(float);
}

int block_attn_launch(const b200kv_block_cache* c, const b200kv_block_attn_args* a, void* stream) {
  const int bad = block_cache_check(c);
  if (bad != B200KV_OK) return bad;
  if (!a || !a->q || !a->out || !a->cu_seqlens_q || !a->seq_lens) return B200KV_ERR_INVALID_ARG;
  if (a->num_tokens < 0 || a->max_qlen <= 0 || a->max_seq_len < 0 || a->num_q_heads <= 0 || a->window < 0 ||
      a->sinks < 0 || a->num_q_heads % c->num_kv_heads)
    return B200KV_ERR_INVALID_ARG;
  if (a->num_q_heads / c->num_kv_heads > kMaxGroup) return B200KV_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->out)) & 15) return B200KV_ERR_MISALIGNED;
  if ((a->q_stride_tok | a->q_stride_head | a->out_stride_tok | a->out_stride_head) & 7)
    return B200KV_ERR_MISALIGNED;
  if (!a->workspace || a->workspace_bytes < block_attn_workspace_bytes(c->num_seqs, c->num_kv_heads))
    return B200KV_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(a->workspace) & 255) return B200KV_ERR_MISALIGNED;
  if (sm_major_current_device() < 10) return B200KV_ERR_NO_DEVICE;
  if (a->num_tokens == 0) return B200KV_OK;
  BlockAttnParams p;
  p.q = static_cast<const __nv_bfloat16*>(a->q);
  p.out = static_cast<__nv_bfloat16*>(a->out);
  p.q_st = a->q_stride_tok; p.q_sh = a->q_stride_head;
  p.o_st = a->out_stride_tok; p.o_sh = a->out_stride_head;
  p.cu = a->cu_seqlens_q;
  p.lens = a->seq_lens;
  p.bt = c->block_table;
  p.bt_stride = c->bt_stride;
  p.kc = static_cast<const uint8_t*>(c->k);
  p.vc = static_cast<const uint8_t*>(c->v);
  p.ks = c->k_scales;
  p.vs = c->v_scales;
  p.sk0 = c->sk0; p.sk1 = c->sk1; p.sk2 = c->sk2;
  p.sv0 = c->sv0; p.sv1 = c->sv1; p.sv2 = c->sv2;
  p.ks0 = c->ks0; p.ks1 = c->ks1; p.vs0 = c->vs0; p.vs1 = c->vs1;
  p.sm_scale = a->sm_scale;
  p.num_seqs = c->num_seqs;
  p.group = a->num_q_heads / c->num_kv_heads;
  p.shift = __builtin_ctz((unsigned)c->block_size);
  p.num_blocks = c->num_blocks;
  p.max_blocks = c->max_blocks < (0x7fffffff >> p.shift) ? c->max_blocks : 0x7fffffff >> p.shift;
  p.window = a->window;
  p.sinks = a->sinks;
  p.hkv = c->num_kv_heads;
  p.counters = static_cast<int*>(a->workspace);
  p.partials = reinterpret_cast<float*>(static_cast<char*>(a->workspace) +
                                        align_up((size_t)c->num_seqs * c->num_kv_heads * sizeof(int), 256));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  CUtensorMap km, vm;
  if (!encode_paged_kv(&km, c->k, kHead, (uint32_t)c->num_kv_heads, (uint32_t)c->block_size, (uint64_t)c->num_blocks,
                       (uint64_t)c->sk2, (uint64_t)c->sk1, (uint64_t)c->sk0) ||
      !encode_paged_kv(&vm, c->v, kHead, (uint32_t)c->num_kv_heads, (uint32_t)c->block_size, (uint64_t)c->num_blocks,
                       (uint64_t)c->sv2, (uint64_t)c->sv1, (uint64_t)c->sv0))
    return B200KV_ERR_UNSUPPORTED;
  const int64_t rows = (int64_t)a->max_qlen * p.group;
  if (block_decode_launch(km, vm, p, rows < kMaxRows ? (int)rows : kMaxRows, st) != cudaSuccess)
    return B200KV_ERR_LAUNCH;
  if (rows <= kMaxRows) return B200KV_OK;
  block_attn_plain_kernel<<<dim3(a->num_tokens, c->num_kv_heads), kHead, 0, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? B200KV_OK : B200KV_ERR_LAUNCH;
}

}  // namespace b200kv
