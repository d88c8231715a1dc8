// Append to a block-scaled fp8 paged cache (sm_100a): rotary embedding of q and
// k, k and v into e4m3 codes with one power-of-two scale per (block, kv head).
//
// For the new values x of one block and head: s = 2^e, the smallest with
// max |x| <= 448 s, and code = e4m3(x / s).  A power of two makes x / s exact, so
// the code is the one rounding of the fp32 value, and a block that outgrows its
// scale (s > old) has its earlier codes rounded again from code * (old / s), which
// is exact down to e4m3's subnormals.  Rotation as rope_pair (the RoPE + KV-write
// kernel's arithmetic), not rounded to bf16 before the codes.
//
// A block is written by one CTA per kv head: the scale needs the maximum over the
// block's new rows, so a CTA owns (sequence, block, head) with the block's up to
// 128 tokens, keeps their rotated k and v in registers between the maximum and
// the codes, and rotates the head's group of q rows of the same tokens, whose
// angles it then reads once.  No atomics on memory: two runs give the same bytes.

#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <stdint.h>

#include "b200kv.h"
#include "b200kv_common.cuh"

namespace b200kv {
namespace {

constexpr int kHead = 128;
constexpr int kMinExp = -64, kMaxExp = 100;  // exponents of the scales written

struct AppendParams {
  const __nv_bfloat16* qkv;
  int64_t qkv_st;
  const float* cos_sin;
  int max_pos;
  __nv_bfloat16* q_out;
  int64_t q_st, q_sh;
  const int32_t* cu;
  const int32_t* lens;
  const int32_t* bt;
  int64_t bt_stride;
  uint8_t* kc;
  uint8_t* vc;
  float* ks;
  float* vs;
  int64_t sk0, sk1, sk2, sv0, sv1, sv2, ks0, ks1, vs0, vs1;
  int num_seqs, hq, hkv, shift, num_blocks, max_blocks;
};

// Items (sequence, block) of the batch are numbered without a prefix sum: the
// sequence that starts at row c touches at most qlen and at most qlen / block + 2
// blocks, so numbering them from min(c, c / block + 2 s) leaves room for each.
__device__ __host__ __forceinline__ int first_item(int c, int s, int shift) {
  const int a = c, b = (c >> shift) + 2 * s;
  return a < b ? a : b;
}

__device__ __forceinline__ float bf_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf_hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
__device__ __forceinline__ uint32_t bf_pack(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// the bits of |x|, 0 where x is not finite: an unsigned maximum of them is the
// maximum of the finite magnitudes
__device__ __forceinline__ uint32_t finite_bits(float x) {
  const uint32_t b = __float_as_uint(x) & 0x7FFFFFFFu;
  return b < 0x7F800000u ? b : 0u;
}
// smallest power of two s with amax <= 448 s (448 = 1.75 * 2^8)
__device__ __forceinline__ float scale_for(uint32_t amax_bits) {
  const int x = (int)(amax_bits >> 23) - 127;  // amax = m 2^x, 1 <= m < 2 (subnormals end at the floor)
  int e = (amax_bits & 0x7FFFFFu) <= 0x600000u ? x - 8 : x - 7;
  e = max(kMinExp, min(kMaxExp, e));
  return __uint_as_float((uint32_t)(e + 127) << 23);
}
__device__ __forceinline__ uint32_t codes2(float a, float b) {
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
// x / s; a power of two is divided by through its exact reciprocal
struct Divider {
  float s, inv;
  bool pow2;
  __device__ __forceinline__ explicit Divider(float s_) : s(s_) {
    const uint32_t b = __float_as_uint(s_);
    pow2 = (b & 0x7FFFFFu) == 0 && b >= 0x01000000u && b < 0x7E800000u;
    inv = pow2 ? __uint_as_float(0x7F000000u - b) : 0.f;
  }
  __device__ __forceinline__ float operator()(float x) const { return pow2 ? x * inv : __fdiv_rn(x, s); }
};

// e4m3 codes of one 32-bit word times r, rounded again
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float r) {
  uint32_t out = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (16 * i)), __NV_E4M3);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    out |= codes2(f.x * r, f.y * r) << (16 * i);
  }
  return out;
}

// TPW tokens of the block per warp, NW warps; lane l holds elements 2l, 2l+1 and
// 64+2l, 64+2l+1 of each row: two rotary pairs.
template <int TPW, int NW>
__global__ void __launch_bounds__(NW * 32) block_append_kernel(const AppendParams p) {
  __shared__ int s_count[NW];
  __shared__ uint32_t s_amax[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int item = blockIdx.x, kh = blockIdx.y;
  if (tid == 0) griddep_launch_dependents();
  if (tid < 2) s_amax[tid] = 0;
  griddep_wait();

  // the sequence of this item: the last one whose first item is not past it
  const int c0 = p.cu[0];
  int cnt = 0;
  for (int s = tid; s < p.num_seqs; s += NW * 32) cnt += first_item(p.cu[s] - c0, s, p.shift) <= item;
  cnt = __reduce_add_sync(0xffffffffu, cnt);
  if (lane == 0) s_count[warp] = cnt;
  __syncthreads();
  int seq = -1;
#pragma unroll
  for (int w = 0; w < NW; ++w) seq += s_count[w];
  const int row_s = p.cu[seq], qlen = p.cu[seq + 1] - row_s, total = p.lens[seq];
  const int begin = total - qlen;
  const int page = (begin >> p.shift) + (item - first_item(row_s - c0, seq, p.shift));
  if (qlen <= 0 || page > ((total - 1) >> p.shift)) return;
  const int lo = max(begin, page << p.shift), hi = min(total, (page + 1) << p.shift);
  const int nt = hi - lo, row0 = row_s + (lo - begin);
  const int kept = lo - (page << p.shift);  // earlier tokens of this block

  int blk = -1;
  if (page >= 0 && page < p.max_blocks) blk = p.bt[(int64_t)seq * p.bt_stride + page];
  const bool ok = blk >= 0 && blk < p.num_blocks;
  if (!ok && tid == 0) atomicExch(&g_device_status, kDevIndexRange);
  float* ksp = p.ks + (int64_t)(ok ? blk : 0) * p.ks0 + kh * p.ks1;
  float* vsp = p.vs + (int64_t)(ok ? blk : 0) * p.vs0 + kh * p.vs1;
  const float old_k = ok ? *ksp : 0.f, old_v = ok ? *vsp : 0.f;

  const int group = p.hq / p.hkv;
  float kr[TPW][4];
  uint32_t vr[TPW][2];
  uint32_t amax_k = 0, amax_v = 0;
#pragma unroll
  for (int i = 0; i < TPW; ++i) {
    const int t = warp + i * NW;
    if (t < nt) {
      const __nv_bfloat16* row = p.qkv + (int64_t)(row0 + t) * p.qkv_st;
      const int pos = min(max(lo + t, 0), p.max_pos - 1);
      const float2 c = *reinterpret_cast<const float2*>(p.cos_sin + (int64_t)pos * kHead + 2 * lane);
      const float2 s = *reinterpret_cast<const float2*>(p.cos_sin + (int64_t)pos * kHead + 64 + 2 * lane);
      const uint32_t* kw = reinterpret_cast<const uint32_t*>(row + (int64_t)(p.hq + kh) * kHead);
      const uint32_t* vw = reinterpret_cast<const uint32_t*>(row + (int64_t)(p.hq + p.hkv + kh) * kHead);
      const uint32_t k1 = kw[lane], k2 = kw[32 + lane];
      vr[i][0] = vw[lane];
      vr[i][1] = vw[32 + lane];
      for (int h = 0; h < group; ++h) {
        const uint32_t* qw = reinterpret_cast<const uint32_t*>(row + (int64_t)(kh * group + h) * kHead);
        const uint32_t x1 = qw[lane], x2 = qw[32 + lane];
        float a1, a2, b1, b2;
        rope_pair(bf_lo(x1), bf_lo(x2), c.x, s.x, a1, a2);
        rope_pair(bf_hi(x1), bf_hi(x2), c.y, s.y, b1, b2);
        uint32_t* o = reinterpret_cast<uint32_t*>(p.q_out + (int64_t)(row0 + t) * p.q_st +
                                                  (int64_t)(kh * group + h) * p.q_sh);
        o[lane] = bf_pack(a1, b1);
        o[32 + lane] = bf_pack(a2, b2);
      }
      rope_pair(bf_lo(k1), bf_lo(k2), c.x, s.x, kr[i][0], kr[i][2]);
      rope_pair(bf_hi(k1), bf_hi(k2), c.y, s.y, kr[i][1], kr[i][3]);
#pragma unroll
      for (int e = 0; e < 4; ++e) amax_k = max(amax_k, finite_bits(kr[i][e]));
#pragma unroll
      for (int e = 0; e < 2; ++e)
        amax_v = max(amax_v, max(finite_bits(bf_lo(vr[i][e])), finite_bits(bf_hi(vr[i][e]))));
    }
  }
  if (!ok) return;  // CTA-uniform
  amax_k = __reduce_max_sync(0xffffffffu, amax_k);
  amax_v = __reduce_max_sync(0xffffffffu, amax_v);
  if (lane == 0) {
    atomicMax(&s_amax[0], amax_k);
    atomicMax(&s_amax[1], amax_v);
  }
  __syncthreads();
  float new_k = scale_for(s_amax[0]), new_v = scale_for(s_amax[1]);
  uint8_t* kb = p.kc + (int64_t)blk * p.sk0 + (int64_t)kh * p.sk2;
  uint8_t* vb = p.vc + (int64_t)blk * p.sv0 + (int64_t)kh * p.sv2;
  if (kept > 0) {
    new_k = fmaxf(new_k, old_k);
    new_v = fmaxf(new_v, old_v);
    const float rk = __fdiv_rn(old_k, new_k), rv = __fdiv_rn(old_v, new_v);
    for (int t = warp; t < kept; t += NW) {
      if (new_k != old_k) {
        uint32_t* w = reinterpret_cast<uint32_t*>(kb + (int64_t)t * p.sk1) + lane;
        *w = rescale4(*w, rk);
      }
      if (new_v != old_v) {
        uint32_t* w = reinterpret_cast<uint32_t*>(vb + (int64_t)t * p.sv1) + lane;
        *w = rescale4(*w, rv);
      }
    }
  }
  if (tid == 0) {
    *ksp = new_k;
    *vsp = new_v;
  }
  const Divider dk(new_k), dv(new_v);
#pragma unroll
  for (int i = 0; i < TPW; ++i) {
    const int t = warp + i * NW;
    if (t < nt) {
      uint16_t* kw = reinterpret_cast<uint16_t*>(kb + (int64_t)(kept + t) * p.sk1);
      uint16_t* vw = reinterpret_cast<uint16_t*>(vb + (int64_t)(kept + t) * p.sv1);
      kw[lane] = (uint16_t)codes2(dk(kr[i][0]), dk(kr[i][1]));
      kw[32 + lane] = (uint16_t)codes2(dk(kr[i][2]), dk(kr[i][3]));
#pragma unroll
      for (int e = 0; e < 2; ++e)
        vw[32 * e + lane] = (uint16_t)codes2(dv(bf_lo(vr[i][e])), dv(bf_hi(vr[i][e])));
    }
  }
}

}  // namespace

// What every entry point asks of a cache.
int block_cache_check(const b200kv_block_cache* c) {
  if (!c || !c->k || !c->v || !c->k_scales || !c->v_scales || !c->block_table) return B200KV_ERR_INVALID_ARG;
  if (c->num_blocks <= 0 || c->num_kv_heads <= 0 || c->max_blocks <= 0 || c->num_seqs <= 0 ||
      c->bt_stride < c->max_blocks || c->num_kv_heads > 65535)
    return B200KV_ERR_INVALID_ARG;
  if (c->head_dim != kHead) return B200KV_ERR_UNSUPPORTED;
  if (c->block_size != 16 && c->block_size != 32 && c->block_size != 64 && c->block_size != 128)
    return B200KV_ERR_UNSUPPORTED;
  const int64_t st[6] = {c->sk0, c->sk1, c->sk2, c->sv0, c->sv1, c->sv2};
  for (int i = 0; i < 6; ++i)
    if (st[i] % 16) return B200KV_ERR_MISALIGNED;
  if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15) return B200KV_ERR_MISALIGNED;
  return B200KV_OK;
}

int block_append_launch(const b200kv_block_cache* c, const void* qkv, int64_t qkv_st, const float* cos_sin,
                        int max_pos, void* q_out, int64_t q_st, int64_t q_sh, const int32_t* cu,
                        const int32_t* lens, int num_tokens, int hq, void* stream) {
  const int bad = block_cache_check(c);
  if (bad != B200KV_OK) return bad;
  if (!qkv || !cos_sin || !q_out || !cu || !lens || max_pos <= 0 || num_tokens < 0 || hq <= 0 ||
      hq % c->num_kv_heads)
    return B200KV_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q_out) |
       reinterpret_cast<uintptr_t>(cos_sin)) & 15)
    return B200KV_ERR_MISALIGNED;
  if (qkv_st % 8 || q_st % 8 || q_sh % 8) return B200KV_ERR_MISALIGNED;
  if (sm_major_current_device() < 10) return B200KV_ERR_NO_DEVICE;
  if (num_tokens == 0) return B200KV_OK;
  AppendParams p;
  p.qkv = static_cast<const __nv_bfloat16*>(qkv);
  p.qkv_st = qkv_st;
  p.cos_sin = cos_sin;
  p.max_pos = max_pos;
  p.q_out = static_cast<__nv_bfloat16*>(q_out);
  p.q_st = q_st;
  p.q_sh = q_sh;
  p.cu = cu;
  p.lens = lens;
  p.bt = c->block_table;
  p.bt_stride = c->bt_stride;
  p.kc = static_cast<uint8_t*>(c->k);
  p.vc = static_cast<uint8_t*>(c->v);
  p.ks = c->k_scales;
  p.vs = c->v_scales;
  p.sk0 = c->sk0; p.sk1 = c->sk1; p.sk2 = c->sk2;
  p.sv0 = c->sv0; p.sv1 = c->sv1; p.sv2 = c->sv2;
  p.ks0 = c->ks0; p.ks1 = c->ks1; p.vs0 = c->vs0; p.vs1 = c->vs1;
  p.num_seqs = c->num_seqs;
  p.hq = hq;
  p.hkv = c->num_kv_heads;
  p.shift = __builtin_ctz((unsigned)c->block_size);
  p.num_blocks = c->num_blocks;
  p.max_blocks = c->max_blocks;
  const int64_t items = (int64_t)(num_tokens >> p.shift) + 2 * (int64_t)c->num_seqs;
  cudaLaunchConfig_t lc = {};
  lc.gridDim = dim3((unsigned)(items < num_tokens ? items : num_tokens), c->num_kv_heads, 1);
  lc.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  lc.attrs = attr;
  lc.numAttrs = pdl_enabled() ? 1 : 0;
  cudaError_t e;
  switch (c->block_size) {
    case 16: lc.blockDim = dim3(256); e = cudaLaunchKernelEx(&lc, block_append_kernel<2, 8>, p); break;
    case 32: lc.blockDim = dim3(256); e = cudaLaunchKernelEx(&lc, block_append_kernel<4, 8>, p); break;
    case 64: lc.blockDim = dim3(512); e = cudaLaunchKernelEx(&lc, block_append_kernel<4, 16>, p); break;
    default: lc.blockDim = dim3(512); e = cudaLaunchKernelEx(&lc, block_append_kernel<8, 16>, p); break;
  }
  return e == cudaSuccess ? B200KV_OK : B200KV_ERR_LAUNCH;
}

}  // namespace b200kv
