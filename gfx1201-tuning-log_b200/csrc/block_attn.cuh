// What the attention kernels over a block-scaled cache share.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

namespace b200kv {

constexpr int kMaxGroup = 16;  // query heads per kv head
constexpr int kMaxRows = 64;   // (query token, head) rows of a kv head that the few-query kernel takes
constexpr int kMaxCtas = 160;  // shares of a batch it is cut into, at most

// Whether something was done once on the current device (a kernel's attribute set).
class PerDevice {
 public:
  bool done() const {
    const int d = device();
    return d >= 0 && done_[d].load(std::memory_order_acquire);
  }
  void set() {
    const int d = device();
    if (d >= 0) done_[d].store(true, std::memory_order_release);
  }

 private:
  static constexpr int kDevices = 64;
  static int device() {
    int d = -1;
    return cudaGetDevice(&d) == cudaSuccess && d < kDevices ? d : -1;
  }
  std::atomic<bool> done_[kDevices] = {};
};

struct BlockAttnParams {
  const __nv_bfloat16* q;
  __nv_bfloat16* out;
  int64_t q_st, q_sh, o_st, o_sh;
  const int32_t* cu;
  const int32_t* lens;
  const int32_t* bt;
  int64_t bt_stride;
  const uint8_t* kc;
  const uint8_t* vc;
  const float* ks;
  const float* vs;
  int64_t sk0, sk1, sk2, sv0, sv1, sv2, ks0, ks1, vs0, vs1;
  float sm_scale;
  int num_seqs, hkv, group, shift, num_blocks, max_blocks, window, sinks;
  int heads, slots;  // of the few-query kernel: kv heads a CTA walks, CTAs that share a range
  float* partials;  // [2 kMaxCtas][kMaxRows x (128 + m + l)]
  int* counters;    // [num_seqs][hkv], zero between calls
};

// sequences with at most kMaxRows rows per kv head; `rows` bounds them in this batch
cudaError_t block_decode_launch(const CUtensorMap& km, const CUtensorMap& vm, BlockAttnParams p, int rows,
                                cudaStream_t st);

}  // namespace b200kv
