// Attention over the 8-bit paged cache: what its kernels share.
//
// With codes c and row scales s, and q scaled by a power of two f_i:
//     x_ij = sm_scale * log2(e) / f_i * (sum_d q'_id ck_jd) * sk_j      p_ij = 2^(x_ij - m_i)
//     o_i  = sum_j (p_ij sv_j) cv_j / sum_j p_ij
// The first product runs on fp16 operands for few rows (q' below 2^15, exact) and on e4m3 operands
// for many (see there). The second runs on fp16: e4m3 codes are exact in it, and P' = p_ij sv_j
// 2^(6 - e), with e the largest exponent of the sv seen so far, is rounded to it (relative error
// 2^-11, below half a step of the output; P' < 2^15, and its range reaches 2^-30 below the row's
// largest p). Sums, statistics and scales are fp32.
#pragma once

#include "kv8_common.cuh"
#include "ptx_sm100.cuh"

namespace fa2kv {

struct AttnArgs {
  Cache c;
  const uint16_t* q;
  uint16_t* o;
  int64_t q_st[3], o_st[3];  // (b, h, n)
  const int* bt;
  const int* lens;
  const int* cu_q;  // packed queries, else nullptr
  int* err;
  float* o_part;    // split partials: O / l in fp32 ...
  float* lse_part;  // ... and log2 of the row's sum
  int64_t bt_stride;
  long long timeout;
  int pages_per_seq, batch, group, heads_kv, n_q, total_q, max_k;
  int causal, bottom_right;
  int splits, split_keys;  // key ranges [s * split_keys, (s + 1) * split_keys)
  int row_blocks, rows_pad;
  float qk_scale;
};

constexpr float RESCALE_TH = 8.0f;  // log2: the reference max moves when a row's max grows by more
constexpr int P_SHIFT = 6;          // P' = p * sv * 2^(P_SHIFT - e), see above
constexpr int EB_MIN = 8;           // smallest exponent field used for e (a multiplier stays finite)

struct Seq {
  int n_q, q0, len, off;  // queries, first packed row, keys, causal offset
};

// Sequence b, checked: nothing its numbers lead to is outside the tensors.
__device__ __forceinline__ Seq sequence(const AttnArgs& a, int b) {
  Seq s;
  s.n_q = a.n_q;
  s.q0 = 0;
  if (a.cu_q != nullptr) {
    s.q0 = __ldg(a.cu_q + b);
    const int64_t end = __ldg(a.cu_q + b + 1);
    const int64_t n = end - s.q0;
    if (s.q0 < 0 || n < 0 || n > a.n_q || end > a.total_q) {
      report(a.err, FA2_ERR_SHAPE);
      s.n_q = 0;
    } else {
      s.n_q = static_cast<int>(n);
    }
  }
  s.len = __ldg(a.lens + b);
  if (s.len < 0 || s.len > a.max_k || s.len > static_cast<int64_t>(a.pages_per_seq) * a.c.page_size) {
    report(a.err, FA2_ERR_SHAPE);
    s.len = 0;
  }
  s.off = a.bottom_right ? s.len - s.n_q : 0;
  return s;
}

// Keys that the rows [row0, row0 + count) of a (sequence, kv head) see at most: [0, result).
__device__ __forceinline__ int keys_end(const AttnArgs& a, const Seq& s, int row0, int count) {
  if (!a.causal) return s.len;
  const int i = min((row0 + count - 1) / a.group, s.n_q - 1);
  return max(0, min(s.len, i + s.off + 1));
}

// The last key that query i sees (-1: none).
__device__ __forceinline__ int last_key(const AttnArgs& a, const Seq& s, int i) {
  return a.causal ? min(s.len - 1, i + s.off) : s.len - 1;
}

__device__ __forceinline__ const uint16_t* q_row(const AttnArgs& a, const Seq& s, int b, int h, int row) {
  const int i = row / a.group, g = row - i * a.group;
  const int64_t bb = a.cu_q != nullptr ? 0 : b;
  return a.q + bb * a.q_st[0] + static_cast<int64_t>(h * a.group + g) * a.q_st[1] + static_cast<int64_t>(s.q0 + i) * a.q_st[2];
}

__device__ __forceinline__ uint16_t* o_row(const AttnArgs& a, const Seq& s, int b, int h, int row) {
  const int i = row / a.group, g = row - i * a.group;
  const int64_t bb = a.cu_q != nullptr ? 0 : b;
  return a.o + bb * a.o_st[0] + static_cast<int64_t>(h * a.group + g) * a.o_st[1] + static_cast<int64_t>(s.q0 + i) * a.o_st[2];
}

__device__ __forceinline__ float pow2f(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }  // -126 <= e <= 127

// Exponent e such that a row with largest magnitude `top` (bits) times 2^(14 - e) stays below 2^15.
__device__ __forceinline__ int row_exponent(uint32_t top_bits) {
  return min(127, max(-100, static_cast<int>(top_bits >> 23) - 127));
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  const int n = valid ? 16 : 0;  // 0: zeros are written, nothing is read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async16_full(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool valid) {
  const int n = valid ? 4 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

}  // namespace fa2kv
