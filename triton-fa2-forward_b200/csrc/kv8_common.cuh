// Shared pieces of the serving kernels (rotary positions, 8-bit paged K/V cache): page arithmetic,
// e4m3 conversions, error reports, and the host's checks of a cache.
#pragma once

#include <atomic>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "fa2_kvcache_sm100.h"

namespace fa2kv {

constexpr float E4M3_MAX = 448.0f;

// One tensor of codes or scales on the device side.
struct Cache {
  const uint8_t* k;
  const uint8_t* v;
  const float* ks;
  const float* vs;
  int num_pages, page_size, page_shift;           // shift >= 0 where page_size is a power of two
  int heads_kv;
  // Strides in 32 bits (page strides of codes in 16-byte units), for offsets that are one widening
  // product each.
  int k_page16, v_page16, ks_page, vs_page, k_row, v_row, ks_row, vs_row, k_head, v_head, ks_head, vs_head;
};

// What the tests run on the host as well: reads and reports in both forms.
#define FA2_HOST_DEVICE __host__ __device__ __forceinline__
FA2_HOST_DEVICE int load_int(const int* p) {
#ifdef __CUDA_ARCH__
  return __ldg(p);
#else
  return *p;
#endif
}

__device__ __forceinline__ int page_of(const Cache& c, int pos) {
  return c.page_shift >= 0 ? pos >> c.page_shift : pos / c.page_size;
}

FA2_HOST_DEVICE void report(int* err, int code) {
  if (err == nullptr) return;
#ifdef __CUDA_ARCH__
  atomicCAS(err, 0, code);  // the first report wins
#else
  if (*err == 0) *err = code;
#endif
}

// Two values to two e4m3 codes (low byte: lo), round to nearest even, saturated at +-448.
__device__ __forceinline__ uint16_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// The same with e5m2 (5 exponent bits, 2 mantissa bits: smallest step 2^-16, saturated at +-57344).
__device__ __forceinline__ uint16_t e5m2x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// Two e5m2 codes to fp16 (exact: e5m2 is its upper byte).
__device__ __forceinline__ uint32_t f16x2_of_e5m2x2(uint16_t c) {
  uint32_t r;
  asm("cvt.rn.f16x2.e5m2x2 %0, %1;" : "=r"(r) : "h"(c));
  return r;
}

// Two e4m3 codes to fp16 (exact: fp16 holds every e4m3 value).
__device__ __forceinline__ uint32_t f16x2_of_e4m3x2(uint16_t c) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(c));
  return r;
}

__device__ __forceinline__ float2 float2_of_f16x2(uint32_t h) {
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

template <bool BF16>
__device__ __forceinline__ float2 float2_of_x2(uint32_t w) {
  if constexpr (BF16) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  } else {
    return float2_of_f16x2(w);
  }
}

template <bool BF16>
__device__ __forceinline__ float float_of_16(uint16_t w) {
  if constexpr (BF16) {
    return __uint_as_float(static_cast<uint32_t>(w) << 16);
  } else {
    return __half2float(__ushort_as_half(w));
  }
}

template <bool BF16>
__device__ __forceinline__ uint32_t x2_of_floats(float lo, float hi) {
  uint32_t r;
  if constexpr (BF16) {
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  } else {
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  }
  return r;
}

template <bool BF16>
__device__ __forceinline__ uint16_t x1_of_float(float x) {
  if constexpr (BF16) {
    return __bfloat16_as_ushort(__float2bfloat16_rn(x));
  } else {
    return __half_as_ushort(__float2half_rn(x));
  }
}

// The sequence whose packed rows hold row `t`: the largest b with cu[b] <= t among b0.. (cu is
// non-decreasing where it is right; where it is not, the caller's own range test refuses the row).
// The block's first row is located by all its threads at once (one round of loads for as many
// sequences as it has threads, 128 in the kernels here), the others by walking on from there.
__device__ __forceinline__ int block_first_sequence(const int* cu, int batch, int t) {
  int n = 0;
  for (int base = 0; base < batch; base += static_cast<int>(blockDim.x)) {
    const int i = base + static_cast<int>(threadIdx.x);
    n += __syncthreads_count(i < batch && __ldg(cu + i + 1) <= t);
  }
  return n;
}
__device__ __forceinline__ int walk_sequence(const int* cu, int batch, int b, int t) {
  while (b < batch && __ldg(cu + b + 1) <= t) ++b;
  return b;
}

// Sums that fall, or go past the tensor's `total` rows, are reported, by the first block.
__device__ __forceinline__ void check_sums(const int* cu, int batch, int total, int* err) {
  if (blockIdx.x != 0) return;
  for (int i = static_cast<int>(threadIdx.x); i < batch; i += static_cast<int>(blockDim.x)) {
    const int from = __ldg(cu + i), to = __ldg(cu + i + 1);
    if (from < 0 || to < from || to > total) report(err, FA2_ERR_SHAPE);
  }
}

// n / d by a multiplication, 0 <= n < 2^31: hi(n mul) >> shift with mul = 2^(31 + s) / d + 1, d <= 2^s
// (too large by less than n 2^-(31 + s) < 1 / d).
struct Divisor {
  int d;
  uint32_t mul;
  int shift;
};
FA2_HOST_DEVICE int divide(const Divisor& v, int n) {
#ifdef __CUDA_ARCH__
  const uint32_t hi = __umulhi(static_cast<uint32_t>(n), v.mul);
#else
  const uint32_t hi = static_cast<uint32_t>(static_cast<uint64_t>(static_cast<uint32_t>(n)) * v.mul >> 32);
#endif
  return v.d == 1 ? n : static_cast<int>(hi >> v.shift);
}

// ------------------------------------------------------------------------------------ host
inline Divisor divisor(int d) {
  Divisor v{d, 0, 0};
  if (d > 1) {
    int log = 1;
    while ((1ll << log) < d) ++log;
    v.mul = static_cast<uint32_t>((1ull << (31 + log)) / static_cast<uint64_t>(d) + 1);
    v.shift = log - 1;
  }
  return v;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

inline bool page_size_ok(int n) { return n == 16 || n == 32 || n == 64 || (n >= 128 && n % 128 == 0); }

inline int check_cache(const Fa2Kv8Cache& c) {
  if (c.k == nullptr || c.v == nullptr || c.k_scale == nullptr || c.v_scale == nullptr) return FA2_ERR_NULL;
  if (c.num_pages < 1 || c.heads_kv < 1 || !page_size_ok(c.page_size)) return FA2_ERR_SHAPE;
  if (c.head_dim != 16 && c.head_dim != 32 && c.head_dim != 64 && c.head_dim != 128) return FA2_ERR_HEAD_DIM;
  if (!aligned16(c.k) || !aligned16(c.v)) return FA2_ERR_LAYOUT;
  if ((reinterpret_cast<uintptr_t>(c.k_scale) & 3u) != 0 || (reinterpret_cast<uintptr_t>(c.v_scale) & 3u) != 0) {
    return FA2_ERR_LAYOUT;
  }
  const int64_t n[3] = {c.num_pages, c.page_size, c.heads_kv};
  for (int i = 0; i < 3; ++i) {
    if (n[i] <= 1) continue;  // the stride of a single entry is never used
    if (((c.k_stride[i] | c.v_stride[i]) & 15) != 0) return FA2_ERR_LAYOUT;
    const int64_t most = i == 0 ? 0x7fffffffll * 16 : 0x7fffffffll, most_s = 0x7fffffffll;
    if (c.k_stride[i] < 0 || c.v_stride[i] < 0 || c.ks_stride[i] < 0 || c.vs_stride[i] < 0 || c.k_stride[i] > most ||
        c.v_stride[i] > most || c.ks_stride[i] > most_s || c.vs_stride[i] > most_s) {
      return FA2_ERR_LAYOUT;
    }
  }
  return FA2_OK;
}

inline Cache device_cache(const Fa2Kv8Cache& c) {
  Cache d{};
  d.k = static_cast<const uint8_t*>(c.k);
  d.v = static_cast<const uint8_t*>(c.v);
  d.ks = c.k_scale;
  d.vs = c.v_scale;
  d.num_pages = c.num_pages;
  d.page_size = c.page_size;
  d.page_shift = -1;
  for (int s = 4; s < 31; ++s) {
    if (c.page_size == (1 << s)) d.page_shift = s;
  }
  d.heads_kv = c.heads_kv;
  if (c.num_pages > 1) {
    d.k_page16 = static_cast<int>(c.k_stride[0] / 16);
    d.v_page16 = static_cast<int>(c.v_stride[0] / 16);
    d.ks_page = static_cast<int>(c.ks_stride[0]);
    d.vs_page = static_cast<int>(c.vs_stride[0]);
  }
  d.k_row = static_cast<int>(c.k_stride[1]);
  d.v_row = static_cast<int>(c.v_stride[1]);
  d.ks_row = static_cast<int>(c.ks_stride[1]);
  d.vs_row = static_cast<int>(c.vs_stride[1]);
  if (c.heads_kv > 1) {
    d.k_head = static_cast<int>(c.k_stride[2]);
    d.v_head = static_cast<int>(c.v_stride[2]);
    d.ks_head = static_cast<int>(c.ks_stride[2]);
    d.vs_head = static_cast<int>(c.vs_stride[2]);
  }
  return d;
}

constexpr int MAX_DEVICES = 64;

// The current device, or -1 where it is not an sm_100 one. Each device is asked once: the two
// attribute queries cost as much as a launch. (Threads that race here write the same value.)
inline int sm100_device() {
  static std::atomic<signed char> known[MAX_DEVICES];  // 0: not asked, 1: sm_100, -1: another
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= MAX_DEVICES) return -1;
  signed char k = known[dev].load(std::memory_order_relaxed);
  if (k == 0) {
    int major = 0, minor = 0;
    if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, dev) != cudaSuccess) {
      return -1;
    }
    k = major == 10 && minor == 0 ? 1 : -1;
    known[dev].store(k, std::memory_order_relaxed);
  }
  return k > 0 ? dev : -1;
}

inline int launch_status() { return cudaGetLastError() == cudaSuccess ? FA2_OK : FA2_ERR_LAUNCH; }

}  // namespace fa2kv
