// Rotary positions for sm_100a: q and k of one call in one launch.
//
// A pair (a, c) of a head's values at position p turns by t = p * f_i. The angle is kept in turns
// and in 64 bits until its whole turns are gone: u = p * (f_i / 2 pi), u - rint(u) in [-1/2, 1/2]
// (error about p * 2^-54 turns, 4e-10 radians at p = 10^6, where 32 bits would be off by 0.06),
// then sincospi in fp32. Memory bound: every value is read and written once, 4 bytes a 16-bit
// value; no table of angles is read.
//
// Split: a thread owns 8 pairs of a token (16 values of each head) and turns them in up to
// HEADS_PER_THREAD heads, so the sines are computed once for several heads and all their loads are
// in flight together. Few tokens take one head a thread instead, which fills more SMs. Measured:
// 53 us in a graph for 16384 tokens of 32 + 8 heads of 128 (336 MB: 6.3 TB/s, 0.97 of the copy rate; 59 us
// as ordinary calls), 2.8 us for 8 tokens, which is the launch. 3000 tokens of 16 heads take one head a
// thread and form their angles in each: 6.2 us.

#include "kv8_common.cuh"

namespace {

using namespace fa2kv;

struct RotArgs {
  const uint16_t* x[2];  // q, k
  uint16_t* y[2];
  int64_t xs[2][4], ys[2][4];  // (b, h, n, d)
  const void* pos;
  int64_t pos_st[2];
  const double* freq;
  int pos64;
  int n;            // tokens of a batch entry
  int heads[2];     // q, k
  int chunks;       // head chunks of a token
  int units;        // threads of a head chunk
  int d, rd;
  float mag, sign;
  int64_t rows;     // batch * n * chunks
};

constexpr double INV_2PI = 0.15915494309189535;

__device__ __forceinline__ double position(const RotArgs& a, int64_t b, int64_t n) {
  const int64_t at = b * a.pos_st[0] + n * a.pos_st[1];
  return a.pos64 ? static_cast<double>(__ldg(static_cast<const long long*>(a.pos) + at))
                 : static_cast<double>(__ldg(static_cast<const int*>(a.pos) + at));
}

__device__ __forceinline__ void sine(const RotArgs& a, double pos, int i, float& s, float& c) {
  const double u = pos * (__ldg(a.freq + i) * INV_2PI);
  const float r = static_cast<float>(u - rint(u));
  sincospif(2.0f * r, &s, &c);
  s *= a.sign;
  c *= a.mag;
}

// row -> (b, n, chunk), in 32 bits where they do (the common case).
__device__ __forceinline__ void locate(const RotArgs& a, int64_t row, int64_t& b, int64_t& n, int& chunk) {
  if (a.rows <= 0xffffffffll) {
    const uint32_t r = static_cast<uint32_t>(row);
    const uint32_t t = r / static_cast<uint32_t>(a.chunks);
    chunk = static_cast<int>(r - t * a.chunks);
    const uint32_t bb = t / static_cast<uint32_t>(a.n);
    b = bb;
    n = t - bb * static_cast<uint32_t>(a.n);
  } else {
    const int64_t t = row / a.chunks;
    chunk = static_cast<int>(row - t * a.chunks);
    b = t / a.n;
    n = t - b * a.n;
  }
}

// 16-byte loads: rows of 16 * units values, the first rd / 16 units rotated, the others copied.
template <bool BF16, bool INTER, int HPT>
__global__ void __launch_bounds__(128) rotary_vec_kernel(const RotArgs a) {
  const int64_t idx = static_cast<int64_t>(blockIdx.x) * 128 + threadIdx.x;
  const int shift = 31 - __clz(a.units);  // units is a power of two here
  const int u = static_cast<int>(idx) & (a.units - 1);
  const int64_t row = idx >> shift;
  if (row >= a.rows) return;
  int64_t b, n;
  int chunk;
  locate(a, row, b, n, chunk);
  const int h0 = chunk * HPT;
  const int heads = a.heads[0] + a.heads[1];
  const bool turn = u * 16 < a.rd;
  // This thread's two 8-value pieces of a head.
  const int d0 = (INTER || !turn) ? u * 16 : u * 8;
  const int d1 = (INTER || !turn) ? u * 16 + 8 : u * 8 + a.rd / 2;
  uint4 w[HPT][2];
#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    const int h = h0 + i;
    if (h < heads) {
      const int z = h >= a.heads[0];
      const uint16_t* x = a.x[z] + b * a.xs[z][0] + (h - (z ? a.heads[0] : 0)) * a.xs[z][1] + n * a.xs[z][2];
      w[i][0] = *reinterpret_cast<const uint4*>(x + d0);
      w[i][1] = *reinterpret_cast<const uint4*>(x + d1);
    }
  }
  float s[8], c[8];
  if (turn) {
    const double pos = position(a, b, n);
#pragma unroll
    for (int i = 0; i < 8; ++i) sine(a, pos, u * 8 + i, s[i], c[i]);
  }
#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    const int h = h0 + i;
    if (h >= heads) break;
    if (turn) {
      uint32_t* p = reinterpret_cast<uint32_t*>(w[i]);
      if constexpr (INTER) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float2 v = float2_of_x2<BF16>(p[e]);
          p[e] = x2_of_floats<BF16>(v.x * c[e] - v.y * s[e], v.x * s[e] + v.y * c[e]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 v0 = float2_of_x2<BF16>(p[e]), v1 = float2_of_x2<BF16>(p[e + 4]);
          p[e] = x2_of_floats<BF16>(v0.x * c[2 * e] - v1.x * s[2 * e], v0.y * c[2 * e + 1] - v1.y * s[2 * e + 1]);
          p[e + 4] = x2_of_floats<BF16>(v0.x * s[2 * e] + v1.x * c[2 * e], v0.y * s[2 * e + 1] + v1.y * c[2 * e + 1]);
        }
      }
    }
    const int z = h >= a.heads[0];
    uint16_t* y = a.y[z] + b * a.ys[z][0] + (h - (z ? a.heads[0] : 0)) * a.ys[z][1] + n * a.ys[z][2];
    *reinterpret_cast<uint4*>(y + d0) = w[i][0];
    *reinterpret_cast<uint4*>(y + d1) = w[i][1];
  }
}

// Any strides and sizes: one pair (or two copied values) of one head a thread.
template <bool BF16>
__global__ void __launch_bounds__(128) rotary_any_kernel(const RotArgs a, int inter) {
  const int64_t idx = static_cast<int64_t>(blockIdx.x) * 128 + threadIdx.x;
  const int64_t row = idx / a.units;
  if (row >= a.rows) return;
  const int u = static_cast<int>(idx - row * a.units);
  int64_t b, n;
  int h;
  locate(a, row, b, n, h);
  const int z = h >= a.heads[0];
  const int hz = h - (z ? a.heads[0] : 0);
  const uint16_t* x = a.x[z] + b * a.xs[z][0] + hz * a.xs[z][1] + n * a.xs[z][2];
  uint16_t* y = a.y[z] + b * a.ys[z][0] + hz * a.ys[z][1] + n * a.ys[z][2];
  if (2 * u < a.rd) {
    const int i0 = inter ? 2 * u : u, i1 = inter ? 2 * u + 1 : u + a.rd / 2;
    const float v0 = float_of_16<BF16>(x[i0 * a.xs[z][3]]), v1 = float_of_16<BF16>(x[i1 * a.xs[z][3]]);
    float s, c;
    sine(a, position(a, b, n), u, s, c);
    y[i0 * a.ys[z][3]] = x1_of_float<BF16>(v0 * c - v1 * s);
    y[i1 * a.ys[z][3]] = x1_of_float<BF16>(v0 * s + v1 * c);
  } else {
    for (int i = 2 * u; i < min(2 * u + 2, a.d); ++i) y[i * a.ys[z][3]] = x[i * a.xs[z][3]];
  }
}

bool vec_layout(const void* p, const int64_t st[4], const int64_t n[3]) {
  if (!aligned16(p) || st[3] != 1) return false;
  for (int i = 0; i < 3; ++i) {
    if (n[i] > 1 && (st[i] & 7) != 0) return false;
  }
  return true;
}

template <bool BF16, bool INTER>
int launch_vec(RotArgs& a, int64_t tokens, int heads, cudaStream_t s) {
  // Heads a thread: 1 until a launch of one-head threads would be several waves of the GPU's
  // thread slots, then 4.
  const bool few = tokens * heads * a.units <= 148ll * 2048;
  const int hpt = few ? 1 : 4;
  a.chunks = (heads + hpt - 1) / hpt;
  a.rows = tokens * a.chunks;
  const int64_t blocks = (a.rows * a.units + 127) / 128;
  if (blocks > 0x7fffffffll) return FA2_ERR_SHAPE;
  if (few) {
    rotary_vec_kernel<BF16, INTER, 1><<<static_cast<unsigned>(blocks), 128, 0, s>>>(a);
  } else {
    rotary_vec_kernel<BF16, INTER, 4><<<static_cast<unsigned>(blocks), 128, 0, s>>>(a);
  }
  return launch_status();
}

}  // namespace

extern "C" {

int fa2_rotary_sm100_check(const Fa2RotaryParams* p) {
  if (p == nullptr || p->q == nullptr || p->q_out == nullptr || p->positions == nullptr || p->inv_freq == nullptr) {
    return FA2_ERR_NULL;
  }
  if ((p->k == nullptr) != (p->heads_kv == 0) || (p->k != nullptr && p->k_out == nullptr)) return FA2_ERR_NULL;
  if (p->batch < 1 || p->seqlen < 1 || p->heads_q < 1 || p->heads_kv < 0) return FA2_ERR_SHAPE;
  if (p->heads_q > (1 << 20) || p->heads_kv > (1 << 20)) return FA2_ERR_SHAPE;
  if (p->dtype != FA2_DTYPE_FP16 && p->dtype != FA2_DTYPE_BF16) return FA2_ERR_DTYPE;
  if (p->head_dim < 2 || p->head_dim > (1 << 16) || p->rotary_dim < 2 || p->rotary_dim > p->head_dim ||
      (p->rotary_dim & 1) != 0) {
    return FA2_ERR_HEAD_DIM;
  }
  if (!(p->magnitude > 0.0f) || p->magnitude > 3.0e38f) return FA2_ERR_SCALE;
  return FA2_OK;
}

int fa2_rotary_sm100(const Fa2RotaryParams* p, void* stream) {
  const int rc = fa2_rotary_sm100_check(p);
  if (rc != FA2_OK) return rc;
  if (sm100_device() < 0) return FA2_ERR_DEVICE;
  RotArgs a{};
  a.x[0] = static_cast<const uint16_t*>(p->q);
  a.x[1] = static_cast<const uint16_t*>(p->k);
  a.y[0] = static_cast<uint16_t*>(p->q_out);
  a.y[1] = static_cast<uint16_t*>(p->k_out);
  for (int i = 0; i < 4; ++i) {
    a.xs[0][i] = p->q_stride[i];
    a.xs[1][i] = p->k_stride[i];
    a.ys[0][i] = p->q_out_stride[i];
    a.ys[1][i] = p->k_out_stride[i];
  }
  a.pos = p->positions;
  a.pos_st[0] = p->pos_stride[0];
  a.pos_st[1] = p->pos_stride[1];
  a.freq = p->inv_freq;
  a.pos64 = p->pos_is_64;
  a.n = p->seqlen;
  a.heads[0] = p->heads_q;
  a.heads[1] = p->heads_kv;
  a.d = p->head_dim;
  a.rd = p->rotary_dim;
  a.mag = p->magnitude;
  a.sign = p->inverse ? -p->magnitude : p->magnitude;
  const int heads = p->heads_q + p->heads_kv;
  const int64_t tokens = static_cast<int64_t>(p->batch) * p->seqlen;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf = p->dtype == FA2_DTYPE_BF16;
  const int units = p->head_dim / 16;
  bool vec = p->head_dim % 16 == 0 && (units & (units - 1)) == 0 && p->rotary_dim % 16 == 0;
  const int64_t nq[3] = {p->batch, p->heads_q, p->seqlen}, nk[3] = {p->batch, p->heads_kv, p->seqlen};
  vec = vec && vec_layout(p->q, p->q_stride, nq) && vec_layout(p->q_out, p->q_out_stride, nq);
  if (p->k != nullptr) vec = vec && vec_layout(p->k, p->k_stride, nk) && vec_layout(p->k_out, p->k_out_stride, nk);
  if (vec) {
    a.units = units;
    if (p->interleaved) return bf ? launch_vec<true, true>(a, tokens, heads, s) : launch_vec<false, true>(a, tokens, heads, s);
    return bf ? launch_vec<true, false>(a, tokens, heads, s) : launch_vec<false, false>(a, tokens, heads, s);
  }
  a.units = (p->head_dim + 1) / 2;
  a.chunks = heads;
  a.rows = tokens * heads;
  const int64_t blocks = (a.rows * a.units + 127) / 128;
  if (blocks > 0x7fffffffll) return FA2_ERR_SHAPE;
  if (bf) {
    rotary_any_kernel<true><<<static_cast<unsigned>(blocks), 128, 0, s>>>(a, p->interleaved);
  } else {
    rotary_any_kernel<false><<<static_cast<unsigned>(blocks), 128, 0, s>>>(a, p->interleaved);
  }
  return launch_status();
}

}  // extern "C"
