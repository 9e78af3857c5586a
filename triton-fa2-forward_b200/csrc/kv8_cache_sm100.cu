// The 8-bit paged K/V cache for sm_100a: rows of 16-bit keys and values are quantised to e4m3 as
// they are written into their pages, and read back. Memory bound both ways: 3 bytes a value and 4
// a row.
//
// A row of D values is held by D / 16 neighbouring lanes, 8 values of each half, so that every load
// and store of a row is of consecutive bytes (16 values in a piece took 87 us in place of 76 for the
// reading below: half-filled sectors). The largest magnitude comes by shuffles among them. A thread has
// the key's and the value's row of the same token and head: they share the page, and four loads are
// in flight. Heads run fastest, as the packed tokens have them in memory.
//
// Measured in a graph: append of 17,000 tokens of 8 heads of 128, 103 MB, 26 us (4.0 TB/s, 0.61 of the copy
// rate): the way from the sums over the table to the page lies before the stores, and a row costs
// some 300 instructions a lane for its maximum, quotients and codes (with divisions 39 us). Read of
// 157,000 tokens, 471 MB, 76 us (6.2 TB/s, 0.95); two or four rows a thread were no faster.

#include "kv8_common.cuh"

#include <algorithm>
#include <utility>

namespace {

using namespace fa2kv;

struct RowArgs {
  Cache c;
  const uint16_t* x[2];        // k, v (append) or the outputs (read)
  int64_t st[2][4];            // (b, h, n, d)
  const int* bt;
  const int* lens;
  const int* cu;
  int* err;
  int64_t bt_stride;
  int pages_per_seq, batch, n;  // n: tokens of a sequence, or all packed rows
  int rows;                     // tokens * heads
  Divisor by_heads, by_n;
  bool wide;  // an input stride needs more than 32 bits
};

// Where a token lives: its page and row, or false where it is not to be touched.
__device__ __forceinline__ bool find_row(const RowArgs& a, int b, int pos, int& page, int& row) {
  const int pi = page_of(a.c, pos);
  if (pi >= a.pages_per_seq) {
    report(a.err, FA2_ERR_SHAPE);
    return false;
  }
  const int pg = __ldg(a.bt + b * a.bt_stride + pi);
  if (pg < 0 || pg >= a.c.num_pages) {
    report(a.err, FA2_ERR_PAGE);
    return false;
  }
  page = pg;
  row = pos - pi * a.c.page_size;
  return true;
}

__device__ __forceinline__ void token_head(const RowArgs& a, int row, int& t, int& h) {
  t = divide(a.by_heads, row);
  h = row - t * a.c.heads_kv;
}

// Bytes (codes) or entries (scales) from a tensor's start to a row: widening 32-bit products.
__device__ __forceinline__ int64_t codes_at(const Cache& c, bool v, int page, int row, int h) {
  return (static_cast<int64_t>(page) * (v ? c.v_page16 : c.k_page16) << 4) + static_cast<int64_t>(row) * (v ? c.v_row : c.k_row) +
         static_cast<int64_t>(h) * (v ? c.v_head : c.k_head);
}
__device__ __forceinline__ int64_t scale_at(const Cache& c, bool v, int page, int row, int h) {
  return static_cast<int64_t>(page) * (v ? c.vs_page : c.ks_page) + static_cast<int64_t>(row) * (v ? c.vs_row : c.ks_row) +
         static_cast<int64_t>(h) * (v ? c.vs_head : c.ks_head);
}

// An input row. Strides fit 32 bits unless the host says otherwise.
__device__ __forceinline__ const uint16_t* row_at(const RowArgs& a, int z, int b, int h, int n) {
  if (a.wide) return a.x[z] + b * a.st[z][0] + h * a.st[z][1] + n * a.st[z][2];
  return a.x[z] + static_cast<int64_t>(b) * static_cast<int>(a.st[z][0]) + static_cast<int64_t>(h) * static_cast<int>(a.st[z][1]) +
         static_cast<int64_t>(n) * static_cast<int>(a.st[z][2]);
}

// A lane's 16 values of a row, as they are in memory and as floats: 8 in each half, so that the lanes
// of a row ask for (and write) consecutive bytes.
template <int D, bool VEC>
__device__ __forceinline__ void load16(const uint16_t* x, int64_t d_stride, uint32_t (&w)[8]) {
  if constexpr (VEC) {
    const uint4 w0 = __ldcs(reinterpret_cast<const uint4*>(x)), w1 = __ldcs(reinterpret_cast<const uint4*>(x + D / 2));
    w[0] = w0.x;
    w[1] = w0.y;
    w[2] = w0.z;
    w[3] = w0.w;
    w[4] = w1.x;
    w[5] = w1.y;
    w[6] = w1.z;
    w[7] = w1.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int at = i < 4 ? 2 * i : D / 2 + 2 * i - 8;
      w[i] = static_cast<uint32_t>(x[at * d_stride]) | (static_cast<uint32_t>(x[(at + 1) * d_stride]) << 16);
    }
  }
}
template <bool BF16>
__device__ __forceinline__ void floats16(const uint32_t (&w)[8], float (&f)[16]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 v = float2_of_x2<BF16>(w[i]);
    f[2 * i] = v.x;
    f[2 * i + 1] = v.y;
  }
}

// The row's scale from its lanes' values; NaN where a value is not finite. The magnitudes' largest is
// taken two at a time in the type itself (exact; a NaN wins).
template <int L, bool BF16>
__device__ __forceinline__ float row_scale(const uint32_t (&w)[8]) {
  auto larger = [](uint32_t x, uint32_t y) -> uint32_t {
    uint32_t r;
    if constexpr (BF16) {
      asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y));
    } else {
      asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y));
    }
    return r;
  };
  uint32_t m = w[0] & 0x7fff7fffu;
#pragma unroll
  for (int i = 1; i < 8; ++i) m = larger(m, w[i] & 0x7fff7fffu);
  m = larger(m, __byte_perm(m, m, 0x1032));
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) m = larger(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float top = float2_of_x2<BF16>(m).x;
  return top < INFINITY ? top / E4M3_MAX : __uint_as_float(0x7fc00000u);
}

// x / scale, correctly rounded, by Markstein's theorem (1990): with r the rounded reciprocal of scale
// and q = x r, q + r (x - q scale) in fused multiply-adds is the rounded quotient. Three instructions
// where the division takes about ten; for scales where r or the remainder could leave the normal
// range (a largest value below 2^-71) the division itself.
__device__ __forceinline__ uint4 codes16(const float (&f)[16], float scale) {
  const bool some = scale > 0.0f;  // false for a zero row and for a NaN scale: codes 0
  const bool plain = scale > 0x1p-80f && scale < 0x1p120f;
  const float r = plain ? 1.0f / scale : 0.0f;
  float q[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float q0 = f[i] * r;
    q[i] = fmaf(fmaf(-q0, scale, f[i]), r, q0);
  }
  if (some && !plain) {
#pragma unroll 1
    for (int i = 0; i < 16; ++i) {
#pragma unroll
      for (int j = 0; j < 16; ++j) q[j] = j == i ? f[j] / scale : q[j];
    }
  }
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = some ? static_cast<uint32_t>(e4m3x2(q[4 * i], q[4 * i + 1])) | (static_cast<uint32_t>(e4m3x2(q[4 * i + 2], q[4 * i + 3])) << 16)
                : 0u;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int D, bool BF16, bool VEC>
__global__ void __launch_bounds__(128) append_kernel(const RowArgs a) {
  constexpr int L = D / 16;
  constexpr int ROWS = 128 / L;  // of a block
  const int first = static_cast<int>(blockIdx.x) * ROWS;
  const int part = threadIdx.x % L, row_id = first + static_cast<int>(threadIdx.x) / L;
  bool on = row_id < a.rows;
  int t = 0, h = 0, b, i, n_new;
  token_head(a, on ? row_id : a.rows - 1, t, h);
  // The rows are asked for before the way to their pages is walked.
  uint32_t raw[2][8];
  const int tb = a.cu != nullptr ? 0 : divide(a.by_n, t), tn = a.cu != nullptr ? t : t - tb * a.n;
#pragma unroll
  for (int z = 0; z < 2; ++z) {
    load16<D, VEC>(row_at(a, z, tb, h, tn) + part * 8 * a.st[z][3], a.st[z][3], raw[z]);
  }
  if (a.cu != nullptr) {
    int t0, h0;
    token_head(a, first, t0, h0);
    b = walk_sequence(a.cu, a.batch, block_first_sequence(a.cu, a.batch, t0), t);
    if (b >= a.batch) {  // behind the last sequence
      on = false;
      b = a.batch - 1;
    }
    const int start = __ldg(a.cu + b), end = __ldg(a.cu + b + 1);
    n_new = end - start;
    i = t - start;
    if (i < 0 || end > a.n) on = false;  // a row before the first sequence; a sequence that goes past the tensor
  } else {
    b = tb;
    i = tn;
    n_new = a.n;
  }
  const int len = __ldg(a.lens + b);
  if (a.cu == nullptr && len == 0) on = false;  // no sequence in this slot
  const int pos = len - n_new + i;
  if (on && (pos < 0 || len < n_new)) {
    report(a.err, FA2_ERR_SHAPE);
    on = false;
  }
  int page = 0, row = 0;
  if (on) on = find_row(a, b, pos, page, row);
#pragma unroll
  for (int z = 0; z < 2; ++z) {
    float f[16];
    floats16<BF16>(raw[z], f);
    const float scale = row_scale<L, BF16>(raw[z]);  // shuffles: all lanes
    if (on) {
      uint8_t* dst = const_cast<uint8_t*>(z ? a.c.v : a.c.k) + codes_at(a.c, z != 0, page, row, h) + part * 8;
      const uint4 w = codes16(f, scale);
      *reinterpret_cast<uint2*>(dst) = make_uint2(w.x, w.y);
      *reinterpret_cast<uint2*>(dst + D / 2) = make_uint2(w.z, w.w);
      if (part == 0) const_cast<float*>(z ? a.c.vs : a.c.ks)[scale_at(a.c, z != 0, page, row, h)] = scale;
    }
  }
  if (a.cu != nullptr) check_sums(a.cu, a.batch, a.n, a.err);
}

template <int D, bool BF16>
__global__ void __launch_bounds__(128) read_kernel(const RowArgs a) {
  constexpr int L = D / 16;
  constexpr int ROWS = 128 / L;  // of a block
  const int first = static_cast<int>(blockIdx.x) * ROWS;
  const int part = threadIdx.x % L, row_id = first + static_cast<int>(threadIdx.x) / L;
  int t, h, t0, h0;
  token_head(a, min(row_id, a.rows - 1), t, h);
  token_head(a, first, t0, h0);
  const int b = walk_sequence(a.cu, a.batch, block_first_sequence(a.cu, a.batch, t0), t);
  check_sums(a.cu, a.batch, a.n, a.err);
  if (row_id >= a.rows || b >= a.batch) return;
  const int pos = t - __ldg(a.cu + b);
  if (pos < 0) return;
  int page = 0, row = 0;
  uint2 w[2][2] = {};
  float scale[2] = {};
  const bool whole = __ldg(a.cu + b + 1) <= a.n;  // a sequence that goes past the tensor: zeros
  if (find_row(a, b, pos, page, row) && whole) {
#pragma unroll
    for (int z = 0; z < 2; ++z) {
      const uint8_t* src = (z ? a.c.v : a.c.k) + codes_at(a.c, z != 0, page, row, h) + part * 8;
      w[z][0] = __ldcs(reinterpret_cast<const uint2*>(src));
      w[z][1] = __ldcs(reinterpret_cast<const uint2*>(src + D / 2));
      scale[z] = (z ? a.c.vs : a.c.ks)[scale_at(a.c, z != 0, page, row, h)];
    }
  }
#pragma unroll
  for (int z = 0; z < 2; ++z) {
    uint16_t* dst = const_cast<uint16_t*>(a.x[z]) + static_cast<int64_t>(row_id) * D + part * 8;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t c[2] = {w[z][i].x, w[z][i].y};
      uint32_t o[4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float2 lo = float2_of_f16x2(f16x2_of_e4m3x2(static_cast<uint16_t>(c[j])));
        const float2 hi = float2_of_f16x2(f16x2_of_e4m3x2(static_cast<uint16_t>(c[j] >> 16)));
        o[2 * j] = x2_of_floats<BF16>(lo.x * scale[z], lo.y * scale[z]);
        o[2 * j + 1] = x2_of_floats<BF16>(hi.x * scale[z], hi.y * scale[z]);
      }
      *reinterpret_cast<uint4*>(dst + i * (D / 2)) = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
}

template <int D>
int launch_append(const RowArgs& a, bool bf, bool vec, cudaStream_t s) {
  constexpr int ROWS = 128 / (D / 16);
  const unsigned g = (static_cast<unsigned>(a.rows) + ROWS - 1) / ROWS;
  if (bf) {
    if (vec) append_kernel<D, true, true><<<g, 128, 0, s>>>(a);
    else append_kernel<D, true, false><<<g, 128, 0, s>>>(a);
  } else {
    if (vec) append_kernel<D, false, true><<<g, 128, 0, s>>>(a);
    else append_kernel<D, false, false><<<g, 128, 0, s>>>(a);
  }
  return launch_status();
}

template <int D>
int launch_read(const RowArgs& a, bool bf, cudaStream_t s) {
  constexpr int ROWS = 128 / (D / 16);
  const unsigned g = (static_cast<unsigned>(a.rows) + ROWS - 1) / ROWS;
  if (bf) read_kernel<D, true><<<g, 128, 0, s>>>(a);
  else read_kernel<D, false><<<g, 128, 0, s>>>(a);
  return launch_status();
}

// Whether the rows of a cache tensor, `inner` values each, lie apart: sorted by stride, each dimension's
// step is past all that the smaller ones span (as in every slice of a dense tensor).
bool rows_apart(const Fa2Kv8Cache& c, const int64_t (&stride)[3], int64_t inner) {
  std::pair<int64_t, int64_t> dims[3] = {{stride[0], c.num_pages}, {stride[1], c.page_size}, {stride[2], c.heads_kv}};
  std::sort(dims, dims + 3);
  int64_t span = inner;
  for (const auto& [step, n] : dims) {
    if (n <= 1) continue;
    if (step < span) return false;
    span += step * (n - 1);
  }
  return true;
}

bool vec_rows(const void* p, const int64_t st[4], int64_t nb, int64_t nh, int64_t nn) {
  return aligned16(p) && st[3] == 1 && (nb <= 1 || (st[0] & 7) == 0) && (nh <= 1 || (st[1] & 7) == 0) &&
         (nn <= 1 || (st[2] & 7) == 0);
}

}  // namespace

extern "C" {

int fa2_kvcache_sm100_abi_version(void) { return FA2_KVCACHE_ABI_VERSION; }

int64_t fa2_kvcache_sm100_params_size(int32_t which) {
  switch (which) {
    case 0: return static_cast<int64_t>(sizeof(Fa2RotaryParams));
    case 1: return static_cast<int64_t>(sizeof(Fa2Kv8AppendParams));
    case 2: return static_cast<int64_t>(sizeof(Fa2Kv8ReadParams));
    case 3: return static_cast<int64_t>(sizeof(Fa2Kv8AttnParams));
    default: return -1;
  }
}

int fa2_kv8_append_sm100_check(const Fa2Kv8AppendParams* p) {
  if (p == nullptr || p->k == nullptr || p->v == nullptr || p->block_table == nullptr || p->cache_seqlens == nullptr) {
    return FA2_ERR_NULL;
  }
  const int rc = check_cache(p->cache);
  if (rc != FA2_OK) return rc;
  const Fa2Kv8Cache& c = p->cache;
  if (!rows_apart(c, c.k_stride, c.head_dim) || !rows_apart(c, c.v_stride, c.head_dim) || !rows_apart(c, c.ks_stride, 1) ||
      !rows_apart(c, c.vs_stride, 1)) {
    return FA2_ERR_LAYOUT;
  }
  if (p->batch < 1 || p->seqlen < 0 || p->pages_per_seq < 1) return FA2_ERR_SHAPE;
  // Rows (tokens x heads) are counted in 31 bits.
  if (static_cast<int64_t>(p->cu_seqlens != nullptr ? 1 : p->batch) * p->seqlen > 0x7fff0000ll / p->cache.heads_kv) return FA2_ERR_SHAPE;
  if (p->dtype != FA2_DTYPE_FP16 && p->dtype != FA2_DTYPE_BF16) return FA2_ERR_DTYPE;
  return FA2_OK;
}

int fa2_kv8_append_sm100(const Fa2Kv8AppendParams* p, void* stream) {
  const int rc = fa2_kv8_append_sm100_check(p);
  if (rc != FA2_OK || p->seqlen == 0) return rc;
  if (sm100_device() < 0) return FA2_ERR_DEVICE;
  RowArgs a{};
  a.c = device_cache(p->cache);
  a.x[0] = static_cast<const uint16_t*>(p->k);
  a.x[1] = static_cast<const uint16_t*>(p->v);
  for (int i = 0; i < 4; ++i) {
    a.st[0][i] = p->k_in_stride[i];
    a.st[1][i] = p->v_in_stride[i];
  }
  a.bt = p->block_table;
  a.lens = p->cache_seqlens;
  a.cu = p->cu_seqlens;
  a.err = p->err_flag;
  a.bt_stride = p->block_table_stride;
  a.pages_per_seq = p->pages_per_seq;
  a.batch = p->batch;
  a.n = p->seqlen;
  const int64_t tokens = p->cu_seqlens != nullptr ? p->seqlen : static_cast<int64_t>(p->batch) * p->seqlen;
  a.rows = static_cast<int>(tokens * p->cache.heads_kv);
  a.by_heads = divisor(p->cache.heads_kv);
  a.by_n = divisor(p->seqlen);
  for (int z = 0; z < 2; ++z) {
    for (int i = 0; i < 3; ++i) a.wide = a.wide || a.st[z][i] < -0x7fffffffll || a.st[z][i] > 0x7fffffffll;
  }
  const int64_t nb = p->cu_seqlens != nullptr ? 1 : p->batch;
  const bool vec = vec_rows(p->k, p->k_in_stride, nb, p->cache.heads_kv, p->seqlen) &&
                   vec_rows(p->v, p->v_in_stride, nb, p->cache.heads_kv, p->seqlen);
  const bool bf = p->dtype == FA2_DTYPE_BF16;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (p->cache.head_dim) {
    case 16: return launch_append<16>(a, bf, vec, s);
    case 32: return launch_append<32>(a, bf, vec, s);
    case 64: return launch_append<64>(a, bf, vec, s);
    default: return launch_append<128>(a, bf, vec, s);
  }
}

int fa2_kv8_read_sm100_check(const Fa2Kv8ReadParams* p) {
  if (p == nullptr || p->k_out == nullptr || p->v_out == nullptr || p->block_table == nullptr || p->cu_seqlens == nullptr) {
    return FA2_ERR_NULL;
  }
  const int rc = check_cache(p->cache);
  if (rc != FA2_OK) return rc;
  if (p->batch < 1 || p->total < 0 || p->pages_per_seq < 1 || p->total > 0x7fff0000 / p->cache.heads_kv) return FA2_ERR_SHAPE;
  if (p->dtype != FA2_DTYPE_FP16 && p->dtype != FA2_DTYPE_BF16) return FA2_ERR_DTYPE;
  if (!aligned16(p->k_out) || !aligned16(p->v_out)) return FA2_ERR_LAYOUT;
  return FA2_OK;
}

int fa2_kv8_read_sm100(const Fa2Kv8ReadParams* p, void* stream) {
  const int rc = fa2_kv8_read_sm100_check(p);
  if (rc != FA2_OK || p->total == 0) return rc;
  if (sm100_device() < 0) return FA2_ERR_DEVICE;
  RowArgs a{};
  a.c = device_cache(p->cache);
  a.x[0] = static_cast<const uint16_t*>(p->k_out);
  a.x[1] = static_cast<const uint16_t*>(p->v_out);
  a.bt = p->block_table;
  a.cu = p->cu_seqlens;
  a.err = p->err_flag;
  a.bt_stride = p->block_table_stride;
  a.pages_per_seq = p->pages_per_seq;
  a.batch = p->batch;
  a.n = p->total;
  a.rows = p->total * p->cache.heads_kv;
  a.by_heads = divisor(p->cache.heads_kv);
  const bool bf = p->dtype == FA2_DTYPE_BF16;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (p->cache.head_dim) {
    case 16: return launch_read<16>(a, bf, s);
    case 32: return launch_read<32>(a, bf, s);
    case 64: return launch_read<64>(a, bf, s);
    default: return launch_read<128>(a, bf, s);
  }
}

}  // extern "C"
