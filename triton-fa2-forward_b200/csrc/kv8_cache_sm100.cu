// The 8-bit paged K/V cache for sm_100a: rows of 16-bit keys and values are quantised to e4m3 as
// they are written into their pages, and read back. Memory bound both ways: 3 bytes a value and 4
// a row.
//
// A row of D values is held by D / 16 neighbouring lanes, 16 values each (two 16-byte loads, one
// 16-byte store of codes), the largest magnitude by shuffles among them. A thread has the key's
// and the value's row of the same token and head: they share the page, and four loads are in
// flight. Heads run fastest, as the packed tokens have them in memory.

#include "kv8_common.cuh"

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
  int64_t rows;                 // tokens * heads
};

// Where a token lives: its page and row, or false where it is not to be touched.
__device__ __forceinline__ bool find_row(const RowArgs& a, int b, int pos, int64_t& page, int& row) {
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

// Token t and head h of a block's thread. 32-bit arithmetic: the host bounds rows * L below 2^40
// and the tokens below 2^31.
__device__ __forceinline__ void token_head(const RowArgs& a, int64_t row, int& t, int& h) {
  if (a.rows <= 0xffffffffll) {
    const uint32_t q = static_cast<uint32_t>(row) / static_cast<uint32_t>(a.c.heads_kv);
    t = static_cast<int>(q);
    h = static_cast<int>(static_cast<uint32_t>(row) - q * a.c.heads_kv);
  } else {
    const int64_t q = row / a.c.heads_kv;
    t = static_cast<int>(q);
    h = static_cast<int>(row - q * a.c.heads_kv);
  }
}

template <bool BF16, bool VEC>
__device__ __forceinline__ void load16(const uint16_t* x, int64_t d_stride, float (&f)[16]) {
  if constexpr (VEC) {
    const uint4 w0 = *reinterpret_cast<const uint4*>(x), w1 = *reinterpret_cast<const uint4*>(x + 8);
    const uint32_t w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 v = float2_of_x2<BF16>(w[i]);
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) f[i] = float_of_16<BF16>(x[i * d_stride]);
  }
}

// The row's scale from its lanes' values; NaN where a value is not finite.
template <int L>
__device__ __forceinline__ float row_scale(const float (&f)[16]) {
  uint32_t m = 0;  // magnitudes compare as integers, NaN above infinity: nothing is lost in the max
#pragma unroll
  for (int i = 0; i < 16; ++i) m = max(m, __float_as_uint(f[i]) & 0x7fffffffu);
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m < 0x7f800000u ? __uint_as_float(m) / E4M3_MAX : __uint_as_float(0x7fc00000u);
}

__device__ __forceinline__ uint4 codes16(const float (&f)[16], float scale) {
  const bool some = scale > 0.0f;  // false for a zero row and for a NaN scale: codes 0
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float q[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) q[j] = some ? f[4 * i + j] / scale : 0.0f;
    w[i] = static_cast<uint32_t>(e4m3x2(q[0], q[1])) | (static_cast<uint32_t>(e4m3x2(q[2], q[3])) << 16);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int D, bool BF16, bool VEC>
__global__ void __launch_bounds__(128) append_kernel(const RowArgs a) {
  constexpr int L = D / 16;
  const int64_t idx0 = static_cast<int64_t>(blockIdx.x) * 128;
  const int64_t row_id = (idx0 + threadIdx.x) / L;
  const int part = threadIdx.x % L;
  bool on = row_id < a.rows;
  int t = 0, h = 0, b, i, n_new;
  token_head(a, on ? row_id : a.rows - 1, t, h);
  if (a.cu != nullptr) {
    int t0, h0;
    token_head(a, min(idx0 / L, a.rows - 1), t0, h0);
    b = walk_sequence(a.cu, a.batch, block_first_sequence(a.cu, a.batch, t0), t);
    if (b >= a.batch) {  // behind the last sequence
      on = false;
      b = a.batch - 1;
    }
    const int start = __ldg(a.cu + b);
    n_new = __ldg(a.cu + b + 1) - start;
    i = t - start;
    if (i < 0) on = false;  // a row before the first sequence
  } else {
    b = t / a.n;
    i = t - b * a.n;
    n_new = a.n;
  }
  const int len = __ldg(a.lens + b);
  if (a.cu == nullptr && len == 0) on = false;  // no sequence in this slot
  const int pos = len - n_new + i;
  if (on && (pos < 0 || len < n_new)) {
    report(a.err, FA2_ERR_SHAPE);
    on = false;
  }
  int64_t page = 0;
  int row = 0;
  if (on) on = find_row(a, b, pos, page, row);
  float f[2][16] = {};
  if (on) {
#pragma unroll
    for (int z = 0; z < 2; ++z) {
      const int64_t bi = a.cu != nullptr ? 0 : b, ni = a.cu != nullptr ? t : i;
      load16<BF16, VEC>(a.x[z] + bi * a.st[z][0] + h * a.st[z][1] + ni * a.st[z][2] + part * 16 * a.st[z][3],
                        a.st[z][3], f[z]);
    }
  }
#pragma unroll
  for (int z = 0; z < 2; ++z) {
    const float scale = row_scale<L>(f[z]);  // shuffles: all lanes
    if (on) {
      const int64_t* st = z ? a.c.v_st : a.c.k_st;
      const int64_t* sst = z ? a.c.vs_st : a.c.ks_st;
      uint8_t* dst = const_cast<uint8_t*>(z ? a.c.v : a.c.k) + page * st[0] + row * st[1] + h * st[2] + part * 16;
      *reinterpret_cast<uint4*>(dst) = codes16(f[z], scale);
      if (part == 0) const_cast<float*>(z ? a.c.vs : a.c.ks)[page * sst[0] + row * sst[1] + h * sst[2]] = scale;
    }
  }
}

template <int D, bool BF16>
__global__ void __launch_bounds__(128) read_kernel(const RowArgs a) {
  constexpr int L = D / 16;
  const int64_t idx0 = static_cast<int64_t>(blockIdx.x) * 128;
  const int64_t row_id = (idx0 + threadIdx.x) / L;
  const int part = threadIdx.x % L;
  int t, h, t0, h0;
  token_head(a, min(row_id, a.rows - 1), t, h);
  token_head(a, min(idx0 / L, a.rows - 1), t0, h0);
  const int b = walk_sequence(a.cu, a.batch, block_first_sequence(a.cu, a.batch, t0), t);
  if (row_id >= a.rows || b >= a.batch) return;
  const int pos = t - __ldg(a.cu + b);
  if (pos < 0) return;
  int64_t page = 0;
  int row = 0;
  const bool on = find_row(a, b, pos, page, row);
  uint4 w[2] = {};
  float scale[2] = {};
  if (on) {
#pragma unroll
    for (int z = 0; z < 2; ++z) {
      const int64_t* st = z ? a.c.v_st : a.c.k_st;
      const int64_t* sst = z ? a.c.vs_st : a.c.ks_st;
      w[z] = *reinterpret_cast<const uint4*>((z ? a.c.v : a.c.k) + page * st[0] + row * st[1] + h * st[2] + part * 16);
      scale[z] = (z ? a.c.vs : a.c.ks)[page * sst[0] + row * sst[1] + h * sst[2]];
    }
  }
#pragma unroll
  for (int z = 0; z < 2; ++z) {
    const uint32_t c[4] = {w[z].x, w[z].y, w[z].z, w[z].w};
    uint32_t o[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 lo = float2_of_f16x2(f16x2_of_e4m3x2(static_cast<uint16_t>(c[i])));
      const float2 hi = float2_of_f16x2(f16x2_of_e4m3x2(static_cast<uint16_t>(c[i] >> 16)));
      o[2 * i] = x2_of_floats<BF16>(lo.x * scale[z], lo.y * scale[z]);
      o[2 * i + 1] = x2_of_floats<BF16>(hi.x * scale[z], hi.y * scale[z]);
    }
    uint16_t* dst = const_cast<uint16_t*>(a.x[z]) + row_id * D + part * 16;
    *reinterpret_cast<uint4*>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
    *reinterpret_cast<uint4*>(dst + 8) = make_uint4(o[4], o[5], o[6], o[7]);
  }
}

template <int D>
int launch_append(const RowArgs& a, bool bf, bool vec, cudaStream_t s) {
  const int64_t blocks = (a.rows * (D / 16) + 127) / 128;
  if (blocks > 0x7fffffffll) return FA2_ERR_SHAPE;
  const unsigned g = static_cast<unsigned>(blocks);
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
  const int64_t blocks = (a.rows * (D / 16) + 127) / 128;
  if (blocks > 0x7fffffffll) return FA2_ERR_SHAPE;
  const unsigned g = static_cast<unsigned>(blocks);
  if (bf) read_kernel<D, true><<<g, 128, 0, s>>>(a);
  else read_kernel<D, false><<<g, 128, 0, s>>>(a);
  return launch_status();
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
  if (p->batch < 1 || p->seqlen < 0 || p->pages_per_seq < 1) return FA2_ERR_SHAPE;
  if (static_cast<int64_t>(p->batch) * (p->cu_seqlens != nullptr ? 1 : p->seqlen) > 0x7fffffffll) return FA2_ERR_SHAPE;
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
  a.rows = tokens * p->cache.heads_kv;
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
  if (p->batch < 1 || p->total < 0 || p->pages_per_seq < 1) return FA2_ERR_SHAPE;
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
  a.rows = static_cast<int64_t>(p->total) * p->cache.heads_kv;
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
