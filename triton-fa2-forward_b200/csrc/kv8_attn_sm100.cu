// Attention of new tokens over the 8-bit paged cache, for sm_100a.

#include "kv8_attn.cuh"
#include "kv8_chunk.cuh"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace {

using namespace fa2kv;

// ------------------------------------------------------------------ few rows (decode)
// At most 16 rows (queries x heads of a group) a CTA. Bound by the bytes of the cache, 2 (D + 4) a
// key, as long as the instructions for them fit under the copies. So the tensor work runs on
// warp-wide products that take the codes straight from registers (two codes to fp16 in one
// instruction), and the rows are the products' narrow side: S^T = K Q^T and O^T = V^T P^T, 16 keys or
// 16 columns by 8 rows a product, so that 1 to 8 rows waste half of what 16-row tiles would.
// Every warp streams its own 32-key groups through its own ring of asynchronous copies (no barrier
// between warps) and keeps its own running max, sum and output; the four warps are merged once at
// the end. A 128-row tile would be 1/16 full and the way through shared memory and TMEM would cost
// more than the bytes. (Warp-wide e4m3 products in place of conversions and fp16 ones were slower, 162
// against 137 us at the time.) Measured in a graph: 4 sequences of 65536 keys, 8 kv heads of 128, one token,
// 554 MB, 92 us (6.0 TB/s, 0.92 of the copy rate), 16 rows in place of 4 113 us; one of 700 keys 11.6 us,
// most of it two launches and the way to the first key; 48 of up to 8192 keys, 2 kv heads of 64, 54 MB, 28 us.
// Ordinary calls of these: 96, 24 (the host's) and 29 us.
//
// Operand layouts, lane (g, c) = (lane / 4, lane % 4). The products sum over d (QK^T) and over keys
// (PV) in any order, so both operands use the order in which a lane's bytes lie in memory: for QK^T
// a lane reads D / 4 contiguous bytes of the keys g and g + 8, four to a 16-wide step; for PV D / 8
// contiguous bytes at column g D / 8 of the keys 2c, 2c + 1, 2c + 8, 2c + 9, and interleaves pairs of
// keys, so it holds D / 8 contiguous output columns of the rows 2c and 2c + 1. P^T comes out of the
// first product with a lane's keys g, g + 8 and is turned by 8 x 8 transposes.

constexpr int DEC_WARPS = 4;
constexpr int DEC_KEYS = 32;   // of a group
constexpr int DEC_STAGES = 2;  // 12 warps an SM x one group on its way: 96 KB
constexpr int DEC_CTAS = 3;    // an SM at most
// CTAs an SM that the work is shared among: two, three where rows of codes are shorter. Two / three for 4
// sequences of 65536 keys and 8 kv heads: 128 dims 91 / 98 us, 64 59 / 55, 32 49 / 44, 16 46 / 40; for 48 of up
// to 8192 and 2 kv heads 38.5 / 37, 30 / 28, 25 / 23, 22.6 / 21; the same in fp16.
constexpr int dec_shares(int head_dim) { return head_dim > 64 ? 2 : 3; }

template <int D>
struct Dec {
  static constexpr int PIECES = D / 16;                    // 16-byte pieces of a row of codes
  static constexpr int CODES = DEC_KEYS * D;               // bytes of a group's K (or V) codes
  static constexpr int STAGE = 2 * CODES + 2 * DEC_KEYS * 4;  // and the scales
  static constexpr int OUT = 16 * (D + 4) * 4;             // the warp's output, later, in the same place
  static constexpr int RING = DEC_STAGES * STAGE > OUT ? DEC_STAGES * STAGE : OUT;
  static constexpr int SMEM = DEC_WARPS * RING + DEC_WARPS * 2 * 16 * 4;
  // 16-byte pieces of a row are stored at piece ^ swz(row): spreads the lanes' reads over the banks.
  __device__ static constexpr int swz_k(int row) { return D == 128 ? (row & 1) << 2 : 0; }
  __device__ static constexpr int swz_v(int row) { return D == 128 ? row & 6 : D == 64 ? (row >> 1) & 3 : 0; }
};

// c += a * b, fp16 operands, 16 x 8 x 16.
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
__device__ __forceinline__ uint32_t f16_lo(uint32_t w) { return f16x2_of_e4m3x2(static_cast<uint16_t>(w)); }
__device__ __forceinline__ uint32_t f16_hi(uint32_t w) { return f16x2_of_e4m3x2(static_cast<uint16_t>(w >> 16)); }

// N bytes (2, 4, 8, 16) of shared memory into words.
template <int N>
__device__ __forceinline__ void lds(uint32_t addr, uint32_t* w) {
  if constexpr (N == 16) {
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr));
  } else if constexpr (N == 8) {
    asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
  } else if constexpr (N == 4) {
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[0]) : "r"(addr));
  } else {
    uint16_t h;
    asm volatile("ld.shared.b16 %0, [%1];" : "=h"(h) : "r"(addr));
    w[0] = h;
  }
}

// Over the lanes of one c: the keys of a row.
__device__ __forceinline__ float keys_max(float x) {
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
  return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
}
__device__ __forceinline__ float keys_sum(float x) {
  x += __shfl_xor_sync(0xffffffffu, x, 4);
  x += __shfl_xor_sync(0xffffffffu, x, 8);
  return x + __shfl_xor_sync(0xffffffffu, x, 16);
}

// NT: 8-row tiles of the row block (1 or 2).
// One worker's part of the keys of one (sequence, kv head): keys [k0, k1). `slot`: where a partial
// result goes, -1 for a whole one.
template <int D, bool BF16, int NT>
__device__ __forceinline__ void decode_part(const AttnArgs& a, uint8_t* smem, const Seq& sq, int b, int h, int k0, int k1, int slot) {
  using C = Dec<D>;
  constexpr int ROWS = 8 * NT;
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x) >> 5, 0), lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  const int rows = sq.n_q * a.group;

  const uint32_t ring = fa2::smem_u32(smem) + warp * C::RING;
  const int n_groups = (k1 - k0 + DEC_KEYS - 1) / DEC_KEYS;
  const int mine = n_groups > warp ? (n_groups - warp + DEC_WARPS - 1) / DEC_WARPS : 0;
  const int* bt = a.bt + b * a.bt_stride;
  // A lane copies piece lane % PIECES of the rows lane / PIECES + STEP * i of a group, and the scales
  // of key `lane`.
  constexpr int STEP = 32 / C::PIECES;
  const int my_row = lane / C::PIECES, my_piece = lane % C::PIECES;
  const uint8_t* kh = a.c.k + static_cast<int64_t>(h) * a.c.k_head + my_piece * 16;
  const uint8_t* vh = a.c.v + static_cast<int64_t>(h) * a.c.v_head + my_piece * 16;
  const float* ksh = a.c.ks + static_cast<int64_t>(h) * a.c.ks_head;
  const float* vsh = a.c.vs + static_cast<int64_t>(h) * a.c.vs_head;
  auto group_pos = [&](int it) { return k0 + DEC_KEYS * (warp + DEC_WARPS * it); };
  // The next group's place: its page's index in the table, its first row there, and the page itself,
  // fetched one group ahead. Each half of a group, 16 keys, lies in one page; both do unless pages
  // have 16 rows. A warp's groups are 128 keys apart.
  const bool two = a.c.page_size == 16;
  int pi = page_of(a.c, group_pos(0)), row_in = group_pos(0) - pi * a.c.page_size;
  int next_page[2] = {0, 0};
  auto fetch_pages = [&](int it) {
    if (it >= mine) return;
    next_page[0] = next_page[1] = __ldg(bt + pi);
    if (two && group_pos(it) + 16 < sq.len) next_page[1] = __ldg(bt + pi + 1);
  };
  fetch_pages(0);
  // This lane's offsets within a stage and a page.
  const uint32_t to_k = my_row * D + ((my_piece ^ C::swz_k(my_row)) << 4);
  const uint32_t to_v = my_row * D + ((my_piece ^ C::swz_v(my_row)) << 4);
  const int64_t step_k = static_cast<int64_t>(STEP) * a.c.k_row, step_v = static_cast<int64_t>(STEP) * a.c.v_row;
  auto issue = [&](int it) {
    if (it < mine) {
      const int page[2] = {next_page[0], next_page[1]}, r0 = row_in, pos0 = group_pos(it);
      if (a.c.page_size < 128) {
        pi += 128 >> a.c.page_shift;
      } else {
        row_in += 128;
        if (row_in >= a.c.page_size) {
          row_in -= a.c.page_size;
          ++pi;
        }
      }
      fetch_pages(it + 1);
      const uint32_t st = ring + (it % DEC_STAGES) * C::STAGE;
      const uint32_t sc = st + 2 * C::CODES + lane * 4;
      const bool good[2] = {static_cast<unsigned>(page[0]) < static_cast<unsigned>(a.c.num_pages),
                            static_cast<unsigned>(page[1]) < static_cast<unsigned>(a.c.num_pages)};
      if (good[0] && good[1] && pos0 + DEC_KEYS <= sq.len && STEP <= 16) {
        const uint8_t* kp = kh + (static_cast<int64_t>(page[0]) * a.c.k_page16 << 4) + static_cast<int64_t>(r0 + my_row) * a.c.k_row;
        const uint8_t* vp = vh + (static_cast<int64_t>(page[0]) * a.c.v_page16 << 4) + static_cast<int64_t>(r0 + my_row) * a.c.v_row;
#pragma unroll
        for (int i = 0; i < C::PIECES; ++i) {
          if (i == C::PIECES / 2 && two) {
            kp = kh + (static_cast<int64_t>(page[1]) * a.c.k_page16 << 4) + static_cast<int64_t>(my_row) * a.c.k_row;
            vp = vh + (static_cast<int64_t>(page[1]) * a.c.v_page16 << 4) + static_cast<int64_t>(my_row) * a.c.v_row;
          }
          // Row i STEP + my_row; its swizzle differs from my_row's by that of i STEP.
          cp_async16_full(st + i * STEP * D + (to_k ^ (C::swz_k(i * STEP) << 4)), kp);
          cp_async16_full(st + C::CODES + i * STEP * D + (to_v ^ (C::swz_v(i * STEP) << 4)), vp);
          kp += step_k;
          vp += step_v;
        }
        const int pg = lane < 16 ? page[0] : page[1], r = two ? lane & 15 : r0 + lane;
        cp_async4(sc, ksh + static_cast<int64_t>(pg) * a.c.ks_page + static_cast<int64_t>(r) * a.c.ks_row, true);
        cp_async4(sc + DEC_KEYS * 4, vsh + static_cast<int64_t>(pg) * a.c.vs_page + static_cast<int64_t>(r) * a.c.vs_row, true);
      } else {
        // Rows past the end hold anything: zeros instead. A refused page: zeros and NaN scales,
        // queries that see its keys get NaN.
        if (!good[0] || !good[1]) report(a.err, FA2_ERR_PAGE);
        for (int i = 0; i < C::PIECES; ++i) {
          const int row = i * STEP + my_row;
          const bool ok = row < 16 ? good[0] : good[1], in = ok && pos0 + row < sq.len;
          const int pg = in ? (row < 16 ? page[0] : page[1]) : 0, r = in ? (two ? row & 15 : r0 + row) : 0;
          cp_async16(st + row * D + ((my_piece ^ C::swz_k(row)) << 4),
                     kh + (static_cast<int64_t>(pg) * a.c.k_page16 << 4) + static_cast<int64_t>(r) * a.c.k_row, in);
          cp_async16(st + C::CODES + row * D + ((my_piece ^ C::swz_v(row)) << 4),
                     vh + (static_cast<int64_t>(pg) * a.c.v_page16 << 4) + static_cast<int64_t>(r) * a.c.v_row, in);
        }
        const bool ok = lane < 16 ? good[0] : good[1], in = ok && pos0 + lane < sq.len;
        const int pg = in ? (lane < 16 ? page[0] : page[1]) : 0, r = in ? (two ? lane & 15 : r0 + lane) : 0;
        if (ok) {
          cp_async4(sc, ksh + static_cast<int64_t>(pg) * a.c.ks_page + static_cast<int64_t>(r) * a.c.ks_row, in);
          cp_async4(sc + DEC_KEYS * 4, vsh + static_cast<int64_t>(pg) * a.c.vs_page + static_cast<int64_t>(r) * a.c.vs_row, in);
        } else {
          asm volatile("st.shared.b32 [%0], %1;" ::"r"(sc), "r"(0x7fc00000u) : "memory");
          asm volatile("st.shared.b32 [%0], %1;" ::"r"(sc + DEC_KEYS * 4), "r"(0u) : "memory");
        }
      }
    }
    cp_async_commit();  // also where there is nothing: the group count stays in step
  };
#pragma unroll
  for (int it = 0; it < DEC_STAGES; ++it) issue(it);

  // Q: this lane holds values of the rows 8 t + g, in the order described above, times the power of
  // two that brings the row's largest value below 2^15 (exact in fp16).
  uint32_t qb[NT][D / 16][2];
  __shared__ float q_scale[DEC_WARPS][16];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int row = 8 * t + g;
    constexpr int NB = D >= 64 ? 16 : D / 4;  // values of a contiguous piece
    uint32_t w[D / 8];                        // D / 4 values
    uint32_t top = 0;
    const bool in = row < rows;
    const uint16_t* src = q_row(a, sq, b, h, in ? row : 0);
#pragma unroll
    for (int p = 0; p < D / 4 / NB; ++p) {
      const uint32_t* s = reinterpret_cast<const uint32_t*>(src + p * 64 + c * NB);
#pragma unroll
      for (int i = 0; i < NB / 2; ++i) {
        w[p * NB / 2 + i] = in ? __ldg(s + i) : 0u;
        const float2 v = float2_of_x2<BF16>(w[p * NB / 2 + i]);
        top = max(top, max(__float_as_uint(v.x) & 0x7fffffffu, __float_as_uint(v.y) & 0x7fffffffu));
      }
    }
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int e = row_exponent(top);
    const float f = top < 0x7f800000u ? pow2f(14 - e) : __uint_as_float(0x7fc00000u);  // NaN, infinity: a NaN row
    if (c == 0) q_scale[warp][8 * t + g] = a.qk_scale * pow2f(max(-126, e - 14));
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      const float2 lo = float2_of_x2<BF16>(w[2 * s]), hi = float2_of_x2<BF16>(w[2 * s + 1]);
      qb[t][s][0] = x2_of_floats<false>(lo.x * f, lo.y * f);
      qb[t][s][1] = x2_of_floats<false>(hi.x * f, hi.y * f);
    }
  }
  __syncwarp();
  // From here on this lane's rows are 8 t + 2c + i.
  float row_sc[NT][2], m[NT][2], l[NT][2];
  int lim[NT][2];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = 8 * t + 2 * c + i;
      row_sc[t][i] = q_scale[warp][r];
      lim[t][i] = r < rows ? last_key(a, sq, query_of(a, r)) : -1;
      m[t][i] = -INFINITY;
      l[t][i] = 0.0f;
    }
  }
  const int lim_first = last_key(a, sq, query_of(a, 0));  // the smallest of the block's rows

  float o[NT][D / 16][4];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) o[t][j][i] = 0.0f;
    }
  }
  int eb = EB_MIN;  // exponent field of the largest finite sv so far ...
  uint32_t low = 0xffffffffu;  // ... and the smallest but zero that this lane has met, its bits - 1
  int er[NT][2];  // the rows' exponents, of their own once those are too far apart
  constexpr int HALVES = DEC_KEYS / 16;

  // A group of keys. `wide`: rows have exponents of their own. False (and nothing is done) where they should.
  auto group = [&](auto is_wide, int it) -> bool {
    constexpr bool wide = decltype(is_wide)::value;
    cp_async_wait<DEC_STAGES - 1>();
    __syncwarp();
    const uint32_t st = ring + (it % DEC_STAGES) * C::STAGE;
    const int pos0 = group_pos(it);

    // Scores: s[t][z][0..3] = (key 16 z + g, rows 8 t + 2c, + 1), (key 16 z + g + 8, the same rows).
    float s[NT][HALVES][4];
#pragma unroll
    for (int z = 0; z < HALVES; ++z) {
      const int r = 16 * z + g;
      constexpr int NB = D >= 64 ? 16 : D / 4;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) s[t][z][i] = 0.0f;
      }
#pragma unroll
      for (int p = 0; p < D / 4 / NB; ++p) {
        uint32_t w0[4], w1[4];
        const int byte = p * 64 + c * NB;
        lds<NB>(st + r * D + (((byte >> 4) ^ C::swz_k(r)) << 4) + (byte & 15), w0);
        lds<NB>(st + (r + 8) * D + (((byte >> 4) ^ C::swz_k(r + 8)) << 4) + (byte & 15), w1);
#pragma unroll
        for (int i = 0; i < NB / 4; ++i) {
          const uint32_t a0 = f16_lo(w0[i]), a1 = f16_lo(w1[i]), a2 = f16_hi(w0[i]), a3 = f16_hi(w1[i]);
#pragma unroll
          for (int t = 0; t < NT; ++t) mma_f16(s[t][z], a0, a1, a2, a3, qb[t][p * 4 + i][0], qb[t][p * 4 + i][1]);
        }
      }
    }
    // Scales of this lane's keys: 16 z + 8 y + g.
    float sk[HALVES][2], sv[HALVES][2];
    uint32_t top = 0;
#pragma unroll
    for (int z = 0; z < HALVES; ++z) {
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        uint32_t w;
        lds<4>(st + 2 * C::CODES + (16 * z + 8 * y + g) * 4, &w);
        sk[z][y] = __uint_as_float(w);
        lds<4>(st + 2 * C::CODES + (DEC_KEYS + 16 * z + 8 * y + g) * 4, &w);
        sv[z][y] = __uint_as_float(w);
        top = max(top, w & 0x7fffffffu);
        low = min(low, (w & 0x7fffffffu) - 1u);
      }
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (top >= 0x7f800000u) {
      // A value row that is not finite makes its key's score NaN instead (0 * NaN in the second
      // product would reach the rows that do not see the key).
      top = 0;
#pragma unroll
      for (int z = 0; z < HALVES; ++z) {
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          if (!(fabsf(sv[z][y]) < INFINITY)) {
            sk[z][y] = __uint_as_float(0x7fc00000u);
            sv[z][y] = 0.0f;
          }
          top = max(top, __float_as_uint(sv[z][y]) & 0x7fffffffu);
        }
      }
      top = __reduce_max_sync(0xffffffffu, top);
    }
    const bool masked = pos0 + DEC_KEYS - 1 > lim_first;
    const int eb_new = max(eb, static_cast<int>(top >> 23));  // the same in every lane
    bool bump = !wide && (eb_new > eb || too_wide(eb_new, low));
    float cand[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int z = 0; z < HALVES; ++z) {
#pragma unroll
        for (int i = 0; i < 4; ++i) s[t][z][i] *= sk[z][i >> 1];
      }
      if (masked) {
#pragma unroll
        for (int z = 0; z < HALVES; ++z) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (pos0 + 16 * z + 8 * (i >> 1) + g > lim[t][i & 1]) s[t][z][i] = -INFINITY;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float v = fmaxf(s[t][0][i], s[t][0][i + 2]);
#pragma unroll
        for (int z = 1; z < HALVES; ++z) v = fa2::fmax3(v, s[t][z][i], s[t][z][i + 2]);
        cand[t][i] = keys_max(v) * row_sc[t][i];
        if constexpr (!wide) bump = bump || cand[t][i] > m[t][i] + RESCALE_TH;
      }
    }
    uint32_t pb[NT][HALVES][2];
    if constexpr (!wide) {
      if (__any_sync(0xffffffffu, bump)) {
        if (__any_sync(0xffffffffu, too_wide(eb_new, low))) return false;
        const float fe = eb_new - eb > 126 ? 0.0f : pow2f(eb - eb_new);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          float al[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            al[i] = 1.0f;
            if (cand[t][i] > m[t][i] + RESCALE_TH) {
              al[i] = fa2::ex2_mufu(m[t][i] - cand[t][i]);  // 0 the first time (m = -inf)
              m[t][i] = cand[t][i];
            }
            l[t][i] *= al[i];
            al[i] *= fe;
          }
#pragma unroll
          for (int j = 0; j < D / 16; ++j) {
#pragma unroll
            for (int i = 0; i < 4; ++i) o[t][j][i] *= al[i & 1];
          }
        }
        eb = eb_new;
      }
      const float gs = __uint_as_float(static_cast<uint32_t>(254 + P_SHIFT - eb) << 23);
#pragma unroll
      for (int z = 0; z < HALVES; ++z) {
        sv[z][0] *= gs;
        sv[z][1] *= gs;
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float m0 = m[t][0] == -INFINITY ? 0.0f : m[t][0], m1 = m[t][1] == -INFINITY ? 0.0f : m[t][1];
#pragma unroll
        for (int z = 0; z < HALVES; ++z) {
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const float p0 = fa2::ex2_mufu(fmaf(s[t][z][2 * y], row_sc[t][0], -m0));
            const float p1 = fa2::ex2_mufu(fmaf(s[t][z][2 * y + 1], row_sc[t][1], -m1));
            l[t][0] += p0;
            l[t][1] += p1;
            pb[t][z][y] = transpose8x8(x2_of_floats<false>(p0 * sv[z][y], p1 * sv[z][y]));
          }
        }
      }
    } else {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float gs[2], f[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float al = 1.0f, most = 0.0f;
          if (cand[t][i] > m[t][i] + RESCALE_TH) {
            al = fa2::ex2_mufu(m[t][i] - cand[t][i]);
            m[t][i] = cand[t][i];
          }
          l[t][i] *= al;
          const float mi = m[t][i] == -INFINITY ? 0.0f : m[t][i];
#pragma unroll
          for (int z = 0; z < HALVES; ++z) {
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const float p = fa2::ex2_mufu(fmaf(s[t][z][2 * y + i], row_sc[t][i], -mi));
              l[t][i] += p;
              s[t][z][2 * y + i] = p * sv[z][y];
              most = fmaxf(most, fabsf(s[t][z][2 * y + i]));
            }
          }
          er[t][i] = row_unit(static_cast<int>(__float_as_uint(keys_max(most)) >> 23), er[t][i], al, f[i]);
          gs[i] = __uint_as_float(static_cast<uint32_t>(254 + P_SHIFT - er[t][i]) << 23);
        }
#pragma unroll
        for (int z = 0; z < HALVES; ++z) {
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            pb[t][z][y] = transpose8x8(x2_of_floats<false>(s[t][z][2 * y] * gs[0], s[t][z][2 * y + 1] * gs[1]));
          }
        }
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
#pragma unroll
          for (int i = 0; i < 4; ++i) o[t][j][i] *= f[i & 1];
        }
      }
    }
    // O^T += V^T P'^T, 16 keys at a time.
#pragma unroll
    for (int z = 0; z < HALVES; ++z) {
      uint32_t v0[4], v1[4], v2[4], v3[4];
      constexpr int NB = D / 8;
      const int byte = g * NB;
      const uint32_t vst = st + C::CODES;
      auto at = [&](int r) { return vst + r * D + (((byte >> 4) ^ C::swz_v(r)) << 4) + (byte & 15); };
      lds<NB>(at(16 * z + 2 * c), v0);
      lds<NB>(at(16 * z + 2 * c + 1), v1);
      lds<NB>(at(16 * z + 2 * c + 8), v2);
      lds<NB>(at(16 * z + 2 * c + 9), v3);
#pragma unroll
      for (int w = 0; w < (D + 31) / 32; ++w) {
        const uint32_t e0 = __byte_perm(v0[w], v1[w], 0x5140), e1 = __byte_perm(v2[w], v3[w], 0x5140);
        const uint32_t a0 = f16_lo(e0), a1 = f16_hi(e0), a2 = f16_lo(e1), a3 = f16_hi(e1);
#pragma unroll
        for (int t = 0; t < NT; ++t) mma_f16(o[t][2 * w], a0, a1, a2, a3, pb[t][z][0], pb[t][z][1]);
        if constexpr (D >= 32) {
          const uint32_t f0 = __byte_perm(v0[w], v1[w], 0x7362), f1 = __byte_perm(v2[w], v3[w], 0x7362);
          const uint32_t c0 = f16_lo(f0), c1 = f16_hi(f0), c2 = f16_lo(f1), c3 = f16_hi(f1);
#pragma unroll
          for (int t = 0; t < NT; ++t) mma_f16(o[t][2 * w + 1], c0, c1, c2, c3, pb[t][z][0], pb[t][z][1]);
        }
      }
    }
    __syncwarp();  // every lane has read the stage before it is filled again
    issue(it + DEC_STAGES);
    return true;
  };
  int it = 0;
  while (it < mine && group(std::false_type{}, it)) ++it;
#pragma unroll
  for (int t = 0; t < NT; ++t) er[t][0] = er[t][1] = eb;
  for (; it < mine; ++it) group(std::true_type{}, it);
  cp_async_wait<0>();
  __syncwarp();

  // Merge the warps: (m, l, O / 2^above(l)) of each in shared memory. Rows of O are D + 4 floats apart: the four rows
  // that the lanes of one g write lie in different banks.
  float* wo = reinterpret_cast<float*>(smem + warp * C::RING);
  float* wm = reinterpret_cast<float*>(smem + DEC_WARPS * C::RING);  // [warp][16]
  float* wl = wm + DEC_WARPS * 16;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float sum = keys_sum(l[t][i]);
      const int r = 8 * t + 2 * c + i;
      if (g == 0) {
        wm[warp * 16 + r] = m[t][i];
        wl[warp * 16 + r] = sum;
      }
      // Out of the unit 2^(e - 127 - P_SHIFT), as two factors so that neither leaves the normal range, and over
      // the power of two above the sum: an average of the values stays in range where a sum may not.
      const int ex = er[t][i] - 127 - P_SHIFT - above(sum);
      const float u0 = pow2f(ex / 2), u1 = pow2f(ex - ex / 2);
      float* dst = wo + r * (D + 4) + g * (D / 8);
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        *reinterpret_cast<float2*>(dst + 2 * j) = make_float2(o[t][j][i] * u0 * u1, o[t][j][2 + i] * u0 * u1);
      }
    }
  }
  __syncthreads();
  constexpr int PARTS = DEC_WARPS * 32 / ROWS;  // threads of a row
  const int r = static_cast<int>(threadIdx.x) / PARTS, part = static_cast<int>(threadIdx.x) % PARTS;
  if (r >= rows) return;  // (no barrier follows in here)
  float mx = -INFINITY;
#pragma unroll
  for (int w = 0; w < DEC_WARPS; ++w) mx = fmaxf(mx, wm[w * 16 + r]);
  float sum = 0.0f, f[DEC_WARPS];
#pragma unroll
  for (int w = 0; w < DEC_WARPS; ++w) {
    const float mw = wm[w * 16 + r], lw = wl[w * 16 + r];
    // A warp that saw no key of the row has m = -inf and l = 0; a NaN sum is kept.
    f[w] = mw == -INFINITY ? (lw == 0.0f ? 0.0f : 1.0f) : exp2f(mw - mx);
    sum = f[w] == 0.0f ? sum : fmaf(f[w], lw, sum);
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
  for (int w = 0; w < DEC_WARPS; ++w) f[w] = f[w] == 0.0f ? 0.0f : f[w] * pow2f(above(wl[w * 16 + r])) * inv;
  const int64_t part_row = static_cast<int64_t>(slot) * ROWS + r;
  constexpr int PER = D / PARTS > 0 ? (D / PARTS < 8 ? D / PARTS : 8) : 1;  // neighbouring columns at a time
  for (int d = part * PER; d < D; d += PARTS * PER) {
    float acc[PER] = {};
#pragma unroll
    for (int w = 0; w < DEC_WARPS; ++w) {
      if (f[w] == 0.0f) continue;
      const float* src = reinterpret_cast<const float*>(smem + w * C::RING) + r * (D + 4) + d;
#pragma unroll
      for (int j = 0; j < PER; ++j) acc[j] = fmaf(f[w], src[j], acc[j]);
    }
    if (slot >= 0) {
#pragma unroll
      for (int j = 0; j < PER; ++j) a.o_part[part_row * D + d + j] = acc[j];
    } else {
      uint16_t* dst = o_row(a, sq, b, h, r) + d;
      if constexpr (PER >= 2) {
#pragma unroll
        for (int j = 0; j < PER; j += 2) {
          *reinterpret_cast<uint32_t*>(dst + j) = x2_of_floats<BF16>(acc[j], acc[j + 1]);
        }
      } else {
        dst[0] = x1_of_float<BF16>(acc[0]);
      }
    }
  }
  if (slot >= 0 && part == 0) a.lse_part[part_row] = sum == 0.0f ? -INFINITY : (mx == -INFINITY ? 0.0f : mx) + log2f(sum);
}

template <int D, bool BF16, int NT>
__global__ void __launch_bounds__(DEC_WARPS * 32, DEC_CTAS) decode_kernel(const AttnArgs a) {
  extern __shared__ __align__(128) uint8_t smem[];  // (rows of codes start on their banks)
  allow_next();
  __shared__ Piece piece;
  __shared__ int more;
  Pieces pieces;
  if (threadIdx.x < 32) pieces.begin(a, static_cast<int>(blockIdx.x));
  while (true) {
    if (threadIdx.x < 32) {  // warp 0 walks the share
      Piece o{};
      const bool m = pieces.next(a, o);
      if (threadIdx.x == 0) {
        piece = o;
        more = m;
      }
    }
    __syncthreads();
    if (!more) break;
    // (Broadcasts: what follows from these is then kept in uniform registers.)
    Piece o;
    o.sq.n_q = __shfl_sync(0xffffffffu, piece.sq.n_q, 0);
    o.sq.q0 = __shfl_sync(0xffffffffu, piece.sq.q0, 0);
    o.sq.len = __shfl_sync(0xffffffffu, piece.sq.len, 0);
    o.sq.off = __shfl_sync(0xffffffffu, piece.sq.off, 0);
    o.b = __shfl_sync(0xffffffffu, piece.b, 0);
    o.h = __shfl_sync(0xffffffffu, piece.h, 0);
    o.t0 = __shfl_sync(0xffffffffu, piece.t0, 0);
    o.tiles = __shfl_sync(0xffffffffu, piece.tiles, 0);
    o.kend = __shfl_sync(0xffffffffu, piece.kend, 0);
    o.slot = __shfl_sync(0xffffffffu, piece.slot, 0);
    decode_part<D, BF16, NT>(a, smem, o.sq, o.b, o.h, o.t0 * 128, min(o.kend, (o.t0 + o.tiles) * 128), o.slot);
    __syncthreads();  // the shared memory is free again
  }
}

// ------------------------------------------------------------------ merge of the partial results
// o = sum_s 2^(lse_s - max) o_s / sum_s 2^(lse_s - max) over a cut block's parts, in the line's order, a
// warp a row (four rows side by side in the 256-row kernel): CTA (x, y) has 4 R rows of the block that
// share x + 1 is the first to cut. Loads wait for no other part's: with a branch around each the
// merge of 32 parts alone took 14 us.
// The last ZERO_CTAS write zeros for the blocks without a tile, which no worker has.
constexpr int ZERO_CTAS = 16;
constexpr int merge_rows(int block) { return block < 256 ? 4 : 16; }

template <int N>
__device__ __forceinline__ void load_floats(const float* p, float (&v)[N]) {
  if constexpr (N == 4) {
    const float4 x = *reinterpret_cast<const float4*>(p);
    v[0] = x.x;
    v[1] = x.y;
    v[2] = x.z;
    v[3] = x.w;
  } else if constexpr (N == 2) {
    const float2 x = *reinterpret_cast<const float2*>(p);
    v[0] = x.x;
    v[1] = x.y;
  } else {
    v[0] = *p;
  }
}

template <int D, bool BF16, int R>
__global__ void __launch_bounds__(128) merge_kernel(const AttnArgs a) {
  constexpr int MERGE_ROWS = 4 * R;  // a warp's: row_first + warp + 4 k
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row_first = static_cast<int>(blockIdx.y) * MERGE_ROWS;
  const int w = static_cast<int>(blockIdx.x) + 1;
  wait_for_previous();  // every thread: what follows this kernel must not overtake the one before it
  if (w >= a.workers) {
    for (int b = w - a.workers; b < a.batch; b += ZERO_CTAS) {
      const Seq sq = sequence(a, b);
      const int rows = sq.n_q * a.group;
      for (int rb = 0; rb * a.block < rows; ++rb) {
        if (Line::tiles(a, sq, rb) > 0) continue;
        const int row0 = rb * a.block + row_first, n = min(min(MERGE_ROWS, a.block - row_first), rows - row0);
        for (int i = threadIdx.x; i < n * a.heads_kv; i += 128) {
          uint4* dst = reinterpret_cast<uint4*>(o_row(a, sq, b, i / n, row0 + i % n));
#pragma unroll 1
          for (int j = 0; j < D / 8; ++j) dst[j] = make_uint4(0, 0, 0, 0);
        }
      }
    }
    return;
  }
  const Cut cut = a.cuts[w];
  Seq sq{};
  sq.q0 = cut.q0;
  const int rows = min(a.block, cut.n_q * a.group - cut.row0);
  constexpr int PER = D >= 32 ? D / 32 : 1;
  const bool on = lane * PER < D;
  auto part = [&](int i, int r) -> int64_t {  // its row
    return static_cast<int64_t>(i == 0 ? cut.first_slot : 2 * (w - 1 + i)) * a.block + r;
  };
  if (cut.n_parts == 0 || row_first >= rows) return;
  const int r0 = row_first + warp;
  float mx[R], sum[R] = {}, acc[R][PER] = {};
#pragma unroll
  for (int k = 0; k < R; ++k) mx[k] = -INFINITY;
  for (int i = lane; i < cut.n_parts; i += 32) {
#pragma unroll
    for (int k = 0; k < R; ++k) {
      if (r0 + 4 * k < rows) mx[k] = fmaxf(mx[k], a.lse_part[part(i, r0 + 4 * k)]);
    }
  }
#pragma unroll
  for (int k = 0; k < R; ++k) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx[k] = fmaxf(mx[k], __shfl_xor_sync(0xffffffffu, mx[k], o));
  }
  // 2^-j <= 1 / n_parts on every weight: the sum of the parts stays in range as its average does.
  const float down = pow2f(-(32 - __clz(cut.n_parts - 1)));
  for (int i0 = 0; i0 < cut.n_parts; i0 += 32) {
    float f[R];
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const float v = i0 + lane < cut.n_parts && r0 + 4 * k < rows ? a.lse_part[part(i0 + lane, r0 + 4 * k)] : -INFINITY;
      f[k] = v == -INFINITY ? 0.0f : exp2f(v - (mx[k] == -INFINITY ? 0.0f : mx[k])) * down;  // a NaN stays one
    }
    const int n = min(32, cut.n_parts - i0);
    constexpr int AT_ONCE = R == 1 ? 8 : 2;
    for (int i = 0; i < n; i += AT_ONCE) {
      float v[AT_ONCE][R][PER];
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
#pragma unroll
        for (int k = 0; k < R; ++k) {
          const int64_t at = part(i0 + min(i + u, n - 1), min(r0 + 4 * k, rows - 1)) * D + (on ? lane * PER : 0);
          load_floats<PER>(a.o_part + at, v[u][k]);
        }
      }
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
#pragma unroll
        for (int k = 0; k < R; ++k) {
          const float fi = __shfl_sync(0xffffffffu, f[k], i + u);  // 0 from part n on
          sum[k] += fi;
#pragma unroll
          for (int j = 0; j < PER; ++j) {  // a part without a key has weight 0, and may hold anything
            acc[k][j] = fi != 0.0f ? fmaf(fi, v[u][k][j], acc[k][j]) : acc[k][j];
          }
        }
      }
    }
  }
#pragma unroll
  for (int k = 0; k < R; ++k) {
    if (!on || r0 + 4 * k >= rows) continue;
    const float inv = sum[k] == 0.0f ? 0.0f : 1.0f / sum[k];
    uint16_t* dst = o_row(a, sq, cut.b, cut.h, cut.row0 + r0 + 4 * k) + lane * PER;
#pragma unroll
    for (int j = 0; j < PER; ++j) dst[j] = x1_of_float<BF16>(acc[k][j] * inv);
  }
}

// ------------------------------------------------------------------------------------ host
struct Plan {
  int block = 8;  // rows of a block: 8 or 16 (decode_kernel), 256 (chunk_kernel)
  int workers = 1;
  int64_t cut_bytes = 0, lse_floats = 0, bytes = 0;
};

constexpr int MAX_SPLITS = 256;

// The kernel, the workers and the workspace of a call, from its sizes alone.
Plan plan(const Fa2Kv8AttnParams* p) {
  Plan r;
  const int64_t rows = static_cast<int64_t>(p->seqlen_q) * (p->heads_q / p->cache.heads_kv);
  r.block = rows <= 8 ? 8 : rows <= 16 ? 16 : 256;
  const int64_t units = static_cast<int64_t>(p->batch) * p->cache.heads_kv * std::max<int64_t>(1, (rows + r.block - 1) / r.block);
  // One wave: dec_shares() CTAs, or one of the 256-row kernel, on each of 148 SMs.
  const int64_t most = r.block == 256 ? 148 : 148 * dec_shares(p->cache.head_dim);
  const int64_t per_unit = (static_cast<int64_t>(p->max_seqlen_k) + 127) / 128, tiles = units * per_unit;
  int64_t w = most;
  if (p->num_splits > 0) {
    w = units * p->num_splits;
  } else if (units <= most) {
    // With fewer (sequence, head, block)s than that a multiple of their number cuts equal ones alike.
    const int64_t alike = most / units * units;
    if (r.block < 256) {
      // Three tiles a share at least: more shares cost their finding and merging, fewer their keys. Us for 8
      // heads of one sequence with one, two, three and more tiles a share: 700 keys 10.3, 11.0, 11.7, 12.3 (6
      // tiles); 2000 keys 12.3, 11.6, 12.3, 12.3 (4), 14.4 (6); 8192 keys 17 (2), 16.4 (3), 14.6 (4), 15.8 (6),
      // 16.4 (8), 19 (11). Short sequences would take one or two, long ones four.
      const int64_t least = std::max<int64_t>(3, (per_unit + most / units - 1) / (most / units));
      w = std::max<int64_t>(1, (per_unit + least - 1) / least) * units;
    } else {
      // Shares that hold one whole block each need no merge (15 us), and those of one block alone start
      // and end one piece less (10 us): taken where a CTA has at most as much more to do.
      const int64_t more = (tiles + alike - 1) / alike - tiles / most;
      if (more <= (alike == units ? 6 : 3)) w = alike;
    }
  }
  if (w > 148 * 16) w = 148 * 16;
  if (w > tiles) w = tiles;
  r.workers = static_cast<int>(w < 1 ? 1 : w);
  // A Cut and two partial results a worker.
  const int64_t slots = 2ll * r.workers * r.block;
  r.lse_floats = (slots + 3) / 4 * 4;
  r.cut_bytes = static_cast<int64_t>(sizeof(Cut)) * r.workers;
  r.bytes = r.cut_bytes + 4 * (r.lse_floats + slots * p->cache.head_dim);
  return r;
}

int check_core(const Fa2Kv8AttnParams* p) {
  if (p == nullptr || p->q == nullptr || p->o == nullptr || p->block_table == nullptr || p->cache_seqlens == nullptr) {
    return FA2_ERR_NULL;
  }
  const int rc = check_cache(p->cache);
  if (rc != FA2_OK) return rc;
  if (p->batch < 1 || p->heads_q < 1 || p->seqlen_q < 0 || p->max_seqlen_k < 0 || p->pages_per_seq < 1) return FA2_ERR_SHAPE;
  if (p->cu_seqlens_q != nullptr && p->total_q < 0) return FA2_ERR_SHAPE;
  if (p->heads_q % p->cache.heads_kv != 0) return FA2_ERR_GQA;
  if (p->num_splits < 0 || p->num_splits > MAX_SPLITS) return FA2_ERR_SHAPE;
  if (p->causal && p->causal_align != FA2_CAUSAL_TOP_LEFT && p->causal_align != FA2_CAUSAL_BOTTOM_RIGHT) return FA2_ERR_SHAPE;
  if (p->dtype != FA2_DTYPE_FP16 && p->dtype != FA2_DTYPE_BF16) return FA2_ERR_DTYPE;
  if (!(p->qk_scale > 0.0f) || !std::isfinite(p->qk_scale)) return FA2_ERR_SCALE;
  // Rows of q and o are moved 16 bytes at a time.
  if (!aligned16(p->q) || !aligned16(p->o) || p->q_stride[3] != 1 || p->o_stride[3] != 1) return FA2_ERR_LAYOUT;
  const int64_t n[3] = {p->cu_seqlens_q != nullptr ? 1 : p->batch, p->heads_q, p->cu_seqlens_q != nullptr ? p->total_q : p->seqlen_q};
  for (int i = 0; i < 3; ++i) {
    if (n[i] > 1 && ((p->q_stride[i] | p->o_stride[i]) & 7) != 0) return FA2_ERR_LAYOUT;
  }
  // Row numbers and grids stay in 31 bits, the line of tiles (four cost units each, and 16 a block) below
  // LONGEST_LINE.
  const int64_t rows = static_cast<int64_t>(p->seqlen_q) * (p->heads_q / p->cache.heads_kv);
  if (rows > (1ll << 30) || static_cast<int64_t>(p->batch) * p->cache.heads_kv > (1ll << 26)) return FA2_ERR_SHAPE;
  int64_t blocks = static_cast<int64_t>(p->batch) * ((rows + 255) / 256);
  if (p->cu_seqlens_q != nullptr) {
    blocks = std::min(blocks, static_cast<int64_t>(p->total_q) * (p->heads_q / p->cache.heads_kv) / 256 + p->batch);
  }
  const int64_t units = blocks * p->cache.heads_kv, tiles = (static_cast<int64_t>(p->max_seqlen_k) + 127) / 128;
  if (units > (1ll << 24) || units * tiles > (1ll << 27)) return FA2_ERR_SHAPE;
  return FA2_OK;
}

// Raises a kernel's shared memory limit, once for each device. `done` is the kernel's own.
template <typename K>
bool allow_smem(K kernel, int bytes, int dev, std::atomic<bool> (&done)[MAX_DEVICES]) {
  if (done[dev].load(std::memory_order_acquire)) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
  done[dev].store(true, std::memory_order_release);
  return true;
}

// Launches the merge behind the kernel that was just launched. It may start early: it works out where
// the parts lie, then waits for them.
template <int D, bool BF16>
int launch_merge(const AttnArgs& a, cudaStream_t s) {
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(a.workers - 1 + ZERO_CTAS), a.block / merge_rows(a.block));
  cfg.blockDim = dim3(128);
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = a.block < 256 ? cudaLaunchKernelEx(&cfg, merge_kernel<D, BF16, merge_rows(8) / 4>, a)
                                      : cudaLaunchKernelEx(&cfg, merge_kernel<D, BF16, merge_rows(256) / 4>, a);
  return e == cudaSuccess ? FA2_OK : FA2_ERR_LAUNCH;
}

template <int D, bool BF16>
int launch(const AttnArgs& a, cudaStream_t s, int dev) {
  static std::atomic<bool> done[3][MAX_DEVICES];
  const unsigned ctas = static_cast<unsigned>(a.workers);
  if (a.block == 256) {
    auto kernel = chunk_kernel<D, BF16>;
    if (!allow_smem(kernel, Ch<D, BF16>::SMEM, dev, done[2])) return FA2_ERR_LAUNCH;
    kernel<<<ctas, CH_THREADS, Ch<D, BF16>::SMEM, s>>>(a);
  } else if (a.block == 16) {
    auto kernel = decode_kernel<D, BF16, 2>;
    if (!allow_smem(kernel, Dec<D>::SMEM, dev, done[1])) return FA2_ERR_LAUNCH;
    kernel<<<ctas, DEC_WARPS * 32, Dec<D>::SMEM, s>>>(a);
  } else {
    auto kernel = decode_kernel<D, BF16, 1>;
    if (!allow_smem(kernel, Dec<D>::SMEM, dev, done[0])) return FA2_ERR_LAUNCH;
    kernel<<<ctas, DEC_WARPS * 32, Dec<D>::SMEM, s>>>(a);
  }
  const int rc = launch_status();
  return rc != FA2_OK ? rc : launch_merge<D, BF16>(a, s);
}

}  // namespace

extern "C" {

int fa2_kv8_attn_sm100_check(const Fa2Kv8AttnParams* p) {
  const int rc = check_core(p);
  if (rc != FA2_OK) return rc;
  const Plan r = plan(p);
  if (r.bytes > 0 && (p->workspace == nullptr || !aligned16(p->workspace) || p->workspace_bytes < r.bytes)) {
    return FA2_ERR_WORKSPACE;
  }
  return FA2_OK;
}

int64_t fa2_kv8_attn_sm100_workspace_bytes(const Fa2Kv8AttnParams* p) {
  return check_core(p) == FA2_OK ? plan(p).bytes : -1;
}

int fa2_kv8_attn_sm100(const Fa2Kv8AttnParams* p, void* stream) {
  const int rc = fa2_kv8_attn_sm100_check(p);
  if (rc != FA2_OK) return rc;
  if (p->seqlen_q == 0 || (p->cu_seqlens_q != nullptr && p->total_q == 0)) return FA2_OK;
  const int dev = sm100_device();
  if (dev < 0) return FA2_ERR_DEVICE;
  const Plan r = plan(p);
  AttnArgs a{};
  a.c = device_cache(p->cache);
  a.q = static_cast<const uint16_t*>(p->q);
  a.o = static_cast<uint16_t*>(p->o);
  for (int i = 0; i < 3; ++i) {
    a.q_st[i] = p->q_stride[i];
    a.o_st[i] = p->o_stride[i];
  }
  a.bt = p->block_table;
  a.lens = p->cache_seqlens;
  a.cu_q = p->cu_seqlens_q;
  a.err = p->err_flag;
  a.bt_stride = p->block_table_stride;
  a.timeout = p->timeout_cycles;
  a.pages_per_seq = p->pages_per_seq;
  a.batch = p->batch;
  a.group = p->heads_q / p->cache.heads_kv;
  a.by_group = divisor(a.group);
  a.heads_kv = p->cache.heads_kv;
  a.n_q = p->seqlen_q;
  a.total_q = p->total_q;
  a.max_k = std::min(p->max_seqlen_k, MAX_KEYS);
  a.causal = p->causal;
  a.bottom_right = p->causal && p->causal_align == FA2_CAUSAL_BOTTOM_RIGHT;
  a.workers = r.workers;
  a.block = r.block;
  a.qk_scale = p->qk_scale;
  a.cuts = static_cast<Cut*>(p->workspace);
  a.lse_part = reinterpret_cast<float*>(static_cast<uint8_t*>(p->workspace) + r.cut_bytes);
  a.o_part = a.lse_part + r.lse_floats;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf = p->dtype == FA2_DTYPE_BF16;
  switch (p->cache.head_dim) {
    case 16: return bf ? launch<16, true>(a, s, dev) : launch<16, false>(a, s, dev);
    case 32: return bf ? launch<32, true>(a, s, dev) : launch<32, false>(a, s, dev);
    case 64: return bf ? launch<64, true>(a, s, dev) : launch<64, false>(a, s, dev);
    default: return bf ? launch<128, true>(a, s, dev) : launch<128, false>(a, s, dev);
  }
}

}  // extern "C"
