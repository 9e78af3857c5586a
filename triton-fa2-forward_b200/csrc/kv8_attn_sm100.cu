// Attention of new tokens over the 8-bit paged cache, for sm_100a.

#include "kv8_attn.cuh"
#include "kv8_chunk.cuh"

#include <cmath>

namespace {

using namespace fa2kv;

// ------------------------------------------------------------------ few rows (decode)
// At most 16 rows (queries x heads of a group) a CTA. Bound by the bytes of the cache: 2 (D + 4) a
// key. So the tensor work runs on warp-wide 16 x 8 x 16 products, which take the codes straight
// from registers: every warp streams its own 16-key groups through its own ring of asynchronous
// copies (no barrier between warps), converts them in registers and keeps its own running max, sum
// and output; the four warps are merged once at the end. A 128-row tile would be 1/8 full at most
// and its conversion to shared memory would cost more than the bytes allow.
//
// Operand layouts. The products sum over d (QK^T) and over keys (PV) in any order, so both
// operands use the order in which a lane's bytes lie in memory: in QK^T lane (g, c) = (lane / 4,
// lane % 4) reads D / 4 contiguous bytes of key g's row, four to a 16-wide step; in PV it reads D / 8
// contiguous bytes at column g D / 8 of the keys 2c, 2c + 1, 2c + 8, 2c + 9 and interleaves pairs of
// keys, so its sums hold 2 x D / 8 contiguous output columns.

constexpr int DEC_WARPS = 4;
constexpr int DEC_STAGES = 4;

template <int D>
struct Dec {
  static constexpr int ROW = D;                       // bytes of a row of codes
  static constexpr int STAGE = 2 * 16 * ROW + 128;    // K, V codes of 16 keys, their scales
  static constexpr int RING = DEC_STAGES * STAGE;     // a warp's ring, later its output (64 D bytes)
  static constexpr int SMEM = DEC_WARPS * RING + DEC_WARPS * 2 * 16 * 4;
  static_assert(RING >= 16 * D * 4, "the ring is reused for the warp's output");
  // 16-byte pieces of a row are stored at piece ^ swz(row): spreads the lanes' reads over the banks.
  __device__ static int swz_k(int row) { return D == 128 ? (row & 1) << 2 : 0; }
  __device__ static int swz_v(int row) { return D == 128 ? row & 6 : D == 64 ? (row >> 1) & 3 : 0; }
};

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

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

__device__ __forceinline__ float quad_max(float x) {
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
  return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
}
__device__ __forceinline__ float quad_sum(float x) {
  x += __shfl_xor_sync(0xffffffffu, x, 1);
  return x + __shfl_xor_sync(0xffffffffu, x, 2);
}

template <int D, bool BF16>
__global__ void __launch_bounds__(DEC_WARPS * 32) decode_kernel(const AttnArgs a) {
  using C = Dec<D>;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  // Row blocks of one key range run next to one another: they share its bytes in L2.
  int x = static_cast<int>(blockIdx.x);
  const int rb = x % a.row_blocks;
  x /= a.row_blocks;
  const int split = x % a.splits;
  x /= a.splits;
  const int h = x % a.heads_kv, b = x / a.heads_kv;
  const Seq sq = sequence(a, b);
  const int rows = sq.n_q * a.group, row0 = rb * 16;
  if (row0 >= rows) return;
  const int kend = keys_end(a, sq, row0, min(16, rows - row0));
  const int k0 = split * a.split_keys;
  const int k1 = min(kend, k0 + a.split_keys);
  if (k1 <= k0 && a.splits > 1) return;  // the merge kernel does not read this split

  const uint32_t ring = fa2::smem_u32(smem) + warp * C::RING;
  const int n_groups = k1 > k0 ? (k1 - k0 + 15) / 16 : 0;
  const int mine = n_groups > warp ? (n_groups - warp + DEC_WARPS - 1) / DEC_WARPS : 0;
  const int* bt = a.bt + b * a.bt_stride;
  const uint8_t* kh = a.c.k + h * a.c.k_st[2];
  const uint8_t* vh = a.c.v + h * a.c.v_st[2];
  const float* ksh = a.c.ks + h * a.c.ks_st[2];
  const float* vsh = a.c.vs + h * a.c.vs_st[2];
  auto group_pos = [&](int it) { return k0 + 16 * (warp + DEC_WARPS * it); };
  // A 16-key group lies in one page. Its table entry is fetched one group ahead.
  int next_page = mine > 0 ? __ldg(bt + page_of(a.c, group_pos(0))) : 0;
  auto issue = [&](int it) {
    if (it < mine) {
      const int pos0 = group_pos(it);
      const int64_t page = next_page;
      if (it + 1 < mine) next_page = __ldg(bt + page_of(a.c, group_pos(it + 1)));
      const int r0 = pos0 - page_of(a.c, pos0) * a.c.page_size;
      const uint32_t st = ring + (it % DEC_STAGES) * C::STAGE;
      const bool ok = page >= 0 && page < a.c.num_pages;
      if (!ok) report(a.err, FA2_ERR_PAGE);
      const int64_t pg = ok ? page : 0;
      constexpr int PIECES = D / 16;  // of a row
#pragma unroll
      for (int i = 0; i < (16 * PIECES + 31) / 32; ++i) {
        const int e = i * 32 + lane;
        const int r = e / PIECES, piece = e % PIECES;
        if (16 * PIECES % 32 == 0 || e < 16 * PIECES) {
          const bool in = ok && pos0 + r < sq.len;  // rows past the end hold anything: zeros instead
          cp_async16(st + r * C::ROW + ((piece ^ C::swz_k(r)) << 4),
                     kh + pg * a.c.k_st[0] + (in ? r0 + r : 0) * a.c.k_st[1] + piece * 16, in);
          cp_async16(st + 16 * C::ROW + r * C::ROW + ((piece ^ C::swz_v(r)) << 4),
                     vh + pg * a.c.v_st[0] + (in ? r0 + r : 0) * a.c.v_st[1] + piece * 16, in);
        }
      }
      const int r = lane & 15;
      const bool in = ok && pos0 + r < sq.len;
      const float* src = lane < 16 ? ksh + pg * a.c.ks_st[0] + (in ? r0 + r : 0) * a.c.ks_st[1]
                                   : vsh + pg * a.c.vs_st[0] + (in ? r0 + r : 0) * a.c.vs_st[1];
      const uint32_t dst = st + 32 * C::ROW + lane * 4;
      if (ok) {
        cp_async4(dst, src, in);
      } else {  // a refused page: queries that see its keys get NaN
        asm volatile("st.shared.b32 [%0], %1;" ::"r"(dst), "r"(0x7fc00000u) : "memory");
      }
    }
    cp_async_commit();  // also where there is nothing: the group count stays in step
  };
  for (int it = 0; it < DEC_STAGES - 1; ++it) issue(it);

  // Q, scaled by a power of two, in the order described above: this lane's rows are g and g + 8.
  uint32_t qa[D / 16][4];
  float row_sc[2];
  int lim[2];
#pragma unroll
  for (int rr = 0; rr < 2; ++rr) {
    const int row = row0 + g + 8 * rr;
    constexpr int NB = D >= 64 ? 16 : D / 4;  // values of a contiguous piece
    uint32_t w[D / 8];                        // D / 4 values
    uint32_t top = 0;
    const bool in = row < rows;
    const uint16_t* src = q_row(a, sq, b, h, in ? row : row0);
#pragma unroll
    for (int p = 0; p < D / 4 / NB; ++p) {
      const uint16_t* s = src + p * 64 + c * NB;
#pragma unroll
      for (int i = 0; i < NB / 2; ++i) {
        w[p * NB / 2 + i] = in ? *reinterpret_cast<const uint32_t*>(s + 2 * i) : 0;
        const float2 v = float2_of_x2<BF16>(w[p * NB / 2 + i]);
        top = max(top, max(__float_as_uint(v.x) & 0x7fffffffu, __float_as_uint(v.y) & 0x7fffffffu));
      }
    }
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int e = row_exponent(top);
    const float f = pow2f(14 - e);
    row_sc[rr] = a.qk_scale * pow2f(max(-126, e - 14));
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      const float2 lo = float2_of_x2<BF16>(w[2 * s]), hi = float2_of_x2<BF16>(w[2 * s + 1]);
      qa[s][rr] = x2_of_floats<false>(lo.x * f, lo.y * f);
      qa[s][2 + rr] = x2_of_floats<false>(hi.x * f, hi.y * f);
    }
    lim[rr] = in ? last_key(a, sq, row / a.group) : -1;
  }
  const int lim_first = last_key(a, sq, row0 / a.group);  // the smallest of the block's rows

  float o[D / 8][4];
#pragma unroll
  for (int j = 0; j < D / 8; ++j) {
#pragma unroll
    for (int i = 0; i < 4; ++i) o[j][i] = 0.0f;
  }
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
  int eb = EB_MIN;  // exponent field of the largest finite sv so far

  for (int it = 0; it < mine; ++it) {
    issue(it + DEC_STAGES - 1);
    cp_async_wait<DEC_STAGES - 1>();
    __syncwarp();
    const uint32_t st = ring + (it % DEC_STAGES) * C::STAGE;
    const int pos0 = group_pos(it);

    float s[2][4] = {};
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int r = t * 8 + g;
      constexpr int NB = D >= 64 ? 16 : D / 4;
#pragma unroll
      for (int p = 0; p < D / 4 / NB; ++p) {
        uint32_t w[4];
        const int byte = p * 64 + c * NB;
        lds<NB>(st + r * C::ROW + (((byte >> 4) ^ C::swz_k(r)) << 4) + (byte & 15), w);
#pragma unroll
        for (int i = 0; i < NB / 4; ++i) {
          mma16816(s[t], qa[p * 4 + i], f16x2_of_e4m3x2(static_cast<uint16_t>(w[i])),
                   f16x2_of_e4m3x2(static_cast<uint16_t>(w[i] >> 16)));
        }
      }
    }
    // Scales of this lane's keys: 2c, 2c + 1 (tile 0) and 8 + 2c, 8 + 2c + 1 (tile 1).
    float sk[2][2], sv[2][2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      uint32_t w[2];
      lds<8>(st + 32 * C::ROW + (t * 8 + 2 * c) * 4, w);
      sk[t][0] = __uint_as_float(w[0]);
      sk[t][1] = __uint_as_float(w[1]);
      lds<8>(st + 32 * C::ROW + 64 + (t * 8 + 2 * c) * 4, w);
      sv[t][0] = __uint_as_float(w[0]);
      sv[t][1] = __uint_as_float(w[1]);
    }
    uint32_t sv_top = 0;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t v = __float_as_uint(sv[t][i]) & 0x7fffffffu;
        sv_top = max(sv_top, v < 0x7f800000u ? v : 0u);
      }
    }
    sv_top = max(sv_top, __shfl_xor_sync(0xffffffffu, sv_top, 1));
    sv_top = max(sv_top, __shfl_xor_sync(0xffffffffu, sv_top, 2));

    const bool masked = pos0 + 15 > lim_first || row0 + 16 > rows;
    float cand[2];
#pragma unroll
    for (int rr = 0; rr < 2; ++rr) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float v = s[t][2 * rr + i] * sk[t][i];
          if (masked && pos0 + t * 8 + 2 * c + i > lim[rr]) v = -INFINITY;
          s[t][2 * rr + i] = v;
        }
      }
      cand[rr] = quad_max(fmaxf(fmaxf(s[0][2 * rr], s[0][2 * rr + 1]), fmaxf(s[1][2 * rr], s[1][2 * rr + 1]))) * row_sc[rr];
    }
    const int eb_new = max(eb, static_cast<int>(sv_top >> 23));  // the same in every lane
    const bool bump = cand[0] > m[0] + RESCALE_TH || cand[1] > m[1] + RESCALE_TH || eb_new > eb;
    if (__any_sync(0xffffffffu, bump)) {
      const float fe = eb_new - eb > 126 ? 0.0f : pow2f(eb - eb_new);
      float al[2];
#pragma unroll
      for (int rr = 0; rr < 2; ++rr) {
        al[rr] = 1.0f;
        if (cand[rr] > m[rr] + RESCALE_TH) {
          al[rr] = fa2::ex2_mufu(m[rr] - cand[rr]);  // 0 the first time (m = -inf)
          m[rr] = cand[rr];
        }
        l[rr] *= al[rr];
        al[rr] *= fe;
      }
#pragma unroll
      for (int j = 0; j < D / 8; ++j) {
        o[j][0] *= al[0];
        o[j][1] *= al[0];
        o[j][2] *= al[1];
        o[j][3] *= al[1];
      }
      eb = eb_new;
    }
    const float gs = __uint_as_float(static_cast<uint32_t>(254 + P_SHIFT - eb) << 23);
    uint32_t pa[4];
#pragma unroll
    for (int rr = 0; rr < 2; ++rr) {
      const float mr = m[rr] == -INFINITY ? 0.0f : m[rr];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        float p[2], w[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float v = s[t][2 * rr + i];
          p[i] = fa2::ex2_mufu(fmaf(v, row_sc[rr], -mr));
          // A masked key's scale may be anything: its weight is 0, not 0 * sv.
          w[i] = masked && pos0 + t * 8 + 2 * c + i > lim[rr] ? 0.0f : p[i] * (sv[t][i] * gs);
        }
        l[rr] += p[0] + p[1];
        pa[rr + 2 * t] = x2_of_floats<false>(w[0], w[1]);
      }
    }
    // O += P' V.
    uint32_t v0[4], v1[4], v2[4], v3[4];
    {
      constexpr int NB = D / 8;
      const int byte = g * NB;
      const uint32_t vst = st + 16 * C::ROW;
      auto at = [&](int r) { return vst + r * C::ROW + (((byte >> 4) ^ C::swz_v(r)) << 4) + (byte & 15); };
      lds<NB>(at(2 * c), v0);
      lds<NB>(at(2 * c + 1), v1);
      lds<NB>(at(2 * c + 8), v2);
      lds<NB>(at(2 * c + 9), v3);
    }
#pragma unroll
    for (int w = 0; w < (D + 31) / 32; ++w) {
      const uint32_t e0 = __byte_perm(v0[w], v1[w], 0x5140), e1 = __byte_perm(v2[w], v3[w], 0x5140);
      mma16816(o[4 * w], pa, f16x2_of_e4m3x2(static_cast<uint16_t>(e0)), f16x2_of_e4m3x2(static_cast<uint16_t>(e1)));
      mma16816(o[4 * w + 1], pa, f16x2_of_e4m3x2(static_cast<uint16_t>(e0 >> 16)), f16x2_of_e4m3x2(static_cast<uint16_t>(e1 >> 16)));
      if constexpr (D >= 32) {
        const uint32_t f0 = __byte_perm(v0[w], v1[w], 0x7362), f1 = __byte_perm(v2[w], v3[w], 0x7362);
        mma16816(o[4 * w + 2], pa, f16x2_of_e4m3x2(static_cast<uint16_t>(f0)), f16x2_of_e4m3x2(static_cast<uint16_t>(f1)));
        mma16816(o[4 * w + 3], pa, f16x2_of_e4m3x2(static_cast<uint16_t>(f0 >> 16)), f16x2_of_e4m3x2(static_cast<uint16_t>(f1 >> 16)));
      }
    }
    __syncwarp();  // every lane has read the stage before it is filled again
  }
  cp_async_wait<0>();
  __syncwarp();

  // Merge the warps: (m, l, O) of each in shared memory, O in the sv's own units.
  float* wo = reinterpret_cast<float*>(smem + warp * C::RING);
  float* wm = reinterpret_cast<float*>(smem + DEC_WARPS * C::RING);  // [warp][16]
  float* wl = wm + DEC_WARPS * 16;
  // 2^(eb - 127 - P_SHIFT), as two factors so that neither leaves the normal range.
  const float u0 = pow2f((eb - 127 - P_SHIFT) / 2), u1 = pow2f((eb - 127 - P_SHIFT) - (eb - 127 - P_SHIFT) / 2);
#pragma unroll
  for (int rr = 0; rr < 2; ++rr) {
    const float sum = quad_sum(l[rr]);
    const int r = g + 8 * rr;
    if (c == 0) {
      wm[warp * 16 + r] = m[rr];
      wl[warp * 16 + r] = sum;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float* dst = wo + r * D + (2 * c + i) * (D / 8);
#pragma unroll
      for (int j = 0; j < D / 8; ++j) dst[j] = o[j][2 * rr + i] * u0 * u1;
    }
  }
  __syncthreads();
  const int r = threadIdx.x >> 3, part = threadIdx.x & 7;  // 128 threads: 16 rows x 8 parts
  const int row = row0 + r;
  if (row >= rows) return;
  constexpr int PER = D / 8;
  float mx = -INFINITY;
#pragma unroll
  for (int w = 0; w < DEC_WARPS; ++w) mx = fmaxf(mx, wm[w * 16 + r]);
  float sum = 0.0f, acc[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) acc[j] = 0.0f;
#pragma unroll
  for (int w = 0; w < DEC_WARPS; ++w) {
    const float mw = wm[w * 16 + r], lw = wl[w * 16 + r];
    // A warp that saw no key of the row has m = -inf and l = 0; a NaN sum is kept.
    const float f = mw == -INFINITY ? (lw == 0.0f ? 0.0f : 1.0f) : exp2f(mw - mx);
    if (f == 0.0f) continue;
    sum = fmaf(f, lw, sum);
    const float* src = reinterpret_cast<const float*>(smem + w * C::RING) + r * D + part * PER;
#pragma unroll
    for (int j = 0; j < PER; ++j) acc[j] = fmaf(f, src[j], acc[j]);
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
  for (int j = 0; j < PER; ++j) acc[j] *= inv;
  if (a.splits > 1) {
    const int64_t slot = (static_cast<int64_t>(b * a.heads_kv + h) * a.splits + split) * a.rows_pad + row;
    float* dst = a.o_part + slot * D + part * PER;
#pragma unroll
    for (int j = 0; j < PER; ++j) dst[j] = acc[j];
    if (part == 0) a.lse_part[slot] = sum == 0.0f ? -INFINITY : (mx == -INFINITY ? 0.0f : mx) + log2f(sum);
  } else {
    uint32_t* dst = reinterpret_cast<uint32_t*>(o_row(a, sq, b, h, row) + part * PER);
#pragma unroll
    for (int j = 0; j < PER; j += 2) dst[j / 2] = x2_of_floats<BF16>(acc[j], acc[j + 1]);
  }
}

// ------------------------------------------------------------------ merge of the key ranges
// One warp a row: o = sum_s 2^(lse_s - max) o_s / sum_s 2^(lse_s - max) in split order.
template <int D, bool BF16, int ROWS>
__global__ void __launch_bounds__(128) merge_kernel(const AttnArgs a) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t x = static_cast<int64_t>(blockIdx.x) * 4 + warp;
  const int row = static_cast<int>(x % a.rows_pad);
  const int bh = static_cast<int>(x / a.rows_pad);
  if (bh >= a.batch * a.heads_kv) return;
  const int b = bh / a.heads_kv, h = bh - b * a.heads_kv;
  const Seq sq = sequence(a, b);
  const int rows = sq.n_q * a.group;
  if (row >= rows) return;
  const int row0 = row / ROWS * ROWS;
  const int ns = (keys_end(a, sq, row0, min(ROWS, rows - row0)) + a.split_keys - 1) / a.split_keys;
  const float* lse = a.lse_part + static_cast<int64_t>(bh) * a.splits * a.rows_pad + row;
  const float* op = a.o_part + (static_cast<int64_t>(bh) * a.splits * a.rows_pad + row) * D;
  float mx = -INFINITY;
  for (int s = lane; s < ns; s += 32) mx = fmaxf(mx, lse[static_cast<int64_t>(s) * a.rows_pad]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  constexpr int PER = D >= 32 ? D / 32 : 1;
  const bool on = lane * PER < D;
  float acc[PER] = {}, sum = 0.0f;
  for (int s0 = 0; s0 < ns; s0 += 32) {
    float w = 0.0f;
    if (s0 + lane < ns) {
      const float v = lse[static_cast<int64_t>(s0 + lane) * a.rows_pad];
      w = v == -INFINITY ? 0.0f : exp2f(v - (mx == -INFINITY ? 0.0f : mx));  // a NaN stays one
    }
    const int n = min(32, ns - s0);
#pragma unroll 4
    for (int s = 0; s < n; ++s) {
      const float f = __shfl_sync(0xffffffffu, w, s);
      if (on && f != 0.0f) {
        const float* src = op + static_cast<int64_t>(s0 + s) * a.rows_pad * D + lane * PER;
#pragma unroll
        for (int i = 0; i < PER; ++i) acc[i] = fmaf(f, src[i], acc[i]);
      }
      sum += f;
    }
  }
  if (!on) return;
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  uint16_t* dst = o_row(a, sq, b, h, row) + lane * PER;
#pragma unroll
  for (int i = 0; i < PER; ++i) dst[i] = x1_of_float<BF16>(acc[i] * inv);
}

// ------------------------------------------------------------------------------------ host
struct Plan {
  bool chunk = false;  // the 256-row kernel
  int row_blocks = 1, rows_pad = 16, splits = 1, split_keys = 0;
  int64_t lse_floats = 0, bytes = 0;
};

constexpr int MAX_SPLITS = 256;

// The kernel and the key ranges of a call, from its sizes alone.
Plan plan(const Fa2Kv8AttnParams* p) {
  Plan r;
  const int64_t rows = static_cast<int64_t>(p->seqlen_q) * (p->heads_q / p->cache.heads_kv);
  r.chunk = rows > 16;
  const int per_block = r.chunk ? 256 : 16;
  r.row_blocks = static_cast<int>((rows + per_block - 1) / per_block);
  r.rows_pad = r.row_blocks * per_block;
  int64_t units = static_cast<int64_t>(p->batch) * p->cache.heads_kv * r.row_blocks;
  if (units < 1) units = 1;
  // Few rows: one wave of three CTAs on each of 148 SMs, at least two 16-key groups for each of a
  // CTA's warps. Many rows: one wave of one CTA an SM, at least four 128-key tiles each.
  const int unit_keys = r.chunk ? 128 : 64;
  int64_t s = p->num_splits > 0 ? p->num_splits : (r.chunk ? 148 : 148 * 3) / units;
  const int64_t least = p->num_splits > 0 ? unit_keys : r.chunk ? 512 : 128;
  const int64_t most = (p->max_seqlen_k + least - 1) / least;
  if (s > most) s = most;
  if (s > MAX_SPLITS) s = MAX_SPLITS;
  if (s < 1) s = 1;
  const int64_t per = (p->max_seqlen_k + s - 1) / s;
  const int64_t keys = (per + unit_keys - 1) / unit_keys * unit_keys;
  r.split_keys = static_cast<int>(keys < unit_keys ? unit_keys : keys > (1ll << 30) ? (1ll << 30) : keys);
  r.splits = static_cast<int>((static_cast<int64_t>(p->max_seqlen_k) + r.split_keys - 1) / r.split_keys);
  if (r.splits < 1) r.splits = 1;
  if (r.splits > 1) {
    const int64_t slots = static_cast<int64_t>(p->batch) * p->cache.heads_kv * r.splits * r.rows_pad;
    r.lse_floats = (slots + 3) / 4 * 4;
    r.bytes = 4 * (r.lse_floats + slots * p->cache.head_dim);
  }
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
  // Row numbers and the grid stay in 31 bits.
  const int64_t rows = static_cast<int64_t>(p->seqlen_q) * (p->heads_q / p->cache.heads_kv);
  if (rows > (1ll << 30)) return FA2_ERR_SHAPE;
  if (static_cast<int64_t>(p->batch) * p->cache.heads_kv > (1ll << 26)) return FA2_ERR_SHAPE;
  const Plan r = plan(p);
  if (static_cast<int64_t>(p->batch) * p->cache.heads_kv * r.splits > (1ll << 32) / (r.rows_pad > 0 ? r.rows_pad : 1)) {
    return FA2_ERR_SHAPE;
  }
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

template <int D, bool BF16>
int launch(const AttnArgs& a, bool chunk, cudaStream_t s, int dev) {
  static std::atomic<bool> done[2][MAX_DEVICES];
  const unsigned ctas = static_cast<unsigned>(static_cast<int64_t>(a.batch) * a.heads_kv * a.splits * a.row_blocks);
  if (chunk) {
    auto kernel = chunk_kernel<D, BF16>;
    if (!allow_smem(kernel, Ch<D, BF16>::SMEM, dev, done[1])) return FA2_ERR_LAUNCH;
    kernel<<<ctas, CH_THREADS, Ch<D, BF16>::SMEM, s>>>(a);
  } else {
    auto kernel = decode_kernel<D, BF16>;
    if (!allow_smem(kernel, Dec<D>::SMEM, dev, done[0])) return FA2_ERR_LAUNCH;
    kernel<<<ctas, DEC_WARPS * 32, Dec<D>::SMEM, s>>>(a);
  }
  const int rc = launch_status();
  if (rc != FA2_OK || a.splits <= 1) return rc;
  const int64_t rows = static_cast<int64_t>(a.batch) * a.heads_kv * a.rows_pad;
  const unsigned blocks = static_cast<unsigned>((rows + 3) / 4);
  if (chunk) {
    merge_kernel<D, BF16, 256><<<blocks, 128, 0, s>>>(a);
  } else {
    merge_kernel<D, BF16, 16><<<blocks, 128, 0, s>>>(a);
  }
  return launch_status();
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
  a.heads_kv = p->cache.heads_kv;
  a.n_q = p->seqlen_q;
  a.total_q = p->total_q;
  a.max_k = p->max_seqlen_k;
  a.causal = p->causal;
  a.bottom_right = p->causal && p->causal_align == FA2_CAUSAL_BOTTOM_RIGHT;
  a.splits = r.splits;
  a.split_keys = r.split_keys;
  a.row_blocks = r.row_blocks;
  a.rows_pad = r.rows_pad;
  a.qk_scale = p->qk_scale;
  a.lse_part = static_cast<float*>(p->workspace);
  a.o_part = r.splits > 1 ? a.lse_part + r.lse_floats : nullptr;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf = p->dtype == FA2_DTYPE_BF16;
  switch (p->cache.head_dim) {
    case 16: return bf ? launch<16, true>(a, r.chunk, s, dev) : launch<16, false>(a, r.chunk, s, dev);
    case 32: return bf ? launch<32, true>(a, r.chunk, s, dev) : launch<32, false>(a, r.chunk, s, dev);
    case 64: return bf ? launch<64, true>(a, r.chunk, s, dev) : launch<64, false>(a, r.chunk, s, dev);
    default: return bf ? launch<128, true>(a, r.chunk, s, dev) : launch<128, false>(a, r.chunk, s, dev);
  }
}

}  // extern "C"
