// Attention over the 8-bit paged cache for many rows (chunks of prompts): tcgen05 products.
//
// Bound by the tensor cores (4 D operations a score) and, inside a step, by the exponentials
// (16 a clock and SM), the issue slots and shared memory. A CTA owns 256 rows (queries x heads of a
// group) as two 128-row tiles that take turns: while one tile's scores go through the softmax, the
// tensor core works on the other. With 128 rows or fewer both tiles hold the same rows and take
// every other 128-key tile, merged at the end.
//
// QK^T runs on the codes as they are stored: K is an e4m3 operand, and a row of Q, times the power
// of two that brings its largest value into [128, 256), is the sum of two e4m3 operands for bf16
// (8 significant bits: 4 and a sign's 4) or three for fp16 (11 bits). That is exact but for values
// more than 2^10 below the row's largest, which are off by at most 2^-17 of it. 8-bit products run
// at twice the rate of 16-bit ones, so the second operand costs nothing over converting K to fp16
// (64 instructions less for each 16 values).
//
// PV runs on fp16: P' needs 11 bits. V is converted on its way into shared memory. Its row scales:
// bf16 queries fold them into that conversion (code * s_j in fp16, one rounding of at most 2^-11, an
// eighth of the output's half step); for fp16 queries, whose half step is 2^-11 itself, the codes
// stay exact and each probability is multiplied by its key's scale in fp32. K's scales multiply the
// scores.
//
// Warps 0-3 / 4-7: softmax of tile 0 / 1, one thread a row (scores and P' live in TMEM, P' feeds the
// second product from there). Warps 8-11: bring the tiles in from their pages: K by asynchronous
// copies, two tiles ahead, V through registers. Warp 12: issues the products.
#pragma once

#include <type_traits>

#include "kv8_attn.cuh"

namespace fa2kv {

using fa2::mbar_arrive;
using fa2::mbar_init;
using fa2::mbar_wait;
using fa2::mbar_wait_warp;
using fa2::mma_commit;
using fa2::smem_u32;
using fa2::tc_fence_after;
using fa2::tc_fence_before;

constexpr int CH_THREADS = 512;
constexpr int CH_CONV_WARP = 8, CH_CONV_THREADS = 128, CH_MMA_WARP = 12;
constexpr int CH_KSLOTS = 3, CH_VSLOTS = 2;  // rings of K (codes) and V (fp16) tiles
constexpr int CH_ENTRIES = 8;                // ring of the tiles' scales
constexpr int CH_REGS = 128;                 // a thread at launch, then by warpgroup:
constexpr int CH_REGS_SM = 176, CH_REGS_CONV = 88, CH_REGS_MMA = 72;
static_assert(256 * CH_REGS_SM + 128 * CH_REGS_CONV + 128 * CH_REGS_MMA <= CH_THREADS * CH_REGS, "register split");
constexpr long long CH_TIMEOUT = 2000000000ll;
constexpr int FOLD_SHIFT = 6;   // folded scales: the largest lies in [2^6, 2^7), times 448 below 2^16

template <int D, bool BF16>
struct Ch {
  static constexpr int TERMS = BF16 ? 2 : 3;          // e4m3 operands of Q
  static constexpr int KSTEPS = D > 32 ? D / 32 : 1;  // 32-wide steps of QK^T (D = 16: zeros beyond)
  static constexpr int CODES = 128 * 128;             // bytes of a tile of codes: 128-byte rows
  static constexpr int CHUNKS = D > 64 ? D / 64 : 1;  // 64-column pieces of an fp16 tile
  static constexpr int CHUNK = 128 * 128;
  static constexpr int VTILE = CHUNKS * CHUNK;
  static constexpr int OFF_Q = 0;  // [tile][term]
  static constexpr int OFF_K = 2 * TERMS * CODES;
  static constexpr int OFF_V = OFF_K + CH_KSLOTS * CODES;
  static constexpr int OFF_SC = OFF_V + CH_VSLOTS * VTILE;      // [entry][2][128] words
  static constexpr int OFF_HEAD = OFF_SC + CH_ENTRIES * 1024;   // [entry] exponent field of sv
  static constexpr int OFF_MAX = OFF_HEAD + CH_ENTRIES * 4;     // [2][4 warps]
  static constexpr int OFF_BAR = OFF_MAX + 32;
  static constexpr int OFF_TMEM = OFF_BAR + 256;
  static constexpr int SMEM = OFF_TMEM + 16 + 1024;             // and slack to align the base
  // The merge of two tiles of the same rows: O of tile 1 in fp32 over the rings.
  static constexpr int MERGE = 128 * D * 4 + 2 * 128 * 4;
  static_assert(OFF_K + MERGE <= OFF_SC, "merge area");
  static_assert(SMEM <= 227 * 1024, "shared memory");
  static constexpr int TMEM_O = 256;
};

enum ChBar { CB_Q = 0, CB_S = 2, CB_P = 4, CB_PL = 6, CB_O = 8, CB_KF = 10, CB_KE = CB_KF + CH_KSLOTS,
             CB_VF = CB_KE + CH_KSLOTS, CB_VE = CB_VF + CH_VSLOTS, CB_SC = CB_VE + CH_VSLOTS,
             CB_DONE = CB_SC + CH_ENTRIES, CB_COUNT };
static_assert(CB_COUNT * 8 <= 256, "barriers");

// A shared-memory descriptor's upper word (128-byte swizzle, 8-row groups 1024 bytes apart), and the
// lower one of a tile at `addr` with `lbo` bytes between 64-column pieces.
constexpr uint32_t DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lbo) { return ((addr >> 4) & 0x3fffu) | ((lbo >> 4) << 16); }

// The products take their operands as tile + compile-time offset and put the descriptor together in
// place: kept in variables, the unrolled steps' descriptors cost the issuing thread 50 registers.
// D[tmem] (+)= A[smem] * B[smem], both e4m3 (32 wide steps), fp32 sums.
template <int A_OFF, int B_OFF>
__device__ __forceinline__ void mma_e4m3(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b32 x, y;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "add.u32 x, %1, %5;\n\tadd.u32 y, %2, %6;\n\tmov.b64 da, {x, %7};\n\tmov.b64 db, {y, %7};\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(add), "n"(A_OFF >> 4), "n"(B_OFF >> 4), "r"(DESC_HI)
      : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem], both fp16 (16 wide steps).
template <int A_OFF, int B_OFF>
__device__ __forceinline__ void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc, uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b32 x, y;\n\t.reg .b64 db;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "add.u32 x, %1, %5;\n\tadd.u32 y, %2, %6;\n\tmov.b64 db, {y, %7};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [x], db, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "r"(b_lo), "r"(idesc), "r"(add), "n"(A_OFF), "n"(B_OFF >> 4), "r"(DESC_HI)
      : "memory");
}
template <int I, int N, typename F>
__device__ __forceinline__ void steps(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    steps<I + 1, N>(static_cast<F&&>(f));
  }
}
// Instruction descriptor of kind::f8f6f4: fp32 D, e4m3 A and B (type codes 0), both K-major.
__host__ __device__ constexpr uint32_t idesc_e4m3(int M, int N) {
  return (1u << 4) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}

__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}

// A scale as two fp16 parts (high | low << 16): 22 bits of it.
__device__ __forceinline__ uint32_t split_scale(float s) {
  const __half hi = __float2half_rn(s);
  const float rest = s - __half2float(hi);  // NaN where s is NaN or infinite
  return static_cast<uint32_t>(__half_as_ushort(hi)) |
         (static_cast<uint32_t>(__half_as_ushort(__float2half_rn(rest))) << 16);
}

// The four loading warps meet; false where one of them gave up, in all of them alike.
__device__ __forceinline__ bool conv_sync(bool ok) {
  uint32_t bad = ok ? 0u : 1u;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %0, 0;\n\t"
      "bar.red.or.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "+r"(bad)::"memory");
  return bad == 0;
}

template <int D, bool BF16>
__global__ void __launch_bounds__(CH_THREADS, 1) chunk_kernel(const AttnArgs a) {
  using C = Ch<D, BF16>;
  constexpr bool FOLD = BF16;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t sraw = smem_u32(smem_raw);
  const uint32_t sbase = (sraw + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (sbase - sraw);
  auto bar = [&](int i) -> uint32_t { return sbase + C::OFF_BAR + 8u * static_cast<uint32_t>(i); };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // Row blocks of one key range run next to one another (they share its bytes in L2), the last,
  // which see most keys, first.
  int x = static_cast<int>(blockIdx.x);
  const int rb = a.row_blocks - 1 - x % a.row_blocks;
  x /= a.row_blocks;
  const int split = x % a.splits;
  x /= a.splits;
  const int h = x % a.heads_kv, b = x / a.heads_kv;
  const Seq sq = sequence(a, b);
  const int rows = sq.n_q * a.group, row0 = rb * 256;
  if (row0 >= rows) return;  // (uniform, before any barrier)
  const int n_rows = min(256, rows - row0);
  const int kend = keys_end(a, sq, row0, n_rows);
  const int k0 = split * a.split_keys, k1 = min(kend, k0 + a.split_keys);
  const int tiles = k1 > k0 ? (k1 - k0 + 127) / 128 : 0;
  if (tiles == 0) {
    if (a.splits > 1) return;  // the merge kernel does not read this split
    for (int r = threadIdx.x; r < n_rows; r += CH_THREADS) {
      uint4* dst = reinterpret_cast<uint4*>(o_row(a, sq, b, h, row0 + r));
#pragma unroll
      for (int i = 0; i < D / 8; ++i) dst[i] = make_uint4(0, 0, 0, 0);
    }
    return;
  }
  const bool dual = n_rows <= 128;
  const int ahead = dual && tiles > 1 ? 2 : 1;  // score tiles under way
  const long long timeout = a.timeout > 0 ? a.timeout : CH_TIMEOUT;

  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(bar(CB_Q + t), 128);
      mbar_init(bar(CB_S + t), 1);
      mbar_init(bar(CB_P + t), 128);
      mbar_init(bar(CB_PL + t), 128);
      mbar_init(bar(CB_O + t), 1);
    }
    for (int s = 0; s < CH_KSLOTS; ++s) {
      mbar_init(bar(CB_KF + s), CH_CONV_THREADS);
      mbar_init(bar(CB_KE + s), 1);
    }
    for (int s = 0; s < CH_VSLOTS; ++s) {
      mbar_init(bar(CB_VF + s), CH_CONV_THREADS);
      mbar_init(bar(CB_VE + s), 1);
    }
    for (int s = 0; s < CH_ENTRIES; ++s) mbar_init(bar(CB_SC + s), CH_CONV_THREADS);
    mbar_init(bar(CB_DONE), 1);
    fa2::fence_mbar_init();
    fa2::fence_proxy_async_smem();
  }
  if (warp == CH_MMA_WARP) {
    __syncwarp();
    fa2::tmem_alloc(sbase + C::OFF_TMEM, 512);
    fa2::tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + C::OFF_TMEM);
  bool ok = true;

  if (warp >= CH_CONV_WARP && warp < CH_MMA_WARP) {
    // -------------------------------------------------------------- K codes, V codes -> fp16
    fa2::reg_dealloc<CH_REGS_CONV>();
    const int tid = static_cast<int>(threadIdx.x) - CH_CONV_WARP * 32;
    constexpr int PIECES = D / 16;  // 16-byte pieces of a row
    const int* bt = a.bt + b * a.bt_stride;
    const int ps = a.c.page_size;
    const bool small = ps < 128;
    const int slots = small ? 128 / ps : 1;
    // Pages of a tile: lane l holds page slot l's index (-1: no keys there, -2: refused).
    auto pages_of = [&](int n) -> int {
      const int key = k0 + n * 128 + lane * ps;
      if (lane >= slots || key >= sq.len || n >= tiles) return -1;
      const int pg = __ldg(bt + page_of(a.c, key));
      return pg >= 0 && pg < a.c.num_pages ? pg : -2;
    };
    const uint8_t* kh = a.c.k + h * a.c.k_st[2];
    const uint8_t* vh = a.c.v + h * a.c.v_st[2];

    // K: thread tid copies piece tid % PIECES of the rows tid / PIECES + K_ROWS * it, to rows of 128
    // bytes whose 16-byte parts are xor-ed with the row's number (128-byte swizzle).
    constexpr int K_ROWS = CH_CONV_THREADS / PIECES, K_IT = PIECES;
    const int k_row = tid / PIECES, k_piece = tid % PIECES;
    auto copy_k = [&](int n, int pg) {
      const uint32_t slot = sbase + C::OFF_K + (n % CH_KSLOTS) * C::CODES;
      const int keys = sq.len - (k0 + n * 128);
      const int page0 = __shfl_sync(0xffffffffu, pg, 0);
      const uint8_t* p0 = kh + k_piece * 16;
      if (!small) p0 += max(page0, 0) * a.c.k_st[0] + static_cast<int64_t>((k0 + n * 128) % ps + k_row) * a.c.k_st[1];
#pragma unroll
      for (int it = 0; it < K_IT; ++it) {
        const int r = it * K_ROWS + k_row;
        int page = page0;
        const uint8_t* p = p0 + it * K_ROWS * a.c.k_st[1];
        if (small) {
          page = __shfl_sync(0xffffffffu, pg, r >> a.c.page_shift);
          p = p0 + max(page, 0) * a.c.k_st[0] + (r & (ps - 1)) * a.c.k_st[1];
        }
        const bool in = r < keys && page >= 0;
        cp_async16(slot + r * 128 + ((k_piece ^ (r & 7)) << 4), in ? p : kh, in);
      }
    };

    // V: thread tid has piece tid % PC of the rows tid / PC + V_ROWS * it, 64 columns at a time, so
    // that eight neighbouring lanes write two rows and do not meet in a bank.
    constexpr int PC = PIECES < 4 ? PIECES : 4;
    constexpr int V_ROWS = CH_CONV_THREADS / PC, V_IT = 128 / V_ROWS * C::CHUNKS;
    const int v_row = tid / PC, v_piece = tid % PC;
    uint4 w[V_IT];  // the next tile's codes, in flight
    auto fetch_v = [&](int n, int pg) {
      const int keys = sq.len - (k0 + n * 128);
      const int page0 = __shfl_sync(0xffffffffu, pg, 0);
      const uint8_t* p0 = vh + v_piece * 16;
      if (!small) {
        p0 += max(page0, 0) * a.c.v_st[0] + static_cast<int64_t>((k0 + n * 128) % ps + v_row) * a.c.v_st[1];
        if (page0 >= 0 && keys >= 128) {
#pragma unroll
          for (int it = 0; it < V_IT; ++it) {
            w[it] = __ldg(reinterpret_cast<const uint4*>(p0 + (it % (128 / V_ROWS)) * V_ROWS * a.c.v_st[1] + it / (128 / V_ROWS) * 64));
          }
          return;
        }
      }
#pragma unroll
      for (int it = 0; it < V_IT; ++it) {
        const int r = (it % (128 / V_ROWS)) * V_ROWS + v_row;
        int page = page0;
        const uint8_t* p = p0 + (it % (128 / V_ROWS)) * V_ROWS * a.c.v_st[1] + it / (128 / V_ROWS) * 64;
        if (small) {
          page = __shfl_sync(0xffffffffu, pg, r >> a.c.page_shift);
          p = p0 + max(page, 0) * a.c.v_st[0] + (r & (ps - 1)) * a.c.v_st[1] + it / (128 / V_ROWS) * 64;
        }
        w[it] = make_uint4(0, 0, 0, 0);
        if (r < keys && page >= 0) w[it] = __ldg(reinterpret_cast<const uint4*>(p));
      }
    };
    auto convert_v = [&](int n) {
      uint8_t* dst = smem + C::OFF_V + (n % CH_VSLOTS) * C::VTILE + v_row * 128;
      const uint32_t part = (static_cast<uint32_t>(v_piece) * 2) ^ static_cast<uint32_t>(v_row & 7);
      const uint32_t* sc = reinterpret_cast<const uint32_t*>(smem + C::OFF_SC) + (n % CH_ENTRIES) * 256 + 128 + v_row;
      uint32_t ws[V_IT];
#pragma unroll
      for (int it = 0; it < V_IT; ++it) ws[it] = FOLD ? sc[(it % (128 / V_ROWS)) * V_ROWS] : 0u;
#pragma unroll
      for (int it = 0; it < V_IT; ++it) {
        const uint32_t c[4] = {w[it].x, w[it].y, w[it].z, w[it].w};
        uint32_t o[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          o[2 * i] = f16x2_of_e4m3x2(static_cast<uint16_t>(c[i]));
          o[2 * i + 1] = f16x2_of_e4m3x2(static_cast<uint16_t>(c[i] >> 16));
        }
        if constexpr (FOLD) {
          const uint32_t hi = __byte_perm(ws[it], ws[it], 0x1010), lo = __byte_perm(ws[it], ws[it], 0x3232);
#pragma unroll
          for (int i = 0; i < 8; ++i) o[i] = hfma2(o[i], hi, hmul2(o[i], lo));
        }
        uint8_t* row = dst + (it % (128 / V_ROWS)) * V_ROWS * 128 + it / (128 / V_ROWS) * C::CHUNK;
        *reinterpret_cast<uint4*>(row + (part << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
        *reinterpret_cast<uint4*>(row + ((part ^ 1u) << 4)) = make_uint4(o[4], o[5], o[6], o[7]);
      }
    };
    static_assert(V_ROWS % 8 == 0, "a thread's rows have the same swizzle");

    float sk = 0.0f, sv = 0.0f;  // of key tid of the next tile
    auto fetch_scales = [&](int n, int pg) {
      const int page = __shfl_sync(0xffffffffu, pg, small ? tid >> a.c.page_shift : 0);
      const int row = small ? tid & (ps - 1) : (k0 + n * 128) % ps + tid;
      const bool in = k0 + n * 128 + tid < sq.len;
      sk = sv = 0.0f;
      if (page >= 0 && in) {
        sk = __ldg(a.c.ks + h * a.c.ks_st[2] + page * a.c.ks_st[0] + row * a.c.ks_st[1]);
        sv = __ldg(a.c.vs + h * a.c.vs_st[2] + page * a.c.vs_st[0] + row * a.c.vs_st[1]);
      } else if (page == -2 && in) {  // queries that see a key of a refused page get NaN
        sv = __uint_as_float(0x7fc00000u);
        report(a.err, FA2_ERR_PAGE);
      }
    };
    int eb = EB_MIN;  // exponent field of the largest finite sv so far
    // Scales of tile n into its entry, and the exponent that they are relative to.
    auto store_scales = [&](int n) {
      // A value row that is not finite makes its key's score NaN instead (0 * NaN in the second
      // product would reach the rows that do not see the key).
      if (!(fabsf(sv) < INFINITY)) {
        sk = __uint_as_float(0x7fc00000u);
        sv = 0.0f;
      }
      const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(sv) & 0x7fffffffu);
      uint32_t* wm = reinterpret_cast<uint32_t*>(smem + C::OFF_MAX) + (n & 1) * 4;
      if (lane == 0) wm[warp - CH_CONV_WARP] = top;
      conv_sync(true);
      eb = max(eb, static_cast<int>(max(max(wm[0], wm[1]), max(wm[2], wm[3])) >> 23));
      const int en = n % CH_ENTRIES;
      const float fv = __uint_as_float(static_cast<uint32_t>(254 + FOLD_SHIFT - eb) << 23);
      uint32_t* dst = reinterpret_cast<uint32_t*>(smem + C::OFF_SC) + en * 256 + tid;
      dst[0] = __float_as_uint(sk);
      dst[128] = FOLD ? split_scale(sv * fv) : __float_as_uint(sv * fv);
      if (tid == 0) reinterpret_cast<int*>(smem + C::OFF_HEAD)[en] = eb;
      mbar_arrive(bar(CB_SC + en));
      if (FOLD) conv_sync(true);  // the conversion reads the scales of the others' keys
    };

    if constexpr (D < 32) {  // the second half of the only 32-wide step
      for (int i = tid; i < CH_KSLOTS * 128 * 8; i += CH_CONV_THREADS) {
        *reinterpret_cast<uint4*>(smem + C::OFF_K + i * 16) = make_uint4(0, 0, 0, 0);
      }
      conv_sync(true);
    }
    // Step n: K_n has landed; K_(n + 2) is asked for; V_n is converted from registers and V_(n + 1)
    // fetched into them. The page numbers of tile n + 3 are on their way.
    int pg0 = pages_of(0), pg1 = pages_of(1), pg2 = pages_of(2);
    copy_k(0, pg0);
    cp_async_commit();
    if (tiles > 1) copy_k(1, pg1);
    cp_async_commit();
    fetch_v(0, pg0);
    fetch_scales(0, pg0);
    for (int n = 0; n < tiles; ++n) {
      const int pg3 = pages_of(n + 3);
      bool go = true;
      if (n + 2 < tiles) {
        const int s = (n + 2) % CH_KSLOTS;
        go = mbar_wait_warp(bar(CB_KE + s), (static_cast<uint32_t>((n + 2) / CH_KSLOTS) & 1u) ^ 1u, timeout, a.err);
        if (go) copy_k(n + 2, pg2);
      }
      cp_async_commit();
      cp_async_wait<2>();
      fa2::fence_proxy_async_smem();
      mbar_arrive(bar(CB_KF + n % CH_KSLOTS));
      go = go && mbar_wait_warp(bar(CB_VE + n % CH_VSLOTS), (static_cast<uint32_t>(n / CH_VSLOTS) & 1u) ^ 1u, timeout, a.err);
      ok = conv_sync(go);
      if (!ok) break;
      store_scales(n);
      convert_v(n);
      if (n + 1 < tiles) {
        fetch_v(n + 1, pg1);
        fetch_scales(n + 1, pg1);
      }
      fa2::fence_proxy_async_smem();
      mbar_arrive(bar(CB_VF + n % CH_VSLOTS));
      pg1 = pg2;
      pg2 = pg3;
    }
    cp_async_wait<0>();
  } else if (warp == CH_MMA_WARP) {
    // -------------------------------------------------------------- products
    fa2::reg_dealloc<CH_REGS_MMA>();
    if (lane == 0) {
      constexpr uint32_t idesc_qk = idesc_e4m3(128, 128);
      constexpr uint32_t idesc_pv = fa2::idesc_f16(false, 128, D, true);
      const uint32_t dq = desc_lo(sbase + C::OFF_Q, 16), dk = desc_lo(sbase + C::OFF_K, 16);
      const uint32_t dv = desc_lo(sbase + C::OFF_V, C::CHUNK);
      auto wait = [&](int i, uint32_t parity) -> bool { return mbar_wait(bar(i), parity, timeout, a.err); };
      auto qk = [&](int t, int n) {
        const uint32_t qd = dq + static_cast<uint32_t>(((dual ? 0 : t) * C::TERMS * C::CODES) >> 4);
        const uint32_t kd = dk + static_cast<uint32_t>(((n % CH_KSLOTS) * C::CODES) >> 4);
        steps<0, C::TERMS * C::KSTEPS>([&](auto i) {
          constexpr int term = decltype(i)::value / C::KSTEPS, kk = decltype(i)::value % C::KSTEPS;
          mma_e4m3<term * C::CODES + kk * 32, kk * 32>(tmem + t * 128, qd, kd, idesc_qk, term + kk > 0 ? 1u : 0u);
        });
        mma_commit(bar(CB_S + t));
      };
      // P' of tile t comes in two parts: 96 keys, then 32.
      auto pv = [&](int t, int n, bool acc, uint32_t parity) -> bool {
        const uint32_t vd = dv + static_cast<uint32_t>(((n % CH_VSLOTS) * C::VTILE) >> 4);
        const uint32_t td = tmem + C::TMEM_O + t * D, tp = tmem + t * 128 + 64;
        if (!wait(CB_P + t, parity)) return false;
        tc_fence_after();
        steps<0, 6>([&](auto kk) {
          mma_f16_ts<decltype(kk)::value * 8, decltype(kk)::value * 16 * 128>(td, tp, vd, idesc_pv, (acc || decltype(kk)::value > 0) ? 1u : 0u);
        });
        if (!wait(CB_PL + t, parity)) return false;
        tc_fence_after();
        mma_f16_ts<6 * 8, 6 * 16 * 128>(td, tp, vd, idesc_pv, 1u);
        mma_f16_ts<7 * 8, 7 * 16 * 128>(td, tp, vd, idesc_pv, 1u);
        return true;
      };
      auto take_k = [&](int n) -> bool {
        if (!wait(CB_KF + n % CH_KSLOTS, static_cast<uint32_t>(n / CH_KSLOTS) & 1u)) return false;
        tc_fence_after();
        return true;
      };
      auto take_v = [&](int n) -> bool {
        if (!wait(CB_VF + n % CH_VSLOTS, static_cast<uint32_t>(n / CH_VSLOTS) & 1u)) return false;
        tc_fence_after();
        return true;
      };
      auto drop_k = [&](int n) { mma_commit(bar(CB_KE + n % CH_KSLOTS)); };
      auto drop_v = [&](int n) { mma_commit(bar(CB_VE + n % CH_VSLOTS)); };
      ok = wait(CB_Q + 0, 0) && (dual || wait(CB_Q + 1, 0));
      if (ok && dual) {
        for (int n = 0; ok && n < ahead; ++n) {
          ok = take_k(n);
          if (ok) {
            qk(n & 1, n);
            drop_k(n);
          }
        }
        for (int n = 0; ok && n < tiles; ++n) {
          const int t = n & 1;
          ok = take_v(n) && pv(t, n, n > 1, static_cast<uint32_t>(n >> 1) & 1u);
          if (!ok) break;
          if (n + 2 >= tiles) mma_commit(bar(CB_O + t));
          drop_v(n);
          if (n + ahead < tiles) {
            ok = take_k(n + ahead);
            if (!ok) break;
            qk((n + ahead) & 1, n + ahead);
            drop_k(n + ahead);
          }
        }
      } else if (ok) {
        ok = take_k(0);
        if (ok) {
          qk(0, 0);
          qk(1, 0);
          drop_k(0);
        }
        for (int n = 0; ok && n < tiles; ++n) {
          const bool more = n + 1 < tiles;
          const uint32_t parity = static_cast<uint32_t>(n) & 1u;
          for (int t = 0; t < 2 && ok; ++t) {
            ok = (t > 0 || take_v(n)) && pv(t, n, n > 0, parity);
            if (!ok) break;
            if (!more) mma_commit(bar(CB_O + t));
            if (t == 1) drop_v(n);
            if (more) {
              ok = t > 0 || take_k(n + 1);
              if (!ok) break;
              qk(t, n + 1);
              if (t == 1) drop_k(n + 1);
            }
          }
        }
      }
      // Every product has retired before TMEM is given back.
      mma_commit(bar(CB_DONE));
      if (!mbar_wait(bar(CB_DONE), 0, CH_TIMEOUT, nullptr)) ok = false;
    }
    __syncwarp();
  } else if (warp > CH_MMA_WARP) {
    fa2::reg_dealloc<CH_REGS_MMA>();
  } else {
    // -------------------------------------------------------------- softmax: one thread a row
    fa2::reg_alloc<CH_REGS_SM>();
    const int t = warp >> 2, q = warp & 3;
    const int r = q * 32 + lane;  // row of the tile
    const int row = row0 + (dual ? 0 : t * 128) + r;
    const bool have = row < row0 + n_rows;
    const uint32_t lane_addr = static_cast<uint32_t>(q * 32) << 16;
    const uint32_t tS = tmem + t * 128 + lane_addr, tP = tS + 64, tO = tmem + C::TMEM_O + t * D + lane_addr;

    // Q: this row as e4m3 terms, times the power of two that brings its largest value into [128, 256).
    // Each term is the rounding of what the terms before leave (an exact difference in fp32).
    float row_sc;
    {
      uint32_t top = 0;
      const uint4* src = reinterpret_cast<const uint4*>(q_row(a, sq, b, h, have ? row : row0));
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        const uint4 v = have ? __ldg(src + i) : make_uint4(0, 0, 0, 0);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f2 = float2_of_x2<BF16>(w[j]);
          top = max(top, max(__float_as_uint(f2.x) & 0x7fffffffu, __float_as_uint(f2.y) & 0x7fffffffu));
        }
      }
      const int e = row_exponent(top);
      const float f = top < 0x7f800000u ? pow2f(7 - e) : __uint_as_float(0x7fc00000u);  // NaN, infinity: a NaN row
      row_sc = a.qk_scale * pow2f(max(-126, e - 7));
      if (!dual || t == 0) {
        const uint32_t dst = sbase + C::OFF_Q + t * C::TERMS * C::CODES + r * 128;
#pragma unroll
        for (int i = 0; i < (D + 15) / 16; ++i) {
          float x[16];
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            const uint4 v = have ? __ldg(src + 2 * i + z) : make_uint4(0, 0, 0, 0);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 f2 = float2_of_x2<BF16>(w[j]);
              x[8 * z + 2 * j] = f2.x * f;
              x[8 * z + 2 * j + 1] = f2.y * f;
            }
          }
#pragma unroll
          for (int term = 0; term < C::TERMS; ++term) {
            uint32_t o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint16_t lo = e4m3x2(x[4 * j], x[4 * j + 1]), hi = e4m3x2(x[4 * j + 2], x[4 * j + 3]);
              const float2 y0 = float2_of_f16x2(f16x2_of_e4m3x2(lo)), y1 = float2_of_f16x2(f16x2_of_e4m3x2(hi));
              x[4 * j] -= y0.x;
              x[4 * j + 1] -= y0.y;
              x[4 * j + 2] -= y1.x;
              x[4 * j + 3] -= y1.y;
              o[j] = static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
            }
            fa2::st_shared_v4(dst + term * C::CODES + ((i ^ (r & 7)) << 4), o[0], o[1], o[2], o[3]);
            if constexpr (D < 32) fa2::st_shared_v4(dst + term * C::CODES + ((1 ^ (r & 7)) << 4), 0, 0, 0, 0);
          }
        }
        fa2::fence_proxy_async_smem();
        mbar_arrive(bar(CB_Q + t));
      }
    }
    const int lim_row = have ? last_key(a, sq, row / a.group) : -1;  // last visible key
    const int tile_row0 = row0 + (dual ? 0 : t * 128);
    // All keys up to here are seen by every row of the tile (rows that are not there are zeros).
    const int lim_all = last_key(a, sq, tile_row0 / a.group);

    float m = -INFINITY, l = 0.0f;
    int eb = EB_MIN;
    const int step = dual ? 2 : 1;
    int done = 0;
    for (int n = dual ? t : 0; n < tiles; n += step, ++done) {
      const int en = n % CH_ENTRIES;
      if (!mbar_wait_warp(bar(CB_S + t), static_cast<uint32_t>(done) & 1u, timeout, a.err) ||
          !mbar_wait_warp(bar(CB_SC + en), static_cast<uint32_t>(n / CH_ENTRIES) & 1u, timeout, a.err)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t sc_addr = sbase + C::OFF_SC + en * 1024;
      int eb_new;
      asm volatile("ld.shared.b32 %0, [%1];" : "=r"(eb_new) : "r"(sbase + C::OFF_HEAD + en * 4));
      const int col0 = k0 + n * 128;
      const float sc = row_sc;
      const bool masked = col0 + 127 > lim_all;
      const int lim = lim_row - col0;

      uint32_t s[4][32];
      fa2::tmem_ld64(tS, s[0], s[1]);
      fa2::tmem_ld64(tS + 64, s[2], s[3]);
      fa2::tmem_wait_ld();
#pragma unroll
      for (int c = 0; c < 4; ++c) fa2::reg_fence32(s[c]);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          uint64_t k0, k1;
          asm volatile("ld.shared.v2.b64 {%0,%1}, [%2];" : "=l"(k0), "=l"(k1) : "r"(sc_addr + (c * 32 + i) * 4));
          float u0, u1, u2, u3;
          fa2::f2_unpack(fa2::f2_mul(fa2::f2_pack(__uint_as_float(s[c][i]), __uint_as_float(s[c][i + 1])), k0), u0, u1);
          fa2::f2_unpack(fa2::f2_mul(fa2::f2_pack(__uint_as_float(s[c][i + 2]), __uint_as_float(s[c][i + 3])), k1), u2, u3);
          s[c][i] = __float_as_uint(u0);
          s[c][i + 1] = __float_as_uint(u1);
          s[c][i + 2] = __float_as_uint(u2);
          s[c][i + 3] = __float_as_uint(u3);
        }
      }
      if (masked) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            if (c * 32 + i > lim) s[c][i] = 0xff800000u;
          }
        }
      }
      float mx[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        mx[c] = __uint_as_float(s[c][0]);
#pragma unroll
        for (int i = 1; i < 31; i += 2) mx[c] = fa2::fmax3(mx[c], __uint_as_float(s[c][i]), __uint_as_float(s[c][i + 1]));
        mx[c] = fmaxf(mx[c], __uint_as_float(s[c][31]));
      }
      // Folded: the reference lies FOLD_SHIFT below the maximum, so that P' uses fp16's range up to 2^14.
      const float cand = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sc - (FOLD ? static_cast<float>(P_SHIFT) : 0.0f);
      const bool bump = cand > m + RESCALE_TH;  // the first tile with a visible key: always
      float alpha = 1.0f;
      if (bump) {
        alpha = fa2::ex2_mufu(m - cand);
        m = cand;
      }
      l *= alpha;
      if (done > 0 && __any_sync(0xffffffffu, bump || eb_new > eb)) {
        // (PV of the step before has retired: this step's scores were committed after it.)
        alpha *= eb_new - eb > 126 ? 0.0f : pow2f(eb - eb_new);
        const uint64_t a2 = fa2::f2_pack(alpha, alpha);
#pragma unroll 1
        for (int c = 0; c < D / 16; ++c) {
          uint32_t o[16];
          fa2::tmem_ld16(tO + c * 16, o);
          fa2::tmem_wait_ld();
          fa2::reg_fence16(o);
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            float u, v;
            fa2::f2_unpack(fa2::f2_mul(fa2::f2_pack(__uint_as_float(o[i]), __uint_as_float(o[i + 1])), a2), u, v);
            o[i] = __float_as_uint(u);
            o[i + 1] = __float_as_uint(v);
          }
          fa2::tmem_st16(tO + c * 16, o);
        }
        fa2::tmem_wait_st();
      }
      eb = eb_new;
      const float mr = m == -INFINITY ? 0.0f : m;  // a row that has seen no key yet: p = 0, not NaN
      const uint64_t sc2 = fa2::f2_pack(sc, sc), nm2 = fa2::f2_pack(-mr, -mr);
      uint64_t sum2[4] = {0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          float p[4];
#pragma unroll
          for (int j = 0; j < 4; j += 2) {
            float x0, x1;
            fa2::f2_unpack(fa2::f2_fma(fa2::f2_pack(__uint_as_float(s[c][i + j]), __uint_as_float(s[c][i + j + 1])), sc2, nm2), x0, x1);
            p[j] = fa2::ex2_mufu(x0);
            p[j + 1] = fa2::ex2_mufu(x1);
            sum2[(i + j) / 2 & 3] = fa2::f2_add(sum2[(i + j) / 2 & 3], fa2::f2_pack(p[j], p[j + 1]));
          }
          if constexpr (!FOLD) {
            float v[4];
            asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];"
                         : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(sc_addr + 512 + (c * 32 + i) * 4));
#pragma unroll
            for (int j = 0; j < 4; ++j) p[j] *= v[j];
          }
          pk[i / 2] = x2_of_floats<false>(p[0], p[1]);
          pk[i / 2 + 1] = x2_of_floats<false>(p[2], p[3]);
        }
        fa2::tmem_st16(tP + c * 16, pk);
        if (c == 2) {
          fa2::tmem_wait_st();
          tc_fence_before();
          mbar_arrive(bar(CB_P + t));
        }
      }
      fa2::tmem_wait_st();
      tc_fence_before();
      mbar_arrive(bar(CB_PL + t));
      float s0, s1;
      fa2::f2_unpack(fa2::f2_add(fa2::f2_add(sum2[0], sum2[1]), fa2::f2_add(sum2[2], sum2[3])), s0, s1);
      l += s0 + s1;
    }
    // O, in the units of the last exponent: * 2^(eb - 127 - shift).
    if (ok && done > 0 && !mbar_wait_warp(bar(CB_O + t), 0, timeout, a.err)) ok = false;
    tc_fence_after();
    const int ex = eb - 127 - FOLD_SHIFT;
    const float u0 = pow2f(ex / 2), u1 = pow2f(ex - ex / 2);
    float* area = reinterpret_cast<float*>(smem + C::OFF_K);  // [D / 4][128] float4
    float* area_m = area + 128 * D;
    float* area_l = area_m + 128;
    if (dual) {
      // Once the last products of both tiles have retired the ring is free for tile 1's output.
      if (t == 1) {
        if (ok && !mbar_wait_warp(bar(CB_O + 0), 0, timeout, a.err)) ok = false;
        if (done > 0 && ok) {
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            uint32_t o[16];
            fa2::tmem_ld16(tO + c * 16, o);
            fa2::tmem_wait_ld();
            fa2::reg_fence16(o);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              reinterpret_cast<float4*>(area)[(c * 4 + i) * 128 + r] =
                  make_float4(__uint_as_float(o[4 * i]) * u0 * u1, __uint_as_float(o[4 * i + 1]) * u0 * u1,
                              __uint_as_float(o[4 * i + 2]) * u0 * u1, __uint_as_float(o[4 * i + 3]) * u0 * u1);
            }
          }
        }
        area_m[r] = m;
        area_l[r] = done > 0 ? l : 0.0f;
      }
      asm volatile("bar.sync 2, 256;" ::: "memory");
    }
    if (ok && !(dual && t == 1)) {  // (uniform in a warp: TMEM is read by whole warps)
      float f0 = 1.0f, f1 = 0.0f, mx = m, sum = l;
      if (dual) {
        const float m1 = area_m[r], l1 = area_l[r];
        mx = fmaxf(m, m1);
        // A tile that saw no key has m = -inf and l = 0; a NaN sum is kept.
        f0 = m == -INFINITY ? (l == 0.0f ? 0.0f : 1.0f) : exp2f(m - mx);
        f1 = m1 == -INFINITY ? (l1 == 0.0f ? 0.0f : 1.0f) : exp2f(m1 - mx);
        sum = f0 * l + f1 * l1;
      }
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      const float g0 = f0 * inv, g1 = f1 * inv;
      const int64_t part = (static_cast<int64_t>(b * a.heads_kv + h) * a.splits + split) * a.rows_pad + row;
#pragma unroll 1
      for (int c = 0; c < D / 16; ++c) {
        uint32_t o[16];
        __syncwarp();
        fa2::tmem_ld16(tO + c * 16, o);
        fa2::tmem_wait_ld();
        fa2::reg_fence16(o);
        if (!have) continue;
        float y[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) y[i] = sum == 0.0f ? 0.0f : __uint_as_float(o[i]) * u0 * u1 * g0;
        if (f1 != 0.0f) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float4 v = reinterpret_cast<const float4*>(area)[(c * 4 + i) * 128 + r];
            y[4 * i] = fmaf(v.x, g1, f0 == 0.0f ? 0.0f : y[4 * i]);
            y[4 * i + 1] = fmaf(v.y, g1, f0 == 0.0f ? 0.0f : y[4 * i + 1]);
            y[4 * i + 2] = fmaf(v.z, g1, f0 == 0.0f ? 0.0f : y[4 * i + 2]);
            y[4 * i + 3] = fmaf(v.w, g1, f0 == 0.0f ? 0.0f : y[4 * i + 3]);
          }
        }
        if (a.splits > 1) {
          float4* dst = reinterpret_cast<float4*>(a.o_part + part * D + c * 16);
#pragma unroll
          for (int i = 0; i < 4; ++i) dst[i] = make_float4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
        } else {
          uint32_t z[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) z[i] = x2_of_floats<BF16>(y[2 * i], y[2 * i + 1]);
          uint4* dst = reinterpret_cast<uint4*>(o_row(a, sq, b, h, row) + c * 16);
          dst[0] = make_uint4(z[0], z[1], z[2], z[3]);
          dst[1] = make_uint4(z[4], z[5], z[6], z[7]);
        }
      }
      if (have && a.splits > 1) a.lse_part[part] = sum == 0.0f ? -INFINITY : (mx == -INFINITY ? 0.0f : mx) + log2f(sum);
    }
  }

  if (!ok) report(a.err, FA2_ERR_TIMEOUT);
  tc_fence_before();
  __syncthreads();
  if (warp == CH_MMA_WARP) {
    __syncwarp();
    tc_fence_after();
    fa2::tmem_dealloc(tmem, 512);
  }
}

}  // namespace fa2kv
