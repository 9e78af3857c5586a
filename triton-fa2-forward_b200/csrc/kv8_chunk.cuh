// Attention over the 8-bit paged cache for many rows (chunks of prompts): tcgen05 products.
//
// Bound by the tensor cores (4 D operations a score) and, inside a step, by the exponentials
// (16 a clock and SM) and shared memory. A CTA owns 256 rows (queries x heads of a group) as two
// 128-row tiles that take turns: while one tile's scores go through the softmax, the tensor core
// works on the other. With 128 rows or fewer both tiles hold the same rows and take every other
// 128-key tile, merged at the end.
//
// Warps 0-3 / 4-7: softmax of tile 0 / 1, one thread a row (scores and P' live in TMEM, P' feeds the
// second product from there). Warps 8-10: bring the codes of 128-key tiles in from their pages and
// convert them to fp16, swizzled as the tensor core reads them, through a ring of three 16-bit
// tiles. Warp 11: issues the products.
//
// Where the row scales go. bf16 queries: into the conversion (code * s_j in fp16, one rounding of at
// most 2^-11, an eighth of the output's half step), which leaves nothing to do for each score. fp16
// queries, whose half step is 2^-11 itself: the codes stay exact and each score and probability is
// multiplied by its key's scale in fp32.
#pragma once

#include "kv8_attn.cuh"

namespace fa2kv {

using fa2::mbar_arrive;
using fa2::mbar_init;
using fa2::mbar_wait;
using fa2::mbar_wait_warp;
using fa2::mma_commit;
using fa2::mma_ss;
using fa2::mma_ts;
using fa2::smem_u32;
using fa2::tc_fence_after;
using fa2::tc_fence_before;

constexpr int CH_THREADS = 384;
constexpr int CH_CONV_WARP = 8, CH_CONV_THREADS = 96, CH_MMA_WARP = 11;
constexpr int CH_SLOTS = 3;     // ring of converted tiles
constexpr int CH_ENTRIES = 8;   // ring of the tiles' scales
constexpr int CH_REGS = 168;    // a thread at launch; then CH_REGS_SM / CH_REGS_OTHER
constexpr int CH_REGS_SM = 200, CH_REGS_OTHER = 104;
static_assert(256 * CH_REGS_SM + 128 * CH_REGS_OTHER <= CH_THREADS * CH_REGS, "register split");
constexpr long long CH_TIMEOUT = 2000000000ll;
constexpr int FOLD_SHIFT = 6;   // folded scales: the largest lies in [2^6, 2^7), times 448 below 2^16

template <int D>
struct Ch {
  static constexpr int CHUNKS = D > 64 ? D / 64 : 1;  // 64-column pieces of a 16-bit tile
  static constexpr int CHUNK = 128 * 128;             // bytes
  static constexpr int TILE = CHUNKS * CHUNK;
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_RING = 2 * TILE;
  static constexpr int OFF_SC = OFF_RING + CH_SLOTS * TILE;     // [entry][2][128] words
  static constexpr int OFF_HEAD = OFF_SC + CH_ENTRIES * 1024;   // [entry]{key scale of the tile, exponent of sv}
  static constexpr int OFF_MAX = OFF_HEAD + CH_ENTRIES * 8;     // [2][3 warps][2]
  static constexpr int OFF_BAR = OFF_MAX + 64;
  static constexpr int OFF_TMEM = OFF_BAR + 256;
  static constexpr int SMEM = OFF_TMEM + 16 + 1024;             // and slack to align the base
  // The merge of two tiles of the same rows: O of tile 1 in fp32 over the ring and what follows it.
  static constexpr int MERGE = 128 * D * 4 + 2 * 128 * 4 + 512;
  static_assert(OFF_RING + MERGE <= OFF_HEAD, "merge area");
  static_assert(SMEM <= 227 * 1024, "shared memory");
  static constexpr int TMEM_O = 256;
};

enum ChBar { CB_Q = 0, CB_S = 2, CB_P = 4, CB_PL = 6, CB_O = 8, CB_FULL = 10, CB_EMPTY = CB_FULL + CH_SLOTS,
             CB_SC = CB_EMPTY + CH_SLOTS, CB_DONE = CB_SC + CH_ENTRIES, CB_COUNT };
static_assert(CB_COUNT * 8 <= 256, "barriers");

// Order of the converted tiles, which is the order of the products: the first `ahead` K tiles, then
// V_n, K_(n + ahead) in turn, then the V tiles that are left. i -> (is V, n).
struct TileOrder {
  int tiles, ahead;
  __device__ void at(int i, bool& is_v, int& n) const {
    if (i < ahead) {
      is_v = false;
      n = i;
    } else if (i < 2 * tiles - ahead) {
      const int k = i - ahead;
      is_v = (k & 1) == 0;
      n = (k >> 1) + (is_v ? 0 : ahead);
    } else {
      is_v = true;
      n = i - tiles;
    }
  }
};

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

// The three converting warps meet; false where one of them gave up, in all of them alike.
__device__ __forceinline__ bool conv_sync(bool ok) {
  uint32_t bad = ok ? 0u : 1u;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %0, 0;\n\t"
      "bar.red.or.pred q, 1, 96, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "+r"(bad)::"memory");
  return bad == 0;
}

template <int D, bool BF16>
__global__ void __launch_bounds__(CH_THREADS, 1) chunk_kernel(const AttnArgs a) {
  using C = Ch<D>;
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
  TileOrder order;
  order.tiles = tiles;
  order.ahead = dual && tiles > 1 ? 2 : 1;
  const long long timeout = a.timeout > 0 ? a.timeout : CH_TIMEOUT;

  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(bar(CB_Q + t), 128);
      mbar_init(bar(CB_S + t), 1);
      mbar_init(bar(CB_P + t), 128);
      mbar_init(bar(CB_PL + t), 128);
      mbar_init(bar(CB_O + t), 1);
    }
    for (int s = 0; s < CH_SLOTS; ++s) {
      mbar_init(bar(CB_FULL + s), CH_CONV_THREADS);
      mbar_init(bar(CB_EMPTY + s), 1);
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
    // -------------------------------------------------------------- codes -> fp16 tiles
    fa2::reg_dealloc<CH_REGS_OTHER>();
    const int tid = static_cast<int>(threadIdx.x) - CH_CONV_WARP * 32;
    constexpr int PIECES = D / 16;                                     // 16-byte pieces of a row
    constexpr int N_IT = (128 * PIECES + CH_CONV_THREADS - 1) / CH_CONV_THREADS;
    const int* bt = a.bt + b * a.bt_stride;
    const int ps = a.c.page_size;
    const bool small = ps < 128;
    const int slots = small ? 128 / ps : 1;
    // Pages of a tile: lane l holds page slot l's index (-1: no keys there, -2: refused).
    auto pages_of = [&](int n) -> int {
      const int key = k0 + n * 128 + lane * ps;
      if (lane >= slots || key >= sq.len) return -1;
      const int pg = __ldg(bt + page_of(a.c, small ? key : k0 + n * 128));
      return pg >= 0 && pg < a.c.num_pages ? pg : -2;
    };
    auto page_row = [&](int pg, int n, int r, int& row) -> int {
      row = small ? r & (ps - 1) : (k0 + n * 128) % ps + r;
      return __shfl_sync(0xffffffffu, pg, small ? r >> a.c.page_shift : 0);
    };
    uint4 w[N_IT];  // the next tile's codes, in flight
    auto fetch_piece = [&](int it, int n, bool is_v, int pg) {
      const int e = it * CH_CONV_THREADS + tid;
      const int r = min(e / PIECES, 127), piece = e % PIECES;
      int row;
      const int page = page_row(pg, n, r, row);  // a shuffle: every lane
      w[it] = make_uint4(0, 0, 0, 0);
      if (e < 128 * PIECES && page >= 0 && k0 + n * 128 + r < sq.len) {
        const uint8_t* base = is_v ? a.c.v + h * a.c.v_st[2] + page * a.c.v_st[0] + row * a.c.v_st[1]
                                   : a.c.k + h * a.c.k_st[2] + page * a.c.k_st[0] + row * a.c.k_st[1];
        w[it] = __ldg(reinterpret_cast<const uint4*>(base + piece * 16));
      }
    };
    float sc[2][2] = {};  // (key tid, key tid + 96) x (sk, sv) of the next K tile
    auto fetch_scales = [&](int n, int pg) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = min(tid + 96 * i, 127);
        int row;
        const int page = page_row(pg, n, r, row);
        sc[i][0] = sc[i][1] = page == -2 ? __uint_as_float(0x7fc00000u) : 0.0f;
        if (page >= 0 && k0 + n * 128 + r < sq.len) {
          sc[i][0] = __ldg(a.c.ks + h * a.c.ks_st[2] + page * a.c.ks_st[0] + row * a.c.ks_st[1]);
          sc[i][1] = __ldg(a.c.vs + h * a.c.vs_st[2] + page * a.c.vs_st[0] + row * a.c.vs_st[1]);
        }
        // A value row that is not finite makes its key's score NaN instead (0 * NaN in the second
        // product would reach the rows that do not see the key).
        if (!(fabsf(sc[i][1]) < INFINITY)) {
          sc[i][0] = __uint_as_float(0x7fc00000u);
          sc[i][1] = 0.0f;
        }
        if (page == -2 && tid + 96 * i < 128 && k0 + n * 128 + r < sq.len) report(a.err, FA2_ERR_PAGE);
      }
    };
    int eb = EB_MIN;  // exponent field of the largest finite sv so far
    // Scales of tile n, from sc: into its entry, with the tile's exponents.
    auto store_scales = [&](int n) {
      uint32_t top[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (tid + 96 * i < 128) {
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            const uint32_t v = __float_as_uint(sc[i][z]) & 0x7fffffffu;
            if (v < 0x7f800000u) top[z] = max(top[z], v);
          }
        }
      }
      top[0] = __reduce_max_sync(0xffffffffu, top[0]);
      top[1] = __reduce_max_sync(0xffffffffu, top[1]);
      uint32_t* wm = reinterpret_cast<uint32_t*>(smem + C::OFF_MAX) + (n & 1) * 6;
      if (lane < 2) wm[(warp - CH_CONV_WARP) * 2 + lane] = top[lane];
      conv_sync(true);
      const int ek = max(EB_MIN, static_cast<int>(max(wm[0], max(wm[2], wm[4])) >> 23));
      eb = max(eb, static_cast<int>(max(wm[1], max(wm[3], wm[5])) >> 23));
      const int en = n % CH_ENTRIES;
      uint32_t* dst = reinterpret_cast<uint32_t*>(smem + C::OFF_SC) + en * 256;
      const float fk = __uint_as_float(static_cast<uint32_t>(254 + FOLD_SHIFT - ek) << 23);
      const float fv = __uint_as_float(static_cast<uint32_t>(254 + FOLD_SHIFT - eb) << 23);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = tid + 96 * i;
        if (r < 128) {
          dst[r] = FOLD ? split_scale(sc[i][0] * fk) : __float_as_uint(sc[i][0]);
          dst[128 + r] = FOLD ? split_scale(sc[i][1] * fv) : __float_as_uint(sc[i][1] * fv);
        }
      }
      if (tid == 0) {
        uint32_t* head = reinterpret_cast<uint32_t*>(smem + C::OFF_HEAD) + en * 2;
        // 2^(ek - 127 - FOLD_SHIFT): what a folded score is to be multiplied by.
        head[0] = FOLD ? (static_cast<uint32_t>(max(1, ek - FOLD_SHIFT)) << 23) : 0x3f800000u;
        head[1] = static_cast<uint32_t>(eb);
      }
      mbar_arrive(bar(CB_SC + en));
      if (FOLD) conv_sync(true);  // the conversion reads the scales of the others' keys
    };
    auto store_piece = [&](int it, int n, bool is_v, uint32_t dst) {
      const int e = it * CH_CONV_THREADS + tid;
      if (128 * PIECES % CH_CONV_THREADS != 0 && e >= 128 * PIECES) return;
      const int r = e / PIECES, piece = e % PIECES;
      const uint32_t c[4] = {w[it].x, w[it].y, w[it].z, w[it].w};
      uint32_t o[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        o[2 * i] = f16x2_of_e4m3x2(static_cast<uint16_t>(c[i]));
        o[2 * i + 1] = f16x2_of_e4m3x2(static_cast<uint16_t>(c[i] >> 16));
      }
      if constexpr (FOLD) {
        const uint32_t s = reinterpret_cast<const uint32_t*>(smem + C::OFF_SC)[(n % CH_ENTRIES) * 256 + (is_v ? 128 : 0) + r];
        const uint32_t hi = __byte_perm(s, s, 0x1010), lo = __byte_perm(s, s, 0x3232);
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = hfma2(o[i], hi, hmul2(o[i], lo));
      }
      // 64 columns a 128-byte row, 16-byte parts xor-ed with the row's number (128-byte swizzle).
      // The upper half of a row stores its parts in the other order: no two lanes meet in a bank.
      const uint32_t row = dst + (piece >> 2) * C::CHUNK + r * 128;
      const uint32_t flip = D > 64 ? static_cast<uint32_t>(piece >> 2) : 0u;
      const uint32_t part = (static_cast<uint32_t>(piece & 3) * 2) ^ static_cast<uint32_t>(r & 7);
      const bool f = flip != 0;
      fa2::st_shared_v4(row + ((part ^ flip) << 4), f ? o[4] : o[0], f ? o[5] : o[1], f ? o[6] : o[2], f ? o[7] : o[3]);
      fa2::st_shared_v4(row + ((part ^ flip ^ 1u) << 4), f ? o[0] : o[4], f ? o[1] : o[5], f ? o[2] : o[6], f ? o[3] : o[7]);
    };

    // Tile i is converted from registers while tile i + 1 is fetched into them, piece by piece; the
    // page numbers of tile i + 2 are on their way.
    const int total = 2 * tiles;
    bool cur_v = false, next_v, then_v = false;
    int cur_n = 0, next_n, then_n = 0, pg_next, pg_then = 0;
    {
      const int pg = pages_of(0);
#pragma unroll
      for (int it = 0; it < N_IT; ++it) fetch_piece(it, 0, false, pg);
      fetch_scales(0, pg);
    }
    order.at(1, next_v, next_n);
    pg_next = pages_of(next_n);
    for (int i = 0; i < total; ++i) {
      if (i + 2 < total) {
        order.at(i + 2, then_v, then_n);
        pg_then = pages_of(then_n);
      }
      const int slot = i % CH_SLOTS;
      const uint32_t ph = static_cast<uint32_t>(i / CH_SLOTS) & 1u;
      ok = conv_sync(mbar_wait_warp(bar(CB_EMPTY + slot), ph ^ 1u, timeout, a.err));
      if (!ok) break;
      if (!cur_v) store_scales(cur_n);
      const uint32_t dst = sbase + C::OFF_RING + slot * C::TILE;
      if (i + 1 < total) {
#pragma unroll
        for (int it = 0; it < N_IT; ++it) {
          store_piece(it, cur_n, cur_v, dst);
          fetch_piece(it, next_n, next_v, pg_next);
        }
        if (!next_v) fetch_scales(next_n, pg_next);
      } else {
#pragma unroll
        for (int it = 0; it < N_IT; ++it) store_piece(it, cur_n, cur_v, dst);
      }
      fa2::fence_proxy_async_smem();
      mbar_arrive(bar(CB_FULL + slot));
      cur_v = next_v;
      cur_n = next_n;
      next_v = then_v;
      next_n = then_n;
      pg_next = pg_then;
    }
  } else if (warp == CH_MMA_WARP) {
    // -------------------------------------------------------------- products
    fa2::reg_dealloc<CH_REGS_OTHER>();
    if (lane == 0) {
      constexpr uint32_t idesc_qk = fa2::idesc_f16(false, 128, 128, false);
      constexpr uint32_t idesc_pv = fa2::idesc_f16(false, 128, D, true);
      const uint64_t dq = fa2::sdesc_sw128(sbase + C::OFF_Q, 16, 1024);
      const uint64_t dk = fa2::sdesc_sw128(sbase + C::OFF_RING, 16, 1024);
      const uint64_t dv = fa2::sdesc_sw128(sbase + C::OFF_RING, C::CHUNK, 1024);
      auto wait = [&](int i, uint32_t parity) -> bool { return mbar_wait(bar(i), parity, timeout, a.err); };
      auto qk = [&](int t, int slot) {
        const uint64_t qd = dq + static_cast<uint64_t>(((dual ? 0 : t) * C::TILE) >> 4);
        const uint64_t kd = dk + static_cast<uint64_t>((slot * C::TILE) >> 4);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint64_t off = static_cast<uint64_t>(((kk >> 2) * C::CHUNK + (kk & 3) * 32) >> 4);
          mma_ss(tmem + t * 128, qd + off, kd + off, idesc_qk, kk > 0 ? 1u : 0u);
        }
        mma_commit(bar(CB_S + t));
      };
      // P' of tile t comes in two parts: 96 keys, then 32.
      auto pv = [&](int t, int slot, bool acc, uint32_t parity) -> bool {
        const uint64_t vd = dv + static_cast<uint64_t>((slot * C::TILE) >> 4);
        if (!wait(CB_P + t, parity)) return false;
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < 6; ++kk) {
          mma_ts(tmem + C::TMEM_O + t * D, tmem + t * 128 + 64 + kk * 8, vd + static_cast<uint64_t>((kk * 16 * 128) >> 4),
                 idesc_pv, (acc || kk > 0) ? 1u : 0u);
        }
        if (!wait(CB_PL + t, parity)) return false;
        tc_fence_after();
#pragma unroll
        for (int kk = 6; kk < 8; ++kk) {
          mma_ts(tmem + C::TMEM_O + t * D, tmem + t * 128 + 64 + kk * 8, vd + static_cast<uint64_t>((kk * 16 * 128) >> 4),
                 idesc_pv, 1u);
        }
        return true;
      };
      int at = 0;  // place in the tile order
      auto take = [&](int i) -> bool {
        if (!wait(CB_FULL + i % CH_SLOTS, static_cast<uint32_t>(i / CH_SLOTS) & 1u)) return false;
        tc_fence_after();
        return true;
      };
      auto drop = [&](int i) { mma_commit(bar(CB_EMPTY + i % CH_SLOTS)); };
      ok = wait(CB_Q + 0, 0) && (dual || wait(CB_Q + 1, 0));
      if (ok && dual) {
        for (int t = 0; ok && t < order.ahead; ++t) {
          ok = take(at);
          if (ok) {
            qk(t, at % CH_SLOTS);
            drop(at++);
          }
        }
        for (int n = 0; ok && n < tiles; ++n) {
          const int t = n & 1;
          ok = take(at) && pv(t, at % CH_SLOTS, n > 1, static_cast<uint32_t>(n >> 1) & 1u);
          if (!ok) break;
          if (n + 2 >= tiles) mma_commit(bar(CB_O + t));
          drop(at++);
          if (n + order.ahead < tiles) {
            ok = take(at);
            if (!ok) break;
            qk((n + order.ahead) & 1, at % CH_SLOTS);
            drop(at++);
          }
        }
      } else if (ok) {
        ok = take(at);
        if (ok) {
          qk(0, 0);
          qk(1, 0);
          drop(at++);
        }
        for (int n = 0; ok && n < tiles; ++n) {
          const bool more = n + 1 < tiles;
          const uint32_t parity = static_cast<uint32_t>(n) & 1u;
          const int iv = at, ik = at + 1;
          for (int t = 0; t < 2 && ok; ++t) {
            ok = (t > 0 || take(iv)) && pv(t, iv % CH_SLOTS, n > 0, parity);
            if (!ok) break;
            if (!more) mma_commit(bar(CB_O + t));
            if (t == 1) drop(iv);
            if (more) {
              ok = t > 0 || take(ik);
              if (!ok) break;
              qk(t, ik % CH_SLOTS);
              if (t == 1) drop(ik);
            }
          }
          at += 2;
        }
      }
      // Every product has retired before TMEM is given back.
      mma_commit(bar(CB_DONE));
      if (!mbar_wait(bar(CB_DONE), 0, CH_TIMEOUT, nullptr)) ok = false;
    }
    __syncwarp();
  } else {
    // -------------------------------------------------------------- softmax: one thread a row
    fa2::reg_alloc<CH_REGS_SM>();
    const int t = warp >> 2, q = warp & 3;
    const int r = q * 32 + lane;  // row of the tile
    const int row = row0 + (dual ? 0 : t * 128) + r;
    const bool have = row < row0 + n_rows;
    const uint32_t lane_addr = static_cast<uint32_t>(q * 32) << 16;
    const uint32_t tS = tmem + t * 128 + lane_addr, tP = tS + 64, tO = tmem + C::TMEM_O + t * D + lane_addr;

    // Q: this row in fp16, times the power of two that brings its largest value below 2^15.
    float row_sc = a.qk_scale;
    if (!dual || t == 0) {
      uint32_t w[D / 2];
      uint32_t top = 0;
      const uint16_t* src = q_row(a, sq, b, h, have ? row : row0);
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        const uint4 v = have ? __ldg(reinterpret_cast<const uint4*>(src) + i) : make_uint4(0, 0, 0, 0);
        w[4 * i] = v.x;
        w[4 * i + 1] = v.y;
        w[4 * i + 2] = v.z;
        w[4 * i + 3] = v.w;
      }
#pragma unroll
      for (int i = 0; i < D / 2; ++i) {
        const float2 v = float2_of_x2<BF16>(w[i]);
        top = max(top, max(__float_as_uint(v.x) & 0x7fffffffu, __float_as_uint(v.y) & 0x7fffffffu));
      }
      const int e = row_exponent(top);
      const float f = pow2f(14 - e);
      row_sc = a.qk_scale * pow2f(max(-126, e - 14));
      const uint32_t dst = sbase + C::OFF_Q + t * C::TILE + r * 128;
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 v = float2_of_x2<BF16>(w[4 * i + j]);
          o[j] = x2_of_floats<false>(v.x * f, v.y * f);
        }
        fa2::st_shared_v4(dst + (i >> 3) * C::CHUNK + (((i & 7) ^ (r & 7)) << 4), o[0], o[1], o[2], o[3]);
      }
      fa2::fence_proxy_async_smem();
      mbar_arrive(bar(CB_Q + t));
    } else {  // the same rows as tile 0's: only their scale
      uint32_t top = 0;
      const uint16_t* src = q_row(a, sq, b, h, have ? row : row0);
      for (int i = 0; i < D / 8; ++i) {
        const uint4 v = have ? __ldg(reinterpret_cast<const uint4*>(src) + i) : make_uint4(0, 0, 0, 0);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f2 = float2_of_x2<BF16>(w[j]);
          top = max(top, max(__float_as_uint(f2.x) & 0x7fffffffu, __float_as_uint(f2.y) & 0x7fffffffu));
        }
      }
      row_sc = a.qk_scale * pow2f(max(-126, row_exponent(top) - 14));
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
      const uint32_t head_addr = sbase + C::OFF_HEAD + en * 8;
      const uint32_t sc_addr = sbase + C::OFF_SC + en * 1024;
      float k_sc;
      int eb_new;
      asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=f"(k_sc), "=r"(eb_new) : "r"(head_addr));
      const float sc = row_sc * k_sc;
      const int col0 = k0 + n * 128;
      const bool masked = col0 + 127 > lim_all;
      const int lim = lim_row - col0;

      uint32_t s[4][32];
      fa2::tmem_ld128(tS, s[0], s[1], s[2], s[3]);
      fa2::tmem_wait_ld();
#pragma unroll
      for (int c = 0; c < 4; ++c) fa2::reg_fence32(s[c]);
      if constexpr (!FOLD) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            float k[4];
            asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];"
                         : "=f"(k[0]), "=f"(k[1]), "=f"(k[2]), "=f"(k[3]) : "r"(sc_addr + (c * 32 + i) * 4));
#pragma unroll
            for (int j = 0; j < 4; ++j) s[c][i + j] = __float_as_uint(__uint_as_float(s[c][i + j]) * k[j]);
          }
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
    float* area = reinterpret_cast<float*>(smem + C::OFF_RING);  // [D / 4][128] float4
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
