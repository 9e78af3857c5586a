// Attention over the 8-bit paged cache for many rows (chunks of prompts): tcgen05 products.
//
// The floor is the tensor cores' (4 D operations a score). What sets the step is a row tile's chain of
// scores, softmax, PV and the next scores, which the other tile fills in part: tensor pipe 45%, issue
// slots 49% and exponentials 47% busy, none of them full. Longer chains cost at once: an eighth of the
// exponentials on the FMA pipe made it 5% slower. Measured: 2 chunks of 512 tokens over 16384 keys, 32
// heads of 128 over 8, 271 GFLOP, 289 us in short runs of a graph (938 TFLOP/s, 0.57 of the bf16 peak), 318 us
// as ordinary calls in a row (850 TFLOP/s, at lower clocks), in fp16 350 us (a third operand of Q, shorter
// rings); 20 rows a kv head in place of 2048 51 us, of which the bytes are 11. A step of 256 rows and 128 keys
// takes 2.35 us, a piece of work 10 us beside its steps.
//
// A CTA owns 256 rows (queries x heads of a group) as two 128-row tiles that take turns: while one
// tile's scores go through the softmax, the tensor core works on the other. With 128 rows or fewer both tiles hold the same rows and take
// every other 128-key tile, merged at the end. One CTA an SM works through the pieces of its share of
// the work (see Line); the rings and barriers carry over from one piece to the next.
//
// QK^T runs on the codes as they are stored: K is an e4m3 operand, and a row of Q, times the power
// of two that brings its largest value into [128, 256), is the sum of an e4m3 operand and one (bf16) or
// two (fp16) e5m2 operands, each the rounding of what the ones before leave. From 2^-6 on the first one has
// 4 significant bits and leaves at most 8 units of the last place of a bf16 value, or 64 of an fp16 value:
// whole numbers up to 8 have 3 significant bits, as e5m2 has, and of those up to 64 a second e5m2 term takes
// the at most 4 units that the first leaves. So every value within 2^13 of its row's largest is exact.
// A smaller one is off by at most 2^-14 (bf16) or 2^-17 (fp16: half of e5m2's smallest step), which is
// 2^-21 or 2^-24 of the largest. (With e4m3 for all terms, whose smallest step is 2^-9, exactness ended
// 2^6 to 2^10 below the largest.) 8-bit products run at twice the rate of 16-bit ones, so the second
// operand costs nothing over converting K to fp16 (64 instructions less for each 16 values).
//
// PV runs on fp16: P' needs 11 bits. V is converted on its way into shared memory. Its row scales:
// bf16 queries fold them into that conversion (code * s_j in fp16, one rounding of at most 2^-11, an
// eighth of the output's half step); for fp16 queries, whose half step is 2^-11 itself, the codes
// stay exact and each probability is multiplied by its key's scale in fp32. K's scales multiply the
// scores. From the tile on where a piece's value scales lie more than 2^WIDE apart, nothing is folded and
// rows have exponents of their own (kv8_attn.cuh). That costs ordinary tiles up to 2% (the chunks above with
// heads of 64 dims: 245 to 250 us, of 128: 300 to 301).
//
// Warps 0-3 / 4-7: softmax of tile 0 / 1, one thread a row (scores and P' live in TMEM, P' feeds the
// second product from there). Warps 8-11: convert V. Warp 12: issues the products. Warps 13 and 14:
// bring K and V in from their pages by asynchronous copies. Warp 15: walks the CTA's share of the
// work and hands the pieces out. Every loop but the softmax's is kept rolled: the roles share the
// instruction caches, and code that runs once costs a fetch from far away for each eight
// instructions (an unrolled start of a piece took 12,000 cycles).
#pragma once

#include "kv8_attn.cuh"

namespace fa2kv {

using fa2::mbar_arrive;
using fa2::mbar_init;
using fa2::mbar_wait_warp;
using fa2::smem_u32;
using fa2::tc_fence_after;
using fa2::tc_fence_before;

constexpr int CH_THREADS = 512;
constexpr int CH_CONV_WARP = 8, CH_CONV_THREADS = 128;
constexpr int CH_MMA_WARP = 12, CH_K_WARP = 13, CH_V_WARP = 14, CH_PLAN_WARP = 15;
constexpr int CH_VSLOTS = 2;   // ring of V (fp16) tiles
constexpr int CH_ENTRIES = 8;  // ring of the tiles' scales
constexpr int CH_PIECES = 4;   // ring of pieces
constexpr int CH_READERS = 15; // warps that read a piece
constexpr int CH_REGS = 128;   // a thread at launch, then by warpgroup:
constexpr int CH_REGS_SM = 176, CH_REGS_CONV = 88, CH_REGS_MMA = 72;
static_assert(256 * CH_REGS_SM + 128 * CH_REGS_CONV + 128 * CH_REGS_MMA <= CH_THREADS * CH_REGS, "register split");
constexpr long long CH_TIMEOUT = 2000000000ll;
constexpr int FOLD_SHIFT = 6;   // folded scales: the largest lies in [2^6, 2^7), times 448 below 2^16

template <int D, bool BF16>
struct Ch {
  static constexpr int TERMS = BF16 ? 2 : 3;          // operands of Q: e4m3, then e5m2
  static constexpr int KSLOTS = BF16 ? 3 : 2;         // rings of K codes ...
  static constexpr int RAW = BF16 ? 2 : 1;            // ... and V codes
  static constexpr int KSTEPS = D > 32 ? D / 32 : 1;  // 32-wide steps of QK^T (D = 16: zeros beyond)
  static constexpr int CODES = 128 * 128;             // bytes of a tile of codes: 128-byte rows
  static constexpr int CHUNKS = D > 64 ? D / 64 : 1;  // 64-column pieces of an fp16 tile
  static constexpr int CHUNK = 128 * 128;
  static constexpr int VTILE = CHUNKS * CHUNK;
  static constexpr int OFF_Q = 0;  // [tile][term]
  static constexpr int OFF_K = 2 * TERMS * CODES;
  static constexpr int OFF_V = OFF_K + KSLOTS * CODES;
  static constexpr int OFF_RAW = OFF_V + CH_VSLOTS * VTILE;
  static constexpr int OFF_SC = OFF_RAW + RAW * CODES;          // [entry][2][128] words
  static constexpr int OFF_HEAD = OFF_SC + CH_ENTRIES * 1024;   // [entry] exponent field of sv, or -1: each row its own
  static constexpr int OFF_MAX = OFF_HEAD + CH_ENTRIES * 4;     // [2][4 warps] largest and smallest sv
  static constexpr int OFF_ML = OFF_MAX + 64;                   // [2][128]: tile 1's max and sum, for the merge
  static constexpr int OFF_QS = OFF_ML + 1024;                  // [2][128]: the rows' score factors
  static constexpr int OFF_PIECE = OFF_QS + 1024;               // [piece] 12 words
  static constexpr int OFF_BAR = OFF_PIECE + CH_PIECES * 48;
  static constexpr int OFF_TMEM = OFF_BAR + 384;
  static constexpr int OFF_STOP = OFF_TMEM + 8;
  static constexpr int SMEM = OFF_TMEM + 16 + 1024;             // and slack to align the base
  // The merge of two tiles of the same rows: 64 columns of tile 1's O at a time, where its Q would be.
  static constexpr int COLS = D < 64 ? D : 64;
  static_assert(128 * COLS * 4 <= TERMS * CODES, "merge area");
  static_assert(SMEM <= 227 * 1024, "shared memory");
  static constexpr int TMEM_O = 256;
};

enum ChBar { CB_Q = 0, CB_S = 2, CB_P = 4, CB_PL = 6, CB_O = 8, CB_KF = 10, CB_KE = CB_KF + 3, CB_VF = CB_KE + 3,
             CB_VE = CB_VF + CH_VSLOTS, CB_RF = CB_VE + CH_VSLOTS, CB_RE = CB_RF + 2, CB_SC = CB_RE + 2,
             CB_X = CB_SC + CH_ENTRIES, CB_Y, CB_PF, CB_PE = CB_PF + CH_PIECES, CB_DONE = CB_PE + CH_PIECES, CB_COUNT };
static_assert(CB_COUNT * 8 <= 384, "barriers");

// A shared-memory descriptor's upper word (128-byte swizzle, 8-row groups 1024 bytes apart), and the
// lower one of a tile at `addr` with `lbo` bytes between 64-column pieces.
constexpr uint32_t DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lbo) { return ((addr >> 4) & 0x3fffu) | ((lbo >> 4) << 16); }

// The issuing warp runs converged and its lane 0 issues (`lead`, a predicate and no branch): the
// descriptors stay in uniform registers, which the products take. Issued inside a branch of one lane
// every operand is moved there first, and a step of the loop took 1.3 to 2 times as long.
// D[tmem] (+)= A[smem] * B[smem], 8-bit floats by `idesc` (32 wide steps), fp32 sums. Operands: lower descriptor words.
__device__ __forceinline__ void mma_f8(uint32_t lead, uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
      "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(add), "r"(DESC_HI), "r"(lead)
      : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem], both fp16 (16 wide steps).
__device__ __forceinline__ void mma_f16_ts(uint32_t lead, uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc, uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 db;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %6, 0;\n\tmov.b64 db, {%2, %5};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "r"(b_lo), "r"(idesc), "r"(add), "r"(DESC_HI), "r"(lead)
      : "memory");
}
// Arrives on `bar` once all products issued so far have completed.
__device__ __forceinline__ void commit_to(uint32_t lead, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(lead)
      : "memory");
}
// Instruction descriptor of kind::f8f6f4: fp32 D, A in e4m3 (type code 0) or e5m2 (1), B in e4m3, both
// K-major.
__host__ __device__ constexpr uint32_t idesc_f8(int M, int N, bool a_e5m2) {
  return (1u << 4) | (a_e5m2 ? 1u << 7 : 0u) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
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

// The four converting warps meet; false where one of them gave up, in all of them alike.
__device__ __forceinline__ bool conv_sync(bool ok) {
  uint32_t bad = ok ? 0u : 1u;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %0, 0;\n\t"
      "bar.red.or.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "+r"(bad)::"memory");
  return bad == 0;
}

__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), "r"(v[0]), "r"(v[1]),
               "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
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
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x) >> 5, 0), lane = threadIdx.x & 31;
  const long long timeout = a.timeout > 0 ? a.timeout : CH_TIMEOUT;
  // Not zero once a wait of this CTA has run out: the others' waits end too. (Not the caller's error word:
  // that one may hold a refused page or length, of this call or an earlier one, which stops nobody.)
  int* const stop = reinterpret_cast<int*>(smem + C::OFF_STOP);
  allow_next();

  if (warp == 0) {
    if (lane == 0) *stop = 0;
    auto count_of = [&](int i) -> uint32_t {
      if (i < CB_S) return 128;                     // a tile's softmax threads: Q is written
      if (i < CB_P) return 1;                       // products' commits
      if (i < CB_O) return 128;                     // P', in two parts
      if (i < CB_KF) return 1;
      if (i < CB_KE) return 32;                     // the copying warp
      if (i < CB_VF) return 1;
      if (i < CB_VE) return CH_CONV_THREADS;
      if (i < CB_RF) return 1;
      if (i < CB_RE) return 32;
      if (i < CB_X) return CH_CONV_THREADS;         // CB_RE, CB_SC
      if (i < CB_PF) return 128;                    // CB_X, CB_Y
      if (i < CB_PE) return 1;
      return i < CB_DONE ? CH_READERS : 1;
    };
    for (int i = lane; i < CB_COUNT; i += 32) mbar_init(bar(i), count_of(i));
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

  auto wait_warp = [&](int i, uint32_t parity) -> bool { return mbar_wait_warp(bar(i), parity, timeout, stop); };
  auto piece_at = [&](int i) -> volatile int* {
    return reinterpret_cast<volatile int*>(smem + C::OFF_PIECE + (i % CH_PIECES) * 48);
  };
  // The next piece of this CTA's share, for a whole warp; false after the last one, or on a time-out.
  int piece_n = 0;
  auto next_piece = [&](Piece& o) -> bool {
    if (!wait_warp(CB_PF + piece_n % CH_PIECES, static_cast<uint32_t>(piece_n / CH_PIECES) & 1u)) {
      ok = false;
      return false;
    }
    volatile int* w = piece_at(piece_n);
    o.sq.n_q = w[0];
    o.sq.q0 = w[1];
    o.sq.len = w[2];
    o.sq.off = w[3];
    o.b = w[4];
    o.h = w[5];
    o.rb = w[6];
    o.t0 = w[7];
    o.tiles = w[8];
    o.kend = w[9];
    o.slot = w[10];
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(CB_PE + piece_n % CH_PIECES));
    ++piece_n;
    return o.tiles > 0;
  };

  if (warp == CH_PLAN_WARP) {
    // -------------------------------------------------------------- the pieces of the share
    fa2::reg_dealloc<CH_REGS_MMA>();
    const int worker = static_cast<int>(blockIdx.x);
    Pieces pieces;
    pieces.begin(a, worker);
    Piece o{};
    bool more = true;
    for (int i = 0; ok && more; ++i) {
      more = pieces.next(a, o);
      if (!wait_warp(CB_PE + i % CH_PIECES, (static_cast<uint32_t>(i / CH_PIECES) & 1u) ^ 1u)) {
        ok = false;
        break;
      }
      if (lane == 0) {
        volatile int* w = piece_at(i);
        w[0] = o.sq.n_q;
        w[1] = o.sq.q0;
        w[2] = o.sq.len;
        w[3] = o.sq.off;
        w[4] = o.b;
        w[5] = o.h;
        w[6] = o.rb;
        w[7] = o.t0;
        w[8] = more ? o.tiles : 0;
        w[9] = o.kend;
        w[10] = o.slot;
        mbar_arrive(bar(CB_PF + i % CH_PIECES));
      }
      __syncwarp();
      const int first = o.rb * 256, end = more ? min(first + 256, o.sq.n_q * a.group) : 0;
      for (int r = first + lane; r < end; r += 32) {  // its queries, towards L2
        const uint16_t* src = q_row(a, o.sq, o.b, o.h, r);
        asm volatile("prefetch.global.L2 [%0];" ::"l"(src));
        if constexpr (D > 64) asm volatile("prefetch.global.L2 [%0];" ::"l"(src + 64));
      }
    }
  } else if (warp == CH_K_WARP || warp == CH_V_WARP) {
    // -------------------------------------------------------------- codes: pages -> shared memory
    fa2::reg_dealloc<CH_REGS_MMA>();
    const bool is_v = warp == CH_V_WARP;
    constexpr int PIECES = D / 16;                              // 16-byte pieces of a row
    constexpr int ROWS = 32 / PIECES < 16 ? 32 / PIECES : 16;   // rows a copy instruction covers
    constexpr int COPIES = 16 / ROWS;                           // for 16 rows, which lie in one page
    const int my_row = lane / PIECES, my_piece = lane % PIECES;
    const bool on = my_row < 16;                                // (D = 16: half the lanes)
    // K's 16-byte parts are xor-ed with the row's number (128-byte swizzle), V's change halves from
    // row to row (eight converting lanes read two rows).
    uint32_t to[COPIES];
#pragma unroll
    for (int j = 0; j < COPIES; ++j) {
      const int r = j * ROWS + my_row;
      to[j] = r * 128 + ((my_piece ^ (is_v ? (r & 1) << 2 : r & 7)) << 4);
    }
    const int ps = a.c.page_size;
    const bool small = ps < 128;
    const int row_st = is_v ? a.c.v_row : a.c.k_row, page16 = is_v ? a.c.v_page16 : a.c.k_page16;
    const int64_t step = static_cast<int64_t>(ROWS) * row_st;
    const int ring = is_v ? C::RAW : C::KSLOTS, full = is_v ? CB_RF : CB_KF, empty = is_v ? CB_RE : CB_KE;
    const uint32_t ring_at = sbase + (is_v ? C::OFF_RAW : C::OFF_K);
    if (D < 32 && !is_v) {  // the second half of the only 32-wide step stays zero
      for (int i = lane; i < C::KSLOTS * 128 * 8; i += 32) {
        *reinterpret_cast<uint4*>(smem + C::OFF_K + i * 16) = make_uint4(0, 0, 0, 0);
      }
      __syncwarp();
    }
    auto landed = [&](int u) {  // this lane's copies of tile u have
      if (!is_v) fa2::fence_proxy_async_smem();  // K is read by the tensor core
      mbar_arrive(bar(full + u % ring));
    };
    int base = 0;  // tiles so far
    Piece o{};
    while (next_piece(o)) {
      const int k0 = o.t0 * 128;
      const int* bt = a.bt + o.b * a.bt_stride;
      const uint8_t* head = (is_v ? a.c.v + static_cast<int64_t>(o.h) * a.c.v_head : a.c.k + static_cast<int64_t>(o.h) * a.c.k_head) + my_piece * 16;
      // Pages of a tile: lane l has the one of rows 16 l (or of them all). -1: none, or refused.
      auto page_for = [&](int n) -> int {
        const int key = k0 + n * 128 + 16 * lane;
        if (n >= o.tiles || lane >= 8 || key >= o.sq.len) return -1;
        const int pg = __ldg(bt + page_of(a.c, key));
        return static_cast<unsigned>(pg) < static_cast<unsigned>(a.c.num_pages) ? pg : -1;
      };
      int pages = page_for(0);
      for (int n = 0; n < o.tiles; ++n) {
        const int u = base + n;
        const int pages_next = page_for(n + 1);
        if (!wait_warp(empty + u % ring, (static_cast<uint32_t>(u / ring) & 1u) ^ 1u)) {
          ok = false;
          break;
        }
        const uint32_t slot = ring_at + (u % ring) * C::CODES;
        const int keys = o.sq.len - (k0 + n * 128), first = small ? 0 : (k0 + n * 128) % ps;
#pragma unroll 1
        for (int g = 0; g < 8; ++g) {
          const int page = __shfl_sync(0xffffffffu, pages, g);
          const int row = (small ? (g * 16) & (ps - 1) : first + g * 16) + my_row;
          const uint8_t* p = head + (static_cast<int64_t>(max(page, 0)) * page16 << 4) + static_cast<int64_t>(row) * row_st;
#pragma unroll
          for (int j = 0; j < COPIES; ++j) {
            const bool in = page >= 0 && g * 16 + j * ROWS + my_row < keys;
            if (on) cp_async16(slot + g * 2048 + to[j], in ? p : head, in);  // zeros where there is nothing
            p += step;
          }
        }
        cp_async_commit();
        if (C::RAW == 1 && is_v) {
          cp_async_wait<0>();
          landed(u);
        } else if (n > 0) {
          cp_async_wait<1>();
          landed(u - 1);
        }
        pages = pages_next;
      }
      if (!ok) break;
      if (!(C::RAW == 1 && is_v)) {
        cp_async_wait<0>();
        landed(base + o.tiles - 1);
      }
      base += o.tiles;
    }
    cp_async_wait<0>();
  } else if (warp >= CH_CONV_WARP && warp < CH_MMA_WARP) {
    // -------------------------------------------------------------- scales, V codes -> fp16
    fa2::reg_dealloc<CH_REGS_CONV>();
    const int tid = static_cast<int>(threadIdx.x) - CH_CONV_WARP * 32;
    // Thread tid has piece tid % PC of the rows tid / PC + V_ROWS * it, 64 columns at a time, so that
    // eight neighbouring lanes write two rows and do not meet in a bank.
    constexpr int PC = D / 16 < 4 ? D / 16 : 4;
    constexpr int V_ROWS = CH_CONV_THREADS / PC, V_IT = 128 / V_ROWS;
    static_assert(V_ROWS % 8 == 0, "a thread's rows have the same swizzle");
    const int v_row = tid / PC, v_piece = tid % PC;
    const uint32_t part = (static_cast<uint32_t>(v_piece) * 2) ^ static_cast<uint32_t>(v_row & 7);
    int base = 0;
    Piece o{};
    auto next = [&]() -> int { return next_piece(o) ? 1 : ok ? 0 : -1; };
    ok = pieces_together(next, conv_sync, [&]() -> bool {
      const int k0 = o.t0 * 128;
      const int* bt = a.bt + o.b * a.bt_stride;
      // Key tid of a tile: its page (-1: no key, -2: refused), then its scales.
      auto page_for = [&](int n) -> int {
        const int key = k0 + n * 128 + tid;
        if (n >= o.tiles || key >= o.sq.len) return -1;
        const int pg = __ldg(bt + page_of(a.c, key));
        return static_cast<unsigned>(pg) < static_cast<unsigned>(a.c.num_pages) ? pg : -2;
      };
      float sk = 0.0f, sv = 0.0f;
      auto fetch_scales = [&](int n, int page) {
        const int key = k0 + n * 128 + tid, row = key - page_of(a.c, key) * a.c.page_size;
        sk = sv = 0.0f;
        if (page >= 0) {
          sk = __ldg(a.c.ks + static_cast<int64_t>(o.h) * a.c.ks_head + static_cast<int64_t>(page) * a.c.ks_page + static_cast<int64_t>(row) * a.c.ks_row);
          sv = __ldg(a.c.vs + static_cast<int64_t>(o.h) * a.c.vs_head + static_cast<int64_t>(page) * a.c.vs_page + static_cast<int64_t>(row) * a.c.vs_row);
        } else if (page == -2) {  // queries that see a key of a refused page get NaN
          sk = __uint_as_float(0x7fc00000u);
          report(a.err, FA2_ERR_PAGE);
        }
      };
      int eb = EB_MIN;  // exponent field of the largest finite sv so far ...
      uint32_t low = 0xffffffffu;  // ... and the smallest but zero, its bits - 1
      bool wide = false;  // too far apart: from here on rows have exponents of their own, and V is not folded
      fetch_scales(0, page_for(0));
      int page = page_for(1);
#pragma unroll 1
      for (int n = 0; n < o.tiles; ++n) {
        const int u = base + n, en = u % CH_ENTRIES;
        // The scales, and the exponent that sv is relative to. A value row that is not finite makes its
        // key's score NaN instead (0 * NaN in the second product would reach the rows that do not see
        // the key).
        if (!(fabsf(sv) < INFINITY)) {
          sk = __uint_as_float(0x7fc00000u);
          sv = 0.0f;
        }
        const uint32_t bits = __float_as_uint(sv) & 0x7fffffffu;
        const uint32_t top = __reduce_max_sync(0xffffffffu, bits), least = __reduce_min_sync(0xffffffffu, bits - 1u);
        const uint32_t wm = sbase + C::OFF_MAX + (u & 1) * 32;
        if (lane == 0) {
          asm volatile("st.shared.b32 [%0], %1;" ::"r"(wm + (warp - CH_CONV_WARP) * 4), "r"(top) : "memory");
          asm volatile("st.shared.b32 [%0], %1;" ::"r"(wm + 16 + (warp - CH_CONV_WARP) * 4), "r"(least) : "memory");
        }
        conv_sync(true);
        uint32_t tops[4], lows[4];
        asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(tops[0]), "=r"(tops[1]), "=r"(tops[2]), "=r"(tops[3]) : "r"(wm) : "memory");
        asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(lows[0]), "=r"(lows[1]), "=r"(lows[2]), "=r"(lows[3]) : "r"(wm + 16) : "memory");
        eb = max(eb, static_cast<int>(max(max(tops[0], tops[1]), max(tops[2], tops[3])) >> 23));
        low = min(low, min(min(lows[0], lows[1]), min(lows[2], lows[3])));
        wide = wide || too_wide(eb, low);
        const float fv = __uint_as_float(static_cast<uint32_t>(254 + FOLD_SHIFT - eb) << 23);
        uint32_t* entry = reinterpret_cast<uint32_t*>(smem + C::OFF_SC) + en * 256;
        entry[tid] = __float_as_uint(sk);
        entry[128 + tid] = wide ? __float_as_uint(sv) : FOLD ? split_scale(sv * fv) : __float_as_uint(sv * fv);
        if (tid == 0) reinterpret_cast<int*>(smem + C::OFF_HEAD)[en] = wide ? -1 : eb;
        mbar_arrive(bar(CB_SC + en));
        fetch_scales(n + 1, page);  // on their way while V is converted
        page = page_for(n + 2);
        const bool go = wait_warp(CB_RF + u % C::RAW, static_cast<uint32_t>(u / C::RAW) & 1u) &&
                        wait_warp(CB_VE + u % CH_VSLOTS, (static_cast<uint32_t>(u / CH_VSLOTS) & 1u) ^ 1u);
        if (!conv_sync(go)) return false;  // (also: the conversion reads the scales of the others' keys)
        const uint8_t* src = smem + C::OFF_RAW + (u % C::RAW) * C::CODES + v_row * 128;
        uint8_t* dst = smem + C::OFF_V + (u % CH_VSLOTS) * C::VTILE + v_row * 128;
        const uint32_t* vsc = entry + 128 + v_row;
#pragma unroll 4
        for (int i = 0; i < V_IT * C::CHUNKS; ++i) {
          const int it = i % V_IT, half = i / V_IT;
          const uint4 w = *reinterpret_cast<const uint4*>(src + it * V_ROWS * 128 + (((half * 4 + v_piece) ^ ((v_row & 1) << 2)) << 4));
          const uint32_t c[4] = {w.x, w.y, w.z, w.w};
          uint32_t y[8];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            y[2 * j] = f16x2_of_e4m3x2(static_cast<uint16_t>(c[j]));
            y[2 * j + 1] = f16x2_of_e4m3x2(static_cast<uint16_t>(c[j] >> 16));
          }
          if constexpr (FOLD) {
            const uint32_t ws = wide ? 0x3c00u : vsc[it * V_ROWS];  // (one: the codes as they are)
            const uint32_t hi = __byte_perm(ws, ws, 0x1010), lo = __byte_perm(ws, ws, 0x3232);
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = hfma2(y[j], hi, hmul2(y[j], lo));
          }
          uint8_t* row = dst + it * V_ROWS * 128 + half * C::CHUNK;
          *reinterpret_cast<uint4*>(row + (part << 4)) = make_uint4(y[0], y[1], y[2], y[3]);
          *reinterpret_cast<uint4*>(row + ((part ^ 1u) << 4)) = make_uint4(y[4], y[5], y[6], y[7]);
        }
        mbar_arrive(bar(CB_RE + u % C::RAW));
        fa2::fence_proxy_async_smem();
        mbar_arrive(bar(CB_VF + u % CH_VSLOTS));
      }
      base += o.tiles;
      return true;
    });
  } else if (warp == CH_MMA_WARP) {
    // -------------------------------------------------------------- products
    fa2::reg_dealloc<CH_REGS_MMA>();
    constexpr uint32_t idesc_qk = idesc_f8(128, 128, false), idesc_qk5 = idesc_f8(128, 128, true);
    constexpr uint32_t idesc_pv = fa2::idesc_f16(false, 128, D, true);
    const uint32_t dq = desc_lo(sbase + C::OFF_Q, 16), dk = desc_lo(sbase + C::OFF_K, 16);
    const uint32_t dv = desc_lo(sbase + C::OFF_V, C::CHUNK);
    const uint32_t lead = lane == 0 ? 1u : 0u;
    uint32_t p_at = 0, q_at = 0;  // parities of the next P' and Q, bit t: tile t's
    int base = 0;
    Piece o{};
    while (next_piece(o)) {
      // Event e of a piece is one tile's PV: of row tile e & 1, on key tile e / 2, or e where both row
      // tiles hold the same rows. It is followed by the scores of event e + 2.
      const int tiles = __shfl_sync(0xffffffffu, o.tiles, 0);
      const int shift = __shfl_sync(0xffffffffu, o.sq.n_q * a.group - o.rb * 256 <= 128 ? 0 : 1, 0);
      const bool dual = shift == 0;
      const int events = tiles << shift;
      ok = wait_warp(CB_Q + 0, q_at & 1u) && (dual || wait_warp(CB_Q + 1, (q_at >> 1) & 1u));
      tc_fence_after();
#pragma unroll 1
      for (int e = -2; ok && e < events; ++e) {
        const int t = e & 1;
        const bool last_use = dual || t == 1;  // of the key tile
        if (e >= 0) {
          // O_t (+)= P'_t V_u. P' comes in two parts: 96 keys, then 32.
          const int u = base + (e >> shift);
          const uint32_t vd = dv + static_cast<uint32_t>(((u % CH_VSLOTS) * C::VTILE) >> 4);
          const uint32_t td = tmem + C::TMEM_O + t * D, tp = tmem + t * 128, parity = (p_at >> t) & 1u;
          p_at ^= 1u << t;
          ok = wait_warp(CB_VF + u % CH_VSLOTS, static_cast<uint32_t>(u / CH_VSLOTS) & 1u) && wait_warp(CB_P + t, parity);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < 6; ++kk) {
            mma_f16_ts(lead, td, tp + kk * 8, vd + kk * (16 * 128 / 16), idesc_pv, (e >= 2 || kk > 0) ? 1u : 0u);
          }
          ok = wait_warp(CB_PL + t, parity);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int kk = 6; kk < 8; ++kk) mma_f16_ts(lead, td, tp + kk * 8, vd + kk * (16 * 128 / 16), idesc_pv, 1u);
          if (e + 2 >= events) commit_to(lead, bar(CB_O + t));
          if (last_use) commit_to(lead, bar(CB_VE + u % CH_VSLOTS));
        }
        if (e + 2 < events) {
          // S_t = Q_t K_u.
          const int u = base + ((e + 2) >> shift);
          ok = wait_warp(CB_KF + u % C::KSLOTS, static_cast<uint32_t>(u / C::KSLOTS) & 1u);
          if (!ok) break;
          tc_fence_after();
          const uint32_t qd = dq + static_cast<uint32_t>(((dual ? 0 : t) * C::TERMS * C::CODES) >> 4);
          const uint32_t kd = dk + static_cast<uint32_t>(((u % C::KSLOTS) * C::CODES) >> 4);
#pragma unroll
          for (int i = 0; i < C::TERMS * C::KSTEPS; ++i) {
            const uint32_t kk = static_cast<uint32_t>(i % C::KSTEPS), term = static_cast<uint32_t>(i / C::KSTEPS);
            mma_f8(lead, tmem + t * 128, qd + (term * C::CODES + kk * 32) / 16, kd + kk * 2, term == 0 ? idesc_qk : idesc_qk5,
                   i > 0 ? 1u : 0u);
          }
          commit_to(lead, bar(CB_S + t));
          if (last_use) commit_to(lead, bar(CB_KE + u % C::KSLOTS));
        }
      }
      if (!ok) break;
      q_at ^= dual ? 1u : 3u;
      base += tiles;
    }
    // Every product has retired before TMEM is given back.
    commit_to(lead, bar(CB_DONE));
    if (!mbar_wait_warp(bar(CB_DONE), 0, CH_TIMEOUT, nullptr)) ok = false;
  } else {
    // -------------------------------------------------------------- softmax: one thread a row
    fa2::reg_alloc<CH_REGS_SM>();
    const int t = warp >> 2, q = warp & 3;
    const int r = q * 32 + lane;  // row of the tile
    const uint32_t lane_addr = static_cast<uint32_t>(q * 32) << 16;
    const uint32_t tS = tmem + t * 128 + lane_addr, tO = tmem + C::TMEM_O + t * D + lane_addr;
    uint32_t s_at = 0, o_at = 0, x_at = 0;  // S's, O's and merges so far
    int base = 0;
    Piece o{};
    while (ok && next_piece(o)) {
      const int rows = o.sq.n_q * a.group, row0 = o.rb * 256, k0 = o.t0 * 128;
      const bool dual = rows - row0 <= 128;
      const int tile_row0 = row0 + (dual ? 0 : t * 128), row = tile_row0 + r;
      // Q: a warp's 32 rows as 8-bit terms, 8 lanes (D / 16) a row, 16 values each; every row times the power
      // of two that brings its largest value into [128, 256). Each term is the rounding of what the
      // terms before leave (an exact difference in fp32). The raw values come by asynchronous copies, all
      // under way at once, to where this lane's first two terms go: it alone reads and overwrites them.
      float row_sc;
      {
        constexpr int LANES = D / 16, STEP = 32 / LANES;  // lanes of a row, rows at a time
        const int part = lane % LANES;
        float* scales = reinterpret_cast<float*>(smem + C::OFF_QS) + t * 128 + q * 32;  // of the warp's rows
        const uint32_t dst = sbase + C::OFF_Q + t * C::TERMS * C::CODES;
        auto place = [&](int i) -> uint32_t {  // of this lane's part of its row in term 0
          const int rt = q * 32 + i * STEP + lane / LANES;
          return dst + rt * 128 + ((part ^ (rt & 7)) << 4);
        };
#pragma unroll 2
        for (int i = 0; i < LANES; ++i) {
          const int qr = tile_row0 + q * 32 + i * STEP + lane / LANES;
          const uint16_t* src = q_row(a, o.sq, o.b, o.h, qr < rows ? qr : row0) + part * 16;
          cp_async16(place(i), src, qr < rows);
          cp_async16(place(i) + C::CODES, src + 8, qr < rows);
        }
        cp_async_commit();
        cp_async_wait<0>();
#pragma unroll 2
        for (int i = 0; i < LANES; ++i) {
          const int rw = i * STEP + lane / LANES, rt = q * 32 + rw;
          uint4 v[2];
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(v[z].x), "=r"(v[z].y), "=r"(v[z].z), "=r"(v[z].w) : "r"(place(i) + z * C::CODES) : "memory");
          }
          const uint32_t w[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
          float x[16];
          uint32_t top = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float2 f2 = float2_of_x2<BF16>(w[j]);
            x[2 * j] = f2.x;
            x[2 * j + 1] = f2.y;
            top = max(top, max(__float_as_uint(f2.x) & 0x7fffffffu, __float_as_uint(f2.y) & 0x7fffffffu));
          }
#pragma unroll
          for (int z = LANES / 2; z > 0; z >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, z));
          const int e = row_exponent(top);
          const float f = top < 0x7f800000u ? pow2f(7 - e) : __uint_as_float(0x7fc00000u);  // NaN, infinity: a NaN row
          if (part == 0) scales[rw] = a.qk_scale * pow2f(max(-126, e - 7));
          if (!dual || t == 0) {
#pragma unroll
            for (int j = 0; j < 16; ++j) x[j] *= f;
#pragma unroll
            for (int term = 0; term < C::TERMS; ++term) {
              uint32_t y[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const uint16_t lo = term == 0 ? e4m3x2(x[4 * j], x[4 * j + 1]) : e5m2x2(x[4 * j], x[4 * j + 1]);
                const uint16_t hi = term == 0 ? e4m3x2(x[4 * j + 2], x[4 * j + 3]) : e5m2x2(x[4 * j + 2], x[4 * j + 3]);
                if (term + 1 < C::TERMS) {
                  const float2 y0 = float2_of_f16x2(term == 0 ? f16x2_of_e4m3x2(lo) : f16x2_of_e5m2x2(lo));
                  const float2 y1 = float2_of_f16x2(term == 0 ? f16x2_of_e4m3x2(hi) : f16x2_of_e5m2x2(hi));
                  x[4 * j] -= y0.x;
                  x[4 * j + 1] -= y0.y;
                  x[4 * j + 2] -= y1.x;
                  x[4 * j + 3] -= y1.y;
                }
                y[j] = static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
              }
              fa2::st_shared_v4(place(i) + term * C::CODES, y[0], y[1], y[2], y[3]);
              if constexpr (D < 32) fa2::st_shared_v4(dst + term * C::CODES + rt * 128 + ((1 ^ (rt & 7)) << 4), 0, 0, 0, 0);
            }
          }
        }
        __syncwarp();
        row_sc = scales[lane];
        if (!dual || t == 0) {
          fa2::fence_proxy_async_smem();
          mbar_arrive(bar(CB_Q + t));
        }
      }
      const int lim_row = row < rows ? last_key(a, o.sq, query_of(a, row)) : -1;  // last visible key
      // All keys up to here are seen by every row of the tile (rows that are not there are zeros).
      const int lim_all = last_key(a, o.sq, query_of(a, tile_row0));

      float m = -INFINITY, l = 0.0f;
      int eb = EB_MIN;
      const int step = dual ? 2 : 1;
      int done = 0;
#pragma unroll 1
      for (int n = dual ? t : 0; n < o.tiles; n += step, ++done) {
        const int u = base + n, en = u % CH_ENTRIES;
        if (!wait_warp(CB_S + t, s_at & 1u) || !wait_warp(CB_SC + en, static_cast<uint32_t>(u / CH_ENTRIES) & 1u)) {
          ok = false;
          break;
        }
        ++s_at;
        tc_fence_after();
        const uint32_t sc_addr = sbase + C::OFF_SC + en * 1024;
        int eb_new;
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(eb_new) : "r"(sbase + C::OFF_HEAD + en * 4));
        const int col0 = k0 + n * 128;
        const bool masked = col0 + 127 > lim_all;
        const int lim = lim_row - col0;

        uint32_t s[4][32];  // x without the row's factor, masked
        fa2::tmem_ld64(tS, s[0], s[1]);
        fa2::tmem_ld64(tS + 64, s[2], s[3]);
        fa2::tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < 4; ++c) fa2::reg_fence32(s[c]);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            uint64_t f0, f1;
            asm volatile("ld.shared.v2.b64 {%0,%1}, [%2];" : "=l"(f0), "=l"(f1) : "r"(sc_addr + (c * 32 + i) * 4));
            float x0, x1, x2, x3;
            fa2::f2_unpack(fa2::f2_mul(fa2::f2_pack(__uint_as_float(s[c][i]), __uint_as_float(s[c][i + 1])), f0), x0, x1);
            fa2::f2_unpack(fa2::f2_mul(fa2::f2_pack(__uint_as_float(s[c][i + 2]), __uint_as_float(s[c][i + 3])), f1), x2, x3);
            s[c][i] = __float_as_uint(x0);
            s[c][i + 1] = __float_as_uint(x1);
            s[c][i + 2] = __float_as_uint(x2);
            s[c][i + 3] = __float_as_uint(x3);
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
        float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            mx0 = fa2::fmax3(mx0, __uint_as_float(s[c][i]), __uint_as_float(s[c][i + 1]));
            mx1 = fa2::fmax3(mx1, __uint_as_float(s[c][i + 2]), __uint_as_float(s[c][i + 3]));
          }
        }
        // Folded: the reference lies P_SHIFT below the maximum, so that P' uses fp16's range up to 2^14.
        const float cand = fmaxf(mx0, mx1) * row_sc - (FOLD ? static_cast<float>(P_SHIFT) : 0.0f);
        const bool bump = cand > m + RESCALE_TH;  // the first tile with a visible key: always
        float alpha = 1.0f;
        if (bump) {
          alpha = fa2::ex2_mufu(m - cand);
          m = cand;
        }
        l *= alpha;
        // O times a factor. (PV of the step before has retired: this step's scores were committed after it.)
        auto scale_o = [&](float f) {
          const uint64_t a2 = fa2::f2_pack(f, f);
#pragma unroll 1
          for (int c = 0; c < D / 16; ++c) {
            uint32_t y[16];
            fa2::tmem_ld16(tO + c * 16, y);
            fa2::tmem_wait_ld();
            fa2::reg_fence16(y);
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
              float y0, y1;
              fa2::f2_unpack(fa2::f2_mul(fa2::f2_pack(__uint_as_float(y[i]), __uint_as_float(y[i + 1])), a2), y0, y1);
              y[i] = __float_as_uint(y0);
              y[i + 1] = __float_as_uint(y1);
            }
            fa2::tmem_st16(tO + c * 16, y);
          }
          fa2::tmem_wait_st();
        };
        const float mr = m == -INFINITY ? 0.0f : m;  // a row that has seen no key yet: p = 0, not NaN
        if (__builtin_expect(eb_new < 0, 0)) {
          // The row's own exponent: products p sv (2^-8 of them: p reaches 2^14) take the scores' place, then P'
          // takes theirs, each 16 columns at a time (rare: small code, no registers kept).
          float sum = 0.0f, most = 0.0f;
#pragma unroll 1
          for (int c = 0; c < 128; c += 16) {
            uint32_t y[16];
            fa2::tmem_ld16(tS + c, y);
            fa2::tmem_wait_ld();
            fa2::reg_fence16(y);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              uint32_t k, v;
              asm volatile("ld.shared.b32 %0, [%1];" : "=r"(k) : "r"(sc_addr + (c + i) * 4));
              asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(sc_addr + 512 + (c + i) * 4));
              const float x = masked && c + i > lim ? -INFINITY : __uint_as_float(y[i]) * __uint_as_float(k);
              const float p = fa2::ex2_mufu(fmaf(x, row_sc, -mr));
              sum += p;
              const float z = p * 0x1p-8f * __uint_as_float(v);
              most = fmaxf(most, fabsf(z));
              y[i] = __float_as_uint(z);
            }
            fa2::tmem_st16(tS + c, y);
          }
          fa2::tmem_wait_st();
          l += sum;
          const int product = static_cast<int>(__float_as_uint(most) >> 23);
          float factor;
          eb = row_unit(product > 0 ? product + 8 : 0, eb, alpha, factor);
          if (done > 0 && __any_sync(0xffffffffu, factor != 1.0f)) scale_o(factor);
          const float gs = __uint_as_float(static_cast<uint32_t>(254 + FOLD_SHIFT + 8 - eb) << 23);
#pragma unroll 1
          for (int c = 0; c < 64; c += 8) {
            uint32_t y[16], pk[8];
            fa2::tmem_ld16(tS + 2 * c, y);
            fa2::tmem_wait_ld();
            fa2::reg_fence16(y);
#pragma unroll
            for (int i = 0; i < 8; ++i) pk[i] = x2_of_floats<false>(__uint_as_float(y[2 * i]) * gs, __uint_as_float(y[2 * i + 1]) * gs);
            tmem_st8(tS + c, pk);
          }
          fa2::tmem_wait_st();
          tc_fence_before();
          mbar_arrive(bar(CB_P + t));
          mbar_arrive(bar(CB_PL + t));
          continue;
        }
        if (done > 0 && __any_sync(0xffffffffu, bump || eb_new > eb)) {
          scale_o(alpha * (eb_new - eb > 126 ? 0.0f : pow2f(eb - eb_new)));
        }
        eb = eb_new;
        const uint64_t sc2 = fa2::f2_pack(row_sc, row_sc), nm2 = fa2::f2_pack(-mr, -mr);
        uint64_t sum2[4] = {0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t (&v)[32] = s[c];
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            float p[4];
#pragma unroll
            for (int j = 0; j < 4; j += 2) {
              float x0, x1;
              fa2::f2_unpack(fa2::f2_fma(fa2::f2_pack(__uint_as_float(v[i + j]), __uint_as_float(v[i + j + 1])), sc2, nm2), x0, x1);
              p[j] = fa2::ex2_mufu(x0);
              p[j + 1] = fa2::ex2_mufu(x1);
              sum2[(i + j) / 2 & 3] = fa2::f2_add(sum2[(i + j) / 2 & 3], fa2::f2_pack(p[j], p[j + 1]));
            }
            if constexpr (!FOLD) {
              float f[4];
              asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];"
                           : "=f"(f[0]), "=f"(f[1]), "=f"(f[2]), "=f"(f[3]) : "r"(sc_addr + 512 + (c * 32 + i) * 4));
#pragma unroll
              for (int j = 0; j < 4; ++j) p[j] *= f[j];
            }
            pk[i / 2] = x2_of_floats<false>(p[0], p[1]);
            pk[i / 2 + 1] = x2_of_floats<false>(p[2], p[3]);
          }
          fa2::tmem_st16(tS + c * 16, pk);
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
      // O, in the units of the last exponent: * 2^(eb - 127 - shift), over the power of two above the sum: an
      // average of the values stays in range where a sum may not.
      if (ok && done > 0) {
        ok = wait_warp(CB_O + t, o_at & 1u);
        ++o_at;
      }
      tc_fence_after();
      const int ex = eb - 127 - FOLD_SHIFT - above(l);
      const float u0 = pow2f(ex / 2), u1 = pow2f(ex - ex / 2);
      float4* area = reinterpret_cast<float4*>(smem + C::OFF_Q + C::TERMS * C::CODES);  // [COLS / 4][128]
      float* ml = reinterpret_cast<float*>(smem + C::OFF_ML);
      float f0 = 1.0f, f1 = 0.0f, mx = m, sum = l, inv = 0.0f;
      const int64_t part_row = static_cast<int64_t>(o.slot) * 256 + (row - row0);
      // 64 columns at a time. With the same rows in both tiles: tile 1 leaves its part, tile 0 takes it.
#pragma unroll 1
      for (int half = 0; ok && half < C::CHUNKS; ++half) {
        if (dual && t == 1) {
          if (half == 0) {
            ml[r] = m;
            ml[128 + r] = l;
          }
          if (done > 0) {
#pragma unroll 1
            for (int c = 0; c < C::COLS / 16; ++c) {
              uint32_t y[16];
              fa2::tmem_ld16(tO + half * 64 + c * 16, y);
              fa2::tmem_wait_ld();
              fa2::reg_fence16(y);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                area[(c * 4 + i) * 128 + r] =
                    make_float4(__uint_as_float(y[4 * i]) * u0 * u1, __uint_as_float(y[4 * i + 1]) * u0 * u1,
                                __uint_as_float(y[4 * i + 2]) * u0 * u1, __uint_as_float(y[4 * i + 3]) * u0 * u1);
              }
            }
          }
          mbar_arrive(bar(CB_X));
          // (Also the last time: the next piece's Q may go where the part lies.)
          ok = wait_warp(CB_Y, x_at & 1u);
          ++x_at;
          continue;
        }
        if (dual) {
          ok = wait_warp(CB_X, x_at & 1u);
          ++x_at;
          if (!ok) break;
        }
        if (half == 0) {
          if (dual) {
            const float m1 = ml[r], l1 = ml[128 + r];
            mx = fmaxf(m, m1);
            // A tile that saw no key has m = -inf and l = 0; a NaN sum is kept.
            f0 = m == -INFINITY ? (l == 0.0f ? 0.0f : 1.0f) : exp2f(m - mx);
            f1 = m1 == -INFINITY ? (l1 == 0.0f ? 0.0f : 1.0f) : exp2f(m1 - mx);
            sum = (f0 == 0.0f ? 0.0f : f0 * l) + (f1 == 0.0f ? 0.0f : f1 * l1);
            f1 *= pow2f(above(l1));
          }
          inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        }
        const float g0 = f0 * inv * pow2f(above(l)), g1 = f1 * inv;
        // The warp's 32 rows go through where its rows of Q were, which are done with, so that rows are
        // stored in whole lines: 32 columns a term, 16-byte parts xor-ed with the row's number.
        uint8_t* stage = smem + C::OFF_Q + t * C::TERMS * C::CODES + q * 32 * 128;
        auto staged = [&](int rw, int p) -> float4& {
          return *reinterpret_cast<float4*>(stage + (p >> 3) * C::CODES + rw * 128 + (((p & 7) ^ (rw & 7)) << 4));
        };
        __syncwarp();  // the columns before have been read
#pragma unroll 1
        for (int c = 0; c < C::COLS / 16; ++c) {
          uint32_t w[16];
          fa2::tmem_ld16(tO + half * 64 + c * 16, w);
          fa2::tmem_wait_ld();
          fa2::reg_fence16(w);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = g0 == 0.0f ? 0.0f : __uint_as_float(w[4 * i + j]) * u0 * u1 * g0;
            if (g1 != 0.0f) {
              const float4 v = area[(c * 4 + i) * 128 + r];
              y[0] = fmaf(v.x, g1, y[0]);
              y[1] = fmaf(v.y, g1, y[1]);
              y[2] = fmaf(v.z, g1, y[2]);
              y[3] = fmaf(v.w, g1, y[3]);
            }
            staged(lane, c * 4 + i) = make_float4(y[0], y[1], y[2], y[3]);
          }
        }
        __syncwarp();
        constexpr int OUT_LANES = C::COLS / 8;  // lanes of a row, 8 columns each
#pragma unroll 1
        for (int i = 0; i < OUT_LANES; ++i) {
          const int rw = i * (32 / OUT_LANES) + lane / OUT_LANES, p8 = lane % OUT_LANES;
          const int out_row = tile_row0 + q * 32 + rw;
          const float4 y0 = staged(rw, 2 * p8), y1 = staged(rw, 2 * p8 + 1);
          if (out_row >= rows) continue;
          if (o.slot >= 0) {
            float4* dst = reinterpret_cast<float4*>(a.o_part + (static_cast<int64_t>(o.slot) * 256 + (out_row - row0)) * D + half * 64 + p8 * 8);
            dst[0] = y0;
            dst[1] = y1;
          } else {
            *reinterpret_cast<uint4*>(o_row(a, o.sq, o.b, o.h, out_row) + half * 64 + p8 * 8) =
                make_uint4(x2_of_floats<BF16>(y0.x, y0.y), x2_of_floats<BF16>(y0.z, y0.w),
                           x2_of_floats<BF16>(y1.x, y1.y), x2_of_floats<BF16>(y1.z, y1.w));
          }
        }
        if (half == 0 && row < rows && o.slot >= 0) {
          a.lse_part[part_row] = sum == 0.0f ? -INFINITY : (mx == -INFINITY ? 0.0f : mx) + log2f(sum);
        }
        if (dual) mbar_arrive(bar(CB_Y));
      }
      tc_fence_before();
      __syncwarp();
      base += o.tiles;
    }
  }

  if (!ok) {
    *static_cast<volatile int*>(stop) = 1;
    report(a.err, FA2_ERR_TIMEOUT);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == CH_MMA_WARP) {
    __syncwarp();
    tc_fence_after();
    fa2::tmem_dealloc(tmem, 512);
  }
}

}  // namespace fa2kv
