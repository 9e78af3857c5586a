// Attention over the 8-bit paged cache: what its kernels share.
//
// With codes c and row scales s, and q scaled by a power of two f_i:
//     x_ij = sm_scale * log2(e) / f_i * (sum_d q'_id ck_jd) * sk_j      p_ij = 2^(x_ij - m_i)
//     o_i  = sum_j (p_ij sv_j) cv_j / sum_j p_ij
// The first product runs on fp16 operands for few rows (q' below 2^15, exact) and on 8-bit ones for
// many (see there). The second runs on fp16: e4m3 codes are exact in it, and P' = p_ij sv_j
// 2^(6 - e), with e the largest exponent of the sv seen so far, is rounded to it (2^-11 of each: an
// eighth of half a bf16 step of the output; for fp16 as much as half a step, so such outputs are about 1.5 times
// as far from the exact ones as their own rounding alone would put them, as with any 16-bit P; a second
// term of P' would double this product). P' < 2^15. Sums, statistics and scales are fp32.
//
// One e for all rows is right as long as the sv lie within 2^WIDE of one another: then P' of a row's largest
// product is 2^-6 or more and 2^-25, half of fp16's smallest step, is 2^-19 of that. Beyond, from the group
// or tile of keys on where they first do, every row has an e of its own, that of its largest product p_ij
// sv_j: a value row of 10^30 does not touch the queries that do not see it or give it no weight. Exponents of
// a row also fall, with its sums, when its maximum grows.
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
  float* o_part;    // partial results: O / l in fp32 ...
  float* lse_part;  // ... and log2 of the row's sum
  struct Cut* cuts;  // [workers]
  int64_t bt_stride;
  long long timeout;
  int pages_per_seq, batch, group, heads_kv, n_q, total_q, max_k;
  Divisor by_group;  // rows to queries
  int causal, bottom_right;
  int workers;  // CTAs that share the work
  int block;    // rows of a block: 8, 16 or 256
  float qk_scale;
};

constexpr float RESCALE_TH = 8.0f;  // log2: the reference max moves when a row's max grows by more
constexpr int P_SHIFT = 6;          // P' = p * sv * 2^(P_SHIFT - e), see above
constexpr int MAX_KEYS = 0x7fffffff - 1023;  // of a sequence: positions a few tiles further fit 32 bits
constexpr int EB_MIN = 16;          // smallest exponent field used for e (a multiplier stays finite)
constexpr int WIDE = 12;            // log2: scales further apart than that give every row its own e, see above

FA2_HOST_DEVICE int query_of(const AttnArgs& a, int row) { return divide(a.by_group, row); }

struct Seq {
  int n_q, q0, len, off;  // queries, first packed row, keys, causal offset
};

// Sequence b, checked: nothing its numbers lead to is outside the tensors.
FA2_HOST_DEVICE Seq sequence(const AttnArgs& a, int b) {
  Seq s;
  s.n_q = a.n_q;
  s.q0 = 0;
  if (a.cu_q != nullptr) {
    s.q0 = load_int(a.cu_q + b);
    const int64_t end = load_int(a.cu_q + b + 1);
    const int64_t n = end - s.q0;
    if (s.q0 < 0 || n < 0 || n > a.n_q || end > a.total_q) {
      report(a.err, FA2_ERR_SHAPE);
      s.n_q = 0;
    } else {
      s.n_q = static_cast<int>(n);
    }
  }
  s.len = load_int(a.lens + b);
  if (s.len < 0 || s.len > a.max_k || s.len > static_cast<int64_t>(a.pages_per_seq) * a.c.page_size) {
    report(a.err, FA2_ERR_SHAPE);
    s.len = 0;
  }
  s.off = a.bottom_right ? s.len - s.n_q : 0;
  return s;
}

// Keys that the rows [row0, row0 + count) of a (sequence, kv head) see at most: [0, result).
FA2_HOST_DEVICE int keys_end(const AttnArgs& a, const Seq& s, int row0, int count) {
  if (!a.causal) return s.len;
  const int i = min(query_of(a, row0 + count - 1), s.n_q - 1);
  return max(0, min(s.len, i + s.off + 1));
}

// The last key that query i sees (-1: none).
__device__ __forceinline__ int last_key(const AttnArgs& a, const Seq& s, int i) {
  return a.causal ? min(s.len - 1, i + s.off) : s.len - 1;
}

__device__ __forceinline__ const uint16_t* q_row(const AttnArgs& a, const Seq& s, int b, int h, int row) {
  const int i = query_of(a, row), g = row - i * a.group;
  const int64_t bb = a.cu_q != nullptr ? 0 : b;
  return a.q + bb * a.q_st[0] + static_cast<int64_t>(h * a.group + g) * a.q_st[1] + static_cast<int64_t>(s.q0 + i) * a.q_st[2];
}

__device__ __forceinline__ uint16_t* o_row(const AttnArgs& a, const Seq& s, int b, int h, int row) {
  const int i = query_of(a, row), g = row - i * a.group;
  const int64_t bb = a.cu_q != nullptr ? 0 : b;
  return a.o + bb * a.o_st[0] + static_cast<int64_t>(h * a.group + g) * a.o_st[1] + static_cast<int64_t>(s.q0 + i) * a.o_st[2];
}

// A row block that is cut for the first time by the start of worker w's share, written by that worker
// for the merge kernel: its parts are those of the workers w - 1, w, w + 1, ...
struct Cut {
  int n_parts;  // 0: this share's start cuts no block, or not as the first
  int b, h, row0;
  int q0, n_q;     // of the sequence
  int first_slot;  // of worker w - 1's part; worker v's is 2 v from w on
  int unused;
};

// The work of a call, as one line of tiles: sequence by sequence, kv head by kv head, row block by
// row block, 128 keys a tile. Worker w of W takes [w N / W, (w + 1) N / W) of the line's N cost units,
// whatever the sequences' lengths: nobody waits for a longer sequence, and the lengths may live on the
// device. A (sequence, head, block) that lies in one worker's share is written as the result; one
// that is cut leaves a partial result for each share (a worker has at most two: where its share
// begins and where it ends) and the merge kernel puts them together in the line's order.
// A tile of few rows costs 1. In the 256-row kernel it costs 4, or 3 where a CTA has one 128-row tile of
// rows to do for it (2.35 and 1.7 us), and a block adds what its start and end take (10 us: 16) where
// the shares are long enough for that to matter.
struct Line {
  // Tiles and tile cost of row block rb of sequence s, and the sum over a sequence's blocks.
  FA2_HOST_DEVICE static int blocks(const AttnArgs& a, const Seq& s) { return (s.n_q * a.group + a.block - 1) / a.block; }
  FA2_HOST_DEVICE static int tiles(const AttnArgs& a, const Seq& s, int rb) {
    const int rows = s.n_q * a.group, row0 = rb * a.block;
    return (keys_end(a, s, row0, min(a.block, rows - row0)) + 127) / 128;
  }
  FA2_HOST_DEVICE static int tile_cost(const AttnArgs& a, const Seq& s, int rb) {
    return a.block < 256 ? 1 : s.n_q * a.group - rb * 256 > 128 ? 4 : 3;
  }
  // A kv head's tiles (cost) and blocks that have any.
  FA2_HOST_DEVICE static void head_cost(const AttnArgs& a, const Seq& s, int& tiles_cost, int& n_blocks) {
    tiles_cost = n_blocks = 0;
    for (int rb = 0; rb < blocks(a, s); ++rb) {
      const int n = tiles(a, s, rb);
      tiles_cost += n * tile_cost(a, s, rb);
      n_blocks += n > 0 ? 1 : 0;
    }
  }
  // From the tiles' cost: the workers that get something, and a block's own cost. Every share is at
  // least as long as a block's own cost and a tile, so one that begins or ends inside a block but for
  // its first tile holds one of its tiles.
  FA2_HOST_DEVICE static int workers(const AttnArgs& a, int cost) { return min(a.workers, a.block < 256 ? cost : max(1, cost / 4)); }
  FA2_HOST_DEVICE static int block_cost(const AttnArgs& a, int cost) {
    return a.block < 256 ? 0 : min(16, max(0, cost / a.workers - 4));
  }
  // Where worker w's share starts, and the worker whose share holds position x.
  FA2_HOST_DEVICE static int start(int w, int workers, int total) {  // w total / workers, in 32 bits
    const uint32_t q = static_cast<uint32_t>(total) / static_cast<uint32_t>(workers), r = total - q * workers;
    return static_cast<int>(w * q + w * r / static_cast<uint32_t>(workers));  // (w r < workers^2)
  }
  FA2_HOST_DEVICE static int holder(int x, int workers, int total) {
    int w = min(workers - 1, static_cast<int>((x + 0.5f) * workers / total));  // off by one at most
    while (w > 0 && start(w, workers, total) > x) --w;
    while (w + 1 < workers && start(w + 1, workers, total) <= x) ++w;
    return w;
  }
};

// A worker's share of the line and a sequence at or before its start.
struct Share {
  int total, workers, block_cost;
  int p0, p1;         // this worker's share
  int b, start_b;     // the first sequence of the run that holds p0, and where it starts
};
// A line of LONGEST_LINE cost units or more is refused and nothing is done. The host's limits keep every
// line of sequences that do not overlap below it; sums of query lengths that go back and forth could
// count the same queries many times. Positions are 32 bits, so the sums over the line stop there.
constexpr int LONGEST_LINE = (1 << 30) - 1;
FA2_HOST_DEVICE int line_sum(int x, int y) { return x + y < LONGEST_LINE ? x + y : LONGEST_LINE; }

// Tiles' cost and blocks of a run of sequences.
struct Run {
  int b0, cost, blocks;
};
// Those of lane `lane`, one of the 32 runs that the sequences are divided into. (A sequence alone is below
// 2^29: the host's limits hold for each.)
FA2_HOST_DEVICE Run run_of(const AttnArgs& a, int lane) {
  const int per = (a.batch + 31) / 32, first = lane * per;
  Run r{first < a.batch ? first : a.batch, 0, 0};
  const int end = r.b0 + per < a.batch ? r.b0 + per : a.batch;
#pragma unroll 1
  for (int b = r.b0; b < end; ++b) {
    int cost, n;
    Line::head_cost(a, sequence(a, b), cost, n);
    r.cost = line_sum(r.cost, a.heads_kv * cost);
    r.blocks = line_sum(r.blocks, a.heads_kv * n);
  }
  return r;
}
// Worker w's share of a line of tiles that cost `cost` in `blocks` blocks; false where it is refused.
FA2_HOST_DEVICE bool share_of(const AttnArgs& a, int w, int cost, int blocks, Share& r) {
  r = Share{};
  const int block_cost = Line::block_cost(a, cost);
  const int64_t total = cost + static_cast<int64_t>(block_cost) * blocks;  // (blocks <= cost)
  if (total >= LONGEST_LINE) return false;
  r.workers = Line::workers(a, cost);
  r.block_cost = block_cost;
  r.total = static_cast<int>(total);
  if (w < r.workers) {
    r.p0 = Line::start(w, r.workers, r.total);
    r.p1 = Line::start(w + 1, r.workers, r.total);
  }
  return true;
}

// Finds a worker's share with a warp: each lane adds up a run.
__device__ __forceinline__ Share find_share(const AttnArgs& a, int w) {
  const int lane = static_cast<int>(threadIdx.x) & 31;
  const Run run = run_of(a, lane);
  int sum = run.cost, sum_blocks = run.blocks;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, sum, o), n = __shfl_up_sync(0xffffffffu, sum_blocks, o);
    if (lane >= o) {
      sum = line_sum(sum, v);
      sum_blocks = line_sum(sum_blocks, n);
    }
  }
  Share r;
  if (!share_of(a, w, __shfl_sync(0xffffffffu, sum, 31), __shfl_sync(0xffffffffu, sum_blocks, 31), r)) {
    report(a.err, FA2_ERR_SHAPE);
    return r;
  }
  const int own = run.cost + r.block_cost * run.blocks, before = sum + r.block_cost * sum_blocks - own;
  const uint32_t at = __ballot_sync(0xffffffffu, before <= r.p0 && r.p0 < before + own);
  const int from = at != 0 ? __ffs(at) - 1 : 0;
  r.b = __shfl_sync(0xffffffffu, run.b0, from);
  r.start_b = __shfl_sync(0xffffffffu, before, from);
  return r;
}

// A row block and where it lies in the line.
struct Block {
  Seq sq;
  int b, h, rb;
  int at, tiles, cost;  // position of the first tile, tiles, cost of each
  int first;            // position of the block
  // The first tile at or behind position p. A share that begins or ends inside a tile: the tile
  // belongs to the earlier worker.
  FA2_HOST_DEVICE int tile_of(int p) const { return p <= at ? 0 : min(tiles, (p - at + cost - 1) / cost); }
};
// The block that holds position p, walking on from sequence b, which starts at `start`.
FA2_HOST_DEVICE void find_block(const AttnArgs& a, int block_cost, int p, int& b, int& start, Block& o) {
  int hc;
  while (true) {
    o.sq = sequence(a, b);
    int n;
    Line::head_cost(a, o.sq, hc, n);
    hc += n * block_cost;
    if (p < start + hc * a.heads_kv) break;
    start += hc * a.heads_kv;
    ++b;
  }
  o.b = b;
  o.h = (p - start) / hc;
  o.first = start + o.h * hc;
  for (o.rb = 0;; ++o.rb) {
    o.tiles = Line::tiles(a, o.sq, o.rb);
    o.cost = Line::tile_cost(a, o.sq, o.rb);
    o.at = o.first + (o.tiles > 0 ? block_cost : 0);
    if (p < o.at + o.tiles * o.cost) return;
    o.first = o.at + o.tiles * o.cost;
  }
}

// A piece of a worker's share: tiles of one row block.
struct Piece {
  Seq sq;
  int b, h, rb;
  int t0, tiles;  // the first tile and how many
  int kend;       // keys that the block's rows see: [0, kend)
  int slot;       // where a partial result goes, -1 for a whole one
};
// The pieces of a share in order; a warp walks them (uniformly) and also leaves the share's Cut.
struct Pieces {
  Share s;
  int p, w;
  __device__ void begin(const AttnArgs& a, int worker) {
    s = find_share(a, worker);
    p = s.p0;
    w = worker;
    if (s.p0 >= s.p1) a.cuts[w].n_parts = 0;
  }
  FA2_HOST_DEVICE bool next(const AttnArgs& a, Piece& o) {
    while (p < s.p1) {
      Block k;
      find_block(a, s.block_cost, p, s.b, s.start_b, k);
      o.sq = k.sq;
      o.b = k.b;
      o.h = k.h;
      o.rb = k.rb;
      o.t0 = k.tile_of(p);
      o.tiles = k.tile_of(s.p1) - o.t0;
      const int row0 = o.rb * a.block;
      o.kend = keys_end(a, o.sq, row0, min(a.block, o.sq.n_q * a.group - row0));
      if (p == s.p0) {
        const int before = w > 0 ? Line::start(w - 1, s.workers, s.total) : 0;
        Cut c{};
        if (o.tiles > 0 && o.t0 > 0 && k.tile_of(before) == 0) {
          // (A tile is its start's holder's.)
          c.n_parts = Line::holder(k.at + (k.tiles - 1) * k.cost, s.workers, s.total) - w + 2;
          c.b = o.b;
          c.h = o.h;
          c.row0 = row0;
          c.q0 = o.sq.q0;
          c.n_q = o.sq.n_q;
          c.first_slot = 2 * (w - 1) + (before >= k.first ? 0 : 1);
        }
        a.cuts[w] = c;
      }
      o.slot = o.tiles == k.tiles ? -1 : 2 * w + (p == s.p0 ? 0 : 1);
      p = min(s.p1, k.at + k.tiles * k.cost);
      if (o.tiles > 0) return true;
    }
    return false;
  }
};

// The pieces of a share for warps that meet at a barrier without a time limit, which each of them runs:
// next() is 1 where a piece came, 0 after the last one, -1 where the wait for it ran out; agree(ok) is
// the barrier, the same in every warp: whether all are ok; work() does a piece and ends as agree()
// ended last. A warp that gave up still comes to the barrier, once, and all leave together: none
// waits there for one that has left.
#pragma nv_exec_check_disable
template <typename Next, typename Agree, typename Work>
__host__ __device__ __forceinline__ bool pieces_together(Next next, Agree agree, Work work) {
  while (true) {
    const int got = next();
    if (!agree(got >= 0)) return false;
    if (got == 0) return true;
    if (!work()) return false;
  }
}

// A later kernel of the stream may start before this one ends (it waits for its results itself).
__device__ __forceinline__ void allow_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Whether scales of which the smallest but zero is `low` (its bits - 1: a zero counts as the largest) and the
// largest has the exponent field eb lie further apart than one unit for all rows takes.
__device__ __forceinline__ bool too_wide(int eb, uint32_t low) { return low < (static_cast<uint32_t>(eb - WIDE) << 23) - 1u; }
// A row's exponent from that of its largest new product (as a field, 0: none) and the one it had, and what its
// sums are multiplied by; `alpha`: by what its maximum's growth scales them.
__device__ __forceinline__ int row_unit(int product, int had, float alpha, float& factor) {
  const int fall = 127 - static_cast<int>(__float_as_uint(alpha) >> 23);  // alpha <= 1; 127 for 0
  const int e = max(max(EB_MIN, product), alpha > 0.0f ? had - fall : 0);
  const int up = had - e;  // <= fall
  factor = alpha > 0.0f && up >= -126 ? alpha * __uint_as_float(static_cast<uint32_t>(up + 127) << 23) : 0.0f;
  return e;
}

__device__ __forceinline__ float pow2f(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }  // -126 <= e <= 127

// The exponent of the power of two above a row's sum (0 and NaN: any, the row's O is 0 or NaN).
__device__ __forceinline__ int above(float sum) { return min(static_cast<int>(__float_as_uint(sum) >> 23), 253) - 126; }

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
