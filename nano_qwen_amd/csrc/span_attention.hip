// Attention over chosen spans of the cache, for gfx950: a sliding window with
// sinks (prefill and decode), and trees of drafted tokens.  No counterpart in
// the reference, whose attention (layers/attention.py:64-74) is causal over
// the whole context.
//
// Rows.  Sequence s has Lq query tokens at positions P + t, P = Lk - Lq, of
// its Lk cached tokens (Lq = 1: decode).  Row r = t * G + i is query head
// kvh * G + i of token t: the rows of one kv head, tokens and heads packed, so
// that a tile of M rows reads each K/V byte once for all of them whatever the
// group size, and a tree of n nodes fills M = n * G rows.
//
// Visible keys of the row of token t, position p = P + t:
//   window: j <= p and (j > p - window or j < sinks);
//   tree:   j < C = Lk - Lq (the context), or node j - C in the row's mask.
// Either way they lie in at most two runs of 32-key tiles -- the sinks' and
// the rest -- so an item (row tile of a sequence) is a list of tiles: the
// first `ts` tiles, then those from `tlo` on.  Keys of a tile that only some
// rows see are masked; whole tiles outside the list are never read, so pages
// that hold no visible key may be missing from the table.
//
// Products as in the other attention kernels: S^T = K Q^T and O^T += V^T P^T
// on v_mfma_f32_16x16x32, whose S^T accumulator is the B operand of the second
// product; V^T through transposing LDS reads; fp8 K/V stay codes in LDS and
// are widened (exactly) in registers, with the scales on the scores and the
// output.  Softmax in the log2 domain, statistics and sums in fp32; the
// maximum of a row moves only when it grows by more than 2^8 (P <= 256, so
// rounding P to 16 bits loses no more than it does at P <= 1).
//
// NaN and infinities in keys or values that a row does not see do not reach
// it: masked scores are replaced before use, and an item whose outputs are not
// all finite is done again with the values that are not finite taken out of the
// products and given back to the rows that see them (odd_values, poison, clean).
// Checking every masked tile's values in the first pass cost more than the rare
// second one: a prompt pair of 8000 tokens, window 2048, 757 us against 570.
//
// Work.  Few long items are cut into equal ranges of the tiles laid end to end,
// one per workgroup, and joined by a second kernel; many are dealt out whole
// (launch).  A workgroup's copies run on from an item into the next, kAhead
// tiles before the tile at work.
//
// What bounds it, measured: prefill, the matrix cores and the exponentials
// beside them: two prompts of 8016 and 8089 tokens, 32 query heads of 8 kv heads
// at D = 128, window 2048, 574-592 us, 800-820 TFLOP/s (products busy 38 % of the
// time, other vector instructions 41 %); full causal of 8192 980.  Trees of 64
// nodes and 64 query heads over 16000-32768 fp8 tokens 254-262 us, 740-760
// TFLOP/s (35 % and 52 %: the conversions share the vector unit with the
// exponentials).  Batched decode, HBM: 96 rows through a window of 4096, 265 us,
// 5.5 TB/s.  Single requests, a chain of round trips to memory: 12 us, and 4-6
// for the second kernel.
#include <algorithm>
#include <type_traits>

#include "nq_device.hpp"

namespace nq {
namespace {

constexpr int kKeys = 32;         // keys per tile
constexpr float kRescale = 8.0f;  // log2 growth of a row maximum that moves it
constexpr int kMaxNodes = 256;    // of a tree: 8 mask words of 32 bits per row

// 16-byte chunk c of key row r of a 16-bit tile lies at chunk c ^ swz(r), so
// that the operand reads (16 rows x one chunk of K; 4 rows x 2 chunks of V^T)
// meet no bank twice; fp8 tiles of D-byte rows likewise in 16-byte units.
__device__ inline int swz_k(int row) { return row & 15; }
__device__ inline int swz_v(int row) { return ((row & 7) << 1) | ((row >> 3) & 1); }
template <int D>
__device__ inline int swz8(int row) {
  const int b = ((row >> 3) ^ (row >> 4)) & 1;
  return D == 128 ? (((row >> 1) & 3) | (b << 2)) : ((row & 7) | (b << 3));
}

struct SpanArgs {
  const uint8_t *q;
  int64_t q_rs, q_hs;  // bytes
  const uint8_t *k;
  const uint8_t *v;
  int64_t kv_rs;        // bytes per K/V row (token)
  const int32_t *cu_q;  // null: one row per sequence (decode)
  const int32_t *cu_k;  // prefix sums of the lengths; decode: the lengths themselves
  int total_q, total_k;  // rows of q and, packed K/V, of k: sequences are clamped to them
  int max_q, max_k;      // most query tokens and keys of a sequence (further ones are never touched)
  const int32_t *block_tables;  // null: packed K/V
  int64_t bt_stride;
  int max_blocks, num_blocks;
  uint8_t *out;
  int64_t o_rs, o_hs;
  const uint8_t *gate;  // null, or the output gate, of the type of out
  int64_t g_rs, g_hs;
  int Hq, Hkv, G, block_size, num_seqs;
  int window, sinks;     // window 0: trees
  const uint64_t *mask;  // [total_q, words] rows of mask_rs words
  int64_t mask_rs;
  int words;
  float scale_log2;
  const float *k_scale;
  const float *v_scale;
  // Decode: the new token's rows to store [num_seqs, Hkv, D] (null: none), of type new_dtype.
  const uint8_t *k_new;
  const uint8_t *v_new;
  int64_t kn_rs, vn_rs;  // bytes
  const int32_t *slot_mapping;
  int new_dtype;
  // Equal ranges: n_ranges per kv head (0: one item per workgroup), the partial
  // outputs of range w's slots 2 w and 2 w + 1 (fp32, normalised, as the lanes
  // hold them), their rows' log2-sum-exp, and what they are.
  int n_ranges, min_range;
  int stride;  // whole items: from a workgroup's item to its next
  float *part_o;
  float *part_l;
  int4 *part_desc;  // (sequence, row tile, kind, 0)
};
constexpr int kPieceNone = -1, kPieceMore = 0, kPieceLast = 1;

// Launch shape: RW waves of QS x 16 rows each that share every tile (M rows),
// a ring of SLOTS tiles.
//  * one wave (M = 16): decode and the smallest trees.  Its ring is its own:
//    no barriers, and K and V of SLOTS tiles are in flight at all times.
//  * four waves of 16 or 32 rows (eight of 16 at head_dim 256; four of 32, with
//    400 registers and so one per SIMD, ran 147 us for six prompts of 200-2567
//    tokens where these took 124, before the rules of launch() brought them to
//    113).  A barrier per tile; copies run SLOTS - 1 tiles ahead.  (The 16-bit
//    shapes at head_dim 256 spill one and five registers, in the items' set-up.)
template <int D_, bool FP8, int RW_, int QS_, int SLOTS_>
struct Shape {
  static constexpr int D = D_, RW = RW_, QS = QS_, SLOTS = SLOTS_;
  static constexpr int M = RW * QS * 16;
  static constexpr int SRC_ROWB = FP8 ? D : 2 * D;
  static constexpr int TILE_B = kKeys * SRC_ROWB, SLOT_B = 2 * TILE_B;
  static constexpr int LPR = SRC_ROWB / 16;        // lanes (16-byte pieces) per row
  static constexpr int COPS = TILE_B / 1024 / RW;  // copies per wave of a K (or V) tile
  static constexpr int RING_B = SLOTS * SLOT_B;
  static constexpr int MASK_WORDS = kMaxNodes / 32 + 1;  // LDS row of a token's mask (odd: no bank pattern)
  static constexpr int TOKENS = M + 1;                   // of a row tile, at most
  static constexpr int SEQS = 256;  // sequences whose bounds are kept in LDS
  // ring, masks, flags of odd tiles, sequences' bounds and positions
  static constexpr int MASK_AT = RING_B, ODD_AT = MASK_AT + (TOKENS * MASK_WORDS * 4 + 15) / 16 * 16,
                       SEQ_AT = ODD_AT + 128, POS_AT = SEQ_AT + SEQS * 16, NEW_AT = POS_AT + SEQS * 8,
                       LDS_B = NEW_AT + (RW == 1 ? 2 * SRC_ROWB : 0);  // (the new token's K and V rows)
  static constexpr int NKK = D / 32, NJ = D / 16;
  static_assert(COPS >= 1, "every wave copies");
};

// The kernel's arguments, read from its argument segment where they are used:
// held in registers, the many that only an item's start needs would crowd the
// tile loop's out.  (The address is opaque, so that no read is moved.)
typedef const __attribute__((address_space(4))) SpanArgs KernArgs;
__device__ __forceinline__ KernArgs *kernel_args() {
  KernArgs *p = (KernArgs *)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return p;
}

// ---------------------------------------------------------------- items
struct Seq {
  int s, q0, Lq, k0, Lk;
};
template <class A>
__device__ __forceinline__ Seq seq_of(const A &a, int s, bool uniform) {
  Seq x{};
  x.s = s;
  if (!a.cu_q) {
    x.q0 = s;
    x.Lq = 1;
    x.Lk = uniform ? ld_const(a.cu_k + s) : a.cu_k[s];
  } else {
    const int qa = uniform ? ld_const(a.cu_q + s) : a.cu_q[s], qb = uniform ? ld_const(a.cu_q + s + 1) : a.cu_q[s + 1];
    const int ka = uniform ? ld_const(a.cu_k + s) : a.cu_k[s], kb = uniform ? ld_const(a.cu_k + s + 1) : a.cu_k[s + 1];
    x.q0 = max(0, min(qa, a.total_q));
    x.Lq = max(0, min(min(qb, a.total_q) - x.q0, a.max_q));
    x.k0 = max(0, min(ka, a.total_k));
    x.Lk = a.block_tables ? kb - ka : min(kb, a.total_k) - x.k0;
  }
  x.Lk = max(0, min(x.Lk, a.max_k));
  return x;
}
// floor(n / d) for 0 <= n < 2^22, 1 <= d < 2^22: the float estimate is within
// one of the quotient.
__device__ __forceinline__ int small_div(int n, int d) {
  int q = static_cast<int>(static_cast<float>(n) * __builtin_amdgcn_rcpf(static_cast<float>(d)));
  if (q * d > n)
    --q;
  else if ((q + 1) * d <= n)
    ++q;
  return q;
}
// A value that every lane has, in a scalar register (small_div leaves it in a
// vector one).
__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }
// The tiles of a row tile whose tokens are ta .. tb.
struct Tiles {
  int ts, tlo, n;  // tiles 0 .. ts - 1, then tlo, tlo + 1, ...: n in all
};
template <class A>
__device__ __forceinline__ Tiles tiles_of(const A &a, const Seq &q, int ta, int tb) {
  Tiles t{0, 0, 0};
  if (a.window == 0) {
    t.n = (q.Lk + kKeys - 1) / kKeys;
    return t;
  }
  const int P = q.Lk - q.Lq;
  const int end = P + tb + 1;  // keys before it may be seen
  if (end <= 0) return t;
  t.ts = (min(a.sinks, end) + kKeys - 1) / kKeys;
  t.tlo = max(t.ts, max(0, P + ta - a.window + 1) / kKeys);
  t.n = t.ts + max(0, (end + kKeys - 1) / kKeys - t.tlo);
  return t;
}
// Cost of each row tile of a sequence in key tiles: an item's fixed cost and
// its tiles (of several windowed row tiles: the most that one can have).
template <class S>
struct Cost {
  // one wave: Q and first-tile latency, in the time of a tile; more waves: the
  // same in their faster tiles
  static constexpr int kItem = S::RW == 1 ? 1 : 4;
  // A range has at least kMinRange tiles, and enough that the longest item is cut
  // into about kPieces.  Fewer pieces leave compute units idle, more are a longer
  // merge: one tree of 16 rows behind 8192 tokens 58 us in ranges of 2 tiles (128
  // pieces), 21 in ranges of 8; one of 64 rows 54 in ranges of 2, 34 of 8, 26 of
  // 16; a decode of 1028 tokens 14.4 in ranges of 2, 15.3 of 4.  The larger a
  // piece's partials, the longer its range: trees of 8 nodes (64 rows) behind 800
  // tokens 17.8 in ranges of 4, 18.9 of 8 (D = 256: 19.5 and 22.3); a prefill of
  // 100 tokens (128 rows) behind 2000 49 and 34.
  static constexpr int kMinRange = S::RW == 1 ? 2 : S::M <= 64 ? 4 : 8, kPieces = S::RW == 1 ? 32 : 16;
  // What cutting costs, in the time of a tile: partials written, a second launch.
  static constexpr int kCut = S::RW == 1 ? 20 : 28;
};
template <class S, class A>
__device__ __forceinline__ int row_tiles(const A &a, const Seq &q) {
  return (q.Lq * a.G + S::M - 1) / S::M;
}
template <class S, class A>
__device__ __forceinline__ int item_cost(const A &a, const Seq &q) {
  if (q.Lq <= 0) return 0;
  int n;
  if (q.Lq * a.G <= S::M) {
    n = tiles_of(a, q, 0, q.Lq - 1).n;
  } else {
    n = (q.Lk + kKeys - 1) / kKeys;
    if (a.window > 0)
      n = min(n, (min(a.sinks, q.Lk) + kKeys - 1) / kKeys + (min(a.window, q.Lk) + S::M + 2 * kKeys - 2) / kKeys);
  }
  return Cost<S>::kItem + n;
}

// ---------------------------------------------------------------- the kernel
template <class T, bool FP8, class S>
__device__ __forceinline__ void span_body() {
  constexpr int D = S::D, RW = S::RW, QS = S::QS, M = S::M, SLOTS = S::SLOTS, COPS = S::COPS;
  constexpr int NKK = S::NKK, NJ = S::NJ, TILE_B = S::TILE_B, SLOT_B = S::SLOT_B, SRC_ROWB = S::SRC_ROWB;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  const int lane = threadIdx.x & 63;
  const int rw = RW == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m = lane & 15, g = lane >> 4;
  KernArgs &a0 = *kernel_args();  // (of the prologue)
  const bool paged = a0.block_tables != nullptr;
  const int n_ranges = a0.n_ranges;
  const bool ranges = n_ranges > 0;

  // kv head and range (or item) of this workgroup.  Workgroup L runs on XCD
  // L % 8: a kv head stays on one XCD (or, of fewer than 8, on 8 / Hkv, which
  // take contiguous ranges, or items in turn), so that the row tiles that read
  // the same keys share an L2.
  const int L = blockIdx.x;
  int h, w;
  if (a0.Hkv < 8 && 8 % a0.Hkv == 0) {
    const int per = 8 / a0.Hkv, x = L & 7;
    h = x % a0.Hkv;
    w = ranges ? (x / a0.Hkv) * (n_ranges / per) + (L >> 3) : (L >> 3) * per + x / a0.Hkv;
  } else {
    h = L % a0.Hkv;
    w = L / a0.Hkv;
  }

  // The batch's row tiles laid end to end.  In equal ranges each counts as its
  // cost.  Whole items are dealt out in rounds, every other round in reverse:
  // first the row tiles whose window is full, which cost the same, then those
  // nearer their sequence's start, each sequence's from the costly end (`ramp`
  // of them), so that the workgroups' sums stay even.
  // Of up to SEQS sequences the bounds and the positions of their ends are kept
  // in LDS, so that finding an item is no chain of round trips to memory; with
  // more of them whole items are dealt out in order.
  int4 *const lds_seq = reinterpret_cast<int4 *>(smem + S::SEQ_AT);
  int2 *const lds_pos = reinterpret_cast<int2 *>(smem + S::POS_AT);
  const bool listed = a0.num_seqs <= S::SEQS;
  auto weight_of = [&](KernArgs &a, const Seq &q) -> int { return ranges ? item_cost<S>(a, q) : (q.Lq > 0 ? 1 : 0); };
  auto ramp_of = [&](KernArgs &a, const Seq &q, int tiles) -> int {
    if (ranges || !listed || a.window == 0) return 0;
    const int short_of = min(a.window - 1 - (q.Lk - q.Lq), q.Lq);  // tokens whose window is not full
    return max(0, min(tiles, (short_of * a.G + M - 1) / M));
  };
  int total = 0, total_ramp = 0;
  for (int b = 0; b < a0.num_seqs; b += 64) {
    int c = 0, ramp = 0;
    Seq q{};
    if (b + lane < a0.num_seqs) {
      q = seq_of(a0, b + lane, false);
      c = row_tiles<S>(a0, q);
      ramp = ramp_of(a0, q, c);
      c = (c - ramp) * weight_of(a0, q);
    }
    const int incl = total + wave_iscan(c), incl_ramp = total_ramp + wave_iscan(ramp);
    if (listed && rw == 0 && b + lane < a0.num_seqs) {
      lds_seq[b + lane] = int4{q.q0, q.Lq, q.k0, q.Lk};
      lds_pos[b + lane] = int2{incl, incl_ramp};
    }
    total = __builtin_amdgcn_readlane(incl, 63);
    total_ramp = __builtin_amdgcn_readlane(incl_ramp, 63);
  }
  if (listed) {
    if constexpr (RW == 1)
      wave_lds_sync();
    else
      __syncthreads();
  }
  // Where this workgroup is: its next position (ranges), or its next round.
  int pos0 = 0, pos1 = total + total_ramp;
  int w_of = 0;  // the range's partials
  if (ranges) {
    w_of = h * n_ranges + w;
    const int W = min(n_ranges, max(1, total / a0.min_range));
    pos0 = w < W ? static_cast<int>(static_cast<int64_t>(w) * total / W) : 0;
    pos1 = w < W ? static_cast<int>(static_cast<int64_t>(w + 1) * total / W) : 0;
  }
  int cuts = 0;  // which of the range's two partial pieces have been described to the merge
  // The first item from `at` (a position or a round) on that this workgroup has
  // to do something for (live: there is one).
  struct Item {
    bool live;
    Seq q;
    int rt, lo, hi, at, next;  // its row tile, its part of the tiles, where it and the next are looked for
    int r_first, r_last, t_first, t_last;
    Tiles tl;
  };
  auto describe = [&](int at) -> Item {
    KernArgs &a = *kernel_args();
    Item it{};
    for (;;) {
      const int pos = ranges ? at : at * a.stride + ((at & 1) ? a.stride - 1 - w : w);
      if (ranges ? pos >= pos1 : at * a.stride >= pos1) return it;
      it.at = at;
      it.next = at + 1;
      if (pos >= pos1) {  // the last round is a part of one
        at = it.next;
        continue;
      }
      const bool ramp = pos >= total;
      const int want = ramp ? pos - total : pos;
      int start = 0, cost = 1;  // where the sequence's row tiles start, and each one's weight
      if (listed) {
        for (int b = 0;; b += 64) {
          const int2 e = lds_pos[min(b + lane, a.num_seqs - 1)];
          const uint64_t hit = __builtin_amdgcn_ballot_w64((ramp ? e.y : e.x) > want);
          if (hit == 0) continue;  // (the last entry's is the total: past `want`)
          const int s = b + static_cast<int>(__builtin_ctzll(hit));
          const int4 x = lds_seq[s];
          it.q.s = s;
          it.q.q0 = __builtin_amdgcn_readfirstlane(x.x);
          it.q.Lq = __builtin_amdgcn_readfirstlane(x.y);
          it.q.k0 = __builtin_amdgcn_readfirstlane(x.z);
          it.q.Lk = __builtin_amdgcn_readfirstlane(x.w);
          if (s > 0) {
            const int2 before = lds_pos[s - 1];
            start = __builtin_amdgcn_readfirstlane(ramp ? before.y : before.x);
          }
          break;
        }
        cost = weight_of(a, it.q);
      } else {
        int base = 0;
        for (int b = 0; b < a.num_seqs; b += 64) {
          int c = 0;
          if (b + lane < a.num_seqs) {
            const Seq q = seq_of(a, b + lane, false);
            c = row_tiles<S>(a, q) * weight_of(a, q);
          }
          const int incl = base + wave_iscan(c);
          const uint64_t hit = __builtin_amdgcn_ballot_w64(incl > want);
          if (hit != 0) {
            const int l = static_cast<int>(__builtin_ctzll(hit));
            it.q = seq_of(a, b + l, true);
            start = __builtin_amdgcn_readlane(incl - c, l);
            break;
          }
          base = __builtin_amdgcn_readlane(incl, 63);
        }
        cost = weight_of(a, it.q);
      }
      it.rt = uni(static_cast<int>(static_cast<unsigned>(want - start) / static_cast<unsigned>(cost)));
      const int X = start + it.rt * cost;
      if (!ranges && listed) {
        const int n_ramp = ramp_of(a, it.q, row_tiles<S>(a, it.q));
        it.rt = ramp ? n_ramp - 1 - it.rt : n_ramp + it.rt;
      }
      it.r_first = it.rt * M;
      it.r_last = min(it.r_first + M, it.q.Lq * a.G) - 1;
      it.t_first = uni(small_div(it.r_first, a.G));
      it.t_last = uni(small_div(it.r_last, a.G));
      it.tl = tiles_of(a, it.q, it.t_first, it.t_last);
      it.lo = 0;
      it.hi = it.tl.n;
      if (ranges) {
        it.lo = max(0, min(it.tl.n, pos0 - X - Cost<S>::kItem));
        it.hi = max(0, min(it.tl.n, pos1 - X - Cost<S>::kItem));
        it.next = X + cost;
      }
      // an item without tiles is written (zeros) where it starts
      it.live = it.hi > it.lo || (it.tl.n == 0 && (!ranges || X >= pos0));
      if (it.live) return it;
      at = it.next;
    }
  };

  // ---------------------------------------------------------------- copies
  const uint32_t lds0 = static_cast<uint32_t>(
      reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t *)(smem)));
  uint32_t *const lds_mask = reinterpret_cast<uint32_t *>(smem + S::MASK_AT);
  const int kv_rs = own_sgpr(static_cast<int>(a0.kv_rs));
  // Lane l's piece of copy c lands at row drow, piece l % LPR of the tile; it
  // fetches the piece that the swizzle puts there.
  uint32_t src_k[COPS], src_v[COPS];
#pragma unroll
  for (int c = 0; c < COPS; ++c) {
    const int drow = (rw * COPS + c) * (64 / S::LPR) + lane / S::LPR;
    const uint32_t row_off = static_cast<uint32_t>(drow * kv_rs);
    if constexpr (FP8) {
      src_k[c] = src_v[c] = row_off + (((lane % S::LPR) ^ swz8<D>(drow)) << 4);
    } else {
      src_k[c] = row_off + (((lane % S::LPR) ^ swz_k(drow)) << 4);
      src_v[c] = row_off + (((lane % S::LPR) ^ swz_v(drow)) << 4);
    }
  }
  const int64_t v_minus_k = own_sgpr(static_cast<int64_t>(a0.v - a0.k));
  // The copies are a stream of ring entries, kAhead of them ahead of the tile
  // at work, which runs on into the next item's tiles.  Lane l of `list` holds
  // where the l-th of 64 tiles lies (in tiles of 32 rows; -1: its page is missing).
  int st_pos = 0;          // entries issued so far
  uint32_t st_dst = lds0;  // ring slot of the next one
  int st_list = 0, st_l = 0, st_left = 0;  // the item being copied: its list, the next lane, tiles left
  int st_at = 0, st_chunk = 0;             // the item, and the lists of 64 before this one
  const uint8_t *st_base = a0.k;           // what its tiles count from (the kv head of row 0)
  uint32_t st_last = 0;                    // bytes that the copies of its last tile may read
  // the item queued to be copied next, and the entry of its first tile once started
  bool nx_queued = false;
  int nx_list = 0, nx_left = 0, nx_at = 0, nx_first = 0;
  const uint8_t *nx_base = a0.k;
  uint32_t nx_last = 0;
  bool bad_seen = false;  // some tile lay in a missing page: from then on every tile is looked up
  auto list_of = [&](KernArgs &a, const Item &it, int chunk) -> int {
    const int i = it.lo + 64 * chunk + lane;
    int at = 0;
    if (i < it.hi) {
      const int tile = i < it.tl.ts ? i : i - it.tl.ts + it.tl.tlo;
      at = tile;
      if (paged) {
        const int per = a.block_size / kKeys, e = small_div(tile, per);
        const int blk = e < a.max_blocks ? a.block_tables[it.q.s * a.bt_stride + e] : -1;
        at = blk >= 0 && blk < a.num_blocks ? blk * per + (tile - e * per) : -1;
      }
    }
    bad_seen = uni(bad_seen | (__builtin_amdgcn_ballot_w64(at < 0) != 0)) != 0;
    return at;
  };
  auto queue = [&](const Item &it) {
    nx_queued = it.live && it.hi > it.lo;
    if (!nx_queued) return;
    KernArgs &a = *kernel_args();
    nx_list = list_of(a, it, 0);
    nx_at = it.at;
    nx_left = uni(it.hi - it.lo);
    nx_base = a.k + (paged ? 0 : static_cast<int64_t>(it.q.k0) * kv_rs) + h * SRC_ROWB;
    const int last = it.hi - 1 < it.tl.ts ? it.hi - 1 : it.hi - 1 - it.tl.ts + it.tl.tlo;
    nx_last = uni(min(kKeys, it.q.Lk - last * kKeys) * kv_rs);
  };
  // Source and readable bytes of the next entry's copies (0 bytes: zeros).
  auto next_tile = [&](const uint8_t *&src, uint32_t &nrec) {
    src = st_base;
    nrec = 0;
    if (st_left == 0 && nx_queued) {
      nx_queued = false;
      nx_first = st_pos;
      st_list = nx_list;
      st_l = 0;
      st_left = nx_left;
      st_at = nx_at;
      st_chunk = 0;
      st_base = nx_base;
      st_last = nx_last;
    }
    ++st_pos;
    if (st_left == 0) return;
    if (st_l == 64) {
      ++st_chunk;
      st_l = 0;
      st_list = list_of(*kernel_args(), describe(st_at), st_chunk);
      // (here, where the list is needed at once: a load that the compiler cannot
      // see waited for on every path, it waits for in the loop, with the copies)
      __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
    }
    const int at = __builtin_amdgcn_readlane(st_list, st_l);
    src = st_base + static_cast<int64_t>(static_cast<uint32_t>(max(at, 0))) * static_cast<uint32_t>(kKeys * kv_rs);
    nrec = at < 0 ? 0u : st_left == 1 ? st_last : static_cast<uint32_t>(kKeys * kv_rs);
    ++st_l;
    --st_left;
  };
  auto copy_k = [&](uint32_t dst, const uint8_t *src, uint32_t nrec) {
    dma16_group(dst + rw * COPS * 1024, rsrc_words(src, nrec), src_k);
  };
  auto copy_v = [&](uint32_t dst, const uint8_t *src, uint32_t nrec) {
    dma16_group(dst + TILE_B + rw * COPS * 1024, rsrc_words(src + v_minus_k, nrec), src_v);
  };

  // ---------------------------------------------------------------- operands
  // K operand kk: key rows m and m + 16, dims 32 kk + 8 g ..; V^T operand j:
  // keys 4 g + i and 16 + 4 g + i (the order of P), dims 16 j + m.
  uint32_t kbase_l, kx_l, vbase_l, vx_l;
  if constexpr (FP8) {
    const int s8 = 2 * swz8<D>(m);
    kbase_l = m * D + ((g ^ (s8 & 3)) << 3);
    kx_l = (s8 & ~3) << 3;
    const int rho = (lane & 15) >> 1, vp = lane & 1;
    const int r = rho < 4 ? 4 * g + rho : 12 + 4 * g + rho;
    vbase_l = r * D + (vp << 3);
    vx_l = (2 * swz8<D>(r)) << 3;
  } else {
    kbase_l = m * 2 * D + ((g ^ (swz_k(m) & 3)) << 4);
    kx_l = (swz_k(m) & 12) << 4;
    const int vk = (lane >> 2) & 3, vq = lane & 3;
    const int r0 = 4 * g + vk;
    vbase_l = r0 * 2 * D + (((vq >> 1) ^ (swz_v(r0) & 1)) << 4) + (vq & 1) * 8;
    vx_l = (swz_v(r0) & 14) << 4;
  }
  auto widen8 = [](const u32x2 &c) {
    return u32x4{T::template fp8x2<false>(c[0]), T::template fp8x2<true>(c[0]), T::template fp8x2<false>(c[1]),
                 T::template fp8x2<true>(c[1])};
  };
  // as read from LDS: 16-bit values, or fp8 codes that `op` widens
  using KV = std::conditional_t<FP8, u32x2, u32x4>;
  auto op = [&](const KV &x) -> u32x4 {
    if constexpr (FP8)
      return widen8(x);
    else
      return x;
  };
  auto k_read = [&](uint32_t kt, int kk, int ks) -> KV {
    if constexpr (FP8) {
      constexpr int KF = D == 128 ? 2 : 4;  // swz8: rows m + 16 flip this bit of kk
      const uint32_t at = (((ks ? kk ^ KF : kk) << 5) ^ kx_l) + (kt + kbase_l);
      return ks ? lds_load_b64<16 * D>(at) : lds_load_b64<0>(at);
    } else {
      const uint32_t at = ((kk << 6) ^ kx_l) + (kt + kbase_l);
      return ks ? lds_load_b128<16 * 2 * D>(at) : lds_load_b128<0>(at);
    }
  };
  auto v_read = [&](uint32_t kt, int j) -> KV {
    if constexpr (FP8) {
      return lds_load_tr8(((j << 4) ^ vx_l) + (kt + TILE_B + vbase_l));
    } else {
      const uint32_t at = ((j << 5) ^ vx_l) + (kt + TILE_B + vbase_l);
      const u32x2 lo = lds_load_tr16<0>(at), hi = lds_load_tr16<16 * 2 * D>(at);
      return u32x4{lo[0], lo[1], hi[0], hi[1]};
    }
  };
  // keeps the compiler from turning an operand's offset into one loop-invariant
  // register per operand
  auto unhoist = [&]() { asm volatile("" : "+v"(kx_l), "+v"(vx_l)); };

  // (never 0: a masked score, -inf, must stay that under a scale of 0)
  const float sl2 = FP8 ? fmaxf(a0.scale_log2 * ld_const(a0.k_scale + h), 0x1p-126f) : a0.scale_log2;

  constexpr int kAhead = RW == 1 ? SLOTS : SLOTS - 1;
  const uint8_t *src;
  uint32_t nrec;
  auto next_slot = [&](uint32_t x) { return x == lds0 + (SLOTS - 1) * SLOT_B ? lds0 : x + SLOT_B; };
  auto issue = [&]() {
    next_tile(src, nrec);
    copy_k(st_dst, src, nrec);
    copy_v(st_dst, src, nrec);
    st_dst = next_slot(st_dst);
  };

  // ---------------------------------------------------------------- items
  Item cur = describe(pos0);
  bool careful = false;  // (see odd_values)
  queue(cur);
  // the item whose output is still in registers
  struct Done {
    bool live, whole;
    int q0, r0, r_last, unit;
  };
  Done done{};
  int turn = 0;
  float m_use[QS], lsum[QS];
  float mref[QS];  // what P's exponents subtract: m_use, or 0 while a row has seen nothing
  f32x4 o[QS][NJ];
  for (;;) {
    // this wave's rows and their tokens (a wave past the last row sees no key
    // and stores nothing)
    const Seq q = cur.q;
    const int r0 = cur.r_first + rw * QS * 16, r_last = cur.r_last;
    const bool wave_live = cur.live && r0 <= r_last;
    const int t_first = cur.t_first, t_last = cur.t_last;
    int tok[QS];  // of this lane's rows
    u32x4 qf[QS][NKK];
    // Its copies, as far as they are not under way: the first item's, and those
    // behind items of few tiles, whose empty entries may lie in the slot that
    // another wave still works on.
    const bool tiles = cur.live && cur.hi > cur.lo;
    if (RW > 1 && tiles && (nx_queued || st_pos < nx_first + kAhead)) {
      wait_lgkmcnt0();
      raw_barrier();
    }
    if (tiles && nx_queued) issue();
    const int p0 = nx_first;  // entry of its first tile
    if (tiles)
      while (st_pos < p0 + kAhead) issue();
    // Q, with it the next item's list, then the output of the item before.  (No
    // live item: some row's.)
    KernArgs &a = *kernel_args();
#pragma unroll
    for (int qs = 0; qs < QS; ++qs) {
      const int r = cur.live ? min(r0 + 16 * qs + m, r_last) : 0;
      tok[qs] = small_div(r, a.G);
      const uint8_t *qp = a.q + static_cast<int64_t>(cur.live ? q.q0 + tok[qs] : 0) * a.q_rs +
                          (h * a.G + r - tok[qs] * a.G) * a.q_hs;
#pragma unroll
      for (int kk = 0; kk < NKK; ++kk) qf[qs][kk] = load16(qp + (8 * g + 32 * kk) * 2);
    }
    if (cur.live) queue(describe(cur.next));
    if (done.live) {
      const float vscale = FP8 ? ld_const(a.v_scale + h) : 1.f;
      // lane (m, g) holds dims 16 j + 4 g .. +3 of row 16 qs + m
#pragma unroll
      for (int qs = 0; qs < QS; ++qs) {
        const float l = sum32(sum16(lsum[qs]));
        const float inv = (l > 0.f ? 1.0f / l : 0.f) * vscale;
        const int r = done.r0 + 16 * qs + m;
        if (!done.whole) {
          const int64_t unit = static_cast<int64_t>(done.unit) + qs;
          f32x4 *po = reinterpret_cast<f32x4 *>(a.part_o) + unit * NJ * 64 + lane;
          if (r <= done.r_last) {
#pragma unroll
            for (int j = 0; j < NJ; ++j) po[j * 64] = o[qs][j] * inv;
            if (g == 0) a.part_l[unit * 16 + m] = l == 0.f ? kNegInf : m_use[qs] + __log2f(l);
          }
        } else if (r <= done.r_last) {
          const int t = small_div(r, a.G), head = h * a.G + r - t * a.G;
          uint8_t *op = a.out + static_cast<int64_t>(done.q0 + t) * a.o_rs + head * a.o_hs + 8 * g;
          const uint8_t *gp = a.gate + static_cast<int64_t>(done.q0 + t) * a.g_rs + head * a.g_hs + 8 * g;
#pragma unroll
          for (int j = 0; j < NJ; ++j) {
            const f32x4 v = o[qs][j] * inv;
            *reinterpret_cast<u32x2 *>(op + 32 * j) =
                a.gate ? gate4<T>(v, *reinterpret_cast<const u32x2 *>(gp + 32 * j))
                       : u32x2{T::pack2(v[0], v[1]), T::pack2(v[2], v[3])};
          }
        }
      }
    }
    if (!cur.live) break;
    {
      const Tiles tl = cur.tl;
      const int lo = cur.lo, hi = cur.hi, n = hi - lo;
      const int P = q.Lk - q.Lq;
      const int ta = uni(small_div(min(r0, r_last), a.G)), tb = uni(small_div(min(r0 + QS * 16 - 1, r_last), a.G));
      uint32_t slot = lds0 + (static_cast<unsigned>(p0) % SLOTS) * SLOT_B;  // of the tile computed next
      const int window = own_sgpr(a.window), sinks = own_sgpr(a.sinks);
      const bool tree = window == 0;
      if (tree) {
        // the masks of the tile's tokens, 32-bit words
        if constexpr (RW > 1) {  // the last item's have been read
          wait_lgkmcnt0();
          raw_barrier();
        }
        const int w32 = 2 * a.words, cnt = (t_last - t_first + 1) * w32;
        const uint32_t *mp = reinterpret_cast<const uint32_t *>(a.mask);
        for (int i = threadIdx.x; i < cnt; i += 64 * RW) {
          const int t = small_div(i, w32), c = i - t * w32;
          lds_mask[t * S::MASK_WORDS + c] = mp[(static_cast<int64_t>(q.q0 + t_first + t) * a.mask_rs) * 2 + c];
        }
        if constexpr (RW == 1)
          wave_lds_sync();
        else
          __syncthreads();
      }
      // The compiler waits for Q here, once (it counts the loads that it knows,
      // and waits for the copies in flight with them), not in the loop.
#pragma unroll
      for (int qs = 0; qs < QS; ++qs)
#pragma unroll
        for (int kk = 0; kk < NKK; ++kk) asm volatile("" : "+v"(qf[qs][kk]));
      asm volatile("" : "+v"(nx_list));
#pragma unroll
      for (int qs = 0; qs < QS; ++qs) {
        m_use[qs] = kNegInf;
        mref[qs] = 0.f;
        lsum[qs] = 0.f;
#pragma unroll
        for (int j = 0; j < NJ; ++j) o[qs][j] = f32x4{0, 0, 0, 0};
      }

      auto key_of = [&](int i) { return (i < tl.ts ? i : i - tl.ts + tl.tlo) * kKeys; };
      // List positions [first, first + count) of tiles that the tokens ta .. tb all
      // see whole, while no page is missing (sinks that a window does not reach
      // are not among them).
      struct Plain {
        int first;
        unsigned count;
      };
      auto plain_of = [&](int ta, int tb) -> Plain {
        int t0 = 0, t1;  // tiles
        if (!tree) {
          t0 = max(tl.ts == tl.tlo ? 0 : tl.tlo, (max(P + tb - window, -kKeys) + kKeys) / kKeys);
          t1 = max(0, P + ta + 1) / kKeys;
        } else {
          t1 = max(0, P) / kKeys;
        }
        return Plain{uni(t0 - tl.tlo + tl.ts), static_cast<unsigned>(uni(max(0, t1 - t0)))};
      };
      // Keys of the tile at `key0` that row block qs of this lane sees: bit
      // 4 ks + r for key 16 ks + 4 g + r.
      auto seen = [&](int qs, int key0) -> uint32_t {
        uint32_t v = 0;
        if (!tree) {
          const int top = P + tok[qs], bot = top - window;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int key = key0 + 16 * (i >> 2) + 4 * g + (i & 3);
            v |= (key <= top && (key > bot || key < sinks)) ? 1u << i : 0u;
          }
        } else {
          const int rel = key0 - P, w32 = 2 * kernel_args()->words;
          const uint32_t *mr = lds_mask + (tok[qs] - t_first) * S::MASK_WORDS;
          uint32_t bits;
          if (rel < 0) {
            bits = rel <= -32 ? ~0u : (mr[0] << -rel) | ((1u << -rel) - 1u);
          } else {
            const int c = rel >> 5, sh = rel & 31;
            const uint32_t b0 = c < w32 ? mr[c] : 0u, b1 = c + 1 < w32 ? mr[c + 1] : 0u;
            bits = sh ? (b0 >> sh) | (b1 << (32 - sh)) : b0;
          }
          const int left = q.Lk - key0;
          if (left < 32) bits &= (1u << left) - 1u;
          v = ((bits >> (4 * g)) & 15u) | (((bits >> (16 + 4 * g)) & 15u) << 4);
        }
        return v;
      };

      f32x4 sc[QS][2];  // scores of the tile whose P is formed next
      u32x4 pb[QS];     // P, in the second product's operand form
      uint32_t vis[QS];
      // The scores of keys that the rows do not see, replaced.  (Of a window, keys
      // past the sinks: one comparison of the distance to its first key.)
      auto missing = [&](int key0) -> bool {  // the tile's page
        KernArgs &a = *kernel_args();
        if (!paged) return false;
        const int e = small_div(key0 / kKeys, a.block_size / kKeys);
        const int blk = e < a.max_blocks ? ld_const(a.block_tables + q.s * a.bt_stride + e) : -1;
        return blk < 0 || blk >= a.num_blocks;
      };
      auto mask_tile = [&](int i, bool live) {
        const int key0 = key_of(i);
        if (!live || (bad_seen && missing(key0))) {
#pragma unroll
          for (int qs = 0; qs < QS; ++qs) {
            vis[qs] = 0;
            sc[qs][0] = sc[qs][1] = f32x4{kNegInf, kNegInf, kNegInf, kNegInf};
          }
          return;
        }
        if (!tree && !careful && key0 >= sinks) {
#pragma unroll
          for (int qs = 0; qs < QS; ++qs) {
            const int d0 = key0 + 4 * g - (P + tok[qs] - window + 1);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int d = d0 + 16 * (e >> 2) + (e & 3);
              sc[qs][e >> 2][e & 3] = static_cast<unsigned>(d) < static_cast<unsigned>(window) ? sc[qs][e >> 2][e & 3] : kNegInf;
            }
          }
          return;
        }
#pragma unroll
        for (int qs = 0; qs < QS; ++qs) {
          vis[qs] = seen(qs, key0);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (!((vis[qs] >> e) & 1u)) sc[qs][e >> 2][e & 3] = kNegInf;
        }
      };
      // The rows' maxima over the tile's scores against the running ones.  A maximum moves when some score exceeds it by
      // more than kRescale; then every row's is brought up to date, alpha holds
      // the factors for o, and the result is true.
      auto check = [&](float (&alpha)[QS]) -> bool {
        float mloc[QS];
        bool grow = false;
#pragma unroll
        for (int qs = 0; qs < QS; ++qs) {
          mloc[qs] = max3(max3(sc[qs][0][0], sc[qs][0][1], sc[qs][0][2]),
                          max3(sc[qs][0][3], sc[qs][1][0], sc[qs][1][1]),
                          __builtin_elementwise_maximum(sc[qs][1][2], sc[qs][1][3])) * sl2;
          grow |= mloc[qs] > m_use[qs] + kRescale;
        }
        if (__builtin_amdgcn_ballot_w64(grow) == 0) return false;
#pragma unroll
        for (int qs = 0; qs < QS; ++qs) {
          const float mn = fmaxf(m_use[qs], max32_raw(max16_raw(mloc[qs])));
          alpha[qs] = m_use[qs] == kNegInf ? 0.f : __builtin_amdgcn_exp2f(m_use[qs] - mn);
          lsum[qs] *= alpha[qs];
          m_use[qs] = mn;
          mref[qs] = mn == kNegInf ? 0.f : mn;
        }
        return true;
      };
      auto rescale = [&](const float (&alpha)[QS]) {
#pragma unroll
        for (int qs = 0; qs < QS; ++qs)
#pragma unroll
          for (int j = 0; j < NJ; ++j) o[qs][j] *= alpha[qs];
      };
      // Elements 2 t, 2 t + 1 of a row block: P, its sum, packed.
      auto p_unit = [&](int qs, int t) -> uint32_t {
        const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[qs][t >> 1][2 * (t & 1)], sl2, -mref[qs]));
        const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[qs][t >> 1][2 * (t & 1) + 1], sl2, -mref[qs]));
        lsum[qs] += e0 + e1;
        return T::pack2(e0, e1);
      };
      auto scores = [&](uint32_t kt) {
#pragma unroll
        for (int qs = 0; qs < QS; ++qs) sc[qs][0] = sc[qs][1] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int kk = 0; kk < NKK; ++kk)
#pragma unroll
          for (int ks = 0; ks < 2; ++ks) {
            const u32x4 kf = op(k_read(kt, kk, ks));
#pragma unroll
            for (int qs = 0; qs < QS; ++qs) sc[qs][ks] = T::mfma16x16x32(kf, qf[qs][kk], sc[qs][ks]);
          }
      };
      // 0 * NaN must not reach a row through a key it does not see.  An item whose
      // outputs are not all finite is done again, carefully: when a tile that not
      // every row sees whole then holds values that are not finite
      // (`odd_values`), `poison` adds them to the outputs of the rows that see
      // them and `clean` takes them out of the tile.  The waves that share the
      // tile check and clean a part of it each.
      constexpr uint32_t kExp = T::dtype == NQ_BF16 ? 0x7f80u : 0x7c00u;
      constexpr uint32_t kMant = T::dtype == NQ_BF16 ? 0x007fu : 0x03ffu;
      // top bit of every half (fp8: byte) of w that is not finite: its exponent
      // (and, of e4m3, its mantissa) is all ones, and the carry reaches that bit
      auto odd_bits = [](uint32_t w) -> uint32_t {
        if constexpr (FP8) return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
        constexpr uint32_t e = kExp | kExp << 16, lsb = (kMant + 1) | (kMant + 1) << 16;
        return ((w & e) + lsb) & 0x80008000u;
      };
      constexpr int kPart = TILE_B / RW / 64;  // bytes of the tile's values per lane
      auto part_of = [&](uint32_t kt, int c) { return kt + TILE_B + (rw * (kPart / 16) + c) * 1024 + lane * 16; };
      uint32_t *const lds_odd = reinterpret_cast<uint32_t *>(smem + S::ODD_AT);
      auto odd_values = [&](uint32_t kt) -> bool {
        uint32_t any = 0;
#pragma unroll 2
        for (int c = 0; c < kPart / 16; ++c) {
          const u32x4 x = lds_load_b128<0>(part_of(kt, c));
          any |= odd_bits(x[0]) | odd_bits(x[1]) | odd_bits(x[2]) | odd_bits(x[3]);
        }
        bool odd = __builtin_amdgcn_ballot_w64(any != 0) != 0;
        if constexpr (RW > 1) {
          if (lane == 0) lds_odd[rw] = odd;
          wait_lgkmcnt0();
          raw_barrier();
          odd = __builtin_amdgcn_ballot_w64(lane < RW && lds_odd[lane & (RW - 1)] != 0) != 0;
        }
        return odd;
      };
      auto clean = [&](uint32_t kt) {
        wait_lgkmcnt0();
        if constexpr (RW > 1) raw_barrier();  // every wave has looked at the tile
#pragma unroll 1
        for (int c = 0; c < kPart / 16; ++c) {
          u32x4 x = lds_load_b128<0>(part_of(kt, c));
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const uint32_t b = odd_bits(x[t]);
            x[t] &= ~((b - (b >> (FP8 ? 7 : 15))) | b);
          }
          lds_store_b128(part_of(kt, c), x);
        }
        wait_lgkmcnt0();
        if constexpr (RW > 1) raw_barrier();
      };
      // This lane's outputs (dims 16 j + 4 g + r of its rows) from every value
      // that is not finite and whose key the row sees.  Rare: written for size.
      auto poison = [&](uint32_t kt) {
#pragma unroll
        for (int qs = 0; qs < QS; ++qs) {
          uint64_t nan = 0, up = 0, down = 0;  // bit 4 j + r
#pragma unroll 1
          for (int key = 0; key < kKeys; ++key) {
            const uint32_t theirs = __shfl(vis[qs], ((key >> 2) & 3) * 16 + m);  // of the lane that holds the key
            if (!((theirs >> (4 * (key >> 4) + (key & 3))) & 1u)) continue;
#pragma unroll 1
            for (int j = 0; j < NJ; ++j) {
              if constexpr (FP8) {
                const uint32_t at = kt + TILE_B + key * D + ((j ^ swz8<D>(key)) << 4) + 4 * g;
                const uint32_t x = *reinterpret_cast<const __attribute__((address_space(3))) uint32_t *>(
                    static_cast<uintptr_t>(at));
#pragma unroll
                for (int r = 0; r < 4; ++r)
                  nan |= static_cast<uint64_t>(((x >> (8 * r)) & 0x7fu) == 0x7fu) << (4 * j + r);
              } else {
                const u32x2 x = lds_load_b64<0>(kt + TILE_B + key * 2 * D + (((2 * j + (g >> 1)) ^ swz_v(key)) << 4) +
                                                (g & 1) * 8);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                  const uint32_t e = (x[r >> 1] >> (16 * (r & 1))) & 0xffffu;
                  const uint64_t odd = (e & kExp) == kExp, is_nan = odd && (e & kMant) != 0;
                  nan |= is_nan << (4 * j + r);
                  up |= static_cast<uint64_t>(odd && !is_nan && !(e & 0x8000u)) << (4 * j + r);
                  down |= static_cast<uint64_t>(odd && !is_nan && (e & 0x8000u)) << (4 * j + r);
                }
              }
            }
          }
#pragma unroll
          for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              // added as bits (a bit's sign extension and the value's): no select per output
              const int bit = (4 * j + r) & 31;
              auto term = [&](uint64_t set, uint32_t value) {
                const uint32_t half = static_cast<uint32_t>(4 * j + r < 32 ? set : set >> 32);
                return u2f(static_cast<uint32_t>(__builtin_amdgcn_sbfe(static_cast<int>(half), bit, 1)) & value);
              };
              o[qs][j][r] += term(nan, 0x7fc00000u);
              if constexpr (!FP8) o[qs][j][r] = (o[qs][j][r] + term(up, 0x7f800000u)) + term(down, 0xff800000u);
            }
        }
      };
      float alpha[QS];
      if constexpr (RW == 1) {
        const Plain plain = plain_of(ta, tb);
        // The new token: the piece that holds the sequence's last tile (or the
        // item without tiles) stores its rows, and takes them from there for the
        // tile, when its cache row is the one they go to: the store and the
        // attention need no order.
        uint8_t *const lds_new = smem + S::NEW_AT;
        int new_row = -1;  // of the last tile
        if (a.k_new && hi == tl.n) {
          const int slot_of = ld_const(a.slot_mapping + q.s), have = ld_const(a.cu_k + q.s);
          if (n > 0 && have == q.Lk) {
            const int at = q.Lk - 1, e = small_div(at / kKeys, a.block_size / kKeys);
            const int blk = e < a.max_blocks ? ld_const(a.block_tables + q.s * a.bt_stride + e) : -1;
            if (blk >= 0 && blk < a.num_blocks &&
                slot_of == static_cast<int64_t>(blk) * a.block_size + (at - e * a.block_size))
              new_row = at % kKeys;
          }
          constexpr int NC = D / 8;  // lane l: elements 8 c .. of K (l < NC) or V
          const bool is_v = lane >= NC;
          const int c = is_v ? lane - NC : lane;
          if (lane < 2 * NC) {
            const uint8_t *row = is_v ? a.v_new + q.s * a.vn_rs : a.k_new + q.s * a.kn_rs;
            uint8_t *cache = const_cast<uint8_t *>(is_v ? a.v : a.k) + slot_of * a.kv_rs + h * SRC_ROWB;
            const bool stored = slot_of >= 0 && slot_of < static_cast<int64_t>(a.num_blocks) * a.block_size;
            if constexpr (FP8) {
              float x[8];
              if (a.new_dtype == NQ_F32) {
                const float *f = reinterpret_cast<const float *>(row) + h * D + 8 * c;
                const f32x4 w0 = *reinterpret_cast<const f32x4 *>(f), w1 = *reinterpret_cast<const f32x4 *>(f + 4);
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                  x[t] = w0[t];
                  x[4 + t] = w1[t];
                }
              } else {
                const u32x4 w = load16(row + (h * D + 8 * c) * 2);
#pragma unroll
                for (int t = 0; t < 8; ++t) {
                  const uint16_t b = static_cast<uint16_t>(w[t >> 1] >> (16 * (t & 1)));
                  x[t] = a.new_dtype == NQ_F16 ? F16::to_float(b) : BF16::to_float(b);
                }
              }
              const float inv = 1.0f / (is_v ? a.v_scale : a.k_scale)[h];
              const u32x2 codes{fp8x4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv),
                                fp8x4(x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv)};
              if (stored) *reinterpret_cast<u32x2 *>(cache + 8 * c) = codes;
              *reinterpret_cast<u32x2 *>(lds_new + (is_v ? SRC_ROWB : 0) + 8 * c) = codes;
            } else {
              const u32x4 w = load16(row + (h * D + 8 * c) * 2);
              if (stored) store16(cache + 16 * c, w);
              *reinterpret_cast<u32x4 *>(lds_new + (is_v ? SRC_ROWB : 0) + 16 * c) = w;
            }
          }
          wave_lds_sync();
        }
        // the row over the one that was copied, a 16-byte piece per lane
        auto patch = [&](uint32_t tile, bool is_v) {
          if (lane < S::LPR) {
            const u32x4 w = *reinterpret_cast<const u32x4 *>(lds_new + (is_v ? SRC_ROWB : 0) + 16 * lane);
            const int sw = FP8 ? swz8<D>(new_row) : is_v ? swz_v(new_row) : swz_k(new_row);
            lds_store_b128(tile + (is_v ? TILE_B : 0) + new_row * SRC_ROWB + ((lane ^ sw) << 4), w);
          }
          wave_lds_sync();
        };
        for (int i = lo; i < hi; ++i) {
          wait_vmcnt<(2 * SLOTS - 1) * COPS>();  // K of this tile (younger: its V and the tiles after it)
          asm volatile("" ::: "memory");
          const bool patched = new_row >= 0 && i == tl.n - 1;
          if (patched) patch(slot, false);
          scores(slot);
          wait_lgkmcnt0();  // the K operands are read: the slot's K is free
          const bool whole_tile = static_cast<unsigned>(i - plain.first) < plain.count && !bad_seen;
          if (!whole_tile) mask_tile(i, true);
          next_tile(src, nrec);
          copy_k(slot, src, nrec);
          if (check(alpha)) rescale(alpha);
#pragma unroll
          for (int t = 0; t < 4; ++t) pb[0][t] = p_unit(0, t);
          wait_vmcnt<(2 * SLOTS - 1) * COPS>();  // V of this tile
          asm volatile("" ::: "memory");
          if (patched) patch(slot, true);
          if (careful && !whole_tile && odd_values(slot)) {
            poison(slot);
            clean(slot);
          }
#pragma unroll
          for (int j = 0; j < NJ; ++j) o[0][j] = T::mfma16x16x32(op(v_read(slot, j)), pb[0], o[0][j]);
          wait_lgkmcnt0();
          copy_v(slot, src, nrec);
          slot = next_slot(slot);
          st_dst = next_slot(st_dst);
        }
      } else if (n > 0) {
        // One tile per step, three tiles at work: P of tile i is formed among the
        // products of P V of tile i - 1, and the V operands of tile i are read
        // among the products of K Q of tile i + 1, so that the matrix core, the
        // exponentials and the LDS reads overlap within a wave.
        constexpr int NP = NJ * QS, U = 4 * QS, PPU = NP / U;  // products of P V, units of P, products per unit
        constexpr int CV = FP8 ? 4 * NJ / U : 0;               // conversions per unit
        constexpr int NQ = NKK * 2 * QS, PPV = NQ / NJ;        // products of K Q, of them per V operand
        static_assert(PPU == 2 || PPU == 4, "2 or 4 products per unit of P");
        static_assert(PPV == 1 || PPV == 2, "one V operand per one or two products");
        KV vf[NJ];  // V operands of the tile whose products are pending
        const Plain plain_w = wave_live ? plain_of(ta, tb) : Plain{0, 0}, plain_wg = plain_of(t_first, t_last);
        bool pend = false;
        auto step = [&](auto first_tag, int i) {
          constexpr bool FIRST = decltype(first_tag)::value;
          unhoist();
          if (!FIRST && pend) rescale(alpha);  // tile i - 1's maxima, before its products join o
          const bool whole_tile = static_cast<unsigned>(i - plain_w.first) < plain_w.count && !bad_seen;
          if (!whole_tile) mask_tile(i, wave_live);
          pend = check(alpha);
          // (for all of the workgroup's waves alike)
          if (careful && !(static_cast<unsigned>(i - plain_wg.first) < plain_wg.count && !bad_seen) && odd_values(slot)) {
            // o is brought up to date before the odd values join it
            if constexpr (!FIRST) {
#pragma unroll
              for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int qs = 0; qs < QS; ++qs) o[qs][j] = T::mfma16x16x32(op(vf[j]), pb[qs], o[qs][j]);
#pragma unroll
              for (int j = 0; j < NJ; ++j) vf[j] = KV{};
            }
            if (pend) rescale(alpha);
            pend = false;
            if (whole_tile) {
#pragma unroll
              for (int qs = 0; qs < QS; ++qs) vis[qs] = 0xffu;
            }
            poison(slot);
            clean(slot);
          }
          issue();
          KV kf[NKK][2];
          {
            const uint32_t slot_next = next_slot(slot);
#pragma unroll
            for (int kk = 0; kk < NKK; ++kk)
#pragma unroll
              for (int ks = 0; ks < 2; ++ks) kf[kk][ks] = k_read(slot_next, kk, ks);
            uint32_t pw[QS][4];
            if constexpr (FIRST) {
#pragma unroll
              for (int u = 0; u < U; ++u) pw[u / 4][u % 4] = p_unit(u / 4, u % 4);
            } else {
              u32x4 vw[NJ];
              constexpr int JPU = NJ / U > 0 ? NJ / U : 1;  // V operands per unit (rounded up)
#pragma unroll
              for (int j = 0; j < JPU; ++j) vw[j] = op(vf[j]);
#pragma unroll
              for (int x = 0; x < NP; ++x) {
                const int j = x / QS, qs = x % QS, u = x / PPU;
                if (FP8 && x % PPU == 0) {
#pragma unroll
                  for (int jn = (u + 1) * NJ / U; jn < (u + 2) * NJ / U && jn < NJ; ++jn)
                    if (jn >= JPU) vw[jn] = op(vf[jn]);
                }
                o[qs][j] = T::mfma16x16x32(FP8 ? vw[j] : op(vf[j]), pb[qs], o[qs][j]);
                if (x % PPU == PPU - 1) pw[u / 4][u % 4] = p_unit(u / 4, u % 4);
              }
              if (FP8) __builtin_amdgcn_sched_group_barrier(0x002, CV, 0);  // VALU: the first operands
#pragma unroll
              for (int u = 0; u < U; ++u) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                // MFMA
                __builtin_amdgcn_sched_group_barrier(0x002, 2 + CV / 2, 0);       // VALU
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                // MFMA
                __builtin_amdgcn_sched_group_barrier(0x400, 2, 0);                // transcendental
                if (PPU == 4) __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
                __builtin_amdgcn_sched_group_barrier(0x002, 3 + CV - CV / 2, 0);  // VALU
                if (PPU == 4) __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
                // DS read (K): halfway; fp8 codes (half the registers) after the first unit
                if (u == (FP8 ? 0 : U / 2 - 1)) __builtin_amdgcn_sched_group_barrier(0x100, 2 * NKK, 0);
              }
            }
#pragma unroll
            for (int qs = 0; qs < QS; ++qs) pb[qs] = u32x4{pw[qs][0], pw[qs][1], pw[qs][2], pw[qs][3]};
          }
          __builtin_amdgcn_sched_barrier(0);  // the two sections are scheduled apart
          {
            f32x4 sn[QS][2];
#pragma unroll
            for (int qs = 0; qs < QS; ++qs) sn[qs][0] = sn[qs][1] = f32x4{0, 0, 0, 0};
            u32x4 kw[NKK][2];  // fp8: each K operand widened while the one before it is at work
            if constexpr (FP8) kw[0][0] = op(kf[0][0]);
#pragma unroll
            for (int x = 0; x < NQ; ++x) {
              const int kk = x / (2 * QS), ks = (x / QS) % 2, qs = x % QS;
              if (FP8 && qs == 0 && 2 * kk + ks + 1 < 2 * NKK) {
                const int nx = 2 * kk + ks + 1;
                kw[nx >> 1][nx & 1] = op(kf[nx >> 1][nx & 1]);
              }
              sn[qs][ks] = T::mfma16x16x32(FP8 ? kw[kk][ks] : op(kf[kk][ks]), qf[qs][kk], sn[qs][ks]);
              if (x % PPV == 0) vf[x / PPV] = v_read(slot, x / PPV);
            }
            constexpr int CK = FP8 ? 4 / QS : 0;  // conversions per product
            if (FP8) __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);  // VALU: the first K operand
#pragma unroll
            for (int x = 0; x < NQ; ++x) {
              __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);        // MFMA
              __builtin_amdgcn_sched_group_barrier(0x100, 2 / PPV, 0);  // DS read
              if (FP8) __builtin_amdgcn_sched_group_barrier(0x002, CK, 0);
            }
#pragma unroll
            for (int qs = 0; qs < QS; ++qs) {
              sc[qs][0] = sn[qs][0];
              sc[qs][1] = sn[qs][1];
            }
          }
          slot = next_slot(slot);
        };
        wait_vmcnt<2 * COPS * (kAhead - 1)>();  // this wave's part of the first tile
        raw_barrier();
        unhoist();
        scores(slot);
        // Tile i + 1 has landed, and tile i - 1's slot is free.
        auto sync = [&]() {
          wait_vmcnt<2 * COPS * (kAhead - 2)>();
          wait_lgkmcnt0();
          raw_barrier();
        };
        sync();
        step(std::true_type{}, lo);
        for (int i = lo + 1; i < hi; ++i) {
          sync();
          step(std::false_type{}, i);
        }
        if (pend) rescale(alpha);
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int qs = 0; qs < QS; ++qs) o[qs][j] = T::mfma16x16x32(op(vf[j]), pb[qs], o[qs][j]);
      }

      // outputs that are not finite: carefully, again (every wave alike)
      float zero = 0.f;
#pragma unroll
      for (int qs = 0; qs < QS; ++qs)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) zero = __builtin_fmaf(o[qs][j][r], 0.f, zero);
      bool again = __builtin_amdgcn_ballot_w64(zero != 0.f) != 0;
      if constexpr (RW > 1) {
        // (flags by turns: a wave may be an item ahead of another's reads)
        uint32_t *const flags = lds_odd + 8 + (turn & 1) * 8;
        ++turn;
        if (lane == 0) flags[rw] = again;
        wait_lgkmcnt0();
        raw_barrier();
        again = __builtin_amdgcn_ballot_w64(lane < RW && flags[lane & (RW - 1)] != 0) != 0;
      }
      if (again && !careful) {
        // the copies under way are given up, and the item is queued anew
        wait_vmcnt<0>();
        wait_lgkmcnt0();
        if constexpr (RW > 1) raw_barrier();
        st_left = 0;
        careful = true;
        queue(cur);
        done.live = false;
        continue;
      }
      const bool whole = lo == 0 && hi == tl.n;
      done = Done{true, whole, q.q0, r0, r_last, ((2 * w_of + (lo > 0 ? 0 : 1)) * RW + rw) * QS};
      if (!whole) {
        const int at = lo > 0 ? 0 : 1;
        cuts |= 1 << at;
        if (rw == 0 && lane == 0)
          kernel_args()->part_desc[2 * w_of + at] = int4{q.s, cur.rt, hi == tl.n ? kPieceLast : kPieceMore, 0};
      }
    }
    cur = describe(cur.next);
    careful = false;
  }
  if (ranges && rw == 0 && lane == 0) {
    int4 *d = kernel_args()->part_desc + 2 * w_of;
    const int4 none{0, 0, kPieceNone, 0};
    if (!(cuts & 1)) d[0] = none;
    if (!(cuts & 2)) d[1] = none;
  }
  wait_vmcnt<0>();  // no copy outlives the workgroup's LDS
}

template <class T, bool FP8, class S>
__global__ __launch_bounds__(64 * S::RW) __attribute__((amdgpu_waves_per_eu(S::RW == 1 ? 1 : 2)))
void span_attention_kernel(const SpanArgs a) {
  span_body<T, FP8, S>();
}

// Merge of the items that ranges cut: workgroup (range, part) takes the item
// whose first piece lies in the range's slot 1; its other pieces are the slots
// 0 of the next ranges, up to the one marked last.  A wave takes J 16-dim
// blocks of one row block, kMergeUnroll pieces in flight: the chain is two round
// trips to memory and one per eight pieces, or per 32 where SPREAD = 4 waves
// share them and join through LDS.  Latency bounds it (4-6 us, half of that the
// launch), or reading the partials: 13 us for trees of 16-32 nodes, 16 sequences.
constexpr int kMergeUnroll = 8;
template <class S>
struct MergeShape {
  static constexpr int J = S::NJ >= 16 ? 4 : S::RW == 1 ? 2 : 4;
  static constexpr int WAVES = S::RW * S::QS * S::NJ / J;
  static_assert(WAVES % 4 == 0, "workgroups of four waves");
};
template <class T, class S, int SPREAD>
__global__ __launch_bounds__(256) void span_merge_kernel(const SpanArgs a) {
  constexpr int NJ = S::NJ, M = S::M, J = MergeShape<S>::J;
  const int w = blockIdx.x, h = w / a.n_ranges, w_end = (h + 1) * a.n_ranges;
  const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const int4 d = a.part_desc[2 * w + 1];
  auto kind = [&](int b) { return a.part_desc[2 * min(b + lane, w_end - 1)].z; };
  int next = kind(w + 1);
  if (d.z == kPieceNone) return;
  const int wave = threadIdx.x >> 6, e = SPREAD > 1 ? blockIdx.y : blockIdx.y * 4 + wave;
  const int unit = e / (NJ / J), j0 = e % (NJ / J) * J;
  const Seq q = seq_of(a, d.x, true);
  const int r = d.y * M + unit * 16 + m;
  int pieces = 1;
  for (int b = w + 1;; b += 64) {
    const uint64_t last = __builtin_amdgcn_ballot_w64(b + lane < w_end && next == kPieceLast);
    if (last != 0) {
      pieces += static_cast<int>(__builtin_ctzll(last)) + 1;
      break;
    }
    if (b + 64 >= w_end) return;  // not reached: every cut item has a last piece
    pieces += 64;
    next = kind(b + 64);
  }
  const bool live = r < q.Lq * a.G;
  float mx = kNegInf, W = 0.f;
  f32x4 acc[J];
#pragma unroll
  for (int j = 0; j < J; ++j) acc[j] = f32x4{0, 0, 0, 0};
  for (int c = (SPREAD > 1 ? wave * kMergeUnroll : 0); c < pieces; c += SPREAD * kMergeUnroll) {
    float l[kMergeUnroll];
    f32x4 p[kMergeUnroll][J];
#pragma unroll
    for (int u = 0; u < kMergeUnroll; ++u) {
      l[u] = kNegInf;
      if (live && c + u < pieces) {
        const int64_t at = static_cast<int64_t>(2 * (w + c + u) + (c + u == 0 ? 1 : 0)) * S::RW * S::QS + unit;
        l[u] = a.part_l[at * 16 + m];
#pragma unroll
        for (int j = 0; j < J; ++j) p[u][j] = reinterpret_cast<const f32x4 *>(a.part_o)[(at * NJ + j0 + j) * 64 + lane];
      }
    }
    float mc = mx;
#pragma unroll
    for (int u = 0; u < kMergeUnroll; ++u) mc = fmaxf(mc, l[u]);
    const float mu = mc == kNegInf ? 0.f : mc;
    const float f = __builtin_amdgcn_exp2f(mx - mu);
    W *= f;
#pragma unroll
    for (int j = 0; j < J; ++j) acc[j] *= f;
    mx = mc;
#pragma unroll
    for (int u = 0; u < kMergeUnroll; ++u)
      if (l[u] != kNegInf) {
        const float x = __builtin_amdgcn_exp2f(l[u] - mu);
        W += x;
#pragma unroll
        for (int j = 0; j < J; ++j) acc[j] += p[u][j] * x;
      }
  }
  if constexpr (SPREAD > 1) {
    if (pieces > kMergeUnroll) {
      __shared__ float states[SPREAD - 1][J * 4 + 2][64];
      if (wave > 0) {
        float(*const st)[64] = states[wave - 1];
#pragma unroll
        for (int i = 0; i < 4 * J; ++i) st[i][lane] = acc[i >> 2][i & 3];
        st[4 * J][lane] = mx;
        st[4 * J + 1][lane] = W;
      }
      __syncthreads();
      if (wave == 0) {
#pragma unroll
        for (int u = 0; u < SPREAD - 1; ++u) {
          const float mo = states[u][4 * J][lane], mn = fmaxf(mx, mo), mu = mn == kNegInf ? 0.f : mn;
          const float f0 = __builtin_amdgcn_exp2f(mx - mu), f1 = __builtin_amdgcn_exp2f(mo - mu);
          W = W * f0 + states[u][4 * J + 1][lane] * f1;
#pragma unroll
          for (int i = 0; i < 4 * J; ++i) acc[i >> 2][i & 3] = acc[i >> 2][i & 3] * f0 + states[u][i][lane] * f1;
          mx = mn;
        }
      }
    }
    if (wave > 0) return;
  }
  if (!live) return;
  const float inv = W > 0.f ? 1.0f / W : 0.f;
  const int t = small_div(r, a.G), head = h * a.G + r - t * a.G;
  uint8_t *op = a.out + static_cast<int64_t>(q.q0 + t) * a.o_rs + head * a.o_hs + 32 * j0 + 8 * g;
  const uint8_t *gp = a.gate + static_cast<int64_t>(q.q0 + t) * a.g_rs + head * a.g_hs + 32 * j0 + 8 * g;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const f32x4 v = acc[j] * inv;
    *reinterpret_cast<u32x2 *>(op + 32 * j) =
        a.gate ? gate4<T>(v, *reinterpret_cast<const u32x2 *>(gp + 32 * j))
               : u32x2{T::pack2(v[0], v[1]), T::pack2(v[2], v[3])};
  }
}

// ---------------------------------------------------------------- launch
int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }

template <class T, bool FP8, class S>
int launch(SpanArgs a, int64_t max_rows, int per_cu, void *workspace, int64_t workspace_bytes, int64_t *need,
           hipStream_t stream) {
  // row tiles of the batch, at most: every sequence's last one may be partial
  const int64_t by_total = static_cast<int64_t>(a.total_q) * a.G / S::M + a.num_seqs;
  const int64_t items = std::min(by_total, a.num_seqs * ((max_rows + S::M - 1) / S::M));
  const int64_t slots = static_cast<int64_t>(device_cus()) * per_cu;
  const int64_t max_tiles = (static_cast<int64_t>(a.max_k) + kKeys - 1) / kKeys, max_cost = max_tiles + Cost<S>::kItem;
  a.n_ranges = 0;
  // the tiles that an item can have: all, or those of its tokens' windows and the sinks'
  int64_t item_tiles = max_tiles;
  if (a.window > 0)
    item_tiles = std::min(item_tiles, (static_cast<int64_t>(a.window) + a.sinks + std::min<int64_t>(S::M, max_rows)) / kKeys + 2);
  // Equal ranges where they beat whole items, whose last round may be nearly empty
  // (both as if every item were as large as it can be).  Measured, whole items
  // against ranges, D = 128, 8 kv heads, window 1024: one prompt of 512 tokens 24
  // against 27 us, 1024 37 - 42, 2048 51 - 55, 8192 176 - 177; chats of 81-333
  // tokens behind 4000-8000 fp8 ones, four of them, 43 - 47; decode of 64 rows
  // 49 - 54, of 256 206 - 211.  The other way round: trees of 32 nodes for 16
  // sequences of 4096 111 - 77, decode of one row 31 - 14.
  const int64_t n = items * a.Hkv, c = item_tiles + Cost<S>::kItem, rounds = (n + slots - 1) / slots;
  const bool cut = rounds * c * slots > n * c + Cost<S>::kCut * slots;
  if (cut && by_total * max_cost < (int64_t{1} << 31)) {
    const int per = a.Hkv < 8 && 8 % a.Hkv == 0 ? 8 / a.Hkv : 1;
    a.min_range = static_cast<int>(std::max<int64_t>(Cost<S>::kMinRange, item_tiles / Cost<S>::kPieces));
    const int64_t most = by_total * max_cost / a.min_range + 1;  // ranges that can have work
    int64_t W = std::max<int64_t>(1, std::min(slots / a.Hkv, most));
    W = (W + per - 1) / per * per;
    const int64_t parts = W * a.Hkv * 2;
    const int64_t o_bytes = align256(parts * S::M * S::D * 4), l_bytes = align256(parts * S::M * 4);
    const int64_t bytes = o_bytes + l_bytes + align256(parts * 16);
    if (!workspace || workspace_bytes < bytes) {
      if (!need)
        return fail(NQ_EINVAL, "span attention: workspace %lld bytes < %lld", (long long)workspace_bytes,
                    (long long)bytes);
      *need = bytes;
      return 1;
    }
    if (!aligned(workspace, 256)) return fail(NQ_EINVAL, "span attention: workspace must be 256-byte aligned");
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    a.n_ranges = static_cast<int>(W);
    a.part_o = reinterpret_cast<float *>(ws);
    a.part_l = reinterpret_cast<float *>(ws + o_bytes);
    a.part_desc = reinterpret_cast<int4 *>(ws + o_bytes + l_bytes);
    span_attention_kernel<T, FP8, S><<<dim3(static_cast<unsigned>(W * a.Hkv)), 64 * S::RW, S::LDS_B, stream>>>(a);
    const int rc = check_launch("span attention");
    if (rc != NQ_OK || W <= 1) return rc;
    const unsigned n_wg = static_cast<unsigned>(W * a.Hkv);
    // Four waves to an element where items have many pieces, unless that is many
    // workgroups: decode of one row 14.4 us against 15.4 with one wave, a tree of 4
    // nodes behind 8192 tokens 21 against 26 (2080 workgroups); of 32 rows of 4096 fp8
    // tokens (4 pieces each) 67 against 61, and trees of 4 nodes for 16 sequences at
    // D = 256, fp8 (16 pieces each, 4096 workgroups) 59 against 52.
    if (W > kMergeUnroll * items && n_wg * MergeShape<S>::WAVES < 16u * static_cast<unsigned>(device_cus()))
      span_merge_kernel<T, S, 4><<<dim3(n_wg, MergeShape<S>::WAVES), 256, 0, stream>>>(a);
    else
      span_merge_kernel<T, S, 1><<<dim3(n_wg, MergeShape<S>::WAVES / 4), 256, 0, stream>>>(a);
    return check_launch("span attention (merge)");
  }
  // Whole items, dealt out in turn to the workgroups that the chip holds at once
  // (a multiple of 8 where kv heads share XCDs, and of the kv heads otherwise).
  const int per = a.Hkv < 8 && 8 % a.Hkv == 0 ? 8 / a.Hkv : 1;
  const int64_t unit = static_cast<int64_t>(a.Hkv) * per;
  const int64_t grid = unit * std::max<int64_t>(1, std::min((items + per - 1) / per, slots / unit));
  a.stride = static_cast<int>(grid / a.Hkv);
  span_attention_kernel<T, FP8, S><<<dim3(static_cast<unsigned>(grid)), 64 * S::RW, S::LDS_B, stream>>>(a);
  return check_launch("span attention");
}

template <class T, bool FP8>
int launch_shape(const SpanArgs &a, int D, int64_t max_rows, void *ws, int64_t ws_bytes, int64_t *need, hipStream_t s) {
  // The smallest shape that holds the longest sequence's rows.  One row block in
  // the four waves' shape: decode of 32 rows of 4096 tokens 110 us against 107, of
  // fp8 80 against 58.  Up to 64 rows in the largest: trees of 8 nodes for 16
  // sequences of 4096 61 against 59, fp8 64 against 50 (D = 256: 67 against 59).
  if (D == 256) {
    if (max_rows <= 16)
      return launch<T, FP8, Shape<256, FP8, 1, 1, 2>>(a, max_rows, FP8 ? 4 : 2, ws, ws_bytes, need, s);
    if (max_rows <= 64)
      return launch<T, FP8, Shape<256, FP8, 4, 1, 4>>(a, max_rows, FP8 ? 2 : 1, ws, ws_bytes, need, s);
    return launch<T, FP8, Shape<256, FP8, 8, 1, 4>>(a, max_rows, 1, ws, ws_bytes, need, s);
  }
  if (max_rows <= 16)
    return launch<T, FP8, Shape<128, FP8, 1, 1, FP8 ? 4 : 2>>(a, max_rows, 4, ws, ws_bytes, need, s);
  if (max_rows <= 64) return launch<T, FP8, Shape<128, FP8, 4, 1, 4>>(a, max_rows, 2, ws, ws_bytes, need, s);
  return launch<T, FP8, Shape<128, FP8, 4, 2, 4>>(a, max_rows, 2, ws, ws_bytes, need, s);
}

// What the three entry points share: checks and the launch of `a`, whose
// pointers, byte strides and mode are set.
int run(const char *what, SpanArgs a, int head_dim, int64_t max_rows, int q_dtype, int kv_dtype, void *workspace,
        int64_t workspace_bytes, int64_t *need, void *stream) {
  const bool fp8 = kv_dtype == NQ_FP8_E4M3;
  if (a.num_seqs < 0 || a.Hq <= 0 || a.Hkv <= 0 || a.Hkv > 65535 || a.total_q < 0)
    return fail(NQ_EINVAL, "%s: bad sequence or head counts", what);
  if (a.Hq % a.Hkv != 0)
    return fail(NQ_EINVAL, "%s: num_q_heads %d not a multiple of num_kv_heads %d", what, a.Hq, a.Hkv);
  a.G = a.Hq / a.Hkv;
  if (a.G > 16) return fail(NQ_EUNSUPPORTED, "%s: GQA group %d > 16", what, a.G);
  if (head_dim != 128 && head_dim != 256)
    return fail(NQ_EUNSUPPORTED, "%s: head_dim %d (built: 128, 256)", what, head_dim);
  if (q_dtype != NQ_BF16 && q_dtype != NQ_F16)
    return fail(NQ_EUNSUPPORTED, "%s: q dtype %d (need f16/bf16)", what, q_dtype);
  if (!fp8 && kv_dtype != q_dtype)
    return fail(NQ_EUNSUPPORTED, "%s: kv dtype %d with q dtype %d", what, kv_dtype, q_dtype);
  if (fp8 && (!a.k_scale || !a.v_scale)) return fail(NQ_EINVAL, "%s: fp8 K/V needs scales", what);
  if (!(a.scale_log2 > 0.f)) return fail(NQ_EINVAL, "%s: softmax_scale must be positive", what);
  if (a.num_seqs == 0 || a.total_q == 0) return NQ_OK;
  if (!a.q || !a.k || !a.v || !a.cu_k || !a.out) return fail(NQ_EINVAL, "%s: null pointer", what);
  if (a.block_tables) {
    if (a.block_size <= 0 || a.block_size % kKeys != 0 || a.block_size > 1 << 26)
      return fail(NQ_EUNSUPPORTED, "%s: block_size %d must be a multiple of 32", what, a.block_size);
    if (a.max_blocks <= 0 || a.bt_stride < a.max_blocks) return fail(NQ_EINVAL, "%s: block table width", what);
    // a tile's place in the pool is an int
    if (static_cast<int64_t>(a.num_blocks) * (a.block_size / kKeys) > 0x7fffffff)
      return fail(NQ_EINVAL, "%s: a pool of %d pages of %d tokens", what, a.num_blocks, a.block_size);
  }
  if (a.q_rs % 16 || a.q_hs % 16 || !aligned(a.q, 16) || !aligned(a.k, 16) || !aligned(a.v, 16) || a.kv_rs % 16 ||
      a.o_rs % 8 || a.o_hs % 8 || !aligned(a.out, 8))
    return fail(NQ_EINVAL, "%s: alignment (q, K/V rows: 16 bytes; out: 8)", what);
  if (a.kv_rs <= 0 || a.kv_rs > (1 << 20)) return fail(NQ_EINVAL, "%s: K/V row stride %lld bytes", what, (long long)a.kv_rs);
  if (a.gate && (a.g_rs % 8 || a.g_hs % 8 || !aligned(a.gate, 8)))
    return fail(NQ_EINVAL, "%s: gate must be 8-byte aligned", what);
  // rows of a sequence and tiles of its keys are divided by small_div
  if (max_rows <= 0 || max_rows >= 1 << 22 || static_cast<int64_t>(a.total_q) * a.G > (int64_t{1} << 30))
    return fail(NQ_EINVAL, "%s: %lld rows per kv head", what, (long long)max_rows);
  if (a.max_k < 0 || a.max_k >= 1 << 26) return fail(NQ_EINVAL, "%s: %d tokens in a sequence", what, a.max_k);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (q_dtype == NQ_BF16)
    return fp8 ? launch_shape<BF16, true>(a, head_dim, max_rows, workspace, workspace_bytes, need, s)
               : launch_shape<BF16, false>(a, head_dim, max_rows, workspace, workspace_bytes, need, s);
  return fp8 ? launch_shape<F16, true>(a, head_dim, max_rows, workspace, workspace_bytes, need, s)
             : launch_shape<F16, false>(a, head_dim, max_rows, workspace, workspace_bytes, need, s);
}

}  // namespace
}  // namespace nq

using namespace nq;

extern "C" int nq_tree_attention(const void *q, int64_t q_row_stride, int64_t q_head_stride, const void *k_cache,
                                 const void *v_cache, const int32_t *cu_seqlens_q, const int32_t *cu_seqlens_k,
                                 int max_seqlen_q, int max_seqlen_k, const int32_t *block_tables, int64_t bt_stride,
                                 int max_blocks_per_seq, int64_t num_blocks, const int64_t *tree_mask,
                                 int64_t mask_row_stride, int mask_words, void *out, int64_t out_row_stride,
                                 int64_t out_head_stride, int num_seqs, int64_t total_q, int num_q_heads,
                                 int num_kv_heads, int head_dim, int block_size, float softmax_scale, int q_dtype,
                                 int kv_dtype, const float *k_scale, const float *v_scale, const void *gate,
                                 int64_t gate_row_stride, int64_t gate_head_stride, void *workspace,
                                 int64_t workspace_bytes, int64_t *need, void *stream) {
  const char *what = "tree_attention";
  if (max_seqlen_q < 0 || max_seqlen_q > kMaxNodes)
    return fail(NQ_EUNSUPPORTED, "%s: trees of %d nodes (at most %d)", what, max_seqlen_q, kMaxNodes);
  if (mask_words < (max_seqlen_q + 63) / 64 || mask_words > kMaxNodes / 64 || mask_row_stride < mask_words)
    return fail(NQ_EINVAL, "%s: %d mask words for %d nodes", what, mask_words, max_seqlen_q);
  if (num_seqs > 0 && total_q > 0 && (!block_tables || !tree_mask || !cu_seqlens_q || !aligned(tree_mask, 8)))
    return fail(NQ_EINVAL, "%s: null (or unaligned) pointer", what);
  if (total_q > 0x7fffffff) return fail(NQ_EINVAL, "%s: %lld rows", what, (long long)total_q);
  if (max_seqlen_q == 0) return NQ_OK;
  SpanArgs a{};
  a.q = static_cast<const uint8_t *>(q);
  a.q_rs = q_row_stride * 2;
  a.q_hs = q_head_stride * 2;
  a.k = static_cast<const uint8_t *>(k_cache);
  a.v = static_cast<const uint8_t *>(v_cache);
  a.kv_rs = static_cast<int64_t>(num_kv_heads) * head_dim * elem_size(kv_dtype);
  a.cu_q = cu_seqlens_q;
  a.cu_k = cu_seqlens_k;
  a.total_q = static_cast<int>(total_q);
  a.max_q = max_seqlen_q;
  a.max_k = static_cast<int>(std::min<int64_t>(max_seqlen_k, static_cast<int64_t>(max_blocks_per_seq) * block_size));
  a.block_tables = block_tables;
  a.bt_stride = bt_stride;
  a.max_blocks = max_blocks_per_seq;
  a.num_blocks = static_cast<int>(std::min<int64_t>(num_blocks, 0x7fffffff));
  a.out = static_cast<uint8_t *>(out);
  a.o_rs = out_row_stride * 2;
  a.o_hs = out_head_stride * 2;
  a.gate = static_cast<const uint8_t *>(gate);
  a.g_rs = gate_row_stride * 2;
  a.g_hs = gate_head_stride * 2;
  a.Hq = num_q_heads;
  a.Hkv = num_kv_heads;
  a.block_size = block_size;
  a.num_seqs = num_seqs;
  a.mask = reinterpret_cast<const uint64_t *>(tree_mask);
  a.mask_rs = mask_row_stride;
  a.words = mask_words;
  a.scale_log2 = softmax_scale * kLog2e;
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  return run(what, a, head_dim, static_cast<int64_t>(max_seqlen_q) * (num_kv_heads > 0 ? num_q_heads / num_kv_heads : 1),
             q_dtype, kv_dtype, workspace, workspace_bytes, need, stream);
}

extern "C" int nq_window_prefill(const void *q, int64_t q_row_stride, int64_t q_head_stride, const void *k,
                                 const void *v, int64_t kv_row_stride, int64_t total_k, const int32_t *cu_seqlens_q,
                                 const int32_t *cu_seqlens_k, int max_seqlen_q, int max_seqlen_k,
                                 const int32_t *block_tables, int64_t bt_stride, int max_blocks_per_seq,
                                 int64_t num_blocks, int window, int num_sinks, void *out, int64_t out_row_stride,
                                 int64_t out_head_stride, int num_seqs, int64_t total_q, int num_q_heads,
                                 int num_kv_heads, int head_dim, int block_size, float softmax_scale, int q_dtype,
                                 int kv_dtype, const float *k_scale, const float *v_scale, const void *gate,
                                 int64_t gate_row_stride, int64_t gate_head_stride, void *workspace,
                                 int64_t workspace_bytes, int64_t *need, void *stream) {
  const char *what = "window_prefill";
  if (window <= 0 || num_sinks < 0) return fail(NQ_EINVAL, "%s: window %d, sinks %d", what, window, num_sinks);
  if (num_seqs > 0 && total_q > 0 && !cu_seqlens_q) return fail(NQ_EINVAL, "%s: null pointer", what);
  if (total_q > 0x7fffffff || total_k > 0x7fffffff || max_seqlen_q < 0)
    return fail(NQ_EINVAL, "%s: %lld rows, %lld keys", what, (long long)total_q, (long long)total_k);
  if (max_seqlen_q == 0) return NQ_OK;
  SpanArgs a{};
  a.q = static_cast<const uint8_t *>(q);
  a.q_rs = q_row_stride * 2;
  a.q_hs = q_head_stride * 2;
  a.k = static_cast<const uint8_t *>(k);
  a.v = static_cast<const uint8_t *>(v);
  const int64_t row = static_cast<int64_t>(num_kv_heads) * head_dim;
  a.kv_rs = (block_tables ? row : kv_row_stride) * elem_size(kv_dtype);
  if (!block_tables && kv_row_stride < row)
    return fail(NQ_EINVAL, "%s: K/V row stride %lld < %lld", what, (long long)kv_row_stride, (long long)row);
  a.cu_q = cu_seqlens_q;
  a.cu_k = cu_seqlens_k;
  a.total_q = static_cast<int>(total_q);
  a.max_q = max_seqlen_q;
  a.total_k = static_cast<int>(total_k);
  a.max_k = block_tables ? static_cast<int>(std::min<int64_t>(max_seqlen_k,
                                                              static_cast<int64_t>(max_blocks_per_seq) * block_size))
                         : max_seqlen_k;
  a.block_tables = block_tables;
  a.bt_stride = bt_stride;
  a.max_blocks = max_blocks_per_seq;
  a.num_blocks = static_cast<int>(std::min<int64_t>(num_blocks, 0x7fffffff));
  a.out = static_cast<uint8_t *>(out);
  a.o_rs = out_row_stride * 2;
  a.o_hs = out_head_stride * 2;
  a.gate = static_cast<const uint8_t *>(gate);
  a.g_rs = gate_row_stride * 2;
  a.g_hs = gate_head_stride * 2;
  a.Hq = num_q_heads;
  a.Hkv = num_kv_heads;
  a.block_size = block_size;
  a.num_seqs = num_seqs;
  a.window = std::min(window, 1 << 28);
  a.sinks = std::min(num_sinks, 1 << 28);
  a.scale_log2 = softmax_scale * kLog2e;
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  return run(what, a, head_dim, static_cast<int64_t>(max_seqlen_q) * (num_kv_heads > 0 ? num_q_heads / num_kv_heads : 1),
             q_dtype, kv_dtype, workspace, workspace_bytes, need, stream);
}

extern "C" int nq_window_decode(const void *q, int64_t q_batch_stride, int64_t q_head_stride, void *k_cache,
                                void *v_cache, const int32_t *block_tables, int64_t bt_stride,
                                int max_blocks_per_seq, const int32_t *context_lens, int window, int num_sinks,
                                const void *k_new, int64_t k_new_row_stride, const void *v_new,
                                int64_t v_new_row_stride, const int32_t *slot_mapping, int new_dtype, void *out,
                                int64_t out_batch_stride, int64_t out_head_stride, int batch, int num_q_heads, int num_kv_heads, int head_dim, int block_size, int64_t num_blocks,
                                float softmax_scale, int q_dtype, int kv_dtype, const float *k_scale,
                                const float *v_scale, const void *gate, int64_t gate_batch_stride,
                                int64_t gate_head_stride, void *workspace, int64_t workspace_bytes, int64_t *need,
                                void *stream) {
  const char *what = "window_decode";
  if (window <= 0 || num_sinks < 0) return fail(NQ_EINVAL, "%s: window %d, sinks %d", what, window, num_sinks);
  if (batch > 0 && !block_tables) return fail(NQ_EINVAL, "%s: null pointer", what);
  const int64_t new_size = elem_size(new_dtype), row = static_cast<int64_t>(num_kv_heads) * head_dim;
  if (k_new) {
    if (!v_new || !slot_mapping) return fail(NQ_EINVAL, "%s: null v_new or slot_mapping", what);
    if (new_size == 0 || new_dtype == NQ_FP8_E4M3 || (kv_dtype != NQ_FP8_E4M3 && new_dtype != kv_dtype))
      return fail(NQ_EUNSUPPORTED, "%s: new rows of dtype %d into a cache of dtype %d", what, new_dtype, kv_dtype);
    if (k_new_row_stride < row || v_new_row_stride < row || (k_new_row_stride * new_size) % 16 ||
        (v_new_row_stride * new_size) % 16 || !aligned(k_new, 16) || !aligned(v_new, 16))
      return fail(NQ_EINVAL, "%s: k_new/v_new rows must be 16-byte aligned [Hkv, D] rows", what);
  }
  SpanArgs a{};
  a.q = static_cast<const uint8_t *>(q);
  a.q_rs = q_batch_stride * 2;
  a.q_hs = q_head_stride * 2;
  a.k = static_cast<const uint8_t *>(k_cache);
  a.v = static_cast<const uint8_t *>(v_cache);
  a.kv_rs = static_cast<int64_t>(num_kv_heads) * head_dim * elem_size(kv_dtype);
  a.cu_k = context_lens;
  a.total_q = batch;
  a.max_q = 1;
  a.max_k = static_cast<int>(std::min<int64_t>(static_cast<int64_t>(max_blocks_per_seq) * block_size, (1 << 26) - 1));
  a.block_tables = block_tables;
  a.bt_stride = bt_stride;
  a.max_blocks = max_blocks_per_seq;
  a.num_blocks = static_cast<int>(std::min<int64_t>(num_blocks, 0x7fffffff));
  a.out = static_cast<uint8_t *>(out);
  a.o_rs = out_batch_stride * 2;
  a.o_hs = out_head_stride * 2;
  a.gate = static_cast<const uint8_t *>(gate);
  a.g_rs = gate_batch_stride * 2;
  a.g_hs = gate_head_stride * 2;
  a.Hq = num_q_heads;
  a.Hkv = num_kv_heads;
  a.block_size = block_size;
  a.num_seqs = batch;
  a.window = std::min(window, 1 << 28);
  a.sinks = std::min(num_sinks, 1 << 28);
  if (k_new) {
    a.k_new = static_cast<const uint8_t *>(k_new);
    a.v_new = static_cast<const uint8_t *>(v_new);
    a.kn_rs = k_new_row_stride * new_size;
    a.vn_rs = v_new_row_stride * new_size;
    a.slot_mapping = slot_mapping;
    a.new_dtype = new_dtype;
  }
  a.scale_log2 = softmax_scale * kLog2e;
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  return run(what, a, head_dim, num_kv_heads > 0 ? num_q_heads / num_kv_heads : 1, q_dtype, kv_dtype, workspace,
             workspace_bytes, need, stream);
}
