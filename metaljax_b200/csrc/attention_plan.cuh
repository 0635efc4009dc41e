// How the work of an attention call is shared out, from lengths that only the device knows.
//
// An item is a tile of query rows of one sequence and key head: row r of a sequence's n * group rows is new token r / group, query
// head r % group of the key head's (so that a group's heads read its keys once). RowTiles takes R rows a tile, wherever tokens begin; TokenTiles (whose
// queries come as boxes of whole tokens) two halves of tile_tokens tokens. A unit is a block of B positions of an item's keys. All units stand in
// one order (sequence, head, tile, block), and CTA c of C works on those from c * quota on: every CTA has the same number of units whatever the lengths are. An item whose units fall to several CTAs
// leaves a partial result with each (two slots a CTA: an item that it finishes, and one that it begins), which a second launch joins: that one works
// out the same order. There are no atomics and no state between calls, and sums do not depend on timing.
#pragma once

#include "paged_cache.cuh"

namespace qmm {

struct AttentionWork {
  const int32_t* cu_q;
  const int32_t* kv_lens;      // NULL: a sequence's keys are its own tokens'
  int64_t tokens;
  int64_t longest;             // positions that a table has room for
  int32_t seqs, heads, kv_heads, group;
  int32_t causal;
  int32_t tile_tokens;         // TokenTiles: tokens of half a tile
  int* status;
};

// A sequence's rows of q and its positions, made safe: within the tensors whatever the lengths say.
struct SeqSpan {
  int q0, n, len;
};
__device__ __forceinline__ SeqSpan span_of(const AttentionWork& w, int s) {
  SeqSpan r;
  if (w.cu_q) {
    const int a = __ldg(w.cu_q + s), b = __ldg(w.cu_q + s + 1);
    r.q0 = a < 0 ? 0 : a > w.tokens ? static_cast<int>(w.tokens) : a;
    const int e = b > w.tokens ? static_cast<int>(w.tokens) : b;
    r.n = e > r.q0 ? e - r.q0 : 0;
    if (a < 0 || b > w.tokens || b < a) report_index(w.status);
  } else {
    r.q0 = s;
    r.n = 1;
  }
  r.len = r.n;
  if (w.kv_lens) {
    r.len = __ldg(w.kv_lens + s);
    if (r.len < 0 || r.len > w.longest) {
      report_index(w.status);
      r.len = r.len < 0 ? 0 : static_cast<int>(w.longest);
    }
  }
  return r;
}

// Positions up to which the last of a sequence's first `tokens` new tokens sees.
__device__ __forceinline__ int seen_by(const AttentionWork& w, const SeqSpan& s, int64_t tokens) {
  const int end = w.causal ? s.len - s.n + (tokens < s.n ? static_cast<int>(tokens) : s.n) : s.len;
  return end < 0 ? 0 : end;
}

// (rows of a sequence can pass 2^31: 64 heads of a group times its tokens)
template <int R, int B>
struct RowTiles {
  static __device__ __forceinline__ int tiles(const AttentionWork& w, const SeqSpan& s) {
    return static_cast<int>((static_cast<int64_t>(s.n) * w.group + R - 1) / R);
  }
  // One unit at least, which writes the zeros of rows that see nothing.
  static __device__ __forceinline__ int units(const AttentionWork& w, const SeqSpan& s, int t) {
    const int u = (seen_by(w, s, ((static_cast<int64_t>(t) + 1) * R - 1) / w.group + 1) + B - 1) / B;
    return u < 1 ? 1 : u;
  }
};

template <int B>
struct TokenTiles {
  static __device__ __forceinline__ int tiles(const AttentionWork& w, const SeqSpan& s) {
    return (s.n + 2 * w.tile_tokens - 1) / (2 * w.tile_tokens);
  }
  static __device__ __forceinline__ int units(const AttentionWork& w, const SeqSpan& s, int t) {
    const int u = (seen_by(w, s, (static_cast<int64_t>(t) + 1) * 2 * w.tile_tokens) + B - 1) / B;
    return u < 1 ? 1 : u;
  }
};

// A place in the order of units.
struct UnitCursor {
  int s, h, t, u, units;
  SeqSpan span;
};

// One warp: a sequence's units of one head, its lanes over the tiles.
template <typename Tiles>
__device__ __forceinline__ int64_t warp_units(const AttentionWork& w, const SeqSpan& s) {
  const int n = Tiles::tiles(w, s);
  int64_t sum = 0;
  for (int t = threadIdx.x & 31; t < n; t += 32) sum += Tiles::units(w, s, t);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return sum;
}

// One warp: units of one head of 32 sequences from `base` on, a lane each (0 behind the last).
template <typename Tiles>
__device__ __forceinline__ int64_t lane_units(const AttentionWork& w, int base, SeqSpan* mine) {
  const int s = base + (threadIdx.x & 31);
  SeqSpan span = {0, 0, 0};
  if (s < w.seqs) span = span_of(w, s);
  const int tiles = Tiles::tiles(w, span);
  int64_t sum = 0;
  if (tiles <= 4)
    for (int t = 0; t < tiles; ++t) sum += Tiles::units(w, span, t);
  unsigned many = __ballot_sync(0xffffffffu, tiles > 4);
  while (many) {
    const int l = __ffs(many) - 1;
    many &= many - 1;
    const SeqSpan other = {__shfl_sync(0xffffffffu, span.q0, l), __shfl_sync(0xffffffffu, span.n, l), __shfl_sync(0xffffffffu, span.len, l)};
    const int64_t all = warp_units<Tiles>(w, other);
    if ((threadIdx.x & 31) == l) sum = all;
  }
  *mine = span;
  return sum;
}

__device__ __forceinline__ int64_t warp_sum(int64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ int64_t warp_scan(int64_t v) {          // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) >= o) v += x;
  }
  return v;
}

// One warp: the units of a call, and the place of unit `index(total)` in their order (false: there is none).
template <typename Tiles, typename Index>
__device__ __forceinline__ bool find_unit(const AttentionWork& w, Index index, int64_t* total_out, UnitCursor* at) {
  const int lane = threadIdx.x & 31;
  SeqSpan span;
  int64_t mine = 0, total = 0;
  for (int base = 0; base < w.seqs; base += 32) {
    mine = lane_units<Tiles>(w, base, &span);
    total += warp_sum(mine) * w.kv_heads;
  }
  *total_out = total;
  int64_t left = index(total);
  if (left < 0 || left >= total) return false;
  int64_t per_head = 0;
  for (int base = 0; base < w.seqs; base += 32) {
    if (w.seqs > 32) mine = lane_units<Tiles>(w, base, &span);       // (the only ones are still there)
    const int64_t upto = warp_scan(mine) * w.kv_heads;
    const unsigned past = __ballot_sync(0xffffffffu, upto > left);
    if (past) {
      const int l = __ffs(past) - 1;
      at->s = base + l;
      at->span = {__shfl_sync(0xffffffffu, span.q0, l), __shfl_sync(0xffffffffu, span.n, l), __shfl_sync(0xffffffffu, span.len, l)};
      per_head = __shfl_sync(0xffffffffu, mine, l);
      left -= __shfl_sync(0xffffffffu, upto, l) - per_head * w.kv_heads;
      break;
    }
    left -= __shfl_sync(0xffffffffu, upto, 31);
  }
  at->h = 0;
  while (left >= per_head) {                            // (a few heads: a division of 64 bits is a call, and spills)
    left -= per_head;
    ++at->h;
  }
  const int tiles = Tiles::tiles(w, at->span);
  for (int base = 0; base < tiles; base += 32) {
    const int64_t u = base + lane < tiles ? Tiles::units(w, at->span, base + lane) : 0;
    const int64_t upto = warp_scan(u);
    const unsigned past = __ballot_sync(0xffffffffu, upto > left);
    if (past) {
      const int l = __ffs(past) - 1;
      at->t = base + l;
      at->units = static_cast<int>(__shfl_sync(0xffffffffu, u, l));
      at->u = static_cast<int>(left - (__shfl_sync(0xffffffffu, upto, l) - at->units));
      return true;
    }
    left -= __shfl_sync(0xffffffffu, upto, 31);
  }
  return false;                                        // (not reached: the sums are the same)
}

// To the first unit of the next item (which there has to be).
template <typename Tiles>
__device__ __forceinline__ void next_item(const AttentionWork& w, UnitCursor& c) {
  c.u = 0;
  if (++c.t >= Tiles::tiles(w, c.span)) {
    c.t = 0;
    if (++c.h >= w.kv_heads) {
      c.h = 0;
      do {
        ++c.s;
        c.span = c.s < w.seqs ? span_of(w, c.s) : SeqSpan{0, 1, 0};
      } while (c.span.n == 0);
    }
  }
  c.units = Tiles::units(w, c.span, c.t);
}

// Units of a CTA: at least `least`, below which a CTA's share does not pay for a part of an item to be joined. (Divisions of 64 bits are calls, and spill
// what is live around them.)
__device__ __forceinline__ int64_t quota_of(int64_t total, int ctas, int least) {
  int shift = 0;
  while ((total + ctas) >> shift >> 32) shift += 8;     // (a larger share than need be where units pass 2^32)
  const int64_t q = shift ? (static_cast<int64_t>(static_cast<uint32_t>(total >> shift) / ctas) + 1) << shift : static_cast<uint32_t>(total + ctas - 1) / ctas;
  return q < least ? least : q;
}
// CTAs that have a part of an item of which `after` units lie behind the end of the first one's share.
__device__ __forceinline__ int parts_of(int after, int64_t quota) {
  return 1 + (quota >> 31 ? 1 : static_cast<int>((static_cast<uint32_t>(after) + static_cast<uint32_t>(quota) - 1) / static_cast<uint32_t>(quota)));
}

// The workspace: a note of every CTA, written by each, then two partial results a CTA. The note says what the second launch has to join at the end of a
// CTA's share: the item that it began and did not finish, and how many CTAs have a part of it (0: there is none).
struct JoinNote {
  int32_t parts, q0, n, len, h, t, pad[2];
};
__device__ __forceinline__ JoinNote note_of(const UnitCursor& c, int begun, int ended, int64_t quota) {
  const int parts = begun == 0 && ended < c.units ? parts_of(c.units - ended, quota) : 0;
  return {parts, c.span.q0, c.span.n, c.span.len, c.h, c.t, {0, 0}};
}

// A partial result in the workspace: R rows of D float32 sums, then R maxima (base 2) and R sums of weights.
template <int R, int D>
constexpr int64_t partial_floats() { return static_cast<int64_t>(R) * (D + 2); }

}  // namespace qmm
