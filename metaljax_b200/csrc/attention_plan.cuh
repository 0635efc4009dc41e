// How the work of an attention call is shared out, from lengths that only the device knows.
//
// An item is a tile of query rows of one sequence and key head: row r of a sequence's n * group rows is new token r / group, query
// head r % group of the key head's (so that a group's heads read its keys once). RowTiles takes R rows a tile, wherever tokens begin; TokenTiles (whose
// queries come as boxes of whole tokens) two halves of tile_tokens tokens. A unit is a block of B positions of an item's keys. An item weighs its units
// and kCost more (queries in, results out). All items stand in one order (sequence, head, tile), and CTA c of C takes the weights from c * quota to
// (c + 1) * quota, so that every CTA has about as much to do whatever the lengths are. Items of fewer than kWhole units go to one CTA, that of their beginning; longer
// ones are cut where a share ends, and each CTA leaves a partial result (two slots a CTA: an item that it finishes, and one that it begins), which a second
// launch joins. There are no atomics and no state between calls, and sums do not depend on timing.
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
__device__ __forceinline__ int seen_by(const AttentionWork& w, const SeqSpan& s, int tokens) {
  const int end = w.causal ? s.len - s.n + (tokens < s.n ? tokens : s.n) : s.len;
  return end < 0 ? 0 : end;
}

// (a sequence's rows are fewer than 2^31: the entry points see to that)
// kCost, kWhole: an item's ends measured in units. 64 sequences of 2000 to 8000 e4m3 positions: kCost 2 and 3 188 us, 5 193, 8 198.
template <int R, int B>
struct RowTiles {
  static constexpr int kCost = 3, kWhole = 2;
  static __device__ __forceinline__ int tiles(const AttentionWork& w, const SeqSpan& s) { return static_cast<int>((static_cast<unsigned>(s.n) * w.group + R - 1) / R); }
  // One unit at least, which writes the zeros of rows that see nothing.
  static __device__ __forceinline__ int units(const AttentionWork& w, const SeqSpan& s, int t) {
    const int u = (seen_by(w, s, static_cast<int>((static_cast<unsigned>(t) * R + R - 1) / static_cast<unsigned>(w.group)) + 1) + B - 1) / B;
    return u < 1 ? 1 : u;
  }
};

// 16 prompts of some 700 tokens with heads of 64 / 4 of some 150 / one of 8192 / 8 chunks of 64 over up to 8000, us: kCost 3 and kWhole 8 46.0 / 16 / 469 / 64; kCost 2
// 45.1 / 16 / 470 / 65, 1 45.3 / 16 / 497 / 69; kCost 2 and kWhole 5 47.0 / 16 / 469 / 63.
template <int B>
struct TokenTiles {
  static constexpr int kCost = 3, kWhole = 8;
  static __device__ __forceinline__ int tiles(const AttentionWork& w, const SeqSpan& s) {
    return static_cast<int>((s.n + 2u * w.tile_tokens - 1) / (2u * w.tile_tokens));
  }
  static __device__ __forceinline__ int units(const AttentionWork& w, const SeqSpan& s, int t) {
    const int u = (seen_by(w, s, (t + 1) * 2 * w.tile_tokens) + B - 1) / B;
    return u < 1 ? 1 : u;
  }
};

// A CTA's place in the order: units u to before `end` of an item are its; `room`: weights from the item's beginning to the end of its share.
struct UnitCursor {
  int s, h, t, u, end, units;
  SeqSpan span;
  int64_t room;
};

// Units of an item before the place `room` weights behind its beginning, where one share ends and the next begins: no share of a single unit.
template <typename Tiles>
__device__ __forceinline__ int cut(int units, int64_t room) {
  if (room >= units + Tiles::kCost) return units;
  if (units < Tiles::kWhole) return room > 0 ? units : 0;
  const int u = static_cast<int>(room) - Tiles::kCost;
  return u < 2 ? 0 : units - u < 2 ? units : u;
}

__device__ __forceinline__ int64_t warp_sum(int64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <typename I>
__device__ __forceinline__ I warp_scan(I v) {                      // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const I x = __shfl_up_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) >= o) v += x;
  }
  return v;
}

// One warp: weight of one head's items of 32 sequences from `base` on, a lane each (0 behind the last).
template <typename Tiles>
__device__ __forceinline__ int64_t lane_weights(const AttentionWork& w, int base) {
  const int lane = threadIdx.x & 31, s = base + lane;
  SeqSpan span = {0, 0, 0};
  if (s < w.seqs) span = span_of(w, s);
  const int tiles = Tiles::tiles(w, span);
  int64_t sum = 0;
  if (tiles <= 32)
    for (int t = 0; t < tiles; ++t) sum += Tiles::units(w, span, t) + Tiles::kCost;
  unsigned many = __ballot_sync(0xffffffffu, tiles > 32);
  while (many) {                                        // long ones: all lanes over the tiles
    const int l = __ffs(many) - 1;
    many &= many - 1;
    const SeqSpan other = {__shfl_sync(0xffffffffu, span.q0, l), __shfl_sync(0xffffffffu, span.n, l), __shfl_sync(0xffffffffu, span.len, l)};
    const int n = Tiles::tiles(w, other);
    int64_t part = 0;
    for (int t = lane; t < n; t += 32) part += Tiles::units(w, other, t) + Tiles::kCost;
    part = warp_sum(part);
    if (lane == l) sum = part;
  }
  return sum;
}

// Weights of a CTA's share: at least a single unit with what its item costs (less makes parts to join out of nothing). (Divisions of 64
// bits are calls, and spill what is live around them.)
template <typename Tiles>
__device__ __forceinline__ int64_t quota_of(int64_t total, int ctas) {
  constexpr int kLeast = Tiles::kCost + 1;
  int shift = 0;
  while ((total + ctas) >> shift >> 32) shift += 8;     // (a larger share than need be where weights pass 2^32)
  const int64_t q = shift ? (static_cast<int64_t>(static_cast<uint32_t>(total >> shift) / ctas) + 1) << shift : static_cast<uint32_t>(total + ctas - 1) / ctas;
  return q < kLeast ? kLeast : q;
}

// To the beginning of the next item; whether there is one.
template <typename Tiles>
__device__ __forceinline__ bool step_item(const AttentionWork& w, UnitCursor& c) {
  if (++c.t >= Tiles::tiles(w, c.span)) {
    c.t = 0;
    if (++c.h >= w.kv_heads) {
      c.h = 0;
      do {
        if (++c.s >= w.seqs) return false;
        c.span = span_of(w, c.s);
      } while (c.span.n == 0);
    }
  }
  c.units = Tiles::units(w, c.span, c.t);
  return true;
}

// To this CTA's part of the next item; whether it has one.
template <typename Tiles>
__device__ __forceinline__ bool next_item(const AttentionWork& w, UnitCursor& c) {
  c.room -= c.units + Tiles::kCost;
  if (c.room <= 0 || !step_item<Tiles>(w, c)) return false;
  c.u = 0;
  c.end = cut<Tiles>(c.units, c.room);
  return c.end > 0;
}

// `left` weights into its item, and `quota` of them this CTA's: where it begins; false where it has nothing to do.
template <typename Tiles>
__device__ __forceinline__ bool begin_share(const AttentionWork& w, int64_t left, int64_t quota, UnitCursor* at) {
  at->u = left > 0 ? cut<Tiles>(at->units, left) : 0;
  at->room = quota + left;
  if (at->u == at->units) return next_item<Tiles>(w, *at);
  at->end = cut<Tiles>(at->units, at->room);
  return at->end > at->u;
}

// One warp: the item of a sequence at->s and head at->h that is `left` weights behind its first one's beginning; returns what is left of them.
template <typename Tiles, typename I>
__device__ __forceinline__ I find_tile(const AttentionWork& w, I left, UnitCursor* at) {
  const int lane = threadIdx.x & 31, tiles = Tiles::tiles(w, at->span);
  at->t = 0;
  at->units = Tiles::units(w, at->span, 0);
  if (tiles == 1) return left;
  for (int base = 0; base < tiles; base += 32) {
    const int units = base + lane < tiles ? Tiles::units(w, at->span, base + lane) : 0;
    const int upto = warp_scan(base + lane < tiles ? units + Tiles::kCost : 0);        // (32 items: fewer than 2^30)
    const unsigned past = __ballot_sync(0xffffffffu, upto > left);
    if (past) {
      const int l = __ffs(past) - 1;
      at->t = base + l;
      at->units = __shfl_sync(0xffffffffu, units, l);
      return left - (__shfl_sync(0xffffffffu, upto, l) - (at->units + Tiles::kCost));
    }
    left -= __shfl_sync(0xffffffffu, upto, 31);
  }
  return left;                                          // (not reached: the sums are the same)
}

// One warp: where CTA `cta` of `ctas` begins; false where it has nothing to do. `share`: what a CTA takes.
template <typename Tiles>
__device__ __forceinline__ bool find_share(const AttentionWork& w, int cta, int ctas, UnitCursor* at, int64_t* share) {
  // ordinary calls: up to 128 sequences, looked at once, and sums of 32 bits (a call waits 2 us for this, and more with 64-bit sums over two looks)
  constexpr int kGroups = 4;
  if (w.seqs <= 32 * kGroups) {
    int mine[kGroups], sum = 0;
    bool small = true;
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      mine[i] = 0;
      if (i * 32 >= w.seqs) continue;
      const int64_t weight = lane_weights<Tiles>(w, i * 32);
      small = small && weight < (1 << 23) / w.kv_heads;
      mine[i] = static_cast<int>(weight) * w.kv_heads;
      sum += mine[i];
    }
    if (__all_sync(0xffffffffu, small)) {
      const int total = __reduce_add_sync(0xffffffffu, sum);
      int quota = static_cast<int>(static_cast<unsigned>(total + ctas - 1) / static_cast<unsigned>(ctas));
      if (quota < Tiles::kCost + 1) quota = Tiles::kCost + 1;
      *share = quota;
      if (static_cast<int64_t>(quota) * cta >= total) return false;
      int left = quota * cta;
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
        if (i * 32 >= w.seqs) break;
        const int upto = warp_scan(mine[i]);
        const unsigned past = __ballot_sync(0xffffffffu, upto > left);
        if (past) {
          const int l = __ffs(past) - 1, all = __shfl_sync(0xffffffffu, mine[i], l);
          at->s = i * 32 + l;
          at->span = span_of(w, at->s);
          left -= __shfl_sync(0xffffffffu, upto, l) - all;
          const unsigned per_head = static_cast<unsigned>(all) / static_cast<unsigned>(w.kv_heads);
          at->h = static_cast<int>(static_cast<unsigned>(left) / per_head);
          left = find_tile<Tiles>(w, left - at->h * static_cast<int>(per_head), at);
          return begin_share<Tiles>(w, left, quota, at);
        }
        left -= __shfl_sync(0xffffffffu, upto, 31);
      }
      return false;                                     // (not reached)
    }
  }
  int64_t total = 0;
  for (int base = 0; base < w.seqs; base += 32) total += warp_sum(lane_weights<Tiles>(w, base)) * w.kv_heads;
  const int64_t quota = quota_of<Tiles>(total, ctas);
  *share = quota;
  int64_t left = quota * cta;
  if (left >= total) return false;
  for (int base = 0; base < w.seqs; base += 32) {
    const int64_t mine = lane_weights<Tiles>(w, base);
    const int64_t upto = warp_scan(mine) * w.kv_heads;
    const unsigned past = __ballot_sync(0xffffffffu, upto > left);
    if (past) {
      const int l = __ffs(past) - 1;
      at->s = base + l;
      at->span = span_of(w, at->s);
      const int64_t per_head = __shfl_sync(0xffffffffu, mine, l);
      left -= __shfl_sync(0xffffffffu, upto, l) - per_head * w.kv_heads;
      at->h = 0;
      while (left >= per_head) {
        left -= per_head;
        ++at->h;
      }
      left = find_tile<Tiles>(w, left, at);
      return begin_share<Tiles>(w, left, quota, at);
    }
    left -= __shfl_sync(0xffffffffu, upto, 31);
  }
  return false;                                         // (not reached)
}

// The workspace: a note of every CTA, written by each, then two partial results a CTA. The note says what the second launch has to join at the end of a
// CTA's share: the item that it began and did not finish, and how many CTAs have a part of it (0: there is none).
struct JoinNote {
  int32_t parts, q0, n, len, h, t, pad[2];
};
// (the shares behind the first one's end take `share` units each, the last one what is left, and a single unit more)
__device__ __forceinline__ JoinNote note_of(const UnitCursor& c, int begun, int64_t share) {
  int parts = 0;
  if (begun == 0 && c.end < c.units) {
    const int rest = c.units - 1 - c.end;
    parts = 1 + (share > rest ? 1 : static_cast<int>((static_cast<uint32_t>(rest) + static_cast<uint32_t>(share) - 1) / static_cast<uint32_t>(share)));
  }
  return {parts, c.span.q0, c.span.n, c.span.len, c.h, c.t, {0, 0}};
}

// A partial result in the workspace: R rows of D float32 sums, then R maxima (base 2) and R sums of weights.
template <int R, int D>
constexpr int64_t partial_floats() { return static_cast<int64_t>(R) * (D + 2); }

}  // namespace qmm
