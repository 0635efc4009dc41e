// Attention of query tiles of 16, 32 or 64 rows over keys and values in pages (16-bit or e4m3) or in rows, on mma.sync: what one new token a
// sequence, or a few, take. With few rows a key is used for too little arithmetic to be anything but a stream, so the kernel is
// built like one: 128 threads, two CTAs an SM (three of codes), shares of the work by weight or clusters by item, chunks of 64 positions on their way (cp.async, 16-byte pieces under an XOR swizzle that makes
// ldmatrix conflict-free) while one is worked on, also across the ends of items.
//
// One pass: a warp holds 16 rows' queries as A fragments, takes scores of its positions of a chunk, the running maximum m and sum l of
// 2^(s - m), and adds 2^(s - m) v to its 16 x D sums in registers. RW warps share a tile's rows; the KW = 4 / RW
// warps on the same rows take 64 / KW positions of a chunk each, and are joined when the item ends. With one row of 16 (RW = 1) a warp reads only what it has asked
// for itself, and the CTA does not meet but at the ends of items. Pages of bf16 are bound by the memory: the same 64 sequences 206 us, 6.5 TB/s.
//
// e4m3 codes: with one row of 16 a warp takes them straight into its B fragments as f16, one conversion a pair (a bf16 takes five
// instructions a pair, with which 64 sequences of 2000 to 8000 positions took 249 us; now 171, 3.9 TB/s, bound by instructions: 680 for 16
// positions): of keys four codes of a row a step (the queries' elements in the order that makes), of values the codes of its four positions,
// paired by a byte permutation. A row's queries become f16 under a power of two of its own, the rows' powers of two go to the scores and to the weights. Where warps share positions, the one that asked for a chunk's rows turns them into bf16 (exactly) next to the chunk in
// shared memory.
//
// Masked positions: scores are selected, not added to. A value that is no number at a masked position would still be 0 * NaN in the sum, so
// rows of v behind a sequence's end are zeros (the copies fill them in), and in chunks that some rows see and others do not infinities and NaN
// are taken out, and put into the sums of the rows that see them at the end (`Specials`).
#include <climits>
#include <type_traits>

#include "attention.h"
#include "qmm_tcgen05.cuh"

namespace qmm {
namespace {

using namespace ptx;

constexpr int kThreads = 128, kChunk = 64;

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t lds8(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint32_t lds16(uint32_t addr) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ float remote_ld32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Whether a pair of 16-bit floats has one without a finite value.
template <typename T>
__device__ __forceinline__ bool odd_pair(uint32_t w) {
  constexpr uint32_t kExp = std::is_same<T, __nv_bfloat16>::value ? 0x7f80u : 0x7c00u;
  return (w & kExp) == kExp || (w >> 16 & kExp) == kExp;
}

enum Source { kRowsSource, kPages16, kPages8 };

template <int D, int SOURCE, int RW>
struct RowsLayout {
  static constexpr bool kE4m3 = SOURCE == kPages8, kDirect = kE4m3 && RW == 1;
  static constexpr int kCtas = kDirect ? 3 : 2;                          // an SM

  static constexpr int kStages = 3;
  static constexpr int kRowBytes = D * (kE4m3 ? 1 : 2);
  static constexpr int kHalf = kChunk * kRowBytes;                       // keys of a chunk; values follow, then (e4m3) both rows' bytes
  static constexpr int kStage = 2 * kHalf + (kE4m3 ? 2 * kChunk : 0);
  static constexpr int kValues = kE4m3 && !kDirect ? 2 * kChunk * D * 2 : 0;         // an e4m3 chunk as bf16
  static constexpr int kRing = kStages * kStage;
  static constexpr int kSpecials = 3 * D * 4 + 16;
  static constexpr int kStats = kChunk * 2 * 4;                          // (maximum, sum) of a warp's rows
  static constexpr int kBytes = kRing + kValues + kSpecials + kStats + 64;
};

// Four elements of a row's result. No weight at all: a row that sees nothing is zero; one that sees only scores of -inf has no softmax.
template <typename T>
__device__ __forceinline__ void store_row(const RowsParams& p, const UnitCursor& c, int tok, int g, int d, int dim, const float (&v)[4], float l, int seen) {
  const float inv = l == 0.0f ? (seen < 0 ? 0.0f : NAN) : 1.0f / l;
  uint2 out;
  out.x = pack2<T>(v[0] * inv, v[1] * inv);
  out.y = pack2<T>(v[2] * inv, v[3] * inv);
  *reinterpret_cast<uint2*>(p.out + (((static_cast<int64_t>(c.span.q0) + tok) * p.work.heads + c.h * p.work.group + g) * dim + d) * 2) = out;
}

// CTAS = 1: shares by weight, which attend_join_kernel joins. CTAS > 1: clusters of CTAS take whole items (in turn, if there are more than clusters), every CTA an
// equal run of the units, and join them out of one another's shared memory: the first stages of the ring, and maxima and sums of weights behind everything else.
// (They are two an SM at most, and have the registers of two: 8 sequences of up to 2000 positions of codes, two tokens each, 18.1 us, with those of three 21.2.)
template <typename Tiles>
__device__ __forceinline__ bool cluster_item(const AttentionWork& w, int item, int rank, int ctas, UnitCursor* at) {
  int n = item / w.kv_heads;                            // tile of all sequences'
  at->h = item - n * w.kv_heads;
  if (!w.cu_q) {
    at->span.n = 1;
    const int per = Tiles::tiles(w, at->span);
    at->s = n / per;
    if (at->s >= w.seqs) return false;
    at->t = n - at->s * per;
    at->span = span_of(w, at->s);
  } else {
    for (int base = 0;; base += 32) {
      if (base >= w.seqs) return false;
      SeqSpan span = {0, 0, 0};
      if (base + (threadIdx.x & 31) < w.seqs) span = span_of(w, base + (threadIdx.x & 31));
      const int tiles = Tiles::tiles(w, span);
      const int64_t upto = warp_scan<int64_t>(tiles);
      const unsigned past = __ballot_sync(0xffffffffu, upto > n);
      if (past) {
        const int l = __ffs(past) - 1;
        at->s = base + l;
        at->t = n - static_cast<int>(__shfl_sync(0xffffffffu, upto - tiles, l));
        at->span = {__shfl_sync(0xffffffffu, span.q0, l), __shfl_sync(0xffffffffu, span.n, l), __shfl_sync(0xffffffffu, span.len, l)};
        break;
      }
      n -= static_cast<int>(__shfl_sync(0xffffffffu, upto, 31));
    }
  }
  at->units = Tiles::units(w, at->span, at->t);
  const int each = (at->units + ctas - 1) / ctas;
  at->u = rank * each < at->units ? rank * each : at->units;
  at->end = at->u + each < at->units ? at->u + each : at->units;
  at->room = 0;                                         // (no item behind it)
  return true;
}

template <typename T, int D, int RW, int SOURCE, int CTAS>
__global__ void __launch_bounds__(kThreads, (CTAS > 1 ? 2 : RowsLayout<D, SOURCE, RW>::kCtas)) attend_rows_kernel(const RowsParams p) {
  using L = RowsLayout<D, SOURCE, RW>;
  constexpr bool kPaged = SOURCE != kRowsSource, kE4m3 = L::kE4m3;
  constexpr int R = 16 * RW, KW = 4 / RW, SN = kChunk / KW;               // rows of a tile; warps on the same rows; a warp's positions of a chunk
  constexpr bool kDirect = L::kDirect;                                    // codes straight into fragments: no other warp wants them
  using MT = typename std::conditional<kDirect, __half, T>::type;         // ... f16, which holds a code in one conversion of two
  using Tiles = RowTiles<R, kChunk>;
  extern __shared__ __align__(128) uint8_t smem[];
  int* const special = reinterpret_cast<int*>(smem + L::kRing + L::kValues);           // first positions of +inf, -inf, NaN in each column of v
  int* const any_special = special + 3 * D;
  float* const stats = reinterpret_cast<float*>(smem + L::kRing + L::kValues + L::kSpecials);
  constexpr bool kCluster = CTAS > 1;
  static_assert(!kCluster || (R * D * 4 <= (kE4m3 && !kDirect ? L::kRing : L::kStage) && 4 * (kDirect ? 8 : 16) * D * 4 <= (kE4m3 && !kDirect ? L::kValues : L::kStage)),
                "a part, and what it is made of, in the ring");
  [[maybe_unused]] float* const part_rows = reinterpret_cast<float*>(smem);
  [[maybe_unused]] float* const part_stats = reinterpret_cast<float*>(smem + L::kBytes);          // R maxima, R sums of weights
  const uint32_t ring = smem_u32(smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rw = warp / KW, kw = warp % KW;
  const AttentionWork& w = p.work;

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  UnitCursor c;
  [[maybe_unused]] int64_t share = 0;
  if constexpr (kCluster) {
    if (!cluster_item<Tiles>(w, blockIdx.x / CTAS, blockIdx.x % CTAS, CTAS, &c)) return;
  } else {
    if (tid == 0) p.notes[blockIdx.x].parts = 0;
    // every warp works out where this CTA begins by itself
    if (!find_share<Tiles>(w, blockIdx.x, gridDim.x, &c, &share)) return;
  }
  UnitCursor load = c;                                  // where the copies are
  bool loading = c.u < c.end;

  // ---- copies: a warp asks for rows 16 * warp .. of a chunk (which lie in one page) ----
  int pages = 0, pages_at = 0;                          // lane i: the page of this warp's rows of chunk pages_at + i
  auto look_up = [&]() {
    if constexpr (kPaged) {
      pages_at = load.u;
      const int u = load.u + lane, pos = u * kChunk + 16 * warp;
      int64_t page = 0;
      if (u < load.end && pos < load.span.len) page = page_of(p.cache, load.s, pos, w.status);
      pages = page < 0 ? 0 : static_cast<int>(page);
    }
  };
  auto request = [&](int loaded) {                      // the chunk that `load` stands at into the ring, and `load` on
    if (loading) {
      const uint32_t stage = ring + (loaded % L::kStages) * L::kStage;
      constexpr int kPieces = L::kRowBytes / 16;
      const int pos0 = load.u * kChunk + 16 * warp;
      // (16 positions of a page are one run of bytes)
      const int64_t page = kPaged ? __shfl_sync(0xffffffffu, pages, load.u - pages_at) : 0;
      const int64_t run = kPaged ? ((page * w.kv_heads + load.h) << p.cache.page_shift) + (pos0 & ((1 << p.cache.page_shift) - 1)) : 0;
      const bool whole = pos0 + 16 <= load.span.len;
#pragma unroll
      for (int i = 0; i < 16 * kPieces / 32; ++i) {
        const int piece = i * 32 + lane, r = piece / kPieces, col = piece % kPieces;
        const uint32_t line = stage + (16 * warp + r) * L::kRowBytes;
        const int k_col = kDirect ? (D == 128 ? col ^ ((r & 1) << 2) : col) : kE4m3 ? col : col ^ (r & 7);
        const int v_col = kDirect ? (D == 128 ? col ^ (r & 6) : col ^ (r & 2)) : k_col;
        const uint32_t k_dst = line + (k_col << 4), v_dst = line + (v_col << 4) + L::kHalf;
        if constexpr (kPaged) {
          const uint8_t* const ks = p.cache.k + run * L::kRowBytes + piece * 16;
          const uint8_t* const vs = p.cache.v + run * L::kRowBytes + piece * 16;
          if (whole) {
            cp_async16(k_dst, ks);
            cp_async16(v_dst, vs);
          } else {
            const int there = pos0 + r < load.span.len ? 16 : 0;
            cp_async16(k_dst, ks, there);
            cp_async16(v_dst, vs, there);
          }
        } else {
          const int there = pos0 + r < load.span.len ? 16 : 0;
          const int64_t row = there ? load.span.q0 + pos0 + r : 0;
          cp_async16(k_dst, p.k + (row * p.k_row + load.h * p.k_head) * 2 + col * 16, there);
          cp_async16(v_dst, p.v + (row * p.v_row + load.h * p.v_head) * 2 + col * 16, there);
        }
      }
      if constexpr (kE4m3) {
        if (lane < 2)                                   // the 16 rows' exponent bytes, of k and of v (the positions behind the end: of no use)
          cp_async16(stage + 2 * L::kHalf + lane * kChunk + 16 * warp, (lane ? p.cache.v_exp : p.cache.k_exp) + run, pos0 < load.span.len ? 16 : 0);
      }
      if (++load.u >= load.end) {
        loading = next_item<Tiles>(w, load);
        if (loading) look_up();
      } else if (load.u - pages_at == 32) {
        look_up();
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  uint32_t q[D / 16][4];
  float o[D / 8][4];
  float m[2], l[2];
  int limit[2];                                          // last position that the thread's two rows see (-1: none)
  int tile_first_limit = 0, tile_rows = 0;
  int begun = 0;                                         // first unit of this item here
  [[maybe_unused]] float q_scale[2] = {};                // (codes) the power of two of the queries of the thread's two rows, and the scale
  // (codes) The weights of the values, p * 2^e with e a row's exponent, are f16 too, times a power of two for each row of queries, `v_unit`, which its sums have as
  // well: 2^(6 - t), where 2^(t - 4) is about the largest weight that this row has had (0: none yet). So a weight loses bits 2^18 below the largest and is lost
  // 2^27 below it, however far the rows' exponents are apart, and rows that a query does not see, or gives no weight, count for nothing. No weight is above
  // 2^(e + 8): while e <= t + 1 none is above f16's range, and the weights themselves are looked at in chunks with a larger exponent only.
  constexpr int kNone = -1000;
  [[maybe_unused]] float v_unit[2] = {};
  [[maybe_unused]] int t_low = kNone, t_high = kNone;     // the least and the largest t of the warp's rows (t_low kNone: one has none, or they are to be looked at)
  auto unit_of = [](int t) { return __uint_as_float(static_cast<uint32_t>(133 - t) << 23); };
  auto exponent_of = [](float unit) { return 133 - static_cast<int>(__float_as_uint(unit) >> 23); };

  auto begin_item = [&]() {
    begun = c.u;
    const int row0 = c.t * R, rows = c.span.n * w.group - row0;
    tile_rows = rows < R ? rows : R;
    tile_first_limit = w.causal ? c.span.len - c.span.n + row0 / w.group : c.span.len - 1;
    [[maybe_unused]] float big[2] = {};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = rw * 16 + (lane >> 2) + 8 * i;
      m[i] = -INFINITY;
      l[i] = 0.0f;
      limit[i] = -1;
      const int tok = (row0 + r) / w.group, g = row0 + r - tok * w.group;
      const bool live = r < tile_rows;
      if (live) limit[i] = w.causal ? c.span.len - c.span.n + tok : c.span.len - 1;
      const uint8_t* src = p.q + ((c.span.q0 + (live ? tok : 0)) * p.q_row + (c.h * w.group + (live ? g : 0)) * p.q_head) * 2;
      if constexpr (kDirect) {
        // elements in the order in which codes come: 16 of a piece a lane, four a step
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint2 x = live ? __ldg(reinterpret_cast<const uint2*>(src + ((kk / 4 * 4 + (lane & 3)) * 16 + kk % 4 * 4) * 2)) : make_uint2(0, 0);
          q[kk][i] = x.x;
          q[kk][i + 2] = x.y;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float2 f = unpack2<T>(e ? x.y : x.x);
            if (fabsf(f.x) <= 3.402823466e38f) big[i] = fmaxf(big[i], fabsf(f.x));
            if (fabsf(f.y) <= 3.402823466e38f) big[i] = fmaxf(big[i], fabsf(f.y));
          }
        }
      } else {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          q[kk][i] = live ? __ldg(reinterpret_cast<const uint32_t*>(src + (lane & 3) * 4 + kk * 32)) : 0;
          q[kk][i + 2] = live ? __ldg(reinterpret_cast<const uint32_t*>(src + (lane & 3) * 4 + kk * 32 + 16)) : 0;
        }
      }
    }
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[n][i] = 0.0f;
    if constexpr (kDirect) {
      // f16 under a power of two for each row, that brings its largest element to [2^14, 2^15): elements down to 2^-31 of it keep all their bits
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        big[i] = fmaxf(big[i], __shfl_xor_sync(0xffffffffu, big[i], 1));
        big[i] = fmaxf(big[i], __shfl_xor_sync(0xffffffffu, big[i], 2));
        int e = 0;
        if (big[i] > 0.0f) frexpf(big[i], &e);
        e = e < -100 ? -100 : e;
        const float up = __uint_as_float(static_cast<uint32_t>(15 - e + 127) << 23);
        q_scale[i] = __uint_as_float(static_cast<uint32_t>(e - 15 + 127) << 23) * p.scale_log2;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
          for (int j = i; j < 4; j += 2) {
            const float2 f = unpack2<T>(q[kk][j]);
            q[kk][j] = pack2<__half>(f.x * up, f.y * up);
          }
      }
      v_unit[0] = v_unit[1] = 0.0f;
      t_low = t_high = kNone;
    }
  };

  for (int item = blockIdx.x / CTAS;;) {                  // (CTAS = 1: once, with a share's items below)
    look_up();
    begin_item();                                          // (its queries before the stream of keys and values, which they would wait behind)
#pragma unroll
    for (int i = 0; i < L::kStages - 1; ++i) request(i);
    if (tid == 0) *any_special = 0;
    for (int i = tid; i < 3 * D; i += kThreads) special[i] = INT_MAX;
    __syncthreads();

    for (int done = 0; !kCluster || c.u < c.end; ++done) {
      asm volatile("cp.async.wait_group %0;" ::"n"(L::kStages - 2) : "memory");
      if constexpr (KW == 4) __syncwarp(); else __syncthreads();
      request(done + L::kStages - 1);
      const uint32_t stage = ring + (done % L::kStages) * L::kStage;
      const int pos0 = c.u * kChunk;
      uint32_t keys = stage, values = stage + L::kHalf;
      if constexpr (kE4m3 && !kDirect) {
        // this warp's 16 rows of both as bf16
        keys = ring + L::kRing;
        values = keys + kChunk * D * 2;
        if constexpr (KW != 4) __syncthreads();             // (the last chunk's are read by other warps)
        constexpr int kPieces = D / 16;
        static_assert(16 * kPieces % 32 == 0, "whole passes of a warp");
#pragma unroll
        for (int half = 0; half < 2; ++half) {
#pragma unroll
          for (int i = 0; i < 16 * kPieces / 32; ++i) {
            const int piece = i * 32 + lane, r = 16 * warp + piece / kPieces, col = piece % kPieces;
            const uint4 c16 = lds128<0>(stage + half * L::kHalf + r * D + col * 16);
            uint32_t byte = 127;
            if (pos0 + r < c.span.len) byte = lds8(stage + 2 * L::kHalf + half * kChunk + r);
            const uint32_t codes[4] = {c16.x, c16.y, c16.z, c16.w};
            uint32_t v[8];
            row_values(codes, row_factors(byte), v);
            const uint32_t row = (half ? values : keys) + r * D * 2;
            const uint32_t at0 = row + (((2 * col) ^ (r & 7)) << 4), at1 = row + (((2 * col + 1) ^ (r & 7)) << 4);
            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at0), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at1), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
          }
        }
        if constexpr (KW == 4) __syncwarp(); else __syncthreads();
      }
      // a chunk with positions that are this sequence's, but not every row's (codes by themselves are always numbers)
      if (!kDirect && pos0 + kChunk - 1 > tile_first_limit && tile_first_limit < c.span.len - 1) {
        constexpr int kPieces = D / 8;
        for (int i = 0; i < 16 * kPieces / 32; ++i) {
          const int piece = i * 32 + lane, r = 16 * warp + piece / kPieces, col = piece % kPieces;
          const uint32_t at = values + r * D * 2 + ((col ^ (r & 7)) << 4);
          const uint4 v = lds128<0>(at);
          if (odd_pair<T>(v.x) || odd_pair<T>(v.y) || odd_pair<T>(v.z) || odd_pair<T>(v.w)) {
            uint32_t u[4] = {v.x, v.y, v.z, v.w};
            for (int e = 0; e < 8; ++e) {
              const float2 pair = unpack2<T>(u[e >> 1]);
              const float x = e & 1 ? pair.y : pair.x;
              if (!(fabsf(x) <= 3.402823466e38f)) {
                atomicMin(special + (x > 0.0f ? 0 : x < 0.0f ? D : 2 * D) + col * 8 + e, pos0 + r);
                *any_special = 1;
                u[e >> 1] &= e & 1 ? 0x0000ffffu : 0xffff0000u;
              }
            }
            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]) : "memory");
          }
        }
        if constexpr (KW == 4) __syncwarp(); else __syncthreads();
      }
      // ---- scores of this warp's positions ----
      float s[SN / 8][4];
#pragma unroll
      for (int n = 0; n < SN / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[n][i] = 0.0f;
      [[maybe_unused]] float k_scale[SN / 8][2], v_scale[SN / 8][2];        // (codes: of the thread's columns; positions behind the end: 1 and 0)
      [[maybe_unused]] uint32_t v_bytes[SN / 8];
      [[maybe_unused]] bool plain = true;
      [[maybe_unused]] int low = 0, high = 0;               // (codes) exponents of this warp's rows of values
      [[maybe_unused]] float s2[SN / 8][4] = {};            // (two chains of products)
      if constexpr (kDirect) {
        const uint32_t bytes = stage + 2 * L::kHalf + kw * SN;
        const bool there = lane < SN && kw * SN + lane < c.span.len - pos0;
        const int k_byte = there ? static_cast<int>(lds8(bytes + lane)) : 127, v_byte = there ? static_cast<int>(lds8(bytes + kChunk + lane)) : 255;
        high = __reduce_max_sync(0xffffffffu, v_byte == 255 ? kNone : v_byte - 127);
        low = __reduce_min_sync(0xffffffffu, v_byte == 255 ? 1000 : v_byte - 127);
        // ordinary rows: all there, and numbers
        plain = __all_sync(0xffffffffu, lane >= SN || (there && k_byte != 255 && k_byte != 0 && v_byte != 255 && v_byte != 0));
#pragma unroll
        for (int n = 0; n < SN / 8; ++n) {
          const uint32_t k2 = lds16(bytes + n * 8 + (lane & 3) * 2);
          v_bytes[n] = lds16(bytes + kChunk + n * 8 + (lane & 3) * 2);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t kb = e ? k2 >> 8 : k2 & 255;
            k_scale[n][e] = plain ? __uint_as_float(kb << 23) : kw * SN + n * 8 + (lane & 3) * 2 + e < c.span.len - pos0 ? row_scale(kb) : 1.0f;
          }
          const int r = kw * SN + n * 8 + (lane >> 2);
#pragma unroll
          for (int h = 0; h < D / 64; ++h) {
            const int piece = h * 4 + (lane & 3);
            const uint4 codes = lds128<0>(keys + r * D + ((D == 128 ? piece ^ ((r & 1) << 2) : piece) << 4));
            const uint32_t word[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) mma16816<MT>(h == 0 ? s[n] : s2[n], q[h * 4 + i], code_half2(word[i]), code_half2(word[i] >> 16));
          }
          if constexpr (D == 128) {
#pragma unroll
            for (int i = 0; i < 4; ++i) s[n][i] += s2[n][i];
          }
        }
      } else
#pragma unroll
      for (int n = 0; n < SN / 16; ++n) {
        const int r = kw * SN + n * 16 + (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          uint32_t b[4];
          ldmatrix4(b, keys + r * D * 2 + (((kk * 2 + ((lane >> 3) & 1)) ^ (r & 7)) << 4));
          mma16816<MT>(s[2 * n], q[kk], b[0], b[1]);
          mma16816<MT>(s[2 * n + 1], q[kk], b[2], b[3]);
        }
      }
      const int warp_pos = pos0 + kw * SN;
      const bool edge = warp_pos + SN - 1 > tile_first_limit;          // (rows behind the tile's last: whatever their sums are, none reads them)
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int n = 0; n < SN / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[n][i] *= kDirect ? k_scale[n][i & 1] * q_scale[i >> 1] : p.scale_log2;
        }
      if (edge) {
#pragma unroll
        for (int n = 0; n < SN / 8; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (warp_pos + n * 8 + (lane & 3) * 2 + (i & 1) > limit[i >> 1]) s[n][i] = -INFINITY;
      }
#pragma unroll
      for (int n = 0; n < SN / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) top[i >> 1] = fmaxf(top[i >> 1], s[n][i]);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
        top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
      }
      // the maximum is followed loosely: sums are scaled down when a row's has risen by more than a factor of 2^8, for all rows of the warp at once
      if (__any_sync(0xffffffffu, top[0] > m[0] + 8.0f || top[1] > m[1] + 8.0f)) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float now = fmaxf(m[i], top[i]), base = now == -INFINITY ? 0.0f : now;
          float shrink = ex2(m[i] - base);
          l[i] *= shrink;
          if constexpr (kDirect) {                          // the weights so far shrink, and their power of two with them
            if (v_unit[i] > 0.0f && now > m[i]) {
              const int t = exponent_of(v_unit[i]), fall = min(static_cast<int>(fminf(now - m[i], 300.0f)), t + 117);
              v_unit[i] = unit_of(t - fall);
              shrink = ex2(m[i] - base + static_cast<float>(fall));
            }
          }
          m[i] = now;
#pragma unroll
          for (int n = 0; n < D / 8; ++n) {
            o[n][2 * i] *= shrink;
            o[n][2 * i + 1] *= shrink;
          }
        }
        t_low = kNone;
      }
      if constexpr (kDirect) {
#pragma unroll
        for (int n = 0; n < SN / 8; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t vb = e ? v_bytes[n] >> 8 : v_bytes[n] & 255;
            v_scale[n][e] = plain ? __uint_as_float(vb << 23) : warp_pos + n * 8 + (lane & 3) * 2 + e < c.span.len ? row_scale(vb) : 0.0f;
          }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float base = m[i] == -INFINITY ? 0.0f : m[i];
#pragma unroll
        for (int n = 0; n < SN / 8; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float x = ex2(s[n][2 * i + e] - base);
            l[i] += x;
            s[n][2 * i + e] = kDirect ? x * v_scale[n][e] : x;           // (the values' power of two goes to their weights)
          }
      }
      if (kDirect && edge) {                                // a masked weight is zero whatever that is
#pragma unroll
        for (int n = 0; n < SN / 8; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (warp_pos + n * 8 + (lane & 3) * 2 + (i & 1) > limit[i >> 1]) s[n][i] = 0.0f;
      }
      // Rows of values more than 2^14 below t would lose bits where their weights are small: rows of queries that see one take this chunk's weights in bf16.
      [[maybe_unused]] bool wide[2] = {false, false}, any_wide = false, all_wide = false;
      if constexpr (kDirect) {
        const bool apart = warp_pos + SN - 1 > tile_first_limit && tile_first_limit < c.span.len - 1;        // positions that only some rows see: all that follows is by what a row sees
        if (high > t_low + 1 || t_high - low > 14 || apart) {
          int least = 1000, most = kNone, mine[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float big = 0.0f;
#pragma unroll
            for (int n = 0; n < SN / 8; ++n) big = fmaxf(big, fmaxf(s[n][2 * i], s[n][2 * i + 1]));
            big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
            big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
            const int old = v_unit[i] > 0.0f ? exponent_of(v_unit[i]) : kNone, t = max(static_cast<int>(__float_as_uint(big) >> 23) - 127 + 4, -117);
            mine[i] = old;
            if (big > 0.0f && t > old) {
              if (old != kNone) {
                const float down = t - old > 126 ? 0.0f : __uint_as_float(static_cast<uint32_t>(127 - (t - old)) << 23);
#pragma unroll
                for (int n = 0; n < D / 8; ++n) {
                  o[n][2 * i] *= down;
                  o[n][2 * i + 1] *= down;
                }
              }
              v_unit[i] = unit_of(t);
              mine[i] = t;
            }
            if (limit[i] >= 0) {
              least = min(least, mine[i]);
              most = max(most, mine[i]);
            }
          }
          t_low = __reduce_min_sync(0xffffffffu, least);
          t_high = __reduce_max_sync(0xffffffffu, most);
          if (t_high - low > 14) {
            // the least exponent of the first 1, 2, .. 16 positions, in a lane each
            const int byte = lane < SN && warp_pos + lane < c.span.len ? static_cast<int>(lds8(stage + 2 * L::kHalf + kChunk + kw * SN + lane)) : 255;
            int upto = byte == 255 ? 1000 : byte - 127;
#pragma unroll
            for (int d = 1; d < SN; d <<= 1) {
              const int x = __shfl_up_sync(0xffffffffu, upto, d);
              if (lane >= d) upto = min(upto, x);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int last = limit[i] - warp_pos, seen = __shfl_sync(0xffffffffu, upto, last < 0 ? 0 : last < SN ? last : SN - 1);
              wide[i] = last >= 0 && mine[i] - seen > 14;
            }
            any_wide = __any_sync(0xffffffffu, wide[0] || wide[1]);
            all_wide = __all_sync(0xffffffffu, (wide[0] || limit[0] < 0) && (wide[1] || limit[1] < 0));
          }
        }
#pragma unroll
        for (int n = 0; n < SN / 8; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[n][i] *= v_unit[i >> 1];
      }
      // ---- weights times values ----
#pragma unroll
      for (int n = 0; n < SN / 16; ++n) {
        uint32_t a[4] = {pack2<MT>(s[2 * n][0], s[2 * n][1]), pack2<MT>(s[2 * n][2], s[2 * n][3]), pack2<MT>(s[2 * n + 1][0], s[2 * n + 1][1]),
                         pack2<MT>(s[2 * n + 1][2], s[2 * n + 1][3])};
        if constexpr (kDirect) {
          // a thread's D / 8 codes of the four positions that its B fragments hold: column `lane / 4` of every fragment
          const int r = kw * SN + n * 16 + (lane & 3) * 2, g = lane >> 2;
          uint32_t codes[4][D / 32];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int row = r + (i & 1) + (i >> 1) * 8;
            const uint32_t at = values + row * D;
            if constexpr (D == 128) {
              const uint4 v = lds128<0>(at + ((g ^ (row & 6)) << 4));
              codes[i][0] = v.x;
              codes[i][1] = v.y;
              codes[i][2] = v.z;
              codes[i][3] = v.w;
            } else {
              const uint2 v = lds64<0>(at + (((g >> 1) ^ (row & 2)) << 4) + (g & 1) * 8);
              codes[i][0] = v.x;
              codes[i][1] = v.y;
            }
          }
          if (any_wide) {
            uint32_t b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              b[i] = wide[i & 1] ? pack2<T>(s[2 * n + (i >> 1)][(i & 1) * 2], s[2 * n + (i >> 1)][(i & 1) * 2 + 1]) : 0;
              if (wide[i & 1]) a[i] = 0;
            }
#pragma unroll
            for (int x = 0; x < D / 32; ++x) {
              mma16816<T>(o[4 * x], b, code_pair<0>(codes[0][x], codes[1][x]), code_pair<0>(codes[2][x], codes[3][x]));
              mma16816<T>(o[4 * x + 1], b, code_pair<1>(codes[0][x], codes[1][x]), code_pair<1>(codes[2][x], codes[3][x]));
              mma16816<T>(o[4 * x + 2], b, code_pair<2>(codes[0][x], codes[1][x]), code_pair<2>(codes[2][x], codes[3][x]));
              mma16816<T>(o[4 * x + 3], b, code_pair<3>(codes[0][x], codes[1][x]), code_pair<3>(codes[2][x], codes[3][x]));
            }
          }
          if (!all_wide) {
#pragma unroll
            for (int x = 0; x < D / 32; ++x) {
              mma16816<MT>(o[4 * x], a, code_half2<0>(codes[0][x], codes[1][x]), code_half2<0>(codes[2][x], codes[3][x]));
              mma16816<MT>(o[4 * x + 1], a, code_half2<1>(codes[0][x], codes[1][x]), code_half2<1>(codes[2][x], codes[3][x]));
              mma16816<MT>(o[4 * x + 2], a, code_half2<2>(codes[0][x], codes[1][x]), code_half2<2>(codes[2][x], codes[3][x]));
              mma16816<MT>(o[4 * x + 3], a, code_half2<3>(codes[0][x], codes[1][x]), code_half2<3>(codes[2][x], codes[3][x]));
            }
          }
        } else {
          const int r = kw * SN + n * 16 + (lane & 7) + (((lane >> 3) & 1) << 3);
#pragma unroll
          for (int dd = 0; dd < D / 16; ++dd) {
            uint32_t b[4];
            ldmatrix4t(b, values + r * D * 2 + (((dd * 2 + (lane >> 4)) ^ (r & 7)) << 4));
            mma16816<MT>(o[2 * dd], a, b[0], b[1]);
            mma16816<MT>(o[2 * dd + 1], a, b[2], b[3]);
          }
        }
      }
      ++c.u;
      if (c.u < c.end) continue;

      // ---- the item, or this CTA's part of it, ends: its warps' sums meet where the chunk was (e4m3: where its values were) ----
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
      }
      if constexpr (kDirect) {
        // In units of one, and both sums with the maximum under a power of two that leaves them 2^12 below the largest value: what joins up to as many of them
        // stays in float32's range as the result does. (Of small values less: one factor in range.)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int t = v_unit[i] > 0.0f ? exponent_of(v_unit[i]) : 6;
          const int below = min(12 + min(max(static_cast<int>(__float_as_uint(l[i]) >> 23) - 126, 0), 48), t + 120);
          const float unit = __uint_as_float(static_cast<uint32_t>(127 + t - 6 - below) << 23);
          l[i] *= __uint_as_float(static_cast<uint32_t>(127 - below) << 23);
          m[i] += static_cast<float>(below);
#pragma unroll
          for (int n = 0; n < D / 8; ++n) {
            o[n][2 * i] *= unit;
            o[n][2 * i + 1] *= unit;
          }
        }
      }
      __syncthreads();
      float* const sums = reinterpret_cast<float*>(smem + (kE4m3 && !kDirect ? L::kRing : kCluster ? L::kStage : stage - ring));
      constexpr int kPasses = kDirect ? 2 : 1, kPart = 16 / kPasses;       // a stage of codes holds eight rows of each warp's sums, the other places all sixteen
      const bool first = begun == 0, last = c.u == c.units;
      const bool odd = *any_special != 0;
      float* const part = p.partial + (2 * static_cast<int64_t>(blockIdx.x) + (first ? 1 : 0)) * partial_floats<R, D>();
      constexpr int kVec = D / 4;                           // threads of a row
#pragma unroll
      for (int pass = 0; pass < kPasses; ++pass) {
        if (pass * kPart >= tile_rows) break;
        if (pass) __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = (lane >> 2) + 8 * i, sr = warp * kPart + (kDirect ? lane >> 2 : r);
          if (pass == 0 && (lane & 3) == 0) {
            stats[warp * 16 + r] = m[i];
            stats[kChunk + warp * 16 + r] = l[i];
          }
          if (kDirect && i != pass) continue;
#pragma unroll
          for (int n = 0; n < D / 8; ++n)
            *reinterpret_cast<float2*>(sums + sr * D + ((n * 8 + (lane & 3) * 2) ^ ((sr & 3) << 3))) = make_float2(o[n][2 * i], o[n][2 * i + 1]);
        }
        __syncthreads();
        const int row_end = kDirect && tile_rows > (pass + 1) * kPart ? (pass + 1) * kPart : tile_rows;
        for (int i = pass * kPart * kVec + tid; i < row_end * kVec; i += kThreads) {
          const int r = i / kVec, d = (i % kVec) * 4;
          const int tok = (c.t * R + r) / w.group, g = c.t * R + r - tok * w.group;
          const int seen = w.causal ? c.span.len - c.span.n + tok : c.span.len - 1;
          float mm = -INFINITY, ll = 0.0f, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int k = 0; k < KW; ++k) mm = fmaxf(mm, stats[((r / 16) * KW + k) * 16 + r % 16]);
          const float base = mm == -INFINITY ? 0.0f : mm;
#pragma unroll
          for (int k = 0; k < KW; ++k) {
            const int at = ((r / 16) * KW + k) * 16 + r % 16, sr = ((r / 16) * KW + k) * kPart + r % kPart;
            const float f = ex2(stats[at] - base);
            ll = fmaf(f, stats[kChunk + at], ll);
            if constexpr (kDirect) {                        // fragment t, column n: element n * D / 8 + t
#pragma unroll
              for (int e = 0; e < 4; ++e) v[e] = fmaf(f, sums[sr * D + (((d + e) % (D / 8) * 8 + d / (D / 8)) ^ ((sr & 3) << 3))], v[e]);
            } else {
              const float4 x = *reinterpret_cast<const float4*>(sums + sr * D + (d ^ ((sr & 3) << 3)));
              v[0] = fmaf(f, x.x, v[0]);
              v[1] = fmaf(f, x.y, v[1]);
              v[2] = fmaf(f, x.z, v[2]);
              v[3] = fmaf(f, x.w, v[3]);
            }
          }
          if (odd) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (special[d + e] <= seen) v[e] += INFINITY;
              if (special[D + d + e] <= seen) v[e] -= INFINITY;
              if (special[2 * D + d + e] <= seen) v[e] = NAN;
            }
          }
          if constexpr (kCluster) {
            *reinterpret_cast<float4*>(part_rows + r * D + d) = make_float4(v[0], v[1], v[2], v[3]);
            if (d == 0) {
              part_stats[r] = mm;
              part_stats[R + r] = ll;
            }
          } else if (first && last) {
            store_row<T>(p, c, tok, g, d, D, v, ll, seen);
          } else {
            *reinterpret_cast<float4*>(part + r * D + d) = make_float4(v[0], v[1], v[2], v[3]);
            if (d == 0) {
              part[R * D + r] = mm;
              part[R * D + R + r] = ll;
            }
          }
        }
      }
      if (odd) {
        __syncthreads();
        for (int i = tid; i < 3 * D; i += kThreads) special[i] = INT_MAX;
        if (tid == 0) *any_special = 0;
      }
      if constexpr (kCluster) break;
      __syncthreads();
      if (c.end < c.units && tid == 0) p.notes[blockIdx.x] = note_of(c, begun, share);
      if (!next_item<Tiles>(w, c)) break;
      begin_item();
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if constexpr (!kCluster) return;
    if (begun == c.end) {                                   // a CTA without positions: no weight, and zeros
      for (int i = tid; i < R * D; i += kThreads) part_rows[i] = 0.0f;
      for (int i = tid; i < 2 * R; i += kThreads) part_stats[i] = i < R ? -INFINITY : 0.0f;
    }
    tc::cluster_barrier();                                  // the parts are there
    constexpr int kVec = D / 4;
    const int rank = blockIdx.x % CTAS;
    for (int i = tid; i < (tile_rows - rank + CTAS - 1) / CTAS * kVec; i += kThreads) {
      const int r = rank + i / kVec * CTAS, d = i % kVec * 4;
      const int tok = (c.t * R + r) / w.group, g = c.t * R + r - tok * w.group;
      const int seen = w.causal ? c.span.len - c.span.n + tok : c.span.len - 1;
      float m_of[CTAS], l_of[CTAS], mm = -INFINITY, ll = 0.0f, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      float4 x[CTAS];
#pragma unroll
      for (int k = 0; k < CTAS; ++k) {
        const uint32_t stats_at = tc::in_cta(smem_u32(part_stats), k) + r * 4;
        x[k] = tc::remote_ld128(tc::in_cta(ring, k) + (r * D + d) * 4);
        m_of[k] = remote_ld32(stats_at);
        l_of[k] = remote_ld32(stats_at + R * 4);
        mm = fmaxf(mm, m_of[k]);
      }
      const float base = mm == -INFINITY ? 0.0f : mm;
#pragma unroll
      for (int k = 0; k < CTAS; ++k) {
        const float f = ex2(m_of[k] - base);
        ll = fmaf(f, l_of[k], ll);
        v[0] = fmaf(f, x[k].x, v[0]);
        v[1] = fmaf(f, x[k].y, v[1]);
        v[2] = fmaf(f, x[k].z, v[2]);
        v[3] = fmaf(f, x[k].w, v[3]);
      }
      store_row<T>(p, c, tok, g, d, D, v, ll, seen);
    }
    tc::cluster_barrier();                                  // ... and have been read
    item += gridDim.x / CTAS;
    if (!cluster_item<Tiles>(w, item, rank, CTAS, &c)) return;
    load = c;
    loading = c.u < c.end;
  }
}

// Items whose units fell to several CTAs: block (b, y) joins eight rows of the one that CTA b began and did not finish, a warp each.
constexpr int kJoinThreads = 256, kJoinRows = kJoinThreads / 32;
template <typename T, int D, int R>
__global__ void __launch_bounds__(kJoinThreads) attend_join_kernel(const JoinParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const AttentionWork& w = p.work;
  const JoinNote c = p.notes[blockIdx.x];
  const int r = blockIdx.y * kJoinRows + (threadIdx.x >> 5), lane = threadIdx.x & 31, row = c.t * R + r;
  if (c.parts == 0 || row >= c.n * w.group) return;
  constexpr int V = D / 32;                                                       // elements of a lane
  // (the first part lies behind this CTA's finished item, the others are the first of theirs)
  const float* const first = p.partial + (2 * static_cast<int64_t>(blockIdx.x) + 1) * partial_floats<R, D>();
  const float* const others = p.partial + 2 * static_cast<int64_t>(blockIdx.x) * partial_floats<R, D>();
  auto part_of = [&](int i) { return i == 0 ? first : others + 2ll * i * partial_floats<R, D>(); };
  // eight parts' loads on their way at once
  constexpr int kBatch = 8;
  float mm = -INFINITY, ll = 0.0f, v[V] = {};
  for (int i0 = 0; i0 < c.parts; i0 += kBatch) {
    float x[kBatch][V], m[kBatch], l[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const float* const part = part_of(i0 + i < c.parts ? i0 + i : i0);
      m[i] = part[R * D + r];
      l[i] = part[R * D + R + r];
      if constexpr (V == 4) {
        const float4 y = *reinterpret_cast<const float4*>(part + r * D + lane * V);
        x[i][0] = y.x;
        x[i][1] = y.y;
        x[i][2] = y.z;
        x[i][3] = y.w;
      } else {
        const float2 y = *reinterpret_cast<const float2*>(part + r * D + lane * V);
        x[i][0] = y.x;
        x[i][1] = y.y;
      }
    }
    float top = mm;
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      if (i0 + i < c.parts) top = fmaxf(top, m[i]);
    const float base = top == -INFINITY ? 0.0f : top, shrink = ex2(mm - base);
    mm = top;
    ll *= shrink;
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] *= shrink;
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      if (i0 + i < c.parts) {
        const float f = ex2(m[i] - base);
        ll = fmaf(f, l[i], ll);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = fmaf(f, x[i][e], v[e]);
      }
  }
  const int tok = row / w.group, g = row - tok * w.group;
  const int seen = w.causal ? c.len - c.n + tok : c.len - 1;
  const float inv = ll == 0.0f ? (seen < 0 ? 0.0f : NAN) : 1.0f / ll;
  uint8_t* dst = p.out + ((static_cast<int64_t>(c.q0) + tok) * w.heads + c.h * w.group + g) * D * 2 + lane * V * 2;
#pragma unroll
  for (int e = 0; e < V; e += 2) *reinterpret_cast<uint32_t*>(dst + e * 2) = pack2<T>(v[e] * inv, v[e + 1] * inv);
}

template <typename T, int D, int RW, int SOURCE>
int launch_one(const RowsParams& p, cudaStream_t stream) {
  const int ctas = RowsLayout<D, SOURCE, RW>::kCtas * device_sm_count();
  static bool done[kMaxDevices] = {};
  const int dev = current_device();
  if (dev < 0) return QMM_ERR_DEVICE;
  if (!done[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(attend_rows_kernel<T, D, RW, SOURCE, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, RowsLayout<D, SOURCE, RW>::kBytes);
    if (e != cudaSuccess) return fail(QMM_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    done[dev] = true;
  }
  launch_early(attend_rows_kernel<T, D, RW, SOURCE, 1>, ctas, kThreads, RowsLayout<D, SOURCE, RW>::kBytes, stream, p);
  count_launch();
  if (int rc = check_launch("attend_rows_kernel")) return rc;
  // sequences of one chunk at most: nothing to join
  const int64_t longest = SOURCE == kRowsSource ? p.work.tokens : p.work.longest;
  if (ctas < 2 || longest <= kChunk) return QMM_OK;
  static_assert(RowTiles<16 * RW, kChunk>::kWhole == 2, "items of one unit are whole");
  JoinParams j = {p.work, p.out, p.notes, p.partial};
  launch_early(attend_join_kernel<T, D, 16 * RW>, dim3(ctas - 1, 16 * RW / kJoinRows), kJoinThreads, 0, stream, j);
  count_launch();
  return check_launch("attend_join_kernel");
}

template <typename T, int D, int RW, int SOURCE, int CTAS>
int launch_clusters(const RowsParams& p, cudaStream_t stream) {
  static bool done[kMaxDevices] = {};
  const int dev = current_device();
  if (dev < 0) return QMM_ERR_DEVICE;
  auto kernel = attend_rows_kernel<T, D, RW, SOURCE, CTAS>;
  constexpr int kBytes = RowsLayout<D, SOURCE, RW>::kBytes + 2 * 16 * RW * 4;
  if (!done[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
    if (e != cudaSuccess) return fail(QMM_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    done[dev] = true;
  }
  // (a sequence's last tile may be short; items beyond what the device holds at once are taken in turn)
  const int64_t items = (p.work.tokens * p.work.group / (16 * RW) + p.work.seqs) * p.work.kv_heads, room = 2 * device_sm_count() / CTAS;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(items < room ? items : room) * CTAS);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CTAS;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaLaunchKernelEx(&cfg, kernel, p);
  count_launch();
  return check_launch("attend_rows_kernel");
}

template <typename T, int D, int RW, int SOURCE>
int launch_tiles(const RowsParams& p, cudaStream_t stream) {
  const int ctas = attend_cluster_ctas(p, SOURCE, 16 * RW);
  if (ctas == 8) return launch_clusters<T, D, RW, SOURCE, 8>(p, stream);
  if (ctas == 4) return launch_clusters<T, D, RW, SOURCE, 4>(p, stream);
  return launch_one<T, D, RW, SOURCE>(p, stream);
}

template <typename T, int D, int SOURCE>
int launch_rows_of(const RowsParams& p, int rows, cudaStream_t stream) {
  if (rows <= 16) return launch_tiles<T, D, 1, SOURCE>(p, stream);
  if (rows <= 32) return launch_tiles<T, D, 2, SOURCE>(p, stream);
  return launch_tiles<T, D, 4, SOURCE>(p, stream);
}

template <typename T, int D>
int launch_source(const RowsParams& p, int source, int rows, cudaStream_t stream) {
  if (source == kRowsSource) return launch_one<T, D, 2, kRowsSource>(p, stream);
  if (source == kPages16) return launch_rows_of<T, D, kPages16>(p, rows, stream);
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return launch_rows_of<T, D, kPages8>(p, rows, stream);
  return fail(QMM_ERR_UNSUPPORTED, "attention: an e4m3 cache is attended with bf16 queries");
}

}  // namespace

// Clusters want neither the order of all units (2 us) nor a second launch to join (3.5 us): eight CTAs a sequence and key head where the device holds as many for all, at
// two an SM, else four. They pay while no CTA has many positions to do: without shares by weight no others help it, and codes want three CTAs an SM. Measured with 8
// key heads of 128, us, clusters / shares, two calls' inputs in turn. Tiles of 16 rows: 1 sequence of 2000 positions 8.1 / 11.7, 8000 15.6 / 16.2, 16000 26.9 / 23.6; 8 of
// 500 to 2000 11.6 / 12.8, 1000 to 4000 20.6 / 21.1, 2000 to 8000 36.0 / 35.1; of codes: 1 of 2000 10.8 / 15.3, 4000 15.0 / 16.5, 8000 23.6 / 20.1; 8 of 500 to 2000 16.2 / 18.1,
// 1000 to 4000 26.0 / 22.2. (Heads of 64: 1 of 8000 11.4 / 13.2, 16000 17.9 / 16.0; 8 of 1000 to 4000 13.9 / 14.0; of codes: 1 of 4000 12.7 / 13.2, 8000 20.0 / 15.4; 8 of
// 500 to 2000 13.4 / 14.1, 1000 to 4000 22.0 / 16.6.) Tiles of 32 rows: 1 of 4000 15.5 / 17.0, 8000 23.2 / 20.0; 8 of 2000 19.6 / 24.0, 1000 to 4000 27.1 / 28.1; of codes
// 22.1 / 20.7, 36.3 / 23.8, 24.9 / 29.2, 40.4 / 35.7. Tiles of 64 rows, against the kernel of 2 x 128: 1 of 4000 21.1 / 23.2; 8 of 2000 26.6 / 31.4; of codes 29.2 / 28.8,
// 32.0 / 38.7; 8 of 500 to 2000 with 40 rows on average and up to 76 in two tiles 26.5 / 21.7.
int attend_cluster_ctas(const RowsParams& p, int source, int rows) {
  const int64_t items = static_cast<int64_t>(p.work.seqs) * p.work.kv_heads, room = 2 * device_sm_count();
  const int ctas = items * 8 <= room ? 8 : 4;
  const bool few = source == kPages16 && rows <= 16 ? p.work.longest <= 1024 * ctas : p.work.longest <= 512 * ctas;
  return source != kRowsSource && rows <= 64 && items * ctas <= room && few ? ctas : 0;
}

int attend_rows_ctas() { return 3 * device_sm_count(); }

int64_t attend_rows_workspace(int head_dim, int ctas) {
  return ctas * (sizeof(JoinNote) + 2ll * (head_dim == 64 ? partial_floats<64, 64>() : partial_floats<64, 128>()) * 4);
}

int launch_attend_rows(const RowsParams& p, int elem, int head_dim, int source, int rows, cudaStream_t stream) {
  if (elem == QMM_BF16) return head_dim == 64 ? launch_source<__nv_bfloat16, 64>(p, source, rows, stream) : launch_source<__nv_bfloat16, 128>(p, source, rows, stream);
  return head_dim == 64 ? launch_source<__half, 64>(p, source, rows, stream) : launch_source<__half, 128>(p, source, rows, stream);
}

}  // namespace qmm
