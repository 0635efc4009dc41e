// Attention of query tiles of up to 2 x 128 rows on tcgen05: prompts, and chunks of new tokens over a cache.
//
//   S = Q K^T             both from shared memory (TMA, 128-byte swizzle), [128 x 128] float32 in tensor memory
//   P = 2^(S scale - m)   by the thread that owns the row: tcgen05.ld -> registers -> 16-bit -> tcgen05.st over S's own columns
//   O += P V              P is the A operand in tensor memory, V the B operand as it lies, positions by elements (MN-major)
//
// A tile is two halves of 128 rows (whole tokens of the group's heads, so that a key is read once for all of them) on the same keys: while one
// half's 128 threads take the exponentials of a block of 128 positions, the tensor cores work for the other one. Tensor memory is full with both
// halves' S and O (512 columns), so one CTA an SM, persistent: its share of the call's units is a range of their order (attention_plan.cuh).
//
// The running maximum is followed loosely: O is only scaled down when a row's maximum has risen by more than a factor of 2^8 (no warp does it for less),
// so that O stays in tensor memory; weights up to 2^8 are as exact as ones below 1 in a floating format. S's barrier says that the block before has
// been added up (MMAs complete in order), so scaling O needs none of its own.
//
// Masked positions: scores are selected. Two helper warps look at the blocks of v that some row does not see all of, before the tensor cores
// do: rows behind the sequence's end become zeros (0 times what stands in a page behind the end may be NaN), and infinities and NaN that only some
// rows see are taken out and put into those rows' sums at the end.
//
// An e4m3 cache's blocks arrive as codes, and six helpers turn them into bf16 in the products' layout (exactly); there the only values that are no numbers
// are rows whose exponent byte says so.
//
// Warps: 0..3 and 4..7 the halves' rows, 8 the MMAs' issuer, 9 the copies, from 10 on helpers. Waits are bounded, as everywhere.
#include <climits>
#include <type_traits>

#include "attention.h"
#include "qmm_tcgen05.cuh"

namespace qmm {
namespace {

using namespace tc;

constexpr int kBlock = 128;
enum Source { kRowsSource, kPages16, kPages8 };
using Tiles = TokenTiles<kBlock>;

template <int D, int SOURCE>
struct TcLayout {
  static constexpr bool kE4m3 = SOURCE == kPages8;
  static constexpr int kHelpers = kE4m3 ? 6 : 2, kThreads = (10 + kHelpers) * 32;
  static constexpr int kTile = D / 64 * 16384;         // 128 rows: columns of 64 elements, 128 bytes a row, one behind the other
  static constexpr int kKeys = D == 64 ? (kE4m3 ? 3 : 5) : 2, kValues = D == 64 ? (kE4m3 ? 3 : 5) : kE4m3 ? 2 : 3;       // blocks on their way or at work
  static constexpr int kCodes = kE4m3 ? 2 : 0;         // blocks of codes on their way, keys and values in turn
  static constexpr int kKeyRing = 2 * kTile;           // behind Q's halves
  static constexpr int kValueRing = kKeyRing + kKeys * kTile;
  static constexpr int kCodeRing = kValueRing + kValues * kTile;
  static constexpr int kExps = kCodeRing + kCodes * kBlock * D;          // the codes' rows' exponent bytes
  static constexpr int kSpecials = kExps + kCodes * kBlock;
  static constexpr int kBars = kSpecials + (kE4m3 ? 0 : kHelpers * 3 * D * 2);           // 16-bit places, a set for each helper
  static constexpr int kNumBars = 2 * kKeys + 3 * kValues + 2 * kCodes + 15;
  static constexpr int kWords = kBars + 8 * kNumBars;  // tensor memory's address, abort flag, and counters
  static constexpr int kBytes = kWords + 128 + 1024;   // (what is swizzled begins at a multiple of 1024)
};

// A, B in shared memory, both K-major: D / 16 steps of 16 elements.
#define QMM_SS(AO, BO, ACC)                                                                                  \
  "add.u32 al, %1, " AO "; add.u32 bl, %2, " BO "; mov.b64 a, {al, %3}; mov.b64 b, {bl, %3};"               \
  "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, " ACC ";"
template <int D>
__device__ __forceinline__ void mma_scores(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc) {
  if constexpr (D == 64)
    asm volatile("{ .reg .pred e, t, f; .reg .b32 al, bl; .reg .b64 a, b; elect.sync _|e, 0xffffffff; setp.eq.b32 t, 0, 0; setp.ne.b32 f, 0, 0;"
                 QMM_SS("0", "0", "f") QMM_SS("2", "2", "t") QMM_SS("4", "4", "t") QMM_SS("6", "6", "t") "}" ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc) : "memory");
  else
    asm volatile("{ .reg .pred e, t, f; .reg .b32 al, bl; .reg .b64 a, b; elect.sync _|e, 0xffffffff; setp.eq.b32 t, 0, 0; setp.ne.b32 f, 0, 0;"
                 QMM_SS("0", "0", "f") QMM_SS("2", "2", "t") QMM_SS("4", "4", "t") QMM_SS("6", "6", "t")
                 QMM_SS("1024", "1024", "t") QMM_SS("1026", "1026", "t") QMM_SS("1028", "1028", "t") QMM_SS("1030", "1030", "t") "}"
                 ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc) : "memory");
}
// A in tensor memory (8 columns a step of 16 positions), B in shared memory as rows of positions: 16 of them are 2048 bytes.
#define QMM_TS(COL, BO, ACC)                                                                                 \
  "add.u32 a, %1, " COL "; add.u32 bl, %2, " BO "; mov.b64 b, {bl, %3};"                                    \
  "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %4, " ACC ";"
__device__ __forceinline__ void mma_values(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{ .reg .pred e, p, t; .reg .b32 a, bl; .reg .b64 b; elect.sync _|e, 0xffffffff; setp.ne.b32 p, %5, 0; setp.eq.b32 t, 0, 0;"
               QMM_TS("0", "0", "p") QMM_TS("8", "128", "t") QMM_TS("16", "256", "t") QMM_TS("24", "384", "t") "}"
               ::"r"(d), "r"(a), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate) : "memory");
}
// MN-major operand in the 128-byte swizzle: columns of 64 elements (leading byte offset) and groups of 8 positions (stride byte offset).
__device__ __forceinline__ uint32_t desc_low_mn(uint32_t saddr) { return ((saddr & 0x3FFFFu) >> 4) | ((16384u >> 4) << 16); }

__device__ __forceinline__ void tma_load_3d(const CUtensorMap* map, uint32_t dst, uint32_t bar, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"(map), "r"(bar), "r"(c0),
               "r"(c1), "r"(c2)
               : "memory");
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {       // 16-byte aligned, a multiple of 16 bytes
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
__device__ __forceinline__ uint64_t pack_f32(float a, float b) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  return v;
}
__device__ __forceinline__ float2 unpack_f32(uint64_t v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      QMM_ASM_R(0), QMM_ASM_R(8), QMM_ASM_R(16), QMM_ASM_R(24)
      : "memory");
}

template <typename T>
__device__ __forceinline__ bool odd_pair(uint32_t w) {
  constexpr uint32_t kExp = std::is_same<T, __nv_bfloat16>::value ? 0x7f80u : 0x7c00u;
  return (w & kExp) == kExp || (w >> 16 & kExp) == kExp;
}

// A place in a ring. Keys and values have rings of their own: a wait knows a phase only from the one before it, so whoever waits for a ring's copies has
// to wait for each of them in turn (or could take the phase before for the one it wants: copies do not land in order), and has to hold up the
// next ones (or could be lapped). The issuer does so for keys, the helpers for values.
template <int N>
struct Slot {
  uint32_t slot, phase;
  __device__ __forceinline__ void next() {
    if (++slot == N) {
      slot = 0;
      phase ^= 1u;
    }
  }
};

// 32 bytes of a row: a sector at once where the result is aligned to that, else (16 bytes) in two stores.
__device__ __forceinline__ void store32(uint8_t* at, const uint32_t (&v)[8], bool sector) {
  if (sector) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
  } else {
    reinterpret_cast<uint4*>(at)[0] = make_uint4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<uint4*>(at)[1] = make_uint4(v[4], v[5], v[6], v[7]);
  }
}

// What a CTA does of an item: units from `begin` on, of which each half sees those before its own `last`.
struct Part {
  int begin, seen[2], last[2], load_end;
  bool live;
};
__device__ __forceinline__ Part part_of(const AttentionWork& w, const UnitCursor& c) {
  Part r;
  r.begin = c.u;
  const int token = c.t * 2 * w.tile_tokens;
  r.seen[0] = seen_by(w, c.span, token + w.tile_tokens);
  r.seen[1] = token + w.tile_tokens < c.span.n ? seen_by(w, c.span, token + 2 * w.tile_tokens) : 0;
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int u = (r.seen[x] + kBlock - 1) / kBlock;
    r.last[x] = u < c.end ? u : c.end;
    if (r.last[x] < r.begin) r.last[x] = r.begin;
  }
  r.load_end = r.last[0] > r.last[1] ? r.last[0] : r.last[1];
  r.live = r.load_end > r.begin;
  return r;
}

// Blocks that are looked at begin no more than 127 before the first position that the tile's first row does not see, and end less than 128 behind the
// last that its last row sees: a place counted from here has 10 bits. (An unwritten one, 0xffff, is above every row's.)
__device__ __forceinline__ int place_of(int first_limit) { return (first_limit > 0 ? first_limit : 0) - 127; }

template <typename T, int D, int SOURCE>
__global__ void __launch_bounds__((TcLayout<D, SOURCE>::kThreads), 1)
attend_tc_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                 const RowsParams p) {
  using L = TcLayout<D, SOURCE>;
  constexpr bool PAGED = SOURCE != kRowsSource, kE4m3 = L::kE4m3;
  constexpr int kHelpers = L::kHelpers, kTags = 2, kHelped = 8, kWritten = 14, kNanPlace = 22;      // words
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* const smem = smem_raw + (base - raw);
  uint16_t* const special = reinterpret_cast<uint16_t*>(smem + L::kSpecials);      // [helper][+inf, -inf, NaN][D]: first place with one in a column of v
  // [kTags + helper] item whose specials its set holds, [kHelped + helper] items it has been through, [kWritten + warp of rows] items it has written
  volatile int* const words = reinterpret_cast<volatile int*>(smem + L::kWords);
  const uint32_t key_ring = base + L::kKeyRing, value_ring = base + L::kValueRing, bars = base + L::kBars;
  const uint32_t q_full = bars, q_empty = bars + 16, k_full = bars + 32, k_empty = k_full + 8 * L::kKeys;
  const uint32_t v_full = k_empty + 8 * L::kKeys, v_empty = v_full + 8 * L::kValues, v_clean = v_empty + 8 * L::kValues;
  const uint32_t c_full = v_clean + 8 * L::kValues, c_empty = c_full + 8 * L::kCodes;
  const uint32_t s_full = c_empty + 8 * L::kCodes, p_full = s_full + 16, o_full = p_full + 32, o_free = o_full + 16, done = o_free + 16;
  const uint32_t tmem_slot = base + L::kWords, abort_at = tmem_slot + 4;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const AttentionWork& w = p.work;

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid == 0) {
    auto init = [](uint32_t bar, int n) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(n)); };
    for (int i = 0; i < L::kKeys; ++i) {
      init(k_full + 8 * i, kE4m3 ? kHelpers : 1);
      init(k_empty + 8 * i, 1);
    }
    for (int i = 0; i < L::kValues; ++i) {
      init(v_full + 8 * i, 1);
      init(v_empty + 8 * i, 1);
      init(v_clean + 8 * i, kHelpers);
    }
    for (int i = 0; i < L::kCodes; ++i) {
      init(c_full + 8 * i, 1);
      init(c_empty + 8 * i, kHelpers);
    }
    for (int x = 0; x < 2; ++x) {
      init(q_full + 8 * x, 1);
      init(q_empty + 8 * x, 1);
      init(s_full + 8 * x, 1);
      init(p_full + 16 * x, 4);
      init(p_full + 16 * x + 8, 4);
      init(o_full + 8 * x, 1);
      init(o_free + 8 * x, 4);
    }
    init(done, 1);
    for (int i = 1; i < 32; ++i) words[i] = 0;
    mbar_init_fence();
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(tmem_slot) : "memory");
  tmem = __shfl_sync(0xffffffffu, tmem, 0);

  asm volatile("griddepcontrol.wait;" ::: "memory");
  UnitCursor c;
  int64_t share;
  bool more = find_share<Tiles>(w, blockIdx.x, gridDim.x, &c, &share);
  // every lane waits, and all go on or none does
  auto wait = [&](uint32_t bar, uint32_t parity, int where) -> bool { return __all_sync(0xffffffffu, wait_phase(bar, parity, abort_at, where)); };
  // ... for `n` counters of this CTA, a lane each
  auto wait_count = [&](int word, int n, int count, int where) -> bool {
    bool ok = true;
    if (lane < n && words[word + lane] < count) {
      const long long t0 = clock64();
      while (words[word + lane] < count) {
        if (words[1]) {
          ok = false;
          break;
        }
        if (clock64() - t0 > kSpinLimit) {
          words[1] = where;
          ok = false;
          break;
        }
      }
    }
    ok = __all_sync(0xffffffffu, ok);
    __threadfence_block();
    return ok;
  };
  bool ok = true;
  // registers a thread at the launch: 168 (128 x 104 + 256 x 200 = 384 x 168), or with more helpers 128 (256 x 64 + 256 x 192 = 512 x 128)
  if (warp >= 8) {
    if constexpr (kE4m3) asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
    if (warp == 9) {
      // ---------------- copies ----------------
      if (lane == 0) p.notes[blockIdx.x].parts = 0;         // (also where this CTA gives up)
      Slot<L::kKeys> key = {0, 0};
      Slot<L::kValues> value = {0, 0};
      [[maybe_unused]] Slot<kE4m3 ? L::kCodes : 1> code = {0, 0};
      int items[2] = {0, 0};
      const int page_size = 1 << p.cache.page_shift;
      const int per_block = PAGED ? (page_size < kBlock ? kBlock / page_size : 1) : 1;       // pages of a block
      while (ok && more) {
        const Part it = part_of(w, c);
        if (it.live) {
          for (int x = 0; x < 2; ++x) {
            if (it.last[x] == it.begin) continue;
            if (!(ok = wait(q_empty + 8 * x, (items[x] & 1) ^ 1, 31))) break;
            ++items[x];
            if (lane == 0) {
              mbar_expect_tx(q_full + 8 * x, (D / 64) * w.tile_tokens * w.group * 128);
              for (int i = 0; i < D / 64; ++i)
                tma_load_3d(&q_map, base + x * L::kTile + i * 16384, q_full + 8 * x, i * 64, c.h * w.group, c.span.q0 + (2 * c.t + x) * w.tile_tokens);
            }
            __syncwarp();
          }
          if (!ok) break;
          int64_t page = 0;
          auto look_up = [&](int u) {                    // lane i: page i of block u
            if constexpr (PAGED) {
              const int pos = u * kBlock + lane * page_size;
              page = 0;
              if (lane < per_block && u < it.load_end && pos < c.span.len) page = page_of(p.cache, c.s, pos, w.status);
              if (page < 0) page = 0;
            }
          };
          look_up(it.begin);
          for (int u = it.begin; ok && u < it.load_end; ++u) {
            int there = 1;                                // pages of the block that the sequence has
            if constexpr (PAGED) {
              const int pages = (c.span.len - u * kBlock + page_size - 1) >> p.cache.page_shift;
              there = pages < per_block ? pages : per_block;
            }
            const int64_t here = page;
            look_up(u + 1);
#pragma unroll
            for (int which = 0; which < 2; ++which) {
              if constexpr (kE4m3) {
                if (!(ok = wait(c_empty + 8 * code.slot, code.phase ^ 1u, 32))) break;
                const uint32_t dst = base + L::kCodeRing + code.slot * (kBlock * D), exps = base + L::kExps + code.slot * kBlock, bar = c_full + 8 * code.slot;
                const int rows = page_size < kBlock ? page_size : kBlock;
                if (lane == 0) mbar_expect_tx(bar, there * rows * (D + 1));
                __syncwarp();
                if (lane < there) {
                  const int64_t row = ((here * w.kv_heads + c.h) << p.cache.page_shift) + ((u * kBlock) & (page_size - 1));
                  tma_load_2d(which ? &v_map : &k_map, dst + lane * rows * D, bar, 0, static_cast<int>(row));
                  bulk_load(exps + lane * rows, (which ? p.cache.v_exp : p.cache.k_exp) + row, rows, bar);
                }
                __syncwarp();
                code.next();
                continue;
              }
              const uint32_t slot = which ? value.slot : key.slot;
              if (!(ok = wait((which ? v_empty : k_empty) + 8 * slot, (which ? value.phase : key.phase) ^ 1u, 32))) break;
              const uint32_t dst = (which ? value_ring : key_ring) + slot * L::kTile, bar = (which ? v_full : k_full) + 8 * slot;
              if constexpr (PAGED) {
                const int rows = page_size < kBlock ? page_size : kBlock;
                if (lane == 0) mbar_expect_tx(bar, there * rows * D * 2);
                __syncwarp();
                if (lane < there) {
                  const int row = static_cast<int>(((here * w.kv_heads + c.h) << p.cache.page_shift) + ((u * kBlock) & (page_size - 1)));
                  for (int i = 0; i < D / 64; ++i) tma_load_2d(which ? &v_map : &k_map, dst + i * 16384 + lane * rows * 128, bar, i * 64, row);
                }
              } else if (lane == 0) {
                mbar_expect_tx(bar, kBlock * D * 2);
                for (int i = 0; i < D / 64; ++i) tma_load_3d(which ? &v_map : &k_map, dst + i * 16384, bar, i * 64, c.h, c.span.q0 + u * kBlock);
              }
              __syncwarp();
              if (which) value.next(); else key.next();
            }
          }
        }
        if (c.end < c.units && lane == 0) p.notes[blockIdx.x] = note_of(c, it.begin, share);
        more = next_item<Tiles>(w, c);
      }
      if (!ok) {                                          // given up: what is on its way lands first
        auto drain = [&](uint32_t bars_of, int n, uint32_t slot, uint32_t phase) {
          for (int i = 0; i < n; ++i) mbar_drain(bars_of + 8 * i, i < static_cast<int>(slot) ? phase : phase ^ 1u);
        };
        if constexpr (kE4m3) {
          drain(c_full, L::kCodes, code.slot, code.phase);
        } else {
          drain(k_full, L::kKeys, key.slot, key.phase);
          drain(v_full, L::kValues, value.slot, value.phase);
        }
        for (int x = 0; x < 2; ++x)
          if (items[x]) mbar_drain(q_full + 8 * x, (items[x] - 1) & 1);
      }
    } else if (kE4m3 && warp >= 10) {
      // ---------------- helpers: codes into bf16, in the products' layout ----------------
      Slot<L::kKeys> key = {0, 0};
      Slot<L::kValues> value = {0, 0};
      Slot<kE4m3 ? L::kCodes : 1> code = {0, 0};
      int live = 0;
      while (ok && more) {
        const Part it = part_of(w, c);
        if (it.live) {
          const int first_limit = w.causal ? c.span.len - c.span.n + c.t * 2 * w.tile_tokens : c.span.len - 1;
          const int seen = it.seen[0] > it.seen[1] ? it.seen[0] : it.seen[1];
          bool mine = false;                              // the first row of no numbers is this item's
          for (int u = it.begin; ok && u < it.load_end; ++u) {
#pragma unroll 1
            for (int which = 0; which < 2; ++which) {
              if (!(ok = wait(c_full + 8 * code.slot, code.phase, 33))) break;
              if (!(ok = wait((which ? v_empty : k_empty) + 8 * (which ? value.slot : key.slot), (which ? value.phase : key.phase) ^ 1u, 45))) break;
              const uint32_t from = base + L::kCodeRing + code.slot * (kBlock * D), exps = base + L::kExps + code.slot * kBlock;
              const uint32_t to = which ? value_ring + value.slot * L::kTile : key_ring + key.slot * L::kTile;
              const int pos0 = u * kBlock;
              constexpr int kPieces = D / 16;
              // rows of values that some rows see and others do not, or none
              const int some = which ? (first_limit + 1 > pos0 ? first_limit + 1 - pos0 : 0) : kBlock, none = which ? seen - pos0 : kBlock;
              auto convert = [&](int i, uint32_t byte, bool zero) {
                const int r = i / kPieces, col = i % kPieces;
                const uint4 c16 = lds128<0>(from + i * 16);
                const uint32_t codes[4] = {c16.x, c16.y, c16.z, c16.w};
                uint32_t v[8];
                row_values(codes, row_factors(byte), v);
                if (zero) {
#pragma unroll
                  for (int n = 0; n < 8; ++n) v[n] = 0;
                }
                const uint32_t line = to + (col >> 2) * 16384 + r * 128, piece = 2 * col & 7;
                asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(line + ((piece ^ (r & 7)) << 4)), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
                asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(line + (((piece + 1) ^ (r & 7)) << 4)), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
              };
              const int mine0 = (warp - 10) * 32 + lane;
              if (some >= kBlock && none >= kBlock) {
#pragma unroll 3
                for (int i = mine0; i < kBlock * kPieces; i += kHelpers * 32) convert(i, lds8(exps + i / kPieces), false);
              } else {
                for (int i = mine0; i < kBlock * kPieces; i += kHelpers * 32) {
                  const int r = i / kPieces;
                  const uint32_t byte = lds8(exps + r);
                  const bool odd = r >= some && r < none && byte == 255;
                  if (__any_sync(0xffffffffu, odd) && !mine) {
                    if (!(ok = wait_count(kWritten, 8, live, 34))) break;
                    if (lane == 0) words[kNanPlace + warp - 10] = 0x7fffffff;
                    if (lane == 0) words[kTags + warp - 10] = live + 1;
                    __syncwarp();
                    mine = true;
                  }
                  if (odd) atomicMin(const_cast<int*>(&words[kNanPlace + warp - 10]), pos0 + r);
                  convert(i, byte, odd || r >= none);
                }
              }
              fence_proxy_async();
              __syncwarp();
              if (lane == 0) {
                mbar_arrive(c_empty + 8 * code.slot);
                mbar_arrive(which ? v_clean + 8 * value.slot : k_full + 8 * key.slot);
              }
              code.next();
              if (which) value.next(); else key.next();
            }
          }
          __threadfence_block();
          __syncwarp();
          if (lane == 0) words[kHelped + warp - 10] = live + 1;
          ++live;
        }
        more = next_item<Tiles>(w, c);
      }
    } else if (warp >= 10) {
      // ---------------- helpers: blocks of v that some row does not see all of ----------------
      Slot<L::kValues> at = {0, 0};
      int live = 0;
      while (ok && more) {
        const Part it = part_of(w, c);
        if (it.live) {
          const int first_limit = w.causal ? c.span.len - c.span.n + c.t * 2 * w.tile_tokens : c.span.len - 1;
          const int place0 = place_of(first_limit);
          uint16_t* const set = special + (warp - 10) * 3 * D;
          bool mine = false;                              // the set is this item's
          for (int u = it.begin; ok && u < it.load_end; ++u) {
            const uint32_t slot = at.slot;
            if (!(ok = wait(v_full + 8 * slot, at.phase, 33))) break;
            const int pos0 = u * kBlock;
            if (pos0 + kBlock - 1 > first_limit) {
              constexpr int kPieces = D / 8;
              const int some = first_limit + 1 > pos0 ? first_limit + 1 - pos0 : 0;                                   // rows up to here: seen by all
              const int seen = it.seen[0] > it.seen[1] ? it.seen[0] : it.seen[1];
              const int none = seen - pos0 < kBlock ? seen - pos0 : kBlock;                                           // from here on: by none
              auto place = [&](int i) {
                const int r = i / kPieces, col = i % kPieces;
                return value_ring + slot * L::kTile + (col >> 3) * 16384 + r * 128 + (((col & 7) ^ (r & 7)) << 4);
              };
              const int mine0 = (warp - 10) * 32 + lane;
              for (int i = none * kPieces + mine0; i < kBlock * kPieces; i += kHelpers * 32)
                asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(place(i)), "r"(0) : "memory");
              constexpr int kBatch = 4;
              for (int i0 = some * kPieces; i0 < none * kPieces; i0 += kBatch * kHelpers * 32) {
                uint4 v[kBatch];
                unsigned odd = 0;
#pragma unroll
                for (int b = 0; b < kBatch; ++b) {
                  const int i = i0 + b * kHelpers * 32 + mine0;
                  v[b] = i < none * kPieces ? lds128<0>(place(i)) : make_uint4(0, 0, 0, 0);
                }
#pragma unroll
                for (int b = 0; b < kBatch; ++b)
                  if (odd_pair<T>(v[b].x) || odd_pair<T>(v[b].y) || odd_pair<T>(v[b].z) || odd_pair<T>(v[b].w)) odd |= 1u << b;
                if (!__any_sync(0xffffffffu, odd)) continue;
                if (!mine) {                            // the items before this one are written: what the set held goes
                  if (!(ok = wait_count(kWritten, 8, live, 34))) break;
                  for (int n = lane; n < 3 * D; n += 32) set[n] = 0xffff;
                  if (lane == 0) words[kTags + warp - 10] = live + 1;
                  __syncwarp();
                  mine = true;
                }
                for (int l = 0; l < 32; ++l) {          // a lane at a time: two may have the same column
                  if (l == lane && odd) {
#pragma unroll
                    for (int b = 0; b < kBatch; ++b) {
                      if (!(odd >> b & 1)) continue;
                      const int i = i0 + b * kHelpers * 32 + mine0, r = i / kPieces, col = i % kPieces;
                      uint32_t word[4] = {v[b].x, v[b].y, v[b].z, v[b].w};
#pragma unroll
                      for (int e = 0; e < 8; ++e) {
                        const float2 pair = unpack2<T>(word[e >> 1]);
                        const float x = e & 1 ? pair.y : pair.x;
                        if (!(fabsf(x) <= 3.402823466e38f)) {
                          uint16_t* const first = set + (x > 0.0f ? 0 : x < 0.0f ? D : 2 * D) + col * 8 + e;
                          if (pos0 + r - place0 < *first) *first = static_cast<uint16_t>(pos0 + r - place0);
                          word[e >> 1] &= e & 1 ? 0x0000ffffu : 0xffff0000u;
                        }
                      }
                      asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(place(i)), "r"(word[0]), "r"(word[1]), "r"(word[2]), "r"(word[3]) : "memory");
                    }
                  }
                  __syncwarp();
                }
              }
              fence_proxy_async();
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(v_clean + 8 * slot);
            at.next();
          }
          __threadfence_block();
          __syncwarp();
          if (lane == 0) words[kHelped + warp - 10] = live + 1;
          ++live;
        }
        more = next_item<Tiles>(w, c);
      }
    } else {
      // ---------------- the MMAs' issuer ----------------
      constexpr uint32_t kFmt = kBf16 ? 1 : 0;
      const uint32_t id_scores = instr_desc(kFmt, 128) | (static_cast<uint32_t>(kBlock / 8) << 17);
      const uint32_t id_values = instr_desc(kFmt, 128) | (static_cast<uint32_t>(D / 8) << 17) | (1u << 16);       // B is MN-major
      Slot<L::kKeys> key = {0, 0};
      Slot<L::kValues> value = {0, 0};
      uint32_t items[2] = {0, 0}, p_ph[2] = {0, 0};
      auto scores = [&](int x, uint32_t key_slot, bool last) {
        mma_scores<D>(tmem + x * 128, desc_low(base + x * L::kTile), desc_low(key_ring + key_slot * L::kTile), kDescHigh, id_scores);
        tc_commit<false>(s_full + 8 * x, 0);
        if (last) tc_commit<false>(q_empty + 8 * x, 0);    // the next item's queries may come
      };
      while (ok && more) {
        const Part it = part_of(w, c);
        if (it.live) {
          if (!(ok = wait(k_full + 8 * key.slot, key.phase, 36))) break;
          for (int x = 0; x < 2; ++x) {
            if (it.last[x] == it.begin) continue;
            if (!(ok = wait(q_full + 8 * x, items[x] & 1, 35))) break;
            tc_fence_after();
            scores(x, key.slot, it.begin + 1 == it.last[x]);
          }
          if (!ok) break;
          tc_commit<false>(k_empty + 8 * key.slot, 0);
          key.next();
          for (int u = it.begin; ok && u < it.load_end; ++u) {
            const bool next = u + 1 < it.load_end;
            if (!(ok = wait(v_clean + 8 * value.slot, value.phase, 37))) break;
            if (next && !(ok = wait(k_full + 8 * key.slot, key.phase, 38))) break;
            for (int x = 0; x < 2; ++x) {
              if (u >= it.last[x]) continue;
              if (u == it.begin) {                        // the rows' last item has been read out of O
                if (!(ok = wait(o_free + 8 * x, (items[x] & 1) ^ 1, 39))) break;
              }
              for (int part = 0; part < 2; ++part) {      // P comes in two parts of 64 positions
                if (!(ok = wait(p_full + 16 * x + 8 * part, p_ph[x], 40))) break;
                tc_fence_after();
                mma_values(tmem + 256 + x * D, tmem + x * 128 + part * 32, desc_low_mn(value_ring + value.slot * L::kTile + part * 8192), kDescHigh, id_values,
                           part | (u > it.begin));
              }
              if (!ok) break;
              p_ph[x] ^= 1u;
              if (u + 1 < it.last[x]) {
                scores(x, key.slot, u + 2 == it.last[x]);
              } else {
                tc_commit<false>(o_full + 8 * x, 0);
                ++items[x];
              }
            }
            if (!ok) break;
            tc_commit<false>(v_empty + 8 * value.slot, 0);
            value.next();
            if (next) {
              tc_commit<false>(k_empty + 8 * key.slot, 0);
              key.next();
            }
          }
        }
        more = next_item<Tiles>(w, c);
      }
      // The arrivals of all MMAs so far, given up or not, reach their barriers before the CTA leaves.
      tc_commit<false>(done, 0);
      mbar_drain(done, 0);
    }
  } else {
    if constexpr (kE4m3) asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    else asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    // ---------------- rows ----------------
    const int x = warp >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + x * 128 + lanes, o_at = tmem + 256 + x * D + lanes;
    const int tok_in = r / w.group, g = r - tok_in * w.group;
    const uint64_t scale = pack_f32(p.scale_log2, p.scale_log2);
    uint32_t s_ph = 0, o_ph = 0;
    int live = 0;
    while (ok && more) {
      const Part it = part_of(w, c);
      const int tok0 = (2 * c.t + x) * w.tile_tokens, tok = tok0 + tok_in;
      const bool mine = tok_in < w.tile_tokens && tok < c.span.n;
      const int limit = w.causal ? c.span.len - c.span.n + tok : c.span.len - 1;
      const int first_limit = w.causal ? c.span.len - c.span.n + tok0 : c.span.len - 1;
      const int first_item_limit = w.causal ? c.span.len - c.span.n + 2 * c.t * w.tile_tokens : c.span.len - 1;
      float top = -INFINITY, sum = 0.0f;                // running maximum (times the scale, base 2) that O stands for
      for (int u = it.begin; u < it.last[x]; ++u) {
        if (!(ok = wait(s_full + 8 * x, s_ph, 41))) break;
        s_ph ^= 1u;
        tc_fence_after();
        uint32_t s[4][32];
#pragma unroll
        for (int i = 0; i < 4; ++i) tmem_ld(s_at + i * 32, s[i]);
        tmem_wait_ld();
        if (u * kBlock + kBlock - 1 > first_limit) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int seen = limit - u * kBlock - i * 32;             // columns 0 .. seen of these 32 are seen: a bit each
            const uint32_t mask = seen < 0 ? 0u : seen >= 31 ? ~0u : (2u << seen) - 1u;
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (!(mask & 1u << j)) s[i][j] = 0xff800000u;
          }
        }
        float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 32; j += 2) m[j >> 1 & 3] = max3(m[j >> 1 & 3], __uint_as_float(s[i][j]), __uint_as_float(s[i][j + 1]));
        const float now = fmaxf(max3(m[0], m[1], m[2]), m[3]) * p.scale_log2;
        if (u == it.begin) {
          top = now;
        } else if (__any_sync(0xffffffffu, now > top + 8.0f)) {
          float shrink = 1.0f;
          if (now > top + 8.0f) {
            shrink = ex2(top - now);
            top = now;
            sum *= shrink;
          }
#pragma unroll 1
          for (int i = 0; i < D / 32; ++i) {
            uint32_t o[32];
            tmem_ld(o_at + i * 32, o);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * shrink);
            tmem_st(o_at + i * 32, o);
          }
        }
        const float off = top == -INFINITY ? 0.0f : -top;
        const uint64_t off2 = pack_f32(off, off);
        uint64_t sums[2] = {0, 0};
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          uint32_t out[32];
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const uint32_t(&v)[32] = s[2 * part + i];
              const float2 e = unpack_f32(fma2(pack_f32(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1])), scale, off2));
              const float a = ex2(e.x), b = ex2(e.y);
              sums[j & 1] = add2(sums[j & 1], pack_f32(a, b));
              out[i * 16 + j] = pack2<T>(a, b);
            }
          tmem_st(s_at + part * 32, out);
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(p_full + 16 * x + 8 * part);
        }
        const float2 both = unpack_f32(add2(sums[0], sums[1]));
        sum += both.x + both.y;
      }
      if (!ok) break;
      // ---- the item, or this CTA's part of it, ends (the next one is worked out while its last product runs) ----
      UnitCursor after = c;
      const bool again = next_item<Tiles>(w, after);
      const bool has = it.last[x] > it.begin;
      bool odd[kHelpers] = {};
      if (has) {
        if (!(ok = wait(o_full + 8 * x, o_ph, 42))) break;
        o_ph ^= 1u;
        tc_fence_after();
        if (!(ok = wait_count(kHelped, kHelpers, live + 1, 43))) break;
        for (int n = 0; n < kHelpers; ++n) odd[n] = words[kTags + n] == live + 1;
      }
      const bool sector = (reinterpret_cast<uintptr_t>(p.out) & 31) == 0;
      const bool whole = it.begin == 0 && c.end == c.units;
      const float inv = sum == 0.0f ? (limit < 0 ? 0.0f : NAN) : 1.0f / sum;
      uint8_t* const out = p.out + ((static_cast<int64_t>(c.span.q0) + tok) * w.heads + c.h * w.group + g) * D * 2;
      float4* const part = reinterpret_cast<float4*>(p.partial + (2 * static_cast<int64_t>(blockIdx.x) + (it.begin == 0 ? 1 : 0)) * partial_floats<256, D>());
      const int row = x * 128 + r;
#pragma unroll 1
      for (int i = 0; i < D / 64; ++i) {
        uint32_t o[2][32];
        if (has) {
          tmem_ld(o_at + i * 64, o[0]);
          tmem_ld(o_at + i * 64 + 32, o[1]);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int j = 0; j < 64; ++j) o[j >> 5][j & 31] = 0;
        }
#pragma unroll
        for (int n = 0; n < kHelpers; ++n)
          if (kE4m3 && odd[n]) {
            if (words[kNanPlace + n] <= limit) {
#pragma unroll
              for (int j = 0; j < 64; ++j) o[j >> 5][j & 31] = 0x7fc00000u;
            }
          } else if (!kE4m3 && odd[n]) {
            const uint16_t* const set = special + n * 3 * D + i * 64;
            const int seen = limit - place_of(first_item_limit);
#pragma unroll
            for (int j = 0; j < 64; ++j) {
              float v = __uint_as_float(o[j >> 5][j & 31]);
              if (set[j] <= seen) v += INFINITY;
              if (set[D + j] <= seen) v -= INFINITY;
              if (set[2 * D + j] <= seen) v = NAN;
              o[j >> 5][j & 31] = __float_as_uint(v);
            }
          }
        if (!mine) continue;
        if (whole) {
#pragma unroll
          for (int j = 0; j < 64; j += 16) {
            uint32_t v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
              v[e] = pack2<T>(__uint_as_float(o[j >> 5][(j & 31) + 2 * e]) * inv, __uint_as_float(o[j >> 5][(j & 31) + 2 * e + 1]) * inv);
            store32(out + (i * 64 + j) * 2, v, sector);
          }
        } else {
          // four elements of 256 rows side by side: neighbouring threads write neighbouring 16 bytes
#pragma unroll
          for (int j = 0; j < 64; j += 4)
            part[((i * 64 + j) / 4) * 256 + row] = make_float4(__uint_as_float(o[j >> 5][j & 31]), __uint_as_float(o[j >> 5][(j & 31) + 1]),
                                                               __uint_as_float(o[j >> 5][(j & 31) + 2]), __uint_as_float(o[j >> 5][(j & 31) + 3]));
        }
      }
      if (!whole && mine) {
        reinterpret_cast<float*>(part)[256 * D + row] = top;
        reinterpret_cast<float*>(part)[256 * D + 256 + row] = sum;
      }
      if (has) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(o_free + 8 * x);
      }
      if (it.live) {
        __threadfence_block();
        __syncwarp();
        if (lane == 0) words[kWritten + warp] = live + 1;
        ++live;
      }
      more = again;
      c = after;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
  if (tid == 0 && words[1]) atomicCAS(w.status, 0, words[1]);
}

// Items whose units fell to several CTAs: block (b, y) looks at the end of CTA b's share, and joins 16 columns of the item there if it is cut there
// first. A thread has a row.
constexpr int kJoinColumns = 16;
template <typename T, int D>
__global__ void __launch_bounds__(256) attend_tc_join_kernel(const JoinParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const AttentionWork& w = p.work;
  const JoinNote c = p.notes[blockIdx.x];
  if (c.parts == 0) return;
  const int row = threadIdx.x, x = row >> 7, r = row & 127;
  const int tok_in = r / w.group, g = r - tok_in * w.group, tok = (2 * c.t + x) * w.tile_tokens + tok_in;
  if (tok_in >= w.tile_tokens || tok >= c.n) return;
  auto slot = [&](int i) { return p.partial + (2 * (static_cast<int64_t>(blockIdx.x) + i) + (i == 0 ? 1 : 0)) * partial_floats<256, D>(); };
  float top = -INFINITY;
  for (int i = 0; i < c.parts; ++i) top = fmaxf(top, slot(i)[256 * D + row]);
  const float base = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f, v[kJoinColumns] = {};
#pragma unroll 2
  for (int i = 0; i < c.parts; ++i) {
    const float* s = slot(i);
    const float f = ex2(s[256 * D + row] - base);
    sum = fmaf(f, s[256 * D + 256 + row], sum);
#pragma unroll
    for (int j = 0; j < kJoinColumns / 4; ++j) {
      const float4 y = reinterpret_cast<const float4*>(s)[(blockIdx.y * (kJoinColumns / 4) + j) * 256 + row];
      v[4 * j] = fmaf(f, y.x, v[4 * j]);
      v[4 * j + 1] = fmaf(f, y.y, v[4 * j + 1]);
      v[4 * j + 2] = fmaf(f, y.z, v[4 * j + 2]);
      v[4 * j + 3] = fmaf(f, y.w, v[4 * j + 3]);
    }
  }
  const int limit = w.causal ? c.len - c.n + tok : c.len - 1;
  const float inv = sum == 0.0f ? (limit < 0 ? 0.0f : NAN) : 1.0f / sum;
  uint8_t* const out = p.out + (((static_cast<int64_t>(c.q0) + tok) * w.heads + c.h * w.group + g) * D + blockIdx.y * kJoinColumns) * 2;
#pragma unroll
  for (int j = 0; j < kJoinColumns; j += 8)
    *reinterpret_cast<uint4*>(out + j * 2) = make_uint4(pack2<T>(v[j] * inv, v[j + 1] * inv), pack2<T>(v[j + 2] * inv, v[j + 3] * inv),
                                                        pack2<T>(v[j + 4] * inv, v[j + 5] * inv), pack2<T>(v[j + 6] * inv, v[j + 7] * inv));
}

template <typename T, int D, int SOURCE>
int launch_one(const RowsParams& p, const CUtensorMap (&maps)[3], int ctas, cudaStream_t stream) {
  static bool done[kMaxDevices] = {};
  const int dev = current_device();
  if (dev < 0) return QMM_ERR_DEVICE;
  auto kernel = attend_tc_kernel<T, D, SOURCE>;
  using L = TcLayout<D, SOURCE>;
  if (!done[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes);
    if (e != cudaSuccess) return fail(QMM_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    done[dev] = true;
  }
  launch_early(kernel, ctas, L::kThreads, L::kBytes, stream, maps[0], maps[1], maps[2], p);
  count_launch();
  if (int rc = check_launch("attend_tc_kernel")) return rc;
  // items too short to be cut, however sequences are: nothing to join, and the launch that would find that out (2 us) is left out
  const int64_t longest = SOURCE == kRowsSource ? p.work.tokens : p.work.longest;
  if (ctas < 2 || longest <= (Tiles::kWhole - 1) * kBlock) return QMM_OK;
  JoinParams j = {p.work, p.out, p.notes, p.partial};
  launch_early(attend_tc_join_kernel<T, D>, dim3(ctas - 1, D / kJoinColumns), 256, 0, stream, j);
  count_launch();
  return check_launch("attend_tc_join_kernel");
}

template <typename T, int D>
int launch_of(const RowsParams& p, const CUtensorMap (&maps)[3], int source, int ctas, cudaStream_t stream) {
  if (source == kRowsSource) return launch_one<T, D, kRowsSource>(p, maps, ctas, stream);
  if (source == kPages16) return launch_one<T, D, kPages16>(p, maps, ctas, stream);
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return launch_one<T, D, kPages8>(p, maps, ctas, stream);
  return fail(QMM_ERR_UNSUPPORTED, "attention: an e4m3 cache is attended with bf16 queries");
}

}  // namespace

int attend_tc_ctas() { return device_sm_count(); }

int64_t attend_tc_workspace(int head_dim, int ctas) {
  return ctas * (sizeof(JoinNote) + 2ll * (head_dim == 64 ? partial_floats<256, 64>() : partial_floats<256, 128>()) * 4);
}

int launch_attend_tc(const RowsParams& given, int elem, int head_dim, int source, int ctas, cudaStream_t stream) {
  RowsParams p = given;
  AttentionWork& w = p.work;
  w.tile_tokens = 128 / w.group;
  CUtensorMap maps[3];
  if (int rc = tensor_map_3d(&maps[0], elem, p.q, head_dim, w.heads, w.tokens, p.q_head * 2, p.q_row * 2, 64, w.group, w.tile_tokens)) return rc;
  if (source != kRowsSource) {
    const int page = 1 << p.cache.page_shift, rows = page < kBlock ? page : kBlock;
    const uint64_t all = static_cast<uint64_t>(p.cache.pages) * w.kv_heads << p.cache.page_shift;
    const bool codes = source == kPages8;              // as they lie; values in the products' swizzle, 64 elements a row
    for (int i = 0; i < 2; ++i)
      if (int rc = tensor_map_2d(&maps[1 + i], codes ? QMM_U8 : elem, i ? p.cache.v : p.cache.k, head_dim, all, head_dim * (codes ? 1 : 2), codes ? head_dim : 64, rows, codes ? 0 : 1))
        return rc;
  } else {
    if (int rc = tensor_map_3d(&maps[1], elem, p.k, head_dim, w.kv_heads, w.tokens, p.k_head * 2, p.k_row * 2, 64, 1, kBlock)) return rc;
    if (int rc = tensor_map_3d(&maps[2], elem, p.v, head_dim, w.kv_heads, w.tokens, p.v_head * 2, p.v_row * 2, 64, 1, kBlock)) return rc;
  }
  if (elem == QMM_BF16) return head_dim == 64 ? launch_of<__nv_bfloat16, 64>(p, maps, source, ctas, stream) : launch_of<__nv_bfloat16, 128>(p, maps, source, ctas, stream);
  return head_dim == 64 ? launch_of<__half, 64>(p, maps, source, ctas, stream) : launch_of<__half, 128>(p, maps, source, ctas, stream);
}

}  // namespace qmm
