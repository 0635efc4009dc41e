// Writing new tokens into a paged cache and reading a cache's rows back.
//
// Both are streams of rows, bound by memory where there are many and by a chain of dependent loads (starts, length, table, row) where there are few, so a warp works by
// itself, without a barrier: it looks up its token or positions (32 starts at a time), and has the loads of several rows on their way at once.
//
// append: a head's row of D elements is D / 8 lanes of 16 bytes, so that norm, largest magnitude and rotation stay within a group of lanes (shuffles). A
// token's angles are the same for all of its heads: two lanes' worth each take position * frequency in float64 (a position of 10^5 times a float32 frequency
// is off by 0.006 radians), reduce it to a fraction of a turn there, and hand sine and cosine round through shared memory. A token's heads go to one
// warp, or to up to eight where there are few tokens.
#include <type_traits>

#include "paged_cache.cuh"

namespace qmm {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;

// One warp: sequence of packed row `row`: the last s with starts[s] <= row, or -1 for a row of none.
__device__ __forceinline__ int warp_sequence_of(const int32_t* __restrict__ starts, int seqs, int row, int* end) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = seqs + 1;                            // among starts[lo .. lo + n), of which the first is <= row
  for (;;) {
    const int step = (n + 31) / 32, at = lane * step;
    const int v = at < n ? __ldg(starts + lo + at) : 0x7fffffff;
    const unsigned below = __ballot_sync(0xffffffffu, at < n && v <= row);
    if (!below) return -1;
    const int k = 31 - __clz(below);                   // (starts that fall would still leave it within them)
    if (step == 1) {
      lo += k;
      const int next = __shfl_sync(0xffffffffu, v, k + 1 < 32 ? k + 1 : 31);
      *end = k + 1 < n && k + 1 < 32 ? next : lo < seqs ? __ldg(starts + lo + 1) : 0;
      return lo < seqs && row < *end ? lo : -1;
    }
    lo += k * step;
    n = n - k * step < step ? n - k * step : step;
  }
}

struct AppendParams {
  CacheView c;
  const uint8_t* qkv;
  uint8_t* q_out;
  const double* freqs;
  const uint8_t* q_norm;
  const uint8_t* k_norm;
  const int32_t* kv_lens;
  const int32_t* cu_q;
  int* status;
  int64_t row_stride;          // elements
  int32_t seqs, heads, rotary_dim, interleaved;
  int32_t tokens, token_warps;  // warps of a token
  float eps;
};

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& w, float (&f)[8]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = unpack2<T>(u[i]);
    f[2 * i] = v.x;
    f[2 * i + 1] = v.y;
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
}

// Pairs of floats in one instruction.
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  return v;
}
__device__ __forceinline__ float2 floats_of(uint64_t v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
template <typename T>
__device__ __forceinline__ void pairs_of(const uint4& w, uint64_t (&f)[4]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = unpack2<T>(u[i]);
    f[i] = pair_of(v.x, v.y);
  }
}
__device__ __forceinline__ float max_nan(float a, float b) {            // NaN if one is
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// T: type of the projection's rows; E4M3: the cache holds codes, else values of T. Queries, keys and values are a pass each: what an element and its pair's other
// one are multiplied with (norm's weight times cosine, and sine) stays in registers for all heads, and the root mean square comes last.
// Bound by instructions at three CTAs an SM (some 6700 tokens of 32 + 2 x 8 heads of 128 with norms into e4m3 49.7 us, 4.1 TB/s; 8192 into bf16 44, 4.5 TB/s). Before heads were
// asked for a batch ahead, with four rows a batch: 52.7; four CTAs 53.6, with two rows 58.1; two CTAs with six 60.4; two warps a token 72.
template <typename T, int D, bool E4M3>
__global__ void __launch_bounds__(kThreads, 3) append_kernel(const AppendParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int kLanes = D / 8, kRows = 32 / kLanes;   // lanes of a head's row; rows of a warp
  constexpr int kBatch = 4;                            // rows whose loads are on their way at once, kRows heads each
  __shared__ float2 turns[kWarps][D / 2];              // (sine, cosine) of a token's angles
  const int warp = threadIdx.x >> 5, lane32 = threadIdx.x & 31, lane = lane32 % kLanes, slot = lane32 / kLanes;
  const int id = blockIdx.x * kWarps + warp, token = id / p.token_warps, part = id - token * p.token_warps;
  if (token >= p.tokens) return;
  const int stride = p.token_warps * kRows;
  const uint4* const rows = reinterpret_cast<const uint4*>(p.qkv) + token * p.row_stride / 8;
  // Pieces of this warp's next heads, asked for a batch ahead, also of the next pass; the first ones before it is known where the token stands.
  uint4 x[kBatch];
  const int head_at = part * kRows + slot;
  auto ask = [&](int begin, int count, int head) {
    return head < count ? __ldg(rows + static_cast<int64_t>(begin + head) * kLanes + lane) : make_uint4(0, 0, 0, 0);
  };
#pragma unroll
  for (int b = 0; b < kBatch; ++b) x[b] = ask(0, p.heads, head_at + b * stride);
  int seq = token, end = 0, pos;
  if (p.cu_q) {
    seq = warp_sequence_of(p.cu_q, p.seqs, token, &end);
    if (seq < 0) return;                               // a row behind the last sequence
    pos = __ldg(p.kv_lens + seq) - (end - token);
  } else {
    pos = __ldg(p.kv_lens + seq) - 1;
  }
  const int64_t page = page_of(p.c, seq, pos, p.status);
  const int row = pos & ((1 << p.c.page_shift) - 1);
  for (int i = lane32; i < p.rotary_dim / 2; i += 32) {
    // a fraction of a turn, off by some 2^-52 of the number of turns: 2^-35 at position 2^20, 2^-25 at 2^30, the last that a table allows, where a radian is a
    // position; sine and cosine rounded once (from a fraction in 32 bits a third more of an e4m3 cache's codes of keys
    // were a step off: 15 in five million, now 10)
    const double turned = static_cast<double>(pos) * (__ldg(p.freqs + i) * 0.15915494309189533576888376337251);
    double s, c;
    sincospi(2.0 * (turned - rint(turned)), &s, &c);
    turns[warp][i] = make_float2(static_cast<float>(s), static_cast<float>(c));
  }
  __syncwarp();
  const int pairs = p.rotary_dim / 16;                 // lanes of the first elements of split pairs
  const bool first = lane < pairs, turned = lane < 2 * pairs;
  const int partner = p.interleaved || !turned ? lane : first ? lane + pairs : lane - pairs;

  auto pass = [&](auto kind_of, int begin, int count, const uint8_t* weight, int next_begin, int next_count) {
    constexpr int kKind = decltype(kind_of)::value;      // 0 queries, 1 keys, 2 values
    const bool turns_on = kKind != 2 && pairs > 0, scaled = kKind != 2 && weight != nullptr;
    uint64_t own[4], across[4];                           // factors of an element and of its pair's other one
    if (kKind != 2) {
#pragma unroll
      for (int i = 0; i < 4; ++i) own[i] = across[i] = pair_of(1.0f, 1.0f);
      if (scaled) {
        pairs_of<T>(__ldg(reinterpret_cast<const uint4*>(weight) + lane), own);
        pairs_of<T>(__ldg(reinterpret_cast<const uint4*>(weight) + partner), across);
      }
      if (turned) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (p.interleaved) {
            const float2 t = turns[warp][lane * 4 + i], v = floats_of(across[i]);
            across[i] = pair_of(-t.x * v.y, t.x * v.x);
            own[i] = mul2(own[i], pair_of(t.y, t.y));
          } else {
            const float2 a = turns[warp][(first ? lane : partner) * 8 + 2 * i], b = turns[warp][(first ? lane : partner) * 8 + 2 * i + 1];
            across[i] = mul2(across[i], first ? pair_of(-a.x, -b.x) : pair_of(a.x, b.x));
            own[i] = mul2(own[i], pair_of(a.y, b.y));
          }
        }
      }
    }
    for (int head0 = head_at;; head0 += kBatch * stride) {
      const bool more = __any_sync(0xffffffffu, head0 + kBatch * stride < count);
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int head = head0 + b * stride;
        const uint4 mine = x[b];
        x[b] = more ? ask(begin, count, head + kBatch * stride) : ask(next_begin, next_count, head_at + b * stride);
        if (!__any_sync(0xffffffffu, head < count)) continue;
        uint4 out = mine;
        uint64_t f[4];
        if (kKind != 2 || E4M3) {
          pairs_of<T>(mine, f);
          uint64_t inv2 = pair_of(1.0f, 1.0f);
          if (scaled) {
            uint64_t ss2 = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) ss2 = fma2(f[i], f[i], ss2);
            const float2 two = floats_of(ss2);
            float ss = two.x + two.y;
#pragma unroll
            for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            const float inv = rsqrtf(ss / static_cast<float>(D) + p.eps);
            inv2 = pair_of(inv, inv);
          }
          if (turns_on) {
            uint64_t g[4];                               // the pairs' other elements
            if (p.interleaved) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float2 v = floats_of(f[i]);
                g[i] = pair_of(v.y, v.x);
              }
            } else {
              const uint4 other = make_uint4(__shfl_sync(0xffffffffu, mine.x, partner, kLanes), __shfl_sync(0xffffffffu, mine.y, partner, kLanes),
                                             __shfl_sync(0xffffffffu, mine.z, partner, kLanes), __shfl_sync(0xffffffffu, mine.w, partner, kLanes));
              pairs_of<T>(other, g);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint64_t y = mul2(f[i], own[i]);
              f[i] = turned ? fma2(g[i], across[i], y) : y;            // (elements that are not turned: infinities and NaN beside them or not)
            }
          } else if (scaled) {
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = mul2(f[i], own[i]);
          }
          if (scaled) {
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = mul2(f[i], inv2);
          }
          if (!(E4M3 && kKind != 0)) {
            float2 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = floats_of(f[i]);
            out = make_uint4(pack2<T>(v[0].x, v[0].y), pack2<T>(v[1].x, v[1].y), pack2<T>(v[2].x, v[2].y), pack2<T>(v[3].x, v[3].y));
          }
        }
        if (kKind == 0) {
          if (head < count) reinterpret_cast<uint4*>(p.q_out)[(static_cast<int64_t>(token) * p.heads + head) * kLanes + lane] = out;
          continue;
        }
        const int64_t at = ((page * p.c.kv_heads + head) << p.c.page_shift) + row;
        if constexpr (E4M3) {
          float big = 0.0f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 v = floats_of(f[i]);
            big = max_nan(big, max_nan(fabsf(v.x), fabsf(v.y)));
          }
#pragma unroll
          for (int o = kLanes / 2; o > 0; o >>= 1) big = max_nan(big, __shfl_xor_sync(0xffffffffu, big, o));
          const bool fine = big <= 3.402823466e38f;
          const int e = fine ? row_exponent(big) : 0;
          const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);      // 2^-e: a normal number, and the product is exact
          uint32_t u[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 v = floats_of(mul2(f[i], pair_of(down, down)));
            u[i] = fine ? e4m3_pair(v.x, v.y) : 0;
          }
          if (head < count && page >= 0) {
            reinterpret_cast<uint2*>(kKind == 2 ? p.c.v : p.c.k)[at * kLanes + lane] = make_uint2(u[0] | u[1] << 16, u[2] | u[3] << 16);
            if (lane == 0) (kKind == 2 ? p.c.v_exp : p.c.k_exp)[at] = static_cast<uint8_t>(fine ? e + 127 : 255);
          }
        } else if (head < count && page >= 0) {
          reinterpret_cast<uint4*>(kKind == 2 ? p.c.v : p.c.k)[at * kLanes + lane] = out;
        }
      }
      if (!more) break;
    }
  };
  pass(std::integral_constant<int, 0>{}, 0, p.heads, p.q_norm, p.heads, p.c.kv_heads);
  pass(std::integral_constant<int, 1>{}, p.heads, p.c.kv_heads, p.k_norm, p.heads + p.c.kv_heads, p.c.kv_heads);
  pass(std::integral_constant<int, 2>{}, p.heads + p.c.kv_heads, p.c.kv_heads, nullptr, 0, 0);
}

struct ReadParams {
  CacheView c;
  uint8_t* k_out;
  uint8_t* v_out;
  const int32_t* cu_kv;
  int* status;
  int32_t seqs, warp_rows;     // positions of a warp
  int64_t total;
};

// A warp takes warp_rows positions one behind the other, all heads of each; a lane's pieces are 16 bytes of the cache.
template <typename T, int D, bool E4M3>
__global__ void __launch_bounds__(kThreads) read_kernel(const ReadParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int kLanes = D / (E4M3 ? 16 : 8), kRows = 32 / kLanes;      // lanes of a head's row; heads of a warp
  constexpr int kBatch = 2;                                             // loads of k, and as many of v, on their way at once
  const int lane32 = threadIdx.x & 31, lane = lane32 % kLanes, slot = lane32 / kLanes;
  const int64_t first = (static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5)) * p.warp_rows;
  int seq = -1, start = 0, end = 0;
  for (int64_t out_row = first; out_row < first + p.warp_rows && out_row < p.total; ++out_row) {
    if (seq < 0 || out_row >= end) {
      seq = warp_sequence_of(p.cu_kv, p.seqs, static_cast<int>(out_row), &end);
      if (seq < 0) continue;                            // a row of no sequence
      start = __ldg(p.cu_kv + seq);
    }
    const int pos = static_cast<int>(out_row) - start;
    int64_t page = page_of(p.c, seq, pos, p.status);
    if (page < 0) page = 0;
    const int64_t row0 = ((page * p.c.kv_heads) << p.c.page_shift) + (pos & ((1 << p.c.page_shift) - 1));
    for (int head0 = slot; head0 < p.c.kv_heads; head0 += kBatch * kRows) {
      uint4 w[2][kBatch];
      uint32_t byte[2][kBatch];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int head = head0 + b * kRows;
        const int64_t at = row0 + (static_cast<int64_t>(head) << p.c.page_shift);
#pragma unroll
        for (int which = 0; which < 2; ++which) {
          if (head < p.c.kv_heads) {
            w[which][b] = __ldg(reinterpret_cast<const uint4*>(which ? p.c.v : p.c.k) + at * kLanes + lane);
            if constexpr (E4M3) byte[which][b] = __ldg((which ? p.c.v_exp : p.c.k_exp) + at);
          }
        }
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int head = head0 + b * kRows;
        if (head >= p.c.kv_heads) break;
        const int64_t to = (out_row * p.c.kv_heads + head) * (D / 8) + lane * (E4M3 ? 2 : 1);
#pragma unroll
        for (int which = 0; which < 2; ++which) {
          uint4* const out = reinterpret_cast<uint4*>(which ? p.v_out : p.k_out) + to;
          if constexpr (E4M3) {
            const uint32_t codes[4] = {w[which][b].x, w[which][b].y, w[which][b].z, w[which][b].w};
            uint32_t v[8];
            row_values(codes, row_factors(byte[which][b]), v);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              uint4 x = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
              if constexpr (!std::is_same<T, __nv_bfloat16>::value) {
                float e[8];
                unpack8<__nv_bfloat16>(x, e);
                x = pack8<T>(e);
              }
              out[i] = x;
            }
          } else {
            *out = w[which][b];
          }
        }
      }
    }
  }
}

template <typename Params>
int launch(const char* what, void (*kernel)(Params), int64_t blocks, cudaStream_t stream, const Params& p) {
  launch_early(kernel, static_cast<unsigned>(blocks), kThreads, 0, stream, p);
  count_launch();
  return check_launch(what);
}

}  // namespace

int launch_append(const CacheView& c, const qmm_append_args& a, int head_dim, bool e4m3, int* status, cudaStream_t stream) {
  AppendParams p = {};
  p.c = c;
  p.qkv = static_cast<const uint8_t*>(a.qkv);
  p.q_out = static_cast<uint8_t*>(a.q_out);
  p.freqs = a.freqs;
  p.q_norm = static_cast<const uint8_t*>(a.q_norm);
  p.k_norm = static_cast<const uint8_t*>(a.k_norm);
  p.kv_lens = a.kv_lens;
  p.cu_q = a.cu_q;
  p.status = status;
  p.row_stride = a.row_stride;
  p.tokens = static_cast<int32_t>(a.tokens);
  // a warp a token fills the machine from some 2000 tokens on; fewer share their heads out
  p.token_warps = 1;
  while (p.token_warps < kWarps && a.tokens * p.token_warps < 12ll * device_sm_count()) p.token_warps *= 2;
  p.seqs = static_cast<int32_t>(a.seqs);
  p.heads = a.heads;
  p.rotary_dim = a.rotary_dim;
  p.interleaved = a.interleaved;
  p.eps = a.eps;
  void (*kernel)(AppendParams) = nullptr;
  if (a.elem == QMM_BF16) {
    if (e4m3) kernel = head_dim == 64 ? append_kernel<__nv_bfloat16, 64, true> : append_kernel<__nv_bfloat16, 128, true>;
    else kernel = head_dim == 64 ? append_kernel<__nv_bfloat16, 64, false> : append_kernel<__nv_bfloat16, 128, false>;
  } else {
    if (e4m3) kernel = head_dim == 64 ? append_kernel<__half, 64, true> : append_kernel<__half, 128, true>;
    else kernel = head_dim == 64 ? append_kernel<__half, 64, false> : append_kernel<__half, 128, false>;
  }
  return launch("append_kernel", kernel, (a.tokens * p.token_warps + kWarps - 1) / kWarps, stream, p);
}

int launch_cache_read(const CacheView& c, int64_t seqs, const int32_t* cu_kv, int64_t total, int head_dim, int elem, bool e4m3, void* k_out,
                      void* v_out, int* status, cudaStream_t stream) {
  ReadParams p = {};
  p.c = c;
  p.k_out = static_cast<uint8_t*>(k_out);
  p.v_out = static_cast<uint8_t*>(v_out);
  p.cu_kv = cu_kv;
  p.status = status;
  p.seqs = static_cast<int32_t>(seqs);
  p.total = total;
  void (*kernel)(ReadParams) = nullptr;
  if (!e4m3) kernel = head_dim == 64 ? read_kernel<__nv_bfloat16, 64, false> : read_kernel<__nv_bfloat16, 128, false>;    // (16-bit rows are copied, whatever they hold)
  else if (elem == QMM_BF16) kernel = head_dim == 64 ? read_kernel<__nv_bfloat16, 64, true> : read_kernel<__nv_bfloat16, 128, true>;
  else kernel = head_dim == 64 ? read_kernel<__half, 64, true> : read_kernel<__half, 128, true>;
  // four positions a warp (one look into the starts), one where that would leave warps without any
  p.warp_rows = total >= 4ll * 48 * device_sm_count() ? 4 : 1;
  return launch("read_kernel", kernel, (total + static_cast<int64_t>(p.warp_rows) * kWarps - 1) / (static_cast<int64_t>(p.warp_rows) * kWarps), stream, p);
}

}  // namespace qmm
