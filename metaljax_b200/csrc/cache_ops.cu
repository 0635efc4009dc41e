// Writing new tokens into a paged cache and reading a cache's rows back.
//
// append: one CTA per token. A head's row of D elements is D / 8 lanes of 16 bytes, so that norm, largest magnitude and rotation
// stay within one group of lanes (shuffles), and a CTA of 256 threads works on 16 or 32 heads' rows at once. A token's angles are the same for all of its
// heads: one thread each takes position * frequency in float64 (a position of 10^5 times a float32 frequency is off by 0.006 radians), reduces it to a
// fraction of a turn there, and leaves sine and cosine in shared memory.
#include <type_traits>

#include "paged_cache.cuh"

namespace qmm {
namespace {

constexpr int kThreads = 256;

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

// T: type of the projection's rows; E4M3: the cache holds codes, else values of T.
template <typename T, int D, bool E4M3>
__global__ void __launch_bounds__(kThreads) append_kernel(const AppendParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int kLanes = D / 8;                        // of a head's row
  constexpr int kRows = kThreads / kLanes;             // heads' rows at once
  __shared__ float2 turn[D / 2];                       // (sine, cosine) of the token's angles
  __shared__ int where[2];                             // its sequence and position
  const int token = blockIdx.x, tid = threadIdx.x;
  const int lane = tid % kLanes, slot = tid / kLanes;
  const int all = p.heads + 2 * p.c.kv_heads;
  if (tid == 0) {
    const int seq = p.cu_q ? sequence_of(p.cu_q, p.seqs, token) : token;
    where[0] = seq;
    where[1] = seq < 0 ? 0 : p.kv_lens[seq] - (p.cu_q ? p.cu_q[seq + 1] - token : 1);
  }
  __syncthreads();
  const int seq = where[0], pos = where[1];
  if (seq < 0) return;                                 // a row behind the last sequence
  for (int i = tid; i < p.rotary_dim / 2; i += kThreads) {
    // a fraction of a turn, exact to 2^-30 for positions up to 2^31, before it becomes a float
    const double turns = static_cast<double>(pos) * (p.freqs[i] * 0.15915494309189533576888376337251);
    float s, c;
    sincospif(2.0f * static_cast<float>(turns - rint(turns)), &s, &c);
    turn[i] = make_float2(s, c);
  }
  __syncthreads();
  const int64_t page = page_of(p.c, seq, pos, p.status);
  const int row = pos & ((1 << p.c.page_shift) - 1);
  const int pairs = p.rotary_dim / 16;                 // lanes of the first elements of split pairs
  for (int head0 = 0; head0 < all; head0 += kRows) {
    const int head = head0 + slot;
    const bool live = head < all;
    float f[8] = {};
    if (live) unpack8<T>(__ldg(reinterpret_cast<const uint4*>(p.qkv) + (token * p.row_stride + head * D) / 8 + lane), f);
    const bool is_q = head < p.heads, is_v = head >= p.heads + p.c.kv_heads;
    const uint8_t* weight = is_v ? nullptr : is_q ? p.q_norm : p.k_norm;
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(f[i], f[i], ss);
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (weight) {
      float w[8];
      unpack8<T>(__ldg(reinterpret_cast<const uint4*>(weight) + lane), w);
      const float inv = rsqrtf(ss / static_cast<float>(D) + p.eps);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = f[i] * inv * w[i];
    }
    // the partner's elements for split pairs: rotary_dim / 16 lanes further on or back
    const int partner = lane < pairs ? lane + pairs : lane - pairs;
    const bool turned = !is_v && lane < 2 * pairs;
    float other[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) other[i] = __shfl_sync(0xffffffffu, f[i], turned ? partner : lane, kLanes);
    if (turned) {
      if (p.interleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 t = turn[lane * 4 + i];
          const float a = f[2 * i], b = f[2 * i + 1];
          f[2 * i] = a * t.y - b * t.x;
          f[2 * i + 1] = b * t.y + a * t.x;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 t = turn[(lane % pairs) * 8 + i];
          f[i] = lane < pairs ? f[i] * t.y - other[i] * t.x : f[i] * t.y + other[i] * t.x;
        }
      }
    }
    if constexpr (E4M3) {
      float big = 0.0f;
      bool fine = true;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        big = fmaxf(big, fabsf(f[i]));
        fine = fine && fabsf(f[i]) <= 3.402823466e38f;
      }
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) {
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
        fine = __shfl_xor_sync(0xffffffffu, fine ? 1 : 0, o) && fine;
      }
      if (live && !is_q && page >= 0) {
        const int e = fine ? row_exponent(big) : 0;
        const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);      // 2^-e: a normal number, and the product is exact
        const int64_t at = ((page * p.c.kv_heads + (head - p.heads - (is_v ? p.c.kv_heads : 0))) << p.c.page_shift) + row;
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = fine ? e4m3_pair(f[2 * i] * down, f[2 * i + 1] * down) : 0;
        reinterpret_cast<uint2*>(is_v ? p.c.v : p.c.k)[at * kLanes + lane] = make_uint2(u[0] | u[1] << 16, u[2] | u[3] << 16);
        if (lane == 0) (is_v ? p.c.v_exp : p.c.k_exp)[at] = static_cast<uint8_t>(fine ? e + 127 : 255);
      }
      if (live && is_q) reinterpret_cast<uint4*>(p.q_out)[(static_cast<int64_t>(token) * p.heads + head) * kLanes + lane] = pack8<T>(f);
    } else {
      if (live) {
        const uint4 w = pack8<T>(f);
        if (is_q) {
          reinterpret_cast<uint4*>(p.q_out)[(static_cast<int64_t>(token) * p.heads + head) * kLanes + lane] = w;
        } else if (page >= 0) {
          const int64_t at = ((page * p.c.kv_heads + (head - p.heads - (is_v ? p.c.kv_heads : 0))) << p.c.page_shift) + row;
          reinterpret_cast<uint4*>(is_v ? p.c.v : p.c.k)[at * kLanes + lane] = w;
        }
      }
    }
  }
}

struct ReadParams {
  CacheView c;
  uint8_t* k_out;
  uint8_t* v_out;
  const int32_t* cu_kv;
  int* status;
  int32_t seqs;
  int64_t total;
};

// A position's row of all heads at a time: kv_heads * D / 8 threads of 16 bytes (of k, then of v).
template <typename T, int D, bool E4M3>
__global__ void __launch_bounds__(kThreads) read_kernel(const ReadParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int kLanes = D / 8;
  const int per_row = p.c.kv_heads * kLanes;
  const int64_t pieces = p.total * per_row;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < pieces; i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int64_t out_row = i / per_row;
    const int piece = static_cast<int>(i - out_row * per_row), head = piece / kLanes, lane = piece % kLanes;
    const int seq = sequence_of(p.cu_kv, p.seqs, static_cast<int>(out_row));
    if (seq < 0) continue;
    const int pos = static_cast<int>(out_row) - p.cu_kv[seq];
    int64_t page = page_of(p.c, seq, pos, p.status);
    if (page < 0) page = 0;
    const int64_t at = ((page * p.c.kv_heads + head) << p.c.page_shift) + (pos & ((1 << p.c.page_shift) - 1));
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const uint8_t* src = which ? p.c.v : p.c.k;
      uint4 w;
      if constexpr (E4M3) {
        const uint2 codes = __ldg(reinterpret_cast<const uint2*>(src) + at * kLanes + lane);
        const RowFactors f = row_factors(__ldg((which ? p.c.v_exp : p.c.k_exp) + at));
        const uint2 a = row_values(codes.x, f), b = row_values(codes.y, f);
        w = make_uint4(a.x, a.y, b.x, b.y);
        if constexpr (!std::is_same<T, __nv_bfloat16>::value) {
          float v[8];
          unpack8<__nv_bfloat16>(w, v);
          w = pack8<T>(v);
        }
      } else {
        w = __ldg(reinterpret_cast<const uint4*>(src) + at * kLanes + lane);
      }
      reinterpret_cast<uint4*>(which ? p.v_out : p.k_out)[i] = w;
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
  return launch("append_kernel", kernel, a.tokens, stream, p);
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
  const int64_t pieces = total * c.kv_heads * (head_dim / 8);
  int64_t blocks = (pieces + kThreads - 1) / kThreads;
  const int64_t most = static_cast<int64_t>(device_sm_count()) * 16;
  return launch("read_kernel", kernel, blocks < most ? blocks : most, stream, p);
}

}  // namespace qmm
