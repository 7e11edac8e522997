// rotary.cu -- rotary positions of queries and keys (and their gradients).
//
// Each head's first 2 * half elements are `half` pairs; pair i of a token at position p is
// turned by the angle p * frequency[i]:
//   (a, b) -> amplitude * (a cos - b sin, b cos + a sin)
// Pairs are (i, i + half) or, interleaved, (2i, 2i + 1); the rest of the head is copied.  The
// gradient is the rotation by the negative angle (`inverse`).
//
// The angle of a far position is large (2^17 radians and more), so the product with the
// frequency and its reduction to a fraction of a turn are done in 64 bits -- in 32 the error
// of a position of 2^17 would be 2^-7 radians -- and only the fraction goes to 32 bits, for
// sincospif.  A cosine and sine are computed once per token and pair, into shared memory,
// and used by every head: 1 / (query_heads + kv_heads) of the work of computing them where
// they are used.
//
// What bounds it: the bytes of the queries and keys, read and written once.
#include <cuda_runtime.h>

#include "rk_device.cuh"
#include "rk_internal.h"

namespace rk {
namespace {

constexpr int THREADS = 256;

struct RotaryParams {
  const void* in[2];    // queries, keys
  void* out[2];         // dense [tokens, heads, head_dim]
  int64_t token_stride[2], head_stride[2];  // of the inputs, in elements
  const void* positions;
  const double* frequencies;
  int64_t tokens;
  int query_heads, heads;  // heads: query_heads + kv_heads
  int head_dim, half;
  int units;        // work items per head
  int turn_units;   // the first of them that rotate
  int index_bits;
  float amplitude;
  int inverse;
};

// One 16-byte vector of each half (HALVES) or of neighbouring pairs (INTERLEAVED), turned.
template <typename T>
__device__ __forceinline__ void turn_halves(uint4& a, uint4& b, const float2* cs) {
  uint32_t* pa = reinterpret_cast<uint32_t*>(&a);
  uint32_t* pb = reinterpret_cast<uint32_t*>(&b);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 x = Pack2<T>::to_floats(pa[j]), y = Pack2<T>::to_floats(pb[j]);
    const float4 t = *reinterpret_cast<const float4*>(cs + 2 * j);  // cos, sin, cos, sin
    pa[j] = Pack2<T>::from_floats(x.x * t.x - y.x * t.y, x.y * t.z - y.y * t.w);
    pb[j] = Pack2<T>::from_floats(y.x * t.x + x.x * t.y, y.y * t.z + x.y * t.w);
  }
}

template <typename T>
__device__ __forceinline__ void turn_pairs(uint4& a, const float2* cs) {
  uint32_t* pa = reinterpret_cast<uint32_t*>(&a);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 x = Pack2<T>::to_floats(pa[j]);
    const float2 t = cs[j];
    pa[j] = Pack2<T>::from_floats(x.x * t.x - x.y * t.y, x.y * t.x + x.x * t.y);
  }
}

// VEC: 16-byte vectors (head sizes, strides and pointers allow them); otherwise one pair or
// one element per item.  `tokens_per_cta` tokens share a CTA and its table of cosines.
template <typename T, bool INTERLEAVED, bool VEC>
__global__ void __launch_bounds__(THREADS) rotary_kernel(RotaryParams p, int tokens_per_cta) {
  extern __shared__ float2 table[];  // [tokens_per_cta][half]
  pdl_begin();
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * tokens_per_cta;
  const int nt = static_cast<int>(min(static_cast<int64_t>(tokens_per_cta), p.tokens - t0));
  for (int i = threadIdx.x; i < nt * p.half; i += THREADS) {
    const int t = i / p.half, f = i - t * p.half;
    const double position = p.index_bits == 32
                                ? static_cast<double>(static_cast<const int32_t*>(p.positions)[t0 + t])
                                : static_cast<double>(static_cast<const int64_t*>(p.positions)[t0 + t]);
    const double turns = position * (p.frequencies[f] * 0.15915494309189533577);  // 1 / (2 pi)
    float s, c;
    sincospif(2.0f * static_cast<float>(turns - rint(turns)), &s, &c);
    table[i] = make_float2(c * p.amplitude, (p.inverse ? -s : s) * p.amplitude);
  }
  __syncthreads();
  const int items = nt * p.heads * p.units;
  for (int item = threadIdx.x; item < items; item += THREADS) {
    const int row = item / p.units, unit = item - row * p.units;
    const int t = row / p.heads, h = row - t * p.heads;
    const int which = h >= p.query_heads;
    const int head = which ? h - p.query_heads : h;
    const int nheads = which ? p.heads - p.query_heads : p.query_heads;
    const T* in = static_cast<const T*>((which ? p.in[1] : p.in[0])) + (t0 + t) * (which ? p.token_stride[1] : p.token_stride[0]) + head * (which ? p.head_stride[1] : p.head_stride[0]);
    T* out = static_cast<T*>((which ? p.out[1] : p.out[0])) + ((t0 + t) * nheads + head) * p.head_dim;
    const float2* cs = table + t * p.half;
    if (VEC) {
      if (unit < p.turn_units) {
        if (INTERLEAVED) {
          uint4 a = ld_stream_v4(in + unit * 8);
          turn_pairs<T>(a, cs + unit * 4);
          *reinterpret_cast<uint4*>(out + unit * 8) = a;
        } else {
          uint4 a = ld_stream_v4(in + unit * 8);
          uint4 b = ld_stream_v4(in + p.half + unit * 8);
          turn_halves<T>(a, b, cs + unit * 8);
          *reinterpret_cast<uint4*>(out + unit * 8) = a;
          *reinterpret_cast<uint4*>(out + p.half + unit * 8) = b;
        }
      } else {
        const int at = 2 * p.half + (unit - p.turn_units) * 8;
        *reinterpret_cast<uint4*>(out + at) = ld_stream_v4(in + at);
      }
    } else {
      if (unit < p.turn_units) {
        const int ia = INTERLEAVED ? 2 * unit : unit, ib = INTERLEAVED ? 2 * unit + 1 : unit + p.half;
        const float a = to_f32(in[ia]), b = to_f32(in[ib]);
        const float2 t2 = cs[unit];
        out[ia] = from_f32<T>(a * t2.x - b * t2.y);
        out[ib] = from_f32<T>(b * t2.x + a * t2.y);
      } else {
        const int at = 2 * p.half + unit - p.turn_units;
        out[at] = in[at];
      }
    }
  }
}

template <typename T>
cudaError_t launch(const RotaryParams& p, bool interleaved, bool vec, int per_cta, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>((p.tokens + per_cta - 1) / per_cta));
  const size_t smem = static_cast<size_t>(per_cta) * p.half * sizeof(float2);
  if (interleaved)
    return vec ? launch_kernel(rotary_kernel<T, true, true>, grid, dim3(THREADS), smem, s, 0, p, per_cta)
               : launch_kernel(rotary_kernel<T, true, false>, grid, dim3(THREADS), smem, s, 0, p, per_cta);
  return vec ? launch_kernel(rotary_kernel<T, false, true>, grid, dim3(THREADS), smem, s, 0, p, per_cta)
             : launch_kernel(rotary_kernel<T, false, false>, grid, dim3(THREADS), smem, s, 0, p, per_cta);
}

}  // namespace

rk_status rotary_launch(const RotaryArgs& a, cudaStream_t s) {
  if (a.tokens == 0) return RK_OK;
  RotaryParams p{};
  p.in[0] = a.query;
  p.in[1] = a.key;
  p.out[0] = a.query_out;
  p.out[1] = a.key_out;
  p.token_stride[0] = a.query_token_stride;
  p.token_stride[1] = a.key_token_stride;
  p.head_stride[0] = a.query_head_stride;
  p.head_stride[1] = a.key_head_stride;
  p.positions = a.positions;
  p.frequencies = a.frequencies;
  p.tokens = a.tokens;
  p.query_heads = static_cast<int>(a.query_heads);
  p.heads = static_cast<int>(a.query_heads + a.kv_heads);
  p.head_dim = static_cast<int>(a.head_dim);
  p.half = static_cast<int>(a.rotary_dim / 2);
  p.index_bits = a.index_bits;
  p.amplitude = a.amplitude;
  p.inverse = a.inverse ? 1 : 0;
  bool vec = a.head_dim % 8 == 0 && (a.interleaved ? p.half % 4 == 0 : p.half % 8 == 0);
  for (int w = 0; w < 2; ++w)
    vec = vec && aligned16(p.in[w]) && aligned16(p.out[w]) && p.token_stride[w] % 8 == 0 && p.head_stride[w] % 8 == 0;
  if (vec) {
    p.turn_units = a.interleaved ? p.half / 4 : p.half / 8;
    p.units = p.turn_units + (p.head_dim - 2 * p.half) / 8;
  } else {
    p.turn_units = p.half;
    p.units = p.half + p.head_dim - 2 * p.half;
  }
  // Few tokens: one CTA each, so that they spread over the SMs.  Many: four to a CTA.
  const int per_cta = p.tokens >= 16 * static_cast<int64_t>(device_sm_count()) ? 4 : 1;
  const cudaError_t e = a.dt == RK_DTYPE_BF16 ? launch<__nv_bfloat16>(p, a.interleaved, vec, per_cta, s)
                                              : launch<__half>(p, a.interleaved, vec, per_cta, s);
  note_launch("rotary_kernel");
  return cuda_status(e);
}

}  // namespace rk
