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
// What bounds it: the bytes of the queries and keys, read and written once (8192 tokens of 32 + 8
// heads of 128 in bf16: 168 MB in 29.2 us, 5.7 TB/s; 16 tokens: 2.4 us, the launch).  Heads whose
// sizes allow only 8- or 4-byte vectors: 5000 tokens of 28 + 2 heads of 80, 40 or 20 of them turned,
// 48 MB in 13.9 us (50.8 an element at a time).
#include <cuda_runtime.h>

#include "rk_device.cuh"
#include "rk_internal.h"

namespace rk {
namespace {

constexpr int THREADS = 256;
constexpr int MOST_TOKENS = 8;  // of a CTA: a table of 32 KB at most
// Rows of a thread in flight, of two vectors each.
constexpr int rows_ahead(int width) { return width == 8 ? 2 : 4; }

struct RotaryParams {
  const void* in[2];    // queries, keys
  void* out[2];         // dense [tokens, heads, head_dim]
  int64_t token_stride[2], head_stride[2];  // of the inputs, in elements
  const void* positions;
  const double* frequencies;
  int64_t tokens;
  int query_heads, heads;  // heads: query_heads + kv_heads
  int head_dim, half;
  int units;        // work items per head: two vectors each (or elements, without vectors)
  int turn_units;   // the first of them that rotate
  int index_bits;
  float amplitude;
  int inverse;
};

// Where a pair's cosine and sine lie in its token's row of the table.  Lanes read 16 bytes each,
// 64 apart (8 pairs, one unit): in order, four of every eight would meet in the same banks (8192
// tokens of 32 + 8 heads of 128: 32.8 us instead of 29.2), so the unit's number exchanges its four.
__device__ __forceinline__ int table_at(int pair) { return pair ^ ((pair >> 3) & 6); }

// W elements of 16 bits, loaded and stored at once.
template <int W>
struct Vector {
  uint32_t w[W / 2];
};
template <>
struct Vector<1> {};
template <int W>
__device__ __forceinline__ Vector<W> load_vector(const void* from) {
  Vector<W> v;
  if constexpr (W == 8) {
    const uint4 x = ld_stream_v4(from);
    v.w[0] = x.x;
    v.w[1] = x.y;
    v.w[2] = x.z;
    v.w[3] = x.w;
  } else if constexpr (W == 4) {
    const uint2 x = __ldcs(static_cast<const uint2*>(from));
    v.w[0] = x.x;
    v.w[1] = x.y;
  } else {
    v.w[0] = __ldcs(static_cast<const uint32_t*>(from));
  }
  return v;
}
template <int W>
__device__ __forceinline__ void store_vector(void* to, const Vector<W>& v) {
  if constexpr (W == 8) {
    *static_cast<uint4*>(to) = make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]);
  } else if constexpr (W == 4) {
    *static_cast<uint2*>(to) = make_uint2(v.w[0], v.w[1]);
  } else {
    *static_cast<uint32_t*>(to) = v.w[0];
  }
}

// Cosine and sine of two neighbouring pairs, the j-th (even) of those that begin at `at` =
// table_at(a multiple of their number).
__device__ __forceinline__ float4 turns_of(const float2* row, int at, int j) {
  return *reinterpret_cast<const float4*>(row + (at ^ j));
}

// Two vectors that a lane turns: the first and second elements of W pairs from `pair` on.
template <typename T, int W>
__device__ __forceinline__ void turn_halves(Vector<W>& a, Vector<W>& b, const float2* row, int pair) {
  const int at = table_at(pair);
#pragma unroll
  for (int j = 0; j < W / 2; ++j) {
    const float2 x = Pack2<T>::to_floats(a.w[j]), y = Pack2<T>::to_floats(b.w[j]);
    const float4 t = turns_of(row, at, 2 * j);  // cos, sin, cos, sin
    a.w[j] = Pack2<T>::from_floats(x.x * t.x - y.x * t.y, x.y * t.z - y.y * t.w);
    b.w[j] = Pack2<T>::from_floats(y.x * t.x + x.x * t.y, y.y * t.z + x.y * t.w);
  }
}

// A vector of W / 2 neighbouring pairs from `pair` on.
template <typename T, int W>
__device__ __forceinline__ void turn_pairs(Vector<W>& a, const float2* row, int pair) {
  if constexpr (W == 2) {
    const float2 t = row[table_at(pair)];
    const float2 x = Pack2<T>::to_floats(a.w[0]);
    a.w[0] = Pack2<T>::from_floats(x.x * t.x - x.y * t.y, x.y * t.x + x.x * t.y);
  } else {
    const int at = table_at(pair);
#pragma unroll
    for (int j = 0; j < W / 2; j += 2) {
      const float4 t = turns_of(row, at, j);
      const float2 x = Pack2<T>::to_floats(a.w[j]), y = Pack2<T>::to_floats(a.w[j + 1]);
      a.w[j] = Pack2<T>::from_floats(x.x * t.x - x.y * t.y, x.y * t.x + x.x * t.y);
      a.w[j + 1] = Pack2<T>::from_floats(y.x * t.z - y.y * t.w, y.y * t.z + y.x * t.w);
    }
  }
}

// Pairs of a row of the table: whole units.
__host__ __device__ constexpr int table_stride(int half) { return (half + 7) & ~7; }

// A CTA takes some tokens.  Each thread keeps one unit of a head (no division in the loop) and
// walks over the heads of the tokens, ROWS of them in flight; the first are on their way while
// the threads fill the table of the tokens' cosines and sines.  W: elements of a vector, the most
// that head sizes, strides and pointers allow; 1: a pair or an element at a time.
template <typename T, bool INTERLEAVED, int W>
__global__ void __launch_bounds__(THREADS, W == 8 ? 6 : 5) rotary_kernel(RotaryParams p, int tokens_per_cta) {
  constexpr bool VEC = W > 1;
  constexpr int ROWS = VEC ? rows_ahead(W) : 1;
  extern __shared__ __align__(16) float2 table[];  // [tokens_per_cta][stride]
  const int stride = table_stride(p.half);
  pdl_begin();
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * tokens_per_cta;
  const int nt = static_cast<int>(min(static_cast<int64_t>(tokens_per_cta), p.tokens - t0));
  const int rows = nt * p.heads;
  const int side = min(p.units, THREADS);  // threads of a row
  const int step = THREADS / side;         // rows side by side; threads left over take none
  const int row0 = threadIdx.x / side;
  int unit = row0 < step ? threadIdx.x - row0 * side : p.units;

  // Elements of the unit's two vectors, and whether there is a second.
  int first = 0, second = 0;
  bool turns = false, both = false;
  const auto look_at_unit = [&] {
    turns = unit < p.turn_units;
    if (!VEC) {
      first = turns ? (INTERLEAVED ? 2 * unit : unit) : unit + p.half;  // behind the pairs one element each
      second = INTERLEAVED ? first + 1 : first + p.half;
      both = turns;
    } else if (INTERLEAVED || !turns) {
      first = INTERLEAVED ? unit * 2 * W : 2 * p.half + (unit - p.turn_units) * 2 * W;
      second = first + W;
      both = second < p.head_dim;
    } else {
      first = unit * W;
      second = first + p.half;
      both = true;
    }
  };
  // Walks over ROWS rows from (t, h) on, handing each its place in the loop.
  const auto walk = [&](int row, int t, int h, const auto& visit) {
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      if (row + k * step < rows) visit(k, t, h);
      h += step;
      while (h >= p.heads) {
        h -= p.heads;
        ++t;
      }
    }
  };
  Vector<W> a[ROWS], b[ROWS];
  const auto source = [&](int t, int h) {
    const bool key = h >= p.query_heads;
    return static_cast<const T*>(key ? p.in[1] : p.in[0]) + (t0 + t) * (key ? p.token_stride[1] : p.token_stride[0]) +
           (key ? h - p.query_heads : h) * (key ? p.head_stride[1] : p.head_stride[0]);
  };
  const auto load = [&](int k, int t, int h) {
    if constexpr (VEC) {
      const T* in = source(t, h);
      a[k] = load_vector<W>(in + first);
      if (both) b[k] = load_vector<W>(in + second);
    }
  };
  const auto turn_and_store = [&](int k, int t, int h) {
    const bool key = h >= p.query_heads;
    const int head = key ? h - p.query_heads : h, nheads = key ? p.heads - p.query_heads : p.query_heads;
    T* out = static_cast<T*>(key ? p.out[1] : p.out[0]) + ((t0 + t) * nheads + head) * p.head_dim;
    const float2* cs = table + t * stride;
    if constexpr (VEC) {
      if (INTERLEAVED) {
        // The border between turned and copied elements lies on a vector's.
        if (first < 2 * p.half) turn_pairs<T, W>(a[k], cs, unit * W);
        if (second < 2 * p.half) turn_pairs<T, W>(b[k], cs, unit * W + W / 2);
      } else if (turns) {
        turn_halves<T, W>(a[k], b[k], cs, first);
      }
      store_vector<W>(out + first, a[k]);
      if (both) store_vector<W>(out + second, b[k]);
    } else {
      const T* in = source(t, h);
      if (turns) {
        const float x = to_f32(in[first]), y = to_f32(in[second]);
        const float2 c = cs[table_at(unit)];
        out[first] = from_f32<T>(x * c.x - y * c.y);
        out[second] = from_f32<T>(y * c.x + x * c.y);
      } else {
        out[first] = in[first];
      }
    }
  };

  const int start_t = row0 / p.heads, start_h = row0 - start_t * p.heads;
  int row = unit < p.units ? row0 : rows, t = start_t, h = start_h;
  look_at_unit();
  walk(row, t, h, load);

  for (int i = threadIdx.x; i < nt * p.half; i += THREADS) {
    const int at = i / p.half, f = i - at * p.half;
    const double position = p.index_bits == 32
                                ? static_cast<double>(static_cast<const int32_t*>(p.positions)[t0 + at])
                                : static_cast<double>(static_cast<const int64_t*>(p.positions)[t0 + at]);
    const double turned = position * (p.frequencies[f] * 0.15915494309189533577);  // 1 / (2 pi)
    float s, c;
    sincospif(2.0f * static_cast<float>(turned - rint(turned)), &s, &c);
    table[at * stride + table_at(f)] = make_float2(c * p.amplitude, (p.inverse ? -s : s) * p.amplitude);
  }
  __syncthreads();

#pragma unroll 1
  while (row < rows) {
    walk(row, t, h, turn_and_store);
    row += ROWS * step;
    h += ROWS * step;
    while (h >= p.heads) {
      h -= p.heads;
      ++t;
    }
    if (row >= rows && unit + side < p.units) {  // heads of more units than threads
      unit += side;
      row = row0;
      t = start_t;
      h = start_h;
      look_at_unit();
    }
    walk(row, t, h, load);
  }
}

template <typename T, bool INTERLEAVED>
cudaError_t launch(const RotaryParams& p, int width, int per_cta, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>((p.tokens + per_cta - 1) / per_cta));
  const size_t smem = static_cast<size_t>(per_cta) * table_stride(p.half) * sizeof(float2);
  switch (width) {
    case 8: return launch_kernel(rotary_kernel<T, INTERLEAVED, 8>, grid, dim3(THREADS), smem, s, 0, p, per_cta);
    case 4: return launch_kernel(rotary_kernel<T, INTERLEAVED, 4>, grid, dim3(THREADS), smem, s, 0, p, per_cta);
    case 2: return launch_kernel(rotary_kernel<T, INTERLEAVED, 2>, grid, dim3(THREADS), smem, s, 0, p, per_cta);
    default: return launch_kernel(rotary_kernel<T, INTERLEAVED, 1>, grid, dim3(THREADS), smem, s, 0, p, per_cta);
  }
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
  // The most elements that every vector's place and size allow.
  int64_t places = a.head_dim | (a.interleaved ? 2 * p.half : p.half);
  for (int w = 0; w < 2; ++w)
    places |= p.token_stride[w] | p.head_stride[w] |
              static_cast<int64_t>((reinterpret_cast<uintptr_t>(p.in[w]) | reinterpret_cast<uintptr_t>(p.out[w])) / sizeof(uint16_t));
  const int width = places % 8 == 0 ? 8 : places % 4 == 0 ? 4 : places % 2 == 0 ? 2 : 1;
  if (width > 1) {
    // Two vectors to a unit: neighbours, or the two halves of the pairs.
    p.turn_units = p.half / width;  // interleaved units look at their elements
    const int two = 2 * width;
    p.units = a.interleaved ? (p.head_dim + two - 1) / two : p.turn_units + (p.head_dim - 2 * p.half + two - 1) / two;
  } else {
    p.turn_units = p.half;
    p.units = p.half + p.head_dim - 2 * p.half;
  }
  // Few tokens: one CTA each, so that they spread over the SMs.  Many: as many to a CTA as keep its
  // threads busy, but 4 CTAs for each SM (8192 tokens of 32 + 8 heads of 128: 29.1 us with two,
  // 33.9 with one, 30.0 with four; 1000 tokens: 7.4, 5.9, 10.5).
  const int64_t fill = (rows_ahead(width) * THREADS + p.heads * p.units - 1) / (p.heads * p.units);
  const int64_t spread = p.tokens / (4 * static_cast<int64_t>(device_sm_count()));
  const int64_t most = fill < spread ? fill : spread;
  const int per_cta = static_cast<int>(most < 1 ? 1 : most > MOST_TOKENS ? MOST_TOKENS : most);
  cudaError_t e;
  if (a.dt == RK_DTYPE_BF16)
    e = a.interleaved ? launch<__nv_bfloat16, true>(p, width, per_cta, s) : launch<__nv_bfloat16, false>(p, width, per_cta, s);
  else
    e = a.interleaved ? launch<__half, true>(p, width, per_cta, s) : launch<__half, false>(p, width, per_cta, s);
  note_launch("rotary_kernel");
  return cuda_status(e);
}

}  // namespace rk
