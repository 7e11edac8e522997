// paged_append8.cu -- new keys and values into a paged cache of 8 bits, with one fp32 scale
// per block and head.
//
// For one cache, block and head, with x the new rows and s the block's scale so far:
//   need = the least power of two with max |x| <= LARGEST * need
//   s'   = need where the block is new (the call writes its first slot), else max(s, need)
//   stored(x) = round(x / s')
//   rows that stay below the last new one, where s' > s: round(stored * s / s')
// Scales are powers of two because blocks fill one token at a time: a growing scale then
// moves E4m3 values by whole exponents, which loses nothing but what falls under the
// smallest step, and a block is re-rounded only when its largest value doubles -- an exact
// fit (max |x| / LARGEST) would re-round a block of 16 about three times while it fills, with
// half a step of error each time.  The price is up to one bit of an Int8 value; E4m3, a
// floating type, pays none.
//
// Work: a token starts a run if the one before it goes to another block or not to a lower
// slot.  A run is one block's tokens, so a warp that owns (run, head, K or V) owns
// (block, head, K or V) alone: it takes the largest magnitude over the run's rows, holds them
// in registers (8 x 16 bytes a lane: 16 rows at head_dim 128), and stores them with the
// new scale.  No atomics, no second pass over the data.  A block whose tokens are not
// adjacent would have two owners: only the first run is stored, the others are skipped and
// reported.  Up to SCAN_TOKENS tokens every CTA looks through the earlier slots itself;
// beyond that a claim per block (workspace) is taken in a launch before.
//
// What bounds it: latency for a decode step, the bytes (2 in, 1 out per element) for a prefill.
#include <cuda_runtime.h>

#include "rk_cache8.cuh"
#include "rk_device.cuh"
#include "rk_internal.h"

namespace rk {
namespace {

constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int SPAN = 64;           // tokens of a CTA at most
constexpr int SCAN_TOKENS = 2048;  // more tokens than this: claims
constexpr int HELD = 8;            // 16-byte vectors a lane keeps

struct AppendParams {
  const void* rows[2];  // keys, values
  int64_t token_stride[2], head_stride[2];
  uint8_t* cache[2];
  float* scales[2];
  const void* slots;
  const int32_t* claims;  // per block: the first token of its first run; null: look through the slots
  int64_t tokens, capacity;  // capacity: num_blocks * block_size
  int heads, block_size, span, index_bits;
};

__device__ __forceinline__ int64_t slot_of(const void* slots, int index_bits, int64_t t) {
  return index_bits == 32 ? static_cast<int64_t>(static_cast<const int32_t*>(slots)[t])
                          : static_cast<const int64_t*>(slots)[t];
}

// Whether token t starts a run; `slot` is its slot, inside the cache.
__device__ __forceinline__ bool starts_run(const void* slots, int index_bits, int64_t t, int64_t slot, int block_size) {
  if (t == 0) return true;
  const int64_t before = slot_of(slots, index_bits, t - 1);
  return before < 0 || before >= slot || before / block_size != slot / block_size;
}

__global__ void __launch_bounds__(THREADS)
    append_claim_kernel(const void* slots, int index_bits, int64_t tokens, int64_t capacity, int block_size,
                        int32_t* claims) {
  pdl_begin();
  const int64_t t = static_cast<int64_t>(blockIdx.x) * THREADS + threadIdx.x;
  if (t >= tokens) return;
  const int64_t slot = slot_of(slots, index_bits, t);
  if (slot < 0 || slot >= capacity) return;
  if (starts_run(slots, index_bits, t, slot, block_size)) atomicMin(claims + slot / block_size, static_cast<int32_t>(t));
}

template <typename T>
__device__ __forceinline__ float amax8(const uint4& v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  float m = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = Pack2<T>::to_floats(w[j]);
    const float a = fabsf(f.x), b = fabsf(f.y);
    m = fmaxf(m, a < INFINITY ? a : 0.f);  // infinities and NaN set no scale
    m = fmaxf(m, b < INFINITY ? b : 0.f);
  }
  return m;
}

template <typename T, typename C>
__device__ __forceinline__ uint2 store8(const uint4& v, float inv) {
  const float2 a = Pack2<T>::to_floats(v.x), b = Pack2<T>::to_floats(v.y);
  const float2 c = Pack2<T>::to_floats(v.z), d = Pack2<T>::to_floats(v.w);
  return make_uint2(C::pack4(a.x * inv, a.y * inv, b.x * inv, b.y * inv),
                    C::pack4(c.x * inv, c.y * inv, d.x * inv, d.y * inv));
}

template <typename C>
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float was, float inv) {
  uint32_t lo, hi;
  C::halves(w, lo, hi);
  const float2 a = Pack2<__half>::to_floats(lo), b = Pack2<__half>::to_floats(hi);
  return C::pack4((a.x * was) * inv, (a.y * was) * inv, (b.x * was) * inv, (b.y * was) * inv);
}

template <typename T, typename C, int D>
__global__ void __launch_bounds__(THREADS) paged_append8_kernel(AppendParams p, KernelCtl ctl) {
  constexpr int LANES = D / 8;     // lanes of a row, 8 elements each
  constexpr int ROWS = 32 / LANES;  // rows side by side
  __shared__ int64_t s_token[SPAN];  // first token of each run that starts here
  __shared__ int64_t s_slot[SPAN];   // and its slot
  __shared__ int s_len[SPAN];
  __shared__ int s_drop[SPAN];
  __shared__ int s_runs;
  pdl_begin();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * p.span;
  const int span = static_cast<int>(min(static_cast<int64_t>(p.span), p.tokens - t0));
  if (threadIdx.x == 0) s_runs = 0;
  __syncthreads();
  if (threadIdx.x < span) {
    const int64_t t = t0 + threadIdx.x;
    const int64_t slot = slot_of(p.slots, p.index_bits, t);
    if (slot >= p.capacity) {
      atomicOr(ctl.status, RK_DEV_ERR_BAD_INDEX);
    } else if (slot >= 0 && starts_run(p.slots, p.index_bits, t, slot, p.block_size)) {
      const int at = atomicAdd(&s_runs, 1);  // any order: runs are independent
      s_token[at] = t;
      s_slot[at] = slot;
      s_drop[at] = p.claims != nullptr && p.claims[slot / p.block_size] != t;
    }
  }
  __syncthreads();
  const int runs = s_runs;
  for (int i = warp; i < runs; i += WARPS) {
    // Length of the run: 32 tokens at a time, until one does not continue it.
    const int64_t first = s_token[i], block = s_slot[i] / p.block_size;
    int64_t len = 1;
    for (;;) {
      const int64_t t = first + len + lane;
      bool on = false;
      if (t < p.tokens) {
        const int64_t slot = slot_of(p.slots, p.index_bits, t), before = slot_of(p.slots, p.index_bits, t - 1);
        on = slot > before && slot < p.capacity && before >= 0 && slot / p.block_size == block;
      }
      const uint32_t off = ~__ballot_sync(0xffffffffu, on);
      if (off != 0) {
        len += __ffs(off) - 1;
        break;
      }
      len += 32;
    }
    if (p.claims == nullptr) {
      bool seen = false;
      for (int64_t t = lane; t < first; t += 32) {
        const int64_t slot = slot_of(p.slots, p.index_bits, t);
        seen = seen || (slot >= 0 && slot < p.capacity && slot / p.block_size == block);
      }
      if (lane == 0) s_drop[i] = 0;
      __syncwarp();
      if (__any_sync(0xffffffffu, seen) && lane == 0) s_drop[i] = 1;
    }
    if (lane == 0) {
      s_len[i] = static_cast<int>(len);  // slots ascend within a block: at most block_size
      if (s_drop[i]) atomicOr(ctl.status, RK_DEV_ERR_BAD_INDEX);
    }
  }
  __syncthreads();

  const int pairs = 2 * p.heads;
  const int y_pairs = min(WARPS, pairs - static_cast<int>(blockIdx.y) * WARPS);  // of this CTA
  const int row = lane / LANES, at = (lane - row * LANES) * 8;
  for (int item = warp; item < runs * y_pairs; item += WARPS) {
    const int i = item / y_pairs;
    const int pair = static_cast<int>(blockIdx.y) * WARPS + item - i * y_pairs;
    if (s_drop[i]) continue;
    const int which = pair >= p.heads, head = which ? pair - p.heads : pair;
    const int64_t first = s_token[i], slot0 = s_slot[i];
    const int64_t block = slot0 / p.block_size;
    const int offset0 = static_cast<int>(slot0 - block * p.block_size);
    const int len = s_len[i];
    const int64_t stride = which ? p.token_stride[1] : p.token_stride[0];
    const T* src = static_cast<const T*>(which ? p.rows[1] : p.rows[0]) + first * stride +
                   head * (which ? p.head_stride[1] : p.head_stride[0]) + at;
    const int64_t slot_bytes = static_cast<int64_t>(p.heads) * D;
    uint8_t* dst = (which ? p.cache[1] : p.cache[0]) + block * p.block_size * slot_bytes + static_cast<int64_t>(head) * D + at;
    float* scale = (which ? p.scales[1] : p.scales[0]) + block * p.heads + head;
    const float was_raw = offset0 == 0 ? 0.f : *scale;
    const float was = was_raw > 0.f && was_raw < INFINITY ? was_raw : 0.f;

    uint4 held[HELD];
    float amax = 0.f;
#pragma unroll
    for (int k = 0; k < HELD; ++k) {
      const int r = row + k * ROWS;
      held[k] = make_uint4(0, 0, 0, 0);
      if (r < len) held[k] = ld_stream_v4(src + r * stride);
    }
#pragma unroll
    for (int k = 0; k < HELD; ++k) amax = fmaxf(amax, amax8<T>(held[k]));
    for (int r = row + HELD * ROWS; r < len; r += ROWS)
      amax = fmaxf(amax, amax8<T>(*reinterpret_cast<const uint4*>(src + r * stride)));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const float now = fmaxf(was, C::scale_for(amax));
    const float inv = 1.0f / now;

    const int last = static_cast<int>(slot_of(p.slots, p.index_bits, first + len - 1) - block * p.block_size);
    if (offset0 > 0 && now != was) {
      // Rows that stay: those below the last new one that the run does not write.
      const bool dense = last - offset0 == len - 1;
      for (int r = row; r < last; r += ROWS) {
        bool stays = r < offset0;
        if (!stays && !dense) {
          int lo = 0, hi = len - 1;  // the run's slots ascend
          while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (slot_of(p.slots, p.index_bits, first + mid) - block * p.block_size >= r) hi = mid;
            else lo = mid + 1;
          }
          stays = slot_of(p.slots, p.index_bits, first + lo) - block * p.block_size != r;
        }
        if (stays) {
          uint2* cell = reinterpret_cast<uint2*>(dst + r * slot_bytes);
          uint2 v = *cell;
          v.x = rescale4<C>(v.x, was, inv);
          v.y = rescale4<C>(v.y, was, inv);
          *cell = v;
        }
      }
    }
#pragma unroll
    for (int k = 0; k < HELD; ++k) {
      const int r = row + k * ROWS;
      if (r < len) {
        const int64_t o = slot_of(p.slots, p.index_bits, first + r) - block * p.block_size;
        *reinterpret_cast<uint2*>(dst + o * slot_bytes) = store8<T, C>(held[k], inv);
      }
    }
    for (int r = row + HELD * ROWS; r < len; r += ROWS) {
      const int64_t o = slot_of(p.slots, p.index_bits, first + r) - block * p.block_size;
      *reinterpret_cast<uint2*>(dst + o * slot_bytes) =
          store8<T, C>(*reinterpret_cast<const uint4*>(src + r * stride), inv);
    }
    __syncwarp();  // every lane has read the old scale
    if (lane == 0) *scale = now;
  }
}

template <typename T, typename C>
cudaError_t launch_d(const AppendParams& p, int64_t head_dim, const KernelCtl& ctl, dim3 grid, cudaStream_t s) {
  switch (head_dim) {
    case 64: return launch_kernel(paged_append8_kernel<T, C, 64>, grid, dim3(THREADS), 0, s, 0, p, ctl);
    case 128: return launch_kernel(paged_append8_kernel<T, C, 128>, grid, dim3(THREADS), 0, s, 0, p, ctl);
    default: return launch_kernel(paged_append8_kernel<T, C, 256>, grid, dim3(THREADS), 0, s, 0, p, ctl);
  }
}

}  // namespace

size_t paged_append8_workspace_bytes(int64_t tokens, int64_t num_blocks) {
  return tokens > SCAN_TOKENS ? static_cast<size_t>(num_blocks) * sizeof(int32_t) : 0;
}

rk_status paged_append8_launch(const PagedAppend8Args& a, void* workspace, size_t workspace_bytes, cudaStream_t s) {
  if (a.tokens == 0) return RK_OK;
  const size_t need = paged_append8_workspace_bytes(a.tokens, a.num_blocks);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return RK_ERR_INVALID_ARGUMENT;
  LaunchCtl lc;
  const rk_status st = launch_ctl(&lc);
  if (st != RK_OK) return st;
  const KernelCtl ctl{lc.status, lc.timeout_ns, 0};
  AppendParams p{};
  p.rows[0] = a.key;
  p.rows[1] = a.value;
  p.token_stride[0] = a.key_token_stride;
  p.token_stride[1] = a.value_token_stride;
  p.head_stride[0] = a.key_head_stride;
  p.head_stride[1] = a.value_head_stride;
  p.cache[0] = static_cast<uint8_t*>(a.key_cache);
  p.cache[1] = static_cast<uint8_t*>(a.value_cache);
  p.scales[0] = a.key_scales;
  p.scales[1] = a.value_scales;
  p.slots = a.slot_mapping;
  p.index_bits = a.index_bits;
  p.tokens = a.tokens;
  p.capacity = a.num_blocks * a.block_size;
  p.heads = static_cast<int>(a.kv_heads);
  p.block_size = static_cast<int>(a.block_size);
  if (need > 0) {
    p.claims = static_cast<const int32_t*>(workspace);
    cudaError_t e = cudaMemsetAsync(workspace, 0x7F, need, s);  // above every token index
    if (e == cudaSuccess)
      e = launch_kernel(append_claim_kernel, dim3(static_cast<unsigned>((a.tokens + THREADS - 1) / THREADS)),
                        dim3(THREADS), 0, s, 0, a.slot_mapping, a.index_bits, a.tokens, p.capacity, p.block_size,
                        static_cast<int32_t*>(workspace));
    note_launch("append_claim_kernel");
    if (e != cudaSuccess) return cuda_status(e);
  }
  // One token to a CTA while that fills the GPU, up to SPAN beyond.
  const int64_t even = a.tokens / (4 * static_cast<int64_t>(device_sm_count()));
  p.span = static_cast<int>(even < 1 ? 1 : (even > SPAN ? SPAN : even));
  const dim3 grid(static_cast<unsigned>((a.tokens + p.span - 1) / p.span),
                  static_cast<unsigned>((2 * p.heads + WARPS - 1) / WARPS));
  const bool bf16 = a.dt == RK_DTYPE_BF16, e4m3 = a.cache == RK_CACHE_E4M3;
  const cudaError_t e =
      bf16 ? (e4m3 ? launch_d<__nv_bfloat16, E4m3>(p, a.head_dim, ctl, grid, s)
                   : launch_d<__nv_bfloat16, Int8>(p, a.head_dim, ctl, grid, s))
           : (e4m3 ? launch_d<__half, E4m3>(p, a.head_dim, ctl, grid, s) : launch_d<__half, Int8>(p, a.head_dim, ctl, grid, s));
  note_launch("paged_append8_kernel");
  return cuda_status(e);
}

}  // namespace rk
