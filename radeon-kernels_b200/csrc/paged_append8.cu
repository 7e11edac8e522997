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
// new scale.  Where blocks are larger than that, teams of 2 to 8 warps do, and agree on the
// magnitude in shared memory.  No atomics on data, no second pass over it.  A block whose
// tokens are not adjacent would have two owners: only the first run is stored, the others are
// skipped and reported.
//
// Up to SCAN_TOKENS tokens a CTA per token looks for its run and through the earlier slots by
// itself, in one launch.  Beyond that those looks would be quadratic: in a launch before, each
// run leaves its token in its block's claim (workspace), and only where a claim shows a second
// run of the block are the earlier slots read.  The claims need no clearing: whatever they
// held is checked against the slots.  The storing launch starts beside it and waits for it only
// when its first rows are there (13k tokens of 4 heads of 64: 9.0 us, 0.8 more with the runs listed by
// the first launch).
//
// What bounds it.  A decode step: launch and latency (a token each of 128 requests, 8 heads of
// 128: 3.6 us on the device).  A prefill: the bytes, 2 in and 1 out per element (43k
// tokens of 8 heads of 128 in bf16: 265 MB in 51 us, 5.2 TB/s), with 5 us of start and end; the
// instructions are near (60 % of the issue slots with magnitudes taken in fp32, and 56 us).
#include <cuda_runtime.h>

#include <type_traits>

#include "rk_cache8.cuh"
#include "rk_device.cuh"
#include "rk_internal.h"

namespace rk {
namespace {

constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
// More tokens than this: claims, and CTAs that list runs (300 requests with a token each, 8 heads of 128:
// 6.3 us in one launch, 7.0 in two; 600 requests 9.6 and 9.1; 390 of up to 9 tokens 12.1, 8.8).
constexpr int SCAN_TOKENS = 256;
constexpr int HELD = 8;            // 16-byte vectors a lane keeps
constexpr int APPEND_CTAS = 3;      // resident on an SM; four spill registers
constexpr int HELPERS = 8;          // tokens of a long run whose CTAs store it

// The tokens of one block: `len` from `token` on, ascending from `offset` to `last` in `block`.
struct Run {
  int32_t token, block;
  int16_t offset, len, last, unused;
};

struct AppendParams {
  const void* rows[2];  // keys, values
  int64_t token_stride[2], head_stride[2];
  uint8_t* cache[2];
  float* scales[2];
  const void* slots;
  int32_t* claims;  // per block: a token that starts a run of it; or anything
  uint8_t* rivals;  // per token that starts a run: whether another run of its block is known
  int parts;        // CTAs that share THREADS tokens
  int team;         // warps that hold a full block of a head
  int64_t capacity;  // num_blocks * block_size
  int32_t tokens;
  int heads, block_size, index_bits;
};

__device__ __forceinline__ int64_t slot_of(const AppendParams& p, int64_t t) {
  return p.index_bits == 32 ? static_cast<int64_t>(static_cast<const int32_t*>(p.slots)[t])
                            : static_cast<const int64_t*>(p.slots)[t];
}
__device__ __forceinline__ int block_of(const AppendParams& p, int64_t slot) {
  return p.capacity <= INT32_MAX ? static_cast<int>(static_cast<uint32_t>(slot) / static_cast<uint32_t>(p.block_size))
                                 : static_cast<int>(slot / p.block_size);
}

// Whether a token in `slot`, inside the cache, goes on with the run of one in `before`.
__device__ __forceinline__ bool goes_on(const AppendParams& p, int64_t before, int64_t slot, int block) {
  return before >= 0 && before < slot && before >= static_cast<int64_t>(block) * p.block_size;
}

// Tokens after `from` that go on with the run of `block`, counted by a warp.
__device__ __forceinline__ int more_tokens(const AppendParams& p, int64_t from, int block, int lane) {
  int more = 0;
  for (;;) {
    const int64_t t = from + 1 + more + lane;
    bool on = false;
    if (t < p.tokens) {
      const int64_t slot = slot_of(p, t);
      on = slot < p.capacity && slot < (static_cast<int64_t>(block) + 1) * p.block_size && goes_on(p, slot_of(p, t - 1), slot, block);
    }
    const uint32_t off = ~__ballot_sync(0xffffffffu, on);
    if (off != 0) return more + __ffs(off) - 1;
    more += 32;  // slots ascend within a block, so this ends after block_size of them
  }
}

// Whether `other` is a token that starts a run of `block`.
__device__ __forceinline__ bool starts_run(const AppendParams& p, int32_t other, int block) {
  if (other < 0 || other >= p.tokens) return false;
  const int64_t slot = slot_of(p, other), first = static_cast<int64_t>(block) * p.block_size;
  return slot >= first && slot < first + p.block_size && !(other > 0 && goes_on(p, slot_of(p, other - 1), slot, block));
}

__device__ __forceinline__ void wait_for_earlier_kernels() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Looks for blocks that have several runs.  A thread per token.  Each run leaves its
// token in its block's claim and sees what was there: anything, since nothing clears the
// claims, or the token of a run that came before it, which the slots tell apart.  Of several
// runs of a block all but the first to come see another, and the first finds another's token
// in the claim afterwards.
__global__ void __launch_bounds__(THREADS) append_claims_kernel(AppendParams p, KernelCtl ctl) {
  // The next kernel reads the call's inputs before it waits for this one: it may start once they
  // are there.
  wait_for_earlier_kernels();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t t = static_cast<int64_t>(blockIdx.x) * THREADS + threadIdx.x;
  if (t >= p.tokens) return;
  const int64_t slot = slot_of(p, t), before = t > 0 ? slot_of(p, t - 1) : -1;
  if (slot >= p.capacity) atomicOr(ctl.status, RK_DEV_ERR_BAD_INDEX);
  if (slot < 0 || slot >= p.capacity) return;
  const int block = block_of(p, slot);
  if (goes_on(p, before, slot, block)) return;
  const int32_t claimed = atomicExch(p.claims + block, static_cast<int32_t>(t));
  p.rivals[t] = claimed != static_cast<int32_t>(t) && starts_run(p, claimed, block);
}

// The runs that start in THREADS tokens from t0 on, in their order; returns how many, and whether one
// is longer than `held`.
__device__ __forceinline__ int list_runs(const AppendParams& p, int64_t t0, Run* runs, int held, bool* longer) {
  __shared__ int64_t s_slots[THREADS];
  __shared__ uint32_t s_breaks[WARPS];  // tokens that do not go on with the one before
  __shared__ uint32_t s_starts[WARPS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t t = t0 + threadIdx.x;
  int64_t slot = -1;
  int block = -1;
  bool on = false;
  if (t < p.tokens) {
    slot = slot_of(p, t);
    const int64_t before = t > 0 ? slot_of(p, t - 1) : -1;
    if (slot >= p.capacity) slot = -1;
    if (slot >= 0) {
      block = block_of(p, slot);
      on = goes_on(p, before, slot, block);
    }
  }
  const bool starts = slot >= 0 && !on;
  const uint32_t breaks = ~__ballot_sync(0xffffffffu, on), who = __ballot_sync(0xffffffffu, starts);
  s_slots[threadIdx.x] = slot;
  if (lane == 0) {
    s_breaks[warp] = breaks;
    s_starts[warp] = who;
  }
  __syncthreads();
  int len = 0;
  bool open = false;  // no break behind it in this CTA
  if (starts) {
    uint32_t rest = breaks & (lane == 31 ? 0u : ~0u << (lane + 1));
    int w = warp;
    while (rest == 0 && ++w < WARPS) rest = s_breaks[w];
    open = w == WARPS;
    len = (open ? THREADS : w * 32 + __ffs(rest) - 1) - static_cast<int>(threadIdx.x);
  }
  // At most one run of a CTA is open: its warp follows it.
  const uint32_t opens = __ballot_sync(0xffffffffu, open);
  int more = 0;
  if (opens != 0) more = more_tokens(p, t0 + THREADS - 1, __shfl_sync(0xffffffffu, block, __ffs(opens) - 1), lane);
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    const int n = __popc(s_starts[w]);
    before += w < warp ? n : 0;
    all += n;
  }
  if (starts) {
    const int64_t first = static_cast<int64_t>(block) * p.block_size;
    const int64_t last = open && more > 0 ? slot_of(p, t0 + THREADS - 1 + more) : s_slots[threadIdx.x + len - 1];
    runs[before + __popc(who & ((1u << lane) - 1))] =
        Run{static_cast<int32_t>(t), block, static_cast<int16_t>(slot - first),
            static_cast<int16_t>(open ? len + more : len), static_cast<int16_t>(last - first), 0};
  }
  *longer = __syncthreads_or((open ? len + more : len) > held) != 0;
  return all;
}

// The largest magnitude of 8 elements; infinities and NaN set no scale.
template <typename T>
__device__ __forceinline__ float amax8(const uint4& v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  float m = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = Pack2<T>::to_floats(w[j]);
    const float a = fabsf(f.x), b = fabsf(f.y);
    m = fmaxf(m, a < INFINITY ? a : 0.f);
    m = fmaxf(m, b < INFINITY ? b : 0.f);
  }
  return m;
}

// The same, pair by pair in 16 bits, but for infinities, which it returns.
template <typename T>
__device__ __forceinline__ uint32_t max2(uint32_t m, const uint4& v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t magnitude = w[j] & 0x7FFF7FFFu;
    if constexpr (std::is_same<T, __half>::value)
      asm("max.f16x2 %0, %0, %1;" : "+r"(m) : "r"(magnitude));  // NaN against a number: the number
    else
      asm("max.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(magnitude));
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

// Warps that store a run's head together: one, or `size`, a power of two.
struct Alone {
  static constexpr int size = 1, rank = 0, UNROLL = 1;
  __device__ __forceinline__ float largest(float x, int) { return x; }
};
struct Team {
  static constexpr int UNROLL = 4;  // of the rows that are not held
  int size, rank, barrier;
  float* most;  // [2][size] in shared memory
  int turn;
  __device__ __forceinline__ Team(int warps, int warp, float* places)
      : size(warps), rank(warp % warps), barrier(1 + warp / warps), most(places + warp / warps * warps), turn(0) {}
  // The largest of all warps' values.  A warp can be one call ahead of another at most, so two sets of
  // places are enough.
  __device__ __forceinline__ float largest(float x, int lane) {
    if (size == 1) return x;
    float* const at = most + turn * WARPS;
    turn ^= 1;
    if (lane == 0) at[rank] = x;
    asm volatile("bar.sync %0, %1;" ::"r"(barrier), "r"(size * 32) : "memory");
    for (int i = 0; i < size; ++i) x = fmaxf(x, at[i]);
    return x;
  }
};

// Rows of a head that a warp keeps in registers.
__host__ __device__ constexpr int held_rows(int head_dim) { return HELD * (256 / head_dim); }

// One run of one head of K or V (`pair` < heads: K), by a team.  `is_first` says whether the run
// is the first of its block; it is asked when the rows are there, before anything is stored.
template <typename T, typename C, int D, typename Warps, typename First>
__device__ __forceinline__ void append_run(const AppendParams& p, const Run& run, int pair, int lane, Warps& team,
                                           const First& is_first) {
  constexpr int LANES = D / 8;      // lanes of a row, 8 elements each
  constexpr int ROWS = 32 / LANES;  // rows of a warp side by side
  const int side = ROWS * team.size;
  const int row = lane / LANES + ROWS * team.rank, at = (lane % LANES) * 8;
  const bool which = pair >= p.heads;
  const int head = which ? pair - p.heads : pair;
  const int64_t stride = which ? p.token_stride[1] : p.token_stride[0];
  const T* src = static_cast<const T*>(which ? p.rows[1] : p.rows[0]) + run.token * stride +
                 head * (which ? p.head_stride[1] : p.head_stride[0]) + at;
  const int rows = run.len - row;  // from this lane's first on, `side` apart
  uint4 held[HELD];
  {
    const T* from = src + row * stride;
#pragma unroll
    for (int k = 0; k < HELD; ++k) {
      held[k] = make_uint4(0, 0, 0, 0);
      if (k * side < rows) held[k] = ld_stream_v4(from);
      from += side * stride;
    }
  }
  const int64_t slot_bytes = static_cast<int64_t>(p.heads) * D;
  const int64_t slot0 = static_cast<int64_t>(run.block) * p.block_size;
  uint8_t* dst = (which ? p.cache[1] : p.cache[0]) + slot0 * slot_bytes + static_cast<int64_t>(head) * D + at;
  float* scale = (which ? p.scales[1] : p.scales[0]) + static_cast<int64_t>(run.block) * p.heads + head;
  const float was_raw = run.offset == 0 ? 0.f : *scale;
  const float was = was_raw > 0.f && was_raw < INFINITY ? was_raw : 0.f;

  uint32_t most = 0;
#pragma unroll
  for (int k = 0; k < HELD; ++k) most = max2<T>(most, held[k]);
  const float2 of_most = Pack2<T>::to_floats(most);
  float amax = fmaxf(of_most.x, of_most.y);
  if (amax == INFINITY) {
    amax = 0.f;
#pragma unroll
    for (int k = 0; k < HELD; ++k) amax = fmaxf(amax, amax8<T>(held[k]));
  }
  // Unpacked again for the store: kept from here, their fp32 values would take twice the
  // registers of the rows themselves.
#pragma unroll
  for (int k = 0; k < HELD; ++k) asm volatile("" : "+r"(held[k].x), "+r"(held[k].y), "+r"(held[k].z), "+r"(held[k].w));
#pragma unroll Warps::UNROLL
  for (int r = row + HELD * side; r < run.len; r += side)
    amax = fmaxf(amax, amax8<T>(*reinterpret_cast<const uint4*>(src + r * stride)));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  amax = team.largest(amax, lane);  // and every warp has read the old scale
  const float now = fmaxf(was, C::scale_for(amax));
  const float inv = 1.0f / now;

  if (!is_first()) return;
  const bool dense = run.last - run.offset == run.len - 1;  // no holes
  if (run.offset > 0 && now != was) {
    // Rows that stay: those below the last new one that the run does not write.
#pragma unroll 1
    for (int r = row; r < run.last; r += side) {
      bool stays = r < run.offset;
      if (!stays && !dense) {
        int lo = 0, hi = run.len - 1;  // the run's slots ascend
        while (lo < hi) {
          const int mid = (lo + hi) >> 1;
          if (slot_of(p, run.token + mid) - slot0 >= r) hi = mid;
          else lo = mid + 1;
        }
        stays = slot_of(p, run.token + lo) - slot0 != r;
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
  if (dense) {
    uint8_t* to = dst + (run.offset + row) * slot_bytes;
#pragma unroll
    for (int k = 0; k < HELD; ++k) {
      if (k * side < rows) *reinterpret_cast<uint2*>(to) = store8<T, C>(held[k], inv);
      to += side * slot_bytes;
    }
  }
#pragma unroll Warps::UNROLL
  for (int r = row + (dense ? HELD * side : 0); r < run.len; r += side) {
    const int64_t o = dense ? run.offset + r : slot_of(p, run.token + r) - slot0;
    *reinterpret_cast<uint2*>(dst + o * slot_bytes) = store8<T, C>(*reinterpret_cast<const uint4*>(src + r * stride), inv);
  }
  __syncwarp();  // every lane has read the old scale
  if (lane == 0 && team.rank == 0) *scale = now;
}

// Few tokens: a CTA (of each 8 heads of K and V) per token, which goes on if a run starts there.  The CTAs
// of the next tokens of a run help if it is longer than a warp holds: teams of p.team warps store it.
template <typename T, typename C, int D, bool TEAMS>
__global__ void __launch_bounds__(THREADS) paged_append8_kernel(AppendParams p, KernelCtl ctl) {
  __shared__ float s_most[2 * WARPS];
  pdl_begin();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t t = blockIdx.x;
  const int64_t slot = slot_of(p, t);
  const int64_t before = t > 0 ? slot_of(p, t - 1) : -1;
  if (slot >= p.capacity && threadIdx.x == 0 && blockIdx.y == 0) atomicOr(ctl.status, RK_DEV_ERR_BAD_INDEX);
  if (slot < 0 || slot >= p.capacity) return;
  const int block = block_of(p, slot);
  const int64_t slot0 = static_cast<int64_t>(block) * p.block_size;
  int helps = 0;  // the token's number in its run
  int64_t first = slot;
  if (goes_on(p, before, slot, block)) {
    if (!TEAMS) return;
    // The run's first token, if it is one of the last few.
    const int64_t u = t - lane;
    int64_t here = -1;
    bool on = false;
    if (u > 0 && lane < HELPERS) {
      here = slot_of(p, u);
      on = here < slot0 + p.block_size && goes_on(p, slot_of(p, u - 1), here, block);
    } else if (u == 0) {
      here = slot_of(p, u);
    }
    helps = __ffs(~__ballot_sync(0xffffffffu, on)) - 1;
    if (helps >= HELPERS) return;
    t -= helps;
    first = __shfl_sync(0xffffffffu, here, helps);
  }
  const int len = 1 + more_tokens(p, t, block, lane);
  if (helps > 0 && len <= held_rows(D)) return;
  // A block that an earlier token went to has been stored by that run.
  bool seen = false;
  for (int64_t i = threadIdx.x; i < t; i += THREADS) {
    const int64_t other = slot_of(p, i);
    seen = seen || (other >= slot0 && other < slot0 + p.block_size);
  }
  if (__syncthreads_or(seen)) {
    if (threadIdx.x == 0 && blockIdx.y == 0 && helps == 0) atomicOr(ctl.status, RK_DEV_ERR_BAD_INDEX);
    return;
  }
  const Run run{static_cast<int32_t>(t), block, static_cast<int16_t>(first - slot0), static_cast<int16_t>(len),
                static_cast<int16_t>((len == 1 ? first : slot_of(p, t + len - 1)) - slot0), 0};
  const auto is_first = [] { return true; };
  if (TEAMS && len > held_rows(D)) {
    Team team(p.team, warp, s_most);
    const int pair = (helps * static_cast<int>(gridDim.y) + static_cast<int>(blockIdx.y)) * (WARPS / team.size) + warp / team.size;
    if (pair < 2 * p.heads) append_run<T, C, D>(p, run, pair, lane, team, is_first);
  } else {
    Alone team;
    const int pair = static_cast<int>(blockIdx.y) * WARPS + warp;
    if (pair < 2 * p.heads) append_run<T, C, D>(p, run, pair, lane, team, is_first);
  }
}

// Many tokens: `parts` CTAs for each THREADS of them, whose warps, or teams if a run is longer than a warp
// holds, take the runs' heads of K and V in turn.  Each CTA lists the runs for itself and loads its first rows while the claims are still
// being made.
template <typename T, typename C, int D, bool TEAMS>
__global__ void __launch_bounds__(THREADS, APPEND_CTAS) paged_append8_runs_kernel(AppendParams p, KernelCtl ctl) {
  __shared__ __align__(16) Run s_runs[THREADS];
  __shared__ float s_most[2 * WARPS];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int list = static_cast<int>(blockIdx.x) / p.parts, part = static_cast<int>(blockIdx.x) - list * p.parts;
  const int pairs = 2 * p.heads;
  bool longer;
  const int items = list_runs(p, static_cast<int64_t>(list) * THREADS, s_runs, held_rows(D), &longer) * pairs;
  bool waited = false;
  const auto store = [&](auto& team, int item) {
    const int at = item / pairs, pair = item - at * pairs;
    const int4 raw = *reinterpret_cast<const int4*>(s_runs + at);
    const Run run{raw.x, raw.y, static_cast<int16_t>(raw.z & 0xFFFF), static_cast<int16_t>(raw.z >> 16),
                  static_cast<int16_t>(raw.w & 0xFFFF), 0};
    int32_t claim = 0;
    uint32_t rival = 0;
    const auto look = [&] {
      claim = __ldcg(p.claims + run.block);
      rival = __ldcg(p.rivals + run.token);
    };
    if (waited) look();
    append_run<T, C, D>(p, run, pair, lane, team, [&] {
      if (!waited) {
        wait_for_earlier_kernels();
        waited = true;
        look();
      }
      if (rival == 0 && claim == run.token) return true;
      // The block has several runs: the first is stored, the others are not.
      const int64_t slot0 = static_cast<int64_t>(run.block) * p.block_size;
      bool seen = false;
      for (int t0 = 0; t0 < run.token && !seen; t0 += 32) {
        const int64_t slot = t0 + lane < run.token ? slot_of(p, t0 + lane) : -1;
        seen = __any_sync(0xffffffffu, slot >= slot0 && slot < slot0 + p.block_size) != 0;
      }
      if (seen && lane == 0 && pair == 0 && team.rank == 0) atomicOr(ctl.status, RK_DEV_ERR_BAD_INDEX);
      return !seen;
    });
  };
  if (TEAMS && longer) {
    const int teams = WARPS / p.team;
    Team team(p.team, warp, s_most);
#pragma unroll 1
    for (int item = part * teams + warp / p.team; item < items; item += p.parts * teams) store(team, item);
  } else {
    Alone team;
#pragma unroll 1
    for (int item = part * WARPS + warp; item < items; item += p.parts * WARPS) store(team, item);
  }
  if (!waited) wait_for_earlier_kernels();
}

int64_t lists_of(int64_t tokens) { return (tokens + THREADS - 1) / THREADS; }

template <typename T, typename C, int D, bool TEAMS>
cudaError_t launch(const AppendParams& p, const KernelCtl& ctl, cudaStream_t s) {
  if (p.claims == nullptr) {
    const dim3 grid(static_cast<unsigned>(p.tokens), static_cast<unsigned>((2 * p.heads + WARPS - 1) / WARPS));
    note_launch("paged_append8_kernel");
    return launch_kernel(paged_append8_kernel<T, C, D, TEAMS>, grid, dim3(THREADS), 0, s, 0, p, ctl);
  }
  const int64_t lists = lists_of(p.tokens);
  note_launch("paged_append8_runs_kernel");
  return launch_kernel(paged_append8_runs_kernel<T, C, D, TEAMS>, dim3(static_cast<unsigned>(lists * p.parts)),
                       dim3(THREADS), 0, s, 0, p, ctl);
}

template <typename T, typename C, int D>
cudaError_t launch(const AppendParams& p, const KernelCtl& ctl, cudaStream_t s) {
  return p.team > 1 ? launch<T, C, D, true>(p, ctl, s) : launch<T, C, D, false>(p, ctl, s);
}

template <typename T, typename C>
cudaError_t launch_d(const AppendParams& p, int64_t head_dim, const KernelCtl& ctl, cudaStream_t s) {
  switch (head_dim) {
    case 64: return launch<T, C, 64>(p, ctl, s);
    case 128: return launch<T, C, 128>(p, ctl, s);
    default: return launch<T, C, 256>(p, ctl, s);
  }
}

}  // namespace

size_t paged_append8_workspace_bytes(int64_t tokens, int64_t num_blocks) {
  if (tokens <= SCAN_TOKENS) return 0;
  return static_cast<size_t>(num_blocks) * sizeof(int32_t) + static_cast<size_t>(tokens);
}

rk_status paged_append8_launch(const PagedAppend8Args& a, void* workspace, size_t workspace_bytes, cudaStream_t s) {
  if (a.tokens == 0) return RK_OK;
  const size_t need = paged_append8_workspace_bytes(a.tokens, a.num_blocks);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned16(workspace))) return RK_ERR_INVALID_ARGUMENT;
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
  p.tokens = static_cast<int32_t>(a.tokens);
  p.capacity = a.num_blocks * a.block_size;
  p.heads = static_cast<int>(a.kv_heads);
  p.block_size = static_cast<int>(a.block_size);
  // Warps that together hold a full block of a head: rows read once and a block's worth of loads at
  // once (36k tokens of 8 heads of 256 in blocks of 128: 142 us with one warp, 57 with eight).
  p.team = 1;
  while (p.team < WARPS && p.team * held_rows(static_cast<int>(a.head_dim)) < p.block_size) p.team *= 2;
  if (need > 0) {
    const int64_t lists = lists_of(a.tokens);
    p.claims = static_cast<int32_t*>(workspace);
    p.rivals = reinterpret_cast<uint8_t*>(p.claims + a.num_blocks);
    // CTAs that fill the GPU four times (43k tokens: the same from three to six; each lists its runs,
    // so not more), each with a run for every warp if blocks fill up -- but at least once, for
    // blocks that get a token each (600 tokens of 8 heads: 20 us with a run for every warp).
    const int64_t once = static_cast<int64_t>(device_sm_count()) * APPEND_CTAS, fill = 4 * once;
    const int64_t most = (THREADS / p.block_size + 1) * 2 * static_cast<int64_t>(p.heads) * p.team / WARPS + 1;
    const int64_t parts = (fill + lists - 1) / lists, least = (once + lists - 1) / lists;
    p.parts = static_cast<int>(parts < most ? parts : most < least ? least : most);
    const cudaError_t e = launch_kernel(append_claims_kernel, dim3(static_cast<unsigned>(lists)), dim3(THREADS), 0, s, 0, p, ctl);
    note_launch("append_claims_kernel");
    if (e != cudaSuccess) return cuda_status(e);
  }
  const bool bf16 = a.dt == RK_DTYPE_BF16, e4m3 = a.cache == RK_CACHE_E4M3;
  return cuda_status(bf16 ? (e4m3 ? launch_d<__nv_bfloat16, E4m3>(p, a.head_dim, ctl, s)
                                  : launch_d<__nv_bfloat16, Int8>(p, a.head_dim, ctl, s))
                          : (e4m3 ? launch_d<__half, E4m3>(p, a.head_dim, ctl, s)
                                  : launch_d<__half, Int8>(p, a.head_dim, ctl, s)));
}

}  // namespace rk
