// paged_attention8.cu -- decode attention over a paged K/V cache of 8 bits (E4m3 or Int8) with
// one fp32 scale per block and head, one query token per sequence:
//
//   s_t = scale * ks(t) * (q . k_t),  p_t = exp(s_t - max s),
//   out = sum_t p_t * vs(t) * v_t / sum_t p_t,        t < context_lengths[b]
//
// with k_t, v_t the stored 8-bit values of position t and ks, vs the scales of its block and
// head.  Query head h reads KV head h / (query_heads / kv_heads).
//
// Work.  The positions of every sequence are cut into units of 32 (16 at head_dim 256), and the
// units of all sequences and head tiles (a KV head and up to 8 or 16 of its query heads), laid
// end to end, are dealt out evenly to all warps of the GPU: each takes one stretch.  So one
// long sequence among short ones, or few sequences, load every SM alike, whatever the width of
// the block table.  A (sequence, head tile) is a range; RANGE_COST places between ranges stand
// for what starting and ending one costs.
//
// A range that a warp holds whole goes to the output from its registers.  Of one that is cut,
// each warp leaves the unnormalised sums and their statistics: the warps of a CTA join theirs
// in shared memory, CTAs meet in the workspace, where every CTA counts its parts in and the
// last to come joins them all -- of ranges over many CTAs, those of a group of neighbours, and
// the last group to be joined all groups --, in their order, so that results do not depend on
// timing.
// Nothing waits for another CTA.  (A second launch for the join measured 3 to 6 us more on
// 16 x 2048 positions, and a device-wide fence at each CTA's end 2 us: hence one count
// and one fence.)
//
// A warp feeds itself: a ring of two units of K and V with their scales in shared memory,
// filled by cp.async and running on across the ends of ranges; block-table entries 32 at a time
// and queries are loaded a range ahead.  No barrier until the warp's stretch is done.
//
// The matrix products are mma.sync m16n8k16 on f16 operands:
//   S^T[16 positions, 8 heads] = K[16, D] Q^T      O^T[16 dims, 8 heads] += V^T[16 dims, 16] P^T
// so a KV head's query heads fill the 8 columns, and each 8-bit value is unpacked once, in
// registers: both E4m3 and Int8 values are f16 numbers, exactly.  The order of a head's
// dimensions within the products is free; it is chosen such that a lane's operands are 16
// consecutive bytes of a row, and its results 16 neighbouring dimensions.  16 MMAs go with 4 KB
// of cache (D 128), a few per cent of the tensor pipe, so the products bound nothing; tcgen05
// would add a round trip through tensor memory and unpacked operands in shared memory.
//
// Numbers.  Queries are brought to f16 by a power of two per head (exact unless a component is
// below 2^-14 of the head's largest: then it keeps 2^-25 of that).  Scores, maxima, sums and
// accumulators are fp32.  The weights of V carry its scales, w_t = p_t * vs(t) * c with c =
// 2^(m - mo) for m the reference of the scores s (in powers of two) and mo that of s + log2 vs, each
// HEADROOM below the running maximum, and are rounded to f16 for the product: half a step, 2^-11, of
// each that is at least 2^-25 of the largest, however the scales differ from block to block,
// and 2^-36 of the largest for smaller ones, which vanish below that.  (With the largest near 1, 11 powers
// of two less, a first position that takes the weight and has no value left what lies 2^-25
// below it nothing.)  The denominator sums the p in fp32, unrounded, so n positions lose n * 2^-36 of
// the largest weight at most.  The maxima are raised
// only when a weight passes SLACK; in between p and w may reach that, inside the
// range of both types, and the sums need no rescaling.
//
// What bounds it: the bytes of K and V, 1.07 GB in 203 to 211 us at 4 x 131072 positions of 8 heads of
// 128 (5.1 TB/s; without the products it streamed them in 187 us, and some SMs finish
// their equal share 20 % before others).  At 16 x 2048 positions (67 MB, 21.5 us) the
// start and the end: 2.2 us until the first loads leave (lengths, then table, then rows: each
// waits for the one before), 4 us from the last tile to the last join.
#include <cuda_runtime.h>

#include <atomic>
#include <chrono>

#include "rk_cache8.cuh"
#include "rk_device.cuh"
#include "rk_internal.h"
#include "rk_paged8_shares.h"

namespace rk {
namespace pa8 {

constexpr int THREADS = WARPS * 32;
// Units of a warp's ring.  Three kept more bytes under way and cost more (8 x 15317 positions of 3 heads
// of 256: 51.9 us, and 46.5 with two; 61 sequences of 1 to 16 Ki, 4 heads of 128: 26.4, 25.3; 4 x 128
// Ki the same).
constexpr int STAGES = 2;
// Ranges over more CTAs than JOIN_ONCE are joined in two steps, JOIN_CTAS at a time first (one
// sequence of 20000 positions, one KV head of 128 with 4 query heads, 40 CTAs: 32 us at once, 15 in
// two steps; 17 CTAs of head_dim 256 with 8 query heads: 18.6 and 21.4).
constexpr int JOIN_ONCE = 24, JOIN_CTAS = 16;
// The largest weight lies HEADROOM powers of two above the reference that its maximum is, so that the f16
// weights of V reach far below it; the maxima are raised when a weight passes SLACK, inside f16's range.
// The less lies between the two, the more often (32 x 3000 positions of 4 KV heads with 16 query
// heads each: 35.9 us with 8 powers of two, 36.7 with these 4, 38.0 with 2; up to 8 query heads
// the same within 1 %).
constexpr float HEADROOM = 11.0f, SLACK = 32768.0f;
constexpr float NONE = -3.402823466e38f;  // a maximum before any score: finite, so that -inf - NONE = -inf

// CTAs of an SM, which the registers allow (held to 168 for three: 4 x 128 Ki positions 209 -> 215
// us, 16 x 2048 21.5 -> 23.9).
constexpr int CTAS_PER_SM = 2;

// Shared memory of a tile.  The 16-byte chunks of a row are exchanged by its number (chunk ^
// row % 8), so that the 128-bit reads of the MMA operands touch every bank once; at D 64,
// where 64-bit reads of V pair with 64-byte rows, V's rows are padded instead.
template <int D>
struct Layout {
  static constexpr int TILE = unit_of(D);
  static constexpr int V_STRIDE = D == 64 ? 80 : D;
  static constexpr int K_BYTES = TILE * D;
  static constexpr int SCALES = K_BYTES + TILE * V_STRIDE;  // of K, then of V
  static constexpr int MASK = SCALES + 2 * TILE * 4;        // which rows hold a position
  static constexpr int STAGE = MASK + 16;
  static constexpr int RING = WARPS * STAGES * STAGE;
  static __device__ __forceinline__ int k_at(int row, int chunk) {
    return row * D + (D == 64 ? chunk : chunk ^ (row & 7)) * 16;
  }
  static __device__ __forceinline__ int v_at(int row, int chunk) {
    return K_BYTES + row * V_STRIDE + (D == 64 ? chunk : chunk ^ (row & 7)) * 16;
  }
};

// A head's part in the workspace: the unnormalised sum, then m, mo, l and nothing.
__host__ __device__ constexpr int part_stride(int head_dim) { return head_dim + 4; }

struct Params {
  const void* q;
  const uint8_t* k;
  const uint8_t* v;
  const float* ks;
  const float* vs;
  const void* tables;
  const void* lens;
  void* out;
  float* part;      // [warp][2][heads of a tile][part_stride]: part 0 continues a range, part 1 begins one
  // [2][warp]: `tag` plus the parts that have been written -- of the range that the warp begins, then of
  // groups of CTAs of ranges that are joined in two steps -- or anything.
  uint64_t* arrivals;
  uint64_t tag;        // of this launch; its low 16 bits are 0, the others not all
  int batch, hq, hkv, group, head_groups;
  int num_blocks, block_size, max_blocks;
  uint32_t block_multiplier;  // t / block_size = t * block_multiplier >> block_shift for t < 2^31
  int block_shift;
  int index_bits, bf16;
  float scale_log2;
};

// A launch constant, hidden from the compiler, which would otherwise keep a copy of a loop for each
// value of each flag (5 KB of 62 at head_dim 128).
__device__ __forceinline__ int flag_of(int v) {
  asm volatile("" : "+r"(v));
  return v;
}

// An index as loaded: nothing waits for the load until value_of.
struct Raw {
  uint32_t lo, hi;
};
__device__ __forceinline__ Raw load_raw(const void* p, int bits, int64_t i) {
  Raw r{0, 0};
  if (flag_of(bits) == 32) {
    r.lo = __ldg(static_cast<const uint32_t*>(p) + i);
  } else {
    const uint2 v = __ldg(static_cast<const uint2*>(p) + i);
    r.lo = v.x;
    r.hi = v.y;
  }
  return r;
}
__device__ __forceinline__ int64_t value_of(Raw r, int bits) {
  return flag_of(bits) == 32 ? static_cast<int64_t>(static_cast<int32_t>(r.lo))
                    : static_cast<int64_t>(static_cast<uint64_t>(r.hi) << 32 | r.lo);
}

__device__ __forceinline__ int context_of(const Params& p, Raw raw) {
  const int64_t n = value_of(raw, p.index_bits);
  const int64_t room = static_cast<int64_t>(p.max_blocks) * p.block_size;  // below 2^31
  return static_cast<int>(n < 0 ? 0 : (n > room ? room : n));
}

__device__ __forceinline__ int context_of(const Params& p, int b) {
  return context_of(p, load_raw(p.lens, p.index_bits, b));
}

// The block of position t, by a multiplication (the host's multiplier is 2^block_shift /
// block_size, rounded up; with 31 bits more than block_size's that is exact below 2^31).
__device__ __forceinline__ int block_of(const Params& p, int t) {
  return static_cast<int>(static_cast<uint64_t>(static_cast<uint32_t>(t)) * p.block_multiplier >> p.block_shift);
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <typename T>
__device__ __forceinline__ T at_smem(const uint8_t* smem, int offset) {
  return *reinterpret_cast<const T*>(smem + offset);
}
// D[16 x 8] += A[16 x 16] B[16 x 8], f16 operands, fp32 accumulators.
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Transposes an 8 x 8 matrix of 16-bit values held across the warp.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float lg2_approx(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The parts in the workspace of a range that starts at `place`: that of the warp that begins it,
// one of each later CTA (of its first warp), and one of the warp that ends it where that
// is no CTA's first and went on to other ranges (otherwise it joined its neighbours').
struct Parts {
  int begin, end, ctas, count;
  Parts() = default;
  __device__ __forceinline__ Parts(uint32_t place, int units, const Shares& shares) {
    begin = static_cast<int>(shares.owner(place));
    end = static_cast<int>(shares.owner(place + units - 1));
    ctas = end / WARPS - begin / WARPS;
    const bool went_on = shares.start(end + 1) > place + units + RANGE_COST;
    count = 1 + ctas + (end % WARPS != 0 && end != begin && went_on ? 1 : 0);
  }
  __device__ __forceinline__ int warp(int i) const {
    return i == 0 ? begin : (i <= ctas ? (begin / WARPS + i) * WARPS : end);
  }
  // Part i in the workspace: 1 where the warp begins the range, 0 where it goes on with it.
  __device__ __forceinline__ int slot(int i) const { return i == 0 ? 1 : 0; }
  // Ranges over many CTAs are joined in two steps: JOIN_CTAS neighbours at a time, into the first
  // one's part, then those.
  __device__ __forceinline__ int groups() const { return ctas < JOIN_ONCE ? 1 : ctas / JOIN_CTAS + 1; }
  __device__ __forceinline__ int group_of(int cta) const { return (cta - begin / WARPS) / JOIN_CTAS; }
  __device__ __forceinline__ int parts_of(int group) const {
    return group + 1 < groups() ? JOIN_CTAS : count - group * JOIN_CTAS;
  }
  // Where a group's parts are counted, a warp of its first CTA.  Only one range goes from a CTA to the
  // next, so a CTA begins one group at most, and goes on with one.
  __device__ __forceinline__ int counter(int group) const {
    return (begin / WARPS + group * JOIN_CTAS) * WARPS + (group == 0 ? 1 : 0);
  }
};

// A range of which a warp holds a part.
struct Piece {
  uint32_t place;  // of the range's first unit
  int row, heads;  // of the output; no heads: there is no piece
  int begins, ends;  // whether the part holds the range's first and last unit
  Parts parts;
};

// Adds `parts` to the arrivals of a range and returns whether that makes `all`.  A word that does not
// carry the launch's tag counts as none; the last to arrive leaves 0, so that the next launch
// of a captured graph, whose tag is the same, starts anew.  The word was seen as `seen`: once
// tagged it stays so until the last arrival, so an addition is enough (tens of CTAs can come
// at once, and exchanges would repeat); the first to come to an untagged word tags it.
// Nothing waits for another CTA.
__device__ __forceinline__ bool arrive(uint64_t* word, uint64_t seen, uint64_t tag, int parts, int all) {
  auto* const at = reinterpret_cast<unsigned long long*>(word);
  uint64_t before = tag;
  for (;;) {
    if ((seen & ~uint64_t{0xFFFF}) == tag) {
      before = atomicAdd(at, static_cast<unsigned long long>(parts));
      break;
    }
    const uint64_t found = atomicCAS(at, seen, tag + parts);
    if (found == seen) break;
    seen = found;
  }
  const bool last = static_cast<int>(before & 0xFFFF) + parts == all;
  if (last) *word = 0;
  return last;
}
__device__ __forceinline__ void fence_gpu() { asm volatile("fence.acq_rel.gpu;" ::: "memory"); }

// The chunk (16 bytes of a row) that lane column c reads as its i-th of K.
template <int D>
__device__ __forceinline__ int k_chunk(int c, int i) {
  return D == 64 ? c : 2 * c + (i & 1) + 8 * (i >> 1);
}

// A place with its sequence's length; the next sequence's is loaded a sequence ahead.
struct Walk : Place {
  int context;
  Raw next;
};

// To the first unit of the next (sequence, head tile).  Past the last sequence the walk holds
// some valid length and is not used (left <= 0).
template <int D>
__device__ __forceinline__ void next_range(const Params& p, Walk& w) {
  if (!next_tile(w, p.hkv, p.head_groups)) return;
  w.context = context_of(p, w.next);
  w.units = units_of<D>(w.context);
  w.next = load_raw(p.lens, p.index_bits, min(w.b + 1, p.batch - 1));
}

template <int D>
__device__ __forceinline__ void next_unit(const Params& p, Walk& w) {
  ++w.c;
  --w.left;
  if (w.c == w.units) next_range<D>(p, w);
}

// N (a multiple of 4) neighbouring elements of an output row times f.
template <int N>
__device__ __forceinline__ void write_out(const Params& p, int64_t element, const float* v, float f) {
  uint32_t w[N / 2];
  const int bf16 = flag_of(p.bf16);
#pragma unroll
  for (int i = 0; i < N / 2; ++i)
    w[i] = bf16 ? Pack2<__nv_bfloat16>::from_floats(v[2 * i] * f, v[2 * i + 1] * f)
                  : Pack2<__half>::from_floats(v[2 * i] * f, v[2 * i + 1] * f);
  uint32_t* out = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.out) + element);
  if (N % 8 == 0) {
#pragma unroll
    for (int i = 0; i < N / 8; ++i)
      reinterpret_cast<uint4*>(out)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) reinterpret_cast<uint2*>(out)[i] = make_uint2(w[2 * i], w[2 * i + 1]);
  }
}

// What brings the sums to the output: the weights' sum, and from the one maximum to the
// other.  Without a position it is 1 / 0, and the sums 0.
__device__ __forceinline__ float last_factor(float m, float mo, float l) { return ex2_approx(mo - m) / l; }

template <int D, int HEADS>
__device__ __forceinline__ float* part_of(const Params& p, int warp, int k) {
  return p.part + (static_cast<int64_t>(warp) * 2 + k) * (HEADS * part_stride(D));
}

// Sums of one head, spread over the 16 lanes of half a warp.
template <int D>
struct Sums {
  static constexpr int V = D / 16;  // neighbouring dimensions of a lane
  float m, mo, l, v[V];
  __device__ __forceinline__ void start() {
    m = mo = NONE;
    l = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = 0.f;
  }
  // To maxima that are at least the present ones.
  __device__ __forceinline__ void raise(float bm, float bo) {
    l *= ex2_approx(m - bm);
    const float f = ex2_approx(mo - bo);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] *= f;
    m = bm;
    mo = bo;
  }
  __device__ __forceinline__ void add(const float (&x)[V], float f) {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = fmaf(x[j], f, v[j]);
  }
  static __device__ __forceinline__ void load(float (&x)[V], const float* row, int lane) {
#pragma unroll
    for (int j = 0; j < V; j += 4) {
      const float4 y = *reinterpret_cast<const float4*>(row + V * lane + j);
      x[j] = y.x;
      x[j + 1] = y.y;
      x[j + 2] = y.z;
      x[j + 3] = y.w;
    }
  }
  __device__ __forceinline__ void store(float* row, int lane) const {
#pragma unroll
    for (int j = 0; j < V; j += 4)
      *reinterpret_cast<float4*>(row + V * lane + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
    if (lane == 0) *reinterpret_cast<float4*>(row + D) = make_float4(m, mo, l, 0.f);
  }
  __device__ __forceinline__ void write(const Params& p, int64_t row, int lane) const {
    write_out<V>(p, row * D + V * lane, v, last_factor(m, mo, l));
  }
};

// The heads of a range from `count` of its parts, `step` apart from `from` on, by a CTA: into the
// output, or into the first of the parts.  They were written by other SMs: read past L1, some
// at a time, by half a warp for each head.
template <int D, int HEADS>
__device__ __forceinline__ void join(const Params& p, const Piece& piece, int from, int step, int count, bool out) {
  constexpr int AHEAD = 4;
  const Parts parts = piece.parts;
  const int column = threadIdx.x & 15;
#pragma unroll 1
  for (int h = threadIdx.x >> 4; h < piece.heads; h += THREADS / 16) {
    Sums<D> sums{};
    sums.start();
#pragma unroll 1
    for (int i0 = 0; i0 < count; i0 += AHEAD) {
      float x[AHEAD][Sums<D>::V];
      float4 st[AHEAD];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const int i = from + min(i0 + j, count - 1) * step;
        const float* row = part_of<D, HEADS>(p, parts.warp(i), parts.slot(i)) + h * part_stride(D);
        st[j] = __ldcg(reinterpret_cast<const float4*>(row + D));
#pragma unroll
        for (int k = 0; k < Sums<D>::V; k += 4) {
          const float4 y = __ldcg(reinterpret_cast<const float4*>(row + Sums<D>::V * column + k));
          x[j][k] = y.x;
          x[j][k + 1] = y.y;
          x[j][k + 2] = y.z;
          x[j][k + 3] = y.w;
        }
      }
      float bm = sums.m, bo = sums.mo;
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        bm = fmaxf(bm, st[j].x);  // a part that is loaded twice changes no maximum
        bo = fmaxf(bo, st[j].y);
      }
      sums.raise(bm, bo);
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        if (i0 + j < count) {
          sums.l = fmaf(st[j].z, ex2_approx(st[j].x - bm), sums.l);
          sums.add(x[j], ex2_approx(st[j].y - bo));
        }
      }
    }
    if (out) {
      sums.write(p, static_cast<int64_t>(piece.row) + h, column);
    } else {
      __syncwarp(0xFFFFu << (threadIdx.x & 16));  // all lanes of the head have read the statistics that lane 0 replaces
      sums.store(part_of<D, HEADS>(p, parts.warp(from), parts.slot(from)) + h * part_stride(D), column);
    }
  }
}

template <typename C, int D, int NT>
__global__ void __launch_bounds__(THREADS, CTAS_PER_SM) paged_attention8_kernel(Params p, KernelCtl ctl) {
  using L = Layout<D>;
  constexpr int TILE = L::TILE, SUB = TILE / 16;  // MMA tiles of 16 positions
  constexpr int KC = D / 64;   // 16-byte chunks of a K row per lane
  constexpr int MT = D / 16;   // MMA tiles of 16 dimensions
  constexpr int HEADS = 8 * NT;
  constexpr uint32_t FULL = TILE == 32 ? 0xFFFFFFFFu : 0xFFFFu;
  static_assert(HEADS * part_stride(D) * 4 <= STAGES * L::STAGE, "a warp's sums fit its ring");
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ Piece s_last[WARPS];   // of each warp's last range: the part is in its ring
  __shared__ Piece s_ended[WARPS];  // of its first, which others began: the part is in the workspace
  __shared__ __align__(16) uint32_t s_place[WARPS];
  __shared__ int s_join[2 * WARPS], s_heads[WARPS];

  pdl_begin();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, c4 = lane & 3;
  const int tiles = p.hkv * p.head_groups;
  const int me = static_cast<int>(blockIdx.x) * WARPS + warp;

  // ---- this warp's share: a sequence to a lane, 32 at a time, the next lengths under way.
  Walk run{};
  Shares shares;
  uint32_t place0;  // of this warp's range: the place of its first unit
  {
    const auto raw_of = [&](int base) { return load_raw(p.lens, p.index_bits, min(base + lane, p.batch - 1)); };
    const auto places_of = [&](int base, int context) -> uint32_t {
      return base + lane < p.batch ? units_of<D>(context) + RANGE_COST : 0;
    };
    Raw raw = raw_of(0);
    int context = 0;
    uint32_t total = 0;
#pragma unroll 1
    for (int base = 0; base < p.batch; base += 32) {
      const Raw next = raw_of(base + 32);
      context = context_of(p, raw);
      total += places_of(base, context);
      raw = next;
    }
    uint32_t upto = total;  // of the lanes up to this one
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    total = __shfl_sync(0xffffffffu, upto, 31);
    shares.set(total * tiles, gridDim.x * WARPS);
    const bool idle = me >= static_cast<int>(shares.warps);  // fewer places than warps
    const uint32_t u0 = shares.start(idle ? 0 : me);
    run.left = idle ? 0 : static_cast<int>(shares.start(me + 1) - u0);
    // The sequence that holds place u0.
    uint32_t before = 0;  // places, of one head tile, of earlier rounds
#pragma unroll 1
    for (int base = 0; base < p.batch; base += 32) {
      if (p.batch > 32) {
        context = context_of(p, raw_of(base));
        upto = places_of(base, context);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t x = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += x;
        }
      }
      const uint32_t past = __ballot_sync(0xffffffffu, (before + upto) * tiles > u0);
      if (past != 0) {
        const int at = __ffs(past) - 1;
        run.b = base + at;
        run.context = __shfl_sync(0xffffffffu, context, at);
        run.units = units_of<D>(run.context);
        const uint32_t prior = before + __shfl_sync(0xffffffffu, upto, at) - (run.units + RANGE_COST);
        const uint32_t in = u0 - prior * tiles;
        const int tile = static_cast<int>(quotient(in, run.units + RANGE_COST));
        run.c = static_cast<int>(in) - tile * (run.units + RANGE_COST);
        run.h = p.head_groups == 1 ? tile : tile / p.head_groups;
        run.hg = tile - run.h * p.head_groups;
        place0 = u0 - run.c;
        break;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
  }
  run.next = load_raw(p.lens, p.index_bits, min(run.b + 1, p.batch - 1));
  if (run.c >= run.units) {  // the share starts behind a range
    place0 += run.units + RANGE_COST;
    next_range<D>(p, run);
  }

  // ---- this warp's ring; `load` runs ahead of `run`.
  Walk load = run;
  const int ring = warp * (STAGES * L::STAGE);
  const uint32_t smem_base = smem_u32(smem);
  const int64_t slot_bytes = static_cast<int64_t>(p.hkv) * D;
  constexpr int CHUNKS = D / 16, PER = 32 / CHUNKS;  // chunks of a row, rows side by side
  const int r0 = lane / CHUNKS, ch = lane - r0 * CHUNKS;
  // Where this lane's chunk of row r0 + i * PER lies: the row's number, modulo 8, is r0 ^ (i * PER
  // % 8), so that the exchange of chunks is one XOR with a constant.
  const int lane_chunk = (D == 64 ? ch : ch ^ r0) * 16;
  const int64_t lane_bytes = r0 * slot_bytes + ch * 16, step_bytes = PER * slot_bytes, to_v = p.v - p.k;

  // The block table, 32 entries at a time: lane i holds the block of page `first` + i, -1 where
  // that is no page of the sequence or no block of the cache.  They serve the tiles before
  // `until`; the entries after them -- of this range or the next -- are loaded ahead.
  int page_block = -1, first = 0, until = 0, ahead_first = 0;
  Raw ahead{0, 0};
  auto load_pages = [&](int b, int from, int context) {
    ahead_first = from;
    const int pages = context > 0 ? block_of(p, context - 1) + 1 : 0;
    ahead = from + lane < pages ? load_raw(p.tables, p.index_bits, static_cast<int64_t>(b) * p.max_blocks + from + lane)
                                : Raw{0xFFFFFFFFu, 0xFFFFFFFFu};
  };
  auto turn_page = [&](const Walk& w) {
    first = ahead_first;
    const int pages = w.context > 0 ? block_of(p, w.context - 1) + 1 : 0;
    const int64_t value = value_of(ahead, p.index_bits);
    const bool found = value >= 0 && value < p.num_blocks;
    if (first + lane < pages && !found) atomicOr(ctl.status, RK_DEV_ERR_BAD_INDEX);
    page_block = found ? static_cast<int>(value) : -1;
    until = first + 32 < pages ? (first + 32) * p.block_size / TILE : w.units;
    if (until < w.units) {
      load_pages(w.b, block_of(p, until * TILE), w.context);
    } else {
      const bool same = w.h + 1 < p.hkv || w.hg + 1 < p.head_groups;  // sequence
      load_pages(same ? w.b : min(w.b + 1, p.batch - 1), 0, same ? w.context : context_of(p, w.next));
    }
  };
  auto issue = [&](const Walk& w, int stage) {
    const int offset = ring + stage * L::STAGE;
    const uint32_t base = smem_base + offset;
    const int t = w.c * TILE + (lane & (TILE - 1));
    const int page = block_of(p, t), off = t - page * p.block_size;
    const int held = __shfl_sync(0xffffffffu, page_block, (page - first) & 31);
    const int blk = t < w.context ? held : -1;
    const uint32_t mask = __ballot_sync(0xffffffffu, blk >= 0);
    if (lane == 0)
      *reinterpret_cast<uint32_t*>(smem + offset + L::MASK) = TILE == 32 ? mask : mask & 0xFFFFu;
    const int64_t scale_at = static_cast<int64_t>(blk < 0 ? 0 : blk) * p.hkv + w.h;
    const uint32_t scale_bytes = blk < 0 ? 0u : 4u;
    if (TILE == 32) {
      cp_async4(base + L::SCALES + lane * 4, p.ks + scale_at, scale_bytes);
      cp_async4(base + L::SCALES + 128 + lane * 4, p.vs + scale_at, scale_bytes);
    } else {
      cp_async4(base + L::SCALES + lane * 4, (lane < 16 ? p.ks : p.vs) + scale_at, scale_bytes);
    }
    // Bytes from the start of a cache to this lane's row.
    const int64_t row_bytes = (static_cast<int64_t>(blk < 0 ? 0 : blk) * p.block_size + (blk < 0 ? 0 : off)) * slot_bytes;
    const int head_bytes = w.h * D;
    if (mask == 0xFFFFFFFFu && flag_of(p.block_size) % 16 == 0) {
      // Full tiles whose 16 positions lie side by side.
#pragma unroll
      for (int sub = 0; sub < SUB; ++sub) {
        const uint8_t* from = p.k + __shfl_sync(0xffffffffu, row_bytes, 16 * sub) + head_bytes + lane_bytes;
#pragma unroll
        for (int i = 0; i < 16 / PER; ++i) {
          const int r = 16 * sub + i * PER;  // and r0
          const uint32_t chunk = base + (D == 64 ? lane_chunk : lane_chunk ^ ((i * PER % 8) * 16));
          cp_async16(chunk + r0 * D + r * D, from, 16);
          cp_async16(chunk + r0 * L::V_STRIDE + L::K_BYTES + r * L::V_STRIDE, from + to_v, 16);
          from += step_bytes;
        }
      }
    } else {
#pragma unroll 4
      for (int i = 0; i < TILE / PER; ++i) {
        const int r = i * PER + r0;
        const uint8_t* from = p.k + __shfl_sync(0xffffffffu, row_bytes, r) + head_bytes + ch * 16;
        const uint32_t bytes = (mask >> r) & 1u ? 16u : 0u;  // rows without a position: zeros
        cp_async16(base + L::k_at(r, ch), from, bytes);
        cp_async16(base + L::v_at(r, ch), from + to_v, bytes);
      }
    }
  };

  if (has_units(load)) load_pages(load.b, block_of(p, load.c * TILE), load.context);
  auto load_next = [&](int stage) {  // always a group, so that the groups count the tiles
    if (has_units(load)) {
      if (load.c >= until) turn_page(load);
      issue(load, stage);
      const int c = load.c;
      next_unit<D>(p, load);
      if (load.c <= c) until = 0;  // another range
    }
    cp_async_commit();
  };
  // Queries of a head tile: lane (g, c4) holds head g's dimensions of its K chunks.  Where the
  // registers allow it they are loaded a range ahead.
  constexpr bool QUERIES_AHEAD = NT == 1 && D <= 128;
  uint2 queries[NT][4 * KC];
  auto load_queries = [&](int b, int h, int hg) {
    const int64_t row0 = static_cast<int64_t>(b) * p.hq + h * p.group + hg * HEADS;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const bool live = nt * 8 + g < p.group - hg * HEADS;
      const uint16_t* row = static_cast<const uint16_t*>(p.q) + (row0 + nt * 8 + g) * D;
#pragma unroll
      for (int j = 0; j < 4 * KC; ++j) {
        queries[nt][j] = make_uint2(0, 0);
        if (live) queries[nt][j] = __ldg(reinterpret_cast<const uint2*>(row + k_chunk<D>(c4, j >> 2) * 16 + (j & 3) * 4));
      }
    }
  };
  if (has_units(run)) load_queries(run.b, run.h, run.hg);
  const uint32_t place_first = place0;

#pragma unroll 1
  for (int s = 0; s < STAGES; ++s) load_next(s);
  // The arrivals of the range that this warp may begin: tagged early where the last launch left
  // them at 0.
  if (lane == 0) atomicCAS(reinterpret_cast<unsigned long long*>(p.arrivals + me), 0ull, p.tag);

  // Offsets of this lane's operands within a tile: K's chunks 2 c4 (and + 1: XOR 16) of row g, V's
  // chunk g of rows 2 c4 (and + 1); rows 8 and 16 further on keep their place modulo 8.
  const int k_lane = L::k_at(g, D == 64 ? c4 : 2 * c4), v_lane = L::K_BYTES + 2 * c4 * L::V_STRIDE + (g ^ (2 * c4)) * 16;

  int stage = 0;
  Piece mine{}, ended{};
  bool alone = false;
  float* const sums = reinterpret_cast<float*>(smem + ring);  // for the last range's part: no tile is left then
  while (has_units(run)) {
    const int length = min(run.units - run.c, run.left);  // units of the range that this warp holds
    const int head0 = run.h * p.group + run.hg * HEADS;
    const int nheads = min(HEADS, p.group - run.hg * HEADS);
    const int64_t row0 = static_cast<int64_t>(run.b) * p.hq + head0;
    if (!QUERIES_AHEAD && place0 != place_first) load_queries(run.b, run.h, run.hg);
    uint32_t qf[NT][4 * KC][2];
    float factor[NT][2];
    float o[NT][MT][4];
    float m[NT][2], mo[NT][2], c[NT][2], l[NT][2];  // of heads 2 c4, 2 c4 + 1: c = 2^(m - mo)
    const int bf16 = flag_of(p.bf16);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float f[4 * KC][4];
      float amax = 0.f;
#pragma unroll
      for (int j = 0; j < 4 * KC; ++j) {
        const uint2 raw = queries[nt][j];
        const float2 a = bf16 ? Pack2<__nv_bfloat16>::to_floats(raw.x) : Pack2<__half>::to_floats(raw.x);
        const float2 b = bf16 ? Pack2<__nv_bfloat16>::to_floats(raw.y) : Pack2<__half>::to_floats(raw.y);
        f[j][0] = a.x;
        f[j][1] = a.y;
        f[j][2] = b.x;
        f[j][3] = b.y;
#pragma unroll
        for (int e = 0; e < 4; ++e) amax = fmaxf(amax, fabsf(f[j][e]));
      }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      // 2^-e with 2^e <= amax < 2^(e+1), kept where both it and its inverse are normal.
      const int e = min(max(static_cast<int>(__float_as_uint(amax) >> 23), 2), 252);
      const float down = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
      const float up = __uint_as_float(static_cast<uint32_t>(e) << 23) * p.scale_log2;
#pragma unroll
      for (int j = 0; j < 4 * KC; ++j) {
        qf[nt][j][0] = Pack2<__half>::from_floats(f[j][0] * down, f[j][1] * down);
        qf[nt][j][1] = Pack2<__half>::from_floats(f[j][2] * down, f[j][3] * down);
      }
      // Lane (g, c4) holds the scores of heads 2 c4 and 2 c4 + 1.
      factor[nt][0] = __shfl_sync(0xffffffffu, up, 8 * c4);
      factor[nt][1] = __shfl_sync(0xffffffffu, up, 8 * c4 + 4);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        m[nt][i] = mo[nt][i] = NONE;
        l[nt][i] = c[nt][i] = 0.f;
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[nt][mt][i] = 0.f;
    }

    if (QUERIES_AHEAD && run.left > run.units + RANGE_COST - run.c) {
      const bool more = run.hg + 1 < p.head_groups, same = more || run.h + 1 < p.hkv;
      load_queries(same ? run.b : run.b + 1, more ? run.h : same ? run.h + 1 : 0, more ? run.hg + 1 : 0);
    }

    for (int step = 0; step < length; ++step) {
      cp_async_wait<STAGES - 1>();
      __syncwarp();
      const uint8_t* tile = smem + ring + stage * L::STAGE;
      const uint32_t mask = at_smem<uint32_t>(tile, L::MASK);
      if (mask != 0) {
        float s[NT][SUB][4], s2[NT][SUB][4];  // two chains of products: half the latency
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int t = 0; t < SUB; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[nt][t][i] = s2[nt][t][i] = 0.f;
#pragma unroll
        for (int i = 0; i < KC; ++i) {
#pragma unroll
          for (int t = 0; t < SUB; ++t) {
            const int at = (k_lane ^ ((i & 1) * 16)) + (i >> 1) * 128 + 16 * t * D;
            const uint4 ka = at_smem<uint4>(tile, at), kb = at_smem<uint4>(tile, at + 8 * D);
            const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              uint32_t a0, a1, a2, a3;
              C::halves(wa[j], a0, a2);
              C::halves(wb[j], a1, a3);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                mma16816((j & 1) ? s2[nt][t] : s[nt][t], a0, a1, a2, a3, qf[nt][4 * i + j][0], qf[nt][4 * i + j][1]);
            }
          }
        }
        // Rows g and g + 8 of each 16: p = 2^(score - m), and the weights of V, w = p * vs * c.
        float weight[NT][SUB][4];
        float most = 0.f;
#pragma unroll
        for (int t = 0; t < SUB; ++t) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int row = 16 * t + 8 * r + g;
            const float ks = at_smem<float>(tile, L::SCALES + row * 4), vs = at_smem<float>(tile, L::SCALES + (TILE + row) * 4);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const int e = 2 * r + i;
                s[nt][t][e] += s2[nt][t][e];
                float x = fmaf(s[nt][t][e], ks * factor[nt][i], -m[nt][i]);
                if (mask != FULL && !((mask >> row) & 1u)) x = -INFINITY;
                const float pw = ex2_approx(x);
                s2[nt][t][e] = pw;
                weight[nt][t][e] = (pw * c[nt][i]) * vs;  // in this order: see below
                most = fmax3(most, pw, weight[nt][t][e]);
              }
            }
          }
        }
        if (__any_sync(0xffffffffu, most > SLACK)) {
          // The maxima are raised to what they have become, and all sums brought to them.
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float bm = NONE, bo = NONE;
#pragma unroll
              for (int t = 0; t < SUB; ++t) {
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                  const int row = 16 * t + 8 * r + g;
                  const float ks = at_smem<float>(tile, L::SCALES + row * 4), vs = at_smem<float>(tile, L::SCALES + (TILE + row) * 4);
                  const float x = (mask >> row) & 1u ? s[nt][t][2 * r + i] * (ks * factor[nt][i]) : -INFINITY;
                  bm = fmaxf(bm, x);
                  bo = fmaxf(bo, x + lg2_approx(vs));
                }
              }
#pragma unroll
              for (int x = 4; x < 32; x <<= 1) {
                bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, x));
                bo = fmaxf(bo, __shfl_xor_sync(0xffffffffu, bo, x));
              }
              bm = fmaxf(m[nt][i], bm - HEADROOM);
              bo = fmaxf(mo[nt][i], bo - HEADROOM);
              // c = 2^(m - mo) and its inverse are kept normal numbers, for ex2.approx flushes the others
              // (scales of 2^127 or 2^-126, or none but zeros), and c at most 2^110: then p * c is finite
              // up to SLACK, and 0 where p is, so that a weight is NaN only where p or vs is -- whatever
              // scales follow blocks of smaller ones or of zeros.
              bo = bm - fminf(fmaxf(bm - bo, -125.f), 110.f);
              l[nt][i] *= ex2_approx(m[nt][i] - bm);
              const float down = ex2_approx(mo[nt][i] - bo);
              c[nt][i] = ex2_approx(bm - bo);
              m[nt][i] = bm;
              mo[nt][i] = bo;
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) {
                o[nt][mt][i] *= down;
                o[nt][mt][i + 2] *= down;
              }
#pragma unroll
              for (int t = 0; t < SUB; ++t) {
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                  const int row = 16 * t + 8 * r + g;
                  const float ks = at_smem<float>(tile, L::SCALES + row * 4), vs = at_smem<float>(tile, L::SCALES + (TILE + row) * 4);
                  float x = fmaf(s[nt][t][2 * r + i], ks * factor[nt][i], -bm);
                  if (!((mask >> row) & 1u)) x = -INFINITY;
                  s2[nt][t][2 * r + i] = ex2_approx(x);
                  weight[nt][t][2 * r + i] = (s2[nt][t][2 * r + i] * c[nt][i]) * vs;
                }
              }
            }
          }
        }
        uint32_t pf[NT][SUB][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int t = 0; t < SUB; ++t) {
#pragma unroll
            for (int i = 0; i < 4; ++i) l[nt][i & 1] += s2[nt][t][i];
            pf[nt][t][0] = transpose8x8(Pack2<__half>::from_floats(weight[nt][t][0], weight[nt][t][1]));
            pf[nt][t][1] = transpose8x8(Pack2<__half>::from_floats(weight[nt][t][2], weight[nt][t][3]));
          }
        }
        // V^T: a lane's 16 (D 64: 8) bytes of positions 2 c4, 2 c4 + 1, and those + 8, byte by
        // byte side by side, are two rows of the operand.
#pragma unroll
        for (int t = 0; t < SUB; ++t) {
          if (D == 64) {
            const int row = 16 * t + 2 * c4;
            const int at = L::K_BYTES + g * 8;
            const uint2 va = at_smem<uint2>(tile, at + row * L::V_STRIDE), vb = at_smem<uint2>(tile, at + (row + 1) * L::V_STRIDE);
            const uint2 vc = at_smem<uint2>(tile, at + (row + 8) * L::V_STRIDE), vd = at_smem<uint2>(tile, at + (row + 9) * L::V_STRIDE);
            const uint32_t w0[2] = {va.x, va.y}, w1[2] = {vb.x, vb.y}, w2[2] = {vc.x, vc.y}, w3[2] = {vd.x, vd.y};
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                const uint32_t pick = x == 0 ? 0x5140u : 0x7362u;
                uint32_t a0, a1, a2, a3;
                C::halves(__byte_perm(w0[j], w1[j], pick), a0, a1);
                C::halves(__byte_perm(w2[j], w3[j], pick), a2, a3);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                  mma16816(o[nt][(2 * j + x) % MT], a0, a1, a2, a3, pf[nt][t][0], pf[nt][t][1]);
              }
            }
          } else {
#pragma unroll
            for (int h = 0; h < D / 128; ++h) {
              const int at = v_lane + h * 128 + 16 * t * D, next = (v_lane ^ 16) + h * 128 + (16 * t + 1) * D;
              const uint4 va = at_smem<uint4>(tile, at), vb = at_smem<uint4>(tile, next);
              const uint4 vc = at_smem<uint4>(tile, at + 8 * D), vd = at_smem<uint4>(tile, next + 8 * D);
              const uint32_t w0[4] = {va.x, va.y, va.z, va.w}, w1[4] = {vb.x, vb.y, vb.z, vb.w};
              const uint32_t w2[4] = {vc.x, vc.y, vc.z, vc.w}, w3[4] = {vd.x, vd.y, vd.z, vd.w};
#pragma unroll
              for (int j = 0; j < 4; ++j) {
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                  const uint32_t pick = x == 0 ? 0x5140u : 0x7362u;
                  uint32_t a0, a1, a2, a3;
                  C::halves(__byte_perm(w0[j], w1[j], pick), a0, a1);
                  C::halves(__byte_perm(w2[j], w3[j], pick), a2, a3);
#pragma unroll
                  for (int nt = 0; nt < NT; ++nt)
                    mma16816(o[nt][(8 * h + 2 * j + x) % MT], a0, a1, a2, a3, pf[nt][t][0], pf[nt][t][1]);
                }
              }
            }
          }
        }
      }
      __syncwarp();  // the tile is read
      load_next(stage);
      stage = stage + 1 == STAGES ? 0 : stage + 1;
    }

    // The end of a range.  A lane holds 16 (D 64: 8) neighbouring dimensions of two heads.
    const bool whole = length == run.units;
    const bool final = run.left <= run.units + RANGE_COST - run.c;  // no other range follows
    float* part = sums;
    if (!whole) {
      const Piece piece{place0, static_cast<int>(row0), nheads, run.c == 0, run.c + length == run.units,
                        Parts(place0, run.units, shares)};
      if (final) {
        mine = piece;
        // Whether it is the last range of a neighbour in the CTA, too.
        alone = (warp == 0 || piece.begins) &&
                (warp == WARPS - 1 || piece.ends || shares.start(me + 2) > place0 + run.units + RANGE_COST);
        if (alone) part = part_of<D, HEADS>(p, me, piece.begins);
      } else {  // part 0: it ends its range
        part = part_of<D, HEADS>(p, me, 0);
        ended = piece;
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[nt][i] += __shfl_xor_sync(0xffffffffu, l[nt][i], x);
        const int h = nt * 8 + 2 * c4 + i;
        constexpr int N = D == 64 ? 8 : 16;
        if (h < nheads) {
          float* row = part + h * part_stride(D);
          const float f = last_factor(m[nt][i], mo[nt][i], l[nt][i]);
#pragma unroll
          for (int k = 0; k < MT * 2 / N; ++k) {
            float v[N];
#pragma unroll
            for (int j = 0; j < N / 2; ++j) {
              v[2 * j] = o[nt][k * (N / 2) + j][i];
              v[2 * j + 1] = o[nt][k * (N / 2) + j][i + 2];
            }
            const int d = N * g + 128 * k;
            if (whole) {
              write_out<N>(p, (row0 + h) * D + d, v, f);
            } else {
#pragma unroll
              for (int j = 0; j < N / 4; ++j)
                reinterpret_cast<float4*>(row + d)[j] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
            }
          }
          if (!whole && g == 0) *reinterpret_cast<float4*>(row + D) = make_float4(m[nt][i], mo[nt][i], l[nt][i], 0.f);
        }
      }
    place0 += run.units + RANGE_COST;
    next_range<D>(p, run);
  }

  // ---- the warps' last ranges: neighbours that hold parts of one range join them, in the output
  // if they hold it all.
  if (lane == 0) {
    s_last[warp] = mine;
    s_ended[warp] = ended;
    s_place[warp] = mine.heads > 0 ? mine.place : ~uint32_t(warp);  // no place: unlike any other
    s_heads[warp] = alone ? 0 : mine.heads;                          // to join here
    s_join[2 * warp] = s_join[2 * warp + 1] = 0;
  }
  __syncthreads();
  const int me0 = me - warp;
  const uint4 places = *reinterpret_cast<const uint4*>(s_place);
  // Bit w: warp w's last range is that of the warp before.
  const uint32_t joined = (places.x == places.y ? 2u : 0u) | (places.y == places.z ? 4u : 0u) | (places.z == places.w ? 8u : 0u);

  // Lane 2 w + k of warp 0 stands for part k of warp w, if that stands for itself in the
  // workspace; its range's arrivals are looked at already.
  bool stands = false;
  uint64_t seen = 0;
  uint64_t* word = nullptr;
  int all = 0;
  const Piece* piece = nullptr;
  if (warp == 0 && lane < 2 * WARPS) {
    const int w = lane >> 1, k = lane & 1;
    piece = k == 0 && s_ended[w].heads > 0 ? &s_ended[w] : &s_last[w];
    const int end = __ffs(~joined & (~1u << w)) - 1;  // behind the warps that share warp w's last range
    const bool first = (joined >> w & 1u) == 0;
    stands = piece == &s_ended[w] ||
             (first && piece->heads > 0 && piece->begins == k && !(piece->begins && s_last[end - 1].ends));
    if (stands) {
      const Parts& parts = piece->parts;
      const bool grouped = parts.groups() > 1;
      const int group = parts.group_of(blockIdx.x);
      word = p.arrivals + (grouped ? gridDim.x * WARPS + parts.counter(group) : parts.begin);
      all = grouped ? parts.parts_of(group) : parts.count;
      seen = *reinterpret_cast<volatile uint64_t*>(word);
    }
  }
#pragma unroll 1
  for (int w = 0; w < WARPS;) {
    const int end = __ffs(~joined & (~1u << w)) - 1;
    const int heads = s_heads[w];
    const bool begins = s_last[w].begins, whole = begins && s_last[end - 1].ends;
#pragma unroll 1
    for (int h = threadIdx.x >> 4; h < heads; h += THREADS / 16) {
      Sums<D> sums{};
      sums.start();
      float4 st[WARPS];
#pragma unroll
      for (int i = 0; i < WARPS; ++i) {
        const float* row = reinterpret_cast<const float*>(smem + min(w + i, end - 1) * (STAGES * L::STAGE)) + h * part_stride(D);
        st[i] = *reinterpret_cast<const float4*>(row + D);
      }
      float bm = NONE, bo = NONE;
#pragma unroll
      for (int i = 0; i < WARPS; ++i) {
        bm = fmaxf(bm, st[i].x);
        bo = fmaxf(bo, st[i].y);
      }
      sums.raise(bm, bo);
#pragma unroll
      for (int i = 0; i < WARPS; ++i) {
        if (w + i < end) {
          const float* row = reinterpret_cast<const float*>(smem + (w + i) * (STAGES * L::STAGE)) + h * part_stride(D);
          float x[Sums<D>::V];
          Sums<D>::load(x, row, lane & 15);
          sums.l = fmaf(st[i].z, ex2_approx(st[i].x - bm), sums.l);
          sums.add(x, ex2_approx(st[i].y - bo));
        }
      }
      if (whole) {
        sums.write(p, static_cast<int64_t>(s_last[w].row) + h, lane & 15);
      } else {
        sums.store(part_of<D, HEADS>(p, me0 + w, begins) + h * part_stride(D), lane & 15);
      }
    }
    w = end;
  }

  // ---- ranges that several CTAs, or this one through the workspace, hold parts of.  Every CTA
  // counts its parts in; the last to come joins them all, in their order.
  if (!__syncthreads_or(stands)) return;
  bool last_here = false;
  if (stands) {
    const uint32_t same = __match_any_sync(__activemask(), piece->place);  // this CTA's parts of one range
    if (lane == __ffs(same) - 1) {
      fence_gpu();  // the CTA's parts before their count
      if (arrive(word, seen, p.tag, __popc(same), all)) {
        fence_gpu();  // the count before the parts
        s_join[lane] = 1;
        last_here = true;
      }
    }
  }
  if (!__syncthreads_or(last_here)) return;
#pragma unroll 1
  for (int i = 0; i < 2 * WARPS; ++i) {
    if (s_join[i] == 0) continue;
    const Piece& whose = (i & 1) == 0 && s_ended[i >> 1].heads > 0 ? s_ended[i >> 1] : s_last[i >> 1];
    const Parts& parts = whose.parts;
    const int groups = parts.groups(), group = parts.group_of(blockIdx.x);
    bool out = groups == 1;
    int from = out ? 0 : group * JOIN_CTAS, step = 1, count = out ? parts.count : parts.parts_of(group);
    for (;;) {
      join<D, HEADS>(p, whose, from, step, count, out);
      if (out) break;
      __syncthreads();
      bool last = false;
      if (threadIdx.x == 0) {
        fence_gpu();  // the joined part before its count
        uint64_t* const counted = p.arrivals + parts.begin;
        last = arrive(counted, *reinterpret_cast<volatile uint64_t*>(counted), p.tag, 1, groups);
        if (last) fence_gpu();
      }
      if (!__syncthreads_or(last)) break;
      out = true;
      from = 0;
      step = JOIN_CTAS;
      count = groups;
    }
  }
}

// A number that no workspace holds by chance: a count of the launches, spread over 64 bits by
// an odd factor (2^64 over the golden ratio), from a start that differs from process to
// process.
uint64_t next_tag() {
  static const uint64_t start = static_cast<uint64_t>(std::chrono::steady_clock::now().time_since_epoch().count()) << 20;
  static std::atomic<uint64_t> launches{1};
  const uint64_t x = (start + launches.fetch_add(1, std::memory_order_relaxed)) * 0x9E3779B97F4A7C15ull & ~uint64_t{0xFFFF};
  return x != 0 ? x : 0x10000;
}

struct Plan {
  int nt, head_groups;
};

Plan plan(int64_t hq, int64_t hkv, int64_t head_dim) {
  const int64_t group = hq / hkv;
  // Two column tiles of 8 heads where a KV head has more than 8 query heads: K and V are
  // read and unpacked once for up to 16.  At head_dim 256 the accumulators of one fill the
  // registers.
  const int nt = group > 8 && head_dim < 256 ? 2 : 1;
  return {nt, static_cast<int>((group + 8 * nt - 1) / (8 * nt))};
}

template <typename C, int D, int NT>
rk_status launch(const Params& p, const KernelCtl& ctl, cudaStream_t s) {
  constexpr size_t SMEM = Layout<D>::RING;
  auto kernel = paged_attention8_kernel<C, D, NT>;
  static std::atomic<int> residents[64];  // CTAs per SM, by device; 0: not asked yet
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_status(e);
  int resident = residents[dev & 63].load(std::memory_order_relaxed);
  if (resident == 0) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(SMEM));
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, kernel, THREADS, SMEM);
    if (e != cudaSuccess) return cuda_status(e);
    if (resident < 1) return RK_ERR_UNSUPPORTED;
    residents[dev & 63].store(resident, std::memory_order_relaxed);
  }
  const int64_t ranges = static_cast<int64_t>(p.batch) * p.hkv * p.head_groups;
  const int64_t per_range = (static_cast<int64_t>(p.max_blocks) * p.block_size + unit_of(D) - 1) / unit_of(D);
  // Places are counted in 32 bits, and a warp's share stays below 2^21 of them (see quotient).
  if (ranges > INT32_MAX / (per_range + RANGE_COST)) {
    note_error("the block tables hold too many positions for one call");
    return RK_ERR_UNSUPPORTED;
  }
  const int64_t ctas =
      ctas_of(ranges, per_range, static_cast<int64_t>(device_sm_count()) * (resident < CTAS_PER_SM ? resident : CTAS_PER_SM));
  e = launch_kernel(kernel, dim3(static_cast<unsigned>(ctas)), dim3(THREADS), SMEM, s, 0, p, ctl);
  note_launch("paged_attention8_kernel");
  return cuda_status(e);
}

template <typename C>
rk_status launch_d(const Params& p, int64_t head_dim, int nt, const KernelCtl& ctl, cudaStream_t s) {
  switch (head_dim) {
    case 64: return nt == 1 ? launch<C, 64, 1>(p, ctl, s) : launch<C, 64, 2>(p, ctl, s);
    case 128: return nt == 1 ? launch<C, 128, 1>(p, ctl, s) : launch<C, 128, 2>(p, ctl, s);
    default: return launch<C, 256, 1>(p, ctl, s);
  }
}

}  // namespace pa8

size_t paged_attention8_workspace_bytes(int64_t hq, int64_t hkv, int64_t head_dim) {
  const pa8::Plan pl = pa8::plan(hq, hkv, head_dim);
  const size_t warps = static_cast<size_t>(device_sm_count()) * pa8::CTAS_PER_SM * pa8::WARPS;
  return warps * (2 * sizeof(uint64_t) + 2 * 8 * pl.nt * pa8::part_stride(static_cast<int>(head_dim)) * sizeof(float));
}

rk_status paged_attention8_launch(const PagedAttention8Args& a, void* workspace, size_t workspace_bytes, cudaStream_t s) {
  if (workspace == nullptr || !aligned16(workspace) || workspace_bytes < paged_attention8_workspace_bytes(a.hq, a.hkv, a.head_dim))
    return RK_ERR_INVALID_ARGUMENT;
  LaunchCtl lc;
  const rk_status st = launch_ctl(&lc);
  if (st != RK_OK) return st;
  const KernelCtl ctl{lc.status, lc.timeout_ns, 0};
  const pa8::Plan pl = pa8::plan(a.hq, a.hkv, a.head_dim);
  pa8::Params p{};
  p.q = a.query;
  p.k = static_cast<const uint8_t*>(a.key_cache);
  p.v = static_cast<const uint8_t*>(a.value_cache);
  p.ks = a.key_scales;
  p.vs = a.value_scales;
  p.tables = a.block_tables;
  p.lens = a.context_lengths;
  p.out = a.out;
  p.arrivals = static_cast<uint64_t*>(workspace);
  p.part = reinterpret_cast<float*>(p.arrivals + 2 * device_sm_count() * pa8::CTAS_PER_SM * pa8::WARPS);
  p.tag = pa8::next_tag();
  p.batch = static_cast<int>(a.batch);
  p.hq = static_cast<int>(a.hq);
  p.hkv = static_cast<int>(a.hkv);
  p.group = static_cast<int>(a.hq / a.hkv);
  p.head_groups = pl.head_groups;
  p.num_blocks = static_cast<int>(a.num_blocks);
  p.block_size = static_cast<int>(a.block_size);
  p.max_blocks = static_cast<int>(a.max_blocks);
  int bits = 0;  // of block_size, rounded up to a power of two
  while ((int64_t{1} << bits) < a.block_size) ++bits;
  p.block_shift = 31 + bits;
  p.block_multiplier = static_cast<uint32_t>((uint64_t{1} << p.block_shift) / static_cast<uint64_t>(a.block_size) + 1);
  p.index_bits = a.index_bits;
  p.bf16 = a.dt == RK_DTYPE_BF16;
  p.scale_log2 = a.scale * 1.44269504088896340736f;
  return a.cache == RK_CACHE_E4M3 ? pa8::launch_d<E4m3>(p, a.head_dim, pl.nt, ctl, s)
                                  : pa8::launch_d<Int8>(p, a.head_dim, pl.nt, ctl, s);
}

}  // namespace rk
