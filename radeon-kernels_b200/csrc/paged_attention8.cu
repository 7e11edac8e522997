// paged_attention8.cu -- decode attention over a paged K/V cache of 8 bits (E4m3 or Int8) with
// one fp32 scale per block and head, one query token per sequence:
//
//   s_t = scale * ks(t) * (q . k_t),  p_t = exp(s_t - max s),
//   out = sum_t p_t * vs(t) * v_t / sum_t p_t,        t < context_lengths[b]
//
// with k_t, v_t the stored 8-bit values of position t and ks, vs the scales of its block and
// head.  Query head h reads KV head h / (query_heads / kv_heads).
//
// Work: the positions of every sequence are cut into units of 64, and the units of all
// sequences and KV heads, laid end to end, are dealt out evenly: CTA w of W takes the units
// [w * total / W, (w + 1) * total / W).  So one long sequence among short ones, or few
// sequences, load every SM alike, whatever the width of the block table.  A CTA writes the
// (sequence, KV head) ranges that it covers whole; of a range that it shares it leaves the
// unnormalised sum and its statistics in the workspace, and a second kernel joins the parts in
// CTA order (no atomics: results do not depend on timing).
//
// A CTA is 4 warps; a unit is a tile of 16 positions for each, and the warps meet only at
// the end of a range.  Each warp feeds itself through its own ring of shared memory
// (cp.async, STAGES tiles of K and V with their scales), which runs on across the ends of
// ranges.  The matrix products are mma.sync m16n8k16 on f16 operands:
//   S^T[16 positions, 8 heads] = K[16, D] Q^T      O^T[16 dims, 8 heads] += V^T[16 dims, 16] P^T
// so a KV head's query heads fill the 8 columns, and each 8-bit value is unpacked once, in
// registers: both E4m3 and Int8 values are f16 numbers, exactly.  The order of a head's
// dimensions within the products is free; it is chosen such that a lane's operands are 16
// consecutive bytes of a row.  The 8-query-head tile of a unit needs 16 MMAs per 4 KB of
// cache (D 128), a few per cent of the tensor pipe, so the products bound nothing; tcgen05
// would add a round trip through tensor memory and need unpacked operands in shared memory.
//
// Numbers: queries are brought to f16 by a power of two per head (exact unless a component is
// 2^-14 of the head's largest: then it keeps 2^-25 of that).  Scores, maxima, sums and
// accumulators are fp32.  The weights of V carry its scales, w_t = p_t * vs(t), and are
// rounded to f16 for the product, relative to a maximum of their own (of s_t + log2 vs(t)), so
// that the rounding is 2^-12 of the largest terms however the scales differ from block to block.
// The running maxima are raised only when a value passes them by 2^8; in between p and w
// may reach 2^8, far inside the range of both types.
//
// What bounds it: the bytes of K and V.
#include <cuda_runtime.h>

#include <atomic>

#include "rk_cache8.cuh"
#include "rk_device.cuh"
#include "rk_internal.h"

namespace rk {
namespace pa8 {

constexpr int WARPS = 4;
constexpr int THREADS = WARPS * 32;
constexpr int STAGES = 3;
constexpr int MAX_CTAS_PER_SM = 4;   // sizes the workspace
constexpr int RANGE_COST = 2;        // what starting and ending a range costs, in units
constexpr float SLACK = 8.0f;        // a running maximum is raised when it is passed by 2^SLACK
constexpr float NONE = -3.402823466e38f;  // a maximum before any score: finite, so that -inf - NONE = -inf

// Positions of a unit, which is one tile of a warp.
__host__ __device__ constexpr int unit_of(int head_dim) { return head_dim == 256 ? 16 : 32; }

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

// A part in the workspace: per head the unnormalised sum, then m, mo and l.
__host__ __device__ constexpr int part_stride(int head_dim) { return head_dim + 4; }

// What a warp leaves in the workspace about its parts.  Part 1 of a warp begins a range that
// later CTAs end (row, heads and last describe it); part 0 continues one that an earlier CTA
// began.  Parts of one CTA's warps are joined before, into the first of them.
struct Shared {
  int row;    // of the range that part 1 begins: its first row of the output,
  int heads;  // its rows (0: there is no part 1),
  int last;   // and the warp that ends it
  int kept;   // whether part 0 stands for itself
};

struct Params {
  const void* q;
  const uint8_t* k;
  const uint8_t* v;
  const float* ks;
  const float* vs;
  const void* tables;
  const void* lens;
  void* out;
  float* part;     // [warp][2][heads of a tile][part_stride]
  Shared* shared;  // [warp]
  int batch, hq, hkv, group, head_groups, tile_heads;
  int num_blocks, block_size, block_shift, max_blocks;
  int index_bits, bf16;
  float scale_log2;
};

// An index as loaded: nothing waits for the load until value_of.
struct Raw {
  uint32_t lo, hi;
};
__device__ __forceinline__ Raw load_raw(const void* p, int bits, int64_t i) {
  Raw r{0, 0};
  if (bits == 32) {
    r.lo = __ldg(static_cast<const uint32_t*>(p) + i);
  } else {
    const uint2 v = __ldg(static_cast<const uint2*>(p) + i);
    r.lo = v.x;
    r.hi = v.y;
  }
  return r;
}
__device__ __forceinline__ int64_t value_of(Raw r, int bits) {
  return bits == 32 ? static_cast<int64_t>(static_cast<int32_t>(r.lo))
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

// Units of one (sequence, head tile); an empty sequence has one, which writes its NaN.
template <int D>
__device__ __forceinline__ int units_of(int context) {
  return context <= unit_of(D) ? 1 : (context + unit_of(D) - 1) / unit_of(D);
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

// A warp's last range, of which it holds a part in shared memory.
struct Last {
  int64_t place;  // of the range's first unit; -1: the warp has no such part
  int row, heads, last;
  int begins, ends;  // whether the part holds the range's first and last unit
};

// The chunk (16 bytes of a row) that lane column c reads as its i-th of K.
template <int D>
__device__ __forceinline__ int k_chunk(int c, int i) {
  return D == 64 ? c : 2 * c + (i & 1) + 8 * (i >> 1);
}

// A place in the row of all units: sequence b, head tile h, unit c of its `units`; `left` units
// of this warp's share from here on.  Every range is followed by RANGE_COST places that hold
// no unit, so that shares with many short ranges hold fewer units.  The next sequence's
// length is loaded a sequence ahead.
struct Walk {
  int b, h, c, units, left, context;
  Raw next;
};

// To the first unit of the next (sequence, head tile).  Past the last sequence the walk holds
// some valid length and is not used (left <= 0).
template <int D>
__device__ __forceinline__ void next_range(const Params& p, Walk& w, int tiles) {
  w.left -= w.units + RANGE_COST - w.c;
  w.c = 0;
  if (++w.h < tiles) return;
  w.h = 0;
  ++w.b;
  w.context = context_of(p, w.next);
  w.units = units_of<D>(w.context);
  w.next = load_raw(p.lens, p.index_bits, min(w.b + 1, p.batch - 1));
}

template <int D>
__device__ __forceinline__ void next_unit(const Params& p, Walk& w, int tiles) {
  ++w.c;
  --w.left;
  if (w.c == w.units) next_range<D>(p, w, tiles);
}

// N (a multiple of 4) neighbouring elements of an output row times f.
template <int N>
__device__ __forceinline__ void write_out(const Params& p, int64_t element, const float* v, float f) {
  uint32_t w[N / 2];
#pragma unroll
  for (int i = 0; i < N / 2; ++i)
    w[i] = p.bf16 ? Pack2<__nv_bfloat16>::from_floats(v[2 * i] * f, v[2 * i + 1] * f)
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

template <int V>
__device__ __forceinline__ void write_lane(const Params& p, int64_t element, const float* v, float f) {
  if constexpr (V % 4 == 0) {
    write_out<V>(p, element, v, f);
  } else {
    static_cast<uint32_t*>(p.out)[element >> 1] = p.bf16 ? Pack2<__nv_bfloat16>::from_floats(v[0] * f, v[1] * f)
                                                         : Pack2<__half>::from_floats(v[0] * f, v[1] * f);
  }
}

// What brings the sums to the output: the weights' sum, and from the one maximum to the
// other.  Without a position it is 1 / 0, and the sums 0.
__device__ __forceinline__ float last_factor(float m, float mo, float l) { return ex2_approx(mo - m) / l; }

// First place of warp w's share.  The division is 32 bits wide where it can be.
__device__ __forceinline__ int64_t share_of(uint32_t w, int64_t total, int64_t warps) {
  const uint64_t product = static_cast<uint64_t>(w) * static_cast<uint64_t>(total);
  if (product >> 32 == 0) return static_cast<uint32_t>(product) / static_cast<uint32_t>(warps);
  return static_cast<int64_t>(product / static_cast<uint64_t>(warps));
}

// The warp whose share holds place u: the largest w with floor(w * total / warps) <= u.
__device__ __forceinline__ int owner_of(int64_t u, int64_t total, int64_t warps) {
  return static_cast<int>(((u + 1) * warps - 1) / total);
}

template <typename C, int D, int NT>
__global__ void __launch_bounds__(THREADS, 2) paged_attention8_kernel(Params p, KernelCtl ctl) {
  using L = Layout<D>;
  constexpr int TILE = L::TILE, SUB = TILE / 16;  // MMA tiles of 16 positions
  constexpr int KC = D / 64;   // 16-byte chunks of a K row per lane
  constexpr int MT = D / 16;   // MMA tiles of 16 dimensions
  constexpr int HEADS = 8 * NT;
  static_assert(HEADS * part_stride(D) * 4 <= STAGES * L::STAGE, "a warp's sums fit its ring");
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ Last s_last[WARPS];

  pdl_begin();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, c4 = lane & 3;
  const int tiles = p.hkv * p.head_groups;
  const int me = static_cast<int>(blockIdx.x) * WARPS + warp;
  Shared shared{0, 0, 0, 0};

  // ---- this warp's share, found 128 sequences at a time (four neighbours to a lane, so that
  // the loads of a round are in flight together).
  Walk run{};
  int64_t place0, total = 0, warps;  // of this warp's range: the place of its first unit
  {
    constexpr int ROUND = 128;
    int unit[4];
    auto load_round = [&](int base) -> int {  // the units of a lane's four sequences
      Raw raw[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) raw[i] = load_raw(p.lens, p.index_bits, min(base + 4 * lane + i, p.batch - 1));
      int sum = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        unit[i] = base + 4 * lane + i < p.batch ? units_of<D>(context_of(p, raw[i])) + RANGE_COST : 0;
        sum += unit[i];
      }
      return sum;
    };
    int mine = 0;
    for (int base = 0; base < p.batch; base += ROUND) {
      mine = load_round(base);
      int64_t sum = mine;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      total += sum;
    }
    total *= tiles;
    warps = min(static_cast<int64_t>(gridDim.x) * WARPS, total);
    const bool idle = me >= warps;  // fewer places than warps
    const int64_t u0 = share_of(idle ? 0 : me, total, warps);
    run.left = idle ? 0 : static_cast<int>(share_of(me + 1, total, warps) - u0);
    // The sequence that holds place u0.
    int64_t before = 0;  // places, of one head tile, of earlier rounds
    for (int base = 0; base < p.batch; base += ROUND) {
      if (p.batch > ROUND) mine = load_round(base);
      int64_t upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, (before + upto) * tiles > u0);
      if (past != 0) {
        const int at = __ffs(past) - 1;
        int64_t prior = __shfl_sync(0xffffffffu, before + upto - mine, at);
        int b = base + 4 * at, units = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int n = __shfl_sync(0xffffffffu, unit[i], at);
          if (units == 0) {
            if ((prior + n) * tiles > u0) {
              units = n;
            } else {
              prior += n;
              ++b;
            }
          }
        }
        const uint32_t in = static_cast<uint32_t>(u0 - prior * tiles);  // below tiles * units, which the host checked
        run.b = b;
        run.h = static_cast<int>(in / static_cast<uint32_t>(units));
        run.c = static_cast<int>(in - static_cast<uint32_t>(run.h) * units);
        run.units = units - RANGE_COST;
        place0 = u0 - run.c;
        break;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
  }
  run.context = context_of(p, run.b);
  run.next = load_raw(p.lens, p.index_bits, min(run.b + 1, p.batch - 1));

  if (run.c >= run.units) {  // the share starts behind a range
    place0 += run.units + RANGE_COST;
    next_range<D>(p, run, tiles);
  }

  // ---- this warp's ring; `load` runs ahead of `run`.
  Walk load = run;
  const int ring = warp * (STAGES * L::STAGE);
  const uint32_t smem_base = smem_u32(smem);
  const int64_t slot_bytes = static_cast<int64_t>(p.hkv) * D;
  constexpr int CHUNKS = D / 16, PER = 32 / CHUNKS;  // chunks of a row, rows side by side
  const int r0 = lane / CHUNKS, ch = lane - r0 * CHUNKS;
  const int64_t lane_bytes = r0 * slot_bytes + ch * 16, step_bytes = PER * slot_bytes, to_v = p.v - p.k;

  // The table entry of the row that this lane (lane % TILE) looks up for the tile of `w`.
  auto look_up = [&](const Walk& w) -> Raw {
    const int t = w.c * TILE + (lane & (TILE - 1));
    const int j = p.block_shift >= 0 ? t >> p.block_shift : t / p.block_size;
    return t < w.context ? load_raw(p.tables, p.index_bits, static_cast<int64_t>(w.b) * p.max_blocks + j) : Raw{0, 0};
  };
  auto issue = [&](const Walk& w, Raw entry, int stage) {
    const int offset = ring + stage * L::STAGE;
    const uint32_t base = smem_base + offset;
    const int kvh = p.head_groups == 1 ? w.h : w.h / p.head_groups;
    const int t = w.c * TILE + (lane & (TILE - 1));
    const int off = p.block_shift >= 0 ? t & (p.block_size - 1) : t % p.block_size;
    const int64_t value = value_of(entry, p.index_bits);
    const bool in = t < w.context, found = value >= 0 && value < p.num_blocks;
    if (in && !found && lane < TILE) atomicOr(ctl.status, RK_DEV_ERR_BAD_INDEX);
    const int blk = in && found ? static_cast<int>(value) : -1;
    const uint32_t mask = __ballot_sync(0xffffffffu, blk >= 0);
    if (lane == 0)
      *reinterpret_cast<uint32_t*>(smem + offset + L::MASK) = TILE == 32 ? mask : mask & 0xFFFFu;
    const int64_t scale_at = static_cast<int64_t>(blk < 0 ? 0 : blk) * p.hkv + kvh;
    const uint32_t scale_bytes = blk < 0 ? 0u : 4u;
    if (TILE == 32) {
      cp_async4(base + L::SCALES + lane * 4, p.ks + scale_at, scale_bytes);
      cp_async4(base + L::SCALES + 128 + lane * 4, p.vs + scale_at, scale_bytes);
    } else {
      cp_async4(base + L::SCALES + lane * 4, (lane < 16 ? p.ks : p.vs) + scale_at, scale_bytes);
    }
    // Bytes from the start of a cache to this lane's row.
    const int64_t row_bytes = (static_cast<int64_t>(blk < 0 ? 0 : blk) * p.block_size + (blk < 0 ? 0 : off)) * slot_bytes;
    const int head_bytes = kvh * D;
    if (mask == 0xFFFFFFFFu && p.block_size % 16 == 0) {
      // Full tiles whose 16 positions lie side by side.
#pragma unroll
      for (int sub = 0; sub < SUB; ++sub) {
        const uint8_t* from = p.k + __shfl_sync(0xffffffffu, row_bytes, 16 * sub) + head_bytes + lane_bytes;
#pragma unroll
        for (int i = 0; i < 16 / PER; ++i) {
          const int r = 16 * sub + i * PER + r0;
          cp_async16(base + L::k_at(r, ch), from, 16);
          cp_async16(base + L::v_at(r, ch), from + to_v, 16);
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

  Raw entry{0, 0};
  if (load.left > 0) entry = look_up(load);
  auto load_next = [&](int stage) {  // always a group, so that the groups count the tiles
    if (load.left > 0) {
      issue(load, entry, stage);
      next_unit<D>(p, load, tiles);
      if (load.left > 0) entry = look_up(load);
    }
    cp_async_commit();
  };
#pragma unroll
  for (int s = 0; s < STAGES; ++s) load_next(s);

  int stage = 0;
  Last mine{-1, 0, 0, 0, 0, 0};
  float* const sums = reinterpret_cast<float*>(smem + ring);  // for the last range's part: no tile is left then
  while (run.left > 0) {
    const int length = min(run.units - run.c, run.left);  // units of the range that this warp holds
    const int kvh = p.head_groups == 1 ? run.h : run.h / p.head_groups, hg = run.h - kvh * p.head_groups;
    const int head0 = kvh * p.group + hg * HEADS;
    const int nheads = min(HEADS, p.group - hg * HEADS);
    const int64_t row0 = static_cast<int64_t>(run.b) * p.hq + head0;
    uint32_t qf[NT][4 * KC][2];
      float factor[NT][2];
      float o[NT][MT][4];
      float m[NT][2], mo[NT][2], l[NT][2];
      // Queries of the head tile: lane (g, c4) holds head g's dimensions of its K chunks.
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const bool live = nt * 8 + g < nheads;
        const int64_t row = (row0 + nt * 8 + g) * D;
        float f[4 * KC][4];
        float amax = 0.f;
#pragma unroll
        for (int j = 0; j < 4 * KC; ++j) {
          uint2 raw = make_uint2(0, 0);
          const int64_t at = row + k_chunk<D>(c4, j >> 2) * 16 + (j & 3) * 4;
          if (live) raw = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p.q) + at));
          const float2 a = p.bf16 ? Pack2<__nv_bfloat16>::to_floats(raw.x) : Pack2<__half>::to_floats(raw.x);
          const float2 b = p.bf16 ? Pack2<__nv_bfloat16>::to_floats(raw.y) : Pack2<__half>::to_floats(raw.y);
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
          l[nt][i] = 0.f;
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[nt][mt][i] = 0.f;
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
              const uint4 ka = at_smem<uint4>(tile, L::k_at(16 * t + g, k_chunk<D>(c4, i)));
              const uint4 kb = at_smem<uint4>(tile, L::k_at(16 * t + g + 8, k_chunk<D>(c4, i)));
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
          // Rows g and g + 8 of each 16.
          bool raise = false;
          float w[NT][SUB][4];
#pragma unroll
          for (int t = 0; t < SUB; ++t) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const int row = 16 * t + 8 * r + g;
              const float ks = at_smem<float>(tile, L::SCALES + row * 4);
              const float lv = lg2_approx(at_smem<float>(tile, L::SCALES + (TILE + row) * 4));
              const bool in = (mask >> row) & 1u;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                  float& x = s[nt][t][2 * r + i];
                  x = in ? (x + s2[nt][t][2 * r + i]) * (ks * factor[nt][i]) : -INFINITY;
                  w[nt][t][2 * r + i] = in ? x + lv : -INFINITY;
                  raise = raise || x > m[nt][i] + SLACK || w[nt][t][2 * r + i] > mo[nt][i] + SLACK;
                }
              }
            }
          }
          if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                float a = m[nt][i], b = mo[nt][i];
#pragma unroll
                for (int t = 0; t < SUB; ++t) {
                  a = fmax3(a, s[nt][t][i], s[nt][t][i + 2]);
                  b = fmax3(b, w[nt][t][i], w[nt][t][i + 2]);
                }
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) {
                  a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, x));
                  b = fmaxf(b, __shfl_xor_sync(0xffffffffu, b, x));
                }
                const float down_l = ex2_approx(m[nt][i] - a), down_o = ex2_approx(mo[nt][i] - b);
                m[nt][i] = a;
                mo[nt][i] = b;
                l[nt][i] *= down_l;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                  o[nt][mt][i] *= down_o;
                  o[nt][mt][i + 2] *= down_o;
                }
              }
            }
          }
          uint32_t pf[NT][SUB][2];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int t = 0; t < SUB; ++t) {
              float e[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                l[nt][i & 1] += ex2_approx(s[nt][t][i] - m[nt][i & 1]);
                e[i] = ex2_approx(w[nt][t][i] - mo[nt][i & 1]);
              }
              pf[nt][t][0] = transpose8x8(Pack2<__half>::from_floats(e[0], e[1]));
              pf[nt][t][1] = transpose8x8(Pack2<__half>::from_floats(e[2], e[3]));
            }
          }
          // V^T: a lane's 16 (D 64: 8) bytes of positions 2 c4, 2 c4 + 1, and those + 8, byte by
          // byte side by side, are two rows of the operand.
#pragma unroll
          for (int t = 0; t < SUB; ++t) {
            const int row = 16 * t + 2 * c4;
            if (D == 64) {
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
                const uint4 va = at_smem<uint4>(tile, L::v_at(row, g + 8 * h)), vb = at_smem<uint4>(tile, L::v_at(row + 1, g + 8 * h));
                const uint4 vc = at_smem<uint4>(tile, L::v_at(row + 8, g + 8 * h)), vd = at_smem<uint4>(tile, L::v_at(row + 9, g + 8 * h));
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
        if (final) {
          mine.place = place0;
          mine.row = static_cast<int>(row0);
          mine.heads = nheads;
          mine.last = owner_of(place0 + run.units - 1, total, warps);
          mine.begins = run.c == 0;
          mine.ends = run.c + length == run.units;
        } else {
          part = p.part + static_cast<int64_t>(me) * 2 * HEADS * part_stride(D);  // part 0: it ends its range
          shared.kept = 1;
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
    next_range<D>(p, run, tiles);
  }

  // ---- the warps' last ranges: neighbours that hold parts of one range join them.
  if (lane == 0) s_last[warp] = mine;
  __syncthreads();
  for (int w = 0; w < WARPS;) {
    const Last first = s_last[w];
    int end = w + 1;  // behind the warps that share it
    if (first.place < 0) {
      ++w;
      continue;
    }
    while (end < WARPS && s_last[end].place == first.place) ++end;
    const bool whole = first.begins && s_last[end - 1].ends;
    for (int h = warp; h < first.heads; h += WARPS) {
      constexpr int V = D / 32;  // neighbouring dimensions of a lane
      float m = NONE, mo = NONE, l = 0.f, v[V];
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = 0.f;
      const auto row = [&](int i) {
        return reinterpret_cast<const float*>(smem + i * (STAGES * L::STAGE)) + h * part_stride(D);
      };
      for (int i = w; i < end; ++i) {
        m = fmaxf(m, row(i)[D]);
        mo = fmaxf(mo, row(i)[D + 1]);
      }
      for (int i = w; i < end; ++i) {
        l = fmaf(row(i)[D + 2], ex2_approx(row(i)[D] - m), l);
        const float f = ex2_approx(row(i)[D + 1] - mo);
#pragma unroll
        for (int j = 0; j < V; j += 2) {
          const float2 x = *reinterpret_cast<const float2*>(row(i) + V * lane + j);
          v[j] = fmaf(x.x, f, v[j]);
          v[j + 1] = fmaf(x.y, f, v[j + 1]);
        }
      }
      if (whole) {
        write_lane<V>(p, (static_cast<int64_t>(first.row) + h) * D + V * lane, v, last_factor(m, mo, l));
      } else {
        float* part = p.part + ((static_cast<int64_t>(me - warp + w) * 2 + (first.begins ? 1 : 0)) * HEADS + h) * part_stride(D);
#pragma unroll
        for (int j = 0; j < V; j += 2) *reinterpret_cast<float2*>(part + V * lane + j) = make_float2(v[j], v[j + 1]);
        if (lane == 0) *reinterpret_cast<float4*>(part + D) = make_float4(m, mo, l, 0.f);
      }
    }
    if (warp == w && !whole) {
      if (first.begins) {
        shared.row = first.row;
        shared.heads = first.heads;
        shared.last = first.last;
      } else {
        shared.kept = 1;
      }
    }
    w = end;
  }
  if (lane == 0) p.shared[me] = shared;
}

// Joins the parts of the ranges that several CTAs of the attention shared.  One CTA for those
// that CTA blockIdx.x began, a warp for each head; the parts in order of their CTAs.
constexpr int JOIN_THREADS = 256;

template <int D>
__global__ void __launch_bounds__(JOIN_THREADS, 4) paged_attention8_join_kernel(Params p) {
  constexpr int V = D / 32;              // neighbouring dimensions of a lane
  constexpr int AHEAD = D == 256 ? 4 : 8;  // parts whose sums are loaded together
  pdl_begin();
  const int lane = threadIdx.x & 31;
  const int4* const all = reinterpret_cast<const int4*>(p.shared);
  const int64_t part_floats = static_cast<int64_t>(p.tile_heads) * part_stride(D);
  int4 info[WARPS];
#pragma unroll
  for (int w = 0; w < WARPS; ++w) info[w] = __ldg(all + blockIdx.x * WARPS + w);
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    const Shared shared{info[w].x, info[w].y, info[w].z, info[w].w};
    if (shared.heads == 0) continue;
    // The part that begins the range, one of each later CTA's first warp, and one of the
    // warp that ends it where that is no CTA's first and did not join its neighbours.
    const int ctas = shared.last / WARPS - static_cast<int>(blockIdx.x);
    const int n = 1 + ctas + (shared.last % WARPS != 0 && __ldg(all + shared.last).w != 0 ? 1 : 0);
    const float* const first = p.part + (static_cast<int64_t>(blockIdx.x) * WARPS + w) * 2 * part_floats + part_floats;
    for (int h = threadIdx.x >> 5; h < shared.heads; h += JOIN_THREADS / 32) {
      const auto row = [&](int i) -> const float* {
        if (i == 0) return first + h * part_stride(D);
        const int64_t from = i <= ctas ? (static_cast<int64_t>(blockIdx.x) + i) * WARPS : shared.last;
        return p.part + from * 2 * part_floats + h * part_stride(D);
      };
      float m = NONE, mo = NONE, l = 0.f, v[V];
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = 0.f;
      for (int i0 = 0; i0 < n; i0 += 32) {  // a lane for the statistics of each of 32 parts
        const int count = min(32, n - i0);
        float4 st = make_float4(NONE, NONE, 0.f, 0.f);
        if (lane < count) st = *reinterpret_cast<const float4*>(row(i0 + lane) + D);
        float bm = fmaxf(m, st.x), bo = fmaxf(mo, st.y);
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) {
          bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, x));
          bo = fmaxf(bo, __shfl_xor_sync(0xffffffffu, bo, x));
        }
        float dl = st.z * ex2_approx(st.x - bm);
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) dl += __shfl_xor_sync(0xffffffffu, dl, x);
        l = fmaf(l, ex2_approx(m - bm), dl);
        const float fo = ex2_approx(mo - bo), fi = ex2_approx(st.y - bo);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] *= fo;
        m = bm;
        mo = bo;
        for (int j0 = 0; j0 < count; j0 += AHEAD) {
          float x[AHEAD][V];
#pragma unroll
          for (int j = 0; j < AHEAD; ++j) {
            const float* from = row(i0 + min(j0 + j, count - 1)) + V * lane;
#pragma unroll
            for (int k = 0; k < V; k += 2) {
              const float2 y = *reinterpret_cast<const float2*>(from + k);
              x[j][k] = y.x;
              x[j][k + 1] = y.y;
            }
          }
#pragma unroll
          for (int j = 0; j < AHEAD; ++j) {
            const float f = __shfl_sync(0xffffffffu, fi, (j0 + j) & 31);
            if (j0 + j < count) {
#pragma unroll
              for (int k = 0; k < V; ++k) v[k] = fmaf(x[j][k], f, v[k]);
            }
          }
        }
      }
      write_lane<V>(p, (static_cast<int64_t>(shared.row) + h) * D + V * lane, v, last_factor(m, mo, l));
    }
  }
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
  // A warp counts its places, and a sequence's over its heads, in 32 bits.
  if (static_cast<int64_t>(p.hkv) * p.head_groups > INT32_MAX / (per_range + RANGE_COST) ||
      ranges > (int64_t{1} << 38) / (per_range + RANGE_COST))
    return RK_ERR_UNSUPPORTED;
  int64_t ctas = static_cast<int64_t>(device_sm_count()) * (resident < MAX_CTAS_PER_SM ? resident : MAX_CTAS_PER_SM);
  // Not more warps than units; RANGE_COST places of a range hold none.
  if (ranges <= ctas * WARPS && ranges * (per_range + RANGE_COST) < ctas * WARPS)
    ctas = (ranges * (per_range + RANGE_COST) + WARPS - 1) / WARPS;
  e = launch_kernel(kernel, dim3(static_cast<unsigned>(ctas)), dim3(THREADS), SMEM, s, 0, p, ctl);
  note_launch("paged_attention8_kernel");
  if (e == cudaSuccess && per_range > 1) {
    e = launch_kernel(paged_attention8_join_kernel<D>, dim3(static_cast<unsigned>(ctas)), dim3(JOIN_THREADS), 0, s, 0, p);
    note_launch("paged_attention8_join_kernel");
  }
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
  const size_t warps = static_cast<size_t>(device_sm_count()) * pa8::MAX_CTAS_PER_SM * pa8::WARPS;
  return warps * (sizeof(pa8::Shared) + 2 * 8 * pl.nt * pa8::part_stride(static_cast<int>(head_dim)) * sizeof(float));
}

rk_status paged_attention8_launch(const PagedAttention8Args& a, void* workspace, size_t workspace_bytes, cudaStream_t s) {
  if (workspace == nullptr || workspace_bytes < paged_attention8_workspace_bytes(a.hq, a.hkv, a.head_dim))
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
  p.shared = static_cast<pa8::Shared*>(workspace);
  p.part = reinterpret_cast<float*>(p.shared + device_sm_count() * pa8::MAX_CTAS_PER_SM * pa8::WARPS);
  p.batch = static_cast<int>(a.batch);
  p.hq = static_cast<int>(a.hq);
  p.hkv = static_cast<int>(a.hkv);
  p.group = static_cast<int>(a.hq / a.hkv);
  p.head_groups = pl.head_groups;
  p.tile_heads = 8 * pl.nt;
  p.num_blocks = static_cast<int>(a.num_blocks);
  p.block_size = static_cast<int>(a.block_size);
  p.max_blocks = static_cast<int>(a.max_blocks);
  p.block_shift = -1;
  for (int i = 0; i < 31; ++i)
    if ((int64_t{1} << i) == a.block_size) p.block_shift = i;
  p.index_bits = a.index_bits;
  p.bf16 = a.dt == RK_DTYPE_BF16;
  p.scale_log2 = a.scale * 1.44269504088896340736f;
  return a.cache == RK_CACHE_E4M3 ? pa8::launch_d<E4m3>(p, a.head_dim, pl.nt, ctl, s)
                                  : pa8::launch_d<Int8>(p, a.head_dim, pl.nt, ctl, s);
}

}  // namespace rk
