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
constexpr int TILE = 16;             // positions of a warp's tile
constexpr int UNIT = WARPS * TILE;   // positions of a unit
constexpr int STAGES = 3;
constexpr int MAX_CTAS_PER_SM = 4;   // sizes the workspace
constexpr float SLACK = 8.0f;        // a running maximum is raised when it is passed by 2^SLACK

// Shared-memory layout.  A row of K or V is D bytes; the pads make the 128-bit (V at D 64:
// 64-bit) reads of the MMA operands free of bank conflicts.
template <int D>
struct Layout {
  static constexpr int K_STRIDE = D == 64 ? 64 : D + 16;
  static constexpr int V_STRIDE = D + 16;
  static constexpr int K_BYTES = TILE * K_STRIDE;
  static constexpr int V_BYTES = TILE * V_STRIDE;
  static constexpr int SCALES = K_BYTES + V_BYTES;       // 16 of K, 16 of V
  static constexpr int MASK = SCALES + 2 * TILE * 4;     // which rows hold a position
  static constexpr int STAGE = MASK + 16;
  static constexpr int RING = WARPS * STAGES * STAGE;
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
  float* part;  // [CTA][2][heads of a tile][D + 3 (rounded up)]: see part_floats
  int batch, hq, hkv, group, head_groups, tile_heads;
  int num_blocks, block_size, block_shift, max_blocks;
  int index_bits, bf16;
  float scale_log2;
};

__host__ __device__ constexpr int part_stride(int head_dim) { return head_dim + 4; }  // sum, then m, mo, l

__device__ __forceinline__ int64_t index_at(const void* p, int bits, int64_t i) {
  return bits == 32 ? static_cast<int64_t>(__ldg(static_cast<const int32_t*>(p) + i))
                    : static_cast<int64_t>(__ldg(static_cast<const long long*>(p) + i));
}

__device__ __forceinline__ int context_of(const Params& p, int b) {
  const int64_t n = index_at(p.lens, p.index_bits, b);
  const int64_t room = static_cast<int64_t>(p.max_blocks) * p.block_size;  // below 2^31
  return static_cast<int>(n < 0 ? 0 : (n > room ? room : n));
}

// Units of one (sequence, head tile); an empty sequence has one, which writes its NaN.
__device__ __forceinline__ int units_of(int context) { return context <= UNIT ? 1 : (context + UNIT - 1) / UNIT; }

// Sum of v over the CTA, in every thread.
__device__ __forceinline__ int64_t cta_sum(int64_t v, int64_t* scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) total += scratch[w];
  return total;
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

__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a) : "memory");
  return r;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 r;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(a) : "memory");
  return r;
}
__device__ __forceinline__ float lds_f32(uint32_t a) {
  float r;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(r) : "r"(a) : "memory");
  return r;
}
__device__ __forceinline__ uint32_t lds_u32(uint32_t a) {
  uint32_t r;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r) : "r"(a) : "memory");
  return r;
}
__device__ __forceinline__ void sts_u32(uint32_t a, uint32_t v) {
  asm volatile("st.shared.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
}

// D[16 x 8] += A[16 x 16] B[16 x 8], f16 operands, fp32 accumulators.
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Transposes an 8 x 8 matrix of 16-bit values held across the warp.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float lg2_approx(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The chunk (16 bytes of a row) that lane column c reads as its i-th of K.
template <int D>
__device__ __forceinline__ int k_chunk(int c, int i) {
  return D == 64 ? c : 2 * c + (i & 1) + 8 * (i >> 1);
}

// Which dimension an accumulator stands for: MMA tile mt, lane row g, half e.
template <int D>
__device__ __forceinline__ int o_dim(int mt, int g, int e) {
  return D == 64 ? 8 * g + 2 * mt + e : (mt >> 3) * 128 + 16 * g + 2 * (mt & 7) + e;
}

// A walk over units: sequence b, head tile h, unit c of its `units`.
struct Walk {
  int b, h, c, units, context;
};

__device__ __forceinline__ void walk_on(const Params& p, Walk& w, int tiles) {
  if (++w.c < w.units) return;
  w.c = 0;
  if (++w.h < tiles) return;
  w.h = 0;
  if (++w.b < p.batch) {
    w.context = context_of(p, w.b);
    w.units = units_of(w.context);
  }
}

// The CTA that holds unit u when CTA w holds [floor(w * total / ctas), ...).
__device__ __forceinline__ int64_t owner_of(int64_t u, int64_t total, int64_t ctas) {
  return ((u + 1) * ctas - 1) / total;
}

template <typename C, int D, int NT>
__global__ void __launch_bounds__(THREADS) paged_attention8_kernel(Params p, KernelCtl ctl) {
  using L = Layout<D>;
  constexpr int KC = D / 64;   // 16-byte chunks of a K row per lane
  constexpr int MT = D / 16;   // MMA tiles of 16 dimensions
  constexpr int HEADS = 8 * NT;
  constexpr int O_STRIDE = D + 4;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int64_t s_scratch[WARPS];
  __shared__ int s_at[3];
  __shared__ float s_stats[WARPS][HEADS][3];
  float* s_out = reinterpret_cast<float*>(smem + L::RING);  // [warp][head][O_STRIDE]

  pdl_begin();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, c4 = lane & 3;
  const int tiles = p.hkv * p.head_groups;

  // ---- this CTA's units
  int64_t total = 0;
  for (int base = 0; base < p.batch; base += THREADS) {
    const int b = base + threadIdx.x;
    total += cta_sum(b < p.batch ? units_of(context_of(p, b)) : 0, s_scratch);
  }
  total *= tiles;
  const int64_t ctas = min(static_cast<int64_t>(gridDim.x), total);  // each has a unit at least
  if (blockIdx.x >= ctas) return;
  const int64_t u0 = blockIdx.x * total / ctas, u1 = (blockIdx.x + 1) * total / ctas;
  {
    // The sequence that holds unit u0: sums over 32 sequences at a time, by every warp alike.
    int64_t before = 0;  // units (of one head tile) of earlier sequences
    const int64_t want = u0;
    for (int base = 0; base < p.batch; base += 32) {
      const int b = base + lane;
      const int mine = b < p.batch ? units_of(context_of(p, b)) : 0;
      int64_t upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, (before + upto) * tiles > want);
      if (past != 0) {
        const int at = __ffs(past) - 1;
        const int64_t prior = __shfl_sync(0xffffffffu, before + upto - mine, at);
        const int units = __shfl_sync(0xffffffffu, mine, at);
        if (threadIdx.x == 0) {
          const int64_t in = want - prior * tiles;
          s_at[0] = base + at;
          s_at[1] = static_cast<int>(in / units);
          s_at[2] = static_cast<int>(in % units);
        }
        break;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
  }
  __syncthreads();
  Walk run{s_at[0], s_at[1], s_at[2], 0, context_of(p, s_at[0])};
  run.units = units_of(run.context);
  Walk load = run;

  const uint32_t ring = smem_u32(smem) + warp * (STAGES * L::STAGE);
  const int64_t slot_bytes = static_cast<int64_t>(p.hkv) * D;

  // Block of the row that this lane (lane % 16) looks up for the tile of `w`; -1: no position.
  auto look_up = [&](const Walk& w) -> int {
    const int t = w.c * UNIT + warp * TILE + (lane & 15);
    if (t >= w.context) return -1;
    const int j = p.block_shift >= 0 ? t >> p.block_shift : t / p.block_size;
    const int64_t blk = index_at(p.tables, p.index_bits, static_cast<int64_t>(w.b) * p.max_blocks + j);
    if (blk < 0 || blk >= p.num_blocks) {
      if (lane < 16) atomicOr(ctl.status, RK_DEV_ERR_BAD_INDEX);
      return -1;
    }
    return static_cast<int>(blk);
  };
  auto issue = [&](const Walk& w, int blk, int stage) {
    const uint32_t base = ring + stage * L::STAGE;
    const int kvh = w.h / p.head_groups;
    const int t = w.c * UNIT + warp * TILE + (lane & 15);
    const int off = p.block_shift >= 0 ? t & (p.block_size - 1) : t % p.block_size;
    const int64_t slot = blk < 0 ? 0 : static_cast<int64_t>(blk) * p.block_size + off;
    const uint32_t mask = __ballot_sync(0xffffffffu, blk >= 0) & 0xFFFFu;
    if (lane == 0) sts_u32(base + L::MASK, mask);
    const int64_t sc = static_cast<int64_t>(blk < 0 ? 0 : blk) * p.hkv + kvh;
    cp_async4(base + L::SCALES + lane * 4, (lane < 16 ? p.ks : p.vs) + sc, blk < 0 ? 0u : 4u);
    constexpr int CHUNKS = D / 16, PER = 32 / CHUNKS;  // chunks of a row, rows side by side
    const int r0 = lane / CHUNKS, ch = lane - r0 * CHUNKS;
#pragma unroll
    for (int i = 0; i < TILE / PER; ++i) {
      const int r = r0 + i * PER;
      const int64_t row_slot = __shfl_sync(0xffffffffu, slot, r);
      const uint32_t bytes = (mask >> r) & 1u ? 16u : 0u;
      const int64_t from = row_slot * slot_bytes + kvh * D + ch * 16;
      cp_async16(base + r * L::K_STRIDE + ch * 16, p.k + from, bytes);
      cp_async16(base + L::K_BYTES + r * L::V_STRIDE + ch * 16, p.v + from, bytes);
    }
  };

  int64_t loaded = u0;
  int blk = look_up(load);
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) {
    if (loaded < u1) {
      issue(load, blk, s);
      walk_on(p, load, tiles);
      if (++loaded < u1) blk = look_up(load);
    }
    cp_async_commit();
  }

  uint32_t qf[NT][4 * KC][2];
  float factor[NT][2];
  float o[NT][MT][4];
  float m[NT][2], mo[NT][2], l[NT][2];
  int64_t range0 = u0;  // first unit of the current range that this CTA holds
  bool fresh = true;
  int stage = 0;

  for (int64_t u = u0; u < u1; ++u) {
    const int kvh = run.h / p.head_groups, hg = run.h - kvh * p.head_groups;
    const int head0 = kvh * p.group + hg * HEADS;
    const int nheads = min(HEADS, p.group - hg * HEADS);
    if (fresh) {
      // Queries of the head tile: lane (g, c4) holds head g's dimensions of its K chunks.
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const bool live = nt * 8 + g < nheads;
        const int64_t row = (static_cast<int64_t>(run.b) * p.hq + head0 + nt * 8 + g) * D;
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
          m[nt][i] = mo[nt][i] = -INFINITY;
          l[nt][i] = 0.f;
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[nt][mt][i] = 0.f;
      }
      fresh = false;
    }

    cp_async_wait<STAGES - 2>();
    __syncwarp();
    {
      const int next = stage + STAGES - 1 >= STAGES ? stage - 1 : stage + STAGES - 1;
      if (loaded < u1) {
        issue(load, blk, next);
        walk_on(p, load, tiles);
        if (++loaded < u1) blk = look_up(load);
      }
      cp_async_commit();
    }
    const uint32_t base = ring + stage * L::STAGE;
    stage = stage + 1 == STAGES ? 0 : stage + 1;
    const uint32_t mask = lds_u32(base + L::MASK);
    if (mask != 0) {
      float s[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[nt][i] = 0.f;
#pragma unroll
      for (int i = 0; i < KC; ++i) {
        const uint32_t at = base + k_chunk<D>(c4, i) * 16;
        const uint4 ka = lds128(at + g * L::K_STRIDE), kb = lds128(at + (g + 8) * L::K_STRIDE);
        const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t a0, a1, a2, a3;
          C::halves(wa[j], a0, a2);
          C::halves(wb[j], a1, a3);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma16816(s[nt], a0, a1, a2, a3, qf[nt][4 * i + j][0], qf[nt][4 * i + j][1]);
        }
      }
      // Rows g and g + 8 of the tile.
      const float ks0 = lds_f32(base + L::SCALES + g * 4), ks1 = lds_f32(base + L::SCALES + (g + 8) * 4);
      const float lv0 = lg2_approx(lds_f32(base + L::SCALES + 64 + g * 4));
      const float lv1 = lg2_approx(lds_f32(base + L::SCALES + 64 + (g + 8) * 4));
      const bool in0 = (mask >> g) & 1u, in1 = (mask >> (g + 8)) & 1u;
      bool raise = false;
      float w[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool in = i < 2 ? in0 : in1;
          s[nt][i] = in ? s[nt][i] * ((i < 2 ? ks0 : ks1) * factor[nt][i & 1]) : -INFINITY;
          w[nt][i] = in ? s[nt][i] + (i < 2 ? lv0 : lv1) : -INFINITY;
          raise = raise || s[nt][i] > m[nt][i & 1] + SLACK || w[nt][i] > mo[nt][i & 1] + SLACK;
        }
      }
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float a = fmax3(m[nt][i], s[nt][i], s[nt][i + 2]), b = fmax3(mo[nt][i], w[nt][i], w[nt][i + 2]);
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) {
              a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, x));
              b = fmaxf(b, __shfl_xor_sync(0xffffffffu, b, x));
            }
            // A maximum of -inf has nothing behind it to scale.
            const float down_l = m[nt][i] == -INFINITY ? 0.f : ex2_approx(m[nt][i] - a);
            const float down_o = mo[nt][i] == -INFINITY ? 0.f : ex2_approx(mo[nt][i] - b);
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
      uint32_t pf[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // Against a maximum of -inf every weight is 0 (2^-inf), not 2^(inf - inf).
          const float ms = m[nt][i & 1] == -INFINITY ? 0.f : m[nt][i & 1];
          const float mw = mo[nt][i & 1] == -INFINITY ? 0.f : mo[nt][i & 1];
          l[nt][i & 1] += ex2_approx(s[nt][i] - ms);
          e[i] = ex2_approx(w[nt][i] - mw);
        }
        pf[nt][0] = transpose8x8(Pack2<__half>::from_floats(e[0], e[1]));
        pf[nt][1] = transpose8x8(Pack2<__half>::from_floats(e[2], e[3]));
      }
      // V^T: a lane's 16 (D 64: 8) bytes of positions 2 c4, 2 c4 + 1, and those + 8, byte by
      // byte side by side, are two rows of the operand.
      const uint32_t vb = base + L::K_BYTES;
      if (D == 64) {
        const uint2 va = lds64(vb + (2 * c4) * L::V_STRIDE + g * 8), vc = lds64(vb + (2 * c4 + 1) * L::V_STRIDE + g * 8);
        const uint2 vd = lds64(vb + (2 * c4 + 8) * L::V_STRIDE + g * 8), ve = lds64(vb + (2 * c4 + 9) * L::V_STRIDE + g * 8);
        const uint32_t w0[2] = {va.x, va.y}, w1[2] = {vc.x, vc.y}, w2[2] = {vd.x, vd.y}, w3[2] = {ve.x, ve.y};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const uint32_t pick = x == 0 ? 0x5140u : 0x7362u;
            uint32_t a0, a1, a2, a3;
            C::halves(__byte_perm(w0[j], w1[j], pick), a0, a1);
            C::halves(__byte_perm(w2[j], w3[j], pick), a2, a3);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816(o[nt][2 * j + x], a0, a1, a2, a3, pf[nt][0], pf[nt][1]);
          }
        }
      } else {
#pragma unroll
        for (int h = 0; h < D / 128; ++h) {
          const uint32_t at = vb + g * 16 + h * 128;
          const uint4 va = lds128(at + (2 * c4) * L::V_STRIDE), vc = lds128(at + (2 * c4 + 1) * L::V_STRIDE);
          const uint4 vd = lds128(at + (2 * c4 + 8) * L::V_STRIDE), ve = lds128(at + (2 * c4 + 9) * L::V_STRIDE);
          const uint32_t w0[4] = {va.x, va.y, va.z, va.w}, w1[4] = {vc.x, vc.y, vc.z, vc.w};
          const uint32_t w2[4] = {vd.x, vd.y, vd.z, vd.w}, w3[4] = {ve.x, ve.y, ve.z, ve.w};
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
                mma16816(o[nt][8 * h + 2 * j + x], a0, a1, a2, a3, pf[nt][0], pf[nt][1]);
            }
          }
        }
      }
    }
    __syncwarp();  // the stage is read before it is filled again

    if (run.c + 1 == run.units || u + 1 == u1) {
      // End of a range: join the warps.  Accumulator (mt, g, e) of a head lies at
      // [16 mt + 2 g + e], which keeps the stores free of bank conflicts.
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) l[nt][i] += __shfl_xor_sync(0xffffffffu, l[nt][i], x);
          if (g == 0) {
            float* st = s_stats[warp][nt * 8 + 2 * c4 + i];
            st[0] = m[nt][i];
            st[1] = mo[nt][i];
            st[2] = l[nt][i];
          }
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
            *reinterpret_cast<float2*>(s_out + (warp * HEADS + nt * 8 + 2 * c4 + i) * O_STRIDE + 16 * mt + 2 * g) =
                make_float2(o[nt][mt][i], o[nt][mt][i + 2]);
        }
      __syncthreads();
      const bool whole = run.c + 1 == run.units && u + 1 - range0 == run.units;
      const int slot = range0 == u0 ? 0 : 1;
      for (int idx = threadIdx.x; idx < nheads * (D / 2); idx += THREADS) {
        const int h = idx / (D / 2), at = (idx - h * (D / 2)) * 2;
        float am = -INFINITY, ao = -INFINITY;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
          am = fmaxf(am, s_stats[w][h][0]);
          ao = fmaxf(ao, s_stats[w][h][1]);
        }
        float sum = 0.f, x = 0.f, y = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
          const float wm = s_stats[w][h][0], wo = s_stats[w][h][1];
          // A warp without a maximum has sums of 0, or NaN from NaN scores, which stay.
          sum += s_stats[w][h][2] * (wm == -INFINITY ? 1.f : ex2_approx(wm - am));
          const float f = wo == -INFINITY ? 1.f : ex2_approx(wo - ao);
          const float2 v = *reinterpret_cast<const float2*>(s_out + (w * HEADS + h) * O_STRIDE + at);
          x = fmaf(v.x, f, x);
          y = fmaf(v.y, f, y);
        }
        if (whole) {
          const float f = (ao == -INFINITY || am == -INFINITY ? 1.f : ex2_approx(ao - am)) / sum;
          const int d = o_dim<D>(at >> 4, (at & 15) >> 1, 0);
          const int64_t row = (static_cast<int64_t>(run.b) * p.hq + head0 + h) * D + d;
          static_cast<uint32_t*>(p.out)[row >> 1] =
              p.bf16 ? Pack2<__nv_bfloat16>::from_floats(x * f, y * f) : Pack2<__half>::from_floats(x * f, y * f);
        } else {
          float* part = p.part + ((static_cast<int64_t>(blockIdx.x) * 2 + slot) * HEADS + h) * part_stride(D);
          *reinterpret_cast<float2*>(part + at) = make_float2(x, y);
          if (at == 0) {
            part[D] = am;
            part[D + 1] = ao;
            part[D + 2] = sum;
          }
        }
      }
      __syncthreads();
      range0 = u + 1;
      fresh = true;
    }
    walk_on(p, run, tiles);
  }
}

// Joins the parts of the ranges that several CTAs shared.  One CTA per (sequence, head tile).
template <int D>
__global__ void __launch_bounds__(THREADS) paged_attention8_join_kernel(Params p, int64_t grid) {
  __shared__ int64_t s_scratch[WARPS];
  pdl_begin();
  const int tiles = p.hkv * p.head_groups;
  const int b = blockIdx.x / tiles, tile = blockIdx.x - b * tiles;
  int64_t total = 0, before = 0;
  for (int base = 0; base < p.batch; base += THREADS) {
    const int i = base + threadIdx.x;
    const int64_t units = i < p.batch ? units_of(context_of(p, i)) : 0;
    total += units;
    if (i < b) before += units;
  }
  total = cta_sum(total, s_scratch) * tiles;
  before = cta_sum(before, s_scratch) * tiles;
  const int64_t ctas = min(grid, total);
  const int64_t units = units_of(context_of(p, b));
  const int64_t first = before + tile * units;
  const int64_t w0 = owner_of(first, total, ctas), w1 = owner_of(first + units - 1, total, ctas);
  if (w0 == w1) return;  // written by its one CTA
  const int slot0 = w0 * total / ctas == first ? 0 : 1;
  const int kvh = tile / p.head_groups, hg = tile - kvh * p.head_groups;
  const int nheads = min(p.tile_heads, p.group - hg * p.tile_heads);
  const int64_t head0 = static_cast<int64_t>(b) * p.hq + kvh * p.group + hg * p.tile_heads;
  const int64_t step = static_cast<int64_t>(2) * p.tile_heads * part_stride(D);  // from CTA to CTA
  for (int idx = threadIdx.x; idx < nheads * (D / 2); idx += THREADS) {
    const int h = idx / (D / 2), at = (idx - h * (D / 2)) * 2;
    const float* head = p.part + w0 * step + (static_cast<int64_t>(slot0) * p.tile_heads + h) * part_stride(D);
    const float* rest = p.part + (w0 + 1) * step + static_cast<int64_t>(h) * part_stride(D);
    const int n = static_cast<int>(w1 - w0);
    float am = head[D], ao = head[D + 1];
    for (int i = 0; i < n; ++i) {
      am = fmaxf(am, rest[i * step + D]);
      ao = fmaxf(ao, rest[i * step + D + 1]);
    }
    float sum = 0.f, x = 0.f, y = 0.f;
    for (int i = -1; i < n; ++i) {
      const float* part = i < 0 ? head : rest + i * step;
      const float wm = part[D], wo = part[D + 1];
      sum += part[D + 2] * (wm == -INFINITY ? 1.f : ex2_approx(wm - am));
      const float f = wo == -INFINITY ? 1.f : ex2_approx(wo - ao);
      const float2 v = *reinterpret_cast<const float2*>(part + at);
      x = fmaf(v.x, f, x);
      y = fmaf(v.y, f, y);
    }
    const float f = (ao == -INFINITY || am == -INFINITY ? 1.f : ex2_approx(ao - am)) / sum;
    const int d = o_dim<D>(at >> 4, (at & 15) >> 1, 0);
    static_cast<uint32_t*>(p.out)[((head0 + h) * D + d) >> 1] =
        p.bf16 ? Pack2<__nv_bfloat16>::from_floats(x * f, y * f) : Pack2<__half>::from_floats(x * f, y * f);
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
  constexpr size_t SMEM = Layout<D>::RING + static_cast<size_t>(WARPS) * 8 * NT * (D + 4) * sizeof(float);
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
  const int64_t per_range = (static_cast<int64_t>(p.max_blocks) * p.block_size + UNIT - 1) / UNIT;
  int64_t ctas = static_cast<int64_t>(device_sm_count()) * (resident < MAX_CTAS_PER_SM ? resident : MAX_CTAS_PER_SM);
  if (ranges <= ctas && ranges * per_range < ctas) ctas = ranges * per_range;
  e = launch_kernel(kernel, dim3(static_cast<unsigned>(ctas)), dim3(THREADS), SMEM, s, 0, p, ctl);
  note_launch("paged_attention8_kernel");
  if (e == cudaSuccess && per_range > 1) {
    e = launch_kernel(paged_attention8_join_kernel<D>, dim3(static_cast<unsigned>(ranges)), dim3(THREADS), 0, s, 0, p, ctas);
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
  return static_cast<size_t>(device_sm_count()) * pa8::MAX_CTAS_PER_SM * 2 * 8 * pl.nt *
         pa8::part_stride(static_cast<int>(head_dim)) * sizeof(float);
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
  p.part = static_cast<float*>(workspace);
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
