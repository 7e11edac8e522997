// paged_slots.cu -- block tables and slot maps of one step, from the requests' lengths.
//
// Request b holds h_b tokens and gets n_b more.  Its blocks grow from ceil(h_b / block_size)
// to ceil((h_b + n_b) / block_size); the new ones come from the list of free blocks in request
// order, so request b takes the list from the exclusive sum of those differences on, and
// its tokens take the output from the exclusive sum of n on.  Both sums are a scan over the
// requests.
//
// One launch, no workspace: every CTA repeats the whole scan (a few KB from L2) and then
// handles its own stretch of tokens and its own share of the table rows, so no CTA waits for
// another.  New entries are taken from the free list by both the CTA that writes them and
// those that need them; entries of blocks that a request had are only read.
//
// What bounds it: launch and latency -- lengths, scan, table or free list, slot -- at all sizes of
// use (a token each of 256 requests 3.3 us on the device, of 896 requests 5.1; 64k tokens of 61
// requests 4.4 us for 1 MB written).
#include <cuda_runtime.h>

#include "rk_device.cuh"
#include "rk_internal.h"

namespace rk {
namespace {

constexpr int FEW = 256, MANY = 1024;  // threads of a CTA, by the number of requests

template <typename Index>
struct SlotParams {
  Index* tables;
  const Index* has;
  const Index* gets;
  const Index* free_blocks;
  int64_t* slots;
  Index* positions;
  Index* lengths;
  Index* used;
  int64_t batch, max_blocks, block_size, free_count, tokens;
  int64_t most_block;  // whose slots fit 64 bits
};

// Inclusive sums over the lanes of two values.
__device__ __forceinline__ void scan_lanes2(int64_t& a, int64_t& b, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o);
    if (lane >= o) {
      a += x;
      b += y;
    }
  }
}

// Inclusive sums over the CTA of two values, in thread order.
template <int WARPS>
__device__ __forceinline__ void scan2(int64_t& a, int64_t& b, int64_t (*warp_sums)[2]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  scan_lanes2(a, b, lane);
  if (lane == 31) {
    warp_sums[warp][0] = a;
    warp_sums[warp][1] = b;
  }
  __syncthreads();
  if constexpr (WARPS <= 8) {
    for (int w = 0; w < warp; ++w) {
      a += warp_sums[w][0];
      b += warp_sums[w][1];
    }
  } else {
    static_assert(WARPS == 32, "a lane for each warp");
    int64_t x = warp_sums[lane][0], y = warp_sums[lane][1];
    scan_lanes2(x, y, lane);
    x = __shfl_sync(0xffffffffu, x, (warp + 31) & 31);
    y = __shfl_sync(0xffffffffu, y, (warp + 31) & 31);
    if (warp > 0) {
      a += x;
      b += y;
    }
  }
}

template <typename Index, int THREADS>
__global__ void __launch_bounds__(THREADS) paged_slots_kernel(SlotParams<Index> p, KernelCtl ctl) {
  __shared__ int64_t warp_sums[THREADS / 32][2];
  __shared__ int64_t s_end[THREADS];    // tokens of the requests up to and with this one
  __shared__ int64_t s_has[THREADS];    // tokens that the request had
  __shared__ int64_t s_first[THREADS];  // its first entry of the free list
  __shared__ int64_t s_old[THREADS], s_want[THREADS];  // its blocks before and after
  pdl_begin();
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * (2 * THREADS);
  const int64_t t1 = min(t0 + 2 * THREADS, p.tokens);
  const int64_t room = p.max_blocks * p.block_size;
  // Dividends below 2^32: lengths and block_size are below 2^31, and so is the number of tokens.
  const auto blocks_of = [&](int64_t n) -> int64_t { return static_cast<uint32_t>(n) / static_cast<uint32_t>(p.block_size); };
  int64_t token_base = 0, free_base = 0;  // sums over the requests of earlier rounds
  bool bad = false;
  for (int64_t base = 0; base < p.batch; base += THREADS) {
    const int64_t r = base + threadIdx.x;
    int64_t has = 0, gets = 0;
    if (r < p.batch) {
      has = static_cast<int64_t>(p.has[r]);
      gets = static_cast<int64_t>(p.gets[r]);
      bad = bad || has < 0 || gets < 0 || has > room || gets > room || has + gets > room;
      has = min(max(has, int64_t{0}), room);
      gets = max(gets, int64_t{0});
    }
    const int64_t end = min(has + min(gets, room), room);
    // A larger count overruns the token buffer by itself: said here, for the sum no longer shows it.
    bad = bad || gets > p.tokens;
    gets = min(gets, p.tokens);
    const int64_t old = blocks_of(has + p.block_size - 1);
    const int64_t want = blocks_of(end + p.block_size - 1);
    int64_t tokens = gets, blocks = want - old;
    scan2<THREADS / 32>(tokens, blocks, warp_sums);
    const int64_t first = free_base + blocks - (want - old);
    s_end[threadIdx.x] = token_base + tokens;
    s_has[threadIdx.x] = has;
    s_first[threadIdx.x] = first;
    s_old[threadIdx.x] = old;
    s_want[threadIdx.x] = want;
    __syncthreads();
    const int n = static_cast<int>(min(static_cast<int64_t>(THREADS), p.batch - base));
    if (blockIdx.x == 0 && r < p.batch) p.lengths[r] = static_cast<Index>(end);
    // Table rows of this CTA's share of the requests.  Most steps give a request one block or
    // none: a thread writes that of its own; the further ones a warp writes together.
    const auto entry = [&](int64_t request, int64_t j, int64_t at) {
      if (at >= p.free_count) bad = true;
      p.tables[request * p.max_blocks + j] = at < p.free_count ? p.free_blocks[at] : static_cast<Index>(-1);
    };
    const bool mine = r < p.batch && threadIdx.x % gridDim.x == blockIdx.x;
    if (mine && want > old) entry(r, old, first);
    for (uint32_t more = __ballot_sync(0xffffffffu, mine && want > old + 1); more != 0; more &= more - 1) {
      const int i = (threadIdx.x & ~31) + __ffs(more) - 1;
      for (int64_t j = s_old[i] + 1 + (threadIdx.x & 31); j < s_want[i]; j += 32) entry(base + i, j, s_first[i] + j - s_old[i]);
    }
    // Tokens of these requests that fall into this CTA's stretch.
    const int64_t from = max(t0, token_base), to = min(t1, s_end[n - 1]);
    for (int64_t t = from + threadIdx.x; t < to; t += THREADS) {
      int lo = 0, hi = n - 1;  // the first request whose end is behind t
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (s_end[mid] > t) hi = mid;
        else lo = mid + 1;
      }
      const int64_t before = lo == 0 ? token_base : s_end[lo - 1];
      const int64_t position = s_has[lo] + t - before;
      const int64_t j = blocks_of(position);
      int64_t block = -1;
      if (j < s_old[lo]) {
        block = static_cast<int64_t>(p.tables[(base + lo) * p.max_blocks + j]);
      } else if (j < s_want[lo]) {
        const int64_t at = s_first[lo] + j - s_old[lo];
        if (at < p.free_count) block = static_cast<int64_t>(p.free_blocks[at]);
      }
      if (block > p.most_block) block = -1;
      bad = bad || block < 0;
      p.slots[t] = block < 0 ? -1 : block * p.block_size + position - j * p.block_size;
      p.positions[t] = static_cast<Index>(position);
    }
    token_base = s_end[THREADS - 1];  // threads past the batch add nothing
    free_base = s_first[THREADS - 1] + s_want[THREADS - 1] - s_old[THREADS - 1];
    __syncthreads();  // the arrays are written again
  }
  for (int64_t t = max(t0, token_base) + threadIdx.x; t < t1; t += THREADS) {
    p.slots[t] = -1;
    p.positions[t] = 0;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    p.used[0] = static_cast<Index>(free_base);
    bad = bad || token_base > p.tokens;
  }
  if (bad) atomicOr(ctl.status, RK_DEV_ERR_BAD_INDEX);
}

template <typename Index, int THREADS>
cudaError_t launch(const SlotParams<Index>& p, const KernelCtl& ctl, cudaStream_t s) {
  const int64_t ctas = (p.tokens + 2 * THREADS - 1) / (2 * THREADS);
  return launch_kernel(paged_slots_kernel<Index, THREADS>, dim3(static_cast<unsigned>(ctas < 1 ? 1 : ctas)), dim3(THREADS), 0,
                       s, 0, p, ctl);
}

template <typename Index>
cudaError_t launch(const PagedSlotsArgs& a, const KernelCtl& ctl, cudaStream_t s) {
  SlotParams<Index> p{};
  p.tables = static_cast<Index*>(a.block_tables);
  p.has = static_cast<const Index*>(a.context_lengths);
  p.gets = static_cast<const Index*>(a.new_lengths);
  p.free_blocks = static_cast<const Index*>(a.free_blocks);
  p.slots = a.slot_mapping;
  p.positions = static_cast<Index*>(a.positions);
  p.lengths = static_cast<Index*>(a.lengths_out);
  p.used = static_cast<Index*>(a.blocks_used);
  p.batch = a.batch;
  p.max_blocks = a.max_blocks;
  p.block_size = a.block_size;
  p.free_count = a.free_count;
  p.tokens = a.tokens;
  p.most_block = (INT64_MAX - (a.block_size - 1)) / a.block_size;
  // One round of the scan for up to 1024 requests.
  return a.batch > FEW ? launch<Index, MANY>(p, ctl, s) : launch<Index, FEW>(p, ctl, s);
}

}  // namespace

rk_status paged_slots_launch(const PagedSlotsArgs& a, cudaStream_t s) {
  LaunchCtl lc;
  const rk_status st = launch_ctl(&lc);
  if (st != RK_OK) return st;
  const KernelCtl ctl{lc.status, lc.timeout_ns, 0};
  const cudaError_t e = a.index_bits == 32 ? launch<int32_t>(a, ctl, s) : launch<int64_t>(a, ctl, s);
  note_launch("paged_slots_kernel");
  return cuda_status(e);
}

}  // namespace rk
