// Tables of one serving step, built on the GPU from the requests' lengths: pages are taken from and
// given back to a stack of free pages, and every token row gets its position and its cache slot.
//
// With P = block_size, n_i = max(new_lens[i], 0), c_i = context_lens[i]:
//   rows      end_i  = sum_{j <= i} n_j; request i owns token rows [end_i - n_i, end_i)
//   released  requests with new_lens[i] < 0 push their ceil(c_i / P) pages, in request order
//   need_i    = ceil((c_i + n_i) / P) - ceil(c_i / P) for requests whose pages fit the table row and
//               whose rows fit the row capacity
//   served    need_i == 0, or sum_{j <= i} need_j <= free pages: a prefix of those that need pages
//   slot      of position p: block_table[i][p / P] * P + p % P
//
// The reference builds these tables on the host, page by page, and copies them over on every step.
// Three prefix sums over the requests are all that the rows, pops and pushes have in common, so every
// CTA computes them for itself in shared memory (a few thousand lengths: 32 KB; an exchange between
// CTAs was not tried), and then the token rows, the popped and the pushed pages are dealt over the grid's
// threads, each of which finds its request by bisection of a prefix.  Prefixes saturate at 2^31 - 1,
// beyond every limit.  Nothing of what the grid writes is read again by it (a page popped from the
// part of the stack that this step pushes is looked up in the releasing request's table row), so no
// barrier is needed, except for callers that pass the same tensor for lengths before and after: their
// grid is one thread-block cluster of up to eight CTAs with a barrier between the sums and the writes (4000
// decoding requests 6.7 us instead of 6.1, 61 prompts of 73000 rows in all 12 instead of 8 in a first call).
// Bound by latency: a load, three block-wide sums, a bisection, a load and a store in a chain.  64
// decoding requests: 3.0 us; 4000 with pages of 16: 7.1 us; 61 prompts of 74000 rows in all: 6.0 us.
#include <cooperative_groups.h>

#include "common.cuh"

namespace b200moe {
namespace {

namespace cg = cooperative_groups;

constexpr int kMaxRequests = 8192;
constexpr int kMaxThreads = 1024;
constexpr int kMaxCluster = 8;
constexpr int kMaxGrid = 64;
constexpr int kRowsPerThread = 4;  // consecutive token rows: one 16-byte store of slots
constexpr int32_t kIntMax = 0x7fffffff;

struct Params {
  const int32_t* context_lens;
  const int32_t* new_lens;
  int32_t* block_table;
  int32_t* free_blocks;
  const int32_t* free_count;
  int32_t* seq_lens;
  int32_t* cu_seqlens;
  int32_t* slot_mapping;
  int64_t* positions;
  int32_t* free_count_out;
  int32_t* num_refused;
  int64_t table_stride;
  int32_t requests, max_blocks, block_size, free_capacity, num_rows, vector_rows;
  FastDiv by_block;
  int32_t in_place;  // outputs overwrite inputs: the grid is one cluster
};

// Sum of two non-negative values, at most kIntMax.  Associative, so prefixes may be built in any order; a
// prefix that reached kIntMax lies beyond every limit it is compared with.
__device__ __forceinline__ int32_t add_sat(int32_t a, int32_t b) {
  return static_cast<int32_t>(min(static_cast<uint32_t>(a) + static_cast<uint32_t>(b), static_cast<uint32_t>(kIntMax)));
}

// Exclusive prefixes of N values over the block (added by add_sat) and their totals, with one barrier.
// Every warp adds up the warps' sums for itself.  `s_warp` must not be in use by another scan.
template <int N>
__device__ __forceinline__ void block_scan(const int32_t (&v)[N], int32_t (*s_warp)[32], int32_t (&before)[N],
                                           int32_t (&total)[N]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int32_t inc[N];
#pragma unroll
  for (int k = 0; k < N; ++k) inc[k] = v[k];
#pragma unroll
  for (int d = 1; d < 32; d <<= 1)
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int32_t o = __shfl_up_sync(0xffffffffu, inc[k], d);
      if (lane >= d) inc[k] = add_sat(inc[k], o);
    }
  if (lane == 31)
#pragma unroll
    for (int k = 0; k < N; ++k) s_warp[k][warp] = inc[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; ++k) {
    int32_t w = lane < warps ? s_warp[k][lane] : 0;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int32_t o = __shfl_up_sync(0xffffffffu, w, d);
      if (lane >= d) w = add_sat(w, o);
    }
    total[k] = __shfl_sync(0xffffffffu, w, 31);
    const int32_t earlier = __shfl_sync(0xffffffffu, w, warp ? warp - 1 : 0);
    const int32_t own = __shfl_up_sync(0xffffffffu, inc[k], 1);
    before[k] = add_sat(warp ? earlier : 0, lane ? own : 0);
  }
}

// First index in [lo, n) with a[index] > key (n if none); `a` does not decrease.
__device__ __forceinline__ int first_above(const int32_t* a, int lo, int n, int32_t key) {
  while (lo < n) {
    const int mid = (lo + n) >> 1;
    if (a[mid] > key) n = mid; else lo = mid + 1;
  }
  return lo;
}

// What the blocks know after the sums.
struct Sums {
  const int32_t* end;    // rows, inclusive prefix
  const int32_t* upto;   // pages needed, inclusive prefix
  const int32_t* rel;    // pages released, inclusive prefix
  const int32_t* ctx;    // tokens before the step; ~tokens for requests that are not served
  int32_t top, avail;    // free pages before and after the pushes
  int requests;
};

__device__ __forceinline__ int32_t prefix_before(const int32_t* inclusive, int r) { return r ? inclusive[r - 1] : 0; }

// Where page v of the stack, as it stands after the pushes, is to be read.
__device__ __forceinline__ const int32_t* stack_at(const Params& p, const Sums& s, int32_t v) {
  if (v < s.top) return p.free_blocks + v;
  const int r = first_above(s.rel, 0, s.requests, v - s.top);
  return p.block_table + r * p.table_stride + (v - s.top - prefix_before(s.rel, r));
}

// Slots and positions of kN consecutive rows from n0.
template <int kN>
__device__ __forceinline__ void place_rows(const Params& p, const Sums& s, int64_t n0, int used_rows) {
  const int32_t* from[kN];  // table or stack entry of the row's page; null: no slot
  int32_t off[kN];
  int64_t pos[kN];
  int r = 0, page_before = -1;
  int32_t end = 0, start = 0;
  const int32_t* at = nullptr;
#pragma unroll
  for (int u = 0; u < kN; ++u) {
    const int64_t n = n0 + u;
    from[u] = nullptr;
    pos[u] = 0;
    off[u] = 0;
    if (n >= used_rows) continue;
    if (n >= end) {  // u == 0, or the next request begins here
      r = first_above(s.end, u ? r + 1 : 0, s.requests, static_cast<int32_t>(n));
      end = s.end[r];
      start = prefix_before(s.end, r);
      page_before = -1;
    }
    const int32_t c = s.ctx[r];
    const int32_t base = c < 0 ? ~c : c;
    pos[u] = static_cast<int64_t>(base) + (n - start);
    if (c < 0) continue;  // not served: no slot
    const int32_t i = static_cast<int32_t>(pos[u]);  // served: within the table row
    const int page = p.by_block(i);
    if (page != page_before) {
      page_before = page;
      const int have = p.by_block(base + p.block_size - 1);
      at = page < have ? p.block_table + r * p.table_stride + page
                       : stack_at(p, s, s.avail - 1 - prefix_before(s.upto, r) - (page - have));
    }
    from[u] = at;
    off[u] = i - page * p.block_size;
  }
  int32_t page_id[kN], slot[kN];
#pragma unroll
  for (int u = 0; u < kN; ++u) page_id[u] = from[u] ? *from[u] : -1;
#pragma unroll
  for (int u = 0; u < kN; ++u) {
    const int64_t at_slot = static_cast<int64_t>(page_id[u]) * p.block_size + off[u];
    slot[u] = page_id[u] >= 0 && at_slot <= kIntMax ? static_cast<int32_t>(at_slot) : -1;
  }
  if (kN == 4 && p.vector_rows && n0 + kN <= p.num_rows) {
    *reinterpret_cast<int4*>(p.slot_mapping + n0) = make_int4(slot[0], slot[1 % kN], slot[2 % kN], slot[3 % kN]);
    if (p.positions) {
      *reinterpret_cast<longlong2*>(p.positions + n0) = make_longlong2(pos[0], pos[1 % kN]);
      *reinterpret_cast<longlong2*>(p.positions + n0 + 2) = make_longlong2(pos[2 % kN], pos[3 % kN]);
    }
  } else {
#pragma unroll
    for (int u = 0; u < kN; ++u) {
      if (n0 + u < p.num_rows) {
        p.slot_mapping[n0 + u] = slot[u];
        if (p.positions) p.positions[n0 + u] = pos[u];
      }
    }
  }
}

template <int kPer>  // requests per thread
__global__ void __launch_bounds__(kMaxThreads)
paged_schedule_kernel(const Params p) {
  extern __shared__ int32_t smem[];
  __shared__ int32_t s_warp[3][32];
  __shared__ int s_refused, s_taken;
  const int R = p.requests, P = p.block_size;
  int32_t* s_end = smem;
  int32_t* s_upto = s_end + R;
  int32_t* s_rel = s_upto + R;
  int32_t* s_ctx = s_rel + R;
  if (threadIdx.x == 0) { s_refused = 0; s_taken = 0; }
  pdl_wait();
  pdl_launch_dependents();

  const int32_t count = *p.free_count;
  const int i0 = threadIdx.x * kPer;
  int32_t rows[kPer], ctx[kPer];
  int32_t sum[2] = {0, 0}, before[2], total[2];  // rows, released pages
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    const bool live = i0 + u < R;
    ctx[u] = live ? p.context_lens[i0 + u] : 0;
    rows[u] = live ? p.new_lens[i0 + u] : 0;
  }
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    ctx[u] = min(max(ctx[u], 0), p.max_blocks * P);
    if (rows[u] > 0) sum[0] = add_sat(sum[0], rows[u]);
    else if (rows[u] < 0) sum[1] = add_sat(sum[1], p.by_block(ctx[u] + P - 1));
  }
  block_scan<2>(sum, s_warp, before, total);
  const int32_t top = min(max(count, 0), p.free_capacity);
  const int32_t avail = min(add_sat(top, total[1]), p.free_capacity);

  int32_t need[kPer], sum_need[1] = {0}, need_before[1], total_need[1];
  bool fits[kPer];
  int32_t at_rows = before[0], at_rel = before[1];
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    need[u] = 0;
    fits[u] = false;
    if (i0 + u < R) {
      const int32_t have = p.by_block(ctx[u] + P - 1);
      if (rows[u] > 0) {
        at_rows = add_sat(at_rows, rows[u]);
        fits[u] = rows[u] <= p.max_blocks * P - ctx[u] && at_rows <= p.num_rows;
        if (fits[u]) need[u] = p.by_block(ctx[u] + rows[u] + P - 1) - have;
      } else if (rows[u] < 0) {
        at_rel = add_sat(at_rel, have);
      }
      s_end[i0 + u] = at_rows;
      s_rel[i0 + u] = at_rel;
      sum_need[0] = add_sat(sum_need[0], need[u]);
    }
  }
  block_scan<1>(sum_need, s_warp + 2, need_before, total_need);
  int refused = 0, taken = 0;
  int32_t at_need = need_before[0];
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    if (i0 + u < R) {
      at_need = add_sat(at_need, need[u]);
      const bool ok = fits[u] && (need[u] == 0 || at_need <= avail);
      s_upto[i0 + u] = at_need;
      s_ctx[i0 + u] = ok ? ctx[u] : ~ctx[u];
      if (rows[u] > 0 && !ok) ++refused;
      if (ok) taken += need[u];  // the sum over all threads is at most avail
    }
  }
  if (refused) atomicAdd(&s_refused, refused);
  if (taken) atomicAdd(&s_taken, taken);
  __syncthreads();
  // Every CTA of the cluster holds its own copy of the lengths now: they may be overwritten.
  if (p.in_place) cg::this_cluster().sync();

  // The work is dealt over the grid's threads as one sequence: groups of rows, popped pages, pushed
  // pages, requests.
  const Sums s = {s_end, s_upto, s_rel, s_ctx, top, avail, R};
  const int first = blockIdx.x * blockDim.x + threadIdx.x, stride = gridDim.x * blockDim.x;
  const int used_rows = min(total[0], p.num_rows);
  const int per_group = p.num_rows > stride ? kRowsPerThread : 1;
  const int64_t groups = per_group == 1 ? p.num_rows : (p.num_rows - 1) / kRowsPerThread + 1;
  const int64_t pops = groups + s_taken, pushes = pops + (avail - top), all = pushes + R;
  for (int64_t w = first; w < all; w += stride) {
    if (w < groups) {
      if (per_group == 1) place_rows<1>(p, s, w, used_rows);
      else place_rows<kRowsPerThread>(p, s, w * kRowsPerThread, used_rows);
    } else if (w < pops) {
      const int k = static_cast<int>(w - groups);
      const int r = first_above(s_upto, 0, R, k);
      const int col = p.by_block(s_ctx[r] + P - 1) + (k - prefix_before(s_upto, r));
      p.block_table[r * p.table_stride + col] = *stack_at(p, s, avail - 1 - k);
    } else if (w < pushes) {
      const int v = top + static_cast<int>(w - pops);
      p.free_blocks[v] = *stack_at(p, s, v);
    } else {
      const int i = static_cast<int>(w - pushes);
      const int32_t c = s_ctx[i];
      const int32_t n = min(s_end[i], p.num_rows), n_prev = min(prefix_before(s_end, i), p.num_rows);
      p.cu_seqlens[i + 1] = n;
      p.seq_lens[i] = c >= 0 ? c + (n - n_prev) : s_rel[i] > prefix_before(s_rel, i) ? 0 : ~c;
    }
  }
  if (first == 0) {
    p.cu_seqlens[0] = 0;
    *p.free_count_out = avail - s_taken;
    *p.num_refused = s_refused;
  }
}

}  // namespace
}  // namespace b200moe

extern "C" int b200moe_paged_schedule_max_requests(void) { return b200moe::kMaxRequests; }

extern "C" int b200moe_paged_schedule(const int32_t* context_lens, const int32_t* new_lens,
                                      int32_t* block_table, int32_t* free_blocks,
                                      const int32_t* free_count, int64_t num_requests,
                                      int64_t max_blocks_per_seq, int64_t table_row_stride,
                                      int block_size, int64_t free_capacity, int64_t num_rows,
                                      int32_t* seq_lens, int32_t* cu_seqlens, int32_t* slot_mapping,
                                      int64_t* positions, int32_t* free_count_out,
                                      int32_t* num_refused, b200moe_stream_t stream) {
  using namespace b200moe;
  const char* name = "paged_schedule";
  if (num_requests < 0 || num_requests > kMaxRequests)
    return fail(B200MOE_ERR_SHAPE, "%s: %lld requests; at most %d are supported", name,
                (long long)num_requests, kMaxRequests);
  if (block_size < 1 || max_blocks_per_seq < 1 || table_row_stride < max_blocks_per_seq ||
      max_blocks_per_seq > (kIntMax - block_size) / block_size)
    return fail(B200MOE_ERR_SHAPE, "%s: block_size=%d max_blocks_per_seq=%lld row stride %lld (a table "
                "row must name fewer than 2^31 tokens)", name, block_size,
                (long long)max_blocks_per_seq, (long long)table_row_stride);
  if (free_capacity < 0 || free_capacity >= kIntMax || num_rows < 0 || num_rows >= kIntMax)
    return fail(B200MOE_ERR_SHAPE, "%s: free_capacity=%lld num_rows=%lld", name,
                (long long)free_capacity, (long long)num_rows);
  if (!free_count || !cu_seqlens || !free_count_out || !num_refused || (num_rows > 0 && !slot_mapping) ||
      (free_capacity > 0 && !free_blocks) ||
      (num_requests > 0 && (!context_lens || !new_lens || !block_table || !seq_lens)))
    return fail(B200MOE_ERR_NULL, "%s: null pointer", name);
  Params p;
  p.context_lens = context_lens; p.new_lens = new_lens; p.block_table = block_table;
  p.free_blocks = free_blocks; p.free_count = free_count; p.seq_lens = seq_lens;
  p.cu_seqlens = cu_seqlens; p.slot_mapping = slot_mapping; p.positions = positions;
  p.free_count_out = free_count_out; p.num_refused = num_refused;
  p.table_stride = table_row_stride;
  p.requests = static_cast<int32_t>(num_requests);
  p.max_blocks = static_cast<int32_t>(max_blocks_per_seq);
  p.block_size = block_size;
  p.by_block = FastDiv::by(static_cast<uint32_t>(block_size));
  p.free_capacity = static_cast<int32_t>(free_capacity);
  p.num_rows = static_cast<int32_t>(num_rows);
  p.vector_rows = aligned_to(slot_mapping, 16) && aligned_to(positions, 16);

  // One CTA of 256 threads for small steps; else 1024 threads and a grid that grows with the work, which is
  // the rows, the requests and the pages that move (a few per request, the host does not know).
  p.in_place = seq_lens == context_lens || free_count_out == free_count;
  const int64_t items = num_rows + 4 * num_requests;
  const int threads = items <= 512 ? 256 : kMaxThreads;
  const int most = p.in_place ? kMaxCluster : kMaxGrid;
  int ncta = 1;
  while (ncta < most && items > static_cast<int64_t>(ncta) * kMaxThreads) ncta *= 2;
  if (ncta == 1) p.in_place = 0;  // the block's own barriers are enough
  const size_t smem = static_cast<size_t>(num_requests) * 4 * sizeof(int32_t);
  const int64_t per = ceil_div64(num_requests, threads);
  const auto kernel = per <= 1 ? paged_schedule_kernel<1> : per <= 2 ? paged_schedule_kernel<2>
                    : per <= 4 ? paged_schedule_kernel<4> : paged_schedule_kernel<kMaxRequests / kMaxThreads>;
  if (smem > 48 * 1024 - 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               kMaxRequests * 4 * static_cast<int>(sizeof(int32_t)));
    if (e != cudaSuccess) return fail(B200MOE_ERR_CUDA, "%s: %s", name, cudaGetErrorString(e));
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ncta);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.in_place ? ncta : 1;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaLaunchKernelEx(&cfg, kernel, p);
  return check_launch(name);
}
