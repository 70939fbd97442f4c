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
// CTA of one thread-block cluster computes them for itself in shared memory (a few thousand
// lengths: 32 KB, cheaper than any exchange), and then the token rows, the popped and the pushed
// pages are dealt over the cluster's threads, each of which finds its request by bisection of a
// prefix.  Nothing of what the cluster writes is read again by it (a page popped from
// the part of the stack that this step pushes is looked up in the releasing request's table row), so
// the one barrier between the sums and the writes only serves callers that pass the same tensor for
// lengths before and after.  Bound by latency: a load, three block-wide sums, a bisection, a load and a
// store in a chain.
#include <cooperative_groups.h>

#include "common.cuh"

namespace b200moe {
namespace {

namespace cg = cooperative_groups;

constexpr int kMaxRequests = 8192;
constexpr int kMaxThreads = 1024;
constexpr int kMaxPerThread = kMaxRequests / kMaxThreads;
constexpr int kMaxCluster = 8;
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
};

__device__ __forceinline__ int32_t saturate(int64_t v) {
  return v > kIntMax ? kIntMax : static_cast<int32_t>(v);
}

// Exclusive prefix of `v` over the block; `total` receives the sum.  All threads must call it.
__device__ int64_t block_scan(int64_t v, int64_t* s_warp, int64_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int64_t inc = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t o = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += o;
  }
  __syncthreads();  // s_warp may still be read from the previous scan
  if (lane == 31) s_warp[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    int64_t w = lane < warps ? s_warp[lane] : 0;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t o = __shfl_up_sync(0xffffffffu, w, d);
      if (lane >= d) w += o;
    }
    s_warp[lane] = w;  // inclusive over warps; lanes past the last warp repeat the total
  }
  __syncthreads();
  total = s_warp[31];
  return inc - v + (warp ? s_warp[warp - 1] : 0);
}

// First index in [lo, n) with a[index] > key (n if none); `a` does not decrease.
__device__ __forceinline__ int first_above(const int32_t* a, int lo, int n, int32_t key) {
  while (lo < n) {
    const int mid = (lo + n) >> 1;
    if (a[mid] > key) n = mid; else lo = mid + 1;
  }
  return lo;
}

__global__ void __launch_bounds__(kMaxThreads)
paged_schedule_kernel(const Params p) {
  extern __shared__ int32_t smem[];
  __shared__ int64_t s_warp[32];
  __shared__ int s_refused, s_taken;
  const int R = p.requests, P = p.block_size;
  int32_t* s_end = smem;          // rows, inclusive prefix
  int32_t* s_upto = s_end + R;    // pages needed, inclusive prefix
  int32_t* s_rel = s_upto + R;    // pages released, inclusive prefix
  int32_t* s_ctx = s_rel + R;     // tokens before the step; ~tokens for requests that are not served
  cg::cluster_group cluster = cg::this_cluster();
  const int ncta = static_cast<int>(cluster.num_blocks());
  const int rank = static_cast<int>(cluster.block_rank());
  pdl_wait();
  pdl_launch_dependents();

  if (threadIdx.x == 0) { s_refused = 0; s_taken = 0; }
  const int per = (R + blockDim.x - 1) / blockDim.x;
  const int i0 = threadIdx.x * per;
  int32_t rows[kMaxPerThread], ctx[kMaxPerThread];
  int64_t sum_rows = 0, sum_rel = 0;
#pragma unroll
  for (int u = 0; u < kMaxPerThread; ++u) {
    rows[u] = 0;
    ctx[u] = 0;
    if (u < per && i0 + u < R) {
      ctx[u] = min(max(p.context_lens[i0 + u], 0), p.max_blocks * P);
      rows[u] = p.new_lens[i0 + u];
      if (rows[u] > 0) sum_rows += rows[u];
      else if (rows[u] < 0) sum_rel += (ctx[u] + P - 1) / P;
    }
  }
  int64_t total_rows, total_rel, total_need;
  int64_t at_rows = block_scan(sum_rows, s_warp, total_rows);
  int64_t at_rel = block_scan(sum_rel, s_warp, total_rel);
  const int32_t top = min(max(*p.free_count, 0), p.free_capacity);
  const int32_t avail = static_cast<int32_t>(min(top + total_rel, static_cast<int64_t>(p.free_capacity)));

  int64_t need[kMaxPerThread], sum_need = 0;
  bool fits[kMaxPerThread];
#pragma unroll
  for (int u = 0; u < kMaxPerThread; ++u) {
    need[u] = 0;
    fits[u] = false;
    if (u < per && i0 + u < R) {
      const int64_t have = (ctx[u] + P - 1) / P;
      if (rows[u] > 0) {
        at_rows += rows[u];
        const int64_t want = (static_cast<int64_t>(ctx[u]) + rows[u] + P - 1) / P;
        fits[u] = want <= p.max_blocks && at_rows <= p.num_rows;
        if (fits[u]) need[u] = want - have;
      } else if (rows[u] < 0) {
        at_rel += have;
      }
      s_end[i0 + u] = saturate(at_rows);
      s_rel[i0 + u] = saturate(at_rel);
      sum_need += need[u];
    }
  }
  int64_t at_need = block_scan(sum_need, s_warp, total_need);
  int refused = 0, taken = 0;
#pragma unroll
  for (int u = 0; u < kMaxPerThread; ++u) {
    if (u < per && i0 + u < R) {
      at_need += need[u];
      const bool ok = fits[u] && (need[u] == 0 || at_need <= avail);
      s_upto[i0 + u] = saturate(at_need);
      s_ctx[i0 + u] = ok ? ctx[u] : ~ctx[u];
      if (rows[u] > 0 && !ok) ++refused;
      if (ok) taken += static_cast<int>(need[u]);  // the sum over all threads is at most avail
    }
  }
  if (refused) atomicAdd(&s_refused, refused);
  if (taken) atomicAdd(&s_taken, taken);
  __syncthreads();
  // Every CTA holds its own copy of the lengths now: they may be overwritten (seq_lens may be
  // context_lens, free_count_out may be free_count).
  if (ncta > 1) cluster.sync();

  const int first = rank * blockDim.x + threadIdx.x, stride = ncta * blockDim.x;
  const int used_rows = static_cast<int>(min(total_rows, static_cast<int64_t>(p.num_rows)));

  // Page v of the stack as it stands after the pushes.
  auto stack = [&](int32_t v) -> int32_t {
    if (v < top) return p.free_blocks[v];
    const int r = first_above(s_rel, 0, R, v - top);
    return p.block_table[r * p.table_stride + (v - top - (r ? s_rel[r - 1] : 0))];
  };

  // Token rows.
  for (int64_t n0 = static_cast<int64_t>(first) * kRowsPerThread; n0 < p.num_rows;
       n0 += static_cast<int64_t>(stride) * kRowsPerThread) {
    int32_t slot[kRowsPerThread];
    int64_t pos[kRowsPerThread];
    int r = 0, last_page = -1;
    int32_t end = 0, start = 0, page_id = -1;
#pragma unroll
    for (int u = 0; u < kRowsPerThread; ++u) {
      const int64_t n = n0 + u;
      slot[u] = -1;
      pos[u] = 0;
      if (n >= used_rows) continue;
      if (n >= end) {  // u == 0, or the next request begins here
        r = first_above(s_end, u ? r + 1 : 0, R, static_cast<int32_t>(n));
        end = s_end[r];
        start = r ? s_end[r - 1] : 0;
        last_page = -1;
      }
      const int32_t c = s_ctx[r];
      const int32_t base = c < 0 ? ~c : c;
      pos[u] = static_cast<int64_t>(base) + (n - start);
      if (c < 0) continue;  // not served: no slot
      const int32_t pi = static_cast<int32_t>(pos[u]);  // served: within the table row
      const int page = pi / P, have = (base + P - 1) / P;
      if (page != last_page) {
        last_page = page;
        page_id = page < have ? p.block_table[r * p.table_stride + page]
                              : stack(avail - 1 - (r ? s_upto[r - 1] : 0) - (page - have));
      }
      const int64_t s = static_cast<int64_t>(page_id) * P + (pi - page * P);
      if (page_id >= 0 && s <= kIntMax) slot[u] = static_cast<int32_t>(s);
    }
    if (p.vector_rows && n0 + kRowsPerThread <= p.num_rows) {
      *reinterpret_cast<int4*>(p.slot_mapping + n0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
      if (p.positions) {
        *reinterpret_cast<longlong2*>(p.positions + n0) = make_longlong2(pos[0], pos[1]);
        *reinterpret_cast<longlong2*>(p.positions + n0 + 2) = make_longlong2(pos[2], pos[3]);
      }
    } else {
#pragma unroll
      for (int u = 0; u < kRowsPerThread; ++u) {
        if (n0 + u < p.num_rows) {
          p.slot_mapping[n0 + u] = slot[u];
          if (p.positions) p.positions[n0 + u] = pos[u];
        }
      }
    }
  }

  // Popped pages into the table rows, pushed pages onto the stack.
  for (int k = first; k < s_taken; k += stride) {
    const int r = first_above(s_upto, 0, R, k);
    const int col = (s_ctx[r] + P - 1) / P + (k - (r ? s_upto[r - 1] : 0));
    p.block_table[r * p.table_stride + col] = stack(avail - 1 - k);
  }
  for (int v = top + first; v < avail; v += stride) p.free_blocks[v] = stack(v);

  // Lengths and offsets.
  for (int i = first; i < R; i += stride) {
    const int32_t c = s_ctx[i];
    const int32_t n = min(s_end[i], p.num_rows), n_prev = i ? min(s_end[i - 1], p.num_rows) : 0;
    const int32_t rel = s_rel[i] - (i ? s_rel[i - 1] : 0);
    p.cu_seqlens[i + 1] = n;
    p.seq_lens[i] = c >= 0 ? c + (n - n_prev) : rel > 0 ? 0 : ~c;
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
  if (free_capacity < 0 || free_capacity > kIntMax || num_rows < 0 || num_rows >= kIntMax)
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
  p.free_capacity = static_cast<int32_t>(free_capacity);
  p.num_rows = static_cast<int32_t>(num_rows);
  p.vector_rows = aligned_to(slot_mapping, 16) && aligned_to(positions, 16);

  // One CTA of 256 threads for small steps, else 1024 threads and a cluster that grows with the rows.
  const int threads = num_requests <= 256 && num_rows <= 1024 ? 256 : kMaxThreads;
  int ncta = 1;
  while (ncta < kMaxCluster && num_rows > static_cast<int64_t>(ncta) * kMaxThreads * kRowsPerThread) ncta *= 2;
  const size_t smem = static_cast<size_t>(num_requests) * 4 * sizeof(int32_t);
  const cudaError_t e = cudaFuncSetAttribute(paged_schedule_kernel,
                                             cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             kMaxRequests * 4 * static_cast<int>(sizeof(int32_t)));
  if (e != cudaSuccess) return fail(B200MOE_ERR_CUDA, "%s: %s", name, cudaGetErrorString(e));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ncta);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ncta;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaLaunchKernelEx(&cfg, paged_schedule_kernel, p);
  return check_launch(name);
}
