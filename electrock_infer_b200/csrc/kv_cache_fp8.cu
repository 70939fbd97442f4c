// Paged KV-cache store in 8 bits: new key and value rows become e4m3 codes under one scale per page
// and KV head (layout and scales: fp8_cache.cuh).
//
//   key, value        [num_tokens, num_kv_heads, 128], row strides in elements
//   k_cache, v_cache  [num_blocks, block_size, num_kv_heads, 128] codes
//   k_scale, v_scale  [num_blocks, num_kv_heads] fp32
//   slot_mapping      [num_tokens] int32: slot = block * block_size + offset; negative = skip
//
// For every page that the call stores to, with amax over the call's finite values of page and head:
//   needed = smallest 2^e with amax <= 448 * 2^e;  scale = max(needed, old scale)
//   a grown scale moves the page's old codes by old / new; new codes = e4m3(x / scale)
// A call that stores to a page's first slot begins the page anew: its old scale and codes count for
// nothing.  The tokens of one page must follow one another in the call, with nothing but skipped entries
// between them (slot maps are built request by request); such a run is the unit of work, and nothing has to
// be exchanged between runs.
//
// The reference has no 8-bit cache; its store (src/store_kv_cache.hip:12-63) copies.  This one has to know
// a run's largest value before it can write the first code, so the rows of a run are held in registers
// between the two: short runs (decode: one token) by one warp, longer ones by the whole CTA.  A run that
// does not fit is read a second time (from L2).  Every CTA finds the runs of its segment of tokens for
// itself, 3 us that a list written by a kernel of its own did not make up for.  Prompts: bound by the
// phases of a CTA that follow one another (16 prompts of 512-1024 tokens with 8 heads in 28.0 us, of which
// finding the runs 8, reading 10, converting and writing 7; 75.7 MB would take 11.6).  Decode steps: bound by
// latency (slot -> rows and old scale -> codes; 64 tokens in 3.3 us) as long as no scale grows.  Where one does, a
// warp goes through the page four rows at a time, each load behind the last store: 1.5 us more with pages of 16
// tokens, 7 with 64, 33 with 256, whether one page grows or four do (43 when all 1024 do).  Skipped entries behind the
// last token cost 2 to 3 us up to 448 of them, 5 for 960, 19 for 4032: its run is followed to its end.
#include "fp8_cache.cuh"

namespace b200moe {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxSegment = 256;   // tokens whose runs one CTA may own
// 16-byte pieces of a run that a thread holds: 16 rows of 16-bit elements for a warp, 128 for the CTA.
// Twice as many leave room for two CTAs per SM instead of three: 37 prompts of 26-53 tokens 9.3 us instead
// of 7.0, 16 prompts of 512-1024 tokens 27.2 us instead of 28.3.
constexpr int kPieces = 8;

struct Side {  // keys or values
  const uint8_t* src;
  uint8_t* cache;
  float* scale;
  int64_t src_stride;  // bytes
};
struct Params {
  Side key, value;
  const int32_t* slots;
  int64_t num_tokens, num_slots;
  int heads, block_size, segment;
  FastDiv by_block;
};

// How a thread holds a 16-byte piece of a row.  Sizes (|x|) are compared as integers, two 16-bit ones at
// once: the order of the bits is the order of the values.
template <typename T> struct Row;
template <> struct Row<__nv_bfloat16> {
  static constexpr int kElems = 8;
  static constexpr uint32_t kInfinity = 0x7f80;
  __device__ static uint32_t size_bits(uint32_t size) { return size << 16; }  // as fp32
  __device__ static void up(uint4 v, float (&x)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};
template <> struct Row<__half> {
  static constexpr int kElems = 8;
  static constexpr uint32_t kInfinity = 0x7c00;
  __device__ static uint32_t size_bits(uint32_t size) {
    return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(size))));
  }
  __device__ static void up(uint4 v, float (&x)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
};
template <> struct Row<float> {
  static constexpr int kElems = 4;
  static constexpr uint32_t kInfinity = 0x7f800000;
  __device__ static uint32_t size_bits(uint32_t size) { return size; }
  __device__ static void up(uint4 v, float (&x)[4]) {
    x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y);
    x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w);
  }
};

// The larger of `size` and the sizes in `v`; 16-bit sizes are kept two to a word.
template <typename T>
__device__ __forceinline__ uint32_t larger_size(uint32_t size, uint4 v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    size = sizeof(T) == 2 ? __vmaxu2(size, w[i] & 0x7fff7fffu) : max(size, w[i] & 0x7fffffffu);
  return size;
}
// `v` with zeros in place of infinities and NaN.
template <typename T>
__device__ uint4 finite_only(uint4 v) {
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 2) {
      if ((w[i] & 0x7fffu) >= Row<T>::kInfinity) w[i] &= 0xffff0000u;
      if (((w[i] >> 16) & 0x7fffu) >= Row<T>::kInfinity) w[i] &= 0xffffu;
    } else if ((w[i] & 0x7fffffffu) >= Row<T>::kInfinity) {
      w[i] = 0;
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Slot of token `i`; -1 when it has none, or one outside the cache.
__device__ __forceinline__ int32_t slot_of(const Params& p, int64_t i) {
  const int32_t s = p.slots[i];
  return s >= 0 && s < p.num_slots ? s : -1;
}
// Page of token `i`; -1 when the token has no slot.
__device__ __forceinline__ int page_of(const Params& p, int64_t i) {
  const int32_t s = slot_of(p, i);
  return s >= 0 ? p.by_block(s) : -1;
}

// Stores the run of `len` tokens from `first`, all in page `page` or skipped, for one head of keys or
// values.  kGroupWarps warps work together (1, or the whole CTA); each thread holds up to kU pieces.
template <typename T, int kGroupWarps, int kU>
__device__ void store_run(const Params& p, const Side& side, int head, int64_t first, int64_t len, int page,
                          uint32_t* s_red) {
  constexpr int kLanes = kCodeHeadDim / Row<T>::kElems;      // lanes per row
  constexpr int kRowsPerStep = kGroupWarps * 32 / kLanes;    // rows the group loads at once
  const int gt = kGroupWarps == 1 ? (threadIdx.x & 31) : threadIdx.x;
  const int row0 = gt / kLanes, col = gt % kLanes;
  const uint8_t* src = side.src + static_cast<int64_t>(head) * kCodeHeadDim * sizeof(T) + col * 16;
  const int64_t row_bytes = static_cast<int64_t>(p.heads) * kCodeHeadDim;
  uint8_t* cache = side.cache + static_cast<int64_t>(head) * kCodeHeadDim;
  float* scale_at = side.scale + static_cast<int64_t>(page) * p.heads + head;
  const float old = usable_scale(*scale_at);
  const int32_t page_slot = page * p.block_size;
  constexpr int kWindow = kRowsPerStep * kU;

  uint4 held[kU];
  int32_t slot[kU];
  auto load = [&](int64_t w) {
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int64_t r = w + row0 + u * kRowsPerStep;
      slot[u] = -1;
      if (r < len) {
        held[u] = ld_stream_16(src + (first + r) * side.src_stride);
        slot[u] = slot_of(p, first + r);
      }
    }
  };
  // The run's largest size over the group; infinities and NaN do not count in the second form, which is
  // only needed when the first has met one.
  int begins = 0;
  auto largest = [&](bool only_finite) {
    uint32_t size = 0;
    for (int64_t w = 0; w < len; w += kWindow) {
      if (!only_finite || len > kWindow) load(w);
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        if (slot[u] < 0) continue;
        size = larger_size<T>(size, only_finite ? finite_only<T>(held[u]) : held[u]);
        begins |= slot[u] == page_slot;
      }
    }
    if (sizeof(T) == 2) size = max(size & 0xffffu, size >> 16);
    size = __reduce_max_sync(0xffffffffu, size);
    if (kGroupWarps == 1) {
      begins = __any_sync(0xffffffffu, begins);
    } else {
      begins = __syncthreads_or(begins);  // also: s_red has been read
      if ((threadIdx.x & 31) == 0) s_red[threadIdx.x >> 5] = size;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kGroupWarps; ++i) size = max(size, s_red[i]);
    }
    return size;
  };
  uint32_t size = largest(false);
  if (size >= Row<T>::kInfinity) size = largest(true);
  const float needed = scale_for(Row<T>::size_bits(size));
  const float scale = begins ? needed : fmaxf(needed, old);
  if (!begins && scale > old) {
    // The page's old codes under the new scale, rows of this run included (they are overwritten below).
    const float ratio = old / scale;
    for (int r = gt / 8; r < p.block_size; r += kGroupWarps * 4) {
      uint4* at = reinterpret_cast<uint4*>(cache + (static_cast<int64_t>(page_slot) + r) * row_bytes) + gt % 8;
      uint4 c = *at;
      c.x = rescale_codes4(c.x, ratio); c.y = rescale_codes4(c.y, ratio);
      c.z = rescale_codes4(c.z, ratio); c.w = rescale_codes4(c.w, ratio);
      *at = c;
    }
  }
  if (kGroupWarps > 1) __syncthreads(); else __syncwarp();
  if (gt == 0) *scale_at = scale;
  const float inv = 1.f / scale;  // exact: a power of two
  for (int64_t w = 0; w < len; w += kWindow) {
    if (len > kWindow) load(w);  // otherwise the rows are still held
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      if (slot[u] < 0) continue;
      float x[Row<T>::kElems];
      Row<T>::up(held[u], x);
      uint32_t codes[Row<T>::kElems / 4];
#pragma unroll
      for (int j = 0; j < Row<T>::kElems / 4; ++j)
        codes[j] = to_codes4(x[4 * j] * inv, x[4 * j + 1] * inv, x[4 * j + 2] * inv, x[4 * j + 3] * inv);
      uint8_t* dst = cache + slot[u] * row_bytes + col * Row<T>::kElems;
      if constexpr (Row<T>::kElems == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(codes[0], codes[1]);
      else *reinterpret_cast<uint32_t*>(dst) = codes[0];
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 3)
paged_store_fp8_kernel(const Params p) {
  __shared__ int s_begin[kMaxSegment], s_begin_page[kMaxSegment], s_page[kMaxSegment], s_long[kMaxSegment];
  __shared__ int s_num_begin, s_num_long, s_at;
  __shared__ int s_last[kWarps];
  __shared__ uint32_t s_red[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int head = blockIdx.x >> 1;
  const Side side = blockIdx.x & 1 ? p.value : p.key;
  const int64_t seg0 = static_cast<int64_t>(blockIdx.y) * p.segment;
  if (threadIdx.x == 0) { s_num_begin = 0; s_num_long = 0; }
  pdl_wait();
  pdl_launch_dependents();

  // Runs that begin in this segment: a token whose page differs from that of the last token before it
  // that has one.
  const int64_t mine = seg0 + threadIdx.x;
  const int page = threadIdx.x < p.segment && mine < p.num_tokens ? page_of(p, mine) : -1;
  int before_page = seg0 > 0 ? page_of(p, seg0 - 1) : -1;  // the last page before the segment
  int last = page >= 0 ? static_cast<int>(threadIdx.x) : -1;  // inclusive maximum over the threads
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, last, d);
    if (lane >= d) last = max(last, o);
  }
  if (lane == 31) s_last[warp] = last;
  s_page[threadIdx.x] = page;
  __syncthreads();
  int prev = __shfl_up_sync(0xffffffffu, last, 1);
  if (lane == 0) prev = -1;
  bool any = false;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) prev = max(prev, s_last[w]);
    any |= s_last[w] >= 0;
  }
  if (!any) return;  // nothing but skipped tokens
  // Skipped tokens right before the segment: look further back, kThreads tokens at a time.
  for (int64_t end = seg0 - 1; before_page < 0 && end > 0; end -= kThreads) {
    __syncthreads();
    if (threadIdx.x == 0) s_at = -1;
    __syncthreads();
    const int64_t j = end - 1 - threadIdx.x;
    const int other = j >= 0 ? page_of(p, j) : -1;
    if (other >= 0) atomicMax(&s_at, kThreads - 1 - static_cast<int>(threadIdx.x));
    __syncthreads();
    if (s_at >= 0) before_page = page_of(p, end - kThreads + s_at);
  }
  if (page >= 0 && page != (prev >= 0 ? s_page[prev] : before_page)) {
    const int k = atomicAdd(&s_num_begin, 1);
    s_begin[k] = threadIdx.x;
    s_begin_page[k] = page;
  }
  __syncthreads();

  // One warp per run that ends within the next 32 tokens; the others wait for the whole CTA.
  for (int k = warp; k < s_num_begin; k += kWarps) {
    const int64_t i = seg0 + s_begin[k];
    const int run_page = s_begin_page[k];
    int at = -1;
    if (i + lane < p.num_tokens) at = page_of(p, i + lane); else at = -2;
    const uint32_t out = __ballot_sync(0xffffffffu, at != run_page && at != -1);
    if (out == 0) {
      if (lane == 0) s_long[atomicAdd(&s_num_long, 1)] = k;
      continue;
    }
    store_run<T, 1, kPieces>(p, side, head, i, __ffs(out) - 1, run_page, s_red);
  }
  __syncthreads();
  for (int k = 0; k < s_num_long; ++k) {
    const int64_t i = seg0 + s_begin[s_long[k]];
    const int run_page = s_begin_page[s_long[k]];
    // Length of the run: the first token, looking kThreads at a time, that is elsewhere.
    int64_t len = 0;
    while (true) {
      __syncthreads();  // s_at and s_red of the previous turn have been read
      if (threadIdx.x == 0) s_at = kThreads;
      __syncthreads();
      const int64_t j = i + len + threadIdx.x;
      const int other = j < p.num_tokens ? page_of(p, j) : -2;
      if (other != run_page && other != -1) atomicMin(&s_at, static_cast<int>(threadIdx.x));
      __syncthreads();
      len += s_at;
      if (s_at < kThreads) break;
    }
    // Skipped tokens at its end (a padded batch) need not be gone through: back to the last that has a slot.
    while (page_of(p, i + len - 1) < 0) {
      __syncthreads();
      if (threadIdx.x == 0) s_at = -1;
      __syncthreads();
      const int64_t j = i + len - 1 - threadIdx.x;
      if (j >= i && page_of(p, j) >= 0) atomicMax(&s_at, kThreads - 1 - static_cast<int>(threadIdx.x));
      __syncthreads();
      len -= s_at >= 0 ? kThreads - 1 - s_at : kThreads;
    }
    store_run<T, kWarps, kPieces>(p, side, head, i, len, run_page, s_red);
  }
}

template <typename T>
int launch(Params p, cudaStream_t st) {
  // Segments short enough that the grid fills the GPU several times over, at least one token per warp.
  const int64_t want = ceil_div64(p.num_tokens * 2 * p.heads, 8ll * sm_count());
  p.segment = kWarps;
  while (p.segment < kMaxSegment && p.segment < want) p.segment *= 2;
  const int64_t segments = ceil_div64(p.num_tokens, p.segment);
  if (segments > 65535)
    return fail(B200MOE_ERR_SHAPE, "paged_store_kvcache_fp8: num_tokens=%lld; at most %d", (long long)p.num_tokens,
                65535 * kMaxSegment);
  launch_pdl(paged_store_fp8_kernel<T>, dim3(2 * p.heads, static_cast<unsigned>(segments)), dim3(kThreads), 0,
             st, p);
  return check_launch("paged_store_kvcache_fp8");
}

}  // namespace
}  // namespace b200moe

extern "C" int b200moe_paged_store_kvcache_fp8(const void* key, const void* value, void* k_cache,
                                               void* v_cache, float* k_scale, float* v_scale,
                                               const int32_t* slot_mapping, int dtype,
                                               int64_t num_tokens, int num_kv_heads, int head_dim,
                                               int64_t key_row_stride, int64_t value_row_stride,
                                               int64_t num_blocks, int block_size,
                                               b200moe_stream_t stream) {
  using namespace b200moe;
  const char* name = "paged_store_kvcache_fp8";
  int elem = 0;
  switch (dtype) {
    case B200MOE_F32: elem = 4; break;
    case B200MOE_F16:
    case B200MOE_BF16: elem = 2; break;
    default: return fail(B200MOE_ERR_DTYPE, "%s: unsupported dtype %d", name, dtype);
  }
  if (head_dim != kCodeHeadDim)
    return fail(B200MOE_ERR_SHAPE, "%s: head_dim must be 128, got %d", name, head_dim);
  if (num_tokens < 0 || num_kv_heads < 1 || num_kv_heads > 0x3fffffff || num_blocks < 0 || block_size < 1)
    return fail(B200MOE_ERR_SHAPE, "%s: num_tokens=%lld kv_heads=%d num_blocks=%lld block_size=%d", name,
                (long long)num_tokens, num_kv_heads, (long long)num_blocks, block_size);
  const int64_t row_elems = static_cast<int64_t>(num_kv_heads) * head_dim;
  if (key_row_stride < row_elems || value_row_stride < row_elems)
    return fail(B200MOE_ERR_SHAPE, "%s: row strides (%lld, %lld) smaller than a row (%lld)", name,
                (long long)key_row_stride, (long long)value_row_stride, (long long)row_elems);
  if (num_tokens == 0) return B200MOE_OK;
  if (!key || !value || !k_cache || !v_cache || !k_scale || !v_scale || !slot_mapping)
    return fail(B200MOE_ERR_NULL, "%s: null pointer", name);
  if (key_row_stride * elem % 16 != 0 || value_row_stride * elem % 16 != 0 || !aligned_to(key, 16) ||
      !aligned_to(value, 16) || !aligned_to(k_cache, 16) || !aligned_to(v_cache, 16))
    return fail(B200MOE_ERR_ALIGN, "%s: row strides and base pointers must be multiples of 16 bytes", name);
  Params p;
  p.key = {static_cast<const uint8_t*>(key), static_cast<uint8_t*>(k_cache), k_scale, key_row_stride * elem};
  p.value = {static_cast<const uint8_t*>(value), static_cast<uint8_t*>(v_cache), v_scale,
             value_row_stride * elem};
  p.slots = slot_mapping;
  p.num_tokens = num_tokens;
  p.num_slots = num_blocks * static_cast<int64_t>(block_size);
  p.heads = num_kv_heads;
  p.block_size = block_size;
  p.segment = 0;
  p.by_block = FastDiv::by(static_cast<uint32_t>(block_size));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case B200MOE_BF16: return launch<__nv_bfloat16>(p, st);
    case B200MOE_F16: return launch<__half>(p, st);
    default: return launch<float>(p, st);
  }
}
