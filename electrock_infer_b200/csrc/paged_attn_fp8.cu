// Decode attention over the 8-bit paged cache: one query token per sequence, grouped query heads.
//
//   q, out            [batch, q_heads, 128] bf16 or fp16 (q rows may be strided)
//   k_cache, v_cache  [num_blocks, block_size, kv_heads, 128] e4m3 codes
//   k_scale, v_scale  [num_blocks, kv_heads] fp32, value = code * scale
//   block_table       [batch, max_blocks] int32, context_lens [batch] int32
//   out[b, h] = softmax(scale * q[b, h] . K[b, h / group, :ctx]) @ V[b, h / group, :ctx]
//
// The reference has no 8-bit cache; its kernel (src/paged_attn_gqa_varlen.hip:17-213) streams a 16-bit
// one once per QUERY head.  Half the bytes per token also means half the time per token, so what
// the 16-bit kernel of this library spends per token beside its loads is too much here.  Both products
// are therefore taken transposed:
//
//   S^T = K q^T   16 tokens x 8 heads, A = codes of K widened to fp16 in registers, B = q^T
//   O^T = V^T P^T 16 dims x 8 heads,   A = codes of V widened to fp16, B = P^T
//
// with m16n8k16: the tile is 8 heads wide, not 16 rows high, so groups of up to 8 query heads cost half
// the tensor instructions, exponentials and accumulators of a 16-row query tile (groups of 9 to 16 take
// two such tiles).  Fragments come from 16-byte shared-memory reads, not from matrix loads: the
// contraction index of S and the output rows of O may be permuted at will, so a lane takes 16
// consecutive codes of its token and the query is laid out to match; V's pairs of neighbouring tokens
// are interleaved by byte permutes before they are widened.  fp16 holds every e4m3 value exactly, so
// widening rounds nothing; q rows are scaled by a power of two into fp16's range (exact for values within 2^-28,
// fp16, or 2^-31, bf16, of the row's largest; smaller ones are kept to 2^-39 of it), P is rounded to fp16, all sums,
// maxima and the outputs are fp32.  P's rounding, 2^-11 of a weight, is as large as that of an fp16 output and an eighth
// of a bf16 one's, and the errors of many tokens average out; P in bf16 would err eight times as much, and a second
// fp16 number for what is left would take half as many products again.
//
// Four warps stream their own 32-token chunks through rings of asynchronous 16-byte copies
// (rows of 128 bytes, XOR-swizzled).  A page's K scale multiplies the scores; its V scale is the unit that
// the accumulators are kept in, which is exchanged only where a warp comes to another page.  With
// num_splits > 1 the context is cut into ranges for separate CTAs: 2, 4 or 8 of them form a thread-block
// cluster and merge through distributed shared memory where every CTA has an SM to itself; else they go
// through a workspace and a second kernel.
// (The tensor cores of sm_100a take codes directly only through tcgen05; m16n8k32 of codes is carried out as
// conversions and products of fp16, and measured a tenth slower than converting here.)
// Bound by HBM: 256 bytes per token and KV head.  128 sequences of 4096-8192 tokens with 8 x 4 heads: 251 us, 6.4
// TB/s; 4 of 30000-60000 with 16 query heads on one KV head: 20.1 us, bound by instructions; 1 of 700: 5.2 us.
#include <cooperative_groups.h>

#include "fp8_cache.cuh"
#include "warp_mma.cuh"

namespace b200moe {
namespace {

namespace cg = cooperative_groups;

constexpr int kDim = kCodeHeadDim;
constexpr int kTile = 16;                  // tokens of one product; a tile never crosses a page
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kChunkTiles = 2;             // tiles per ring stage
constexpr int kChunk = kTile * kChunkTiles;
constexpr int kHalfBytes = kChunk * kDim;  // 4 KiB of K, as much of V
constexpr int kStageBytes = 2 * kHalfBytes;
// kNT = tiles of 8 query heads.  One tile: a two-stage ring and three CTAs per SM (measured 5 to 15 % faster
// than three stages and two CTAs); two tiles need the registers of two CTAs per SM, whose rings then have
// three stages.
template <int kNT> struct Ring {
  static constexpr int kStages = kNT == 1 ? 2 : 3;
  static constexpr int kCtas = kNT == 1 ? 3 : 2;
  static constexpr int kBytes = kWarps * kStages * kStageBytes;
  static constexpr int kSmemBytes = kBytes + kWarps * kStages * 2 * kChunkTiles * static_cast<int>(sizeof(float));
};
constexpr int kMaxCluster = 8;             // splits that merge through distributed shared memory
constexpr int kMaxGroup = 16;
constexpr int kMaxSplits = 64;
constexpr int kMaxContext = 0x7fffffff - 4 * kTile;  // so that rounding up to chunks stays in range
// Exponentials are taken relative to a reference point kLift powers of two below the running maximum, and that
// point follows the maximum only when it has risen by more than kSlack: P reaches 2^(kLift + kSlack), half of
// fp16's range.  Without the lift, weights under 2^-14 of the largest would be subnormal and those under 2^-25 lost,
// which a long tail of them shows; with it these are 2^-21 and 2^-32.
constexpr float kSlack = 8.f;
constexpr float kLift = 7.f;
constexpr float kLog2e = 1.4426950408889634f;

struct Params {
  const void* q;
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  const float* k_scale;
  const float* v_scale;
  void* out;
  const int32_t* block_table;
  const int32_t* context_lens;
  float* ws_o;   // [batch, q_heads, splits, 128] un-normalised partial outputs
  float* ws_ml;  // [batch, q_heads, splits, 2] reference point (log2 domain) and sum
  int64_t q_stride, num_blocks, table_stride;
  int q_heads, kv_heads, group, block_size, max_blocks, num_splits;
  FastDiv by_block;
  bool chunk_in_page;  // pages are whole chunks
  float scale_log2;
};

// 2^x with results below 2^-126 flushed to zero.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Byte offset of 16-byte column `col` of token row `row` in a swizzled tile of 128-byte rows.
__device__ __forceinline__ uint32_t tile_offset(int row, int col) {
  return static_cast<uint32_t>(row * kDim + ((col ^ (row & 7)) << 4));
}

template <typename T, int kNT>
__global__ void __launch_bounds__(kThreads, Ring<kNT>::kCtas)
paged_attn_fp8_kernel(const Params p) {
  constexpr int kStages = Ring<kNT>::kStages;
  extern __shared__ __align__(128) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int split = blockIdx.x % p.num_splits;
  const int kvh = (blockIdx.x / p.num_splits) % p.kv_heads;
  const int seq = blockIdx.x / (p.num_splits * p.kv_heads);
  pdl_wait();
  pdl_launch_dependents();

  // The table row is on its way while the context length is being read.
  const int32_t* table = p.block_table + seq * p.table_stride;
  if (threadIdx.x * 32 < p.max_blocks) asm volatile("prefetch.global.L1 [%0];" ::"l"(table + threadIdx.x * 32));
  // A context never reaches past the pages the table row can name.
  const int ctx = static_cast<int>(min(static_cast<int64_t>(min(max(p.context_lens[seq], 0), kMaxContext)),
                                       static_cast<int64_t>(p.max_blocks) * p.block_size));
  // (Ranges of one length for all sequences, so that shorter contexts take fewer CTAs, measured 5 to 20 % slower.)
  int per_split = (ctx - 1) / p.num_splits + 1;
  per_split = ((per_split - 1) / kChunk + 1) * kChunk;
  const int t_begin = static_cast<int>(min(static_cast<int64_t>(split) * per_split, static_cast<int64_t>(ctx)));
  const int t_end = per_split < ctx - t_begin ? t_begin + per_split : ctx;
  const int num_chunks = (t_end - t_begin + kChunk - 1) / kChunk;

  const uint32_t ring = smem_addr(smem) + warp * kStages * kStageBytes;
  float* scales = reinterpret_cast<float*>(smem + Ring<kNT>::kBytes) + warp * kStages * 2 * kChunkTiles;
  const uint32_t scales_addr = smem_addr(scales);
  const int64_t row_bytes = static_cast<int64_t>(p.kv_heads) * kDim;

  // What a lane copies of every tile: column `col` of rows `row`, row + 4, row + 8, row + 12.
  const int row = lane >> 3, col = lane & 7;
  const uint32_t dst_even = ring + tile_offset(row, col), dst_odd = ring + tile_offset(row + 4, col);
  const int64_t row_at = row * row_bytes + kvh * kDim + col * 16;
  const int64_t v_minus_k = p.v_cache - p.k_cache;
  const int64_t four_rows = 4 * row_bytes;

  // Issues the copies of the CTA's chunk `ci` into ring slot `stage`.  A page outside the cache is
  // replaced by page 0, tokens past the range are filled with zeros (0 * NaN would poison the output).
  auto page_of = [&](int tok, int& off) {
    const int index = p.by_block(tok);
    const int page = table[index];
    off = tok - index * p.block_size;
    return page < 0 || page >= p.num_blocks ? 0 : page;
  };
  auto copy_tile = [&](const uint8_t* k, uint32_t to) {
#pragma unroll
    for (int j = 0; j < kTile / 4; ++j, k += four_rows) {
      const uint32_t dst = (j & 1 ? dst_odd : dst_even) + to + (j & ~1) * 4 * kDim;
      cp_async_16(dst, k, 16);
      cp_async_16(dst + kHalfBytes, k + v_minus_k, 16);
    }
  };
  auto issue = [&](int ci, int stage) {
    const int tok0 = t_begin + ci * kChunk;
    const uint32_t scales_to = scales_addr + stage * 2 * kChunkTiles * 4;
    if (ci < num_chunks && p.chunk_in_page && tok0 + kChunk <= t_end) {
      // A whole chunk, in one page.
      int off;
      const int page = page_of(tok0, off);
      const uint8_t* k = p.k_cache + (static_cast<int64_t>(page) * p.block_size + off) * row_bytes + row_at;
#pragma unroll
      for (int tile = 0; tile < kChunkTiles; ++tile, k += 4 * four_rows)
        copy_tile(k, stage * kStageBytes + tile * kTile * kDim);
      if (lane < 2 * kChunkTiles)
        cp_async_4(scales_to + lane * 4,
                   (lane & 1 ? p.v_scale : p.k_scale) + static_cast<int64_t>(page) * p.kv_heads + kvh);
    } else if (ci < num_chunks) {
#pragma unroll
      for (int tile = 0; tile < kChunkTiles; ++tile) {
        const int tok = tok0 + tile * kTile;
        int page = 0, off = 0;
        if (tok < t_end) page = page_of(tok, off);
        const uint8_t* k = p.k_cache + (static_cast<int64_t>(page) * p.block_size + off) * row_bytes + row_at;
        const uint32_t to = stage * kStageBytes + tile * kTile * kDim;
        if (tok + kTile <= t_end) {
          copy_tile(k, to);
        } else {
#pragma unroll
          for (int j = 0; j < kTile / 4; ++j) {
            const int bytes = tok + row + j * 4 < t_end ? 16 : 0;
            const uint8_t* from = bytes ? k + j * four_rows : p.k_cache;
            const uint32_t dst = (j & 1 ? dst_odd : dst_even) + to + (j & ~1) * 4 * kDim;
            cp_async_16(dst, from, bytes);
            cp_async_16(dst + kHalfBytes, from + v_minus_k, bytes);
          }
        }
        if (lane < 2)
          cp_async_4(scales_to + (tile * 2 + lane) * 4,
                     (lane ? p.v_scale : p.k_scale) + static_cast<int64_t>(page) * p.kv_heads + kvh);
      }
    }
    cp_async_commit();
  };

  // Warp w owns chunks w, w + kWarps, w + 2 * kWarps, ... of the CTA's range.
  const int my_chunks = num_chunks > warp ? (num_chunks - warp + kWarps - 1) / kWarps : 0;
  auto chunk_index = [&](int i) { return i < my_chunks ? warp + i * kWarps : num_chunks; };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) issue(chunk_index(s), s);

  // Query rows as B fragments: column n = head, and the contraction index of step 4 * i + w in lane t
  // is the dims (2 t + i) * 16 + 4 w .. + 3, the order in which the lane reads its tokens' codes.
  uint32_t qb[kNT][kDim / 16][2];
  float qmul[kNT][2];  // score factor of heads 2 t and 2 t + 1 (the columns of a lane's accumulators); its sign is in q
#pragma unroll
  for (int n = 0; n < kNT; ++n) {
    const bool live = n * 8 + g < p.group;
    const T* q = static_cast<const T*>(p.q) + seq * p.q_stride +
                 (static_cast<int64_t>(kvh) * p.group + (live ? n * 8 + g : 0)) * kDim;
    float x[2][16];
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 v = live ? *reinterpret_cast<const uint4*>(q + (2 * t + i) * 16 + h * 8) : make_uint4(0, 0, 0, 0);
        const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x[i][h * 8 + j] = Mma<T>::to_float(e[j]);
          const uint32_t b = __float_as_uint(x[i][h * 8 + j]) & 0x7fffffffu;
          amax = max(amax, b < 0x7f800000u ? b : 0u);
        }
      }
    }
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    // 2^up brings the row's largest value to [2^14, 2^15).
    const int up = amax >> 23 ? min(max(14 + 127 - static_cast<int>(amax >> 23), -126), 126) : 0;
    const float f = copysignf(__uint_as_float(static_cast<uint32_t>(127 + up) << 23), p.scale_log2);
    const float back = __uint_as_float(static_cast<uint32_t>(127 - up) << 23);
    qmul[n][0] = __shfl_sync(0xffffffffu, back, 8 * t) * fabsf(p.scale_log2);
    qmul[n][1] = __shfl_sync(0xffffffffu, back, 8 * t + 4) * fabsf(p.scale_log2);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        qb[n][i * 4 + w][0] = Mma<__half>::pack(x[i][4 * w] * f, x[i][4 * w + 1] * f);
        qb[n][i * 4 + w][1] = Mma<__half>::pack(x[i][4 * w + 2] * f, x[i][4 * w + 3] * f);
      }
  }

  // o[n][m]: dims g * 16 + 2 m (elements 0, 1) and g * 16 + 2 m + 1 (2, 3) of heads 2 t and 2 t + 1.
  float o[kNT][kDim / 16][4];
#pragma unroll
  for (int n = 0; n < kNT; ++n)
#pragma unroll
    for (int m = 0; m < kDim / 16; ++m)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[n][m][j] = 0.f;
  float mx[kNT][2], sum[kNT][2];  // reference point of the exponentials; this lane's part of the sum
#pragma unroll
  for (int n = 0; n < kNT; ++n) {
    mx[n][0] = mx[n][1] = -INFINITY;
    sum[n][0] = sum[n][1] = 0.f;
  }
  float unit = 1.f;  // V scale that o is expressed in

  for (int i = 0; i < my_chunks; ++i) {
    const int stage = i % kStages;
    issue(chunk_index(i + kStages - 1), (i + kStages - 1) % kStages);
    cp_async_wait<kStages - 1>();
    __syncwarp();
    const uint32_t ksm = ring + stage * kStageBytes, vsm = ksm + kHalfBytes;
    static_assert(kChunkTiles == 2, "the scales of a stage are K, V, K, V");
    const float4 sc = *reinterpret_cast<const float4*>(scales + stage * 2 * kChunkTiles);
    const float ks[kChunkTiles] = {usable_scale(sc.x), usable_scale(sc.z)};
    const float vs_of[kChunkTiles] = {usable_scale(sc.y), usable_scale(sc.w)};
    const int tok0 = t_begin + (warp + i * kWarps) * kChunk;

    float s[kChunkTiles][kNT][4];
#pragma unroll
    for (int tile = 0; tile < kChunkTiles; ++tile) {
#pragma unroll
      for (int n = 0; n < kNT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[tile][n][j] = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 lo = lds_16(ksm + tile_offset(tile * kTile + g, 2 * t + h));
        const uint4 hi = lds_16(ksm + tile_offset(tile * kTile + g + 8, 2 * t + h));
        const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t a[4];
          codes_to_half2(wl[w], a[0], a[2]);
          codes_to_half2(wh[w], a[1], a[3]);
#pragma unroll
          for (int n = 0; n < kNT; ++n) Mma<__half>::run(s[tile][n], a, qb[n][h * 4 + w][0], qb[n][h * 4 + w][1]);
        }
      }
    }
    const bool cut = tok0 + kChunk > t_end;  // tokens past the range do not count
    auto past = [&](int tile, int j) { return tok0 + tile * kTile + g + (j >> 1) * 8 >= t_end; };
    if (cut) {
#pragma unroll
      for (int tile = 0; tile < kChunkTiles; ++tile)
#pragma unroll
        for (int n = 0; n < kNT; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (past(tile, j)) s[tile][n][j] = -INFINITY;
    }
    // As long as the reference point stays where it is nothing has to be rescaled, and the lanes need not agree on the
    // chunk's maximum.  (A chunk holds at least one token of the range, so its maxima are finite.)  A score is rounded
    // to fp32 before it is compared, moves the reference point or is measured against that: a product kept exact in
    // one of these places would, from 2^24 on, be off the others by more than P has room for.
    uint32_t pb[kChunkTiles][kNT][2];  // P^T as B fragments
#pragma unroll
    for (int n = 0; n < kNT; ++n) {
      float top[2];  // this lane's maxima
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        top[c] = -INFINITY;
#pragma unroll
        for (int tile = 0; tile < kChunkTiles; ++tile) {
          const float f = qmul[n][c] * ks[tile];  // into the exp2 domain; not negative
          s[tile][n][c] = __fmul_rn(s[tile][n][c], f);
          s[tile][n][c + 2] = __fmul_rn(s[tile][n][c + 2], f);
          top[c] = fmaxf(top[c], fmaxf(s[tile][n][c], s[tile][n][c + 2]));
        }
      }
      if (__any_sync(0xffffffffu, top[0] - mx[n][0] > kLift + kSlack || top[1] - mx[n][1] > kLift + kSlack)) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          top[c] = fmaxf(top[c], __shfl_xor_sync(0xffffffffu, top[c], 4));
          top[c] = fmaxf(top[c], __shfl_xor_sync(0xffffffffu, top[c], 8));
          top[c] = fmaxf(top[c], __shfl_xor_sync(0xffffffffu, top[c], 16));
          top[c] = fmaxf(mx[n][c], top[c] - kLift);
          const float a = exp2_fast(mx[n][c] - top[c]);  // 0 on the first chunk
          mx[n][c] = top[c];
          sum[n][c] *= a;
#pragma unroll
          for (int m = 0; m < kDim / 16; ++m) {
            o[n][m][c] *= a;
            o[n][m][c + 2] *= a;
          }
        }
      }
#pragma unroll
      for (int tile = 0; tile < kChunkTiles; ++tile)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[tile][n][j] = exp2_fast(s[tile][n][j] - mx[n][j & 1]);
      if (cut) {  // also where the factor is 0
#pragma unroll
        for (int tile = 0; tile < kChunkTiles; ++tile)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (past(tile, j)) s[tile][n][j] = 0.f;
      }
#pragma unroll
      for (int tile = 0; tile < kChunkTiles; ++tile)
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[n][j & 1] += s[tile][n][j];
#pragma unroll
      for (int tile = 0; tile < kChunkTiles; ++tile) {
        pb[tile][n][0] = transpose_8x8(Mma<__half>::pack(s[tile][n][0], s[tile][n][1]));
        pb[tile][n][1] = transpose_8x8(Mma<__half>::pack(s[tile][n][2], s[tile][n][3]));
      }
    }
#pragma unroll
    for (int tile = 0; tile < kChunkTiles; ++tile) {
      const float vs = vs_of[tile];
      if (vs != unit && tok0 + tile * kTile < t_end) {
        const float f = unit / vs;
        unit = vs;
#pragma unroll
        for (int n = 0; n < kNT; ++n)
#pragma unroll
          for (int m = 0; m < kDim / 16; ++m)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[n][m][j] *= f;
      }
      uint32_t w[4][4];  // rows 2 t, 2 t + 1, 2 t + 8, 2 t + 9 of the tile, 16 dims each
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint4 v = lds_16(vsm + tile_offset(tile * kTile + 2 * t + (r & 1) + (r >> 1) * 8, g));
        w[r][0] = v.x; w[r][1] = v.y; w[r][2] = v.z; w[r][3] = v.w;
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        // Bytes of two tokens interleaved: each half is one dim's pair.
        const uint32_t lo0 = __byte_perm(w[0][q], w[1][q], 0x5140), lo1 = __byte_perm(w[0][q], w[1][q], 0x7362);
        const uint32_t hi0 = __byte_perm(w[2][q], w[3][q], 0x5140), hi1 = __byte_perm(w[2][q], w[3][q], 0x7362);
        uint32_t a0[4], a1[4];
        codes_to_half2(lo0, a0[0], a0[1]);
        codes_to_half2(hi0, a0[2], a0[3]);
        codes_to_half2(lo1, a1[0], a1[1]);
        codes_to_half2(hi1, a1[2], a1[3]);
#pragma unroll
        for (int n = 0; n < kNT; ++n) {
          Mma<__half>::run(o[n][2 * q], a0, pb[tile][n][0], pb[tile][n][1]);
          Mma<__half>::run(o[n][2 * q + 1], a1, pb[tile][n][0], pb[tile][n][1]);
        }
      }
    }
    __syncwarp();  // the slot is refilled by the next iteration's copies
  }
  cp_async_wait<0>();
  __syncthreads();

  // Merge the warps through shared memory (the ring is free now).  Columns are spread by two words in
  // 16 and rows by 20 against bank conflicts.
  constexpr int kHeads = kNT * 8, kPitch = kDim + 20;
  float* sm_o = reinterpret_cast<float*>(smem);              // [warps][kHeads][kPitch]
  float* sm_ml = sm_o + kWarps * kHeads * kPitch;            // [warps][kHeads][2]: reference point, sum
  float* sm_f = sm_ml + kWarps * kHeads * 2;                 // [kHeads][warps]: the warps' weights
  float* sm_total = sm_f + kHeads * kWarps;                  // [kHeads][2]: the CTA's reference point and sum
  float* sm_acc = sm_total + kHeads * 2;                     // [kHeads][128]: the CTA's output
#pragma unroll
  for (int n = 0; n < kNT; ++n) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float l = sum[n][c];
      l += __shfl_xor_sync(0xffffffffu, l, 4);
      l += __shfl_xor_sync(0xffffffffu, l, 8);
      l += __shfl_xor_sync(0xffffffffu, l, 16);
      const int row = warp * kHeads + n * 8 + 2 * t + c;
      float* wo = sm_o + row * kPitch + g * 18;
#pragma unroll
      for (int m = 0; m < kDim / 16; ++m)
        *reinterpret_cast<float2*>(wo + 2 * m) = make_float2(o[n][m][c] * unit, o[n][m][c + 2] * unit);
      if (g == 0) {
        sm_ml[row * 2] = mx[n][c];
        sm_ml[row * 2 + 1] = l;
      }
    }
  }
  __syncthreads();
  if (threadIdx.x < kHeads) {
    float2 ml[kWarps];
    float top = -INFINITY, l = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      ml[w] = *reinterpret_cast<const float2*>(sm_ml + (w * kHeads + threadIdx.x) * 2);
      top = fmaxf(top, ml[w].x);
    }
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = ml[w].y == 0.f ? 0.f : exp2f(ml[w].x - top);  // a warp without tokens has sum 0
      sm_f[threadIdx.x * kWarps + w] = f;
      l += f * ml[w].y;
    }
    sm_total[threadIdx.x * 2] = top;
    sm_total[threadIdx.x * 2 + 1] = l;
  }
  __syncthreads();
  const int64_t head0 = static_cast<int64_t>(seq) * p.q_heads + static_cast<int64_t>(kvh) * p.group;
  const bool in_cluster = p.num_splits > 1 && p.ws_o == nullptr;
#pragma unroll 2
  for (int i = threadIdx.x; i < p.group * kDim; i += kThreads) {
    const int r = i / kDim, d = i % kDim;
    const float* wo = sm_o + r * kPitch + d + 2 * (d / 16);
    float acc = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) acc += sm_f[r * kWarps + w] * wo[w * kHeads * kPitch];
    if (p.num_splits == 1) {
      // An empty context gives zeros (the reference divides 0 by 0 there).
      const float l = sm_total[r * 2 + 1];
      static_cast<T*>(p.out)[head0 * kDim + i] = Mma<T>::from_float(l == 0.f ? 0.f : acc / l);
    } else if (in_cluster) {
      sm_acc[i] = acc;
    } else {
      p.ws_o[((head0 + r) * p.num_splits + split) * kDim + d] = acc;
      if (d < 2) p.ws_ml[((head0 + r) * p.num_splits + split) * 2 + d] = sm_total[r * 2 + d];
    }
  }
  if (in_cluster) {
    // The splits of this (sequence, KV head) are the CTAs of one cluster: each finishes its share of the
    // outputs from all of them.
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    const int outputs = p.group * kDim, share = (outputs + p.num_splits - 1) / p.num_splits;
    const int end = min((split + 1) * share, outputs);
    for (int i = split * share + threadIdx.x; i < end; i += kThreads) {
      const int r = i / kDim;
      float2 ml[kMaxCluster];
      float v[kMaxCluster], top = -INFINITY, l = 0.f, acc = 0.f;
#pragma unroll
      for (int s = 0; s < kMaxCluster; ++s) {
        if (s < p.num_splits) {
          ml[s] = *reinterpret_cast<const float2*>(cluster.map_shared_rank(sm_total, s) + r * 2);
          v[s] = cluster.map_shared_rank(sm_acc, s)[i];
        }
      }
#pragma unroll
      for (int s = 0; s < kMaxCluster; ++s)
        if (s < p.num_splits) top = fmaxf(top, ml[s].x);
#pragma unroll
      for (int s = 0; s < kMaxCluster; ++s) {
        if (s < p.num_splits) {
          const float f = ml[s].y == 0.f ? 0.f : exp2f(ml[s].x - top);
          l += f * ml[s].y;
          acc += f * v[s];
        }
      }
      static_cast<T*>(p.out)[head0 * kDim + i] = Mma<T>::from_float(l == 0.f ? 0.f : acc / l);
    }
    cluster.sync();  // no CTA leaves while another may still read its part
  }
}

// Merges the splits of one (sequence, query head).  The splits' weights are worked out by one lane each.  kParts
// threads share a dimension, every kParts-th split each, so that all partial outputs are on their way at once: four
// where there are more than 16 splits (4 sequences x 16 heads x 64 splits: 2.3 us less), one otherwise (128 x 32
// heads x 4 splits: 9 us less).
template <typename T, int kMergeParts>
__global__ void __launch_bounds__(kDim * kMergeParts)
paged_attn_fp8_merge_kernel(const float* __restrict__ ws_o, const float* __restrict__ ws_ml,
                            T* __restrict__ out, int num_splits) {
  __shared__ float s_weight[kMaxSplits];
  __shared__ float s_sum, s_part[kMergeParts][kDim];
  pdl_wait();
  pdl_launch_dependents();
  const int64_t head = blockIdx.x;
  const int d = threadIdx.x % kDim, part = threadIdx.x / kDim;
  const float2* ml = reinterpret_cast<const float2*>(ws_ml) + head * num_splits;
  const float* o = ws_o + head * num_splits * kDim + d;
  constexpr int kEach = 16;  // splits of a thread
  static_assert(kMaxSplits <= 4 * kEach, "four parts take all splits");
  float v[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) v[i] = i * kMergeParts + part < num_splits ? o[(i * kMergeParts + part) * kDim] : 0.f;
  if (threadIdx.x < 32) {
    float2 w[kMaxSplits / 32];
    float top = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < kMaxSplits / 32; ++i) {
      w[i] = d + i * 32 < num_splits ? ml[d + i * 32] : make_float2(-INFINITY, 0.f);
      top = fmaxf(top, w[i].x);
    }
#pragma unroll
    for (int x = 16; x >= 1; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
#pragma unroll
    for (int i = 0; i < kMaxSplits / 32; ++i) {
      const float f = w[i].y == 0.f ? 0.f : exp2f(w[i].x - top);
      s_weight[d + i * 32] = f;
      l += f * w[i].y;
    }
#pragma unroll
    for (int x = 16; x >= 1; x >>= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
    if (d == 0) s_sum = l;
  }
  __syncthreads();
  float acc = 0.f;
#pragma unroll
  for (int i = 0; i < kEach; ++i)
    if (i * kMergeParts + part < num_splits) acc += s_weight[i * kMergeParts + part] * v[i];
  if (kMergeParts > 1) {
    s_part[part][d] = acc;
    __syncthreads();
  }
  if (part == 0) {
#pragma unroll
    for (int i = 1; i < kMergeParts; ++i) acc += s_part[i][d];
    const float l = s_sum;
    out[head * kDim + d] = Mma<T>::from_float(l == 0.f ? 0.f : acc / l);
  }
}

// Whether the splits of `pairs` (sequence, KV head) pairs merge inside the kernel.  Clusters start and end
// together, which costs more than the second kernel once CTAs have to share SMs (128 sequences x 8 heads x
// 8192 tokens in 8 splits: 338 us as clusters).
inline bool merges_in_cluster(int64_t pairs, int num_splits, int64_t sms) {
  return (num_splits == 2 || num_splits == 4 || num_splits == kMaxCluster) && pairs * num_splits <= sms;
}

template <typename T, int kNT>
int launch(const Params& p, int batch, cudaStream_t st) {
  const char* name = "paged_attn_varlen_fp8";
  const auto kernel = paged_attn_fp8_kernel<T, kNT>;
  const bool in_cluster = merges_in_cluster(static_cast<int64_t>(batch) * p.kv_heads, p.num_splits, sm_count());
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_shared_memory(kernel, Ring<kNT>::kSmemBytes, done);
  if (e != cudaSuccess) return fail(B200MOE_ERR_CUDA, "%s: %s", name, cudaGetErrorString(e));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(static_cast<int64_t>(batch) * p.kv_heads * p.num_splits));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Ring<kNT>::kSmemBytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = p.num_splits;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = in_cluster ? 2 : 1;
  cudaLaunchKernelEx(&cfg, kernel, p);
  if (int rc = check_launch(name)) return rc;
  if (p.num_splits > 1 && !in_cluster) {
    const bool many = p.num_splits > 16;
    launch_pdl(many ? paged_attn_fp8_merge_kernel<T, 4> : paged_attn_fp8_merge_kernel<T, 1>,
               dim3(static_cast<unsigned>(batch * p.q_heads)), dim3(many ? 4 * kDim : kDim), 0, st,
               static_cast<const float*>(p.ws_o), static_cast<const float*>(p.ws_ml), static_cast<T*>(p.out),
               p.num_splits);
    return check_launch("paged_attn_varlen_fp8 (merge)");
  }
  return B200MOE_OK;
}

}  // namespace
}  // namespace b200moe

extern "C" int b200moe_paged_attn_fp8_num_splits(int batch, int q_heads, int kv_heads, int64_t max_context) {
  using namespace b200moe;
  if (batch < 1 || kv_heads < 1 || q_heads < kv_heads || max_context < 1) return 1;
  // Estimated time of each number of splits, from measurements with 1 to 128 sequences of 100 to 60000
  // tokens (1 x 8 heads x 700 tokens: 7.7 us unsplit, 5.2 us in 8 splits; 16 x 8 x 8192: 54 us unsplit, 43 us
  // in 3; 128 x 8 x 8192: 275 us unsplit, 257 us in 4; 16 x 8 x 1024: 9.8 us unsplit, 10.8 us in 3).  In ns:
  // a CTA takes 6.0 a token when it has an SM to itself, 10.2 and 13.6 with one and two others beside it
  // (8.7 and 13 with two head tiles); beyond one wave the GPU is filled evenly, but for a last wave of half
  // a CTA's time and 1.2 us per CTA and wave; merging takes 1.5 us in a cluster, else 1.6 us and 40 ns a split.
  const bool wide = q_heads / kv_heads > 8;
  const int64_t pairs = static_cast<int64_t>(batch) * kv_heads, sms = sm_count();
  const int64_t slots = sms * (wide ? Ring<2>::kCtas : Ring<1>::kCtas);
  const double by_share[3] = {wide ? 8.7 : 6.0, wide ? 13.0 : 10.2, 13.6};
  int best = 1;
  double best_cost = 0;
  for (int s = 1; s <= kMaxSplits; ++s) {
    if (s > 1 && max_context < static_cast<int64_t>(s - 1) * kChunk) break;
    const int64_t ctas = pairs * s;
    const double tokens = static_cast<double>(max_context) / s;
    const int64_t per_sm = ceil_div64(ctas < slots ? ctas : slots, sms);
    double cost = tokens * by_share[per_sm - 1];
    if (ctas > slots) cost *= static_cast<double>(ctas) / slots + 0.5;
    if (ctas > slots) cost += 1200.0 * ctas / slots;
    if (s > 1) cost += merges_in_cluster(pairs, s, sms) ? 1500.0 : 1600.0 + 40.0 * s;
    if (s == 1 || cost < best_cost) { best = s; best_cost = cost; }
  }
  return best;
}

extern "C" size_t b200moe_paged_attn_fp8_workspace_bytes(int batch, int q_heads, int kv_heads, int num_splits) {
  using namespace b200moe;
  if (batch < 1 || q_heads < 1 || kv_heads < 1 || num_splits <= 1 || num_splits > kMaxSplits ||
      merges_in_cluster(static_cast<int64_t>(batch) * kv_heads, num_splits, sm_count()))
    return 0;
  return static_cast<size_t>(batch) * q_heads * num_splits * (kDim + 2) * sizeof(float);
}

extern "C" int b200moe_paged_attn_varlen_fp8(const void* q, const void* k_cache, const void* v_cache,
                                             const float* k_scale, const float* v_scale, void* out,
                                             const int32_t* block_table, const int32_t* context_lens,
                                             int dtype, int batch, int q_heads, int kv_heads,
                                             int head_dim, int64_t q_row_stride, int64_t num_blocks,
                                             int block_size, int max_blocks_per_seq,
                                             int64_t table_row_stride, float softmax_scale,
                                             int num_splits, void* workspace, size_t workspace_bytes,
                                             b200moe_stream_t stream) {
  using namespace b200moe;
  const char* name = "paged_attn_varlen_fp8";
  if (dtype != B200MOE_BF16 && dtype != B200MOE_F16)
    return fail(B200MOE_ERR_DTYPE, "%s: bf16 or fp16 queries only, got dtype %d", name, dtype);
  if (head_dim != kDim) return fail(B200MOE_ERR_SHAPE, "%s: head_dim must be 128, got %d", name, head_dim);
  if (batch < 0 || q_heads < 1 || kv_heads < 1 || q_heads % kv_heads != 0)
    return fail(B200MOE_ERR_SHAPE, "%s: batch=%d q_heads=%d kv_heads=%d (q_heads must be a multiple "
                "of kv_heads)", name, batch, q_heads, kv_heads);
  const int group = q_heads / kv_heads;
  if (group > kMaxGroup)
    return fail(B200MOE_ERR_UNSUPPORTED, "%s: at most %d query heads per KV head, got %d", name,
                kMaxGroup, group);
  if (block_size < kTile || block_size % kTile != 0)
    return fail(B200MOE_ERR_SHAPE, "%s: block_size must be a multiple of %d, got %d", name, kTile, block_size);
  if (num_blocks < 1 || num_blocks > 0x7fffffffLL || max_blocks_per_seq < 1 ||
      table_row_stride < max_blocks_per_seq || num_splits < 1 || num_splits > kMaxSplits)
    return fail(B200MOE_ERR_SHAPE, "%s: num_blocks=%lld max_blocks_per_seq=%d (row stride %lld) num_splits=%d",
                name, (long long)num_blocks, max_blocks_per_seq, (long long)table_row_stride, num_splits);
  if (q_row_stride < static_cast<int64_t>(q_heads) * head_dim)
    return fail(B200MOE_ERR_SHAPE, "%s: query row stride %lld smaller than a row", name, (long long)q_row_stride);
  if (batch == 0) return B200MOE_OK;
  if (!q || !k_cache || !v_cache || !k_scale || !v_scale || !out || !block_table || !context_lens)
    return fail(B200MOE_ERR_NULL, "%s: null pointer", name);
  if (!aligned_to(q, 16) || q_row_stride % 8 != 0 || !aligned_to(k_cache, 16) || !aligned_to(v_cache, 16))
    return fail(B200MOE_ERR_ALIGN, "%s: q, its row stride and the caches must be 16-byte aligned", name);
  if (static_cast<int64_t>(batch) * kv_heads * num_splits > 0x7fffffffLL ||
      static_cast<int64_t>(batch) * q_heads > 0x7fffffffLL)
    return fail(B200MOE_ERR_SHAPE, "%s: too many CTAs", name);
  Params p;
  p.q = q; p.out = out; p.q_stride = q_row_stride;
  p.k_cache = static_cast<const uint8_t*>(k_cache); p.v_cache = static_cast<const uint8_t*>(v_cache);
  p.k_scale = k_scale; p.v_scale = v_scale;
  p.block_table = block_table; p.context_lens = context_lens; p.table_stride = table_row_stride;
  p.ws_o = nullptr; p.ws_ml = nullptr;
  p.q_heads = q_heads; p.kv_heads = kv_heads; p.group = group; p.block_size = block_size;
  p.max_blocks = max_blocks_per_seq; p.num_splits = num_splits; p.num_blocks = num_blocks;
  p.scale_log2 = softmax_scale * kLog2e;
  p.by_block = FastDiv::by(static_cast<uint32_t>(block_size));
  p.chunk_in_page = block_size % kChunk == 0;
  const size_t need = b200moe_paged_attn_fp8_workspace_bytes(batch, q_heads, kv_heads, num_splits);
  if (need > 0) {
    if (!workspace || workspace_bytes < need || !aligned_to(workspace, 16))
      return fail(B200MOE_ERR_WORKSPACE, "%s: num_splits=%d needs a 16-byte aligned workspace of "
                  "%zu bytes, got %zu", name, num_splits, need, workspace_bytes);
    p.ws_o = static_cast<float*>(workspace);
    p.ws_ml = p.ws_o + static_cast<size_t>(batch) * q_heads * num_splits * kDim;
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == B200MOE_BF16)
    return group <= 8 ? launch<__nv_bfloat16, 1>(p, batch, st) : launch<__nv_bfloat16, 2>(p, batch, st);
  return group <= 8 ? launch<__half, 1>(p, batch, st) : launch<__half, 2>(p, batch, st);
}
