// The whole mixture-of-experts layer for a few tokens (1 to 32), in two kernels.
//
//   kernel 1   act[p, j] = weight_p * silu(x_t . w13[e, j]) * (x_t . w13[e, inter + j])
//   kernel 2   out[t, h] = bf16( sum over the token's two pairs p of  act[p] . w2[e, h] )
//
// p = (t, e) runs over the pairs that the router (softmax, top-2) picks; both kernels route for themselves
// from the logits, 32 lanes for 32 tokens, which is cheaper than handing the result over.
//
// The grouped GEMMs of this library pad every expert to 128 rows and go through six launches; with a few
// tokens all that counts is to read the weights of the experts that were hit, once, at the rate of HBM:
// 6 * H * I bytes an expert.  So the weights are the 16-row operand of m16n8k16 and the tokens its 8
// columns; a tile is 16 or 32 weight rows with the whole contraction, split over the eight warps of a CTA.
// Each warp streams 4 KiB of weights per step, with the tokens' elements that belong to them, through a ring of
// its own (asynchronous 16-byte copies, 192 KiB an SM), never waiting for another warp except to add up a
// finished tile (kernel 1 with a short contraction: each warp has its own tiles; kernel 2 with few tiles: a
// thread-block cluster shares one).  Tiles are dealt round-robin; that some CTAs get one more does not cost much,
// because an SM alone can draw well over 1/148 of the HBM rate.
//
// * Fragments come from matrix loads, whose registers are the products' operands as they are (16-byte
//   reads of a row and a permuted contraction index need as many reads, and four moves for each product).
// * A tile of kernel 1 has 8 gate rows over the 8 matching up rows in each 16, so that gate and up of one
//   element meet in one lane's accumulators.
// * Only the tokens that are routed to a tile's expert are copied and multiplied: columns are their places
//   in the expert's list.  A stage has room for 16; an expert with more is gone through twice, its weights
//   then coming from L2.  Kernel 2 adds its columns to the tokens' sums whenever the expert changes.
// * Up to 8 tokens take 16-row tiles (the finest deal); more take 32-row tiles, which halve the copies of
//   tokens per weight.
// * act is kept as the sum of two bf16 numbers (16 bits of mantissa): kernel 2 multiplies both by
//   the weights and adds in fp32, so that the only rounding that shows is the output's.
// * Kernel 2 is launched with programmatic stream serialisation and fills its rings with w2 before it
//   waits for kernel 1.
//
// Measured at hidden 4096: 32 tokens and width 14336 415 us (6.8 TB/s of weights), 7 tokens 336 us, one token and width
// 1792 19.8 us; the general path takes 464 us for 32 tokens, 58 us for the one.  The reference runs the same batch through its general path (layers/moe/fused_moe.py:170-293).
#include <cooperative_groups.h>
#include <type_traits>

#include "warp_mma.cuh"

namespace b200moe {
namespace {

namespace cg = cooperative_groups;

constexpr int kExperts = 8;
constexpr int kMaxCluster = 8;
constexpr int kMaxTokens = 32;
constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kWeightBytes = 4096;     // weights of a ring stage
constexpr int kGroup = 16;             // tokens of a ring stage
constexpr int kRingBytes = 192 * 1024;

struct Params {
  const __nv_bfloat16* x;
  const void* logits;
  const __nv_bfloat16* w;  // w13 or w2
  uint4* act;              // [2 * tokens][inter / 8][2]: eight high parts, eight low parts
  __nv_bfloat16* out;
  int tokens, hidden, inter, logits_dtype, renormalize;
  int cluster;  // CTAs that share the contraction of a tile of kernel 2
};

// Experts that were hit, in ascending order, and their tokens.
struct Routing {
  int num_active;
  int expert[kExperts];                 // number of the a-th active expert
  int count[kExperts];                  // its tokens
  int begin[kExperts + 1];              // prefix of (units * groups of tokens), see the kernel
  int8_t token[kExperts][kMaxTokens];   // its tokens, ascending
  int8_t pair[kExperts][kMaxTokens];    // the pairs' indices, in the same order
  float weight[kExperts][kMaxTokens];   // and their routing weights
};

__device__ __forceinline__ float load_logit(const void* p, int dtype, int i) {
  if (dtype == B200MOE_F32) return static_cast<const float*>(p)[i];
  if (dtype == B200MOE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}

// Softmax and top-2 of up to 32 tokens, one lane each (one warp).  Equal logits: the lower index wins.
// `units`: tiles or steps of one expert, of which the sequence that r.begin divides is made.
__device__ void route(const Params& p, Routing& r, int units) {
  const int t = threadIdx.x;
  int first = -1, second = -1;
  float w1 = 0.f, w2 = 0.f;
  if (t < p.tokens) {
    float v[kExperts];
#pragma unroll
    for (int e = 0; e < kExperts; ++e) v[e] = load_logit(p.logits, p.logits_dtype, t * kExperts + e);
    float b1 = v[0], b2 = -INFINITY;
    first = 0;
#pragma unroll
    for (int e = 1; e < kExperts; ++e) {
      if (v[e] > b1) { b2 = b1; second = first; b1 = v[e]; first = e; }
      else if (v[e] > b2) { b2 = v[e]; second = e; }
    }
    if (second < 0) second = first == 0 ? 1 : 0;  // nothing above -inf is left
    const float e2 = expf(b2 - b1);
    float sum = 1.f + e2;
    if (!p.renormalize) {
      sum = 0.f;
#pragma unroll
      for (int e = 0; e < kExperts; ++e) sum += expf(v[e] - b1);
    }
    w1 = 1.f / sum;
    w2 = e2 / sum;
  }
  int n = 0, at = 0;
#pragma unroll
  for (int e = 0; e < kExperts; ++e) {
    const int slot = first == e ? 0 : second == e ? 1 : -1;
    const uint32_t hit = __ballot_sync(0xffffffffu, slot >= 0);
    if (hit == 0) continue;
    const int rank = __popc(hit & ((1u << t) - 1));
    if (slot >= 0) {
      r.token[n][rank] = static_cast<int8_t>(t);
      r.pair[n][rank] = static_cast<int8_t>(2 * t + slot);
      r.weight[n][rank] = slot == 0 ? w1 : w2;
    }
    const int count = __popc(hit);
    if (t == 0) {
      r.expert[n] = e;
      r.count[n] = count;
      r.begin[n] = at;
    }
    at += units * ((count + kGroup - 1) / kGroup);
    ++n;
  }
  if (t == 0) {
    r.num_active = n;
    r.begin[n] = at;
  }
}

// A warp's way through the sequence of (active expert, unit, group of tokens).  Kernel 1: units are tiles, and
// the groups of one tile follow one another, so that its weights come from L2 the second time.  Kernel 2: units
// are contraction steps, and the groups go through all of them one after the other, so that the columns
// change seldom (an expert's rows of a tile stay in L2).
template <bool kDown>
struct Place {
  int a, until, unit, group;  // `until`: end of the part of the sequence with the same expert and (kernel 2) group
  // Moves forward to position `at` of the sequence.
  __device__ __forceinline__ void seek(const Routing& r, int at, int units) {
    while (at >= r.begin[a + 1]) ++a;
    const int rest = at - r.begin[a];
    const bool two = r.count[a] > kGroup;
    if (kDown) {
      group = two && rest >= units ? 1 : 0;
      unit = rest - group * units;
      until = r.begin[a] + (group + 1) * units;
    } else {
      unit = two ? rest >> 1 : rest;
      group = two ? rest & 1 : 0;
      until = r.begin[a + 1];
    }
  }
};

// kCT = tiles of 8 tokens that a stage has room for, kRT = tiles of 16 weight rows.
// kAlone (kernel 1): a warp takes whole tiles by itself instead of an eighth of every tile.
template <int kCT_, int kRT_, bool kDown_, bool kAlone_>
struct Shape {
  static constexpr int kCT = kCT_, kRT = kRT_;
  static constexpr bool kDown = kDown_, kAlone = kAlone_;
  static constexpr int kStep = 128 / kRT;                      // contraction elements of a stage
  static constexpr int kPieces = kStep / 8;                    // 16-byte pieces of a weight row
  static constexpr int kParts = kDown ? 2 : 1;                 // numbers that an element is the sum of
  static constexpr int kSlots = 8 * kCT;                       // tokens that a stage has room for
  static constexpr int kTokenPieces = kPieces * kParts;
  static constexpr int kStageBytes = kWeightBytes + kSlots * kTokenPieces * 16;
  static constexpr int kStages = kRingBytes / kWarps / kStageBytes;
  static constexpr int kRows = 16 * kRT;
  static constexpr int kSets = kCT * kRT == 1 ? 2 : 1;         // accumulator sets, against dependent products
  static constexpr int kMaxT = kCT == 1 ? 8 : kMaxTokens;      // tokens of the batch
  // What the warps add up through: kernel 1 two buffers of accumulators, kernel 2 a tile per warp.
  static constexpr int kSumFloats = kDown ? kRows * kMaxT : kAlone ? 4 : 2 * kRT * kCT * 32 * 4;
  static_assert(kStages >= 2, "the ring is too small");
};

// Byte offsets in a stage: piece `col` of weight row `row`; piece `piece` of token slot `slot`.  Eight rows or
// slots in a row never meet in a bank.
template <typename S> __device__ __forceinline__ uint32_t weight_offset(int row, int col) {
  return static_cast<uint32_t>((row * S::kPieces + (col ^ (row & 7))) * 16);
}
template <typename S> __device__ __forceinline__ uint32_t token_offset(int slot, int piece) {
  return static_cast<uint32_t>(kWeightBytes + (slot * S::kTokenPieces + (piece ^ (slot & 7))) * 16);
}

template <typename S>
__global__ void __launch_bounds__(kThreads, 1)
few_tokens_kernel(const Params p) {
  constexpr int kCT = S::kCT, kRT = S::kRT;
  constexpr bool kDown = S::kDown;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Routing r;
  __shared__ __align__(16) float s_sum[kWarps * S::kSumFloats];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int K = kDown ? p.inter : p.hidden;
  const int steps = (K + S::kStep - 1) / S::kStep;                             // of one expert
  const int expert_tiles = kDown ? p.hidden / S::kRows : p.inter / (S::kRows / 2);
  // Kernel 2 may look at the logits before kernel 1 is through: kernel 1 lets it start only after its own
  // wait, that is after everything before it in the stream has finished.
  if (!kDown) pdl_wait();
  if (warp == 0) route(p, r, kDown ? steps : expert_tiles);
  if (kDown)
    for (int i = threadIdx.x; i < kWarps * S::kSumFloats; i += kThreads) s_sum[i] = 0.f;
  __syncthreads();
  pdl_launch_dependents();

  const int chunks = kDown ? r.begin[r.num_active] : steps;                    // of one tile
  const int tiles = kDown ? expert_tiles : r.begin[r.num_active];
  const int units = kDown ? steps : expert_tiles;
  // The warp's chunks of a tile: every eighth (kernel 1; kernel 2: of those of the cluster that works on the tile,
  // side by side for the sake of DRAM pages), all (kernel 1, alone), or, where an expert has too few for that, a
  // range, so that the columns do not change all the time.
  const int shares = kDown ? p.cluster * kWarps : S::kAlone ? 1 : kWarps;
  const int share = kDown ? static_cast<int>(blockIdx.x % p.cluster) * kWarps + warp : S::kAlone ? 0 : warp;
  const bool range = kDown && steps < 8 * shares;
  const int next_chunk = range ? 1 : shares;
  const int chunk0 = range ? static_cast<int>(static_cast<int64_t>(chunks) * share / shares) : share;
  const int my_chunks = range ? static_cast<int>(static_cast<int64_t>(chunks) * (share + 1) / shares) - chunk0
                      : chunks > share ? (chunks - share + shares - 1) / shares : 0;
  const int tile0 = kDown ? blockIdx.x / p.cluster : S::kAlone ? warp * gridDim.x + blockIdx.x : blockIdx.x;
  const int tile_step = kDown ? gridDim.x / p.cluster : S::kAlone ? gridDim.x * kWarps : gridDim.x;
  const uint32_t ring = smem_addr(smem) + warp * S::kStages * S::kStageBytes;
  const int64_t row_bytes = static_cast<int64_t>(K) * 2;
  const int64_t expert_rows = kDown ? p.hidden : 2 * static_cast<int64_t>(p.inter);

  // ---- The copying side.  The warp's chunks of all its tiles are one sequence; what a lane copies of a
  // chunk is at fixed distances from what it copied of the last one, until the expert or the tile changes.
  constexpr int kRowsAtOnce = 32 / S::kPieces;                     // weight rows of one copy instruction
  constexpr int kTokenCopies = S::kSlots * S::kTokenPieces / 32;   // copy instructions of the tokens
  const int w_row = lane / S::kPieces, w_col = lane % S::kPieces;
  Place<kDown> ahead = {0, 0, 0, 0};
  int ahead_tile = my_chunks ? tile0 : tiles, ahead_chunk = 0, filled = 0;
  int step = 0;                        // contraction step of the next chunk
  const uint8_t* w_src = nullptr;      // of the next chunk
  const uint8_t* t_src[kTokenCopies];
  int live = 0;                        // tokens of the group

  auto locate = [&]() {  // the next chunk has another expert, group or tile than the last one
    ahead.seek(r, kDown ? chunk0 + ahead_chunk * next_chunk : ahead_tile, units);
    step = kDown ? ahead.unit : chunk0;
    const int row0 = kDown ? ahead_tile * S::kRows : ahead.unit * (S::kRows / 2);
    w_src = reinterpret_cast<const uint8_t*>(p.w) + (r.expert[ahead.a] * expert_rows + row0 + w_row) * row_bytes +
            (static_cast<int64_t>(step) * S::kStep + w_col * 8) * 2;
    live = min(r.count[ahead.a] - ahead.group * kGroup, kGroup);
#pragma unroll
    for (int i = 0; i < kTokenCopies; ++i) {
      const int slot = (i * 32 + lane) / S::kTokenPieces, piece = (i * 32 + lane) % S::kTokenPieces;
      const int at = ahead.group * kGroup + slot;
      const int token = slot < live ? r.token[ahead.a][at] : 0;
      const int64_t k = static_cast<int64_t>(step) * S::kStep + piece / S::kParts * 8;
      t_src[i] = kDown ? reinterpret_cast<const uint8_t*>(p.act) +
                             (static_cast<int64_t>(slot < live ? r.pair[ahead.a][at] : 0) * p.inter + k) * 4 +
                             piece % S::kParts * 16
                       : reinterpret_cast<const uint8_t*>(p.x) + (static_cast<int64_t>(token) * p.hidden + k) * 2;
    }
  };
  const int64_t rows_down = kRowsAtOnce * row_bytes;
  // Kernel 1: rows 16 m + 0..7 of a tile are gate rows 8 m + 0..7, rows 16 m + 8..15 the same up rows.
  const int64_t gate_to_up = (p.inter - 8 + kRowsAtOnce) * row_bytes;
  const int64_t up_to_gate = (kRowsAtOnce - p.inter) * row_bytes;
  // kRows rows x kStep elements of weights; zeros past K.
  auto issue_weights = [&](uint32_t to) {
    const uint8_t* src = w_src;
    const uint32_t dst = to + weight_offset<S>(w_row, w_col), dst_odd = to + weight_offset<S>(w_row + 4, w_col);
    const int bytes = (step + 1) * S::kStep <= K || step * S::kStep + w_col * 8 < K ? 16 : 0;
    if (bytes == 0) src = reinterpret_cast<const uint8_t*>(p.w);
#pragma unroll
    for (int j = 0; j < S::kRows / kRowsAtOnce; ++j) {
      const int base = j * kRowsAtOnce;  // rows base + w_row of the tile
      if (kRowsAtOnce == 4) {
        // Rows 4 apart differ in the swizzle, rows 8 apart do not.
        cp_async_16((base & 4 ? dst_odd : dst) + (base & ~7) * S::kPieces * 16, src, bytes);
      } else {
        cp_async_16(to + weight_offset<S>(base + w_row, w_col), src, bytes);
      }
      const int next = base + kRowsAtOnce;
      if (bytes) src += kDown || next % 8 != 0 ? rows_down : next % 16 == 8 ? gate_to_up : up_to_gate;
    }
  };
  // The elements of the group's tokens that belong to them.
  auto issue_tokens = [&](uint32_t to) {
    const bool whole = (step + 1) * S::kStep <= K;
#pragma unroll
    for (int i = 0; i < kTokenCopies; ++i) {
      const int slot = (i * 32 + lane) / S::kTokenPieces, piece = (i * 32 + lane) % S::kTokenPieces;
      if (slot < live) {
        const bool inside = whole || step * S::kStep + piece / S::kParts * 8 < K;
        cp_async_16(to + token_offset<S>(slot, piece), inside ? t_src[i] : reinterpret_cast<const uint8_t*>(p.w),
                    inside ? 16 : 0);
      }
    }
  };
  auto advance = [&]() {
    filled = filled + 1 == S::kStages ? 0 : filled + 1;
    if (ahead_tile >= tiles) return;
    if (++ahead_chunk >= my_chunks) {
      ahead_chunk = 0;
      ahead_tile += tile_step;
      if (kDown) ahead.a = 0;
      if (ahead_tile < tiles) locate();
    } else if (kDown && chunk0 + ahead_chunk * next_chunk >= ahead.until) {
      locate();
    } else {
      step += next_chunk;
      const uint32_t bytes = static_cast<uint32_t>(next_chunk) * (S::kStep * 2);
      w_src += bytes;
#pragma unroll
      for (int i = 0; i < kTokenCopies; ++i) t_src[i] += bytes * S::kParts;
    }
  };
  auto issue_next = [&]() {
    if (ahead_tile < tiles) {
      issue_weights(ring + filled * S::kStageBytes);
      issue_tokens(ring + filled * S::kStageBytes);
    }
    cp_async_commit();
    advance();
  };
  if (ahead_tile < tiles) locate();
  if constexpr (kDown) {
    // Weights first, then, once kernel 1 is through, the activations that go with them.
    for (int s = 0; s < S::kStages - 1; ++s) {
      if (ahead_tile < tiles) issue_weights(ring + filled * S::kStageBytes);
      advance();
    }
    ahead_tile = my_chunks ? tile0 : tiles; ahead_chunk = 0; filled = 0; ahead.a = 0;
    if (ahead_tile < tiles) locate();
    pdl_wait();
    for (int s = 0; s < S::kStages - 1; ++s) {
      if (ahead_tile < tiles) issue_tokens(ring + filled * S::kStageBytes);
      cp_async_commit();
      advance();
    }
  } else {
#pragma unroll 1
    for (int s = 0; s < S::kStages - 1; ++s) issue_next();
  }

  // ---- The computing side.  Columns of the products are the slots of a stage; what is left in slots
  // without a token stays in columns that nobody reads.
  // Matrix loads: lane l names row l % 8 of matrix l / 8.  Weights: rows 0..7 and 8..15 of 8 elements, then
  // the same of the next 8.  Tokens: eight slots of 8 elements, four times in a row.
  const int m_row = lane & 15, m_col = lane >> 4;
  int stage = 0, parity = 0, here_live = 0;
  Place<kDown> here = {0, 0, 0, 0};
  float acc[S::kSets][kRT][kCT][4];
  auto clear = [&]() {
#pragma unroll
    for (int s = 0; s < S::kSets; ++s)
#pragma unroll
      for (int m = 0; m < kRT; ++m)
#pragma unroll
        for (int n = 0; n < kCT; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[s][m][n][j] = 0.f;
  };
  auto look_up = [&](int at) {
    here.seek(r, at, units);
    here_live = min(r.count[here.a] - here.group * kGroup, kGroup);
  };
  // Element (row, token) of a warp's tile in kernel 2; rows shifted against bank conflicts.
  auto sum_at = [&](int w, int row, int token) -> float& {
    return s_sum[w * S::kSumFloats + row * S::kMaxT + (token ^ ((row & 7) << 2) % S::kMaxT)];
  };
  // Kernel 2, when the expert or the group changes: adds the columns to the tokens they belong to.
  auto flush = [&]() {
#pragma unroll
    for (int n = 0; n < kCT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int slot = n * 8 + 2 * t + c;
        if (slot < here_live) {
          const int token = r.token[here.a][here.group * kGroup + slot];
#pragma unroll
          for (int m = 0; m < kRT; ++m) {
            float lo = acc[0][m][n][c], hi = acc[0][m][n][c + 2];
            if (S::kSets == 2) { lo += acc[S::kSets - 1][m][n][c]; hi += acc[S::kSets - 1][m][n][c + 2]; }
            sum_at(warp, m * 16 + g, token) += lo;
            sum_at(warp, m * 16 + g + 8, token) += hi;
          }
        }
      }
    clear();
  };
  // Products of one stage with the first kN column tiles.
  auto multiply = [&](uint32_t at, auto tiles_of_8) {
    constexpr int kN = decltype(tiles_of_8)::value;
#pragma unroll
    for (int kk = 0; kk < S::kStep / 32; ++kk) {
      uint32_t a[2][kRT][4], b[kN][S::kParts][4];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int m = 0; m < kRT; ++m)
          ldmatrix_x4(a[h][m], at + weight_offset<S>(m * 16 + m_row, kk * 4 + h * 2 + m_col));
#pragma unroll
      for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int part = 0; part < S::kParts; ++part)
          ldmatrix_x4(b[n][part], at + token_offset<S>(n * 8 + (lane & 7), (kk * 4 + (lane >> 3)) * S::kParts + part));
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int part = 0; part < S::kParts; ++part)
#pragma unroll
          for (int n = 0; n < kN; ++n)
#pragma unroll
            for (int m = 0; m < kRT; ++m)
              Mma<__nv_bfloat16>::run(acc[h * (S::kSets - 1)][m][n], a[h][m], b[n][part][2 * h], b[n][part][2 * h + 1]);
    }
  };

  for (int tile = tile0; tile < tiles; tile += tile_step) {
    clear();
    if (kDown) { here = {0, 0, 0, 0}; here_live = 0; } else look_up(tile);

    for (int i = 0; i < my_chunks; ++i) {
      if (kDown && chunk0 + i * next_chunk >= here.until) {
        flush();
        look_up(chunk0 + i * next_chunk);
      }
      issue_next();
      cp_async_wait<S::kStages - 1>();
      __syncwarp();
      const uint32_t at = ring + stage * S::kStageBytes;
      if (kCT == 1 || here_live <= 8) multiply(at, std::integral_constant<int, 1>());
      else multiply(at, std::integral_constant<int, kCT>());
      __syncwarp();  // the stage is refilled by a later iteration's copies
      stage = stage + 1 == S::kStages ? 0 : stage + 1;
    }

    // Add the warps up, in their order.
    if constexpr (kDown) {
      flush();
      __syncthreads();
      if (p.cluster == 1) {
        for (int i = threadIdx.x; i < S::kRows * S::kMaxT; i += kThreads) {
          const int row = i % S::kRows, token = i / S::kRows;
          float v = 0.f;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) {
            v += sum_at(w, row, token);
            sum_at(w, row, token) = 0.f;
          }
          if (token < p.tokens)
            p.out[static_cast<int64_t>(token) * p.hidden + tile * S::kRows + row] = __float2bfloat16_rn(v);
        }
        __syncthreads();
      } else {
        // Every CTA of the cluster adds up its warps in place of the first, then a share of the tile over the
        // CTAs, in their order.
        for (int i = threadIdx.x; i < S::kRows * S::kMaxT; i += kThreads) {
          const int row = i % S::kRows, token = i / S::kRows;
          float v = 0.f;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) {
            v += sum_at(w, row, token);
            sum_at(w, row, token) = 0.f;
          }
          sum_at(0, row, token) = v;
        }
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        const int outputs = S::kRows * p.tokens, rank = static_cast<int>(blockIdx.x % p.cluster);
        for (int i = rank * kThreads + threadIdx.x; i < outputs; i += p.cluster * kThreads) {
          const int row = i % S::kRows, token = i / S::kRows;
          float v = 0.f;
          for (int c = 0; c < p.cluster; ++c) v += *cluster.map_shared_rank(&sum_at(0, row, token), c);
          p.out[static_cast<int64_t>(token) * p.hidden + tile * S::kRows + row] = __float2bfloat16_rn(v);
        }
        cluster.sync();
        for (int i = threadIdx.x; i < S::kSumFloats; i += kThreads) s_sum[i] = 0.f;
        __syncthreads();
      }
    } else {
      // Gate element g and up element g of row tile m (v.x, v.y and v.z, v.w), for slots 2 t and 2 t + 1 of column
      // tile n.
      auto finish = [&](int m, int n, float4 v) {
        const float gate[2] = {v.x, v.y}, up[2] = {v.z, v.w};
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int slot = n * 8 + 2 * t + c, place = here.group * kGroup + slot;
          if (slot < here_live) {
            const float value = r.weight[here.a][place] * (gate[c] / (1.f + expf(-gate[c])) * up[c]);
            const __nv_bfloat16 high = __float2bfloat16_rn(value);
            const float rest = __hisinf(high) ? 0.f : value - __bfloat162float(high);  // not inf - inf
            __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(
                p.act + (static_cast<int64_t>(r.pair[here.a][place]) * (p.inter / 8) + here.unit * kRT + m) * 2);
            o[g] = high;
            o[8 + g] = __float2bfloat16_rn(rest);
          }
        }
      };
      auto own = [&](int m, int n) {
        float4 v = make_float4(acc[0][m][n][0], acc[0][m][n][1], acc[0][m][n][2], acc[0][m][n][3]);
        if (S::kSets == 2) {
          v.x += acc[S::kSets - 1][m][n][0]; v.y += acc[S::kSets - 1][m][n][1];
          v.z += acc[S::kSets - 1][m][n][2]; v.w += acc[S::kSets - 1][m][n][3];
        }
        return v;
      };
      if constexpr (S::kAlone) {
#pragma unroll
        for (int m = 0; m < kRT; ++m)
#pragma unroll
          for (int n = 0; n < kCT; ++n) finish(m, n, own(m, n));
      } else {
        // Two buffers in turn make one barrier per tile enough.
        float4* sums = reinterpret_cast<float4*>(s_sum) + parity * kWarps * kRT * kCT * 32;
        parity ^= 1;
#pragma unroll
        for (int m = 0; m < kRT; ++m)
#pragma unroll
          for (int n = 0; n < kCT; ++n) sums[(warp * kRT * kCT + m * kCT + n) * 32 + lane] = own(m, n);
        __syncthreads();
        if (warp < kRT * kCT) {
          float4 v = sums[warp * 32 + lane];
#pragma unroll
          for (int w = 1; w < kWarps; ++w) {
            const float4 o = sums[(w * kRT * kCT + warp) * 32 + lane];
            v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
          }
          finish(warp / kCT, warp % kCT, v);
        }
      }
    }
  }
  cp_async_wait<0>();
}

template <typename S>
int launch(Params p, const void* w, int64_t tiles, int cluster, cudaStream_t st) {
  const char* name = "moe_few_tokens";
  const auto kernel = few_tokens_kernel<S>;
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_shared_memory(kernel, kRingBytes, done);
  if (e != cudaSuccess) return fail(B200MOE_ERR_CUDA, "%s: %s", name, cudaGetErrorString(e));
  const int64_t sms = sm_count();
  p.cluster = cluster;
  p.w = static_cast<const __nv_bfloat16*>(w);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((tiles < sms ? tiles : sms) * cluster));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kRingBytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  cudaLaunchKernelEx(&cfg, kernel, p);
  return check_launch(name);
}

template <int kCT, int kRT>
int launch_up(const Params& p, const void* w13, int experts_hit, cudaStream_t st) {
  const int64_t tiles = static_cast<int64_t>(experts_hit) * p.inter / (8 * kRT), sms = sm_count();
  const int steps = (p.hidden + 128 / kRT - 1) / (128 / kRT);
  // Where a tile has no more steps than the CTA has warps, adding them up takes longer than the tile: with tiles
  // for every warp of the GPU, each warp takes its own (8 tokens, hidden 256, width 14336: 96 us together, 43
  // alone; hidden 1024, width 3584: 37 and 32).  Longer tiles are better shared (hidden 4096, width 1792: 52
  // together, 55 alone), because they come out even.
  const bool alone = steps <= kWarps && tiles >= kWarps * sms;
  return alone ? launch<Shape<kCT, kRT, false, true>>(p, w13, tiles, 1, st)
               : launch<Shape<kCT, kRT, false, false>>(p, w13, tiles, 1, st);
}

template <int kCT, int kRT>
int launch_down(const Params& p, const void* w2, int experts_hit, cudaStream_t st) {
  const int64_t tiles = p.hidden / (16 * kRT);
  // Where there are tiles for half of the SMs or fewer, clusters of two to eight CTAs share them, as long as every
  // warp has eight steps (32 tokens, hidden 1024, width 3584: 57 us without clusters, 38 with them; 3 tokens,
  // hidden and width 256: 8.4 and 13.6, a cluster takes longer to start and to add up).
  const int64_t steps = static_cast<int64_t>(experts_hit) * (p.inter / (128 / kRT));
  int cluster = 1;
  while (cluster < kMaxCluster && tiles * cluster * 2 <= sm_count() && steps >= 8ll * kWarps * cluster * 2) cluster *= 2;
  return launch<Shape<kCT, kRT, true, false>>(p, w2, tiles, cluster, st);
}

// 32-row tiles where there are more than 8 tokens, the sizes allow it and, in kernel 2, tiles for three quarters of
// the SMs are left (16 tokens, hidden and width 2048: 49 us with 32-row tiles in kernel 2, 39 with 16-row tiles).
template <int kCT>
int launch(const Params& p, const void* w13, const void* w2, cudaStream_t st) {
  constexpr int kRT = kCT;
  const int experts_hit = 2 * p.tokens < kExperts ? 2 * p.tokens : kExperts;
  if (int rc = p.inter % (8 * kRT) == 0 ? launch_up<kCT, kRT>(p, w13, experts_hit, st)
                                        : launch_up<kCT, 1>(p, w13, experts_hit, st))
    return rc;
  const bool wide = p.hidden % (16 * kRT) == 0 && p.hidden / (16 * kRT) * 4 >= 3 * sm_count();
  return wide ? launch_down<kCT, kRT>(p, w2, experts_hit, st) : launch_down<kCT, 1>(p, w2, experts_hit, st);
}

}  // namespace
}  // namespace b200moe

extern "C" int b200moe_few_tokens_max(void) { return b200moe::kMaxTokens; }

extern "C" size_t b200moe_few_tokens_workspace_bytes(int64_t num_tokens, int64_t inter) {
  if (num_tokens < 1 || num_tokens > b200moe::kMaxTokens || inter < 1) return 0;
  return static_cast<size_t>(num_tokens) * 2 * static_cast<size_t>(inter) * 4;
}

extern "C" int b200moe_few_tokens(const void* hidden_states, const void* gating_output, int logits_dtype,
                                  const void* w13, const void* w2, void* output, int64_t num_tokens,
                                  int num_experts, int top_k, int64_t hidden, int64_t inter,
                                  int renormalize, void* workspace, size_t workspace_bytes,
                                  b200moe_stream_t stream) {
  using namespace b200moe;
  const char* name = "moe_few_tokens";
  if (num_experts != kExperts || top_k != 2)
    return fail(B200MOE_ERR_SHAPE, "%s: compiled for num_experts=8 and top_k=2, got %d and %d", name, num_experts, top_k);
  if (num_tokens < 0 || num_tokens > kMaxTokens)
    return fail(B200MOE_ERR_SHAPE, "%s: 0 to %d tokens, got %lld", name, kMaxTokens, (long long)num_tokens);
  if (hidden < 16 || hidden % 16 != 0 || inter < 8 || inter % 8 != 0 || hidden > (1 << 20) || inter > (1 << 20))
    return fail(B200MOE_ERR_SHAPE, "%s: hidden=%lld must be a multiple of 16 and inter=%lld of 8 (at most 2^20)", name,
                (long long)hidden, (long long)inter);
  if (logits_dtype != B200MOE_F32 && logits_dtype != B200MOE_F16 && logits_dtype != B200MOE_BF16)
    return fail(B200MOE_ERR_DTYPE, "%s: unsupported logits dtype %d", name, logits_dtype);
  if (num_tokens == 0) return B200MOE_OK;
  if (!hidden_states || !gating_output || !w13 || !w2 || !output)
    return fail(B200MOE_ERR_NULL, "%s: null pointer", name);
  if (!aligned_to(hidden_states, 16) || !aligned_to(w13, 16) || !aligned_to(w2, 16))
    return fail(B200MOE_ERR_ALIGN, "%s: hidden_states, w13 and w2 must be 16-byte aligned", name);
  const size_t need = b200moe_few_tokens_workspace_bytes(num_tokens, inter);
  if (!workspace || workspace_bytes < need || !aligned_to(workspace, 16))
    return fail(B200MOE_ERR_WORKSPACE, "%s: needs a 16-byte aligned workspace of %zu bytes, got %zu", name, need,
                workspace_bytes);
  Params p;
  p.x = static_cast<const __nv_bfloat16*>(hidden_states);
  p.logits = gating_output;
  p.w = nullptr;
  p.act = static_cast<uint4*>(workspace);
  p.out = static_cast<__nv_bfloat16*>(output);
  p.tokens = static_cast<int>(num_tokens);
  p.hidden = static_cast<int>(hidden);
  p.inter = static_cast<int>(inter);
  p.logits_dtype = logits_dtype;
  p.renormalize = renormalize;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return num_tokens <= 8 ? launch<1>(p, w13, w2, st) : launch<2>(p, w13, w2, st);
}
