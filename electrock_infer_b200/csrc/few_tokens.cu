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
// finished tile.  Tiles are dealt round-robin; that some CTAs get one more does not cost much,
// because an SM alone can draw well over 1/148 of the HBM rate.
//
// * The contraction index may be permuted at will, so fragments are 16-byte reads of eight consecutive
//   elements from shared memory (pieces swizzled by the row's parity: no bank conflicts).
// * A tile of kernel 1 has 8 gate rows over the 8 matching up rows in each 16, so that gate and up of one
//   element meet in one lane's accumulators.
// * Only the tokens that are routed to a tile's expert are copied; the columns of the others are zeros that
//   are not read from anywhere, and products with eight such columns are left out.  A stage has room
//   for 16 tokens: an expert with more is gone through twice, its weights then coming from L2.
// * Up to 8 tokens take 16-row tiles (the finest deal); more take 32-row tiles, which halve the copies of
//   tokens per weight.
// * act is kept as the sum of two bf16 numbers (16 bits of mantissa): kernel 2 multiplies both by
//   the weights and adds in fp32, so that the only rounding that shows is the output's.
// * Kernel 2 is launched with programmatic stream serialisation and fills its rings with w2 before it
//   waits for kernel 1.
//
// The reference runs the same batch through its general path (layers/moe/fused_moe.py:170-293).
#include "warp_mma.cuh"

namespace b200moe {
namespace {

constexpr int kExperts = 8;
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
};

// Experts that were hit, in ascending order, and their tokens.
struct Routing {
  int num_active;
  int expert[kExperts];                 // number of the a-th active expert
  int count[kExperts];                  // its tokens
  int begin[kExperts + 1];              // prefix of (units * groups of tokens), see the kernel
  int8_t token[kExperts][kMaxTokens];   // its tokens, ascending
  int8_t rank[kExperts][kMaxTokens];    // place of a token in that list, -1: not routed to it
  int8_t pair[kExperts][kMaxTokens];    // index of the pair, by token
  float weight[kExperts][kMaxTokens];
  uint8_t tiles[kExperts][2];           // column tiles that hold a token of group 0, 1
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
    if (slot >= 0) r.token[n][rank] = static_cast<int8_t>(t);
    r.rank[n][t] = static_cast<int8_t>(slot < 0 ? -1 : rank);
    r.pair[n][t] = static_cast<int8_t>(2 * t + slot);
    r.weight[n][t] = slot == 0 ? w1 : w2;
    const int count = __popc(hit);
    uint32_t tiles[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < kMaxTokens / 8; ++i)
#pragma unroll
      for (int q = 0; q < 2; ++q)
        if (__any_sync(0xffffffffu, slot >= 0 && t / 8 == i && rank / kGroup == q)) tiles[q] |= 1u << i;
    if (t == 0) {
      r.expert[n] = e;
      r.count[n] = count;
      r.begin[n] = at;
      r.tiles[n][0] = static_cast<uint8_t>(tiles[0]);
      r.tiles[n][1] = static_cast<uint8_t>(tiles[1]);
    }
    at += units * ((count + kGroup - 1) / kGroup);
    ++n;
  }
  if (t == 0) {
    r.num_active = n;
    r.begin[n] = at;
  }
}

// A place in the sequence of (active expert, unit, group of tokens): units are tiles of kernel 1 and
// contraction steps of kernel 2, the groups of one unit follow one another.
struct Place {
  int a, unit, group;
  // Moves forward to position `at` of the sequence.
  __device__ __forceinline__ void seek(const Routing& r, int at) {
    while (at >= r.begin[a + 1]) ++a;
    const int rest = at - r.begin[a];
    const bool two = r.count[a] > kGroup;
    unit = two ? rest >> 1 : rest;
    group = two ? rest & 1 : 0;
  }
};

// kNT = tiles of 8 tokens, kRT = tiles of 16 weight rows.
template <int kNT, int kRT, bool kDown>
struct Shape {
  static constexpr int kStep = 128 / kRT;                      // contraction elements of a stage
  static constexpr int kPieces = kStep / 8;                    // 16-byte pieces of a weight row
  static constexpr int kParts = kDown ? 2 : 1;                 // numbers that an element is the sum of
  static constexpr int kSlots = kNT == 1 ? 8 : kGroup;         // tokens that a stage has room for
  static constexpr int kTokenPieces = kPieces * kParts;
  static constexpr int kStageBytes = kWeightBytes + kSlots * kTokenPieces * 16;
  static constexpr int kStages = kRingBytes / kWarps / kStageBytes;
  static constexpr int kRows = 16 * kRT;
  static constexpr int kSets = kNT * kRT == 1 ? 2 : 1;         // accumulator sets, against dependent products
  static_assert(kStages >= 2, "the ring is too small");
};

// Byte offsets in a stage: piece `col` of weight row `row`; piece `col`, part `part` of token slot `slot`.
// Two rows or slots of different parity never meet in a bank where a quarter of a warp reads them.
template <typename S> __device__ __forceinline__ uint32_t weight_offset(int row, int col) {
  return static_cast<uint32_t>((row * S::kPieces + (col ^ ((row & 1) << 2))) * 16);
}
template <typename S> __device__ __forceinline__ uint32_t token_offset(int slot, int piece) {
  const int mixed = S::kParts == 2 ? piece ^ (slot & 1) : piece ^ ((slot & 1) << 2);
  return static_cast<uint32_t>(kWeightBytes + (slot * S::kTokenPieces + mixed) * 16);
}

template <int kNT, int kRT, bool kDown>
__global__ void __launch_bounds__(kThreads, 1)
few_tokens_kernel(const Params p) {
  using S = Shape<kNT, kRT, kDown>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Routing r;
  __shared__ float4 s_sum[kNT * kRT <= 2 ? 2 : 1][kWarps][kNT * kRT][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int K = kDown ? p.inter : p.hidden;
  const int steps = (K + S::kStep - 1) / S::kStep;                             // of one expert
  const int expert_tiles = kDown ? p.hidden / S::kRows : p.inter / (S::kRows / 2);
  // Kernel 2 may look at the logits before kernel 1 is through: kernel 1 lets it start only after its own
  // wait, that is after everything before it in the stream has finished.
  if (!kDown) pdl_wait();
  if (warp == 0) route(p, r, kDown ? steps : expert_tiles);
  __syncthreads();
  pdl_launch_dependents();

  const int chunks = kDown ? r.begin[r.num_active] : steps;                    // of one tile
  const int tiles = kDown ? expert_tiles : r.begin[r.num_active];
  const int my_chunks = chunks > warp ? (chunks - warp + kWarps - 1) / kWarps : 0;  // of one tile
  const uint32_t ring = smem_addr(smem) + warp * S::kStages * S::kStageBytes;
  const int64_t row_bytes = static_cast<int64_t>(K) * 2;
  const int64_t up_gap = kDown ? 0 : static_cast<int64_t>(p.inter - 8) * row_bytes;  // from gate rows to up rows

  // Copies of the weights of chunk `c` of a tile: kRows rows x kStep elements, zeros past K.
  auto issue_weights = [&](int tile, const Place& at, int step, uint32_t to) {
    const int k0 = step * S::kStep;
    const int row0 = kDown ? tile * S::kRows : at.unit * (S::kRows / 2);
    const int64_t expert_rows = kDown ? p.hidden : 2 * static_cast<int64_t>(p.inter);
    constexpr int kRowsAtOnce = 32 / S::kPieces;   // 2 or 4, of one row tile's eight upper or lower rows
    const int row = lane / S::kPieces, col = lane % S::kPieces;
    const int bytes = k0 + col * 8 < K ? 16 : 0;
    const uint8_t* src = reinterpret_cast<const uint8_t*>(p.w) +
                         (r.expert[at.a] * expert_rows + row0 + row) * row_bytes + (bytes ? (k0 + col * 8) * 2 : 0);
#pragma unroll
    for (int j = 0; j < S::kRows / kRowsAtOnce; ++j) {
      const int base = j * kRowsAtOnce;            // rows base + row of the tile
      // Kernel 1: rows 16 m + 0..7 are gate rows 8 m + 0..7, rows 16 m + 8..15 the same up rows.
      const int from = kDown ? base : base / 16 * 8 + base % 8;
      cp_async_16(to + weight_offset<S>(base + row, col),
                  src + from * row_bytes + (!kDown && base % 16 >= 8 ? up_gap + 8 * row_bytes : 0), bytes);
    }
  };
  // Copies of the group's tokens that belong to them.
  auto issue_tokens = [&](const Place& at, int step, uint32_t to) {
    const int live = min(r.count[at.a] - at.group * kGroup, kGroup);
    const int k0 = step * S::kStep;
#pragma unroll
    for (int i = 0; i < S::kSlots * S::kTokenPieces / 32; ++i) {
      const int index = i * 32 + lane;
      const int slot = index / S::kTokenPieces, piece = index % S::kTokenPieces;
      if (slot < live) {
        const int token = r.token[at.a][at.group * kGroup + slot];
        const int k = k0 + piece / S::kParts * 8;
        const int bytes = k < K ? 16 : 0;
        const void* src;
        if constexpr (kDown) {
          src = p.act + (static_cast<int64_t>(r.pair[at.a][token]) * (p.inter / 8) + (bytes ? k / 8 : 0)) * 2 +
                piece % S::kParts;
        } else {
          src = p.x + static_cast<int64_t>(token) * p.hidden + (bytes ? k : 0);
        }
        cp_async_16(to + token_offset<S>(slot, piece), src, bytes);
      }
    }
  };

  // The warp's chunks of all its tiles as one sequence, of which `ahead` is the next to be issued.
  Place ahead = {0, 0, 0};
  int ahead_tile = my_chunks ? blockIdx.x : tiles, ahead_chunk = 0, filled = 0;
  auto ahead_step = [&]() {  // seeks the place, returns the contraction step
    const int c = warp + ahead_chunk * kWarps;
    if (kDown) {
      if (ahead_chunk == 0) ahead.a = 0;
      ahead.seek(r, c);
      return ahead.unit;
    }
    if (ahead_chunk == 0) ahead.seek(r, ahead_tile);
    return c;
  };
  auto advance = [&]() {
    filled = filled + 1 == S::kStages ? 0 : filled + 1;
    if (++ahead_chunk >= my_chunks) { ahead_chunk = 0; if (ahead_tile < tiles) ahead_tile += gridDim.x; }
  };
  auto issue_next = [&]() {
    if (ahead_tile < tiles) {
      const int step = ahead_step();
      const uint32_t to = ring + filled * S::kStageBytes;
      issue_weights(ahead_tile, ahead, step, to);
      issue_tokens(ahead, step, to);
    }
    cp_async_commit();
    advance();
  };
  if constexpr (kDown) {
    // Weights first, then, once kernel 1 is through, the activations that go with them.
    const int tile0 = ahead_tile;
    for (int s = 0; s < S::kStages - 1; ++s) {
      if (ahead_tile < tiles) {
        const int step = ahead_step();
        issue_weights(ahead_tile, ahead, step, ring + filled * S::kStageBytes);
      }
      advance();
    }
    ahead_tile = tile0; ahead_chunk = 0; filled = 0; ahead = {0, 0, 0};
    pdl_wait();
    for (int s = 0; s < S::kStages - 1; ++s) {
      if (ahead_tile < tiles) {
        const int step = ahead_step();
        issue_tokens(ahead, step, ring + filled * S::kStageBytes);
      }
      cp_async_commit();
      advance();
    }
  } else {
#pragma unroll
    for (int s = 0; s < S::kStages - 1; ++s) issue_next();
  }

  int stage = 0, parity = 0;
  Place here = {0, 0, 0};
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    float acc[S::kSets][kRT][kNT][4];
#pragma unroll
    for (int s = 0; s < S::kSets; ++s)
#pragma unroll
      for (int m = 0; m < kRT; ++m)
#pragma unroll
        for (int n = 0; n < kNT; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[s][m][n][j] = 0.f;
    if (kDown) here = {0, 0, 0}; else here.seek(r, tile);

    for (int i = 0; i < my_chunks; ++i) {
      if (kDown) here.seek(r, warp + i * kWarps);
      issue_next();
      cp_async_wait<S::kStages - 1>();
      __syncwarp();
      const uint32_t at = ring + stage * S::kStageBytes;
      int slot[kNT];  // where the lane's token of each column tile stands in the stage; -1: a zero column
      const uint32_t used = r.tiles[here.a][here.group];
#pragma unroll
      for (int n = 0; n < kNT; ++n) {
        const int rank = r.rank[here.a][n * 8 + g] - here.group * kGroup;
        slot[n] = rank < kGroup ? rank : -1;
      }
#pragma unroll
      for (int kk = 0; kk < S::kStep / 32; ++kk) {
        uint32_t a0[kRT][4], a1[kRT][4];
#pragma unroll
        for (int m = 0; m < kRT; ++m) {
          const uint4 lo = lds_16(at + weight_offset<S>(m * 16 + g, kk * 4 + t));
          const uint4 hi = lds_16(at + weight_offset<S>(m * 16 + g + 8, kk * 4 + t));
          a0[m][0] = lo.x; a0[m][1] = hi.x; a0[m][2] = lo.y; a0[m][3] = hi.y;
          a1[m][0] = lo.z; a1[m][1] = hi.z; a1[m][2] = lo.w; a1[m][3] = hi.w;
        }
#pragma unroll
        for (int n = 0; n < kNT; ++n) {
          if (kNT > 1 && !(used >> n & 1)) continue;
#pragma unroll
          for (int h = 0; h < S::kParts; ++h) {
            uint4 b = make_uint4(0, 0, 0, 0);
            if (slot[n] >= 0) b = lds_16(at + token_offset<S>(slot[n], (kk * 4 + t) * S::kParts + h));
#pragma unroll
            for (int m = 0; m < kRT; ++m) {
              Mma<__nv_bfloat16>::run(acc[0][m][n], a0[m], b.x, b.y);
              Mma<__nv_bfloat16>::run(acc[S::kSets - 1][m][n], a1[m], b.z, b.w);
            }
          }
        }
      }
      __syncwarp();  // the stage is refilled by a later iteration's copies
      stage = stage + 1 == S::kStages ? 0 : stage + 1;
    }

    // Add the warps up, in their order.
    if (sizeof(s_sum) / sizeof(s_sum[0]) == 1) __syncthreads();  // with two buffers, one barrier per tile is enough
#pragma unroll
    for (int m = 0; m < kRT; ++m)
#pragma unroll
      for (int n = 0; n < kNT; ++n) {
        float4 v = make_float4(acc[0][m][n][0], acc[0][m][n][1], acc[0][m][n][2], acc[0][m][n][3]);
        if (S::kSets == 2) {
          v.x += acc[S::kSets - 1][m][n][0]; v.y += acc[S::kSets - 1][m][n][1];
          v.z += acc[S::kSets - 1][m][n][2]; v.w += acc[S::kSets - 1][m][n][3];
        }
        s_sum[parity][warp][m * kNT + n][lane] = v;
      }
    __syncthreads();
    if (warp < kNT * kRT) {
      float4 v = s_sum[parity][0][warp][lane];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) {
        const float4 o = s_sum[parity][w][warp][lane];
        v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
      }
      const int m = warp / kNT, n = warp % kNT;
      // Elements (row g, tokens 2 t, 2 t + 1) and (row g + 8, the same tokens) of row tile m.
      const float top[2] = {v.x, v.y}, bottom[2] = {v.z, v.w};
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int token = n * 8 + 2 * t + c;
        if constexpr (kDown) {
          if (token < p.tokens) {
            __nv_bfloat16* o = p.out + static_cast<int64_t>(token) * p.hidden + tile * S::kRows + m * 16 + g;
            o[0] = __float2bfloat16_rn(top[c]);
            o[8] = __float2bfloat16_rn(bottom[c]);
          }
        } else {
          const int rank = r.rank[here.a][token];
          if (rank >= 0 && rank / kGroup == here.group) {
            const float value = r.weight[here.a][token] * (top[c] / (1.f + expf(-top[c])) * bottom[c]);
            const __nv_bfloat16 high = __float2bfloat16_rn(value);
            const float rest = value - __bfloat162float(high);
            __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(
                p.act + (static_cast<int64_t>(r.pair[here.a][token]) * (p.inter / 8) + here.unit * kRT + m) * 2);
            o[g] = high;
            o[8 + g] = __float2bfloat16_rn(rest);
          }
        }
      }
    }
    if (sizeof(s_sum) / sizeof(s_sum[0]) == 2) parity ^= 1;
  }
  cp_async_wait<0>();
}

template <int kNT, int kRT, bool kDown>
int launch(const Params& p, int64_t tiles, cudaStream_t st) {
  const char* name = "moe_few_tokens";
  const auto kernel = few_tokens_kernel<kNT, kRT, kDown>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes);
  if (e != cudaSuccess) return fail(B200MOE_ERR_CUDA, "%s: %s", name, cudaGetErrorString(e));
  const int64_t sms = sm_count();
  launch_pdl(kernel, dim3(static_cast<unsigned>(tiles < sms ? tiles : sms)), dim3(kThreads), kRingBytes, st, p);
  return check_launch(name);
}

// 32-row tiles where there are more than 8 tokens and the sizes allow it.
template <int kNT>
int launch(Params p, const void* w13, const void* w2, cudaStream_t st) {
  const int experts_hit = 2 * p.tokens < kExperts ? 2 * p.tokens : kExperts;
  constexpr int kRT = kNT == 1 ? 1 : 2;
  const bool wide_up = p.inter % (8 * kRT) == 0, wide_down = p.hidden % (16 * kRT) == 0;
  p.w = static_cast<const __nv_bfloat16*>(w13);
  const int64_t up_tiles = static_cast<int64_t>(experts_hit) * p.inter / 8;
  if (int rc = wide_up ? launch<kNT, kRT, false>(p, up_tiles / kRT, st) : launch<kNT, 1, false>(p, up_tiles, st)) return rc;
  p.w = static_cast<const __nv_bfloat16*>(w2);
  return wide_down ? launch<kNT, kRT, true>(p, p.hidden / (16 * kRT), st) : launch<kNT, 1, true>(p, p.hidden / 16, st);
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
  if (num_tokens <= 8) return launch<1>(p, w13, w2, st);
  if (num_tokens <= 16) return launch<2>(p, w13, w2, st);
  return launch<4>(p, w13, w2, st);
}
