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
// columns; a tile is 16 weight rows with the whole contraction, split over the eight warps of a CTA.  Each
// warp streams 16 x 128 weights per step through a ring of its own (asynchronous 16-byte copies, 20 KiB a
// warp, 160 KiB an SM in flight), never waiting for another warp except to add up a finished tile.  Tiles
// are dealt round-robin; that some CTAs get one more does not cost much, because an SM alone can
// draw well over 1/148 of the HBM rate.
//
// * The contraction index may be permuted at will, so fragments are 16-byte reads of eight consecutive
//   elements: of the weights from shared memory (columns swizzled by the row's parity: no bank
//   conflicts), of the tokens straight from global memory (L1 and L2 hold them).
// * A tile of kernel 1 is 8 gate rows over the 8 matching up rows, so that gate and up of one
//   element meet in one lane's accumulators.
// * Tokens that are not routed to a tile's expert are zero columns: nothing is loaded for them.
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
constexpr int kRows = 16;                        // weight rows of a tile
constexpr int kStep = 128;                       // contraction elements of a ring stage
constexpr int kStages = 5;
constexpr int kStageBytes = kRows * kStep * 2;   // 4 KiB
constexpr int kRingBytes = kWarps * kStages * kStageBytes;  // 160 KiB

struct Params {
  const __nv_bfloat16* x;
  const void* logits;
  const __nv_bfloat16* w;  // w13 or w2
  uint4* act;              // [2 * tokens][inter / 8][2]: eight high parts, eight low parts
  __nv_bfloat16* out;
  int tokens, hidden, inter, logits_dtype, renormalize;
};

struct Routing {
  int active[kExperts];                 // the experts that were hit, ascending
  int num_active;
  int8_t pair[kExperts][kMaxTokens];    // pair index of (expert, token), -1: not routed
  float weight[kExperts][kMaxTokens];
};

__device__ __forceinline__ float load_logit(const void* p, int dtype, int i) {
  if (dtype == B200MOE_F32) return static_cast<const float*>(p)[i];
  if (dtype == B200MOE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}

// Softmax and top-2 of up to 32 tokens, one lane each (one warp).  Equal logits: the lower index wins.
__device__ void route(const Params& p, Routing& r) {
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
  int n = 0;
#pragma unroll
  for (int e = 0; e < kExperts; ++e) {
    const int slot = first == e ? 0 : second == e ? 1 : -1;
    r.pair[e][t] = static_cast<int8_t>(slot < 0 ? -1 : 2 * t + slot);
    r.weight[e][t] = slot == 0 ? w1 : w2;
    if (__any_sync(0xffffffffu, slot >= 0)) {
      if (t == 0) r.active[n] = e;
      ++n;
    }
  }
  if (t == 0) r.num_active = n;
}

// Byte offset of 16-byte column `col` of row `row` in a stage of 256-byte rows.
__device__ __forceinline__ uint32_t stage_offset(int row, int col) {
  return static_cast<uint32_t>(row * kStep * 2 + ((col ^ ((row & 1) << 2)) << 4));
}

template <int kNT, bool kDown>  // kNT = tiles of 8 tokens
__global__ void __launch_bounds__(kThreads, 1)
few_tokens_kernel(const Params p) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Routing r;
  __shared__ float4 s_sum[2][kWarps][kNT][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  // Kernel 2 may look at the logits before kernel 1 is through: kernel 1 lets it start only after its own
  // wait, that is after everything before it in the stream has finished.
  if (!kDown) pdl_wait();
  if (warp == 0) route(p, r);
  __syncthreads();
  pdl_launch_dependents();

  const int K = kDown ? p.inter : p.hidden;
  const int steps = (K + kStep - 1) / kStep;                              // of one expert
  const int chunks = kDown ? r.num_active * steps : steps;                // of one tile
  const int expert_tiles = kDown ? p.hidden / kRows : p.inter / (kRows / 2);
  const int tiles = kDown ? expert_tiles : r.num_active * expert_tiles;
  const int my_chunks = chunks > warp ? (chunks - warp + kWarps - 1) / kWarps : 0;  // of one tile
  const uint32_t ring = smem_addr(smem) + warp * kStages * kStageBytes;
  const int64_t row_bytes = static_cast<int64_t>(K) * 2;
  const int64_t up_gap = kDown ? 0 : static_cast<int64_t>(p.inter - kRows / 2) * row_bytes;

  // Issues the copies of chunk `c` of tile `tile`: 16 weight rows x 128 elements, zeros past K.
  auto issue = [&](int tile, int c, int stage) {
    if (tile < tiles) {
      const int a = kDown ? c / steps : tile / expert_tiles;
      const int k0 = (kDown ? c - a * steps : c) * kStep;
      const int row0 = kDown ? tile * kRows : (tile - a * expert_tiles) * (kRows / 2);
      const int64_t expert_rows = kDown ? p.hidden : 2 * static_cast<int64_t>(p.inter);
      const int row = lane >> 4, col = lane & 15;
      const int bytes = k0 + col * 8 < K ? 16 : 0;
      const uint8_t* src = reinterpret_cast<const uint8_t*>(p.w) +
                           (r.active[a] * expert_rows + row0 + row) * row_bytes + (bytes ? (k0 + col * 8) * 2 : 0);
#pragma unroll
      for (int j = 0; j < kRows / 2; ++j)
        cp_async_16(ring + stage * kStageBytes + stage_offset(row + 2 * j, col),
                    src + 2 * j * row_bytes + (j >= kRows / 4 ? up_gap : 0), bytes);
    }
    cp_async_commit();
  };

  // The warp's chunks of all its tiles, as one sequence.
  int ahead_tile = my_chunks ? blockIdx.x : tiles, ahead = 0, filled = 0;
  auto issue_next = [&]() {
    issue(ahead_tile, warp + ahead * kWarps, filled);
    filled = filled + 1 == kStages ? 0 : filled + 1;
    if (++ahead >= my_chunks) { ahead = 0; if (ahead_tile < tiles) ahead_tile += gridDim.x; }
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) issue_next();
  if (kDown) pdl_wait();

  int stage = 0, parity = 0;
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, parity ^= 1) {
    float acc[kNT][4];
#pragma unroll
    for (int n = 0; n < kNT; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[n][j] = 0.f;
    const int tile_expert = kDown ? 0 : r.active[tile / expert_tiles];

    for (int i = 0; i < my_chunks; ++i) {
      const int c = warp + i * kWarps;
      const int a = kDown ? c / steps : 0;
      const int k0 = (kDown ? c - a * steps : c) * kStep;
      const int e = kDown ? r.active[a] : tile_expert;
      // The tokens' side of the products: eight elements from k0 + kk * 32 + t * 8.
      uint4 b[kStep / 32][kNT][kDown ? 2 : 1];
#pragma unroll
      for (int n = 0; n < kNT; ++n) {
        const int pair = r.pair[e][n * 8 + g];
#pragma unroll
        for (int kk = 0; kk < kStep / 32; ++kk) {
          const int k = k0 + kk * 32 + t * 8;
          const bool live = pair >= 0 && k < K;
          if constexpr (kDown) {
            const uint4* at = p.act + (static_cast<int64_t>(pair) * (p.inter / 8) + k / 8) * 2;
            b[kk][n][0] = live ? at[0] : make_uint4(0, 0, 0, 0);
            b[kk][n][1] = live ? at[1] : make_uint4(0, 0, 0, 0);
          } else {
            b[kk][n][0] = live ? __ldg(reinterpret_cast<const uint4*>(
                                     p.x + static_cast<int64_t>(n * 8 + g) * p.hidden + k))
                               : make_uint4(0, 0, 0, 0);
          }
        }
      }
      issue_next();
      cp_async_wait<kStages - 1>();
      __syncwarp();
      const uint32_t at = ring + stage * kStageBytes;
#pragma unroll
      for (int kk = 0; kk < kStep / 32; ++kk) {
        const uint4 lo = lds_16(at + stage_offset(g, kk * 4 + t)), hi = lds_16(at + stage_offset(g + 8, kk * 4 + t));
        const uint32_t a0[4] = {lo.x, hi.x, lo.y, hi.y}, a1[4] = {lo.z, hi.z, lo.w, hi.w};
#pragma unroll
        for (int n = 0; n < kNT; ++n)
#pragma unroll
          for (int h = 0; h < (kDown ? 2 : 1); ++h) {
            Mma<__nv_bfloat16>::run(acc[n], a0, b[kk][n][h].x, b[kk][n][h].y);
            Mma<__nv_bfloat16>::run(acc[n], a1, b[kk][n][h].z, b[kk][n][h].w);
          }
      }
      __syncwarp();  // the stage is refilled by a later iteration's copies
      stage = stage + 1 == kStages ? 0 : stage + 1;
    }

    // Add the warps up, in their order; the two buffers make one barrier per tile enough.
#pragma unroll
    for (int n = 0; n < kNT; ++n) s_sum[parity][warp][n][lane] = make_float4(acc[n][0], acc[n][1], acc[n][2], acc[n][3]);
    __syncthreads();
    if (warp < kNT) {
      float4 v = s_sum[parity][0][warp][lane];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) {
        const float4 o = s_sum[parity][w][warp][lane];
        v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
      }
      // Elements (row g, tokens 2 t, 2 t + 1) and (row g + 8, the same tokens).
      const float top[2] = {v.x, v.y}, bottom[2] = {v.z, v.w};
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int token = warp * 8 + 2 * t + c;
        if constexpr (kDown) {
          if (token < p.tokens) {
            __nv_bfloat16* o = p.out + static_cast<int64_t>(token) * p.hidden + tile * kRows + g;
            o[0] = __float2bfloat16_rn(top[c]);
            o[8] = __float2bfloat16_rn(bottom[c]);
          }
        } else {
          const int pair = r.pair[tile_expert][token];
          if (pair >= 0) {
            const int group = tile % expert_tiles;  // eight elements of the expert's width
            const float value = r.weight[tile_expert][token] * (top[c] / (1.f + expf(-top[c])) * bottom[c]);
            const __nv_bfloat16 high = __float2bfloat16_rn(value);
            const float rest = value - __bfloat162float(high);
            __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(
                p.act + (static_cast<int64_t>(pair) * expert_tiles + group) * 2);
            o[g] = high;
            o[8 + g] = __float2bfloat16_rn(rest);
          }
        }
      }
    }
  }
  cp_async_wait<0>();
}

template <int kNT>
int launch(Params p, const void* w13, const void* w2, cudaStream_t st) {
  const char* name = "moe_few_tokens";
  for (int down = 0; down < 2; ++down) {
    const cudaError_t e =
        down ? cudaFuncSetAttribute(few_tokens_kernel<kNT, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes)
             : cudaFuncSetAttribute(few_tokens_kernel<kNT, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes);
    if (e != cudaSuccess) return fail(B200MOE_ERR_CUDA, "%s: %s", name, cudaGetErrorString(e));
  }
  const int experts_hit = 2 * p.tokens < kExperts ? 2 * p.tokens : kExperts;
  const int64_t up_tiles = static_cast<int64_t>(experts_hit) * p.inter / (kRows / 2), down_tiles = p.hidden / kRows;
  const int64_t sms = sm_count();
  p.w = static_cast<const __nv_bfloat16*>(w13);
  launch_pdl(few_tokens_kernel<kNT, false>, dim3(static_cast<unsigned>(up_tiles < sms ? up_tiles : sms)), dim3(kThreads),
             kRingBytes, st, p);
  if (int rc = check_launch(name)) return rc;
  p.w = static_cast<const __nv_bfloat16*>(w2);
  launch_pdl(few_tokens_kernel<kNT, true>, dim3(static_cast<unsigned>(down_tiles < sms ? down_tiles : sms)), dim3(kThreads),
             kRingBytes, st, p);
  return check_launch(name);
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
  switch ((num_tokens + 7) / 8) {
    case 1: return launch<1>(p, w13, w2, st);
    case 2: return launch<2>(p, w13, w2, st);
    case 3: return launch<3>(p, w13, w2, st);
    default: return launch<4>(p, w13, w2, st);
  }
}
