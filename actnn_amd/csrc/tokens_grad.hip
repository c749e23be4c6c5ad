// Weight gradient of a linear layer from the 8-bit tokens it kept:
//
//     grad_w[o, i] = sum_m grad_out[m, o] * x[m, i],   x[m, i] = codes[m, i] * scale[m]
//
// A token's scale varies along the sum, so it cannot be taken out of it: the codes are turned back into values on their way
// into LDS and rounded to the 16-bit type of grad_out (what the layer would have kept without the 8 bits has the same
// rounding; the sums are fp32).  v_mfma_f32_32x32x16, both tiles in LDS as they lie in memory, [token][column]; the
// transposing read ds_read_b64_tr_b16 gives a lane four consecutive tokens of its column.
//
// Tile: 128 outputs x 128 features, four waves of 64 x 64, 64 tokens a step, two buffers.  A row of a tile is 256
// bytes, all banks once; its 16-byte chunks lie at chunk ^ 4 (row % 4), so that the four rows which 32 lanes of a transposing
// read touch (64 bytes each) fall into the four quarters of the banks.  Everything goes through registers: rows of any length at any
// address, tokens past the end are zeros in both operands.  Few tiles: the tokens are split over blocks that leave fp32 tiles in a
// workspace, a second kernel adds them in a fixed order.
#include <type_traits>

#include "token_math.h"

namespace actnn {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;

template <typename T> ACTNN_DEV f32x16 mma16(u32x4 a, u32x4 b, f32x16 c);
template <> ACTNN_DEV f32x16 mma16<bf16_t>(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <> ACTNN_DEV f32x16 mma16<__half>(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

typedef __attribute__((address_space(3))) uint8_t* lds_ptr_t;
ACTNN_DEV uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint8_t*)p;
}
// four consecutive rows of this lane's column
ACTNN_DEV u32x2 read_transposed(uint32_t at) {
  const i16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(uintptr_t)at);
  return __builtin_bit_cast(u32x2, v);
}

struct Grad {
  const void* g;                         // [M, O], rows `ldg` elements apart
  const int8_t* x;                       // [M, I], rows `ldx` bytes apart
  const float* scale;
  void* out;                             // [O, I], or fp32 [splits][O][I]
  int64_t ldg, ldx;
  int64_t g_last;                        // where the last 16 bytes of g begin
  int M, O, I;
};

template <typename T, typename TY>
__global__ __launch_bounds__(kThreads, 2) void tokens_grad_kernel(Grad p, int splits, int tokens_per_split) {
  constexpr int BO = 128, BI = 128, BK = 64, kRow = 256, kTile = BK * kRow;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[4 * kTile];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wave & 1, wn = wave >> 1;
  const int tiles_i = (p.I + BI - 1) / BI, tiles = (p.O + BO - 1) / BO * tiles_i;
  const int split = blockIdx.x / tiles, tile = blockIdx.x % tiles;
  const int o0 = tile / tiles_i * BO, i0 = tile % tiles_i * BI;
  const int m0 = split * tokens_per_split;
  const int m1 = p.M - m0 < tokens_per_split ? p.M : m0 + tokens_per_split;
  TY* out = static_cast<TY*>(p.out) + (int64_t)split * p.O * p.I;

  // ---- staging: thread -> chunk of eight columns tid % 16, rows tid / 16 + 16 j of both tiles
  const int ch = tid & 15, row0 = tid >> 4;
  const T* last = static_cast<const T*>(p.g) + p.g_last;
  const bool in_x = i0 + ch * 8 < p.I;                  // (a row of codes is whole to the next multiple of 16)
  RowVector rg[4];
  u32x2 rx[4];
  float rs[4];
  auto fetch = [&](int m) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int at = m + row0 + 16 * j;
      const int64_t row = at < m1 ? at : m1 - 1;
      rg[j] = load16_row<T>(static_cast<const T*>(p.g) + row * p.ldg + o0 + ch * 8, at < m1 ? p.O - (o0 + ch * 8) : 0, last);
      rx[j] = *reinterpret_cast<const u32x2*>(p.x + row * p.ldx + (in_x ? i0 + ch * 8 : 0));
      rs[j] = p.scale[row];
    }
  };
  auto stage = [&](int buffer, int m) {
    uint8_t* tg = smem + buffer * 2 * kTile;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = row0 + 16 * j;
      const int at = row * kRow + ((ch ^ ((row & 3) << 2)) << 4);
      *reinterpret_cast<u32x4*>(tg + at) = row_vector_ends<T>(rg[j]);
      float f[8];
      code_values(rx[j], f);
      const bool valid = m + row < m1;
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = valid ? f[e] * rs[j] : 0.0f;
      *reinterpret_cast<u32x4*>(tg + kTile + at) = words_of8(static_cast<const T*>(nullptr), f);
    }
  };

  // ---- fragments: lane -> column n0 + lane % 32, tokens 16 kb + 8 (lane / 32) ..
  const int blk = lane >> 4, r = lane & 15;
  const int f_row = 8 * (blk >> 1) + (r >> 2);
  auto fragment_at = [&](int n0) {
    const int c = n0 / 8 + 2 * (blk & 1) + ((r & 3) >> 1);
    return (uint32_t)(f_row * kRow + ((c ^ ((f_row & 3) << 2)) << 4) + (r & 1) * 8);
  };
  const uint32_t lds0 = lds_address(smem);
  uint32_t ag[2], ax[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    ag[i] = lds0 + fragment_at(wr * 64 + 32 * i);
    ax[i] = lds0 + kTile + fragment_at(wn * 64 + 32 * i);
  }
  f32x16 acc[2][2];
#pragma unroll
  for (int e = 0; e < 2; ++e)
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int c = 0; c < 16; ++c) acc[e][a][c] = 0.0f;

  if (m0 < m1) {
    fetch(m0);
    stage(0, m0);
  }
  __syncthreads();
  int buffer = 0;
  for (int m = m0; m < m1; m += BK) {
    const bool more = m + BK < m1;
    if (more) fetch(m + BK);
    const uint32_t base = buffer * 2 * kTile;
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) {
      u32x4 fg[2], fx[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const u32x2 a = read_transposed(ag[i] + base + kb * 16 * kRow), b = read_transposed(ag[i] + base + (kb * 16 + 4) * kRow);
        fg[i] = (u32x4){a.x, a.y, b.x, b.y};
        const u32x2 c = read_transposed(ax[i] + base + kb * 16 * kRow), d = read_transposed(ax[i] + base + (kb * 16 + 4) * kRow);
        fx[i] = (u32x4){c.x, c.y, d.x, d.y};
      }
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int a = 0; a < 2; ++a) acc[e][a] = mma16<T>(fx[e], fg[a], acc[e][a]);
    }
    if (more) stage(1 - buffer, m + BK);                // (its last readers passed the barrier of the step before)
    __syncthreads();
    buffer = 1 - buffer;
  }

  // accumulator register c of a lane: feature 8 (c / 4) + 4 (lane / 32) + c % 4 of the fragment, output lane % 32
#pragma unroll
  for (int a = 0; a < 2; ++a) {
    const int o = o0 + wr * 64 + 32 * a + (lane & 31);
    if (o >= p.O) continue;
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int i = i0 + wn * 64 + 32 * e + 8 * q + 4 * (lane >> 5);
        TY* to = out + (int64_t)o * p.I + i;
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (i + c < p.I) Conv<TY>::store(to, c, acc[e][a][4 * q + c]);
      }
  }
}

template <typename TY>
__global__ __launch_bounds__(kThreads) void tokens_grad_sum_kernel(const float* __restrict__ part, TY* __restrict__ out,
                                                                   int64_t n, int splits) {
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i >= n) return;
  float v = 0.0f;
  for (int s = 0; s < splits; ++s) v += part[s * n + i];
  Conv<TY>::store(out, i, v);
}

// Blocks that share the tokens of a tile: enough to fill the chip twice, with four steps each at least.
struct Plan { int splits, tokens; };
Plan plan_of(int64_t M, int64_t O, int64_t I) {
  const int64_t tiles = ((O + 127) / 128) * ((I + 127) / 128), steps = (M + 63) / 64;
  int64_t splits = tiles >= 256 ? 1 : 512 / tiles;
  if (splits > steps / 4) splits = steps / 4;
  if (splits < 1) splits = 1;
  const int64_t per = (steps + splits - 1) / splits;
  return Plan{(int)((steps + per - 1) / per), (int)(per * 64)};
}

template <typename T, typename TY>
int launch_grad(Grad p, void* workspace, int64_t workspace_bytes, hipStream_t s) {
  Plan plan = plan_of(p.M, p.O, p.I);
  const int64_t n = (int64_t)p.O * p.I;
  const int64_t whole = ((int64_t)p.M + 63) / 64 * 64;
  if (plan.splits > 1 && (!workspace || workspace_bytes < 4 * n * plan.splits)) plan = Plan{1, (int)whole};
  const int64_t blocks = ((p.O + 127LL) / 128) * ((p.I + 127LL) / 128) * plan.splits;
  if (blocks > 0x7fffffffLL || (n + kThreads - 1) / kThreads > 0x7fffffffLL) return ACTNN_EINVAL;
  const dim3 grid((unsigned)blocks), blk(kThreads);
  if (plan.splits == 1) {
    tokens_grad_kernel<T, TY><<<grid, blk, 0, s>>>(p, 1, plan.tokens);
  } else {
    if (!aligned16(workspace)) return ACTNN_EALIGN;
    TY* out = static_cast<TY*>(p.out);
    p.out = workspace;
    tokens_grad_kernel<T, float><<<grid, blk, 0, s>>>(p, plan.splits, plan.tokens);
    tokens_grad_sum_kernel<TY><<<dim3((unsigned)((n + kThreads - 1) / kThreads)), blk, 0, s>>>(
        static_cast<const float*>(workspace), out, n, plan.splits);
  }
  ACTNN_RETURN_LAUNCH_STATUS();
}
template <typename T>
int launch_out(const Grad& p, int out_dtype, void* workspace, int64_t workspace_bytes, hipStream_t s) {
  if (out_dtype == ACTNN_F32) return launch_grad<T, float>(p, workspace, workspace_bytes, s);
  return launch_grad<T, T>(p, workspace, workspace_bytes, s);
}

}  // namespace
}  // namespace actnn

extern "C" int64_t actnn_tokens_grad_weight_workspace_bytes(int64_t M, int64_t O, int64_t I) {
  using namespace actnn;
  if (M < 1 || O < 1 || I < 1 || M > 0x7fffff00LL || O > 0x7fffff00LL || I > 0x7fffff00LL) return 0;
  const Plan plan = plan_of(M, O, I);
  return plan.splits > 1 ? 4 * O * I * plan.splits : 0;
}

extern "C" int actnn_tokens_grad_weight(const void* grad_out, int64_t ldg, const int8_t* codes, int64_t ldc, const float* scale,
                                        void* grad_w, int64_t M, int64_t O, int64_t I, int go_dtype, int out_dtype,
                                        void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace actnn;
  if (M < 0 || O < 0 || I < 0 || M > 0x7fffff00LL || O > 0x7fffff00LL || I > 0x7fffff00LL) return ACTNN_EINVAL;
  if (ldc < I || ldc % 16 || ldg < 0) return ACTNN_EINVAL;
  if (go_dtype != ACTNN_F16 && go_dtype != ACTNN_BF16) return ACTNN_EDTYPE;
  if (out_dtype != ACTNN_F32 && out_dtype != go_dtype) return ACTNN_EDTYPE;
  if (O == 0 || I == 0) return ACTNN_OK;
  if (M == 0) return ACTNN_EINVAL;                      // (nothing to launch: the caller clears the result)
  if (!grad_out || !codes || !scale || !grad_w) return ACTNN_EINVAL;
  int64_t g_last = (M - 1) * ldg + O - 8;
  if (g_last < 0) {                                     // below 16 bytes: the rows have room behind them
    if (ldg < 8) return ACTNN_EINVAL;
    g_last = (M - 1) * ldg;
  }
  if (!aligned16(codes) || reinterpret_cast<uintptr_t>(grad_out) % 2 || reinterpret_cast<uintptr_t>(scale) % 4 ||
      reinterpret_cast<uintptr_t>(grad_w) % (out_dtype == ACTNN_F32 ? 4 : 2))
    return ACTNN_EALIGN;
  const Grad p{grad_out, codes, scale, grad_w, ldg, ldc, g_last, (int)M, (int)O, (int)I};
  hipStream_t s = static_cast<hipStream_t>(stream);
  return go_dtype == ACTNN_F16 ? launch_out<__half>(p, out_dtype, workspace, workspace_bytes, s)
                               : launch_out<bf16_t>(p, out_dtype, workspace, workspace_bytes, s);
}
