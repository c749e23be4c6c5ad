// Weight gradient of a linear layer from the 8-bit tokens it kept:
//
//     grad_w[o, i] = sum_m grad_out[m, o] * x[m, i],   x[m, i] = codes[m, i] * scale[m]
//
// A token's scale varies along the sum, so it cannot be taken out of it: the codes are turned back into values on their way
// into LDS and rounded to the 16-bit type of grad_out (what the layer would have kept without the 8 bits has the same
// rounding; the sums are fp32).  v_mfma_f32_32x32x16, both tiles in LDS as they lie in memory, [token][column]; the
// transposing read ds_read_b64_tr_b16 gives a lane four consecutive tokens of its column.
//
// Large products take tiles of 256 outputs x 256 features, fed by loads straight into LDS; small ones, and rows of
// grad_out at any address, tiles of 64 or 128 fed through registers.  Few tiles: the tokens are split over blocks that leave fp32
// tiles in a workspace, a second kernel adds them in a fixed order.
#include <type_traits>

#include "matrix_tiles.h"
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

// four consecutive rows of this lane's column
ACTNN_DEV u32x2 read_transposed(uint32_t at) {
  const i16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(uintptr_t)at);
  return __builtin_bit_cast(u32x2, v);
}

// eight codes of a token as values
template <typename T> ACTNN_DEV u32x4 values_of(u32x2 codes, float scale) {
  const uint32_t a = codes.x, b = codes.y;
  return (u32x4){code_pair<T, 0>(a, scale), code_pair<T, 1>(a, scale), code_pair<T, 0>(b, scale), code_pair<T, 1>(b, scale)};
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

// eight columns of a row of grad_out at any address: what lies behind the row's last column only reaches outputs that are not
// stored; a vector that would end behind the tensor is read from its last 16 bytes
template <typename T> ACTNN_DEV u32x4 load_columns(const T* at, const T* last) {
  const int64_t over = at - last;
  u32x4 v = load16_any(over > 0 ? last : at);
  for (int i = 0; i < over && i < 8; ++i)
    v = (u32x4){__builtin_amdgcn_alignbit(v.y, v.x, 16), __builtin_amdgcn_alignbit(v.z, v.y, 16),
                __builtin_amdgcn_alignbit(v.w, v.z, 16), v.w >> 16};
  return v;
}

// ------------------------------------------------------------------------------------------
// Small products, and rows at any address: 64 N outputs x 64 N features a block, four waves of 32 N x 32 N, 64 tokens a step,
// two buffers, everything through registers; tokens past the end are zeros in both operands.  Bound by the latencies of a step
// and by the code's own way into the CUs: bf16 [1000, 100]^T x [1000, 784] takes 9.2 us with the addition of its splits.
// ------------------------------------------------------------------------------------------
template <typename T, typename TY, int N>
__global__ __launch_bounds__(kThreads) void tokens_grad_kernel(Grad p, int splits, int tokens_per_split) {
  constexpr int kEdge = 64 * N, BK = 64, kRow = 2 * kEdge, kTile = BK * kRow;
  constexpr int kChunks = kEdge / 8, kDown = kThreads / kChunks, kRounds = BK / kDown;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[4 * kTile];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wave & 1, wn = wave >> 1;
  const int tiles_i = (p.I + kEdge - 1) / kEdge, tiles = (p.O + kEdge - 1) / kEdge * tiles_i;
  const int split = splits > 1 ? blockIdx.x / tiles : 0, tile = splits > 1 ? blockIdx.x % tiles : blockIdx.x;
  const int o0 = tile / tiles_i * kEdge, i0 = tile % tiles_i * kEdge;
  const int m0 = split * tokens_per_split;
  const int m1 = p.M - m0 < tokens_per_split ? p.M : m0 + tokens_per_split;
  // chunk ch of row k lies at ch ^ swizzle(k): the four rows that 32 lanes of a transposing read touch, 64 bytes each, fall into
  // the four quarters of the banks (rows of 256 bytes; of 128, where two rows share the banks)
  auto swizzle = [](int row) { return N == 2 ? (row & 3) << 2 : ((row >> 1) & 1) << 2; };

  // ---- staging: thread -> chunk of eight columns, rows tid / kChunks + kDown j of both tiles
  const int ch = tid % kChunks, row0 = tid / kChunks;
  const T* g = static_cast<const T*>(p.g);
  const T* last = g + p.g_last;
  const int g_col = o0 + ch * 8 < p.O ? o0 + ch * 8 : o0, x_col = i0 + ch * 8 < p.I ? i0 + ch * 8 : i0;
  u32x4 rg[kRounds];
  u32x2 rx[kRounds];
  float rs[kRounds];
  auto fetch = [&](int m) {
#pragma unroll
    for (int j = 0; j < kRounds; ++j) {
      const int at = m + row0 + kDown * j;
      const int64_t row = at < m1 ? at : m1 - 1;
      rg[j] = load_columns(g + row * p.ldg + g_col, last);
      rx[j] = *reinterpret_cast<const u32x2*>(p.x + row * p.ldx + x_col);
      rs[j] = p.scale[row];
    }
  };
  auto stage = [&](int buffer, int m) {
    uint8_t* tg = smem + buffer * 2 * kTile;
#pragma unroll
    for (int j = 0; j < kRounds; ++j) {
      const int row = row0 + kDown * j;
      const bool valid = m + row < m1;
      const int at = row * kRow + ((ch ^ swizzle(row)) << 4);
      const u32x4 none = {0u, 0u, 0u, 0u};
      *reinterpret_cast<u32x4*>(tg + at) = valid ? rg[j] : none;
      *reinterpret_cast<u32x4*>(tg + kTile + at) = values_of<T>(rx[j], valid ? rs[j] : 0.0f);
    }
  };

  // ---- fragments: lane -> column n0 + lane % 32, tokens 16 kb + 8 (lane / 32) ..
  const int blk = lane >> 4, r = lane & 15;
  const int f_row = 8 * (blk >> 1) + (r >> 2);
  auto fragment_at = [&](int n0) {
    const int c = n0 / 8 + 2 * (blk & 1) + ((r & 3) >> 1);
    return (uint32_t)(f_row * kRow + ((c ^ swizzle(f_row)) << 4) + (r & 1) * 8);
  };
  const uint32_t lds0 = lds_address(smem);
  uint32_t ag[N], ax[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    ag[i] = lds0 + fragment_at(wr * 32 * N + 32 * i);
    ax[i] = lds0 + kTile + fragment_at(wn * 32 * N + 32 * i);
  }
  f32x16 acc[N][N];
#pragma unroll
  for (int e = 0; e < N; ++e)
#pragma unroll
    for (int a = 0; a < N; ++a)
#pragma unroll
      for (int c = 0; c < 16; ++c) acc[e][a][c] = 0.0f;

  fetch(m0);
  stage(0, m0);
  __syncthreads();
  uint32_t base = 0;
  for (int m = m0; m < m1; m += BK) {
    const bool more = m + BK < m1;
    if (more) fetch(m + BK);
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) {
      auto fragment = [&](uint32_t at) {
        const u32x2 a = read_transposed(at + base + kb * 16 * kRow), b = read_transposed(at + base + (kb * 16 + 4) * kRow);
        return (u32x4){a.x, a.y, b.x, b.y};
      };
      u32x4 fg[N], fx[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        fg[i] = fragment(ag[i]);
        fx[i] = fragment(ax[i]);
      }
#pragma unroll
      for (int e = 0; e < N; ++e)
#pragma unroll
        for (int a = 0; a < N; ++a) acc[e][a] = mma16<T>(fx[e], fg[a], acc[e][a]);
    }
    if (more) stage(base ? 0 : 1, m + BK);              // (its last readers passed the barrier of the step before)
    __syncthreads();
    base ^= 2 * kTile;
  }

  // accumulator register c of a lane: feature 8 (c / 4) + 4 (lane / 32) + c % 4 of the fragment, output lane % 32: through
  // LDS, 32 outputs of the wave's features at a time, so that whole lines are stored
  constexpr int kFeatures = 32 * N, kPitch = 4 * kFeatures + 16;
  constexpr int V = 16 / sizeof(TY), kAcross = kFeatures / V, kOutputs = 64 / kAcross;
  static_assert(4 * 32 * kPitch <= 4 * kTile, "the sums of 32 outputs of four waves fit");
  const uint32_t slab = lds0 + (uint32_t)(wave * 32 * kPitch);
  const int feature = i0 + wn * kFeatures + lane % kAcross * V;
  TY* const out = static_cast<TY*>(p.out) + (int64_t)split * p.O * p.I + feature;
#pragma unroll
  for (int a = 0; a < N; ++a) {
#pragma unroll
    for (int e = 0; e < N; ++e)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        lds_store(slab + (uint32_t)((lane & 31) * kPitch + 4 * (32 * e + 8 * q + 4 * (lane >> 5))),
                  (u32x4){as_uint(acc[e][a][4 * q]), as_uint(acc[e][a][4 * q + 1]), as_uint(acc[e][a][4 * q + 2]),
                          as_uint(acc[e][a][4 * q + 3])});
    wave_lds_fence();
    for (int j = lane / kAcross; j < 32; j += kOutputs) {
      const int o = o0 + wr * 32 * N + 32 * a + j;
      float v[V];
#pragma unroll
      for (int i = 0; i < V; i += 4) {
        const u32x4 w = lds_load<u32x4>(slab + (uint32_t)(j * kPitch + (lane % kAcross * V + i) * 4));
        v[i] = as_float(w.x); v[i + 1] = as_float(w.y); v[i + 2] = as_float(w.z); v[i + 3] = as_float(w.w);
      }
      store16_part<false>(out + (int64_t)o * p.I, narrow(static_cast<const TY*>(nullptr), v), o < p.O ? p.I - feature : 0);
    }
    wave_lds_fence();
  }
}

// ------------------------------------------------------------------------------------------
// Large products: 256 outputs x 256 features a block, four waves of 128 x 128, 32 tokens a step.
//
// grad_out's rows go straight into LDS (global_load_lds; rows of whole 16-byte chunks), four buffers, loads three steps ahead.
// The codes go into LDS as they are too, four steps ahead, each wave those of its eight tokens of a step with their scales; one
// step ahead the wave turns them into values in the tile that the transposing reads take (two buffers).  So every load is one
// whose arrival the kernel counts itself, and the step only waits for those of two steps before.  A row of a tile is 512 bytes, its
// 32 chunks at chunk ^ 4 (row % 8).  Everything but the MFMAs stands beside one of them, about six instructions at most: fragment
// reads and loads in the first eight of a group of sixteen, the values two at a time in the other eight.
//
// Bound by the matrix pipes, with the conversion of the codes (two and a half instructions a value) in their shadow: fp16
// [8192, 4096]^T x [8192, 4096] takes 250 us, 1.1 PFLOP/s, as fast as the library's product of two such matrices in 16 bits.
//
// The first tokens, up to a multiple of 128, go through registers, masked: behind the last token there is nothing that may be
// multiplied, an infinite gradient times a zero would be a NaN.
// ------------------------------------------------------------------------------------------
template <typename T, typename TY>
__global__ __launch_bounds__(kThreads, 1) void tokens_grad_large_kernel(Grad p, int splits, int tokens_per_split) {
  constexpr int BO = 256, BI = 256, BK = 32, kRow = 512, kTile = BK * kRow, NA = 4, NE = 4;
  constexpr int kRawWave = 8 * 256 + 256, kRaw = 4 * kRawWave;        // codes and scales of a step
  constexpr int kX = 4 * kTile, kCodes = kX + 2 * kTile;              // where they begin
  constexpr int kGroup = NA * NE, kSlots = 2 * kGroup;
  constexpr int kLoads = 4 + 2 + 1;                                   // of a wave and step
  __shared__ __attribute__((aligned(1024))) uint8_t smem[kCodes + 4 * kRaw];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wave & 1, wn = wave >> 1;
  const int tiles_i = (p.I + BI - 1) / BI, tiles_o = (p.O + BO - 1) / BO, tiles = tiles_o * tiles_i;
  const int split = splits > 1 ? blockIdx.x / tiles : 0;
  const int tile = splits > 1 ? blockIdx.x % tiles : blockIdx.x;
  int tile_o = tile / tiles_i, tile_i = tile % tiles_i;
  if (splits == 1 && tiles_o % 8 == 0) {
    // each XCD gets panels of outputs of its own, and takes them by 8 tiles of features
    const int xcd = blockIdx.x & 7, i = blockIdx.x >> 3, panels = tiles_o / 8;
    const int strip = i / (panels * 8), in = i - strip * panels * 8;
    const int wide = tiles_i - strip * 8 < 8 ? tiles_i - strip * 8 : 8;
    tile_o = xcd * panels + in / wide;
    tile_i = strip * 8 + in % wide;
  }
  const int o0 = tile_o * BO, i0 = tile_i * BI;
  const int m_first = split * tokens_per_split;
  const int count = p.M - m_first < tokens_per_split ? p.M - m_first : tokens_per_split;
  const int masked = count % (4 * BK), steps = count / BK - masked / BK;     // steps: a multiple of four
  const T* g = static_cast<const T*>(p.g) + o0;
  const int8_t* x = p.x + i0;
  const uint32_t lds0 = lds_address(smem);

  // ---- fragments: lane -> column n0 + lane % 32, tokens 16 kb + 8 (lane / 32) ..
  const int blk = lane >> 4, r = lane & 15;
  const int f_row = 8 * (blk >> 1) + (r >> 2);
  auto fragment_at = [&](int n0) {
    const int ch = n0 / 8 + 2 * (blk & 1) + ((r & 3) >> 1);
    return (uint32_t)(f_row * kRow + ((ch ^ ((f_row & 7) << 2)) << 4) + (r & 1) * 8);
  };
  // (the second read of a fragment, four rows on, lies in the other half of the row)
  uint32_t ag[NA], ax[NE], ag2[NA], ax2[NE];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    ag[i] = lds0 + fragment_at(wr * 128 + 32 * i);
    ax[i] = lds0 + kX + fragment_at(wn * 128 + 32 * i);
    ag2[i] = ag[i] ^ 256u;
    ax2[i] = ax[i] ^ 256u;
  }
  f32x16 acc[NE][NA];
#pragma unroll
  for (int e = 0; e < NE; ++e)
#pragma unroll
    for (int a = 0; a < NA; ++a)
#pragma unroll
      for (int c = 0; c < 16; ++c) acc[e][a][c] = 0.0f;
  u32x4 fg[2][NA], fx[2][NE];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i) fg[h][i] = fx[h][i] = (u32x4){0u, 0u, 0u, 0u};
  auto read_fragment = [&](auto BUF, auto KB, auto F) {
    constexpr int buf = decltype(BUF)::value, kb = decltype(KB)::value, f = decltype(F)::value;
    constexpr bool is_g = f < NA;
    constexpr uint32_t at = (is_g ? buf : buf & 1) * kTile + kb * 16 * kRow;
    const u32x2 lo = read_transposed((is_g ? ag[f % 4] : ax[f % 4]) + at);
    const u32x2 hi = read_transposed((is_g ? ag2[f % 4] : ax2[f % 4]) + at + 4 * kRow);
    const u32x4 v = {lo.x, lo.y, hi.x, hi.y};
    if constexpr (is_g) fg[kb][f] = v;
    else fx[kb][f - NA] = v;
  };
  auto mma = [&](auto KB, int e, int a) {
    constexpr int h = decltype(KB)::value;
    acc[e][a] = mma16<T>(fx[h][e], fg[h][a], acc[e][a]);
  };

  // ---- the first tokens, through registers: thread -> chunk tid % 32 of rows tid / 32 + 8 j
  for (int m = 0; m < masked; m += BK) {
    const int ch = tid & 31;
    const bool in_g = o0 + ch * 8 < p.O, in_x = i0 + ch * 8 < p.I;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = (tid >> 5) + 8 * j;
      const bool valid = m + row < masked;
      const int64_t at = m_first + (valid ? m + row : 0);
      const u32x4 none = {0u, 0u, 0u, 0u};
      const u32x4 v = valid && in_g ? load16(g + at * p.ldg + ch * 8) : none;
      const u32x2 q = *reinterpret_cast<const u32x2*>(x + at * p.ldx + (in_x ? ch * 8 : 0));
      const uint32_t to = lds0 + (uint32_t)(row * kRow + ((ch ^ ((row & 7) << 2)) << 4));
      lds_store(to, v);
      lds_store(to + kX, values_of<T>(q, valid ? p.scale[at] : 0.0f));
    }
    __syncthreads();
    for_each<2>([&](auto KB) {
      for_each<NA + NE>([&](auto F) { read_fragment(Const<0>{}, KB, F); });
      for_each<kGroup>([&](auto G) { mma(KB, decltype(G)::value / NA, decltype(G)::value % NA); });
    });
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) fg[1][i] = fx[1][i] = (u32x4){0u, 0u, 0u, 0u};     // (multiplied once more at the start)

  if (steps > 0) {
    __syncthreads();
    const int m0 = m_first + masked;
    // ---- direct loads.  grad_out: one instruction is rows 2 rp and 2 rp + 1, rp = wave + 4 jj, LDS chunk lane % 32
    const int g_row = lane >> 5;
    const int g_chunk = (lane & 31) ^ (((2 * wave + g_row) & 7) << 2);
    const uint32_t g_lane = (uint32_t)g_row * (uint32_t)p.ldg * 2u + (o0 + g_chunk * 8 < p.O ? (uint32_t)g_chunk * 16u : 0u);
    const char* g_wave = reinterpret_cast<const char*>(g + (int64_t)(m0 + 2 * wave) * p.ldg);
    const int64_t g_step = (int64_t)BK * p.ldg * 2, g_piece = (int64_t)8 * p.ldg * 2;
    // codes: one instruction is four of the wave's eight tokens, 16 bytes a lane; scales: the even tokens' and the odd ones'
    const int c_row = lane >> 4;
    const uint32_t c_lane = (uint32_t)c_row * (uint32_t)p.ldx + (i0 + (lane & 15) * 16 < p.I ? (uint32_t)(lane & 15) * 16u : 0u);
    const int8_t* c_wave = x + (int64_t)(m0 + 8 * wave) * p.ldx;
    const int64_t c_step = (int64_t)BK * p.ldx, c_piece = (int64_t)4 * p.ldx;
    const uint32_t s_lane = (uint32_t)((lane & 3) * 2 + ((lane >> 2) & 1)) * 4u;
    const float* s_wave = p.scale + m0 + 8 * wave;
    const uint32_t lds_g = __builtin_amdgcn_readfirstlane(lds0 + wave * 1024);
    const uint32_t lds_c = __builtin_amdgcn_readfirstlane(lds0 + kCodes + wave * kRawWave);
    // (steps past the last load that one again: nobody reads it)
    auto load_g = [&](auto BUF, int t, auto J) {
      const int64_t at = t < steps ? t : steps - 1;
      load_rows(g_wave + at * g_step + decltype(J)::value * g_piece, g_lane,
                lds_g + decltype(BUF)::value * kTile + decltype(J)::value * 4096);
    };
    auto load_codes = [&](auto BUF, int t, auto J) {
      constexpr int j = decltype(J)::value;
      const int64_t at = t < steps ? t : steps - 1;
      const uint32_t to = lds_c + decltype(BUF)::value * kRaw;
      if constexpr (j < 2) load_rows(c_wave + at * c_step + j * c_piece, c_lane, to + j * 1024);
      else load_words(s_wave + at * BK, s_lane, to + 2048);
    };
    auto load_piece = [&](auto BUF, int t, auto I) {      // buffer of step t, which loads grad_out of t + 3 and codes of t + 4
      constexpr int i = decltype(I)::value, buf = decltype(BUF)::value;
      if constexpr (i < 4) load_g(Const<(buf + 3) % 4>{}, t + 3, Const<i>{});
      else load_codes(Const<buf>{}, t + 4, Const<i - 4>{});
    };

    // ---- codes to values: lane -> eight codes (lane % 32) of tokens 2 i + lane / 32 of the wave's
    const int v_row = lane >> 5;
    const uint32_t raw_at = lds0 + kCodes + wave * kRawWave + lane * 8;
    const uint32_t scale_at = lds0 + kCodes + wave * kRawWave + 2048 + v_row * 16;
    const uint32_t value_at = lds0 + kX + (uint32_t)((8 * wave + v_row) * kRow + (((lane & 31) ^ (v_row << 2)) << 4));
    u32x2 raw[4];
    u32x4 scales;
    uint32_t made[4];
    auto read_raw = [&](auto BUF, auto I) {
      constexpr int i = decltype(I)::value;
      if constexpr (i < 4) raw[i] = lds_load<u32x2>(raw_at + decltype(BUF)::value * kRaw + i * 512);
      else scales = lds_load<u32x4>(scale_at + decltype(BUF)::value * kRaw);
    };
    auto make_values = [&](auto BUF, auto I) {            // two of the lane's 32 codes; every fourth call stores 16 bytes
      constexpr int i = decltype(I)::value / 4, w = decltype(I)::value % 4;
      const u32x4 all = scales;
      const uint32_t sc = i == 0 ? all.x : i == 1 ? all.y : i == 2 ? all.z : all.w;
      const u32x2 two = raw[i];
      const uint32_t word = w < 2 ? two.x : two.y;
      made[w] = code_pair<T, w % 2>(word, as_float(sc));
      if constexpr (w == 3)
        lds_store((value_at ^ (i << 7)) + decltype(BUF)::value * kTile + i * 1024, (u32x4){made[0], made[1], made[2], made[3]});
    };

    auto step = [&](auto BUF, int t) {
      constexpr int buf = decltype(BUF)::value;
      for_each<kSlots>([&](auto S) {
        constexpr int slot = decltype(S)::value, in = slot % kGroup;
        mma(Const<1 - slot / kGroup>{}, in / NA, in % NA);
        if constexpr (in < NA + NE) {
          read_fragment(Const<buf>{}, Const<slot / kGroup>{}, Const<in>{});
          if constexpr (slot < 5) read_raw(Const<(buf + 1) % 4>{}, Const<slot>{});
          if constexpr (slot >= kGroup && in < kLoads) load_piece(Const<buf>{}, t, Const<in>{});
        } else {
          make_values(Const<(buf + 1) % 2>{}, Const<(slot / kGroup) * 8 + in - 8>{});
        }
        __builtin_amdgcn_sched_barrier(0);
      });
      __builtin_amdgcn_s_waitcnt(waitcnt_all_but(2 * kLoads));
      __syncthreads();
    };
    for_each<4>([&](auto B) { for_each<3>([&](auto J) { load_codes(B, decltype(B)::value, J); }); });
    for_each<3>([&](auto B) { for_each<4>([&](auto J) { load_g(B, decltype(B)::value, J); }); });
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    for_each<5>([&](auto I) { read_raw(Const<0>{}, I); });
    for_each<16>([&](auto I) { make_values(Const<0>{}, I); });
    __syncthreads();
    for (int t = 0; t < steps; t += 4) {
      step(Const<0>{}, t);
      step(Const<1>{}, t + 1);
      step(Const<2>{}, t + 2);
      step(Const<3>{}, t + 3);
    }
    for_each<kGroup>([&](auto G) { mma(Const<1>{}, decltype(G)::value / NA, decltype(G)::value % NA); });
  }
  __builtin_amdgcn_s_waitcnt(0);                         // (the last steps' loads write into LDS still)
  __syncthreads();

  // accumulator register c of a lane: feature 8 (c / 4) + 4 (lane / 32) + c % 4 of the fragment, output lane % 32: through
  // LDS, 32 outputs of the wave's 128 features at a time, so that whole lines are stored
  constexpr int kPitch = 4 * 128 + 16, V = 16 / sizeof(TY), kAcross = 128 / V, kDown = 64 / kAcross;
  static_assert(4 * 32 * kPitch <= kCodes, "the sums of 32 outputs of four waves fit");
  const uint32_t slab = lds0 + (uint32_t)(wave * 32 * kPitch);
  const int feature = i0 + wn * 128 + lane % kAcross * V;
  TY* const out = static_cast<TY*>(p.out) + (int64_t)split * p.O * p.I + feature;
#pragma unroll
  for (int a = 0; a < NA; ++a) {
#pragma unroll
    for (int e = 0; e < NE; ++e)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        lds_store(slab + (uint32_t)((lane & 31) * kPitch + 4 * (32 * e + 8 * q + 4 * (lane >> 5))),
                  (u32x4){as_uint(acc[e][a][4 * q]), as_uint(acc[e][a][4 * q + 1]), as_uint(acc[e][a][4 * q + 2]),
                          as_uint(acc[e][a][4 * q + 3])});
    wave_lds_fence();
#pragma unroll
    for (int j = 0; j < 32 / kDown; ++j) {
      const int o = o0 + wr * 128 + 32 * a + j * kDown + lane / kAcross;
      const uint32_t at = slab + (uint32_t)((j * kDown + lane / kAcross) * kPitch + lane % kAcross * V * 4);
      float v[V];
#pragma unroll
      for (int i = 0; i < V; i += 4) {
        const u32x4 w = lds_load<u32x4>(at + 4 * i);
        v[i] = as_float(w.x); v[i + 1] = as_float(w.y); v[i + 2] = as_float(w.z); v[i + 3] = as_float(w.w);
      }
      store16_part<false>(out + (int64_t)o * p.I, narrow(static_cast<const TY*>(nullptr), v), o < p.O ? p.I - feature : 0);
    }
    wave_lds_fence();
  }
}

template <typename TY>
__global__ __launch_bounds__(kThreads) void tokens_grad_sum_kernel(const float* __restrict__ part, TY* __restrict__ out,
                                                                   int64_t n, int splits) {
  constexpr int kAhead = 8;                              // loads on their way; the additions keep their order
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i >= n) return;
  float v = 0.0f;
  for (int s0 = 0; s0 < splits; s0 += kAhead) {
    float w[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) w[j] = part[(s0 + j < splits ? s0 + j : 0) * n + i];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) v += s0 + j < splits ? w[j] : 0.0f;
  }
  Conv<TY>::store(out, i, v);
}

// Which kernel (the edge of its tiles), and how many blocks share the tokens of a tile (`tokens` each): the cheapest by this
// estimate, us.  A step of a tile's tokens (32 for the large tiles, 64 for the others) takes step_us for each round of blocks over
// the chip's 256 CUs (the small tiles: two blocks a CU at the same time); the start and the end of a block `fixed`; splits a
// second launch of about 4.5, and their fp32 tiles are written and read back at some 8 TB/s (mostly in the last cache).  (Measured,
// large / 128 / 64: one round of 256 steps 250, two of 16 59, one of 16 12.)
struct Plan { int edge, splits, tokens; double us; };
struct Kernel { int edge, step, unit; double fixed, step_us; int64_t at_once; };
constexpr Kernel kKernels[] = {{64, 64, 64, 3.0, 0.55, 512}, {128, 64, 64, 4.0, 1.0, 256}, {256, 32, 128, 8.0, 0.9, 256}};
Plan plan_of(int64_t M, int64_t O, int64_t I, bool aligned) {
  Plan best{0, 1, 0, 0.0};
  for (const Kernel& k : kKernels) {
    if (k.edge == 256 && (!aligned || M < 512)) continue;
    const int64_t tiles = ((O + k.edge - 1) / k.edge) * ((I + k.edge - 1) / k.edge), units = (M + k.unit - 1) / k.unit;
    for (int64_t n = 1; n <= 64 && n <= units && (n == 1 || n * tiles <= 1024); n += n < 16 ? 1 : 4) {
      const double sums = n > 1 ? 4.5 + 8.0 * (double)n * (double)O * (double)I / 8.0e6 : 0.0;
      if (best.edge != 0 && k.fixed + k.step_us + sums >= best.us) break;
      const int64_t per = (units + n - 1) / n, rounds = (tiles * n + k.at_once - 1) / k.at_once;
      const double us = k.fixed + k.step_us * (double)(rounds * per * (k.unit / k.step)) + sums;
      if (best.edge == 0 || us < best.us) best = Plan{k.edge, (int)((units + per - 1) / per), (int)(per * k.unit), us};
    }
  }
  return best;
}

template <typename T, typename TY>
int launch_grad(Grad p, bool aligned, void* workspace, int64_t workspace_bytes, hipStream_t s) {
  Plan plan = plan_of(p.M, p.O, p.I, aligned);
  const int64_t n = (int64_t)p.O * p.I;
  if (plan.splits > 1 && (!workspace || workspace_bytes < 4 * n * plan.splits)) plan = Plan{plan.edge, 1, p.M, 0.0};
  const int64_t edge = plan.edge, blocks = ((p.O + edge - 1) / edge) * ((p.I + edge - 1) / edge) * plan.splits;
  if (blocks > kMostBlocks) return ACTNN_EINVAL;
  const dim3 grid((unsigned)blocks), blk(kThreads);
  auto go = [&](auto* to) {
    using TO = std::remove_pointer_t<decltype(to)>;
    p.out = to;
    if (edge == 256) tokens_grad_large_kernel<T, TO><<<grid, blk, 0, s>>>(p, plan.splits, plan.tokens);
    else if (edge == 128) tokens_grad_kernel<T, TO, 2><<<grid, blk, 0, s>>>(p, plan.splits, plan.tokens);
    else tokens_grad_kernel<T, TO, 1><<<grid, blk, 0, s>>>(p, plan.splits, plan.tokens);
  };
  TY* out = static_cast<TY*>(p.out);
  if (plan.splits == 1) {
    go(out);
  } else {
    if (!aligned16(workspace)) return ACTNN_EALIGN;
    go(static_cast<float*>(workspace));
    tokens_grad_sum_kernel<TY><<<dim3((unsigned)((n + kThreads - 1) / kThreads)), blk, 0, s>>>(
        static_cast<const float*>(workspace), out, n, plan.splits);
  }
  ACTNN_RETURN_LAUNCH_STATUS();
}
template <typename T>
int launch_out(const Grad& p, int out_dtype, void* workspace, int64_t workspace_bytes, hipStream_t s) {
  // (offsets of rows inside a wave's load are 32-bit)
  const bool aligned = aligned16(p.g) && p.ldg % 8 == 0 && p.O % 8 == 0 && p.ldg < (1 << 24) && p.ldx < (1 << 24);
  if (out_dtype == ACTNN_F32) return launch_grad<T, float>(p, aligned, workspace, workspace_bytes, s);
  return launch_grad<T, T>(p, aligned, workspace, workspace_bytes, s);
}

}  // namespace
}  // namespace actnn

extern "C" int64_t actnn_tokens_grad_weight_workspace_bytes(int64_t M, int64_t O, int64_t I) {
  using namespace actnn;
  if (M < 1 || O < 1 || I < 1 || M > 0x7fffff00LL || O > 0x7fffff00LL || I > 0x7fffff00LL) return 0;
  int64_t most = 0;
  for (const bool aligned : {false, true}) {
    const Plan plan = plan_of(M, O, I, aligned);
    if (plan.splits > 1 && 4 * O * I * plan.splits > most) most = 4 * O * I * plan.splits;
  }
  return most;
}

extern "C" int actnn_tokens_grad_weight_wants_chunks(int64_t M, int64_t O, int64_t I) {
  using namespace actnn;
  if (M < 1 || O < 1 || I < 1 || M > 0x7fffff00LL || O > 0x7fffff00LL || I > 0x7fffff00LL) return 0;
  // (a copy is two launches, and grad_out is read and written once more, at some 4 TB/s)
  return plan_of(M, O, I, true).us + 9.0 + 4.0 * (double)M * (double)O / 4.0e6 < plan_of(M, O, I, false).us;
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
