// Matrix product in 8-bit integers with a scale for each token and each output channel:
//
//     y[m, o] = scale[m] * weight_scale[o] * sum_k codes[m, k] * weight_codes[o, k]  (+ bias[o])
//
// The sum is a 32-bit integer and exact (K <= 131071: K * 2^14 < 2^31); it is converted to fp32, multiplied by the two scales,
// the bias is added, and the result is rounded to the output's type.  Sums that are split over blocks or waves are
// added as integers: the order does not matter.
//
// Three kernels share the work:
//   * few tokens (up to 32, where the estimate below has this cheaper than tiles): a wave's lanes load their 16 bytes of 16
//     channels' rows straight into the operand registers of v_mfma_i32_16x16x64_i8, the waves of a block share the features of
//     the same channels and add their sums in LDS.
//   * tiles of 64, 128 or 256 channels by as many tokens, for everything else ([24, 4096] -> 16384 among it):
//     v_mfma_i32_32x32x32_i8 out of LDS.  Four buffers of 64 or 128 features; both operands go from global memory straight into LDS (global_load_lds, 16 bytes a lane), rows as they
//     lie in memory, their 16-byte chunks permuted so that 16 rows that are read together meet every bank once.
//   * tiles that do not fill the chip take slices of the features; a second kernel adds the slices.
// Rows and channels past the end are read from the last one and not stored; features past the end are read from the
// step's first chunk and masked out of the weight's operand.
#include <type_traits>

#include "matrix_tiles.h"
#include "token_math.h"

namespace actnn {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

constexpr int kThreads = 256;
constexpr int64_t kMostFeatures = 131071;               // the integer sum of so many products fits 32 bits
constexpr int64_t kMostStride = 0x7fffff;               // 256 rows of so many bytes stay below 2 GiB
constexpr int64_t kMostOutputs = 0x3ffffff;             // 16 of them to a block

// the first `valid` of 16 bytes, the others 0
ACTNN_DEV u32x4 first_bytes(u32x4 v, int valid) {
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int n = valid - 4 * i;
    w[i] = n >= 4 ? w[i] : n <= 0 ? 0u : w[i] & ((1u << (8 * n)) - 1u);
  }
  return (u32x4){w[0], w[1], w[2], w[3]};
}

struct Product {
  const int8_t* x;                       // token codes [M, K], rows `ldx` bytes apart
  const float* xs;
  const int8_t* w;                       // weight codes [O, K]
  const float* ws;
  const float* bias;                     // [O] or null
  void* y;                               // [M, O]; slices: int32 [slices][M, O]
  int64_t ldx, ldw;
  int M, K, O;
};

// The sum times the token's scale times the channel's.  Times a scale above 2^90 it may pass the largest number where the result
// does not, if the other scale is small: then that one comes first (and if that passes it too, the result does).
constexpr float kLargeScale = 0x1p90f;
ACTNN_DEV float scaled_usually(int sum, float xs, float ws, float bias) { return __builtin_fmaf((float)sum * xs, ws, bias); }
ACTNN_DEV float scaled(int sum, float xs, float ws, float bias) {
  return xs > kLargeScale ? scaled_usually(sum, ws, xs, bias) : scaled_usually(sum, xs, ws, bias);
}

// four consecutive channels of a token, from their integer sums
template <typename TY> ACTNN_DEV void put4(const Product& p, int64_t token, int channel, const int (&sum)[4], float xs) {
  TY* to = static_cast<TY*>(p.y) + token * p.O + channel;
  float v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = channel + i < p.O ? channel + i : p.O - 1;
    v[i] = scaled(sum[i], xs, p.ws[c], p.bias ? p.bias[c] : 0.0f);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (channel + i < p.O) Conv<TY>::store(to, i, v[i]);
}
// the integer sums of 16 bytes' worth of channels of a token, of which `valid` exist; LARGE: its scale may be above kLargeScale
template <typename TY, bool LARGE, int V>
ACTNN_DEV void put_row(TY* to, int valid, const int (&sum)[V], float xs, const float (&ws)[V], const float (&bias)[V]) {
  u32x4 out;
  if constexpr (std::is_same<TY, int>::value) {
    out = (u32x4){(uint32_t)sum[0], (uint32_t)sum[1], (uint32_t)sum[2], (uint32_t)sum[3]};
    store16_part<false>(reinterpret_cast<float*>(to), out, valid);
  } else {
    float v[V];
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = LARGE ? scaled(sum[i], xs, ws[i], bias[i]) : scaled_usually(sum[i], xs, ws[i], bias[i]);
    store16_part<false>(to, narrow(static_cast<const TY*>(nullptr), v), valid);
  }
}

// ------------------------------------------------------------------------------------------
// Tiles.  Four waves, two by two; a wave has NA x NE fragments of 32 channels x 32 tokens.
//
// Bound by the matrix pipes and by what reaches them: a wave of the largest tile holds 128 x 128 sums in its 256 accumulation
// registers, so that a byte read from LDS meets 64 products.  [8192, 4096] x [4096, 4096] takes 131 to 136 us, 2.0 to 2.1 POPS (the
// library's product of such matrices in bf16: 1.2; the pipes alone, fed from registers, reach 3.2 on such codes, 4.4 on zeros:
// the clock follows the power).  When it took 136 us, 113 remained without the loads into LDS and 87 without the reads from it.
// ------------------------------------------------------------------------------------------
// BK features a step; WHOLE: the features are whole steps.
template <typename TY, int NA, int NE, int BK, bool WHOLE>
__global__ __launch_bounds__(kThreads, 1) void tokens_tile_kernel(Product p, int slices, int steps_per_slice) {
  constexpr int BO = 64 * NA, BT = 64 * NE, kBuffers = 4, kBlocks = BK / 32;
  constexpr int kChunks = BK / 16, kPieceRows = 64 / kChunks;         // 16-byte chunks of a row, rows of a direct load
  constexpr int kBuffer = (BO + BT) * BK;
  constexpr int kGroup = NA * NE, kSlots = kBlocks * kGroup, kFragments = NA + NE;
  constexpr int kReads = (kFragments + kGroup - 1) / kGroup;          // fragment reads beside an MFMA
  constexpr int kPieces = kBuffer / (kThreads * 16), kWeightPieces = BO * BK / (kThreads * 16);   // direct loads of a wave and step
  __shared__ __attribute__((aligned(1024))) uint8_t smem[kBuffers * kBuffer];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = wave & 1, wn = wave >> 1;
  const int tiles_o = (p.O + BO - 1) / BO, tiles_t = (p.M + BT - 1) / BT;
  const int slice = slices > 1 ? blockIdx.x / (tiles_o * tiles_t) : 0;
  const int tile = slices > 1 ? blockIdx.x % (tiles_o * tiles_t) : blockIdx.x;
  int tile_t = tile / tiles_o, tile_o = tile % tiles_o;
  if (slices == 1 && tiles_t % 8 == 0) {
    // Blocks are dealt round-robin to the 8 XCDs: each gets panels of tokens of its own, and takes them by 8 tiles of
    // channels, so that the tiles at work at one time share their operands in its L2.
    const int xcd = blockIdx.x & 7, i = blockIdx.x >> 3, panels = tiles_t / 8;
    const int strip = i / (panels * 8), in = i - strip * panels * 8;
    const int wide = tiles_o - strip * 8 < 8 ? tiles_o - strip * 8 : 8;
    tile_t = xcd * panels + in / wide;
    tile_o = strip * 8 + in % wide;
  }
  const int t0 = tile_t * BT, o0 = tile_o * BO;
  const int all_steps = (p.K + BK - 1) / BK;
  const int first = slice * steps_per_slice;
  int steps = all_steps - first;
  if (slices > 1 && steps > steps_per_slice) steps = steps_per_slice;
  if (slices > 1) p.y = static_cast<int*>(p.y) + (int64_t)slice * p.M * p.O;
  const int chunks = (p.K + 15) / 16;
  const int features = (p.K < (first + steps) * BK ? p.K : (first + steps) * BK) - first * BK;     // of this block

  const uint32_t lds0 = lds_address(smem);
  const uint32_t lds_wave = __builtin_amdgcn_readfirstlane(lds0 + wave * 1024);

  // Chunk c of row r lies at c ^ swizzle(r): 16 rows that are read together meet every bank once.
  auto swizzle = [](int row) { return (row * kChunks / 16) & (kChunks - 1); };

  // ---- direct loads: piece j is kPieceRows rows of the weight's tile or, behind those, of the tokens'; a wave's pieces
  // are 4 kPieceRows rows apart, which leaves the swizzle as it is
  const int row_in = lane / kChunks;
  const int chunk = (lane % kChunks) ^ swizzle(kPieceRows * wave + row_in);
  uint32_t off[kPieces];
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int row = kPieceRows * (wave + 4 * i) + row_in;
    if (i < kWeightPieces) {
      const int at = o0 + row < p.O ? row : p.O - 1 - o0;
      off[i] = (uint32_t)at * (uint32_t)p.ldw + (uint32_t)chunk * 16u;
    } else {
      const int at = t0 + row - BO < p.M ? row - BO : p.M - 1 - t0;
      off[i] = (uint32_t)at * (uint32_t)p.ldx + (uint32_t)chunk * 16u;
    }
  }
  const int8_t* wp = p.w + (int64_t)o0 * p.ldw;
  const int8_t* xp = p.x + (int64_t)t0 * p.ldx;
  // (a step past the block's last loads that one again: nobody reads it)
  auto load_piece = [&](auto BUF, int t, auto I) {
    constexpr int i = decltype(I)::value;
    const int step = first + (t < steps ? t : steps - 1);
    uint32_t at = off[i];
    if constexpr (!WHOLE) {
      if (step * kChunks + chunk >= chunks) at -= (uint32_t)chunk * 16u;     // past the row's end: the step's first chunk
    }
    const int8_t* base = (i < kWeightPieces ? wp : xp) + (int64_t)step * BK;
    load_rows(base, at, lds_wave + decltype(BUF)::value * kBuffer + i * 4096);
  };

  // ---- fragments: lane -> row lane % 32, features 32 kb + 16 (lane / 32) ..
  const uint32_t in_row = (uint32_t)(lane & 31) * BK + (uint32_t)(((lane >> 5) ^ swizzle(lane & 31)) << 4);
  const uint32_t at_w = lds0 + (uint32_t)(wr * 32 * NA) * BK + in_row;
  const uint32_t at_x = lds0 + (uint32_t)(BO + wn * 32 * NE) * BK + in_row;

  i32x16 acc[NE][NA];
#pragma unroll
  for (int e = 0; e < NE; ++e)
#pragma unroll
    for (int a = 0; a < NA; ++a)
#pragma unroll
      for (int c = 0; c < 16; ++c) acc[e][a][c] = 0;
  u32x4 fw[2][NA], fx[2][NE];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int a = 0; a < NA; ++a) fw[h][a] = (u32x4){0u, 0u, 0u, 0u};
#pragma unroll
    for (int e = 0; e < NE; ++e) fx[h][e] = (u32x4){0u, 0u, 0u, 0u};
  }
  auto read_fragment = [&](auto BUF, auto KB, auto F, auto TAIL, int t) {
    constexpr int kb = decltype(KB)::value, f = decltype(F)::value;
    constexpr uint32_t buf = decltype(BUF)::value * kBuffer;
    if constexpr (f < NA) {
      u32x4 v = lds_load<u32x4>((at_w ^ (kb << 5)) + buf + f * 32 * BK);
      if constexpr (decltype(TAIL)::value != 0) v = first_bytes(v, features - (t * BK + kb * 32 + (lane >> 5) * 16));
      fw[kb & 1][f] = v;
    } else {
      fx[kb & 1][f - NA] = lds_load<u32x4>((at_x ^ (kb << 5)) + buf + (f - NA) * 32 * BK);
    }
  };
  auto mma = [&](auto KB, int e, int a) {
    constexpr int h = decltype(KB)::value & 1;
    acc[e][a] = __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, fw[h][a]), __builtin_bit_cast(i32x4, fx[h][e]),
                                                      acc[e][a], 0, 0, 0);
  };

  // Step t is multiplied out of buffer t % 4.  Between two barriers: the MFMAs of the last k-block of the step before (its
  // fragments are in registers) and of all but the last of this one, the fragments of each k-block read beside the MFMAs of the
  // one before, and the direct loads of step t + 3 into the buffer whose last readers passed the barrier before.  The step
  // ends when the loads of step t + 1 have landed: those of two steps may be on their way.
  // (a direct load and what it takes stand beside MFMAs without fragment reads where there are any, half of them in either
  // group: about six instructions fit beside one)
  constexpr bool kRoom = kBlocks == 2 && kGroup >= kFragments + kPieces;
  constexpr auto load_slot = [](int i) {
    return !kRoom ? i * kSlots / kPieces : i < kPieces / 2 ? kFragments + 2 * i : kGroup + kFragments + 2 * (i - kPieces / 2);
  };
  static_assert(load_slot(kPieces - 1) < kSlots, "every load has its place");
  constexpr int kLandedOne = waitcnt_all_but(2 * kPieces);
  // (no branches in a body: the compiler's own waits for LDS then stay exact)
  auto step = [&](auto BUF, auto TAIL, auto AHEAD, int t) {
    constexpr int buf = decltype(BUF)::value;
    constexpr bool ahead = decltype(AHEAD)::value != 0;
    for_each<kSlots>([&](auto S) {
      constexpr int slot = decltype(S)::value, in = slot % kGroup;
      mma(Const<(slot / kGroup + 1) % 2>{}, in / NA, in % NA);              // (of the k-block before: kBlocks is even)
      for_each<kReads>([&](auto R) {
        constexpr int f = in * kReads + decltype(R)::value;
        if constexpr (f < kFragments) read_fragment(Const<buf>{}, Const<slot / kGroup>{}, Const<f>{}, TAIL, t);
      });
      for_each<kPieces>([&](auto I) {
        constexpr int i = decltype(I)::value;
        if constexpr (ahead && slot == load_slot(i)) load_piece(Const<(buf + 3) % kBuffers>{}, t + 3, Const<i>{});
      });
      __builtin_amdgcn_sched_barrier(0);
    });
    __builtin_amdgcn_s_waitcnt(ahead ? kLandedOne : 0);
    __syncthreads();
  };
  for_each<kPieces>([&](auto I) { load_piece(Const<0>{}, 0, I); });
  for_each<kPieces>([&](auto I) { load_piece(Const<1>{}, 1, I); });
  for_each<kPieces>([&](auto I) { load_piece(Const<2>{}, 2, I); });
  __builtin_amdgcn_s_waitcnt(kLandedOne);
  __syncthreads();
  // The last one to four steps, masked, stand behind the loop once, and the steps that are missing there add zeros: with
  // bodies under conditions the accumulators were copied and spilled where their paths met.
  int t = 0;
  for (; t + 4 < steps; t += 4) {
    step(Const<0>{}, Const<0>{}, Const<1>{}, t);
    step(Const<1>{}, Const<0>{}, Const<1>{}, t + 1);
    step(Const<2>{}, Const<0>{}, Const<1>{}, t + 2);
    step(Const<3>{}, Const<0>{}, Const<1>{}, t + 3);
  }
  step(Const<0>{}, Const<1>{}, Const<1>{}, t);
  step(Const<1>{}, Const<1>{}, Const<0>{}, t + 1);
  step(Const<2>{}, Const<1>{}, Const<0>{}, t + 2);
  step(Const<3>{}, Const<1>{}, Const<0>{}, t + 3);
  for_each<kGroup>([&](auto G) { mma(Const<1>{}, decltype(G)::value / NA, decltype(G)::value % NA); });

  // Accumulator register c of a lane: channel 8 (c / 4) + 4 (lane / 32) + c % 4 of the fragment, token lane % 32.  Stored
  // from there a wave would write 8 bytes each into 32 rows.  The sums go through LDS instead (all of it is free: the last
  // fragments were read before the last barrier), 32 tokens of the wave's channels at a time, and come back with a lane's
  // channels side by side: whole lines, and a lane's scales and biases are the same for all its tokens.
  constexpr int kChannels = 32 * NA, kPitch = 4 * kChannels + 16;     // bytes a token; the 16 keep rows off the same banks
  constexpr int V = sizeof(TY) == 2 ? 8 : 4;                          // channels of a 16-byte store
  constexpr int kAcross = kChannels / V, kDown = 64 / kAcross;        // lanes to a token, tokens to an instruction
  static_assert(4 * 32 * kPitch <= kBuffers * kBuffer, "the sums of 32 tokens of four waves fit where the tiles were");
  const uint32_t slab = lds0 + (uint32_t)(wave * 32 * kPitch);
  const int channel = o0 + wr * kChannels + lane % kAcross * V;
  const int valid = p.O - channel;
  float ws[V], bias[V];
  if constexpr (!std::is_same<TY, int>::value) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = channel + i < p.O ? channel + i : p.O - 1;
      ws[i] = p.ws[c];
      bias[i] = p.bias ? p.bias[c] : 0.0f;
    }
  }
  TY* const out = static_cast<TY*>(p.y) + channel;
#pragma unroll
  for (int e = 0; e < NE; ++e) {
    const int first_token = t0 + wn * 32 * NE + 32 * e + lane / kAcross;
    auto scale_of = [&](int j) { return p.xs[first_token + j * kDown < p.M ? first_token + j * kDown : p.M - 1]; };
    float xs[32 / kDown];
    bool large = false;
#pragma unroll
    for (int j = 0; j < 32 / kDown; ++j) {
      xs[j] = scale_of(j);
      large = large || xs[j] > kLargeScale;
    }
#pragma unroll
    for (int a = 0; a < NA; ++a)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        lds_store(slab + (uint32_t)((lane & 31) * kPitch + 4 * (32 * a + 8 * q + 4 * (lane >> 5))),
                    (u32x4){(uint32_t)acc[e][a][4 * q], (uint32_t)acc[e][a][4 * q + 1], (uint32_t)acc[e][a][4 * q + 2],
                            (uint32_t)acc[e][a][4 * q + 3]});
    wave_lds_fence();
    auto put = [&](int j, float scale, auto LARGE) {
      const int64_t token = first_token + j * kDown;
      const uint32_t at = slab + (uint32_t)((j * kDown + lane / kAcross) * kPitch + lane % kAcross * V * 4);
      int sum[V];
#pragma unroll
      for (int i = 0; i < V; i += 4) {
        const u32x4 v = lds_load<u32x4>(at + 4 * i);
        sum[i] = (int)v.x; sum[i + 1] = (int)v.y; sum[i + 2] = (int)v.z; sum[i + 3] = (int)v.w;
      }
      put_row<TY, decltype(LARGE)::value != 0>(out + token * p.O, token < p.M ? valid : 0, sum, scale, ws, bias);
    };
    // (a branch of the wave: a choice for each value takes 4 of the largest product's 133 us)
    if (!std::is_same<TY, int>::value && __builtin_expect(__any(large), 0)) {
#pragma unroll 1
      for (int j = 0; j < 32 / kDown; ++j) put(j, scale_of(j), Const<1>{});
    } else {
#pragma unroll
      for (int j = 0; j < 32 / kDown; ++j) put(j, xs[j], Const<0>{});
    }
    wave_lds_fence();
  }
}

// ------------------------------------------------------------------------------------------
// Few tokens, up to 32: 16 channels a block, MT tiles of 16 tokens; the waves share the features, a run of pieces of 64 each.
// Bound by the latency of a wave's loads, 4 pieces ahead, and past some 4.5 TB/s of weight by those: [12, 4096] -> 4096 takes 5.9.
// ------------------------------------------------------------------------------------------
constexpr int kFew = 32;
template <typename TY, int MT>
__global__ __launch_bounds__(kThreads) void tokens_few_kernel(Product p) {
  constexpr int kAhead = 4, WAVES = kThreads / 64;
  __shared__ i32x4 s_sum[WAVES][MT][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int o0 = blockIdx.x * 16;
  const int row = lane & 15, part = lane >> 4;
  const int8_t *wp = p.w + (int64_t)(o0 + row < p.O ? o0 + row : p.O - 1) * p.ldw, *xp[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) xp[i] = p.x + (int64_t)(16 * i + row < p.M ? 16 * i + row : p.M - 1) * p.ldx;
  i32x4 acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) acc[i] = (i32x4){0, 0, 0, 0};
  const int pieces = (p.K + 63) / 64, per = (pieces + WAVES - 1) / WAVES;
  const int end = (wave + 1) * per < pieces ? (wave + 1) * per : pieces;
  for (int c0 = wave * per; c0 < end; c0 += kAhead) {
    u32x4 fw[kAhead], fx[kAhead][MT];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      int k = (c0 + j) * 64 + part * 16;
      k = k < p.K && c0 + j < end ? k : 0;                             // (masked below)
      fw[j] = load16(wp + k);
#pragma unroll
      for (int i = 0; i < MT; ++i) fx[j][i] = load16(xp[i] + k);
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int left = c0 + j < end ? p.K - (c0 + j) * 64 - part * 16 : 0;
      const u32x4 w = left < 16 ? first_bytes(fw[j], left) : fw[j];
#pragma unroll
      for (int t = 0; t < MT; ++t)
        acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, w), __builtin_bit_cast(i32x4, fx[j][t]),
                                                       acc[t], 0, 0, 0);
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) s_sum[wave][t][lane] = acc[t];
  __syncthreads();
  // accumulator register c of a lane: channel 4 (lane / 16) + c, token lane % 16
  for (int i = threadIdx.x; i < MT * 64; i += kThreads) {
    const int tile = i >> 6, in = i & 63;
    i32x4 v = s_sum[0][tile][in];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) v += s_sum[w][tile][in];
    const int sum[4] = {v.x, v.y, v.z, v.w};
    const int channel = o0 + 4 * (in >> 4), token = 16 * tile + (in & 15);
    if (channel < p.O && token < p.M) put4<TY>(p, token, channel, sum, p.xs[token]);
  }
}

// ------------------------------------------------------------------------------------------
// One to four tokens in full precision: every block turns them into codes for itself, in LDS, while its first pieces of the
// weight are on their way; a launch and the wait between two are saved (one bf16 token x [4096, 4096]: 6.5 us, 9.7 by two
// kernels; its 16.8 MB of codes come at 2.6 TB/s, bound by the latencies of the start).
// ------------------------------------------------------------------------------------------
constexpr int kFused = 4;
constexpr int kFusedFeatures = 16384;
template <typename T>
__global__ __launch_bounds__(kThreads) void tokens_linear_few_kernel(Product p, const T* __restrict__ x, int64_t ld) {
  constexpr int E = kVector<T>, WAVES = kThreads / 64, kAhead = 4;
  extern __shared__ __attribute__((aligned(16))) uint8_t s_codes[];    // [M][K to the next multiple of 64]
  __shared__ uint32_t s_top[WAVES][kFused], s_scale[kFused];
  __shared__ i32x4 s_sum[WAVES][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int o0 = blockIdx.x * 16;
  const int row = lane & 15, part = lane >> 4;
  const int8_t* wp = p.w + (int64_t)(o0 + row < p.O ? o0 + row : p.O - 1) * p.ldw;
  const int pieces = (p.K + 63) / 64, per = (pieces + WAVES - 1) / WAVES, pitch = pieces * 64;
  const int first = wave * per, end = first + per < pieces ? first + per : pieces;
  u32x4 next[kAhead];
  auto fetch = [&](int c0) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int k = (c0 + j) * 64 + part * 16;
      next[j] = load16(wp + (k < p.K && c0 + j < end ? k : 0));        // (the codes behind the last feature are zeros)
    }
  };
  fetch(first);
  const int vectors = p.K / E;
  for (int m = 0; m < p.M; ++m) {
    Top<T> top;
    for (int v = threadIdx.x; v < vectors; v += kThreads) top.add(load16(x + m * ld + (int64_t)v * E));
    const uint32_t largest = lanes_largest(top.one());
    if (lane == 0) s_top[wave][m] = largest;
  }
  __syncthreads();
  for (int m = 0; m < p.M; ++m) {
    uint32_t largest = s_top[0][m];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) largest = largest > s_top[w][m] ? largest : s_top[w][m];
    const float value = Top<T>::value(largest);
    const TokenScale ts = token_scale(value);
    const Coder<T> coder(value);
    typedef typename CodeWords<T>::type Words;
    Words* codes = reinterpret_cast<Words*>(s_codes + m * pitch);
    for (int v = threadIdx.x; v < pitch / E; v += kThreads) {
      float f[E];
      widen(static_cast<const T*>(nullptr), load16(x + m * ld + (int64_t)(v < vectors ? v : 0) * E), f);
      codes[v] = codes_of<T>(coder, f, v < vectors ? ts.keep : 0u);
    }
    if (threadIdx.x == 0) s_scale[m] = as_uint(ts.scale);
  }
  __syncthreads();
  const uint8_t* xp = s_codes + (row < p.M ? row : 0) * pitch;
  i32x4 acc = {0, 0, 0, 0};
  for (int c0 = first; c0 < end; c0 += kAhead) {
    u32x4 fw[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) fw[j] = next[j];
    fetch(c0 + kAhead);
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const u32x4 zero = {0u, 0u, 0u, 0u};
      const u32x4 fx = *reinterpret_cast<const u32x4*>(xp + (c0 + j < end ? c0 + j : first) * 64 + part * 16);
      const u32x4 w = c0 + j < end ? fw[j] : zero;
      acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, w), __builtin_bit_cast(i32x4, fx), acc, 0, 0, 0);
    }
  }
  s_sum[wave][lane] = acc;
  __syncthreads();
  if (wave == 0) {
    i32x4 v = s_sum[0][lane];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) v += s_sum[w][lane];
    const int sum[4] = {v.x, v.y, v.z, v.w};
    const int channel = o0 + 4 * part;
    if (channel < p.O && row < p.M) put4<T>(p, row, channel, sum, as_float(s_scale[row]));
  }
}

// the sum of the slices
template <typename TY>
__global__ __launch_bounds__(kThreads) void tokens_sum_slices_kernel(Product p, const int* __restrict__ part, int slices) {
  const int64_t n = (int64_t)p.M * p.O;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kThreads) {
    int sum = 0;
    for (int s = 0; s < slices; ++s) sum += part[s * n + i];
    const int64_t token = i / p.O;
    const int channel = (int)(i - token * p.O);
    Conv<TY>::store(static_cast<TY*>(p.y), i, scaled(sum, p.xs[token], p.ws[channel], p.bias ? p.bias[channel] : 0.0f));
  }
}

// Which kernel - the tile, 0: few tokens - and slices of the features, of `steps` steps each: the cheapest by this estimate, us.
// A step takes step_us for each round of blocks over the chip's 256 CUs, 0.7 of it for half a round or less (the last round of the
// smaller tiles, two of which share a CU, may be half a round); the start and the end of a block, the fetch of its code among
// them, `fixed`; slices a second launch of about 4.5, and their sums are written and read back at some 8 TB/s.  Measured, tile 64
// by 64 features / 64 by 128 / 128 / 256, us: 256 x 4096 x 4096 (tokens, features, outputs) 12.2, 10.0, 18.9, 42;
// 1024 x 4096 x 4096 36.1, 29.6, 27.9, 42.8; 8192 x 4096 x 4096 248, 205, 169, 125 (133 now); 512 x 1024 x 2048 6.3, 6.6, 7.6, 18.8.  Few
// tokens without tiles: 0.7 (1.1 for more than 16) for every 1024 features that its waves walk alone, or the weight at 4.5 TB/s,
// and 2 for start and end (without tiles / by them: 24 x 4096 x 1024 6.7, 10.8; 24 x 4096 x 16384 21.2, 13.1; 16 x 16384 x 100
// 15.9, 10.1; 61 x 7326 x 1790, which none of it takes, 15.5, 11.8).
struct Plan { int tile, slices, steps; };
struct Tile { int edge, features; double fixed, step_us; };
constexpr Tile kTiles[] = {{0, 1, 0.0, 0.0}, {64, 64, 3.0, 0.15}, {64, 128, 4.0, 0.25}, {128, 64, 5.0, 0.32},
                           {256, 64, 12.0, 0.88}};
Plan plan_of(int64_t M, int64_t K, int64_t O) {
  Plan best{0, 1, 0};
  const bool few = M <= kFew;
  const double alone = (M <= 16 ? 0.7 : 1.1) * (double)K / 1024.0, together = (double)K * (double)O / 4.5e6;
  double least = 2.0 + (alone > together ? alone : together);
  for (int i = 1; i < (int)(sizeof(kTiles) / sizeof(kTiles[0])); ++i) {
    const Tile& t = kTiles[i];
    const int64_t tiles = ((M + t.edge - 1) / t.edge) * ((O + t.edge - 1) / t.edge), steps = (K + t.features - 1) / t.features;
    for (int64_t n = 1; n <= 16 && n <= steps && (n == 1 || n * tiles <= 512); ++n) {
      const double sums = n > 1 ? 4.5 + 8.0 * (double)n * (double)M * (double)O / 8.0e6 : 0.0;
      if ((best.tile != 0 || few) && t.fixed + sums >= least) break;
      const int64_t per = (steps + n - 1) / n;
      const int64_t blocks = tiles * n;
      const double rounds = blocks <= 128    ? 0.7
                            : t.edge == 256 ? (double)((blocks + 255) / 256)
                                            : 0.5 * (double)((blocks + 127) / 128);
      const double us = t.fixed + t.step_us * rounds * (double)per + sums;
      if ((best.tile == 0 && !few) || us < least) {
        least = us;
        best = Plan{i, (int)((steps + per - 1) / per), (int)per};
      }
    }
  }
  return best;
}

template <typename TY, int I> void launch_tiles(const Product& p, const Plan& plan, int64_t blocks, hipStream_t s) {
  constexpr int N = kTiles[I].edge / 64, BK = kTiles[I].features;
  const dim3 grid((unsigned)blocks), blk(kThreads);
  if (p.K % BK == 0) tokens_tile_kernel<TY, N, N, BK, true><<<grid, blk, 0, s>>>(p, plan.slices, plan.steps);
  else tokens_tile_kernel<TY, N, N, BK, false><<<grid, blk, 0, s>>>(p, plan.slices, plan.steps);
}
template <typename TY> void launch_tile(const Product& p, const Plan& plan, int64_t blocks, hipStream_t s) {
  switch (plan.tile) {
    case 1: return launch_tiles<TY, 1>(p, plan, blocks, s);
    case 2: return launch_tiles<TY, 2>(p, plan, blocks, s);
    case 3: return launch_tiles<TY, 3>(p, plan, blocks, s);
    default: return launch_tiles<TY, 4>(p, plan, blocks, s);
  }
}
template <typename TY, int MT> void launch_few(const Product& p, hipStream_t s) {
  tokens_few_kernel<TY, MT><<<dim3((unsigned)((p.O + 15LL) / 16)), dim3(kThreads), 0, s>>>(p);
}

template <typename TY> int product(const Product& p, void* workspace, int64_t workspace_bytes, hipStream_t s) {
  Plan plan = plan_of(p.M, p.K, p.O);
  if (plan.tile == 0) {
    if (p.M <= 16) launch_few<TY, 1>(p, s);
    else launch_few<TY, 2>(p, s);
    ACTNN_RETURN_LAUNCH_STATUS();
  }
  const int64_t n = (int64_t)p.M * p.O;
  if (plan.slices > 1 && (!workspace || workspace_bytes < 4 * n * plan.slices)) plan = Plan{plan.tile, 1, 0};
  const int64_t edge = kTiles[plan.tile].edge;
  const int64_t blocks = (p.M + edge - 1) / edge * ((p.O + edge - 1) / edge) * plan.slices;
  if (blocks > kMostBlocks) return ACTNN_EINVAL;
  if (plan.slices == 1) {
    launch_tile<TY>(p, plan, blocks, s);
  } else {
    if (!aligned16(workspace)) return ACTNN_EALIGN;
    Product parts = p;
    parts.y = workspace;
    launch_tile<int>(parts, plan, blocks, s);
    const int64_t sums = (n + kThreads - 1) / kThreads;
    tokens_sum_slices_kernel<TY><<<dim3((unsigned)(sums < 4096 ? sums : 4096)), dim3(kThreads), 0, s>>>(
        p, static_cast<const int*>(workspace), plan.slices);
  }
  ACTNN_RETURN_LAUNCH_STATUS();
}

}  // namespace
}  // namespace actnn

extern "C" int64_t actnn_tokens_matmul_workspace_bytes(int64_t M, int64_t K, int64_t O) {
  using namespace actnn;
  if (M < 1 || K < 1 || O < 1 || M > 0x7fffff00LL || O > kMostOutputs || K > kMostFeatures) return 0;
  const Plan plan = plan_of(M, K, O);
  return plan.slices > 1 ? 4 * M * O * plan.slices : 0;
}

extern "C" int actnn_tokens_matmul(const int8_t* codes, int64_t ldc, const float* scale, const int8_t* weight_codes,
                                   int64_t ldw, const float* weight_scale, const float* bias, void* out, int64_t M,
                                   int64_t K, int64_t O, int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace actnn;
  if (M < 0 || O < 0 || K < 1 || K > kMostFeatures || M > 0x7fffff00LL || O > kMostOutputs) return ACTNN_EINVAL;
  if (ldc < K || ldc % 16 || ldc > kMostStride || ldw < K || ldw % 16 || ldw > kMostStride) return ACTNN_EINVAL;
  if (dtype != ACTNN_F32 && dtype != ACTNN_F16 && dtype != ACTNN_BF16) return ACTNN_EDTYPE;
  if (M == 0 || O == 0) return ACTNN_OK;
  if (!codes || !scale || !weight_codes || !weight_scale || !out) return ACTNN_EINVAL;
  if (!aligned16(codes) || !aligned16(weight_codes) || reinterpret_cast<uintptr_t>(out) % (dtype == ACTNN_F32 ? 4 : 2) != 0)
    return ACTNN_EALIGN;
  const Product p{codes, scale, weight_codes, weight_scale, bias, out, ldc, ldw, (int)M, (int)K, (int)O};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == ACTNN_F32) return product<float>(p, workspace, workspace_bytes, s);
  if (dtype == ACTNN_F16) return product<__half>(p, workspace, workspace_bytes, s);
  return product<bf16_t>(p, workspace, workspace_bytes, s);
}

namespace actnn {
namespace {
template <typename T> void launch_linear_few(const Product& p, const void* x, int64_t ld, hipStream_t s) {
  const size_t lds = (size_t)p.M * ((p.K + 63) / 64 * 64);
  tokens_linear_few_kernel<T><<<dim3((unsigned)((p.O + 15) / 16)), dim3(kThreads), lds, s>>>(p, static_cast<const T*>(x), ld);
}
}  // namespace
}  // namespace actnn

extern "C" int actnn_tokens_linear_few(const void* data, int64_t ld, const int8_t* weight_codes, int64_t ldw,
                                       const float* weight_scale, const float* bias, void* out, int64_t M, int64_t K, int64_t O,
                                       int dtype, void* stream) {
  using namespace actnn;
  if (M < 0 || M > kFused || K < 1 || K > kFusedFeatures || O < 0 || O > kMostOutputs || ld < 0) return ACTNN_EINVAL;
  if (ldw < K || ldw % 16 || ldw > kMostStride) return ACTNN_EINVAL;
  if (dtype != ACTNN_F32 && dtype != ACTNN_F16 && dtype != ACTNN_BF16) return ACTNN_EDTYPE;
  const int64_t vector = dtype == ACTNN_F32 ? 4 : 8;
  if (K % vector || ld % vector) return ACTNN_EINVAL;
  if (M == 0 || O == 0) return ACTNN_OK;
  if (!data || !weight_codes || !weight_scale || !out) return ACTNN_EINVAL;
  if (!aligned16(data) || !aligned16(weight_codes) || reinterpret_cast<uintptr_t>(out) % (16 / vector)) return ACTNN_EALIGN;
  const Product p{nullptr, nullptr, weight_codes, weight_scale, bias, out, 0, ldw, (int)M, (int)K, (int)O};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == ACTNN_F32) launch_linear_few<float>(p, data, ld, s);
  else if (dtype == ACTNN_F16) launch_linear_few<__half>(p, data, ld, s);
  else launch_linear_few<bf16_t>(p, data, ld, s);
  ACTNN_RETURN_LAUNCH_STATUS();
}
