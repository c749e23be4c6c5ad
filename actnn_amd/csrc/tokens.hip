// 8-bit tokens: rows of features written as codes with one scale a row, and read back.
//
//   codes[m, k] = sign(x) floor(127 |x[m, k]| / top[m] + 1/2),  top[m] = max_k |x[m, k]|,  scale[m] = top[m] / 127
//   out[m, k]   = codes[m, k] * scale[m], rounded to the type
//
// Both are bound by memory: 3 bytes a value for 16-bit types, 5 for fp32, in either direction.  A row is held in registers
// between the search for its top and its codes (one read): by a wave up to 256 vectors of 16 bytes, by a block of four
// waves up to 2048; longer rows are read twice, the second time from a cache.  Rows of codes start at multiples of
// 16 bytes and are filled up with zeros, so that the matrix kernels load them 16 bytes at a time.  bf16 [8192, 4096] there and
// back takes 34.2 us, 201 MB at 5.9 TB/s (in part from the last cache: what was just written is read).
#include "token_math.h"

namespace actnn {
namespace {

constexpr int kThreads = 256;

// A launch counts its work items in 32 bits, so blocks are counted in two dimensions: kAcross to a row.
constexpr int64_t kAcross = 1 << 20;
dim3 grid_of(int64_t blocks) {
  return blocks <= kAcross ? dim3((unsigned)blocks) : dim3((unsigned)kAcross, (unsigned)((blocks + kAcross - 1) / kAcross));
}
ACTNN_DEV int64_t block_number() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }

// first element of a row's vector and how many of its elements the row has
template <typename T> struct TokenRows {
  const T* x;
  int64_t ld, K;
  const T* last;                         // the tensor's last 16 bytes
  ACTNN_DEV u32x4 at(int64_t m, int64_t vec) const {
    constexpr int E = kVector<T>;
    const int64_t k = vec * E;
    return row_vector_ends<T>(load16_row<T>(x + m * ld + k, part_of_row(K, k), last));
  }
};
// rows whose vectors are whole and lie at multiples of 16 bytes
template <typename T> struct WholeRows {
  const T* x;
  int64_t ld, K;
  const T* last;
  ACTNN_DEV u32x4 at(int64_t m, int64_t vec) const { return load16(x + m * ld + vec * kVector<T>); }
};

template <typename T> ACTNN_DEV void store_codes(int8_t* row, int64_t vec, typename CodeWords<T>::type w) {
  reinterpret_cast<typename CodeWords<T>::type*>(row)[vec] = w;
}

// WAVES: waves that share a row (1 or 4); HELD: vectors of it that a lane keeps (0: none, the row is read twice).
// `vectors`: of a row of codes, zeros included (a multiple of 16 codes); those past `K` hold no element.
template <typename T, typename ROWS, int WAVES, int HELD>
__global__ __launch_bounds__(kThreads) void tokens_quantize_kernel(ROWS rows, int8_t* __restrict__ codes, int64_t ldc,
                                                                    float* __restrict__ scale, int64_t M, int64_t vectors,
                                                                    int64_t read) {
  constexpr int E = kVector<T>, kStep = 64 * WAVES;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t m = WAVES == 1 ? block_number() * (kThreads / 64) + wave : block_number();
  if (m >= M) return;                                   // (whole waves; with four to a row whole blocks)
  const int at = WAVES == 1 ? lane : threadIdx.x;
  u32x4 held[HELD > 0 ? HELD : 1];
  Top<T> top;
  const u32x4 none = {0u, 0u, 0u, 0u};
  if constexpr (HELD > 0) {
#pragma unroll
    for (int i = 0; i < HELD; ++i) held[i] = at + i * kStep < read ? rows.at(m, at + i * kStep) : none;
#pragma unroll
    for (int i = 0; i < HELD; ++i) top.add(held[i]);
  } else {
    for (int64_t v = at; v < read; v += kStep) top.add(rows.at(m, v));
  }
  uint32_t largest = lanes_largest(top.one());
  if constexpr (WAVES > 1) {
    __shared__ uint32_t s_top[WAVES];
    if (lane == 0) s_top[wave] = largest;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WAVES; ++i) largest = largest > s_top[i] ? largest : s_top[i];
  }
  const float value = Top<T>::value(largest);
  const TokenScale ts = token_scale(value);
  const Coder<T> coder(value);
  int8_t* row = codes + m * ldc;
  auto put = [&](int64_t v, const u32x4& raw) {
    float f[E];
    widen(static_cast<const T*>(nullptr), raw, f);
    store_codes<T>(row, v, codes_of<T>(coder, f, ts.keep));
  };
  if constexpr (HELD > 0) {
#pragma unroll
    for (int i = 0; i < HELD; ++i)
      if (at + i * kStep < vectors) put(at + i * kStep, held[i]);
  } else {
    for (int64_t v = at; v < vectors; v += kStep) put(v, v < read ? rows.at(m, v) : none);
  }
  if (at == 0) scale[m] = ts.scale;
}

// Tensors below 16 bytes: one thread a row, one element at a time.
template <typename T>
__global__ void tokens_quantize_tiny_kernel(const T* __restrict__ x, int64_t ld, int8_t* __restrict__ codes, int64_t ldc,
                                            float* __restrict__ scale, int M, int K) {
  const int64_t m = (int64_t)blockIdx.x * 64 + threadIdx.x;     // (rows of a stride of 0 may be many)
  if (m >= M) return;
  codes += m * ldc;
  x += m * ld;
  float top = 0.0f;
  bool bad = false;
  for (int k = 0; k < K; ++k) {
    const float v = __builtin_fabsf(Conv<T>::load(x, k));
    bad = bad || !(v <= 3.402823466e38f);
    top = v > top ? v : top;
  }
  if (bad) top = __builtin_nanf("");
  const TokenScale ts = token_scale(top);
  const Coder<T> coder(top);
  for (int k = 0; k < ldc && k < 16; ++k)
    codes[k] = k < K && ts.keep ? (int8_t)coder.code(Conv<T>::load(x, k)) : (int8_t)0;
  scale[m] = ts.scale;
}

template <typename T, typename ROWS>
void launch_quantize(const ROWS& rows, int8_t* codes, int64_t ldc, float* scale, int64_t M, hipStream_t s) {
  constexpr int E = kVector<T>;
  const int64_t read = (rows.K + E - 1) / E, vectors = (rows.K + 15) / 16 * 16 / E;
  const dim3 blk(kThreads), by_wave = grid_of((M + 3) / 4), by_block = grid_of(M);
#define ACTNN_GO(waves, held, grid) \
  tokens_quantize_kernel<T, ROWS, waves, held><<<grid, blk, 0, s>>>(rows, codes, ldc, scale, M, vectors, read)
  // a wave a row while its lanes keep four vectors at most and the rows fill the chip, else a block a row
  if (vectors <= 64) ACTNN_GO(1, 1, by_wave);
  else if (vectors <= 128) ACTNN_GO(1, 2, by_wave);
  else if (vectors <= 256 && M >= 1024) ACTNN_GO(1, 4, by_wave);
  else if (vectors <= 256) ACTNN_GO(4, 1, by_block);
  else if (vectors <= 512) ACTNN_GO(4, 2, by_block);
  else if (vectors <= 1024) ACTNN_GO(4, 4, by_block);
  else if (vectors <= 2048) ACTNN_GO(4, 8, by_block);
  else ACTNN_GO(4, 0, by_block);
#undef ACTNN_GO
}

template <typename T>
int quantize(const void* x, int64_t ldx, int8_t* codes, int64_t ldc, float* scale, int64_t M, int64_t K, hipStream_t s) {
  constexpr int E = kVector<T>;
  const T* p = static_cast<const T*>(x);
  if ((M - 1) * ldx + K < E) {
    tokens_quantize_tiny_kernel<T><<<dim3((unsigned)((M + 63) / 64)), dim3(64), 0, s>>>(p, ldx, codes, ldc, scale, (int)M, (int)K);
  } else {
    const T* last = p + (M - 1) * ldx + K - E;
    if (aligned16(x) && K % E == 0 && ldx % E == 0)
      launch_quantize<T>(WholeRows<T>{p, ldx, K, last}, codes, ldc, scale, M, s);
    else
      launch_quantize<T>(TokenRows<T>{p, ldx, K, last}, codes, ldc, scale, M, s);
  }
  ACTNN_RETURN_LAUNCH_STATUS();
}

// ------------------------------------------------------------------------------------------
// Reading back: a wave takes vectors of one row.
// ------------------------------------------------------------------------------------------
template <typename T, bool WHOLE, int WAVES>
__global__ __launch_bounds__(kThreads) void tokens_dequantize_kernel(const int8_t* __restrict__ codes, int64_t ldc,
                                                                     const float* __restrict__ scale, T* __restrict__ out,
                                                                     int64_t M, int64_t K) {
  constexpr int E = kVector<T>, kStep = 64 * WAVES, kAhead = 4;
  typedef typename CodeWords<T>::type Words;
  const int64_t m = WAVES == 1 ? block_number() * (kThreads / 64) + (threadIdx.x >> 6) : block_number();
  if (m >= M) return;
  const int at = WAVES == 1 ? threadIdx.x & 63 : threadIdx.x;
  const Words* row = reinterpret_cast<const Words*>(codes + m * ldc);
  T* to = out + m * K;
  const float sc = scale[m];
  const int64_t vectors = (K + E - 1) / E;
  for (int64_t v0 = at; v0 < vectors; v0 += kAhead * kStep) {
    Words w[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int64_t v = v0 + i * kStep;
      w[i] = row[v < vectors ? v : v0];
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int64_t v = v0 + i * kStep;
      if (v >= vectors) break;
      float f[E];
      code_values(w[i], f);
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] *= sc;
      const u32x4 o = narrow(static_cast<const T*>(nullptr), f);
      if constexpr (WHOLE) store16(to + v * E, o);
      else store16_part<false>(to + v * E, o, part_of_row(K, v * E));
    }
  }
}

template <typename T>
int dequantize(const int8_t* codes, int64_t ldc, const float* scale, void* out, int64_t M, int64_t K, hipStream_t s) {
  constexpr int E = kVector<T>;
  T* to = static_cast<T*>(out);
  const bool whole = K % E == 0 && aligned16(out);
  const bool wave = (K + E - 1) / E <= 256 && M >= 1024;
  const dim3 blk(kThreads), grid = grid_of(wave ? (M + 3) / 4 : M);
  if (wave && whole) tokens_dequantize_kernel<T, true, 1><<<grid, blk, 0, s>>>(codes, ldc, scale, to, M, K);
  else if (wave) tokens_dequantize_kernel<T, false, 1><<<grid, blk, 0, s>>>(codes, ldc, scale, to, M, K);
  else if (whole) tokens_dequantize_kernel<T, true, 4><<<grid, blk, 0, s>>>(codes, ldc, scale, to, M, K);
  else tokens_dequantize_kernel<T, false, 4><<<grid, blk, 0, s>>>(codes, ldc, scale, to, M, K);
  ACTNN_RETURN_LAUNCH_STATUS();
}

constexpr int64_t kMostRows = 0x7fffffffLL, kMostFeatures = 0x7fffffffLL - 64;

bool code_rows(int64_t ldc, int64_t K) { return ldc % 16 == 0 && ldc >= K; }

}  // namespace
}  // namespace actnn

extern "C" int actnn_tokens_quantize(const void* data, int64_t ld, int8_t* codes, int64_t ldc, float* scale, int64_t M,
                                     int64_t K, int dtype, void* stream) {
  using namespace actnn;
  if (M < 0 || K < 1 || M > kMostRows || K > kMostFeatures || ld < 0 || !code_rows(ldc, K)) return ACTNN_EINVAL;
  if (dtype != ACTNN_F32 && dtype != ACTNN_F16 && dtype != ACTNN_BF16) return ACTNN_EDTYPE;
  if (M == 0) return ACTNN_OK;
  if (!data || !codes || !scale) return ACTNN_EINVAL;
  const uintptr_t size = dtype == ACTNN_F32 ? 4 : 2;
  if (!aligned16(codes) || reinterpret_cast<uintptr_t>(data) % size != 0 || reinterpret_cast<uintptr_t>(scale) % 4 != 0)
    return ACTNN_EALIGN;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == ACTNN_F32) return quantize<float>(data, ld, codes, ldc, scale, M, K, s);
  if (dtype == ACTNN_F16) return quantize<__half>(data, ld, codes, ldc, scale, M, K, s);
  return quantize<bf16_t>(data, ld, codes, ldc, scale, M, K, s);
}

extern "C" int actnn_tokens_dequantize(const int8_t* codes, int64_t ldc, const float* scale, void* out, int64_t M, int64_t K,
                                       int dtype, void* stream) {
  using namespace actnn;
  if (M < 0 || K < 1 || M > kMostRows || K > kMostFeatures || !code_rows(ldc, K)) return ACTNN_EINVAL;
  if (dtype != ACTNN_F32 && dtype != ACTNN_F16 && dtype != ACTNN_BF16) return ACTNN_EDTYPE;
  if (M == 0) return ACTNN_OK;
  if (!codes || !scale || !out) return ACTNN_EINVAL;
  const uintptr_t size = dtype == ACTNN_F32 ? 4 : 2;
  if (!aligned16(codes) || reinterpret_cast<uintptr_t>(out) % size != 0 || reinterpret_cast<uintptr_t>(scale) % 4 != 0)
    return ACTNN_EALIGN;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == ACTNN_F32) return dequantize<float>(codes, ldc, scale, out, M, K, s);
  if (dtype == ACTNN_F16) return dequantize<__half>(codes, ldc, scale, out, M, K, s);
  return dequantize<bf16_t>(codes, ldc, scale, out, M, K, s);
}
