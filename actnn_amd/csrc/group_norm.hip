// Group norm with its activation over channels-last tensors, and its backward pass from an input kept in 8 bits.
//
//   forward    per sample and group: mean, rstd = 1 / sqrt(variance + eps) over the pixels and the group's channels;
//              z = (x - mean) rstd w + b,  y = z  or  z sigmoid(z);  kept: codes of x with one scale per sample and group
//   backward   n = (x' - mean) rstd from the codes' values x' = code * scale (or from x itself), z as above, dz = dy act'(z);
//              db = sum dz,  dw = sum dz n,  u = dz w,  dx = rstd (u - mean(u) - n mean(u n))
//
// All four passes are bound by memory.  A pixel's channels are consecutive, a group's are not: blocks take whole groups side
// by side (128 bytes of a pixel at least), a thread keeps the same 16 bytes of channels from pixel to pixel, so that
// everything that goes by channel stays in its registers, and sums are made per channel first and per group at the end.
// Each direction is two passes over the data with a table of partial results between them: a block of the second pass adds up
// the entries of its own groups before it starts.  The second pass takes the samples in the opposite order: the first one's last
// samples are still in the caches.
//
// Sums and statistics are fp32.  The variance is summed about the mean, not as a difference of moments: a thread sums up to
// 32 pixels about the first of them (which costs at most a factor of 32 of the last bit, however far the
// mean lies from zero) and such partial means and sums of squares are joined by their own differences.
#include "token_math.h"

namespace actnn {
namespace {

constexpr int kThreads = 256;
constexpr int kRun = 32;                 // pixels summed about the same value

// How a tensor [N, pixels, C] in G groups is cut into blocks: `chunk` channels (`per` whole groups, or a part of one wider than
// a block takes), `slice` pixels.
struct Cut {
  int64_t pixels;
  int N, C, G, width;                    // width: channels of a group
  int per;                               // groups of a chunk; 0: `parts` chunks to a group
  int parts, chunk, chunks;              // chunks: over all channels
  int slices, slice;
  __host__ __device__ int slots() const { return slices * parts; }
};

template <typename T> bool whole_vectors(const Cut& c) {
  constexpr int E = kVector<T>;
  return c.C % E == 0 && c.chunk % E == 0 && (c.per || c.width % E == 0);
}

int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

Cut cut_of(int64_t N, int64_t C, int64_t pixels, int64_t G, int E) {
  Cut c;
  c.N = (int)N; c.C = (int)C; c.G = (int)G; c.width = (int)(C / G); c.pixels = pixels;
  const int most = kThreads * E;
  if (c.width > most) {
    c.per = 0;
    c.parts = (c.width + most - 1) / most;
    c.chunk = ((c.width + c.parts - 1) / c.parts + E - 1) / E * E;
    c.parts = (c.width + c.chunk - 1) / c.chunk;
    c.chunks = c.G * c.parts;
  } else {
    // groups that end with a vector, 8 vectors at least
    int unit = E / gcd(c.width, E);
    if ((int64_t)unit * c.width > most || C % E) unit = 1;
    int per = unit;
    while (per < c.G && (int64_t)per * c.width < 8 * E && (int64_t)(per + unit) * c.width <= most) per += unit;
    if (per > c.G) per = c.G;
    c.per = per;
    c.parts = 1;
    c.chunk = per * c.width;
    c.chunks = (c.G + per - 1) / per;
  }
  // slices: some thousand blocks, four rounds of pixels each at least
  const int rows = kThreads / ((c.chunk + E - 1) / E);
  int64_t slices = 2048 / ((int64_t)c.N * c.chunks);
  const int64_t most_slices = (pixels + 4 * rows - 1) / (4 * rows);
  if (slices > most_slices) slices = most_slices;
  if (slices > 64) slices = 64;
  if (slices < 1) slices = 1;
  c.slice = (int)((pixels + slices - 1) / slices);
  c.slices = (int)((pixels + c.slice - 1) / c.slice);
  return c;
}

// The block's place: blocks run over the chunks first, then the slices, then the samples.
struct Place {
  int n, chunk, slice, part;
  int c0, channels, g0, groups;          // first channel, number of them; first group, number of them
  int64_t p0;                            // first pixel, and how many
  int count;
  int cols, rows, col, row;              // vectors of a pixel, pixels of a round; this thread's (row >= rows: none)
  ACTNN_DEV Place(const Cut& c, uint32_t block, int E, bool backwards) {
    chunk = block % c.chunks;
    const uint32_t rest = block / c.chunks;
    slice = rest % c.slices;
    n = rest / c.slices;
    if (backwards) { n = c.N - 1 - n; slice = c.slices - 1 - slice; }
    if (c.per) {
      part = 0;
      g0 = chunk * c.per;
      groups = c.G - g0 < c.per ? c.G - g0 : c.per;
      c0 = g0 * c.width;
      channels = groups * c.width;
    } else {
      part = chunk % c.parts;
      g0 = chunk / c.parts;
      groups = 1;
      c0 = g0 * c.width + part * c.chunk;
      channels = c.width - part * c.chunk < c.chunk ? c.width - part * c.chunk : c.chunk;
    }
    p0 = (int64_t)slice * c.slice;
    count = c.pixels - p0 < c.slice ? (int)(c.pixels - p0) : c.slice;
    cols = (channels + E - 1) / E;
    rows = kThreads / cols;
    col = threadIdx.x % cols;
    row = threadIdx.x / cols;
  }
  ACTNN_DEV int mine() const { return row < rows && row < count ? (count - row + rows - 1) / rows : 0; }     // this thread's pixels
  ACTNN_DEV int of_row(int r) const { return r < count ? (count - r + rows - 1) / rows : 0; }
  ACTNN_DEV int valid(int E) const { return channels - col * E < E ? channels - col * E : E; }
};

// vectors of 16 bytes of a tensor, whole and aligned or not
template <typename T, bool WHOLE> struct Source {
  const T* at;                           // this thread's vector of the slice's first pixel
  const T* last;
  int valid;
  ACTNN_DEV Source(const T* base, const Cut& c, const Place& b) {
    constexpr int E = kVector<T>;
    at = base + ((int64_t)b.n * c.pixels + b.p0) * c.C + b.c0 + b.col * E;
    const int64_t all = (int64_t)c.N * c.pixels * c.C;
    last = base + (all > E ? all - E : 0);               // (a smaller tensor has room for 16 bytes)
    valid = b.valid(E);
  }
  ACTNN_DEV u32x4 get(int64_t offset) const {
    if constexpr (WHOLE) return load16(at + offset);
    else return row_vector_ends<T>(load16_row<T>(at + offset, valid, last));
  }
};
template <typename T, bool WHOLE> ACTNN_DEV void put_vector(T* to, const u32x4& v, int valid) {
  if constexpr (WHOLE) store16(to, v);
  else store16_part<false>(to, v, valid);
}
template <typename T, bool WHOLE> ACTNN_DEV void put_codes(int8_t* to, typename CodeWords<T>::type w, int valid) {
  typedef typename CodeWords<T>::type Words;
  if constexpr (WHOLE) {
    *reinterpret_cast<Words*>(to) = w;
  } else {
    uint32_t words[2];
    if constexpr (sizeof(T) == 4) { words[0] = w; words[1] = 0; } else { words[0] = w.x; words[1] = w.y; }
#pragma unroll
    for (int i = 0; i < kVector<T>; ++i)
      if (i < valid) to[i] = (int8_t)(words[i / 4] >> (8 * (i % 4)));
  }
}
template <typename T, bool WHOLE> ACTNN_DEV typename CodeWords<T>::type get_codes(const int8_t* from, int valid) {
  typedef typename CodeWords<T>::type Words;
  if constexpr (WHOLE) {
    return *reinterpret_cast<const Words*>(from);
  } else {
    uint32_t words[2] = {0u, 0u};
#pragma unroll
    for (int i = 0; i < kVector<T>; ++i)
      if (i < valid) words[i / 4] |= (uint32_t)(uint8_t)from[i] << (8 * (i % 4));
    if constexpr (sizeof(T) == 4) return words[0];
    else return (Words){words[0], words[1]};
  }
}

// ------------------------------------------------------------------------------------------
// Sums over a group by a team of lanes: 1 to 64 lanes of a wave, a power of two of them.
// ------------------------------------------------------------------------------------------
struct Team {
  int size, lane, first, step;           // lanes of a team, this one; the team's first group, and the distance to its next
  ACTNN_DEV explicit Team(int groups) {
    size = 64;
    while (size > 1 && size * groups > kThreads) size >>= 1;
    lane = threadIdx.x & (size - 1);
    first = threadIdx.x / size;
    step = kThreads / size;
  }
  ACTNN_DEV float sum(float v) const {
    for (int d = size >> 1; d > 0; d >>= 1) v += __shfl_xor(v, d);
    return v;
  }
  ACTNN_DEV uint32_t largest(uint32_t v) const {
    for (int d = size >> 1; d > 0; d >>= 1) {
      const uint32_t o = (uint32_t)__shfl_xor((int)v, d);
      v = v > o ? v : o;
    }
    return v;
  }
};

struct Partial { float mean, squares, count, top; };     // top: bits of the largest magnitude, as a float's

// ------------------------------------------------------------------------------------------
// Forward, first pass: partial statistics [N][G][slots].
// ------------------------------------------------------------------------------------------
template <typename T, bool WHOLE>
__global__ __launch_bounds__(kThreads) void group_norm_stats_kernel(const T* __restrict__ x, Partial* __restrict__ table, Cut c) {
  constexpr int E = kVector<T>;
  __shared__ float s_mean[kThreads * E], s_squares[kThreads * E];
  __shared__ uint32_t s_top[kThreads * E];
  const Place b(c, blockIdx.x, E, false);
  const int mine = b.mine();
  const T* none = nullptr;
  float mean[E], squares[E];
  uint32_t top[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int e = 0; e < E; ++e) mean[e] = squares[e] = 0.0f;
  if (mine > 0) {
    const Source<T, WHOLE> src(x, c, b);
    const int64_t step = (int64_t)b.rows * c.C;
    int64_t at = (int64_t)b.row * c.C;
    float done = 0.0f;
    for (int i = 0; i < mine; i += kRun) {
      const int run = mine - i < kRun ? mine - i : kRun;
      float first[E], s1[E], s2[E];
      auto add = [&](const u32x4& raw) {
        float f[E];
        widen(none, raw, f);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float d = f[e] - first[e];
          s1[e] += d;
          s2[e] = __builtin_fmaf(d, d, s2[e]);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) top[k] = Top<T>::larger(top[k], raw[k] & (sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu));
      };
      {
        const u32x4 raw = src.get(at);
        widen(none, raw, first);
#pragma unroll
        for (int e = 0; e < E; ++e) s1[e] = s2[e] = 0.0f;
        add(raw);
        at += step;
      }
      int k = 1;
      for (; k + 4 <= run; k += 4) {
        u32x4 raw[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) raw[j] = src.get(at + j * step);
#pragma unroll
        for (int j = 0; j < 4; ++j) add(raw[j]);
        at += 4 * step;
      }
      for (; k < run; ++k) {
        add(src.get(at));
        at += step;
      }
      const float n = (float)run, total = done + n;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float m = s1[e] / n, q = s2[e] - s1[e] * m, d = first[e] + m - mean[e];
        squares[e] += q + d * d * (done * n / total);
        mean[e] += d * (n / total);
      }
      done = total;
    }
  }
  // per channel and row of threads into LDS, then per group
  if (b.row < b.rows) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int at = (b.row * b.cols + b.col) * E + e;
      s_mean[at] = mean[e];
      s_squares[at] = squares[e];
      s_top[at] = sizeof(T) == 4 ? top[e & 3] : (e & 1) ? top[(e >> 1) & 3] >> 16 : top[(e >> 1) & 3] & 0xffffu;
    }
  }
  __syncthreads();
  const Team team(b.groups);
  const int width = c.per ? c.width : b.channels;        // of a group, in this block
  const float count = (float)b.count * (float)width;
  for (int g = team.first; g < b.groups; g += team.step) {
    const float about = s_mean[g * width];               // (means are summed about one of them, like values)
    float sum = 0.0f;
    uint32_t largest = 0;
    for (int i = team.lane; i < b.rows * width; i += team.size) {
      const int r = i / width, at = r * b.cols * E + g * width + i % width;
      sum += (float)b.of_row(r) * (s_mean[at] - about);
      largest = largest > s_top[at] ? largest : s_top[at];
    }
    // (rows of threads without a pixel have count 0, and mean 0)
    const float m = about + team.sum(sum) / count;
    largest = team.largest(largest);
    float q = 0.0f;
    for (int i = team.lane; i < b.rows * width; i += team.size) {
      const int r = i / width, at = r * b.cols * E + g * width + i % width;
      const float d = s_mean[at] - m;
      q += s_squares[at] + (float)b.of_row(r) * d * d;
    }
    q = team.sum(q);
    if (team.lane == 0)
      table[((int64_t)b.n * c.G + b.g0 + g) * c.slots() + b.slice * c.parts + b.part] = Partial{m, q, count, Top<T>::value(largest)};
  }
}

struct Moments { float mean, rstd, top; };
// a group's statistics from its partial ones, by a team; every lane has them
ACTNN_DEV Moments join(const Team& team, const Partial* p, int slots, float eps) {
  const float about = p[0].mean;
  float n = 0.0f, sum = 0.0f;
  uint32_t top = 0;
  for (int i = team.lane; i < slots; i += team.size) {
    const Partial v = p[i];
    n += v.count;
    sum += v.count * (v.mean - about);
    const uint32_t t = as_uint(v.top);
    top = top > t ? top : t;
  }
  n = team.sum(n);
  const float mean = about + team.sum(sum) / n;
  top = team.largest(top);
  float q = 0.0f;
  for (int i = team.lane; i < slots; i += team.size) {
    const Partial v = p[i];
    const float d = v.mean - mean;
    q += v.squares + v.count * d * d;
  }
  q = team.sum(q);
  return Moments{mean, 1.0f / __builtin_sqrtf(q / n + eps), as_float(top)};
}

ACTNN_DEV float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + __expf(-z)); }

// ------------------------------------------------------------------------------------------
// Forward, second pass.
// ------------------------------------------------------------------------------------------
struct Forward {
  const Partial* table;
  const float *weight, *bias;            // [C] or null
  float *mean, *rstd, *scale;            // [N, G]
  int8_t* codes;
  float eps;
};
template <typename T, bool WHOLE, bool SILU, bool KEEP>
__global__ __launch_bounds__(kThreads) void group_norm_apply_kernel(const T* __restrict__ x, T* __restrict__ y, Forward f, Cut c) {
  constexpr int E = kVector<T>;
  __shared__ Moments s_group[kThreads * E];
  const Place b(c, blockIdx.x, E, true);
  const Team team(b.groups);
  for (int g = team.first; g < b.groups; g += team.step) {
    const int64_t at = (int64_t)b.n * c.G + b.g0 + g;
    const Moments m = join(team, f.table + at * c.slots(), c.slots(), f.eps);
    if (team.lane == 0) {
      s_group[g] = m;
      if (b.slice == 0 && b.part == 0) {
        f.mean[at] = m.mean;
        f.rstd[at] = m.rstd;
        if constexpr (KEEP) f.scale[at] = token_scale(m.top).scale;
      }
    }
  }
  __syncthreads();
  const int mine = b.mine();
  if (mine == 0) return;
  float mean[E], a[E], add[E];
  Coder<T> coder[E] = {};
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int ch = b.col * E + e < b.channels ? b.col * E + e : b.channels - 1;
    const Moments m = s_group[c.per ? ch / c.width : 0];
    mean[e] = m.mean;
    a[e] = f.weight ? m.rstd * f.weight[b.c0 + ch] : m.rstd;
    add[e] = f.bias ? f.bias[b.c0 + ch] : 0.0f;
    if constexpr (KEEP) {
      if (token_scale(m.top).keep) coder[e] = Coder<T>(m.top);      // (else a factor of 0: codes 0)
    }
  }
  const Source<T, WHOLE> src(x, c, b);
  const int64_t step = (int64_t)b.rows * c.C, base = src.at - x;
  int64_t at = (int64_t)b.row * c.C;
  const T* none = nullptr;
  auto put = [&](int64_t offset, const u32x4& raw) {
    float v[E];
    widen(none, raw, v);
    if constexpr (KEEP) {
      int q[E];
#pragma unroll
      for (int e = 0; e < E; ++e) q[e] = coder[e].code(v[e]);
      typename CodeWords<T>::type w;
      if constexpr (E == 4) w = pack_codes(q[0], q[1], q[2], q[3]);
      else w = (u32x2){pack_codes(q[0], q[1], q[2], q[3]), pack_codes(q[4 % E], q[5 % E], q[6 % E], q[7 % E])};
      put_codes<T, WHOLE>(f.codes + base + offset, w, src.valid);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float z = __builtin_fmaf(v[e] - mean[e], a[e], add[e]);
      v[e] = SILU ? z * sigmoid(z) : z;
    }
    put_vector<T, WHOLE>(y + base + offset, narrow(none, v), src.valid);
  };
  int i = 0;
  for (; i + 4 <= mine; i += 4) {
    u32x4 raw[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) raw[j] = src.get(at + j * step);
#pragma unroll
    for (int j = 0; j < 4; ++j) put(at + j * step, raw[j]);
    at += 4 * step;
  }
  for (; i < mine; ++i) {
    put(at, src.get(at));
    at += step;
  }
}

// ------------------------------------------------------------------------------------------
// Backward.
// ------------------------------------------------------------------------------------------
struct Backward {
  const int8_t* codes;                   // the kept input: codes and scale [N, G], or null and x
  const float* scale;
  const float *weight, *bias, *mean, *rstd;
  float* sums;                           // [N][slices][2][C]: sum dz, sum dz n
  float *dweight, *dbias;
};

// What goes by channel for a thread's vector, and n, dz of a vector's elements.
template <typename T, bool WHOLE, bool SILU, bool CODES> struct Slope {
  static constexpr int E = kVector<T>;
  float by[E], less[E], w[E], add[E];    // n = value * by - less
  ACTNN_DEV void init(const Backward& k, const Cut& c, const Place& b) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int ch = b.col * E + e < b.channels ? b.col * E + e : b.channels - 1;
      const int64_t g = (int64_t)b.n * c.G + b.g0 + (c.per ? ch / c.width : 0);
      const float rstd = k.rstd[g];
      if constexpr (CODES) {
        by[e] = k.scale[g] * rstd;
        less[e] = k.mean[g] * rstd;
      } else {
        by[e] = rstd;
        less[e] = k.mean[g];
      }
      w[e] = k.weight ? k.weight[b.c0 + ch] : 1.0f;
      add[e] = k.bias ? k.bias[b.c0 + ch] : 0.0f;
    }
  }
  typedef typename CodeWords<T>::type Words;
  struct Raw { u32x4 dy, x; Words codes; };
  ACTNN_DEV void fetch(Raw& r, const Source<T, WHOLE>& dy, const Source<T, WHOLE>& x, const int8_t* codes, int64_t at) const {
    r.dy = dy.get(at);
    if constexpr (CODES) r.codes = get_codes<T, WHOLE>(codes + at, dy.valid);
    else r.x = x.get(at);
  }
  ACTNN_DEV void values(const Raw& r, float (&n)[E], float (&dz)[E]) const {
    const T* none = nullptr;
    widen(none, r.dy, dz);
    if constexpr (CODES) {
      code_values(r.codes, n);
#pragma unroll
      for (int e = 0; e < E; ++e) n[e] = __builtin_fmaf(n[e], by[e], -less[e]);
    } else {
      widen(none, r.x, n);
#pragma unroll
      for (int e = 0; e < E; ++e) n[e] = (n[e] - less[e]) * by[e];
    }
    if constexpr (SILU) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float z = __builtin_fmaf(n[e], w[e], add[e]), s = sigmoid(z);
        dz[e] *= __builtin_fmaf(z * s, 1.0f - s, s);
      }
    }
  }
};

template <typename T, bool WHOLE, bool SILU, bool CODES>
__global__ __launch_bounds__(kThreads) void group_norm_backward_sums_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                                            Backward k, Cut c) {
  constexpr int E = kVector<T>;
  __shared__ float s_sum[2][kThreads * E];
  const Place b(c, blockIdx.x, E, false);
  const int mine = b.mine();
  float sum[E], by_n[E];
#pragma unroll
  for (int e = 0; e < E; ++e) sum[e] = by_n[e] = 0.0f;
  if (mine > 0) {
    Slope<T, WHOLE, SILU, CODES> slope;
    slope.init(k, c, b);
    const Source<T, WHOLE> sdy(dy, c, b), sx(CODES ? dy : x, c, b);
    const int8_t* codes = k.codes + (sdy.at - dy);
    const int64_t step = (int64_t)b.rows * c.C;
    int64_t at = (int64_t)b.row * c.C;
    typename Slope<T, WHOLE, SILU, CODES>::Raw raw[4];
    auto add = [&](int j) {
      float n[E], dz[E];
      slope.values(raw[j], n, dz);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        sum[e] += dz[e];
        by_n[e] = __builtin_fmaf(dz[e], n[e], by_n[e]);
      }
    };
    int i = 0;
    for (; i + 4 <= mine; i += 4) {
#pragma unroll
      for (int j = 0; j < 4; ++j) slope.fetch(raw[j], sdy, sx, codes, at + j * step);
#pragma unroll
      for (int j = 0; j < 4; ++j) add(j);
      at += 4 * step;
    }
    for (; i < mine; ++i) {
      slope.fetch(raw[0], sdy, sx, codes, at);
      add(0);
      at += step;
    }
  }
  if (b.row < b.rows) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      s_sum[0][(b.row * b.cols + b.col) * E + e] = sum[e];
      s_sum[1][(b.row * b.cols + b.col) * E + e] = by_n[e];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * b.channels; i += kThreads) {
    const int which = i >= b.channels, ch = which ? i - b.channels : i;
    float v = 0.0f;
    for (int r = 0; r < b.rows; ++r) v += s_sum[which][r * b.cols * E + ch];
    k.sums[(((int64_t)b.n * c.slices + b.slice) * 2 + which) * c.C + b.c0 + ch] = v;
  }
}

template <typename T, bool WHOLE, bool SILU, bool CODES>
__global__ __launch_bounds__(kThreads) void group_norm_backward_apply_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                                             T* __restrict__ dx, Backward k, Cut c) {
  constexpr int E = kVector<T>;
  __shared__ float s_mean[2][kThreads * E];
  const Place b(c, blockIdx.x, E, true);
  const Team team(b.groups);
  const float all = 1.0f / ((float)c.pixels * (float)c.width);
  for (int g = team.first; g < b.groups; g += team.step) {
    float first = 0.0f, second = 0.0f;
    const float* sums = k.sums + (int64_t)b.n * c.slices * 2 * c.C + (int64_t)(b.g0 + g) * c.width;
    for (int ch = team.lane; ch < c.width; ch += team.size) {
      float s = 0.0f, t = 0.0f;
      for (int j = 0; j < c.slices; ++j) {
        s += sums[(int64_t)(2 * j) * c.C + ch];
        t += sums[(int64_t)(2 * j + 1) * c.C + ch];
      }
      const float w = k.weight ? k.weight[(b.g0 + g) * c.width + ch] : 1.0f;
      first = __builtin_fmaf(w, s, first);
      second = __builtin_fmaf(w, t, second);
    }
    first = team.sum(first);
    second = team.sum(second);
    if (team.lane == 0) {
      s_mean[0][g] = first * all;
      s_mean[1][g] = second * all;
    }
  }
  __syncthreads();
  const int mine = b.mine();
  if (mine == 0) return;
  Slope<T, WHOLE, SILU, CODES> slope;
  slope.init(k, c, b);
  float rstd[E], first[E], second[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int ch = b.col * E + e < b.channels ? b.col * E + e : b.channels - 1;
    const int g = c.per ? ch / c.width : 0;
    rstd[e] = k.rstd[(int64_t)b.n * c.G + b.g0 + g];
    first[e] = s_mean[0][g] * rstd[e];
    second[e] = s_mean[1][g] * rstd[e];
  }
  const Source<T, WHOLE> sdy(dy, c, b), sx(CODES ? dy : x, c, b);
  const int64_t base = sdy.at - dy;
  const int8_t* codes = k.codes + base;
  const int64_t step = (int64_t)b.rows * c.C;
  int64_t at = (int64_t)b.row * c.C;
  typename Slope<T, WHOLE, SILU, CODES>::Raw raw[4];
  const T* none = nullptr;
  auto put = [&](int j, int64_t offset) {
    float n[E], dz[E];
    slope.values(raw[j], n, dz);
#pragma unroll
    for (int e = 0; e < E; ++e)
      dz[e] = __builtin_fmaf(dz[e], slope.w[e] * rstd[e], -first[e]) - n[e] * second[e];
    put_vector<T, WHOLE>(dx + base + offset, narrow(none, dz), sdy.valid);
  };
  int i = 0;
  for (; i + 4 <= mine; i += 4) {
#pragma unroll
    for (int j = 0; j < 4; ++j) slope.fetch(raw[j], sdy, sx, codes, at + j * step);
#pragma unroll
    for (int j = 0; j < 4; ++j) put(j, at + j * step);
    at += 4 * step;
  }
  for (; i < mine; ++i) {
    slope.fetch(raw[0], sdy, sx, codes, at);
    put(0, at);
    at += step;
  }
}

// dw, db: the table's sums over samples and slices, 64 channels a block, 16 rows of the table at a time.
__global__ __launch_bounds__(1024) void group_norm_backward_parameters_kernel(Backward k, Cut c) {
  __shared__ float s_sum[16][64];
  const int lane = threadIdx.x & 63, row = threadIdx.x >> 6;
  const int which = blockIdx.y, ch = blockIdx.x * 64 + lane;
  const int64_t rows = (int64_t)c.N * c.slices;
  float v = 0.0f;
  if (ch < c.C)
    for (int64_t r = row; r < rows; r += 16) v += k.sums[(2 * r + which) * c.C + ch];
  s_sum[row][lane] = v;
  __syncthreads();
  if (row == 0 && ch < c.C) {
    for (int r = 1; r < 16; ++r) v += s_sum[r][lane];
    float* to = which ? k.dweight : k.dbias;
    if (to) to[ch] = v;
  }
}

enum { kNone = 0, kSilu = 1 };

template <typename T> int forward(const void* x, void* y, Forward f, const Cut& c, bool silu, bool keep, void* ws, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)c.N * c.chunks * c.slices)), blk(kThreads);
  const T* px = static_cast<const T*>(x);
  T* py = static_cast<T*>(y);
  f.table = static_cast<Partial*>(ws);
  auto go = [&](auto whole) {
    constexpr bool W = decltype(whole)::value;
    group_norm_stats_kernel<T, W><<<grid, blk, 0, s>>>(px, static_cast<Partial*>(ws), c);
    if (silu && keep) group_norm_apply_kernel<T, W, true, true><<<grid, blk, 0, s>>>(px, py, f, c);
    else if (silu) group_norm_apply_kernel<T, W, true, false><<<grid, blk, 0, s>>>(px, py, f, c);
    else if (keep) group_norm_apply_kernel<T, W, false, true><<<grid, blk, 0, s>>>(px, py, f, c);
    else group_norm_apply_kernel<T, W, false, false><<<grid, blk, 0, s>>>(px, py, f, c);
  };
  const bool aligned = aligned16(x) && aligned16(y) && reinterpret_cast<uintptr_t>(f.codes) % 8 == 0;
  if (aligned && whole_vectors<T>(c)) go(std::true_type{});
  else go(std::false_type{});
  ACTNN_RETURN_LAUNCH_STATUS();
}

template <typename T>
int backward(const void* dy, const void* x, void* dx, const Backward& k, const Cut& c, bool silu, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)c.N * c.chunks * c.slices)), blk(kThreads);
  const T *pdy = static_cast<const T*>(dy), *px = static_cast<const T*>(x);
  T* pdx = static_cast<T*>(dx);
  auto go = [&](auto whole, auto act, auto codes) {
    constexpr bool W = decltype(whole)::value, S = decltype(act)::value, Q = decltype(codes)::value;
    group_norm_backward_sums_kernel<T, W, S, Q><<<grid, blk, 0, s>>>(pdy, px, k, c);
    if (dx) group_norm_backward_apply_kernel<T, W, S, Q><<<grid, blk, 0, s>>>(pdy, px, pdx, k, c);
    if (k.dweight || k.dbias)
      group_norm_backward_parameters_kernel<<<dim3((unsigned)((c.C + 63) / 64), 2), dim3(1024), 0, s>>>(k, c);
  };
  auto by_source = [&](auto whole, auto act) {
    if (k.codes) go(whole, act, std::true_type{});
    else go(whole, act, std::false_type{});
  };
  auto by_act = [&](auto whole) {
    if (silu) by_source(whole, std::true_type{});
    else by_source(whole, std::false_type{});
  };
  const bool aligned = aligned16(dy) && (!x || aligned16(x)) && (!dx || aligned16(dx)) && reinterpret_cast<uintptr_t>(k.codes) % 8 == 0;
  if (aligned && whole_vectors<T>(c)) by_act(std::true_type{});
  else by_act(std::false_type{});
  ACTNN_RETURN_LAUNCH_STATUS();
}

int check(int64_t N, int64_t C, int64_t P, int64_t G, int dtype) {
  if (N < 0 || C < 1 || P < 0 || G < 1 || C % G || N > 0x7fffff || C > 0x7fffff || P > 0x7fffffffLL) return ACTNN_EINVAL;
  if (dtype != ACTNN_F32 && dtype != ACTNN_F16 && dtype != ACTNN_BF16) return ACTNN_EDTYPE;
  return ACTNN_OK;
}
int64_t forward_bytes(const Cut& c) { return (int64_t)c.N * c.G * c.slots() * (int64_t)sizeof(Partial); }
int64_t backward_bytes(const Cut& c) { return (int64_t)c.N * c.slices * 2 * c.C * 4; }

}  // namespace
}  // namespace actnn

extern "C" int64_t actnn_group_norm_workspace_bytes(int64_t N, int64_t C, int64_t pixels, int64_t groups, int dtype,
                                                    int backward) {
  using namespace actnn;
  if (const int rc = check(N, C, pixels, groups, dtype)) return rc;
  if (N == 0 || pixels == 0) return 0;
  const Cut c = cut_of(N, C, pixels, groups, dtype == ACTNN_F32 ? 4 : 8);
  return backward ? backward_bytes(c) : forward_bytes(c);
}

extern "C" int actnn_group_norm_forward(const void* x, const float* weight, const float* bias, void* y, float* mean,
                                        float* rstd, int8_t* codes, float* scale, int64_t N, int64_t C, int64_t pixels,
                                        int64_t groups, double eps, int activation, int dtype, void* workspace,
                                        int64_t workspace_bytes, void* stream) {
  using namespace actnn;
  if (const int rc = check(N, C, pixels, groups, dtype)) return rc;
  if (activation != kNone && activation != kSilu) return ACTNN_EINVAL;
  if (N == 0 || pixels == 0) return ACTNN_OK;
  if (!x || !y || !mean || !rstd || !workspace || (codes && !scale)) return ACTNN_EINVAL;
  const int64_t size = dtype == ACTNN_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(x) % size || reinterpret_cast<uintptr_t>(y) % size || !aligned16(workspace)) return ACTNN_EALIGN;
  const Cut c = cut_of(N, C, pixels, groups, dtype == ACTNN_F32 ? 4 : 8);
  if (workspace_bytes < forward_bytes(c) || (int64_t)c.N * c.chunks * c.slices > 0x7fffffffLL) return ACTNN_EINVAL;
  Forward f{nullptr, weight, bias, mean, rstd, scale, codes, (float)eps};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool silu = activation == kSilu;
  if (dtype == ACTNN_F32) return forward<float>(x, y, f, c, silu, codes != nullptr, workspace, s);
  if (dtype == ACTNN_F16) return forward<__half>(x, y, f, c, silu, codes != nullptr, workspace, s);
  return forward<bf16_t>(x, y, f, c, silu, codes != nullptr, workspace, s);
}

extern "C" int actnn_group_norm_backward(const void* dy, const int8_t* codes, const float* scale, const void* x,
                                         const float* weight, const float* bias, const float* mean, const float* rstd,
                                         void* dx, float* dweight, float* dbias, int64_t N, int64_t C, int64_t pixels,
                                         int64_t groups, int activation, int dtype, void* workspace, int64_t workspace_bytes,
                                         void* stream) {
  using namespace actnn;
  if (const int rc = check(N, C, pixels, groups, dtype)) return rc;
  if (activation != kNone && activation != kSilu) return ACTNN_EINVAL;
  if (N == 0 || pixels == 0) return ACTNN_EINVAL;       // (nothing to launch: the caller clears the parameters' gradients)
  if (!dy || !mean || !rstd || !workspace || (codes ? !scale : !x)) return ACTNN_EINVAL;
  const int64_t size = dtype == ACTNN_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(dy) % size || reinterpret_cast<uintptr_t>(x) % size || reinterpret_cast<uintptr_t>(dx) % size ||
      !aligned16(workspace))
    return ACTNN_EALIGN;
  const Cut c = cut_of(N, C, pixels, groups, dtype == ACTNN_F32 ? 4 : 8);
  if (workspace_bytes < backward_bytes(c) || (int64_t)c.N * c.chunks * c.slices > 0x7fffffffLL) return ACTNN_EINVAL;
  const Backward k{codes, scale, weight, bias, mean, rstd, static_cast<float*>(workspace), dweight, dbias};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool silu = activation == kSilu;
  if (dtype == ACTNN_F32) return backward<float>(dy, codes ? nullptr : x, dx, k, c, silu, s);
  if (dtype == ACTNN_F16) return backward<__half>(dy, codes ? nullptr : x, dx, k, c, silu, s);
  return backward<bf16_t>(dy, codes ? nullptr : x, dx, k, c, silu, s);
}
