// Group norm with its activation over channels-last tensors, and its backward pass from an input kept in 8 bits.
//
//   forward    per sample and group: mean, rstd = 1 / sqrt(variance + eps) over the pixels and the group's channels;
//              z = (x - mean) rstd w + b,  y = z  or  z sigmoid(z);  kept: codes of x with one scale per sample and group
//   backward   n = (x' - mean) rstd from the codes' values x' = code * scale (or from x itself), z as above, dz = dy act'(z);
//              db = sum dz,  dw = sum dz n,  u = dz w,  dx = rstd (u - mean(u) - n mean(u n))
//
// Large tensors are bound by memory.  A pixel's channels are consecutive, a group's are not: blocks take whole groups side
// by side (128 bytes of a pixel at least), a thread keeps the same 16 bytes of channels from pixel to pixel, so that
// everything that goes by channel stays in its registers, and sums are made per channel first and per group at the end.
// Each direction is two passes over the data with a table of partial results by group between them: a block of the second pass adds
// up the entries of its own groups before it starts.  The second pass takes the samples in the opposite order: the first one's last
// samples are still in the caches.  [128, 56 * 56, 256] bf16 takes 332 us in both directions: the first passes read 205 and 308 MB at
// 3.3 TB/s, the second ones move 514 MB each at 5.8 (a copy: 5.1).
//
// Small tensors are bound by the instructions: a kernel's code comes from the L2 at about a microsecond a kilobyte when it is
// run once.  So small planes take one kernel instead of two, a block to a plane's chunk that reads it twice; loops over
// pixels are unrolled as far as loads need it and no further, and positions come from divisions prepared on the host.
//
// Sums and statistics are fp32.  The variance is summed about the mean, not as a difference of moments: a thread sums up to
// 32 pixels about the first of them (which costs at most a factor of 32 of the last bit, however far the
// mean lies from zero) and such partial means and sums of squares are joined by their own differences.  The backward pass sums by
// runs too.
#include "token_math.h"

namespace actnn {
namespace {

constexpr int kThreads = 256;
constexpr int kWide = 1024;              // of the kernel that adds up the parameters' gradients
constexpr int kRun = 32;                 // pixels summed about the same value
constexpr int64_t kMostBlocks = 0xffffff;   // (a launch counts its work items in 32 bits)

// How a tensor [N, pixels, C] in G groups is cut into blocks: `chunk` channels (`per` whole groups, or a part of one wider than
// a block takes), `slice` pixels.
struct Cut {
  int64_t pixels;
  int N, C, G, width;                    // width: channels of a group
  int per;                               // groups of a chunk; 0: `parts` chunks to a group
  int parts, chunk, chunks;              // chunks: over all channels
  int slices, slice;
  int cols, rows;                        // vectors of a chunk's pixel, pixels of a round of the block's threads
  FastDiv by_chunks, by_slices, by_parts, by_cols, by_rows, by_width;
  __host__ __device__ int slots() const { return slices * parts; }
  int64_t blocks() const { return (int64_t)N * chunks * slices; }
};

// Every chunk has a vector's channels.  Then all vectors are whole: where a chunk's channels are no whole number of them, the last
// one begins earlier and shares channels with the one before (both compute and store the same).  Global memory takes
// 16-byte accesses at any address.
bool whole_vectors(const Cut& c, int E) {
  const int last = c.per ? (c.G - (c.chunks - 1) * c.per) * c.width : c.width - (c.parts - 1) * c.chunk;
  return c.chunk >= E && last >= E;
}

int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

// The groups whose channels end with a line of memory (128 bytes) of every pixel, or 0 where those are more than 128 vectors; where
// the pixels do not begin with lines, all groups.  Blocks that share lines write parts of them, mostly from different XCDs: chunks
// like these and before, both directions, us: [54, 35 * 35, 768] in 32 groups 166, 220; [28, 61 * 81, 366] in 6 169, 208;
// [56, 30 * 33, 504] in 24 90, 102.
constexpr int kWidest = 128;
int groups_of_lines(const Cut& c, int E) {
  const int line = 8 * E, groups = c.C % line ? c.G : line / gcd(c.width, line);
  return (int64_t)groups * c.width <= kWidest * E ? groups : 0;
}

// A chunk of whole groups, of `least` vectors where there are as many channels, in whole `unit`s of groups where it can; unit 0:
// ending with a vector.
void cut_channels(Cut& c, int E, int least, int unit = 0) {
  const int most = kThreads * E;
  if (c.width > most) {
    c.per = 0;
    c.parts = (c.width + most - 1) / most;
    c.chunk = (c.width + c.parts - 1) / c.parts;
    if ((int64_t)(c.parts - 1) * ((c.chunk + E - 1) / E * E) <= c.width - E) c.chunk = (c.chunk + E - 1) / E * E;
    c.chunks = c.G * c.parts;
  } else {
    if (!unit) unit = c.C % E ? 1 : E / gcd(c.width, E);
    if ((int64_t)unit * c.width > most) unit = 1;
    int per = unit;
    while (per < c.G && (int64_t)per * c.width < least * E && (int64_t)(per + unit) * c.width <= most) per += unit;
    if (per > c.G) per = c.G;
    const int chunks = (c.G + per - 1) / per;            // as many groups to each
    per = (c.G + chunks - 1) / chunks;
    const int up = per % unit ? unit - per % unit : 0;   // to whole units
    if (per + up <= c.G && (int64_t)(per + up) * c.width <= most) per += up;
    c.per = per;
    c.parts = 1;
    c.chunk = per * c.width;
    c.chunks = (c.G + per - 1) / per;
  }
  c.cols = (c.chunk + E - 1) / E;
}
void cut_pixels(Cut& c, int64_t slices) {
  c.rows = kThreads / c.cols;
  c.slice = (int)((c.pixels + slices - 1) / slices);
  c.slices = (int)((c.pixels + c.slice - 1) / c.slice);
  c.by_chunks = FastDiv((uint32_t)c.chunks);
  c.by_slices = FastDiv((uint32_t)c.slices);
  c.by_parts = FastDiv((uint32_t)c.parts);
  c.by_cols = FastDiv((uint32_t)c.cols);
  c.by_rows = FastDiv((uint32_t)c.rows);
  c.by_width = FastDiv((uint32_t)c.width);
}

Cut cut_of(int64_t N, int64_t C, int64_t pixels, int64_t G, int E) {
  Cut c;
  c.N = (int)N; c.C = (int)C; c.G = (int)G; c.width = (int)(C / G); c.pixels = pixels;
  // Chunks of 32 vectors (512 bytes of a pixel) while that leaves enough blocks, else of 16 or 8.  The chip holds 1024 blocks at a
  // time; slices for one to eight times as many, of eight rounds of pixels each at least: those with the fewest rounds one after
  // the other, a block's start and end counted as eight (both directions, us: [128, 56 * 56, 256] bf16 with 1024 blocks 333, 2048
  // 357, 4096 414, chunks of 8 vectors 351; slices for a little over 1024 blocks / a little under: [28, 61 * 81, 366] in 6 groups
  // 219 / 204, [10, 122 * 122, 340] in 4 214 / 199).
  int64_t slices = 1;
  auto cut = [&](int least, int unit) {
    cut_channels(c, E, least, unit);
    const int rows = kThreads / c.cols;
    const int64_t planes = (int64_t)c.N * c.chunks;
    int64_t most = (pixels + 8 * rows - 1) / (8 * rows), fewest = 0;
    if (most > 64) most = 64;
    for (int times = 1; times <= 8; ++times) {
      int64_t n = 1024 * times / planes;
      n = n < 1 ? 1 : n > most ? most : n;
      const int64_t cost = (planes * n + 1023) / 1024 * ((pixels + n * rows - 1) / (n * rows) + 8);
      if (fewest == 0 || cost < fewest) {
        fewest = cost;
        slices = n;
      }
    }
    return planes * slices >= 768;
  };
  const int lines = groups_of_lines(c, E);
  bool enough = lines && cut(32, lines);
  for (int least = 32; !enough && least >= 8; least /= 2) enough = cut(least, 0);
  if (!enough) {                                         // few blocks: four rounds ([5, 55 * 55, 96] 30.4 us, 27.9 like this)
    const int rows = kThreads / c.cols;
    int64_t most = (pixels + 4 * rows - 1) / (4 * rows);
    if (most > 64) most = 64;
    const int64_t room = 1024 / ((int64_t)c.N * c.chunks);
    if (most > room) most = room;
    if (slices < most) slices = most;
  }
  const int64_t needed = (pixels * C >> 30) + 1;        // (offsets inside a slice are 32-bit)
  if (slices < needed) slices = needed < pixels ? needed : pixels;
  cut_pixels(c, slices);
  return c;
}

// One kernel, a block to a sample's chunk, both directions against two kernels each, us:
//   * chunks of whole lines whose blocks fill the chip, up to 64 pixels a thread: [64, 28 * 28, 256] bf16 45.9, 67.9 (64 blocks of
//     32 pixels a thread, [16, 32 * 32, 256]: 47.7, 34.0);
//   * chunks of 8 vectors at least where a thread has few pixels, unless the tensor is so large that parts of lines cost more than
//     the launches: [4, 16 * 16, 320] fp16 24.9, 27.4; [190, 8 * 5, 624] in 24 groups 38.7, 50.0; but [200, 16 * 16, 320] 77.3,
//     62.7.
//     Few blocks with several pixels a thread take chunks of 4 vectors (8 vectors / 4: [4, 16 * 16, 320] 25.2 / 20.7,
//     [32, 22 * 22, 64] in 8 groups 30.6 / 22.7) where those have two groups: a wave adds up a group (forward of one in
//     [4, 16 * 16, 1280] 12.1 / 12.8).
// False: none of these, or a group wider than a block.
constexpr int kFewPixels = 16, kSomePixels = 64;
constexpr int64_t kManyValues = 1 << 23;
bool cut_once(Cut& c, int E) {
  if (c.pixels * c.C >> 30) return false;
  Cut once = c;
  auto cut = [&](int least, int unit) {                  // pixels of a thread
    cut_channels(once, E, least, unit);
    return (c.pixels + kThreads / once.cols - 1) / (kThreads / once.cols);
  };
  auto blocks = [&] { return (int64_t)c.N * once.chunks; };
  const int lines = groups_of_lines(c, E);
  if (!lines || cut(8, lines) > kSomePixels || blocks() < 256) {
    const int64_t mine = cut(8, 0);
    if (!once.per || mine > kFewPixels || (lines && blocks() >= 256 && c.N * c.pixels * c.C >= kManyValues)) return false;
    if (mine >= 6 && blocks() < 256 && (cut(4, 0), once.per < 2)) cut(8, 0);
  }
  cut_pixels(once, 1);
  if (once.blocks() > kMostBlocks) return false;
  c = once;
  return true;
}

// The block's place: blocks run over the chunks first, then the slices, then the samples.
struct Place {
  int n, slice, part;
  int c0, channels, g0, groups;          // first channel, number of them; first group, number of them
  int64_t p0;                            // first pixel, and how many
  int count;
  int cs, row;                           // the first channel of this thread's vector in the chunk, and its first pixel
  int rounds, over;                      // pixels of every row of threads, and the rows that have one more
  ACTNN_DEV Place(const Cut& c, int E, bool backwards, bool whole) {
    const uint32_t rest = c.by_chunks.div(blockIdx.x);
    const int chunk = (int)(blockIdx.x - rest * c.chunks);
    n = (int)c.by_slices.div(rest);
    slice = (int)(rest - (uint32_t)n * c.slices);
    if (backwards) { n = c.N - 1 - n; slice = c.slices - 1 - slice; }
    if (c.per) {
      part = 0;
      g0 = chunk * c.per;
      groups = c.G - g0 < c.per ? c.G - g0 : c.per;
      c0 = g0 * c.width;
      channels = groups * c.width;
    } else {
      g0 = (int)c.by_parts.div((uint32_t)chunk);
      part = chunk - g0 * c.parts;
      groups = 1;
      c0 = g0 * c.width + part * c.chunk;
      channels = c.width - part * c.chunk < c.chunk ? c.width - part * c.chunk : c.chunk;
    }
    p0 = (int64_t)slice * c.slice;
    count = c.pixels - p0 < c.slice ? (int)(c.pixels - p0) : c.slice;
    row = (int)c.by_cols.div(threadIdx.x);
    cs = ((int)threadIdx.x - row * c.cols) * E;
    rounds = (int)c.by_rows.div((uint32_t)count);
    over = count - rounds * c.rows;
    at_end = cs >= channels;                             // (the last chunk may have fewer vectors)
    if (whole) cs = cs < channels - E ? cs : channels - E;
    else if (at_end) cs = 0;
  }
  bool at_end;
  ACTNN_DEV int of_row(int r) const { return rounds + (r < over); }
  ACTNN_DEV int mine(const Cut& c) const { return row < c.rows && !at_end ? of_row(row) : 0; }     // this thread's pixels
  ACTNN_DEV int valid(int E) const { return channels - cs < E ? channels - cs : E; }
};

// vectors of 16 bytes of a tensor, whole or not
template <typename T, bool WHOLE> struct Source {
  const T* at;                           // this thread's vector of the slice's first pixel
  const T* last;
  int valid;
  ACTNN_DEV Source(const T* base, const Cut& c, const Place& b) {
    constexpr int E = kVector<T>;
    at = base + ((int64_t)b.n * c.pixels + b.p0) * c.C + b.c0 + b.cs;
    const int64_t all = (int64_t)c.N * c.pixels * c.C;
    last = base + (all > E ? all - E : 0);               // (a smaller tensor has room for 16 bytes)
    valid = b.valid(E);
  }
  ACTNN_DEV u32x4 get(int offset) const {
    if constexpr (WHOLE) return load16_any(at + offset);
    else return row_vector_ends<T>(load16_row<T>(at + offset, valid, last));
  }
};
template <typename T, bool WHOLE> ACTNN_DEV void put_vector(T* to, const u32x4& v, int valid) {
  if constexpr (WHOLE) store16_any<false>(to, v);
  else store16_part<false>(to, v, valid);
}
typedef u32x2 u32x2_a1 __attribute__((aligned(1)));
typedef uint32_t u32_a1 __attribute__((aligned(1)));
template <typename T> struct CodesAnywhere { typedef u32x2_a1 type; };
template <> struct CodesAnywhere<float> { typedef u32_a1 type; };
template <typename T, bool WHOLE> ACTNN_DEV void put_codes(int8_t* to, typename CodeWords<T>::type w, int valid) {
  if constexpr (WHOLE) {
    *reinterpret_cast<typename CodesAnywhere<T>::type*>(to) = w;
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
    return *reinterpret_cast<const typename CodesAnywhere<T>::type*>(from);
  } else {
    uint32_t words[2] = {0u, 0u};
#pragma unroll
    for (int i = 0; i < kVector<T>; ++i)
      if (i < valid) words[i / 4] |= (uint32_t)(uint8_t)from[i] << (8 * (i % 4));
    if constexpr (sizeof(T) == 4) return words[0];
    else return (Words){words[0], words[1]};
  }
}

// A thread's pixels, AHEAD of them on their way while as many before them are worked on (two: four are 2 % faster for the largest
// tensors and 5 to 8 % slower below, by their code): get(offset) loads one, use(vector,
// offset, i) works on it.  No load is guarded, the waits would follow each of them: what does not exist is the thread's
// first vector once more.
template <typename RAW, int AHEAD> struct Walk {
  RAW next[AHEAD];
  int at, step, mine;
  template <typename GET> ACTNN_DEV void begin(const Cut& c, const Place& b, GET get) {
    step = c.rows * c.C;
    at = b.row * c.C;
    mine = b.mine(c);
    ahead(mine, get);
  }
  template <typename GET> ACTNN_DEV void ahead(int left, GET get) {
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) next[j] = get(j < left ? at + j * step : 0);
  }
  template <typename GET, typename USE> ACTNN_DEV void run(GET get, USE use) {
    for (int i = 0; i < mine; i += AHEAD) {
      RAW raw[AHEAD];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) raw[j] = next[j];
      const int here = at;
      at += AHEAD * step;
      ahead(mine - i - AHEAD, get);
#pragma unroll
      for (int j = 0; j < AHEAD; ++j)
        if (i + j < mine) use(raw[j], here + j * step, i + j);
    }
  }
};

// ------------------------------------------------------------------------------------------
// Sums over a group by a team of lanes: 1 to 64 lanes of a wave, a power of two of them.
// ------------------------------------------------------------------------------------------
struct Team {
  int size, lane, first, step;           // lanes of a team, this one; the team's first group, and the distance to its next
  ACTNN_DEV explicit Team(int groups) {
    int shift = 6;
    while (shift > 0 && groups << shift > kThreads) --shift;
    size = 1 << shift;
    lane = threadIdx.x & (size - 1);
    first = threadIdx.x >> shift;
    step = kThreads >> shift;
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

// The entries [rows][width] of a group by the lanes of a team: f(row, channel).
template <typename F> ACTNN_DEV void each_entry(const Team& team, const Cut& c, int width, int rows, F f) {
  // (a part of a wide group has a width of its own)
  const bool usual = width == c.width;
  int r = usual ? (int)c.by_width.div((uint32_t)team.lane) : team.lane / width, ch = team.lane - r * width;
  const int down = usual ? (int)c.by_width.div((uint32_t)team.size) : team.size / width, across = team.size - down * width;
  while (r < rows) {
    f(r, ch);
    r += down;
    ch += across;
    if (ch >= width) { ch -= width; ++r; }
  }
}

struct Partial { float mean, squares, count, top; };     // top: bits of the largest magnitude, as a float's

// ------------------------------------------------------------------------------------------
// Statistics: a thread's, by channel, and from those the block's, by group.
// ------------------------------------------------------------------------------------------
template <typename T> struct ChannelStats {
  static constexpr int E = kVector<T>;
  float mean[E], squares[E];
  uint32_t top[4];
  float first[E], s1[E], s2[E];          // a run of pixels about its first one
  ACTNN_DEV ChannelStats() {
#pragma unroll
    for (int e = 0; e < E; ++e) mean[e] = squares[e] = 0.0f;
#pragma unroll
    for (int q = 0; q < 4; ++q) top[q] = 0u;
  }
  // the thread's pixel number i, the last one being number last
  ACTNN_DEV void add(const u32x4& raw, int i, int last) {
    float f[E];
    widen(static_cast<const T*>(nullptr), raw, f);
    if (i % kRun == 0) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        first[e] = f[e];
        s1[e] = s2[e] = 0.0f;
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float d = f[e] - first[e];
      s1[e] += d;
      s2[e] = __builtin_fmaf(d, d, s2[e]);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) top[q] = Top<T>::larger(top[q], raw[q] & (sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu));
    if (i % kRun == kRun - 1 || i == last) {
      const float run = (float)(i % kRun + 1), done = (float)(i / kRun * kRun);
      const float by_run = 1.0f / run, share = run / (done + run);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float m = s1[e] * by_run, q = s2[e] - s1[e] * m, d = first[e] + m - mean[e];
        squares[e] += q + d * d * (done * share);
        mean[e] += d * share;
      }
    }
  }
  ACTNN_DEV uint32_t top_of(int e) const {
    return sizeof(T) == 4 ? top[e & 3] : (e & 1) ? top[(e >> 1) & 3] >> 16 : top[(e >> 1) & 3] & 0xffffu;
  }
};
// emit(g, partial) by the first lane of each group's team
template <typename T, typename F>
ACTNN_DEV void block_stats(const ChannelStats<T>& mine, const Cut& c, const Place& b, F emit) {
  constexpr int E = kVector<T>;
  __shared__ float s_mean[kThreads * E], s_squares[kThreads * E];
  __shared__ uint32_t s_top[kThreads * E];
  const int pitch = c.cols * E;
  if (b.row < c.rows && !b.at_end) {
    const int at = b.row * pitch + b.cs;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      s_mean[at + e] = mine.mean[e];
      s_squares[at + e] = mine.squares[e];
      s_top[at + e] = mine.top_of(e);
    }
  }
  __syncthreads();
  const Team team(b.groups);
  const int width = c.per ? c.width : b.channels;        // of a group, in this block
  const float count = (float)b.count * (float)width;
  for (int g = team.first; g < b.groups; g += team.step) {
    const int at0 = g * width;
    const float about = s_mean[at0];                     // (means are summed about one of them, like values)
    float sum = 0.0f, m = about, q = 0.0f;
    uint32_t largest = 0;
    // twice: for the mean, and about it (rows of threads without a pixel count 0)
    for (int pass = 0; pass < 2; ++pass) {
      each_entry(team, c, width, c.rows, [&](int r, int ch) {
        const int at = r * pitch + at0 + ch;
        const float d = s_mean[at] - m, n = (float)b.of_row(r);
        sum = __builtin_fmaf(n, d, sum);
        q += __builtin_fmaf(n * d, d, s_squares[at]);
        largest = largest > s_top[at] ? largest : s_top[at];
      });
      if (pass == 0) {
        m = about + team.sum(sum) / count;
        q = 0.0f;
      }
    }
    q = team.sum(q);
    largest = team.largest(largest);
    if (team.lane == 0) emit(g, Partial{m, q, count, Top<T>::value(largest)});
  }
}

// Forward, first pass: partial statistics [N][G][slots].
template <typename T, bool WHOLE>
__global__ __launch_bounds__(kThreads) void group_norm_stats_kernel(const T* __restrict__ x, Partial* __restrict__ table, Cut c) {
  const Place b(c, kVector<T>, false, WHOLE);
  const Source<T, WHOLE> src(x, c, b);
  ChannelStats<T> stats;
  Walk<u32x4, 2> walk;
  auto get = [&](int offset) { return src.get(offset); };
  walk.begin(c, b, get);
  walk.run(get, [&](const u32x4& raw, int, int i) { stats.add(raw, i, walk.mine - 1); });
  block_stats(stats, c, b, [&](int g, const Partial& v) {
    table[((int64_t)b.n * c.G + b.g0 + g) * c.slots() + b.slice * c.parts + b.part] = v;
  });
}

// a group's statistics from its partial ones, by a team; every lane has them
ACTNN_DEV Partial join(const Team& team, const Partial* p, int slots) {
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
  return Partial{mean, team.sum(q), n, as_float(top)};
}

// By the fast exponential and reciprocal, for fp32 tensors too: their errors (2^-24 of the exponent, a step of the reciprocal) are
// those of the rounding before and after.  fp32 [5, 55 * 55, 96] lies 8.1e-8 from the formula in 64 bits (2-norm) and its input's
// gradient 8.4e-8, torch's exponential and division in 32 bits 8.2e-8 and 8.8e-8.
ACTNN_DEV float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + __expf(-z)); }

// A thread's vector of a parameter, `fallback` without one.
template <int E, bool WHOLE> ACTNN_DEV void by_channel(const float* p, const Place& b, float fallback, float (&v)[E]) {
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = fallback;
  if (!p) return;
  const float* from = p + b.c0 + b.cs;
  if constexpr (WHOLE) {
#pragma unroll
    for (int i = 0; i < E; i += 4) {
      const u32x4 w = load16_any(from + i);
      v[i] = as_float(w.x); v[i + 1] = as_float(w.y); v[i + 2] = as_float(w.z); v[i + 3] = as_float(w.w);
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = from[e < b.valid(E) ? e : 0];
  }
}
// f(e, group in the chunk) for the channels of a thread's vector
template <int E, typename F> ACTNN_DEV void by_group(const Cut& c, const Place& b, F f) {
  int g = 0, left = c.C;
  if (c.per) {
    g = (int)c.by_width.div((uint32_t)b.cs);
    left = (g + 1) * c.width - b.cs;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    f(e, g);
    if (--left == 0) {
      left = c.width;
      if (g + 1 < b.groups) ++g;                         // (behind the chunk's last channel: nobody uses it)
    }
  }
}

// ------------------------------------------------------------------------------------------
// Forward: from statistics to outputs and codes.
// ------------------------------------------------------------------------------------------
struct Forward {
  const Partial* table;
  const float *weight, *bias;            // [C] or null
  float *mean, *rstd, *scale;            // [N, G]
  int8_t* codes;
  float eps;
};
template <typename T> struct Group {     // factor 0: every code is 0
  float mean, rstd;
  decltype(Coder<T>::factor) factor;
};
// a group's statistics on their way to the channels and, by the block that has the group's first pixels, to memory
template <typename T, bool KEEP> ACTNN_DEV Group<T> group_of(const Forward& f, const Partial& v, int64_t at, bool first) {
  Group<T> g;
  g.mean = v.mean;
  g.rstd = 1.0f / __builtin_sqrtf(v.squares / v.count + f.eps);
  g.factor = 0;
  if constexpr (KEEP) {
    const TokenScale s = token_scale(v.top);
    if (s.keep) g.factor = Coder<T>(v.top).factor;
    if (first) f.scale[at] = s.scale;
  }
  if (first) {
    f.mean[at] = g.mean;
    f.rstd[at] = g.rstd;
  }
  return g;
}
// what goes by channel for a thread's vector
template <typename T, bool WHOLE, bool SILU, bool KEEP> struct Normalise {
  static constexpr int E = kVector<T>;
  float mean[E], a[E], add[E];
  Coder<T> coder[E];
  ACTNN_DEV void init(const Forward& f, const Group<T>* groups, const Cut& c, const Place& b) {
    by_channel<E, WHOLE>(f.weight, b, 1.0f, a);
    by_channel<E, WHOLE>(f.bias, b, 0.0f, add);
    by_group<E>(c, b, [&](int e, int g) {
      mean[e] = groups[g].mean;
      a[e] *= groups[g].rstd;
      if constexpr (KEEP) coder[e].factor = groups[g].factor;
    });
  }
  ACTNN_DEV void put(T* y, int8_t* codes, const u32x4& raw, int valid) const {
    const T* none = nullptr;
    float v[E];
    widen(none, raw, v);
    if constexpr (KEEP) {
      int q[E];
#pragma unroll
      for (int e = 0; e < E; ++e) q[e] = coder[e].code(v[e]);
      typename CodeWords<T>::type w;
      if constexpr (E == 4) w = pack_codes(q[0], q[1], q[2], q[3]);
      else w = (u32x2){pack_codes(q[0], q[1], q[2], q[3]), pack_codes(q[4 % E], q[5 % E], q[6 % E], q[7 % E])};
      put_codes<T, WHOLE>(codes, w, valid);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float z = __builtin_fmaf(v[e] - mean[e], a[e], add[e]);
      v[e] = SILU ? z * sigmoid(z) : z;
    }
    put_vector<T, WHOLE>(y, narrow(none, v), valid);
  }
};
// ONCE: the statistics too, from this block's own pixels; else from the table.
template <typename T, bool WHOLE, bool SILU, bool KEEP, bool ONCE>
__global__ __launch_bounds__(kThreads) void group_norm_apply_kernel(const T* __restrict__ x, T* __restrict__ y, Forward f, Cut c) {
  __shared__ Group<T> s_group[kThreads * kVector<T>];
  const Place b(c, kVector<T>, !ONCE, WHOLE);
  const Source<T, WHOLE> src(x, c, b);
  auto get = [&](int offset) { return src.get(offset); };
  Walk<u32x4, 2> walk;
  walk.begin(c, b, get);                                 // (before the statistics are joined)
  if constexpr (ONCE) {
    ChannelStats<T> stats;
    walk.run(get, [&](const u32x4& raw, int, int i) { stats.add(raw, i, walk.mine - 1); });
    walk.begin(c, b, get);
    block_stats(stats, c, b, [&](int g, const Partial& v) {
      s_group[g] = group_of<T, KEEP>(f, v, (int64_t)b.n * c.G + b.g0 + g, true);
    });
  } else {
    const Team team(b.groups);
    for (int g = team.first; g < b.groups; g += team.step) {
      const int64_t at = (int64_t)b.n * c.G + b.g0 + g;
      const Partial v = join(team, f.table + at * c.slots(), c.slots());
      if (team.lane == 0) s_group[g] = group_of<T, KEEP>(f, v, at, b.slice == 0 && b.part == 0);
    }
  }
  __syncthreads();
  Normalise<T, WHOLE, SILU, KEEP> norm;
  norm.init(f, s_group, c, b);
  T* to = y + (src.at - x);
  int8_t* codes = f.codes + (src.at - x);
  walk.run(get, [&](const u32x4& raw, int offset, int) { norm.put(to + offset, codes + offset, raw, src.valid); });
}

// ------------------------------------------------------------------------------------------
// Backward.
// ------------------------------------------------------------------------------------------
struct Backward {
  const int8_t* codes;                   // the kept input: codes and scale [N, G], or null and x
  const float* scale;
  const float *weight, *bias, *mean, *rstd;
  float* sums;                           // [N][slices][2][C]: sum dz, sum dz n
  float* group_sums;                     // [N][G][slots][2]: the same times the weight, over a group's channels (joining `sums`
                                         // in the second pass instead: [2, 20 * 20, 4096] in one group 1081 us backward, 24)
  float *dweight, *dbias;
};

// What goes by channel for a thread's vector, and n, dz of a vector's elements.
template <typename T, bool WHOLE, bool SILU, bool CODES> struct Slope {
  static constexpr int E = kVector<T>;
  float by[E], less[E], w[E], add[E];    // n = value * by - less
  ACTNN_DEV void init(const Backward& k, const Cut& c, const Place& b) {
    by_channel<E, WHOLE>(k.weight, b, 1.0f, w);
    if constexpr (SILU) by_channel<E, WHOLE>(k.bias, b, 0.0f, add);
    const int64_t at = (int64_t)b.n * c.G + b.g0;
    by_group<E>(c, b, [&](int e, int g) {
      const float rstd = k.rstd[at + g];
      by[e] = CODES ? k.scale[at + g] * rstd : rstd;
      less[e] = CODES ? k.mean[at + g] * rstd : k.mean[at + g];
    });
  }
  typedef typename CodeWords<T>::type Words;
  struct Raw { u32x4 dy, x; Words codes; };
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
template <typename T, bool WHOLE, bool SILU, bool CODES> struct Saved {
  typedef typename Slope<T, WHOLE, SILU, CODES>::Raw Raw;
  Source<T, WHOLE> dy, x;
  const int8_t* codes;
  ACTNN_DEV Saved(const T* g, const T* in, const int8_t* q, const Cut& c, const Place& b)
      : dy(g, c, b), x(CODES ? g : in, c, b), codes(q + (dy.at - g)) {}
  ACTNN_DEV Raw get(int offset) const {
    Raw r;
    r.dy = dy.get(offset);
    if constexpr (CODES) r.codes = get_codes<T, WHOLE>(codes + offset, dy.valid);
    else r.x = x.get(offset);
    return r;
  }
};
// A thread's sums over its pixels, by channel: dz, dz n.  LONG: of any number of pixels, by runs of kLongRun, so that no sum is of
// more than some hundred additions in a row (4095 equal terms in a row were off by 5.8e-5 of themselves, by runs less than 4e-6).
constexpr int kLongRun = 128;
template <typename T, bool LONG> struct ChannelSums {
  static constexpr int E = kVector<T>, L = LONG ? E : 1;
  float plain[E], by_n[E], runs_plain[L], runs_by_n[L];
  ACTNN_DEV ChannelSums() {
#pragma unroll
    for (int e = 0; e < E; ++e) plain[e] = by_n[e] = 0.0f;
#pragma unroll
    for (int e = 0; e < L; ++e) runs_plain[e] = runs_by_n[e] = 0.0f;
  }
  // the thread's pixel number i
  template <typename SLOPE> ACTNN_DEV void add(const SLOPE& slope, const typename SLOPE::Raw& r, int i) {
    float n[E], dz[E];
    slope.values(r, n, dz);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      plain[e] += dz[e];
      by_n[e] = __builtin_fmaf(dz[e], n[e], by_n[e]);
    }
    if constexpr (LONG) {
      if (i % kLongRun == kLongRun - 1) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          runs_plain[e] += plain[e];
          runs_by_n[e] += by_n[e];
          plain[e] = by_n[e] = 0.0f;
        }
      }
    }
  }
  ACTNN_DEV void end() {
    if constexpr (LONG) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        plain[e] += runs_plain[e];
        by_n[e] += runs_by_n[e];
      }
    }
  }
};
// dx of a pixel: rstd (u - first - n second), the factors with rstd in them
template <typename T, bool WHOLE, bool SILU, bool CODES> struct Gradient {
  static constexpr int E = kVector<T>;
  float by[E], first[E], second[E];
  ACTNN_DEV void init(const Slope<T, WHOLE, SILU, CODES>& slope, const Backward& k, const float* firsts, const float* seconds,
                      const Cut& c, const Place& b) {
    const int64_t at = (int64_t)b.n * c.G + b.g0;
    by_group<E>(c, b, [&](int e, int g) {
      const float rstd = k.rstd[at + g];
      by[e] = slope.w[e] * rstd;
      first[e] = firsts[g] * rstd;
      second[e] = seconds[g] * rstd;
    });
  }
  typedef Slope<T, WHOLE, SILU, CODES> SlopeT;
  ACTNN_DEV void put(T* dx, const SlopeT& slope, const typename SlopeT::Raw& r, int valid) const {
    float n[E], dz[E];
    slope.values(r, n, dz);
#pragma unroll
    for (int e = 0; e < E; ++e) dz[e] = __builtin_fmaf(-n[e], second[e], __builtin_fmaf(dz[e], by[e], -first[e]));
    put_vector<T, WHOLE>(dx, narrow(static_cast<const T*>(nullptr), dz), valid);
  }
};

// the threads' sums by channel, over the rows of threads: emit(which, channel of the chunk, sum)
template <typename T, bool LONG, typename F>
ACTNN_DEV void block_sums(const ChannelSums<T, LONG>& mine, const Cut& c, const Place& b, F emit) {
  constexpr int E = kVector<T>;
  __shared__ float s_sum[2][kThreads * E];
  const int pitch = c.cols * E;
  if (b.row < c.rows && !b.at_end) {
    const int at = b.row * pitch + b.cs;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      s_sum[0][at + e] = mine.plain[e];
      s_sum[1][at + e] = mine.by_n[e];
    }
  }
  __syncthreads();
  // lanes that share a channel: as many as there are threads for
  const Team team(2 * b.channels);
  for (int i = team.first; i < 2 * b.channels; i += team.step) {
    const int which = i >= b.channels, ch = which ? i - b.channels : i;
    float v = 0.0f;
    for (int r = team.lane; r < c.rows; r += team.size) v += s_sum[which][r * pitch + ch];
    v = team.sum(v);
    if (team.lane == 0) emit(which, ch, v);
  }
}
// and over the channels of each group in the block, times the weight: emit(g, sum u, sum u n)
template <typename F>
ACTNN_DEV void block_group_sums(const float* plain, const float* by_n, const float* weight, const Cut& c, const Place& b, F emit) {
  const int width = c.per ? c.width : b.channels;
  const Team team(b.groups);
  for (int g = team.first; g < b.groups; g += team.step) {
    float first = 0.0f, second = 0.0f;
    for (int in = team.lane; in < width; in += team.size) {
      const int ch = g * width + in;
      const float w = weight ? weight[b.c0 + ch] : 1.0f;
      first = __builtin_fmaf(w, plain[ch], first);
      second = __builtin_fmaf(w, by_n[ch], second);
    }
    first = team.sum(first);
    second = team.sum(second);
    if (team.lane == 0) emit(g, first, second);
  }
}

template <typename T, bool WHOLE, bool SILU, bool CODES>
__global__ __launch_bounds__(kThreads) void group_norm_backward_sums_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                                            Backward k, Cut c) {
  const Place b(c, kVector<T>, false, WHOLE);
  typedef Saved<T, WHOLE, SILU, CODES> SavedT;
  const SavedT saved(dy, x, k.codes, c, b);
  auto get = [&](int offset) { return saved.get(offset); };
  Walk<typename SavedT::Raw, 2> walk;
  walk.begin(c, b, get);
  Slope<T, WHOLE, SILU, CODES> slope;
  slope.init(k, c, b);
  ChannelSums<T, true> sums;
  walk.run(get, [&](const typename SavedT::Raw& raw, int, int i) { sums.add(slope, raw, i); });
  sums.end();
  __shared__ float s_total[2][kThreads * kVector<T>];
  block_sums(sums, c, b, [&](int which, int ch, float v) {
    s_total[which][ch] = v;
    k.sums[(((int64_t)b.n * c.slices + b.slice) * 2 + which) * c.C + b.c0 + ch] = v;
  });
  __syncthreads();
  block_group_sums(s_total[0], s_total[1], k.weight, c, b, [&](int g, float first, float second) {
    float* to = k.group_sums + 2 * (((int64_t)b.n * c.G + b.g0 + g) * c.slots() + b.slice * c.parts + b.part);
    to[0] = first;
    to[1] = second;
  });
}

// ONCE: the sums too, from this block's own pixels; else from the table.
template <typename T, bool WHOLE, bool SILU, bool CODES, bool ONCE>
__global__ __launch_bounds__(kThreads) void group_norm_backward_apply_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                                             T* __restrict__ dx, Backward k, Cut c) {
  constexpr int E = kVector<T>;
  typedef Saved<T, WHOLE, SILU, CODES> SavedT;
  __shared__ float s_mean[2][kThreads * E];
  const Place b(c, E, !ONCE, WHOLE);
  const SavedT saved(dy, x, k.codes, c, b);
  auto get = [&](int offset) { return saved.get(offset); };
  Walk<typename SavedT::Raw, 2> walk;
  walk.begin(c, b, get);                                 // (before the sums are joined)
  Slope<T, WHOLE, SILU, CODES> slope;
  slope.init(k, c, b);
  const float all = 1.0f / ((float)c.pixels * (float)c.width);
  auto means = [&](int g, float first, float second) {
    s_mean[0][g] = first * all;
    s_mean[1][g] = second * all;
  };
  if constexpr (ONCE) {
    __shared__ float s_total[2][kThreads * E];
    ChannelSums<T, false> sums;                           // (kSomePixels at most)
    walk.run(get, [&](const typename SavedT::Raw& raw, int, int i) { sums.add(slope, raw, i); });
    walk.begin(c, b, get);
    block_sums(sums, c, b, [&](int which, int ch, float v) {
      s_total[which][ch] = v;
      k.sums[((int64_t)b.n * 2 + which) * c.C + b.c0 + ch] = v;
    });
    __syncthreads();
    if (!dx) return;
    block_group_sums(s_total[0], s_total[1], k.weight, c, b, means);
  } else {
    const Team team(b.groups);
    for (int g = team.first; g < b.groups; g += team.step) {
      const float* from = k.group_sums + 2 * ((int64_t)b.n * c.G + b.g0 + g) * c.slots();
      float first = 0.0f, second = 0.0f;
      for (int i = team.lane; i < c.slots(); i += team.size) {
        first += from[2 * i];
        second += from[2 * i + 1];
      }
      first = team.sum(first);
      second = team.sum(second);
      if (team.lane == 0) means(g, first, second);
    }
  }
  __syncthreads();
  Gradient<T, WHOLE, SILU, CODES> gradient;
  gradient.init(slope, k, s_mean[0], s_mean[1], c, b);
  T* to = dx + (saved.dy.at - dy);
  walk.run(get, [&](const typename SavedT::Raw& raw, int offset, int) { gradient.put(to + offset, slope, raw, saved.dy.valid); });
}

// dw, db: the table's sums over samples and slices, 16 channels a block, 64 rows of the table at a time.
__global__ __launch_bounds__(kWide) void group_norm_backward_parameters_kernel(Backward k, Cut c) {
  constexpr int kChannels = 16, kRows = kWide / kChannels;
  __shared__ float s_sum[kWide / 64][kChannels];
  const int which = blockIdx.y, in = threadIdx.x & (kChannels - 1), ch = blockIdx.x * kChannels + in;
  const int rows = c.N * c.slices;
  const float* from = k.sums + (int64_t)which * c.C + (ch < c.C ? ch : c.C - 1);
  const int64_t pitch = (int64_t)2 * c.C;
  float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  int r = threadIdx.x / kChannels;
  for (; r + 3 * kRows < rows; r += 4 * kRows)
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] += from[(r + j * kRows) * pitch];
  for (; r < rows; r += kRows) v[0] += from[r * pitch];
  float sum = (v[0] + v[1]) + (v[2] + v[3]);
  sum += __shfl_xor(sum, 16);
  sum += __shfl_xor(sum, 32);
  if ((threadIdx.x & 63) < kChannels) s_sum[threadIdx.x >> 6][in] = sum;
  __syncthreads();
  if (threadIdx.x < kChannels && ch < c.C) {
    sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kWide / 64; ++w) sum += s_sum[w][in];
    float* to = which ? k.dweight : k.dbias;
    if (to) to[ch] = sum;
  }
}

enum { kNone = 0, kSilu = 1 };

// picks the template's flags at run time
template <typename F> void with_flag(bool flag, F f) {
  if (flag) f(std::true_type{});
  else f(std::false_type{});
}

template <typename T> int forward(const void* x, void* y, Forward f, Cut c, bool silu, bool keep, void* ws, hipStream_t s) {
  const bool once = cut_once(c, kVector<T>);
  const dim3 grid((unsigned)c.blocks()), blk(kThreads);
  const T* px = static_cast<const T*>(x);
  T* py = static_cast<T*>(y);
  f.table = static_cast<Partial*>(ws);
  with_flag(whole_vectors(c, kVector<T>), [&](auto W) {
    if (!once) group_norm_stats_kernel<T, decltype(W)::value><<<grid, blk, 0, s>>>(px, static_cast<Partial*>(ws), c);
    with_flag(silu, [&](auto S) {
      with_flag(keep, [&](auto K) {
        with_flag(once, [&](auto O) {
          group_norm_apply_kernel<T, decltype(W)::value, decltype(S)::value, decltype(K)::value, decltype(O)::value>
              <<<grid, blk, 0, s>>>(px, py, f, c);
        });
      });
    });
  });
  ACTNN_RETURN_LAUNCH_STATUS();
}

template <typename T>
int backward(const void* dy, const void* x, void* dx, const Backward& k, Cut c, bool silu, hipStream_t s) {
  const bool once = cut_once(c, kVector<T>);
  const dim3 grid((unsigned)c.blocks()), blk(kThreads);
  const T *pdy = static_cast<const T*>(dy), *px = static_cast<const T*>(x);
  T* pdx = static_cast<T*>(dx);
  with_flag(whole_vectors(c, kVector<T>), [&](auto W) {
    with_flag(silu, [&](auto S) {
      with_flag(k.codes != nullptr, [&](auto Q) {
        constexpr bool w = decltype(W)::value, a = decltype(S)::value, q = decltype(Q)::value;
        if (once) {
          group_norm_backward_apply_kernel<T, w, a, q, true><<<grid, blk, 0, s>>>(pdy, px, pdx, k, c);
        } else {
          group_norm_backward_sums_kernel<T, w, a, q><<<grid, blk, 0, s>>>(pdy, px, k, c);
          if (dx) group_norm_backward_apply_kernel<T, w, a, q, false><<<grid, blk, 0, s>>>(pdy, px, pdx, k, c);
        }
      });
    });
  });
  if (k.dweight || k.dbias)
    group_norm_backward_parameters_kernel<<<dim3((unsigned)((c.C + 15) / 16), 2), dim3(kWide), 0, s>>>(k, c);
  ACTNN_RETURN_LAUNCH_STATUS();
}

int check(int64_t N, int64_t C, int64_t P, int64_t G, int dtype) {
  if (N < 0 || C < 1 || P < 0 || G < 1 || C % G || N > 0x7fffff || C > 0x3fffff || P > 0x7fffffffLL) return ACTNN_EINVAL;
  if (dtype != ACTNN_F32 && dtype != ACTNN_F16 && dtype != ACTNN_BF16) return ACTNN_EDTYPE;
  return ACTNN_OK;
}
int64_t forward_bytes(const Cut& c) { return (int64_t)c.N * c.G * c.slots() * (int64_t)sizeof(Partial); }
int64_t backward_bytes(const Cut& c) { return 8 * ((int64_t)c.N * c.slices * c.C + (int64_t)c.N * c.G * c.slots()); }
// (the table's rows are 32-bit)
bool too_many(const Cut& c) { return c.blocks() > kMostBlocks || (int64_t)c.N * c.slices > 0x7fffff00LL; }

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
  if (workspace_bytes < forward_bytes(c) || too_many(c)) return ACTNN_EINVAL;
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
  if (workspace_bytes < backward_bytes(c) || too_many(c)) return ACTNN_EINVAL;
  float* sums = static_cast<float*>(workspace);
  const Backward k{codes, scale, weight, bias, mean, rstd, sums, sums + 2 * (int64_t)c.N * c.slices * c.C, dweight, dbias};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool silu = activation == kSilu;
  if (dtype == ACTNN_F32) return backward<float>(dy, codes ? nullptr : x, dx, k, c, silu, s);
  if (dtype == ACTNN_F16) return backward<__half>(dy, codes ? nullptr : x, dx, k, c, silu, s);
  return backward<bf16_t>(dy, codes ? nullptr : x, dx, k, c, silu, s);
}
