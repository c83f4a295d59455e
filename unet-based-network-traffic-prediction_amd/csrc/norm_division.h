// Group norm: how the work is divided among workgroups and threads, and where a workgroup's values lie in LDS.  Nothing here needs
// a GPU, so that the CPU can check every index that the kernels (norm_impl.h) work out against what the launches allocate.
#pragma once
#include "common.h"

namespace mi {

constexpr int kThreads = 256, kWaves = kThreads / 64, kI = 8;

struct NormGeom {
  int B, P, C, G, cg;
  int nv;                      // vectors per pixel
  int lanes, log_lanes;        // lanes per pixel: power of two, at most 64
  int chunks;                  // ranges of `lanes` vectors that make up a pixel
  int rows;                    // pixels read at a time = kThreads / lanes
  int tiles;                   // per image
  int q, n_slots;              // channels that are summed together (a vector, 4 of a bf16 vector, or 1: must divide cg), pieces per vector
  FastDiv d_tiles, d_chunks, d_cg;
};

// ---------------------------------------------------------------- slabs
constexpr int kSlabThreads = 256, kWideThreads = 1024;
struct Slab {
  int cv;                      // vectors per pixel of a chunk: whole groups
  int lanes, log_lanes;        // power of two >= cv, at most 64
  int chunks;
  int tpi, log_tpi;            // threads per image, a power of two >= lanes
  int nb, img_blocks;          // images per workgroup, workgroups along the images
  int rows;                    // tpi / lanes
  int parts;                   // workgroups that share an image (then nb = 1, tpi = kSlabThreads)
  int merge;                   // lanes of a group that shuffles can sum (a power of two), ...
  int left;                    // ... and what then remains: pieces per group / merge
  int threads, iters;          // nb * tpi, pixels per thread
  int polls;                   // how often a part is looked for before its sums are formed here instead
  FastDiv d_chunks, d_parts;
};

// Where a workgroup's values lie in LDS, as the kernels index it and the launches allocate it.
// Sums of a group's pieces that shuffles leave over lie lanes * ns to an image's chunk: the first piece of the group that
// piece j of a lane belongs to.  A lane behind the chunk and a piece of padding belong to none and take the row's first ones,
// whose sum nobody uses.
__host__ __device__ inline int slab_first_piece(const NormGeom& g, const Slab& s, int ns, int chunk, int lane, int j) {
  if (s.left == 1) return lane * ns + j;
  const int c = (chunk * s.cv + lane) * (ns * g.q) + j * g.q;
  if (lane >= s.cv || c >= g.C) return 0;
  return ((int)fdiv((uint32_t)c, g.d_cg) * g.cg) / g.q - chunk * s.cv * ns;
}
// Groups of a chunk: the first, how many (none where it holds padding alone), and which of them channel c belongs to (one of
// them also where c lies behind them).
__host__ __device__ inline int slab_first_group(const NormGeom& g, const Slab& s, int N, int chunk) { return chunk * s.cv * N / g.cg; }
__host__ __device__ inline int slab_groups(const NormGeom& g, const Slab& s, int N, int chunk) {
  const int all = s.cv * N / g.cg, rest = g.G - slab_first_group(g, s, N, chunk), n = all < rest ? all : rest;
  return n > 0 ? n : 0;
}
__host__ __device__ inline int slab_group_of(const NormGeom& g, const Slab& s, int N, int chunk, int c) {
  const int gi = (int)fdiv((uint32_t)(c < g.C ? c : g.C - 1), g.d_cg) - slab_first_group(g, s, N, chunk), last = slab_groups(g, s, N, chunk) - 1;
  const int in = gi < last ? gi : last;
  return in > 0 ? in : 0;
}
// Where the groups' results (two floats each) lie: behind the 2 * ns sums of slab_sum (parts > 1: one image, all its threads).
__host__ __device__ inline int slab_stats_at(const Slab& s, int ns) {
  return s.tpi <= 64 && s.left == 1 ? 0 : ((s.threads + 63) >> 6) * s.lanes * 2 * ns;
}
// Behind them, the number of a missing part, and the sums of the waves (aligned to 16 bytes).
constexpr int kPartialFloats = kSlabThreads * 4;
__host__ __device__ inline int slab_missing_at(int groups) { return 2 * groups; }
__host__ __device__ inline int slab_partial_at(int groups) { return (2 * groups + 5) & ~3; }
// Floats of slab_sum with `sums` sums, and of the kernels.
inline int slab_sum_floats(const Slab& s, int sums) {
  if (s.tpi <= 64 && s.left == 1) return 0;
  return (s.tpi > 64 ? s.threads >> 6 : s.threads >> s.log_tpi) * s.lanes * sums;
}
// the sums, and with several parts (mean, rstd) of each group of the chunk, a number and the sums of the waves
inline int slab_fwd_floats(const NormGeom& g, const Slab& s, int ns, int N) {
  return slab_sum_floats(s, 2 * ns) + (s.parts > 1 ? 2 * (s.cv * N / g.cg + 1) + 2 + kPartialFloats : 0);
}
// the same for the backward kernels, or the sums of the channels, or ReLU's thresholds
inline int slab_bwd_floats(const NormGeom& g, const Slab& s, int ns, int N, bool params, bool relu) {
  int floats = slab_fwd_floats(g, s, ns, N);
  const int channels = params ? (s.threads >> 6) * s.lanes * 2 * N : 0, thresholds = relu ? (s.threads >> s.log_tpi) * s.lanes * N : 0;
  if (channels > floats) floats = channels;
  return thresholds > floats ? thresholds : floats;
}

// Threads that join the tiles of an (image, group): one wave, or 1024 threads where there are many (norm.hip) and a launch holds
// them -- less than 2^32.
constexpr int kJoinThreads = 1024;
inline int join_threads(const NormGeom& g, bool backward) {
  const bool many = backward ? g.cg > 64 : (int64_t)g.tiles * (g.cg / g.q) > 512;
  return many && (int64_t)g.B * g.G * kJoinThreads < (1ll << 32) ? kJoinThreads : 64;
}

inline unsigned slab_grid(const Slab& s) { return (unsigned)(s.img_blocks * s.parts * s.chunks); }
// 64-bit words that the parts exchange
inline int64_t slab_words(const NormGeom& g, const Slab& s) { return 2 * (int64_t)g.B * s.parts * g.G; }

inline int gcd_int(int a, int b) {
  while (b) { const int t = a % b; a = b; b = t; }
  return a;
}
inline NormGeom norm_geom(int B, int H, int W, int C, int G, int dtype) {
  NormGeom g{};
  const int N = dtype == MI_BF16 ? 8 : 4;
  g.B = B; g.P = H * W; g.C = C; g.G = G; g.cg = C / G;
  g.nv = pad_ch(C) / N;
  while (g.lanes = 1 << g.log_lanes, g.lanes < g.nv && g.lanes < 64) ++g.log_lanes;
  g.chunks = (g.nv + g.lanes - 1) / g.lanes;
  g.rows = kThreads / g.lanes;
  g.tiles = (g.P + g.rows * kI - 1) / (g.rows * kI);
  g.q = gcd_int(g.cg, N);
  if (g.q != N && !(N == 8 && g.q == 4)) g.q = 1;                // the kernels come for 1, 2 (bf16) and N pieces per vector
  g.n_slots = N / g.q;
  g.d_tiles = make_fastdiv(g.tiles);
  g.d_chunks = make_fastdiv(g.chunks);
  g.d_cg = make_fastdiv(g.cg);
  return g;
}
inline int pow2_ceil(int64_t v) {
  int p = 1;
  while (p < v) p <<= 1;
  return p;
}
// How the slab kernels divide the work, or false where they do not apply.
// Up to 64 parts, which run at the same time on a fraction of the card; more have not been measured since the parts of an image
// start next to each other.  Without parts, by the general kernels: 16 images of 128x128x64 bf16 25 us forward and 48 backward,
// with them 17 and 28; 2 of 256x256x32 14 and 24 against 12 and 17; 1024 of 64x64x32 154 and 286 against 109 and 176.
constexpr int kMaxParts = 64;
constexpr int kPolls = 4096;                 // about 1 us each
// The division with `iters` vectors a thread of chunks of cv vectors, up to `most` threads for an image, `most_nb` for several.
inline bool divide_slab(const NormGeom& g, int64_t cv, int iters, int most, int most_nb, Slab* out) {
  Slab s{};
  s.iters = iters;
  s.cv = (int)cv;
  s.lanes = pow2_ceil(cv);
  while ((1 << s.log_lanes) < s.lanes) ++s.log_lanes;
  s.chunks = (int)((g.nv + cv - 1) / cv);
  const int64_t vectors = (int64_t)g.P * s.lanes;
  s.tpi = vectors < iters * most ? pow2_ceil((vectors + iters - 1) / iters) : most;
  if (s.tpi < s.lanes) s.tpi = s.lanes;
  while ((1 << s.log_tpi) < s.tpi) ++s.log_tpi;
  s.rows = s.tpi / s.lanes;
  const int64_t parts = (g.P + (int64_t)s.rows * iters - 1) / ((int64_t)s.rows * iters);
  if (parts > kMaxParts) return false;
  s.parts = (int)parts;
  s.nb = 1;
  if (s.parts == 1)
    while (s.nb * s.tpi < most_nb && s.nb < g.B) s.nb *= 2;
  s.img_blocks = (g.B + s.nb - 1) / s.nb;
  s.threads = s.nb * s.tpi < 64 ? 64 : s.nb * s.tpi;
  const int ppg = g.cg / g.q;
  s.merge = g.n_slots == 1 && (ppg & (ppg - 1)) == 0 ? ppg : 1;
  s.left = ppg / s.merge;
  s.polls = kPolls;
  s.d_chunks = make_fastdiv(s.chunks);
  s.d_parts = make_fastdiv(s.parts);
  *out = s;
  return true;
}
inline bool choose_slab(const NormGeom& g, int N, bool backward, Slab* out) {
  const int unit = g.cg / gcd_int(g.cg, N) < g.nv ? g.cg / gcd_int(g.cg, N) : g.nv;   // vectors after which a group ends with a vector
  if (unit > 64) return false;
  const int64_t most = 16 * kSlabThreads, few = 4 * kSlabThreads;
  const bool small = (int64_t)g.B * g.P * g.nv < 256 * most;     // not enough to give every CU a full workgroup
  int64_t cv = g.nv <= 64 ? g.nv : unit * (64 / unit);
  // Fewer workgroups than CUs: narrower chunks, down to one line of 128 bytes per pixel, or to 64 bytes where an image's
  // chunk then has a workgroup of its own.  Measured, forward / backward: 8 images of 4x4x1024 fp32 4.0 / 7.0 us with whole
  // pixels, 3.7 / 6.5 so; 32 of 16x16x64 bf16 6.0 / 11.3 with 128 bytes, 4.3 / 8.1 with 64 (with 32: 5.0 / 8.7); but
  // 16 of 128x128x64 bf16, which have parts, 14.1 / 24.3 with 128 bytes and 18.8 / 38 with 64.
  // Backward, an image of more than 64 parts is cut into narrower chunks whatever their number: one of 256x256x512 fp32 223 us
  // by the general kernels, 145 in chunks of 64 bytes, 16 of 256x256x64 bf16 133 and 110, 256 of 70x70x256 fp32 1168 and 607.
  // Forward the same gives 86 and 103, 76 and 81, but 739 and 467: not taken, though large batches of wide pixels would gain.
  for (;;) {
    const int64_t lanes = pow2_ceil(cv), size = g.P * lanes, wgs = (int64_t)g.B * ((g.nv + cv - 1) / cv);
    int64_t half = cv / 2 / unit * unit;
    if (2 * pow2_ceil(half) < lanes) half = lanes / 2 / unit * unit;
    const bool cut = backward && size > kMaxParts * most;
    const int64_t least = cut || g.P * (int64_t)pow2_ceil(half) <= most ? 4 : 8;
    if (pow2_ceil(half) < least || (!cut && (wgs >= 256 || size <= 256))) break;
    cv = half;
  }
  // And below that, down to a lane, where it spares an image of a tensor of at most 256 KB its parts, whose words take a
  // launch to empty: one image of 64x64x32 bf16 8.0 us forward and 11.1 backward on the device, with parts 8.0 and 11.7, and
  // 3 us less on the host.  Larger tensors lose more by the lines read in pieces: one image of 64x64x64 11 and 23 us, with
  // parts 7.7 and 11.5; 8 of 64x64x32 10.8 and 19.7, with parts 8.4 and 13.3.
  if ((int64_t)g.B * g.P * g.nv <= 4 * most && g.P * (int64_t)pow2_ceil(cv) > most) {
    int64_t narrow = cv;
    while (narrow >= unit && g.P * (int64_t)pow2_ceil(narrow) > most) narrow = narrow / 2 / unit * unit;
    if (narrow >= unit) cv = narrow;
  }
  const int64_t vectors = (int64_t)g.P * pow2_ceil(cv);
  // 16 vectors a thread, as many as its registers hold, where that leaves every CU a workgroup; else 4, and a fourth of the
  // time.  An image of up to 4096 vectors then has up to 1024 threads, to be spared parts; backward, all images of a chunk
  // share these threads if they can, and no launch has to join the parameter gradients.  Measured, forward / backward:
  // 512 images of 4x4x256 bf16 4.5 / 10 us, with 16 vectors 6.2 / 15.2; 64 of 8x8x512 fp32 5.7 / 9.4 with 1024 threads,
  // 6.6 / 11.3 with 16 vectors and 256; 8 of 4x4x1024 fp32 backward 4.7 and 6.5.
  const bool alone = backward && g.B <= kSlabThreads && pow2_ceil(g.B) * vectors <= most;
  int iters = small ? 4 : 16;
  if (vectors <= pow2_ceil(cv)) iters = 1;
  else if (alone && pow2_ceil(g.B) * vectors <= few) iters = 4;
  const int threads = small && vectors <= most ? kWideThreads : kSlabThreads;
  return divide_slab(g, cv, iters, iters == 4 ? threads : kSlabThreads, alone && iters == 4 ? threads : kSlabThreads, out) ||
         divide_slab(g, cv, 16, kSlabThreads, kSlabThreads, out);
}

}  // namespace mi
