// Group norm: the kernels that do not depend on the stored type, how the work is divided, and the launches by type
// (norm_f32.hip, norm_bf16.hip; the kernels themselves are in norm_impl.h).
#include "norm_impl.h"

#include <algorithm>

namespace mi {

int launch_gn_fwd_f32(const NormArgs& a, const Slab* sl, hipStream_t s);
int launch_gn_fwd_bf16(const NormArgs& a, const Slab* sl, hipStream_t s);
int launch_gn_bwd_f32(const NormArgs& a, const Slab* sl, hipStream_t s);
int launch_gn_bwd_bf16(const NormArgs& a, const Slab* sl, hipStream_t s);

// The sum over a workgroup, the same for all its threads; `shared` holds one value per wave.
template <typename F> __device__ __forceinline__ F block_total(F v, F* shared) {
  v = wave_total(v);
  if (blockDim.x == 64) return v;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
  __syncthreads();
  v = shared[0];
  for (unsigned w = 1; w < blockDim.x >> 6; ++w) v += shared[w];
  return v;
}
// Joins the tiles and pieces of a group.  Piece k of an image's tile covers channels k*q .. k*q + q - 1.  One wave, or 1024
// threads where there are many: a wave takes a memory latency for every 64 (22 images of 75x41x617 fp32 in one group, 60,000
// pieces each, 576 us forward with one wave, 145 so; 9 of 64x64x1024 backward, channels along the threads, 626 and 152).
constexpr int kJoinThreads = 1024;
__global__ __launch_bounds__(kJoinThreads) void gn_join_kernel(const NormArgs a) {
  __shared__ double shared[kJoinThreads / 64];
  const NormGeom& g = a.g;
  const int b = blockIdx.x / g.G, gi = blockIdx.x - b * g.G;
  const int ppg = g.cg / g.q, per_image = g.nv * g.n_slots;
  const int items = g.tiles * ppg;
  const float4* part = (const float4*)a.part + (int64_t)b * g.tiles * per_image + gi * ppg;
  const double n_total = (double)g.P * g.cg;
  double s = 0.0, m2 = 0.0;
  for (int k = threadIdx.x; k < items; k += blockDim.x) {
    const int t = k / ppg;
    const float4 p = part[(int64_t)t * per_image + (k - t * ppg)];
    s += (double)p.w * ((double)p.x + (double)p.y);
  }
  const double mean = block_total(s, shared) / n_total;
  for (int k = threadIdx.x; k < items; k += blockDim.x) {
    const int t = k / ppg;
    const float4 p = part[(int64_t)t * per_image + (k - t * ppg)];
    const double d = (double)p.x + (double)p.y - mean;
    m2 += (double)p.z + (double)p.w * (d * d - (double)p.y * (double)p.y);
  }
  double var = block_total(m2, shared) / n_total;
  var = var < 0.0 ? 0.0 : var;                                   // a NaN stays
  if (threadIdx.x == 0) {
    a.mean[blockIdx.x] = (float)mean;
    a.rstd[blockIdx.x] = (float)(1.0 / sqrt(var + (double)a.eps));
  }
}
// One workgroup per (image, group): the image's sums of each channel, and the group's two means.
__global__ __launch_bounds__(kJoinThreads) void gn_bwd_join_kernel(const NormArgs a, int padded) {
  __shared__ float shared[kJoinThreads / 64];
  const NormGeom& g = a.g;
  const int b = blockIdx.x / g.G, gi = blockIdx.x - b * g.G;
  float m1 = 0.f, m2 = 0.f;
  for (int k = threadIdx.x; k < g.cg; k += blockDim.x) {
    const int c = gi * g.cg + k;
    const float2* part = a.part + (int64_t)b * g.tiles * padded + c;
    float2 s = make_float2(0.f, 0.f);
#pragma unroll 8
    for (int t = 0; t < g.tiles; ++t) {                          // eight loads under way, one order of the sums
      const float2 p = part[(int64_t)t * padded];
      s.x += p.x;
      s.y += p.y;
    }
    a.chan[(int64_t)b * g.C + c] = s;
    const float gamma = a.gamma != nullptr ? a.gamma[c] : 1.f;
    m1 = fmaf(gamma, s.x, m1);
    m2 = fmaf(gamma, s.y, m2);
  }
  m1 = block_total(m1, shared);
  m2 = block_total(m2, shared);
  const float n = (float)g.P * (float)g.cg;
  if (threadIdx.x == 0) a.moments[blockIdx.x] = make_float2(m1 / n, m2 / n);
}
// Sums the rows of channel sums in a fixed order: a workgroup takes 8 channels (one 64-byte piece of a row), 128 threads
// share a channel's rows.  Latency-bound: 4 us for 512 to 1024 rows of 32 channels (256 KB), a launch included.
__global__ __launch_bounds__(1024) void gn_param_grads_kernel(const NormArgs a) {
  __shared__ float2 shared[16][8];
  const int k = threadIdx.x & 7, r = threadIdx.x >> 3, c = blockIdx.x * 8 + k;
  float2 s = make_float2(0.f, 0.f);
  if (c < a.g.C) {
    for (int row = r; row < a.chan_rows; row += 128 * 8) {       // eight loads in flight: the kernel is one memory latency long
      float2 p[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = a.chan[(int64_t)min(row + i * 128, a.chan_rows - 1) * a.chan_stride + c];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        s.x += row + i * 128 < a.chan_rows ? p[i].x : 0.f;
        s.y += row + i * 128 < a.chan_rows ? p[i].y : 0.f;
      }
    }
  }
#pragma unroll
  for (int o = 32; o >= 8; o >>= 1) {
    s.x += __shfl_xor(s.x, o, 64);
    s.y += __shfl_xor(s.y, o, 64);
  }
  if ((threadIdx.x & 63) < 8) shared[threadIdx.x >> 6][k] = s;
  __syncthreads();
  if (threadIdx.x < 8 && c < a.g.C) {
    for (int w = 1; w < 16; ++w) {
      s.x += shared[w][k].x;
      s.y += shared[w][k].y;
    }
    if (a.dgamma) a.dgamma[c] = a.ga * s.y + (a.gb != 0.f ? a.gb * a.dgamma[c] : 0.f);
    if (a.dbeta) a.dbeta[c] = a.ga * s.x + (a.gb != 0.f ? a.gb * a.dbeta[c] : 0.f);
  }
}
// Fills the words that parts exchange (a kernel, not a memset: the call may be captured into a graph).
__global__ __launch_bounds__(256) void gn_empty_kernel(uint64_t* words, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) words[i] = kEmpty;
}
void launch_gn_empty(uint64_t* words, int64_t n, hipStream_t s) {
  const int64_t blocks = (n + 255) / 256;
  hipLaunchKernelGGL(gn_empty_kernel, dim3((unsigned)(blocks < 1024 ? blocks : 1024)), dim3(256), 0, s, words, n);
}
void launch_gn_join(const NormArgs& a, hipStream_t s) {
  const bool many = (int64_t)a.g.tiles * (a.g.cg / a.g.q) > 512;
  hipLaunchKernelGGL(gn_join_kernel, dim3(a.g.B * a.g.G), dim3(many ? kJoinThreads : 64), 0, s, a);
}
void launch_gn_bwd_join(const NormArgs& a, int padded, hipStream_t s) {
  hipLaunchKernelGGL(gn_bwd_join_kernel, dim3(a.g.B * a.g.G), dim3(a.g.cg > 64 ? kJoinThreads : 64), 0, s, a, padded);
}
void launch_gn_param_grads(const NormArgs& a, hipStream_t s) {
  hipLaunchKernelGGL(gn_param_grads_kernel, dim3((a.g.C + 7) / 8), dim3(1024), 0, s, a);
}

// ---------------------------------------------------------------- host
static int gcd_int(int a, int b) {
  while (b) { const int t = a % b; a = b; b = t; }
  return a;
}
static NormGeom norm_geom(int B, int H, int W, int C, int G, int dtype) {
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
static int pow2_ceil(int64_t v) {
  int p = 1;
  while (p < v) p <<= 1;
  return p;
}
// How the slab kernels divide the work, or false where they do not apply.
// Up to 64 parts, which run at the same time on a fraction of the card.  Without parts, by the general kernels: 16 images of 128x128x64
// bf16 20 us forward and 75 backward, with them 14 and 25; 2 of 256x256x32 12.7 and 50 against 13.6 and 20.
constexpr int kMaxParts = 64;
constexpr int kPolls = 4096;                 // about 1 us each
// The division with `iters` vectors a thread of chunks of cv vectors, up to `most` threads for an image, `most_nb` for several.
static bool divide_slab(const NormGeom& g, int64_t cv, int iters, int most, int most_nb, Slab* out) {
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
static bool choose_slab(const NormGeom& g, int N, bool backward, Slab* out) {
  const int unit = g.cg / gcd_int(g.cg, N) < g.nv ? g.cg / gcd_int(g.cg, N) : g.nv;   // vectors after which a group ends with a vector
  if (unit > 64) return false;
  const int64_t most = 16 * kSlabThreads, few = 4 * kSlabThreads;
  const bool small = (int64_t)g.B * g.P * g.nv < 256 * most;     // not enough to give every CU a full workgroup
  int64_t cv = g.nv <= 64 ? g.nv : unit * (64 / unit);
  // Fewer workgroups than CUs: narrower chunks, down to one line of 128 bytes per pixel, or to 64 bytes where an image's
  // chunk then has a workgroup of its own.  Measured, forward / backward: 8 images of 4x4x1024 fp32 4.0 / 7.0 us with whole
  // pixels, 3.7 / 6.5 so; 32 of 16x16x64 bf16 6.0 / 11.3 with 128 bytes, 4.3 / 8.1 with 64 (with 32: 5.0 / 8.7); but
  // 16 of 128x128x64 bf16, which have parts, 14.1 / 24.3 with 128 bytes and 18.8 / 38 with 64.
  // Backward, an image of more than 64 parts is cut into narrower chunks whatever their number: one of 256x256x512 fp32 616 us
  // by the general kernels, 151 in chunks of 64 bytes, 16 of 256x256x64 bf16 225 and 124; forward 120 and 146, 88 and 106.
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
static size_t slab_rows(const Slab& s) { return (size_t)s.img_blocks * s.parts; }   // rows of channel sums
static size_t fwd_part_bytes(const NormGeom& g) { return (size_t)g.B * g.tiles * g.nv * g.n_slots * sizeof(float4); }
static size_t bwd_part_bytes(const NormGeom& g, int dtype) {
  return (size_t)g.B * g.tiles * g.nv * (dtype == MI_BF16 ? 8 : 4) * sizeof(float2);
}
size_t group_norm_ws_bytes(int B, int H, int W, int C, int G, int backward, int dtype) {
  const NormGeom g = norm_geom(B, H, W, C, G, dtype);
  const int N = dtype == MI_BF16 ? 8 : 4;
  Slab s;
  if (!backward) {
    if (choose_slab(g, N, false, &s)) return s.parts > 1 ? slab_words(g, s) * sizeof(uint64_t) : 0;
    return fwd_part_bytes(g);
  }
  if (choose_slab(g, N, true, &s)) return (s.parts > 1 ? slab_words(g, s) / 2 * sizeof(uint64_t) : 0) + (slab_rows(s) > 1 ? slab_rows(s) * C * sizeof(float2) : 0);
  return bwd_part_bytes(g, dtype) + ((size_t)B * C + (size_t)B * G) * sizeof(float2);
}

static int check_range(const NormGeom& g, const char* what) {
  MI_REQUIRE((int64_t)g.B * g.P < (1ll << 31) && (int64_t)g.B * g.G < (1ll << 31) &&
                 (int64_t)g.B * g.tiles * g.chunks < (1ll << 31), std::string(what) + ": tensor too large");
  return MI_OK;
}
// A launch holds less than 2^32 threads.
static int check_threads(const NormGeom& g, const Slab* s, const char* what) {
  const int64_t threads = s ? (int64_t)s->img_blocks * s->parts * s->chunks * s->threads
                            : std::max((int64_t)g.B * g.tiles * g.chunks * kThreads, (int64_t)g.B * g.G * kJoinThreads);
  MI_REQUIRE(threads < (1ll << 32), std::string(what) + ": tensor too large");
  return MI_OK;
}
int launch_group_norm_fwd(const void* x, int xcs, int xco, const float* gamma, const float* beta, void* y, int ycs, int yco,
                          float* mean, float* rstd, int B, int H, int W, int C, int G, int act, float eps,
                          const mi_dropout* drop, int polls, void* ws, size_t ws_bytes, int dtype, hipStream_t s) {
  NormArgs a{};
  int rc = make_drop_args(drop, &a.drop);
  if (rc) return rc;
  a.g = norm_geom(B, H, W, C, G, dtype);
  if ((rc = check_range(a.g, "group_norm_act_fwd"))) return rc;
  if (B == 0) return MI_OK;
  Slab slab;
  const Slab* sl = choose_slab(a.g, dtype == MI_BF16 ? 8 : 4, false, &slab) ? &slab : nullptr;
  if ((rc = check_threads(a.g, sl, "group_norm_act_fwd"))) return rc;
  if (polls >= 0) slab.polls = polls;
  if (ws_bytes < group_norm_ws_bytes(B, H, W, C, G, 0, dtype)) return fail(MI_ESIZE, "group_norm_act_fwd: workspace too small");
  a.x = x; a.xcs = xcs; a.xco = xco;
  a.out = y; a.ocs = ycs; a.oco = yco;
  a.gamma = gamma; a.beta = beta; a.mean = mean; a.rstd = rstd;
  a.act = act; a.eps = eps;
  a.part = (float2*)ws;
  a.words = (uint64_t*)ws;
  return dtype == MI_BF16 ? launch_gn_fwd_bf16(a, sl, s) : launch_gn_fwd_f32(a, sl, s);
}
int launch_group_norm_bwd(const void* x, int xcs, int xco, const void* dy, int ycs, int yco, const float* gamma, const float* beta,
                          const float* mean, const float* rstd, void* dx, int dcs, int dco, float* dgamma, float* dbeta,
                          float ga, float gb, int B, int H, int W, int C, int G, int act, const mi_dropout* drop, int polls,
                          void* ws, size_t ws_bytes, int dtype, hipStream_t s) {
  NormArgs a{};
  int rc = make_drop_args(drop, &a.drop);
  if (rc) return rc;
  a.g = norm_geom(B, H, W, C, G, dtype);
  if ((rc = check_range(a.g, "group_norm_act_bwd"))) return rc;
  Slab slab;
  const Slab* sl = B > 0 && choose_slab(a.g, dtype == MI_BF16 ? 8 : 4, true, &slab) ? &slab : nullptr;
  if ((rc = check_threads(a.g, sl, "group_norm_act_bwd"))) return rc;
  if (polls >= 0) slab.polls = polls;
  if (ws_bytes < group_norm_ws_bytes(B, H, W, C, G, 1, dtype)) return fail(MI_ESIZE, "group_norm_act_bwd: workspace too small");
  a.x = x; a.xcs = xcs; a.xco = xco;
  a.dy = dy; a.ycs = ycs; a.yco = yco;
  a.out = dx; a.ocs = dcs; a.oco = dco;
  a.gamma = gamma; a.beta = beta; a.mean = const_cast<float*>(mean); a.rstd = const_cast<float*>(rstd);
  a.act = act;
  a.chan_stride = C;
  if (sl) {
    a.words = (uint64_t*)ws;
    a.parts = slab.parts;
    a.chan = (float2*)(a.words + (slab.parts > 1 ? slab_words(a.g, slab) / 2 : 0));
    a.chan_rows = (int)slab_rows(slab);
  } else {
    a.part = (float2*)ws;
    a.chan = a.part + bwd_part_bytes(a.g, dtype) / sizeof(float2);
    a.chan_rows = B;
    a.moments = a.chan + (size_t)B * C;
  }
  a.dgamma = dgamma; a.dbeta = dbeta; a.ga = ga; a.gb = gb;
  return dtype == MI_BF16 ? launch_gn_bwd_bf16(a, sl, s) : launch_gn_bwd_f32(a, sl, s);
}

}  // namespace mi
