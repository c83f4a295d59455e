// Group norm: the kernels that do not depend on the stored type, and the launches by type
// (norm_f32.hip, norm_bf16.hip; the kernels themselves are in norm_impl.h, the division in norm_division.h).
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
    m2 += unmarked(p.z) + (double)p.w * (d * d - (double)p.y * (double)p.y);
  }
  double var = block_total(m2, shared) / n_total;
  var = var < 0.0 ? 0.0 : var;                                   // a NaN stays
  if (threadIdx.x == 0) {
    a.mean[blockIdx.x] = (float)mean;
    a.rstd[blockIdx.x] = (float)(1.0 / sqrt(var + (double)a.eps));
  }
}
// One workgroup per (image, group): the image's sums of each channel, and the group's two means.  In 64 bits: an image has
// thousands of tiles, and their sums may all have one sign (8,192 tiles of a constant dy lost 10^-4 of dbias in 32 bits).
__global__ __launch_bounds__(kJoinThreads) void gn_bwd_join_kernel(const NormArgs a, int padded) {
  __shared__ double shared[kJoinThreads / 64];
  const NormGeom& g = a.g;
  const int b = blockIdx.x / g.G, gi = blockIdx.x - b * g.G;
  double m1 = 0.0, m2 = 0.0;
  for (int k = threadIdx.x; k < g.cg; k += blockDim.x) {
    const int c = gi * g.cg + k;
    const float2* part = a.part + (int64_t)b * g.tiles * padded + c;
    double s0 = 0.0, s1 = 0.0;
#pragma unroll 8
    for (int t = 0; t < g.tiles; ++t) {                          // eight loads under way, one order of the sums
      const float2 p = part[(int64_t)t * padded];
      s0 += (double)p.x;
      s1 += (double)p.y;
    }
    a.chan[(int64_t)b * g.C + c] = make_float2((float)s0, (float)s1);
    const double gamma = a.gamma != nullptr ? (double)a.gamma[c] : 1.0;
    m1 = fma(gamma, s0, m1);
    m2 = fma(gamma, s1, m2);
  }
  m1 = block_total(m1, shared);
  m2 = block_total(m2, shared);
  const double n = (double)g.P * g.cg;
  if (threadIdx.x == 0) a.moments[blockIdx.x] = make_float2((float)(m1 / n), (float)(m2 / n));
}
// Sums the rows of channel sums in a fixed order: a workgroup takes 8 channels (one 64-byte piece of a row), 128 threads
// share a channel's rows, of which a thread may have thousands: eight at a time go into 64 bits.  Latency-bound: 4 us for 512
// to 1024 rows of 32 channels (256 KB), a launch included.
__global__ __launch_bounds__(1024) void gn_param_grads_kernel(const NormArgs a) {
  __shared__ float2 shared[16][8];
  const int k = threadIdx.x & 7, r = threadIdx.x >> 3, c = blockIdx.x * 8 + k;
  double s0 = 0.0, s1 = 0.0;
  if (c < a.g.C) {
    for (int row = r; row < a.chan_rows; row += 128 * 8) {       // eight loads in flight: the kernel is one memory latency long
      float2 p[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = a.chan[(int64_t)min(row + i * 128, a.chan_rows - 1) * a.chan_stride + c];
      float2 eight = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        eight.x += row + i * 128 < a.chan_rows ? p[i].x : 0.f;
        eight.y += row + i * 128 < a.chan_rows ? p[i].y : 0.f;
      }
      s0 += (double)eight.x;
      s1 += (double)eight.y;
    }
  }
  float2 s = make_float2((float)s0, (float)s1);
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
  hipLaunchKernelGGL(gn_join_kernel, dim3(a.g.B * a.g.G), dim3(join_threads(a.g, false)), 0, s, a);
}
void launch_gn_bwd_join(const NormArgs& a, int padded, hipStream_t s) {
  hipLaunchKernelGGL(gn_bwd_join_kernel, dim3(a.g.B * a.g.G), dim3(join_threads(a.g, true)), 0, s, a, padded);
}
void launch_gn_param_grads(const NormArgs& a, hipStream_t s) {
  hipLaunchKernelGGL(gn_param_grads_kernel, dim3((a.g.C + 7) / 8), dim3(1024), 0, s, a);
}

// ---------------------------------------------------------------- host
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
static int check_threads(const NormGeom& g, const Slab* s, bool backward, const char* what) {
  const int64_t threads = s ? (int64_t)s->img_blocks * s->parts * s->chunks * s->threads
                            : std::max((int64_t)g.B * g.tiles * g.chunks * kThreads, (int64_t)g.B * g.G * join_threads(g, backward));
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
  if ((rc = check_threads(a.g, sl, false, "group_norm_act_fwd"))) return rc;
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
  if ((rc = check_threads(a.g, sl, true, "group_norm_act_bwd"))) return rc;
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
