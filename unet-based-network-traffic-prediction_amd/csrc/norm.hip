// Group norm with an activation (and dropout) on NHWC views, forward and backward.
//
//   h = (x - mean) * rstd,  z = h * gamma + beta,  y = drop(act(z))            mean, rstd over a group's cg channels x P pixels
//   dz = drop(dy) * act'(z),  t = gamma * dz,  dx = rstd * (t - mean_g(t) - h * mean_g(t * h))
//   dgamma = sum dz * h,  dbeta = sum dz                                        over images and pixels
//
// Both directions are HBM-bound (about 10 and 40 operations per 4 and 6 bytes).  Everything is held in fp32 from the load on;
// what is stored in bf16 is rounded once.
//
// Tiles.  A workgroup owns kI * R pixels of one image and up to 64 vectors (16 bytes: 8 or 4 channels) of each: its
// lanes lie along the channels, so a pixel's 64..1024 bytes are read by neighbours, and R = 256 / lanes-per-pixel rows
// of pixels are read at a time.  A thread keeps its channels for all of its kI pixels: per-channel values are loaded
// once and sums stay in registers until the end.
//
// Precision of the statistics: the corrected two-pass form (Chan, Golub, LeVeque, "Algorithms for computing the sample
// variance", 1983).  A tile's mean m comes first, from registers; then r = sum (x - m) and q = sum (x - m)^2, which give
// the mean m + r / n and the squared deviations q - r^2 / n without m's own rounding; tiles are joined in 64 bits.  Data
// far from zero lose nothing: at a mean of 10^4 standard deviations rstd is off by 1e-7, without r by 2e-5.
// Sums have a fixed order: results repeat bit for bit.
#include "drop.h"

namespace mi {

constexpr int kThreads = 256, kWaves = kThreads / 64, kI = 8;

struct NormGeom {
  int B, P, C, G, cg;
  int nv;                      // vectors per pixel
  int lanes, log_lanes;        // lanes per pixel: power of two, at most 64
  int chunks;                  // ranges of `lanes` vectors that make up a pixel
  int rows;                    // pixels read at a time = kThreads / lanes
  int tiles;                   // per image
  int q, n_slots;              // channels that are summed together, gcd(cg, vector width), and how often they fit a vector
  FastDiv d_tiles, d_chunks, d_cg;
};

struct NormArgs {
  NormGeom g;
  const void* x; int xcs, xco;
  const void* dy; int ycs, yco;        // backward
  void* out; int ocs, oco;             // y or dx
  const float* gamma; const float* beta;
  float* mean; float* rstd;            // [B][G]
  int act;
  float eps;
  float2* part;                        // forward: [B][tiles][pieces] float4; backward: [B][tiles][nv * N] (sum dz, sum dz*h)
  float2* chan;                        // backward: [B][C] (sum dz, sum dz*h) of an image
  float2* moments;                     // backward: [B][G] (mean t, mean t*h)
  float* dgamma; float* dbeta; float ga, gb;
  DropArgs drop;
};

template <typename F> __device__ __forceinline__ F wave_total(F v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// ---------------------------------------------------------------- activations
template <typename T> __device__ __forceinline__ float exp_for(float v);
template <> __device__ __forceinline__ float exp_for<float>(float v) { return expf(v); }
// bf16 results keep 8 bits: the argument's rounding (|v| 2^-24 of the result) is far below that
template <> __device__ __forceinline__ float exp_for<__bf16>(float v) { return __builtin_amdgcn_exp2f(v * 1.44269504f); }

template <typename T> __device__ __forceinline__ float act_value(float z, int act) {
  switch (act) {
    case MI_ACT_RELU: return z > 0.f ? z : (z <= 0.f ? 0.f : z);   // a NaN stays one
    case MI_ACT_SILU: return z * __builtin_amdgcn_rcpf(1.f + exp_for<T>(-z));
    case MI_ACT_GELU: return 0.5f * z * (1.f + erff(z * 0.70710678f));
    default: return z;
  }
}
// act'(z)
template <typename T> __device__ __forceinline__ float act_slope(float z, int act) {
  switch (act) {
    case MI_ACT_RELU: return z > 0.f ? 1.f : 0.f;
    case MI_ACT_SILU: {
      const float s = __builtin_amdgcn_rcpf(1.f + exp_for<T>(-z));
      return s + z * s * (1.f - s);
    }
    case MI_ACT_GELU: return 0.5f * (1.f + erff(z * 0.70710678f)) + z * 0.39894228f * exp_for<T>(-0.5f * z * z);
    default: return 1.f;
  }
}

// ---------------------------------------------------------------- a workgroup's tile
struct Tile {
  int b, t, v, row;            // image, tile, vector of this thread, first pixel of this thread
  int n;                       // how many of this thread's kI pixels exist
  int count;                   // pixels of the tile
  bool live;                   // this thread's vector exists
};
__device__ __forceinline__ Tile my_tile(const NormGeom& g) {
  Tile w;
  const uint32_t i = blockIdx.x, it = fdiv(i, g.d_chunks), chunk = i - it * g.chunks;
  w.b = (int)fdiv(it, g.d_tiles);
  w.t = (int)it - w.b * g.tiles;
  const int lane = (int)threadIdx.x & (g.lanes - 1), r = (int)threadIdx.x >> g.log_lanes;
  w.v = (int)chunk * g.lanes + lane;
  w.live = w.v < g.nv;
  w.v = min(w.v, g.nv - 1);
  const int p0 = w.t * (g.rows * kI);
  w.count = min(g.P - p0, g.rows * kI);
  w.row = p0 + r;
  w.n = w.count > r ? min(kI, (w.count - r + g.rows - 1) >> (31 - __clz(g.rows))) : 0;
  return w;
}
// Loads are unconditional (a pixel behind the tile reads the image's last one instead, and is weighted with zero or not stored).
template <typename T>
__device__ __forceinline__ void load_tile(const Tile& w, const NormGeom& g, const void* base, int cs, int co, u32x4_t* v) {
  const T* p = (const T*)base + (int64_t)w.b * g.P * cs + co + w.v * ActVec<T>::N;
#pragma unroll
  for (int i = 0; i < kI; ++i) v[i] = load_stream(p + (int64_t)min(w.row + i * g.rows, g.P - 1) * cs);
}
// Sums over the rows of the tile: in, NS values per thread; out, shared[lane * NS + slot] for every lane of a pixel.
// `shared` holds kWaves * 64 * NS values.
template <int NS>
__device__ __forceinline__ void tile_sum(const float* v, const NormGeom& g, float* shared) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float r[NS];
#pragma unroll
  for (int j = 0; j < NS; ++j) r[j] = v[j];
  for (int o = 32; o >= g.lanes; o >>= 1) {
#pragma unroll
    for (int j = 0; j < NS; ++j) r[j] += __shfl_xor(r[j], o, 64);
  }
  __syncthreads();
  if (lane < g.lanes) {
#pragma unroll
    for (int j = 0; j < NS; ++j) shared[(wave * 64 + lane) * NS + j] = r[j];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < g.lanes * NS; i += kThreads) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < kWaves; ++k) s += shared[k * 64 * NS + i];
    shared[i] = s;                                               // nobody else reads or writes slot i of wave 0
  }
  __syncthreads();
}

// One value per channel, the same for all pixels: of channel c, or of its group, or a default.
template <int N>
__device__ __forceinline__ void load_channels(const float* p, float none, int c0, int C, float* out) {
#pragma unroll
  for (int j = 0; j < N; ++j) out[j] = p != nullptr ? p[min(c0 + j, C - 1)] : none;
}
template <int N>
__device__ __forceinline__ void load_groups(const float* p, const NormGeom& g, int b, int c0, float* out) {
#pragma unroll
  for (int j = 0; j < N; ++j) out[j] = p[(int64_t)b * g.G + fdiv((uint32_t)min(c0 + j, g.C - 1), g.d_cg)];
}

// Forward, statistics of a tile: (m, r / n, q, n) of each piece (q channels of one vector).
template <typename T, int NS>
__global__ __launch_bounds__(kThreads) void gn_stats_kernel(const NormArgs a) {
  constexpr int N = ActVec<T>::N, Q = N / NS;
  __shared__ float shared[kWaves * 64 * NS];
  const NormGeom& g = a.g;
  const Tile w = my_tile(g);
  u32x4_t v[kI];
  load_tile<T>(w, g, a.x, a.xcs, a.xco, v);
  float s[NS] = {}, m[NS], r[NS] = {}, q[NS] = {};
#pragma unroll
  for (int i = 0; i < kI; ++i) {
    float f[N];
    ActVec<T>::unpack(v[i], f);
#pragma unroll
    for (int j = 0; j < N; ++j) s[j / Q] += i < w.n ? f[j] : 0.f;
  }
  tile_sum<NS>(s, g, shared);
  const float n = (float)w.count * Q;
  const int lane = threadIdx.x & (g.lanes - 1);
#pragma unroll
  for (int j = 0; j < NS; ++j) m[j] = shared[lane * NS + j] / n;
#pragma unroll
  for (int i = 0; i < kI; ++i) {
    float f[N];
    ActVec<T>::unpack(v[i], f);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float d = i < w.n ? f[j] - m[j / Q] : 0.f;
      r[j / Q] += d;
      q[j / Q] = fmaf(d, d, q[j / Q]);
    }
  }
  tile_sum<NS>(r, g, shared);
#pragma unroll
  for (int j = 0; j < NS; ++j) r[j] = shared[lane * NS + j];
  tile_sum<NS>(q, g, shared);
  if ((int)threadIdx.x < g.lanes && w.live) {
    float4* out = (float4*)a.part + (((int64_t)w.b * g.tiles + w.t) * g.nv + w.v) * NS;
#pragma unroll
    for (int j = 0; j < NS; ++j) out[j] = make_float4(m[j], r[j] / n, shared[lane * NS + j], n);
  }
}
// One wave joins the tiles and pieces of a group.  Piece k of an image's tile covers channels k*q .. k*q + q - 1.
__global__ __launch_bounds__(64) void gn_join_kernel(const NormArgs a) {
  const NormGeom& g = a.g;
  const int b = blockIdx.x / g.G, gi = blockIdx.x - b * g.G;
  const int ppg = g.cg / g.q, per_image = g.nv * g.n_slots;
  const int items = g.tiles * ppg;
  const float4* part = (const float4*)a.part + (int64_t)b * g.tiles * per_image + gi * ppg;
  const double n_total = (double)g.P * g.cg;
  double s = 0.0, m2 = 0.0;
  for (int k = threadIdx.x; k < items; k += 64) {
    const int t = k / ppg;
    const float4 p = part[(int64_t)t * per_image + (k - t * ppg)];
    s += (double)p.w * ((double)p.x + (double)p.y);
  }
  const double mean = wave_total(s) / n_total;
  for (int k = threadIdx.x; k < items; k += 64) {
    const int t = k / ppg;
    const float4 p = part[(int64_t)t * per_image + (k - t * ppg)];
    const double d = (double)p.x + (double)p.y - mean;
    m2 += (double)p.z + (double)p.w * (d * d - (double)p.y * (double)p.y);
  }
  double var = wave_total(m2) / n_total;
  var = var < 0.0 ? 0.0 : var;                                   // a NaN stays
  if (threadIdx.x == 0) {
    a.mean[blockIdx.x] = (float)mean;
    a.rstd[blockIdx.x] = (float)(1.0 / sqrt(var + (double)a.eps));
  }
}
template <typename T>
__global__ __launch_bounds__(kThreads) void gn_apply_kernel(const NormArgs a) {
  constexpr int N = ActVec<T>::N;
  const NormGeom& g = a.g;
  const Tile w = my_tile(g);
  const int c0 = w.v * N;
  u32x4_t v[kI];
  load_tile<T>(w, g, a.x, a.xcs, a.xco, v);
  float mean[N], rstd[N], gamma[N], beta[N];
  load_groups<N>(a.mean, g, w.b, c0, mean);
  load_groups<N>(a.rstd, g, w.b, c0, rstd);
  load_channels<N>(a.gamma, 1.f, c0, g.C, gamma);
  load_channels<N>(a.beta, 0.f, c0, g.C, beta);
  const uint64_t offset = a.drop.on ? drop_offset(a.drop) : 0;
  T* out = (T*)a.out + (int64_t)w.b * g.P * a.ocs + a.oco + c0;
  uint32_t bits = 0xff;
  if (a.drop.on && a.drop.per_channel) bits = drop_bits<N>(a.drop, offset, (uint64_t)w.b * (g.nv * N) + c0);
#pragma unroll
  for (int i = 0; i < kI; ++i) {
    const int p = w.row + i * g.rows;
    float f[N];
    ActVec<T>::unpack(v[i], f);
    if (a.drop.on && !a.drop.per_channel) bits = drop_bits<N>(a.drop, offset, ((uint64_t)w.b * g.P + p) * (uint32_t)(g.nv * N) + c0);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      f[j] = act_value<T>(fmaf((f[j] - mean[j]) * rstd[j], gamma[j], beta[j]), a.act);
      if (a.drop.on) f[j] = bits >> j & 1 ? f[j] * a.drop.scale : 0.f;
      if (c0 + j >= g.C) f[j] = 0.f;
    }
    if (w.live && i < w.n) store_stream(out + (int64_t)p * a.ocs, ActVec<T>::pack(f));
  }
}

// ---------------------------------------------------------------- backward
// h and dz of one vector.  ReLU's gate is a border: where z came out smaller than its rounding can be
// (2^-20 |beta|: z = h * gamma + beta, so a small z has |h * gamma| ~ |beta|) its sign is taken from 64 bits.
template <typename T, int N>
__device__ __forceinline__ void norm_dz(const NormArgs& a, const float* x, const float* dy, const float* mean, const float* rstd,
                                        const float* gamma, const float* beta, uint32_t bits, float* h, float* dz) {
#pragma unroll
  for (int j = 0; j < N; ++j) {
    h[j] = (x[j] - mean[j]) * rstd[j];
    float z = fmaf(h[j], gamma[j], beta[j]);
    if (a.act == MI_ACT_RELU && fabsf(z) < fabsf(beta[j]) * 0x1p-20f)
      z = (float)(((double)x[j] - (double)mean[j]) * (double)rstd[j] * (double)gamma[j] + (double)beta[j]);
    float d = dy[j];
    if (a.drop.on) d = bits >> j & 1 ? d * a.drop.scale : 0.f;
    dz[j] = a.act == MI_ACT_RELU ? (z > 0.f ? d : 0.f) : d * act_slope<T>(z, a.act);
  }
}
template <typename T>
struct NormChannels {
  static constexpr int N = ActVec<T>::N;
  float mean[N], rstd[N], gamma[N], beta[N];
  __device__ __forceinline__ void load(const NormArgs& a, int b, int c0) {
    load_groups<N>(a.mean, a.g, b, c0, mean);
    load_groups<N>(a.rstd, a.g, b, c0, rstd);
    load_channels<N>(a.gamma, 1.f, c0, a.g.C, gamma);
    load_channels<N>(a.beta, 0.f, c0, a.g.C, beta);
  }
};
template <typename T>
__global__ __launch_bounds__(kThreads) void gn_bwd_sums_kernel(const NormArgs a) {
  constexpr int N = ActVec<T>::N;
  __shared__ float shared[kWaves * 64 * N];
  const NormGeom& g = a.g;
  const Tile w = my_tile(g);
  const int c0 = w.v * N;
  u32x4_t vx[kI], vd[kI];
  load_tile<T>(w, g, a.x, a.xcs, a.xco, vx);
  load_tile<T>(w, g, a.dy, a.ycs, a.yco, vd);
  NormChannels<T> ch;
  ch.load(a, w.b, c0);
  const uint64_t offset = a.drop.on ? drop_offset(a.drop) : 0;
  uint32_t bits = 0xff;
  if (a.drop.on && a.drop.per_channel) bits = drop_bits<N>(a.drop, offset, (uint64_t)w.b * (g.nv * N) + c0);
  float sa[N] = {}, sq[N] = {};
#pragma unroll
  for (int i = 0; i < kI; ++i) {
    float x[N], dy[N], h[N], dz[N];
    ActVec<T>::unpack(vx[i], x);
    ActVec<T>::unpack(vd[i], dy);
    if (a.drop.on && !a.drop.per_channel)
      bits = drop_bits<N>(a.drop, offset, ((uint64_t)w.b * g.P + w.row + i * g.rows) * (uint32_t)(g.nv * N) + c0);
    norm_dz<T, N>(a, x, dy, ch.mean, ch.rstd, ch.gamma, ch.beta, bits, h, dz);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float d = i < w.n ? dz[j] : 0.f, e = i < w.n ? dz[j] * h[j] : 0.f;
      sa[j] += d;
      sq[j] += e;
    }
  }
  const int lane = threadIdx.x & (g.lanes - 1);
  tile_sum<N>(sa, g, shared);
#pragma unroll
  for (int j = 0; j < N; ++j) sa[j] = shared[lane * N + j];
  tile_sum<N>(sq, g, shared);
  if ((int)threadIdx.x < g.lanes && w.live) {
    float2* out = a.part + (((int64_t)w.b * g.tiles + w.t) * g.nv + w.v) * N;
#pragma unroll
    for (int j = 0; j < N; ++j) out[j] = make_float2(sa[j], shared[lane * N + j]);
  }
}
// One wave per (image, group): the image's sums of each channel, and the group's two means.
__global__ __launch_bounds__(64) void gn_bwd_join_kernel(const NormArgs a, int padded) {
  const NormGeom& g = a.g;
  const int b = blockIdx.x / g.G, gi = blockIdx.x - b * g.G;
  float m1 = 0.f, m2 = 0.f;
  for (int k = threadIdx.x; k < g.cg; k += 64) {
    const int c = gi * g.cg + k;
    const float2* part = a.part + (int64_t)b * g.tiles * padded + c;
    float2 s = make_float2(0.f, 0.f);
    for (int t = 0; t < g.tiles; ++t) {
      const float2 p = part[(int64_t)t * padded];
      s.x += p.x;
      s.y += p.y;
    }
    a.chan[(int64_t)b * g.C + c] = s;
    const float gamma = a.gamma != nullptr ? a.gamma[c] : 1.f;
    m1 = fmaf(gamma, s.x, m1);
    m2 = fmaf(gamma, s.y, m2);
  }
  m1 = wave_total(m1);
  m2 = wave_total(m2);
  const float n = (float)g.P * (float)g.cg;
  if (threadIdx.x == 0) a.moments[blockIdx.x] = make_float2(m1 / n, m2 / n);
}
template <typename T>
__global__ __launch_bounds__(kThreads) void gn_bwd_apply_kernel(const NormArgs a) {
  constexpr int N = ActVec<T>::N;
  const NormGeom& g = a.g;
  const Tile w = my_tile(g);
  const int c0 = w.v * N;
  u32x4_t vx[kI], vd[kI];
  load_tile<T>(w, g, a.x, a.xcs, a.xco, vx);
  load_tile<T>(w, g, a.dy, a.ycs, a.yco, vd);
  NormChannels<T> ch;
  ch.load(a, w.b, c0);
  float m1[N], m2[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const float2 m = a.moments[(int64_t)w.b * g.G + fdiv((uint32_t)min(c0 + j, g.C - 1), g.d_cg)];
    m1[j] = m.x;
    m2[j] = m.y;
  }
  const uint64_t offset = a.drop.on ? drop_offset(a.drop) : 0;
  uint32_t bits = 0xff;
  if (a.drop.on && a.drop.per_channel) bits = drop_bits<N>(a.drop, offset, (uint64_t)w.b * (g.nv * N) + c0);
  T* out = (T*)a.out + (int64_t)w.b * g.P * a.ocs + a.oco + c0;
#pragma unroll
  for (int i = 0; i < kI; ++i) {
    const int p = w.row + i * g.rows;
    float x[N], dy[N], h[N], dz[N], dx[N];
    ActVec<T>::unpack(vx[i], x);
    ActVec<T>::unpack(vd[i], dy);
    if (a.drop.on && !a.drop.per_channel) bits = drop_bits<N>(a.drop, offset, ((uint64_t)w.b * g.P + p) * (uint32_t)(g.nv * N) + c0);
    norm_dz<T, N>(a, x, dy, ch.mean, ch.rstd, ch.gamma, ch.beta, bits, h, dz);
#pragma unroll
    for (int j = 0; j < N; ++j) {
#pragma clang fp contract(off)   // t is rounded before the subtraction, as it was in the sum: a group of one value gives exactly zero
      const float t = ch.gamma[j] * dz[j];
      dx[j] = c0 + j < g.C ? ch.rstd[j] * (t - m1[j] - h[j] * m2[j]) : 0.f;
    }
    if (w.live && i < w.n) store_stream(out + (int64_t)p * a.ocs, ActVec<T>::pack(dx));
  }
}
// Sums over the images in a fixed order: a workgroup takes 8 channels, 32 threads share a channel's images.
__global__ __launch_bounds__(256) void gn_param_grads_kernel(const NormArgs a) {
  __shared__ float2 shared[256];
  const int k = threadIdx.x & 7, r = threadIdx.x >> 3, c = blockIdx.x * 8 + k;
  float2 s = make_float2(0.f, 0.f);
  if (c < a.g.C)
    for (int b = r; b < a.g.B; b += 32) {
      const float2 p = a.chan[(int64_t)b * a.g.C + c];
      s.x += p.x;
      s.y += p.y;
    }
  shared[threadIdx.x] = s;
  __syncthreads();
  if (r == 0 && c < a.g.C) {
    for (int i = 1; i < 32; ++i) {
      s.x += shared[i * 8 + k].x;
      s.y += shared[i * 8 + k].y;
    }
    if (a.dgamma) a.dgamma[c] = a.ga * s.y + (a.gb != 0.f ? a.gb * a.dgamma[c] : 0.f);
    if (a.dbeta) a.dbeta[c] = a.ga * s.x + (a.gb != 0.f ? a.gb * a.dbeta[c] : 0.f);
  }
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
  g.n_slots = N / g.q;
  g.d_tiles = make_fastdiv(g.tiles);
  g.d_chunks = make_fastdiv(g.chunks);
  g.d_cg = make_fastdiv(g.cg);
  return g;
}
static size_t fwd_part_bytes(const NormGeom& g) { return (size_t)g.B * g.tiles * g.nv * g.n_slots * sizeof(float4); }
static size_t bwd_part_bytes(const NormGeom& g, int dtype) {
  return (size_t)g.B * g.tiles * g.nv * (dtype == MI_BF16 ? 8 : 4) * sizeof(float2);
}
size_t group_norm_ws_bytes(int B, int H, int W, int C, int G, int backward, int dtype) {
  const NormGeom g = norm_geom(B, H, W, C, G, dtype);
  if (!backward) return fwd_part_bytes(g) + 16;
  return bwd_part_bytes(g, dtype) + ((size_t)B * C + (size_t)B * G) * sizeof(float2) + 16;
}

template <typename T>
static int launch_fwd(const NormArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)(a.g.B * a.g.tiles * a.g.chunks)), block(kThreads);
  switch (a.g.n_slots) {
    case 1: hipLaunchKernelGGL((gn_stats_kernel<T, 1>), grid, block, 0, s, a); break;
    case 2: hipLaunchKernelGGL((gn_stats_kernel<T, 2>), grid, block, 0, s, a); break;
    case 4: hipLaunchKernelGGL((gn_stats_kernel<T, 4>), grid, block, 0, s, a); break;
    default: hipLaunchKernelGGL((gn_stats_kernel<T, ActVec<T>::N>), grid, block, 0, s, a); break;
  }
  hipLaunchKernelGGL(gn_join_kernel, dim3(a.g.B * a.g.G), dim3(64), 0, s, a);
  hipLaunchKernelGGL((gn_apply_kernel<T>), grid, block, 0, s, a);
  return check_hip(hipGetLastError(), "group_norm_act_fwd");
}
static int check_range(const NormGeom& g, const char* what) {
  MI_REQUIRE((int64_t)g.B * g.P < (1ll << 31) && (int64_t)g.B * g.G < (1ll << 31) &&
                 (int64_t)g.B * g.tiles * g.chunks < (1ll << 31), std::string(what) + ": tensor too large");
  return MI_OK;
}
int launch_group_norm_fwd(const void* x, int xcs, int xco, const float* gamma, const float* beta, void* y, int ycs, int yco,
                          float* mean, float* rstd, int B, int H, int W, int C, int G, int act, float eps,
                          const mi_dropout* drop, void* ws, size_t ws_bytes, int dtype, hipStream_t s) {
  NormArgs a{};
  int rc = make_drop_args(drop, &a.drop);
  if (rc) return rc;
  a.g = norm_geom(B, H, W, C, G, dtype);
  if ((rc = check_range(a.g, "group_norm_act_fwd"))) return rc;
  if (B == 0) return MI_OK;
  if (ws_bytes < group_norm_ws_bytes(B, H, W, C, G, 0, dtype)) return fail(MI_ESIZE, "group_norm_act_fwd: workspace too small");
  a.x = x; a.xcs = xcs; a.xco = xco;
  a.out = y; a.ocs = ycs; a.oco = yco;
  a.gamma = gamma; a.beta = beta; a.mean = mean; a.rstd = rstd;
  a.act = act; a.eps = eps;
  a.part = (float2*)ws;
  return dtype == MI_BF16 ? launch_fwd<__bf16>(a, s) : launch_fwd<float>(a, s);
}
template <typename T>
static int launch_bwd(const NormArgs& a, hipStream_t s) {
  if (a.g.B > 0) {
    const dim3 grid((unsigned)(a.g.B * a.g.tiles * a.g.chunks)), block(kThreads);
    hipLaunchKernelGGL((gn_bwd_sums_kernel<T>), grid, block, 0, s, a);
    hipLaunchKernelGGL(gn_bwd_join_kernel, dim3(a.g.B * a.g.G), dim3(64), 0, s, a, a.g.nv * ActVec<T>::N);
    hipLaunchKernelGGL((gn_bwd_apply_kernel<T>), grid, block, 0, s, a);
  }
  if (a.dgamma || a.dbeta) hipLaunchKernelGGL(gn_param_grads_kernel, dim3((a.g.C + 7) / 8), dim3(256), 0, s, a);
  return check_hip(hipGetLastError(), "group_norm_act_bwd");
}
int launch_group_norm_bwd(const void* x, int xcs, int xco, const void* dy, int ycs, int yco, const float* gamma, const float* beta,
                          const float* mean, const float* rstd, void* dx, int dcs, int dco, float* dgamma, float* dbeta,
                          float ga, float gb, int B, int H, int W, int C, int G, int act, const mi_dropout* drop, void* ws,
                          size_t ws_bytes, int dtype, hipStream_t s) {
  NormArgs a{};
  int rc = make_drop_args(drop, &a.drop);
  if (rc) return rc;
  a.g = norm_geom(B, H, W, C, G, dtype);
  if ((rc = check_range(a.g, "group_norm_act_bwd"))) return rc;
  if (ws_bytes < group_norm_ws_bytes(B, H, W, C, G, 1, dtype)) return fail(MI_ESIZE, "group_norm_act_bwd: workspace too small");
  a.x = x; a.xcs = xcs; a.xco = xco;
  a.dy = dy; a.ycs = ycs; a.yco = yco;
  a.out = dx; a.ocs = dcs; a.oco = dco;
  a.gamma = gamma; a.beta = beta; a.mean = const_cast<float*>(mean); a.rstd = const_cast<float*>(rstd);
  a.act = act;
  a.part = (float2*)ws;
  a.chan = a.part + bwd_part_bytes(a.g, dtype) / sizeof(float2);
  a.moments = a.chan + (size_t)B * C;
  a.dgamma = dgamma; a.dbeta = dbeta; a.ga = ga; a.gb = gb;
  return dtype == MI_BF16 ? launch_bwd<__bf16>(a, s) : launch_bwd<float>(a, s);
}

}  // namespace mi
