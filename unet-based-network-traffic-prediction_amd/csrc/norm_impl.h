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
#pragma once
#include "drop.h"

#include <type_traits>

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
  uint64_t* words;                     // what the parts of an image tell each other
  DropArgs drop;
};

template <typename F> __device__ __forceinline__ F wave_total(F v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// ---------------------------------------------------------------- activations
// exp through the hardware's 2^x: the argument's rounding, |v| 2^-24 relative, enters z * sigmoid(z) and Phi(z) only
// where it meets a factor that falls faster than |v| grows (z^2 s (1 - s) < 0.5, z^2 exp(-z^2 / 2) < 0.75).
__device__ __forceinline__ float exp_fast(float v) { return __builtin_amdgcn_exp2f(v * 1.44269504f); }
__device__ __forceinline__ float sigmoid_fast(float z) { return __builtin_amdgcn_rcpf(1.f + exp_fast(-z)); }
// Phi(z) and exp(-z^2 / 2).  erf by formula 7.1.26 of Abramowitz and Stegun, "Handbook of Mathematical Functions"
// (error at most 1.5e-7, 2.5 half steps of fp32 at 1): its exponential is the Gaussian that the slope needs.
__device__ __forceinline__ float normal_cdf(float z, float* gauss) {
  const float x = fabsf(z) * 0.70710678f, t = __builtin_amdgcn_rcpf(fmaf(0.3275911f, x, 1.f)), e = exp_fast(-0.5f * z * z);
  float p = fmaf(1.061405429f, t, -1.453152027f);
  p = fmaf(p, t, 1.421413741f);
  p = fmaf(p, t, -0.284496736f);
  p = fmaf(p, t, 0.254829592f);
  const float tail = 0.5f * p * t * e;                           // 1 - Phi(|z|)
  *gauss = e;
  return z >= 0.f ? 1.f - tail : tail;
}
template <int ACT> __device__ __forceinline__ float act_value(float z) {
  if constexpr (ACT == MI_ACT_RELU) return __builtin_elementwise_maximum(z, 0.f);   // a NaN stays one
  if constexpr (ACT == MI_ACT_SILU) return z * sigmoid_fast(z);
  if constexpr (ACT == MI_ACT_GELU) {
    float e;
    return z * normal_cdf(z, &e);
  }
  return z;
}
template <int ACT> __device__ __forceinline__ float act_slope(float z) {
  if constexpr (ACT == MI_ACT_RELU) return z > 0.f ? 1.f : 0.f;
  if constexpr (ACT == MI_ACT_SILU) {
    const float s = sigmoid_fast(z);
    return fmaf(z * s, 1.f - s, s);
  }
  if constexpr (ACT == MI_ACT_GELU) {
    float e;
    const float phi = normal_cdf(z, &e);
    return fmaf(z * 0.39894228f, e, phi);
  }
  return 1.f;
}
// The activation code is uniform: one branch per tile, not per value.
#define MI_FOR_ACT(act, CALL)              \
  switch (act) {                           \
    case MI_ACT_RELU: CALL(MI_ACT_RELU); break; \
    case MI_ACT_SILU: CALL(MI_ACT_SILU); break; \
    case MI_ACT_GELU: CALL(MI_ACT_GELU); break; \
    default: CALL(MI_ACT_NONE); break;     \
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
  if (p == nullptr) {
#pragma unroll
    for (int j = 0; j < N; ++j) out[j] = none;
  } else if (C % N == 0 && ((uintptr_t)p & 15) == 0) {           // (a padding vector takes the last one's)
    const float4* q = (const float4*)(p + min(c0, C - N));
#pragma unroll
    for (int j = 0; j < N; j += 4) {
      const float4 f = q[j / 4];
      out[j] = f.x; out[j + 1] = f.y; out[j + 2] = f.z; out[j + 3] = f.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) out[j] = p[min(c0 + j, C - 1)];
  }
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
template <typename T, int ACT>
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
  KeepBits<1, N> keep;
  keep.keep_all();
  if (a.drop.on && a.drop.per_channel) keep.add(0, a.drop, offset, (uint64_t)w.b * (g.nv * N) + c0);
#pragma unroll
  for (int i = 0; i < kI; ++i) {
    const int p = w.row + i * g.rows;
    float f[N];
    ActVec<T>::unpack(v[i], f);
    if (a.drop.on && !a.drop.per_channel) keep.add(0, a.drop, offset, ((uint64_t)w.b * g.P + p) * (uint32_t)(g.nv * N) + c0);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      f[j] = act_value<ACT>(fmaf((f[j] - mean[j]) * rstd[j], gamma[j], beta[j]));
      if (a.drop.on) f[j] = keep.kept(0, j, f[j] * a.drop.scale);
      if (c0 + j >= g.C) f[j] = 0.f;
    }
    if (w.live && i < w.n) store_stream(out + (int64_t)p * a.ocs, ActVec<T>::pack(f));
  }
}

// ---------------------------------------------------------------- slabs: one read of x
// A workgroup's registers hold its part of an image -- all of it, or `parts` workgroups share it --, so x is read once:
// its I vectors per thread stay where they are while the sums are formed, and are normalised from there.  A second
// reading would cost as much as the first (the memory-side cache delivers 6.8 TB/s, HBM 6.2), and the join and apply
// launches ~3 us each, on the host as on the device.
//
// A workgroup owns `nb` images x cv vectors.  Its threads are (image, row, lane): lanes lie along the channels, tpi
// threads share an image.  A group's sum goes over the rows and lanes of a wave by shuffles and over waves through LDS.
struct Slab {
  int cv;                      // vectors per pixel of a chunk: whole groups
  int lanes, log_lanes;        // power of two >= cv, at most 64
  int chunks;
  int tpi, log_tpi;            // threads per image, a power of two >= lanes
  int nb, img_blocks;          // images per workgroup, workgroups along the images
  int rows;                    // tpi / lanes
  int parts, log_parts;        // workgroups that share an image (then nb = 1); rounded up to a power of two
  int merge;                   // lanes of a group that shuffles can sum (a power of two), ...
  int left;                    // ... and what then remains: pieces per group / merge
  int threads, iters;          // nb * tpi, pixels per thread
  int by_xcd;                  // chunks of an image go to one XCD: they share the lines that its L2 holds
  int polls;                   // how often a part is looked for before its sums are formed here instead
  FastDiv d_chunks, d_parts;
};
struct SlabThread {
  int tin, slot, lane, row;    // thread of its image, image of the workgroup, vector of the chunk, row of pixels
  int b, v, part, chunk;       // image, vector
  bool live;
};
__device__ __forceinline__ SlabThread slab_thread(const NormGeom& g, const Slab& s) {
  SlabThread t;
  uint32_t i = blockIdx.x, ib;
  if (s.by_xcd) {                                                // workgroup i runs on XCD i % 8
    const uint32_t j = i >> 3, q = fdiv(j, s.d_chunks);
    t.chunk = (int)(j - q * s.chunks);
    ib = q * 8 + (i & 7);
    t.part = 0;
  } else {
    const uint32_t q = fdiv(i, s.d_chunks);
    t.chunk = (int)(i - q * s.chunks);
    ib = fdiv(q, s.d_parts);
    t.part = (int)(q - ib * s.parts);
  }
  const int tid = threadIdx.x;
  t.slot = tid >> s.log_tpi;
  t.tin = tid & (s.tpi - 1);
  t.lane = t.tin & (s.lanes - 1);
  t.row = t.tin >> s.log_lanes;
  t.b = (int)ib * s.nb + t.slot;
  t.v = t.chunk * s.cv + t.lane;
  t.live = t.slot < s.nb && t.b < g.B && t.lane < s.cv && t.v < g.nv;
  t.b = min(t.b, g.B - 1);
  t.v = min(t.v, g.nv - 1);
  return t;
}
// The pixels of a part: first, how many there are, how many of them are this thread's.
struct SlabPixels { int first, count, mine; bool full; };
template <int I>
__device__ __forceinline__ SlabPixels slab_pixels(const SlabThread& t, const NormGeom& g, const Slab& s, int part) {
  SlabPixels p;
  p.first = part * s.rows * I;
  p.count = min(g.P - p.first, s.rows * I);
  p.mine = t.row < p.count ? (p.count - t.row + s.rows - 1) / s.rows : 0;
  p.full = p.count == s.rows * I;
  return p;
}
// Loads are unconditional (a pixel behind the part reads the image's last one instead); what they bring in is zeroed.
template <typename T, int I>
__device__ __forceinline__ void load_slab(const SlabThread& t, const SlabPixels& px, const NormGeom& g, const Slab& s, const void* base,
                                          int cs, int co, u32x4_t (&v)[I]) {
  const T* p = (const T*)base + (int64_t)t.b * g.P * cs + co + t.v * ActVec<T>::N;
#pragma unroll
  for (int i = 0; i < I; ++i) v[i] = load_stream(p + (int64_t)min(px.first + t.row + i * s.rows, g.P - 1) * cs);
}
template <int I> __device__ __forceinline__ void zero_missing(const SlabPixels& px, u32x4_t (&v)[I]) {
  if (px.full) return;
#pragma unroll
  for (int i = 0; i < I; ++i) v[i] = i < px.mine ? v[i] : u32x4_t{0, 0, 0, 0};
}
// Ends the lifetime of values unpacked from v: without it the compiler keeps all N * I of them from one use to the next
// (bf16: twice the registers of v itself) instead of unpacking again.
template <int I> __device__ __forceinline__ void repack(u32x4_t (&v)[I]) {
#pragma unroll
  for (int i = 0; i < I; ++i) asm volatile("" : "+v"(v[i]));
}
// K sums over each group of each image: in, a thread's K x NS partial sums (of its vector's pieces); out, the sums of the
// groups that its pieces belong to.  `shared`: as much as slab_shared says; free to use again after a barrier.
template <int NS, int K>
__device__ __forceinline__ void slab_sum(float (&v)[K][NS], const NormGeom& g, const Slab& s, const SlabThread& t, float* shared) {
  for (int o = min(64, s.tpi) >> 1; o >= s.lanes; o >>= 1) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < NS; ++j) v[k][j] += __shfl_xor(v[k][j], o, 64);
  }
  for (int o = s.merge >> 1; o > 0; o >>= 1) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < NS; ++j) v[k][j] += __shfl_xor(v[k][j], o, 64);
  }
  if (s.tpi <= 64 && s.left == 1) return;
  const int per = s.lanes * NS * K, tid = threadIdx.x;
  const int segs = s.tpi > 64 ? s.tpi >> 6 : 1;                  // segments (waves, or parts of one) of an image
  const int seg = s.tpi > 64 ? tid >> 6 : t.slot;
  if ((tid & (min(64, s.tpi) - 1)) < s.lanes) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < NS; ++j) shared[seg * per + (k * s.lanes + t.lane) * NS + j] = v[k][j];
  }
  __syncthreads();
  float* mine = shared + t.slot * segs * per;
  if (segs > 1) {
    for (int i = t.tin; i < per; i += s.tpi) {
      float sum = 0.f;
      for (int w = 0; w < segs; ++w) sum += mine[w * per + i];
      mine[i] = sum;                                             // entry i belongs to this thread
    }
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    int first = t.lane * NS + j;
    if (s.left > 1) {                                            // the first piece of this piece's group, within the chunk
      const int c = min((t.chunk * s.cv + t.lane) * (NS * g.q) + j * g.q, g.C - 1);
      first = ((int)fdiv((uint32_t)c, g.d_cg) * g.cg) / g.q - t.chunk * s.cv * NS;
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float sum = 0.f;
      for (int i = 0; i < s.left; ++i) sum += mine[k * s.lanes * NS + first + i];
      v[k][j] = sum;
    }
  }
}
// Sum and sum of squares of a thread's vectors, per piece.
template <int NS, int I>
__device__ __forceinline__ void power_sums(const u32x4_t (&v)[I], float (&s)[2][NS], float) {
#pragma unroll
  for (int i = 0; i < I; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float f = __uint_as_float(v[i][j]);
      s[0][j * NS / 4] += f;
      s[1][j * NS / 4] = fmaf(f, f, s[1][j * NS / 4]);
    }
}
// bf16: two products and the sum in one instruction, products exact, accumulated in fp32, nothing to unpack
template <int NS, int I>
__device__ __forceinline__ void power_sums(const u32x4_t (&v)[I], float (&s)[2][NS], __bf16) {
  typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int i = 0; i < I; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (NS == 8) {
        const float lo = __uint_as_float(v[i][j] << 16), hi = __uint_as_float(v[i][j] & 0xffff0000u);
        s[0][2 * j] += lo;
        s[0][2 * j + 1] += hi;
        s[1][2 * j] = fmaf(lo, lo, s[1][2 * j]);
        s[1][2 * j + 1] = fmaf(hi, hi, s[1][2 * j + 1]);
      } else {
        const bf16x2_t x = __builtin_bit_cast(bf16x2_t, (uint32_t)v[i][j]), one = __builtin_bit_cast(bf16x2_t, 0x3f803f80u);
        s[0][j * NS / 4] = __builtin_amdgcn_fdot2_f32_bf16(x, one, s[0][j * NS / 4], false);
        s[1][j * NS / 4] = __builtin_amdgcn_fdot2_f32_bf16(x, x, s[1][j * NS / 4], false);
      }
    }
}
// Mean (as m + e, m rounded) and squared deviations of the groups over a part.  Sums of x and x^2 first: they do where
// the deviations are not small against the values, 4 q >= sum x^2 -- what is lost then are two bits.  Groups further from
// zero take the corrected two-pass form from the registers.  Which of the two is decided for each group by its own values.
template <typename T, int NS, int I>
__device__ __forceinline__ void slab_moments(u32x4_t (&v)[I], const SlabPixels& px, const NormGeom& g, const Slab& s, const SlabThread& t,
                                             float* shared, float* m, float* e, float* q) {
  constexpr int N = ActVec<T>::N, Q = N / NS;
  const float n = (float)px.count * (float)g.cg, inv = 1.f / n;
  float sum[2][NS] = {};
  power_sums<NS, I>(v, sum, T());
  slab_sum<NS, 2>(sum, g, s, t, shared);
  bool far = false;
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    m[j] = sum[0][j] * inv;
    e[j] = 0.f;
    q[j] = fmaf(-m[j], sum[0][j], sum[1][j]);
    far = far || !(4.f * q[j] >= sum[1][j]);
  }
  if (__syncthreads_or(far && t.live)) {
    repack(v);
    float dev[2][NS] = {};
#pragma unroll
    for (int i = 0; i < I; ++i) {
      float f[N];
      ActVec<T>::unpack(v[i], f);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float d = i < px.mine ? f[j] - m[j / Q] : 0.f;
        dev[0][j / Q] += d;
        dev[1][j / Q] = fmaf(d, d, dev[1][j / Q]);
      }
    }
    slab_sum<NS, 2>(dev, g, s, t, shared);
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      if (4.f * q[j] >= sum[1][j]) continue;
      e[j] = dev[0][j] * inv;
      q[j] = fmaf(-e[j], dev[0][j], dev[1][j]);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------- parts of an image
// Each workgroup of an image publishes its part's sums for the others, two 64-bit words per (image, part, group), and
// takes the sums of all parts in one order, so all get the same bits.  A word is valid as soon as it is not kEmpty,
// which the words are filled with before the launch and which no sum can be: there is nothing else to wait for, and
// plain device-scope loads and stores do (a release would write the whole L2 back).
// A part may take long to come -- its workgroup may not run yet, or never at the same time as this one.  No workgroup
// depends on that: after `polls` looks it forms a missing part's sums itself (the same operations in the same order)
// and publishes them, so every wait ends.
constexpr uint64_t kEmpty = ~0ull;
__device__ __forceinline__ void put_word(uint64_t* p, uint64_t w) { __hip_atomic_store(p, w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ uint64_t get_word(const uint64_t* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// Runs `take(group of the chunk, present, word 0, word 1)` for every (group, part) of the workgroup's image with lane
// % 2^log_parts = part, once all parts are there.  Returns the number of a missing part, or -1.
template <typename F>
__device__ __forceinline__ int slab_collect(const uint64_t* words, const NormGeom& g, const Slab& s, const SlabThread& t, int groups,
                                            int* missing, F take) {
  const int tid = threadIdx.x, lane = tid & 63, per_wave = 64 >> s.log_parts;
  if (tid == 0) *missing = -1;
  __syncthreads();
  const int part = lane & ((1 << s.log_parts) - 1);
  for (int k = (tid >> 6) * per_wave; k < groups; k += (s.threads >> 6) * per_wave) {
    const int group = k + (lane >> s.log_parts);
    const bool needed = part < s.parts && group < groups;
    const uint64_t* w = words + 2 * ((int64_t)min(part, s.parts - 1) * g.G + min(group, groups - 1));
    uint64_t a = kEmpty, b = kEmpty;
    for (int i = 0;; ++i) {
      a = get_word(w);
      b = get_word(w + 1);
      const bool there = !needed || (a != kEmpty && b != kEmpty);
      if (__all(there)) break;
      if (i >= s.polls) {
        if (!there) atomicMax(missing, part);
        break;
      }
      __builtin_amdgcn_s_sleep(1);
    }
    take(group, needed, a, b);
  }
  __syncthreads();
  const int result = *missing;
  __syncthreads();
  return result;
}
// Where the groups' results lie in LDS: behind the 2 * NS sums of slab_sum (parts > 1: one image, all its threads).
template <int NS> __device__ __forceinline__ int slab_stats_at(const Slab& s) {
  return s.tpi <= 64 && s.left == 1 ? 0 : ((s.threads + 63) >> 6) * s.lanes * 2 * NS;
}
// Sum over the lanes that hold the parts of one group.
__device__ __forceinline__ double parts_total(double v, const Slab& s) {
  for (int o = (1 << s.log_parts) >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// Two workgroups a CU (128 registers): one loads or stores while the other sums.  (Eight pieces per vector with parts
// need more; groups of odd channel counts in large images run one workgroup a CU.)
template <typename T, int NS, int I, bool PARTS>
__global__ __launch_bounds__(512, PARTS && NS > 2 ? 2 : 4) void gn_fwd_slab_kernel(const NormArgs a, const Slab s) {
  constexpr int N = ActVec<T>::N, Q = N / NS;
  extern __shared__ float shared[];
  const NormGeom& g = a.g;
  const SlabThread t = slab_thread(g, s);
  const int c0 = t.v * N;
  SlabPixels px = slab_pixels<I>(t, g, s, t.part);
  u32x4_t v[I];
  load_slab<T, I>(t, px, g, s, a.x, a.xcs, a.xco, v);
  float gamma[N], beta[N];
  if constexpr (!PARTS) {
    load_channels<N>(a.gamma, 1.f, c0, g.C, gamma);
    load_channels<N>(a.beta, 0.f, c0, g.C, beta);
  }
  KeepBits<I, N> keep;                                           // while the loads are in flight
  if (a.drop.on) {
    const uint64_t offset = drop_offset(a.drop);
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const uint64_t row = a.drop.per_channel ? (uint64_t)t.b : (uint64_t)t.b * g.P + (px.first + t.row + i * s.rows);
      keep.add(i, a.drop, offset, row * (uint32_t)(g.nv * N) + c0);
    }
  }
  zero_missing(px, v);
  float mean[NS], rstd[NS], e[NS], q[NS];
  if constexpr (!PARTS) {
    slab_moments<T, NS, I>(v, px, g, s, t, shared, mean, e, q);
    const float inv = 1.f / ((float)g.P * (float)g.cg);
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      const float var = q[j] * inv;
      mean[j] += e[j];
      rstd[j] = 1.f / sqrtf((var < 0.f ? 0.f : var) + a.eps);    // a NaN stays
    }
  } else {
    float* stats = shared + slab_stats_at<NS>(s);                // (mean, rstd) of each group of the chunk, then one int
    const int g0 = t.chunk * s.cv * N / g.cg, groups = min(s.cv * N / g.cg, g.G - g0);
    uint64_t* words = a.words + 2 * ((int64_t)t.b * s.parts * g.G + g0);
    int part = t.part;
    for (;;) {
      slab_moments<T, NS, I>(v, px, g, s, t, shared, mean, e, q);
      if (t.row == 0 && t.live) {
#pragma unroll
        for (int j = 0; j < NS; ++j) {
          const int c = c0 + j * Q, gi = (int)fdiv((uint32_t)min(c, g.C - 1), g.d_cg);
          if (c == gi * g.cg) {                                  // a group's first piece
            uint64_t* w = words + 2 * ((int64_t)part * g.G + gi - g0);
            put_word(w, (uint64_t)__double_as_longlong((double)mean[j] + (double)e[j]));
            put_word(w + 1, (uint64_t)__double_as_longlong((double)q[j]));
          }
        }
      }
      if (part != t.part) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      part = slab_collect(words, g, s, t, groups, (int*)(stats + 2 * groups), [&](int group, bool there, uint64_t w0, uint64_t w1) {
        const int p = threadIdx.x & ((1 << s.log_parts) - 1);
        const double n = there ? (double)min(g.P - p * s.rows * I, s.rows * I) * g.cg : 0.0;
        const double m = there ? __longlong_as_double((long long)w0) : 0.0, dev = there ? __longlong_as_double((long long)w1) : 0.0;
        const double all = (double)g.P * g.cg, mu = parts_total(n * m, s) / all, d = m - mu;
        const double var = parts_total(dev + n * d * d, s) / all;
        if (p == 0 && there) {
          stats[2 * group] = (float)mu;
          stats[2 * group + 1] = (float)(1.0 / sqrt((var < 0.0 ? 0.0 : var) + (double)a.eps));
        }
      });
      if (part < 0) break;
      px = slab_pixels<I>(t, g, s, part);
      asm volatile("" : "+v"(px.first));                         // nothing of the addresses is to be kept from the first reading
      load_slab<T, I>(t, px, g, s, a.x, a.xcs, a.xco, v);
      zero_missing(px, v);
    }
    if (px.first != t.part * s.rows * I) {                       // the registers hold another part: read this one again
      px = slab_pixels<I>(t, g, s, t.part);
      asm volatile("" : "+v"(px.first));
      load_slab<T, I>(t, px, g, s, a.x, a.xcs, a.xco, v);
    }
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      const int gi = (int)fdiv((uint32_t)min(c0 + j * Q, g.C - 1), g.d_cg) - g0;
      mean[j] = stats[2 * gi];
      rstd[j] = stats[2 * gi + 1];
    }
    load_channels<N>(a.gamma, 1.f, c0, g.C, gamma);              // only now: the exchange needs the registers
    load_channels<N>(a.beta, 0.f, c0, g.C, beta);
  }
  repack(v);
  if (t.row == 0 && t.live && t.part == 0) {
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      const int c = c0 + j * Q, gi = (int)fdiv((uint32_t)min(c, g.C - 1), g.d_cg);
      if (c == gi * g.cg) {
        a.mean[(int64_t)t.b * g.G + gi] = mean[j];
        a.rstd[(int64_t)t.b * g.G + gi] = rstd[j];
      }
    }
  }
  // z = (x - mean) * (rstd * gamma) + beta; in bf16 x * (rstd * gamma) + (beta - mean * rstd * gamma), whose rounding,
  // 2^-24 of |x| and |mean|, is far below the 2^-9 that x itself was rounded by
  constexpr bool kOneFma = N == 8;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    gamma[j] *= rstd[j / Q];
    if (kOneFma) beta[j] = fmaf(-mean[j / Q], gamma[j], beta[j]);
  }
  T* out = (T*)a.out + ((int64_t)t.b * g.P + px.first + t.row) * a.ocs + a.oco + c0;
  const bool tail = c0 + N > g.C;
  auto emit = [&](auto act) {
#pragma unroll
    for (int i = 0; i < I; ++i) {
      float f[N];
      ActVec<T>::unpack(v[i], f);
#pragma unroll
      for (int j = 0; j < N; ++j) f[j] = act_value<decltype(act)::value>(fmaf(kOneFma ? f[j] : f[j] - mean[j / Q], gamma[j], beta[j]));
      if (a.drop.on) {
#pragma unroll
        for (int j = 0; j < N; ++j) f[j] = keep.kept(i, j, f[j] * a.drop.scale);
      }
      if (tail) {
#pragma unroll
        for (int j = 0; j < N; ++j) f[j] = c0 + j < g.C ? f[j] : 0.f;
      }
      if (t.live && i < px.mine) store_stream(out + (int64_t)(i * s.rows) * a.ocs, ActVec<T>::pack(f));
    }
  };
#define GN_EMIT(A) emit(std::integral_constant<int, A>{})
  MI_FOR_ACT(a.act, GN_EMIT)
#undef GN_EMIT
}

// ---------------------------------------------------------------- backward
// h and dz of one vector.  ReLU's gate is a border: where z came out smaller than its rounding can be
// (2^-20 |beta|: z = h * gamma + beta, so a small z has |h * gamma| ~ |beta|) its sign is taken from 64 bits.
template <int ACT, int N>
__device__ __forceinline__ void norm_dz(const NormArgs& a, const float* x, const float* dy, const float* mean, const float* rstd,
                                        const float* gamma, const float* beta, const KeepBits<1, N>& keep, float* h, float* dz) {
#pragma unroll
  for (int j = 0; j < N; ++j) {
    h[j] = (x[j] - mean[j]) * rstd[j];
    float z = fmaf(h[j], gamma[j], beta[j]);
    if (ACT == MI_ACT_RELU && fabsf(z) < fabsf(beta[j]) * 0x1p-20f)
      z = (float)(((double)x[j] - (double)mean[j]) * (double)rstd[j] * (double)gamma[j] + (double)beta[j]);
    float d = dy[j];
    if (a.drop.on) d = keep.kept(0, j, d * a.drop.scale);
    dz[j] = ACT == MI_ACT_RELU ? (z > 0.f ? d : 0.f) : d * act_slope<ACT>(z);
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
template <typename T, int ACT>
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
  KeepBits<1, N> keep;
  keep.keep_all();
  if (a.drop.on && a.drop.per_channel) keep.add(0, a.drop, offset, (uint64_t)w.b * (g.nv * N) + c0);
  float sa[N] = {}, sq[N] = {};
#pragma unroll
  for (int i = 0; i < kI; ++i) {
    float x[N], dy[N], h[N], dz[N];
    ActVec<T>::unpack(vx[i], x);
    ActVec<T>::unpack(vd[i], dy);
    if (a.drop.on && !a.drop.per_channel)
      keep.add(0, a.drop, offset, ((uint64_t)w.b * g.P + w.row + i * g.rows) * (uint32_t)(g.nv * N) + c0);
    norm_dz<ACT, N>(a, x, dy, ch.mean, ch.rstd, ch.gamma, ch.beta, keep, h, dz);
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
template <typename T, int ACT>
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
  KeepBits<1, N> keep;
  keep.keep_all();
  if (a.drop.on && a.drop.per_channel) keep.add(0, a.drop, offset, (uint64_t)w.b * (g.nv * N) + c0);
  T* out = (T*)a.out + (int64_t)w.b * g.P * a.ocs + a.oco + c0;
#pragma unroll
  for (int i = 0; i < kI; ++i) {
    const int p = w.row + i * g.rows;
    float x[N], dy[N], h[N], dz[N], dx[N];
    ActVec<T>::unpack(vx[i], x);
    ActVec<T>::unpack(vd[i], dy);
    if (a.drop.on && !a.drop.per_channel) keep.add(0, a.drop, offset, ((uint64_t)w.b * g.P + p) * (uint32_t)(g.nv * N) + c0);
    norm_dz<ACT, N>(a, x, dy, ch.mean, ch.rstd, ch.gamma, ch.beta, keep, h, dz);
#pragma unroll
    for (int j = 0; j < N; ++j) {
#pragma clang fp contract(off)   // t is rounded before the subtraction, as it was in the sum: a group of one value gives exactly zero
      const float t = ch.gamma[j] * dz[j];
      dx[j] = c0 + j < g.C ? ch.rstd[j] * (t - m1[j] - h[j] * m2[j]) : 0.f;
    }
    if (w.live && i < w.n) store_stream(out + (int64_t)p * a.ocs, ActVec<T>::pack(dx));
  }
}
// ---------------------------------------------------------------- launches
// in norm.hip
bool choose_slab(const NormGeom& g, int N, Slab* out);
void launch_gn_empty(uint64_t* words, int64_t n, hipStream_t s);
void launch_gn_join(const NormArgs& a, hipStream_t s);
void launch_gn_bwd_join(const NormArgs& a, int padded, hipStream_t s);
void launch_gn_param_grads(const NormArgs& a, hipStream_t s);

inline unsigned slab_grid(const Slab& s) {
  return (unsigned)((s.by_xcd ? (s.img_blocks + 7) / 8 * 8 : s.img_blocks * s.parts) * s.chunks);
}
// 64-bit words that the parts exchange
inline int64_t slab_words(const NormGeom& g, const Slab& s) { return 2 * (int64_t)g.B * s.parts * g.G; }
// LDS floats of slab_sum with K sums of NS pieces
inline int slab_sum_floats(const Slab& s, int sums) {
  if (s.tpi <= 64 && s.left == 1) return 0;
  return (s.tpi > 64 ? s.threads >> 6 : s.threads >> s.log_tpi) * s.lanes * sums;
}
// bf16 vectors of two pieces (groups of 4, 12, 20, ... channels); N / 4 is 1 in fp32, where there is no such kernel
template <typename T> bool two_pieces(const NormGeom& g) { return ActVec<T>::N == 8 && g.n_slots == 2; }
template <typename T, int NS>
void launch_fwd_slab(const NormArgs& a, const Slab& sl, hipStream_t s) {
  const dim3 grid(slab_grid(sl)), block((unsigned)sl.threads);
  // the sums, and with several parts (mean, rstd) of each group of the chunk and a number
  const int floats = slab_sum_floats(sl, 2 * NS) + (sl.parts > 1 ? 2 * (sl.cv * ActVec<T>::N / a.g.cg + 1) + 2 : 0);
  const unsigned lds = (unsigned)(floats * sizeof(float));
  if (sl.parts > 1) launch_gn_empty(a.words, slab_words(a.g, sl), s);
  switch (sl.iters) {
    case 1: hipLaunchKernelGGL((gn_fwd_slab_kernel<T, NS, 1, false>), grid, block, lds, s, a, sl); break;
    case 4: hipLaunchKernelGGL((gn_fwd_slab_kernel<T, NS, 4, false>), grid, block, lds, s, a, sl); break;
    default:
      if (sl.parts == 1) hipLaunchKernelGGL((gn_fwd_slab_kernel<T, NS, 8, false>), grid, block, lds, s, a, sl);
      else hipLaunchKernelGGL((gn_fwd_slab_kernel<T, NS, 8, true>), grid, block, lds, s, a, sl);
  }
}

template <typename T>
int launch_gn_fwd_t(const NormArgs& a, hipStream_t s) {
  Slab sl;
  if (choose_slab(a.g, ActVec<T>::N, &sl)) {
    if (a.g.n_slots == 1) launch_fwd_slab<T, 1>(a, sl, s);
    else if (two_pieces<T>(a.g)) launch_fwd_slab<T, ActVec<T>::N / 4>(a, sl, s);
    else launch_fwd_slab<T, ActVec<T>::N>(a, sl, s);
    return check_hip(hipGetLastError(), "group_norm_act_fwd");
  }
  const dim3 grid((unsigned)(a.g.B * a.g.tiles * a.g.chunks)), block(kThreads);
  if (a.g.n_slots == 1) hipLaunchKernelGGL((gn_stats_kernel<T, 1>), grid, block, 0, s, a);
  else if (two_pieces<T>(a.g)) hipLaunchKernelGGL((gn_stats_kernel<T, ActVec<T>::N / 4>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((gn_stats_kernel<T, ActVec<T>::N>), grid, block, 0, s, a);
  launch_gn_join(a, s);
#define GN_APPLY(A) hipLaunchKernelGGL((gn_apply_kernel<T, A>), grid, block, 0, s, a)
  MI_FOR_ACT(a.act, GN_APPLY)
#undef GN_APPLY
  return check_hip(hipGetLastError(), "group_norm_act_fwd");
}
template <typename T>
int launch_gn_bwd_t(const NormArgs& a, hipStream_t s) {
  if (a.g.B > 0) {
    const dim3 grid((unsigned)(a.g.B * a.g.tiles * a.g.chunks)), block(kThreads);
#define GN_SUMS(A) hipLaunchKernelGGL((gn_bwd_sums_kernel<T, A>), grid, block, 0, s, a)
    MI_FOR_ACT(a.act, GN_SUMS)
#undef GN_SUMS
    launch_gn_bwd_join(a, a.g.nv * ActVec<T>::N, s);
#define GN_DX(A) hipLaunchKernelGGL((gn_bwd_apply_kernel<T, A>), grid, block, 0, s, a)
    MI_FOR_ACT(a.act, GN_DX)
#undef GN_DX
  }
  if (a.dgamma || a.dbeta) launch_gn_param_grads(a, s);
  return check_hip(hipGetLastError(), "group_norm_act_bwd");
}
}  // namespace mi
