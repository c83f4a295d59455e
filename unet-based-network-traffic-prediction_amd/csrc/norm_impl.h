// Group norm with an activation (and dropout) on NHWC views, forward and backward.
//
//   h = (x - mean) * rstd,  z = h * gamma + beta,  y = drop(act(z))            mean, rstd over a group's cg channels x P pixels
//   dz = drop(dy) * act'(z),  t = gamma * dz,  dx = rstd * (t - mean_g(t) - h * mean_g(t * h))
//   dgamma = sum dz * h,  dbeta = sum dz                                        over images and pixels
//
// Everything is held in fp32 from the load on; what is stored in bf16 is rounded once.
//
// Two paths.  The slab kernels (below) read x, and backward dy, once into registers: one launch forward, and backward a
// second for the parameter gradients where several workgroups hold rows of them.  They take every shape but images of more
// than 64 parts (a part: at most 4096 vectors of up to 64 neighbouring ones per pixel) and groups that end together with a
// vector only after more than 64 vectors.  Those take the general kernels, which read x (and dy) twice: sums of tiles, a join, a pass that applies.
// Both are bound by HBM where a call is large, by the launches where it is small; the slab backward works nearly as long
// as it loads (about 20 operations per value, of 6 or 12 bytes, and twice that with dropout).
//
// Tiles of the general kernels.  A workgroup owns kI * R pixels of one image and up to 64 vectors (16 bytes: 8 or 4
// channels) of each: its lanes lie along the channels, so a pixel's 64..1024 bytes are read by neighbours, and R = 256 /
// lanes-per-pixel rows of pixels are read at a time.  A thread keeps its channels for all of its kI pixels: per-channel
// values are loaded once and sums stay in registers until the end.
//
// Precision of the statistics: the corrected two-pass form (Chan, Golub, LeVeque, "Algorithms for computing the sample
// variance", 1983).  A tile's mean m comes first, from registers; then r = sum (x - m) and q = sum (x - m)^2, which give
// the mean m + r / n and the squared deviations q - r^2 / n without m's own rounding; tiles are joined in 64 bits.  Data
// far from zero cost the statistics nothing: at a mean of 10^4 standard deviations rstd is off by 1e-7, without r by 2e-5.  The
// mean is handed on in fp32, as the backward pass gets it: its rounding, 2^-24 |mean| rstd, is in h and y.
// Sums have a fixed order: results repeat bit for bit.
#pragma once
#include "drop.h"
#include "norm_division.h"

#include <type_traits>

namespace mi {

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
  float2* chan;                        // backward: rows of (sum dz, sum dz*h) of each channel, chan_rows of chan_stride
  int chan_rows, chan_stride;
  float2* moments;                     // backward: [B][G] (mean t, mean t*h)
  float* dgamma; float* dbeta; float ga, gb;
  uint64_t* words;                     // what the parts of an image tell each other
  int parts;
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
// Phi(z) and exp(-z^2 / 2), from (1 - Phi(|z|)) exp(z^2 / 2) / t as a polynomial in t = 1 / (1 + k |z|); its exponential is the
// Gaussian that the slope needs.  Tensors of N values a vector:
//   4, fp32: degree 6, fitted here for the least maximum of the error over max(1 - Phi, 10^-3), k = 0.34: 1 - Phi is off by at most
//   1.1e-8, a fifth of fp32's half step at 1, or 1.1e-5 of itself where it is smaller than 10^-3;
//   8, bf16: degree 4, erf by formula 7.1.26 of Abramowitz and Stegun, "Handbook of Mathematical Functions", k, 1 / sqrt 2 and the
//   half of 1 - Phi = (1 - erf) / 2 in the constants: off by at most 7.5e-8, a 2^-15th of bf16's half step at 1.
template <int N> __device__ __forceinline__ float normal_cdf(float z, float* gauss) {
  const float t = __builtin_amdgcn_rcpf(fmaf(N == 4 ? 0.34f : 0.231641888f, fabsf(z), 1.f)), e = __builtin_amdgcn_exp2f(z * -0.72134752f * z);
  float p;
  if constexpr (N == 4) {
    p = fmaf(0.0441167168f, t, -0.197348997f);
    p = fmaf(p, t, 0.258327425f);
    p = fmaf(p, t, -0.0253811497f);
    p = fmaf(p, t, 0.153916016f);
    p = fmaf(p, t, 0.130408421f);
    p = fmaf(p, t, 0.135961592f);
  } else {
    p = fmaf(0.5307027145f, t, -0.7265760135f);
    p = fmaf(p, t, 0.7107068705f);
    p = fmaf(p, t, -0.142248368f);
    p = fmaf(p, t, 0.127414796f);
  }
  const float tail = p * t * e;                                  // 1 - Phi(|z|)
  *gauss = e;
  return z >= 0.f ? 1.f - tail : tail;
}
template <int ACT, int N> __device__ __forceinline__ float act_value(float z) {
  if constexpr (ACT == MI_ACT_RELU) return __builtin_elementwise_maximum(z, 0.f);   // a NaN stays one
  if constexpr (ACT == MI_ACT_SILU) return z * sigmoid_fast(z);
  if constexpr (ACT == MI_ACT_GELU) {
    float e;
    return z * normal_cdf<N>(z, &e);
  }
  return z;
}
template <int ACT, int N> __device__ __forceinline__ float act_slope(float z) {
  if constexpr (ACT == MI_ACT_RELU) return z > 0.f ? 1.f : 0.f;
  if constexpr (ACT == MI_ACT_SILU) {
    const float s = sigmoid_fast(z);
    return fmaf(z * s, 1.f - s, s);
  }
  if constexpr (ACT == MI_ACT_GELU) {
    float e;
    const float phi = normal_cdf<N>(z, &e);
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

__device__ __forceinline__ int opaque(int v) {                   // a value whose uses are not prepared in advance
  asm volatile("" : "+v"(v));
  return v;
}
// Ends the lifetime of what was derived from v: without it the compiler unpacks the vectors of all of a thread's pixels in
// advance and keeps them (bf16: twice the registers of the vectors) from one use to the next.  `after` is a result that
// the use has to wait for; WHICH tells branches of one switch apart, whose common beginnings would otherwise move in front
// of the switch.
template <int WHICH = -1> __device__ __forceinline__ void pin(u32x4_t& v, float after) {
  asm volatile("; %1" : "+v"(v) : "n"(WHICH), "v"(after));
}
// Values whose squares pass fp32's range are summed as their 2^-80th part (which costs nothing: what underflows is too small to
// count among them).  Squared deviations that still pass it are handed on in that scale, with their sign turned.
constexpr float kTiny = 0x1p-80f;
__device__ __forceinline__ float unscaled_or_marked(float q) {
  const float all = q * (1.f / kTiny) * (1.f / kTiny);
  return all < INFINITY ? all : -q;                              // a NaN stays
}
__device__ __forceinline__ double unmarked(float q) { return q < 0.f ? (double)q * -0x1p160 : (double)q; }
// Forward, statistics of a tile: (m, r / n, q, n) of each piece (q channels of one vector).
template <typename T, int NS>
__global__ __launch_bounds__(kThreads) void gn_stats_kernel(const NormArgs a) {
  constexpr int N = ActVec<T>::N, Q = N / NS;
  __shared__ float shared[kWaves * 64 * NS];
  const NormGeom& g = a.g;
  Tile w = my_tile(g);
  const float n = (float)w.count * Q;
  const int lane = threadIdx.x & (g.lanes - 1);
  float m[NS], r[NS], q[NS], scale[NS];
#pragma unroll
  for (int j = 0; j < NS; ++j) scale[j] = 1.f;
  for (bool again = false;; again = true) {                      // mostly once: nothing is kept for a second time
    u32x4_t v[kI];
    w.row = opaque(w.row);
    load_tile<T>(w, g, a.x, a.xcs, a.xco, v);
    float s[NS];
#pragma unroll
    for (int j = 0; j < NS; ++j) s[j] = r[j] = q[j] = 0.f;
#pragma unroll
    for (int i = 0; i < kI; ++i) {
      float f[N];
      ActVec<T>::unpack(v[i], f);
#pragma unroll
      for (int j = 0; j < N; ++j) s[j / Q] = i < w.n ? fmaf(f[j], scale[j / Q], s[j / Q]) : s[j / Q];
    }
    tile_sum<NS>(s, g, shared);
#pragma unroll
    for (int j = 0; j < NS; ++j) m[j] = shared[lane * NS + j] / n;
#pragma unroll
    for (int i = 0; i < kI; ++i) {
      float f[N];
      ActVec<T>::unpack(v[i], f);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float d = i < w.n ? fmaf(f[j], scale[j / Q], -m[j / Q]) : 0.f;
        r[j / Q] += d;
        q[j / Q] = fmaf(d, d, q[j / Q]);
      }
    }
    tile_sum<NS>(r, g, shared);
#pragma unroll
    for (int j = 0; j < NS; ++j) r[j] = shared[lane * NS + j];
    tile_sum<NS>(q, g, shared);
    bool big = false;
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      q[j] = shared[lane * NS + j];
      big = big || !(q[j] < INFINITY);
    }
    if (again || !__syncthreads_or(big && w.live && w.v * N < g.C)) break;
#pragma unroll
    for (int j = 0; j < NS; ++j) scale[j] = q[j] < INFINITY ? 1.f : kTiny;      // the others come out the same again
  }
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    if (scale[j] == 1.f) continue;
    m[j] *= 1.f / kTiny;
    r[j] *= 1.f / kTiny;
    q[j] = unscaled_or_marked(q[j]);
  }
  if ((int)threadIdx.x < g.lanes && w.live) {
    float4* out = (float4*)a.part + (((int64_t)w.b * g.tiles + w.t) * g.nv + w.v) * NS;
#pragma unroll
    for (int j = 0; j < NS; ++j) out[j] = make_float4(m[j], r[j] / n, q[j], n);
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
      f[j] = act_value<ACT, N>(fmaf((f[j] - mean[j]) * rstd[j], gamma[j], beta[j]));
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
struct SlabThread {
  int tin, slot, lane, row;    // thread of its image, image of the workgroup, vector of the chunk, row of pixels
  int b, v, part, chunk;       // image, vector
  int sums;                    // backward: row of the workgroup's channel sums
  bool live;
};
// This thread's place.  The parts of an image's chunk are neighbours in the order in which workgroups start, so they run at
// the same time (3 images of 128x128x1024 fp32, 32 chunks of 32 parts: 280 ms with the chunks next to each other, of which
// more than can run come between two parts; 164 us so).
__device__ __forceinline__ SlabThread slab_thread(const NormGeom& g, const Slab& s) {
  SlabThread t;
  const uint32_t item = fdiv(blockIdx.x, s.d_parts), ib = fdiv(item, s.d_chunks);
  t.part = (int)(blockIdx.x - item * s.parts);
  t.chunk = (int)(item - ib * s.chunks);
  const int tid = threadIdx.x;
  t.slot = tid >> s.log_tpi;
  t.tin = tid & (s.tpi - 1);
  t.lane = t.tin & (s.lanes - 1);
  t.row = t.tin >> s.log_lanes;
  t.v = min(t.chunk * s.cv + t.lane, g.nv - 1);
  t.b = (int)ib * s.nb + t.slot;
  t.live = t.slot < s.nb && t.b < g.B && t.lane < s.cv && t.chunk * s.cv + t.lane < g.nv;
  t.b = min(t.b, g.B - 1);
  t.sums = (int)ib * s.parts + t.part;
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
// K sums over each group of each image: in, a thread's K x NS partial sums (of its vector's pieces); out, the sums of the
// groups that its pieces belong to.  `shared`: as much as slab_sum_floats says; free to use again after a barrier.
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
    const int first = slab_first_piece(g, s, NS, t.chunk, t.lane, j);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float sum = 0.f;
      for (int i = 0; i < s.left; ++i) sum += mine[k * s.lanes * NS + first + i];
      v[k][j] = sum;
    }
  }
}
// Adds a vector to the sums and the sums of squares of its pieces.
template <int NS> __device__ __forceinline__ void power_sums(u32x4_t v, float (&s)[2][NS], float) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float f = __uint_as_float(v[j]);
    s[0][j * NS / 4] += f;
    s[1][j * NS / 4] = fmaf(f, f, s[1][j * NS / 4]);
  }
}
// bf16: two products and the sum in one instruction, products exact, accumulated in fp32, nothing to unpack
template <int NS> __device__ __forceinline__ void power_sums(u32x4_t v, float (&s)[2][NS], __bf16) {
  typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (NS == 8) {
      const float lo = __uint_as_float(v[j] << 16), hi = __uint_as_float(v[j] & 0xffff0000u);
      s[0][2 * j] += lo;
      s[0][2 * j + 1] += hi;
      s[1][2 * j] = fmaf(lo, lo, s[1][2 * j]);
      s[1][2 * j + 1] = fmaf(hi, hi, s[1][2 * j + 1]);
    } else {
      const bf16x2_t x = __builtin_bit_cast(bf16x2_t, (uint32_t)v[j]), one = __builtin_bit_cast(bf16x2_t, 0x3f803f80u);
      s[0][j * NS / 4] = __builtin_amdgcn_fdot2_f32_bf16(x, one, s[0][j * NS / 4], false);
      s[1][j * NS / 4] = __builtin_amdgcn_fdot2_f32_bf16(x, x, s[1][j * NS / 4], false);
    }
  }
}
// A part's vectors: from the registers of its own workgroup, or one after the other from memory.
template <typename T, int I> struct InRegisters {
  static constexpr int kUnroll = I;
  u32x4_t (&v)[I];
  __device__ __forceinline__ u32x4_t operator()(int i, float after) const {
    pin(v[i], after);
    return v[i];
  }
};
template <typename T, int I> struct InMemory {
  static constexpr int kUnroll = 1;
  const T* first;              // this thread's first pixel and vector
  int64_t step;
  int mine;
  __device__ __forceinline__ u32x4_t operator()(int i, float) const { return i < mine ? load_stream(first + i * step) : u32x4_t{0, 0, 0, 0}; }
};
template <typename T, int I>
__device__ __forceinline__ InMemory<T, I> in_memory(const SlabThread& t, const SlabPixels& px, const NormGeom& g, const Slab& s, const void* base,
                                                    int cs, int co) {
  return InMemory<T, I>{(const T*)base + ((int64_t)t.b * g.P + px.first + t.row) * cs + co + t.v * ActVec<T>::N, (int64_t)s.rows * cs, px.mine};
}
// Mean (as m + e, m rounded) and squared deviations of the groups over a part.  Sums of x and x^2 first: they do where
// the deviations are not small against the values, 4 q >= sum x^2 -- what is lost then are two bits.  Groups further from
// zero take the corrected two-pass form, and so do those whose sum of squares passes fp32's range: their values are scaled
// first.  Which of them is decided for each group by its own values.
template <typename T, int NS, int I, typename V>
__device__ __forceinline__ void slab_moments(const V& v, const SlabPixels& px, const NormGeom& g, const Slab& s, const SlabThread& t,
                                             float* shared, float* m, float* e, float* q) {
  constexpr int N = ActVec<T>::N, Q = N / NS;
  const float n = (float)px.count * (float)g.cg, inv = 1.f / n;
  float sum[2][NS] = {};
#pragma unroll V::kUnroll
  for (int i = 0; i < I; ++i) power_sums<NS>(v(i, 0.f), sum, T());
  slab_sum<NS, 2>(sum, g, s, t, shared);
  bool far = false;
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    m[j] = sum[0][j] * inv;
    e[j] = 0.f;
    q[j] = fmaf(-m[j], sum[0][j], sum[1][j]);
    far = far || !(fmaf(4.f, q[j], -sum[1][j]) >= 0.f);          // also where both are infinite
  }
  const bool real = t.live && t.v * N < g.C;                     // vectors of padding may hold anything
  if (__syncthreads_or(far && real)) {
    float scale[NS];
    bool big = false;
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      scale[j] = sum[1][j] < INFINITY ? 1.f : kTiny;
      big = big || scale[j] != 1.f;
    }
    if (__syncthreads_or(big && real)) {
      float sums[1][NS] = {};
#pragma unroll V::kUnroll
      for (int i = 0; i < I; ++i) {
        float f[N];
        ActVec<T>::unpack(v(i, m[0]), f);
#pragma unroll
        for (int j = 0; j < N; ++j) sums[0][j / Q] = fmaf(f[j], scale[j / Q], sums[0][j / Q]);
      }
      slab_sum<NS, 1>(sums, g, s, t, shared);
#pragma unroll
      for (int j = 0; j < NS; ++j) m[j] = scale[j] == 1.f ? m[j] : sums[0][j] * inv;
      __syncthreads();
    }
    float dev[2][NS] = {};
#pragma unroll V::kUnroll
    for (int i = 0; i < I; ++i) {
      float f[N];
      ActVec<T>::unpack(v(i, m[0]), f);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float d = i < px.mine ? fmaf(f[j], scale[j / Q], -m[j / Q]) : 0.f;
        dev[0][j / Q] += d;
        dev[1][j / Q] = fmaf(d, d, dev[1][j / Q]);
      }
    }
    slab_sum<NS, 2>(dev, g, s, t, shared);
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      if (fmaf(4.f, q[j], -sum[1][j]) >= 0.f) continue;
      e[j] = dev[0][j] * inv;
      q[j] = fmaf(-e[j], dev[0][j], dev[1][j]);
      q[j] = q[j] < 0.f ? 0.f : q[j];                            // a NaN stays
      if (scale[j] == 1.f) continue;
      m[j] *= 1.f / kTiny;
      e[j] *= 1.f / kTiny;
      q[j] = unscaled_or_marked(q[j]);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------- parts of an image
// Each workgroup of an image publishes its part's sums for the others, 64-bit words for each (image, part, group), and
// takes the sums of all parts in one order, so all get the same bits.  A word is valid as soon as it is not kEmpty,
// which the words are filled with before the launch and which no sum can be: there is nothing else to wait for, and
// plain device-scope loads and stores do (a release would write the whole L2 back).
// A part may take long to come -- its workgroup may not run yet, or never at the same time as this one.  No workgroup
// depends on that: after `polls` looks it forms a missing part's sums itself (from memory, the same operations in the same
// order) and publishes them, so every wait ends.
constexpr uint64_t kEmpty = ~0ull;
__device__ __forceinline__ void put_word(uint64_t* p, uint64_t w) { __hip_atomic_store(p, w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ uint64_t get_word(const uint64_t* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// For each group of the chunk: `term(part, first word, last word, part 0's first word, s0, s1)` adds a part to two sums, over all
// parts in an order that depends on their number alone, and `take(group, s0, s1, part 0's first word)` gets these.  Returns the
// number of a part that has not come, or -1.
// Threads are (share of the parts, group), up to 64 groups at a time, so that the words of several parts are under way together
// and few sums cross lanes (64 images of 100x100x64 fp32 in 64 groups, before and after this change alone: with the parts along a
// wave's lanes and one group after the other 116 us forward and 127 backward, so 91 and 106).
template <int W, typename Term, typename Take>
__device__ __forceinline__ int slab_collect(const uint64_t* words, const NormGeom& g, const Slab& s, int groups, int* missing,
                                            double2* partial, Term term, Take take) {
  constexpr int U = 4, kWavesOfPart = kSlabThreads / 64;
  const int tid = threadIdx.x, log_w = groups > 1 ? 32 - __clz(min(groups, 64) - 1) : 0, width = 1 << log_w;
  const int own = tid & (width - 1), share = tid >> log_w, shares = kSlabThreads >> log_w;
  bool failed = false;
  if (tid == 0) *missing = -1;
  __syncthreads();
  for (int base = 0; base < groups; base += width) {
    const bool real = base + own < groups;
    const uint64_t* w = words + W * min(base + own, groups - 1);
    uint64_t first = 0, a[U], b[U];
    double s0 = 0.0, s1 = 0.0;
    for (int p0 = share; p0 - share < s.parts && !failed; p0 += shares * U) {
      for (int i = 0;; ++i) {
        bool all = true;
        if constexpr (W == 2) {
          first = get_word(w);
          all = !real || first != kEmpty;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int p = p0 + u * shares;
          a[u] = b[u] = 0;
          if (p - share >= s.parts) continue;                    // uniform: nobody has that many
          const uint64_t* at = w + W * ((int64_t)min(p, s.parts - 1) * g.G);
          a[u] = get_word(at);
          if (W == 2) b[u] = get_word(at + 1);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) all = all && (!real || p0 + u * shares >= s.parts || (a[u] != kEmpty && b[u] != kEmpty));
        if (__all(all)) break;
        if (i >= s.polls) {
          if (real && W == 2 && first == kEmpty) atomicMax(missing, 0);
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (real && p0 + u * shares < s.parts && (a[u] == kEmpty || b[u] == kEmpty)) atomicMax(missing, p0 + u * shares);
          failed = true;
          break;
        }
        __builtin_amdgcn_s_sleep(1);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (p0 + u * shares < s.parts) term(p0 + u * shares, a[u], b[u], first, s0, s1);
    }
    for (int o = 32; o >= width; o >>= 1) {
      s0 += __shfl_xor(s0, o, 64);
      s1 += __shfl_xor(s1, o, 64);
    }
    if ((tid & 63) < width) partial[(tid >> 6) * width + own] = make_double2(s0, s1);
    __syncthreads();
    if (tid < width && real) {
      for (int k = 1; k < kWavesOfPart; ++k) {
        s0 += partial[k * width + own].x;
        s1 += partial[k * width + own].y;
      }
      take(base + own, s0, s1, first);
    }
    __syncthreads();
  }
  const int result = *missing;
  __syncthreads();
  return result;
}
// 256 threads with up to 16 vectors each: what a thread does once -- its place, its channels' parameters, the sums over
// other threads -- is several hundred instructions, worth it for 128 values (512 threads with 8 vectors, forward: 16.3 us
// against 16.4 for 512 images of 32x32x32 bf16).  16 vectors leave three workgroups a CU (up to 168 registers); 4 vectors
// stay within 128, so 1024 threads fit.
// Bound by HBM.  Medians of a kernel trace over rotating tensors: 1024 images of 64x64x32 bf16 with SiLU, four parts each, 108 us
// for 537 MB = 5.0 TB/s, and 4.8 for the launch that empties the words (105 a call for both, back to back); 512 of 32x32x32 with
// ReLU and dropout 10 % 16.4 us for 67 MB = 4.1 TB/s (14.9 a call: the mask's words are worked out while the loads are in
// flight); 512 of 64x64x32 fp32 with SiLU 101 for 537 MB = 5.3 TB/s.  One image of 64x64x32: 8.5 us, of which a launch is 2.8
// and the rest one memory latency after the other.
template <typename T, int NS, int I, bool PARTS>
__global__ __launch_bounds__(I == 4 && !PARTS ? kWideThreads : kSlabThreads, I > 4 || PARTS ? 3 : 4) void gn_fwd_slab_kernel(const NormArgs a, const Slab s) {
  constexpr int N = ActVec<T>::N, Q = N / NS;
  extern __shared__ float shared[];
  const NormGeom& g = a.g;
  const SlabThread t = slab_thread(g, s);
  const int c0 = t.v * N;
  const SlabPixels px = slab_pixels<I>(t, g, s, t.part);
  u32x4_t v[I];
  float gamma[N], beta[N];
  if constexpr (!PARTS) {
    load_channels<N>(a.gamma, 1.f, c0, g.C, gamma);
    load_channels<N>(a.beta, 0.f, c0, g.C, beta);
  }
  load_slab<T, I>(t, px, g, s, a.x, a.xcs, a.xco, v);
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
  slab_moments<T, NS, I>(InRegisters<T, I>{v}, px, g, s, t, shared, mean, e, q);
  if constexpr (!PARTS) {
    const float inv = 1.f / ((float)g.P * (float)g.cg);
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      const float var = q[j] * inv;
      mean[j] += e[j];
      rstd[j] = var < 0.f ? kTiny / sqrtf(-var) : 1.f / sqrtf(var + a.eps);
    }
  } else {
    float* stats = shared + slab_stats_at(s, NS);                // (mean, rstd) of each group of the chunk, then one int
    const int g0 = slab_first_group(g, s, N, t.chunk), groups = slab_groups(g, s, N, t.chunk);
    uint64_t* words = a.words + 2 * ((int64_t)t.b * s.parts * g.G + g0);
    auto publish = [&](int part) {
      if (t.row != 0 || !t.live) return;
      const int c1 = opaque(c0);
#pragma unroll
      for (int j = 0; j < NS; ++j) {
        const int c = c1 + j * Q, gi = (int)fdiv((uint32_t)min(c, g.C - 1), g.d_cg);
        if (c != gi * g.cg) continue;                            // not a group's first piece
        uint64_t* w = words + 2 * ((int64_t)part * g.G + gi - g0);
        put_word(w, (uint64_t)__double_as_longlong((double)mean[j] + (double)e[j]));
        put_word(w + 1, (uint64_t)__double_as_longlong(unmarked(q[j])));
      }
    };
    publish(t.part);
    for (;;) {
      // deviations from part 0's mean: those of the means themselves, so nothing cancels that 64 bits would miss
      const int part = slab_collect<2>(words, g, s, groups, (int*)(stats + slab_missing_at(groups)), (double2*)(stats + slab_partial_at(groups)),
        [&](int p, uint64_t w0, uint64_t w1, uint64_t first, double& s0, double& s1) {
          const double n = (double)min(g.P - p * s.rows * I, s.rows * I) * g.cg;
          const double d = __longlong_as_double((long long)w0) - __longlong_as_double((long long)first);
          s0 = fma(n, d, s0);
          s1 += fma(n * d, d, __longlong_as_double((long long)w1));
        },
        [&](int group, double s0, double s1, uint64_t first) {
          const double all = (double)g.P * g.cg, d = s0 / all, var = s1 / all - d * d;
          stats[2 * group] = (float)(__longlong_as_double((long long)first) + d);
          stats[2 * group + 1] = (float)(1.0 / sqrt((var < 0.0 ? 0.0 : var) + (double)a.eps));
        });
      if (__builtin_expect(part < 0, 1)) break;
      const SlabPixels other = slab_pixels<I>(t, g, s, part);
      slab_moments<T, NS, I>(in_memory<T, I>(t, other, g, s, a.x, a.xcs, a.xco), other, g, s, t, shared, mean, e, q);
      publish(part);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");           // the next look finds it
    }
    const int c1 = opaque(c0);
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      const int gi = slab_group_of(g, s, N, t.chunk, c1 + j * Q);
      mean[j] = stats[2 * gi];
      rstd[j] = stats[2 * gi + 1];
    }
    load_channels<N>(a.gamma, 1.f, c0, g.C, gamma);              // only now: the exchange needs the registers
    load_channels<N>(a.beta, 0.f, c0, g.C, beta);
  }
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
#pragma unroll
  for (int j = 0; j < N; ++j) gamma[j] *= rstd[j / Q];           // z = (x - mean) * (rstd * gamma) + beta
  T* out = (T*)a.out + ((int64_t)t.b * g.P + px.first + t.row) * a.ocs + a.oco + c0;
  const bool ragged = g.C != g.nv * N;                           // uniform: mostly there are no padding channels to look for
  auto emit = [&](auto act) {
#pragma unroll
    for (int i = 0; i < I; ++i) {
      pin<decltype(act)::value>(v[i], rstd[0]);
      float f[N];
      ActVec<T>::unpack(v[i], f);
#pragma unroll
      for (int j = 0; j < N; ++j) f[j] = act_value<decltype(act)::value, N>(fmaf(f[j] - mean[j / Q], gamma[j], beta[j]));
      if (a.drop.on) {
#pragma unroll
        for (int j = 0; j < N; ++j) f[j] = keep.kept(i, j, f[j] * a.drop.scale);
      }
      if (ragged) {
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
    dz[j] = ACT == MI_ACT_RELU ? (z > 0.f ? d : 0.f) : d * act_slope<ACT, N>(z);
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
// ReLU's gate is a border that fp32 rounding of z may cross.  But z > 0 is  sign(gamma) x > sign(gamma) tau  with
// tau = mean - beta / (rstd gamma), and x is an fp32 value: against tau in 64 bits, rounded down to fp32, the comparison is
// exact.  Where x is the mean, as in a group without deviations, z = beta: its sign decides, also where nothing is left of the
// quotient next to the mean.  A channel's tau is worked out once per workgroup; the gate costs two instructions and needs no z.
// The quotient by two steps of Newton's method from the hardware's reciprocal (a library division works a special case per
// operand out besides, one after the other).
__device__ __forceinline__ float relu_threshold(float mean, float rstd, float gamma, float beta) {
  const double d = (double)rstd * (double)gamma;                 // 48 bits: exact
  double r = __builtin_amdgcn_rcp(d);
  r = fma(fma(-d, r, 1.0), r, r);
  r = fma(fma(-d, r, 1.0), r, r);
  double tau = fma(-(double)beta, r, (double)mean);
  tau = gamma < 0.f ? -tau : tau;
  const float f = (float)tau;
  const float below = f > 0.f ? __uint_as_float(__float_as_uint(f) - 1) : __uint_as_float(f < 0.f ? __float_as_uint(f) + 1 : 0x80000001u);
  const bool down = f == (gamma < 0.f ? -mean : mean) ? beta > 0.f : (double)f > tau;
  const float t = down ? below : f;                              // f itself where tau is an fp32 value, infinite or NaN
  return d == 0.0 ? (beta > 0.f ? -INFINITY : INFINITY) : t;     // z = beta
}
__device__ __forceinline__ bool relu_gate(float x, float gamma, float threshold) {
  return __uint_as_float(__builtin_amdgcn_bitop3_b32(__float_as_uint(x), __float_as_uint(gamma), 0x80000000u, 0x78)) > threshold;   // x ^ (gamma & sign)
}
// The thresholds of a thread's channels.  At least N rows of threads share the work: a thread does one at most, they pass
// through LDS (nb * lanes * N floats), and `first`, what it is made of, is read before the tile's loads are issued, which
// complete in order.  Fewer rows: every thread its own, from its channels' values (512 images of 2x2x512 bf16 backward
// 11.9 us where they shared it and fetched what the further ones are made of, 9.6 so).
struct ReluInputs { float mean, rstd, gamma, beta; };
__device__ __forceinline__ ReluInputs relu_inputs(const NormArgs& a, const SlabThread& t, int c0, int k) {
  const int c = min(c0 + k, a.g.C - 1);
  const int64_t gi = (int64_t)t.b * a.g.G + fdiv((uint32_t)c, a.g.d_cg);
  return ReluInputs{a.mean[gi], a.rstd[gi], a.gamma ? a.gamma[c] : 1.f, a.beta ? a.beta[c] : 0.f};
}
template <int NS, int N>
__device__ __forceinline__ void relu_thresholds(const Slab& s, const SlabThread& t, ReluInputs first, const float* mean, const float* rstd,
                                                const float* gamma, const float* beta, float* shared, float* out) {
  if (s.rows < N) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      out[j] = relu_threshold(mean[j * NS / N], rstd[j * NS / N], gamma[j], beta[j]);
      asm volatile("" : "+v"(out[j]));                           // one after the other: eight at a time need the tile's registers
    }
    return;
  }
  float* mine = shared + t.slot * s.lanes * N;
  if (t.tin < s.lanes * N) mine[t.tin] = relu_threshold(first.mean, first.rstd, first.gamma, first.beta);
  __syncthreads();
#pragma unroll
  for (int j = 0; j < N; ++j) out[j] = mine[t.lane * N + j];
  __syncthreads();
}
template <int NS, int N> __device__ __forceinline__ void slab_stats(const NormArgs& a, int b, int c0, float* mean, float* rstd) {
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    const int64_t gi = (int64_t)b * a.g.G + fdiv((uint32_t)min(c0 + j * N / NS, a.g.C - 1), a.g.d_cg);
    mean[j] = a.mean[gi];
    rstd[j] = a.rstd[gi];
  }
}
// Per-channel values of the backward pass: scaled = gamma * rstd.
template <int NS, int N>
__device__ __forceinline__ void slab_channels(const NormArgs& a, int b, int c0, float* mean, float* rstd, float* scaled, float* beta) {
  slab_stats<NS, N>(a, b, c0, mean, rstd);
  load_channels<N>(a.gamma, 1.f, c0, a.g.C, scaled);
  load_channels<N>(a.beta, 0.f, c0, a.g.C, beta);
}
template <int NS, int N> __device__ __forceinline__ void slab_scale(const float* rstd, float* scaled) {
#pragma unroll
  for (int j = 0; j < N; ++j) scaled[j] *= rstd[j * NS / N];
}
// x in units of a power of two near the group's standard deviation, where that is above 1: mean and rstd in these units, and
// the unit's inverse.  Squares of rstd and sums of x would leave fp32's range otherwise (at deviations of 10^20 dx lost its
// third term); a power of two changes no other bit.
template <int NS> __device__ __forceinline__ void slab_units(float* mean, float* rstd, float* unit) {
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    const uint32_t power = __float_as_uint(rstd[j]) & 0x7f800000u;                     // 2^floor(log2 rstd), 0 of a subnormal rstd
    const bool in = power > 0 && rstd[j] < 1.f;
    unit[j] = in ? __uint_as_float(power) : 1.f;
    mean[j] *= unit[j];
    rstd[j] *= in ? __uint_as_float(0x7f000000u - power) : 1.f;
  }
}
// Publishes a part's two sums of each group.
template <int NS, int N>
__device__ __forceinline__ void publish_bwd(const NormArgs& a, const SlabThread& t, int part, const float (&sum)[2][NS]) {
  if (t.row != 0 || !t.live) return;
  const NormGeom& g = a.g;
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    const int c = t.v * N + j * (N / NS), gi = (int)fdiv((uint32_t)min(c, g.C - 1), g.d_cg);
    if (c != gi * g.cg) continue;                                // not a group's first piece
    const uint32_t w0 = sum[0][j] == sum[0][j] ? __float_as_uint(sum[0][j]) : 0x7fc00000u;   // never kEmpty
    const uint32_t w1 = sum[1][j] == sum[1][j] ? __float_as_uint(sum[1][j]) : 0x7fc00000u;
    put_word(a.words + ((int64_t)t.b * a.parts + part) * g.G + gi, (uint64_t)w1 << 32 | w0);
  }
}
// Sums M values over the lanes that differ in bits lanes .. o; every total lands in dst.
template <int M> __device__ __forceinline__ void scatter_sum(const float* v, int o, int lanes, int lane, float* dst) {
  if (o < lanes) {
#pragma unroll
    for (int j = 0; j < M; ++j) dst[j] = v[j];
    return;
  }
  if constexpr (M > 1) {
    const bool up = (lane & o) != 0;
    float r[M / 2];
#pragma unroll
    for (int j = 0; j < M / 2; ++j) r[j] = (up ? v[M / 2 + j] : v[j]) + __shfl_xor(up ? v[j] : v[M / 2 + j], o, 64);
    scatter_sum<M / 2>(r, o >> 1, lanes, lane, dst + (up ? M / 2 : 0));
  } else {
    float r = v[0];
    for (; o >= lanes; o >>= 1) r += __shfl_xor(r, o, 64);
    dst[0] = r;                                                  // lanes that differ in these bits write the same value
  }
}
// A channel's sums: the gradients themselves if there is one row of them, else a row for gn_param_grads_kernel.
__device__ __forceinline__ void store_channel(const NormArgs& a, int row, int c, float sum_dz, float sum_dzh) {
  if (a.chan_rows > 1) {
    a.chan[(int64_t)row * a.chan_stride + c] = make_float2(sum_dz, sum_dzh);
    return;
  }
  if (a.dgamma) a.dgamma[c] = a.ga * sum_dzh + (a.gb != 0.f ? a.gb * a.dgamma[c] : 0.f);
  if (a.dbeta) a.dbeta[c] = a.ga * sum_dz + (a.gb != 0.f ? a.gb * a.dbeta[c] : 0.f);
}
// Adds a vector's dz and dz * (x - mean) to the sums of its channels (d4: dy, dropped units cleared; scaled: gamma * rstd; x as
// slab_units has it).
// What the second pass needs of dy comes back: with gated-off units cleared; in fp32 as dz itself, and so in bf16 with
// SPLIT, the upper halves of dz in d4, the lower ones in `low` (else its slope is worked out again: a bf16 dz would be rounded).
template <typename T, int NS, int ACT, bool SPLIT>
__device__ __forceinline__ void bwd_step(u32x4_t x4, u32x4_t& d4, u32x4_t& low, const float* mean, const float* unit, const float* scaled,
                                         const float* beta, const float* threshold, float* ch) {
  constexpr int N = ActVec<T>::N;
#pragma unroll
  for (int e = 0; e < N / 4; ++e) {
    float x[4], d[4];
    ActVec<T>::unpack4(x4, e, x);
    ActVec<T>::unpack4(d4, e, d);
    if constexpr (ACT == MI_ACT_RELU) {
#pragma unroll
      for (int j = 0; j < 4; ++j) d[j] = relu_gate(x[j], scaled[4 * e + j], threshold[4 * e + j]) ? d[j] : 0.f;
      ActVec<T>::pack4_exact(d, e, d4);
      if (e == N / 4 - 1) pin(d4, mean[0]);                      // what was packed is not kept unpacked besides
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = fmaf(x[j], unit[(4 * e + j) * NS / N], -mean[(4 * e + j) * NS / N]);
    if constexpr (ACT == MI_ACT_SILU || ACT == MI_ACT_GELU) {
#pragma unroll
      for (int j = 0; j < 4; ++j) d[j] *= act_slope<ACT, N>(fmaf(x[j], scaled[4 * e + j], beta[4 * e + j]));
    }
    if constexpr (N == 4 && (ACT == MI_ACT_SILU || ACT == MI_ACT_GELU)) ActVec<T>::pack4(d, e, d4);
    if constexpr (SPLIT) {
      ActVec<T>::split4(d, e, d4, low);
      if (e == N / 4 - 1) {
        pin(d4, mean[0]);
        pin(low, mean[0]);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      ch[4 * e + j] += d[j];
      ch[N + 4 * e + j] = fmaf(d[j], x[j], ch[N + 4 * e + j]);
    }
    __builtin_amdgcn_sched_barrier(0);                           // one group after the other: together they need several times the registers
  }
}
// A group's two sums, of rstd * t and rstd * t * (x - mean), from those of a thread's channels.
template <int NS, int N> __device__ __forceinline__ void bwd_group_sums(const float* ch, const float* scaled, float (&sum)[2][NS]) {
#pragma unroll
  for (int j = 0; j < NS; ++j) sum[0][j] = sum[1][j] = 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    sum[0][j * NS / N] = fmaf(scaled[j], ch[j], sum[0][j * NS / N]);
    sum[1][j * NS / N] = fmaf(scaled[j], ch[N + j], sum[1][j * NS / N]);
  }
}
// The sums of a part whose workgroup has not come, from memory: the same operations in the same order, one vector at a time.
template <typename T, int NS, int I, int ACT>
__device__ __forceinline__ void bwd_other_part(const NormArgs& a, const Slab& s, const SlabThread& t, int part, float* shared) {
  constexpr int N = ActVec<T>::N;
  const NormGeom& g = a.g;
  const SlabPixels px = slab_pixels<I>(t, g, s, part);
  const int c0 = opaque(t.v * N), chunk_c0 = t.chunk * s.cv * N;
  float mean[NS], rstd[NS], unit[NS], scaled[N], beta[N], threshold[N], ch[2 * N] = {}, sum[2][NS];
  slab_channels<NS, N>(a, t.b, c0, mean, rstd, scaled, beta);
  if constexpr (ACT == MI_ACT_RELU)
    relu_thresholds<NS, N>(s, t, relu_inputs(a, t, chunk_c0, t.tin), mean, rstd, scaled, beta, shared, threshold);
  slab_units<NS>(mean, rstd, unit);
  slab_scale<NS, N>(rstd, scaled);
  const auto x = in_memory<T, I>(t, px, g, s, a.x, a.xcs, a.xco), dy = in_memory<T, I>(t, px, g, s, a.dy, a.ycs, a.yco);
#pragma unroll 1
  for (int i = 0; i < I; ++i) {
    u32x4_t d = dy(i, 0.f);
    if (a.drop.on) {
      KeepBits<1, N> keep;
      const uint64_t row = a.drop.per_channel ? (uint64_t)t.b : (uint64_t)t.b * g.P + (px.first + t.row + i * s.rows);
      keep.add(0, a.drop, drop_offset(a.drop), row * (uint32_t)(g.nv * N) + c0);
      d = keep.kept(0, d);
    }
    u32x4_t unused;
    bwd_step<T, NS, ACT, false>(x(i, 0.f), d, unused, mean, unit, scaled, beta, threshold, ch);
  }
  bwd_group_sums<NS, N>(ch, scaled, sum);
  slab_sum<NS, 2>(sum, g, s, t, shared);
  publish_bwd<NS, N>(a, t, part, sum);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");               // the next look finds it
}
// The mask of a part's units, applied to dy's registers.
template <typename T, int I>
__device__ __forceinline__ void bwd_drop(const NormArgs& a, const Slab& s, const SlabThread& t, const SlabPixels& px, u32x4_t (&vd)[I]) {
  constexpr int N = ActVec<T>::N;
  if (!a.drop.on) return;
  KeepBits<I, N> keep;
  const uint64_t offset = drop_offset(a.drop);
#pragma unroll
  for (int i = 0; i < I; ++i) {
    const uint64_t row = a.drop.per_channel ? (uint64_t)t.b : (uint64_t)t.b * a.g.P + (px.first + t.row + i * s.rows);
    keep.add(i, a.drop, offset, row * (uint32_t)(a.g.nv * N) + t.v * N);
  }
#pragma unroll
  for (int i = 0; i < I; ++i) vd[i] = keep.kept(i, vd[i]);
}
// The workgroup's sums of each channel, over rows and images, into row `row` of the parameter gradients: lanes first, each
// stage halves what a lane holds, then the waves through LDS.
template <int N>
__device__ __forceinline__ void bwd_channel_sums(const NormArgs& a, const Slab& s, const SlabThread& t, float (&ch)[2 * N], bool live,
                                                 float scale, int row, float* shared) {
  if (a.dgamma == nullptr && a.dbeta == nullptr) return;
  __syncthreads();
  const int lane = threadIdx.x & 63, waves = s.threads >> 6, c0 = t.chunk * s.cv * N;
  if (!live) {
#pragma unroll
    for (int j = 0; j < 2 * N; ++j) ch[j] = 0.f;
  }
  scatter_sum<2 * N>(ch, 32, s.lanes, lane, shared + ((threadIdx.x >> 6) * s.lanes + (lane & (s.lanes - 1))) * (2 * N));
  __syncthreads();
  for (int k = threadIdx.x; k < s.lanes * N; k += s.threads) {
    const int l = k / N, j = k & (N - 1), c = c0 + k;
    if (l >= s.cv || c >= a.g.C) continue;
    float sa = 0.f, sq = 0.f;
    for (int w = 0; w < waves; ++w) {
      sa += shared[(w * s.lanes + l) * 2 * N + j];
      sq += shared[(w * s.lanes + l) * 2 * N + N + j];
    }
    store_channel(a, row, c, sa * scale, sq * scale);
  }
}
// The means over the groups of a thread's pieces, from all parts of the image; `sum` has this part's sums.
template <typename T, int NS, int I, bool PARTS, int ACT>
__device__ __forceinline__ void bwd_means(const NormArgs& a, const Slab& s, const SlabThread& t, float (&sum)[2][NS], float* shared) {
  constexpr int N = ActVec<T>::N;
  const NormGeom& g = a.g;
  if constexpr (!PARTS) {
    const float inv = 1.f / ((float)g.P * (float)g.cg);
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      sum[0][j] *= inv;
      sum[1][j] *= inv;
    }
  } else {
    const int g0 = slab_first_group(g, s, N, t.chunk), groups = slab_groups(g, s, N, t.chunk);
    const uint64_t* words = a.words + ((int64_t)t.b * s.parts * g.G + g0);
    float* stats = shared + slab_stats_at(s, NS);
    __syncthreads();
    for (;;) {
      const int part = slab_collect<1>(words, g, s, groups, (int*)(stats + slab_missing_at(groups)), (double2*)(stats + slab_partial_at(groups)),
        [&](int, uint64_t w, uint64_t, uint64_t, double& s0, double& s1) {
          s0 += (double)__uint_as_float((uint32_t)w);
          s1 += (double)__uint_as_float((uint32_t)(w >> 32));
        },
        [&](int group, double s0, double s1, uint64_t) {
          const double n = (double)g.P * g.cg;
          stats[2 * group] = (float)(s0 / n);
          stats[2 * group + 1] = (float)(s1 / n);
        });
      if (__builtin_expect(part < 0, 1)) break;
      bwd_other_part<T, NS, I, ACT>(a, s, t, part, shared);
    }
    const int c0 = opaque(t.v * N);
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      const int gi = slab_group_of(g, s, N, t.chunk, c0 + j * (N / NS));
      sum[0][j] = stats[2 * gi];
      sum[1][j] = stats[2 * gi + 1];
    }
  }
}
// dx of a part from the registers:  dx = scaled * dz - M1 - (x - mean) * rstd^2 * M2,  M1 and M2 the means over the group of
// scaled * dz and scaled * dz * (x - mean); times dropout's factor, and by the unit of x.
template <typename T, int NS, int I, int ACT, bool SPLIT>
__device__ __forceinline__ void bwd_emit(const NormArgs& a, const Slab& s, const SlabThread& t, const SlabPixels& px, u32x4_t (&vx)[I],
                                         u32x4_t (&vd)[I], const u32x4_t* low, const float* mean, const float* rstd, const float* unit, const float* scaled,
                                         const float* beta, const float (&sum)[2][NS], float factor) {
  constexpr int N = ActVec<T>::N, Q = N / NS;
  const int c0 = t.v * N;
  T* out = (T*)a.out + ((int64_t)t.b * a.g.P + px.first + t.row) * a.ocs + a.oco + c0;
  const bool ragged = a.g.C != a.g.nv * N;
  // a group of one value passes nothing on; its terms would cancel but for their roundings
  if (a.g.P == 1 && a.g.cg == 1) factor = 0.f;
  float b0[NS], b1[NS], slope[N];
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    b0[j] = -sum[0][j] * (factor * unit[j]);
    b1[j] = -sum[1][j] * rstd[j] * rstd[j] * (factor * unit[j]);
  }
#pragma unroll
  for (int j = 0; j < N; ++j) slope[j] = scaled[j] * (factor * unit[j / Q]);
#pragma unroll
  for (int i = 0; i < I; ++i) {
    pin(vx[i], sum[0][0]);
    pin(vd[i], sum[0][0]);
    u32x4_t lo;
    if constexpr (SPLIT) lo = low[i * kSlabThreads];
#pragma unroll
    for (int e = 0; e < N / 4; ++e) {
      float x[4], d[4];
      ActVec<T>::unpack4(vx[i], e, x);
      if constexpr (SPLIT) ActVec<T>::join4(vd[i], lo, e, d);
      else ActVec<T>::unpack4(vd[i], e, d);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = 4 * e + j, k = c / Q;
        x[j] = fmaf(x[j], unit[k], -mean[k]);
        if constexpr (N == 8 && !SPLIT && (ACT == MI_ACT_SILU || ACT == MI_ACT_GELU)) d[j] *= act_slope<ACT, N>(fmaf(x[j], scaled[c], beta[c]));
        d[j] = fmaf(x[j], b1[k], fmaf(d[j], slope[c], b0[k]));
      }
      if (ragged) {
#pragma unroll
        for (int j = 0; j < 4; ++j) d[j] = c0 + 4 * e + j < a.g.C ? d[j] : 0.f;
      }
      ActVec<T>::pack4(d, e, vd[i]);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (t.live && i < px.mine) store_stream(out + (int64_t)(i * s.rows) * a.ocs, vd[i]);
  }
}
// One read of x and dy: the same division of the work as forward.  Sums of dz and dz * h for each channel come first; a
// group's two sums are made of them.  Dropout's factor is left out of dz and t until the end: dx and the gradients are
// linear in it.
// 16 vectors of x and of dy take 128 registers, all of it up to 256: two workgroups a CU.  Those load together, compute
// together and store together, so the time is near the sum of both.  Medians of a kernel trace over rotating tensors: 64 images of
// 128x128x32 bf16 with SiLU 47 us for 201 MB (32 of memory at 6.2 TB/s), 512 of 32x32x32 with ReLU and dropout 24 for 101 MB (16),
// 256 of 64x64x32 fp32 with ReLU 76 for 403 MB (65).
// SPLIT: the second pass takes dz as the first one had it, in fp32: its upper halves are where dy was, its lower ones in LDS
// (64 KB; each thread its own, nothing to wait for).  Working the slope out again instead took 60 us where it was 53.5 with this
// change alone, and for 1024 images of 64x64x32 with GELU 255 and 185; the bits are the same.  Where a bf16 vector has eight pieces there is no LDS to
// spare beside the sums of two workgroups, and with 4 vectors a thread nothing to gain.
// What did not help there: 8 vectors a thread and three workgroups, a staggered start, workgroups that stay and prefetch
// the next part (their polls and stores queue behind the prefetch: 83 us against 62), loads of x and dy in turn.
template <typename T, int NS, int I, bool PARTS, int ACT>
__global__ __launch_bounds__(I == 4 && !PARTS ? kWideThreads : kSlabThreads, I > 4 || PARTS ? 2 : 4) void gn_bwd_slab_kernel(const NormArgs a, const Slab s) {
  constexpr int N = ActVec<T>::N;
  constexpr bool SPLIT = N == 8 && NS < N && I == 16 && (ACT == MI_ACT_SILU || ACT == MI_ACT_GELU);
  extern __shared__ float shared[];
  __shared__ u32x4_t low[SPLIT ? I * kSlabThreads : 1];          // [vector][thread]: each thread's own
  const NormGeom& g = a.g;
  const SlabThread t = slab_thread(g, s);
  const int c0 = t.v * N;
  const float scale = a.drop.on ? a.drop.scale : 1.f;
  const SlabPixels px = slab_pixels<I>(t, g, s, t.part);
  u32x4_t vx[I], vd[I];
  float mean[NS], rstd[NS], unit[NS], scaled[N], beta[N], threshold[N], sum[2][NS], ch[2 * N] = {};
  ReluInputs first;
  if constexpr (ACT == MI_ACT_RELU) first = relu_inputs(a, t, t.chunk * s.cv * N, t.tin);
  slab_channels<NS, N>(a, t.b, c0, mean, rstd, scaled, beta);
  load_slab<T, I>(t, px, g, s, a.x, a.xcs, a.xco, vx);
  load_slab<T, I>(t, px, g, s, a.dy, a.ycs, a.yco, vd);
  if constexpr (ACT == MI_ACT_RELU) relu_thresholds<NS, N>(s, t, first, mean, rstd, scaled, beta, shared, threshold);
  slab_units<NS>(mean, rstd, unit);
  slab_scale<NS, N>(rstd, scaled);
  bwd_drop<T, I>(a, s, t, px, vd);
  zero_missing(px, vx);
  zero_missing(px, vd);
#pragma unroll
  for (int i = 0; i < I; ++i) {
    pin(vx[i], scaled[0]);
    pin(vd[i], scaled[0]);
    u32x4_t lo;
    bwd_step<T, NS, ACT, SPLIT>(vx[i], vd[i], lo, mean, unit, scaled, beta, threshold, ch);
    if constexpr (SPLIT) low[i * kSlabThreads + threadIdx.x] = lo;
  }
  bwd_group_sums<NS, N>(ch, scaled, sum);
  slab_sum<NS, 2>(sum, g, s, t, shared);
  if constexpr (PARTS) publish_bwd<NS, N>(a, t, t.part, sum);
#pragma unroll
  for (int j = 0; j < N; ++j) ch[N + j] *= rstd[j * NS / N];     // dz * h
  bwd_channel_sums<N>(a, s, t, ch, t.live, scale, t.sums, shared);
  bwd_means<T, NS, I, PARTS, ACT>(a, s, t, sum, shared);
  if constexpr (PARTS) {                                         // the exchange needs their registers
    slab_channels<NS, N>(a, t.b, opaque(c0), mean, rstd, scaled, beta);
    slab_units<NS>(mean, rstd, unit);
    slab_scale<NS, N>(rstd, scaled);
  }
  bwd_emit<T, NS, I, ACT, SPLIT>(a, s, t, px, vx, vd, low + threadIdx.x, mean, rstd, unit, scaled, beta, sum, scale);
}
// ---------------------------------------------------------------- launches
// in norm.hip
void launch_gn_empty(uint64_t* words, int64_t n, hipStream_t s);
void launch_gn_join(const NormArgs& a, hipStream_t s);
void launch_gn_bwd_join(const NormArgs& a, int padded, hipStream_t s);
void launch_gn_param_grads(const NormArgs& a, hipStream_t s);

// bf16 vectors of two pieces (groups of 4, 12, 20, ... channels); N / 4 is 1 in fp32, where there is no such kernel
template <typename T> bool two_pieces(const NormGeom& g) { return ActVec<T>::N == 8 && g.n_slots == 2; }
template <typename T, int NS>
void launch_fwd_slab(const NormArgs& a, const Slab& sl, hipStream_t s) {
  const dim3 grid(slab_grid(sl)), block((unsigned)sl.threads);
  const int floats = slab_fwd_floats(a.g, sl, NS, ActVec<T>::N);
  const unsigned lds = (unsigned)(floats * sizeof(float));
  if (sl.parts > 1) launch_gn_empty(a.words, slab_words(a.g, sl), s);
#define GN_SLAB(I, PARTS) hipLaunchKernelGGL((gn_fwd_slab_kernel<T, NS, I, PARTS>), grid, block, lds, s, a, sl)
  if (sl.iters == 1) GN_SLAB(1, false);
  else if (sl.iters == 4 && sl.parts == 1) GN_SLAB(4, false);
  else if (sl.iters == 4) GN_SLAB(4, true);
  else if (sl.parts == 1) GN_SLAB(16, false);
  else GN_SLAB(16, true);
#undef GN_SLAB
}

template <typename T>
int launch_gn_fwd_t(const NormArgs& a, const Slab* sl, hipStream_t s) {
  if (sl != nullptr) {
    if (a.g.n_slots == 1) launch_fwd_slab<T, 1>(a, *sl, s);
    else if (two_pieces<T>(a.g)) launch_fwd_slab<T, ActVec<T>::N / 4>(a, *sl, s);
    else launch_fwd_slab<T, ActVec<T>::N>(a, *sl, s);
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
template <typename T, int NS, int ACT>
void launch_bwd_slab_act(const NormArgs& a, const Slab& sl, dim3 grid, dim3 block, unsigned lds, hipStream_t s) {
#define GN_SLAB(I, PARTS) hipLaunchKernelGGL((gn_bwd_slab_kernel<T, NS, I, PARTS, ACT>), grid, block, lds, s, a, sl)
  if (sl.iters == 1) GN_SLAB(1, false);
  else if (sl.iters == 4 && sl.parts == 1) GN_SLAB(4, false);
  else if (sl.iters == 4) GN_SLAB(4, true);
  else if (sl.parts == 1) GN_SLAB(16, false);
  else GN_SLAB(16, true);
#undef GN_SLAB
}
template <typename T, int NS>
void launch_bwd_slab(const NormArgs& a, const Slab& sl, hipStream_t s) {
  const dim3 grid(slab_grid(sl)), block((unsigned)sl.threads);
  const int floats = slab_bwd_floats(a.g, sl, NS, ActVec<T>::N, a.dgamma || a.dbeta, a.act == MI_ACT_RELU);
  const unsigned lds = (unsigned)(floats * sizeof(float));
  if (sl.parts > 1) launch_gn_empty(a.words, slab_words(a.g, sl) / 2, s);
#define GN_SLAB(A) launch_bwd_slab_act<T, NS, A>(a, sl, grid, block, lds, s)
  MI_FOR_ACT(a.act, GN_SLAB)
#undef GN_SLAB
}
template <typename T>
int launch_gn_bwd_t(const NormArgs& a, const Slab* sl, hipStream_t s) {
  if (sl != nullptr) {
    if (a.g.n_slots == 1) launch_bwd_slab<T, 1>(a, *sl, s);
    else if (two_pieces<T>(a.g)) launch_bwd_slab<T, ActVec<T>::N / 4>(a, *sl, s);
    else launch_bwd_slab<T, ActVec<T>::N>(a, *sl, s);
    if (a.chan_rows > 1 && (a.dgamma || a.dbeta)) launch_gn_param_grads(a, s);
    return check_hip(hipGetLastError(), "group_norm_act_bwd");
  }
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
