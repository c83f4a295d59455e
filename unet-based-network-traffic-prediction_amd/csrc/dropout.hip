// Dropout on NHWC views: y = residual + keep * scale * x, the mask worked out from a counter (drop.h).
#include "drop.h"

#include <cmath>

namespace mi {

int make_drop_args(const mi_dropout* d, DropArgs* out) {
  *out = DropArgs{};
  if (d == nullptr) return MI_OK;
  MI_REQUIRE(d->p >= 0.0 && d->p <= 1.0, "dropout: p must be between 0 and 1");   // also refuses a NaN
  const uint32_t keep = (uint32_t)std::floor((1.0 - d->p) * 65536.0 + 0.5);
  out->on = keep < 65536;
  out->per_channel = d->per_channel != 0;
  out->keep = keep;
  out->scale = keep ? (float)(65536.0 / keep) : 0.f;
  out->k0 = (uint32_t)d->seed;
  out->k1 = (uint32_t)(d->seed >> 32);
  out->offset = d->offset;
  out->offset_dev = d->offset_dev;
  return MI_OK;
}

struct DropoutArgs {
  const void* x; int xcs, xco;
  const void* r; int rcs, rco;
  void* y; int ycs, yco;
  int64_t total;               // 16-byte vectors
  int C, nv;                   // channels, vectors per pixel
  FastDiv d_nv, d_px;          // by nv, by pixels per image
  DropArgs drop;
};

// HBM-bound: one read (two with a residual) and one write of the tensor.  A workgroup owns kU * 256 consecutive
// vectors and has all its loads in flight before it works the first mask out; one pass and no grid-stride loop
// (a 537 MB copy: 6.33 TB/s against 5.95 with a loop over 4096 workgroups).  Measured: 1024 images of 64x64x32 bf16 87 us for
// 537 MB, 512 of 16x16x64 fp32 with a residual 17.4 us for 101 MB: 6.2 and 5.8 TB/s, the rate of a copy.  The generator
// (one call of ten rounds per 8 units) stays behind the loads.
constexpr int kU = 4;
template <typename T, bool RES>
__global__ __launch_bounds__(256) void dropout_kernel(const DropoutArgs a) {
  constexpr int N = ActVec<T>::N;
  const int64_t base = (int64_t)blockIdx.x * (256 * kU);
  const int64_t px0 = base / a.nv;                               // uniform over the workgroup
  const uint32_t rem = (uint32_t)(base - px0 * a.nv);
  const T* x = (const T*)a.x;
  const T* r = (const T*)a.r;
  T* y = (T*)a.y;
  u32x4_t vx[kU], vr[kU];
  int64_t px[kU];
  int c[kU];
#pragma unroll
  for (int u = 0; u < kU; ++u) {
    const int64_t i = min(base + u * 256 + (int)threadIdx.x, a.total - 1);
    const uint32_t l = rem + (uint32_t)(i - base);
    const uint32_t q = fdiv(l, a.d_nv);
    px[u] = px0 + q;
    c[u] = (int)(l - q * a.nv) * N;
    vx[u] = load_stream(x + px[u] * a.xcs + a.xco + c[u]);
    if (RES) vr[u] = load_stream(r + px[u] * a.rcs + a.rco + c[u]);
  }
  KeepBits<kU, N> keep;
  if (a.drop.on) {
    const uint64_t offset = drop_offset(a.drop);
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const uint64_t row = a.drop.per_channel ? fdiv((uint32_t)px[u], a.d_px) : (uint64_t)px[u];
      keep.add(u, a.drop, offset, row * (uint32_t)(a.nv * N) + c[u]);
    }
  } else {
    keep.keep_all();
  }
#pragma unroll
  for (int u = 0; u < kU; ++u) {
    float f[N], g[N];
    ActVec<T>::unpack(vx[u], f);
#pragma unroll
    for (int j = 0; j < N; ++j) f[j] = keep.kept(u, j, f[j] * a.drop.scale);       // a dropped NaN is a zero
    if (RES) {
      ActVec<T>::unpack(vr[u], g);
#pragma unroll
      for (int j = 0; j < N; ++j) f[j] += g[j];
    }
    if (c[u] + N > a.C) {                                         // padding channels are zero whatever x held there
#pragma unroll
      for (int j = 0; j < N; ++j) f[j] = c[u] + j < a.C ? f[j] : 0.f;
    }
    if (base + u * 256 + (int)threadIdx.x < a.total) store_stream(y + px[u] * a.ycs + a.yco + c[u], ActVec<T>::pack(f));
  }
}

int launch_dropout(const void* x, int xcs, int xco, const void* r, int rcs, int rco, void* y, int ycs, int yco, int B,
                   int H, int W, int C, const mi_dropout* drop, int dtype, hipStream_t s) {
  DropoutArgs a{};
  int rc = make_drop_args(drop, &a.drop);
  if (rc) return rc;
  if (!a.drop.on) a.drop.scale = 1.f;
  a.x = x; a.xcs = xcs; a.xco = xco;
  a.r = r; a.rcs = rcs; a.rco = rco;
  a.y = y; a.ycs = ycs; a.yco = yco;
  a.C = C;
  a.nv = pad_ch(C) / (dtype == MI_BF16 ? 8 : 4);
  a.total = (int64_t)B * H * W * a.nv;
  if (a.total == 0) return MI_OK;
  a.d_nv = make_fastdiv(a.nv);
  a.d_px = make_fastdiv(H * W);
  const int64_t blocks = (a.total + 256 * kU - 1) / (256 * kU);
  MI_REQUIRE(blocks < (1ll << 24), "dropout: tensor too large");           // a launch holds less than 2^32 threads
  const dim3 grid((unsigned)blocks), block(256);
  if (dtype == MI_BF16) {
    if (r) hipLaunchKernelGGL((dropout_kernel<__bf16, true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((dropout_kernel<__bf16, false>), grid, block, 0, s, a);
  } else {
    if (r) hipLaunchKernelGGL((dropout_kernel<float, true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((dropout_kernel<float, false>), grid, block, 0, s, a);
  }
  return check_hip(hipGetLastError(), "dropout");
}

}  // namespace mi
