// Dropout from a counter: what every kernel that drops shares.
//
// Whether a unit survives is a function of (seed, offset, unit number) alone, so the mask is never stored: the
// backward pass, a fused kernel and a stand-alone one work it out again.  The generator is Philox4x32-10 (Salmon,
// Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC11): ten rounds of two 32 x 32 -> 64
// multiplies over a 128-bit counter.  Unit e takes 16 of the 128 bits of call e / 8: half e & 1 of word (e >> 1) & 3.
// One call then serves the eight bf16 values of a 16-byte vector: 20 multiplies (4 cycles a wave each) and 20 three-way
// xors (2 cycles), a fifth of the time that the vector's 32 bytes of traffic take (537 MB copied with a call per
// vector: 5.85 TB/s, without: 5.81); with 32 bits a unit it would be two fifths, on top of a norm's own work.  The price: p counts in steps of 2^-16.  The scale follows the rounded p, so the expectation is exact.
#pragma once
#include "common.h"

namespace mi {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

struct DropArgs {
  int on;                      // 0: nothing is dropped
  int per_channel;             // one unit per (image, channel) instead of one per element
  uint32_t keep;               // a unit survives where its 16 bits are below this (0 .. 65536)
  float scale;                 // 65536 / keep
  uint32_t k0, k1;             // seed
  uint64_t offset;
  const int64_t* offset_dev;   // optional, added to offset (read on the device)
};
// Checks and converts the caller's description; null = no dropout.
int make_drop_args(const mi_dropout* d, DropArgs* out);

__device__ __forceinline__ uint64_t drop_offset(const DropArgs& d) {
  return d.offset + (d.offset_dev != nullptr ? (uint64_t)*d.offset_dev : 0);
}
// Four words of call number n, the halves as signed numbers (each has its top bit turned: u < keep then is a signed
// comparison; for two of the words the turn rides in the last round's key).
__device__ __forceinline__ u32x4_t drop_words(uint64_t n, uint64_t offset, uint32_t k0, uint32_t k1) {
  uint32_t a = (uint32_t)n, b = (uint32_t)(n >> 32), c = (uint32_t)offset, d = (uint32_t)(offset >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p = (uint64_t)a * 0xD2511F53u, q = (uint64_t)c * 0xCD9E8D57u;
    const uint32_t turn = r == 9 ? 0x80008000u : 0u;
    a = __builtin_amdgcn_bitop3_b32((uint32_t)(q >> 32), b, k0 ^ turn, 0x96);    // three-way xor
    b = (uint32_t)q;
    c = __builtin_amdgcn_bitop3_b32((uint32_t)(p >> 32), d, k1 ^ turn, 0x96);
    d = (uint32_t)p;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return u32x4_t{a, b ^ 0x80008000u, c, d ^ 0x80008000u};
}
// The keep bits of I vectors of N units, collected two at a time: the saturated difference of a half and `keep` has the
// answer in its sign.  The bits of a thread's vectors are worked out while their loads are in flight and cost a
// register per 32 units until they are used.
template <int I, int N>
struct KeepBits {
  static constexpr int kWords = I * N / 2, kRegs = (kWords + 15) / 16;
  uint32_t r[kRegs];
  // vector i (a literal after unrolling, 0, 1, 2, ...): its units start at e, a multiple of N
  __device__ __forceinline__ void add(int i, const DropArgs& d, uint64_t offset, uint64_t e) {
    const u32x4_t w = drop_words(e >> 3, offset, d.k0, d.k1);
    typedef short s16x2_t __attribute__((ext_vector_type(2)));
    const s16x2_t k = __builtin_bit_cast(s16x2_t, (d.keep ^ 0x8000u) * 0x10001u);
#pragma unroll
    for (int h = 0; h < N / 2; ++h) {
      const uint32_t word = N == 8 ? w[h] : (e & 4 ? w[2 + h] : w[h]);
      const uint32_t t = __builtin_bit_cast(uint32_t, __builtin_elementwise_sub_sat(__builtin_bit_cast(s16x2_t, word), k));
      const int at = i * (N / 2) + h;
      r[at / 16] = at % 16 == 0 ? t & 0x80008000u : r[at / 16] >> 1 | (t & 0x80008000u);
      // the compiler would rather keep every t than read its sign back from here
      if (at % 16 == 15 || at == kWords - 1) asm("" : "+v"(r[at / 16]));
    }
  }
  // all ones where unit j of vector i survives, else zero
  __device__ __forceinline__ uint32_t mask(int i, int j) const {
    const int at = i * (N / 2) + j / 2, in_reg = at / 16 < kRegs - 1 ? 16 : kWords - 16 * (kRegs - 1);
    const int bit = (j & 1) * 16 + 16 - in_reg + at % 16;
    return (uint32_t)((int32_t)(r[at / 16] << (31 - bit)) >> 31);
  }
  // f where the unit survives, +0 where it does not
  __device__ __forceinline__ float kept(int i, int j, float f) const { return __uint_as_float(__float_as_uint(f) & mask(i, j)); }
  // the same for a whole vector of the stored type
  __device__ __forceinline__ u32x4_t kept(int i, u32x4_t v) const {
#pragma unroll
    for (int h = 0; h < 4; ++h) v[h] &= N == 8 ? __builtin_amdgcn_perm(mask(i, 2 * h + 1), mask(i, 2 * h), 0x05040100) : mask(i, h);
    return v;
  }
  __device__ __forceinline__ void keep_all() {
#pragma unroll
    for (int k = 0; k < kRegs; ++k) r[k] = ~0u;
  }
};

// ---------------------------------------------------------------- 16-byte vectors of activations
// N values; in groups of 4 (group h of a bf16 vector: words 2h and 2h + 1), so that a kernel which has little room for
// unpacked values can take one group after the other.
template <typename T> struct ActVec;
template <> struct ActVec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack4(u32x4_t v, int, float* f) {
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = __uint_as_float(v[j]);
  }
  static __device__ __forceinline__ void pack4(const float* f, int, u32x4_t& v) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = __float_as_uint(f[j]);
  }
  static __device__ __forceinline__ void pack4_exact(const float* f, int, u32x4_t& v) { pack4(f, 0, v); }
  static __device__ __forceinline__ void unpack(u32x4_t v, float* f) { unpack4(v, 0, f); }
  static __device__ __forceinline__ u32x4_t pack(const float* f) {
    u32x4_t v;
    pack4(f, 0, v);
    return v;
  }
};
template <> struct ActVec<__bf16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack4(u32x4_t v, int h, float* f) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      f[2 * j] = __uint_as_float(v[2 * h + j] << 16);
      f[2 * j + 1] = __uint_as_float(v[2 * h + j] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ void pack4(const float* f, int h, u32x4_t& v) {   // to nearest even: one rounding, of the stored result
    typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int j = 0; j < 2; ++j) v[2 * h + j] = __builtin_bit_cast(uint32_t, bf16x2_t{(__bf16)f[2 * j], (__bf16)f[2 * j + 1]});
  }
  static __device__ __forceinline__ void pack4_exact(const float* f, int h, u32x4_t& v) {   // the upper halves: of values that are bf16 already, all of them
#pragma unroll
    for (int j = 0; j < 2; ++j) v[2 * h + j] = __builtin_amdgcn_perm(__float_as_uint(f[2 * j + 1]), __float_as_uint(f[2 * j]), 0x07060302);
  }
  // fp32 values as two vectors of 16-bit halves
  static __device__ __forceinline__ void split4(const float* f, int h, u32x4_t& high, u32x4_t& low) {
    pack4_exact(f, h, high);
#pragma unroll
    for (int j = 0; j < 2; ++j) low[2 * h + j] = __builtin_amdgcn_perm(__float_as_uint(f[2 * j + 1]), __float_as_uint(f[2 * j]), 0x05040100);
  }
  static __device__ __forceinline__ void join4(u32x4_t high, u32x4_t low, int h, float* f) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      f[2 * j] = __uint_as_float(__builtin_amdgcn_perm(high[2 * h + j], low[2 * h + j], 0x05040100));
      f[2 * j + 1] = __uint_as_float(__builtin_amdgcn_perm(high[2 * h + j], low[2 * h + j], 0x07060302));
    }
  }
  static __device__ __forceinline__ void unpack(u32x4_t v, float* f) {
    unpack4(v, 0, f);
    unpack4(v, 1, f + 4);
  }
  static __device__ __forceinline__ u32x4_t pack(const float* f) {
    u32x4_t v;
    pack4(f, 0, v);
    pack4(f + 4, 1, v);
    return v;
  }
};
// Streamed: nothing in these kernels comes back to a line it has read or written.
template <typename T> __device__ __forceinline__ u32x4_t load_stream(const T* p) {
  return __builtin_nontemporal_load((const u32x4_t*)p);
}
template <typename T> __device__ __forceinline__ void store_stream(T* p, u32x4_t v) {
  __builtin_nontemporal_store(v, (u32x4_t*)p);
}

}  // namespace mi
