// Sliding-window operators: a cache of the first `sinks` and the last `window` tokens of every sequence, in 16 or in 4 bits.
//
// A token at position p sees position j if j <= p and (j > p - window or j < sinks).
//
// Rows of a kv row's cache: `sp` rows (sinks rounded up to 16) for the first tokens, then a ring of `ring` rows (window
// rounded up to 16): token t < sinks lies in row t, any other in row sp + (t - sinks) % ring.
//
// 16 bits: k and v are bf16 [kv row][rows][D].
// 4 bits: one array of blocks of 16 rows, [kv row][rows / 16][18 D bytes]: key codes (16 x D/2 bytes), value codes, key
// scales, value scales.  A group of 32 channels shares a scale s = max|x| / 6 rounded to 6 significant bits (bf16); a value
// is held as the nearest e2m1 number (0, .5, 1, 1.5, 2, 3, 4, 6, either sign) to x / s, ties to even.  e2m1 has two
// significant bits: code * s is a bf16 number, what is read back is exactly what the attention uses.  A group with an infinity
// or NaN gets the scale NaN and reads back as NaN; one whose scale would be below the smallest normal number is all zeros.
// Order inside a row, made for the fragments of the token attention's warp-level MMAs (thread (g, t) = (lane / 4, lane % 4)):
//   key codes: 32-bit word t * (D/32) + n holds channels 32 n + 8 t .. + 7 of group n (nibble i = channel i): a thread's
//     channels of all groups are contiguous, and one k-step of 16 channels lies inside one group
//   value codes: 16-bit unit g * (D/32) + n holds channels 32 n + 4 g .. + 3
//   key scales: [row][group];  value scales: [pair of rows][group][2]
#pragma once

#include <cuda_fp16.h>

#include <atomic>

#include "kvm_common.cuh"
#include "kvm_pdl.cuh"
#include "kvm_tc.cuh"

namespace kvm {

struct WindowDev {
  int batch, Hkv, window, sinks, sp, ring, rows;  // rows = sp + ring
  bf16* k;                                        // 16 bits
  bf16* v;
  unsigned char* blocks;                          // 4 bits
  __host__ __device__ __forceinline__ int row_of(int t) const { return t < sinks ? t : sp + (t - sinks) % ring; }
  // rows [0, live) are looked at for a sequence of n tokens
  __host__ __device__ __forceinline__ int live(int n) const { return n <= 0 ? 0 : (n <= sinks ? n : sp + min(ring, n - sinks)); }
};

// Lengths (or positions) of a batch: a device array, or one number for all.
struct SeqInts {
  const int* dev;
  int all;
  __device__ __forceinline__ int at(int b) const { return dev ? dev[b] : all; }
};

// byte offsets inside a block of 16 rows
template <int D>
struct Block4 {
  static constexpr int kKeys = 0, kValues = 8 * D, kKeyScales = 16 * D, kValueScales = 17 * D, kBytes = 18 * D;
  static constexpr int kGroups = D / 32;
};

// The scale of a group from the largest of its magnitudes' bf16 bit patterns: bf16 bits, and a reciprocal for the products
// below.  m / 6 is formed as a product and rounded to 16 significant bits first: m has 8 of them, so a quotient that is not
// on the border between two 6-bit numbers is at least 2^-11 away from it, one that is comes out exactly.
__device__ __forceinline__ unsigned short group_scale(unsigned amax_bits, float& inv) {
  inv = 0.f;
  if (amax_bits >= 0x7f80u) return 0xffffu;  // infinity or NaN (as a 16-bit integer below every scale: a maximum of scales passes it by)
  unsigned u = __float_as_uint(__uint_as_float(amax_bits << 16) * (1.0f / 6.0f));
  u = (u + 0x80u) & ~0xffu;
  u = (u + 0x1ffffu + ((u >> 18) & 1u)) & ~0x3ffffu;
  if (u < 0x00800000u) return 0;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(__uint_as_float(u)));
  return (unsigned short)(u >> 16);
}
// x / s to within 2^-14, exact where it lies on the border between two levels: x has 8 and s 6 significant bits, so a
// quotient off the border is at least 2^-10 away from it (255 / 1024 beside 1 / 4, the nearest of all mantissas and borders), and
// the product with the reciprocal errs by less than 2^-19.  (A sum in [512, 1024) is a multiple of 2^-14.)
__device__ __forceinline__ float2 levels_of(unsigned x2, float inv) {
  return __fadd2_rn(__ffma2_rn(unpack_bf16(x2), make_float2(inv, inv), make_float2(768.f, 768.f)), make_float2(-768.f, -768.f));
}

// levels -> e2m1 codes (the first in the lowest nibble), nearest, ties to even, saturating
__device__ __forceinline__ unsigned e2m1x4(float2 a, float2 b) {
  unsigned r;
  asm("{\n\t.reg .b8 x, y, z;\n\tcvt.rn.satfinite.e2m1x2.f32 x, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 y, %4, %3;\n\tcvt.u8.u32 z, 0;\n\t"
      "mov.b32 %0, {x, y, z, z};\n\t}"
      : "=r"(r)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ unsigned e2m1x8(float2 a, float2 b, float2 c, float2 d) {
  unsigned r;
  asm("{\n\t.reg .b8 x, y, z, w;\n\tcvt.rn.satfinite.e2m1x2.f32 x, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 y, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 z, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 w, %8, %7;\n\tmov.b32 %0, {x, y, z, w};\n\t}"
      : "=r"(r)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y), "f"(d.x), "f"(d.y));
  return r;
}
// 8 codes -> 4 x f16x2 (byte i of the word -> o[i], low nibble in the low half)
__device__ __forceinline__ void e2m1_to_f16x2(uint32_t w, uint32_t& o0, uint32_t& o1, uint32_t& o2, uint32_t& o3) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\tcvt.rn.f16x2.e2m1x2 %1, b1;\n\tcvt.rn.f16x2.e2m1x2 %2, b2;\n\tcvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(o0), "=r"(o1), "=r"(o2), "=r"(o3)
      : "r"(w));
}

// What does not change between launches on a device, asked for once (device ordinals below 64, checked where the calls enter).
inline int window_sm_count() {
  static std::atomic<int> count[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  int n = count[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    count[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}
// Raises a kernel's limit of dynamic shared memory, once per device (`done`: the kernel's own bits).
template <typename F>
inline cudaError_t raise_smem_limit(F kern, int bytes, std::atomic<unsigned long long>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (done.load(std::memory_order_acquire) >> (dev & 63) & 1) return cudaSuccess;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(1ull << (dev & 63), std::memory_order_release);
  return e;
}

}  // namespace kvm
