// Writing tokens into a window cache (in 4 bits: quantised on the way) and reading back what it holds, in order.
// Both are one pass over memory.
#include <algorithm>

#include "kvm_window.cuh"

namespace kvm {

namespace {

constexpr int kStoreThreads = 256;
constexpr int kRowsPerZ = 32768;  // kv rows along y of the grid, the rest along z
constexpr int kStoreUnroll = 4;  // rows in flight per thread

// ring place of the token that is `i`-th behind the sinks (before them: where it would be), once per thread
__device__ __forceinline__ int ring_place(int i, int ring) {
  const int r = i % ring;
  return r < 0 ? r + ring : r;
}

}  // namespace

// A thread's place: piece c (8 channels) of a row, keys in the first half of the block's threads, values in the second, rows
// kRowsPerIter apart.
template <int D>
struct Piece {
  static constexpr int kPerRow = D / 8, kRowsPerIter = kStoreThreads / kPerRow / 2, kTile = kRowsPerIter * kStoreUnroll;
  int c, r0;
  bool value;
  __device__ __forceinline__ Piece() {
    const int half = threadIdx.x & (kStoreThreads / 2 - 1);
    c = half % kPerRow;
    r0 = half / kPerRow;
    value = threadIdx.x >= kStoreThreads / 2;
  }
  // 4 bits: byte of the thread's 8 codes in row 0 of a block, and of its group's scale
  __device__ __forceinline__ int code_at() const {
    constexpr int NG = Block4<D>::kGroups;
    const int n = c >> 2, u = c & 3;  // group, eighth channels inside it
    if (!value) return Block4<D>::kKeys + (u * NG + n) * 4;
    // (units g = 2 u, 2 u + 1 of group n; with the neighbouring group's thread it forms 32-bit words)
    return Block4<D>::kValues + (NG > 1 ? (2 * u + (n & 1)) * (2 * NG) + (n >> 1) * 4 : 4 * u);
  }
  __device__ __forceinline__ int scale_at() const { return value ? Block4<D>::kValueScales + (c >> 2) * 4 : Block4<D>::kKeyScales + (c >> 2) * 2; }
  __device__ __forceinline__ int scale_row(int rr) const {
    constexpr int NG = Block4<D>::kGroups;
    return value ? (rr >> 1) * (4 * NG) + (rr & 1) * 2 : rr * (2 * NG);
  }
};

// Tokens [position, position + length) of every sequence; of a sequence longer than the cache only those are written that
// are still in it behind the last one (no two tokens of a call share a row).
template <int D, int BITS>
__global__ void __launch_bounds__(kStoreThreads)
kvm_window_write_kernel(WindowDev W, Tensor4 k, Tensor4 v, int n_tokens, SeqInts positions, SeqInts lengths) {
  constexpr int RPI = Piece<D>::kRowsPerIter, NG = Block4<D>::kGroups;
  pdl_wait();
  const int kvrow = blockIdx.z * kRowsPerZ + blockIdx.y;
  if (kvrow >= W.batch * W.Hkv) return;
  const int b = kvrow / W.Hkv, h = kvrow % W.Hkv;
  const int pos = positions.at(b), len = min(lengths.at(b), n_tokens);
  const int base = (int)blockIdx.x * Piece<D>::kTile;
  if (pos < 0 || base >= len || pos > 0x7fffffff - len) return;  // (positions that are not representable: left alone)
  const int first = pos + len - W.ring;  // tokens from there on stay in the ring (positions stay below 2^31)
  if (pos + base >= W.sinks && (long long)pos + base + Piece<D>::kTile <= first) return;
  const Piece<D> at;
  const bf16* src = at.value ? v.row(b, h, base + at.r0) + at.c * 8 : k.row(b, h, base + at.r0) + at.c * 8;
  const long long step = (at.value ? v.st : k.st) * RPI;
  uint4 x[kStoreUnroll];
#pragma unroll
  for (int i = 0; i < kStoreUnroll; ++i) {
    x[i] = base + at.r0 + i * RPI < len ? *reinterpret_cast<const uint4*>(src) : make_uint4(0, 0, 0, 0);
    src += step;
  }
  const int ring0 = ring_place(pos + base - W.sinks, W.ring) + at.r0, p0 = pos + base + at.r0;
  bf16* rows16 = (at.value ? W.v : W.k) + (size_t)kvrow * W.rows * D + at.c * 8;
  unsigned char* blocks = W.blocks + (size_t)kvrow * (W.rows / 16) * Block4<D>::kBytes;
  const int code_at = at.code_at(), scale_at = at.scale_at();
  const bool odd = (at.c >> 2) & 1, first_of_group = (at.c & 3) == 0;
#pragma unroll
  for (int i = 0; i < kStoreUnroll; ++i) {
    const int p = p0 + i * RPI;
    const bool write = base + at.r0 + i * RPI < len && (p < W.sinks || p >= first);
    int r = ring0 + i * RPI;
    if (r >= W.ring) r = W.ring >= Piece<D>::kTile ? r - W.ring : r % W.ring;
    r = p < W.sinks ? p : W.sp + r;
    if (BITS == 16) {
      if (write) *reinterpret_cast<uint4*>(rows16 + (size_t)r * D) = x[i];
      continue;
    }
    unsigned m = __vmaxu2(__vmaxu2(x[i].x & 0x7fff7fffu, x[i].y & 0x7fff7fffu), __vmaxu2(x[i].z & 0x7fff7fffu, x[i].w & 0x7fff7fffu));
    m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 2));
    m = max(m & 0xffffu, m >> 16);
    float inv;
    const unsigned short s = group_scale(m, inv);
    unsigned code = e2m1x8(levels_of(x[i].x, inv), levels_of(x[i].y, inv), levels_of(x[i].z, inv), levels_of(x[i].w, inv));
    if (m >= 0x7f80u) code = 0;
    if (at.value && NG > 1) {
      const unsigned other = __shfl_xor_sync(0xffffffffu, code, 4);
      code = odd ? __byte_perm(other, code, 0x7632) : __byte_perm(code, other, 0x5410);
    }
    if (write) {
      unsigned char* block = blocks + (size_t)(unsigned)(r >> 4) * (unsigned)Block4<D>::kBytes;
      const int rr = r & 15;
      *reinterpret_cast<unsigned*>(block + rr * (D / 2) + code_at) = code;
      if (first_of_group) *reinterpret_cast<unsigned short*>(block + at.scale_row(rr) + scale_at) = s;
    }
  }
}

// Rows i < min(n, sinks + window) of the output: the first sinks tokens, then the last `window`; zeros behind them.
template <int D, int BITS>
__global__ void __launch_bounds__(kStoreThreads)
kvm_window_read_kernel(WindowDev W, SeqInts lengths, bf16* __restrict__ k_out, bf16* __restrict__ v_out) {
  constexpr int RPI = Piece<D>::kRowsPerIter, NG = Block4<D>::kGroups;
  pdl_wait();
  const int kvrow = blockIdx.z * kRowsPerZ + blockIdx.y;
  if (kvrow >= W.batch * W.Hkv) return;
  const int b = kvrow / W.Hkv;
  const int keep = W.sinks + W.window, n = max(lengths.at(b), 0), held = min(n, keep);
  const int base = (int)blockIdx.x * Piece<D>::kTile;
  if (base >= keep) return;
  const Piece<D> at;
  const int out0 = base + at.r0, ring0 = ring_place(n - held + base - W.sinks, W.ring) + at.r0;
  const bf16* rows16 = (at.value ? W.v : W.k) + (size_t)kvrow * W.rows * D + at.c * 8;
  const unsigned char* blocks = W.blocks + (size_t)kvrow * (W.rows / 16) * Block4<D>::kBytes;
  const int code_at = at.code_at(), scale_at = at.scale_at();
  const bool odd = (at.c >> 2) & 1;
  uint4 x[kStoreUnroll];  // 4 bits: codes and scale
#pragma unroll
  for (int i = 0; i < kStoreUnroll; ++i) {
    const int to = out0 + i * RPI;
    x[i] = make_uint4(0, 0, 0, 0);
    if (to >= held) continue;
    int r = ring0 + i * RPI;
    if (r >= W.ring) r = W.ring >= Piece<D>::kTile ? r - W.ring : r % W.ring;
    r = to < W.sinks ? to : W.sp + r;
    if (BITS == 16) {
      x[i] = *reinterpret_cast<const uint4*>(rows16 + (size_t)r * D);
    } else {
      const unsigned char* block = blocks + (size_t)(unsigned)(r >> 4) * (unsigned)Block4<D>::kBytes;
      const int rr = r & 15;
      x[i].x = *reinterpret_cast<const unsigned*>(block + rr * (D / 2) + code_at);
      x[i].y = (unsigned)*reinterpret_cast<const unsigned short*>(block + at.scale_row(rr) + scale_at) << 16;
    }
  }
  bf16* dst = (at.value ? v_out : k_out) + ((size_t)kvrow * keep + out0) * D + at.c * 8;
#pragma unroll
  for (int i = 0; i < kStoreUnroll; ++i) {
    uint4 y = x[i];
    if (BITS == 4) {
      unsigned code = x[i].x;
      if (at.value && NG > 1) {  // words of two groups' units back into a thread's own 8 channels
        const unsigned other = __shfl_xor_sync(0xffffffffu, code, 4);
        code = odd ? __byte_perm(other, code, 0x7632) : __byte_perm(code, other, 0x5410);
      }
      const float2 s = make_float2(__uint_as_float(x[i].y), __uint_as_float(x[i].y));
      uint32_t o[4], z[4];
      e2m1_to_f16x2(code, o[0], o[1], o[2], o[3]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = __fmul2_rn(__half22float2(*reinterpret_cast<const __half2*>(&o[j])), s);  // (a bf16 number)
        z[j] = pack_bf16(f.x, f.y);
      }
      y = make_uint4(z[0], z[1], z[2], z[3]);
    }
    if (out0 + i * RPI < keep) *reinterpret_cast<uint4*>(dst + (size_t)(i * RPI) * D) = y;
  }
}

namespace {

// tiles x kv rows
bool store_grid(const WindowDev& W, int n, int rows, dim3& grid) {
  const long long kvrows = (long long)W.batch * W.Hkv, z = (kvrows + kRowsPerZ - 1) / kRowsPerZ;
  grid = dim3((n + rows - 1) / rows, (unsigned)std::min<long long>(kvrows, kRowsPerZ), (unsigned)z);
  return z < 65536;
}
template <int D, int BITS>
cudaError_t launch_write(const WindowDev& W, Tensor4 k, Tensor4 v, int n_tokens, SeqInts positions, SeqInts lengths, cudaStream_t stream) {
  dim3 grid;
  if (!store_grid(W, n_tokens, Piece<D>::kTile, grid)) return cudaErrorInvalidValue;
  return launch_pdl(kvm_window_write_kernel<D, BITS>, grid, dim3(kStoreThreads), 0, stream, true, W, k, v, n_tokens, positions, lengths);
}
template <int D, int BITS>
cudaError_t launch_read(const WindowDev& W, SeqInts lengths, bf16* k_out, bf16* v_out, cudaStream_t stream) {
  dim3 grid;
  if (!store_grid(W, W.sinks + W.window, Piece<D>::kTile, grid)) return cudaErrorInvalidValue;
  return launch_pdl(kvm_window_read_kernel<D, BITS>, grid, dim3(kStoreThreads), 0, stream, true, W, lengths, k_out, v_out);
}

}  // namespace

#define KVM_WINDOW_DISPATCH(fn, ...)                                                    \
  (bits == 4 ? (D == 128 ? fn<128, 4>(__VA_ARGS__) : D == 64 ? fn<64, 4>(__VA_ARGS__) : fn<32, 4>(__VA_ARGS__)) \
             : (D == 128 ? fn<128, 16>(__VA_ARGS__) : D == 64 ? fn<64, 16>(__VA_ARGS__) : fn<32, 16>(__VA_ARGS__)))

cudaError_t window_write_dispatch(int D, int bits, const WindowDev& W, Tensor4 k, Tensor4 v, int n_tokens, SeqInts positions,
                                  SeqInts lengths, cudaStream_t stream) {
  return KVM_WINDOW_DISPATCH(launch_write, W, k, v, n_tokens, positions, lengths, stream);
}
cudaError_t window_read_dispatch(int D, int bits, const WindowDev& W, SeqInts lengths, bf16* k_out, bf16* v_out, cudaStream_t stream) {
  return KVM_WINDOW_DISPATCH(launch_read, W, lengths, k_out, v_out, stream);
}

}  // namespace kvm
