// Writing tokens into a window cache (in 4 bits: quantised on the way) and reading back what it holds, in order.
// Both are one pass over memory.
#include <algorithm>

#include "kvm_window.cuh"

namespace kvm {

namespace {

constexpr int kStoreThreads = 256;
constexpr int kRowsPerZ = 32768;  // kv rows along y of the grid, the rest along z
constexpr int kStoreUnroll = 4;  // rows in flight per thread

__device__ __forceinline__ unsigned abs_max_bits(const uint4& x) {
  unsigned m = 0;
  const unsigned w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
  return max(m & 0xffffu, m >> 16);
}

// ring place of the token that is `i`-th behind the sinks (before them: where it would be), once per thread
__device__ __forceinline__ int ring_place(int i, int ring) {
  const int r = i % ring;
  return r < 0 ? r + ring : r;
}

}  // namespace

// Codes of the 8 channels [8 c, 8 c + 8) of a row, one thread of the row's D/8 consecutive ones, into row `rr` of the block
// (4 threads hold a group of 32).
template <int D>
__device__ __forceinline__ void store_row4(unsigned char* block, int rr, int c, bool value, bool write, const uint4& x) {
  constexpr int NG = Block4<D>::kGroups;
  unsigned m = abs_max_bits(x);
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
  float inv;
  const unsigned short s = group_scale(m, inv);
  unsigned code = e2m1x8(levels_of(x.x, inv), levels_of(x.y, inv), levels_of(x.z, inv), levels_of(x.w, inv));
  if (m >= 0x7f80u) code = 0;
  const int n = c >> 2, u = c & 3;  // group, eighth channels inside it
  if (value) {
    // this thread holds units g = 2 u, 2 u + 1 of group n; with the neighbouring group's thread it forms 32-bit words
    if (NG > 1) {
      const unsigned other = __shfl_xor_sync(0xffffffffu, code, 4);
      const unsigned word = (n & 1) ? __byte_perm(other, code, 0x7632) : __byte_perm(code, other, 0x5410);
      if (write) *reinterpret_cast<unsigned*>(block + Block4<D>::kValues + rr * (D / 2) + (2 * u + (n & 1)) * (2 * NG) + (n >> 1) * 4) = word;
    } else if (write) {
      *reinterpret_cast<unsigned*>(block + Block4<D>::kValues + rr * (D / 2) + 4 * u) = code;
    }
  } else if (write) {
    *reinterpret_cast<unsigned*>(block + Block4<D>::kKeys + rr * (D / 2) + (u * NG + n) * 4) = code;
  }
  if (u == 0 && write) {
    unsigned short* sc = reinterpret_cast<unsigned short*>(block + (value ? Block4<D>::kValueScales : Block4<D>::kKeyScales));
    sc[value ? (rr >> 1) * (2 * NG) + 2 * n + (rr & 1) : rr * NG + n] = s;
  }
}

// Tokens [position, position + length) of every sequence; of a sequence longer than the cache only those are written that
// are still in it behind the last one (no two tokens of a call share a row).
template <int D, int BITS>
__global__ void __launch_bounds__(kStoreThreads)
kvm_window_write_kernel(WindowDev W, Tensor4 k, Tensor4 v, int n_tokens, SeqInts positions,
                        SeqInts lengths) {
  constexpr int TPR = D / 8;                          // threads per row
  constexpr int RPI = kStoreThreads / TPR / 2;        // rows per iteration (keys and values side by side)
  pdl_wait();
  const int kvrow = blockIdx.z * kRowsPerZ + blockIdx.y;
  if (kvrow >= W.batch * W.Hkv) return;
  const int b = kvrow / W.Hkv, h = kvrow % W.Hkv;
  const int pos = positions.at(b), len = min(lengths.at(b), n_tokens);
  if (pos < 0 || len <= 0) return;
  const int tid = threadIdx.x, c = tid % TPR, vr = tid / TPR;
  const bool value = vr >= RPI;
  const int r0 = vr - (value ? RPI : 0);
  const Tensor4& src = value ? v : k;
  const long long end = (long long)pos + len, first = end - W.ring;  // tokens from `first` on stay in the ring
  const int base = (int)blockIdx.x * (RPI * kStoreUnroll);
  if (base >= len || ((long long)pos + base >= W.sinks && (long long)pos + base + RPI * kStoreUnroll <= first)) return;
  uint4 x[kStoreUnroll];
#pragma unroll
  for (int i = 0; i < kStoreUnroll; ++i) {
    const int tok = base + i * RPI + r0;
    x[i] = tok < len ? *reinterpret_cast<const uint4*>(src.row(b, h, tok) + c * 8) : make_uint4(0, 0, 0, 0);
  }
  const int ring0 = ring_place(pos + base - W.sinks, W.ring);
#pragma unroll
  for (int i = 0; i < kStoreUnroll; ++i) {
    const int tok = base + i * RPI + r0;
    const long long p = (long long)pos + tok;
    const bool write = tok < len && (p < W.sinks || p >= first);
    int r = ring0 + i * RPI + r0;
    if (r >= W.ring) r = W.ring >= RPI * kStoreUnroll ? r - W.ring : r % W.ring;
    r = !write ? 0 : (p < W.sinks ? (int)p : W.sp + r);
    if (BITS == 16) {
      if (write) *reinterpret_cast<uint4*>((value ? W.v : W.k) + ((size_t)kvrow * W.rows + r) * D + c * 8) = x[i];
    } else {
      store_row4<D>(W.blocks + ((size_t)kvrow * (W.rows / 16) + (r >> 4)) * Block4<D>::kBytes, r & 15, c, value, write, x[i]);
    }
  }
}

// Rows i < min(n, sinks + window) of the output: the first sinks tokens, then the last `window`; zeros behind them.
template <int D, int BITS>
__global__ void __launch_bounds__(kStoreThreads)
kvm_window_read_kernel(WindowDev W, SeqInts lengths, bf16* __restrict__ k_out, bf16* __restrict__ v_out) {
  constexpr int TPR = D / 8;
  constexpr int RPI = kStoreThreads / TPR / 2;
  constexpr int NG = Block4<D>::kGroups;
  pdl_wait();
  const int keep = W.sinks + W.window;
  const int kvrow = blockIdx.z * kRowsPerZ + blockIdx.y;
  if (kvrow >= W.batch * W.Hkv) return;
  const int b = kvrow / W.Hkv;
  const int n = max(lengths.at(b), 0), held = min(n, keep);
  const int tid = threadIdx.x, c = tid % TPR, vr = tid / TPR;
  const bool value = vr >= RPI;
  const int r0 = vr - (value ? RPI : 0);
  const int base = (int)blockIdx.x * (RPI * kStoreUnroll);
  if (base >= keep) return;
  const int ring0 = ring_place(n - held + base - W.sinks, W.ring);
  uint4 x[kStoreUnroll];
#pragma unroll
  for (int i = 0; i < kStoreUnroll; ++i) {
    const int at = base + i * RPI + r0;
    x[i] = make_uint4(0, 0, 0, 0);
    if (at >= held) continue;
    int r = ring0 + i * RPI + r0;
    if (r >= W.ring) r = W.ring >= RPI * kStoreUnroll ? r - W.ring : r % W.ring;
    r = at < W.sinks ? at : W.sp + r;
    if (BITS == 16) {
      x[i] = *reinterpret_cast<const uint4*>((value ? W.v : W.k) + ((size_t)kvrow * W.rows + r) * D + c * 8);
    } else {
      const unsigned char* block = W.blocks + ((size_t)kvrow * (W.rows / 16) + (r >> 4)) * Block4<D>::kBytes;
      const int rr = r & 15, g = c >> 2, u = c & 3;
      unsigned code;
      if (value) {
        const unsigned char* units = block + Block4<D>::kValues + rr * (D / 2) + g * 2;
        code = *reinterpret_cast<const unsigned short*>(units + 2 * u * (2 * NG)) |
               (unsigned)*reinterpret_cast<const unsigned short*>(units + (2 * u + 1) * (2 * NG)) << 16;
      } else {
        code = *reinterpret_cast<const unsigned*>(block + Block4<D>::kKeys + rr * (D / 2) + (u * NG + g) * 4);
      }
      const unsigned short* sc = reinterpret_cast<const unsigned short*>(block + (value ? Block4<D>::kValueScales : Block4<D>::kKeyScales));
      const float s = __uint_as_float((unsigned)sc[value ? (rr >> 1) * (2 * NG) + 2 * g + (rr & 1) : rr * NG + g] << 16);
      x[i].x = code;
      x[i].y = __float_as_uint(s);
    }
  }
#pragma unroll
  for (int i = 0; i < kStoreUnroll; ++i) {
    const int at = base + i * RPI + r0;
    if (at >= keep) continue;
    uint4 y = x[i];
    if (BITS == 4) {
      const float s = __uint_as_float(x[i].y);
      uint32_t o[4];
      e2m1_to_f16x2(x[i].x, o[0], o[1], o[2], o[3]);
      uint32_t z[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&o[j]));
        const float2 y2 = __fmul2_rn(f, make_float2(s, s));  // exact
        z[j] = pack_bf16(y2.x, y2.y);
      }
      y = make_uint4(z[0], z[1], z[2], z[3]);
    }
    *reinterpret_cast<uint4*>((value ? v_out : k_out) + ((size_t)kvrow * keep + at) * D + c * 8) = y;
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
  if (!store_grid(W, n_tokens, kStoreThreads / (D / 8) / 2 * kStoreUnroll, grid)) return cudaErrorInvalidValue;
  return launch_pdl(kvm_window_write_kernel<D, BITS>, grid, dim3(kStoreThreads), 0, stream, true, W, k, v, n_tokens, positions, lengths);
}
template <int D, int BITS>
cudaError_t launch_read(const WindowDev& W, SeqInts lengths, bf16* k_out, bf16* v_out, cudaStream_t stream) {
  dim3 grid;
  if (!store_grid(W, W.sinks + W.window, kStoreThreads / (D / 8) / 2 * kStoreUnroll, grid)) return cudaErrorInvalidValue;
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
