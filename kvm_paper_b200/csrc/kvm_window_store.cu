// Writing tokens into a window cache (in 4 bits: quantised on the way) and reading back what it holds, in order.
// Both are one pass over memory and bound by it: 4 x 8192 tokens of 16 heads x 128, in 4 bits written in 59 us (5.9 TB/s) and
// read in 62 us (5.5 TB/s; its instructions keep 75 % of the issue slots busy), in 16 bits in 82 and 80 us (6.6 TB/s).
#include <algorithm>

#include "kvm_window.cuh"

namespace kvm {

namespace {

constexpr int kStoreThreads = 256;
constexpr int kRowsPerZ = 32768;  // kv rows along y of the grid, the rest along z
constexpr int kStoreUnroll = 4;  // pieces of 8 channels in flight per thread
constexpr int kGroupUnroll = 2;  // groups of 32 channels in flight per thread

// ring place of the token that is `i`-th behind the sinks (before them: where it would be), once per thread
__device__ __forceinline__ int ring_place(int i, int ring) {
  const int r = i % ring;
  return r < 0 ? r + ring : r;
}
// cache row of the token (or row in order) t that lies `place` behind the ring's start, at most TILE - 1 behind its end
template <int TILE>
__device__ __forceinline__ int row_at(const WindowDev& W, int t, int place) {
  if (place >= W.ring) place = W.ring >= TILE ? place - W.ring : place % W.ring;
  return t < W.sinks ? t : W.sp + place;
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
// are still in it behind the last one (no two tokens of a call share a row).  What both widths share:
struct WriteRange {
  int kvrow, b, h, pos, len, first;  // first: tokens from there on stay in the ring
  bool some;                         // does this block write anything?
  __device__ __forceinline__ WriteRange(const WindowDev& W, int n_tokens, const SeqInts& positions, const SeqInts& lengths, int base, int tile) {
    kvrow = blockIdx.z * kRowsPerZ + blockIdx.y;
    some = false;
    if (kvrow >= W.batch * W.Hkv) return;
    b = kvrow / W.Hkv;
    h = kvrow % W.Hkv;
    pos = positions.at(b);
    len = min(lengths.at(b), n_tokens);
    if (pos < 0 || base >= len || pos > 0x7fffffff - len) return;  // (positions that are not representable: left alone)
    first = pos + len - W.ring;
    some = pos + base < W.sinks || (long long)pos + base + tile > first;
  }
};

template <int D>
__global__ void __launch_bounds__(kStoreThreads)
kvm_window_write16_kernel(WindowDev W, Tensor4 k, Tensor4 v, int n_tokens, SeqInts positions, SeqInts lengths) {
  constexpr int RPI = Piece<D>::kRowsPerIter;
  pdl_wait();
  const int base = (int)blockIdx.x * Piece<D>::kTile;
  const WriteRange w(W, n_tokens, positions, lengths, base, Piece<D>::kTile);
  if (!w.some) return;
  const Piece<D> at;
  const bf16* src = (at.value ? v : k).row(w.b, w.h, base + at.r0) + at.c * 8;
  const long long step = (at.value ? v.st : k.st) * RPI;
  uint4 x[kStoreUnroll];
#pragma unroll
  for (int i = 0; i < kStoreUnroll; ++i) {
    x[i] = base + at.r0 + i * RPI < w.len ? *reinterpret_cast<const uint4*>(src) : make_uint4(0, 0, 0, 0);
    src += step;
  }
  const int ring0 = ring_place(w.pos + base - W.sinks, W.ring) + at.r0;
  bf16* rows16 = (at.value ? W.v : W.k) + (size_t)w.kvrow * W.rows * D + at.c * 8;
#pragma unroll
  for (int i = 0; i < kStoreUnroll; ++i) {
    const int in = base + at.r0 + i * RPI;
    if (in >= w.len) continue;
    const int p = w.pos + in;
    if (p >= W.sinks && p < w.first) continue;
    *reinterpret_cast<uint4*>(rows16 + (size_t)row_at<Piece<D>::kTile>(W, p, ring0 + i * RPI) * D) = x[i];
  }
}

// 4 bits: a thread quantises whole groups, one of a row of keys or values, so that a group's scale and a row's place are
// worked out once per 32 channels.  (With 8 channels per thread the instructions bind, 88 % of the issue slots: 81 us for 4 x 8192
// tokens of 16 heads x 128 instead of 59.)  The loads of a warp are strided, every sector is used whole; the codes are exchanged between the lanes of a row, so
// that each stores 16 bytes in the order of the cache.
template <int D>
__global__ void __launch_bounds__(kStoreThreads)
kvm_window_write4_kernel(WindowDev W, Tensor4 k, Tensor4 v, int n_tokens, SeqInts positions, SeqInts lengths) {
  constexpr int NG = Block4<D>::kGroups, RPI = kStoreThreads / 2 / NG, kTile = RPI * kGroupUnroll;
  constexpr unsigned kAll = 0xffffffffu;
  pdl_wait();
  const int base = (int)blockIdx.x * kTile;
  const WriteRange w(W, n_tokens, positions, lengths, base, kTile);
  if (!w.some) return;
  const bool value = threadIdx.x >= kStoreThreads / 2;
  const int n = threadIdx.x % NG, r0 = (threadIdx.x & (kStoreThreads / 2 - 1)) / NG;  // group, row
  const Tensor4& from = value ? v : k;
  uint4 x[kGroupUnroll][4];
#pragma unroll
  for (int i = 0; i < kGroupUnroll; ++i) {
    const int in = base + r0 + i * RPI;
    const uint4* src = reinterpret_cast<const uint4*>(from.row(w.b, w.h, in) + n * 32);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[i][j] = in < w.len ? src[j] : make_uint4(0, 0, 0, 0);
  }
  const int ring0 = ring_place(w.pos + base - W.sinks, W.ring) + r0;
  unsigned char* blocks = W.blocks + (size_t)w.kvrow * (W.rows / 16) * Block4<D>::kBytes;
#pragma unroll
  for (int i = 0; i < kGroupUnroll; ++i) {
    unsigned m = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const unsigned a = __vmaxu2(x[i][j].x & 0x7fff7fffu, x[i][j].y & 0x7fff7fffu), b = __vmaxu2(x[i][j].z & 0x7fff7fffu, x[i][j].w & 0x7fff7fffu);
      m = __vmaxu2(m, __vmaxu2(a, b));
    }
    m = max(m & 0xffffu, m >> 16);
    float inv;
    const unsigned short s = group_scale(m, inv);
    unsigned c[4];  // codes of channels 8 j .. 8 j + 7
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      c[j] = e2m1x8(levels_of(x[i][j].x, inv), levels_of(x[i][j].y, inv), levels_of(x[i][j].z, inv), levels_of(x[i][j].w, inv));
      if (m >= 0x7f80u) c[j] = 0;
    }
    // lane n of a row: words c[4 n / NG ..] of all its groups, by exchanges of halves
    if constexpr (NG == 4) {
      const bool odd = n & 1, high = n & 2;
      unsigned y = __shfl_xor_sync(kAll, odd ? c[0] : c[1], 1), z = __shfl_xor_sync(kAll, odd ? c[2] : c[3], 1);
      if (odd) { c[0] = y; c[2] = z; } else { c[1] = y; c[3] = z; }
      y = __shfl_xor_sync(kAll, high ? c[0] : c[2], 2);
      z = __shfl_xor_sync(kAll, high ? c[1] : c[3], 2);
      if (high) { c[0] = y; c[1] = z; } else { c[2] = y; c[3] = z; }
    } else if constexpr (NG == 2) {
      const unsigned y = __shfl_xor_sync(kAll, n ? c[0] : c[2], 1), z = __shfl_xor_sync(kAll, n ? c[1] : c[3], 1);
      // (word 2 n of both groups, then word 2 n + 1)
      if (n) { c[0] = y; c[1] = c[2]; c[2] = z; } else { const unsigned c1 = c[1]; c[1] = y; c[2] = c1; c[3] = z; }
    }
    const int in = base + r0 + i * RPI;
    if (in >= w.len) continue;
    const int p = w.pos + in;
    if (p >= W.sinks && p < w.first) continue;
    const int r = row_at<kTile>(W, p, ring0 + i * RPI), rr = r & 15;
    uint4 word = make_uint4(c[0], c[1], c[2], c[3]);
    if (value) {  // 16-bit units, group by group
      if constexpr (NG == 4) word = make_uint4(__byte_perm(c[0], c[1], 0x5410), __byte_perm(c[2], c[3], 0x5410), __byte_perm(c[0], c[1], 0x7632), __byte_perm(c[2], c[3], 0x7632));
      if constexpr (NG == 2) word = make_uint4(__byte_perm(c[0], c[1], 0x5410), __byte_perm(c[0], c[1], 0x7632), __byte_perm(c[2], c[3], 0x5410), __byte_perm(c[2], c[3], 0x7632));
    }
    unsigned char* block = blocks + (size_t)(unsigned)(r >> 4) * (unsigned)Block4<D>::kBytes;
    *reinterpret_cast<uint4*>(block + (value ? Block4<D>::kValues : Block4<D>::kKeys) + rr * (D / 2) + n * 16) = word;
    *reinterpret_cast<unsigned short*>(block + (value ? Block4<D>::kValueScales + (rr >> 1) * (4 * NG) + n * 4 + (rr & 1) * 2
                                                      : Block4<D>::kKeyScales + rr * (2 * NG) + n * 2)) = s;
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
    const int r = row_at<Piece<D>::kTile>(W, to, ring0 + i * RPI);
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
  if (!store_grid(W, n_tokens, BITS == 4 ? kStoreThreads / 2 / Block4<D>::kGroups * kGroupUnroll : Piece<D>::kTile, grid)) return cudaErrorInvalidValue;
  return launch_pdl(BITS == 4 ? kvm_window_write4_kernel<D> : kvm_window_write16_kernel<D>, grid, dim3(kStoreThreads), 0, stream, true, W, k, v, n_tokens, positions, lengths);
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
