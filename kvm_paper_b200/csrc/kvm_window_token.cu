// Attention of one query per sequence over a window cache (16 or 4 bits), the query's own token written on the way if it is
// given; sequences of unequal length.
//
// The rows that the sequences may see, in chunks of 128, form one flat list (sequence, kv head, chunk); every CTA, one per SM,
// takes an equal contiguous range of it.  A producer warp streams the range through a ring of shared-memory stages, eight math
// warps follow it, each with 16 rows of every chunk, and keep a running maximum, sum and output of their own, which are
// joined when the CTA leaves a kv row.  A kv row that lies inside one range is finished there; of one that is cut each CTA
// leaves a partial result (fp32), and kvm_window_join_kernel joins those in the order of the list.  Nothing is counted or
// kept between calls.
//
// Bound by memory: a row is read once for all query heads of its kv head.  The products run on warp-level MMAs with the
// cache rows on the M dimension and the query heads on N (8 or 16 columns).
// 4 bits: the codes become f16 with one conversion instruction per two values.  q is scaled by a power of two per head into
// f16's range.  A key group's scale multiplies the fp32 sum of its group; a value group's scale multiplies the weights, as
// f16 relative to a running power of two R above all scales seen so far (the output is rescaled when R rises, as with the
// softmax maximum): a value scale 2^-24 below the largest of its sequence is lost, which is an error of 2^-24 of that
// largest value.
// The new token: the CTA that reads the chunk with its row patches the stage and writes the row to memory.
#include <algorithm>

#include "kvm_tma_host.cuh"
#include "kvm_window.cuh"

namespace kvm {

namespace {

constexpr int kChunk = 128;                   // rows per chunk
constexpr int kMathWarps = 8;
constexpr int kTokThreads = (kMathWarps + 1) * 32;
constexpr int kMaxStages = 8;
constexpr int kBox = 16;                      // rows per TMA box (16 bits)
constexpr int kMaxSmemBytes = 227 * 1024;
constexpr int kMaxBatch = 1024;               // sequences per launch

template <int D, int BITS>
struct TokGeom {
  static constexpr int kStageKv = BITS == 4 ? kChunk / 16 * Block4<D>::kBytes : 2 * kChunk * D * 2;
  static constexpr int kBoxW = D >= 64 ? 64 : 32;   // elements per box
  static constexpr int kBlocks = D / kBoxW;
};

struct TokSmem {
  int stage_bytes, q, ored, wred, bars, pre, total, stages;
  __host__ __device__ TokSmem(int kv_bytes, int D, int G, int nb, int st) {
    q = kv_bytes;                                            // [G][D] bf16 behind the stage's rows
    stage_bytes = (q + G * D * 2 + 1023) & ~1023;            // (boxes in the 128-byte swizzle start on 1024 bytes)
    stages = st;
    int off = st * stage_bytes;
    ored = off; off += kMathWarps * G * D * 4;
    wred = off; off += 2 * kMathWarps * 16 * 4;
    bars = off; off += 2 * kMaxStages * 8;
    pre = off;  off += (2 * nb + 1) * 4;
    total = (off + 15) & ~15;
  }
};

struct TokMaps {
  CUtensorMap k, v;  // [all rows][D], boxes of 16 rows
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
  const __half2 h = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void math_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kMathWarps * 32) : "memory"); }

// Which rows the last of n tokens sees (WindowDev::visible without its division).
struct Seen {
  int sinks, sp, live, newest, ring, limit;
  __device__ __forceinline__ Seen(const WindowDev& W, int n) {
    const int m = n - W.sinks;
    sinks = min(W.sinks, n);
    sp = W.sp;
    live = W.live(n);
    ring = W.ring;
    newest = m > 0 ? (m - 1) % W.ring : 0;
    limit = min(W.window, m);
  }
  __device__ __forceinline__ bool visible(int r) const {
    const int back = newest - (r - sp);
    return r < live && (r < sp ? r < sinks : (back < 0 ? back + ring : back) < limit);
  }
};

// A place in the flat list.
struct Place {
  int b, h, c, n_chunks;  // sequence, kv head, chunk of the kv row, chunks of the kv row
};

// Partial result of a kv row that a CTA's range cuts: [head][m, l, acc[D]].
__host__ __device__ inline size_t partial_floats(int D, int G) { return (size_t)G * (D + 2); }

// The split of the list, the same in both kernels.  whole_rows: ranges end between kv rows.
struct Split {
  int total, per, active;  // units (chunks, or kv rows) of the list, per CTA, CTAs with work
  __device__ __forceinline__ Split(int units, int grid) {
    total = units;
    per = max(1, (units + grid - 1) / grid);
    active = (units + per - 1) / per;
  }
};

__device__ __forceinline__ int chunks_of(const WindowDev& W, int n) { return (W.live(n) + kChunk - 1) / kChunk; }

// Tokens of every sequence (pre[nb + 1 ..]) and its chunks per kv row as a prefix (pre[0..nb]) in shared memory.
__device__ __forceinline__ void build_prefix(const WindowDev& W, SeqInts lens, int extra, int b0, int nb, int* pre, int tid, int threads) {
  for (int b = tid; b < nb; b += threads) {
    const int n = max(lens.at(b0 + b), -1) + extra;
    pre[nb + 1 + b] = n;
    pre[b + 1] = chunks_of(W, n);
  }
  if (tid == 0) pre[0] = 0;
  __syncthreads();
  if (tid < 32) {
    int carry = 0;
    for (int base = 0; base < nb; base += 32) {
      const int i = base + tid;
      int x = i < nb ? pre[i + 1] : 0;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, d);
        if (tid >= d) x += y;
      }
      if (i < nb) pre[i + 1] = x + carry;
      carry += __shfl_sync(0xffffffffu, x, 31);
    }
  }
  __syncthreads();
}
// sequence whose kv rows hold place f of the list
__device__ __forceinline__ int find_seq(const int* pre, int nb, int Hkv, int f) {
  int lo = 0, hi = nb - 1;  // last b with pre[b] * Hkv <= f among those that have chunks
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (pre[mid] * Hkv <= f) lo = mid; else hi = mid - 1;
  }
  return lo;
}

}  // namespace

template <int D, int BITS, int NH>
__global__ void __launch_bounds__(kTokThreads, 1)
kvm_window_token_kernel(WindowDev W, int G, Tensor4 q, Tensor4 k_new, Tensor4 v_new, SeqInts lens, int b0, int nb, int stages,
                        int whole_rows, float scale_log2, float* __restrict__ partial, bf16* __restrict__ out, int* __restrict__ status,
                        const __grid_constant__ TokMaps maps) {
  using GM = TokGeom<D, BITS>;
  constexpr int NG = D / 32;       // groups of 32 channels
  extern __shared__ __align__(1024) unsigned char smem[];
  const TokSmem lay(GM::kStageKv, D, G, nb, stages);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + lay.bars);
  uint64_t* empty = full + kMaxStages;
  int* pre = reinterpret_cast<int*>(smem + lay.pre);
  const int* tokens = pre + nb + 1;
  __shared__ int s_abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int Hkv = W.Hkv, Hq = Hkv * G;
  const bool with_new = k_new.ptr != nullptr;
  const int extra = with_new ? 1 : 0;  // lens are positions of the new tokens

  if (tid == 0) {
    for (int s = 0; s < stages; ++s) {
      tc::mbar_init(&full[s], 1);
      tc::mbar_init(&empty[s], kMathWarps);
    }
    tc::fence_barrier_init();
    s_abort = 0;
  }
  pdl_trigger();  // (the join kernel may be staged; it waits for this grid)
  pdl_wait();
  build_prefix(W, lens, extra, b0, nb, pre, tid, kTokThreads);
  const int total_f = pre[nb] * Hkv;

  // this CTA's range [f_begin, f_end)
  int f_begin, f_end;
  if (whole_rows) {
    const Split sp(nb * Hkv, gridDim.x);
    const int r0 = min((int)blockIdx.x * sp.per, nb * Hkv), r1 = min(r0 + sp.per, nb * Hkv);
    auto place = [&](int r) { return r >= nb * Hkv ? total_f : pre[r / Hkv] * Hkv + (r % Hkv) * (pre[r / Hkv + 1] - pre[r / Hkv]); };
    f_begin = place(r0);
    f_end = place(r1);
  } else {
    const Split sp(total_f, gridDim.x);
    f_begin = min((int)blockIdx.x * sp.per, total_f);
    f_end = min(f_begin + sp.per, total_f);
  }
  const int nloc = f_end - f_begin;
  // sequences without tokens: zeros
  for (int b = blockIdx.x; b < nb; b += gridDim.x)
    if (pre[b + 1] == pre[b])
      for (int i = tid; i < Hq * D / 8; i += kTokThreads)
        reinterpret_cast<uint4*>(out + (size_t)(b0 + b) * Hq * D)[i] = make_uint4(0, 0, 0, 0);
  if (nloc <= 0) return;

  Place pl;
  pl.b = find_seq(pre, nb, Hkv, f_begin);
  pl.n_chunks = pre[pl.b + 1] - pre[pl.b];
  {
    const int rem = f_begin - pre[pl.b] * Hkv;
    pl.h = rem / pl.n_chunks;
    pl.c = rem % pl.n_chunks;
  }
  auto advance = [&](Place& p) {
    if (++p.c < p.n_chunks) return;
    p.c = 0;
    if (++p.h < Hkv) return;
    p.h = 0;
    do { ++p.b; } while (p.b < nb && pre[p.b + 1] == pre[p.b]);
    if (p.b < nb) p.n_chunks = pre[p.b + 1] - pre[p.b];
  };
  volatile int* abort_flag = &s_abort;

  if (warp == kMathWarps) {
    // ------------------------------------------------------------------------------------ producer
    for (int i = 0; i < nloc; ++i) {
      const int s = i % stages;
      if (i >= stages) {
        const bool ok = tc::mbar_wait(&empty[s], ((i / stages) - 1) & 1) && !*abort_flag;
        if (!__all_sync(0xffffffffu, ok)) {
          if (lane == 0) {
            *abort_flag = 1;
            atomicExch(status, KVM_ERR_DEVICE_TIMEOUT);
            for (int j = i - stages; j < i; ++j) tc::mbar_wait_limit(&full[j % stages], (j / stages) & 1, 1 << 14);  // copies in flight
          }
          __syncwarp();
          break;
        }
      }
      unsigned char* st = smem + s * lay.stage_bytes;
      const int n = tokens[pl.b];
      const int rows = min(kChunk, W.live(n) - pl.c * kChunk), groups = (rows + 15) >> 4;
      const size_t kvrow = (size_t)(b0 + pl.b) * Hkv + pl.h;
      const bool first = i == 0 || pl.c == 0;
      if (lane == 0) {
        const uint32_t bytes = (BITS == 4 ? (uint32_t)groups * Block4<D>::kBytes : (uint32_t)groups * (2u * 16u * D * 2u)) + (first ? (uint32_t)(G * D * 2) : 0u);
        tc::mbar_arrive_expect_tx(&full[s], bytes);
      }
      __syncwarp();
      if (first && lane < G) tc::bulk_g2s(st + lay.q + lane * D * 2, q.row(b0 + pl.b, pl.h * G + lane, 0), D * 2, &full[s]);
      if (BITS == 4) {
        if (lane == 0)
          tc::bulk_g2s(st, W.blocks + (kvrow * (W.rows / 16) + (size_t)pl.c * (kChunk / 16)) * Block4<D>::kBytes, groups * Block4<D>::kBytes, &full[s]);
      } else {
        const int y = (int)(kvrow * W.rows) + pl.c * kChunk;  // (all rows of a cache: below 2^31, checked on the host)
        for (int j = lane; j < groups * GM::kBlocks * 2; j += 32) {
          const int half = j / (groups * GM::kBlocks), k2 = j % (groups * GM::kBlocks), blk = k2 / groups, gr = k2 % groups;
          tc::tma_load_2d(st + half * (kChunk * D * 2) + blk * (kChunk * GM::kBoxW * 2) + gr * (kBox * GM::kBoxW * 2), half ? &maps.v : &maps.k,
                          blk * GM::kBoxW, y + gr * kBox, &full[s]);
        }
      }
      advance(pl);
    }
    return;
  }

  // -------------------------------------------------------------------------------------- math warps
  const int g = lane >> 2, t = lane & 3;
  float* ored = reinterpret_cast<float*>(smem + lay.ored);          // [warp][G][D]
  float* wmax = reinterpret_cast<float*>(smem + lay.wred);          // [warp][16]
  float* wsum = wmax + kMathWarps * 16;
  uint32_t qf[NH][D / 16][2];
  float qs[NH][2];                 // softmax scale (log2) of this thread's heads 2t, 2t + 1
  float o[NH][D / 16][4];          // output rows (channels) x heads
  float m[NH][2], l[NH][2];
  float r_ref = 0.f;               // 4 bits: the power of two that the weights are relative to (0: none yet)
  unsigned r_bits = 0;             // its bf16 exponent field
  const Place start = pl;
  Seen seen(W, 0);
  bool ok = true;  // false: a wait ran out; the warp goes on without data so that it meets the others at their barriers

  for (int i = 0; i < nloc; ++i) {
    const int s = i % stages;
    if (ok) {
      ok = __all_sync(0xffffffffu, tc::mbar_wait(&full[s], (i / stages) & 1) && !*abort_flag);
      if (!ok && lane == 0) {
        *abort_flag = 1;
        atomicExch(status, KVM_ERR_DEVICE_TIMEOUT);
      }
    }
    unsigned char* st = smem + s * lay.stage_bytes;
    const int n = tokens[pl.b];
    if (i == 0 || pl.c == 0) {  // a new kv row: queries as B fragments
      seen = Seen(W, n);
#pragma unroll
      for (int hb = 0; hb < NH; ++hb) {
        const int head = hb * 8 + g;
        const bf16* qrow = reinterpret_cast<const bf16*>(st + lay.q) + (size_t)min(head, G - 1) * D;
        if (BITS == 4) {
          uint4 x[NG];
          unsigned amax = 0;
#pragma unroll
          for (int n2 = 0; n2 < NG; ++n2) {
            x[n2] = *reinterpret_cast<const uint4*>(qrow + n2 * 32 + t * 8);
            const unsigned w[4] = {x[n2].x, x[n2].y, x[n2].z, x[n2].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) amax = __vmaxu2(amax, w[j] & 0x7fff7fffu);
          }
          amax = max(amax & 0xffffu, amax >> 16);
          amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
          amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
          // largest magnitude into [2^14, 2^15): a value loses bits only if it is 2^28 below it.  (2^-e as a float: e in
          // [-126, 127]; infinities and NaN stay what they are)
          const int e = min(max((int)(amax >> 7) - 127, -112), 127);
          const float up = __uint_as_float((unsigned)(127 + 14 - e) << 23 & 0x7f800000u);
          const float upc = amax >= 0x7f80u ? 1.f : up;
          float down = amax >= 0x7f80u ? 1.f : __uint_as_float((unsigned)max(127 - 14 + e, 1) << 23);
#pragma unroll
          for (int n2 = 0; n2 < NG; ++n2) {
            const unsigned w[4] = {x[n2].x, x[n2].y, x[n2].z, x[n2].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 f = unpack_bf16(w[j]);
              qf[hb][n2 * 2 + (j >> 1)][j & 1] = pack_f16(f.x * upc, f.y * upc);
            }
          }
          // this thread's scores are of heads 2t, 2t + 1: their factors lie in lanes 8t, 8t + 4
          qs[hb][0] = __shfl_sync(0xffffffffu, down, 8 * t) * scale_log2;
          qs[hb][1] = __shfl_sync(0xffffffffu, down, 8 * t + 4) * scale_log2;
        } else {
#pragma unroll
          for (int blk = 0; blk < (D >= 64 ? D / 64 : 1); ++blk) {
            constexpr int PER = D >= 64 ? 4 : 2;  // k-steps per 64 (32) channels; a thread's channels are contiguous
#pragma unroll
            for (int j = 0; j < PER; ++j) {
              const uint2 x = *reinterpret_cast<const uint2*>(qrow + blk * 64 + t * (PER * 4) + j * 4);
              qf[hb][blk * PER + j][0] = x.x;
              qf[hb][blk * PER + j][1] = x.y;
            }
          }
          qs[hb][0] = qs[hb][1] = scale_log2;
        }
        m[hb][0] = m[hb][1] = -INFINITY;
        l[hb][0] = l[hb][1] = 0.f;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) o[hb][j][0] = o[hb][j][1] = o[hb][j][2] = o[hb][j][3] = 0.f;
      }
      r_ref = 0.f;
      r_bits = 0;
    }

    // ---- this warp's 16 rows
    const int row0 = pl.c * kChunk + warp * 16;
    const unsigned vis = __ballot_sync(0xffffffffu, seen.visible(row0 + (lane & 15))) & 0xffffu;
    if (vis && ok) {
      const size_t kvrow = (size_t)(b0 + pl.b) * Hkv + pl.h;
      // the new token's row: into the stage (what was loaded there is stale) and into memory
      bool patched = false;
      if (with_new) {
        const int nr = W.row_of(n - 1);
        if ((nr >> 4) == (row0 >> 4)) {
          patched = true;
          const int rr = nr & 15;
          const bf16* kn = k_new.row(b0 + pl.b, pl.h, 0);
          const bf16* vn = v_new.row(b0 + pl.b, pl.h, 0);
          if (BITS == 16) {
            for (int j = lane; j < D / 4; j += 32) {  // 16-byte pieces of K, then of V
              const bool value = j >= D / 8;
              const int c = value ? j - D / 8 : j;
              const uint4 x = *reinterpret_cast<const uint4*>((value ? vn : kn) + c * 8);
              const int r = warp * 16 + rr;
              unsigned char* base = st + (value ? kChunk * D * 2 : 0);
              if (D >= 64) base += (c >> 3) * (kChunk * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
              else base += r * 64 + c * 16;
              *reinterpret_cast<uint4*>(base) = x;
              *reinterpret_cast<uint4*>((value ? W.v : W.k) + (kvrow * W.rows + nr) * D + c * 8) = x;
            }
          } else {
            unsigned char* sb = st + warp * Block4<D>::kBytes;
            unsigned char* gb = W.blocks + (kvrow * (W.rows / 16) + (nr >> 4)) * Block4<D>::kBytes;
#pragma unroll
            for (int it = 0; it < (D == 128 ? 2 : 1); ++it) {  // items: 4 channels of K, then of V
              const int item = it * 32 + lane, value = item >= D / 4, c4 = value ? item - D / 4 : item;
              const bool live_item = item < D / 2;
              const uint2 x = live_item ? *reinterpret_cast<const uint2*>((value ? vn : kn) + c4 * 4) : make_uint2(0, 0);
              unsigned am = __vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu);
              am = max(am & 0xffffu, am >> 16);
#pragma unroll
              for (int d2 = 1; d2 < 8; d2 <<= 1) am = max(am, __shfl_xor_sync(0xffffffffu, am, d2));
              float inv;
              const unsigned short sc = group_scale(am, inv);
              const float2 f0 = unpack_bf16(x.x), f1 = unpack_bf16(x.y);
              unsigned code = e2m1x2(level_of(f0.x, inv), level_of(f0.y, inv)) | e2m1x2(level_of(f1.x, inv), level_of(f1.y, inv)) << 8;
              if (am >= 0x7f80u) code = 0;
              const int grp = c4 >> 3, u = c4 & 7;
              const int off = value ? Block4<D>::kValues + rr * (D / 2) + u * (2 * NG) + grp * 2
                                    : Block4<D>::kKeys + rr * (D / 2) + (u >> 1) * (4 * NG) + grp * 4 + (u & 1) * 2;
              const int soff = value ? Block4<D>::kValueScales + (rr >> 1) * (4 * NG) + grp * 4 + (rr & 1) * 2
                                     : Block4<D>::kKeyScales + rr * (2 * NG) + grp * 2;
              if (live_item) {
                *reinterpret_cast<unsigned short*>(sb + off) = (unsigned short)code;
                *reinterpret_cast<unsigned short*>(gb + off) = (unsigned short)code;
                if (u == 0) {
                  *reinterpret_cast<unsigned short*>(sb + soff) = sc;
                  *reinterpret_cast<unsigned short*>(gb + soff) = sc;
                }
              }
            }
          }
          __syncwarp();
        }
      }
      if (BITS == 4 && vis != 0xffffu) {  // rows that are not to be seen: scale 0 (whatever they hold, they add nothing)
        patched = true;
        unsigned char* sb = st + warp * Block4<D>::kBytes;
        for (int j = lane; j < 16 * NG; j += 32) {
          const int rr = j / NG, grp = j % NG;
          if (!((vis >> rr) & 1)) {
            *reinterpret_cast<unsigned short*>(sb + Block4<D>::kKeyScales + rr * (2 * NG) + grp * 2) = 0;
            *reinterpret_cast<unsigned short*>(sb + Block4<D>::kValueScales + (rr >> 1) * (4 * NG) + grp * 4 + (rr & 1) * 2) = 0;
          }
        }
        __syncwarp();
      }

      // ---- scores: rows g, g + 8 x heads 2t, 2t + 1
      float sc[NH][4];
#pragma unroll
      for (int hb = 0; hb < NH; ++hb) sc[hb][0] = sc[hb][1] = sc[hb][2] = sc[hb][3] = 0.f;
      if (BITS == 4) {
        const unsigned char* sb = st + warp * Block4<D>::kBytes;
        uint32_t kw[2][NG];
        float ks[2][NG];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int rr = g + 8 * r;
          const unsigned char* p = sb + Block4<D>::kKeys + rr * (D / 2) + t * (4 * NG);
          const unsigned char* sp = sb + Block4<D>::kKeyScales + rr * (2 * NG);
          if (NG == 4) {
            const uint4 x = *reinterpret_cast<const uint4*>(p);
            kw[r][0] = x.x; kw[r][NG > 1 ? 1 : 0] = x.y; kw[r][NG > 2 ? 2 : 0] = x.z; kw[r][NG > 3 ? 3 : 0] = x.w;
            const uint2 y = *reinterpret_cast<const uint2*>(sp);
            ks[r][0] = __uint_as_float(y.x << 16); ks[r][NG > 1 ? 1 : 0] = __uint_as_float(y.x & 0xffff0000u);
            ks[r][NG > 2 ? 2 : 0] = __uint_as_float(y.y << 16); ks[r][NG > 3 ? 3 : 0] = __uint_as_float(y.y & 0xffff0000u);
          } else if (NG == 2) {
            const uint2 x = *reinterpret_cast<const uint2*>(p);
            kw[r][0] = x.x; kw[r][NG > 1 ? 1 : 0] = x.y;
            const unsigned y = *reinterpret_cast<const unsigned*>(sp);
            ks[r][0] = __uint_as_float(y << 16); ks[r][NG > 1 ? 1 : 0] = __uint_as_float(y & 0xffff0000u);
          } else {
            kw[r][0] = *reinterpret_cast<const unsigned*>(p);
            ks[r][0] = __uint_as_float((unsigned)*reinterpret_cast<const unsigned short*>(sp) << 16);
          }
        }
#pragma unroll
        for (int n2 = 0; n2 < NG; ++n2) {
          uint32_t a[4], c[4];
          e2m1_to_f16x2(kw[0][n2], a[0], a[1], a[2], a[3]);
          e2m1_to_f16x2(kw[1][n2], c[0], c[1], c[2], c[3]);
#pragma unroll
          for (int hb = 0; hb < NH; ++hb) {
            float acc[4] = {0.f, 0.f, 0.f, 0.f};
            mma_f16(acc, a[0], c[0], a[1], c[1], qf[hb][n2 * 2][0], qf[hb][n2 * 2][1]);
            mma_f16(acc, a[2], c[2], a[3], c[3], qf[hb][n2 * 2 + 1][0], qf[hb][n2 * 2 + 1][1]);
            sc[hb][0] = fmaf(ks[0][n2], acc[0], sc[hb][0]);
            sc[hb][1] = fmaf(ks[0][n2], acc[1], sc[hb][1]);
            sc[hb][2] = fmaf(ks[1][n2], acc[2], sc[hb][2]);
            sc[hb][3] = fmaf(ks[1][n2], acc[3], sc[hb][3]);
          }
        }
      } else {
        const int r = warp * 16 + g;
#pragma unroll
        for (int blk = 0; blk < GM::kBlocks; ++blk) {
          constexpr int PIECES = GM::kBoxW / 32;  // 16-byte pieces per thread and row: 2 (64 channels) or 1
#pragma unroll
          for (int j = 0; j < PIECES; ++j) {
            const int c = t * PIECES + j;
            uint4 x, y;
            if (D >= 64) {
              const unsigned char* base = st + blk * (kChunk * 128) + r * 128 + ((c ^ (r & 7)) << 4);
              x = *reinterpret_cast<const uint4*>(base);
              y = *reinterpret_cast<const uint4*>(base + 8 * 128);
            } else {
              const unsigned char* base = st + r * 64 + c * 16;
              x = *reinterpret_cast<const uint4*>(base);
              y = *reinterpret_cast<const uint4*>(base + 8 * 64);
            }
#pragma unroll
            for (int hb = 0; hb < NH; ++hb) {
              const int kk = (blk * PIECES + j) * 2;
              mma_bf16(sc[hb], x.x, y.x, x.y, y.y, qf[hb][kk][0], qf[hb][kk][1]);
              mma_bf16(sc[hb], x.z, y.z, x.w, y.w, qf[hb][kk + 1][0], qf[hb][kk + 1][1]);
            }
          }
        }
      }
      const bool see0 = (vis >> g) & 1, see1 = (vis >> (g + 8)) & 1;

      // ---- running maximum (raised when a tile exceeds it by 2^8), weights
      float alpha[NH][2];
      bool raise = false;
#pragma unroll
      for (int hb = 0; hb < NH; ++hb) {
#pragma unroll
        for (int j = 0; j < 4; ++j) sc[hb][j] = ((j < 2) ? see0 : see1) ? sc[hb][j] * qs[hb][j & 1] : -INFINITY;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float x = fmaxf(sc[hb][j], sc[hb][j + 2]);
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          const bool up = x > m[hb][j] + 8.f || (m[hb][j] == -INFINITY && x > -INFINITY);
          alpha[hb][j] = 1.f;
          if (up) {
            alpha[hb][j] = m[hb][j] == -INFINITY ? 0.f : ex2(m[hb][j] - x);
            m[hb][j] = x;
            raise = true;
          }
        }
      }
      float r_alpha = 1.f;
      if (BITS == 4) {
        // the exponent of the largest value scale of these rows (NaN does not count: it reaches its own group only)
        const unsigned char* sb = st + warp * Block4<D>::kBytes + Block4<D>::kValueScales;
        unsigned x = lane < 8 * NG ? *reinterpret_cast<const unsigned*>(sb + lane * 4) : 0u;
        const unsigned x0 = x & 0xffffu, x1 = x >> 16;
        x = max(x0 < 0x7f80u ? x0 : 0u, x1 < 0x7f80u ? x1 : 0u);
        x = __reduce_max_sync(0xffffffffu, x) & 0x7f80u;
        if (x > r_bits + (6u << 7) || (r_bits == 0 && x)) {  // a scale is below 2^7 R, a weight at most 2^8: f16 holds the product
          const unsigned old = r_bits;
          r_bits = x;
          r_alpha = old ? __uint_as_float((unsigned)max(127 + (int)(old >> 7) - (int)(x >> 7), 0) << 23) : 0.f;
          r_ref = __uint_as_float(x << 16);
          raise = true;
        }
      }
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int hb = 0; hb < NH; ++hb) {
          l[hb][0] *= alpha[hb][0];
          l[hb][1] *= alpha[hb][1];
          const float a0 = alpha[hb][0] * r_alpha, a1 = alpha[hb][1] * r_alpha;
#pragma unroll
          for (int j = 0; j < D / 16; ++j) {
            o[hb][j][0] *= a0;
            o[hb][j][1] *= a1;
            o[hb][j][2] *= a0;
            o[hb][j][3] *= a1;
          }
        }
      }
      uint32_t pb[NH][2];  // weights as B fragments: rows (2t, 2t + 1), (2t + 8, 2t + 9) of head g
#pragma unroll
      for (int hb = 0; hb < NH; ++hb) {
        float p[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float mm = m[hb][j & 1] == -INFINITY ? 0.f : m[hb][j & 1];
          p[j] = ex2(sc[hb][j] - mm);
        }
        l[hb][0] += p[0] + p[2];
        l[hb][1] += p[1] + p[3];
        pb[hb][0] = movmatrix_trans(BITS == 4 ? pack_f16(p[0], p[1]) : pack_bf16(p[0], p[1]));
        pb[hb][1] = movmatrix_trans(BITS == 4 ? pack_f16(p[2], p[3]) : pack_bf16(p[2], p[3]));
      }

      // ---- output += V^T P
      if (BITS == 4) {
        const unsigned char* sb = st + warp * Block4<D>::kBytes;
        // value scales of row pairs t and t + 4, relative to R, as f16x2
        const float inv = __uint_as_float((254u - (r_bits >> 7)) << 23);
        uint32_t vs[2][NG];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const unsigned char* p = sb + Block4<D>::kValueScales + (t + 4 * r) * (4 * NG);
          uint32_t x[4] = {0, 0, 0, 0};
          if (NG == 4) {
            const uint4 y = *reinterpret_cast<const uint4*>(p);
            x[0] = y.x; x[1] = y.y; x[2] = y.z; x[3] = y.w;
          } else if (NG == 2) {
            const uint2 y = *reinterpret_cast<const uint2*>(p);
            x[0] = y.x; x[1] = y.y;
          } else {
            x[0] = *reinterpret_cast<const uint32_t*>(p);
          }
#pragma unroll
          for (int n2 = 0; n2 < NG; ++n2) {
            vs[r][n2] = pack_f16(__uint_as_float(x[n2] << 16) * inv, __uint_as_float(x[n2] & 0xffff0000u) * inv);
          }
        }
        constexpr int NWD = NG > 1 ? NG / 2 : 1;  // 32-bit words of codes per thread and row
        uint32_t vw[4][NWD];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int rr = 2 * t + (r & 1) + 8 * (r >> 1);
          const unsigned char* p = sb + Block4<D>::kValues + rr * (D / 2) + g * (2 * NG);
          if (NG == 4) {
            const uint2 x = *reinterpret_cast<const uint2*>(p);
            vw[r][0] = x.x; vw[r][NWD - 1] = x.y;
          } else if (NG == 2) {
            vw[r][0] = *reinterpret_cast<const unsigned*>(p);
          } else {
            vw[r][0] = *reinterpret_cast<const unsigned short*>(p);
          }
        }
#pragma unroll
        for (int w = 0; w < NWD; ++w) {
          // rows (2t, 2t + 1) and (2t + 8, 2t + 9) side by side in a byte: even channels in e, odd ones in d
          uint32_t e[2], d[2];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            e[r] = (vw[2 * r][w] & 0x0f0f0f0fu) | ((vw[2 * r + 1][w] << 4) & 0xf0f0f0f0u);
            d[r] = ((vw[2 * r][w] >> 4) & 0x0f0f0f0fu) | (vw[2 * r + 1][w] & 0xf0f0f0f0u);
          }
          uint32_t ea[4], da[4], eb[4], db[4];
          e2m1_to_f16x2(e[0], ea[0], ea[1], ea[2], ea[3]);
          e2m1_to_f16x2(d[0], da[0], da[1], da[2], da[3]);
          e2m1_to_f16x2(e[1], eb[0], eb[1], eb[2], eb[3]);
          e2m1_to_f16x2(d[1], db[0], db[1], db[2], db[3]);
#pragma unroll
          for (int half = 0; half < (NG > 1 ? 2 : 1); ++half) {
            const int n2 = w * 2 + half;
#pragma unroll
            for (int hb = 0; hb < NH; ++hb) {
              const uint32_t p0 = mul_f16x2(pb[hb][0], vs[0][n2]), p1 = mul_f16x2(pb[hb][1], vs[1][n2]);
#pragma unroll
              for (int j = 0; j < 2; ++j)  // channels 32 n2 + 4 g + 2 j (rows g) and + 1 (rows g + 8)
                mma_f16(o[hb][n2 * 2 + j], ea[half * 2 + j], da[half * 2 + j], eb[half * 2 + j], db[half * 2 + j], p0, p1);
            }
          }
        }
      } else {
        const unsigned char* vb = st + kChunk * D * 2;
#pragma unroll
        for (int blk = 0; blk < GM::kBlocks; ++blk) {
          uint4 x[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int rr = warp * 16 + 2 * t + (r & 1) + 8 * (r >> 1);
            if (D >= 64) {
              x[r] = *reinterpret_cast<const uint4*>(vb + blk * (kChunk * 128) + rr * 128 + ((g ^ (rr & 7)) << 4));
            } else {
              const uint2 y = *reinterpret_cast<const uint2*>(vb + rr * 64 + g * 8);
              x[r] = make_uint4(y.x, y.y, 0, 0);
            }
            if (vis != 0xffffu && !((vis >> (rr & 15)) & 1)) x[r] = make_uint4(0, 0, 0, 0);  // (0 x NaN)
          }
          const uint32_t* a = &x[0].x;
          const uint32_t* b = &x[1].x;
          const uint32_t* c = &x[2].x;
          const uint32_t* d = &x[3].x;
          constexpr int WORDS = D >= 64 ? 4 : 2;
#pragma unroll
          for (int w = 0; w < WORDS; ++w) {
            const uint32_t a0 = __byte_perm(a[w], b[w], 0x5410), a1 = __byte_perm(a[w], b[w], 0x7632);
            const uint32_t a2 = __byte_perm(c[w], d[w], 0x5410), a3 = __byte_perm(c[w], d[w], 0x7632);
#pragma unroll
            for (int hb = 0; hb < NH; ++hb) mma_bf16(o[hb][blk * 4 + w], a0, a1, a2, a3, pb[hb][0], pb[hb][1]);
          }
        }
      }
      if (patched) tc::fence_proxy_async();  // before the next copy into this stage
    }
    __syncwarp();
    if (lane == 0) tc::mbar_arrive(&empty[s]);

    // ---- the last chunk of a kv row, or of the range: join the warps
    const Place here = pl;
    const bool row_ends = here.c == here.n_chunks - 1;
    advance(pl);
    if (row_ends || i == nloc - 1) {
#pragma unroll
      for (int hb = 0; hb < NH; ++hb) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float x = l[hb][j];
          x += __shfl_xor_sync(0xffffffffu, x, 4);
          x += __shfl_xor_sync(0xffffffffu, x, 8);
          x += __shfl_xor_sync(0xffffffffu, x, 16);
          if (g == 0) {
            wmax[warp * 16 + hb * 8 + 2 * t + j] = m[hb][j];
            wsum[warp * 16 + hb * 8 + 2 * t + j] = x;
          }
          const int head = hb * 8 + 2 * t + j;
          if (head < G) {
            float* dst = ored + ((size_t)warp * G + head) * D;
            const float up = BITS == 4 ? r_ref : 1.f;
#pragma unroll
            for (int k2 = 0; k2 < D / 16; ++k2) {
              // 4 bits: channels 32 (k2/2) + 4 g + 2 (k2%2) + {0, 1};  16 bits: 64 (k2/4) + 8 g + 2 (k2%4) + {0, 1}, and for
              // D = 32: 4 g + 2 k2 + {0, 1}
              const int ch = BITS == 4 || D == 32 ? (k2 >> 1) * 32 + 4 * g + 2 * (k2 & 1) : (k2 >> 2) * 64 + 8 * g + 2 * (k2 & 3);
              *reinterpret_cast<float2*>(dst + ch) = make_float2(o[hb][k2][j] * up, o[hb][k2][j + 2] * up);
            }
          }
        }
      }
      math_sync();
      const int f_row = f_begin + i - here.c;  // place of the row's first chunk in the list
      const bool whole = f_row >= f_begin && row_ends;
      const int slot = here.b == start.b && here.h == start.h && start.c > 0 ? 0 : 1;  // goes on here, or begins here
      for (int e = tid; e < G * D / 2; e += kMathWarps * 32) {
        const int head = e / (D / 2), ch = (e % (D / 2)) * 2;
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < kMathWarps; ++w) mx = fmaxf(mx, wmax[w * 16 + head]);
        const float mm = mx == -INFINITY ? 0.f : mx;
        float sum = 0.f, a0 = 0.f, a1 = 0.f;
#pragma unroll
        for (int w = 0; w < kMathWarps; ++w) {
          const float f = ex2(wmax[w * 16 + head] - mm);
          const float2 x = *reinterpret_cast<const float2*>(ored + ((size_t)w * G + head) * D + ch);
          sum = fmaf(wsum[w * 16 + head], f, sum);
          a0 = fmaf(x.x, f, a0);
          a1 = fmaf(x.y, f, a1);
        }
        if (whole) {
          *reinterpret_cast<uint32_t*>(out + ((size_t)(b0 + here.b) * Hq + here.h * G + head) * D + ch) = pack_bf16(a0 / sum, a1 / sum);
        } else {
          float* dst = partial + ((size_t)blockIdx.x * 2 + slot) * partial_floats(D, G) + (size_t)head * (D + 2);
          *reinterpret_cast<float2*>(dst + 2 + ch) = make_float2(a0, a1);
          if (ch == 0) *reinterpret_cast<float2*>(dst) = make_float2(mx, sum);
        }
      }
      math_sync();
    }
  }
}

// Joins the partial results of the kv rows that range boundaries cut: block i the row that holds boundary i + 1, if that is
// the row's first.
template <int D>
__global__ void __launch_bounds__(256)
kvm_window_join_kernel(WindowDev W, int G, SeqInts lens, int extra, int b0, int nb, int grid, const float* __restrict__ partial,
                       bf16* __restrict__ out) {
  extern __shared__ int pre[];
  const int tid = threadIdx.x;
  // (the lengths are an earlier kernel's results at the latest: with the wait ahead of them everything else is too)
  pdl_wait();
  build_prefix(W, lens, extra, b0, nb, pre, tid, 256);
  const int Hkv = W.Hkv;
  const Split sp(pre[nb] * Hkv, grid);
  const int f = ((int)blockIdx.x + 1) * sp.per;
  if (f >= sp.total) return;
  const int b = find_seq(pre, nb, Hkv, f);
  const int nc = pre[b + 1] - pre[b], rem = f - pre[b] * Hkv, h = rem / nc, row0 = f - rem % nc, row1 = row0 + nc;
  if (row0 == f || row0 / sp.per != (int)blockIdx.x) return;  // not cut here, or another boundary's
  const int c1 = (row1 - 1) / sp.per;
  for (int e = tid; e < G * D / 2; e += 256) {
    const int head = e / (D / 2), ch = (e % (D / 2)) * 2;
    float mx = -INFINITY, sum = 0.f, a0 = 0.f, a1 = 0.f;
    for (int c = blockIdx.x; c <= c1; ++c) {
      const int slot = c == (int)blockIdx.x ? 1 : 0;  // where the row begins, and where it goes on
      const float* src = partial + ((size_t)c * 2 + slot) * partial_floats(D, G) + (size_t)head * (D + 2);
      const float2 ml = *reinterpret_cast<const float2*>(src), x = *reinterpret_cast<const float2*>(src + 2 + ch);
      const float m2 = fmaxf(mx, ml.x), mm = m2 == -INFINITY ? 0.f : m2;
      const float f0 = ex2(mx - mm), f1 = ex2(ml.x - mm);
      mx = m2;
      sum = sum * f0 + ml.y * f1;
      a0 = a0 * f0 + x.x * f1;
      a1 = a1 * f0 + x.y * f1;
    }
    *reinterpret_cast<uint32_t*>(out + ((size_t)(b0 + b) * Hkv * G + h * G + head) * D + ch) = pack_bf16(a0 / sum, a1 / sum);
  }
}

namespace {

int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return 148;
  return n;
}

template <int D, int BITS, int NH>
cudaError_t launch_token(const WindowDev& W, int G, Tensor4 q, Tensor4 k_new, Tensor4 v_new, SeqInts lens, float scale, float* partial,
                         bf16* out, int* status, cudaStream_t stream) {
  using GM = TokGeom<D, BITS>;
  TokMaps maps = {};
  if (BITS == 16) {
    const cuuint64_t dims[2] = {(cuuint64_t)D, (cuuint64_t)W.batch * W.Hkv * W.rows};
    const cuuint64_t strides[1] = {(cuuint64_t)D * 2};
    const cuuint32_t box[2] = {(cuuint32_t)GM::kBoxW, (cuuint32_t)kBox};
    if (!encode_bf16_map(&maps.k, W.k, 2, dims, strides, box) || !encode_bf16_map(&maps.v, W.v, 2, dims, strides, box))
      return cudaErrorInvalidValue;
  }
  auto kern = kvm_window_token_kernel<D, BITS, NH>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmemBytes - 1024);
  if (e != cudaSuccess) return e;
  const int sms = sm_count();
  const int max_chunks = (W.rows + kChunk - 1) / kChunk;
  for (int b0 = 0; b0 < W.batch; b0 += kMaxBatch) {
    const int nb = std::min(kMaxBatch, W.batch - b0);
    int stages = 1;
    while (stages < kMaxStages && TokSmem(GM::kStageKv, D, G, nb, stages + 1).total <= kMaxSmemBytes - 1024) ++stages;
    // Whole kv rows per CTA where cutting them gains less than the second launch and the partial results cost (about
    // 2.5 us; a chunk streams in about its bytes / 44 GB/s per SM).
    const long long rows = (long long)nb * W.Hkv, chunks = rows * max_chunks;
    const double chunk_us = GM::kStageKv / 44e3;
    const bool whole = (double)((rows + sms - 1) / sms) * max_chunks * chunk_us <= (double)((chunks + sms - 1) / sms) * chunk_us + 2.5;
    const int grid = (int)std::min<long long>(sms, whole ? rows : chunks);
    const TokSmem lay(GM::kStageKv, D, G, nb, stages);
    cudaError_t err = launch_pdl(kern, dim3(grid), dim3(kTokThreads), lay.total, stream, true, W, G, q, k_new, v_new, lens, b0, nb, stages,
                                 whole ? 1 : 0, scale * kLog2e, partial, out, status, maps);
    if (err != cudaSuccess) return err;
    if (!whole && grid > 1) {
      err = launch_pdl(kvm_window_join_kernel<D>, dim3(grid - 1), dim3(256), (2 * nb + 1) * 4, stream, true, W, G, lens,
                       k_new.ptr ? 1 : 0, b0, nb, grid, (const float*)partial, out);
      if (err != cudaSuccess) return err;
    }
  }
  return cudaSuccess;
}

template <int D, int BITS>
cudaError_t launch_token_nh(const WindowDev& W, int G, Tensor4 q, Tensor4 k_new, Tensor4 v_new, SeqInts lens, float scale, float* partial,
                            bf16* out, int* status, cudaStream_t stream) {
  return G <= 8 ? launch_token<D, BITS, 1>(W, G, q, k_new, v_new, lens, scale, partial, out, status, stream)
                : launch_token<D, BITS, 2>(W, G, q, k_new, v_new, lens, scale, partial, out, status, stream);
}

}  // namespace

size_t window_token_workspace(int D, int G) { return (size_t)sm_count() * 2 * partial_floats(D, G) * 4; }

cudaError_t window_token_dispatch(int D, int bits, const WindowDev& W, int G, Tensor4 q, Tensor4 k_new, Tensor4 v_new, SeqInts lens,
                                  float scale, float* partial, bf16* out, int* status, cudaStream_t stream) {
#define KVM_TOKEN(d) (bits == 4 ? launch_token_nh<d, 4>(W, G, q, k_new, v_new, lens, scale, partial, out, status, stream) \
                                : launch_token_nh<d, 16>(W, G, q, k_new, v_new, lens, scale, partial, out, status, stream))
  return D == 128 ? KVM_TOKEN(128) : D == 64 ? KVM_TOKEN(64) : KVM_TOKEN(32);
#undef KVM_TOKEN
}

}  // namespace kvm
