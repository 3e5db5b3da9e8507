// Attention of one query per sequence over a window cache (16 or 4 bits), the query's own token written on the way if it is
// given; sequences of unequal length.
//
// The rows that the sequences may see, in chunks, form one flat list (sequence, kv head, chunk); every CTA takes an equal
// contiguous range of it.  Its chunks stream through a ring of shared-memory stages; eight math warps, each with its own rows
// of every chunk, keep a running maximum, sum and output of their own, which are joined when the CTA leaves a kv row.  A kv row
// that lies inside one range is finished there; of one that is cut each CTA leaves a partial result (fp32), and
// kvm_window_join_kernel joins those in the order of the list.  Nothing is counted or kept between calls.
//
// A row is read once for all query heads of its kv head.  The products run on warp-level MMAs with the cache rows on the M
// dimension and the query heads on N (8 or 16 columns).
// 4 bits: the codes become f16 with one conversion instruction per two values.  q is scaled by a power of two per head into
// f16's range.  A key group's scale multiplies the fp32 sum of its group; a value group's scale multiplies the weights, as
// f16 relative to the largest power of two R in the group's scales so far (its outputs are rescaled when R rises, as with the
// softmax maximum).  Weights go up to 2^8 and scales to 2^7, so that the product uses f16 to its top: scales down to 2^-25 R and
// weights down to 2^-22 of the largest keep all their bits, smaller ones an error of 2^-31 R and 2^-33 of the largest.
// The new token: the CTA that reads the chunk with its row patches the stage and writes the row to memory.
//
// Measured: 4 bits, 64 x 4 kv rows of 16384 x 128 132 us (4.6 TB/s of codes and scales), one sequence of 262144 x 8 kv rows 69 us
// (4.4 TB/s): half of the ALU's and of the issue slots go into unpacking codes, the rest is the latency of a warp's dependent
// steps, for which the registers leave room for eight warps.  16 bits, 64 x 4 kv rows of 4100 x 128 80 us (6.7 TB/s): memory.  A
// few hundred tokens: 5 to 7 us, launch and two round trips to memory.
#include <algorithm>
#include <type_traits>

#include "kvm_tma_host.cuh"
#include "kvm_window.cuh"

namespace kvm {

namespace {

constexpr int kMathWarps = 8;
constexpr int kMaxStages = 8;
constexpr int kBox = 128;                     // rows per TMA box (16 bits; the end of a cache comes in boxes of 16)
constexpr int kSmemPerSm = 228 * 1024;        // of which every CTA takes 1 KB more than it asks for
constexpr int kMaxBatch = 1024;               // sequences per launch
constexpr float kLowest = -3.402823466e38f;   // reference of the weights before the first score: no finite one is below it
constexpr unsigned kScaleUp = 6;              // see R below

// How a variant works.  4 bits: bound by the math warps (conversions and fixed latencies), which is why a warp takes T = 4 groups of
// 16 rows of a chunk side by side; head dimensions below 128 leave the registers for two CTAs per SM.  Short caches of 128
// channels are bound by the changes from kv row to kv row, which two CTAs with smaller chunks (T = 2) overlap: 64 x 8 kv
// rows of 516 tokens 19.9 us against 26.6, 8 x 16 of 4096 25.9 against 23.2 (see kShortRows).  The copies, one per chunk, are
// issued by math warp 0.
// 16 bits: bound by memory (64 x 4 kv rows of 4100 x 128, 4 query heads each: 80 us, 6.7 TB/s): one CTA, chunks of 64 KB at every
// head dimension, copied in boxes of 128 rows (of 16 rows throughout: 97 us; 64 x 8 of 4100 x 32: 48 us against 83) by a
// producer warp of its own (by math warp 0: 64 x 16 of 516 x 128 54 us against 46).
template <int D_, int BITS_, int NH_, int T_>
struct TokGeom {
  static constexpr int D = D_, BITS = BITS_, NH = NH_;           // NH: blocks of 8 query heads per kv head
  static constexpr int kTiles = T_;                              // groups of 16 rows per warp and chunk
  static constexpr int kChunk = kMathWarps * 16 * kTiles;        // rows per chunk
  static constexpr bool kProducer = BITS == 16;
  static constexpr int kThreads = (kMathWarps + (kProducer ? 1 : 0)) * 32;
  static constexpr int kCtas = BITS == 4 && (D * NH < 128 || (D == 128 && NH == 1 && T_ == 2)) ? 2 : 1;  // per SM
  static constexpr int kStageKv = BITS == 4 ? kChunk / 16 * Block4<D>::kBytes : 2 * kChunk * D * 2;
  static constexpr int kBoxW = D >= 64 ? 64 : 32;                // elements per box
  static constexpr int kBlocks = D / kBoxW;
};
constexpr int kShortRows = 1536;  // cache rows per kv row up to which the variant for short caches runs

struct TokSmem {
  int stage_bytes, q, ored, vscale, wred, bars, pre, total;
  template <typename GM>
  __host__ __device__ TokSmem(GM, int G, int nb, int stages) {
    constexpr int D = GM::D;
    q = GM::kStageKv;                                          // [G][D] bf16 behind the stage's rows
    stage_bytes = (q + G * D * 2 + 1023) & ~1023;            // (boxes in the 128-byte swizzle start on 1024 bytes)
    int off = stages * stage_bytes;
    ored = off; off += kMathWarps * G * D * 4;
    vscale = off; off += kMathWarps * GM::kTiles * D;              // a warp's value scales as f16
    wred = off; off += 2 * kMathWarps * 16 * 4;
    bars = off; off += 2 * kMaxStages * 8 + 16;              // full, empty, abort flag
    pre = off;  off += (2 * nb + 1) * 4;
    total = (off + 15) & ~15;
  }
};

struct TokMaps {
  CUtensorMap k, v, k_end, v_end;  // [all rows][D], boxes of kBox rows, of 16 rows
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {  // (2^-23; of 0: infinity)
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mma_f16_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
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

// Which rows the last of n tokens sees: of the ring those whose token is less than `limit` behind the newest.
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
  // chunks [from, to) of n rows are seen whole
  __device__ __forceinline__ void whole_chunks(int n, int& from, int& to) const {
    const int lo = limit == ring ? sp : max(sp, sp + newest - limit + 1);  // (of a ring that has wrapped around, those below the newest row)
    from = (lo + n - 1) / n;
    to = (limit == ring ? live : min(live, sp + newest + 1)) / n;
  }
  // rows [r, r + 16) (r a multiple of 16) as a bit mask, one lane per row
  __device__ __forceinline__ unsigned group(int r, int lane) const {
    return __ballot_sync(0xffffffffu, visible(r + (lane & 15))) & 0xffffu;
  }
};

// A place in the flat list.
struct Place {
  int b, h, c, n_chunks;  // sequence, kv head, chunk of the kv row, chunks of the kv row
};

// Partial result of a kv row that a CTA's range cuts: [head][m, l, output[D]], the output divided by l.
__host__ __device__ inline size_t partial_floats(int D, int G) { return (size_t)G * (D + 2); }

// The split of the list, the same in both kernels.  whole_rows: ranges end between kv rows.
struct Split {
  int total, per;  // units (chunks, or kv rows) of the list, per CTA
  __device__ __forceinline__ Split(int units, int grid) {
    total = units;
    per = max(1, (units + grid - 1) / grid);
  }
};

// Tokens of every sequence (pre[nb + 1 ..]) and its chunks per kv row as a prefix (pre[0..nb]) in shared memory.
__device__ __forceinline__ void build_prefix(const WindowDev& W, SeqInts lens, int extra, int chunk, int b0, int nb, int* pre, int tid,
                                             int threads) {
  for (int b = tid; b < nb; b += threads) {
    const int n = max(lens.at(b0 + b), -1) + extra;
    pre[nb + 1 + b] = n;
    pre[b + 1] = (W.live(n) + chunk - 1) / chunk;
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
  int lo = 0, hi = nb - 1;  // last b with pre[b] * Hkv <= f: one that has chunks
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (pre[mid] * Hkv <= f) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// N 32-bit words from shared memory (16 N-byte, at most 16-byte, aligned)
template <int N>
__device__ __forceinline__ void lds(uint32_t (&x)[N], const void* p) {
  if constexpr (N == 4) {
    const uint4 y = *static_cast<const uint4*>(p);
    x[0] = y.x; x[1] = y.y; x[2] = y.z; x[3] = y.w;
  } else if constexpr (N == 2) {
    const uint2 y = *static_cast<const uint2*>(p);
    x[0] = y.x; x[1] = y.y;
  } else {
    x[0] = *static_cast<const uint32_t*>(p);
  }
}

// The new token's row into row rr of a 4-bit block, in the stage and in memory (whole warp; items of 4 channels of K, then V).
template <int D>
__device__ __forceinline__ void patch4(unsigned char* sb, unsigned char* gb, const bf16* kn, const bf16* vn, int rr, int lane) {
  constexpr int NG = D / 32;
#pragma unroll
  for (int it = 0; it < (D == 128 ? 2 : 1); ++it) {
    const int item = it * 32 + lane, value = item >= D / 4, c4 = value ? item - D / 4 : item;
    const bool some = item < D / 2;
    const uint2 x = some ? *reinterpret_cast<const uint2*>((value ? vn : kn) + c4 * 4) : make_uint2(0, 0);
    unsigned am = __vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu);
    am = max(am & 0xffffu, am >> 16);
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) am = max(am, __shfl_xor_sync(0xffffffffu, am, d));  // 8 lanes hold a group
    float inv;
    const unsigned short sc = group_scale(am, inv);
    unsigned code = e2m1x4(levels_of(x.x, inv), levels_of(x.y, inv));
    if (am >= 0x7f80u) code = 0;
    const int grp = c4 >> 3, u = c4 & 7;
    const int off = value ? Block4<D>::kValues + rr * (D / 2) + u * (2 * NG) + grp * 2
                          : Block4<D>::kKeys + rr * (D / 2) + (u >> 1) * (4 * NG) + grp * 4 + (u & 1) * 2;
    const int soff = value ? Block4<D>::kValueScales + (rr >> 1) * (4 * NG) + grp * 4 + (rr & 1) * 2
                           : Block4<D>::kKeyScales + rr * (2 * NG) + grp * 2;
    if (some) {
      *reinterpret_cast<unsigned short*>(sb + off) = (unsigned short)code;
      *reinterpret_cast<unsigned short*>(gb + off) = (unsigned short)code;
      if (u == 0) {
        *reinterpret_cast<unsigned short*>(sb + soff) = sc;
        *reinterpret_cast<unsigned short*>(gb + soff) = sc;
      }
    }
  }
}

}  // namespace

template <typename GM>
__global__ void __launch_bounds__(GM::kThreads, GM::kCtas)
kvm_window_token_kernel(WindowDev W, int G, Tensor4 q, Tensor4 k_new, Tensor4 v_new, SeqInts lens, int b0, int nb, int stages,
                        int whole_rows, float scale_log2, float* __restrict__ partial, bf16* __restrict__ out, int* __restrict__ status,
                        const __grid_constant__ TokMaps maps) {
  constexpr int D = GM::D, BITS = GM::BITS, NH = GM::NH, NG = D / 32, NT = GM::kTiles, CH = GM::kChunk;
  constexpr uint32_t kAll = 0xffffffffu;
  extern __shared__ __align__(1024) unsigned char smem[];
  const TokSmem lay(GM{}, G, nb, stages);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + lay.bars);
  uint64_t* empty = full + kMaxStages;
  int* pre = reinterpret_cast<int*>(smem + lay.pre);
  const int* tokens = pre + nb + 1;
  volatile int* abort_flag = reinterpret_cast<int*>(empty + kMaxStages);
  const int tid = threadIdx.x, warp = __shfl_sync(kAll, tid >> 5, 0), lane = tid & 31;
  const int Hkv = W.Hkv, Hq = Hkv * G;
  const bool with_new = k_new.ptr != nullptr;

  if (tid == 0) {
    for (int s = 0; s < stages; ++s) {
      tc::mbar_init(&full[s], 1);
      tc::mbar_init(&empty[s], kMathWarps);
    }
    tc::fence_barrier_init();
    *abort_flag = 0;
  }
  pdl_wait();
  pdl_trigger();  // (the join kernel may be staged; it waits for this grid)
  build_prefix(W, lens, with_new ? 1 : 0, CH, b0, nb, pre, tid, GM::kThreads);  // (with a new token lens are its positions)
  const int total_f = pre[nb] * Hkv;

  // this CTA's range [f_begin, f_end) of the list
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
      for (int i = tid; i < Hq * D / 8; i += GM::kThreads)
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
  auto next_row = [&](Place& p) {
    p.c = 0;
    if (++p.h < Hkv) return;
    p.h = 0;
    do { ++p.b; } while (p.b < nb && pre[p.b + 1] == pre[p.b]);
    if (p.b < nb) p.n_chunks = pre[p.b + 1] - pre[p.b];
  };
  auto give_up = [&]() {
    if (lane == 0) {
      *abort_flag = 1;
      atomicExch(status, KVM_ERR_DEVICE_TIMEOUT);
    }
  };

  // Chunk `pp` of the list into stage s, by a whole warp.
  Place pp = pl;
  auto load = [&](int s, bool first_of_range) {
    unsigned char* st = smem + s * lay.stage_bytes;
    const int rows = min(CH, W.live(tokens[pp.b]) - pp.c * CH), groups = (rows + 15) >> 4;
    const size_t kvrow = (size_t)(b0 + pp.b) * Hkv + pp.h;
    const bool first = first_of_range || pp.c == 0;  // the kv row's queries come with its first chunk
    if (lane == 0) {
      const uint32_t bytes = (BITS == 4 ? (uint32_t)groups * Block4<D>::kBytes : (uint32_t)groups * (2u * 16u * D * 2u)) + (first ? (uint32_t)(G * D * 2) : 0u);
      tc::mbar_arrive_expect_tx(&full[s], bytes);
    }
    __syncwarp();
    if (BITS == 4) {
      if (lane == 0)
        tc::bulk_g2s(st, W.blocks + (kvrow * (W.rows / 16) + (size_t)pp.c * (CH / 16)) * Block4<D>::kBytes, groups * Block4<D>::kBytes, &full[s]);
    } else {
      const int y = (int)(kvrow * W.rows) + pp.c * CH;  // (all rows of a cache: below 2^31, checked on the host)
      const int large = groups / (kBox / 16), boxes = large + groups % (kBox / 16);
      for (int j = lane; j < boxes * GM::kBlocks * 2; j += 32) {
        const int half = j / (boxes * GM::kBlocks), k2 = j % (boxes * GM::kBlocks), blk = k2 / boxes, box = k2 % boxes;
        const int row = min(box, large) * kBox + max(box - large, 0) * 16;
        tc::tma_load_2d(st + half * (CH * D * 2) + (blk * CH + row) * (GM::kBoxW * 2),
                        box < large ? (half ? &maps.v : &maps.k) : (half ? &maps.v_end : &maps.k_end), blk * GM::kBoxW, y + row, &full[s]);
      }
    }
    if (first && lane < G) tc::bulk_g2s(st + lay.q + lane * D * 2, q.row(b0 + pp.b, pp.h * G + lane, 0), D * 2, &full[s]);
    if (++pp.c == pp.n_chunks) next_row(pp);
  };
  if (GM::kProducer && warp == kMathWarps) {
    int s = 0, parity = 0;
    for (int i = 0; i < nloc; ++i) {
      if (i >= stages) {
        if (!__all_sync(kAll, tc::mbar_wait(&empty[s], parity ^ 1) && !*abort_flag)) {
          give_up();
          __nanosleep(1000000);  // copies in flight
          break;
        }
      }
      load(s, i == 0);
      if (++s == stages) { s = 0; parity ^= 1; }
    }
    return;
  }
  if (!GM::kProducer && warp == 0)
    for (int i = 0; i < min(stages, nloc); ++i) load(i, i == 0);

  const int g = lane >> 2, t = lane & 3;
  float* ored = reinterpret_cast<float*>(smem + lay.ored);          // [warp][G][D]
  float* wmax = reinterpret_cast<float*>(smem + lay.wred);          // [warp][16]
  float* wsum = wmax + kMathWarps * 16;
  uint32_t* vsc = reinterpret_cast<uint32_t*>(smem + lay.vscale + warp * NT * D);
  bool ok = true;  // false: a wait ran out; the warp goes on without data so that it meets the others at their barriers
  int s = 0, parity = 0;             // stage of the chunk, parity of its use
  int rs = 0, rparity = 0;           // of the chunk before it

  for (int i = 0; i < nloc;) {  // kv rows, or what of them lies in the range
    const int cnt = min(pl.n_chunks - pl.c, nloc - i), n = tokens[pl.b];
    const Seen seen(W, n);
    const int new_row = with_new ? W.row_of(n - 1) : -1, new_chunk = with_new ? new_row / CH : -1;
    int plain_from, plain_to;  // chunks that are seen whole
    seen.whole_chunks(CH, plain_from, plain_to);
    uint32_t qf[NH][D / 16][2];      // queries as B fragments
    float qs[NH][2], qd[NH][2];      // of this thread's heads 2t, 2t + 1: what scores are multiplied by, and 4 bits: a group's sums
    float o[NH][D / 16][4];          // output: channels x heads
    float m[NH][2], l[NH][2];
    unsigned r_bits = 0;             // 4 bits: R of group lane % NG, as the exponent field of a bf16 pattern (0: none yet)
#pragma unroll
    for (int hb = 0; hb < NH; ++hb) {
      m[hb][0] = m[hb][1] = kLowest;
      l[hb][0] = l[hb][1] = 0.f;
#pragma unroll
      for (int j = 0; j < D / 16; ++j) o[hb][j][0] = o[hb][j][1] = o[hb][j][2] = o[hb][j][3] = 0.f;
    }

    for (int j = 0; j < cnt; ++j) {
      const int at = i + j;
      // the stage of the chunk before this one, which the other warps are done with by now or soon, takes a further chunk
      if (!GM::kProducer && warp == 0 && ok && at > 0 && at - 1 + stages < nloc) {
        ok = __all_sync(kAll, tc::mbar_wait(&empty[rs], rparity) && !*abort_flag);
        if (ok) load(rs, false);
        else give_up();
      }
      if (ok) {
        ok = __all_sync(kAll, tc::mbar_wait(&full[s], parity) && !*abort_flag);
        if (!ok) give_up();
      }
      unsigned char* st = smem + s * lay.stage_bytes;
      if (j == 0) {
#pragma unroll
        for (int hb = 0; hb < NH; ++hb) {
          const bf16* qrow = reinterpret_cast<const bf16*>(st + lay.q) + (size_t)min(hb * 8 + g, G - 1) * D;
          if (BITS == 4) {
            uint32_t x[NG][4];
            unsigned amax = 0;
#pragma unroll
            for (int n2 = 0; n2 < NG; ++n2) {
              lds(x[n2], qrow + n2 * 32 + t * 8);
#pragma unroll
              for (int e = 0; e < 4; ++e) amax = __vmaxu2(amax, x[n2][e] & 0x7fff7fffu);
            }
            amax = max(amax & 0xffffu, amax >> 16);
            amax = max(amax, __shfl_xor_sync(kAll, amax, 1));
            amax = max(amax, __shfl_xor_sync(kAll, amax, 2));
            // largest magnitude into [2^14, 2^15): a value loses bits only if it is 2^28 below it (infinities and NaN stay
            // what they are)
            const int e = min(max((int)(amax >> 7) - 127, -112), 127);
            const bool finite = amax < 0x7f80u;
            const float up = finite ? __uint_as_float((unsigned)(127 + 14 - e) << 23) : 1.f;
            const float down = finite ? __uint_as_float((unsigned)(127 - 14 + e) << 23) : 1.f;
#pragma unroll
            for (int n2 = 0; n2 < NG; ++n2)
#pragma unroll
              for (int e2 = 0; e2 < 4; ++e2) {
                const float2 f = unpack_bf16(x[n2][e2]);
                qf[hb][n2 * 2 + (e2 >> 1)][e2 & 1] = pack_f16(f.x * up, f.y * up);
              }
            // this thread's scores are of heads 2t, 2t + 1: their factors lie in lanes 8t, 8t + 4.  The part of a factor that
            // makes sums smaller goes to a group's sums ahead of the keys' scale, the part that makes them larger to the
            // scores: neither passes fp32's range unless the score does.
#pragma unroll
            for (int e2 = 0; e2 < 2; ++e2) {
              const float f = __shfl_sync(kAll, down, 8 * t + 4 * e2) * scale_log2;
              qd[hb][e2] = fminf(f, 1.f);
              qs[hb][e2] = fminf(fmaxf(f, 1.f), 3e38f);
            }
          } else {
            constexpr int PER = D >= 64 ? 4 : 2;  // k-steps per 64 (32) channels; a thread's channels are contiguous
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) lds(qf[hb][kk], qrow + (kk / PER) * 64 + t * (PER * 4) + (kk % PER) * 4);
            qs[hb][0] = qs[hb][1] = scale_log2;
          }
        }
      }

      // ---- this warp's rows: groups of 16, kMathWarps * 16 apart
      const int chunk0 = (pl.c + j) * CH, row0 = chunk0 + warp * 16;
      const bool has_new = pl.c + j == new_chunk;
      // which of this warp's rows are to be seen, 16 bits per group
      constexpr unsigned long long kWhole = NT == 4 ? ~0ull : (1ull << (16 * NT)) - 1;
      unsigned long long seen_rows = ok ? kWhole : 0;
      auto vis = [&](int u) { return (unsigned)(seen_rows >> (16 * u)) & 0xffffu; };
      bool patched = false;
      if (ok && (has_new || pl.c + j < plain_from || pl.c + j >= plain_to)) {
        seen_rows = 0;
#pragma unroll
        for (int u = 0; u < NT; ++u) seen_rows |= (unsigned long long)seen.group(row0 + u * (kMathWarps * 16), lane) << (16 * u);
        // the new token's row: into the stage (what was loaded there is stale) and into memory
#pragma unroll
        for (int u = 0; u < NT; ++u) {
          const int r = row0 + u * (kMathWarps * 16);
          if (has_new && (new_row >> 4) == (r >> 4)) {
            patched = true;
            const size_t kvrow = (size_t)(b0 + pl.b) * Hkv + pl.h;
            const bf16* kn = k_new.row(b0 + pl.b, pl.h, 0);
            const bf16* vn = v_new.row(b0 + pl.b, pl.h, 0);
            if (BITS == 4) {
              patch4<D>(st + (warp + u * kMathWarps) * Block4<D>::kBytes,
                        W.blocks + (kvrow * (W.rows / 16) + (new_row >> 4)) * Block4<D>::kBytes, kn, vn, new_row & 15, lane);
            } else {
              for (int e = lane; e < D / 4; e += 32) {  // 16-byte pieces of K, then of V
                const bool value = e >= D / 8;
                const int c = value ? e - D / 8 : e, rr = new_row - chunk0;
                const uint4 x = *reinterpret_cast<const uint4*>((value ? vn : kn) + c * 8);
                unsigned char* base = st + (value ? CH * D * 2 : 0);
                if (D >= 64) base += (c >> 3) * (CH * 128) + rr * 128 + (((c & 7) ^ (rr & 7)) << 4);
                else base += rr * 64 + c * 16;
                *reinterpret_cast<uint4*>(base) = x;
                *reinterpret_cast<uint4*>((value ? W.v : W.k) + (kvrow * W.rows + new_row) * D + c * 8) = x;
              }
            }
            __syncwarp();
          }
        }
        if (BITS == 4 && seen_rows && seen_rows != kWhole) {  // rows that are not to be seen: scale 0, they add nothing
          patched = true;
#pragma unroll
          for (int u = 0; u < NT; ++u) {
            unsigned char* sb = st + (warp + u * kMathWarps) * Block4<D>::kBytes;
            for (int e = lane; e < 16 * NG; e += 32) {
              const int rr = e / NG, grp = e % NG;
              if (!((vis(u) >> rr) & 1)) {
                *reinterpret_cast<unsigned short*>(sb + Block4<D>::kKeyScales + rr * (2 * NG) + grp * 2) = 0;
                *reinterpret_cast<unsigned short*>(sb + Block4<D>::kValueScales + (rr >> 1) * (4 * NG) + grp * 4 + (rr & 1) * 2) = 0;
              }
            }
          }
          __syncwarp();
        }
      }
      // groups u0 .. u0 + N - 1 of this warp's rows
      auto groups = [&](auto count, int u0) {
        constexpr int N = decltype(count)::value;
        if (BITS == 4) {  // the value scales relative to R as f16, each lane a pair of rows' of a group
          uint32_t x[N], top2 = 0;
#pragma unroll
          for (int u = 0; u < N; ++u) {
            x[u] = lane < 8 * NG ? *reinterpret_cast<const uint32_t*>(st + (warp + (u0 + u) * kMathWarps) * Block4<D>::kBytes + Block4<D>::kValueScales + lane * 4) : 0u;
            top2 = __vmaxs2(top2, x[u]);  // (the NaN of a scale is negative: it reaches its own group only)
          }
          unsigned top = max(top2 & 0xffffu, top2 >> 16) & 0x7f80u;
          if (__any_sync(kAll, top > r_bits)) {  // a group's R rises, to the exponent of the largest of its scales
#pragma unroll
            for (int d = NG; d < 8 * NG; d <<= 1) top = max(top, __shfl_xor_sync(kAll, top, d));
            const float down = top <= r_bits ? 1.f : r_bits ? __uint_as_float((unsigned)max(127 + (int)(r_bits >> 7) - (int)(top >> 7), 0) << 23) : 0.f;
            r_bits = max(r_bits, top);
#pragma unroll
            for (int k2 = 0; k2 < D / 16; ++k2) {
              const float a = __shfl_sync(kAll, down, k2 >> 1);
#pragma unroll
              for (int hb = 0; hb < NH; ++hb)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[hb][k2][e] *= a;
            }
          }
          // (a scale is below 2 R here, a weight at most 2^8: with 2^6 / R, f16 just holds the product)
          const unsigned e_r = r_bits >> 7;
          const float inv = __uint_as_float((254u - e_r + min(e_r, kScaleUp)) << 23);
#pragma unroll
          for (int u = 0; u < N; ++u)
            if (lane < 8 * NG) vsc[u * 8 * NG + lane] = pack_f16(__uint_as_float(x[u] << 16) * inv, __uint_as_float(x[u] & 0xffff0000u) * inv);
          __syncwarp();
        }

        // ---- scores: rows g, g + 8 x heads 2t, 2t + 1
        float sc[N][NH][4];
#pragma unroll
        for (int u = 0; u < N; ++u) {
#pragma unroll
          for (int hb = 0; hb < NH; ++hb) sc[u][hb][0] = sc[u][hb][1] = sc[u][hb][2] = sc[u][hb][3] = 0.f;
          if constexpr (BITS == 4) {
            const unsigned char* sb = st + (warp + (u0 + u) * kMathWarps) * Block4<D>::kBytes;
            uint32_t kw[2][NG];
            float ks[2][NG];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const int rr = g + 8 * r;
              lds(kw[r], sb + Block4<D>::kKeys + rr * (D / 2) + t * (4 * NG));
              const unsigned char* sp = sb + Block4<D>::kKeyScales + rr * (2 * NG);
              if constexpr (NG == 1) {
                ks[r][0] = __uint_as_float((unsigned)*reinterpret_cast<const unsigned short*>(sp) << 16);
              } else {
                uint32_t y[NG / 2];
                lds(y, sp);
#pragma unroll
                for (int e = 0; e < NG; ++e) ks[r][e] = __uint_as_float((e & 1) ? y[e / 2] & 0xffff0000u : y[e / 2] << 16);
              }
            }
#pragma unroll
            for (int n2 = 0; n2 < NG; ++n2) {
              uint32_t a[4], c[4];
              e2m1_to_f16x2(kw[0][n2], a[0], a[1], a[2], a[3]);
              e2m1_to_f16x2(kw[1][n2], c[0], c[1], c[2], c[3]);
#pragma unroll
              for (int hb = 0; hb < NH; ++hb) {
                float acc[4];
                mma_f16_zero(acc, a[0], c[0], a[1], c[1], qf[hb][n2 * 2][0], qf[hb][n2 * 2][1]);
                mma_f16(acc, a[2], c[2], a[3], c[3], qf[hb][n2 * 2 + 1][0], qf[hb][n2 * 2 + 1][1]);
                const float2 f = make_float2(qd[hb][0], qd[hb][1]);
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                  const float2 y = __ffma2_rn(__fmul2_rn(make_float2(acc[2 * r], acc[2 * r + 1]), f), make_float2(ks[r][n2], ks[r][n2]),
                                              make_float2(sc[u][hb][2 * r], sc[u][hb][2 * r + 1]));
                  sc[u][hb][2 * r] = y.x;
                  sc[u][hb][2 * r + 1] = y.y;
                }
              }
            }
          } else {
            const int r = (warp + (u0 + u) * kMathWarps) * 16 + g;
#pragma unroll
            for (int blk = 0; blk < GM::kBlocks; ++blk) {
              constexpr int PIECES = GM::kBoxW / 32;  // 16-byte pieces per thread and row: 2 (64 channels) or 1
#pragma unroll
              for (int pc = 0; pc < PIECES; ++pc) {
                const int c = t * PIECES + pc;
                const unsigned char* base = D >= 64 ? st + blk * (CH * 128) + r * 128 + ((c ^ (r & 7)) << 4) : st + r * 64 + c * 16;
                uint32_t x[4], y[4];
                lds(x, base);
                lds(y, base + 8 * (D >= 64 ? 128 : 64));
#pragma unroll
                for (int hb = 0; hb < NH; ++hb) {
                  const int kk = (blk * PIECES + pc) * 2;
                  mma_bf16(sc[u][hb], x[0], y[0], x[1], y[1], qf[hb][kk][0], qf[hb][kk][1]);
                  mma_bf16(sc[u][hb], x[2], y[2], x[3], y[3], qf[hb][kk + 1][0], qf[hb][kk + 1][1]);
                }
              }
            }
          }
        }

        // ---- in units of log2, each rounded as a number of its own: as a fused product and difference below, a score of 2^31
        // would lie further from its own rounded value than a weight reaches.  (Before the mask: a scale may be as small as to
        // count as 0, and 0 x inf is NaN.)
#pragma unroll
        for (int u = 0; u < N; ++u)
#pragma unroll
          for (int hb = 0; hb < NH; ++hb) {
            // (scalar products: a packed one and a sum may be made one fused operation, even with the rounding named)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[u][hb][e] = __fmul_rn(sc[u][hb][e], qs[hb][e & 1]);
          }
        // ---- weights up to 2^kTop of the largest.  4 bits: f16 holds 2^-24 .. 2^15; the reference m is that much below the running
        // maximum, but from 2^26 on, where the difference might be rounded beyond f16's range, the maximum itself.  16 bits:
        // small enough that 2^24 of the largest bf16 numbers stay inside fp32's range; m is the maximum, kTop a sum of its own.
        constexpr float kTop = BITS == 4 ? 8.f : -24.f;
        float alpha[NH][2];
#pragma unroll
        for (int hb = 0; hb < NH; ++hb) {
          if (seen_rows != kWhole) {
#pragma unroll
            for (int u = 0; u < N; ++u)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (!((vis(u0 + u) >> (g + (e >> 1) * 8)) & 1)) sc[u][hb][e] = -INFINITY;
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = fmaxf(sc[0][hb][e], sc[0][hb][e + 2]);
#pragma unroll
            for (int u = 1; u < N; ++u) x = fmaxf(x, fmaxf(sc[u][hb][e], sc[u][hb][e + 2]));
            x = fmaxf(x, __shfl_xor_sync(kAll, x, 4));
            x = fmaxf(x, __shfl_xor_sync(kAll, x, 8));
            x = fmaxf(x, __shfl_xor_sync(kAll, x, 16));
            const float top = fmaxf(m[hb][e], BITS == 4 && fabsf(x) < 0x1p26f ? x - kTop : x);
            alpha[hb][e] = ex2(m[hb][e] - top);
            m[hb][e] = top;
          }
        }
        // (always: the FMA pipe is idle, and without a branch the rest of the chunk mixes with it)
#pragma unroll
        for (int hb = 0; hb < NH; ++hb) {
          l[hb][0] *= alpha[hb][0];
          l[hb][1] *= alpha[hb][1];
          const float2 a = make_float2(alpha[hb][0], alpha[hb][1]);
#pragma unroll
          for (int e = 0; e < D / 16; ++e) {
            const float2 x = __fmul2_rn(make_float2(o[hb][e][0], o[hb][e][1]), a), y = __fmul2_rn(make_float2(o[hb][e][2], o[hb][e][3]), a);
            o[hb][e][0] = x.x; o[hb][e][1] = x.y; o[hb][e][2] = y.x; o[hb][e][3] = y.y;
          }
        }
        uint32_t pb[N][NH][2];  // weights as B fragments: rows (2t, 2t + 1), (2t + 8, 2t + 9) of head g
#pragma unroll
        for (int u = 0; u < N; ++u)
#pragma unroll
          for (int hb = 0; hb < NH; ++hb) {
            float p[4];
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
              float2 x = __fadd2_rn(make_float2(sc[u][hb][e], sc[u][hb][e + 1]), make_float2(-m[hb][0], -m[hb][1]));
              if (BITS == 16) x = __fadd2_rn(x, make_float2(kTop, kTop));
              p[e] = ex2(x.x);
              p[e + 1] = ex2(x.y);
            }
            l[hb][0] += p[0] + p[2];
            l[hb][1] += p[1] + p[3];
            pb[u][hb][0] = movmatrix_trans(BITS == 4 ? pack_f16(p[0], p[1]) : pack_bf16(p[0], p[1]));
            pb[u][hb][1] = movmatrix_trans(BITS == 4 ? pack_f16(p[2], p[3]) : pack_bf16(p[2], p[3]));
          }

        // ---- output += V^T P
#pragma unroll
        for (int u = 0; u < N; ++u) {
          if constexpr (BITS == 4) {
            const unsigned char* sb = st + (warp + (u0 + u) * kMathWarps) * Block4<D>::kBytes;
            uint32_t vs[2][NG];  // value scales of row pairs t and t + 4
            lds(vs[0], vsc + u * 8 * NG + t * NG);
            lds(vs[1], vsc + u * 8 * NG + (t + 4) * NG);
            constexpr int NWD = NG > 1 ? NG / 2 : 1;  // 32-bit words of codes per thread and row
            uint32_t vw[4][NWD];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const unsigned char* p = sb + Block4<D>::kValues + (2 * t + (r & 1) + 8 * (r >> 1)) * (D / 2) + g * (2 * NG);
              if constexpr (NG > 1) lds(vw[r], p);
              else vw[r][0] = *reinterpret_cast<const unsigned short*>(p);
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
                  const uint32_t p0 = mul_f16x2(pb[u][hb][0], vs[0][n2]), p1 = mul_f16x2(pb[u][hb][1], vs[1][n2]);
#pragma unroll
                  for (int y = 0; y < 2; ++y)  // channels 32 n2 + 4 g + 2 y (rows g) and + 1 (rows g + 8)
                    mma_f16(o[hb][n2 * 2 + y], ea[half * 2 + y], da[half * 2 + y], eb[half * 2 + y], db[half * 2 + y], p0, p1);
                }
              }
            }
          } else {
            const unsigned char* vb = st + CH * D * 2;
#pragma unroll
            for (int blk = 0; blk < GM::kBlocks; ++blk) {
              constexpr int WORDS = D >= 64 ? 4 : 2;
              uint32_t x[4][WORDS];
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const int rr = (warp + (u0 + u) * kMathWarps) * 16 + 2 * t + (r & 1) + 8 * (r >> 1);
                lds(x[r], D >= 64 ? vb + blk * (CH * 128) + rr * 128 + ((g ^ (rr & 7)) << 4) : vb + rr * 64 + g * 8);
                if (seen_rows != kWhole && !((vis(u0 + u) >> (rr & 15)) & 1)) {  // (0 x NaN)
#pragma unroll
                  for (int w = 0; w < WORDS; ++w) x[r][w] = 0;
                }
              }
#pragma unroll
              for (int w = 0; w < WORDS; ++w) {
                const uint32_t a0 = __byte_perm(x[0][w], x[1][w], 0x5410), a1 = __byte_perm(x[0][w], x[1][w], 0x7632);
                const uint32_t a2 = __byte_perm(x[2][w], x[3][w], 0x5410), a3 = __byte_perm(x[2][w], x[3][w], 0x7632);
#pragma unroll
                for (int hb = 0; hb < NH; ++hb) mma_bf16(o[hb][blk * 4 + w], a0, a1, a2, a3, pb[u][hb][0], pb[u][hb][1]);
              }
            }
          }
        }
      };
      if (seen_rows) {
        // side by side; a single group with rows to be seen (the end of a cache) by itself
        const int lowest = (__ffsll((long long)seen_rows) - 1) >> 4;
        if (NT == 1 || (seen_rows >> (16 * lowest)) > 0xffffu) groups(std::integral_constant<int, NT>{}, 0);
        else groups(std::integral_constant<int, 1>{}, lowest);
        if (patched) tc::fence_proxy_async();  // before the next copy into this stage
      }
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&empty[s]);
      rs = s;
      rparity = parity;
      if (++s == stages) { s = 0; parity ^= 1; }
    }

    // ---- join the warps
    // (outputs are divided by their sums at once, so that none passes fp32's range on the way)
    float up[NG];  // what the outputs of a group are to be multiplied by
#pragma unroll
    for (int n2 = 0; n2 < NG; ++n2) {
      const unsigned r = __shfl_sync(kAll, r_bits, n2);
      up[n2] = BITS == 4 ? __uint_as_float(r << 16) * __uint_as_float((127u - min(r >> 7, kScaleUp)) << 23) : 1.f;
    }
#pragma unroll
    for (int hb = 0; hb < NH; ++hb) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x = l[hb][e];
        x += __shfl_xor_sync(kAll, x, 4);
        x += __shfl_xor_sync(kAll, x, 8);
        x += __shfl_xor_sync(kAll, x, 16);
        const float inv = x == 0.f ? 0.f : rcp(x);
        const int head = hb * 8 + 2 * t + e;
        if (g == 0) {
          wmax[warp * 16 + head] = m[hb][e];
          wsum[warp * 16 + head] = x;
        }
        if (head < G) {
          float* dst = ored + ((size_t)warp * G + head) * D;
#pragma unroll
          for (int k2 = 0; k2 < D / 16; ++k2) {
            // 4 bits: channels 32 (k2/2) + 4 g + 2 (k2%2) + {0, 1};  16 bits: 64 (k2/4) + 8 g + 2 (k2%4) + {0, 1}, and for
            // D = 32: 4 g + 2 k2 + {0, 1}
            const int ch = BITS == 4 || D == 32 ? (k2 >> 1) * 32 + 4 * g + 2 * (k2 & 1) : (k2 >> 2) * 64 + 8 * g + 2 * (k2 & 3);
            *reinterpret_cast<float2*>(dst + ch) = make_float2(o[hb][k2][e] * inv * up[k2 >> 1], o[hb][k2][e + 2] * inv * up[k2 >> 1]);
          }
        }
      }
    }
    math_sync();
    const bool whole = pl.c == 0 && cnt == pl.n_chunks;
    const int slot = pl.c > 0 ? 0 : 1;  // of a cut row's partial results: it goes on here, or it begins here
    for (int x = tid; x < G * D / 2; x += kMathWarps * 32) {
      const int head = x / (D / 2), ch = (x % (D / 2)) * 2;
      float mx = kLowest;
#pragma unroll
      for (int w = 0; w < kMathWarps; ++w) mx = fmaxf(mx, wmax[w * 16 + head]);
      float f[kMathWarps], sum = 0.f, a0 = 0.f, a1 = 0.f;
#pragma unroll
      for (int w = 0; w < kMathWarps; ++w) {
        f[w] = ex2(wmax[w * 16 + head] - mx) * wsum[w * 16 + head];
        sum += f[w];
      }
      // (no score above -inf: NaN, 0 x inf, if that is all of the kv row; a share of one that is cut adds zeros)
      const float inv = sum == 0.f && !whole ? 0.f : rcp(sum);
#pragma unroll
      for (int w = 0; w < kMathWarps; ++w) {
        const float2 y = *reinterpret_cast<const float2*>(ored + ((size_t)w * G + head) * D + ch);
        a0 = fmaf(y.x, f[w] * inv, a0);
        a1 = fmaf(y.y, f[w] * inv, a1);
      }
      if (whole) {
        *reinterpret_cast<uint32_t*>(out + ((size_t)(b0 + pl.b) * Hq + pl.h * G + head) * D + ch) = pack_bf16(a0, a1);
      } else {
        float* dst = partial + ((size_t)blockIdx.x * 2 + slot) * partial_floats(D, G) + (size_t)head * (D + 2);
        *reinterpret_cast<float2*>(dst + 2 + ch) = make_float2(a0, a1);
        if (ch == 0) *reinterpret_cast<float2*>(dst) = make_float2(mx, sum);
      }
    }
    math_sync();
    i += cnt;
    next_row(pl);
  }
  if (!ok) __nanosleep(1000000);  // copies in flight
}

// Joins the partial results of a kv row that range boundaries cut, one block per (row, query head): block x is kv row x of the
// launch, or, where there are more kv rows than boundaries, the row that boundary x + 1 cuts first.  The weights of all
// partial results first (one load latency), then their weighted sum with independent loads.  Its launch and latency cost 2.5 us
// behind the main kernel (262144 tokens of one sequence, eight kv rows of 18 or 19 parts: 68 us in all).
template <int D>
__global__ void __launch_bounds__(256)
kvm_window_join_kernel(WindowDev W, int G, SeqInts lens, int extra, int chunk, int b0, int nb, int grid, int by_row,
                       const float* __restrict__ partial, bf16* __restrict__ out) {
  constexpr int COLS = D / 2, GROUPS = 256 / COLS;  // column pairs; partial results are dealt out over GROUPS sets of threads
  extern __shared__ int pre[];
  __shared__ float red[2][8];
  __shared__ float2 part[256];
  const int tid = threadIdx.x, head = blockIdx.y;
  // The main kernel lets this one start once its own wait is over: the lengths may be read ahead of its end.  Blocks without
  // work wait for it all the same: what follows in the stream waits for this grid, and through it for the main one.
  build_prefix(W, lens, extra, chunk, b0, nb, pre, tid, 256);
  float* weight = reinterpret_cast<float*>(pre + 2 * nb + 1);
  const int Hkv = W.Hkv;
  const Split sp(pre[nb] * Hkv, grid);
  int b, h, row0, nc;
  if (by_row) {
    b = blockIdx.x / Hkv;
    h = blockIdx.x % Hkv;
    nc = pre[b + 1] - pre[b];
    row0 = pre[b] * Hkv + h * nc;
  } else {
    const int f = ((int)blockIdx.x + 1) * sp.per;
    if (f >= sp.total) return pdl_wait();
    b = find_seq(pre, nb, Hkv, f);
    nc = pre[b + 1] - pre[b];
    const int rem = f - pre[b] * Hkv;
    h = rem / nc;
    row0 = f - rem % nc;
    if (row0 / sp.per != (int)blockIdx.x) return pdl_wait();  // another boundary's
  }
  if (nc == 0) return pdl_wait();
  const int c0 = row0 / sp.per, c1 = (row0 + nc - 1) / sp.per, n = c1 - c0 + 1;  // CTAs that hold parts of the row
  pdl_wait();
  if (n < 2) return;
  // the row begins in CTA c0 (its second partial result) and goes on in the others (their first)
  auto src = [&](int i) { return partial + ((size_t)(c0 + i) * 2 + (i == 0 ? 1 : 0)) * partial_floats(D, G) + (size_t)head * (D + 2); };
  float mx = kLowest;
  for (int i = tid; i < n; i += 256) mx = fmaxf(mx, src(i)[0]);
  mx = warp_max(mx);
  if ((tid & 31) == 0) red[0][tid >> 5] = mx;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) mx = fmaxf(mx, red[0][w]);
  float sum = 0.f;
  for (int i = tid; i < n; i += 256) {
    const float2 ml = *reinterpret_cast<const float2*>(src(i));
    const float f = ex2(ml.x - mx) * ml.y;
    weight[i] = f;
    sum += f;
  }
  sum = warp_sum(sum);
  if ((tid & 31) == 0) red[1][tid >> 5] = sum;
  __syncthreads();
  sum = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) sum += red[1][w];
  const float inv = rcp(sum);
  const int col = tid % COLS, grp = tid / COLS;
  float2 acc = make_float2(0.f, 0.f);
#pragma unroll 8
  for (int i = grp; i < n; i += GROUPS) {
    const float2 x = *reinterpret_cast<const float2*>(src(i) + 2 + col * 2);
    const float f = weight[i] * inv;
    acc.x = fmaf(f, x.x, acc.x);
    acc.y = fmaf(f, x.y, acc.y);
  }
  part[tid] = acc;
  __syncthreads();
  if (grp == 0) {
    for (int i = 1; i < GROUPS; ++i) {
      acc.x += part[i * COLS + col].x;
      acc.y += part[i * COLS + col].y;
    }
    *reinterpret_cast<uint32_t*>(out + ((size_t)(b0 + b) * Hkv * G + h * G + head) * D + col * 2) = pack_bf16(acc.x, acc.y);
  }
}

namespace {

// How a call of nb sequences is launched.
struct TokPlan {
  // sequences whose lengths fit beside two stages
  template <typename GM>
  static int sequences(int G, int limit) {
    int n = kMaxBatch;
    while (n > 16 && TokSmem(GM{}, G, n, 2).total > limit) n -= 16;
    return n;
  }
  // Whole kv rows per CTA where cutting them gains less than it costs.  Fitted to both ways of 170 calls (1 to 64 sequences of
  // 256 to 16384 tokens, all variants): a chunk takes about 1.7 us (4 bits) or 0.8 us (16 bits), all of them together no less
  // than their bytes at 6.5 TB/s; cutting costs 2.5 us for the second launch (taken as 3.5: outside a graph the host needs 4 us
  // for it) and 2.5 more where a CTA's share covers more than a chunk and so, as a rule, parts of two rows.  8 sequences of 512
  // tokens with 16 heads x 128, 4 bits: 9.1 us whole, 12.4 cut; of 16384 with 4 heads: 73 whole, 26 cut.  The rule's choices
  // take 1 % more than the better ones in sum, 20 % at worst (16 bits, 8 x 2048 tokens, 8 heads x 128: 16.2 for 13.4).
  template <typename GM>
  static bool whole_rows(const WindowDev& W, int nb, int ctas) {
    const int max_chunks = (W.rows + GM::kChunk - 1) / GM::kChunk;
    const long long rows = (long long)nb * W.Hkv, chunks = rows * max_chunks, per = (chunks + ctas - 1) / ctas;
    const double chunk_us = GM::BITS == 4 ? 1.7 : 0.8, copy_us = GM::kStageKv / 6.5e6;
    // (rounds of a row per CTA: the last one may leave CTAs, and the memory, idle)
    const long long rounds = rows / ctas, rest = rows % ctas;
    const double whole = max_chunks * (rounds * std::max(chunk_us, ctas * copy_us) + (rest ? std::max(chunk_us, rest * copy_us) : 0.0));
    return whole <= std::max(per * chunk_us, chunks * copy_us) + (per > 1 ? 5.0 : 3.5);
  }
};

template <typename GM>
struct TokLaunch {
  static constexpr int D = GM::D, BITS = GM::BITS;
  static constexpr int kSmemLimit = kSmemPerSm / GM::kCtas - 1024;

  static size_t workspace(const WindowDev& W, int G) {
    const int ctas = window_sm_count() * GM::kCtas, per = TokPlan::sequences<GM>(G, kSmemLimit);
    for (int b0 = 0; b0 < W.batch; b0 += per)
      if (!TokPlan::whole_rows<GM>(W, std::min(per, W.batch - b0), ctas)) return (size_t)ctas * 2 * partial_floats(D, G) * 4;
    return 0;
  }

  static cudaError_t run(const WindowDev& W, int G, Tensor4 q, Tensor4 k_new, Tensor4 v_new, SeqInts lens, float scale, float* partial,
                         bf16* out, int* status, cudaStream_t stream) {
    TokMaps maps;
    if (BITS == 16) {
      const cuuint64_t dims[2] = {(cuuint64_t)D, (cuuint64_t)W.batch * W.Hkv * W.rows};
      const cuuint64_t strides[1] = {(cuuint64_t)D * 2};
      const cuuint32_t box[2] = {(cuuint32_t)GM::kBoxW, (cuuint32_t)kBox}, end[2] = {(cuuint32_t)GM::kBoxW, 16};
      if (!encode_bf16_map(&maps.k, W.k, 2, dims, strides, box) || !encode_bf16_map(&maps.v, W.v, 2, dims, strides, box) ||
          !encode_bf16_map(&maps.k_end, W.k, 2, dims, strides, end) || !encode_bf16_map(&maps.v_end, W.v, 2, dims, strides, end))
        return cudaErrorInvalidValue;
    }
    auto kern = kvm_window_token_kernel<GM>;
    static std::atomic<unsigned long long> raised{0};
    cudaError_t e = raise_smem_limit(kern, kSmemLimit, raised);
    if (e != cudaSuccess) return e;
    const int ctas = window_sm_count() * GM::kCtas, per = TokPlan::sequences<GM>(G, kSmemLimit);
    const int max_chunks = (W.rows + GM::kChunk - 1) / GM::kChunk;
    for (int b0 = 0; b0 < W.batch; b0 += per) {
      const int nb = std::min(per, W.batch - b0);
      int stages = 2;
      while (stages < kMaxStages && TokSmem(GM{}, G, nb, stages + 1).total <= kSmemLimit) ++stages;
      const bool whole = TokPlan::whole_rows<GM>(W, nb, ctas);
      const long long rows = (long long)nb * W.Hkv;
      const int grid = (int)std::min<long long>(ctas, whole ? rows : rows * max_chunks);
      e = launch_pdl(kern, dim3(grid), dim3(GM::kThreads), TokSmem(GM{}, G, nb, stages).total, stream, true, W, G, q, k_new, v_new,
                     lens, b0, nb, stages, whole ? 1 : 0, scale * kLog2e, partial, out, status, maps);
      if (e != cudaSuccess) return e;
      if (!whole && grid > 1) {
        const bool by_row = rows < grid;
        e = launch_pdl(kvm_window_join_kernel<D>, dim3(by_row ? (int)rows : grid - 1, G), dim3(256), (2 * nb + 1 + grid) * 4, stream, true, W,
                       G, lens, k_new.ptr ? 1 : 0, GM::kChunk, b0, nb, grid, by_row ? 1 : 0, (const float*)partial, out);
        if (e != cudaSuccess) return e;
      }
    }
    return cudaSuccess;
  }
};

template <int D, int NH>
struct TokTiles {  // groups per warp and chunk, 4 bits
  static constexpr int value = D * NH == 256 ? 2 : 4;
};

template <typename F>
auto token_variant(int D, int bits, const WindowDev& W, int G, F f) {
  auto heads = [&](auto d, auto h) {
    constexpr int kD = decltype(d)::value, kH = decltype(h)::value;
    if (bits == 16) return f(TokLaunch<TokGeom<kD, 16, kH, 128 / kD>>{});
    if constexpr (kD == 128 && kH == 1) {
      if (W.rows <= kShortRows) return f(TokLaunch<TokGeom<kD, 4, kH, 2>>{});
    }
    return f(TokLaunch<TokGeom<kD, 4, kH, TokTiles<kD, kH>::value>>{});
  };
  auto width = [&](auto h) {
    return D == 128 ? heads(std::integral_constant<int, 128>{}, h)
                    : D == 64 ? heads(std::integral_constant<int, 64>{}, h) : heads(std::integral_constant<int, 32>{}, h);
  };
  return G <= 8 ? width(std::integral_constant<int, 1>{}) : width(std::integral_constant<int, 2>{});
}

}  // namespace

size_t window_token_workspace(int D, int bits, const WindowDev& W, int G) {
  return token_variant(D, bits, W, G, [&](auto v) { return v.workspace(W, G); });
}

cudaError_t window_token_dispatch(int D, int bits, const WindowDev& W, int G, Tensor4 q, Tensor4 k_new, Tensor4 v_new, SeqInts lens,
                                  float scale, float* partial, bf16* out, int* status, cudaStream_t stream) {
  return token_variant(D, bits, W, G, [&](auto v) { return v.run(W, G, q, k_new, v_new, lens, scale, partial, out, status, stream); });
}

}  // namespace kvm
