// Attention of a prompt, or of a chunk of one behind earlier tokens, with a sliding window and sinks: query t stands at
// position S - T + t and sees position j if j <= p and (j > p - window or j < sinks).  tcgen05 + tensor memory.
//
// One persistent CTA per SM; a work item is two query tiles of 128 rows that share their key and value tiles of 128 rows:
// two query heads of one kv head over the same queries where the heads per kv head are even in number, else 256 queries of
// one head.  The tiles of an item: those of the sinks that lie before the window, then the window's, from the first key that
// the item's first query sees to its last query.
//
//   producer (1 warp)      one thread: tiled TMA copies of the query tiles and, through a ring of slots, of K0, V0, K1, ...
//   MMA (1 warp)           one thread: S = Q K^T into tensor memory; O += P V with P as the tensor-memory A operand, in two
//                          parts (64 keys each) as the softmax delivers them.  P lies over the scores it came from, so the next
//                          scores follow behind P V; while one tile is in its softmax the other has the tensor core.
//   softmax (4 warps per tile)  one query row per thread: scores from tensor memory, mask (only where a tile is not seen
//                          whole), running maximum (raised, and O rescaled, when a tile exceeds it by 2^8), exp2, row sum
//                          (fp32), P as bf16; behind the last tile O / l to global memory.
// Infinities and NaN in values that a row does not see: a masked weight is 0, and 0 x inf would reach the row through the
// product.  Value rows behind a sequence's length are cleared in shared memory; for any other, a row whose sum is finite
// but whose output is not is marked, and formed again from the keys that it sees when its warp's last tile is done (revisit).
// Every wait is bounded; one that runs out sets the status word, and the CTA leaves through its common exit.
//
// Measured (32 / 8 heads x 128, 8192 queries over all earlier tokens): 461 us, 1190 TFLOP/s; 2 x 32768 queries, 16 heads x 128,
// window 4096: 1.86 ms (2.15 ms in a long run, at the power limit of 1000 W and 1.5 GHz); 64 channels, 2 x 8192 queries, 16 / 4
// heads, window 2048: 185 us, 650 TFLOP/s.  With a constant in place of the softmax the first takes 443 us: what bounds it is the tensor
// core (1024 of about 1400 clocks per 128 x 128 tile; its operands and the copies share the bandwidth of shared memory) and the
// hand-overs to the issuing warp, at 64 channels the hand-overs and the exponentials (52 % of the special-function unit).  One issuing warp
// with uniform operands instead of one thread: 615 -> 472 us; registers 208 / 88 instead of 224 / 56, which spills: 712 -> 615.
#include <algorithm>
#include <type_traits>

#include "kvm_tma_host.cuh"
#include "kvm_window.cuh"

namespace kvm {

namespace {

constexpr int kRows = 128;   // queries per tile, keys per tile
constexpr int kThreads = 384;
constexpr int kProducerWarp = 8, kMmaWarp = 9;
constexpr float kRescale = 8.0f;  // log2 units
constexpr int kMaxListed = 500;   // sequences of a batch of unequal lengths whose tiles are listed
constexpr int kSplit = 2;         // of 4 x 32 keys, those whose weights are handed to the MMA warp first (2: 461 us, 3: 465)
constexpr int kPoly = 4;          // of 16 pairs of weights, those formed by polynomial (none: 487 us, 4: 475, 8: 493)
constexpr int kRegsSoftmax = 208, kRegsOther = 88, kRegsLaunch = 168;
static_assert(256 * kRegsSoftmax + 128 * kRegsOther <= kThreads * kRegsLaunch, "register split above the block's registers");

// DP: head dimension as the tiles hold it (64 or 128; one of 32 is padded with zeros by the copies)
template <int DP>
struct PC {
  static constexpr int kTileBytes = kRows * DP * 2;
  static constexpr int kSlots = DP == 128 ? 5 : 8;
  static constexpr int kOffKv = 2 * kTileBytes;
  static constexpr int kOffBar = kOffKv + kSlots * kTileBytes;
  static constexpr int kOffPre = kOffBar + 512;
  static constexpr int kSmem = kOffPre + (kMaxListed + 1) * 4;
  static constexpr uint32_t kColO = 256;  // first column of the outputs; scores of tile i in columns 128 i ..
};

struct PromptBars {
  uint64_t q_full[2], q_empty[2], kv_full[8], kv_empty[8], s_full[2], p_full[2][2], o_final[2], o_free[2];
  uint32_t tmem_base;
};

struct PromptArgs {
  int B, Hq, Hkv, D, T, S, window, sinks, pair_heads, n_items, units, q_tiles;  // units: (sequence, head or head pair)
  float scale_log2;
  const int* lengths;
  bf16* out;
  int* status;
  Tensor4 q, k, v;
  CUtensorMap mq, mk, mv;
  int q_head_inner, k_head_inner, v_head_inner;
};

// What an item is, computed alike by every role.  LISTED: batches of unequal lengths, whose items are the tiles that exist, found
// through a prefix over the sequences (6 padded prompts of up to 2011 tokens, 64 channels: 46 us against 72; a template: the
// few registers cost the others 2 %).  The prefix of larger batches would take too much shared memory from the tiles.
template <bool LISTED>
struct Item {
  int b, hkv, len, lo, s_end, n_sink, n_tiles;  // first window key, end of the sinks before it, their tiles, tiles in all
  int hq[2], t0[2], begin[2], end[2];           // per query tile: head, first query, window tiles [begin, end) in list places
  __device__ __forceinline__ Item(const PromptArgs& a, const int* pre, int x) {
    const int per_seq = a.units / a.B, G = a.Hq / a.Hkv;
    int qt, hu;
    if (LISTED) {  // sequence by sequence, later tiles first
      const int t = x / per_seq;
      int lo_b = 0, hi_b = a.B - 1;  // last b with pre[b] <= t: one that has tiles
      while (lo_b < hi_b) {
        const int mid = (lo_b + hi_b + 1) >> 1;
        if (pre[mid] <= t) lo_b = mid; else hi_b = mid - 1;
      }
      b = lo_b;
      qt = pre[b + 1] - 1 - t;
      hu = x % per_seq;
    } else {  // later, heavier tiles of all sequences first
      qt = a.q_tiles - 1 - x / a.units;
      b = (x % a.units) / per_seq;
      hu = x % per_seq;
    }
    if (a.pair_heads) {
      hq[0] = hu * 2;
      hq[1] = hq[0] + 1;
      t0[0] = t0[1] = qt * kRows;
    } else {
      hq[0] = hq[1] = hu;
      t0[0] = qt * 2 * kRows;
      t0[1] = t0[0] + kRows;
    }
    hkv = hq[0] / G;
    len = a.lengths ? min(max(a.lengths[b], 0), a.S) : a.S;
    const int at = a.S - a.T;
    lo = max(0, at + t0[0] - a.window + 1);
    int hi_all = 0;
    s_end = min(a.sinks, lo);
    n_sink = (s_end + kRows - 1) / kRows;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int p0 = at + t0[i], hi = min(min(at + a.T, p0 + kRows), len);  // first query's position, end of the seen keys
      begin[i] = end[i] = 0;
      if (t0[i] < a.T && p0 < len) {
        // (sinks inside the window's tiles: from its first one on)
        const int lo_i = a.sinks > lo ? lo : max(lo, p0 - a.window + 1);
        begin[i] = n_sink + (lo_i - lo) / kRows;
        end[i] = n_sink + (hi - lo + kRows - 1) / kRows;
      }
      hi_all = max(hi_all, end[i]);
    }
    n_tiles = hi_all;
  }
  __device__ __forceinline__ int key0(int u) const { return u < n_sink ? u * kRows : lo + (u - n_sink) * kRows; }
  // (i: 0 or 1; picked so that the item stays in registers)
  __device__ __forceinline__ int pick(const int (&x)[2], int i) const { return i ? x[1] : x[0]; }
  __device__ __forceinline__ bool uses(int i, int u) const { return u < n_sink ? pick(end, i) > 0 : u >= pick(begin, i) && u < pick(end, i); }
  __device__ __forceinline__ int count(int i) const { return pick(end, i) > 0 ? n_sink + pick(end, i) - pick(begin, i) : 0; }
};

// Bounded wait without pauses of its own between the tries: the roles hand tiles to each other several times per microsecond,
// and a pause that overshoots is on the path of both.  What is waited for comes within microseconds.  A try that fails has
// waited for about 2700 clocks: 2^22 of them are some 6 s.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity) {
  for (uint32_t i = 0; i < (1u << 22); ++i)
    if (tc::mbar_try_wait(bar, parity)) return true;
  return false;
}
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)); }
// One thread of a converged warp, the same one every time.
__device__ __forceinline__ bool elected() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {  // NaN if any of them is
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float fma_sat(float a, float b, float c) {  // clamped to [0, 1]
  float d;
  asm("fma.rn.sat.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// 2^x for two x, given as y = (x + 127) / 256 clamped to [0, 1]: x <= -127 gives exactly 0, as below the smallest number.
// Range reduction to the nearest integer and a polynomial 1 + f (a + b f + c f^2) on [-1/2, 1/2], minimax in the relative error by
// linear programming: 1.07e-4, an eighteenth of the bf16 rounding that follows.  (With a constant term of its own it would be
// 7.5e-5, but 2^-127 no longer the pattern of 0: just below 1 it wraps around to a negative number.)  On the FMA pipes: the
// special-function unit makes 16 exponentials per clock and SM, and both query tiles' softmaxes want 128 x 128 each for every
// 2048 clocks of the tensor core.
__device__ __forceinline__ float2 ex2_fma(float2 y) {
  constexpr float kMagic = 12582912.f;  // 1.5 * 2^23: adding it rounds to an integer, which stands in the low bits
  const float2 t = __ffma2_rn(y, make_float2(256.f, 256.f), make_float2(kMagic - 127.f, kMagic - 127.f));
  const float2 n = __fadd2_rn(t, make_float2(127.f - kMagic, 127.f - kMagic));  // the integer + 127
  const float2 f = __ffma2_rn(y, make_float2(256.f, 256.f), make_float2(-n.x, -n.y));
  float2 p = __ffma2_rn(f, make_float2(0.05500893294811249f, 0.05500893294811249f), make_float2(0.2422109693288803f, 0.2422109693288803f));
  p = __ffma2_rn(f, p, make_float2(0.6932829022407532f, 0.6932829022407532f));
  p = __ffma2_rn(f, p, make_float2(1.f, 1.f));
  return make_float2(__uint_as_float(__float_as_uint(p.x) + (__float_as_uint(t.x) << 23)),
                     __uint_as_float(__float_as_uint(p.y) + (__float_as_uint(t.y) << 23)));
}
__device__ __forceinline__ void load_box(void* dst, const CUtensorMap* m, bool head_inner, int x, int t, int h, int b, uint64_t* bar) {
  if (head_inner) tc::tma_load_4d(dst, m, x, h, t, b, bar);
  else tc::tma_load_4d(dst, m, x, t, h, b, bar);
}
template <int DP>
__device__ __forceinline__ void load_tile(unsigned char* dst, const CUtensorMap* m, bool head_inner, int t, int h, int b, uint64_t* bar) {
  tc::mbar_arrive_expect_tx(bar, PC<DP>::kTileBytes);
#pragma unroll
  for (int x = 0; x < DP; x += 64) load_box(dst + x * kRows * 2, m, head_inner, x, t, h, b, bar);
}

// ------------------------------------------------------------------------------------------ producer
template <int DP, bool LISTED>
__device__ __forceinline__ bool produce(const PromptArgs& a, const int* pre, int n_items, unsigned char* smem, PromptBars* bars) {
  int slot = 0, round = 0;  // of the ring
  auto kv = [&](const CUtensorMap* m, bool hi, int key, const Item<LISTED>& it) {
    if (round > 0 && !wait(&bars->kv_empty[slot], (round - 1) & 1)) return false;
    load_tile<DP>(smem + PC<DP>::kOffKv + slot * PC<DP>::kTileBytes, m, hi, key, it.hkv, it.b, &bars->kv_full[slot]);
    if (++slot == PC<DP>::kSlots) { slot = 0; ++round; }
    return true;
  };
  int nq[2] = {0, 0};
  for (int x = blockIdx.x; x < n_items; x += gridDim.x) {
    const Item<LISTED> it(a, pre, x);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (it.end[i] == 0) continue;
      if (nq[i] > 0 && !wait(&bars->q_empty[i], (nq[i] - 1) & 1)) return false;
      load_tile<DP>(smem + i * PC<DP>::kTileBytes, &a.mq, a.q_head_inner, it.t0[i], it.hq[i], it.b, &bars->q_full[i]);
      ++nq[i];
    }
    for (int u = 0; u < it.n_tiles; ++u) {
      if (!kv(&a.mk, a.k_head_inner, it.key0(u), it)) return false;
      if (!kv(&a.mv, a.v_head_inner, it.key0(u), it)) return false;
    }
  }
  return true;
}

// ------------------------------------------------------------------------------------------ MMA issue
// One thread for both query tiles, so that the products of one tile run as a block (P V of its last tile, then the scores of
// the next) while the other is in its softmax.  (Two issuing threads interleave on the tensor core: both tiles' scores then
// come late and together, both softmaxes run at the same time, and the tensor core idles meanwhile.)  Step u: P V of
// tile u - 1 and Q K of tile u, for query tile 0, then for 1; it goes on from item to item.
// The issuing warp is the narrowest part of the pipeline: operand descriptors differ in the low word's address field only (no
// carry leaves it), so that an MMA costs one 32-bit addition per operand.
__device__ __forceinline__ void mma_ss_lo(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}"
      :
      : "r"(d), "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_ts_lo(uint32_t d, uint32_t a_tmem, uint32_t b_lo, uint32_t hi, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 b, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}"
      :
      : "r"(d), "r"(a_tmem), "r"(b_lo), "r"(hi), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}

template <int DP>
struct Issuer {
  static constexpr uint32_t kIdescQk = tc::make_idesc(kRows, kRows, 0, 0), kIdescPv = tc::make_idesc(kRows, DP, 0, 1);
  static constexpr uint32_t kTile = PC<DP>::kTileBytes >> 4;
  PromptBars* bars;
  uint32_t dq, dk, dv, hi;  // low words of the first query tile's, slot 0's key and value descriptors; the high word
  uint32_t tmem;
  int n[2] = {0, 0}, nq[2] = {0, 0};   // tiles whose P V is issued, items begun
  bool pending[2] = {false, false}, first[2], last[2];
  int pv_slot = 0, pv_parity = 0;      // value slot of the pending tiles
  bool slot_held = false;

  template <int I>
  __device__ __forceinline__ bool pv() {  // of the pending tile
    if (!pending[I]) return true;
    pending[I] = false;
    if (first[I] && nq[I] > 1 && !warp_wait(&bars->o_free[I], (nq[I] - 2) & 1)) return false;  // the last item's output has been read
    if (!warp_wait(&bars->kv_full[pv_slot], pv_parity)) return false;
    const uint32_t v_lo = dv + pv_slot * kTile;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (!warp_wait(&bars->p_full[I][half], n[I] & 1)) return false;
      tc::tc_fence_after_sync();
      if (elected()) {
#pragma unroll
        for (int s = half * kSplit * 2; s < (half ? 8 : kSplit * 2); ++s)
          mma_ts_lo(tmem + PC<DP>::kColO + I * DP, tmem + I * 128 + s * 8, v_lo + s * (2048 >> 4), hi, kIdescPv, !first[I] || s > 0);
        if (half == 1 && last[I]) tc::mma_commit(&bars->o_final[I]);
      }
      __syncwarp();
    }
    ++n[I];
    return true;
  }
  template <int I>
  __device__ __forceinline__ bool qk(int k_slot, bool is_first, bool is_last) {
    if (is_first) {
      if (!warp_wait(&bars->q_full[I], nq[I] & 1)) return false;
      ++nq[I];
    }
    const uint32_t k_lo = dk + k_slot * kTile;
    tc::tc_fence_after_sync();
    if (elected()) {
#pragma unroll
      for (int s = 0; s < DP / 16; ++s) {
        const uint32_t off = ((s >> 2) * (kRows * 128) + (s & 3) * 32) >> 4;
        mma_ss_lo(tmem + I * 128, dq + I * kTile + off, k_lo + off, hi, kIdescQk, s > 0);
      }
      tc::mma_commit(&bars->s_full[I]);
      if (is_last) tc::mma_commit(&bars->q_empty[I]);
    }
    __syncwarp();
    pending[I] = true;
    first[I] = is_first;
    last[I] = is_last;
    return true;
  }
  __device__ __forceinline__ void commit(uint64_t* bar) {
    if (elected()) tc::mma_commit(bar);
    __syncwarp();
  }
};

template <int DP, bool LISTED>
__device__ __forceinline__ bool issue(const PromptArgs& a, const int* pre, int n_items, unsigned char* smem, PromptBars* bars, uint32_t tmem) {
  Issuer<DP> is;
  is.bars = bars;
  is.tmem = tmem;
  const uint64_t d0 = tc::make_desc(tc::smem_u32(smem), 16, 1024);
  is.dq = (uint32_t)d0;
  is.hi = (uint32_t)(d0 >> 32);
  is.dk = (uint32_t)tc::make_desc(tc::smem_u32(smem + PC<DP>::kOffKv), 16, 1024);
  is.dv = (uint32_t)tc::make_desc(tc::smem_u32(smem + PC<DP>::kOffKv), kRows * 128, 1024);  // (the high words are alike)
  int slot = 0, round = 0;
  for (int x = blockIdx.x; x < n_items; x += gridDim.x) {
    const Item<LISTED> it(a, pre, x);
    const int cnt0 = it.count(0), cnt1 = it.count(1);
    int done0 = 0, done1 = 0;
    for (int u = 0; u < it.n_tiles; ++u) {
      const int ks = slot, kr = round & 1;
      if (++slot == PC<DP>::kSlots) { slot = 0; ++round; }
      const int vs = slot, vr = round & 1;
      if (++slot == PC<DP>::kSlots) { slot = 0; ++round; }
      if (!warp_wait(&bars->kv_full[ks], kr)) return false;
      if (!is.template pv<0>()) return false;
      if (it.uses(0, u)) {
        ++done0;
        if (!is.template qk<0>(ks, done0 == 1, done0 == cnt0)) return false;
      }
      if (!is.template pv<1>()) return false;
      if (it.uses(1, u)) {
        ++done1;
        if (!is.template qk<1>(ks, done1 == 1, done1 == cnt1)) return false;
      }
      if (elected()) {
        if (is.slot_held) tc::mma_commit(&bars->kv_empty[is.pv_slot]);
        tc::mma_commit(&bars->kv_empty[ks]);
      }
      __syncwarp();
      is.pv_slot = vs;
      is.pv_parity = vr;
      is.slot_held = true;
    }
  }
  return is.template pv<0>() && is.template pv<1>();
}

// ------------------------------------------------------------------------------------------ softmax
// Rows to be formed again.  The tiles leave a mark in the first column that is concerned, a NaN that no conversion makes: the
// row's scores are numbers, but not all of the tensor core's sums are.  An infinity or NaN among the values did that, of a key that
// the row sees or of one that it does not (0 x inf), or sums beyond fp32.
// Another mark, in the first column, asks for all of the row's columns: its maximum is beyond 2^16.  The tiles form a weight from
// a fused product and difference, which lies off the rounded maximum by up to half a step: 2^-8 there, from 2^31 on more than
// a weight holds.  The second pass rounds every score as it rounds the maximum.  (As a variant of the tiles' weights it took 1 to
// 5 % of every prompt's time.)
constexpr unsigned kAgain = 0x7fc5, kAllAgain = 0x7fc6;
constexpr float kFar = 0x1p16f;

// Columns [c0, c0 + 32) of the 32 query rows of a warp (one per lane), in each row those of `bad`.  First the values that the rows
// see are looked through, a key per lane: columns that hold a NaN or infinity get theirs (NaN for an infinity whose weight is 0).
// What is left is summed again over the keys that the row sees, a row per lane, with normalised weights; their maximum and sum
// are formed once per row (`have`).
struct Again {
  const PromptArgs& a;
  int b, hq, hkv, t, p, lo, ns, n;  // the keys that any of the rows sees: the first ns, then those from lo on
  float m, inv;
  bool have, large_q;  // (large_q: of any row's query)
  static constexpr unsigned kAll = 0xffffffffu;
  static constexpr int kKeys = 8;   // at a time: as many loads in flight
  __device__ __forceinline__ int key(int i) const { return i < ns ? i : lo + i - ns; }
  __device__ __forceinline__ bool sees(int i) const {
    const int j = key(i);
    return i < n && j <= p && (j > p - a.window || j < a.sinks);
  }
  // scores of keys i0 .. i0 + 7, in units of log2
  __device__ __forceinline__ void scores(int i0, float (&x)[kKeys]) const {
    const bf16* qr = a.q.row(b, hq, t);
    float2 s[kKeys];
#pragma unroll
    for (int e = 0; e < kKeys; ++e) s[e] = make_float2(0.f, 0.f);
#pragma unroll 1
    for (int d = 0; d < a.D; d += 8) {
      const uint4 y = *reinterpret_cast<const uint4*>(qr + d);
#pragma unroll
      for (int e = 0; e < kKeys; ++e) {
        const uint4 z = *reinterpret_cast<const uint4*>(a.k.row(b, hkv, key(min(i0 + e, n - 1))) + d);
        s[e] = __ffma2_rn(unpack_bf16(y.x), unpack_bf16(z.x), s[e]);
        s[e] = __ffma2_rn(unpack_bf16(y.y), unpack_bf16(z.y), s[e]);
        s[e] = __ffma2_rn(unpack_bf16(y.z), unpack_bf16(z.z), s[e]);
        s[e] = __ffma2_rn(unpack_bf16(y.w), unpack_bf16(z.w), s[e]);
      }
    }
#pragma unroll
    for (int e = 0; e < kKeys; ++e) x[e] = __fmul_rn(s[e].x + s[e].y, a.scale_log2);
  }
  // Is there a channel of 2^40 or more, an infinity or NaN?  (Of queries and keys below it no score passes fp32's range.)
  static __device__ __forceinline__ bool beyond(const bf16* row, int D) {
    unsigned top = 0;
#pragma unroll 4
    for (int d = 0; d < D; d += 8) {
      const uint4 y = *reinterpret_cast<const uint4*>(row + d);
      top = __vmaxu2(top, __vmaxu2(__vmaxu2(y.x & 0x7fff7fffu, y.y & 0x7fff7fffu), __vmaxu2(y.z & 0x7fff7fffu, y.w & 0x7fff7fffu)));
    }
    return max(top & 0xffffu, top >> 16) >= (127u + 40u) << 7;
  }
  // is the score of key j -inf?
  __device__ __forceinline__ bool weightless(int j) const {
    const bf16 *qr = a.q.row(b, hq, t), *kr = a.k.row(b, hkv, j);
    float2 s = make_float2(0.f, 0.f);
#pragma unroll 4
    for (int d = 0; d < a.D; d += 8) {
      const uint4 y = *reinterpret_cast<const uint4*>(qr + d), z = *reinterpret_cast<const uint4*>(kr + d);
      s = __ffma2_rn(unpack_bf16(y.x), unpack_bf16(z.x), s);
      s = __ffma2_rn(unpack_bf16(y.y), unpack_bf16(z.y), s);
      s = __ffma2_rn(unpack_bf16(y.z), unpack_bf16(z.z), s);
      s = __ffma2_rn(unpack_bf16(y.w), unpack_bf16(z.w), s);
    }
    return s.x + s.y == -INFINITY;
  }
  __device__ __forceinline__ void columns(int c0, unsigned bad, int lane) {
    unsigned nan = 0, pos = 0, neg = 0;
#pragma unroll 2
    for (int i0 = 0; i0 < n; i0 += 32) {
      unsigned is_nan = 0, is_pos = 0, is_neg = 0;  // of the lane's key
      bool may_be = false;                          // weightless, for some row
      if (i0 + lane < n) {
        const uint4* vr = reinterpret_cast<const uint4*>(a.v.row(b, hkv, key(i0 + lane)) + c0);
        uint4 y[4];
        unsigned top = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          y[e] = vr[e];
          top = __vmaxu2(top, __vmaxu2(__vmaxu2(y[e].x & 0x7fff7fffu, y[e].y & 0x7fff7fffu), __vmaxu2(y[e].z & 0x7fff7fffu, y[e].w & 0x7fff7fffu)));
        }
        if (max(top & 0xffffu, top >> 16) >= 0x7f80u) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const unsigned ys[4] = {y[e].x, y[e].y, y[e].z, y[e].w};
#pragma unroll
            for (int z = 0; z < 8; ++z) {
              const unsigned u = (ys[z >> 1] >> (16 * (z & 1))) & 0xffffu, bit = 1u << (8 * e + z);
              if ((u & 0x7fffu) > 0x7f80u) is_nan |= bit;
              else if (u == 0x7f80u) is_pos |= bit;
              else if (u == 0xff80u) is_neg |= bit;
            }
          }
          may_be = large_q || beyond(a.k.row(b, hkv, key(i0 + lane)), a.D);
        }
      }
      const unsigned doubt = __ballot_sync(kAll, may_be);
      unsigned hits = __ballot_sync(kAll, (is_nan | is_pos | is_neg) != 0);
      if (hits == 0) continue;
      for (; hits; hits &= hits - 1) {
        const int src = __ffs(hits) - 1;
        const unsigned x = __shfl_sync(kAll, is_nan, src), y = __shfl_sync(kAll, is_pos, src), z = __shfl_sync(kAll, is_neg, src);
        if (!sees(i0 + src)) continue;
        nan |= x;
        if ((y | z) == 0) continue;
        if ((doubt >> src & 1) && weightless(key(i0 + src))) nan |= y | z;  // (0 x inf, of a key that is seen)
        else { pos |= y; neg |= z; }
      }
      if (!__any_sync(kAll, bad & ~(nan | (pos & neg)))) break;  // (settled whatever follows)
    }
    nan |= pos & neg;
    float acc[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) acc[i] = 0.f;
    if (__any_sync(kAll, bad & ~(nan | pos | neg))) {
      if (!have) {
        float sum = 0.f;
        m = -INFINITY;
#pragma unroll 1
        for (int i0 = 0; i0 < n; i0 += kKeys) {
          float x[kKeys], top = m;
          scores(i0, x);
#pragma unroll
          for (int e = 0; e < kKeys; ++e) {
            if (!sees(i0 + e)) x[e] = -INFINITY;
            top = fmaxf(top, x[e]);
          }
          if (top == -INFINITY) continue;
          sum *= ex2(m - top);
#pragma unroll
          for (int e = 0; e < kKeys; ++e) sum += ex2(x[e] - top);
          m = top;
        }
        inv = 1.0f / sum;
        have = true;
      }
#pragma unroll 1
      for (int i0 = 0; i0 < n; i0 += kKeys) {
        float x[kKeys];
        scores(i0, x);
#pragma unroll
        for (int e = 0; e < kKeys; ++e) {
          const float w = ex2(x[e] - m) * inv;
          const uint4* vr = reinterpret_cast<const uint4*>(a.v.row(b, hkv, key(min(i0 + e, n - 1))) + c0);
          const bool seen = sees(i0 + e);
#pragma unroll
          for (int z = 0; z < 4; ++z) {
            const uint4 y = vr[z];
            const unsigned ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const float2 h = unpack_bf16(ys[u]);
              if (seen) {
                acc[8 * z + 2 * u] = fmaf(w, h.x, acc[8 * z + 2 * u]);
                acc[8 * z + 2 * u + 1] = fmaf(w, h.y, acc[8 * z + 2 * u + 1]);
              }
            }
          }
          asm volatile("" ::: "memory");  // (one key's values at a time: registers)
        }
      }
    }
    bf16* dst = a.out + (((size_t)b * a.T + t) * a.Hq + hq) * a.D + c0;
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (bad >> i & 1)
        dst[i] = __float2bfloat16_rn((nan >> i & 1) ? __int_as_float(0x7fffffff) : (pos >> i & 1) ? INFINITY : (neg >> i & 1) ? -INFINITY : acc[i]);
  }
};

// The marked rows of a softmax warp, once its tiles are done: nobody waits for it any more, however long it takes.  For 32 rows of
// 128 channels: 14 ns per key and 32 columns to look through the values, 2.1 us per key to sum 32 columns again, 1.1 us for each
// further 32 (of 8192 keys 18 ms, all columns 46 ms).  Inside the tiles' loop a call took 2 to 4 % of every prompt's time.
template <bool LISTED>
__device__ __noinline__ void revisit(const PromptArgs& a, const int* pre, int n_items, int I, int row, int lane) {
  constexpr unsigned kAll = 0xffffffffu;
#pragma unroll 1
  for (int x = blockIdx.x; x < n_items; x += gridDim.x) {
    const Item<LISTED> it(a, pre, x);
    const int t = it.pick(it.t0, I) + row, p = a.S - a.T + t, hq = it.pick(it.hq, I);
    bool again = false;
    unsigned bad[4] = {0, 0, 0, 0};  // columns that hold no number
    if (t < a.T && p < it.len) {
      const uint4* src = reinterpret_cast<const uint4*>(a.out + (((size_t)it.b * a.T + t) * a.Hq + hq) * a.D);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        if (e * 8 >= a.D) break;
        const uint4 y = src[e];
        const unsigned ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int z = 0; z < 8; ++z) {
          const unsigned u = (ys[z >> 1] >> (16 * (z & 1))) & 0xffffu;
          if ((u & 0x7f80u) == 0x7f80u) bad[e >> 2] |= 1u << (8 * (e & 3) + z);
          again |= u == kAgain || u == kAllAgain;
          if (u == kAllAgain) bad[0] = bad[1] = bad[2] = bad[3] = 0xffffffffu;
        }
      }
    }
    if (!__any_sync(kAll, again)) continue;
    const int p_lo = __reduce_min_sync(kAll, again ? p : 0x7fffffff), p_hi = __reduce_max_sync(kAll, again ? p : -1);
    const int lo = max(0, p_lo - a.window + 1), ns = min(a.sinks, lo);
    Again rows{a, it.b, hq, it.hkv, again ? t : 0, again ? p : -1, lo, ns, ns + p_hi + 1 - lo, 0.f, 0.f, false, false};
    rows.large_q = __any_sync(kAll, again && Again::beyond(a.q.row(rows.b, rows.hq, rows.t), a.D));
#pragma unroll 1
    for (int c0 = 0; c0 < a.D; c0 += 32) {
      const unsigned mine = !again ? 0 : c0 < 64 ? (c0 < 32 ? bad[0] : bad[1]) : (c0 < 96 ? bad[2] : bad[3]);
      if (__any_sync(kAll, mine)) rows.columns(c0, mine, lane);
    }
  }
}

template <int DP, bool LISTED>
__device__ __forceinline__ bool softmax(const PromptArgs& a, const int* pre, int n_items, unsigned char* smem, PromptBars* bars, uint32_t tmem,
                                        int I, int row, int wq, int lane) {
  const uint32_t lane_addr = tmem + ((uint32_t)(wq * 32) << 16);
  const uint32_t col_s = lane_addr + I * 128, col_o = lane_addr + PC<DP>::kColO + I * DP;
  const float sc = a.scale_log2;
  int slot = 0, round = 0, n = 0, ni = 0;
  bool marked = false;
  for (int x = blockIdx.x; x < n_items; x += gridDim.x) {
    const Item<LISTED> it(a, pre, x);
    const int t = it.pick(it.t0, I) + row, p0 = a.S - a.T + it.pick(it.t0, I), p = p0 + row;
    float m_run = -INFINITY, l_run = 0.f;
    bool poison = false;
    int done = 0;
    for (int u = 0; u < it.n_tiles; ++u) {
      if (++slot == PC<DP>::kSlots) { slot = 0; ++round; }  // (the keys' slot)
      const int vs = slot, vr = round & 1;
      if (++slot == PC<DP>::kSlots) { slot = 0; ++round; }
      if (!it.uses(I, u)) continue;
      const int key0 = it.key0(u);
      if (!warp_wait(&bars->s_full[I], n & 1)) return false;
      tc::tc_fence_after_sync();
      uint32_t sr[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tc::tmem_ld32(col_s + c * 32, sr[c]);
      tc::tmem_ld_wait();
      // is the tile seen whole by all rows?
      const bool sink_tile = u < it.n_sink;
      const bool whole = sink_tile ? key0 + kRows <= it.s_end : key0 + kRows - 1 <= p0 && (key0 > p0 + kRows - 1 - a.window || key0 + kRows <= a.sinks);
      if (!whole) {
        // columns [c_lo, c_hi) and those below c_s are seen
        const int c_hi = sink_tile ? it.s_end - key0 : p + 1 - key0, c_lo = sink_tile ? 0 : p - a.window + 1 - key0;
        const int c_s = sink_tile ? 0 : a.sinks - key0;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          auto below = [](int k) { return k <= 0 ? 0u : (k >= 32 ? 0xffffffffu : (1u << k) - 1u); };
          const unsigned hi = below(c_hi - c * 32), seen = (hi & ~below(c_lo - c * 32)) | (hi & below(c_s - c * 32));
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (!((seen >> i) & 1u)) sr[c][i] = 0xff800000u;  // -inf
        }
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < 32; i += 2) {
#pragma unroll
        for (int c = 0; c < 4; ++c) mx[c] = max3(mx[c], __uint_as_float(sr[c][i]), __uint_as_float(sr[c][i + 1]));
      }
      const float tmax = max3(max3(mx[0], mx[1], mx[2]), mx[3], mx[3]) * sc;
      poison |= !(tmax < INFINITY);  // NaN or +inf among the scores: the row is NaN (the polynomial below does not carry a NaN on)
      const bool need = tmax > m_run + kRescale || (m_run == -INFINITY && tmax > -INFINITY);
      if (__any_sync(0xffffffffu, need)) {
        const float m_new = need ? tmax : m_run;
        const float alpha = m_run == -INFINITY ? 0.f : ex2(m_run - m_new);
        if (done > 0) {  // (P V of the last tile, issued ahead of these scores, is complete with them; that of this tile waits for this warp)
#pragma unroll 1
          for (int c = 0; c < DP; c += 16) {
            uint32_t o[16];
            tc::tmem_ld16(col_o + c, o);
            tc::tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tc::tmem_st16(col_o + c, o);
          }
          tc::tmem_st_wait();
        }
        l_run *= alpha;
        m_run = m_new;
      }
      // value rows behind the sequence's length: padding, cleared before the product reads them
      if (it.len < a.S && key0 + kRows > it.len) {
        if (!warp_wait(&bars->kv_full[vs], vr)) return false;
        if (key0 + row >= it.len) {
          unsigned char* vrow = smem + PC<DP>::kOffKv + vs * PC<DP>::kTileBytes + row * 128;
#pragma unroll
          for (int c = 0; c < DP / 8; ++c) *reinterpret_cast<uint4*>(vrow + (c >> 3) * (kRows * 128) + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
        }
        tc::fence_proxy_async();
      }
      // weights; where every key is seen, some by polynomial
      const float neg_m = m_run == -INFINITY ? 0.f : -m_run;
      const float2 sc2 = make_float2(sc, sc), nm2 = make_float2(neg_m, neg_m);
      const float sc256 = sc * (1.f / 256.f), nm256 = (neg_m + 127.f) * (1.f / 256.f);
      float2 ls = make_float2(0.f, 0.f);
      auto weights = [&](auto poly) {
#pragma unroll
        for (int part = 0; part < 2; ++part) {
#pragma unroll
          for (int c = part * kSplit; c < (part ? 4 : kSplit); ++c) {
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float s0 = __uint_as_float(sr[c][e * 2]), s1 = __uint_as_float(sr[c][e * 2 + 1]);
              float2 w;
              if (decltype(poly)::value && (e * kPoly) / 16 != ((e + 1) * kPoly) / 16) {  // (spread evenly)
                w = ex2_fma(make_float2(fma_sat(s0, sc256, nm256), fma_sat(s1, sc256, nm256)));
              } else {
                const float2 z = __ffma2_rn(make_float2(s0, s1), sc2, nm2);
                w = make_float2(ex2(z.x), ex2(z.y));
              }
              ls = __fadd2_rn(ls, w);
              pk[e] = pack_bf16(w.x, w.y);
            }
            tc::tmem_st16(col_s + c * 16, pk);
          }
          tc::tmem_st_wait();
          tc::tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(&bars->p_full[I][part]);
        }
      };
      if (whole) weights(std::true_type{});
      else weights(std::false_type{});
      l_run += ls.x + ls.y;
      ++done;
      ++n;
    }
    // ---- the item's output
    bf16* dst = a.out + (((size_t)it.b * a.T + t) * a.Hq + it.pick(it.hq, I)) * a.D;
    const bool mine = t < a.T;
    if (done == 0) {
      if (mine)
        for (int c = 0; c < a.D; c += 8) *reinterpret_cast<uint4*>(dst + c) = make_uint4(0, 0, 0, 0);
      continue;
    }
    if (!warp_wait(&bars->o_final[I], ni & 1)) return false;
    ++ni;
    tc::tc_fence_after_sync();
    const bool valid = mine && p < it.len;
    if (poison || m_run == -INFINITY) l_run = __int_as_float(0x7fffffff);  // (no score above -inf: 0 / 0)
    const float inv = valid ? 1.0f / l_run : 0.f;
    float largest = 0.f;  // magnitude among the sums, NaN if there is one
#pragma unroll
    for (int hb = 0; hb < DP / 32; ++hb) {
      uint32_t o[32];
      tc::tmem_ld32(col_o + hb * 32, o);
      tc::tmem_ld_wait();
      if (hb * 32 < a.D && mine) {
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          largest = max3(largest, fabsf(__uint_as_float(o[i])), fabsf(__uint_as_float(o[i + 1])));
          o[i] = valid ? __float_as_uint(__uint_as_float(o[i]) * inv) : 0u;
          o[i + 1] = valid ? __float_as_uint(__uint_as_float(o[i + 1]) * inv) : 0u;
        }
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
          uint4 y;
          y.x = pack_bf16(__uint_as_float(o[i]), __uint_as_float(o[i + 1]));
          y.y = pack_bf16(__uint_as_float(o[i + 2]), __uint_as_float(o[i + 3]));
          y.z = pack_bf16(__uint_as_float(o[i + 4]), __uint_as_float(o[i + 5]));
          y.w = pack_bf16(__uint_as_float(o[i + 6]), __uint_as_float(o[i + 7]));
          *reinterpret_cast<uint4*>(dst + hb * 32 + i) = y;
        }
      }
    }
    tc::tc_fence_before_sync();
    __syncwarp();
    if (lane == 0) tc::mbar_arrive(&bars->o_free[I]);
    if (valid && !poison && fabsf(m_run) > kFar && m_run > -INFINITY) {
      *reinterpret_cast<unsigned short*>(dst) = kAllAgain;
      marked = true;
    } else if (valid && l_run < INFINITY && !(largest < INFINITY)) {
      unsigned short* at = reinterpret_cast<unsigned short*>(dst);
      int c = 0;
      while (c + 1 < a.D && (at[c] & 0x7f80u) != 0x7f80u) ++c;  // (what is not finite is stored so)
      at[c] = kAgain;
      marked = true;
    }
  }
  if (__any_sync(0xffffffffu, marked)) revisit<LISTED>(a, pre, n_items, I, row, lane);
  return true;
}

// Zeros into the output rows of tiles that do not exist (one warp per CTA, beside the others' work).
__device__ __forceinline__ void clear_padding(const PromptArgs& a, const int* pre, int lane) {
  const int rows = a.pair_heads ? kRows : 2 * kRows, per_row = a.Hq * a.D / 8;
  for (int b = 0; b < a.B; ++b)
    for (int t = (pre[b + 1] - pre[b]) * rows + (int)blockIdx.x; t < a.T; t += gridDim.x) {
      uint4* dst = reinterpret_cast<uint4*>(a.out + ((size_t)b * a.T + t) * a.Hq * a.D);
      for (int i = lane; i < per_row; i += 32) dst[i] = make_uint4(0, 0, 0, 0);
    }
}

}  // namespace

template <int DP, bool LISTED>
__global__ void __launch_bounds__(kThreads, 1) kvm_window_prompt_kernel(const __grid_constant__ PromptArgs a) {
  extern __shared__ __align__(1024) unsigned char smem[];
  PromptBars* bars = reinterpret_cast<PromptBars*>(smem + PC<DP>::kOffBar);
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  if ((tc::smem_u32(smem) & 1023u) != 0) {  // operand tiles need 1024-byte alignment
    if (tid == 0) atomicExch(a.status, KVM_ERR_UNSUPPORTED);
    return;
  }
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&bars->q_full[i], 1);
      tc::mbar_init(&bars->q_empty[i], 1);
      tc::mbar_init(&bars->s_full[i], 1);
      tc::mbar_init(&bars->p_full[i][0], 4);
      tc::mbar_init(&bars->p_full[i][1], 4);
      tc::mbar_init(&bars->o_final[i], 1);
      tc::mbar_init(&bars->o_free[i], 4);
    }
    for (int i = 0; i < PC<DP>::kSlots; ++i) {
      tc::mbar_init(&bars->kv_full[i], 1);
      tc::mbar_init(&bars->kv_empty[i], 1);
    }
    tc::fence_barrier_init();
  }
  if (warp == kMmaWarp) tc::tmem_alloc(&bars->tmem_base, 512);
  pdl_wait();
  int* pre = reinterpret_cast<int*>(smem + PC<DP>::kOffPre);
  if (LISTED && warp == 0) {  // tiles of every sequence, prefix
    const int rows = a.pair_heads ? kRows : 2 * kRows;
    int carry = 0;
    for (int base = 0; base < a.B; base += 32) {
      int x = base + lane < a.B ? (max(min(max(a.lengths[base + lane], 0), a.S) - (a.S - a.T), 0) + rows - 1) / rows : 0;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
      }
      if (base + lane < a.B) pre[base + lane + 1] = x + carry;
      carry += __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane == 0) pre[0] = 0;
  }
  tc::tc_fence_before_sync();
  __syncthreads();
  tc::tc_fence_after_sync();
  const uint32_t tmem = __shfl_sync(0xffffffffu, bars->tmem_base, 0);
  const int n_items = LISTED ? __shfl_sync(0xffffffffu, pre[a.B], 0) * (a.units / a.B) : a.n_items;
  bool ok = true;
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    ok = softmax<DP, LISTED>(a, pre, n_items, smem, bars, tmem, warp >> 2, tid & 127, warp & 3, lane);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
    if (warp == kProducerWarp) {
      if (lane == 0) ok = produce<DP, LISTED>(a, pre, n_items, smem, bars);
      __syncwarp();
    } else if (warp == kMmaWarp) {
      // (the whole warp walks the tiles: operands that are uniform over it reach the issuing instructions without detours)
      ok = issue<DP, LISTED>(a, pre, n_items, smem, bars, tmem);
    } else if (LISTED && warp == kMmaWarp + 1) {
      clear_padding(a, pre, lane);
    }
  }
  if (!ok) {
    atomicExch(a.status, KVM_ERR_DEVICE_TIMEOUT);
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);  // copies and products in flight
  }
  tc::tc_fence_before_sync();
  __syncthreads();
  if (warp == kMmaWarp) tc::tmem_dealloc(tmem, 512);
}

namespace {

// [batch][head][row][D] with any strides as a 4-D tensor, boxes of 64 elements x 128 rows; dimensions ordered by stride
bool encode_rows(CUtensorMap* m, const Tensor4& t, int batch, int heads, int rows, int D, int* head_inner) {
  *head_inner = t.sh < t.st && heads > 1;
  auto bytes = [&](long long s, int n) { return (cuuint64_t)(n > 1 ? s * 2 : (long long)D * 2); };  // (one entry: never stepped over)
  const cuuint64_t sh = bytes(t.sh, heads), st = bytes(t.st, rows), sb = bytes(t.sb, batch);
  if (*head_inner) {
    const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)rows, (cuuint64_t)batch}, strides[3] = {sh, st, sb};
    const cuuint32_t box[4] = {64, 1, kRows, 1};
    return encode_bf16_map(m, t.ptr, 4, dims, strides, box);
  }
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)rows, (cuuint64_t)heads, (cuuint64_t)batch}, strides[3] = {st, sh, sb};
  const cuuint32_t box[4] = {64, kRows, 1, 1};
  return encode_bf16_map(m, t.ptr, 4, dims, strides, box);
}

template <int DP, bool LISTED>
cudaError_t launch_prompt(const PromptArgs& a, int sms, cudaStream_t stream) {
  auto kern = kvm_window_prompt_kernel<DP, LISTED>;
  static std::atomic<unsigned long long> raised{0};
  const cudaError_t e = raise_smem_limit(kern, PC<DP>::kSmem, raised);
  if (e != cudaSuccess) return e;
  // the register split draws on what the block is launched with
  static const bool regs_ok = [&] {
    cudaFuncAttributes at;
    return cudaFuncGetAttributes(&at, kern) == cudaSuccess && at.numRegs == kRegsLaunch;
  }();
  if (!regs_ok) return cudaErrorInvalidConfiguration;
  return launch_pdl(kern, dim3(std::min(a.n_items, sms)), dim3(kThreads), PC<DP>::kSmem, stream, true, a);
}

}  // namespace

cudaError_t window_prompt_dispatch(int D, int batch, int Hq, int Hkv, int T, int S, Tensor4 q, Tensor4 k, Tensor4 v, int window,
                                   int sinks, float scale, const int* lengths, bf16* out, int* status, cudaStream_t stream) {
  PromptArgs a;
  a.B = batch; a.Hq = Hq; a.Hkv = Hkv; a.D = D; a.T = T; a.S = S; a.window = window; a.sinks = sinks;
  a.scale_log2 = scale * kLog2e;
  a.lengths = lengths; a.out = out; a.status = status;
  a.q = q; a.k = k; a.v = v;
  a.pair_heads = (Hq / Hkv) % 2 == 0;
  const int rows = a.pair_heads ? kRows : 2 * kRows;
  a.q_tiles = (T + rows - 1) / rows;
  const long long units = (long long)batch * (a.pair_heads ? Hq / 2 : Hq);
  if (units * a.q_tiles > 0x3fffffff) return cudaErrorInvalidValue;
  a.units = (int)units;
  a.n_items = (int)units * a.q_tiles;
  if (!encode_rows(&a.mq, q, batch, Hq, T, D, &a.q_head_inner) || !encode_rows(&a.mk, k, batch, Hkv, S, D, &a.k_head_inner) ||
      !encode_rows(&a.mv, v, batch, Hkv, S, D, &a.v_head_inner))
    return cudaErrorInvalidValue;
  const int sms = window_sm_count();
  if (lengths && batch <= kMaxListed) return D == 128 ? launch_prompt<128, true>(a, sms, stream) : launch_prompt<64, true>(a, sms, stream);
  return D == 128 ? launch_prompt<128, false>(a, sms, stream) : launch_prompt<64, false>(a, sms, stream);
}

}  // namespace kvm
