// Attention of a prompt, or of a chunk of one behind earlier tokens, with a sliding window and sinks: query t stands at
// position S - T + t and sees position j if j <= p and (j > p - window or j < sinks).
#include "kvm_window.cuh"

namespace kvm {

namespace {

// One warp per (sequence, query head, query): lanes take one key each, then D/32 channels each.
template <int D>
__global__ void __launch_bounds__(256)
kvm_window_prompt_kernel(int Hq, int Hkv, int T, int S, Tensor4 q, Tensor4 k, Tensor4 v, int window, int sinks, float scale_log2,
                         const int* __restrict__ lengths, bf16* __restrict__ out) {
  constexpr int CPL = D / 32;
  __shared__ float qs[8][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t = blockIdx.x * 8 + warp, hq = blockIdx.y % Hq, b = blockIdx.y / Hq, h = hq / (Hq / Hkv);
  if (t >= T) return;
  const int p = S - T + t;
  bf16* dst = out + ((size_t)b * T + t) * Hq * D + (size_t)hq * D + lane * CPL;
  float o[CPL], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < CPL; ++i) o[i] = 0.f;
  if (!lengths || p < lengths[b]) {
    for (int i = lane; i < D; i += 32) qs[warp][i] = __bfloat162float(q.row(b, hq, t)[i]) * scale_log2;
    __syncwarp();
    const int lo = max(0, p - window + 1), ns = min(sinks, lo);
    for (int base = 0; base < ns + p + 1 - lo; base += 32) {
      const int i = base + lane, j = i < ns ? i : lo + i - ns;
      float s = -INFINITY;
      if (j <= p) {
        s = 0.f;
        const bf16* kr = k.row(b, h, j);
        for (int d = 0; d < D; ++d) s = fmaf(qs[warp][d], __bfloat162float(kr[d]), s);
      }
      const float mn = fmaxf(m, warp_max(s)), mm = mn == -INFINITY ? 0.f : mn, a = exp2f(m - mm), e = exp2f(s - mm);
      l = l * a + warp_sum(e);
      m = mn;
#pragma unroll
      for (int c = 0; c < CPL; ++c) o[c] *= a;
      for (int x = 0; x < 32; ++x) {
        const float w = __shfl_sync(0xffffffffu, e, x);
        const int jx = __shfl_sync(0xffffffffu, j, x);
        if (jx > p) break;
        const bf16* vr = v.row(b, h, jx) + lane * CPL;
#pragma unroll
        for (int c = 0; c < CPL; ++c) o[c] = fmaf(w, __bfloat162float(vr[c]), o[c]);
      }
    }
#pragma unroll
    for (int c = 0; c < CPL; ++c) o[c] /= l;
  }
#pragma unroll
  for (int c = 0; c < CPL; ++c) dst[c] = __float2bfloat16_rn(o[c]);
}

}  // namespace

cudaError_t window_prompt_dispatch(int D, int batch, int Hq, int Hkv, int T, int S, Tensor4 q, Tensor4 k, Tensor4 v, int window,
                                   int sinks, float scale, const int* lengths, bf16* out, int* status, cudaStream_t stream) {
  (void)status;
  const dim3 grid((T + 7) / 8, batch * Hq);
  auto go = [&](auto kern) {
    kern<<<grid, 256, 0, stream>>>(Hq, Hkv, T, S, q, k, v, window, sinks, scale * kLog2e, lengths, out);
    return cudaGetLastError();
  };
  return D == 128 ? go(kvm_window_prompt_kernel<128>) : D == 64 ? go(kvm_window_prompt_kernel<64>) : go(kvm_window_prompt_kernel<32>);
}

}  // namespace kvm
