// pages_attn.cu -- attention of a batch's rows over the paged 8-bit K/V pools.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "common.cuh"
#include "pages.cuh"

namespace shk {
namespace {

__device__ __forceinline__ float value_of(uint8_t b, uint32_t type) {
  return type == PAGES_I8 ? (float)(int8_t)b : __half2float(__half(__nv_cvt_fp8_to_halfraw(b, __NV_E4M3)));
}
__device__ __forceinline__ float load_dt(const void* p, size_t i, uint32_t dt) {
  if (dt == DT_F32) return static_cast<const float*>(p)[i];
  if (dt == DT_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store_dt(void* p, size_t i, uint32_t dt, float v) {
  if (dt == DT_F32)
    static_cast<float*>(p)[i] = v;
  else if (dt == DT_F16)
    static_cast<__half*>(p)[i] = __float2half_rn(v);
  else
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// One warp per (row, query head): online softmax over the row's positions,
// hd / 32 dims per lane.
template <int HD>
__global__ void __launch_bounds__(256) attend_kernel(const __grid_constant__ PagesAttnArgs a) {
  constexpr int E = HD / 32;
  const uint32_t row = blockIdx.x, lane = threadIdx.x & 31;
  const uint32_t bs = a.pool.block_shift, bt = 1u << bs;
  const int32_t z = a.row_seq ? a.row_seq[row] : (int32_t)row;
  if (z < 0) return;
  int64_t len = (int64_t)a.row_pos[row] + 1;
  if ((uint32_t)z >= a.n_seq || len > (int64_t)a.stride << bs) {
    if (threadIdx.x == 0) set_error(a.err, DERR_BAD_POS);
    len = 0;
  }
  for (uint32_t h = blockIdx.y * 8 + (threadIdx.x >> 5); h < a.n_heads; h += gridDim.y * 8) {
    const uint32_t kvh = h % a.pool.n_kv;
    float q[E], o[E] = {}, m = -INFINITY, l = 0.f;
    for (int e = 0; e < E; ++e) q[e] = load_dt(a.q, row * a.q_stride + (size_t)h * HD + lane * E + e, a.dtype) * a.scale;
    for (int64_t t = 0; t < len; ++t) {
      const int32_t b = a.table[(size_t)z * a.stride + (t >> bs)];
      if ((uint32_t)b >= a.pool.n_blocks) {
        if (lane == 0) set_error(a.err, DERR_BAD_POS);
        continue;
      }
      const size_t bh = (size_t)b * a.pool.n_kv + kvh, at = ((bh << bs) + (t & (bt - 1))) * HD + lane * E;
      float s = 0.f;
      for (int e = 0; e < E; ++e) s += q[e] * value_of(a.pool.k[at + e], a.pool.type);
      s = warp_sum(s) * a.pool.ks[bh];
      const float mn = fmaxf(m, s), c = m == mn ? 1.f : expf(m - mn), p = expf(s - mn);
      m = mn;
      l = l * c + p;
      for (int e = 0; e < E; ++e) o[e] = o[e] * c + p * a.pool.vs[bh] * value_of(a.pool.v[at + e], a.pool.type);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    for (int e = 0; e < E; ++e)
      store_dt(a.out, row * a.out_stride + (size_t)h * HD + lane * E + e, a.dtype, o[e] * inv);
  }
}

}  // namespace

size_t pages_attend_ws_bytes(uint32_t, uint32_t, uint32_t, uint32_t) { return 16; }
cudaError_t pages_attend_init() { return cudaSuccess; }
cudaError_t pages_attend_launch(const PagesAttnArgs& a, int, cudaStream_t st) {
  const dim3 grid(a.n_rows, (a.n_heads + 7) / 8);
  if (a.pool.hd == 64)
    attend_kernel<64><<<grid, 256, 0, st>>>(a);
  else
    attend_kernel<128><<<grid, 256, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace shk
