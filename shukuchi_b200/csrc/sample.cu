// sample.cu -- temperature, top-k, top-p and min-p sampling.
//
// A row's logits z become x = (z - z_max) * (1 / T) and weights w = exp(x),
// both in fp32, and the weights become whole numbers W = floor(w * 2^40):
// every sum below is a sum of integers, so that the token that a random
// number picks does not depend on the order in which threads add.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "common.cuh"
#include "pages.cuh"
#include "sample.cuh"

namespace shk {
namespace {

constexpr int THREADS = 1024;
constexpr int WARPS = THREADS / 32;

template <uint32_t DT>
__device__ __forceinline__ float logit(const void* p, size_t i) {
  float z;
  if constexpr (DT == DT_F32)
    z = static_cast<const float*>(p)[i];
  else if constexpr (DT == DT_F16)
    z = __half2float(static_cast<const __half*>(p)[i]);
  else
    z = __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return z + 0.f;  // -0 becomes +0: the two compare equal, and so do their keys
}

// Larger logits have larger keys; NaN comes last.
__device__ __forceinline__ uint32_t key_of(float z) {
  if (z != z) return 0;
  const uint32_t u = __float_as_uint(z);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float weight_of(float z, float zmax, float inv_t) {
  const float x = (z - zmax) * inv_t;
  if (z == zmax) return 1.f;
  return x <= 0.f ? expf(x) : 0.f;  // NaN (masked or not a number): 0
}
__device__ __forceinline__ uint64_t mass_of(float w) { return (uint64_t)(w * 1099511627776.f); }

__device__ __forceinline__ uint64_t warp_sum64(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct Shared {
  uint64_t mass[256];
  uint32_t count[256];
  uint64_t part[WARPS];
  uint32_t ties[WARPS];
  float red[WARPS];
  uint32_t idx[WARPS];
  uint32_t key;        // radix select: the border key
  uint64_t above;      // mass (or count) of larger keys
};

__device__ __forceinline__ uint64_t block_sum64(uint64_t v, Shared& s) {
  v = warp_sum64(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s.part[threadIdx.x >> 5] = v;
  __syncthreads();
  uint64_t t = 0;
  for (int w = 0; w < WARPS; ++w) t += s.part[w];
  return t;
}

// The largest key at which the running total from the largest key down
// reaches `need`: by count (BY_MASS false) or by mass, over keys >= floor_key.
// Returns the key; `above` is the total of the keys over it.
template <uint32_t DT, bool BY_MASS>
__device__ uint32_t border(const void* z, uint32_t n, float zmax, float inv_t, uint32_t floor_key, uint64_t need,
                           uint64_t& above, Shared& s) {
  uint32_t prefix = 0;
  uint64_t over = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += THREADS) s.mass[i] = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += THREADS) {
      const float v = logit<DT>(z, i);
      const uint32_t key = key_of(v);
      if (key < floor_key || (shift < 24 && (key >> (shift + 8)) != (prefix >> (shift + 8)))) continue;
      const uint64_t add = BY_MASS ? mass_of(weight_of(v, zmax, inv_t)) : 1;
      if (add) atomicAdd(reinterpret_cast<unsigned long long*>(&s.mass[(key >> shift) & 255]), (unsigned long long)add);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      uint64_t c = over;
      int b = 255;
      while (b > 0 && c + s.mass[b] < need) c += s.mass[b--];
      s.key = prefix | ((uint32_t)b << shift);
      s.above = c;
    }
    __syncthreads();
    prefix = s.key;
    over = s.above;
    __syncthreads();
  }
  above = over;
  return prefix;
}

template <uint32_t DT>
__global__ void __launch_bounds__(THREADS) sample_kernel(const __grid_constant__ SampleArgs a) {
  __shared__ Shared s;
  const uint32_t row = blockIdx.x, n = a.n_vocab, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const void* z = static_cast<const uint8_t*>(a.logits) + row * a.row_stride * (DT == DT_F32 ? 4 : 2);

  float m = -INFINITY;
  uint32_t mi = 0xFFFFFFFFu;
  for (uint32_t i = threadIdx.x; i < n; i += THREADS) {
    const float v = logit<DT>(z, i);
    if (v > m) m = v, mi = i;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float v = __shfl_xor_sync(0xffffffffu, m, o);
    const uint32_t i = __shfl_xor_sync(0xffffffffu, mi, o);
    if (v > m || (v == m && i < mi)) m = v, mi = i;
  }
  if (lane == 0) s.red[warp] = m, s.idx[warp] = mi;
  __syncthreads();
  m = s.red[0], mi = s.idx[0];
  for (int w = 1; w < WARPS; ++w)
    if (s.red[w] > m || (s.red[w] == m && s.idx[w] < mi)) m = s.red[w], mi = s.idx[w];

  const float t = a.temperature ? a.temperature[row] : 1.f;
  if (mi == 0xFFFFFFFFu || !(t > 0.f)) {
    if (threadIdx.x == 0) {
      a.out[row] = mi;
      if (a.prob) a.prob[row] = mi == 0xFFFFFFFFu ? 0.f : 1.f;
    }
    return;
  }
  const float inv_t = __frcp_rn(t);

  // the kept tokens are those over `floor_key` and the first `ties` at it
  uint32_t floor_key = 0, ties = 0xFFFFFFFFu;
  const int32_t k = a.top_k ? a.top_k[row] : 0;
  if (k > 0 && (uint32_t)k < n) {
    uint64_t above;
    floor_key = border<DT, false>(z, n, m, inv_t, 0, (uint64_t)k, above, s);
    ties = (uint32_t)(k - above);
  }
  const float top_p = a.top_p ? a.top_p[row] : 1.f;
  if (top_p < 1.f) {
    uint64_t sum = 0;
    for (uint32_t i = threadIdx.x; i < n; i += THREADS) {
      const float v = logit<DT>(z, i);
      if (key_of(v) > floor_key) sum += mass_of(weight_of(v, m, inv_t));
    }
    sum = block_sum64(sum, s);
    uint64_t at = 0;  // one token at the border
    if (ties != 0xFFFFFFFFu) {
      const uint32_t u = (floor_key & 0x80000000u) ? floor_key & 0x7FFFFFFFu : ~floor_key;
      at = floor_key ? mass_of(weight_of(__uint_as_float(u), m, inv_t)) : 0;
      sum += at * ties;
    }
    const double need_d = ceil((double)top_p * (double)sum);
    const uint64_t need = need_d >= 1.0 ? (uint64_t)need_d : 1;
    uint64_t above;
    const uint32_t key = border<DT, true>(z, n, m, inv_t, floor_key, need, above, s);
    const uint32_t u = (key & 0x80000000u) ? key & 0x7FFFFFFFu : ~key;
    const uint64_t one = mass_of(weight_of(__uint_as_float(u), m, inv_t));
    floor_key = key;
    ties = one ? (uint32_t)min((need - above + one - 1) / one, (uint64_t)n) : n;
  }
  float min_p = a.min_p ? a.min_p[row] : 0.f;
  min_p = min_p > 0.f ? fminf(min_p, 1.f) : 0.f;  // the largest weight, 1, always stays

  // each warp takes a run of the vocabulary: ties at the border, then kept mass
  const uint32_t per = ((n + WARPS - 1) / WARPS + 31) & ~31u;
  const uint32_t lo = min(n, warp * per), hi = min(n, lo + per);
  uint32_t mine = 0;
  for (uint32_t i = lo + lane; i < hi; i += 32) mine += key_of(logit<DT>(z, i)) == floor_key;
  mine = __reduce_add_sync(0xffffffffu, mine);
  if (lane == 0) s.ties[warp] = mine;
  __syncthreads();
  uint32_t seen0 = 0;
  for (uint32_t w = 0; w < warp; ++w) seen0 += s.ties[w];
  auto kept = [&](uint32_t i, bool in, uint32_t& seen) -> uint64_t {
    const float v = in ? logit<DT>(z, i) : -INFINITY;
    const uint32_t key = in ? key_of(v) : 0;
    const uint32_t eq = __ballot_sync(0xffffffffu, in && key == floor_key);
    const uint32_t rank = seen + __popc(eq & ((1u << lane) - 1));
    seen += __popc(eq);
    if (!in || key < floor_key || (key == floor_key && rank >= ties)) return 0;
    const float w = weight_of(v, m, inv_t);
    return w < min_p ? 0 : mass_of(w);
  };
  uint64_t sum = 0;
  uint32_t seen = seen0;
  for (uint32_t i0 = lo; i0 < hi; i0 += 32) sum += kept(i0 + lane, i0 + lane < hi, seen);
  sum = warp_sum64(sum);
  __syncthreads();
  if (lane == 0) s.part[warp] = sum;
  __syncthreads();
  uint64_t total = 0, before = 0;
  for (uint32_t w = 0; w < (uint32_t)WARPS; ++w) {
    if (w == warp) before = total;
    total += s.part[w];
  }
  const float uf = a.u[row];
  uint64_t target = uf > 0.f ? (uint64_t)fmin((double)uf * (double)total, 1.8e19) : 0;
  if (target >= total) target = total - 1;
  if (target < before || target >= before + sum) return;
  seen = seen0;
  for (uint32_t i0 = lo; i0 < hi; i0 += 32) {
    const uint64_t w = kept(i0 + lane, i0 + lane < hi, seen);
    uint64_t c = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t u = __shfl_up_sync(0xffffffffu, c, o);
      if (lane >= (uint32_t)o) c += u;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, before + c > target);
    if (hit) {
      if (lane == (uint32_t)__ffs(hit) - 1) {
        a.out[row] = i0 + lane;
        if (a.prob) a.prob[row] = (float)((double)w / (double)total);
      }
      return;
    }
    before += __shfl_sync(0xffffffffu, c, 31);
  }
}

}  // namespace

cudaError_t sample_launch(const SampleArgs& a, int, cudaStream_t st) {
  if (a.dtype == DT_F32)
    sample_kernel<DT_F32><<<a.n_rows, THREADS, 0, st>>>(a);
  else if (a.dtype == DT_F16)
    sample_kernel<DT_F16><<<a.n_rows, THREADS, 0, st>>>(a);
  else
    sample_kernel<DT_BF16><<<a.n_rows, THREADS, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace shk
