// pages.cu -- block tables, append and read of the paged 8-bit K/V pools.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"
#include "pages.cuh"

namespace shk {
namespace {

constexpr int TAB_THREADS = 1024;

__device__ __forceinline__ uint64_t warp_scan64(uint64_t v, uint32_t lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= (uint32_t)o) v += u;
  }
  return v;
}

// Inclusive sum over the block's threads plus `carry`, which becomes the
// total.  part: one slot per warp.
__device__ __forceinline__ uint64_t block_scan64(uint64_t v, uint64_t& carry, uint64_t* part) {
  const uint32_t lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  uint64_t s = warp_scan64(v, lane);
  if (lane == 31) part[w] = s;
  __syncthreads();
  const uint64_t p = warp_scan64(part[lane], lane);  // TAB_THREADS / 32 == 32 partials
  const uint64_t total = __shfl_sync(0xffffffffu, p, 31);
  const uint64_t before = __shfl_sync(0xffffffffu, p, (w + 31) & 31);
  s += carry + (w ? before : 0);
  carry += total;
  __syncthreads();
  return s;
}

// Largest i with start[i] <= r (start[0] == 0, not falling).
__device__ __forceinline__ uint32_t owner_of(const int32_t* start, uint32_t n, int32_t r) {
  uint32_t lo = 0, hi = n;
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) >> 1;
    if (start[mid] <= r)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// Rows and new blocks are two running sums over the requests, both in the
// requests' order, so that the same lengths always give the same tables.
__global__ void __launch_bounds__(TAB_THREADS) assign_kernel(const __grid_constant__ AssignArgs a) {
  extern __shared__ int32_t tab_sm[];
  __shared__ uint64_t part[32];
  int32_t* start = tab_sm;             // first row of each request
  int32_t* held = tab_sm + a.n_seq;    // tokens it holds
  int32_t* base = held + a.n_seq;      // free-stack index of its first new block; -1: refused
  const uint32_t bs = a.block_shift, bt = 1u << bs;
  const int64_t cap = (int64_t)a.stride << bs;
  int32_t n_free = *a.n_free;
  if (n_free < 0 || n_free > (int32_t)a.n_blocks) {
    if (threadIdx.x == 0) set_error(a.err, DERR_BAD_POS);
    n_free = n_free < 0 ? 0 : (int32_t)a.n_blocks;
  }
  uint64_t rows = 0, blocks = 0, took = 0, live = 0, refused = 0;
  for (uint32_t r0 = 0; r0 < a.n_seq; r0 += TAB_THREADS) {
    const uint32_t r = r0 + threadIdx.x;
    const bool in = r < a.n_seq;
    const int32_t h = in ? a.have[r] : 0, n = in ? a.add[r] : 0;
    const bool valid = h >= 0 && n >= 0 && (int64_t)h + n <= cap;
    const uint64_t row_end = block_scan64(n > 0 ? n : 0, rows, part);
    const uint64_t row0 = row_end - (n > 0 ? n : 0);
    bool ok = valid && (n == 0 || row_end <= a.n_rows);
    const uint64_t need = ok ? (((uint64_t)h + n + bt - 1) >> bs) - (((uint64_t)h + bt - 1) >> bs) : 0;
    const uint64_t end = block_scan64(need, blocks, part);
    ok = ok && (need == 0 || end <= (uint64_t)n_free);
    if (in) {
      start[r] = (int32_t)(row0 < a.n_rows ? row0 : a.n_rows);
      held[r] = h;
      // a request without new blocks never reads its base: any value but -1
      base[r] = !ok ? -1 : need ? (int32_t)(n_free - 1 - (int64_t)(end - need)) : 0;
      a.lens[r] = ok ? h + n : h;
      a.last[r] = ok && n > 0 ? (int32_t)(row_end - 1) : -1;
    }
    took += ok && in ? need : 0;
    live += ok && in ? n : 0;
    refused += in && !ok;
  }
  // per-thread tallies -> totals
  uint64_t t0 = 0, t1 = 0, t2 = 0;
  block_scan64(took, t0, part);
  block_scan64(live, t1, part);
  block_scan64(refused, t2, part);
  if (threadIdx.x == 0) {
    a.counts[0] = n_free - (int32_t)t0;
    a.counts[1] = (int32_t)t1;
    a.counts[2] = (int32_t)t2;
  }
  for (uint32_t r = threadIdx.x; r < a.n_rows; r += TAB_THREADS) {
    int32_t slot = -1, pos = -1, seq = -1;
    const uint32_t q = owner_of(start, a.n_seq, (int32_t)r);
    if (r < rows && base[q] >= 0) {
      pos = held[q] + (int32_t)r - start[q];
      seq = (int32_t)q;
      const uint32_t b = (uint32_t)pos >> bs, have_blocks = ((uint32_t)held[q] + bt - 1) >> bs;
      const bool fresh = b >= have_blocks;
      const int32_t id = fresh ? a.free_ids[base[q] - (int32_t)(b - have_blocks)] : a.table[(size_t)q * a.stride + b];
      if ((uint32_t)id < a.n_blocks) {
        slot = (int32_t)(((uint32_t)id << bs) + ((uint32_t)pos & (bt - 1)));
        // a new block's first token is always one of the rows
        if (fresh && ((uint32_t)pos & (bt - 1)) == 0) a.table[(size_t)q * a.stride + b] = id;
      } else {
        set_error(a.err, DERR_BAD_POS);
      }
    }
    a.slots[r] = slot;
    a.pos[r] = pos;
    a.seq[r] = seq;
  }
}

__global__ void __launch_bounds__(TAB_THREADS) release_kernel(const __grid_constant__ ReleaseArgs a) {
  extern __shared__ int32_t tab_sm[];
  __shared__ uint64_t part[32];
  int32_t* start = tab_sm;  // first freed block of each request
  const uint32_t bs = a.block_shift, bt = 1u << bs;
  const int32_t n_free = *a.n_free;
  uint64_t total = 0;
  bool bad = false;
  for (uint32_t r0 = 0; r0 < a.n_seq; r0 += TAB_THREADS) {
    const uint32_t r = r0 + threadIdx.x;
    uint64_t n = 0;
    if (r < a.n_seq && a.done[r] != 0) {
      const int32_t h = a.have[r];
      n = h > 0 ? ((uint64_t)h + bt - 1) >> bs : 0;
      if (h < 0 || n > a.stride) bad = true, n = 0;
    }
    const uint64_t end = block_scan64(n, total, part);
    if (r < a.n_seq) start[r] = (int32_t)min(end - n, (uint64_t)a.n_blocks);
  }
  // a stack that would outgrow the pool means blocks given back twice
  bad = __syncthreads_or(bad || n_free < 0 || (int64_t)n_free + (int64_t)total > (int64_t)a.n_blocks);
  if (bad && threadIdx.x == 0) set_error(a.err, DERR_BAD_POS);
  for (uint32_t i = threadIdx.x; !bad && i < total; i += TAB_THREADS) {
    const uint32_t q = owner_of(start, a.n_seq, (int32_t)i);
    const int32_t id = a.table[(size_t)q * a.stride + (i - start[q])];
    if ((uint32_t)id >= a.n_blocks) set_error(a.err, DERR_BAD_POS);
    a.free_ids[n_free + i] = id;
  }
  for (uint32_t r = threadIdx.x; r < a.n_seq; r += TAB_THREADS) a.lens[r] = !bad && a.done[r] != 0 ? 0 : a.have[r];
  __syncthreads();  // every thread has read *n_free, which n_free_out may be
  if (threadIdx.x == 0) *a.n_free_out = bad ? n_free : n_free + (int32_t)total;
}

// ---- append ----

template <uint32_t DT>
__device__ __forceinline__ float load_as_f32(const void* p, size_t i) {
  if constexpr (DT == DT_F32) return static_cast<const float*>(p)[i];
  if constexpr (DT == DT_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

__device__ __forceinline__ float e4m3_value(uint32_t b) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)b, __NV_E4M3)));
}

// x / s rounded to the pool's type, halves to even; NaN gives 0, as the Q8_0
// quantiser's integer conversion does.
template <uint32_t TYPE>
__device__ __forceinline__ uint8_t to_byte(float y) {
  if (y != y) return 0;
  if constexpr (TYPE == PAGES_I8) return (uint8_t)(int8_t)__float2int_rn(fminf(fmaxf(y, -127.f), 127.f));
  return (uint8_t)__nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3);
}
template <uint32_t TYPE>
__device__ __forceinline__ float from_byte(uint8_t b) {
  if constexpr (TYPE == PAGES_I8) return (float)(int8_t)b;
  return e4m3_value(b);
}

constexpr int APP_WARPS = 16;

// The call's tokens fall into runs of consecutive slots of one block.  The
// CTA of a run's first token writes the run: one warp per (K or V, head)
// finds the largest magnitude, raises the block's scale if need be (the
// block's earlier rows are then rounded to the new scale) and rounds the
// run's rows.  A block whose rows come in two runs of one call would be
// written by two CTAs at once: the later run is refused.
template <uint32_t TYPE, uint32_t DT>
__global__ void __launch_bounds__(32 * APP_WARPS) append_kernel(PagesPool p, uint32_t n, const void* k, const void* v,
                                                                size_t row_stride, const int32_t* slots, int* err) {
  const uint32_t t = blockIdx.x, bs = p.block_shift, bt = 1u << bs;
  const int32_t slot = slots[t];
  if (slot < 0) return;
  const uint32_t b = (uint32_t)slot >> bs, first = (uint32_t)slot & (bt - 1);
  if (b >= p.n_blocks) {
    if (threadIdx.x == 0) set_error(err, DERR_BAD_POS);
    return;
  }
  if (t > 0 && first > 0 && slots[t - 1] == slot - 1) return;  // inside a run
  bool twice = false;
  for (uint32_t i = threadIdx.x; i < t; i += blockDim.x) twice |= slots[i] >= 0 && ((uint32_t)slots[i] >> bs) == b;
  if (__syncthreads_or(twice)) {
    if (threadIdx.x == 0) set_error(err, DERR_BAD_POS);
    return;
  }
  uint32_t len = 1;
  while (first + len < bt && t + len < n && slots[t + len] == slot + (int32_t)len) ++len;

  const uint32_t lane = threadIdx.x & 31;
  constexpr float TOP = TYPE == PAGES_I8 ? 127.f : 448.f;
  for (uint32_t w = threadIdx.x >> 5; w < 2 * p.n_kv; w += blockDim.x >> 5) {
    const uint32_t h = w >> 1;
    const void* x = (w & 1) ? v : k;
    uint8_t* dst = ((w & 1) ? p.v : p.k) + (((size_t)b * p.n_kv + h) << bs) * p.hd;
    float* sp = ((w & 1) ? p.vs : p.ks) + (size_t)b * p.n_kv + h;
    const size_t src = t * row_stride + (size_t)h * p.hd;
    float m = 0.f;
    for (uint32_t i = 0; i < len; ++i)
      for (uint32_t d = lane; d < p.hd; d += 32) m = fmaxf(m, fabsf(load_as_f32<DT>(x, src + i * row_stride + d)));
    m = warp_max(m);
    const float old = first ? *sp : 0.f;
    const float s = fmaxf(old, __fdiv_rn(m, TOP));
    if (first && s > old) {
      const float ratio = __fdiv_rn(old, s);
      for (uint32_t i = lane; i < first * p.hd; i += 32)
        dst[i] = to_byte<TYPE>(from_byte<TYPE>(dst[i]) * ratio);
    }
    for (uint32_t i = 0; i < len; ++i)
      for (uint32_t d = lane; d < p.hd; d += 32) {
        const float y = load_as_f32<DT>(x, src + i * row_stride + d);
        dst[(size_t)(first + i) * p.hd + d] = s > 0.f ? to_byte<TYPE>(__fdiv_rn(y, s)) : 0;
      }
    __syncwarp();
    if (lane == 0) *sp = s;
  }
}

template <uint32_t TYPE>
__global__ void read_kernel(PagesPool p, const int32_t* slots, float* k, float* v, int* err) {
  const int32_t slot = slots[blockIdx.x];
  if (slot < 0) return;
  const uint32_t b = (uint32_t)slot >> p.block_shift, t = (uint32_t)slot & ((1u << p.block_shift) - 1);
  if (b >= p.n_blocks) {
    if (threadIdx.x == 0) set_error(err, DERR_BAD_POS);
    return;
  }
  const uint32_t width = p.n_kv * p.hd;
  for (uint32_t i = threadIdx.x; i < width; i += blockDim.x) {
    const uint32_t h = i / p.hd, d = i % p.hd;
    const size_t bh = (size_t)b * p.n_kv + h, at = ((bh << p.block_shift) + t) * p.hd + d;
    k[(size_t)blockIdx.x * width + i] = from_byte<TYPE>(p.k[at]) * p.ks[bh];
    v[(size_t)blockIdx.x * width + i] = from_byte<TYPE>(p.v[at]) * p.vs[bh];
  }
}

template <uint32_t TYPE>
cudaError_t append_go(const PagesPool& p, uint32_t n, const void* k, const void* v, uint32_t dtype, size_t row_stride,
                      const int32_t* slots, int* err, cudaStream_t st) {
  switch (dtype) {
    case DT_F32: append_kernel<TYPE, DT_F32><<<n, 32 * APP_WARPS, 0, st>>>(p, n, k, v, row_stride, slots, err); break;
    case DT_F16: append_kernel<TYPE, DT_F16><<<n, 32 * APP_WARPS, 0, st>>>(p, n, k, v, row_stride, slots, err); break;
    default: append_kernel<TYPE, DT_BF16><<<n, 32 * APP_WARPS, 0, st>>>(p, n, k, v, row_stride, slots, err); break;
  }
  return cudaGetLastError();
}

}  // namespace

cudaError_t pages_init() {
  cudaError_t e = cudaFuncSetAttribute(assign_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 3 * 4 * 16384);
  if (e != cudaSuccess) return e;
  e = cudaFuncSetAttribute(release_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 4 * 16384);
  return e != cudaSuccess ? e : pages_attend_init();
}

cudaError_t pages_assign_launch(const AssignArgs& a, cudaStream_t st) {
  assign_kernel<<<1, TAB_THREADS, 3 * 4 * a.n_seq, st>>>(a);
  return cudaGetLastError();
}

cudaError_t pages_release_launch(const ReleaseArgs& a, cudaStream_t st) {
  release_kernel<<<1, TAB_THREADS, 4 * a.n_seq, st>>>(a);
  return cudaGetLastError();
}

cudaError_t pages_append_launch(const PagesPool& p, uint32_t n, const void* k, const void* v, uint32_t dtype,
                                size_t row_stride, const int32_t* slots, int* err, cudaStream_t st) {
  return p.type == PAGES_I8 ? append_go<PAGES_I8>(p, n, k, v, dtype, row_stride, slots, err, st)
                            : append_go<PAGES_E4M3>(p, n, k, v, dtype, row_stride, slots, err, st);
}

cudaError_t pages_read_launch(const PagesPool& p, uint32_t n, const int32_t* slots, float* k, float* v, int* err,
                              cudaStream_t st) {
  if (p.type == PAGES_I8)
    read_kernel<PAGES_I8><<<n, 256, 0, st>>>(p, slots, k, v, err);
  else
    read_kernel<PAGES_E4M3><<<n, 256, 0, st>>>(p, slots, k, v, err);
  return cudaGetLastError();
}

}  // namespace shk
