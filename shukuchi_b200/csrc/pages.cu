// pages.cu -- block tables, append and read of the paged 8-bit K/V pools.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "common.cuh"
#include "pages.cuh"

namespace shk {
namespace {

// The tables are running sums over the requests: a few microseconds of loads
// that wait on one another, not bytes.  A cluster of CTAs takes them: each sums
// the lengths for itself (no exchange), and the rows, each of which looks up its
// request and its block, are dealt to all.  The cluster's barrier separates the
// last read of the inputs from the writes to arrays that may be the same.
// Release and assign of 1024 requests with 50k rows 15.9 us together, of 64
// requests 9.0 (five of them the two calls' own).
constexpr int TAB_THREADS = 1024;
constexpr int TAB_CLUSTER = 8;
// Rows that one CTA takes alone (1024 requests, 50k rows: 57 us on one CTA, 12 on
// 8; 64 rows: the same).
constexpr uint32_t TAB_ROWS = 2048;

__device__ __forceinline__ uint64_t warp_scan64(uint64_t v, uint32_t lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= (uint32_t)o) v += u;
  }
  return v;
}

// Inclusive sum over the block's threads plus `carry`, which grows by the
// total.  part: one slot per warp, 32 of them.
__device__ __forceinline__ uint64_t block_scan64(uint64_t v, uint64_t& carry, uint64_t* part) {
  const uint32_t lane = threadIdx.x & 31, w = threadIdx.x >> 5, warps = blockDim.x >> 5;
  uint64_t s = warp_scan64(v, lane);
  if (lane == 31) part[w] = s;
  __syncthreads();
  const uint64_t p = warp_scan64(lane < warps ? part[lane] : 0, lane);
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

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_ctas() {
  uint32_t r;
  asm volatile("mov.u32 %0, %cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// All CTAs of the cluster have read what this kernel may overwrite.
__device__ __forceinline__ void cluster_barrier() {
  cluster_arrive();
  cluster_wait();
}

// One word of CTA `rank`'s shared memory.
__device__ __forceinline__ void cluster_put(const uint32_t* word, uint32_t rank, uint32_t v) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(word)), "r"(rank));
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
}

// Rows and new blocks are two running sums over the requests, both in the
// requests' order, so that the same lengths always give the same tables.
__global__ void __launch_bounds__(TAB_THREADS) assign_kernel(const __grid_constant__ AssignArgs a) {
  extern __shared__ int32_t tab_sm[];
  __shared__ uint64_t part[32];
  __shared__ uint32_t tally[3];        // blocks taken, rows, requests refused
  int32_t* start = tab_sm;             // first row of each request
  int32_t* held = tab_sm + a.n_seq;    // tokens it holds
  int32_t* base = held + a.n_seq;      // free-stack index of its first new block; -1: refused
  const uint32_t bs = a.block_shift, bt = 1u << bs;
  const uint32_t rank = cluster_rank(), ctas = cluster_ctas();
  const int64_t cap = (int64_t)a.stride << bs;
  pdl_trigger();
  pdl_wait();
  int32_t n_free = *a.n_free;
  if (threadIdx.x < 3) tally[threadIdx.x] = 0;
  if (n_free < 0 || n_free > (int32_t)a.n_blocks) {
    if (threadIdx.x == 0) set_error(a.err, DERR_BAD_POS);
    n_free = n_free < 0 ? 0 : (int32_t)a.n_blocks;
  }
  uint64_t rows = 0, blocks = 0;
  for (uint32_t r0 = 0; r0 < a.n_seq; r0 += blockDim.x) {
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
      if (rank == 0) {
        a.last[r] = ok && n > 0 ? (int32_t)(row_end - 1) : -1;
        if (ok && need) atomicAdd(&tally[0], (uint32_t)need);
        if (ok && n) atomicAdd(&tally[1], (uint32_t)n);
        if (!ok) atomicAdd(&tally[2], 1u);
      }
    }
  }
  __syncthreads();
  if (ctas > 1) cluster_barrier();
  if (rank == 0) {
    if (threadIdx.x == 0) {
      a.counts[0] = n_free - (int32_t)tally[0];
      a.counts[1] = (int32_t)tally[1];
      a.counts[2] = (int32_t)tally[2];
    }
    for (uint32_t r = threadIdx.x; r < a.n_seq; r += blockDim.x) {
      const int32_t next = r + 1 < a.n_seq ? start[r + 1] : (int32_t)min(rows, (uint64_t)a.n_rows);
      a.lens[r] = base[r] < 0 ? held[r] : held[r] + (next - start[r]);
    }
  }
  // Where a row's block id stands; null: the row is nobody's.
  auto look_up = [&](uint32_t r, uint32_t q, int32_t& pos, bool& fresh) -> const int32_t* {
    pos = -1;
    if (r >= a.n_rows || r >= rows || base[q] < 0) return nullptr;
    pos = held[q] + (int32_t)r - start[q];
    const uint32_t b = (uint32_t)pos >> bs, have_blocks = ((uint32_t)held[q] + bt - 1) >> bs;
    fresh = b >= have_blocks;
    return fresh ? a.free_ids + (base[q] - (int32_t)(b - have_blocks)) : a.table + (size_t)q * a.stride + b;
  };
  // The row's slot.  A row whose block id lies outside the pool is nobody's either;
  // such a new block leaves -1 in the table, so that no later call takes what
  // stood there before for the request's.
  auto slot_of = [&](int32_t id, uint32_t r, int32_t& pos, int32_t& seq, bool fresh) -> int32_t {
    const uint32_t at = (uint32_t)pos & (bt - 1);
    const bool good = (uint32_t)id < a.n_blocks;
    // a new block's first token is always one of the rows
    if (fresh && at == 0) a.table[(size_t)seq * a.stride + ((uint32_t)pos >> bs)] = good ? id : -1;
    if (good) return (int32_t)(((uint32_t)id << bs) + at);
    set_error(a.err, DERR_BAD_POS);
    if (a.last[seq] == (int32_t)r) a.last[seq] = -1;  // (written before the barrier above)
    return pos = seq = -1;
  };
  const uint32_t me = rank * blockDim.x + threadIdx.x, all = ctas * blockDim.x;
  if (a.n_rows <= all) {
    if (me >= a.n_rows) return;
    const uint32_t q = owner_of(start, a.n_seq, (int32_t)me);
    int32_t pos;
    bool fresh = false;
    const int32_t* at = look_up(me, q, pos, fresh);
    int32_t seq = at ? (int32_t)q : -1;
    a.slots[me] = at ? slot_of(*at, me, pos, seq, fresh) : -1;
    a.pos[me] = pos;
    a.seq[me] = seq;
    return;
  }
  // many rows: four a thread, with one search and 16-byte stores where the arrays allow
  const bool wide = ((reinterpret_cast<uintptr_t>(a.slots) | reinterpret_cast<uintptr_t>(a.pos) |
                      reinterpret_cast<uintptr_t>(a.seq)) & 15) == 0;
  for (uint32_t r0 = 4 * me; r0 < a.n_rows; r0 += 4 * all) {
    int32_t slot[4], pos[4], seq[4], id[4];
    const int32_t* at[4];
    bool fresh[4];
    uint32_t q = owner_of(start, a.n_seq, (int32_t)r0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      while (q + 1 < a.n_seq && (uint32_t)start[q + 1] <= r0 + i) ++q;
      fresh[i] = false;
      at[i] = look_up(r0 + i, q, pos[i], fresh[i]);
      seq[i] = at[i] ? (int32_t)q : -1;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) id[i] = at[i] ? *at[i] : 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) slot[i] = at[i] ? slot_of(id[i], r0 + i, pos[i], seq[i], fresh[i]) : -1;
    if (wide && r0 + 3 < a.n_rows) {
      *reinterpret_cast<int4*>(a.slots + r0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
      *reinterpret_cast<int4*>(a.pos + r0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
      *reinterpret_cast<int4*>(a.seq + r0) = make_int4(seq[0], seq[1], seq[2], seq[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (r0 + i < a.n_rows) a.slots[r0 + i] = slot[i], a.pos[r0 + i] = pos[i], a.seq[r0 + i] = seq[i];
    }
  }
}

// A request that ended gives all its blocks back, one that is cut short those
// behind the last token it keeps.
// Ids outside the pool are looked for where they are copied, and closed up behind
// that by one CTA, which has to wait for the others' word (0.8 us with 8 CTAs).
__global__ void __launch_bounds__(TAB_THREADS) release_kernel(const __grid_constant__ ReleaseArgs a) {
  extern __shared__ int32_t tab_sm[];
  __shared__ uint64_t part[32];
  __shared__ uint32_t odd_ids;  // CTA 0's: some CTA met an id outside the pool
  int32_t* start = tab_sm;             // first freed block of each request
  int32_t* skip = tab_sm + a.n_seq;    // blocks that it keeps
  const uint32_t bs = a.block_shift, bt = 1u << bs;
  const uint32_t rank = cluster_rank(), ctas = cluster_ctas();
  pdl_trigger();
  pdl_wait();
  const int32_t n_free = *a.n_free;
  if (threadIdx.x == 0) odd_ids = 0;
  uint64_t total = 0;
  const auto blocks = [&](int32_t tokens) { return (uint32_t)(((uint64_t)tokens + bt - 1) >> bs); };
  // the tokens that request r keeps of its h
  const auto keeps = [&](uint32_t r, int32_t h) { return a.keep ? min(a.keep[r], h) : a.done[r] != 0 ? 0 : h; };
  // a length that is none, or that its table row cannot hold: the request stays as it is
  const auto wrong = [&](int32_t h, int32_t kept) { return (kept < h && kept < 0) || h < kept || blocks(max(h, 0)) > a.stride; };
  for (uint32_t r0 = 0; r0 < a.n_seq; r0 += blockDim.x) {
    const uint32_t r = r0 + threadIdx.x;
    uint32_t n = 0, first = 0;
    if (r < a.n_seq) {
      const int32_t h = a.have[r], kept = keeps(r, h);
      if (kept != h && !wrong(h, kept)) first = blocks(kept), n = blocks(h) - first;
    }
    const uint64_t end = block_scan64(n, total, part);
    if (r < a.n_seq) start[r] = (int32_t)min(end - n, (uint64_t)a.n_blocks), skip[r] = (int32_t)first;
  }
  // a stack that would outgrow the pool means blocks given back twice
  const bool bad = n_free < 0 || (int64_t)n_free + (int64_t)total > (int64_t)a.n_blocks;
  __syncthreads();
  if (ctas > 1) cluster_barrier();
  bool odd = false;
  for (uint32_t i = rank * blockDim.x + threadIdx.x; !bad && i < total; i += ctas * blockDim.x) {
    const uint32_t q = owner_of(start, a.n_seq, (int32_t)i);
    const int32_t id = a.table[(size_t)q * a.stride + skip[q] + (i - start[q])];
    odd |= (uint32_t)id >= a.n_blocks;
    a.free_ids[n_free + i] = id;
  }
  odd = __syncthreads_or(odd);
  if (ctas > 1) {  // CTA 0 alone waits for the others' ids, and writes the lengths meanwhile
    if (odd && rank && threadIdx.x == 0) cluster_put(&odd_ids, 0, 1);
    cluster_arrive();
  }
  if (rank) return;
  for (uint32_t r = threadIdx.x; r < a.n_seq; r += blockDim.x) {
    const int32_t h = a.have[r];
    const int32_t kept = keeps(r, h);
    const bool no = kept != h && wrong(h, kept);
    if (no) set_error(a.err, DERR_BAD_POS);
    a.lens[r] = bad || no ? h : kept;
  }
  if (ctas > 1) {
    cluster_wait();
    odd |= odd_ids != 0;
  }
  if (odd) {  // the others move up, a block's worth at a time: all of it is read before any of it is written
    uint64_t kept = 0;
    for (uint32_t i0 = 0; i0 < total; i0 += blockDim.x) {
      const uint32_t i = i0 + threadIdx.x;
      const int32_t id = i < total ? a.free_ids[n_free + i] : -1;
      const bool good = (uint32_t)id < a.n_blocks;
      const uint64_t end = block_scan64(good, kept, part);
      if (good) a.free_ids[n_free + (int32_t)end - 1] = id;
    }
    total = kept;
  }
  if ((bad || odd) && threadIdx.x == 0) set_error(a.err, DERR_BAD_POS);
  if (threadIdx.x == 0) *a.n_free_out = bad ? n_free : n_free + (int32_t)total;
}

template <typename Args>
cudaError_t tables_go(void (*kernel)(Args), const Args& a, uint32_t rows, uint32_t arrays, cudaStream_t st) {
  const uint32_t most = a.n_seq > rows ? a.n_seq : rows, ctas = rows > TAB_ROWS ? TAB_CLUSTER : 1;
  return launch_early(kernel, ctas, dim3(ctas), dim3(most >= TAB_THREADS ? TAB_THREADS : (most + 127) / 128 * 128),
                         arrays * 4 * a.n_seq, st, a);
}

// ---- append ----

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
// Four bytes to_byte(x / s), by the division.
template <uint32_t TYPE>
__device__ __noinline__ uint32_t quotients(float4 x, float s) {
  if (!(s > 0.f)) return 0;
  return to_byte<TYPE>(__fdiv_rn(x.x, s)) | to_byte<TYPE>(__fdiv_rn(x.y, s)) << 8 | to_byte<TYPE>(__fdiv_rn(x.z, s)) << 16 |
         (uint32_t)to_byte<TYPE>(__fdiv_rn(x.w, s)) << 24;
}
// The same from products with inv = 1 / s (0: not to be used) where the two
// cannot differ: a product is within 2^-22 of the quotient, so its rounding is
// the quotient's unless a border of the type's grid lies that near.  Divisions
// took three quarters of a long call's instructions.
template <uint32_t TYPE>
__device__ __forceinline__ uint32_t round4(float4 x, float s, float inv) {
  const float r[4] = {x.x * inv, x.y * inv, x.z * inv, x.w * inv};
  const float all = (r[0] + r[1]) + (r[2] + r[3]);  // not a number if one of them is
  if constexpr (TYPE == PAGES_I8) {
    float off = 0.f, big = 0.f;
    uint32_t i[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float m = r[e] + 12582912.f;  // 1.5 * 2^23: the integer, halves to even, in the low bits
      i[e] = __float_as_uint(m);
      off = fmaxf(off, fabsf(r[e] - (m - 12582912.f)));
      big = fmaxf(big, fabsf(r[e]));
    }
    if (inv > 0.f && off < 0.4999f && big < 127.25f && all == all)
      return __byte_perm(__byte_perm(i[0], i[1], 0x0040), __byte_perm(i[2], i[3], 0x0040), 0x5410);
  } else {
    constexpr float LO = 1.f - 0x1p-21f, HI = 1.f + 0x1p-21f;
    const auto two = [](float a, float b) {
      return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    };
    const uint32_t lo = two(r[0] * LO, r[1] * LO) | two(r[2] * LO, r[3] * LO) << 16;
    const uint32_t hi = two(r[0] * HI, r[1] * HI) | two(r[2] * HI, r[3] * HI) << 16;
    if (inv > 0.f && lo == hi && all == all) return lo;
  }
  return quotients<TYPE>(x, s);
}
template <uint32_t TYPE>
__device__ __forceinline__ float from_byte(uint8_t b) {
  if constexpr (TYPE == PAGES_I8) return (float)(int8_t)b;
  return e4m3_value(b);
}

constexpr int APP_THREADS = 256;
constexpr int APP_WARPS = APP_THREADS / 32;
constexpr int APP_TOKENS = APP_THREADS;  // tokens whose runs a CTA lists at a time
constexpr uint32_t APP_HASH = 16384;

// How a warp reads rows of HD elements of a type: LANES lanes a row, ROWS rows
// at once, N elements (16 bytes) a lane.
template <int HD, uint32_t DT>
struct RowLay {
  static constexpr int N = DT == DT_F32 ? 4 : 8;
  static constexpr int HELD = 32 / N;  // pieces that a lane holds
  static constexpr int LANES = HD / N;
  static constexpr int ROWS = 32 / LANES;
};

// N elements from x[at] on, as they lie.
template <uint32_t DT>
__device__ __forceinline__ uint4 load_piece(const void* x, size_t at, bool wide) {
  if constexpr (DT == DT_F32) {
    const uint32_t* u = static_cast<const uint32_t*>(x) + at;
    return wide ? *reinterpret_cast<const uint4*>(u) : make_uint4(u[0], u[1], u[2], u[3]);
  } else {
    const unsigned short* u = static_cast<const unsigned short*>(x) + at;
    if (wide) return *reinterpret_cast<const uint4*>(u);
    auto two = [&](int i) { return (uint32_t)u[i] | (uint32_t)u[i + 1] << 16; };
    return make_uint4(two(0), two(2), two(4), two(6));
  }
}
template <uint32_t DT>
__device__ __forceinline__ float element(const uint4& w, int e) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
  if constexpr (DT == DT_F32) return __uint_as_float(u[e]);
  const uint32_t half = u[e / 2] >> (16 * (e & 1));
  if constexpr (DT == DT_F16) return __half2float(__ushort_as_half((unsigned short)half));
  return __uint_as_float(half << 16);
}

// The largest magnitude of a piece; NaN counts for nothing.
template <uint32_t DT>
__device__ __forceinline__ float largest(const uint4& w) {
  if constexpr (DT == DT_F32) {
    return fmaxf(fmaxf(fabsf(element<DT>(w, 0)), fabsf(element<DT>(w, 1))),
                 fmaxf(fabsf(element<DT>(w, 2)), fabsf(element<DT>(w, 3))));
  } else {
    using H2 = typename std::conditional<DT == DT_F16, __half2, __nv_bfloat162>::type;
    const H2* h = reinterpret_cast<const H2*>(&w);
    const H2 m = __hmax2(__hmax2(__habs2(h[0]), __habs2(h[1])), __hmax2(__habs2(h[2]), __habs2(h[3])));
    const uint32_t u = *reinterpret_cast<const uint32_t*>(&m);
    const float lo = DT == DT_F16 ? __half2float(__ushort_as_half((unsigned short)u)) : __uint_as_float(u << 16);
    const float hi = DT == DT_F16 ? __half2float(__ushort_as_half((unsigned short)(u >> 16))) : __uint_as_float(u & 0xFFFF0000u);
    return fmaxf(lo, hi);
  }
}

// Rows < first of the block to a larger scale, in 16-byte pieces.
template <uint32_t TYPE>
__device__ __forceinline__ void rescale(uint8_t* dst, uint32_t bytes, float ratio, uint32_t from, uint32_t step) {
  for (uint32_t i = from; i < bytes / 16; i += step) {
    uint4 w = reinterpret_cast<uint4*>(dst)[i];
    uint32_t* u = &w.x;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t r = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        r |= (uint32_t)to_byte<TYPE>(from_byte<TYPE>((uint8_t)(u[j] >> (8 * e))) * ratio) << (8 * e);
      u[j] = r;
    }
    reinterpret_cast<uint4*>(dst)[i] = w;
  }
}

// Refuses the listed runs whose block one of the tokens j .. j + n - 1 has already.
__device__ __noinline__ void refuse_runs(const uint32_t* run_block, const uint32_t* run_t, uint32_t* run_len, uint32_t count,
                                         const int32_t* slots, uint32_t j, uint32_t n, uint32_t bs, int* err) {
  for (uint32_t e = j + n; j < e; ++j) {
    const int32_t slot = slots[j];
    for (uint32_t i = 0; slot >= 0 && i < count; ++i)
      if (run_block[i] == (uint32_t)slot >> bs && j < run_t[i]) {
        run_len[i] = 0;
        set_error(err, DERR_BAD_POS);
      }
  }
}

// The call's tokens fall into runs of consecutive slots of one block.  An item
// is one run of one head's K or V; the grid is cut by tokens and by (head, K or
// V), and an item belongs to the CTA that has its run's first token.  A warp
// takes an item: the largest magnitude of its rows raises the block's scale if
// need be (the block's earlier rows are then rounded to the new one), and the rows
// are rounded to it, from registers or, in longer runs, read again from L1 / L2.
// Of a prompt's whole blocks all of a CTA's warps take one item after the other,
// its rows in their registers.
// A block whose rows come in two runs of one call would be written by two CTAs at
// once: the later run is refused, so each CTA looks through the earlier tokens for
// the blocks of its own runs (a bit per hashed block first).  That is a number of
// reads that grows with the square of the call's tokens: nothing to be seen of it
// at 20000 (62 us), a sixth of the time at 65536 (242 us), two fifths at 131072 (694).
//
// 6300 tokens of bf16 (8 heads of 128) into e4m3 blocks of 64: 20 to 22 us (1.8 TB/s)
// in a row of calls, bound by instructions (22 an element, most of them the two
// roundings of round4) at 0.5 a cycle and by 3 or 4 CTAs on an SM; 32 tokens 5 us.
template <int HD, uint32_t TYPE, uint32_t DT>
__global__ void __launch_bounds__(APP_THREADS, 4) append_kernel(PagesPool p, uint32_t n, const void* k, const void* v,
                                                                size_t row_stride, bool wide, const int32_t* slots,
                                                                uint32_t tokens, uint32_t pairs, int* err) {
  using R = RowLay<HD, DT>;
  constexpr uint32_t WARP_ROWS = R::HELD * R::ROWS;  // rows that a warp holds
  constexpr float TOP = TYPE == PAGES_I8 ? 127.f : 448.f;
  __shared__ uint32_t run_t[APP_TOKENS], run_len[APP_TOKENS], run_block[APP_TOKENS];
  __shared__ uint32_t hash[APP_HASH / 32];
  __shared__ uint32_t follows[2 * APP_TOKENS / 32 + 1];  // bit: the token is in its predecessor's run
  __shared__ uint32_t warp_runs[APP_WARPS];
  __shared__ float peak[APP_WARPS];
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, bs = p.block_shift, bt = 1u << bs;
  const uint32_t first_pair = blockIdx.y * pairs, n_pairs = min(pairs, 2 * p.n_kv - first_pair);

  pdl_trigger();
  pdl_wait();
  const uint64_t t_lo = (uint64_t)blockIdx.x * tokens, t_hi = min((uint64_t)n, t_lo + tokens);
  for (uint64_t t0 = t_lo; t0 < t_hi; t0 += APP_TOKENS) {
    // ---- the runs that begin here ----
    __syncthreads();
    for (uint32_t i = tid; i < APP_HASH / 32; i += APP_THREADS) hash[i] = 0;
    int32_t mine = -1;
#pragma unroll
    for (int half = 0; half < 2; ++half) {  // these tokens and the next ones, into which a run may reach
      const uint64_t t = t0 + half * APP_TOKENS + tid;
      const int32_t slot = t < n ? slots[t] : -1;
      const bool f = slot >= 0 && t > 0 && ((uint32_t)slot & (bt - 1)) && slots[t - 1] == slot - 1;
      const uint32_t bits = __ballot_sync(0xffffffffu, f);
      if (lane == 0) follows[half * APP_WARPS + warp] = bits;
      if (half == 0 && slot >= 0 && !f && t < t_hi) mine = slot;
    }
    if (tid == 0) follows[2 * APP_WARPS] = 0;
    const uint32_t leads = __ballot_sync(0xffffffffu, mine >= 0);
    if (lane == 0) warp_runs[warp] = __popc(leads);
    __syncthreads();
    uint32_t count = 0, at = __popc(leads & ((1u << lane) - 1));
#pragma unroll
    for (uint32_t w = 0; w < APP_WARPS; ++w) {
      if (w < warp) at += warp_runs[w];
      count += warp_runs[w];
    }
    if (mine >= 0) {
      const uint32_t i = at, b = (uint32_t)mine >> bs;
      // the run ends where a bit after this token's is 0
      uint32_t w = (tid + 1) >> 5, gap = ~follows[w] & (0xffffffffu << ((tid + 1) & 31));
      while (gap == 0) gap = ~follows[++w];
      run_t[i] = (uint32_t)t0 + tid;
      run_block[i] = b;
      run_len[i] = 32 * w + __ffs(gap) - 1 - tid;
      atomicOr(&hash[(b & (APP_HASH - 1)) >> 5], 1u << (b & 31));
      if (b >= p.n_blocks) {
        run_len[i] = 0;
        set_error(err, DERR_BAD_POS);
      }
    }
    __syncthreads();
    if (count == 0) continue;
    // (this part of the tokens may hold a second run as well)
    const uint32_t look = (uint32_t)min((uint64_t)n, t0 + APP_TOKENS);
    auto maybe = [&](int32_t slot) -> uint32_t {
      const uint32_t b = (uint32_t)slot >> bs;  // (a padding row's bit may be set: refuse_runs looks again)
      return (hash[(b & (APP_HASH - 1)) >> 5] >> (b & 31)) & 1;
    };
    uint32_t j0 = 0;
    if ((reinterpret_cast<uintptr_t>(slots) & 15) == 0) {
      j0 = look & ~3u;
#pragma unroll 4
      for (uint32_t j = 4 * tid; j < j0; j += 4 * APP_THREADS) {
        const int4 v = *reinterpret_cast<const int4*>(slots + j);
        if (maybe(v.x) | maybe(v.y) | maybe(v.z) | maybe(v.w)) refuse_runs(run_block, run_t, run_len, count, slots, j, 4, bs, err);
      }
    }
    for (uint32_t j = j0 + tid; j < look; j += APP_THREADS)
      if (maybe(slots[j])) refuse_runs(run_block, run_t, run_len, count, slots, j, 1, bs, err);
    __syncthreads();

    // ---- the items: one to a warp, then the long ones by all warps together ----
    const uint32_t items = count * n_pairs, long_run = items < APP_WARPS ? WARP_ROWS : 2 * WARP_ROWS;
    bool any = false;
    for (int together = 0; together < 2; ++together) {
      const uint32_t warps = together ? APP_WARPS : 1, w = together ? warp : 0;
      for (uint32_t it = together ? 0 : warp; it < items; it += together ? 1 : APP_WARPS) {
        const uint32_t q = it / n_pairs, len = run_len[q], pair = first_pair + it % n_pairs;
        if (len == 0) continue;
        if ((len > long_run) != (together != 0)) {
          any = true;
          continue;
        }
        const uint32_t rt = run_t[q], b = run_block[q], first = (uint32_t)slots[rt] & (bt - 1), h = pair >> 1;
        const void* x = (pair & 1) ? v : k;
        uint8_t* dst = ((pair & 1) ? p.v : p.k) + (((size_t)b * p.n_kv + h) << bs) * HD;
        float* sp = ((pair & 1) ? p.vs : p.ks) + (size_t)b * p.n_kv + h;
        const uint32_t sub = lane / R::LANES, col = (lane % R::LANES) * R::N;
        const size_t src = rt * row_stride + (size_t)h * HD + col;
        const bool once = len <= warps * WARP_ROWS;  // else the rows are read twice
        const float old = first ? *sp : 0.f;
        uint4 val[R::HELD];
        float m = 0.f;
        auto read_rows = [&](uint32_t r0) {
#pragma unroll
          for (int i = 0; i < R::HELD; ++i) {
            const uint32_t r = r0 + i * R::ROWS + sub;
            val[i] = r < len ? load_piece<DT>(x, src + r * row_stride, wide) : make_uint4(0, 0, 0, 0);
          }
        };
        for (uint32_t r0 = w * WARP_ROWS; r0 < len; r0 += warps * WARP_ROWS) {
          read_rows(r0);
#pragma unroll
          for (int i = 0; i < R::HELD; ++i) m = fmaxf(m, largest<DT>(val[i]));
        }
        m = warp_max(m);
        if (together) {
          __syncthreads();
          if (lane == 0) peak[warp] = m;
          __syncthreads();
          for (uint32_t i = 0; i < APP_WARPS; ++i) m = fmaxf(m, peak[i]);
        }
        const float s = fmaxf(old, __fdiv_rn(m, TOP));
        if (first && s > old) rescale<TYPE>(dst, first * HD, __fdiv_rn(old, s), w * 32 + lane, warps * 32);
        const float inv = s > 1e-30f && s < 1e30f ? __frcp_rn(s) : 0.f;
        for (uint32_t r0 = w * WARP_ROWS; r0 < len; r0 += warps * WARP_ROWS) {
          if (!once) read_rows(r0);
#pragma unroll
          for (int i = 0; i < R::HELD; ++i) {
            const uint32_t r = r0 + i * R::ROWS + sub;
            if (r >= len) continue;
            uint32_t out[R::N / 4];
#pragma unroll
            for (int j = 0; j < R::N; j += 4)
              out[j / 4] = round4<TYPE>(make_float4(element<DT>(val[i], j), element<DT>(val[i], j + 1),
                                                    element<DT>(val[i], j + 2), element<DT>(val[i], j + 3)), s, inv);
            uint8_t* to = dst + (size_t)(first + r) * HD + col;
            if constexpr (R::N == 4)
              *reinterpret_cast<uint32_t*>(to) = out[0];
            else
              *reinterpret_cast<uint2*>(to) = make_uint2(out[0], out[1]);
          }
        }
        if (together)
          __syncthreads();
        else
          __syncwarp();
        if (w == 0 && lane == 0) *sp = s;  // every thread has read the old one
      }
      if (!together && !__syncthreads_or(any)) break;
    }
  }
}

// Four values a thread: 4 bytes in, 16 out, both whole lines to a warp.  Bound by
// memory: 6300 tokens of 8 x 128 (64 MB) 11.7 us, 5.5 TB/s.
template <uint32_t TYPE>
__global__ void __launch_bounds__(256) read_kernel(PagesPool p, uint32_t n, const int32_t* slots, float* k, float* v,
                                                   bool wide, int* err) {
  const uint32_t quads = p.n_kv * p.hd / 4;  // of a row
  pdl_trigger();
  pdl_wait();
  const uint64_t total = (uint64_t)n * quads;
  for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (uint64_t)gridDim.x * blockDim.x) {
    const uint32_t r = (uint32_t)(i / quads), d = 4 * (uint32_t)(i % quads);
    const int32_t slot = slots[r];
    if (slot < 0) continue;
    const uint32_t b = (uint32_t)slot >> p.block_shift, t = (uint32_t)slot & ((1u << p.block_shift) - 1);
    if (b >= p.n_blocks) {
      set_error(err, DERR_BAD_POS);
      continue;
    }
    const size_t bh = (size_t)b * p.n_kv + d / p.hd, at = ((bh << p.block_shift) + t) * p.hd + d % p.hd;
    const uint32_t wk = *reinterpret_cast<const uint32_t*>(p.k + at), wv = *reinterpret_cast<const uint32_t*>(p.v + at);
    const float ks = p.ks[bh], vs = p.vs[bh];
    float a[4], c[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      a[e] = from_byte<TYPE>((uint8_t)(wk >> (8 * e))) * ks;
      c[e] = from_byte<TYPE>((uint8_t)(wv >> (8 * e))) * vs;
    }
    const size_t o = (size_t)r * 4 * quads + d;
    if (wide) {
      *reinterpret_cast<float4*>(k + o) = make_float4(a[0], a[1], a[2], a[3]);
      *reinterpret_cast<float4*>(v + o) = make_float4(c[0], c[1], c[2], c[3]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) k[o + e] = a[e], v[o + e] = c[e];
    }
  }
}

struct AppendCall {
  uint32_t n;
  const void *k, *v;
  size_t row_stride;
  const int32_t* slots;
  int* err;
  dim3 grid;
  uint32_t tokens, pairs;  // of a CTA
  bool wide;
  cudaStream_t st;
};

template <int HD, uint32_t TYPE, uint32_t DT>
cudaError_t append_go(const PagesPool& p, const AppendCall& c) {
  return launch_early(append_kernel<HD, TYPE, DT>, 1, c.grid, dim3(APP_THREADS), 0, c.st, p, c.n, c.k, c.v, c.row_stride, c.wide,
                  c.slots, c.tokens, c.pairs, c.err);
}
template <int HD, uint32_t TYPE>
cudaError_t append_dt(const PagesPool& p, uint32_t dtype, const AppendCall& c) {
  if (dtype == DT_F32) return append_go<HD, TYPE, DT_F32>(p, c);
  return dtype == DT_F16 ? append_go<HD, TYPE, DT_F16>(p, c) : append_go<HD, TYPE, DT_BF16>(p, c);
}

}  // namespace

cudaError_t pages_init() {
  cudaError_t e = cudaFuncSetAttribute(assign_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 3 * 4 * 16384);
  if (e != cudaSuccess) return e;
  e = cudaFuncSetAttribute(release_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * 4 * 16384);
  return e != cudaSuccess ? e : pages_attend_init();
}

cudaError_t pages_assign_launch(const AssignArgs& a, cudaStream_t st) {
  return tables_go(assign_kernel, a, a.n_rows, 3, st);
}

cudaError_t pages_release_launch(const ReleaseArgs& a, cudaStream_t st) {
  // the blocks to give back are at most what the tables can hold, or the pool
  const uint64_t most = (uint64_t)a.n_seq * a.stride;
  return tables_go(release_kernel, a, most < a.n_blocks ? (uint32_t)most : a.n_blocks, 2, st);
}

cudaError_t pages_append_launch(const PagesPool& p, uint32_t n, const void* k, const void* v, uint32_t dtype,
                                size_t row_stride, const int32_t* slots, int* err, int num_sms, cudaStream_t st) {
  // Few tokens, or blocks of 16: short runs, a warp per item, so 8 (head, K or V)
  // pairs to a CTA.  Else one pair to a CTA and whole blocks of tokens to it.
  // (8 heads of 128, bf16 to e4m3: 6300 tokens of prompts in blocks of 64 34 us with
  // 8 pairs, 22 with one; in blocks of 16 18.6 and 20.5.  Runs are known on the
  // device alone, so the rule goes by n and loses where they are unlike that: 4000
  // single tokens in blocks of 64 take 59 us with one pair where 8 would take 35,
  // two prompts of 150 take 22 with 8 where one would take 11.)
  const uint32_t all = 2 * p.n_kv, full = 4 * (uint32_t)num_sms, bt = 1u << p.block_shift;
  const bool by_warp = bt <= 16 || (uint64_t)n * all <= (uint64_t)APP_WARPS * full;
  const uint32_t pairs = by_warp ? APP_WARPS : 1, ny = (all + pairs - 1) / pairs;
  const uint32_t most = (full + ny - 1) / ny, nx = n < most ? n : most;
  uint32_t tokens = (n + nx - 1) / nx;
  if (!by_warp) tokens = (tokens + bt - 1) / bt * bt;
  const size_t es = dtype == DT_F32 ? 4 : 2;
  const bool wide = ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | row_stride * es) & 15) == 0;
  const AppendCall c{n, k, v, row_stride, slots, err, dim3((n + tokens - 1) / tokens, ny), tokens, pairs, wide, st};
  if (p.hd == 64) return p.type == PAGES_I8 ? append_dt<64, PAGES_I8>(p, dtype, c) : append_dt<64, PAGES_E4M3>(p, dtype, c);
  return p.type == PAGES_I8 ? append_dt<128, PAGES_I8>(p, dtype, c) : append_dt<128, PAGES_E4M3>(p, dtype, c);
}

cudaError_t pages_read_launch(const PagesPool& p, uint32_t n, const int32_t* slots, float* k, float* v, int* err,
                              int num_sms, cudaStream_t st) {
  const uint64_t ctas = ((uint64_t)n * p.n_kv * p.hd / 4 + 255) / 256, most = (uint64_t)num_sms * 32;
  const bool wide = ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0;
  const dim3 grid((uint32_t)(ctas < most ? ctas : most));
  return launch_early(p.type == PAGES_I8 ? read_kernel<PAGES_I8> : read_kernel<PAGES_E4M3>, 1, grid, dim3(256), 0, st, p, n, slots, k,
                  v, wide, err);
}

}  // namespace shk
