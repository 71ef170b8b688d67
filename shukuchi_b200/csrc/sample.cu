// sample.cu -- temperature, top-k, top-p and min-p sampling.
//
// A row's logits z become x = (z - z_max) * (1 / T) and weights w = exp(x),
// both in fp32, and the weights become whole numbers W = floor(w * 2^40):
// every sum below is a sum of integers, so that the token that a random
// number picks does not depend on the order in which threads add.
//
// The row is read once: a thread-block cluster takes it, each CTA a run of the
// vocabulary that stays in its shared memory, and what the CTAs need of one
// another (maximum, histograms, sums) goes over distributed shared memory.
// Nothing is sorted.  Tokens are ordered by (logit, lower index), each one's
// place being one 50-bit number c, and top-k and top-p together keep c >= C.
// C is found from a histogram over x, 2048 bins down to the x whose weight is 0:
// of counts for top-k, of weights in 16 bits for top-p (one 32-bit atomic a token;
// sums in 64 bits there took three times as long).  That names the bin of the
// border token; what lies above it is then summed exactly, and the bin's own
// tokens, a hundred or so in a row of 128k, go to every CTA of the cluster, which
// ranks them by comparison (of flat rows' fuller bins only the part with the border:
// 64 rows of 128256, logits N(0, 2.5), T 1.3, top-p 0.97: 84 us without, 69).  Where
// the exact sums disagree with the 16-bit ones the next bin is taken.  A bin with
// more than CAP tokens (equal logits, mostly) is searched by the digits of c instead.
//
// A small top-k takes a shorter way: the k-th largest of the threads' own maxima
// is at most the k-th largest logit, so the tokens from its bin up, not many more
// than k, go to one CTA, which does the rest with them alone.
//
// Bound by instructions: about 100 a token with top-p (two exponentials of libm
// quality, exact integer sums, the bin), IPC 0.58 of 1 with two CTAs an SM, the
// rest barriers.  128256 logits: 11.5 us a row alone, 40 us for 64 rows of mixed
// settings (0.82 TB/s); 333 rows of 32000 51 us with top-p, 31 with temperature alone.
// Slices of 8192 logits (three or four CTAs an SM) 71 to 80 us for the 333 rows,
// of 32768 60 (and 50 against 53 for 64 rows with top-p, 29 against 36 with top-k).
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

constexpr int THREADS = 512;
constexpr int WARPS = THREADS / 32;
constexpr int MAX_CL = 8;
constexpr int OWN = 4;               // bins a thread: 16 bytes of a peer's histogram, whole lines to a warp
constexpr int NB = OWN * THREADS;
constexpr int DIGITS = 2 * THREADS;  // of the search by digits, 10 bits each
constexpr int CAP = 512;             // candidates that are ranked by comparison
constexpr int FINE = 64;             // parts of the border bin, where it has more than FINE_FROM tokens
constexpr int FINE_FROM = 128;
constexpr float X_MIN = -27.75f;     // exp(x) * 2^40 < 1 below
constexpr int IDX_BITS = 18;
constexpr uint32_t IDX_MASK = (1u << IDX_BITS) - 1;
static_assert(SAMPLE_MAX_VOCAB <= 1u << IDX_BITS, "an index fits its bits of c");
constexpr uint32_t MAX_SLICE = SAMPLE_MAX_VOCAB / MAX_CL;

template <uint32_t DT>
__device__ __forceinline__ float logit(const void* p, size_t i) {
  if constexpr (DT == DT_F32) return static_cast<const float*>(p)[i];
  if constexpr (DT == DT_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
// As the row is held: NaN as -inf.
__device__ __forceinline__ float clean(float z) { return fmaxf(z, -INFINITY); }

// Larger logits have larger keys; -0 and +0 compare equal and have one.
__device__ __forceinline__ uint32_t key_of(float z) {
  const uint32_t u = __float_as_uint(z + 0.f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? key & 0x7FFFFFFFu : ~key);
}
__device__ __forceinline__ uint64_t place_of(float z, uint32_t i) {
  return ((uint64_t)key_of(z) << IDX_BITS) | (IDX_MASK - i);
}

// ODD: an infinite maximum or factor, so that differences and products may be NaN.
template <bool ODD>
struct Scale {
  float zmax, inv_t;
  __device__ __forceinline__ float x(float z) const {
    const float v = (z - zmax) * inv_t;
    if constexpr (ODD) return z == zmax ? 0.f : v <= 0.f ? v : -INFINITY;
    return v;
  }
  __device__ __forceinline__ float weight(float z) const { return expf(x(z)); }
};
// Rises as x falls, from bin 0 on; NB for a token without weight.
// (2^23 + the bin, or more than 2^23 + NB.)
__device__ __forceinline__ float bin_float(float x) { return __fmaf_rd(x, NB / X_MIN, 8388608.f); }
__device__ __forceinline__ int bin_of(float x) {
  return x > X_MIN ? (int)(__float_as_uint(bin_float(x)) - 0x4B000000u) : NB;
}

// floor(w * 2^40) for w in [0, 1] as two numbers of 20 bits, rounded down by
// additions of 2^23 (conversions to 64-bit integers run at a fraction of their
// rate), and sums of up to 4096 of them.
struct Mass {
  uint32_t hi = 0, lo = 0;
  __device__ __forceinline__ void add(float w) {
    const float h = __fmaf_rd(w, 1048576.f, 8388608.f);
    const float rest = __fmaf_rn(w, 1048576.f, 8388608.f - h);  // exact
    hi += __float_as_uint(h) - 0x4B000000u;
    lo += __float_as_uint(__fmaf_rd(rest, 1048576.f, 8388608.f)) - 0x4B000000u;
  }
  __device__ __forceinline__ uint64_t value() const { return ((uint64_t)hi << 20) + lo; }
};
__device__ __forceinline__ uint64_t mass_of(float w) {
  Mass m;
  m.add(w);
  return m.value();
}
// Weights of bin b times 2^(16 + bin_scale) fit 16 bits and a bit over.
__device__ __forceinline__ int bin_scale(int b) { return min(24, (b * 1281) >> 16); }

__device__ __forceinline__ uint64_t warp_sum64(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <typename T>
__device__ __forceinline__ T warp_scan(T v, uint32_t lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= (uint32_t)o) v += u;
  }
  return v;
}

// ---- cluster ----
__device__ __forceinline__ uint32_t cl_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cl_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cl_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Another CTA's memory may be touched once that CTA has begun: each says so at
// its start, and waits for the others' word before its first store to them.
__device__ __forceinline__ void cl_begun() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cl_all_begun() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer(const void* p, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ void put32(uint32_t a, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
}
__device__ __forceinline__ void put64(uint32_t a, uint64_t v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(a), "l"(v) : "memory");
}
__device__ __forceinline__ uint4 get32x4(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint2 get32x2(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared::cluster.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ ulonglong2 get64x2(uint32_t a) {
  ulonglong2 v;
  asm volatile("ld.shared::cluster.v2.u64 {%0, %1}, [%2];" : "=l"(v.x), "=l"(v.y) : "r"(a) : "memory");
  return v;
}

struct Fine {  // the border bin's tokens once more, by parts of it
  unsigned long long mass[FINE];
  uint32_t cnt[FINE], n;
  uint64_t above_mass;
  uint32_t part, above_cnt;
  uint16_t list[CAP];  // tokens of the border's part
};

struct Shared {
  uint32_t hist[NB];  // of the slice's tokens: how many, or their weights times 2^(16 + bin_scale)
  union {
    struct {  // the border bin's tokens; two lists in turn, so that one can be written while a peer reads the other
      uint64_t place[2][CAP], mass[2][CAP];
    } cand;
    struct {
      unsigned long long mass[DIGITS];
      uint32_t cnt[DIGITS];
    } digits;
    struct {  // CTA 0: all the tokens that may stay
      uint64_t place[CAP], mass[CAP];
      float w[CAP];
    } few;
  };
  uint64_t part[WARPS], part2[WARPS];
  unsigned long long kept[WARPS];  // weights that stay of each warp's run
  uint64_t xsum[MAX_CL], xabove[2][MAX_CL], xin[2][MAX_CL];
  uint32_t part32[WARPS], xcnt[2][MAX_CL];
  float xmax[MAX_CL];
  // what one thread found
  uint64_t border, inside, above, above_mass;
  uint32_t bin;
  uint32_t next[3];  // CTA 0: places given out in the lists, three counters in turn
  uint32_t own;      // tokens of this CTA in the list
};

// Places for a warp's `mine` tokens (of 4 a lane) in a list whose counter is CTA
// 0's: one atomic for all of them, as it takes as long as a hundred
// instructions.  A lane's first place; its tokens follow one another.
__device__ __forceinline__ uint32_t take_places(uint32_t* counter, uint32_t mine, Shared& s) {
  const uint32_t lane = threadIdx.x & 31, upto = warp_scan(mine, lane);
  uint32_t at = 0;
  if (lane == 31) {
    atomicAdd(&s.own, upto);
    asm volatile("atom.relaxed.cluster.shared::cluster.add.u32 %0, [%1], %2;"
                 : "=r"(at)
                 : "r"(peer(counter, 0)), "r"(upto)
                 : "memory");
  }
  return __shfl_sync(0xffffffffu, at, 31) + upto - mine;
}

// A cluster's totals at this thread's bins (bin 0 holds the largest tokens),
// and the running total before them.
template <int N>
struct Totals {
  uint64_t v[N], before;
};

template <int N>
__device__ __forceinline__ void run_totals(Totals<N>& t, uint64_t* part) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint64_t own = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) own += t.v[i];
  const uint64_t upto = warp_scan(own, lane);
  __syncthreads();
  if (lane == 31) part[warp] = upto;
  __syncthreads();
  t.before = upto - own;
  for (uint32_t w = 0; w < warp; ++w) t.before += part[w];
}

// The bin at which the running total reaches `need` (s.bin; N * THREADS where it
// does not) and the total before it (s.above).
template <int N>
__device__ __forceinline__ void find_bin(const Totals<N>& t, uint64_t need, Shared& s) {
  __syncthreads();
  if (threadIdx.x == 0) s.bin = N * THREADS;
  __syncthreads();
  uint64_t c = t.before;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (c < need && need <= c + t.v[i]) s.bin = N * threadIdx.x + i, s.above = c;
    c += t.v[i];
  }
  __syncthreads();
}

// The nearest bin with tokens before (step -1) or after (1) bin b to s.bin; NB if there is none.
__device__ __forceinline__ void next_bin(const Totals<OWN>& t, int b, int step, Shared& s) {
  __syncthreads();
  if (threadIdx.x == 0) s.own = step > 0 ? NB : 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < OWN; ++i) {
    const int mine = OWN * (int)threadIdx.x + i;
    if (t.v[i] && step > 0 && mine > b) atomicMin(&s.own, (uint32_t)mine);
    if (t.v[i] && step < 0 && mine < b) atomicMax(&s.own, (uint32_t)mine + 1);
  }
  __syncthreads();
  if (threadIdx.x == 0) s.bin = step > 0 ? s.own : s.own ? s.own - 1 : NB;
  __syncthreads();
}

template <bool ODD>
struct Part {  // one CTA's part of a row
  const float* z;
  uint32_t n, base, rank, cl;
  uint32_t run;  // of a warp, a multiple of 4
  Scale<ODD> sc;
  float min_p;
};

// Four tokens at a time (those behind the slice's last are -inf).  What is done
// with each of them has no branch, so that their chains of dependent
// instructions run side by side (top-p's pass over 16k tokens: 7.6k cycles; one
// token after the other, each with a branch, 9.2k).
template <bool ODD, typename F>
__device__ __forceinline__ void each4(const Part<ODD>& p, F f) {
  for (uint32_t i0 = 128 * (threadIdx.x >> 5); i0 < p.n; i0 += 4 * THREADS) {  // whole warps stay together
    const uint32_t i = i0 + 4 * (threadIdx.x & 31);
    float4 v = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    if (i < p.n) v = *reinterpret_cast<const float4*>(p.z + i);
    const float w[4] = {v.x, v.y, v.z, v.w};
    f(i, w);
  }
}
// The same, each warp over its run of the slice.
template <bool ODD, typename F>
__device__ __forceinline__ void each4_of_run(const Part<ODD>& p, F f) {
  const uint32_t lo = min(p.n, (threadIdx.x >> 5) * p.run), hi = min(p.n, lo + p.run);
  for (uint32_t i0 = lo; i0 < hi; i0 += 128) {
    const uint32_t i = i0 + 4 * (threadIdx.x & 31);
    float4 v = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    if (i < hi) v = *reinterpret_cast<const float4*>(p.z + i);
    const float w[4] = {v.x, v.y, v.z, v.w};
    f(i, w);
  }
}
// One token after the other, for what concerns few of them.
template <bool ODD, typename F>
__device__ __forceinline__ void each(const Part<ODD>& p, F f) {
  for (uint32_t i = 4 * threadIdx.x; i < p.n; i += 4 * THREADS) {
    const float4 v = *reinterpret_cast<const float4*>(p.z + i);
    f(i, v.x), f(i + 1, v.y), f(i + 2, v.z), f(i + 3, v.w);
  }
}

// The border token, from s.bin of find_bin on: s.border = its place, and the
// weight of the tokens down to it in s.inside.  need: by rank (BY_MASS false)
// or by weight.  `turn` alternates between the candidate lists.  Returns whether
// s.kept has the weights that stay of each warp's run (it has not where the
// digits were searched).
template <bool BY_MASS, bool ODD>
__device__ bool find_border(const Part<ODD>& p, const Totals<OWN>& t, uint64_t need, uint32_t& turn, Shared& s) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (;;) {
    const int bin = (int)s.bin;
    const uint32_t list = turn & 1;
    uint32_t* place = &s.next[turn % 3];
    const uint64_t above_cnt = s.above;
    if (threadIdx.x == 0) {
      s.own = 0;
      s.next[(turn + 1) % 3] = 0;  // last used two turns ago
    }
    ++turn;
    __syncthreads();
    Mass above_m, in_m, kept_m;
    // Most tokens lie below the border: a lane marks those of its next 32 that do
    // not, and does the rest for these alone, two by two (333 rows of 32000, T 0.7,
    // top-p 0.9: 60 us with every token's exponential, 53 so; a nearly flat row's
    // pass takes a quarter longer).
    const float least = 8388608.f + (float)bin;
    const uint32_t lo = min(p.n, warp * p.run), hi = min(p.n, lo + p.run);
    for (uint32_t i0 = lo; i0 < hi; i0 += 32 * 32) {
      uint32_t marks = 0;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const uint32_t i = i0 + 128 * c + 4 * lane;
        if (i >= hi) continue;
        const float4 v4 = *reinterpret_cast<const float4*>(p.z + i);
        const float v[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (bin_float(p.sc.x(v[j])) <= least) marks |= 1u << (4 * c + j);
      }
      while (__any_sync(0xffffffffu, marks)) {
        float z[2], e[2];
        uint32_t at_i[2], in = 0;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t c = __ffs(marks) - 1;
          at_i[k] = i0 + 32 * (c & 28) + 4 * lane + (c & 3);
          z[k] = marks ? p.z[at_i[k]] : -INFINITY;
          marks &= marks - 1;
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float x = p.sc.x(z[k]);
          e[k] = expf(x);
          const bool here = bin_of(x) == bin;
          in |= here ? 1u << k : 0;
          above_m.add(here ? 0.f : e[k]);
          if (p.min_p > 0.f) kept_m.add(!here && e[k] >= p.min_p ? e[k] : 0.f);
        }
        if (!__any_sync(0xffffffffu, in)) continue;
        uint32_t at = take_places(place, __popc(in), s);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          if (!(in >> k & 1)) continue;
          in_m.add(e[k]);
          if (at < CAP)
            for (uint32_t r = 0; r < p.cl; ++r) {
              put64(peer(&s.cand.place[list][at], r), place_of(z[k], p.base + at_i[k]));
              put64(peer(&s.cand.mass[list][at], r), mass_of(e[k]));
            }
          ++at;
        }
      }
    }
    uint64_t above = warp_sum64(above_m.value()), in = warp_sum64(in_m.value());
    const uint64_t kept = p.min_p > 0.f ? warp_sum64(kept_m.value()) : above;
    if (lane == 0) s.part[warp] = above, s.part2[warp] = in, s.kept[warp] = kept;
    __syncthreads();
    if (threadIdx.x < p.cl) {
      uint64_t x = 0, y = 0;
      for (int w = 0; w < WARPS; ++w) x += s.part[w], y += s.part2[w];
      put64(peer(&s.xabove[list][p.rank], threadIdx.x), x);
      put64(peer(&s.xin[list][p.rank], threadIdx.x), y);
      put32(peer(&s.xcnt[list][p.rank], threadIdx.x), s.own);
    }
    cl_sync();
    above = in = 0;
    uint32_t m = 0;
    for (uint32_t r = 0; r < p.cl; ++r) above += s.xabove[list][r], in += s.xin[list][r], m += s.xcnt[list][r];
    if (BY_MASS && (need <= above || need > above + in)) {
      next_bin(t, bin, need <= above ? -1 : 1, s);
      if (s.bin < NB) continue;
      if (threadIdx.x == 0) s.border = 0, s.inside = above + in;  // not reached: every token stays
      __syncthreads();
      return false;
    }
    const uint64_t left = BY_MASS ? need - above : need - above_cnt;  // of the bin's own
    if (m <= CAP) {
      uint32_t who = threadIdx.x, rivals = m, over = 0;
      uint64_t over_w = 0;
      Fine& fine = *reinterpret_cast<Fine*>(s.hist);  // every CTA has read the histogram
      const bool split = m > FINE_FROM;
      if (split) {  // only the part with the border is ranked
        if (threadIdx.x < FINE) fine.mass[threadIdx.x] = 0, fine.cnt[threadIdx.x] = 0;
        if (threadIdx.x == 0) fine.n = 0;
        __syncthreads();
        uint32_t f = FINE;
        if (threadIdx.x < m) {
          const float x = p.sc.x(value_of((uint32_t)(s.cand.place[list][threadIdx.x] >> IDX_BITS)));
          f = (__float_as_uint(__fmaf_rd(x, FINE * (NB / X_MIN), 8388608.f)) - 0x4B000000u) & (FINE - 1);  // falls as x rises
          atomicAdd(&fine.mass[f], (unsigned long long)s.cand.mass[list][threadIdx.x]);
          atomicAdd(&fine.cnt[f], 1u);
        }
        __syncthreads();
        if (warp == 0) {
          const uint64_t w0 = fine.mass[2 * lane], w1 = fine.mass[2 * lane + 1];
          const uint32_t c0 = fine.cnt[2 * lane], c1 = fine.cnt[2 * lane + 1];
          const uint64_t w = warp_scan(w0 + w1, lane) - w0 - w1;
          const uint32_t c = warp_scan(c0 + c1, lane) - c0 - c1;
          const uint64_t a0 = BY_MASS ? w : c, a1 = a0 + (BY_MASS ? w0 : c0), a2 = a1 + (BY_MASS ? w1 : c1);
          if (a0 < left && left <= a1) fine.part = 2 * lane, fine.above_mass = w, fine.above_cnt = c;
          if (a1 < left && left <= a2) fine.part = 2 * lane + 1, fine.above_mass = w + w0, fine.above_cnt = c + c0;
        }
        __syncthreads();
        if (f == fine.part) fine.list[atomicAdd(&fine.n, 1u)] = (uint16_t)threadIdx.x;
        __syncthreads();
        rivals = fine.n, over = fine.above_cnt, over_w = fine.above_mass;
        if (threadIdx.x < rivals) who = fine.list[threadIdx.x];
      }
      if (threadIdx.x < rivals) {
        const uint64_t me = s.cand.place[list][who], mine = s.cand.mass[list][who];
        for (uint32_t i = 0; i < rivals; ++i) {
          const uint32_t j = split ? fine.list[i] : i;
          if (s.cand.place[list][j] > me) over += 1, over_w += s.cand.mass[list][j];
        }
        const uint64_t o = BY_MASS ? over_w : over, own = BY_MASS ? mine : 1;
        if (o < left && left <= o + own) s.border = me, s.inside = above + over_w + mine;
      }
      __syncthreads();
      if (threadIdx.x < m) {  // the bin's tokens that stay, to the runs of this slice
        const uint64_t me = s.cand.place[list][threadIdx.x];
        const uint32_t i = IDX_MASK - (uint32_t)(me & IDX_MASK) - p.base;  // huge where it is before the slice
        if (me >= s.border && i < p.n && !(p.sc.weight(value_of((uint32_t)(me >> IDX_BITS))) < p.min_p))
          atomicAdd(&s.kept[i / p.run], (unsigned long long)s.cand.mass[list][threadIdx.x]);
      }
      __syncthreads();
      return true;
    }
    // digit by digit, from the top
    uint64_t prefix = 0, over = 0, over_w = 0;
    for (int shift = 40; shift >= 0; shift -= 10) {
      for (int i = threadIdx.x; i < DIGITS; i += THREADS) s.digits.cnt[i] = 0, s.digits.mass[i] = 0;
      __syncthreads();
      each(p, [&](uint32_t i, float v) {
        if (bin_of(p.sc.x(v)) != bin) return;
        const uint64_t c = place_of(v, p.base + i);
        if ((c >> (shift + 10)) != prefix) return;
        const uint32_t d = DIGITS - 1 - ((uint32_t)(c >> shift) & (DIGITS - 1));
        atomicAdd(&s.digits.cnt[d], 1u);
        atomicAdd(&s.digits.mass[d], (unsigned long long)mass_of(p.sc.weight(v)));
      });
      cl_sync();
      Totals<2> c{}, w{};
      for (uint32_t r = 0; r < p.cl; ++r) {
        const uint2 x = get32x2(peer(&s.digits.cnt[2 * threadIdx.x], r));
        const ulonglong2 y = get64x2(peer(&s.digits.mass[2 * threadIdx.x], r));
        c.v[0] += x.x, c.v[1] += x.y;
        w.v[0] += y.x, w.v[1] += y.y;
      }
      run_totals(c, s.part);
      run_totals(w, s.part2);
      find_bin(BY_MASS ? w : c, left - (BY_MASS ? over_w : over), s);
      const uint32_t d = s.bin;
      if (d / 2 == threadIdx.x) s.above = c.before + (d & 1 ? c.v[0] : 0), s.above_mass = w.before + (d & 1 ? w.v[0] : 0);
      __syncthreads();
      over += s.above;
      over_w += s.above_mass;
      prefix = (prefix << 10) | (DIGITS - 1 - d);
      cl_sync();  // every CTA has read the digits
    }
    if (threadIdx.x == 0) {
      s.border = prefix;
      s.inside = above + over_w + mass_of(p.sc.weight(value_of((uint32_t)(prefix >> IDX_BITS))));
    }
    __syncthreads();
    return false;
  }
}

// The draw, from the row's slices in shared memory and its maximum on.
template <bool ODD>
__device__ __forceinline__ void draw(const SampleArgs& a, const Part<ODD>& p, uint32_t row, float own_max, Shared& s) {
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t n = p.n, base = p.base, rank = p.rank, cl = p.cl;
  const float* z = p.z;
  const float uf = a.u[row];
  const float min_p = p.min_p;
  auto target_of = [&](uint64_t total) {
    const uint64_t t = uf > 0.f ? (uint64_t)fmin((double)uf * (double)total, 1.8e19) : 0;
    return t < total ? t : total - 1;
  };
  auto need_of = [](float top_p, uint64_t sum) {
    const double d = ceil((double)top_p * (double)sum);
    return d >= 1.0 ? (uint64_t)d : 1;
  };

  // ---- the border of top-k and top-p ----
  uint64_t border = 0;  // tokens with a place of at least this stay
  bool summed = false;  // s.kept has their weights
  const int32_t k = a.top_k ? a.top_k[row] : 0;
  const float top_p = a.top_p ? a.top_p[row] : 1.f;
  const bool by_k = k > 0 && (uint32_t)k < a.n_vocab, by_p = top_p < 1.f;
  if (by_k || by_p) {
    uint64_t sum = 0;  // of the whole row, then of the top-k set
    Totals<OWN> t{};
    auto gather = [&](bool masses, uint64_t mine) {  // the cluster's histogram, and the sum of what each thread has
      mine = warp_sum64(mine);
      if (lane == 0) s.part2[warp] = mine;
      __syncthreads();
      if (tid < cl) {
        uint64_t v = 0;
        for (int w = 0; w < WARPS; ++w) v += s.part2[w];
        put64(peer(&s.xsum[rank], tid), v);
      }
      cl_sync();
      t = Totals<OWN>{};
      uint4 c[MAX_CL];  // all on their way at once
#pragma unroll
      for (uint32_t r = 0; r < MAX_CL; ++r) c[r] = r < cl ? get32x4(peer(&s.hist[OWN * tid], r)) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (uint32_t r = 0; r < MAX_CL; ++r) t.v[0] += c[r].x, t.v[1] += c[r].y, t.v[2] += c[r].z, t.v[3] += c[r].w;
      if (masses)
#pragma unroll
        for (int i = 0; i < OWN; ++i) t.v[i] <<= 24 - bin_scale(OWN * tid + i);
      mine = 0;
      for (uint32_t r = 0; r < cl; ++r) mine += s.xsum[r];
      run_totals(t, s.part);
      return mine;
    };
    auto clear = [&]() {  // the histogram, once every CTA has read it
      cl_sync();
      for (int i = tid; i < NB; i += THREADS) s.hist[i] = 0;
      __syncthreads();
    };
    if (by_k && k <= CAP) {
      // the bin of the k-th largest of the threads' maxima: k tokens at least are in it or above
      const int own_bin = bin_of(p.sc.x(own_max));
      if (own_bin < NB) atomicAdd(&s.hist[own_bin], 1u);
      gather(false, 0);
      find_bin(t, (uint64_t)k, s);
      const int bin = min((int)s.bin, NB - 1);  // else every token with a weight may stay
      each(p, [&](uint32_t i, float v) {
        const float x = p.sc.x(v);
        if (bin_of(x) > bin) return;
        atomicAdd(&s.own, 1u);
        uint32_t at;
        asm volatile("atom.relaxed.cluster.shared::cluster.add.u32 %0, [%1], 1;" : "=r"(at) : "r"(peer(&s.next[2], 0)) : "memory");
        if (at >= CAP) return;
        const float w = expf(x);
        put64(peer(&s.few.place[at], 0), place_of(v, base + i));
        put64(peer(&s.few.mass[at], 0), mass_of(w));
        put32(peer(&s.few.w[at], 0), __float_as_uint(w));
      });
      __syncthreads();
      if (tid < cl) put32(peer(&s.xcnt[0][rank], tid), s.own);
      cl_sync();
      uint32_t m_few = 0;  // (from here on no CTA touches another's memory: all but CTA 0 may leave)
      for (uint32_t r = 0; r < cl; ++r) m_few += s.xcnt[0][r];
      if (m_few <= CAP) {
        if (rank != 0) return;
        uint64_t me = 0, mine = 0, over_w = 0;
        uint32_t over = 0;
        if (tid < m_few) {
          me = s.few.place[tid];
          mine = s.few.mass[tid];
          for (uint32_t j = 0; j < m_few; ++j)
            if (s.few.place[j] > me) over += 1, over_w += s.few.mass[j];
        }
        auto block_sum = [&](uint64_t v) {
          v = warp_sum64(v);
          __syncthreads();
          if (lane == 0) s.part[warp] = v;
          __syncthreads();
          v = 0;
          for (int w = 0; w < WARPS; ++w) v += s.part[w];
          return v;
        };
        bool stays = tid < m_few && over < (uint32_t)k;
        if (by_p) {
          const uint64_t need = need_of(top_p, block_sum(stays ? mine : 0));
          stays = stays && over_w < need;
        }
        stays = stays && !(s.few.w[tid] < min_p);
        mine = stays ? mine : 0;
        const uint64_t total = block_sum(mine), target = target_of(total);
        if (tid < m_few) s.few.mass[tid] = mine;
        __syncthreads();
        if (mine == 0) return;
        uint64_t before = 0;  // of the tokens of lower index
        for (uint32_t j = 0; j < m_few; ++j)
          if ((s.few.place[j] & IDX_MASK) > (me & IDX_MASK)) before += s.few.mass[j];
        if (before <= target && target < before + mine) {
          a.out[row] = IDX_MASK - (uint32_t)(me & IDX_MASK);
          if (a.prob) a.prob[row] = (float)((double)mine / (double)total);
        }
        return;
      }
      clear();  // more than fit: as with a large k
    }
    uint32_t turn = 0;
    if (by_k) {
      each4(p, [&](uint32_t, const float (&v)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int b = bin_of(p.sc.x(v[j]));
          if (b < NB) atomicAdd(&s.hist[b], 1u);
        }
      });
      gather(false, 0);
      find_bin(t, (uint64_t)k, s);
      if (s.bin < NB) {  // else fewer than k tokens have a weight
        summed = find_border<false, ODD>(p, t, (uint64_t)k, turn, s);
        border = s.border;
        sum = s.inside;
      }
      if (by_p) clear();
    }
    if (by_p) {
      Mass all;
      each4(p, [&](uint32_t, const float (&v)[4]) {
        int b[4];
        uint32_t part[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float x = p.sc.x(v[j]), w = expf(x);
          b[j] = bin_of(x);
          all.add(w);
          const float scale = __uint_as_float((uint32_t)(127 + 16 + bin_scale(b[j])) << 23);
          part[j] = __float_as_uint(__fmaf_rd(w, scale, 8388608.f)) - 0x4B000000u;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (b[j] < NB) atomicAdd(&s.hist[b[j]], part[j]);
      });
      const uint64_t row_sum = gather(true, all.value());
      const uint64_t need = need_of(top_p, border ? sum : row_sum);
      find_bin(t, need, s);
      if (s.bin == NB) next_bin(t, NB, -1, s);  // the 16-bit sums fall short: the last bin with tokens
      summed = find_border<true, ODD>(p, t, need, turn, s);  // (top-p's border is not below top-k's)
      border = max(border, s.border);
    }
    cl_sync();  // xsum is read: it is written again below
  }
  // ---- weights that stay: each warp sums a run of the slice ----
  const float border_z = border ? value_of((uint32_t)(border >> IDX_BITS)) : -INFINITY;
  const uint32_t border_idx = IDX_MASK - ((uint32_t)border & IDX_MASK);
  auto kept = [&](uint32_t i, float v) -> float {
    const float w = p.sc.weight(v);
    return (v < border_z) | ((v == border_z) & (base + i > border_idx)) | (w < min_p) ? 0.f : w;
  };
  if (!summed) {
    Mass sum_m;
    each4_of_run(p, [&](uint32_t i, const float (&v)[4]) {
#pragma unroll
      for (int j = 0; j < 4; ++j) sum_m.add(kept(i + j, v[j]));
    });
    const uint64_t sum = warp_sum64(sum_m.value());
    if (lane == 0) s.kept[warp] = sum;
    __syncthreads();
  }
  const uint32_t run = p.run;
  if (tid < cl) {
    uint64_t v = 0;
    for (int w = 0; w < WARPS; ++w) v += s.kept[w];
    put64(peer(&s.xsum[rank], tid), v);
  }
  cl_sync();
  uint64_t total = 0, before = 0;
  for (uint32_t r = 0; r < cl; ++r) {
    if (r == rank) before = total;
    total += s.xsum[r];
  }
  const uint64_t target = target_of(total);
  if (target < before || target >= before + s.xsum[rank]) return;
  // the warp's run, split again over the warps, then the token
  uint32_t r = 0;
  while (before + s.kept[r] <= target) before += s.kept[r++];
  const uint32_t sub = (run / WARPS + 31) / 32 * 32;
  const uint32_t from = r * run, end = min(n, from + run);
  const uint32_t mine = min(end, from + warp * sub), mine_end = min(end, mine + sub);
  Mass mine_m;
  for (uint32_t i = mine + lane; i < mine_end; i += 32) mine_m.add(kept(i, z[i]));
  const uint64_t v = warp_sum64(mine_m.value());
  if (lane == 0) s.part2[warp] = v;
  __syncthreads();
  if (warp != 0) return;
  uint32_t g = 0;
  while (g + 1 < WARPS && before + s.part2[g] <= target) before += s.part2[g++];
  for (uint32_t i0 = from + g * sub; i0 < end; i0 += 32) {
    const uint32_t i = i0 + lane;
    const uint64_t w = i < end ? mass_of(kept(i, z[i])) : 0;
    const uint64_t to = before + warp_scan(w, lane);
    const uint32_t hit = __ballot_sync(0xffffffffu, to > target);
    if (hit) {
      if (lane == (uint32_t)__ffs(hit) - 1) {
        a.out[row] = base + i;
        if (a.prob) a.prob[row] = (float)((double)w / (double)total);
      }
      return;
    }
    before = __shfl_sync(0xffffffffu, to, 31);
  }
}

template <uint32_t DT>
__global__ void __launch_bounds__(THREADS, 2) sample_kernel(const __grid_constant__ SampleArgs a, uint32_t slice) {
  extern __shared__ __align__(16) uint8_t sample_smem[];
  cl_begun();
  pdl_trigger();
  pdl_wait();
  float* z = reinterpret_cast<float*>(sample_smem);
  Shared& s = *reinterpret_cast<Shared*>(sample_smem + sizeof(float) * slice);
  const uint32_t rank = cl_rank(), cl = cl_size(), row = blockIdx.x / cl;
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t base = min(a.n_vocab, rank * slice), n = min(a.n_vocab - base, slice);

  // ---- the slice, and its first maximum ----
  constexpr int PER = DT == DT_F32 ? 4 : 8;  // logits in 16 bytes
  const uint8_t* src = static_cast<const uint8_t*>(a.logits) + ((size_t)row * a.row_stride + base) * (16 / PER);
  float m = -INFINITY;
  auto take = [&](float v) {
    v = clean(v);
    m = fmaxf(m, v);
    return v;
  };
  uint32_t done = 0;
  if ((reinterpret_cast<uintptr_t>(src) & 15) == 0) {
    done = n / PER * PER;
#pragma unroll 4
    for (uint32_t i = tid; i < n / PER; i += THREADS) {
      const uint4 v = reinterpret_cast<const uint4*>(src)[i];
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < PER; e += 4) {
        float4 f;
        if constexpr (DT == DT_F32)
          f = make_float4(__uint_as_float(w[0]), __uint_as_float(w[1]), __uint_as_float(w[2]), __uint_as_float(w[3]));
        else if constexpr (DT == DT_F16) {
          const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&w[e / 2]));
          const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&w[e / 2 + 1]));
          f = make_float4(x.x, x.y, y.x, y.y);
        } else
          f = make_float4(__uint_as_float(w[e / 2] << 16), __uint_as_float(w[e / 2] & 0xFFFF0000u),
                          __uint_as_float(w[e / 2 + 1] << 16), __uint_as_float(w[e / 2 + 1] & 0xFFFF0000u));
        const uint32_t at = i * PER + e;
        f.x = take(f.x), f.y = take(f.y), f.z = take(f.z), f.w = take(f.w);
        *reinterpret_cast<float4*>(z + at) = f;
      }
    }
  }
  for (uint32_t i = done + tid; i < n; i += THREADS) z[i] = take(logit<DT>(src, i));
  if (tid < ((4 - n) & 3)) z[n + tid] = -INFINITY;  // whole fours
  const float own_max = m;
  m = warp_max(m);
  if (lane == 0) s.part32[warp] = __float_as_uint(m);
  for (int i = tid; i < NB; i += THREADS) s.hist[i] = 0;
  if (tid < 3) s.next[tid] = 0;
  if (tid == 0) s.own = 0;
  __syncthreads();
  cl_all_begun();
  if (tid < cl) {  // thread r tells CTA r
    for (int w = 0; w < WARPS; ++w) m = fmaxf(m, __uint_as_float(s.part32[w]));
    put32(peer(&s.xmax[rank], tid), __float_as_uint(m));
  }
  cl_sync();
  m = s.xmax[0];
  for (uint32_t r = 1; r < cl; ++r) m = fmaxf(m, s.xmax[r]);

  const float temp = a.temperature ? a.temperature[row] : 1.f;
  if (m == -INFINITY || !(temp > 0.f)) {  // nothing, or the first maximum: in the first CTA that has one
    uint32_t r = 0;
    while (r + 1 < cl && s.xmax[r] < m) ++r;
    if (rank != r) return;
    uint32_t first = 0xFFFFFFFFu;
    if (m > -INFINITY)
      for (uint32_t i = tid; i < n && first == 0xFFFFFFFFu; i += THREADS)
        if (z[i] == m) first = base + i;
    first = __reduce_min_sync(0xffffffffu, first);
    if (lane == 0) s.part32[warp] = first;
    __syncthreads();
    if (tid == 0) {
      for (int w = 0; w < WARPS; ++w) first = min(first, s.part32[w]);
      a.out[row] = first;
      if (a.prob) a.prob[row] = m > -INFINITY ? 1.f : 0.f;
    }
    return;
  }
  const float inv_t = __frcp_rn(temp);
  float min_p = a.min_p ? a.min_p[row] : 0.f;
  min_p = min_p > 0.f ? fminf(min_p, 1.f) : 0.f;  // the largest weight, 1, always stays
  if (m < INFINITY && inv_t < INFINITY && inv_t > 0.f)
    draw(a, Part<false>{z, n, base, rank, cl, slice / WARPS, {m, inv_t}, min_p}, row, own_max, s);
  else
    draw(a, Part<true>{z, n, base, rank, cl, slice / WARPS, {m, inv_t}, min_p}, row, own_max, s);
}

template <uint32_t DT>
cudaError_t sample_go(const SampleArgs& a, int num_sms, cudaStream_t st) {
  // As many CTAs a row as its slice needs, more while the rows leave SMs idle: down
  // to 8192 logits each, as below that the cluster's exchanges cost more than the
  // shorter slices save (a row of 32000, top-p: 14.1 us with 8 CTAs, 13.6 with 4,
  // 15.5 with 2; 128256: 22 with 4, 18.7 with 8, 21 with 16).
  uint32_t cl = 1;
  while (cl < MAX_CL && (a.n_vocab > cl * 16384 || (a.n_rows * cl * 2 <= (uint32_t)num_sms && a.n_vocab > cl * 8192))) cl *= 2;
  const uint32_t slice = ((a.n_vocab + cl - 1) / cl + 127) / 128 * 128;
  const size_t smem = sizeof(float) * slice + sizeof(Shared);
  return launch_early(sample_kernel<DT>, cl, dim3(a.n_rows * cl), dim3(THREADS), smem, st, a, slice);
}

}  // namespace

cudaError_t sample_init() {
  const int smem = sizeof(float) * MAX_SLICE + sizeof(Shared);
  const auto big = cudaFuncAttributeMaxDynamicSharedMemorySize;
  cudaError_t e = cudaFuncSetAttribute(sample_kernel<DT_F32>, big, smem);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(sample_kernel<DT_F16>, big, smem);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(sample_kernel<DT_BF16>, big, smem);
  return e;
}

cudaError_t sample_launch(const SampleArgs& a, int num_sms, cudaStream_t st) {
  if (a.dtype == DT_F32) return sample_go<DT_F32>(a, num_sms, st);
  return a.dtype == DT_F16 ? sample_go<DT_F16>(a, num_sms, st) : sample_go<DT_BF16>(a, num_sms, st);
}

}  // namespace shk
