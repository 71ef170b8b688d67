// pages_attn.cu -- attention of a batch's rows over the paged 8-bit K/V pools.
//
// A row reads its request's keys and values once and does 4 hd flops per
// position and query head with them: bound by memory.  So the work is laid out
// by bytes.  An item is the positions that one row reads for up to 8 or 16 query
// heads of one KV head, or that several rows of one request read together, where
// their heads fit; items are cut into units of 128 positions, all units of all items are
// put in one line, and each CTA takes an equal part of it, whatever the
// lengths.  A CTA's part may begin and end inside an item: its (max, sum,
// output) for that piece goes to the workspace and a second, small kernel joins
// the pieces.  Lengths are read on the device only.
//
// Inside a unit each of the 4 warps takes 32 positions: two times 16, which lie
// in one block each and so share one scale of K and one of V.  A warp copies its
// own steps (cp.async: the next V while this step is computed, the next K from
// the moment this one has been multiplied), so no warp waits for another.
//
//   S = q K^T by mma.m16n8k16 in f16: the bytes of both pool types are exact in
//   f16, q is scaled by a power of two and split into two f16 parts (22 bits):
//   head g's high part is row g of the A operand and its low part row g + 8, so
//   both go through one instruction and their sums meet in one lane.
//   O^T = V^T P^T, the weights in two f16 parts as well, one instruction each:
//   lane (g, t) has the scores of head g that its B fragment asks for, and a
//   head's outputs take half the registers that they would as rows.  Additions to
//   an accumulator are cut off by the tensor core, always towards 0: each 16
//   positions begin at 0, and their sum is added to the outputs with rounding (in
//   one chain, outputs over 65536 positions came out 5e-6 too small, now 3e-7; it
//   costs 0.5 us on one row, 3 to 4% on a batch of 64 heads over 8 of 128).
//
// The softmax runs with two maxima per head: m of the scores for the sum, and M
// of score + E, E the exponent of the block's V scale (V = 2^E f byte), for the
// weights 2^(s - M + E) f of the output, so that neither overflows and the largest
// never underflows.  A weight's two f16 parts hold it to 2^-22 of itself or, where
// it is small, to 2^-39 of the row's largest: a block whose V scale is 2^-30 of
// another's is left with 9 bits where that one holds zeros, and with none at
// 2^-40.  A third part would add half of the second product's instructions to all
// calls, for scales that K/V of one model and head do not have.
//
// Measured (64 heads over 8 of 128): 16 requests of 30k to 65k positions, e4m3,
// 313 to 316 us, 5.2 TB/s; 32 of 1 to 8192, i8, 71 us, 3.9 TB/s, of which the join
// is 9; one of 8192 16.9 us, one of 777 (32 heads) 11.5 us, both chains of loads
// that wait on one another.  64 x 4 rows of 100 to 2000 positions (32 heads over 4
// of 64) 41 us: instructions, 800 a warp's step of 32 positions for 16 slots at
// 0.54 a cycle.  Five and six CTAs an SM there: 47 and 52 us.  A prompt's rows have
// no tile of their own, K/V are read and converted again for every 16 / G of them:
// 2048 rows of 32 heads over 8 of 128 on their own causal positions 366 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "common.cuh"
#include "pages.cuh"

namespace shk {
namespace {

constexpr int WARPS = 4;
constexpr int THREADS = 32 * WARPS;
constexpr int HEADS = 8;        // slots (a row's query head each) of a set: the MMA's rows g
constexpr int SUB = 16;         // positions under one pair of scales
constexpr int STEP = 2 * SUB;   // positions of a warp's step
constexpr int UNIT = STEP * WARPS;
constexpr int CTAS_PER_SM = 4;  // 128 registers a thread (two sets: 3, 168)
constexpr int MAX_CTAS = 640;   // 4 x the SMs of a B200 (148), rounded up
// What an item costs besides its positions, in units (32 ragged rows with 0, 1, 2:
// 78, 66, 66 us; 64 x 4: 62, 47, 45).
constexpr int ITEM_UNITS = 2;
constexpr int MIN_UNITS = 2;    // a CTA's part: shorter ones cost more in joining than they save

template <int HD, int SETS>
struct Lay {
  static constexpr int NP = HD / 64;            // 16-byte pieces of a K row per lane
  static constexpr int NW = HD / 32;            // words of a V row per lane
  static constexpr int STEPS = HD / 16;         // k-steps of q K^T
  static constexpr int HALF = SUB * HD;         // bytes of 16 positions of K or V
  static constexpr int KBUF = 2 * HALF;         // a step's K; V has two such buffers behind it
  static constexpr int RING = 3 * KBUF;         // per warp
  static constexpr int CTAS = SETS == 2 ? 3 : CTAS_PER_SM;
  static constexpr int QF = STEPS * 32 * 16;    // a set's q fragments
  static constexpr int HROW = HD + 4;           // floats of a head's outputs in shared memory, padded
  static constexpr int BYTES = WARPS * RING + SETS * QF;
  static constexpr int REC = HEADS * (HD + 3);  // floats of a piece's record of one set: O, m, M, l
  static_assert(SETS * HEADS * HROW * 4 <= RING, "a warp's output fits its ring");
};

struct Header {  // the item that begins in a CTA's part and ends in a later one's
  int32_t row, item, last;
  int32_t slot_rows;  // which of the CTA's two records, and twice the item's rows
};

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

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 2^d / l in two factors, the second a power of two: 2^d for a V scale near the
// smallest floats is below what ex2 gives, and what the output is not.
__device__ __forceinline__ float2 out_factor(float d, float l) {
  const bool low = d < -64.f;
  return make_float2(l == 0.f ? 0.f : ex2(low ? d + 64.f : d) / l, low ? 0x1p-64f : 1.f);
}

__device__ __forceinline__ void copy(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_or_zero(uint32_t dst, const void* src, bool take) {
  const uint32_t n = take ? 16 : 0;  // 0: reads nothing, writes zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

// The low and the high two bytes of a word as f16 pairs, exactly.
template <uint32_t TYPE>
__device__ __forceinline__ void to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (TYPE == PAGES_I8) {
    // byte + 128 under the exponent of 1024, less 1152
    const uint32_t x = w ^ 0x80808080u;
    uint32_t a = __byte_perm(x, 0x64646464u, 0x4140), b = __byte_perm(x, 0x64646464u, 0x4342);
    const __half2 c = __half2half2(__ushort_as_half(0x6480));
    const __half2 ra = __hsub2(*reinterpret_cast<__half2*>(&a), c), rb = __hsub2(*reinterpret_cast<__half2*>(&b), c);
    lo = *reinterpret_cast<const uint32_t*>(&ra);
    hi = *reinterpret_cast<const uint32_t*>(&rb);
  } else {
    asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n cvt.rn.f16x2.e4m3x2 %0, l;\n cvt.rn.f16x2.e4m3x2 %1, h;\n}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  }
}

// x = hi + lo in two f16 parts, for two values at once.
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}

struct Row {
  int32_t z;
  uint32_t len, units, rows;  // of the item: the longest row's positions, units of them, and its rows
};

// Positions of row r of request z.
__device__ __forceinline__ uint32_t row_len(const PagesAttnArgs& a, int32_t z, int32_t p) {
  if ((uint32_t)z >= a.n_seq || (p >= 0 && (uint64_t)p >= ((uint64_t)a.stride << a.pool.block_shift))) {
    if (z >= 0) set_error(a.err, DERR_BAD_POS);
    return 0;
  }
  return z >= 0 && p >= 0 ? (uint32_t)p + 1 : 0;
}

// The item that begins at row r.  MANY: up to a.window rows of one request, one
// behind the other, that begin at a multiple of a.window or where the request
// changes; other rows have no units.  A padding row has none either; live rows
// have at least one, so that rows which see nothing are written (zeros).
template <bool MANY>
__device__ __forceinline__ Row row_of(const PagesAttnArgs& a, uint32_t r) {
  Row w{a.row_seq ? a.row_seq[r] : (int32_t)r, 0, 0, 1};
  w.len = row_len(a, w.z, a.row_pos[r]);
  bool leads = true;
  if (MANY && a.window > 1) {
    const uint32_t in = r % a.window, behind = min(a.window - in, a.n_rows - r);
    leads = in == 0 || a.row_seq[r - 1] != w.z;
    bool same = true;
#pragma unroll 4
    for (uint32_t i = 1; i < behind; ++i) {  // (loads that do not wait on one another)
      const int32_t z = a.row_seq[r + i], p = a.row_pos[r + i];
      same = same && z == w.z;
      if (same) w.len = max(w.len, row_len(a, z, p)), ++w.rows;
    }
  }
  if (w.z >= 0 && leads) w.units = w.len ? (w.len + UNIT - 1) / UNIT : 1;
  return w;
}

struct Sums {
  uint64_t warp[WARPS];
  uint64_t base;
  Row at;
  uint32_t row;
};

// The first row from `row` on that is somebody's, n where there is none: 128 rows
// at a time, by each warp for itself, as a request that was refused whole may leave
// thousands of padding rows between two items (64 rows with 4000 behind the first
// half: 1.47 ms one after the other, 52 us so).
__device__ __forceinline__ uint32_t live_row(const int32_t* row_seq, uint32_t row, uint32_t n) {
  const uint32_t lane = threadIdx.x & 31;
  for (; row < n; row += 128) {
    uint32_t live[4];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      const uint32_t r = row + 32 * i + lane;
      live[i] = __ballot_sync(0xffffffffu, r < n && row_seq[r] >= 0);
    }
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
      if (live[i]) return row + 32 * i + __ffs(live[i]) - 1;
  }
  return n;
}

// Row of a request's position p0 in a pool.
__device__ __forceinline__ size_t first_row(const PagesAttnArgs& a, int32_t id, uint32_t kvh, uint32_t p0) {
  const uint32_t bs = a.pool.block_shift;
  return (((size_t)id * a.pool.n_kv + kvh) << bs) + (p0 & ((1u << bs) - 1));
}

// 16 rows of K or V go to shared memory as they lie, 512 bytes by an
// instruction: quarter warps that reach into several lines halve the rate (V's
// fragments fetched directly, 16 bytes of 4 rows each: 4.4 against 6.0 TB/s).
// 16-byte piece p of 128-byte line r is stored at piece p ^ swizzle(r), which
// spreads the pieces that 8 lanes read at a time over all banks: K's are pieces
// t (+ 4) of rows 2q and 2q + 1, V's pieces g of rows 2t (head_dim 64: two rows
// a line, V's are the halves of piece g / 2 of line t).
template <int HD, bool V>
__device__ __forceinline__ constexpr uint32_t swizzle(uint32_t line) {
  return HD == 64 ? (line & 3) * 2 : V ? line & 6 : (line & 1) * 4;
}
template <int HD, bool V>
__device__ __forceinline__ uint32_t at_piece(uint32_t line, uint32_t piece) {
  return line * 128 + ((piece ^ swizzle<HD, V>(line)) << 4);
}
// Only `rows` of V's positions are the row's.  What lies behind them gets weight
// 0; e4m3 values become zeros here too, as a NaN byte would outlive that.
template <int HD, uint32_t TYPE, bool V>
__device__ __forceinline__ void fetch(const uint8_t* row0, uint32_t dst, uint32_t rows, uint32_t lane) {
  const uint8_t* src = row0 + 16 * lane;
#pragma unroll
  for (int j = 0; j < SUB * HD / 512; ++j) {
    const uint32_t to = dst + at_piece<HD, V>(4 * j + (lane >> 3), lane & 7);
    if constexpr (V && TYPE == PAGES_E4M3)
      copy_or_zero(to, src + 512 * j, (512 * j + 16 * lane) / HD < rows);
    else
      copy(to, src + 512 * j);
  }
}

template <int HD, uint32_t TYPE, int SETS, bool MANY>
__global__ void __launch_bounds__(THREADS, Lay<HD, SETS>::CTAS) attend_kernel(const __grid_constant__ PagesAttnArgs a) {
  using L = Lay<HD, SETS>;
  constexpr uint32_t SLOTS = SETS * HEADS;
  extern __shared__ __align__(16) uint8_t att_smem[];
  __shared__ Sums sums;
  __shared__ int32_t qmax[SLOTS];
  __shared__ float stat[WARPS][SLOTS][3];
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const uint32_t c = blockIdx.x, bs = a.pool.block_shift, n_kv = a.pool.n_kv, G = a.group;
  const uint32_t nsub = a.subs, NI = n_kv * nsub;
  Header* headers = static_cast<Header*>(a.ws);
  float* records = reinterpret_cast<float*>(static_cast<uint8_t*>(a.ws) + MAX_CTAS * sizeof(Header));
  pdl_trigger();
  pdl_wait();

  // ---- this CTA's part of the line of units ----
  if (tid == 0) headers[c] = Header{-1, 0, 0, 0};
  // Its first unit's row: each thread sums what its share of the rows cost, the
  // sums are summed over the CTA, and the share that has the unit is dealt out
  // again until it is one row (65535 rows: three times).
  auto cost = [](const Row& r) -> uint32_t { return r.units ? r.units + ITEM_UNITS : 0; };
  Row rw{-1, 0, 0, 0};
  uint64_t s = 0, end = 0, U = 0, before = 0;
  uint32_t C = 0, row = 0;
  for (uint32_t left = a.n_rows;;) {
    const uint32_t per = (left + THREADS - 1) / THREADS;
    const uint32_t r0 = row + tid * per, r1 = min(row + left, r0 + per);
    uint64_t mine = 0, upto;
#pragma unroll 2
    for (uint32_t r = r0; r < r1; ++r) {
      rw = row_of<MANY>(a, r);
      mine += cost(rw);
    }
    upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t u = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= (uint32_t)o) upto += u;
    }
    if (lane == 31) sums.warp[warp] = upto;
    __syncthreads();
    uint64_t total = 0;
#pragma unroll
    for (uint32_t w = 0; w < WARPS; ++w) {
      if (w < warp) upto += sums.warp[w];
      total += sums.warp[w];
    }
    if (left == a.n_rows) {
      U = NI * total;
      const uint64_t want = U / MIN_UNITS;
      C = want < 1 ? 1 : want < gridDim.x ? (uint32_t)want : gridDim.x;
      if (c >= C || U == 0) return;
      s = c * U / C;
      end = (c + 1) * U / C;
    }
    upto += before;
    if (mine && s >= NI * (upto - mine) && s < NI * upto) {
      sums.row = r0;
      sums.base = upto - mine;
      sums.at = rw;
    }
    __syncthreads();
    row = sums.row;
    before = sums.base;
    if (per == 1) break;
    left = min(per, a.n_rows - row);
  }
  const uint64_t first = s;
  uint64_t base = NI * before;
  rw = sums.at;

  const uint32_t ring = smem_u32(att_smem) + warp * L::RING;
  uint4* qf = reinterpret_cast<uint4*>(att_smem + WARPS * L::RING);

  // where this lane's fragments lie: pieces of K's row g, of V's row 2t (rows 8 further on are swizzled alike)
  uint32_t k_at[L::NP];
#pragma unroll
  for (int i = 0; i < L::NP; ++i)
    k_at[i] = HD == 128 ? at_piece<HD, false>(g, 4 * i + t) : at_piece<HD, false>(g >> 1, 4 * (g & 1) + t);
  const uint32_t v_at = HD == 128 ? at_piece<HD, true>(2 * t, g) : at_piece<HD, true>(t, g >> 1) + 8 * (g & 1);

  while (s < end) {
    // the item, and this piece of it: units ua .. ub - 1 (its first ITEM_UNITS places in the line stand for its fixed cost)
    const uint32_t span = rw.units + ITEM_UNITS;
    const uint32_t item = (uint32_t)((s - base) / span);
    const uint32_t va = (uint32_t)(s - base - (uint64_t)item * span);
    const uint32_t vb = (uint32_t)min((uint64_t)span, va + (end - s));
    const uint32_t ua = va > ITEM_UNITS ? va - ITEM_UNITS : 0, ub = vb > ITEM_UNITS ? vb - ITEM_UNITS : 0;
    const uint64_t start = s;
    s += vb - va;
    const bool next_row = s < end && s == base + (uint64_t)NI * span;
    if (ub > 0) {
      const uint32_t kvh = item / nsub, sub = item % nsub;
      // slot x of the item: head sub * SLOTS + x of its row, or head x % G of row x / G
      const uint32_t slots = MANY && nsub == 1 ? rw.rows * G : min(G - sub * SLOTS, SLOTS);
      auto slot_in = [&](uint32_t x) { return MANY && nsub == 1 ? x * a.inv_group >> 16 : 0; };
      auto slot_row = [&](uint32_t x) { return row + slot_in(x); };
      auto slot_dim = [&](uint32_t x) { return (size_t)((sub * SLOTS + x - slot_in(x) * G) * n_kv + kvh) * HD; };
      const int32_t* table = a.table + (size_t)rw.z * a.stride;  // z is in range where len > 0

      // q of this lane's fragments: k-step st covers, for lane (g, t), the 4 dims of word st % 4 of its piece st / 4
      float q[SETS][L::STEPS / WARPS][4];
      uint32_t len[SETS];  // of the rows of this lane's slots
#pragma unroll
      for (int x = 0; x < SETS; ++x) {
        const uint32_t slot = HEADS * x + g;
        len[x] = rw.len;
        if (MANY && rw.rows > 1 && slot < slots) len[x] = row_len(a, rw.z, a.row_pos[slot_row(slot)]);
#pragma unroll
        for (int i = 0; i < L::STEPS / WARPS; ++i) {
          const uint32_t st = warp + WARPS * i, d = 64 * (st >> 2) + 16 * t + 4 * (st & 3);
          const size_t at = slot < slots ? slot_row(slot) * a.q_stride + slot_dim(slot) + d : 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) q[x][i][e] = slot < slots ? load_dt(a.q, at + e, a.dtype) : 0.f;
        }
      }

      // ---- this warp's steps: units ua .. ub - 1, positions UNIT u + STEP warp ----
      const uint32_t steps = (rw.len + STEP - 1) / STEP;
      const uint32_t last_u = steps > warp ? (steps - warp + WARPS - 1) / WARPS : 0;  // units with a step of this warp
      const int32_t n = (int32_t)min(ub, last_u) - (int32_t)ua;
      auto place = [&](int32_t i, int half) { return (ua + (uint32_t)i) * UNIT + warp * STEP + half * SUB; };
      // a table entry is checked a step after it is read, when it has arrived
      auto entry = [&](int32_t i, int half) -> int32_t {
        const uint32_t p = place(i, half);
        return i < n && p < rw.len ? table[p >> bs] : -1;
      };
      auto checked = [&](int32_t i, int2 id) {
        if ((uint32_t)id.x >= a.pool.n_blocks || (uint32_t)id.y >= a.pool.n_blocks) {
          if (i < n && ((uint32_t)id.x >= a.pool.n_blocks || place(i, 1) < rw.len)) set_error(a.err, DERR_BAD_POS);
          if ((uint32_t)id.x >= a.pool.n_blocks) id.x = -1;
          if ((uint32_t)id.y >= a.pool.n_blocks) id.y = -1;
        }
        return id;
      };
      auto issue_k = [&](int32_t i, int2 id) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if ((h ? id.y : id.x) >= 0)
            fetch<HD, TYPE, false>(a.pool.k + first_row(a, h ? id.y : id.x, kvh, place(i, h)) * HD, ring + h * L::HALF, 0,
                                   lane);
        copy_commit();
      };
      auto issue_v = [&](int32_t i, int2 id) {
        const uint32_t dst = ring + L::KBUF + (i & 1) * L::KBUF;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if ((h ? id.y : id.x) >= 0)
            fetch<HD, TYPE, true>(a.pool.v + first_row(a, h ? id.y : id.x, kvh, place(i, h)) * HD, dst + h * L::HALF,
                                  rw.len - place(i, h), lane);
          else if (TYPE == PAGES_E4M3 && i < n)
            fetch<HD, TYPE, true>(a.pool.v, dst + h * L::HALF, 0, lane);
        }
        copy_commit();
      };
      auto scales = [&](int32_t id) {
        const size_t at = (size_t)(id < 0 ? 0 : id) * n_kv + kvh;
        return make_float2(a.pool.ks[at], a.pool.vs[at]);
      };
      float m[SETS], M[SETS], l[SETS], o[SETS][HD / 16][4];
#pragma unroll
      for (int x = 0; x < SETS; ++x) {
        m[x] = M[x] = -INFINITY, l[x] = 0.f;
#pragma unroll
        for (int j = 0; j < HD / 16; ++j) o[x][j][0] = o[x][j][1] = o[x][j][2] = o[x][j][3] = 0.f;
      }
      int2 id0{-1, -1}, id1{-1, -1};
      float2 sx{}, sy{};
      if (n > 0) {  // the first copies are on their way before q is needed
        id0 = int2{entry(0, 0), entry(0, 1)};
        id1 = int2{entry(1, 0), entry(1, 1)};
        id0 = checked(0, id0);
        issue_k(0, id0);
        issue_v(0, id0);
        sx = scales(id0.x), sy = scales(id0.y);
      }

      // q scaled by a power of two so that the largest magnitude of a head is in [2^14, 2^15)
      if (tid < SLOTS) qmax[tid] = 0;
      __syncthreads();
#pragma unroll
      for (int x = 0; x < SETS; ++x) {
        float big = 0.f;
#pragma unroll
        for (int i = 0; i < L::STEPS / WARPS; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) big = fmaxf(big, fabsf(q[x][i][e]));
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
        if (t == 0) atomicMax(&qmax[HEADS * x + g], __float_as_int(big));
      }
      __syncthreads();
      float qscale[SETS];
#pragma unroll
      for (int x = 0; x < SETS; ++x) {
        const float top = __int_as_float(qmax[HEADS * x + g]);
        int ex = 0;
        if (top > 0.f && top < INFINITY) ex = min(14 - ilogbf(top), 126);
        const float up = ldexpf(1.f, ex);
        qscale[x] = a.scale * 1.4426950408889634f * ldexpf(1.f, -ex);
#pragma unroll
        for (int i = 0; i < L::STEPS / WARPS; ++i) {
          uint4 f;
          split2(q[x][i][0] * up, q[x][i][1] * up, f.x, f.y);
          split2(q[x][i][2] * up, q[x][i][3] * up, f.z, f.w);
          qf[(x * L::STEPS + warp + WARPS * i) * 32 + lane] = f;
        }
      }
      __syncthreads();

      for (int32_t i = 0; i < n; ++i) {
        id1 = checked(i + 1, id1);
        issue_v(i + 1, id1);
        const float2 nx = scales(id1.x), ny = scales(id1.y);
        const int2 id2{entry(i + 2, 0), entry(i + 2, 1)};
        copy_wait<1>();  // this step's K and V; the next V may be on its way
        __syncwarp();
        const uint8_t* here = att_smem + warp * L::RING;
        float acc[SETS][4][4] = {};
#pragma unroll
        for (int pi = 0; pi < L::NP; ++pi) {
          uint32_t kw[4][4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint4 x = *reinterpret_cast<const uint4*>(here + (j >> 1) * L::HALF + k_at[pi] + (j & 1) * 8 * HD);
            kw[j][0] = x.x, kw[j][1] = x.y, kw[j][2] = x.z, kw[j][3] = x.w;
          }
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint4 qa[SETS];
#pragma unroll
            for (int x = 0; x < SETS; ++x) qa[x] = qf[(x * L::STEPS + 4 * pi + w) * 32 + lane];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              uint32_t b0, b1;
              to_f16<TYPE>(kw[j][w], b0, b1);
#pragma unroll
              for (int x = 0; x < SETS; ++x) mma_f16(acc[x][j], qa[x], b0, b1);
            }
          }
        }
        __syncwarp();
        issue_k(i + 1, id1);  // this step's K has been multiplied
        // a V scale is 2^E * vf, vf below 2 (also for a scale of 0, an infinite one or NaN)
        float E[2], vf[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float vs = (h ? id0.y : id0.x) < 0 ? 0.f : h ? sy.y : sx.y;
          const int e8 = max(1, min(254, (int)((__float_as_uint(vs) >> 23) & 255)));
          E[h] = (float)(e8 - 127);
          vf[h] = e8 == 254 ? vs * 0x1p-127f : vs * __int_as_float((254 - e8) << 23);
        }
        // scores in powers of two; lane (g, t) holds slot g at positions 8 j + 2t, 8 j + 2t + 1
        float sv[SETS][4][2], m0[SETS], M0[SETS];
#pragma unroll
        for (int x = 0; x < SETS; ++x) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float f = (j < 2 ? sx.x : sy.x) * qscale[x];
            sv[x][j][0] = (acc[x][j][0] + acc[x][j][2]) * f;
            sv[x][j][1] = (acc[x][j][1] + acc[x][j][3]) * f;
          }
          const int32_t left = (int32_t)(len[x] - place(i, 0));
          if (left < STEP || id0.x < 0 || id0.y < 0) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                if ((int32_t)(8 * j + 2 * t + e) >= left || (j < 2 ? id0.x : id0.y) < 0) sv[x][j][e] = -INFINITY;
          }
          const float c0 = fmaxf(fmaxf(sv[x][0][0], sv[x][0][1]), fmaxf(sv[x][1][0], sv[x][1][1]));
          const float c1 = fmaxf(fmaxf(sv[x][2][0], sv[x][2][1]), fmaxf(sv[x][3][0], sv[x][3][1]));
          float mn = fmaxf(c0, c1), Mn = fmaxf(c0 + E[0], c1 + E[1]);
#pragma unroll
          for (int y = 1; y <= 2; y <<= 1) {
            mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, y));
            Mn = fmaxf(Mn, __shfl_xor_sync(0xffffffffu, Mn, y));
          }
          mn = fmaxf(m[x], mn), Mn = fmaxf(M[x], Mn);
          if (__any_sync(0xffffffffu, mn > m[x] || Mn > M[x])) {
            const float al = m[x] == mn ? 1.f : ex2(m[x] - mn), aM = M[x] == Mn ? 1.f : ex2(M[x] - Mn);
            l[x] *= al;
            // the outputs of lane (g, t) are slots 2t and 2t + 1
            const float a0 = __shfl_sync(0xffffffffu, aM, 8 * t), a1 = __shfl_sync(0xffffffffu, aM, 8 * t + 4);
#pragma unroll
            for (int j = 0; j < HD / 16; ++j) o[x][j][0] *= a0, o[x][j][1] *= a1, o[x][j][2] *= a0, o[x][j][3] *= a1;
            m[x] = mn;
            M[x] = Mn;
          }
          // a step without positions may leave the maxima at -inf: its weights are 0
          m0[x] = m[x] == -INFINITY ? 0.f : m[x], M0[x] = M[x] == -INFINITY ? 0.f : M[x];
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t hi0[SETS], lo0[SETS], hi1[SETS], lo1[SETS];
          const float vo = E[h] + 14.f;  // weights up to 2^15: their low parts stay normal f16
#pragma unroll
          for (int x = 0; x < SETS; ++x) {
            float wt[4];
            // (an infinite scale of positions that the slot does not see)
            const float f = (int32_t)(len[x] - place(i, h)) <= 0 ? 0.f : vf[h];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float y = sv[x][2 * h + (e >> 1)][e & 1];
              l[x] += ex2(y - m0[x]);
              wt[e] = ex2((y - M0[x]) + vo) * f;
            }
            split2(wt[0], wt[1], hi0[x], lo0[x]);
            split2(wt[2], wt[3], hi1[x], lo1[x]);
          }
          const uint8_t* vp = here + L::KBUF + (i & 1) * L::KBUF + h * L::HALF;
          uint32_t vr[4][L::NW];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if constexpr (HD == 128) {
              const uint4 x = *reinterpret_cast<const uint4*>(vp + v_at + ((r & 1) + 8 * (r >> 1)) * HD);
              vr[r][0] = x.x, vr[r][1] = x.y, vr[r][2] = x.z, vr[r][3] = x.w;
            } else {
              const uint2 x = *reinterpret_cast<const uint2*>(vp + (v_at ^ ((r & 1) * 64)) + 8 * (r >> 1) * HD);
              vr[r][0] = x.x, vr[r][1] = x.y;
            }
          }
          // tile j: rows g and g + 8 are dims 2j and 2j + 1 of the lane's run
#pragma unroll
          for (int w = 0; w < L::NW; ++w)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              uint4 va;
              to_f16<TYPE>(__byte_perm(vr[0][w], vr[1][w], e ? 0x7362 : 0x5140), va.x, va.y);
              to_f16<TYPE>(__byte_perm(vr[2][w], vr[3][w], e ? 0x7362 : 0x5140), va.z, va.w);
#pragma unroll
              for (int x = 0; x < SETS; ++x) {
                float s16[4] = {};
                mma_f16(s16, va, lo0[x], lo1[x]);
                mma_f16(s16, va, hi0[x], hi1[x]);
                float(&to)[4] = o[x][2 * w + e];
#pragma unroll
                for (int k = 0; k < 4; k += 2) {
                  const float2 sum = __fadd2_rn(make_float2(to[k], to[k + 1]), make_float2(s16[k], s16[k + 1]));
                  to[k] = sum.x, to[k + 1] = sum.y;
                }
              }
            }
        }
        id0 = id1, id1 = id2;
        sx = nx, sy = ny;
        __syncwarp();  // the next V goes where this one was
      }
      copy_wait<0>();

      // ---- the warps' outputs meet in shared memory (each in its own ring) ----
      const bool whole = ua == 0 && ub == rw.units;
      const uint32_t mine = start == first ? 0 : 1;
      if (!whole && tid == 0 && ua == 0)
        headers[c] = Header{(int32_t)row, (int32_t)item, (int32_t)(((base + (uint64_t)(item + 1) * span) * C - 1) / U),
                            (int32_t)(mine + 2 * (MANY ? rw.rows : 1))};
      __syncwarp();
#pragma unroll
      for (int x = 0; x < SETS; ++x) {
        l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
        l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
        // lane (g, t): slots 2t and 2t + 1, the HD / 8 dims from HD / 8 g
        float* mo = reinterpret_cast<float*>(att_smem + warp * L::RING) + (HEADS * x + 2 * t) * L::HROW + g * (HD / 8);
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int j = 0; j < HD / 16; j += 2)
            *reinterpret_cast<float4*>(mo + r * L::HROW + 2 * j) =
                make_float4(o[x][j][r], o[x][j][r + 2], o[x][j + 1][r], o[x][j + 1][r + 2]);
        float* st = stat[warp][HEADS * x + g];
        if (t == 0) st[0] = m[x], st[1] = M[x], st[2] = l[x];
      }
      __syncthreads();
#pragma unroll
      for (int x = 0; x < SETS; ++x) {
        float* rec = records + ((size_t)(2 * c + mine) * SETS + x) * L::REC;
        constexpr int PER = HD * HEADS / THREADS;  // consecutive dims of one slot per thread
        const uint32_t h = tid / (HD / PER), d = (tid % (HD / PER)) * PER;
        float mm = -INFINITY, MM = -INFINITY, ll = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w)
          mm = fmaxf(mm, stat[w][HEADS * x + h][0]), MM = fmaxf(MM, stat[w][HEADS * x + h][1]);
        float out[PER] = {};
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
          const float lw = stat[w][HEADS * x + h][2];
          if (lw == 0.f) continue;  // a warp without positions
          ll += lw * ex2(stat[w][HEADS * x + h][0] - mm);
          const float f = ex2(stat[w][HEADS * x + h][1] - MM);
          const float* src = reinterpret_cast<const float*>(att_smem + w * L::RING) + (HEADS * x + h) * L::HROW + d;
#pragma unroll
          for (int e = 0; e < PER; ++e) out[e] += src[e] * f;
        }
        if (whole) {
          const uint32_t slot = HEADS * x + h;
          if (slot < slots) {
            // MM - mm is at most the largest exponent of a scale
            const float2 f = out_factor(MM - mm - 14.f, ll);
            const size_t at = slot_row(slot) * a.out_stride + slot_dim(slot) + d;
#pragma unroll
            for (int e = 0; e < PER; ++e) store_dt(a.out, at + e, a.dtype, ll == 0.f ? 0.f : out[e] * f.x * f.y);
          }
        } else {
#pragma unroll
          for (int e = 0; e < PER; e += 4)
            *reinterpret_cast<float4*>(rec + h * HD + d + e) = make_float4(out[e], out[e + 1], out[e + 2], out[e + 3]);
          if (d == 0) rec[HEADS * HD + h] = mm, rec[HEADS * (HD + 1) + h] = MM, rec[HEADS * (HD + 2) + h] = ll;
        }
      }
      __syncthreads();  // the rings and stat are free again
    }
    if (next_row) {
      base = s;
      row += MANY ? rw.rows : 1;
      if (row < a.n_rows && a.row_seq && a.row_seq[row] < 0) row = live_row(a.row_seq, row + 1, a.n_rows);
      if (row >= a.n_rows) return;  // (positions that were changed during the call)
      rw = row_of<MANY>(a, row);
    }
  }
}

// Joins the pieces of set blockIdx.y of the item that begins in CTA blockIdx.x's
// part.  Its time is that of loads that wait on one another, so there are two such
// waits: for the header, then for the pieces' (max, sum) together with their outputs (4 dims a
// thread, the pieces dealt to the thread groups, the first HELD of a group held in
// registers meanwhile).
template <int HD, int SETS, int THREADS_J>
__global__ void __launch_bounds__(THREADS_J) attend_join_kernel(const __grid_constant__ PagesAttnArgs a) {
  using L = Lay<HD, SETS>;
  constexpr uint32_t SLOTS = SETS * HEADS;
  constexpr uint32_t PER_GROUP = HEADS * HD / 4, GROUPS = THREADS_J / PER_GROUP;
  // (8 in a small block of two groups: 64 x 4 rows 42.3 us, 4: 41.0)
  constexpr uint32_t HELD = THREADS_J == 256 ? 8 / GROUPS : 8;
  __shared__ float weight[HEADS][MAX_CTAS + 1];  // of a piece's outputs
  __shared__ float2 fin[HEADS];
  __shared__ float4 sum[THREADS_J];
  const uint32_t c = blockIdx.x, tid = threadIdx.x, lane = tid & 31;
  pdl_wait();
  const Header hd = static_cast<const Header*>(a.ws)[c];
  if (hd.row < 0) return;
  const float* records = reinterpret_cast<const float*>(static_cast<const uint8_t*>(a.ws) + MAX_CTAS * sizeof(Header));
  const uint32_t n_kv = a.pool.n_kv, G = a.group, nsub = a.subs;
  const uint32_t kvh = hd.item / nsub, sub = hd.item % nsub, n = (uint32_t)hd.last - c + 1;
  auto rec = [&](uint32_t i) { return records + ((size_t)(2 * (c + i) + (i == 0 ? hd.slot_rows & 1 : 0)) * SETS + blockIdx.y) * L::REC; };
  const uint32_t grp = tid / PER_GROUP, e = tid % PER_GROUP, h = e / (HD / 4);
  float4 x[HELD];
#pragma unroll
  for (uint32_t k = 0; k < HELD; ++k)
    if (grp + k * GROUPS < n) x[k] = reinterpret_cast<const float4*>(rec(grp + k * GROUPS))[e];
  if (tid < 32 * HEADS) {  // warp h: head h
    const uint32_t hh = tid >> 5;
    float m = -INFINITY, M = -INFINITY, l = 0.f;
    for (uint32_t i = lane; i < n; i += 32) {  // running maxima, and the sum that goes with them
      const float* r = rec(i) + HEADS * HD + hh;
      const float rm = r[0], rM = r[HEADS], rl = r[2 * HEADS];
      weight[hh][i] = rl == 0.f ? -INFINITY : rM;  // no positions: no weight
      if (rl == 0.f) continue;
      const float mn = fmaxf(m, rm);
      l = (m == mn ? l : l * ex2(m - mn)) + (rm == mn ? rl : rl * ex2(rm - mn));
      m = mn;
      M = fmaxf(M, rM);
    }
    const float mm = warp_max(m);
    M = warp_max(M);
    l = warp_sum(l == 0.f ? 0.f : l * ex2(m - mm));
    for (uint32_t i = lane; i < n; i += 32) weight[hh][i] = weight[hh][i] == -INFINITY ? 0.f : ex2(weight[hh][i] - M);
    if (lane == 0) fin[hh] = out_factor(M - mm - 14.f, l);
  }
  __syncthreads();
  float4 o{};
  auto add = [&](const float4& v, uint32_t i) {
    const float f = weight[h][i];
    o.x += v.x * f, o.y += v.y * f, o.z += v.z * f, o.w += v.w * f;
  };
#pragma unroll
  for (uint32_t k = 0; k < HELD; ++k)
    if (grp + k * GROUPS < n) add(x[k], grp + k * GROUPS);
#pragma unroll 4
  for (uint32_t i = grp + HELD * GROUPS; i < n; i += GROUPS) add(reinterpret_cast<const float4*>(rec(i))[e], i);
  sum[tid] = o;
  __syncthreads();
  const uint32_t slot = HEADS * blockIdx.y + h, rows = (uint32_t)hd.slot_rows >> 1;
  if (grp || slot >= (nsub == 1 ? rows * G : min(G - sub * SLOTS, SLOTS))) return;
#pragma unroll
  for (uint32_t k = 1; k < GROUPS; ++k) {
    const float4 v = sum[k * PER_GROUP + e];
    o.x += v.x, o.y += v.y, o.z += v.z, o.w += v.w;
  }
  const float2 f = fin[h];
  const uint32_t in = nsub == 1 ? slot * a.inv_group >> 16 : 0, row = (uint32_t)hd.row + in, head = sub * SLOTS + slot - in * G;
  const size_t at = row * a.out_stride + (size_t)(head * n_kv + kvh) * HD + 4 * (e % (HD / 4));
  store_dt(a.out, at, a.dtype, o.x * f.x * f.y);
  store_dt(a.out, at + 1, a.dtype, o.y * f.x * f.y);
  store_dt(a.out, at + 2, a.dtype, o.z * f.x * f.y);
  store_dt(a.out, at + 3, a.dtype, o.w * f.x * f.y);
}

template <int HD, uint32_t TYPE, int SETS, bool MANY>
cudaError_t attend_sets(PagesAttnArgs a, int num_sms, cudaStream_t st) {
  using L = Lay<HD, SETS>;
  constexpr uint32_t SLOTS = SETS * HEADS;
  a.group = a.n_heads / a.pool.n_kv;
  a.subs = (a.group + SLOTS - 1) / SLOTS;
  a.window = MANY && a.row_seq && a.group < SLOTS ? SLOTS / a.group : 1;
  a.inv_group = 65536 / a.group + 1;
  const uint32_t ctas = (uint32_t)min(num_sms * L::CTAS, MAX_CTAS);
  cudaError_t e = launch_early(attend_kernel<HD, TYPE, SETS, MANY>, 1, dim3(ctas), dim3(THREADS), L::BYTES, st, a);
  if (e != cudaSuccess) return e;
  // the join waits for the kernel above by itself (griddepcontrol.wait)
  // Few items are cut into many pieces each, and only their first CTAs have any
  // to join: large blocks (1 x 8192, 32 pieces an item: 8.4 us against 11).  Many
  // items are cut in two or three, by almost every CTA: small ones.
  const bool many = (uint64_t)a.n_rows * a.pool.n_kv * a.subs * 4 > ctas;
  return launch_early(many ? attend_join_kernel<HD, SETS, 256> : attend_join_kernel<HD, SETS, 1024>, 1, dim3(ctas, SETS),
                      dim3(many ? 256 : 1024), 0, st, a);
}

template <int HD, uint32_t TYPE>
cudaError_t attend_go(const PagesAttnArgs& a, int num_sms, cudaStream_t st) {
  // Where a request's rows have more than 8 heads for a KV head, two sets of slots
  // share what is read and converted, and three CTAs fit an SM instead of four:
  // 32 requests of 2000 positions, 4 rows of 64 heads over 8 of 128: 84 us with
  // one set, 76 with two; 24 heads over 2, one row: 29 and 27; 64 x 4 rows of 32
  // heads over 4 of 64, 2048 positions: 70 and 62; at 8 heads one set is all it takes.
  // Rows of one request share an item of one set as well: 5 rows of 16 heads over 16:
  // 111 us apart, 51 together.  The search for such rows costs other calls 0.5 us
  // of instruction fetches, so they go without.
  // Which rows are live only the device knows, so the rule goes by the arrays' sizes
  // and picks the other variant where padding changes those (32 heads over 8 of 128,
  // lengths to 2000): 64 single rows in 64 rows 44 us, in 256 rows of 64 requests
  // 64; 4 rows each of 32 requests in 128 rows of 32 request slots 39, of 256 slots 67.
  const uint64_t G = a.n_heads / a.pool.n_kv;
  if (a.n_rows * G > (uint64_t)HEADS * min(a.n_seq, a.n_rows)) return attend_sets<HD, TYPE, 2, true>(a, num_sms, st);
  return a.row_seq && a.n_rows > a.n_seq ? attend_sets<HD, TYPE, 1, true>(a, num_sms, st)
                                         : attend_sets<HD, TYPE, 1, false>(a, num_sms, st);
}

template <int HD, uint32_t TYPE>
cudaError_t attend_attributes() {
  const auto big = cudaFuncAttributeMaxDynamicSharedMemorySize;
  cudaError_t e = cudaFuncSetAttribute(attend_kernel<HD, TYPE, 1, false>, big, Lay<HD, 1>::BYTES);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(attend_kernel<HD, TYPE, 1, true>, big, Lay<HD, 1>::BYTES);
  return e == cudaSuccess ? cudaFuncSetAttribute(attend_kernel<HD, TYPE, 2, true>, big, Lay<HD, 2>::BYTES) : e;
}

}  // namespace

size_t pages_attend_ws_bytes(uint32_t, uint32_t, uint32_t, uint32_t hd) {
  return MAX_CTAS * (sizeof(Header) + 2 * 2 * 4 * (size_t)(hd == 64 ? Lay<64, 2>::REC : Lay<128, 2>::REC));
}

cudaError_t pages_attend_init() {
  cudaError_t e = attend_attributes<64, PAGES_I8>();
  if (e == cudaSuccess) e = attend_attributes<64, PAGES_E4M3>();
  if (e == cudaSuccess) e = attend_attributes<128, PAGES_I8>();
  return e == cudaSuccess ? attend_attributes<128, PAGES_E4M3>() : e;
}

cudaError_t pages_attend_launch(const PagesAttnArgs& a, int num_sms, cudaStream_t st) {
  if (a.pool.hd == 64)
    return a.pool.type == PAGES_I8 ? attend_go<64, PAGES_I8>(a, num_sms, st) : attend_go<64, PAGES_E4M3>(a, num_sms, st);
  return a.pool.type == PAGES_I8 ? attend_go<128, PAGES_I8>(a, num_sms, st) : attend_go<128, PAGES_E4M3>(a, num_sms, st);
}

}  // namespace shk
