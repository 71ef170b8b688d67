// pages.cuh -- K/V pools of 8-bit blocks shared by the requests of a batch:
// block tables and slots, append, read and attention launchers.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace shk {

// Types of q, k, v and logits (ggml's codes).
constexpr uint32_t DT_F32 = 0;
constexpr uint32_t DT_F16 = 1;
constexpr uint32_t DT_BF16 = 30;

// Pool types: value = scale * byte, the byte a signed integer or an e4m3 number.
constexpr uint32_t PAGES_I8 = 0;
constexpr uint32_t PAGES_E4M3 = 1;

// One layer's pools.  Block b, head h, token t of the block: k / v at
// ((b * n_kv + h) * block + t) * hd, scales at b * n_kv + h.
struct PagesPool {
  uint8_t* k;
  uint8_t* v;
  float* ks;
  float* vs;
  uint32_t type;
  uint32_t n_blocks, n_kv, hd;
  uint32_t block_shift;  // log2 of the tokens per block
};

struct AssignArgs {
  uint32_t n_seq, block_shift, n_blocks, stride, n_rows;
  const int32_t* have;
  const int32_t* add;
  int32_t* table;
  const int32_t* free_ids;
  const int32_t* n_free;
  int32_t* lens;
  int32_t* counts;
  int32_t* slots;
  int32_t* pos;
  int32_t* seq;
  int32_t* last;
  int* err;
};

struct ReleaseArgs {
  uint32_t n_seq, block_shift, n_blocks, stride;
  const int32_t* table;
  const int32_t* done;
  const int32_t* keep;  // not null: tokens kept, in place of done
  const int32_t* have;
  int32_t* lens;
  int32_t* free_ids;
  const int32_t* n_free;
  int32_t* n_free_out;
  int* err;
};

struct PagesAttnArgs {
  PagesPool pool;
  uint32_t n_rows, n_seq, n_heads;
  uint32_t dtype;  // of q and out
  const void* q;
  void* out;
  size_t q_stride, out_stride;  // elements
  const int32_t* row_seq;       // null: row r is sequence r
  const int32_t* row_pos;
  const int32_t* table;
  uint32_t stride;
  float scale;
  void* ws;
  int* err;
  // set by the launcher
  uint32_t group;      // query heads of a KV head
  uint32_t subs;       // items of a KV head and row
  uint32_t window;     // rows whose heads fit one item
  uint32_t inv_group;  // 2^16 / group + 1: x * inv_group >> 16 is x / group for x < 16
};

cudaError_t pages_init();  // kernel attributes, once per device
cudaError_t pages_assign_launch(const AssignArgs& a, cudaStream_t st);
cudaError_t pages_release_launch(const ReleaseArgs& a, cudaStream_t st);
cudaError_t pages_append_launch(const PagesPool& p, uint32_t n, const void* k, const void* v, uint32_t dtype,
                                size_t row_stride, const int32_t* slots, int* err, int num_sms, cudaStream_t st);
cudaError_t pages_read_launch(const PagesPool& p, uint32_t n, const int32_t* slots, float* k, float* v, int* err,
                              int num_sms, cudaStream_t st);
size_t pages_attend_ws_bytes(uint32_t n_rows, uint32_t n_heads, uint32_t n_kv, uint32_t hd);
cudaError_t pages_attend_init();
cudaError_t pages_attend_launch(const PagesAttnArgs& a, int num_sms, cudaStream_t st);

}  // namespace shk
