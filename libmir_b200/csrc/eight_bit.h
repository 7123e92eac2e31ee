// One call of attention over the 8-bit cache, as the entry points hand it to the kernels' launchers.
#pragma once
#include "eight_bit.cuh"

struct Attention8 {
  const char* what = "";
  const void* q = nullptr;             // packed bf16 rows whose first heads * head_dim columns are the rotated queries
  long long q_stride = 0;
  void* out = nullptr;                 // [tokens, heads * head_dim] bf16
  mir::Cache8 cache{};
  const int* block_table = nullptr;    // [num_rows, table_width]
  int table_width = 0;
  const int* positions = nullptr;      // one token per request: its position; else
  const int* query_starts = nullptr;   // portions
  const int* context_lens = nullptr;
  int num_rows = 0, heads = 0, head_dim = 0;
  float scale = 0.0f;
  int window = 0;
  // keys split over this many partitions, joined by mir_merge_8bit; partition 0: all requests' keys shared out over that many CTAs
  int partition = 0, num_partitions = 1;
  float* scratch = nullptr;
  long long scratch_floats = 0;
  const float* sinks = nullptr;        // [heads] or null
  const int* error = nullptr;          // not 0: partitions may be missing, nothing is joined; null: none ever is
  cudaStream_t stream = nullptr;

  float* partial_o(long long) const { return scratch; }
  float* partial_ml(long long tokens) const {
    return scratch == nullptr ? nullptr : scratch + tokens * heads * num_partitions * head_dim;
  }
};

int mir_attention_8bit_general(const Attention8& a, int tokens);
int mir_merge_8bit(const Attention8& a, int tokens);
// Single tokens on the 5th-generation tensor cores (attention_8bit_decode.cu), where it takes the sizes.
bool mir_decode_8bit_takes(int head_dim, int page_size);
int mir_decode_8bit_ctas(long long most_tiles, int heads, int kv_heads);
long long mir_decode_8bit_floats(int ctas, int group);
int mir_attention_8bit_decode(const Attention8& a);
// Portions on them (attention_8bit_tc.cu), for the same sizes.
int mir_attention_8bit_prefill(const Attention8& a, int tokens);

// The product of rounded rows (codes [m, k], scales [blocks of 128 columns, scale_stride], scale_stride m
// filled up to whole 128) with an 8-bit weight, by tiles of 128 rows
// on the tensor cores (linear_8bit_tc.cu).
int mir_linear_8bit_tiles(const uint8_t* codes, const float* scales, int scale_stride, const uint8_t* weight, const float* w_scales,
                          const void* bias, void* out, long long out_stride, int m, int n, int k, bool out_float, bool accumulate, cudaStream_t stream);
// The same for up to 128 rows, bound by the weight's bytes (linear_8bit_few.cu): codes and scales as above, or, where `rounds` says so,
// bf16 rows.
bool mir_linear_8bit_few_takes(int m, int k);
bool mir_linear_8bit_few_rounds(int m);
int mir_linear_8bit_few(const uint8_t* codes, const float* scales, int scale_stride, const void* x, long long x_stride,
                        const uint8_t* weight, const float* w_scales, const void* bias, void* out, long long out_stride, int m, int n, int k,
                        bool out_float, bool accumulate, cudaStream_t stream);
