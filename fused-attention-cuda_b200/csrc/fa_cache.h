// fa_cache.h -- internal interface between the C-ABI layer of the paged cache (fa_cache.cu) and
// its kernels (fa_cache_append.cu, fa_cache_attn.cu).  Not part of the public ABI.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "fa_launch.h"
#include "fa_sm100.h"

namespace fa_sm100 {

// The cache and the batch as the kernels see them (validated on the host; everything that lives in
// device memory -- page numbers, lengths, offsets -- is checked by the kernels themselves).
struct CacheView {
  unsigned char* k;
  unsigned char* v;
  float* k_scale;
  float* v_scale;
  long long ks[3], vs[3];  // byte strides of (page, kv head, token)
  long long num_pages;
  int page_shift;  // log2(page_size)
  int Hkv;
  const int* block_table;
  long long table_stride;
  int max_pages;
  const int* seq_lens;
  const int* cu_seqlens;  // null: T / n_seqs new tokens for each sequence
  int n_seqs;
  int T;         // packed new tokens (rows of q, k, v)
  unsigned* status;  // the library's status word (kStCacheIndex)
};

struct AppendArgs {
  CacheView c;
  int dtype, H, D;
  const void* k;
  const void* v;
  const void* q;  // may be null
  void* q_out;
  long long sk[2], sv[2], sq[2];  // element strides of (token, head)
  const float* cos;               // null: no rotation
  const float* sin;
  long long table_rows;  // rows of cos / sin
  int rot_dim;
  bool interleaved;
};

struct CacheAttnArgs {
  CacheView c;
  int dtype, H, D;
  const void* q;
  long long sq[2];
  void* o;
  float* lse;
  float scale;
  bool causal;
  void* workspace;
  unsigned long long timeout_ns;
};

cudaError_t launch_cache_append(const AppendArgs& a, cudaStream_t stream);
cudaError_t launch_cache_attention(const CacheAttnArgs& a, cudaStream_t stream);
// Sequences with few query rows on average (fa_cache_attn.cu) or many (fa_cache_tile.cu).
cudaError_t launch_cache_tile(const CacheAttnArgs& a, cudaStream_t stream);
size_t cache_tile_workspace(int D, int sms);
size_t cache_attention_workspace(int H, int Hkv, int D, int T, int n_seqs, int sms);

// Tensor maps of the pages {d, token, kv head, page}, the last three ordered by stride; `pos` packs
// (two bits each) which of the map's dimensions 1-3 holds token, head and page.
struct PageMaps {
  CUtensorMap k, v;
  int k_pos, v_pos;
};
// Boxes of `rows` tokens, swizzled by the row's D bytes.
cudaError_t make_page_maps(PageMaps* m, const CacheView& c, int D, int rows);

// Multiprocessors of the current device (148 when the query fails).
int multiprocessors();

// Device address of the status word on the current device (null on error).
unsigned* status_word(cudaError_t* err);

}  // namespace fa_sm100
