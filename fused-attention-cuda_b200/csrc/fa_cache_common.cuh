// fa_cache_common.cuh -- device helpers shared by the paged cache's kernels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "fa_cache.h"

namespace fa_sm100 {

// One sequence's part of the batch.  Everything here comes from device memory, so it is checked:
// a value out of range is reported through the status word and replaced by one that is safe.
struct SeqInfo {
  int t0;    // first packed row
  int n;     // new tokens
  int len;   // keys held, this call's included; no more than the table has room for, or as it was given
};

__device__ __forceinline__ void report_cache_index(const CacheView& c) {
  atomicOr(c.status, kStCacheIndex);
}

// The packed rows of sequence s lie in the batch, and those of the first one begin it.
__device__ __forceinline__ bool offsets_ok(const CacheView& c, int s, int t0, int end) {
  return t0 >= 0 && end >= t0 && end <= c.T && (s > 0 || t0 == 0);
}

// What a length above the table's room means: the room (KEEP_LONG false), or that the sequence's last tokens
// have no page, which is for the caller to see.
template <bool KEEP_LONG = false>
__device__ __forceinline__ SeqInfo seq_info(const CacheView& c, int s) {
  SeqInfo q;
  int len = c.seq_lens[s];
  if (c.cu_seqlens != nullptr) {
    q.t0 = c.cu_seqlens[s];
    const int end = c.cu_seqlens[s + 1];
    if (!offsets_ok(c, s, q.t0, end)) {
      report_cache_index(c);
      q.t0 = 0;
      q.n = 0;
    } else {
      q.n = end - q.t0;
    }
  } else {
    q.n = c.T / c.n_seqs;
    q.t0 = s * q.n;
  }
  const long long room = static_cast<long long>(c.max_pages) << c.page_shift;
  if (len < 0 || len > room) {
    report_cache_index(c);
    len = len < 0 ? 0 : KEEP_LONG ? len : static_cast<int>(room);
  }
  q.len = len;
  return q;
}

// Packed rows that belong to a sequence; the rows from here to T are behind the last one.
__device__ __forceinline__ int live_rows(const CacheView& c) {
  if (c.cu_seqlens == nullptr) return c.T;
  const int end = c.cu_seqlens[c.n_seqs];
  return end < 0 ? 0 : (end > c.T ? c.T : end);
}

// Zeros in the rows of attention's outputs that belong to no sequence, by all threads of all blocks:
// those behind the last one or, where an offset is out of order, each row that no sequence has.
template <typename T, int D, int THREADS>
__device__ __forceinline__ void zero_stray_rows(const CacheAttnArgs& a) {
  const CacheView& c = a.c;
  if (c.cu_seqlens == nullptr) return;
  const int live = live_rows(c);
  bool bad = false;
  for (int s = threadIdx.x; s < c.n_seqs; s += THREADS) {
    bad |= !offsets_ok(c, s, c.cu_seqlens[s], c.cu_seqlens[s + 1]);
  }
  bad = __syncthreads_or(bad);
  for (int t = (bad ? 0 : live) + static_cast<int>(blockIdx.x); t < c.T; t += gridDim.x) {
    bool stray = true;
    if (bad) {
      for (int s = threadIdx.x; s < c.n_seqs; s += THREADS) {
        const int t0 = c.cu_seqlens[s], end = c.cu_seqlens[s + 1];
        stray &= !(offsets_ok(c, s, t0, end) && t >= t0 && t < end);
      }
      stray = __syncthreads_and(stray);
    }
    if (!stray) continue;
    const long long at = static_cast<long long>(t) * a.H;
    uint4* o = reinterpret_cast<uint4*>(static_cast<T*>(a.o) + at * D);
    for (int i = threadIdx.x; i < a.H * (D / 8); i += THREADS) o[i] = make_uint4(0, 0, 0, 0);
    for (int h = threadIdx.x; h < a.H; h += THREADS) a.lse[at + h] = 0.f;
  }
}

// The page of sequence s that holds its keys [i << page_shift, ...), or -1 (reported).
__device__ __forceinline__ int page_of(const CacheView& c, int s, int i) {
  if (i < 0 || i >= c.max_pages) {
    report_cache_index(c);
    return -1;
  }
  const int p = c.block_table[static_cast<long long>(s) * c.table_stride + i];
  if (p < 0 || p >= c.num_pages) {
    report_cache_index(c);
    return -1;
  }
  return p;
}

// A page's value scale as (log2, reciprocal); exact for powers of two.  P / scale is summed, P at most
// 2^8 and its exponent's range 2^-126, so the scales need a range of their own for the denominator to
// hold: what lies outside of it (zero and what is negative, too) is reported and counts as its nearest end.
// A scale that is NaN makes the scores of the rows that see its page NaN, by way of `add`; `inv` also meets
// the zero weights of rows that do not, so it stays finite.
constexpr float kMinValueScale = 0x1p-64f, kMaxValueScale = 0x1p120f;  // what cache_append writes
__device__ __forceinline__ void value_scale(const CacheView& c, float s, float* add, float* inv) {
  const float in = fminf(fmaxf(s, kMinValueScale), kMaxValueScale);
  if (s < kMinValueScale || s > kMaxValueScale) report_cache_index(c);
  const int bits = __float_as_int(in);
  const float mant = __int_as_float((bits & 0x7fffff) | 0x3f800000);
  *add = s != s ? s : static_cast<float>((bits >> 23) - 127) + log2f(mant);
  *inv = s != s ? 1.f : 1.0f / in;
}

// A key that some rows of a tile see and others do not has weight 0 in the latter, but 0 times NaN is
// NaN.  Where a tile's rows differ in what they see, the kernels therefore take V's NaN out (e4m3 has
// no infinities), note it, and at the end put NaN where it belongs: the columns of nan_columns in the
// rows that see the key.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t v) {  // 0xff in the bytes that are NaN
  return __vcmpeq4(v & 0x7f7f7f7fu, 0x7f7f7f7fu);
}

// Bit i: column col + i (col, COLS multiples of 4) of V is NaN in one of the keys [lo, hi).
template <int COLS>
__device__ __forceinline__ uint32_t nan_columns(const CacheView& c, int s, int head, int lo, int hi,
                                                int col) {
  uint32_t bits = 0;
#pragma unroll 1
  for (int key = lo; key < hi; ++key) {
    const int page = page_of(c, s, key >> c.page_shift);
    if (page < 0) continue;
    const unsigned char* at = c.v + page * c.vs[0] + head * c.vs[1] +
                              (key & ((1 << c.page_shift) - 1)) * c.vs[2] + col;
#pragma unroll
    for (int i = 0; i < COLS / 4; ++i) {
      const uint32_t n = nan_bytes(*reinterpret_cast<const uint32_t*>(at + 4 * i)) & 0x08040201u;
      bits |= ((n | n >> 8 | n >> 16 | n >> 24) & 15u) << (4 * i);
    }
  }
  return bits;
}

// In a kernel launched while the one before it runs: until that one's results are there.  Every block
// of such a kernel comes here, so that its end is the end of both.
__device__ __forceinline__ void wait_for_parts() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

template <typename T>
__device__ __forceinline__ float2 to_float2(uint32_t u);
template <>
__device__ __forceinline__ float2 to_float2<__half>(uint32_t u) {
  return __half22float2(*reinterpret_cast<__half2*>(&u));
}
template <>
__device__ __forceinline__ float2 to_float2<__nv_bfloat16>(uint32_t u) {
  return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&u));
}

template <typename T>
__device__ __forceinline__ uint32_t from_float2(float a, float b);
template <>
__device__ __forceinline__ uint32_t from_float2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t from_float2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

}  // namespace fa_sm100
