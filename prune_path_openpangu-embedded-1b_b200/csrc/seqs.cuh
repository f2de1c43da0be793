// What the paged-cache kernels (rotary.cu, attend.cu) share: the description of a ragged batch of
// newest tokens over a paged key/value cache, and element conversions.
#pragma once
#include <cuda_fp16.h>
#include "common.cuh"

namespace ppmoe {

// Sequence b owns the packed rows [starts[b], starts[b+1]); they are its newest tokens, so row
// starts[b] + i stands at position lengths[b] - (starts[b+1] - starts[b]) + i of lengths[b] keys.
// Position p of sequence b lies in row p % page of page table[b][p / page] of the cache.
struct Seqs {
  const int32_t* starts;   // [batch + 1], not decreasing
  const int32_t* lengths;  // [batch]
  const int32_t* table;    // [batch][max_pages], rows table_stride apart
  int64_t table_stride;
  int batch, max_pages;
};

struct Pages {
  void* k;
  void* v;
  int64_t k_page, k_head, k_row, v_page, v_head, v_row;  // strides in elements; the last one is 1
  int num_pages, page_shift, kv_heads;                   // page size 1 << page_shift
};

// Largest b with starts[b] <= t (-1: t lies before the first sequence), by all lanes of a warp:
// each step probes 32 pivots, so 1024 sequences take two dependent loads and not ten.
__device__ __forceinline__ int find_seq_warp(const int32_t* starts, int batch, int t) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = batch + 1;  // starts[0 .. lo) <= t; starts[hi ..) > t
  while (lo < hi) {
    const int step = (hi - lo + 31) / 32;
    const int i = lo + lane * step;
    const bool le = i < hi && __ldg(starts + i) <= t;
    const int n = __popc(__ballot_sync(0xffffffffu, le));  // pivots 0 .. n-1 are <= t
    if (n == 0) break;
    const int last = lo + (n - 1) * step;  // starts[last] <= t
    const int next = last + step;          // the following pivot, > t (or past hi)
    lo = last + 1;
    hi = next < hi ? next : hi;
  }
  return lo - 1;
}

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Two rounded values in one 32-bit word, the first in the low half.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Host-side checks common to the entry points of both files (kvcache layout and batch tables).
int check_cache(const char* fn, const ppmoe_kv_cache* c, Pages& p);
int check_seqs(const char* fn, const Seqs& s);

}  // namespace ppmoe
