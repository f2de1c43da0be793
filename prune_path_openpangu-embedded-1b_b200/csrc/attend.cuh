// What the two attention kernels (attend.cu: few rows; attend_tiles.cu: many) share.
#pragma once
#include <math_constants.h>
#include <algorithm>
#include <cmath>
#include <type_traits>
#include "seqs.cuh"
#include "umma.cuh"

namespace ppmoe {

struct AttendArgs {
  const void* q;
  int64_t q_t, q_h;
  void* out;
  int64_t o_t, o_h;
  int tokens, q_heads, group;
  float c;         // |scale| log2 e (1 where scale is 0)
  int q_sign;      // -1, 0, 1: what q is multiplied by
  int q_wide16;    // rows of q start on 16-byte boundaries
  int o_wide;      // rows of out start on 16-byte boundaries
  int o_wide32;    // ... on 32-byte boundaries
  int nsplit;      // parts of the keys; above 1 they meet in ws
  int joins;       // the next launch on the stream is attend_join_kernel, which may start early
  float* part_o;   // [nsplit][tokens][q_heads][D]: sum of 2^(x - m) v
  float* part_ml;  // [nsplit][tokens][q_heads][2]: m, l
  Seqs seqs;
  Pages pages;
  uint32_t* status;
};

__device__ __forceinline__ float exp2_ftz(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Sequence b as the kernels see it: its first packed row, its new rows (held to the rows there are), its length.
struct Seq {
  int first, rows, length;
};
__device__ __forceinline__ Seq load_seq(const AttendArgs& a, int b) {
  Seq s;
  s.first = a.seqs.starts[b];
  int end = a.seqs.starts[b + 1];
  s.length = a.seqs.lengths[b];
  if (s.first < 0) s.first = 0;
  if (end > a.tokens) end = a.tokens;
  s.rows = end - s.first;
  return s;
}
// The positions of a sequence that its table can name.
__device__ __forceinline__ int key_cap(const AttendArgs& a, int length) {
  const int64_t cap = (int64_t)a.seqs.max_pages << a.pages.page_shift;
  return length < cap ? length : (int)cap;
}

// What the sum of a row at position pos is multiplied by.  Its weights sum to 0 where it sees no key (its sum is 0 too)
// and where every score that it sees is -inf: softmax has no answer there, so NaN.
__device__ __forceinline__ float inverse_sum(float l, int pos) {
  return l > 0.f ? 1.f / l : l == 0.f && pos < 0 ? 0.f : CUDART_NAN_F;
}

// C rounded values of one row piece, scaled by inv.
template <typename T, int C>
__device__ __forceinline__ void store_row(T* out, const float (&v)[C], float inv, bool wide) {
  if (wide) {
#pragma unroll
    for (int i = 0; i < C; i += 8)
      *reinterpret_cast<uint4*>(out + i) =
          make_uint4(pack2<T>(v[i] * inv, v[i + 1] * inv), pack2<T>(v[i + 2] * inv, v[i + 3] * inv),
                     pack2<T>(v[i + 4] * inv, v[i + 5] * inv), pack2<T>(v[i + 6] * inv, v[i + 7] * inv));
  } else {
#pragma unroll
    for (int i = 0; i < C; ++i) out[i] = from_f32<T>(v[i] * inv);
  }
}

// 16 bytes global -> shared, or 16 zero bytes (the source is then not read).
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}

// What q is multiplied by (-1, 0 or 1), on a packed pair.
__device__ __forceinline__ uint32_t q_pair(uint32_t v, int sign) {
  return sign > 0 ? v : sign < 0 ? v ^ 0x80008000u : 0u;
}

// Fp16 weights below 2^-24 would vanish; lifting every weight by 2^7 (it cancels against l) keeps
// those down to 2^-31 of the largest, and weights of up to 2^8 (attend_tiles.cu) below fp16's
// largest number.  bf16 has fp32's exponents and needs none.
template <typename T>
constexpr float kLift = 0.f;
template <>
constexpr float kLift<__half> = 7.f;

// Exponent field all ones: inf or NaN.
template <typename T>
__device__ __forceinline__ bool not_finite16(uint32_t v) {  // v: the 16 bits
  constexpr uint32_t m = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  return (v & m) == m;
}
template <typename T>
__device__ __forceinline__ uint32_t not_finite2(uint32_t v) {  // bits 15 and 31: of the two halves
  // a one added below an exponent of all ones carries into the sign's place, and no further
  constexpr uint32_t m = std::is_same<T, __half>::value ? 0x7c007c00u : 0x7f807f80u;
  constexpr uint32_t one = std::is_same<T, __half>::value ? 0x04000400u : 0x00800080u;
  return ((v & m) + one) & 0x80008000u;
}

int attend_tiles_launch(AttendArgs& a, int head_dim, int page_size, bool half, int tiles, int groups, cudaStream_t st);

}  // namespace ppmoe
