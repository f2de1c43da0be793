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

// Largest of three, NaN where one is.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
template <int N>
__device__ __forceinline__ bool any_nan(const float (&v)[N]) {
  float top = v[0];
#pragma unroll
  for (int i = 1; i < N; i += 2) top = max3(top, v[i], v[i + 1 < N ? i + 1 : i]);
  return top != top;
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

// Eight rounded values of a row, scaled by inv.
template <typename T>
__device__ __forceinline__ void store_row(T* out, const float (&v)[8], float inv, bool wide) {
  if (wide) {
    *reinterpret_cast<uint4*>(out) =
        make_uint4(pack2<T>(v[0] * inv, v[1] * inv), pack2<T>(v[2] * inv, v[3] * inv), pack2<T>(v[4] * inv, v[5] * inv),
                   pack2<T>(v[6] * inv, v[7] * inv));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = from_f32<T>(v[i] * inv);
  }
}

// 16 bytes global -> shared, or 16 zero bytes (the source is then not read).
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
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

// A packed pair of q times -1, 0 or 1 (0 times what is not finite is NaN).
template <typename T>
__device__ __forceinline__ uint32_t q_pair(uint32_t v, int sign) {
  return sign > 0 ? v : sign < 0 ? v ^ 0x80008000u : (not_finite2<T>(v) >> 15) * 0x7fffu;
}

// Values that are not finite are listed apart: list [NaN, +inf, -inf][D], the first key with one in each column.
// What column col of a row that sees keys up to lim gets from them.
template <int D>
__device__ __forceinline__ float listed_value(const int* list, int col, int lim) {
  float add = 0.f;
  if (list[D + col] <= lim) add += CUDART_INF_F;
  if (list[2 * D + col] <= lim) add -= CUDART_INF_F;
  return list[col] <= lim ? CUDART_NAN_F : add;
}
// Lists one: the bits of key `key`'s value in column col.
template <typename T, int D>
__device__ __forceinline__ void list_value(int* list, uint16_t bits, int key, int col) {
  const float f = to_f32<T>(*reinterpret_cast<const T*>(&bits));
  atomicMin(list + (f != f ? 0 : f > 0.f ? 1 : 2) * D + col, key);
}
// Where a row's weights are fine and a sum over them is NaN, an infinity may have met a weight or a factor that vanished
// (0 * inf); what the sum has to be then follows from the values that are not finite alone.  THREADS threads (a warp or
// the CTA) list those of keys [from, to).  That is paid for where a NaN stands in an early value: 16 prompts of 512
// then take 64 us for 32 (12 heads of 64), 2048 rows over 34816 keys 7.4 ms for 0.93.
template <typename T, int D, int THREADS>
__device__ __noinline__ void list_values(const AttendArgs& a, int b, int kvh, int from, int to, int* list) {
  auto sync = [] {
    if constexpr (THREADS == 32)
      __syncwarp();
    else
      __syncthreads();
  };
  const int me = threadIdx.x % THREADS;
  for (int i = me; i < 3 * D; i += THREADS) list[i] = INT_MAX;
  sync();
  constexpr int CH = D / 8;
  const int32_t* table = a.seqs.table + b * a.seqs.table_stride;
#pragma unroll 4
  for (int64_t i = (int64_t)from * CH + me; i < (int64_t)to * CH; i += THREADS) {
    const int key = (int)(i / CH), col = (int)(i % CH) * 8, page = table[key >> a.pages.page_shift];
    if ((uint32_t)page >= (uint32_t)a.pages.num_pages) continue;
    const int64_t row = key & ((1 << a.pages.page_shift) - 1);
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.pages.v) + page * a.pages.v_page +
                                                         kvh * a.pages.v_head + row * a.pages.v_row + col));
    if (!(not_finite2<T>(v.x) | not_finite2<T>(v.y) | not_finite2<T>(v.z) | not_finite2<T>(v.w))) continue;
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint16_t bits = (uint16_t)(u[e >> 1] >> (16 * (e & 1)));
      if (not_finite16<T>(bits)) list_value<T, D>(list, bits, key, col + e);
    }
  }
  sync();
}
// ... and one thread puts right n columns from col on of row r (of those of kv head kvh, which sees keys up to lim): of the
// result, or (part >= 0) of a part on its way to the join.
template <typename T, int D>
__device__ __noinline__ void mend_row(const AttendArgs& a, const int* list, int64_t first, int r, int kvh, int part, int lim,
                                      int col, int n) {
  const int64_t t = first + r / a.group;
  const int h = kvh * a.group + r % a.group;
  auto go = [&](auto* row) {
    using V = std::remove_pointer_t<decltype(row)>;
#pragma unroll 1
    for (int c = col; c < col + n; ++c) {
      const float v = to_f32<V>(row[c]), right = listed_value<D>(list, c, lim);
      if (v != v && right != 0.f) row[c] = from_f32<V>(right);
    }
  };
  if (part >= 0)
    go(a.part_o + (((int64_t)part * a.tokens + t) * a.q_heads + h) * D);
  else
    go(static_cast<T*>(a.out) + t * a.o_t + h * a.o_h);
}

int attend_tiles_launch(AttendArgs& a, int head_dim, int page_size, bool half, int tiles, int groups, cudaStream_t st);

}  // namespace ppmoe
