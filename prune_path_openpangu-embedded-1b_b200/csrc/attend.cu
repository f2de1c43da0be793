// Causal attention of each sequence's newest tokens over a paged key/value cache.
//
//   out[t, h] = sum_{j <= p(t)} w_j v_j,  w = softmax_j(scale q[t, h] . k_j),  p(t) = position of t
// and 0 where no key is left (p(t) < 0).
//
// One warp per (token, head): one pass over the keys with the running maximum m and sum l of
// the softmax; every lane holds head_dim / 32 values of the query and of the sum.
#include "seqs.cuh"

namespace ppmoe {

struct AttendArgs {
  const void* q;
  int64_t q_t, q_h;
  void* out;
  int64_t o_t, o_h;
  int tokens, q_heads, group;
  float scale;
  Seqs seqs;
  Pages pages;
  uint32_t* status;
};

template <typename T, int D>
__global__ void __launch_bounds__(128) attend_rows_kernel(const __grid_constant__ AttendArgs a) {
  constexpr int N = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int t = (int)(item / a.q_heads), h = (int)(item % a.q_heads);
  if (t >= a.tokens) return;
  const int b = find_seq_warp(a.seqs.starts, a.seqs.batch, t);
  if (b < 0 || b >= a.seqs.batch) return;
  const int pos = a.seqs.lengths[b] - a.seqs.starts[b + 1] + t;
  const int64_t cap = (int64_t)a.seqs.max_pages << a.pages.page_shift;
  const int keys = (int)(pos + 1 < cap ? pos + 1 : cap);
  float q[N], o[N], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    q[i] = to_f32<T>(static_cast<const T*>(a.q)[t * a.q_t + h * a.q_h + lane + 32 * i]) * a.scale;
    o[i] = 0.f;
  }
  for (int j = 0; j < keys; ++j) {
    const int page = a.seqs.table[b * a.seqs.table_stride + (j >> a.pages.page_shift)];
    if (page < 0 || page >= a.pages.num_pages) {
      atomicOr(a.status, DEVERR_PAGE);
      continue;
    }
    const int64_t row = j & ((1 << a.pages.page_shift) - 1);
    const T* k = static_cast<const T*>(a.pages.k) + page * a.pages.k_page + row * a.pages.k_row + (h / a.group) * a.pages.k_head;
    const T* v = static_cast<const T*>(a.pages.v) + page * a.pages.v_page + row * a.pages.v_row + (h / a.group) * a.pages.v_head;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) s += q[i] * to_f32<T>(k[lane + 32 * i]);
    s = warp_sum(s);
    const float m2 = fmaxf(m, s), c = m2 == -INFINITY ? 1.f : __expf(m - m2), p = m2 == -INFINITY ? 0.f : __expf(s - m2);
    m = m2;
    l = l * c + p;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = o[i] * c + p * to_f32<T>(v[lane + 32 * i]);
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    static_cast<T*>(a.out)[t * a.o_t + h * a.o_h + lane + 32 * i] = from_f32<T>(l != 0.f ? o[i] / l : 0.f);
}

template <typename T, int D>
static int launch(const AttendArgs& a, cudaStream_t st) {
  const int64_t items = (int64_t)a.tokens * a.q_heads;
  attend_rows_kernel<T, D><<<(unsigned)((items + 3) / 4), 128, 0, st>>>(a);
  PPMOE_CHECK_CUDA(cudaGetLastError());
  return PPMOE_OK;
}

}  // namespace ppmoe

using namespace ppmoe;

extern "C" size_t ppmoe_attend_workspace_bytes(int tokens, int q_heads, int kv_heads, int head_dim, int batch,
                                               int max_new, int64_t max_length) {
  return 0;
}

extern "C" int ppmoe_attend(const void* q, int64_t q_t, int64_t q_h, int q_heads, int tokens, const void* k_pages,
                            int64_t kp_page, int64_t kp_head, int64_t kp_row, const void* v_pages, int64_t vp_page,
                            int64_t vp_head, int64_t vp_row, int num_pages, int page_size, int kv_heads, int head_dim,
                            const int32_t* starts, const int32_t* lengths, const int32_t* table, int64_t table_stride,
                            int batch, int max_pages, float scale, int max_new, int64_t max_length, void* out,
                            int64_t o_t, int64_t o_h, int dtype, void* status, void* ws, size_t ws_bytes,
                            void* stream) {
  clear_error();
  AttendArgs a{};
  a.pages = {const_cast<void*>(k_pages), const_cast<void*>(v_pages), kp_page, kp_head, kp_row, vp_page, vp_head,
             vp_row, num_pages, 0, kv_heads};
  a.seqs = {starts, lengths, table, table_stride, batch, max_pages};
  if (int rc = check_pages("ppmoe_attend", a.pages, page_size, head_dim)) return rc;
  if (int rc = check_seqs("ppmoe_attend", a.seqs)) return rc;
  if (dtype != PPMOE_BF16 && dtype != PPMOE_F16) {
    set_error("ppmoe_attend: dtype=%d (0 bf16, 1 fp16)", dtype);
    return PPMOE_ERR_UNSUPPORTED;
  }
  if (tokens < 0 || q_heads < 1 || q_heads % kv_heads) {
    set_error("ppmoe_attend: tokens=%d, q_heads=%d must be a positive multiple of kv_heads=%d", tokens, q_heads,
              kv_heads);
    return PPMOE_ERR_INVALID_ARG;
  }
  if (tokens == 0) return PPMOE_OK;
  if (!q || !out || !status) {
    set_error("ppmoe_attend: null pointer");
    return PPMOE_ERR_INVALID_ARG;
  }
  while ((1 << a.pages.page_shift) < page_size) ++a.pages.page_shift;
  a.q = q;
  a.q_t = q_t;
  a.q_h = q_h;
  a.out = out;
  a.o_t = o_t;
  a.o_h = o_h;
  a.tokens = tokens;
  a.q_heads = q_heads;
  a.group = q_heads / kv_heads;
  a.scale = scale;
  a.status = static_cast<uint32_t*>(status);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == PPMOE_BF16)
    return head_dim == 128 ? launch<__nv_bfloat16, 128>(a, st) : launch<__nv_bfloat16, 64>(a, st);
  return head_dim == 128 ? launch<__half, 128>(a, st) : launch<__half, 64>(a, st);
}
