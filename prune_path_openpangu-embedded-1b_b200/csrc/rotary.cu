// Rotary position embedding of queries and keys (forward and gradient), and the append of new
// keys and values to a paged cache with the rotation applied on the way.
//
// Pair i of a head at position p turns by 2 pi p turns[i]:
//   y1 = g (x1 cos - x2 sin),  y2 = g (x2 cos + x1 sin)     (gradient: the same with -angle)
// The angle is reduced in fp64 (p turns[i] minus the nearest integer: up to |p| = 2^31 within 2^-21 radians) and its
// sine and cosine are taken in fp32; values are rounded once, at the store.
//
// Bound by memory: every value is read and written once.  Taking the angle from the position costs one
// fp64 product and one sincospi per pair and token, shared by all heads, and no table that would have
// to be read or sized.  Measured (bf16, 12 + 12 heads of 128, 16384 tokens, 201 MB): 37.0 us, 5.4 TB/s;
// (fp16, 32 + 8 heads of 128, half of each turned, 32768 tokens, 671 MB): 104.7 us, 6.4 TB/s.  Streaming
// loads and stores and CTAs of 2 tokens x 128 threads: 37.0 us; without the hints 41.1; 4 x 256: 38.5.
#include <cuda_fp16.h>
#include "seqs.cuh"

namespace ppmoe {

constexpr int kMaxPairs = 128;  // head_dim <= 256
constexpr int kRotThreads = 128;
constexpr int kRotTokens = 2;   // most tokens of one CTA

// One tensor of heads: rows of head_dim contiguous values; strides in elements.
struct HeadsView {
  const void* in;
  void* out;
  int64_t in_b, in_t, in_h, out_b, out_t, out_h;
  int heads;
};

struct RotaryArgs {
  HeadsView q, k, v;  // v: append only (copied)
  double turns[kMaxPairs];
  const void* positions;  // rotary only
  int64_t pos_b, pos_t;
  int pos64;
  int64_t length, tokens;  // rows of one sequence of the batch, of all
  int head_dim, pairs;     // rotated values: 2 * pairs of head_dim
  float gain, sign;
  int per_cta;
  Seqs seqs;    // append only
  Pages pages;  // append only
  uint32_t* status;
};

template <typename T, int V>
struct alignas(V == 1 ? alignof(T) : 16) Chunk {
  T x[V];
};
template <typename T, int V>
__device__ __forceinline__ Chunk<T, V> load_chunk(const T* p) {
  Chunk<T, V> c;
  if constexpr (V == 1) {
    c.x[0] = *p;
  } else {
    static_assert(sizeof(T) * V == 16, "16-byte chunks");
    *reinterpret_cast<uint4*>(c.x) = __ldcs(reinterpret_cast<const uint4*>(p));  // read once
  }
  return c;
}
template <int V>
__device__ __forceinline__ Chunk<float, V> load_angles(const float* p) {
  Chunk<float, V> c;
  if constexpr (V == 1) {
    c.x[0] = *p;
  } else {  // (V divides the pairs of a token)
#pragma unroll
    for (int i = 0; i < V; i += 4) *reinterpret_cast<float4*>(c.x + i) = *reinterpret_cast<const float4*>(p + i);
  }
  return c;
}
template <typename T, int V>
__device__ __forceinline__ void store_chunk(T* p, const Chunk<T, V>& c) {
  if constexpr (V == 1)
    *p = c.x[0];
  else
    __stcs(reinterpret_cast<uint4*>(p), *reinterpret_cast<const uint4*>(c.x));
}

// A unit is V pairs (two 16-byte chunks of a head, or 2 values where alignment allows no
// more): units [0, pairs / V) of a head are rotated, the rest copied.  A CTA takes a few tokens: offsets of
// their rows, sines and cosines once, into shared memory; then a thread keeps its place in the head and
// goes through (token, head) in equal steps, so that a unit costs no division.
template <typename T, int V, bool INTERLEAVED, bool APPEND>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const __grid_constant__ RotaryArgs a) {
  __shared__ __align__(16) float s_cos[kRotTokens * kMaxPairs], s_sin[kRotTokens * kMaxPairs];
  __shared__ long long s_pos[kRotTokens];
  __shared__ int64_t s_in[kRotTokens][3], s_out[kRotTokens][3];  // q, k, v: elements to the token's first head
  __shared__ bool s_skip[kRotTokens][3];                         // not stored
  const int tid = threadIdx.x;
  const int64_t t0 = (int64_t)blockIdx.x * a.per_cta;
  const int nt = (int)(a.tokens - t0 < a.per_cta ? a.tokens - t0 : a.per_cta);

  // a warp a token: its position and (append) its place in the cache
  static_assert(kRotThreads / 32 >= kRotTokens, "a warp a token");
  if (const int w = tid >> 5; w < nt) {
    const unsigned t = (unsigned)(t0 + w);
    const bool lead = (tid & 31) == 0;
    if constexpr (APPEND) {
      const int b = find_seq_warp(a.seqs.starts, a.seqs.batch, (int)t);
      if (lead) {
        const bool live = b >= 0 && b < a.seqs.batch;
        long long pos = 0;
        bool stored = false;
        if (live) {
          pos = (long long)a.seqs.lengths[b] - a.seqs.starts[b + 1] + t;
          const long long pi = pos >> a.pages.page_shift;
          int page = -1;
          if (pos >= 0 && pi < a.seqs.max_pages) page = a.seqs.table[b * a.seqs.table_stride + pi];
          stored = page >= 0 && page < a.pages.num_pages;
          if (stored) {
            const int64_t row = pos & ((1ll << a.pages.page_shift) - 1);
            s_out[w][1] = page * a.pages.k_page + row * a.pages.k_row;
            s_out[w][2] = page * a.pages.v_page + row * a.pages.v_row;
          } else {
            atomicOr(a.status, DEVERR_PAGE);
          }
        }
        s_pos[w] = pos;
        s_in[w][0] = t * a.q.in_t;
        s_in[w][1] = t * a.k.in_t;
        s_in[w][2] = t * a.v.in_t;
        s_out[w][0] = t * a.q.out_t;
        s_skip[w][0] = !live;
        s_skip[w][1] = s_skip[w][2] = !stored;
      }
    } else if (lead) {
      const unsigned b = t / (unsigned)a.length, l = t - b * (unsigned)a.length;
      const int64_t i = b * a.pos_b + l * a.pos_t;
      s_pos[w] = a.pos64 ? static_cast<const long long*>(a.positions)[i]
                         : (long long)static_cast<const int32_t*>(a.positions)[i];
      s_in[w][0] = b * a.q.in_b + l * a.q.in_t;
      s_in[w][1] = b * a.k.in_b + l * a.k.in_t;
      s_out[w][0] = b * a.q.out_b + l * a.q.out_t;
      s_out[w][1] = b * a.k.out_b + l * a.k.out_t;
    }
  }
  __syncthreads();
  for (int i = tid; i < nt * a.pairs; i += kRotThreads) {
    const int t = i / a.pairs, p = i - t * a.pairs;
    const double turn = (double)s_pos[t] * a.turns[p];
    float s, c;
    sincospif(2.f * (float)(turn - rint(turn)), &s, &c);
    s_cos[t * a.pairs + p] = c * a.gain;
    s_sin[t * a.pairs + p] = s * (a.gain * a.sign);
  }
  __syncthreads();

  const int units = a.head_dim / (2 * V);
  const int heads = a.q.heads + a.k.heads + (APPEND ? a.v.heads : 0);
  const int slots = kRotThreads / units;  // heads taken at once (units <= 128)
  const int slot = tid / units, u = tid - slot * units;
  if (slot >= slots) return;
  const bool turned = u < a.pairs / V;
  const int step_t = slots / heads, step_h = slots - step_t * heads;
  int t = slot / heads, h = slot - t * heads;
  for (; t < nt; t += step_t, h += step_h) {
    if (h >= heads) {
      h -= heads;
      if (++t >= nt) break;
    }
    // which tensor
    const int g = h < a.q.heads ? 0 : !APPEND || h < a.q.heads + a.k.heads ? 1 : 2;
    if (APPEND && s_skip[t][g]) continue;
    const T* in;
    T* out;
    if (g == 0) {
      in = static_cast<const T*>(a.q.in) + s_in[t][0] + h * a.q.in_h;
      out = static_cast<T*>(a.q.out) + s_out[t][0] + h * a.q.out_h;
    } else if (!APPEND || g == 1) {
      const int hh = h - a.q.heads;
      in = static_cast<const T*>(a.k.in) + s_in[t][1] + hh * a.k.in_h;
      out = APPEND ? static_cast<T*>(a.pages.k) + s_out[t][1] + hh * a.pages.k_head
                   : static_cast<T*>(a.k.out) + s_out[t][1] + hh * a.k.out_h;
    } else {
      const int hh = h - a.q.heads - a.k.heads;
      in = static_cast<const T*>(a.v.in) + s_in[t][2] + hh * a.v.in_h;
      out = static_cast<T*>(a.pages.v) + s_out[t][2] + hh * a.pages.v_head;
    }
    const bool rotate = turned && (!APPEND || g < 2);
    // element offsets of the unit's two chunks
    const int e1 = !INTERLEAVED && rotate ? u * V : u * 2 * V, e2 = !INTERLEAVED && rotate ? a.pairs + u * V : e1 + V;
    Chunk<T, V> x = load_chunk<T, V>(in + e1), y = load_chunk<T, V>(in + e2);
    if (rotate) {
      const Chunk<float, V> cs = load_angles<V>(s_cos + t * a.pairs + u * V), sn = load_angles<V>(s_sin + t * a.pairs + u * V);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        T& p1 = INTERLEAVED ? (2 * j < V ? x.x[2 * j] : y.x[2 * j - V]) : x.x[j];
        T& p2 = INTERLEAVED ? (2 * j + 1 < V ? x.x[2 * j + 1] : y.x[2 * j + 1 - V]) : y.x[j];
        const float f1 = to_f32<T>(p1), f2 = to_f32<T>(p2), c = cs.x[j], s = sn.x[j];
        p1 = from_f32<T>(f1 * c - f2 * s);
        p2 = from_f32<T>(f2 * c + f1 * s);
      }
    }
    store_chunk<T, V>(out + e1, x);
    store_chunk<T, V>(out + e2, y);
  }
}

template <typename T, int V, bool APPEND>
static int launch_v(RotaryArgs& a, bool interleaved, cudaStream_t st) {
  const int64_t ctas = (a.tokens + a.per_cta - 1) / a.per_cta;
  if (interleaved)
    rotary_kernel<T, V, true, APPEND><<<(unsigned)ctas, kRotThreads, 0, st>>>(a);
  else
    rotary_kernel<T, V, false, APPEND><<<(unsigned)ctas, kRotThreads, 0, st>>>(a);
  PPMOE_CHECK_CUDA(cudaGetLastError());
  return PPMOE_OK;
}

template <bool APPEND>
static int launch(RotaryArgs& a, bool interleaved, int dtype, bool wide, cudaStream_t st) {
  a.per_cta = a.tokens <= 1024 ? 1 : kRotTokens;  // (few tokens: as many SMs as there are)
  if (dtype == PPMOE_BF16)
    return wide ? launch_v<__nv_bfloat16, 8, APPEND>(a, interleaved, st)
                : launch_v<__nv_bfloat16, 1, APPEND>(a, interleaved, st);
  if (dtype == PPMOE_F16)
    return wide ? launch_v<__half, 8, APPEND>(a, interleaved, st) : launch_v<__half, 1, APPEND>(a, interleaved, st);
  if constexpr (!APPEND)
    return wide ? launch_v<float, 4, false>(a, interleaved, st) : launch_v<float, 1, false>(a, interleaved, st);
  return PPMOE_ERR_UNSUPPORTED;
}

// Whether every row of the view starts on a 16-byte boundary.
static bool wide_view(const void* p, int64_t sb, int64_t st, int64_t sh, int size) {
  const int64_t v = 16 / size;
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && sb % v == 0 && st % v == 0 && sh % v == 0;
}

static int check_rotation(const char* fn, int head_dim, const ppmoe_rotation* r, RotaryArgs& a) {
  const int rotary_dim = r ? r->rotary_dim : 0;
  if (head_dim < 2 || head_dim > 2 * kMaxPairs || head_dim % 2 || rotary_dim < 0 || rotary_dim > head_dim ||
      rotary_dim % 2) {
    set_error("%s: head_dim=%d must be even and in [2, %d], rotary_dim=%d even and in [0, head_dim]", fn, head_dim,
              2 * kMaxPairs, rotary_dim);
    return PPMOE_ERR_UNSUPPORTED;
  }
  a.head_dim = head_dim;
  a.pairs = rotary_dim / 2;
  a.gain = r ? (float)r->gain : 1.f;
  for (int i = 0; i < a.pairs; ++i) a.turns[i] = r->turns[i];
  return PPMOE_OK;
}

int check_cache(const char* fn, const ppmoe_kv_cache* c, Pages& p) {
  if (!c) {
    set_error("%s: null cache", fn);
    return PPMOE_ERR_INVALID_ARG;
  }
  if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1))) {
    set_error("%s: page_size=%d must be 16, 32, 64, 128 or 256", fn, c->page_size);
    return PPMOE_ERR_UNSUPPORTED;
  }
  if (c->head_dim != 64 && c->head_dim != 128) {
    set_error("%s: head_dim=%d must be 64 or 128", fn, c->head_dim);
    return PPMOE_ERR_UNSUPPORTED;
  }
  if (c->dtype != PPMOE_BF16 && c->dtype != PPMOE_F16) {
    set_error("%s: dtype=%d (0 bf16, 1 fp16)", fn, c->dtype);
    return PPMOE_ERR_UNSUPPORTED;
  }
  if (c->num_pages < 1 || c->kv_heads < 1) {
    set_error("%s: num_pages=%d and kv_heads=%d must be positive", fn, c->num_pages, c->kv_heads);
    return PPMOE_ERR_INVALID_ARG;
  }
  if (!c->k || !c->v || !c->status || !wide_view(c->k, c->k_page, c->k_head, c->k_row, 2) ||
      !wide_view(c->v, c->v_page, c->v_head, c->v_row, 2)) {
    set_error("%s: cache tensors must be non-null, 16-byte aligned, with strides of whole 16 bytes", fn);
    return PPMOE_ERR_INVALID_ARG;
  }
  p = {c->k, c->v, c->k_page, c->k_head, c->k_row, c->v_page, c->v_head, c->v_row, c->num_pages, 0, c->kv_heads};
  while ((1 << p.page_shift) < c->page_size) ++p.page_shift;
  return PPMOE_OK;
}

int check_seqs(const char* fn, const Seqs& s) {
  if (s.batch < 1 || s.max_pages < 1) {
    set_error("%s: batch=%d and max_pages=%d must be positive", fn, s.batch, s.max_pages);
    return PPMOE_ERR_INVALID_ARG;
  }
  if (!s.starts || !s.lengths || !s.table) {
    set_error("%s: null starts, lengths or table", fn);
    return PPMOE_ERR_INVALID_ARG;
  }
  return PPMOE_OK;
}

}  // namespace ppmoe

using namespace ppmoe;

extern "C" int ppmoe_rotary(const ppmoe_rotation* rotation, int inverse, const void* q, int64_t q_b, int64_t q_t,
                            int64_t q_h, void* q_out, int64_t qo_b, int64_t qo_t, int64_t qo_h, int q_heads,
                            const void* k, int64_t k_b, int64_t k_t, int64_t k_h, void* k_out, int64_t ko_b,
                            int64_t ko_t, int64_t ko_h, int k_heads, int batch, int64_t length, int head_dim,
                            const void* positions, int positions64, int64_t pos_b, int64_t pos_t, int dtype,
                            void* stream) {
  clear_error();
  RotaryArgs a{};
  if (!rotation) {
    set_error("ppmoe_rotary: null rotation");
    return PPMOE_ERR_INVALID_ARG;
  }
  if (int rc = check_rotation("ppmoe_rotary", head_dim, rotation, a)) return rc;
  if (dtype != PPMOE_BF16 && dtype != PPMOE_F16 && dtype != PPMOE_F32) {
    set_error("ppmoe_rotary: dtype=%d (0 bf16, 1 fp16, 2 fp32)", dtype);
    return PPMOE_ERR_UNSUPPORTED;
  }
  if (batch < 0 || length < 0 || q_heads < 0 || k_heads < 0 || (batch > 0 && length > (int64_t)INT32_MAX / batch)) {
    set_error("ppmoe_rotary: batch=%d, length=%lld (batch * length < 2^31), q_heads=%d, k_heads=%d", batch,
              (long long)length, q_heads, k_heads);
    return PPMOE_ERR_INVALID_ARG;
  }
  if ((int64_t)(q_heads + (int64_t)k_heads) * head_dim > (1 << 24)) {
    set_error("ppmoe_rotary: %d + %d heads of %d are too many", q_heads, k_heads, head_dim);
    return PPMOE_ERR_UNSUPPORTED;
  }
  a.tokens = batch * length;
  if (a.tokens == 0 || q_heads + k_heads == 0) return PPMOE_OK;
  if (!positions || (q_heads && (!q || !q_out)) || (k_heads && (!k || !k_out))) {
    set_error("ppmoe_rotary: null pointer");
    return PPMOE_ERR_INVALID_ARG;
  }
  const int size = dtype == PPMOE_F32 ? 4 : 2, v = 16 / size;
  a.q = {q, q_out, q_b, q_t, q_h, qo_b, qo_t, qo_h, q_heads};
  a.k = {k, k_out, k_b, k_t, k_h, ko_b, ko_t, ko_h, k_heads};
  a.positions = positions;
  a.pos64 = positions64;
  a.pos_b = pos_b;
  a.pos_t = pos_t;
  a.length = length;
  a.sign = inverse ? -1.f : 1.f;
  const bool wide = head_dim % (2 * v) == 0 && rotation->rotary_dim % (2 * v) == 0 &&
                    (!q_heads || (wide_view(q, q_b, q_t, q_h, size) && wide_view(q_out, qo_b, qo_t, qo_h, size))) &&
                    (!k_heads || (wide_view(k, k_b, k_t, k_h, size) && wide_view(k_out, ko_b, ko_t, ko_h, size)));
  return launch<false>(a, rotation->interleaved != 0, dtype, wide, static_cast<cudaStream_t>(stream));
}

extern "C" int ppmoe_kv_append(const ppmoe_kv_cache* cache, const ppmoe_rotation* rotation, const void* q, int64_t q_t,
                               int64_t q_h, void* q_out, int64_t qo_t, int64_t qo_h, int q_heads, const void* k,
                               int64_t k_t, int64_t k_h, const void* v, int64_t v_t, int64_t v_h, int tokens,
                               const int32_t* starts, const int32_t* lengths, const int32_t* table,
                               int64_t table_stride, int batch, int max_pages, void* stream) {
  clear_error();
  RotaryArgs a{};
  a.seqs = {starts, lengths, table, table_stride, batch, max_pages};
  if (int rc = check_cache("ppmoe_kv_append", cache, a.pages)) return rc;
  if (int rc = check_rotation("ppmoe_kv_append", cache->head_dim, rotation, a)) return rc;
  if (int rc = check_seqs("ppmoe_kv_append", a.seqs)) return rc;
  const int kv_heads = cache->kv_heads, head_dim = cache->head_dim;
  if (tokens < 0 || q_heads < 0 || (int64_t)(q_heads + 2ll * kv_heads) * head_dim > (1 << 24)) {
    set_error("ppmoe_kv_append: tokens=%d, q_heads=%d, kv_heads=%d", tokens, q_heads, kv_heads);
    return PPMOE_ERR_INVALID_ARG;
  }
  if (tokens == 0) return PPMOE_OK;
  if (!k || !v || (q_heads && (!q || !q_out))) {
    set_error("ppmoe_kv_append: null pointer");
    return PPMOE_ERR_INVALID_ARG;
  }
  a.q = {q, q_out, 0, q_t, q_h, 0, qo_t, qo_h, q_heads};
  a.k = {k, nullptr, 0, k_t, k_h, 0, 0, 0, kv_heads};
  a.v = {v, nullptr, 0, v_t, v_h, 0, 0, 0, kv_heads};
  a.length = a.tokens = tokens;
  a.sign = 1.f;
  a.status = static_cast<uint32_t*>(cache->status);
  const bool wide = a.pairs % 8 == 0 && wide_view(k, 0, k_t, k_h, 2) && wide_view(v, 0, v_t, v_h, 2) &&
                    (!q_heads || (wide_view(q, 0, q_t, q_h, 2) && wide_view(q_out, 0, qo_t, qo_h, 2)));
  return launch<true>(a, rotation && rotation->interleaved, cache->dtype, wide, static_cast<cudaStream_t>(stream));
}
