// Causal attention of each sequence's newest tokens over a paged key/value cache.
//
//   out[t, h] = sum_{j <= p(t)} w_j v_j,  w = softmax_j(scale q[t, h] . k_j),  p(t) = position of t
// and 0 where no key is left (p(t) < 0).
//
// All query rows of a sequence that read one kv head (its new tokens x the `group` query heads of
// that head) are one matrix of n * group rows; row r is token r / group, head r % group of the group.
// Scores are kept in base 2: x = c q.k with c = |scale| log2 e (a negative scale turns the sign of
// q, which is exact), w = 2^(x - m) / sum.  One pass over the keys keeps the running maximum m
// and sum l in fp32; weights are rounded once to the cache's type for the second product.
//
// A masked key must not reach a row even where its value is not finite (0 * inf = NaN): tiles that
// some row sees in part are searched for such values.  They are taken out of the product, and
// added (they are what the sum becomes) to the rows that see their key.  In other tiles the product carries them, but an
// infinity under a weight, or a running sum's factor, that vanished in its type becomes NaN there: sums that are NaN
// over weights that are not are put right at the end from a list of the values that are not finite, so
// that an answer does not depend on the tiles, parts and order it was computed in.
#include "attend.cuh"

namespace ppmoe {

// ======================================================================== few rows
// Up to 16 rows at a time per (sequence, kv head), or 32 of 64 values: one token per sequence up to a few.  Bound by
// the cache's bytes.  Each warp takes 32 keys at a time through a ring of its own (cp.async, no block
// barrier), m16n8k16 products (rows padded to 16: the tensor pipe has room, it is the loads that
// count), and the warps' and then the parts' (m, l, sum) are joined at the end.
// 64 ragged sequences of up to 8192 keys move 1.144 GB (counted: 1.143 read) in 190 us, 6.0 TB/s; two of 131071
// 1.073 GB in 173 us, 6.2 TB/s.  Short ones are bound by latency: one of 640 keys takes 7 us on the device.
// Small CTAs, several to an SM, so that one's start and end hide behind the others' loads: 64 ragged
// sequences of up to 8192 keys, 32 query and 8 kv heads of 128, in us: 2 warps x 2 stages (3 CTAs an SM) 196,
// 2 x 3 (2) 220, 4 x 3 (1) 235, 1 x 2 (6) 229 (before the clusters).
constexpr int kThinWarps = 2;

template <int D, int MT>  // MT: row tiles of 16 (two of 64 values: with 128 the sums alone fill the registers)
struct ThinShape {
  static_assert(MT == 1 || D == 64, "one row tile of 128 values");
  static constexpr int kKeys = 32;
  static constexpr int kStages = D == 128 ? 2 : 3;
  static constexpr int kCtas = 3;  // per SM
  static constexpr int kTile = kKeys * D * 2;          // bytes of K (or V) of one stage
  static constexpr int kWarp = kStages * 2 * kTile;    // bytes of one warp's ring
  static constexpr int kQ = MT * 16 * D * 2;
  static constexpr int kJoin = (kThinWarps * (D + 4 + 2) + 2) * MT * 16 * 4;
  static constexpr int kBytes = kQ + (kThinWarps * kWarp > kJoin ? kThinWarps * kWarp : kJoin);
};

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Parts of a (sequence, kv head) that are one cluster (2 to 8) meet in shared memory: no workspace, no
// second launch.
constexpr int kMaxCluster = 8;
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t at) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_cluster2(uint32_t at) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
  return v;
}

template <typename T, int D, int MT>
__global__ void __launch_bounds__(kThinWarps * 32, ThinShape<D, MT>::kCtas)
attend_thin_kernel(const __grid_constant__ AttendArgs a) {
  extern __shared__ __align__(1024) uint8_t smem[];
  using S = ThinShape<D, MT>;
  constexpr int KEYS = S::kKeys, STAGES = S::kStages, R = 16 * MT;
  constexpr int KN = KEYS / 8;   // n-tiles of the scores
  constexpr int KS = D / 16;     // k-steps of q.k
  constexpr int NT = D / 8;      // n-tiles of the output
  constexpr int CH = D / 8;      // 16-byte chunks of a row
  constexpr int RPI = 32 / CH;   // rows one copy instruction of the warp takes
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int split = blockIdx.x % a.nsplit;
  const int kvh = (blockIdx.x / a.nsplit) % a.pages.kv_heads;
  const int b = blockIdx.x / (a.nsplit * a.pages.kv_heads);
  if (a.joins) pdl_launch_dependents();
  const Seq sq = load_seq(a, b);
  if (sq.rows <= 0) return;
  const int cap = key_cap(a, sq.length);
  if (cap < sq.length && tid == 0) atomicOr(a.status, DEVERR_PAGE);
  const int pos0 = sq.length - (a.seqs.starts[b + 1] - a.seqs.starts[b]);  // position of row 0
  const int rows = sq.rows * a.group;
  const int32_t* table = a.seqs.table + b * a.seqs.table_stride;
  const int shift = a.pages.page_shift;
  const uint32_t q_s = smem_u32(smem), ring = q_s + S::kQ + warp * S::kWarp;
  float* j_o = reinterpret_cast<float*>(smem + S::kQ);  // [warps][R][D + 4]
  float* j_ml = j_o + kThinWarps * R * (D + 4);         // [warps][R][2]
  float* c_ml = j_ml + kThinWarps * R * 2;              // [R][2]: of all warps, for the cluster
  const bool clustered = a.nsplit > 1 && a.nsplit <= kMaxCluster, joined = a.nsplit > kMaxCluster;  // how parts meet
  static_assert(S::kQ >= 3 * D * 4, "room for the list of values that are not finite");

  for (int r0 = 0; r0 < rows; r0 += R) {
    const int last = r0 + R - 1 < rows ? r0 + R - 1 : rows - 1;
    const int pos_lo = pos0 + r0 / a.group, pos_hi = pos0 + last / a.group;
    const int keys = pos_hi + 1 < cap ? pos_hi + 1 : cap;  // keys some row sees
    const int blocks = keys > 0 ? (keys + KEYS - 1) / KEYS : 0;
    const int per = (blocks + a.nsplit - 1) / a.nsplit;
    const int blk_end = min(blocks, (split + 1) * per);
    int blk = split * per + warp;

    // this thread's rows (lane / 4 and that + 8 of each tile): how far they see (-1: nothing)
    int lim[MT][2];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = r0 + t * 16 + (lane >> 2) + 8 * i;
        lim[t][i] = r < rows ? min(pos0 + r / a.group, cap - 1) : -1;
      }
    }
    // q to shared memory, behind the first keys' page numbers
#pragma unroll
    for (int i = tid; i < R * CH; i += kThinWarps * 32) {
      const int row = i / CH, c = i % CH, r = r0 + row, tok = r / a.group;
      const bool real = r < rows;
      const T* p = static_cast<const T*>(a.q);
      if (real) p += (int64_t)(sq.first + tok) * a.q_t + (int64_t)(kvh * a.group + r - tok * a.group) * a.q_h + c * 8;
      const uint32_t d = q_s + row * (D * 2) + ((c ^ (row & 7)) << 4);
      if (a.q_wide16 && a.q_sign > 0) {
        cp_async16_or_zero(d, p, real);
      } else {
        uint32_t v[4] = {0, 0, 0, 0};
        if (real) {
          const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = q_pair<T>(h[2 * e] | (uint32_t)h[2 * e + 1] << 16, a.q_sign);
        }
        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(d), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
      }
    }
    cp_async_commit();

    // pages of a block's sixteens of keys (pages have 16 rows or more)
    constexpr int NP = KEYS / 16;
    auto ids = [&](int bk, int (&page)[NP]) {
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int key = bk * KEYS + i * 16;
        page[i] = bk < blk_end && key < keys ? __ldg(table + (key >> shift)) : -1;
      }
    };
    auto fetch = [&](int bk, int stage, const int (&page)[NP]) {
      if (bk < blk_end) {
        const int key = bk * KEYS;
        const uint32_t kd = ring + stage * 2 * S::kTile, vd = kd + S::kTile;
        const int c = lane % CH, rr = lane / CH;
        const T* k0 = static_cast<const T*>(a.pages.k) + kvh * a.pages.k_head + c * 8;
        const T* v0 = static_cast<const T*>(a.pages.v) + kvh * a.pages.v_head + c * 8;
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          const bool ok = (uint32_t)page[p] < (uint32_t)a.pages.num_pages;
          if (lane == 0 && !ok && key + p * 16 < keys) atomicOr(a.status, DEVERR_PAGE);
          const int in = (key + p * 16) & ((1 << shift) - 1);
          const T* kp = k0 + (ok ? page[p] * a.pages.k_page + (in + rr) * a.pages.k_row : 0);
          const T* vp = v0 + (ok ? page[p] * a.pages.v_page + (in + rr) * a.pages.v_row : 0);
#pragma unroll
          for (int i = 0; i < 16 / RPI; ++i) {
            const int row = p * 16 + i * RPI + rr;
            const bool real = ok && key + row < keys;
            const uint32_t d = row * (D * 2) + ((c ^ (row & 7)) << 4);
            cp_async16_or_zero(kd + d, kp + (real ? i * RPI * a.pages.k_row : 0), real);
            cp_async16_or_zero(vd + d, vp + (real ? i * RPI * a.pages.v_row : 0), real);
          }
        }
      }
      cp_async_commit();
    };

    float o[MT][NT][4], m[MT][2], l[MT][2];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      m[t][0] = m[t][1] = -CUDART_INF_F;
      l[t][0] = l[t][1] = 0.f;
#pragma unroll
      for (int n = 0; n < NT; ++n) o[t][n][0] = o[t][n][1] = o[t][n][2] = o[t][n][3] = 0.f;
    }

    int page[NP];
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) {
      ids(blk + s * kThinWarps, page);
      fetch(blk + s * kThinWarps, s, page);
    }
    ids(blk + (STAGES - 1) * kThinWarps, page);
    cp_async_wait<STAGES - 1>();  // q
    __syncthreads();
    uint32_t qf[MT == 1 ? KS : 1][4];
    auto load_q = [&](uint32_t (&f)[4], int t, int k) {
      const int row = t * 16 + (lane & 15), ch = k * 2 + (lane >> 4);
      ldsm4(f, q_s + row * (D * 2) + ((ch ^ (row & 7)) << 4));
    };
    if constexpr (MT == 1) {
#pragma unroll
      for (int k = 0; k < KS; ++k) load_q(qf[k], 0, k);
    }
    int stage = 0;
#pragma unroll 1
    for (; blk < blk_end; blk += kThinWarps) {
      {
        const int ahead = blk + (STAGES - 1) * kThinWarps;
        int st = stage + STAGES - 1;
        if (st >= STAGES) st -= STAGES;
        fetch(ahead, st, page);
        ids(ahead + kThinWarps, page);
      }
      cp_async_wait<STAGES - 1>();
      __syncwarp();
      const uint32_t kd = ring + stage * 2 * S::kTile, vd = kd + S::kTile;
      const int key = blk * KEYS;

      float s[MT][KN][4];
#pragma unroll
      for (int t = 0; t < MT; ++t) {
#pragma unroll
        for (int n = 0; n < KN; ++n) s[t][n][0] = s[t][n][1] = s[t][n][2] = s[t][n][3] = 0.f;
      }
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        uint32_t qk[MT][4];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          if constexpr (MT == 1) {
#pragma unroll
            for (int e = 0; e < 4; ++e) qk[t][e] = qf[k][e];
          } else {
            load_q(qk[t], t, k);
          }
        }
#pragma unroll
        for (int h = 0; h < KN / 2; ++h) {
          // matrices: keys h*16 + 0..7 (two k halves), then keys + 8
          const int row = h * 16 + (lane & 7) + ((lane >> 4) << 3);
          const int ch = k * 2 + ((lane >> 3) & 1);
          uint32_t f[4];
          ldsm4(f, kd + row * (D * 2) + ((ch ^ (row & 7)) << 4));
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            mma16<T>(s[t][2 * h], qk[t], f[0], f[1]);
            mma16<T>(s[t][2 * h + 1], qk[t], f[2], f[3]);
          }
        }
      }
      const bool partly = key + KEYS > pos_lo + 1 || key + KEYS > keys;
      uint32_t pf[MT][KN / 2][4];
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        float mx[2] = {m[t][0], m[t][1]};
#pragma unroll
        for (int n = 0; n < KN; ++n) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s[t][n][i] *= a.c;
            if (partly && key + n * 8 + (lane & 3) * 2 + (i & 1) > lim[t][i >> 1]) s[t][n][i] = -CUDART_INF_F;
            mx[i >> 1] = fmaxf(mx[i >> 1], s[t][n][i]);
          }
        }
#pragma unroll
        for (int x = 1; x < 4; x <<= 1) {
          mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], x));
          mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], x));
        }
        if (__any_sync(0xffffffffu, mx[0] > m[t][0] || mx[1] > m[t][1])) {
          // old sums to the new maxima (a row without keys so far has sums of 0)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float f = m[t][i] == -CUDART_INF_F ? 0.f : exp2_ftz(m[t][i] - mx[i]);
            l[t][i] *= f;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              o[t][n][2 * i] *= f;
              o[t][n][2 * i + 1] *= f;
            }
            m[t][i] = mx[i];
          }
        }
        const float sub[2] = {(m[t][0] == -CUDART_INF_F ? 0.f : m[t][0]) - kLift<T>,
                              (m[t][1] == -CUDART_INF_F ? 0.f : m[t][1]) - kLift<T>};
#pragma unroll
        for (int n = 0; n < KN; ++n) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float e0 = exp2_ftz(s[t][n][2 * i] - sub[i]), e1 = exp2_ftz(s[t][n][2 * i + 1] - sub[i]);
            l[t][i] += e0 + e1;
            pf[t][n >> 1][(n & 1) * 2 + i] = pack2<T>(e0, e1);
          }
        }
      }
      if (partly) {  // values that are not finite, of keys that some row does not see
        uint32_t bad = 0;
#pragma unroll 4
        for (int i = lane; i < KEYS * CH; i += 32) {
          uint4 v;
          asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(vd + i * 16) : "memory");
          bad |= not_finite2<T>(v.x) | not_finite2<T>(v.y) | not_finite2<T>(v.z) | not_finite2<T>(v.w);
        }
        if (__any_sync(0xffffffffu, bad != 0)) {
#pragma unroll 1
          for (int j = 0; j < KEYS; ++j) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const uint32_t at = vd + j * (D * 2) + ((n ^ (j & 7)) << 4) + (lane & 3) * 4;
              uint32_t v;
              asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
              __syncwarp();
              uint32_t keep = v;
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const uint16_t bits = (uint16_t)(v >> (16 * e));
                if (not_finite16<T>(bits)) {
                  const float f = to_f32<T>(*reinterpret_cast<const T*>(&bits));
#pragma unroll
                  for (int t = 0; t < MT; ++t) {
                    if (key + j <= lim[t][0]) o[t][n][e] += f;
                    if (key + j <= lim[t][1]) o[t][n][2 + e] += f;
                  }
                  keep &= e ? 0xffffu : 0xffff0000u;
                }
              }
              if (lane < 4 && keep != v) asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(keep) : "memory");
            }
          }
          __syncwarp();
        }
      }
#pragma unroll
      for (int h = 0; h < KN / 2; ++h) {
#pragma unroll
        for (int n = 0; n < NT; n += 2) {
          // matrices: keys h*16 + 0..7 and + 8 of columns n, then of columns n + 1
          const int row = h * 16 + (lane & 15), ch = n + (lane >> 4);
          uint32_t f[4];
          ldsm4_t(f, vd + row * (D * 2) + ((ch ^ (row & 7)) << 4));
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            mma16<T>(o[t][n], pf[t][h], f[0], f[1]);
            mma16<T>(o[t][n + 1], pf[t][h], f[2], f[3]);
          }
        }
      }
      __syncwarp();
      stage = stage + 1 == STAGES ? 0 : stage + 1;
    }
    cp_async_wait<0>();
    __syncthreads();  // every warp is through with its ring
#pragma unroll
    for (int t = 0; t < MT; ++t) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float sum = l[t][i];
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        const int row = warp * R + t * 16 + (lane >> 2) + 8 * i;
        float* to = j_o + row * (D + 4) + (lane & 3) * 2;
#pragma unroll
        for (int n = 0; n < NT; ++n) *reinterpret_cast<float2*>(to + n * 8) = make_float2(o[t][n][2 * i], o[t][n][2 * i + 1]);
        if ((lane & 3) == 0) *reinterpret_cast<float2*>(j_ml + row * 2) = make_float2(m[t][i], sum);
      }
    }
    __syncthreads();
    uint32_t mend = 0;  // which of this thread's pieces of 8 columns have sums that are NaN over weights that are not
    {
      constexpr int TPR = kThinWarps * 32 / R, C = D / TPR;  // threads of a row, columns of one thread
      const int row = tid / TPR, col = (tid % TPR) * C, r = r0 + row;
      if (r < rows) {
        float top = -CUDART_INF_F, sum = 0.f, f[kThinWarps];
#pragma unroll
        for (int w = 0; w < kThinWarps; ++w) top = fmaxf(top, j_ml[(w * R + row) * 2]);
#pragma unroll
        for (int w = 0; w < kThinWarps; ++w) {
          const float mw = j_ml[(w * R + row) * 2];
          f[w] = mw == -CUDART_INF_F ? 0.f : exp2_ftz(mw - top);
          sum += f[w] * j_ml[(w * R + row) * 2 + 1];
        }
        const int tok = r / a.group;
        const int64_t t = sq.first + tok;
        const int h = kvh * a.group + r - tok * a.group;
        const int64_t at = ((int64_t)split * a.tokens + t) * a.q_heads + h;
        const float inv = inverse_sum(sum, pos0 + tok);
#pragma unroll 1
        for (int c = col; c < col + C; c += 8) {
          float acc[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            acc[i] = 0.f;
#pragma unroll
            for (int w = 0; w < kThinWarps; ++w) acc[i] += f[w] * j_o[(w * R + row) * (D + 4) + c + i];
          }
          if (any_nan(acc) && (sum > 0.f || (sum == 0.f && joined))) mend |= 1u << ((c - col) / 8);
          if (!clustered && !joined) {
            store_row<T>(static_cast<T*>(a.out) + t * a.o_t + h * a.o_h + c, acc, inv, a.o_wide);
          } else if (clustered) {  // (over what this thread alone has read)
            *reinterpret_cast<float4*>(j_o + row * (D + 4) + c) = make_float4(acc[0], acc[1], acc[2], acc[3]);
            *reinterpret_cast<float4*>(j_o + row * (D + 4) + c + 4) = make_float4(acc[4], acc[5], acc[6], acc[7]);
          } else {
            *reinterpret_cast<float4*>(a.part_o + at * D + c) = make_float4(acc[0], acc[1], acc[2], acc[3]);
            *reinterpret_cast<float4*>(a.part_o + at * D + c + 4) = make_float4(acc[4], acc[5], acc[6], acc[7]);
          }
        }
        if (a.nsplit > 1 && col == 0)
          *reinterpret_cast<float2*>(clustered ? c_ml + row * 2 : a.part_ml + at * 2) = make_float2(top, sum);
      }
    }
    if (clustered) {
      mend = 0;
      cluster_sync();
      const int n = min(R, rows - r0) * (D / 8);  // pieces of 8 columns, shared out over the cluster's threads
      for (int i = tid + split * kThinWarps * 32, at = 1; i < n; i += a.nsplit * kThinWarps * 32, at <<= 1) {
        const int row = i / (D / 8), c = i % (D / 8) * 8, r = r0 + row;
        // (parts past the last read the last again and count nothing: all loads are in flight at once)
        float2 ml[kMaxCluster];
        float4 x[kMaxCluster], y[kMaxCluster];
#pragma unroll
        for (int w = 0; w < kMaxCluster; ++w) {
          const int from = min(w, a.nsplit - 1);
          ml[w] = ld_cluster2(mapa_u32(c_ml + row * 2, from));
          const uint32_t at = mapa_u32(j_o + row * (D + 4) + c, from);
          x[w] = ld_cluster4(at);
          y[w] = ld_cluster4(at + 16);
        }
        float top = -CUDART_INF_F, sum = 0.f, acc[8] = {};
#pragma unroll
        for (int w = 0; w < kMaxCluster; ++w) top = fmaxf(top, ml[w].x);
#pragma unroll
        for (int w = 0; w < kMaxCluster; ++w) {
          // (a part without a score above -inf has sums of 0, or NaN where a score or a value made them so)
          const float f = ml[w].x == -CUDART_INF_F ? 1.f : exp2_ftz(ml[w].x - top);
          if (w < a.nsplit) {
            sum += f * ml[w].y;
            acc[0] += f * x[w].x;
            acc[1] += f * x[w].y;
            acc[2] += f * x[w].z;
            acc[3] += f * x[w].w;
            acc[4] += f * y[w].x;
            acc[5] += f * y[w].y;
            acc[6] += f * y[w].z;
            acc[7] += f * y[w].w;
          }
        }
        if (any_nan(acc) && sum > 0.f) mend |= at;
        const int tok = r / a.group;
        store_row<T>(static_cast<T*>(a.out) + (sq.first + tok) * a.o_t + (int64_t)(kvh * a.group + r - tok * a.group) * a.o_h + c,
                        acc, inverse_sum(sum, pos0 + tok), a.o_wide);
      }
      cluster_sync();  // every part has been read
    }
    if (__syncthreads_or(mend != 0)) {  // (and before the next rows' copies)
      int* list = reinterpret_cast<int*>(smem);  // where q was
      const int from = joined ? min(split * per * KEYS, keys) : 0, to = joined ? min(blk_end * KEYS, keys) : keys;
      list_values<T, D, kThinWarps * 32>(a, b, kvh, from, to, list);
      for (int p = 0; mend >> p; ++p) {
        if (!(mend >> p & 1)) continue;
        constexpr int TPR = kThinWarps * 32 / R;
        const int piece = clustered ? tid + (split + p * a.nsplit) * kThinWarps * 32 : 0;
        const int row = clustered ? piece / (D / 8) : tid / TPR;
        const int col = clustered ? piece % (D / 8) * 8 : tid % TPR * (D / TPR) + p * 8;
        const int r = r0 + row;
        mend_row<T, D>(a, list, sq.first, r, kvh, joined ? split : -1, min(pos0 + r / a.group, cap - 1), col, 8);
      }
      __syncthreads();
    }
  }
}

// ======================================================================== joining the parts
// out = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s: a CTA per (token, head), its warps taking the parts in
// turn and meeting in warp order, so the order of every sum is fixed.
constexpr int kJoinWarps = 4;
template <typename T, int D>
__global__ void __launch_bounds__(kJoinWarps * 32) attend_join_kernel(const __grid_constant__ AttendArgs a) {
  constexpr int C = D / 32;
  __shared__ float s_o[kJoinWarps][D], s_l[kJoinWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t item = blockIdx.x, items = gridDim.x;
  const int t = (int)(item / a.q_heads), h = (int)(item - (int64_t)t * a.q_heads);
  const int first = a.seqs.starts[0], end = a.seqs.starts[a.seqs.batch];
  pdl_wait();  // the parts are complete and visible
  if (t < first || t >= end) return;
  float m = -CUDART_INF_F, mine[4], ls[4];  // this lane's parts: lane, lane + 32, ... (128 at most)
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int s = lane + 32 * i;
    const float2 v = s < a.nsplit ? *reinterpret_cast<const float2*>(a.part_ml + (s * items + item) * 2)
                                  : make_float2(-CUDART_INF_F, 0.f);
    mine[i] = v.x;
    ls[i] = v.y;
    m = fmaxf(m, v.x);
  }
  m = warp_max(m);
  float l = 0.f, acc[C];
#pragma unroll
  for (int i = 0; i < C; ++i) acc[i] = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    mine[i] = mine[i] == -CUDART_INF_F ? 0.f : exp2_ftz(mine[i] - m);  // the part's factor
    const int n = min(32, a.nsplit - 32 * i);
#pragma unroll 4
    for (int s = warp; s < n; s += kJoinWarps) {
      const float f = __shfl_sync(0xffffffffu, mine[i], s);
      l += f * __shfl_sync(0xffffffffu, ls[i], s);
      const float* p = a.part_o + ((s + 32 * i) * items + item) * D + lane * C;
      if constexpr (C == 4) {
        const float4 v = *reinterpret_cast<const float4*>(p);
        acc[0] += f * v.x;
        acc[1] += f * v.y;
        acc[2] += f * v.z;
        acc[3] += f * v.w;
      } else {
        const float2 v = *reinterpret_cast<const float2*>(p);
        acc[0] += f * v.x;
        acc[1] += f * v.y;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < C; ++i) s_o[warp][lane * C + i] = acc[i];
  if (lane == 0) s_l[warp] = l;
  __syncthreads();
  l = 0.f;
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) l += s_l[w];
  int pos = 0;
  if (l == 0.f) {  // (all threads alike)
    const int b = find_seq_warp(a.seqs.starts, a.seqs.batch, t);
    pos = a.seqs.lengths[b] - a.seqs.starts[b + 1] + t;
  }
  const float inv = inverse_sum(l, pos);
  T* out = static_cast<T*>(a.out) + t * a.o_t + h * a.o_h;
  for (int c = threadIdx.x; c < D; c += kJoinWarps * 32) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) v += s_o[w][c];
    if (v != v && l > 0.f) {  // an infinity in a part whose factor vanished, perhaps: it stays one
      v = 0.f;
      for (int s = 0; s < a.nsplit; ++s) {
        const float ms = a.part_ml[(s * items + item) * 2], x = a.part_o[(s * items + item) * D + c];
        const float f = ms == -CUDART_INF_F ? 0.f : exp2_ftz(ms - m);
        v += f == 0.f && fabsf(x) == CUDART_INF_F ? x : f * x;
      }
    }
    out[c] = from_f32<T>(v * inv);
  }
}

// ======================================================================== host
struct Plan {
  int tiles;   // 128-row tiles of a CTA (1 or 2); 0: the kernel for few rows
  int groups;  // CTAs' worth of row tiles of the longest sequence; few rows: 16-row tiles taken at once (1 or 2)
  int nsplit;  // parts the keys of a (sequence, kv head) are cut into
};

static Plan make_plan(int tokens, int q_heads, int kv_heads, int head_dim, int batch, int max_new, int64_t max_length) {
  auto up = [](int64_t x, int64_t y) { return (x + y - 1) / y; };
  const int64_t rows = (int64_t)max_new * (q_heads / kv_heads), base = (int64_t)batch * kv_heads;
  Plan p;
  // Few rows, where the other kernel's tiles would be empty for the most part: 24 ragged sequences x 5 tokens over up to
  // 4000 keys, in us, here and there: 20 rows of 64 values 23 and 39; of 128 (8 kv heads) 65 (two row
  // tiles at once, 16 keys at a time) and 57.
  if (rows <= (head_dim == 64 ? 32 : 16)) {
    // Parts of 128 keys (two blocks of each warp) as far as they make two CTAs an SM, since there latency
    // counts; parts of 768 as far as they make 1184 CTAs, so that ragged lengths even out; whichever are more.
    p.tiles = 0;
    p.groups = rows <= 16 ? 1 : 2;
    const int64_t n1 = std::min(up(max_length, 128), up(296, base));
    const int64_t n2 = std::min(up(max_length, 768), up(1184, base));
    p.nsplit = (int)std::max<int64_t>(1, std::min<int64_t>(128, std::max(n1, n2)));
  } else {
    // (A CTA goes on to further groups where there are fewer CTAs than groups: batches so wide that most
    // of a larger grid would find nothing to do.)
    // One tile to a CTA (two CTAs to an SM) for few rows, and for so few keys that a CTA's start and end weigh more
    // than its loop: prompts of 12 heads of 128, in us, with one and with two: 16 of 256 20.7 and 24.7, 16 of 512 39 and
    // 41 (of 64: 31 and 35), 8 of 1024 50.5 and 49.9, 4 of 2048 72.8 and 69.2; 2048 rows over 34816 keys 1134 and 999.
    p.tiles = rows <= 128 || max_length <= 768 ? 1 : 2;
    p.groups = (int)std::min(up(rows, 128 * p.tiles), std::max<int64_t>(1, (1 << 18) / base));
    // Parts where they fill the last wave better than they cost: measured us of a block of keys and of a CTA's start
    // and end, and the parts' way through memory at 5 TB/s (2048 rows x 32 heads: 1030 us in one part, 1085 in four,
    // so a gain of less than a tenth is left alone).
    const double block = p.tiles == 2 ? 1.65 : 1.07, ends = p.tiles == 2 ? 6. : 5.;
    const int64_t slots = p.tiles == 2 ? 148 : 296, blocks = up(max_length, 64 * p.tiles);
    double best = 0.;
    for (int n = 1; n <= 32 && (n == 1 || n * 512 <= max_length); ++n) {
      const double t = up(base * p.groups * n, slots) * (up(blocks, n) * block + ends);
      const double all = n == 1 ? t : 1.1 * t + 4. + n * (tokens * 1e-6 * q_heads * head_dim * 8. / 5.);
      if (n == 1 || all < best) {
        best = all;
        p.nsplit = n;
      }
    }
  }
  return p;
}

// Whether parts meet by way of the workspace and a second launch.
static bool joins(const Plan& p) { return p.nsplit > (p.tiles ? 1 : kMaxCluster); }

static size_t plan_bytes(const Plan& p, int tokens, int q_heads, int head_dim) {
  return joins(p) ? (size_t)p.nsplit * tokens * q_heads * (head_dim + 2) * 4 : 0;
}

template <typename T, int D, int MT>
static int launch_thin(const AttendArgs& a, cudaStream_t st) {
  constexpr int bytes = ThinShape<D, MT>::kBytes;
  auto fn = attend_thin_kernel<T, D, MT>;
  PPMOE_CHECK_CUDA(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  const int64_t ctas = (int64_t)a.nsplit * a.pages.kv_heads * a.seqs.batch;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(kThinWarps * 32);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = a.nsplit <= kMaxCluster ? a.nsplit : 1;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  PPMOE_CHECK_CUDA(cudaLaunchKernelEx(&cfg, fn, a));
  return PPMOE_OK;
}

template <typename T, int D>
static int launch(AttendArgs& a, const Plan& p, cudaStream_t st) {
  if (p.tiles) {
    if (int rc = attend_tiles_launch(a, D, 1 << a.pages.page_shift, std::is_same<T, __half>::value, p.tiles, p.groups, st)) return rc;
  } else {
    int rc;
    if constexpr (D == 64)
      rc = p.groups == 1 ? launch_thin<T, D, 1>(a, st) : launch_thin<T, D, 2>(a, st);
    else
      rc = launch_thin<T, D, 1>(a, st);
    if (rc) return rc;
  }
  if (a.joins) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)((int64_t)a.tokens * a.q_heads));
    cfg.blockDim = dim3(kJoinWarps * 32);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    PPMOE_CHECK_CUDA(cudaLaunchKernelEx(&cfg, attend_join_kernel<T, D>, a));
  }
  return PPMOE_OK;
}

}  // namespace ppmoe

using namespace ppmoe;

// What both entry points make of their hints: max_new and max_length held to what can be.
static Plan plan_of(int tokens, int q_heads, int kv_heads, int head_dim, int batch, int max_new, int64_t max_length) {
  max_new = max_new < 1 ? 1 : max_new > tokens ? tokens : max_new;
  max_length = max_length < 1 ? 1 : max_length > INT32_MAX ? INT32_MAX : max_length;
  return make_plan(tokens, q_heads, kv_heads, head_dim, batch, max_new, max_length);
}

extern "C" size_t ppmoe_attend_workspace_bytes(int tokens, int q_heads, int kv_heads, int head_dim, int batch,
                                               int max_new, int64_t max_length) {
  if (tokens < 1 || kv_heads < 1 || q_heads < kv_heads || head_dim < 1 || batch < 1) return 0;
  return plan_bytes(plan_of(tokens, q_heads, kv_heads, head_dim, batch, max_new, max_length), tokens, q_heads, head_dim);
}

extern "C" int ppmoe_attend(const ppmoe_kv_cache* cache, const void* q, int64_t q_t, int64_t q_h, int q_heads,
                            int tokens, const int32_t* starts, const int32_t* lengths, const int32_t* table,
                            int64_t table_stride, int batch, int max_pages, float scale, int max_new,
                            int64_t max_length, void* out, int64_t o_t, int64_t o_h, void* ws, size_t ws_bytes,
                            void* stream) {
  clear_error();
  AttendArgs a{};
  a.seqs = {starts, lengths, table, table_stride, batch, max_pages};
  if (int rc = check_cache("ppmoe_attend", cache, a.pages)) return rc;
  if (int rc = check_seqs("ppmoe_attend", a.seqs)) return rc;
  const int kv_heads = cache->kv_heads, head_dim = cache->head_dim;
  if (tokens < 0 || q_heads < 1 || q_heads % kv_heads) {
    set_error("ppmoe_attend: tokens=%d, q_heads=%d must be a positive multiple of kv_heads=%d", tokens, q_heads,
              kv_heads);
    return PPMOE_ERR_INVALID_ARG;
  }
  if (tokens == 0) return PPMOE_OK;
  if ((int64_t)batch * kv_heads > (1 << 20) || (int64_t)tokens * q_heads > INT32_MAX) {
    set_error("ppmoe_attend: batch * kv_heads = %lld (at most 2^20) or tokens * q_heads = %lld (below 2^31)",
              (long long)batch * kv_heads, (long long)tokens * q_heads);
    return PPMOE_ERR_UNSUPPORTED;
  }
  // (the kernels count keys in 32 bits, up to some blocks past the last)
  if ((int64_t)max_pages * cache->page_size > INT32_MAX - 8192) {
    set_error("ppmoe_attend: a table of %d pages of %d names too many positions (at most 2^31 - 8193)", max_pages, cache->page_size);
    return PPMOE_ERR_UNSUPPORTED;
  }
  if (!q || !out) {
    set_error("ppmoe_attend: null pointer");
    return PPMOE_ERR_INVALID_ARG;
  }
  if (!std::isfinite(scale * 1.4426950408889634f)) {
    set_error("ppmoe_attend: scale (times log2 e) is not finite");
    return PPMOE_ERR_INVALID_ARG;
  }
  const Plan p = plan_of(tokens, q_heads, kv_heads, head_dim, batch, max_new, max_length);
  const size_t need = plan_bytes(p, tokens, q_heads, head_dim);
  if (need && (!ws || ws_bytes < need || reinterpret_cast<uintptr_t>(ws) % 32)) {
    set_error("ppmoe_attend: workspace of %zu bytes (32-byte aligned) needed, %zu given", need, ws ? ws_bytes : 0);
    return PPMOE_ERR_WORKSPACE;
  }
  a.q = q;
  a.q_t = q_t;
  a.q_h = q_h;
  a.out = out;
  a.o_t = o_t;
  a.o_h = o_h;
  a.tokens = tokens;
  a.q_heads = q_heads;
  a.group = q_heads / kv_heads;
  a.c = scale == 0.f ? 1.f : std::fabs(scale) * 1.4426950408889634f;
  a.q_sign = scale > 0.f ? 1 : scale < 0.f ? -1 : 0;
  auto on = [](const void* x, int64_t s1, int64_t s2, int n) {
    return reinterpret_cast<uintptr_t>(x) % (2 * n) == 0 && s1 % n == 0 && s2 % n == 0;
  };
  a.q_wide16 = on(q, q_t, q_h, 8);
  a.o_wide = on(out, o_t, o_h, 8);
  a.o_wide32 = on(out, o_t, o_h, 16);
  a.nsplit = p.nsplit;
  a.joins = joins(p);
  a.part_o = static_cast<float*>(ws);
  a.part_ml = a.part_o + (size_t)p.nsplit * tokens * q_heads * head_dim;
  a.status = static_cast<uint32_t*>(cache->status);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (cache->dtype == PPMOE_BF16)
    return head_dim == 128 ? launch<__nv_bfloat16, 128>(a, p, st) : launch<__nv_bfloat16, 64>(a, p, st);
  return head_dim == 128 ? launch<__half, 128>(a, p, st) : launch<__half, 64>(a, p, st);
}
