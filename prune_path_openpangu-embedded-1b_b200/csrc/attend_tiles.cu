// Paged causal attention of many rows: tcgen05 products over 128 x 128 tiles of scores.
// (The mathematics and the layout of rows: attend.cu.)
//
// A CTA takes two tiles of 128 rows of one (sequence, kv head) over the same keys, 128 at a time:
//   S_t = Q_t K^T (TMEM, fp32)  ->  softmax warps of tile t: w = 2^(c S - m), rounded, into the first
//   half of S_t's columns  ->  O_t += W_t V (A operand from TMEM).
// One warp issues both tiles' products, so that tile 1's run while tile 0's softmax does and the other way
// round.  A thread of the softmax warps owns a row: maxima and sums need no exchange.  The
// reference maximum m of a row moves only when a tile's maximum exceeds it by 2^8 (weights then
// reach 2^8, which fp32 sums and both 16-bit types hold; m cancels in the end), so the
// sums are rescaled seldom.  That needs no wait: S_t(j) comes after O_t += W_t(j-1) V(j-1).
// K and V tiles arrive by TMA, a box per page and 64 columns, in one ring.
// Two more warps look after V tiles that some row sees in part: rows past the last key become
// zero (pages end inside a tile), values that are not finite are taken out and listed.
#include <cuda.h>
#include <mutex>
#include "attend.cuh"

namespace ppmoe {

constexpr int kTileRows = 128;
constexpr int kTileKeys = 128;
constexpr int kTilesThreads = 384;  // 8 softmax warps, products, loads, 2 guards

template <int D>
struct TilesSmem {
  static constexpr int kQ = kTileRows * D * 2;     // one q tile: [D / 64][128 rows][128 bytes]
  static constexpr int kStage = kTileKeys * D * 2; // a K or V tile, the same way
  static constexpr int kStages = D == 128 ? 5 : 8;
  static constexpr int kBars = 2 * kQ + kStages * kStage;
  static constexpr int kNumBars = 4 * kStages + 6;
  static constexpr int kList = kBars + ((kNumBars * 8 + 16 + 15) / 16) * 16;  // [3][D] ints
  static constexpr int kBytes = kList + 3 * D * 4 + 1024;
};

// Bounded wait that records a timeout; any earlier timeout ends it soon.
__device__ __forceinline__ void wait_bar(uint64_t* bar, uint32_t parity, uint32_t* status) {
  const uint32_t at = smem_u32(bar);
#pragma unroll 1
  for (uint32_t i = 0; i < kSpinLimit; ++i) {
    if (mbar_try_wait(at, parity)) return;
    if (i > 16384) __nanosleep(32);
    if ((i & 1023u) == 1023u && (*reinterpret_cast<volatile uint32_t*>(status) & DEVERR_TIMEOUT)) return;
  }
  atomicOr(status, DEVERR_TIMEOUT);
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar)) : "memory");
}

// D (TMEM) += A (TMEM, 16-bit pairs) * B (shared memory).
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
      ::"r"(d), "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}

// Descriptor of a V tile as the B operand with its columns contiguous ("MN-major"), 128-byte
// swizzle: 64 columns x 8 keys are 1024 bytes; 8 keys further on: 1024 bytes; 64 columns further
// on: a half tile.
__device__ __forceinline__ uint64_t desc_v(uint32_t saddr) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr >> 4) & 0x3FFF);
  d |= (uint64_t)((kTileKeys * 128) >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

// D fp32, A and B of type T, M = 128; b_mn: B's columns are contiguous.
template <typename T>
constexpr uint32_t idesc_of(int n, bool b_mn) {
  const uint32_t f = std::is_same<T, __half>::value ? 0u : 1u;
  return (1u << 4) | (f << 7) | (f << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(kTileRows >> 4) << 24);
}

__device__ __forceinline__ void tmem_ld32_async(uint32_t taddr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
        "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
        "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}

// What every warp of a CTA derives alike for one pair of tiles.
struct Pair {
  int r0, tiles;      // first row, tiles with rows (1 or 2)
  int b0, count[2];   // first block of keys, blocks of each tile
  int keys;           // keys some row sees
  int clear;          // keys every row sees: blocks within need no guard
  __device__ Pair(const AttendArgs& a, int pair, int rows, int pos0, int cap, int split) {
    r0 = pair * 2 * kTileRows;
    tiles = r0 + kTileRows < rows ? 2 : 1;
    int n[2] = {0, 0};
    keys = 0;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      if (t >= tiles) continue;
      const int last = min(r0 + (t + 1) * kTileRows, rows) - 1;
      keys = max(0, min(pos0 + last / a.group + 1, cap));
      n[t] = (keys + kTileKeys - 1) / kTileKeys;
    }
    const int most = max(n[0], n[1]), per = (most + a.nsplit - 1) / a.nsplit;
    b0 = split * per;
    const int b1 = min(most, b0 + per);
    count[0] = max(0, min(b1, n[0]) - b0);
    count[1] = max(0, min(b1, n[1]) - b0);
    clear = min(pos0 + r0 / a.group + 1, cap);
  }
  __device__ int blocks() const { return max(count[0], count[1]); }
  __device__ bool guarded(int block) const { return (block + 1) * kTileKeys > clear; }
};

template <typename T, int D>
__global__ void __launch_bounds__(kTilesThreads, 1)
attend_tiles_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                    const __grid_constant__ AttendArgs a, int box_rows, int pairs_hint) {
  extern __shared__ uint8_t smem_raw[];
  using S = TilesSmem<D>;
  constexpr int NS = S::kStages;
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBars);
  // A V tile that needs a guard arrives at g_full, is handed on at v_ok, and leaves kv_full alone: whoever waits
  // for a barrier waits for every phase of it.
  uint64_t *kv_full = bars, *kv_empty = bars + NS, *g_full = bars + 2 * NS, *v_ok = bars + 3 * NS;
  uint64_t *s_full = bars + 4 * NS, *p_ready = s_full + 2, *q_full = s_full + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + S::kNumBars);
  int* any_odd = reinterpret_cast<int*>(tmem_slot + 1);
  int* odd = reinterpret_cast<int*>(smem + S::kList);  // [nan, +inf, -inf][D]: first key with one in that column

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_launch_dependents();
  // blocks of work, the rows with most keys first: pair (slowest, descending), sequence, kv head, part
  int x = blockIdx.x;
  const int split = x % a.nsplit;
  x /= a.nsplit;
  const int kvh = x % a.pages.kv_heads;
  x /= a.pages.kv_heads;
  const int b = x % a.seqs.batch;
  const int pair_of = pairs_hint - 1 - x / a.seqs.batch;
  const Seq sq = load_seq(a, b);
  const int rows = sq.rows > 0 ? sq.rows * a.group : 0;
  if ((int64_t)pair_of * (2 * kTileRows) >= rows) return;
  const int cap = key_cap(a, sq.length);
  if (cap < sq.length && tid == 0) atomicOr(a.status, DEVERR_PAGE);
  const int pos0 = sq.length - (a.seqs.starts[b + 1] - a.seqs.starts[b]);

  if (tid == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(kv_full + i, 1);
      mbar_init(kv_empty + i, 1);
      mbar_init(g_full + i, 1);
      mbar_init(v_ok + i, 2);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(s_full + t, 1);
      mbar_init(p_ready + t, kTileRows);
      mbar_init(q_full + t, kTileRows);
    }
    *any_odd = 0;
    fence_mbar_init();
  }
  for (int i = tid; i < 3 * D; i += kTilesThreads) odd[i] = INT_MAX;
  if (warp == 8) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t ring = smem_u32(smem) + 2 * S::kQ;

  // running counts, alike in every role: ring uses, barrier phases
  int loads = 0;            // K and V tiles so far
  uint32_t ph_s[2] = {0, 0}, ph_p[2] = {0, 0}, ph_q[2] = {0, 0};
  uint32_t ph_full = 0, ph_v = 0;  // a bit a stage: kv_full; g_full (guards) or v_ok (products)

#pragma unroll 1
  for (int64_t pair = pair_of; pair * (2 * kTileRows) < rows; pair += pairs_hint) {
    const Pair w(a, (int)pair, rows, pos0, cap, split);
    const int blocks = w.blocks();
    if (warp < 8) {
      // ------------------------------------------------------------ softmax, tile t, one row a thread
      const int t = warp >> 2, row = tid & 127;
      if (t < w.tiles) {
        const int r = w.r0 + t * kTileRows + row;
        {
          const int base = w.r0 + t * kTileRows;
          constexpr int CH = D / 8;
#pragma unroll 4
          for (int i = row; i < kTileRows * CH; i += kTileRows) {
            const int rr = i / CH, c = i % CH, q_row = base + rr;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (q_row < rows) {
              const int tok = q_row / a.group;
              const T* p = static_cast<const T*>(a.q) + (int64_t)(sq.first + tok) * a.q_t +
                           (int64_t)(kvh * a.group + q_row - tok * a.group) * a.q_h + c * 8;
              if (a.q_wide16) {
                v = __ldg(reinterpret_cast<const uint4*>(p));
              } else {
                const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
                v = make_uint4(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16, h[4] | (uint32_t)h[5] << 16,
                               h[6] | (uint32_t)h[7] << 16);
              }
              v = make_uint4(q_pair(v.x, a.q_sign), q_pair(v.y, a.q_sign), q_pair(v.z, a.q_sign), q_pair(v.w, a.q_sign));
            }
            *reinterpret_cast<uint4*>(smem + t * S::kQ + (c >> 3) * (kTileRows * 128) + sw128_offset(rr, c & 7)) = v;
          }
          fence_proxy_async();
          mbar_arrive(q_full + t);
        }
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // this warp's 32 TMEM lanes
        const uint32_t t_s = tmem + t * kTileKeys + lanes, t_o = tmem + 2 * kTileKeys + t * D + lanes;
        const int tok = r / a.group;
        const int lim = r < rows ? min(pos0 + tok, cap - 1) : -1;
        const int all_see = min(pos0 + (w.r0 + t * kTileRows) / a.group, cap - 1);  // last key the first row sees
        const float c = a.c;
        float m = -CUDART_INF_F, l = 0.f;
        const int count = w.count[t];
#pragma unroll 1
        for (int j = 0; j < count; ++j) {
          float s[kTileKeys];
          wait_bar(s_full + t, ph_s[t], a.status);
          ph_s[t] ^= 1;
          tc_fence_after();
#pragma unroll
          for (int i = 0; i < kTileKeys; i += 32) tmem_ld32_async(t_s + i, s + i);
          tmem_ld_wait();
          const int key0 = (w.b0 + j) * kTileKeys;
          if (key0 + kTileKeys - 1 > all_see) {
            const int n = lim - key0;  // columns 0 .. n are seen
#pragma unroll
            for (int i = 0; i < kTileKeys; ++i) s[i] = i <= n ? s[i] : -CUDART_INF_F;
          }
          float mx = s[0], mx2 = s[1];
#pragma unroll
          for (int i = 2; i < kTileKeys; i += 2) {
            mx = fmaxf(mx, s[i]);
            mx2 = fmaxf(mx2, s[i + 1]);
          }
          mx = fmaxf(mx, mx2);
          const bool move = (mx - m) * c > 8.f;  // false where both are -inf
          if (__any_sync(0xffffffffu, move)) {
            if (j > 0) {
              const float f = move ? exp2_ftz((m - mx) * c) : 1.f;
              l *= f;
#pragma unroll 1
              for (int i = 0; i < D; i += 32) {
                float o[32];
                tmem_ld32_async(t_o + i, o);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] *= f;
                tmem_st32(t_o + i, reinterpret_cast<uint32_t*>(o));
              }
              tmem_st_wait();
            }
            if (move) m = mx;
          }
          const float sub = (m == -CUDART_INF_F ? 0.f : m * c) - kLift<T>;
          float sum[2] = {0.f, 0.f};
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t p[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const float e0 = exp2_ftz(fmaf(s[h * 64 + 2 * i], c, -sub)), e1 = exp2_ftz(fmaf(s[h * 64 + 2 * i + 1], c, -sub));
              sum[0] += e0;
              sum[1] += e1;
              p[i] = pack2<T>(e0, e1);
            }
            tmem_st32(t_s + h * 32, p);
          }
          l += sum[0] + sum[1];
          tmem_st_wait();
          tc_fence_before();
          mbar_arrive(p_ready + t);
        }
        // the sums
        if (count > 0) {
          wait_bar(s_full + t, ph_s[t], a.status);
          ph_s[t] ^= 1;
          tc_fence_after();
        }
        const bool listed = *reinterpret_cast<volatile int*>(any_odd) != 0;
        const float inv = a.nsplit > 1 ? 1.f : l > 0.f ? 1.f / l : l == l ? 0.f : l;
        const int64_t token = sq.first + tok;
        const int h = kvh * a.group + r - tok * a.group;
        const int64_t at = ((int64_t)split * a.tokens + token) * a.q_heads + h;
#pragma unroll 1
        for (int i = 0; i < D; i += 32) {
          float o[32];
          if (count > 0) {
            tmem_ld32_async(t_o + i, o);
            tmem_ld_wait();
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = 0.f;
          }
          if (listed) {
#pragma unroll 1
            for (int e = 0; e < 32; ++e) {
              float add = 0.f;
              if (odd[D + i + e] <= lim) add += CUDART_INF_F;
              if (odd[2 * D + i + e] <= lim) add -= CUDART_INF_F;
              if (odd[i + e] <= lim) add = CUDART_NAN_F;
              if (!(add == 0.f)) {
#pragma unroll
                for (int z = 0; z < 32; ++z) o[z] = z == e ? o[z] + add : o[z];
              }
            }
          }
          if (r < rows) {
            if (a.nsplit == 1) {
              store_row<T, 32>(static_cast<T*>(a.out) + token * a.o_t + h * a.o_h + i, o, inv, a.o_wide);
            } else {
#pragma unroll
              for (int e = 0; e < 32; e += 4)
                *reinterpret_cast<float4*>(a.part_o + at * D + i + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
            }
          }
        }
        if (a.nsplit > 1 && r < rows) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(m * c, l);
        tc_fence_before();
      }
    } else if (warp == 8) {
      // ------------------------------------------------------------ products
      constexpr uint32_t id_s = idesc_of<T>(kTileKeys, false), id_o = idesc_of<T>(D, true);
      auto stage_of = [&](int i) { return ring + (uint32_t)((loads + i) % NS) * S::kStage; };
      auto wait_tile = [&](int st) {
        wait_bar(kv_full + st, (ph_full >> st) & 1, a.status);
        ph_full ^= 1u << st;
      };
      auto qk = [&](int t, int j) {
        if (lane == 0) {
          const uint32_t qa = smem_u32(smem) + t * S::kQ, kb = stage_of(2 * j);
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t off = (k >> 2) * (kTileRows * 128) + (k & 3) * 32;
            umma_bf16(tmem + t * kTileKeys, umma_desc_sw128(qa + off), umma_desc_sw128(kb + off), id_s, k > 0);
          }
          umma_commit(s_full + t);
        }
      };
      for (int t = 0; t < w.tiles; ++t) {
        wait_bar(q_full + t, ph_q[t], a.status);
        ph_q[t] ^= 1;
      }
      if (blocks > 0) {
        wait_tile(loads % NS);
        tc_fence_after();
        for (int t = 0; t < w.tiles; ++t)
          if (w.count[t] > 0) qk(t, 0);
        if (lane == 0) umma_commit(kv_empty + loads % NS);
      }
#pragma unroll 1
      for (int j = 0; j < blocks; ++j) {
        const int vi = loads + 2 * j + 1, vs = vi % NS;
        if (w.guarded(w.b0 + j)) {
          wait_bar(v_ok + vs, (ph_v >> vs) & 1, a.status);
          ph_v ^= 1u << vs;
        } else {
          wait_tile(vs);
        }
        if (j + 1 < blocks) wait_tile((vi + 1) % NS);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (j >= w.count[t]) continue;
          wait_bar(p_ready + t, ph_p[t], a.status);
          ph_p[t] ^= 1;
          tc_fence_after();
          if (lane == 0) {
            const uint32_t vb = ring + vs * S::kStage;
#pragma unroll
            for (int k = 0; k < kTileKeys / 16; ++k)
              umma_ts(tmem + 2 * kTileKeys + t * D, tmem + t * kTileKeys + k * 8, desc_v(vb + k * 2048), id_o, j > 0 || k > 0);
          }
          if (j + 1 < w.count[t])
            qk(t, j + 1);
          else if (lane == 0)
            umma_commit(s_full + t);
          __syncwarp();
        }
        if (lane == 0) {
          umma_commit(kv_empty + vs);
          if (j + 1 < blocks) umma_commit(kv_empty + (vi + 1) % NS);
        }
      }
    } else if (warp == 9) {
      // ------------------------------------------------------------ loads
      const int shift = a.pages.page_shift;
      const int32_t* table = a.seqs.table + b * a.seqs.table_stride;
      const int boxes = kTileKeys / box_rows;  // pages of a block, 1 to 8
#pragma unroll 1
      for (int j = 0; j < blocks; ++j) {
        const int key0 = (w.b0 + j) * kTileKeys;
        const int here = min(boxes, (w.keys - key0 + box_rows - 1) / box_rows);  // boxes with keys
        const int box = lane % 8, half = lane / 8;  // lane -> box and 64-column half
        const bool mine = box < here && half < D / 64;
        int page = 0;
        if (mine) {
          page = __ldg(table + ((key0 + box * box_rows) >> shift));
          if ((uint32_t)page >= (uint32_t)a.pages.num_pages) {
            atomicOr(a.status, DEVERR_PAGE);
            page = a.pages.num_pages;  // out of bounds: filled with zeros
          }
        }
        const int in_page = (key0 + box * box_rows) & ((1 << shift) - 1);
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const int i = loads + 2 * j + kv, st = i % NS;
          wait_bar(kv_empty + st, ((i / NS) & 1) ^ 1, a.status);
          uint64_t* full = (kv && w.guarded(w.b0 + j) ? g_full : kv_full) + st;
          if (lane == 0) mbar_arrive_expect_tx(full, here * box_rows * 128 * (D / 64));
          __syncwarp();
          if (mine)
            tma_load_4d(ring + st * S::kStage + half * (kTileKeys * 128) + box * box_rows * 128, kv ? &map_v : &map_k,
                        half * 64, in_page, kvh, page, full);
          __syncwarp();
        }
      }
      // every tile has been read before the CTA may end
      const int n = 2 * blocks;
      for (int i = max(0, n - NS); i < n; ++i)
        wait_bar(kv_empty + (loads + i) % NS, ((loads + i) / NS) & 1, a.status);
    } else {
      // ------------------------------------------------------------ guards
      const int g = tid - 320;
#pragma unroll 1
      for (int j = 0; j < blocks; ++j) {
        const int block = w.b0 + j;
        if (!w.guarded(block)) continue;
        const int vi = loads + 2 * j + 1, vs = vi % NS;
        wait_bar(g_full + vs, (ph_v >> vs) & 1, a.status);
        ph_v ^= 1u << vs;
        uint8_t* v = smem + 2 * S::kQ + vs * S::kStage;
        const int key0 = block * kTileKeys, here = min(kTileKeys, w.keys - key0);
        constexpr int CH = D / 8;
        uint32_t bad = 0;
#pragma unroll 4
        for (int i = g; i < kTileKeys * CH; i += 64) {  // 16-byte chunk i of the tile, as it lies
          const int key = (i >> 3) & (kTileKeys - 1);
          uint4* p = reinterpret_cast<uint4*>(v) + i;
          if (key >= here) {
            *p = make_uint4(0, 0, 0, 0);
          } else {
            const uint4 u = *p;
            bad |= not_finite2<T>(u.x) | not_finite2<T>(u.y) | not_finite2<T>(u.z) | not_finite2<T>(u.w);
          }
        }
        if (bad) {
          *any_odd = 1;
#pragma unroll 1
          for (int i = g; i < here * 8; i += 64) {
#pragma unroll 1
            for (int half = 0; half < D / 64; ++half) {
              const int key = i >> 3, chunk = (i & 7) ^ (key & 7);
              uint16_t* p = reinterpret_cast<uint16_t*>(v + half * (kTileKeys * 128) + i * 16);
#pragma unroll 1
              for (int e = 0; e < 8; ++e) {
                if (!not_finite16<T>(p[e])) continue;
                const uint16_t bits = p[e];
                const float f = to_f32<T>(*reinterpret_cast<const T*>(&bits));
                atomicMin(odd + (f != f ? 0 : f > 0.f ? 1 : 2) * D + half * 64 + chunk * 8 + e, key0 + key);
                p[e] = 0;
              }
            }
          }
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(v_ok + vs);
      }
    }
    loads += 2 * blocks;
    __syncthreads();
    if ((pair + pairs_hint) * (2 * kTileRows) < rows) {
      if (*any_odd) {
        __syncthreads();
        for (int i = tid; i < 3 * D; i += kTilesThreads) odd[i] = INT_MAX;
        if (tid == 0) *any_odd = 0;
      }
      __syncthreads();
      tc_fence_after();
    }
  }
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ======================================================================== host
typedef CUresult (*TiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                            const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                            CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static int map_pages(CUtensorMap* m, const void* base, int head_dim, int page_size, int kv_heads, int num_pages,
                     int64_t row, int64_t head, int64_t page, bool half) {
  static TiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<TiledFn>(p);
  });
  if (!fn) {
    set_error("cuTensorMapEncodeTiled is unavailable from the driver");
    return PPMOE_ERR_CUDA;
  }
  const cuuint64_t dims[4] = {(cuuint64_t)head_dim, (cuuint64_t)page_size, (cuuint64_t)kv_heads, (cuuint64_t)num_pages};
  const cuuint64_t strides[3] = {(cuuint64_t)row * 2, (cuuint64_t)head * 2, (cuuint64_t)page * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)std::min(page_size, kTileKeys), 1, 1}, es[4] = {1, 1, 1, 1};
  const CUresult r = fn(m, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                        const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("ppmoe_attend: cuTensorMapEncodeTiled failed (%d)", (int)r);
    return PPMOE_ERR_CUDA;
  }
  return PPMOE_OK;
}

template <typename T, int D>
static int launch(const CUtensorMap& mk, const CUtensorMap& mv, const AttendArgs& a, int page_size, int pairs,
                  cudaStream_t st) {
  auto fn = attend_tiles_kernel<T, D>;
  PPMOE_CHECK_CUDA(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, TilesSmem<D>::kBytes));
  const int64_t ctas = (int64_t)pairs * a.nsplit * a.pages.kv_heads * a.seqs.batch;
  fn<<<(unsigned)ctas, kTilesThreads, TilesSmem<D>::kBytes, st>>>(mk, mv, a, std::min(page_size, kTileKeys), pairs);
  PPMOE_CHECK_CUDA(cudaGetLastError());
  return PPMOE_OK;
}

int attend_tiles_launch(AttendArgs& a, int head_dim, int page_size, bool half, int pairs, cudaStream_t st) {
  CUtensorMap mk, mv;
  const Pages& p = a.pages;
  if (int rc = map_pages(&mk, p.k, head_dim, page_size, p.kv_heads, p.num_pages, p.k_row, p.k_head, p.k_page, half)) return rc;
  if (int rc = map_pages(&mv, p.v, head_dim, page_size, p.kv_heads, p.num_pages, p.v_row, p.v_head, p.v_page, half)) return rc;
  if (half)
    return head_dim == 128 ? launch<__half, 128>(mk, mv, a, page_size, pairs, st)
                           : launch<__half, 64>(mk, mv, a, page_size, pairs, st);
  return head_dim == 128 ? launch<__nv_bfloat16, 128>(mk, mv, a, page_size, pairs, st)
                         : launch<__nv_bfloat16, 64>(mk, mv, a, page_size, pairs, st);
}

}  // namespace ppmoe
