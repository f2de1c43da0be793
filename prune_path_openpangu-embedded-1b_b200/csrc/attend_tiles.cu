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
// CTAs of one row tile (few rows, short prompts; two CTAs to an SM) take 64 keys at a time and have two S tiles in turn:
// the next scores are computed while the softmax is at the last ones.
// K and V tiles arrive by TMA, a box per page and 64 columns, in one ring.
// Two more warps look after V tiles that some row sees in part: rows past the last key become
// zero (pages end inside a tile), values that are not finite are taken out and listed.
//
// Long contexts are bound by the chain score -> softmax -> product of each tile, which the other tile's overlaps:
// 3000 cycles a block of 128 keys, of which the tensor pipe is busy for 2048 (68%; over a launch, with its start and
// the tail of its last wave, 62% measured, the special function pipe the same); over seconds the power limit takes
// another tenth.  2048 rows over 34816 keys, 32 query and 8 kv heads of 128, bf16: 930-945 us cold, 1000-1087 us
// sustained (1.2 and 1.1 PFLOP/s).  Tried and slower: a products' warp for each tile (1283 us: the tiles' products
// interleave and both softmaxes wait at once), part of the exponentials as polynomials, and, with the one-tile CTAs of
// then (one S tile), persistent CTAs with the next item's loads ahead (1033; prompts of 512 44-48 us for 41).
// Short prompts are bound by a CTA's start and end (7 + 2 thousand cycles).
#include <cuda.h>
#include <mutex>
#include "attend.cuh"

namespace ppmoe {

constexpr int kTileRows = 128;

// Shape of a CTA: TILES row tiles, KEYS keys at a time, of D values.
template <int D, int TILES, int KEYS>
struct TilesShape {
  static constexpr int kSoftmaxWarps = 4 * TILES;
  static constexpr int kThreads = 32 * (kSoftmaxWarps + 4);  // and products, loads, 2 guards
  static constexpr int kCtas = TILES == 2 ? 1 : 2;           // per SM
  static constexpr int kQ = kTileRows * D * 2;  // one q tile: [D / 64][128 rows][128 bytes]
  static constexpr int kStage = KEYS * D * 2;   // a K or V tile, the same way
  static constexpr int kStages = D == 128 ? (TILES == 2 ? 5 : 4) : (TILES == 2 ? 8 : 10);
  static constexpr int kBars = TILES * kQ + kStages * kStage;
  static constexpr int kNumBars = 4 * kStages + 10;
  static constexpr int kList = kBars + ((kNumBars * 8 + 16 + 15) / 16) * 16;  // [3][D] ints
  static constexpr int kBytes = kList + 3 * D * 4 + 1024;
  static constexpr int kO = 2 * KEYS;           // TMEM columns: two S tiles (of both row tiles; of one, in turn), then O tiles
  static constexpr int kTmem = TILES == 2 ? 512 : 256;
  static_assert(kO + TILES * D <= kTmem, "TMEM");
  static constexpr int kEarly = KEYS / 4 * 3;  // keys whose weights are handed on first
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

// Which of four barriers have passed a phase (bit i: barrier i), asked all at once.  A question takes the products'
// warp about 220 cycles whatever the answer (it queues behind the softmax warps' exponentials and TMEM
// accesses), so it asks for a tile's barriers together and waits only for those that were not ready.
__device__ __forceinline__ uint32_t test_bars(uint64_t* b0, uint32_t ph0, uint64_t* b1, uint32_t ph1, uint64_t* b2, uint32_t ph2,
                                              uint64_t* b3, uint32_t ph3) {
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p0, p1, p2, p3;\n .reg .b32 a, b, c;\n"
      " mbarrier.test_wait.parity.shared::cta.b64 p0, [%1], %2;\n"
      " mbarrier.test_wait.parity.shared::cta.b64 p1, [%3], %4;\n"
      " mbarrier.test_wait.parity.shared::cta.b64 p2, [%5], %6;\n"
      " mbarrier.test_wait.parity.shared::cta.b64 p3, [%7], %8;\n"
      " selp.b32 %0, 1, 0, p0;\n selp.b32 a, 2, 0, p1;\n selp.b32 b, 4, 0, p2;\n selp.b32 c, 8, 0, p3;\n"
      " or.b32 %0, %0, a;\n or.b32 b, b, c;\n or.b32 %0, %0, b;\n}\n"
      : "=&r"(r)
      : "r"(smem_u32(b0)), "r"(ph0), "r"(smem_u32(b1)), "r"(ph1), "r"(smem_u32(b2)), "r"(ph2), "r"(smem_u32(b3)), "r"(ph3)
      : "memory");
  return r;
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar)) : "memory");
}

// One lane of a converged warp.  The compiler knows that a single lane runs what follows; under
// `lane == 0` every product cost its warp about 100 cycles to issue (1.33 -> 1.08 ms for 2048 rows over
// 32768 keys, 32 heads).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p));
  return p != 0;
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
template <int KEYS>
__device__ __forceinline__ uint64_t desc_v(uint32_t saddr) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr >> 4) & 0x3FFF);
  d |= (uint64_t)((KEYS * 128) >> 4) << 16;
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

// 32 columns of this thread's TMEM lane; the values are there after tmem_ld_wait, and only what
// passed tmem_ld_bind after it is safe from being used before it.
__device__ __forceinline__ void tmem_ld32_async(uint32_t taddr, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
        "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]),
        "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]),
        "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld_bind(float* v) {
  asm volatile("" : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
               "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]));
  asm volatile("" : "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]),
               "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]), "+f"(v[30]),
               "+f"(v[31]));
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// Pairs of fp32 in one 64-bit register.
__device__ __forceinline__ uint64_t two(float a, float b) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  return v;
}
__device__ __forceinline__ void untwo(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// What every warp of a CTA derives alike for one group of TILES row tiles.
template <int TILES, int KEYS>
struct Group {
  int r0, tiles;         // first row, tiles with rows
  int b0, count[TILES];  // first block of keys, blocks of each tile
  int keys;              // keys some row sees
  int clear;             // keys every row sees: blocks within need no guard
  __device__ Group(const AttendArgs& a, int64_t group, int rows, int pos0, int cap, int split) {
    r0 = (int)group * TILES * kTileRows;
    tiles = TILES == 2 && r0 + kTileRows < rows ? 2 : 1;
    int n[TILES];
    keys = 0;
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      n[t] = 0;
      if (t >= tiles) continue;
      const int last = min(r0 + (t + 1) * kTileRows, rows) - 1;
      keys = max(0, min(pos0 + last / a.group + 1, cap));
      n[t] = (keys + KEYS - 1) / KEYS;
    }
    const int most = n[tiles - 1], per = (most + a.nsplit - 1) / a.nsplit;
    b0 = split * per;
    const int b1 = min(most, b0 + per);
#pragma unroll
    for (int t = 0; t < TILES; ++t) count[t] = max(0, min(b1, n[t]) - b0);
    clear = min(pos0 + r0 / a.group + 1, cap);
  }
  __device__ int blocks() const { return TILES == 2 ? max(count[0], count[TILES - 1]) : count[0]; }
  __device__ bool guarded(int block) const { return (block + 1) * KEYS > clear; }
};

// Where a row of (token, head of the group) lies in a tensor of these strides, and the rows `step` further on each
// time, without a division for each.
struct RowWalk {
  int64_t off, inc, wrap;
  unsigned head, d_head, group;
  __device__ RowWalk(unsigned row, unsigned step, unsigned g, int64_t s_tok, int64_t s_head) : group(g) {
    const unsigned tok = row / g, d_tok = step / g;
    head = row - tok * g;
    d_head = step - d_tok * g;
    off = tok * s_tok + head * s_head;
    inc = d_tok * s_tok + d_head * s_head;
    wrap = s_tok - (int64_t)g * s_head;
  }
  __device__ void step() {
    off += inc;
    head += d_head;
    if (head >= group) {
      head -= group;
      off += wrap;
    }
  }
};

// 32 bytes at once.
__device__ __forceinline__ void st_global32(void* p, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}

template <typename T, int D, int TILES, int KEYS>
__global__ void __launch_bounds__(TilesShape<D, TILES, KEYS>::kThreads, TilesShape<D, TILES, KEYS>::kCtas)
attend_tiles_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                    const __grid_constant__ AttendArgs a, int box_rows, int groups_hint) {
  extern __shared__ uint8_t smem_raw[];
  using S = TilesShape<D, TILES, KEYS>;
  constexpr int NS = S::kStages, SW = S::kSoftmaxWarps;
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBars);
  // A V tile that needs a guard arrives at g_full, is handed on at v_ok, and leaves kv_full alone: whoever waits
  // for a barrier waits for every phase of it.
  uint64_t *kv_full = bars, *kv_empty = bars + NS, *g_full = bars + 2 * NS, *v_ok = bars + 3 * NS;
  uint64_t *s_full = bars + 4 * NS, *p_early = s_full + 2, *p_late = s_full + 4, *q_full = s_full + 6;
  // one tile: after each product with V (waited for only by whoever must, see there), and after the last
  uint64_t *pv_done = s_full + 8, *o_full = s_full + 9;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + S::kNumBars);
  int* any_odd = reinterpret_cast<int*>(tmem_slot + 1);
  int* odd = reinterpret_cast<int*>(smem + S::kList);  // [nan, +inf, -inf][D]: first key with one in that column

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (a.joins) pdl_launch_dependents();  // (anyone else's launch may write q or read out before its own wait)
  // blocks of work, the rows with most keys first: group (slowest, descending), sequence, kv head, part
  int x = blockIdx.x;
  const int split = x % a.nsplit;
  x /= a.nsplit;
  const int kvh = x % a.pages.kv_heads;
  x /= a.pages.kv_heads;
  const int b = x % a.seqs.batch;
  const int group_of = groups_hint - 1 - x / a.seqs.batch;
  const Seq sq = load_seq(a, b);
  const int rows = sq.rows > 0 ? sq.rows * a.group : 0;
  constexpr int kRows = TILES * kTileRows;
  if ((int64_t)group_of * kRows >= rows) return;
  const int cap = key_cap(a, sq.length);
  if (cap < sq.length && tid == 0) atomicOr(a.status, DEVERR_PAGE);
  const int pos0 = sq.length - (a.seqs.starts[b + 1] - a.seqs.starts[b]);

  // q tile of this thread's softmax group, rows from `base`: all copies in flight at once, the first group's
  // behind the set-up
  constexpr int CH = D / 8, STEP = kTileRows / CH;  // 16-byte chunks of a row, rows 128 threads take at once
  auto load_q = [&](int base) {
    const int row = tid & 127, ch = row % CH;
    uint8_t* q_s = smem + (warp >> 2) * S::kQ + (ch >> 3) * (kTileRows * 128);
    RowWalk at(base + row / CH, STEP, a.group, a.q_t, a.q_h);
    const T* q = static_cast<const T*>(a.q) + sq.first * a.q_t + (int64_t)kvh * a.group * a.q_h + ch * 8;
    if (a.q_wide16 && a.q_sign > 0) {
#pragma unroll
      for (int i = 0; i < CH; ++i, at.step()) {
        const int rr = row / CH + i * STEP;
        const bool real = base + rr < rows;
        cp_async16_or_zero(smem_u32(q_s + sw128_offset(rr, ch & 7)), q + (real ? at.off : 0), real);
      }
    } else {
#pragma unroll 1
      for (int i = 0; i < CH; ++i, at.step()) {
        const int rr = row / CH + i * STEP;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (base + rr < rows) {
          const uint16_t* h = reinterpret_cast<const uint16_t*>(q + at.off);
          v = make_uint4(q_pair<T>(h[0] | (uint32_t)h[1] << 16, a.q_sign), q_pair<T>(h[2] | (uint32_t)h[3] << 16, a.q_sign),
                         q_pair<T>(h[4] | (uint32_t)h[5] << 16, a.q_sign), q_pair<T>(h[6] | (uint32_t)h[7] << 16, a.q_sign));
        }
        *reinterpret_cast<uint4*>(q_s + sw128_offset(rr, ch & 7)) = v;
      }
    }
    cp_async_commit();
  };

  if (warp < SW) {
    const int base = group_of * kRows + (warp >> 2) * kTileRows;
    if (base < rows) load_q(base);
  } else if (warp == SW) {
    tmem_alloc(tmem_slot, S::kTmem);
  } else if (warp == SW + 1) {
    if (lane == 0) {
      for (int i = 0; i < NS; ++i) {
        mbar_init(kv_full + i, 1);
        mbar_init(kv_empty + i, 1);
        mbar_init(g_full + i, 1);
        mbar_init(v_ok + i, 2);
      }
      for (int t = 0; t < 2; ++t) {
        mbar_init(s_full + t, 1);
        mbar_init(p_early + t, kTileRows);
        mbar_init(p_late + t, kTileRows);
        mbar_init(q_full + t, kTileRows);
      }
      mbar_init(pv_done, 1);
      mbar_init(o_full, 1);
      *any_odd = 0;
      fence_mbar_init();
      asm volatile("prefetch.tensormap [%0];" ::"l"(&map_k) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(&map_v) : "memory");
    }
  } else {
    for (int i = tid - 32 * (SW + 2); i < 3 * D; i += 64) odd[i] = INT_MAX;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t ring = smem_u32(smem) + TILES * S::kQ;

  // Between two groups of one CTA: everything of the first is over.
  auto next_group = [&](int64_t group) {
    tc_fence_before();
    __syncthreads();
    if ((group + groups_hint) * kRows < rows) {
      for (int i = tid; i < 3 * D; i += S::kThreads) odd[i] = INT_MAX;
      if (tid == 0) *any_odd = 0;
      __syncthreads();
    }
    tc_fence_after();
  };

  if (warp < SW) {
    // -------------------------------------------------------------- softmax, tile t, one row a thread
    const int t = warp >> 2, row = tid & 127;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // this warp's 32 TMEM lanes
    const uint32_t t_s0 = tmem + t * KEYS + lanes, t_o = tmem + S::kO + t * D + lanes;
    const float c = a.c;
    uint32_t ph_s = 0;  // two tiles: the phase of s_full
    uint32_t ph_o = 0;
    int done = 0;       // one tile: blocks so far; block n has S tile n % 2
#pragma unroll 1
    for (int64_t group = group_of; group * kRows < rows; group += groups_hint) {
      const Group<TILES, KEYS> w(a, group, rows, pos0, cap, split);
      if (t < w.tiles) {
        const int base = w.r0 + t * kTileRows, r = base + row;
        if (group != group_of) load_q(base);
        cp_async_wait<0>();
        fence_proxy_async();
        mbar_arrive(q_full + t);
        const int tok = r / a.group;
        const int lim = r < rows ? min(pos0 + tok, cap - 1) : -1;      // last key this row sees
        const int all_see = min(pos0 + base / a.group, cap - 1);       // ... the tile's first row
        const int count = w.count[t];
        float m = -CUDART_INF_F, l = 0.f;
        bool far = false;  // some row of the warp has |c m| > 2^16
#pragma unroll 1
        for (int j = 0; j < count; ++j) {
          float s[KEYS];
          const int at_s = TILES == 1 ? done & 1 : t;  // S tile and its barriers
          const uint32_t t_s = TILES == 1 ? t_s0 + at_s * KEYS : t_s0;
          wait_bar(s_full + at_s, TILES == 1 ? (done >> 1) & 1 : ph_s, a.status);
          ph_s ^= 1;
          ++done;
          tc_fence_after();
#pragma unroll
          for (int i = 0; i < KEYS; i += 32) tmem_ld32_async(t_s + i, s + i);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < KEYS; i += 32) tmem_ld_bind(s + i);
          const int key0 = (w.b0 + j) * KEYS;
          const bool masked = key0 + KEYS - 1 > all_see;
          if (masked) {
            const int n = lim - key0;  // columns 0 .. n are seen
#pragma unroll
            for (int i = 0; i < KEYS; ++i) s[i] = i <= n ? s[i] : -CUDART_INF_F;
          }
          float mx[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) mx[e] = s[e];
#pragma unroll
          for (int i = 8; i < KEYS; i += 16) {
#pragma unroll
            for (int e = 0; e < 8; ++e) mx[e] = i + 8 < KEYS ? max3(mx[e], s[i + e], s[i + 8 + e]) : max3(mx[e], s[i + e], s[i + e]);
          }
          mx[0] = max3(max3(mx[0], mx[1], mx[2]), max3(mx[3], mx[4], mx[5]), max3(mx[6], mx[7], mx[7]));
          // false where both are -inf; a NaN takes the row for good
          const bool move = (mx[0] - m) * c > 8.f || mx[0] != mx[0];
          if (__any_sync(0xffffffffu, move)) {
            if (j > 0) {
              if constexpr (TILES == 1) {
                // The product of block done - 2.  Its phase is the one running or the one before: the product before it came
                // before these scores, the one after it needs this thread's weights.
                wait_bar(pv_done, (done - 2) & 1, a.status);
                tc_fence_after();
              }
              const float f = move ? exp2_ftz((m - mx[0]) * c) : 1.f;
              l *= f;
#pragma unroll 1
              for (int i = 0; i < D; i += 16) {
                uint32_t o[16];
                asm volatile(
                    "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
                    "tcgen05.wait::ld.sync.aligned;"
                    : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3]), "=r"(o[4]), "=r"(o[5]), "=r"(o[6]), "=r"(o[7]),
                      "=r"(o[8]), "=r"(o[9]), "=r"(o[10]), "=r"(o[11]), "=r"(o[12]), "=r"(o[13]), "=r"(o[14]), "=r"(o[15])
                    : "r"(t_o + i) : "memory");
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                tmem_st16(t_o + i, o);
              }
              tmem_st_wait();
            }
            if (move) m = mx[0];
            // c s - c m carries the rounding of c m, the same factor for every weight of the row: it cancels, but
            // from |c m| = 2^24 on it could leave the types' range.  Such scores are taken from m first.
            far = __any_sync(0xffffffffu, fabsf(m * c) > 65536.f && m != -CUDART_INF_F);
          }
          const float from = m == -CUDART_INF_F ? 0.f : m;
          const uint64_t c2 = two(c, c), from2 = two(-from, -from), lift2 = two(kLift<T>, kLift<T>);
          const uint64_t sub2 = two(kLift<T> - from * c, kLift<T> - from * c);
          uint64_t sum[2] = {0, 0};
          // weights, in eights of pairs: the first three quarters are handed on while the last is computed
          // (all of them by the special-function pipe: a quarter or half by a polynomial on the FMA pipe took 1 and
          // 5% longer)
          auto weights = [&](auto is_far, int first, int to) {
#pragma unroll
            for (int g = first; g < to; g += 16) {
              uint32_t p[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                float x0, x1;
                const uint64_t s2 = two(s[g + 2 * i], s[g + 2 * i + 1]);
                untwo(decltype(is_far)::value ? fma2(add2(s2, from2), c2, lift2) : fma2(s2, c2, sub2), x0, x1);
                const float e0 = exp2_ftz(x0), e1 = exp2_ftz(x1);
                sum[i & 1] = add2(sum[i & 1], two(e0, e1));
                p[i] = pack2<T>(e0, e1);
              }
              tmem_st8(t_s + g / 2, p);
            }
          };
          auto part = [&](int first, int to) {
            if (far)
              weights(std::true_type{}, first, to);
            else
              weights(std::false_type{}, first, to);
          };
          part(0, S::kEarly);
          tmem_st_wait();
          tc_fence_before();
          mbar_arrive(p_early + at_s);
          part(S::kEarly, KEYS);
          tmem_st_wait();
          tc_fence_before();
          mbar_arrive(p_late + at_s);
          float l0, l1;
          untwo(add2(sum[0], sum[1]), l0, l1);
          l += l0 + l1;
        }
        // the sums
        if (count > 0) {
          if constexpr (TILES == 1) {
            wait_bar(o_full, ph_o, a.status);
            ph_o ^= 1;
          } else {
            wait_bar(s_full + t, ph_s, a.status);
            ph_s ^= 1;
          }
          tc_fence_after();
        }
        const bool listed = *reinterpret_cast<volatile int*>(any_odd) != 0;
        const float inv = a.nsplit > 1 ? 1.f : inverse_sum(l, pos0 + tok);
        const int64_t token = sq.first + tok;
        const int h = kvh * a.group + r - tok * a.group;
        const int64_t at = ((int64_t)split * a.tokens + token) * a.q_heads + h;
        T* out = static_cast<T*>(a.out) + token * a.o_t + h * a.o_h;
        bool nan = false;  // some sum is
        constexpr int W = D / 2;  // columns held at once
#pragma unroll 1
        for (int i = 0; i < D; i += W) {
          float o[W];
          if (count > 0) {
#pragma unroll
            for (int e = 0; e < W; e += 32) tmem_ld32_async(t_o + i + e, o + e);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < W; e += 32) tmem_ld_bind(o + e);
          } else {
#pragma unroll
            for (int e = 0; e < W; ++e) o[e] = 0.f;
          }
          nan |= any_nan(o);
          if (listed) {
#pragma unroll 1
            for (int e = 0; e < W; ++e) {
              const float add = listed_value<D>(odd, i + e, lim);
              if (!(add == 0.f)) {
#pragma unroll
                for (int z = 0; z < W; ++z) o[z] = z == e ? o[z] + add : o[z];
              }
            }
          }
          if (r < rows) {  // whole 32-byte sectors of this thread's row
            if (a.nsplit > 1) {
#pragma unroll
              for (int e = 0; e < W; e += 8) {
                uint32_t v[8];
#pragma unroll
                for (int z = 0; z < 8; ++z) v[z] = __float_as_uint(o[e + z]);
                st_global32(a.part_o + at * D + i + e, v);
              }
            } else if (a.o_wide32) {
#pragma unroll
              for (int e = 0; e < W; e += 16) {
                uint32_t v[8];
#pragma unroll
                for (int z = 0; z < 8; ++z) v[z] = pack2<T>(o[e + 2 * z] * inv, o[e + 2 * z + 1] * inv);
                st_global32(out + i + e, v);
              }
            } else {
#pragma unroll
              for (int e = 0; e < W; ++e) out[i + e] = from_f32<T>(o[e] * inv);
            }
          }
        }
        if (a.nsplit > 1 && r < rows) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(m * c, l);
        nan &= r < rows && (l > 0.f || (l == 0.f && a.nsplit > 1));
        // Sums to put right (attend.cuh), by each warp for itself.  16 prompts of 512 take 37.5 us in a graph with this look at
        // the sums and 36.6 without; joined with the barrier behind it, and by the whole CTA, 38.
        if (__any_sync(0xffffffffu, nan)) {
          static_assert(S::kQ / 4 >= 3 * D * 4, "room for a list");
          int* list = reinterpret_cast<int*>(smem + t * S::kQ + (warp & 3) * (S::kQ / 4));  // this tile's q has been read
          list_values<T, D, 32>(a, b, kvh, w.b0 * KEYS, min((w.b0 + count) * KEYS, w.keys), list);
          if (nan) mend_row<T, D>(a, list, sq.first, r, kvh, a.nsplit > 1 ? split : -1, lim, 0, D);
        }
      }
      next_group(group);
    }
  } else {
    int loads = 0;  // K and V tiles so far: use i of the ring is in stage i % NS
    if (warp == SW) {
      // ------------------------------------------------------------ products
      constexpr uint32_t id_s = idesc_of<T>(KEYS, false), id_o = idesc_of<T>(D, true);
      const uint64_t q_desc = umma_desc_sw128(smem_u32(smem)), k_desc = umma_desc_sw128(ring), v_desc = desc_v<KEYS>(ring);
      uint32_t ph_p[TILES] = {}, ph_q[TILES] = {}, ph_full = 0, ph_v = 0;  // the last two: a bit a stage
      int done = 0;  // one tile: blocks so far
#pragma unroll 1
      for (int64_t group = group_of; group * kRows < rows; group += groups_hint) {
        const Group<TILES, KEYS> w(a, group, rows, pos0, cap, split);
        const int blocks = w.blocks();
        if (elect_one()) {
          auto wait_tile = [&](int st) {
            wait_bar(kv_full + st, (ph_full >> st) & 1, a.status);
            ph_full ^= 1u << st;
          };
          // S tile i = q tile t times the K tile in a stage; O tile t += W tile i times a V tile
          auto qk = [&](int t, int i, int st) {
            const uint64_t qd = q_desc + (uint64_t)(t * (S::kQ >> 4)), kd = k_desc + (uint64_t)(st * (S::kStage >> 4));
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
              umma_f16(tmem + i * KEYS, qd + (((k >> 2) * (kTileRows * 128) + (k & 3) * 32) >> 4),
                        kd + (((k >> 2) * (KEYS * 128) + (k & 3) * 32) >> 4), id_s, k > 0);
            umma_commit(s_full + i);
          };
          auto pv = [&](int t, int i, uint64_t vd, int from, int to, bool fresh) {
#pragma unroll
            for (int k = from; k < to; ++k)
              umma_ts(tmem + S::kO + t * D, tmem + i * KEYS + k * 8, vd + k * 128, id_o, !fresh || k > 0);
          };
#pragma unroll
          for (int t = 0; t < TILES; ++t) {
            if (t >= w.tiles) continue;
            wait_bar(q_full + t, ph_q[t], a.status);
            ph_q[t] ^= 1;
          }
          if constexpr (TILES == 1) {
            // One row tile has no other to fill its softmax's time; its next scores are computed ahead, into the other S tile.
            auto k_stage = [&](int j) { return (loads + 2 * j) % NS; };
#pragma unroll 1
            for (int j = 0; j < 2 && j < blocks; ++j) {
              wait_tile(k_stage(j));
              tc_fence_after();
              qk(0, (done + j) & 1, k_stage(j));
              umma_commit(kv_empty + k_stage(j));
            }
#pragma unroll 1
            for (int j = 0; j < blocks; ++j, ++done) {
              const int at_s = done & 1, ph = (done >> 1) & 1, vs = (loads + 2 * j + 1) % NS, ks = k_stage(j + 2);
              const bool guarded = w.guarded(w.b0 + j);
              uint64_t* v_bar = guarded ? v_ok + vs : kv_full + vs;
              const uint32_t v_ph = ((guarded ? ph_v : ph_full) >> vs) & 1;
              (guarded ? ph_v : ph_full) ^= 1u << vs;
              const uint32_t there = test_bars(p_early + at_s, ph, p_late + at_s, ph, v_bar, v_ph, kv_full + ks, (ph_full >> ks) & 1);
              if (!(there & 4)) wait_bar(v_bar, v_ph, a.status);
              if (!(there & 1)) wait_bar(p_early + at_s, ph, a.status);
              tc_fence_after();
              const uint64_t vd = v_desc + (uint64_t)(vs * (S::kStage >> 4));
              pv(0, at_s, vd, 0, S::kEarly / 16, j == 0);
              if (!(there & 2)) wait_bar(p_late + at_s, ph, a.status);
              tc_fence_after();
              pv(0, at_s, vd, S::kEarly / 16, KEYS / 16, false);
              umma_commit(pv_done);
              if (j + 1 == blocks) umma_commit(o_full);
              umma_commit(kv_empty + vs);
              if (j + 2 < blocks) {
                if (!(there & 8)) wait_bar(kv_full + ks, (ph_full >> ks) & 1, a.status);
                ph_full ^= 1u << ks;
                tc_fence_after();
                qk(0, at_s, ks);
                umma_commit(kv_empty + ks);
              }
            }
          } else {
            int ks = loads % NS;  // stage of the next K tile
            if (blocks > 0) {
              wait_tile(ks);
              tc_fence_after();
#pragma unroll
              for (int t = 0; t < TILES; ++t)
                if (w.count[t] > 0) qk(t, t, ks);
              umma_commit(kv_empty + ks);
            }
#pragma unroll 1
            for (int j = 0; j < blocks; ++j) {
              const int vs = ks + 1 == NS ? 0 : ks + 1;
              ks = vs + 1 == NS ? 0 : vs + 1;
              const bool guarded = w.guarded(w.b0 + j);
              bool v_due = true, next = j + 1 < blocks;  // V's, the next K's tile: not seen to be there yet
              const uint64_t vd = v_desc + (uint64_t)(vs * (S::kStage >> 4));
              auto take_v = [&](bool ready) {
                if (!ready) wait_bar(guarded ? v_ok + vs : kv_full + vs, ((guarded ? ph_v : ph_full) >> vs) & 1, a.status);
                (guarded ? ph_v : ph_full) ^= 1u << vs;
                v_due = false;
              };
              auto take_k = [&](bool ready) {
                if (!ready) wait_bar(kv_full + ks, (ph_full >> ks) & 1, a.status);
                ph_full ^= 1u << ks;
                next = false;
              };
#pragma unroll
              for (int t = 0; t < TILES; ++t) {
                if (j >= w.count[t]) continue;
                const uint32_t there = test_bars(p_early + t, ph_p[t], p_late + t, ph_p[t], guarded ? v_ok + vs : kv_full + vs,
                                                 ((guarded ? ph_v : ph_full) >> vs) & 1, kv_full + ks, (ph_full >> ks) & 1);
                if (v_due) take_v(there & 4);
                if (!(there & 1)) wait_bar(p_early + t, ph_p[t], a.status);
                tc_fence_after();
                pv(t, t, vd, 0, S::kEarly / 16, j == 0);
                if (next) take_k(there & 8);
                if (!(there & 2)) wait_bar(p_late + t, ph_p[t], a.status);
                ph_p[t] ^= 1;
                tc_fence_after();
                pv(t, t, vd, S::kEarly / 16, KEYS / 16, false);
                if (j + 1 < w.count[t])
                  qk(t, t, ks);
                else
                  umma_commit(s_full + t);
              }
              if (v_due) take_v(false);
              if (next) take_k(false);
              umma_commit(kv_empty + vs);
              if (j + 1 < blocks) umma_commit(kv_empty + ks);
            }
          }
        }
        __syncwarp();
        loads += 2 * blocks;
        next_group(group);
      }
    } else if (warp == SW + 1) {
      // ------------------------------------------------------------ loads
      const int shift = a.pages.page_shift;
      const int32_t* table = a.seqs.table + b * a.seqs.table_stride;
      const int boxes = KEYS / box_rows;  // boxes of a block, 1 to 8
#pragma unroll 1
      for (int64_t group = group_of; group * kRows < rows; group += groups_hint) {
        const Group<TILES, KEYS> w(a, group, rows, pos0, cap, split);
        const int blocks = w.blocks();
        // lane i looks up box i's page; one elected lane issues (see elect_one: 16 lanes with a box each took
        // 2000 cycles a tile of 16-row pages)
        constexpr int kMaxBoxes = KEYS / 16;
        auto page_id = [&](int j) {
          const int key = (w.b0 + j) * KEYS + lane * box_rows;
          return j < blocks && lane < boxes && key < w.keys ? __ldg(table + (key >> shift)) : 0;
        };
        int next = page_id(0);
#pragma unroll 1
        for (int j = 0; j < blocks; ++j) {
          const int key0 = (w.b0 + j) * KEYS;
          const int here = min(boxes, (w.keys - key0 + box_rows - 1) / box_rows);  // boxes with keys
          int page = next;
          next = page_id(j + 1);
          if (lane < here && (uint32_t)page >= (uint32_t)a.pages.num_pages) {
            atomicOr(a.status, DEVERR_PAGE);
            page = a.pages.num_pages;  // out of bounds: filled with zeros
          }
          int pages[kMaxBoxes];
#pragma unroll
          for (int i = 0; i < kMaxBoxes; ++i) pages[i] = __shfl_sync(0xffffffffu, page, i);
          const int in_page = key0 & ((1 << shift) - 1);  // (not 0 only where a page holds more than a block)
          if (elect_one()) {
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
              const int i = loads + 2 * j + kv, st = i % NS;
              wait_bar(kv_empty + st, ((i / NS) & 1) ^ 1, a.status);
              uint64_t* full = (kv && w.guarded(w.b0 + j) ? g_full : kv_full) + st;
              mbar_arrive_expect_tx(full, here * box_rows * 128 * (D / 64));
              uint32_t to = ring + st * S::kStage;
#pragma unroll
              for (int bx = 0; bx < kMaxBoxes; ++bx, to += box_rows * 128) {
                if (bx >= here) break;
                tma_load_4d(to, kv ? &map_v : &map_k, 0, in_page, kvh, pages[bx], full);
                if constexpr (D == 128) tma_load_4d(to + KEYS * 128, kv ? &map_v : &map_k, 64, in_page, kvh, pages[bx], full);
              }
            }
          }
          __syncwarp();
        }
        // every tile has been read before the CTA may end
        const int n = 2 * blocks;
        for (int i = max(0, n - NS); i < n; ++i)
          wait_bar(kv_empty + (loads + i) % NS, ((loads + i) / NS) & 1, a.status);
        loads += n;
        next_group(group);
      }
    } else {
      // ------------------------------------------------------------ guards
      const int g = tid - 32 * (SW + 2);
      uint32_t ph_v = 0;
#pragma unroll 1
      for (int64_t group = group_of; group * kRows < rows; group += groups_hint) {
        const Group<TILES, KEYS> w(a, group, rows, pos0, cap, split);
        const int blocks = w.blocks();
#pragma unroll 1
        for (int j = 0; j < blocks; ++j) {
          const int block = w.b0 + j;
          if (!w.guarded(block)) continue;
          const int vs = (loads + 2 * j + 1) % NS;
          wait_bar(g_full + vs, (ph_v >> vs) & 1, a.status);
          ph_v ^= 1u << vs;
          uint8_t* v = smem + TILES * S::kQ + vs * S::kStage;
          const int key0 = block * KEYS, here = min(KEYS, w.keys - key0);
          uint32_t bad = 0;
          // 16-byte chunk i of the tile, as it lies; eight loads in flight
#pragma unroll 1
          for (int i0 = g; i0 < KEYS * CH; i0 += 64 * 8) {
            uint4 u[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) u[e] = reinterpret_cast<const uint4*>(v)[i0 + 64 * e];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const uint32_t x = not_finite2<T>(u[e].x) | not_finite2<T>(u[e].y) | not_finite2<T>(u[e].z) | not_finite2<T>(u[e].w);
              bad |= ((i0 + 64 * e) >> 3 & (KEYS - 1)) < here ? x : 0;
            }
          }
          if (here < KEYS) {
#pragma unroll 4
            for (int i = g; i < KEYS * CH; i += 64)
              if ((i >> 3 & (KEYS - 1)) >= here) reinterpret_cast<uint4*>(v)[i] = make_uint4(0, 0, 0, 0);
          }
          if (bad) {
            *any_odd = 1;
#pragma unroll 1
            for (int i = g; i < KEYS * CH; i += 64) {
              const int key = (i >> 3) & (KEYS - 1), col = i / (8 * KEYS) * 64 + (((i & 7) ^ (key & 7)) * 8);
              uint16_t* p = reinterpret_cast<uint16_t*>(v + i * 16);
#pragma unroll 1
              for (int e = 0; e < 8; ++e) {
                const uint16_t bits = p[e];
                if (!not_finite16<T>(bits)) continue;
                list_value<T, D>(odd, bits, key0 + key, col + e);
                p[e] = 0;
              }
            }
          }
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(v_ok + vs);
        }
        loads += 2 * blocks;
        next_group(group);
      }
    }
  }
  if (warp == SW) tmem_dealloc(tmem, S::kTmem);
}

// ======================================================================== host
typedef CUresult (*TiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                            const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                            CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static int map_pages(CUtensorMap* m, const void* base, int head_dim, int page_size, int kv_heads, int num_pages,
                     int64_t row, int64_t head, int64_t page, int box_rows, bool half) {
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
  const cuuint32_t box[4] = {64, (cuuint32_t)box_rows, 1, 1}, es[4] = {1, 1, 1, 1};
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

template <typename T, int D, int TILES, int KEYS>
static int launch(const AttendArgs& a, int page_size, int groups, cudaStream_t st) {
  using S = TilesShape<D, TILES, KEYS>;
  constexpr bool half = std::is_same<T, __half>::value;
  const Pages& p = a.pages;
  const int box = std::min(page_size, KEYS);
  CUtensorMap mk, mv;
  if (int rc = map_pages(&mk, p.k, D, page_size, p.kv_heads, p.num_pages, p.k_row, p.k_head, p.k_page, box, half)) return rc;
  if (int rc = map_pages(&mv, p.v, D, page_size, p.kv_heads, p.num_pages, p.v_row, p.v_head, p.v_page, box, half)) return rc;
  auto fn = attend_tiles_kernel<T, D, TILES, KEYS>;
  PPMOE_CHECK_CUDA(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes));
  const int64_t ctas = (int64_t)groups * a.nsplit * p.kv_heads * a.seqs.batch;
  fn<<<(unsigned)ctas, S::kThreads, S::kBytes, st>>>(mk, mv, a, box, groups);
  PPMOE_CHECK_CUDA(cudaGetLastError());
  return PPMOE_OK;
}

int attend_tiles_launch(AttendArgs& a, int head_dim, int page_size, bool half, int tiles, int groups, cudaStream_t st) {
  auto go = [&](auto type, auto dim) {
    using T = decltype(type);
    constexpr int D = decltype(dim)::value;
    return tiles == 2 ? launch<T, D, 2, 128>(a, page_size, groups, st) : launch<T, D, 1, 64>(a, page_size, groups, st);
  };
  std::integral_constant<int, 128> d128;
  std::integral_constant<int, 64> d64;
  if (half) return head_dim == 128 ? go(__half{}, d128) : go(__half{}, d64);
  return head_dim == 128 ? go(__nv_bfloat16{}, d128) : go(__nv_bfloat16{}, d64);
}

}  // namespace ppmoe
