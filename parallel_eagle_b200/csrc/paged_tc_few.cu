// Attention over the paged key/value cache for few rows per request (decode steps, drafts)
// on the 5th-generation tensor cores.  bf16, fp32 softmax, head sizes 64 and 128.
//
// A request's rows (new tokens x query heads of one KV head's group) number 7 for a decode
// step of the 7B-class drafter and 35 for a draft of five: far below the 128 rows of a
// tcgen05 tile, and each key is used so little that the keys' and values' way from HBM
// bounds the kernel.  So the product is turned round: the 128 keys of a tile are the M side,
// the rows the N side,
//
//   S^T [128 keys x N] = K Q^T          P^T = 2^(c S^T - m)         O^T [hd x N] += V^T P^T
//
// with N = 16, 32 or 64.  A matrix product then costs its operand's way through shared
// memory (the K or V tile, read once), the softmax N exponentials per key, and nothing is
// padded to 128.  Every byte of K and V moves once: TMA pages -> shared memory -> tensor
// core.
//
//   warp 0      TMA: K and V tiles (boxes of one page's keys) through two rings; it runs
//               ahead over segment borders, so the loads never pause
//   warp 1      tcgen05.mma: S^T(i) into a double-buffered TMEM tile, then O^T += of i - 1
//   warp 2      walks the line of work and publishes segments; warps 2..3 fetch Q rows
//   warps 4..   softmax: a thread is a key (TMEM lane); from 32 rows on two groups of four
//               warps halve the columns, so that every scheduler has two warps and no
//               register spills.  Sums of the probabilities stay per thread until the
//               segment ends.  A row's maximum is over keys, that is over threads: it is
//               kept as a stale bound in shared memory and only raised, by a reduction
//               over the group, when some score passes it by 2^8 (one vote per tile), as
//               the probabilities then still fit bf16 and fp32.
// TMEM: S^T 2 x N columns, O^T 2 x N (two segments: the next one starts while this one's
// result is read).
//
// P is rounded to bf16, as the tensor core's operand has to be; its sum is not.  Each rounding
// is off by at most 2^-8: results are 2.3e-3 (rms, relative) from 64 bits, 1.7e-3 of it the
// result's own rounding.  (Another product with what the rounding leaves would take 16 KB of
// shared memory and the value product's tensor work again.)
//
// Measured (28/4 heads of 128, device time with the join): 64 requests x 1 row, 1.1M keys in
// all, 330 us, 6.7 TB/s -- the rate of a plain copy; 8 drafts of 5..9 rows, 36K keys in all,
// 31 us: 6 us to a block's first scores (lengths, then block table, then keys), 10 us of
// tiles, 2 us for a segment's results (the last block, which has two, ends 20.7 us after the
// first one's start), 4 us the join, the rest the start and end of two launches; one row over
// 600 keys 11.6 us, 12.5 under a wide table (cut, and joined).
// Code that runs once per segment is kept short (rolled loops): its time is mostly the
// instructions' way from L2 (an unrolled epilogue made the drafts 39 us).
#include "paged.cuh"
#include "sm100.cuh"

namespace pe {
namespace paged {
namespace {

using namespace sm100;

constexpr int kTile = 128;                    // keys per tile
constexpr uint32_t kChunk = kTile * 128;      // 128 keys x 64 columns, 128-byte swizzled
constexpr int kOver = 6 * kTile;              // a segment's start and end, in keys
constexpr float kRaise = 8.f;                 // log2 of what a score may pass the bound by

template <int N, int HDC>
struct Few {
  static constexpr int kStages = HDC == 2 ? 3 : 6;
  static constexpr int kQBufs = N <= 32 ? 2 : 1;
  static constexpr int kGroups = N <= 16 ? 1 : 2;      // softmax groups of 128 threads
  static constexpr int kCols = N / kGroups;            // rows (S^T columns) of a group
  static constexpr int kThreads = 128 + 128 * kGroups;
  static constexpr uint32_t kTileBytes = HDC * kChunk;
  static constexpr uint32_t kQBytes = HDC * N * 128;
  static constexpr uint32_t kTmem = 4 * N;  // columns
  struct Small {
    float mneg[N];       // minus the rows' bounds (log2 units); the result's scale at the end
    float mx[4][N];      // per-warp maxima; per-warp sums
    float fac[N];        // what a raised bound multiplies the sums and the accumulator by
    int64_t scratch[kThreads / 32 + 4];
    Seg seg[2];
    uint64_t seg_full[2], seg_empty[2];
    uint64_t k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
    uint64_t s_full[2], s_empty[2], p_full, p_empty;
    uint64_t q_full[kQBufs], q_empty[kQBufs], o_full[2], o_empty[2];
    uint32_t tmem;
  };
  // K ring, V ring, P^T, Q.  (With 64 columns the V^T operand's rows 64..127 read the 16 KB
  // behind a V tile: the next tile or P^T; their results are not used.)
  static constexpr size_t kSmem = 1024 + 2 * kStages * kTileBytes + kChunk + kQBufs * kQBytes +
                                  sizeof(Small);
  static_assert(kSmem <= 227 * 1024, "shared memory");
};

__device__ __forceinline__ uint32_t swz128(int r, int u) {
  return (uint32_t)(r * 128 + ((u ^ (r & 7)) << 4));
}

__device__ __forceinline__ void cp_async16(void* dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src),
               "r"(valid ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() {
  asm volatile("cp.async.wait_all;" ::: "memory");
}
// the 128 threads of a softmax group
__device__ __forceinline__ void bar_group(int id) {
  asm volatile("barrier.cta.sync %0, 128;" ::"r"(id) : "memory");
}
// ... and whether any of them votes
__device__ __forceinline__ bool vote_group(int id, bool mine) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, %2, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "r"((uint32_t)mine), "r"(id)
      : "memory");
  return any != 0;
}
__device__ __forceinline__ float redux_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

template <int N>
__device__ __forceinline__ void tmem_ldn(uint32_t addr, float* v) {
  if constexpr (N == 16) {
    tmem_ld16(addr, v);
  } else {
#pragma unroll
    for (int c = 0; c < N; c += 32) tmem_ld32(addr + c, v + c);
  }
}
// Sum v[0..N) over the 32 lanes with about N exchanges: halve the columns a lane answers
// for with every step.  Lane i ends with column i (N = 32) or i / 2 (16).
template <int N>
__device__ __forceinline__ void lane_sums(float (&v)[N], int lane) {
  int w = N / 2;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if (w >= 1) {
      const bool up = lane & o;
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        if (i >= w) break;
        const float send = up ? v[i] : v[i + w], keep = up ? v[i + w] : v[i];
        v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
      }
      w >>= 1;
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
    }
  }
}

template <int N, int HDC>
__global__ void __launch_bounds__(Few<N, HDC>::kThreads, 1)
paged_few_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                 const __grid_constant__ Args a, int shift) {
  using F = Few<N, HDC>;
  constexpr int ST = F::kStages, QB = F::kQBufs, NG = F::kGroups, CW = F::kCols;
  constexpr int HD = 64 * HDC;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint8_t* sK = smem;
  uint8_t* sV = sK + ST * F::kTileBytes;
  uint8_t* sP = sV + ST * F::kTileBytes;
  uint8_t* sQ = sP + kChunk;
  typename F::Small& sm = *reinterpret_cast<typename F::Small*>(sQ + QB * F::kQBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int* status = a.status;

  start_next_kernel();
  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(&sm.k_full[i], 1);
      mbar_init(&sm.k_empty[i], 1);
      mbar_init(&sm.v_full[i], 1);
      mbar_init(&sm.v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.seg_full[i], 1);
      mbar_init(&sm.seg_empty[i], 4 + 4 * NG);  // every warp reads it
      mbar_init(&sm.s_full[i], 1);
      mbar_init(&sm.s_empty[i], 4 * NG);
      mbar_init(&sm.o_full[i], 1);
      mbar_init(&sm.o_empty[i], 4 * NG);
    }
    mbar_init(&sm.p_full, 4 * NG);
    mbar_init(&sm.p_empty, 1);
    for (int i = 0; i < QB; ++i) {
      mbar_init(&sm.q_full[i], 2);
      mbar_init(&sm.q_empty[i], 1);
    }
    fence_barrier_init();
    fence_proxy_async();
    prefetch_tmap(&tmK);
    prefetch_tmap(&tmV);
    a.open[blockIdx.x].parts = 0;
  }
  if (warp == 1) {
    tmem_alloc(&sm.tmem, F::kTmem);
    tmem_relinquish();
  }
  Sched<N, kTile, kOver, 2 * kTile> w(a);
  if (w.requests() > w.kWarpRequests)
    w.init(sm.scratch);
  else if (warp == 2)
    w.init_warp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tS = sm.tmem, tO = sm.tmem + 2 * N;

  // segment s, copied out of shared memory and released; false: the wait ran out
  auto take = [&](int s, Seg& g) -> bool {
    const bool ok = mbar_wait(&sm.seg_full[s & 1], (s >> 1) & 1, status, 401);
    if (!__all_sync(0xffffffffu, ok)) return false;
    g = sm.seg[s & 1];
    __syncwarp();
    if (lane == 0) mbar_arrive(&sm.seg_empty[s & 1]);
    return true;
  };

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA ----
    const int per_chunk = kTile >> shift, boxes = per_chunk * HDC;  // of a chunk, of a tile
    const int box = 1 << shift;                                     // keys of a box
    const int at = lane % per_chunk, ch = lane / per_chunk;         // this lane's box
    const int total_rows = (int)(a.num_pages * a.Hkv * a.page), kbeg = (int)a.kbeg;
    bool ok = true;
    int i = 0;
    uint32_t st = 0, ph = 0;
    Seg g;
    PageWalk pw;
    for (int s = 0; ok; ++s) {
      ok = take(s, g);
      if (!ok || g.end) break;
      const int kend = (int)g.kend;
      if (g.t0 < g.t1)
        pw.start(g.pages, (kbeg + g.t0 * kTile) / a.page, (kend + a.page - 1) / a.page);
      for (int t = g.t0; t < g.t1; ++t, ++i) {
        const int k0 = kbeg + t * kTile;
        const int live = min(per_chunk, (kend - k0 + box - 1) >> shift);
        const bool mine = lane < boxes && at < live;
        const int key = k0 + (mine ? at << shift : 0), pi = (int)((uint32_t)key / (uint32_t)a.page);
        pw.advance((int)((uint32_t)k0 / (uint32_t)a.page));
        const int id = pw.entry(pi, (int)((uint32_t)(k0 + kTile - 1) / (uint32_t)a.page));
        // (an entry outside the pool reads as zeros)
        const int row = id >= 0 && id < a.num_pages
                            ? (id * a.Hkv + g.kvh) * a.page + (key - pi * a.page) : total_rows;
        const uint32_t off = st * F::kTileBytes + ch * kChunk + at * box * 128;
        const uint32_t bytes = (uint32_t)live * HDC * box * 128;
        ok = mbar_wait(&sm.k_empty[st], ph ^ 1u, status, 402);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(&sm.k_full[st], bytes);
        __syncwarp();
        if (mine) tma_load_2d(sK + off, &tmK, &sm.k_full[st], ch * 64, row);
        ok = mbar_wait(&sm.v_empty[st], ph ^ 1u, status, 403);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) {
          mbar_wait(&sm.k_full[st], ph, nullptr, 0);  // its copies land before the block ends
          break;
        }
        if (lane == 0) mbar_arrive_expect_tx(&sm.v_full[st], bytes);
        __syncwarp();
        if (mine) tma_load_2d(sV + off, &tmV, &sm.v_full[st], ch * 64, row);
        if (++st == ST) { st = 0; ph ^= 1u; }
      }
    }
    if (!ok) {  // copies in flight: the stages before this one, as far as they were filled
      for (int back = 1; back <= ST && back <= i; ++back) {
        const int j = i - back;
        mbar_wait(&sm.k_full[j % ST], (j / ST) & 1, nullptr, 0);
        mbar_wait(&sm.v_full[j % ST], (j / ST) & 1, nullptr, 0);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA ----
    constexpr uint32_t ID_S = idesc_bf16(kTile, N, false, false);
    constexpr uint32_t ID_O = idesc_bf16(128, N, true, true);
    const uint32_t k_base = smem_u32(sK), v_base = smem_u32(sV);
    const uint32_t p_base = smem_u32(sP), q_base = smem_u32(sQ);
    bool ok = true;
    int i = 0, seq = 0;
    int p_st = -1, p_i = 0, p_par = 0, p_use = 0;  // the tile whose value product is due
    bool p_first = false, p_last = false;
    auto value_product = [&]() -> bool {
      if (!mbar_wait(&sm.p_full, p_i & 1, status, 404)) return false;
      if (!mbar_wait(&sm.v_full[p_st], (p_i / ST) & 1, status, 405)) return false;
      if (p_first && !mbar_wait(&sm.o_empty[p_par], (p_use & 1) ^ 1u, status, 406)) return false;
      tc_fence_after();
      const uint32_t vb = v_base + p_st * F::kTileBytes;
#pragma unroll
      for (int kk = 0; kk < kTile / 16; ++kk)
        mma_bf16_ss(tO + p_par * N, sw128_desc(vb + kk * 2048, kChunk, 1024),
                    sw128_desc(p_base + kk * 2048, kChunk, 1024), ID_O,
                    (!p_first || kk > 0) ? 1u : 0u);
      mma_commit(&sm.v_empty[p_st]);
      mma_commit(&sm.p_empty);
      if (p_last) mma_commit(&sm.o_full[p_par]);
      return true;
    };
    Seg g;
    for (int s = 0; ok; ++s) {
      ok = take(s, g);
      if (!ok || g.end) break;
      if (g.t1 <= g.t0) continue;
      if (elect_one()) {
        const int qb = seq % QB;
        ok = mbar_wait(&sm.q_full[qb], (seq / QB) & 1, status, 407);
        for (int t = g.t0, j = i; t < g.t1 && ok; ++t, ++j) {
          const int st = j % ST, sb = j & 1;
          if (!mbar_wait(&sm.k_full[st], (j / ST) & 1, status, 408)) { ok = false; break; }
          if (!mbar_wait(&sm.s_empty[sb], ((j >> 1) & 1) ^ 1u, status, 409)) { ok = false; break; }
          tc_fence_after();
          const uint32_t kb = k_base + st * F::kTileBytes, qa = q_base + qb * F::kQBytes;
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk)
            mma_bf16_ss(tS + sb * N,
                        sw128_desc(kb + (kk >> 2) * kChunk + (kk & 3) * 32, 16, 1024),
                        sw128_desc(qa + (kk >> 2) * (N * 128) + (kk & 3) * 32, 16, 1024), ID_S,
                        kk > 0 ? 1u : 0u);
          mma_commit(&sm.s_full[sb]);
          mma_commit(&sm.k_empty[st]);
          if (t + 1 == g.t1) mma_commit(&sm.q_empty[qb]);
          if (p_st >= 0 && !value_product()) { ok = false; break; }
          p_st = st;
          p_i = j;
          p_par = seq & 1;
          p_use = seq >> 1;
          p_first = t == g.t0;
          p_last = t + 1 == g.t1;
        }
        if (ok) ok = value_product();  // the segment's last
        p_st = -1;
      }
      ok = __all_sync(0xffffffffu, ok);
      i += g.t1 - g.t0;
      ++seq;
    }
  } else if (warp < 4) {
    // ------------------------------------------------- line of work, Q rows ----
    const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a.q);
    bool ok = true;
    int seq = 0;
    Seg g;
    for (int s = 0; ok; ++s) {
      if (warp == 2) {
        ok = mbar_wait(&sm.seg_empty[s & 1], ((s >> 1) & 1) ^ 1u, status, 410);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const bool have = w.next();
        if (lane == 0) {
          if (have) {
            w.describe(sm.seg[s & 1]);
            if (w.first && !w.last) w.record_open();
          } else {
            sm.seg[s & 1].end = 1;
          }
          mbar_arrive(&sm.seg_full[s & 1]);
        }
        __syncwarp();
      }
      ok = take(s, g);
      if (!ok || g.end) break;
      if (g.t1 <= g.t0) continue;
      const int qb = seq % QB;
      ok = mbar_wait(&sm.q_empty[qb], ((seq / QB) & 1) ^ 1u, status, 411);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      constexpr int U = HD / 8;  // 16-byte units of a row
      uint8_t* dst = sQ + qb * F::kQBytes;
      for (int x = threadIdx.x - 64; x < N * U; x += 64) {
        const int r = x / U, u = x % U;
        const bool valid = r < g.rows;
        const int pr = g.r0 + (valid ? r : 0), tok = pr / a.G;
        cp_async16(dst + (u >> 3) * (N * 128) + swz128(r, u & 7),
                   q + (int64_t)(g.row0 + tok) * a.q_ld +
                       (int64_t)(g.kvh * a.G + pr - tok * a.G) * HD + u * 8,
                   valid);
      }
      cp_async_wait_all();
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.q_full[qb]);
      ++seq;
    }
  } else {
    // ------------------------------------------------------------- softmax ----
    const int grp = (warp - 4) >> 2, bar = 1 + grp, cb = grp * CW;  // columns cb .. cb + CW
    const int quarter = warp & 3, tid = (threadIdx.x - 128) & 127;  // key, TMEM lane
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    float* mneg = sm.mneg + cb;
    float* fac = sm.fac + cb;
    // A wait that runs out only marks its thread: the group leaves together, at the next
    // barrier that all of its threads reach.
    bool bad = false, joined = false;
    int i = 0, seq = 0;
    Seg g;
    for (int s = 0;; ++s) {
      bad |= !take(s, g);
      if (vote_group(bar, bad) || g.end) break;
      const int par = seq & 1;
      float l[CW];
#pragma unroll
      for (int c = 0; c < CW; ++c) l[c] = 0.f;
      float m = -INFINITY;  // the bound of row cb + tid (tid < CW)
      const int tok0 = (g.r0 + cb) / a.G, rem0 = g.r0 + cb - tok0 * a.G;
      // keys that row cb sees
      const int64_t lim0 = a.all_rows ? g.kend : min(g.kend, g.lim0 + tok0 - g.r0 / a.G);
      bool left = false;
      for (int t = g.t0; t < g.t1; ++t, ++i) {
        const int st = i % ST, sb = i & 1;
        const int64_t k0 = a.kbeg + (int64_t)t * kTile;
        bad |= !mbar_wait(&sm.s_full[sb], (i >> 1) & 1, status, 412);
        tc_fence_after();
        float x[CW];
        tmem_ldn<CW>(tS + sb * N + cb + lane_off, x);
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.s_empty[sb]);
        if (k0 + kTile > lim0) {  // some row does not see all of the tile
          const int key = tid, kend = (int)min(g.kend - k0, (int64_t)kTile);
          int rem = rem0, lim = (int)max(min(lim0 - k0, (int64_t)kTile), -(int64_t)(1 << 30));
#pragma unroll
          for (int c = 0; c < CW; ++c) {
            x[c] = key < lim ? x[c] : -INFINITY;
            if (!a.all_rows && ++rem == a.G) {
              rem = 0;
              lim = min(lim + 1, kend);
            }
          }
        }
        // does any score pass its row's bound by more than 2^8?
        bool raise = bad || t == g.t0 || (tid < CW && m == -INFINITY);
        if (t > g.t0) {
          float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int c = 0; c < CW; c += 8) {
            const float4 n0 = *reinterpret_cast<const float4*>(&mneg[c]);
            const float4 n1 = *reinterpret_cast<const float4*>(&mneg[c + 4]);
            top[0] = max3f(top[0], fmaf(x[c], a.scale_log2, n0.x), fmaf(x[c + 1], a.scale_log2, n0.y));
            top[1] = max3f(top[1], fmaf(x[c + 2], a.scale_log2, n0.z), fmaf(x[c + 3], a.scale_log2, n0.w));
            top[2] = max3f(top[2], fmaf(x[c + 4], a.scale_log2, n1.x), fmaf(x[c + 5], a.scale_log2, n1.y));
            top[3] = max3f(top[3], fmaf(x[c + 6], a.scale_log2, n1.z), fmaf(x[c + 7], a.scale_log2, n1.w));
          }
          raise |= max3f(top[0], top[1], fmaxf(top[2], top[3])) > kRaise;
        }
        if (vote_group(bar, raise)) {
#pragma unroll
          for (int c = 0; c < CW; ++c) {
            const float wm = redux_max(x[c]);
            if (lane == c) sm.mx[quarter][cb + c] = wm;
          }
          if (vote_group(bar, bad)) {
            left = true;
            break;
          }
          if (tid < CW) {
            const int c = cb + tid;
            const float mt = fmaxf(fmaxf(sm.mx[0][c], sm.mx[1][c]),
                                   fmaxf(sm.mx[2][c], sm.mx[3][c])) * a.scale_log2;
            float f = 1.f;
            if (mt > m + kRaise || (m == -INFINITY && mt > m)) {
              f = m == -INFINITY ? 0.f : exp2f(m - mt);
              m = mt;
            }
            mneg[tid] = m == -INFINITY ? 0.f : -m;
            fac[tid] = f;
          }
          bar_group(bar);
          if (t > g.t0) {
#pragma unroll
            for (int c = 0; c < CW; ++c) l[c] *= fac[c];
            // the accumulator of the tiles before this one
            bad |= !mbar_wait(&sm.p_empty, (i - 1) & 1, status, 413);
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < CW; c += 16) {
              float ov[16];
              uint32_t ou[16];
              tmem_ld16(tO + par * N + cb + c + lane_off, ov);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) ou[e] = __float_as_uint(ov[e] * fac[c + e]);
              tmem_st16(tO + par * N + cb + c + lane_off, ou);
            }
            tmem_wait_st();
          }
        }
        // probabilities, rounded to bf16 for the tensor core (their sum is not: see above)
        if (i > 0) bad |= !mbar_wait(&sm.p_empty, (i - 1) & 1, status, 414);
#pragma unroll
        for (int u = 0; u < CW / 8; ++u) {
          uint32_t pk[4];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int c = 8 * u + 4 * e;
            const float4 n0 = *reinterpret_cast<const float4*>(&mneg[c]);
            const float p0 = ex2_approx(fmaf(x[c], a.scale_log2, n0.x));
            const float p1 = ex2_approx(fmaf(x[c + 1], a.scale_log2, n0.y));
            const float p2 = ex2_approx(fmaf(x[c + 2], a.scale_log2, n0.z));
            const float p3 = ex2_approx(fmaf(x[c + 3], a.scale_log2, n0.w));
            l[c] += p0;
            l[c + 1] += p1;
            l[c + 2] += p2;
            l[c + 3] += p3;
            pk[2 * e] = pack_bf16x2(p0, p1);
            pk[2 * e + 1] = pack_bf16x2(p2, p3);
          }
          *reinterpret_cast<uint4*>(sP + swz128(tid, cb / 8 + u)) =
              make_uint4(pk[0], pk[1], pk[2], pk[3]);
        }
        if (k0 + kTile > g.kend) {
          // what lies behind the last key (another request's rows, or anything at all)
          // must not meet its zero probabilities: 0 x NaN.  (Two groups write the same
          // zeros, each before its own part of P is handed over.)
          bad |= !mbar_wait(&sm.v_full[st], (i / ST) & 1, status, 415);
          if (k0 + tid >= g.kend) {
#pragma unroll
            for (int u = 0; u < 8 * HDC; ++u)
              *reinterpret_cast<uint4*>(sV + st * F::kTileBytes + (u >> 3) * kChunk +
                                        swz128(tid, u & 7)) = make_uint4(0, 0, 0, 0);
          }
        }
        fence_proxy_async();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.p_full);
      }
      if (left) break;
      // ---- the segment's rows ----
      const bool any = g.t1 > g.t0, whole = g.slot < 0;
      const int live = min(CW, g.rows - cb);  // this group's rows (none below 1)
      lane_sums<CW>(l, lane);
      if constexpr (CW == 32) {
        sm.mx[quarter][cb + lane] = l[0];
      } else {
        if (!(lane & 1)) sm.mx[quarter][cb + (lane >> 1)] = l[0];
      }
      if (vote_group(bar, bad)) break;
      if (a.pre_lse && !joined) {
        wait_kernel_before();  // the prefix's rows
        joined = true;
      }
      if (tid < live) {
        const int c = cb + tid;
        const float sum = (sm.mx[0][c] + sm.mx[1][c]) + (sm.mx[2][c] + sm.mx[3][c]);
        if (whole) {
          const int pr = g.r0 + c, tok = pr / a.G;
          const int row = g.row0 + tok, head = g.kvh * a.G + pr - tok * a.G;
          const RowScale f = finish_row(a, row, head, m, sum);
          mneg[tid] = f.own;
          fac[tid] = f.pre;
          a.lse[(int64_t)head * a.T + row] = f.lse;
        } else {
          const int64_t row = (int64_t)g.slot * N + c;
          a.part_ml[2 * row] = m;
          a.part_ml[2 * row + 1] = sum;
        }
      }
      bar_group(bar);
      if (any) {
        bad |= !mbar_wait(&sm.o_full[par], (seq >> 1) & 1, status, 416);
        tc_fence_after();
      }
      // elements of the group's first row in o and in the fp32 rows; the next row is one
      // head on, or in the next token's row
      int rem = rem0;
      const int64_t trow = g.row0 + tok0, thead = g.kvh * a.G + rem0;
      int64_t o_at = trow * a.o_ld + thead * HD + tid, f_at = (trow * a.Hq + thead) * HD + tid;
      float* part = whole ? nullptr : a.part_o + ((int64_t)g.slot * N + cb) * HD + tid;
#pragma unroll 1
      for (int c0 = 0; c0 < live; c0 += 8) {
        float ov[8];
        if (any) {
          tmem_ld8(tO + par * N + cb + c0 + lane_off, ov);
          tmem_wait_ld();
        }
        if (tid >= HD) continue;
        if (part) {
          if (any) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (c0 + e < live) part[(c0 + e) * HD] = ov[e];
          }
          continue;
        }
        float pv[8];
        int64_t at[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          at[e] = a.o32 ? f_at : o_at;
          // (loads without branches, so that the chunk's eight are in flight together)
          pv[e] = a.pre_o ? a.pre_o[c0 + e < live ? f_at : tid] : 0.f;
          f_at += HD;
          o_at += HD;
          if (++rem == a.G) {
            rem = 0;
            f_at += (int64_t)(a.Hq - a.G) * HD;
            o_at += a.o_ld - (int64_t)a.G * HD;
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (c0 + e >= live) continue;
          const float own = mneg[c0 + e], pre = fac[c0 + e];
          const float v = (!any || own == 0.f ? 0.f : ov[e] * own) + (pre == 0.f ? 0.f : pre * pv[e]);
          if (a.o32)
            a.o32[at[e]] = v;
          else
            static_cast<__nv_bfloat16*>(a.o)[at[e]] = __float2bfloat16_rn(v);
        }
      }
      if (any) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.o_empty[par]);
        ++seq;
      }
      // (the vote at the next segment's start: mneg, fac and mx are its own from there)
    }
  }

  wait_kernel_before();  // (also where nothing was joined: the kernels end in order)
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(sm.tmem, F::kTmem);
  }
}

template <int N, int HDC>
int launch(const Args& a, int blocks, bool dependent, cudaStream_t st) {
  int shift = 7;  // boxes of up to a tile's keys that divide a page (a multiple of 16)
  while (a.page % (1 << shift)) --shift;
  CUtensorMap tk, tv;
  const uint64_t rows = (uint64_t)a.num_pages * a.Hkv * a.page;
  int rc = make_tmap_2d(&tk, a.kc, 64 * HDC, rows, 128 * HDC, 64, 1u << shift);
  if (!rc) rc = make_tmap_2d(&tv, a.vc, 64 * HDC, rows, 128 * HDC, 64, 1u << shift);
  if (rc) return rc;
  auto kern = paged_few_kernel<N, HDC>;
  constexpr int smem = (int)Few<N, HDC>::kSmem;
  const int rcs = allow_smem<paged_few_kernel<N, HDC>>(smem);
  if (rcs) return rcs;
  return launch_kernel(kern, dim3((unsigned)blocks), Few<N, HDC>::kThreads, smem, st, dependent, tk,
                       tv, a, shift);
}

}  // namespace

int launch_few(const Args& a, int rows, int blocks, bool dependent, cudaStream_t st) {
  const bool wide = a.hd == 128;
  switch (rows) {
    case 16: return wide ? launch<16, 2>(a, blocks, dependent, st) : launch<16, 1>(a, blocks, dependent, st);
    case 32: return wide ? launch<32, 2>(a, blocks, dependent, st) : launch<32, 1>(a, blocks, dependent, st);
    default: return wide ? launch<64, 2>(a, blocks, dependent, st) : launch<64, 1>(a, blocks, dependent, st);
  }
}

}  // namespace paged
}  // namespace pe
