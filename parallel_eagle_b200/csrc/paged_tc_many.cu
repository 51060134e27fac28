// Attention over the paged key/value cache for many rows -- prompts in chunks, and the rows
// of a whole batch against its shared prefix -- on the 5th-generation tensor cores.  bf16,
// fp32 softmax, head sizes 64 and 128.
//
// With hundreds of rows per key the two products bound the kernel (4 hd operations per row
// and key against 4 hd bytes per key).  A block holds 256 packed rows (new tokens x query
// heads of a KV head's group) as two 128-row tiles A and B, so the tensor core always has
// one tile's products to run while the other tile's softmax executes:
//
//   warp 0       TMA: K and V tiles of 64 keys, boxes of one page's keys, through two rings
//   warp 1       tcgen05.mma, per key tile:  PV_A(j) S_A(j+2) PV_B(j) S_B(j+2)
//                (S = Q K^T into TMEM; P read from TMEM as the A operand)
//   warp 2       walks the line of work and publishes segments; warps 2..3 fetch Q rows
//   warps 4..7   softmax of tile A, one thread per row (TMEM lane); warps 8..11 of tile B
//
// TMEM: O_A columns 0..127, O_B 128..255, two S of 64 columns for A and two for B behind
// them; P overwrites the first 32 columns of its S as packed bf16 pairs.  With two S a tile
// the next scores are there when a softmax ends, so both tiles' softmax run all the time;
// with one S of 128 keys they took turns with their own products (3840 cycles per 128
// keys, the tensor pipe half idle).  A row's maximum is only raised (and O rescaled) when
// it grows by more than 2^8.  The exponentials all run on the SFU: a share of them on the FMA
// pipe was no faster (1/8, 1/4) or slower (1/2), and costs power.  P is rounded to bf16, as the
// tensor core's operand has to be (its sum is not): off by at most 2^-8 each, results 2.3e-3
// (rms, relative) from 64 bits, 1.7e-3 of it their own rounding.
//
// Measured: 1600 packed rows a KV head over a prefix of 64K keys, 40/8 heads of 128, 450 us
// in single calls, 950 TFLOP/s (0.56 of the burst rate), and about 500 us when repeated
// under the power cap; two prompts of ~1000 rows over ~4K keys, 28/4 heads, 135 us.  A few
// registers spill (16 to 24 bytes).  Three
// things take about as long each: without the softmax 390 us, without the products 380 us,
// copies and barriers alone 300 us.  With 64 keys a tile the scores read Q from shared
// memory once per 64 columns, which bounds their products; 128 keys leave TMEM for one S a
// tile only (slower, above).
#include "paged.cuh"
#include "sm100.cuh"

namespace pe {
namespace paged {
namespace {

using namespace sm100;

constexpr int kThreads = 384;
constexpr int kRows = 256;                    // packed rows per block
constexpr int kHalf = 128;                    // rows per softmax group
constexpr int kTile = 64;                     // keys per tile
constexpr int kStages = 4;                    // K tiles, V tiles in shared memory
constexpr uint32_t kChunk = kTile * 128;      // 64 keys x 64 columns, 128-byte swizzled
constexpr uint32_t kQChunk = kHalf * 128;     // 128 rows x 64 columns
constexpr int kOver = 4 * kTile;              // a segment's start and end, in keys
constexpr float kRaise = 8.f;

struct Small {
  Seg seg[2];
  int64_t scratch[kThreads / 32 + 4];
  uint64_t seg_full[2], seg_empty[2];
  uint64_t k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
  uint64_t q_full, q_empty, o_full[2], o_empty[2];
  uint64_t s_full[2][2], p_full[2][2], pv_done[2];  // [row tile] ([S buffer])
  uint32_t tmem;
};

template <int HDC>
constexpr size_t smem_bytes() {
  return 1024 + 2 * HDC * kQChunk /* Q_A, Q_B */ + 2 * kStages * HDC * kChunk + sizeof(Small);
}

__device__ __forceinline__ uint32_t swz128(int r, int u) {
  return (uint32_t)(r * 128 + ((u ^ (r & 7)) << 4));
}
// 32 bytes, a whole sector, by one thread (rows lie one to a thread)
__device__ __forceinline__ void st_v8(float* p, const float* v) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0]),
               "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}
__device__ __forceinline__ void cp_async16(void* dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src),
               "r"(valid ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() {
  asm volatile("cp.async.wait_all;" ::: "memory");
}

template <int HDC>
__global__ void __launch_bounds__(kThreads, 1)
paged_many_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                  const __grid_constant__ Args a, int shift, int o_vec) {
  constexpr int HD = 64 * HDC;
  constexpr uint32_t kTileBytes = HDC * kChunk, kQBytes = HDC * kQChunk;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint8_t* sQ = smem;  // row tile h at + h * kQBytes
  uint8_t* sK = sQ + 2 * kQBytes;
  uint8_t* sV = sK + kStages * kTileBytes;
  Small& sm = *reinterpret_cast<Small*>(sV + kStages * kTileBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int* status = a.status;

  start_next_kernel();
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.seg_full[i], 1);
      mbar_init(&sm.seg_empty[i], kThreads / 32);  // every warp reads it
      mbar_init(&sm.o_full[i], 1);
      mbar_init(&sm.o_empty[i], 4);
      mbar_init(&sm.pv_done[i], 1);
      for (int j = 0; j < 2; ++j) {
        mbar_init(&sm.s_full[i][j], 1);
        mbar_init(&sm.p_full[i][j], 4);
      }
    }
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&sm.k_full[i], 1);
      mbar_init(&sm.k_empty[i], 1);
      mbar_init(&sm.v_full[i], 1);
      mbar_init(&sm.v_empty[i], 1);
    }
    mbar_init(&sm.q_full, 2);
    mbar_init(&sm.q_empty, 1);
    fence_barrier_init();
    fence_proxy_async();
    prefetch_tmap(&tmK);
    prefetch_tmap(&tmV);
    a.open[blockIdx.x].parts = 0;
  }
  if (warp == 1) {
    tmem_alloc(&sm.tmem, 512);
    tmem_relinquish();
  }
  Sched<kRows, kTile, kOver, 4 * kTile> w(a);
  if (w.requests() > w.kWarpRequests)
    w.init(sm.scratch);
  else if (warp == 2)
    w.init_warp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem;

  // segment s, copied out of shared memory and released; false: the wait ran out
  auto take = [&](int s, Seg& g) -> bool {
    const bool ok = mbar_wait(&sm.seg_full[s & 1], (s >> 1) & 1, status, 421);
    if (!__all_sync(0xffffffffu, ok)) return false;
    g = sm.seg[s & 1];
    __syncwarp();
    if (lane == 0) mbar_arrive(&sm.seg_empty[s & 1]);
    return true;
  };
  // keys that tile A's last row sees
  auto kend_a = [&](const Seg& g) -> int64_t {
    if (a.all_rows || g.rows <= kHalf) return g.kend;
    return min(g.kend, g.lim0 + (g.r0 + kHalf - 1) / a.G - g.r0 / a.G);
  };

  if (warp < 4) {
    if (warp == 0) {
      // ---------------------------------------------------------------- TMA ----
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
          const uint32_t bytes = (uint32_t)live * HDC * box * 128;
          const uint32_t off = st * kTileBytes + ch * kChunk + at * box * 128;
          ok = mbar_wait(&sm.k_empty[st], ph ^ 1u, status, 422);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          if (lane == 0) mbar_arrive_expect_tx(&sm.k_full[st], bytes);
          __syncwarp();
          if (mine) tma_load_2d(sK + off, &tmK, &sm.k_full[st], ch * 64, row);
          ok = mbar_wait(&sm.v_empty[st], ph ^ 1u, status, 423);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) {
            mbar_wait(&sm.k_full[st], ph, nullptr, 0);  // its copies land before the block ends
            break;
          }
          if (lane == 0) mbar_arrive_expect_tx(&sm.v_full[st], bytes);
          __syncwarp();
          if (mine) tma_load_2d(sV + off, &tmV, &sm.v_full[st], ch * 64, row);
          if (++st == kStages) { st = 0; ph ^= 1u; }
        }
      }
      if (!ok) {  // copies in flight land before the block ends
        for (int back = 1; back <= kStages && back <= i; ++back) {
          const int j = i - back;
          mbar_wait(&sm.k_full[j % kStages], (j / kStages) & 1, nullptr, 0);
          mbar_wait(&sm.v_full[j % kStages], (j / kStages) & 1, nullptr, 0);
        }
      }
    } else if (warp == 1) {
      // ---------------------------------------------------------------- MMA ----
      constexpr uint32_t ID_S = idesc_bf16(kHalf, kTile, false, false);
      constexpr uint32_t ID_O = idesc_bf16(kHalf, HD, false, true);
      const uint32_t q_lo = sw128_lo(smem_u32(sQ), 16);
      const uint32_t k_lo = sw128_lo(smem_u32(sK), 16);
      const uint32_t v_lo = sw128_lo(smem_u32(sV), kChunk);
      auto issue_s = [&](int h, int j) {
        const uint32_t qa = q_lo + h * (kQBytes >> 4);
        const uint32_t kb = k_lo + (j % kStages) * (kTileBytes >> 4);
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
          mma_bf16_ss_lo(tmem + 256 + h * 128 + (j & 1) * 64,
                         qa + (((kk >> 2) * kQChunk + (kk & 3) * 32) >> 4),
                         kb + (((kk >> 2) * kChunk + (kk & 3) * 32) >> 4), ID_S, kk > 0 ? 1u : 0u);
      };
      auto issue_pv = [&](int h, int j, bool first) {
        const uint32_t vb = v_lo + (j % kStages) * (kTileBytes >> 4);
        const uint32_t p = tmem + 256 + h * 128 + (j & 1) * 64;
#pragma unroll
        for (int kk = 0; kk < kTile / 16; ++kk)
          mma_bf16_ts_lo(tmem + h * 128, p + kk * 8, vb + kk * (2048 >> 4), ID_O,
                         kk > 0 ? 1u : first ? 0u : 1u);
      };
      bool ok = true;
      int i = 0, seq = 0;
      Seg g;
      for (int s = 0; ok; ++s) {
        ok = take(s, g);
        if (!ok || g.end) break;
        if (g.t1 <= g.t0) continue;
        const int64_t ka = kend_a(g);
        const bool two = g.rows > kHalf;
        const int n = g.t1 - g.t0;
        // tiles of the segment that tile A sees
        const int na = (int)max((int64_t)0, min((int64_t)n, (ka - a.kbeg + kTile - 1) / kTile - g.t0));
        if (elect_one()) {
          // scores of the segment's tile u into the buffer that tile u - 2 left
          auto scores = [&](int h, int u) -> bool {
            const int j = i + u;
            if (h == 0) {
              if (!mbar_wait(&sm.k_full[j % kStages], (j / kStages) & 1, status, 425)) return false;
              tc_fence_after();
            }
            if (h == 0 ? u < na : two) issue_s(h, j);
            mma_commit(&sm.s_full[h][j & 1]);
            if (h == 1) {
              mma_commit(&sm.k_empty[j % kStages]);
              if (u + 1 == n) mma_commit(&sm.q_empty);
            }
            return true;
          };
          ok = mbar_wait(&sm.q_full, seq & 1, status, 424);
          for (int u = 0; u < 2 && u < n && ok; ++u) ok = scores(0, u) && scores(1, u);
          for (int u = 0; u < n && ok; ++u) {
            const int j = i + u;
            ok = mbar_wait(&sm.v_full[j % kStages], (j / kStages) & 1, status, 426) &&
                 mbar_wait(&sm.p_full[0][j & 1], (j >> 1) & 1, status, 427) &&
                 (u > 0 || (mbar_wait(&sm.o_empty[0], (seq & 1) ^ 1u, status, 428) &&
                            mbar_wait(&sm.o_empty[1], (seq & 1) ^ 1u, status, 429)));
            if (!ok) break;
            tc_fence_after();
            if (u < na) issue_pv(0, j, u == 0);
            mma_commit(&sm.pv_done[0]);
            if (u + 2 < n && !scores(0, u + 2)) { ok = false; break; }
            ok = mbar_wait(&sm.p_full[1][j & 1], (j >> 1) & 1, status, 430);
            if (!ok) break;
            tc_fence_after();
            if (two) issue_pv(1, j, u == 0);
            mma_commit(&sm.pv_done[1]);
            mma_commit(&sm.v_empty[j % kStages]);
            if (u + 2 < n && !scores(1, u + 2)) { ok = false; break; }
          }
          if (ok) {
            mma_commit(&sm.o_full[0]);
            mma_commit(&sm.o_full[1]);
          }
        }
        ok = __all_sync(0xffffffffu, ok);
        i += n;
        ++seq;
      }
    } else {
      // ----------------------------------------------- line of work, Q rows ----
      const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a.q);
      bool ok = true;
      int seq = 0;
      Seg g;
      for (int s = 0; ok; ++s) {
        if (warp == 2) {
          ok = mbar_wait(&sm.seg_empty[s & 1], ((s >> 1) & 1) ^ 1u, status, 432);
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
        ok = mbar_wait(&sm.q_empty, (seq & 1) ^ 1u, status, 433);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        // unit u of rows r0, r0 + step, ...: the address moves on by heads, and to the next
        // token's row where a group ends
        constexpr int U = HD / 8, step = 64 / U;
        const int n = g.rows > kHalf ? kRows : kHalf;
        const int u = (threadIdx.x - 64) % U;
        int r = (threadIdx.x - 64) / U;
        const int tok = (g.r0 + r) / a.G;
        int rem = g.r0 + r - tok * a.G;
        const __nv_bfloat16* src = q + (int64_t)(g.row0 + tok) * a.q_ld +
                                   (int64_t)(g.kvh * a.G + rem) * HD + u * 8;
        uint8_t* dst = sQ + (u >> 3) * kQChunk;
#pragma unroll 8
        for (; r < n; r += step) {
          const bool valid = r < g.rows;
          cp_async16(dst + (r >> 7) * kQBytes + swz128(r & 127, u & 7), valid ? src : q, valid);
          src += step * HD;
          rem += step;
          while (rem >= a.G) {
            rem -= a.G;
            src += a.q_ld - (int64_t)a.G * HD;
          }
        }
        cp_async_wait_all();
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.q_full);
        ++seq;
      }
    }
  } else {
    // --------------------------------------------------------------- softmax ----
    const int h = (warp - 4) >> 2;  // row tile A or B
    const int quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const uint32_t tO = tmem + h * 128 + lane_off;
    const float scale = a.scale_log2;
    bool ok = true, joined = false;
    int i = 0, seq = 0;
    Seg g;
    for (int s = 0; ok; ++s) {
      ok = take(s, g);
      if (!ok || g.end) break;
      const int rr = g.r0 + h * kHalf + row;  // packed row of the request
      const bool valid = h * kHalf + row < g.rows;
      const int tok = rr / a.G;
      const int64_t lim = !valid ? -1 : a.all_rows ? g.kend
                          : min(g.kend, g.lim0 + tok - g.r0 / a.G);
      // the group's tiles: those some row of it sees
      const int64_t gend = h == 0 ? kend_a(g) : g.rows > kHalf ? g.kend : -1;
      float m = -INFINITY, l = 0.f;
      for (int t = g.t0; t < g.t1; ++t, ++i) {
        const uint32_t tS = tmem + 256 + h * 128 + (i & 1) * 64 + lane_off;
        ok = mbar_wait(&sm.s_full[h][i & 1], (i >> 1) & 1, status, 434);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        const int64_t k0 = a.kbeg + (int64_t)t * kTile;
        if (k0 < gend) {
          float x[64];
          tmem_ld32(tS, x);
          tmem_ld32(tS + 32, x + 32);
          tmem_wait_ld();
          if (k0 + kTile > lim) {
            const int see = (int)max((int64_t)0, lim - k0);
#pragma unroll
            for (int c = 0; c < 64; ++c) x[c] = c < see ? x[c] : -INFINITY;
          }
          float mp[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) mp[u] = -INFINITY;
#pragma unroll
          for (int c = 0; c < 64; c += 8) {
#pragma unroll
            for (int u = 0; u < 4; ++u) mp[u] = max3f(mp[u], x[c + 2 * u], x[c + 2 * u + 1]);
          }
          const float mt = max3f(mp[0], mp[1], fmaxf(mp[2], mp[3])) * scale;
          float alpha = 1.f;
          if (mt > m + kRaise || (m == -INFINITY && mt > m)) {
            alpha = m == -INFINITY ? 0.f : ex2_approx(m - mt);
            m = mt;
            l *= alpha;
          }
          const float nm = m == -INFINITY ? 0.f : -m;
          float2 rs[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) rs[u] = make_float2(0.f, 0.f);
          const float2 sc = make_float2(scale, scale), off = make_float2(nm, nm);
          uint32_t pk[32];
#pragma unroll
          for (int c = 0; c < 64; c += 2) {
            const float2 y = fma2(make_float2(x[c], x[c + 1]), sc, off);
            const float2 p = make_float2(ex2_approx(y.x), ex2_approx(y.y));
            rs[(c >> 1) & 3] = add2(rs[(c >> 1) & 3], p);
            pk[c / 2] = pack_bf16x2(p.x, p.y);
          }
          tmem_st32(tS, pk);
          const float2 rsum = add2(add2(rs[0], rs[1]), add2(rs[2], rs[3]));
          l += rsum.x + rsum.y;
          // O holds the tiles before this one, once their product is done
          if (__any_sync(0xffffffffu, alpha != 1.f) && t > g.t0) {
            ok = mbar_wait(&sm.pv_done[h], (i - 1) & 1, status, 437);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < HD; c += 32) {
              float ov[32];
              tmem_ld32(tO + c, ov);
              tmem_wait_ld();
              uint32_t ou[32];
#pragma unroll
              for (int u = 0; u < 32; ++u) ou[u] = __float_as_uint(ov[u] * alpha);
              tmem_st32(tO + c, ou);
            }
          }
          tmem_wait_st();
          if (k0 + kTile > g.kend) {
            // what lies behind the last key must not meet its zero probabilities (0 x NaN);
            // both row tiles write the same zeros
            ok = mbar_wait(&sm.v_full[i % kStages], (i / kStages) & 1, status, 435);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            if (row < kTile && k0 + row >= g.kend) {
              uint8_t* v = sV + (i % kStages) * kTileBytes;
#pragma unroll
              for (int u = 0; u < 8 * HDC; ++u)
                *reinterpret_cast<uint4*>(v + (u >> 3) * kChunk + swz128(row, u & 7)) =
                    make_uint4(0, 0, 0, 0);
            }
          }
          fence_proxy_async();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.p_full[h][i & 1]);
      }
      if (!ok) break;
      // ---- the segment's rows ----
      const bool any = g.t1 > g.t0;
      if (any) {
        ok = mbar_wait(&sm.o_full[h], seq & 1, status, 436);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
      }
      if (a.pre_lse && !joined) {
        wait_kernel_before();  // the prefix's rows
        joined = true;
      }
      const int orow = g.row0 + tok, head = g.kvh * a.G + rr - tok * a.G;
      RowScale f{0.f, 0.f, 0.f};
      float* po = nullptr;
      if (g.slot >= 0) {
        const int64_t prow = (int64_t)g.slot * kRows + h * kHalf + row;
        po = a.part_o + prow * HD;
        if (valid) {
          a.part_ml[2 * prow] = m;
          a.part_ml[2 * prow + 1] = l;
        }
      } else if (valid) {
        f = finish_row(a, orow, head, m, l);
        a.lse[(int64_t)head * a.T + orow] = f.lse;
      }
#pragma unroll 1
      for (int c = 0; c < HD; c += 32) {
        float ov[32];
        if (any) {
          tmem_ld32(tO + c, ov);
          tmem_wait_ld();
        }
        if (!valid) continue;
        if (po) {
          if (l != 0.f) {
#pragma unroll
            for (int e = 0; e < 32; e += 8) st_v8(po + c + e, ov + e);
          }
          continue;
        }
#pragma unroll
        for (int e = 0; e < 32; ++e) ov[e] = f.own == 0.f ? 0.f : ov[e] * f.own;
        const int64_t at = ((int64_t)orow * a.Hq + head) * HD + c;
        if (f.pre != 0.f) {
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const float4 pv = *reinterpret_cast<const float4*>(a.pre_o + at + e);
            ov[e] += f.pre * pv.x;
            ov[e + 1] += f.pre * pv.y;
            ov[e + 2] += f.pre * pv.z;
            ov[e + 3] += f.pre * pv.w;
          }
        }
        if (a.o32) {
#pragma unroll
          for (int e = 0; e < 32; e += 8) st_v8(a.o32 + at + e, ov + e);
        } else {
          __nv_bfloat16* dst =
              static_cast<__nv_bfloat16*>(a.o) + (int64_t)orow * a.o_ld + head * HD + c;
          if (o_vec) {
#pragma unroll
            for (int e = 0; e < 32; e += 8)
              *reinterpret_cast<uint4*>(dst + e) =
                  make_uint4(pack_bf16x2(ov[e], ov[e + 1]), pack_bf16x2(ov[e + 2], ov[e + 3]),
                             pack_bf16x2(ov[e + 4], ov[e + 5]), pack_bf16x2(ov[e + 6], ov[e + 7]));
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) dst[e] = __float2bfloat16_rn(ov[e]);
          }
        }
      }
      if (any) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.o_empty[h]);
        ++seq;
      }
    }
  }

  wait_kernel_before();  // (also where nothing was joined: the kernels end in order)
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int HDC>
int launch(const Args& a, int blocks, bool dependent, cudaStream_t st) {
  int shift = 6;  // boxes of up to a tile's keys that divide a page (a multiple of 16)
  while (a.page % (1 << shift)) --shift;
  CUtensorMap tk, tv;
  const uint64_t rows = (uint64_t)a.num_pages * a.Hkv * a.page;
  int rc = make_tmap_2d(&tk, a.kc, 64 * HDC, rows, 128 * HDC, 64, 1u << shift);
  if (!rc) rc = make_tmap_2d(&tv, a.vc, 64 * HDC, rows, 128 * HDC, 64, 1u << shift);
  if (rc) return rc;
  auto kern = paged_many_kernel<HDC>;
  constexpr int smem = (int)smem_bytes<HDC>();
  static_assert(smem <= 227 * 1024, "shared memory");
  const int rcs = allow_smem<paged_many_kernel<HDC>>(smem);
  if (rcs) return rcs;
  const int o_vec = (reinterpret_cast<uintptr_t>(a.o) & 15u) == 0 && a.o_ld % 8 == 0;
  return launch_kernel(kern, dim3((unsigned)blocks), kThreads, smem, st, dependent, tk, tv, a, shift,
                       o_vec);
}

}  // namespace

int launch_many(const Args& a, int blocks, bool dependent, cudaStream_t st) {
  return a.hd == 128 ? launch<2>(a, blocks, dependent, st) : launch<1>(a, blocks, dependent, st);
}

}  // namespace paged
}  // namespace pe
