// Attention over the paged key/value cache for many rows -- prompts in chunks, and the rows
// of a whole batch against its shared prefix -- on the 5th-generation tensor cores.  bf16,
// fp32 softmax, head sizes 64 and 128.
//
// With hundreds of rows per key the two products bound the kernel (4 hd operations per row
// and key against 4 hd bytes per key).  A block holds 256 packed rows (new tokens x query
// heads of a KV head's group) as two 128-row tiles A and B, so the tensor core always has
// one tile's products to run while the other tile's softmax executes:
//
//   warp 0       TMA: K and V tiles of 128 keys, boxes of one page's keys, two stages
//   warp 1       tcgen05.mma, per key tile:  PV_A(j) S_A(j+1) PV_B(j) S_B(j+1)
//                (S = Q K^T into TMEM; P read from TMEM as the A operand)
//   warp 2       walks the line of work and publishes segments; warps 2..3 fetch Q rows
//   warps 4..7   softmax of tile A, one thread per row (TMEM lane); warps 8..11 of tile B
//
// TMEM: O_A columns 0..127, O_B 128..255, S_A 256..383, S_B 384..511; P overwrites the first
// 64 columns of its S as packed bf16 pairs.  A row's maximum is only raised (and O rescaled)
// when it grows by more than 2^8.  Every fourth pair of exponentials runs on the FMA pipe,
// as the SFU's 16 per clock would take longer than the products.
#include "paged.cuh"
#include "sm100.cuh"

namespace pe {
namespace paged {
namespace {

using namespace sm100;

constexpr int kThreads = 384;
constexpr int kRows = 256;                    // packed rows per block
constexpr int kTile = 128;                    // keys per tile, rows per softmax group
constexpr uint32_t kChunk = kTile * 128;      // 128 rows x 64 columns, 128-byte swizzled
constexpr int kRegsLow = 88, kRegsHigh = 208; // 128 x 88 + 256 x 208 = 384 x 168
constexpr float kRaise = 8.f;
constexpr int kEmuEvery = 4;

struct Small {
  Seg seg[2];
  int64_t scratch[kThreads / 32 + 4];
  uint64_t seg_full[2], seg_empty[2], kv_full[2], kv_empty[2];
  uint64_t q_full, q_empty, s_full[2], p_full[2], o_full[2], o_empty[2];
  uint32_t tmem;
};

template <int HDC>
constexpr size_t smem_bytes() {
  return 1024 + 6 * HDC * kChunk /* Q_A, Q_B, two stages of K and V */ + sizeof(Small);
}

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

template <int HDC>
__global__ void __launch_bounds__(kThreads, 1)
paged_many_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                  const __grid_constant__ Args a, int box, int o_vec) {
  constexpr int HD = 64 * HDC;
  constexpr uint32_t kTileBytes = HDC * kChunk;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint8_t* sQ = smem;                    // tile t at + t * kTileBytes
  uint8_t* sKV = sQ + 2 * kTileBytes;    // stage s: K at + s * 2 * kTileBytes, V behind it
  Small& sm = *reinterpret_cast<Small*>(sKV + 4 * kTileBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int* status = a.status;

  start_next_kernel();
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.seg_full[i], 1);
      mbar_init(&sm.seg_empty[i], 12);  // every warp reads it
      mbar_init(&sm.kv_full[i], 1);
      mbar_init(&sm.kv_empty[i], 1);
      mbar_init(&sm.s_full[i], 1);
      mbar_init(&sm.p_full[i], 4);
      mbar_init(&sm.o_full[i], 1);
      mbar_init(&sm.o_empty[i], 4);
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
  Sched<kRows, kTile> w(a);
  w.init(sm.scratch);
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
    if (a.all_rows || g.rows <= kTile) return g.kend;
    return min(g.kend, g.lim0 + (g.r0 + kTile - 1) / a.G - g.r0 / a.G);
  };

  if (warp < 4) {
    setmaxnreg_dec<kRegsLow>();
    if (warp == 0) {
      // ---------------------------------------------------------------- TMA ----
      const int per_chunk = kTile / box, boxes = per_chunk * HDC;
      const int at = lane % per_chunk, ch = lane / per_chunk;
      const int total_rows = (int)(a.num_pages * a.Hkv * a.page);
      bool ok = true;
      int i = 0;
      Seg g;
      for (int s = 0; ok; ++s) {
        ok = take(s, g);
        if (!ok || g.end) break;
        for (int t = g.t0; t < g.t1; ++t, ++i) {
          const int64_t k0 = a.kbeg + (int64_t)t * kTile;
          const int live = min(per_chunk, (int)((g.kend - k0 + box - 1) / box));
          const bool mine = lane < boxes && at < live;
          int row = total_rows;  // (reads as zeros)
          if (mine) {
            const int64_t key = k0 + at * box, pi = key / a.page;
            const int id = g.pages[pi];
            if (id >= 0 && id < a.num_pages)
              row = (int)(((int64_t)id * a.Hkv + g.kvh) * a.page + (key - pi * a.page));
          }
          const int st = i & 1;
          ok = mbar_wait(&sm.kv_empty[st], ((i >> 1) & 1) ^ 1u, status, 422);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          uint8_t* dst = sKV + st * 2 * kTileBytes + ch * kChunk + at * box * 128;
          if (lane == 0)
            mbar_arrive_expect_tx(&sm.kv_full[st], (uint32_t)live * 2 * HDC * box * 128);
          __syncwarp();
          if (mine) {
            tma_load_2d(dst, &tmK, &sm.kv_full[st], ch * 64, row);
            tma_load_2d(dst + kTileBytes, &tmV, &sm.kv_full[st], ch * 64, row);
          }
        }
      }
      if (!ok) {  // copies in flight land before the block ends
        for (int back = 1; back <= 2 && back <= i; ++back)
          mbar_wait(&sm.kv_full[(i - back) & 1], ((i - back) >> 1) & 1, nullptr, 0);
      }
    } else if (warp == 1) {
      // ---------------------------------------------------------------- MMA ----
      constexpr uint32_t ID_S = idesc_bf16(kTile, kTile, false, false);
      constexpr uint32_t ID_O = idesc_bf16(kTile, HD, false, true);
      const uint32_t q_lo = sw128_lo(smem_u32(sQ), 16);
      const uint32_t kv_lo = sw128_lo(smem_u32(sKV), 16);
      const uint32_t v_lo = sw128_lo(smem_u32(sKV) + kTileBytes, kChunk);
      auto issue_s = [&](int h, int st) {
        const uint32_t qa = q_lo + h * (kTileBytes >> 4), kb = kv_lo + st * (2 * kTileBytes >> 4);
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
          const uint32_t off = ((kk >> 2) * kChunk + (kk & 3) * 32) >> 4;
          mma_bf16_ss_lo(tmem + 256 + h * 128, qa + off, kb + off, ID_S, kk > 0 ? 1u : 0u);
        }
      };
      auto issue_pv = [&](int h, int st, bool first) {
        const uint32_t vb = v_lo + st * (2 * kTileBytes >> 4);
        const uint32_t p = tmem + 256 + h * 128;
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
        const bool two = g.rows > kTile;
        if (elect_one()) {
          auto use_a = [&](int t) { return a.kbeg + (int64_t)t * kTile < ka; };
          ok = mbar_wait(&sm.q_full, seq & 1, status, 423) &&
               mbar_wait(&sm.kv_full[i & 1], (i >> 1) & 1, status, 424);
          if (ok) {
            tc_fence_after();
            if (use_a(g.t0)) issue_s(0, i & 1);
            mma_commit(&sm.s_full[0]);
            if (two) issue_s(1, i & 1);
            mma_commit(&sm.s_full[1]);
            if (g.t0 + 1 == g.t1) mma_commit(&sm.q_empty);
          }
          bool pv_a = false, pv_b = false;
          for (int t = g.t0, j = i; t < g.t1 && ok; ++t, ++j) {
            const int st = j & 1, sn = st ^ 1;
            const bool more = t + 1 < g.t1;
            if (!mbar_wait(&sm.p_full[0], j & 1, status, 425)) { ok = false; break; }
            if (t == g.t0 && (!mbar_wait(&sm.o_empty[0], (seq & 1) ^ 1u, status, 426) ||
                              !mbar_wait(&sm.o_empty[1], (seq & 1) ^ 1u, status, 427))) {
              ok = false;
              break;
            }
            tc_fence_after();
            if (use_a(t)) {
              issue_pv(0, st, !pv_a);
              pv_a = true;
            }
            if (more) {
              if (!mbar_wait(&sm.kv_full[sn], ((j + 1) >> 1) & 1, status, 428)) { ok = false; break; }
              tc_fence_after();
              if (use_a(t + 1)) issue_s(0, sn);
              mma_commit(&sm.s_full[0]);
            }
            if (!mbar_wait(&sm.p_full[1], j & 1, status, 429)) { ok = false; break; }
            tc_fence_after();
            if (two) {
              issue_pv(1, st, !pv_b);
              pv_b = true;
            }
            if (more) {
              if (two) issue_s(1, sn);
              mma_commit(&sm.s_full[1]);
              if (t + 2 == g.t1) mma_commit(&sm.q_empty);
            }
            mma_commit(&sm.kv_empty[st]);
          }
          if (ok) {
            mma_commit(&sm.o_full[0]);
            mma_commit(&sm.o_full[1]);
          }
        }
        ok = __all_sync(0xffffffffu, ok);
        i += g.t1 - g.t0;
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
          ok = mbar_wait(&sm.seg_empty[s & 1], ((s >> 1) & 1) ^ 1u, status, 430);
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
        ok = mbar_wait(&sm.q_empty, (seq & 1) ^ 1u, status, 431);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        constexpr int U = HD / 8;
        const int n = g.rows > kTile ? kRows : kTile;
        for (int x = threadIdx.x - 64; x < n * U; x += 64) {
          const int r = x / U, u = x % U;
          const bool valid = r < g.rows;
          const int pr = g.r0 + (valid ? r : 0), tok = pr / a.G;
          cp_async16(sQ + (r >> 7) * kTileBytes + (u >> 3) * kChunk + swz128(r & 127, u & 7),
                     q + (int64_t)(g.row0 + tok) * a.q_ld +
                         (int64_t)(g.kvh * a.G + pr - tok * a.G) * HD + u * 8,
                     valid);
        }
        cp_async_wait_all();
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.q_full);
        ++seq;
      }
    }
  } else {
    setmaxnreg_inc<kRegsHigh>();
    // --------------------------------------------------------------- softmax ----
    const int h = (warp - 4) >> 2;  // row tile A or B
    const int quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const uint32_t tS = tmem + 256 + h * 128 + lane_off, tO = tmem + h * 128 + lane_off;
    const float scale = a.scale_log2;
    bool ok = true, joined = false;
    int i = 0, seq = 0;
    Seg g;
    for (int s = 0; ok; ++s) {
      ok = take(s, g);
      if (!ok || g.end) break;
      const int rr = g.r0 + h * kTile + row;  // packed row of the request
      const bool valid = h * kTile + row < g.rows;
      const int tok = rr / a.G;
      const int64_t lim = !valid ? -1 : a.all_rows ? g.kend
                          : min(g.kend, g.lim0 + tok - g.r0 / a.G);
      // the group's tiles: those some row of it sees
      const int64_t gend = h == 0 ? kend_a(g) : g.rows > kTile ? g.kend : -1;
      float m = -INFINITY, l = 0.f;
      for (int t = g.t0; t < g.t1; ++t, ++i) {
        ok = mbar_wait(&sm.s_full[h], i & 1, status, 432);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        const int64_t k0 = a.kbeg + (int64_t)t * kTile;
        if (k0 < gend) {
          float x[128];
#pragma unroll
          for (int c = 0; c < 128; c += 32) tmem_ld32(tS + c, x + c);
          tmem_wait_ld();
          if (k0 + kTile > lim) {
            const int see = (int)max((int64_t)0, lim - k0);
#pragma unroll
            for (int c = 0; c < 128; ++c) x[c] = c < see ? x[c] : -INFINITY;
          }
          float mp[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) mp[u] = -INFINITY;
#pragma unroll
          for (int c = 0; c < 128; c += 8) {
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
#pragma unroll
          for (int c0 = 0; c0 < 128; c0 += 32) {
            uint32_t pk[16];
#pragma unroll
            for (int c = 0; c < 32; c += 2) {
              const float2 y = fma2(make_float2(x[c0 + c], x[c0 + c + 1]), sc, off);
              float2 p;
              if (kEmuEvery > 0 && (c / 2) % kEmuEvery == kEmuEvery - 1) {
                p = exp2_poly2(y);
              } else {
                p.x = ex2_approx(y.x);
                p.y = ex2_approx(y.y);
              }
              rs[(c >> 1) & 3] = add2(rs[(c >> 1) & 3], p);
              pk[c / 2] = pack_bf16x2(p.x, p.y);
            }
            tmem_st16(tS + c0 / 2, pk);
          }
          const float2 rsum = add2(add2(rs[0], rs[1]), add2(rs[2], rs[3]));
          l += rsum.x + rsum.y;
          // O holds the tiles before this one (their PV completed before this S did)
          if (__any_sync(0xffffffffu, alpha != 1.f) && t > g.t0) {
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
          if (k0 + kTile > g.kend && k0 + row >= g.kend) {
            // what lies behind the last key must not meet its zero probabilities (0 x NaN);
            // both groups write the same zeros
            uint8_t* v = sKV + (i & 1) * 2 * kTileBytes + kTileBytes;
#pragma unroll
            for (int u = 0; u < 8 * HDC; ++u)
              *reinterpret_cast<uint4*>(v + (u >> 3) * kChunk + swz128(row, u & 7)) =
                  make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.p_full[h]);
      }
      if (!ok) break;
      // ---- the segment's rows ----
      const bool any = g.t1 > g.t0;
      if (any) {
        ok = mbar_wait(&sm.o_full[h], seq & 1, status, 433);
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
        const int64_t prow = (int64_t)g.slot * kRows + h * kTile + row;
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
            for (int e = 0; e < 32; e += 4)
              *reinterpret_cast<float4*>(po + c + e) =
                  make_float4(ov[e], ov[e + 1], ov[e + 2], ov[e + 3]);
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
          for (int e = 0; e < 32; e += 4)
            *reinterpret_cast<float4*>(a.o32 + at + e) =
                make_float4(ov[e], ov[e + 1], ov[e + 2], ov[e + 3]);
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
  int box = kTile;
  while (a.page % box) box >>= 1;  // (pages are multiples of 16)
  CUtensorMap tk, tv;
  const uint64_t rows = (uint64_t)a.num_pages * a.Hkv * a.page;
  int rc = make_tmap_2d(&tk, a.kc, 64 * HDC, rows, 128 * HDC, 64, (uint32_t)box);
  if (!rc) rc = make_tmap_2d(&tv, a.vc, 64 * HDC, rows, 128 * HDC, 64, (uint32_t)box);
  if (rc) return rc;
  auto kern = paged_many_kernel<HDC>;
  constexpr int smem = (int)smem_bytes<HDC>();
  static_assert(smem <= 227 * 1024, "shared memory");
  PE_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  {
    // the warpgroups' register re-split assumes the launch grants 168 per thread:
    // with fewer, setmaxnreg.inc would wait for registers that never free up
    cudaFuncAttributes fa;
    PE_CUDA_TRY(cudaFuncGetAttributes(&fa, kern));
    PE_CHECK_ARG(fa.numRegs * kThreads >= 128 * kRegsLow + 256 * kRegsHigh,
                 "attn_paged: kernel compiled with too few registers");
  }
  const int o_vec = (reinterpret_cast<uintptr_t>(a.o) & 15u) == 0 && a.o_ld % 8 == 0;
  return launch_kernel(kern, dim3((unsigned)blocks), kThreads, smem, st, dependent, tk, tv, a, box,
                       o_vec);
}

}  // namespace

int launch_many(const Args& a, int blocks, bool dependent, cudaStream_t st) {
  return a.hd == 128 ? launch<2>(a, blocks, dependent, st) : launch<1>(a, blocks, dependent, st);
}

}  // namespace paged
}  // namespace pe
