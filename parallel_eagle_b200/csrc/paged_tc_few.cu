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
//   warps 2..3  Q rows -> shared memory, per segment
//   warps 4..7  softmax: a thread is a key (TMEM lane), its N scores in registers; sums of
//               the probabilities stay per thread until the segment ends.  The per-row
//               maximum is over keys, that is over threads: it is kept as a stale bound in
//               shared memory and only raised, by a reduction over the warps, when some
//               score passes it by 2^8 (one vote per tile), as the probabilities then
//               still fit bf16 and fp32.
// TMEM: S^T 2 x N columns, O^T 2 x N (two segments: the next one starts while this one's
// result is read).
#include "paged.cuh"
#include "sm100.cuh"

namespace pe {
namespace paged {
namespace {

using namespace sm100;

constexpr int kThreads = 256;
constexpr int kTile = 128;                    // keys per tile
constexpr uint32_t kChunk = kTile * 128;      // 128 keys x 64 columns, 128-byte swizzled
constexpr float kRaise = 8.f;                 // log2 of what a score may pass the bound by

template <int N, int HDC>
struct Few {
  static constexpr int kStages = HDC == 2 ? 3 : 6;
  static constexpr int kQBufs = N <= 32 ? 2 : 1;
  static constexpr uint32_t kTileBytes = HDC * kChunk;
  static constexpr uint32_t kQBytes = HDC * N * 128;
  static constexpr uint32_t kTmem = 4 * N;  // columns
  struct Small {
    float mneg[N];       // minus the rows' bounds (log2 units); the result's scale at the end
    float mx[4][N];      // per-warp maxima; per-warp sums
    float fac[N];        // what a raised bound multiplies the sums and the accumulator by
    int64_t scratch[kThreads / 32 + 4];
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

__device__ __forceinline__ void bar_softmax() {
  asm volatile("barrier.cta.sync 1, 128;" ::: "memory");
}
// all 128 softmax threads: whether any of them votes
__device__ __forceinline__ bool vote_softmax(bool mine) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, 1, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "r"((uint32_t)mine)
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
template <int N>
__device__ __forceinline__ void tmem_stn(uint32_t addr, const uint32_t* v) {
  if constexpr (N == 16) {
    tmem_st16(addr, v);
  } else {
#pragma unroll
    for (int c = 0; c < N; c += 32) tmem_st32(addr + c, v + c);
  }
}

// Sum v[0..N) over the 32 lanes with about N exchanges: halve the columns a lane answers
// for with every step.  Lane i ends with columns 2i, 2i + 1 (N = 64), i (32) or i / 2 (16).
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
__global__ void __launch_bounds__(kThreads, 1)
paged_few_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                 const __grid_constant__ Args a, int box) {
  using F = Few<N, HDC>;
  constexpr int ST = F::kStages, QB = F::kQBufs;
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

  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(&sm.k_full[i], 1);
      mbar_init(&sm.k_empty[i], 1);
      mbar_init(&sm.v_full[i], 1);
      mbar_init(&sm.v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.s_full[i], 1);
      mbar_init(&sm.s_empty[i], 4);
      mbar_init(&sm.o_full[i], 1);
      mbar_init(&sm.o_empty[i], 4);
    }
    mbar_init(&sm.p_full, 4);
    mbar_init(&sm.p_empty, 1);
    for (int i = 0; i < QB; ++i) {
      mbar_init(&sm.q_full[i], 2);
      mbar_init(&sm.q_empty[i], 1);
    }
    fence_barrier_init();
    fence_proxy_async();
    a.open[blockIdx.x].parts = 0;
  }
  if (warp == 1) {
    tmem_alloc(&sm.tmem, F::kTmem);
    tmem_relinquish();
  }
  Sched<N, kTile> w(a);
  w.init(sm.scratch);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tS = sm.tmem, tO = sm.tmem + 2 * N;

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA ----
    const int per_chunk = kTile / box;               // boxes of one 64-column chunk
    const int boxes = per_chunk * HDC;               // of one tile
    const int total_rows = (int)(a.num_pages * a.Hkv * a.page);
    bool ok = true;
    int i = 0;
    uint32_t st = 0, ph = 0;
    while (ok && w.next()) {
      const int32_t* pages = w.pages();
      for (int t = w.t0; t < w.t1; ++t, ++i) {
        const int64_t k0 = a.kbeg + (int64_t)t * kTile;
        const int live = min(per_chunk, (int)((w.kend - k0 + box - 1) / box));
        // lane -> box: key offset, column chunk and the pool row it starts at
        const int u = lane < boxes ? lane : 0;
        const int at = u % per_chunk, ch = u / per_chunk;
        const bool mine = lane < boxes && at < live;
        int row = total_rows;  // (reads as zeros)
        if (mine) {
          const int64_t key = k0 + at * box, pi = key / a.page;
          const int id = pages[pi];
          if (id >= 0 && id < a.num_pages)
            row = (int)(((int64_t)id * a.Hkv + w.kvh) * a.page + (key - pi * a.page));
        }
        const uint32_t off = st * F::kTileBytes + ch * kChunk + at * box * 128;
        const uint32_t bytes = (uint32_t)live * HDC * box * 128;
        ok = mbar_wait(&sm.k_empty[st], ph ^ 1u, status, 401);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        if (lane == 0) mbar_arrive_expect_tx(&sm.k_full[st], bytes);
        __syncwarp();
        if (mine) tma_load_2d(sK + off, &tmK, &sm.k_full[st], ch * 64, row);
        ok = mbar_wait(&sm.v_empty[st], ph ^ 1u, status, 402);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
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
    if (elect_one()) {
      constexpr uint32_t ID_S = idesc_bf16(kTile, N, false, false);
      constexpr uint32_t ID_O = idesc_bf16(128, N, true, true);
      const uint32_t k_base = smem_u32(sK), v_base = smem_u32(sV);
      const uint32_t p_base = smem_u32(sP), q_base = smem_u32(sQ);
      bool ok = true;
      int i = 0, seq = 0;
      int p_st = -1, p_i = 0, p_par = 0, p_use = 0;
      bool p_first = false, p_last = false;
      auto value_product = [&]() -> bool {
        if (!mbar_wait(&sm.p_full, p_i & 1, status, 403)) return false;
        if (!mbar_wait(&sm.v_full[p_st], (p_i / ST) & 1, status, 404)) return false;
        if (p_first && !mbar_wait(&sm.o_empty[p_par], (p_use & 1) ^ 1u, status, 405)) return false;
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
      while (ok && w.next()) {
        if (w.t1 <= w.t0) continue;
        const int qb = seq % QB;
        ok = mbar_wait(&sm.q_full[qb], (seq / QB) & 1, status, 406);
        for (int t = w.t0; t < w.t1 && ok; ++t, ++i) {
          const int st = i % ST, sb = i & 1;
          if (!mbar_wait(&sm.k_full[st], (i / ST) & 1, status, 407)) { ok = false; break; }
          if (!mbar_wait(&sm.s_empty[sb], ((i >> 1) & 1) ^ 1u, status, 408)) { ok = false; break; }
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
          if (t + 1 == w.t1) mma_commit(&sm.q_empty[qb]);
          if (p_st >= 0 && !value_product()) { ok = false; break; }
          p_st = st;
          p_i = i;
          p_par = seq & 1;
          p_use = seq >> 1;
          p_first = t == w.t0;
          p_last = t + 1 == w.t1;
        }
        ++seq;
      }
      if (ok && p_st >= 0) value_product();
    }
  } else if (warp < 4) {
    // -------------------------------------------------------------- Q rows ----
    const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a.q);
    int seq = 0;
    while (w.next()) {
      if (w.t1 <= w.t0) continue;
      const int qb = seq % QB, rows = w.tile_rows();
      const bool ok = mbar_wait(&sm.q_empty[qb], ((seq / QB) & 1) ^ 1u, status, 409);
      if (!__all_sync(0xffffffffu, ok)) break;
      uint8_t* dst = sQ + qb * F::kQBytes;
      constexpr int U = HD / 8;  // 16-byte units of a row
#pragma unroll 4
      for (int x = threadIdx.x - 64; x < N * U; x += 64) {
        const int r = x / U, u = x % U;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (r < rows) {
          const int pr = w.rt * N + r, tok = pr / a.G;
          v = *reinterpret_cast<const uint4*>(q + (int64_t)(w.rq.row0 + tok) * a.q_ld +
                                              (int64_t)(w.kvh * a.G + pr - tok * a.G) * HD + u * 8);
        }
        *reinterpret_cast<uint4*>(dst + (u >> 3) * (N * 128) + swz128(r, u & 7)) = v;
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.q_full[qb]);
      ++seq;
    }
  } else {
    // ------------------------------------------------------------- softmax ----
    const int quarter = warp & 3, tid = threadIdx.x - 128;  // this thread's key and TMEM lane
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    // A wait that runs out only marks its thread: the group leaves together, at the next
    // barrier that all of its threads reach.
    bool bad = false;
    int i = 0, seq = 0;
    while (w.next()) {
      const int rows = w.tile_rows(), r0 = w.rt * N;
      const int par = seq & 1;
      float l[N];
#pragma unroll
      for (int c = 0; c < N; ++c) l[c] = 0.f;
      float m = -INFINITY;  // the bound of row tid (tid < N)
      const int64_t lim0 = w.limit(r0);
      const int tok0 = r0 / a.G, rem0 = r0 - tok0 * a.G;
      bool left = false;
      for (int t = w.t0; t < w.t1; ++t, ++i) {
        const int st = i % ST, sb = i & 1;
        const int64_t k0 = a.kbeg + (int64_t)t * kTile, key = k0 + tid;
        bad |= !mbar_wait(&sm.s_full[sb], (i >> 1) & 1, status, 410);
        tc_fence_after();
        float x[N];
        tmem_ldn<N>(tS + sb * N + lane_off, x);
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.s_empty[sb]);
        if (k0 + kTile > lim0) {  // some row does not see all of the tile
          int rem = rem0;
          int64_t lim = lim0;
#pragma unroll
          for (int c = 0; c < N; ++c) {
            x[c] = key < lim ? x[c] : -INFINITY;
            if (++rem == a.G) {
              rem = 0;
              lim = min(lim + 1, w.kend);
            }
          }
        }
        // does any score pass its row's bound by more than 2^8?
        bool raise = bad || t == w.t0 || (tid < N && m == -INFINITY);
        if (t > w.t0) {
          float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int c = 0; c < N; c += 8) {
            const float4 n0 = *reinterpret_cast<const float4*>(&sm.mneg[c]);
            const float4 n1 = *reinterpret_cast<const float4*>(&sm.mneg[c + 4]);
            top[0] = max3f(top[0], fmaf(x[c], a.scale_log2, n0.x), fmaf(x[c + 1], a.scale_log2, n0.y));
            top[1] = max3f(top[1], fmaf(x[c + 2], a.scale_log2, n0.z), fmaf(x[c + 3], a.scale_log2, n0.w));
            top[2] = max3f(top[2], fmaf(x[c + 4], a.scale_log2, n1.x), fmaf(x[c + 5], a.scale_log2, n1.y));
            top[3] = max3f(top[3], fmaf(x[c + 6], a.scale_log2, n1.z), fmaf(x[c + 7], a.scale_log2, n1.w));
          }
          raise |= max3f(top[0], top[1], fmaxf(top[2], top[3])) > kRaise;
        }
        if (vote_softmax(raise)) {
#pragma unroll
          for (int c = 0; c < N; ++c) {
            const float wm = redux_max(x[c]);
            if (lane == (c & 31)) sm.mx[quarter][c] = wm;
          }
          if (vote_softmax(bad)) {
            left = true;
            break;
          }
          if (tid < N) {
            const float mt = fmaxf(fmaxf(sm.mx[0][tid], sm.mx[1][tid]),
                                   fmaxf(sm.mx[2][tid], sm.mx[3][tid])) * a.scale_log2;
            float f = 1.f;
            if (mt > m + kRaise || (m == -INFINITY && mt > m)) {
              f = m == -INFINITY ? 0.f : exp2f(m - mt);
              m = mt;
            }
            sm.mneg[tid] = m == -INFINITY ? 0.f : -m;
            sm.fac[tid] = f;
          }
          bar_softmax();
          if (t > w.t0) {
#pragma unroll
            for (int c = 0; c < N; ++c) l[c] *= sm.fac[c];
            // the accumulator of the tiles before this one
            bad |= !mbar_wait(&sm.p_empty, (i - 1) & 1, status, 411);
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < N; c += 16) {
              float ov[16];
              uint32_t ou[16];
              tmem_ld16(tO + par * N + lane_off + c, ov);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) ou[e] = __float_as_uint(ov[e] * sm.fac[c + e]);
              tmem_st16(tO + par * N + lane_off + c, ou);
            }
            tmem_wait_st();
          }
        }
        // probabilities, rounded to bf16 for the tensor core (their sum is not)
        if (i > 0) bad |= !mbar_wait(&sm.p_empty, (i - 1) & 1, status, 412);
#pragma unroll
        for (int u = 0; u < N / 8; ++u) {
          uint32_t pk[4];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int c = 8 * u + 4 * e;
            const float4 n0 = *reinterpret_cast<const float4*>(&sm.mneg[c]);
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
          *reinterpret_cast<uint4*>(sP + swz128(tid, u)) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
        }
        if (k0 + kTile > w.kend) {
          // what lies behind the last key (another request's rows, or anything at all)
          // must not meet its zero probabilities: 0 x NaN
          bad |= !mbar_wait(&sm.v_full[st], (i / ST) & 1, status, 413);
          if (key >= w.kend) {
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
      const bool any = w.t1 > w.t0, whole = w.whole();
      lane_sums<N>(l, lane);
      if constexpr (N == 64) {
        sm.mx[quarter][2 * lane] = l[0];
        sm.mx[quarter][2 * lane + 1] = l[1];
      } else if constexpr (N == 32) {
        sm.mx[quarter][lane] = l[0];
      } else {
        if (!(lane & 1)) sm.mx[quarter][lane >> 1] = l[0];
      }
      if (vote_softmax(bad)) break;
      if (tid < rows) {
        const float sum = (sm.mx[0][tid] + sm.mx[1][tid]) + (sm.mx[2][tid] + sm.mx[3][tid]);
        if (whole) {
          const int pr = r0 + tid, tok = pr / a.G;
          const int row = w.rq.row0 + tok, head = w.kvh * a.G + pr - tok * a.G;
          const RowScale f = finish_row(a, row, head, m, sum);
          sm.mneg[tid] = f.own;
          sm.mx[0][tid] = f.pre;
          a.lse[(int64_t)head * a.T + row] = f.lse;
        } else {
          const int64_t row = (int64_t)w.slot() * N + tid;
          a.part_ml[2 * row] = m;
          a.part_ml[2 * row + 1] = sum;
        }
      }
      if (!whole && w.first && tid == 0) w.record_open();
      bar_softmax();
      float ov[N];
      if (any) {
        bad |= !mbar_wait(&sm.o_full[par], (seq >> 1) & 1, status, 414);
        tc_fence_after();
        tmem_ldn<N>(tO + par * N + lane_off, ov);
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.o_empty[par]);
        ++seq;
      }
      if (tid < HD) {
        if (whole) {
          int tok = tok0, rem = rem0;
#pragma unroll
          for (int c = 0; c < N; ++c) {
            if (c < rows) {
              const int row = w.rq.row0 + tok, head = w.kvh * a.G + rem;
              const int64_t at = ((int64_t)row * a.Hq + head) * HD + tid;
              const float own = sm.mneg[c], pre = sm.mx[0][c];
              float v = !any || own == 0.f ? 0.f : ov[c] * own;
              if (pre != 0.f) v += pre * a.pre_o[at];
              if (a.o32)
                a.o32[at] = v;
              else
                static_cast<__nv_bfloat16*>(a.o)[(int64_t)row * a.o_ld + head * HD + tid] =
                    __float2bfloat16_rn(v);
            }
            if (++rem == a.G) {
              rem = 0;
              ++tok;
            }
          }
        } else if (any) {
          float* dst = a.part_o + (int64_t)w.slot() * N * HD + tid;
#pragma unroll
          for (int c = 0; c < N; ++c)
            if (c < rows) dst[c * HD] = ov[c];
        }
      }
      bar_softmax();  // mneg / mx are the next segment's from here
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(sm.tmem, F::kTmem);
  }
}

template <int N, int HDC>
int launch(const Args& a, int blocks, cudaStream_t st) {
  int box = kTile;
  while (a.page % box) box >>= 1;  // (pages are multiples of 16)
  CUtensorMap tk, tv;
  const uint64_t rows = (uint64_t)a.num_pages * a.Hkv * a.page;
  int rc = make_tmap_2d(&tk, a.kc, 64 * HDC, rows, 128 * HDC, 64, (uint32_t)box);
  if (!rc) rc = make_tmap_2d(&tv, a.vc, 64 * HDC, rows, 128 * HDC, 64, (uint32_t)box);
  if (rc) return rc;
  auto kern = paged_few_kernel<N, HDC>;
  constexpr int smem = (int)Few<N, HDC>::kSmem;
  PE_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  kern<<<blocks, kThreads, smem, st>>>(tk, tv, a, box);
  PE_LAUNCHED();
  return PE_OK;
}

}  // namespace

int launch_few(const Args& a, int rows, int blocks, cudaStream_t st) {
  const bool wide = a.hd == 128;
  switch (rows) {
    case 16: return wide ? launch<16, 2>(a, blocks, st) : launch<16, 1>(a, blocks, st);
    case 32: return wide ? launch<32, 2>(a, blocks, st) : launch<32, 1>(a, blocks, st);
    default: return wide ? launch<64, 2>(a, blocks, st) : launch<64, 1>(a, blocks, st);
  }
}

}  // namespace paged
}  // namespace pe
