// Attention over the paged key/value cache: entry points, kernel choice, the join of split
// entities, and the CUDA-core kernel that serves every type, head size and page size.
//
// Row (t, head) of request b sees keys [0, lens[b] - n_b + j + 1), j its index among the
// request's n_b new rows: real rows are causal, and a draft's prediction slots, which follow
// the last real row, see the context and the slots before them -- the rule of the reference's
// masks (src/pe/masks.py:43-61) for one anchor.  softmax(q k / sqrt(hd)) v, statistics fp32.
#include <algorithm>

#include "paged.cuh"

namespace pe {
namespace paged {
namespace {

// ------------------------------------------------------------- CUDA-core kernel ----
// A block holds 16 packed rows (fp32) and walks its key tiles, 32 keys at a time, through
// two shared-memory buffers: the next tile's copies run while this one is computed.  8
// threads share a row's scores, statistics and output columns.  It serves fp32 (whose
// products the tensor cores would round) and what the tensor-core kernels do not take.
// Bound by shared-memory reads: a key's element is read once per 4 rows of a warp for the
// scores and once for the output.  Measured: 16 requests of 1..5 rows, 17K keys in all, 4/2
// heads of 64, fp32: 26.4 us with the join, of which half is a block's start, its one or two
// results and the join.
constexpr int kThreads = 128;
constexpr int kSimtRows = 16;
constexpr int kTK = 32;
constexpr int kLdP = kTK + 8;  // a warp's four rows of probabilities in different banks

__device__ __forceinline__ float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 load4(const __nv_bfloat16* p) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  const float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.x));
  const float2 y = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.y));
  return make_float4(x.x, x.y, y.x, y.y);
}
__device__ __forceinline__ void copy16(void* dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                   (uint32_t)__cvta_generic_to_shared(dst)),
               "l"(src), "r"(valid ? 16 : 0)
               : "memory");
}

// shared-memory row of a K or V tile, in elements: padded so that 8 keys' 16-byte (fp32)
// or 8-byte (bf16) pieces fall into different banks
__host__ __device__ constexpr int simt_ld(int hdp, int es) { return hdp + 16 / es; }
inline size_t simt_smem(int hdp, int es) {
  return 4ull * kTK * simt_ld(hdp, es) * es + (size_t)kSimtRows * (hdp + 4 + kLdP) * sizeof(float);
}

// Blocks that an SM's registers hold: 128 a thread for fp32, 160 for bf16 (whose conversions
// want more).  The grid is one wave of them, as all pieces are equal.  With a fourth bf16 block
// an SM, which waits for a place, 64 tokens over up to 4K keys took 237 us, 132 with three
// (12/3 heads of 80), and 804 against 450 (16/16 heads of 40).
template <typename T>
constexpr int kSimtBlocks = sizeof(T) == 4 ? 4 : 3;

template <typename T>
__global__ void __launch_bounds__(kThreads, kSimtBlocks<T>)
paged_simt_kernel(const __grid_constant__ Args a, int hdp, int vec) {
  constexpr int Mt = kSimtRows;
  extern __shared__ __align__(16) uint8_t smem[];
  const int ldk = simt_ld(hdp, sizeof(T)), ldq = hdp + 4;
  T* sKV = reinterpret_cast<T*>(smem);  // [buffer][K, V][kTK][ldk]
  float* sQ = reinterpret_cast<float*>(sKV + 4 * kTK * ldk);  // [Mt][ldq]
  float* sP = sQ + Mt * ldq;                                  // [Mt][kLdP]
  __shared__ int64_t scratch[kThreads / 32 + 4];
  const int tid = threadIdx.x, r = tid >> 3, c = tid & 7;
  const T* q = static_cast<const T*>(a.q);
  const T* kc = static_cast<const T*>(a.kc);
  const T* vc = static_cast<const T*>(a.vc);
  const int groups = hdp >> 2;  // float4 columns of the output
  bool joined = false;

  start_next_kernel();
  Sched<Mt, kTK, kTK, 3 * kTK> w(a);
  w.init(scratch);
  if (tid == 0) a.open[blockIdx.x].parts = 0;
  while (w.next()) {
    const int rows = w.tile_rows();
    const int rr = w.rt * Mt + r;  // this thread's packed row
    const bool valid = r < rows;
    const bool active = (tid >> 5) * 4 < rows;  // some of this warp's four rows
    const int64_t lim = valid ? w.limit(rr) : 0;
    // start the copies of tile t (zeros behind the last key and outside the pool)
    auto fetch = [&](int t) {
      const int key = tid >> 2, part = tid & 3;
      const int64_t at = a.kbeg + (int64_t)t * kTK + key;
      const T *kr = kc, *vr = vc;
      bool live = false;
      if (at < w.kend) {
        const int64_t pi = div_pos(at, a.page);
        const int id = w.pages()[pi];
        if (id >= 0 && id < a.num_pages) {
          const int64_t off = (((int64_t)id * a.Hkv + w.kvh) * a.page + (at - pi * a.page)) * a.hd;
          kr = kc + off;
          vr = vc + off;
          live = true;
        }
      }
      T* dk = sKV + (t & 1) * 2 * kTK * ldk + key * ldk;
      T* dv = dk + kTK * ldk;
      if (vec) {
        constexpr int N = 16 / sizeof(T);
        for (int u = part * N; u < hdp; u += 4 * N) {
          copy16(dk + u, kr + u, live);
          copy16(dv + u, vr + u, live);
        }
      } else {
        for (int d = part; d < hdp; d += 4) {
          dk[d] = live && d < a.hd ? kr[d] : from_f<T>(0.f);
          dv[d] = live && d < a.hd ? vr[d] : from_f<T>(0.f);
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    __syncthreads();  // the segment before is read
    if (w.t0 < w.t1) fetch(w.t0);
    {
      const int tok = rr / a.G;
      const T* qr = q + (int64_t)(w.rq.row0 + tok) * a.q_ld +
                    (int64_t)(w.kvh * a.G + rr - tok * a.G) * a.hd;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int d = 4 * (c + 8 * i);
        if (d >= hdp) break;
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = valid && d + e < a.hd ? to_f(qr[d + e]) : 0.f;
        *reinterpret_cast<float4*>(sQ + r * ldq + d) = make_float4(x[0], x[1], x[2], x[3]);
      }
    }
    float4 acc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    float m = -INFINITY, l = 0.f;
    for (int t = w.t0; t < w.t1; ++t) {
      const int64_t k0 = a.kbeg + (int64_t)t * kTK;
      asm volatile("cp.async.wait_all;" ::: "memory");
      __syncthreads();  // tile t is here, tile t - 1 is read
      if (t + 1 < w.t1) fetch(t + 1);
      if (!active) continue;
      const T* sK = sKV + (t & 1) * 2 * kTK * ldk;
      const T* sV = sK + kTK * ldk;
      float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
      for (int d = 0; d < hdp; d += 4) {
        const float4 qv = load4(sQ + r * ldq + d);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float4 kv = load4(sK + (c + 8 * i) * ldk + d);
          s[i] = fmaf(qv.x, kv.x, fmaf(qv.y, kv.y, fmaf(qv.z, kv.z, fmaf(qv.w, kv.w, s[i]))));
        }
      }
      float mt = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[i] = k0 + c + 8 * i < lim ? s[i] * a.scale_log2 : -INFINITY;
        mt = fmaxf(mt, s[i]);
      }
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, o));
      const float m_new = fmaxf(m, mt);
      const float m_use = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = m == m_new ? 1.f : exp2f(m - m_use);
      float rs = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p = exp2f(s[i] - m_use);
        rs += p;
        sP[r * kLdP + c + 8 * i] = p;
      }
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) rs += __shfl_xor_sync(0xffffffffu, rs, o);
      l = l * alpha + rs;
      m = m_new;
      __syncwarp();  // a row's 8 threads are in one warp
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (c + 8 * i >= groups) break;
        float4 o = acc[i];
        o.x *= alpha; o.y *= alpha; o.z *= alpha; o.w *= alpha;
        const T* vcol = sV + 4 * (c + 8 * i);
#pragma unroll 2
        for (int kk = 0; kk < kTK; kk += 4) {
          const float4 p = load4(sP + r * kLdP + kk);
          const float4 v0 = load4(vcol + kk * ldk), v1 = load4(vcol + (kk + 1) * ldk);
          const float4 v2 = load4(vcol + (kk + 2) * ldk), v3 = load4(vcol + (kk + 3) * ldk);
          o.x = fmaf(p.w, v3.x, fmaf(p.z, v2.x, fmaf(p.y, v1.x, fmaf(p.x, v0.x, o.x))));
          o.y = fmaf(p.w, v3.y, fmaf(p.z, v2.y, fmaf(p.y, v1.y, fmaf(p.x, v0.y, o.y))));
          o.z = fmaf(p.w, v3.z, fmaf(p.z, v2.z, fmaf(p.y, v1.z, fmaf(p.x, v0.z, o.z))));
          o.w = fmaf(p.w, v3.w, fmaf(p.z, v2.w, fmaf(p.y, v1.w, fmaf(p.x, v0.w, o.w))));
        }
        acc[i] = o;
      }
      __syncwarp();
    }
    if (a.pre_lse && !joined) {
      wait_kernel_before();  // the prefix's rows
      joined = true;
    }
    if (w.whole()) {
      if (valid) {
        const int tok = w.rq.row0 + rr / a.G, head = w.kvh * a.G + rr % a.G;
        const RowScale f = finish_row(a, tok, head, m, l);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (c + 8 * i >= groups) break;
          const float v[4] = {acc[i].x, acc[i].y, acc[i].z, acc[i].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int d = 4 * (c + 8 * i) + e;
            if (d >= a.hd) continue;
            const int64_t at = ((int64_t)tok * a.Hq + head) * a.hd + d;
            float x = f.own == 0.f ? 0.f : v[e] * f.own;
            if (f.pre != 0.f) x += f.pre * a.pre_o[at];
            if (a.o32)
              a.o32[at] = x;
            else
              static_cast<T*>(a.o)[(int64_t)tok * a.o_ld + (int64_t)head * a.hd + d] = from_f<T>(x);
          }
        }
        if (c == 0) a.lse[(int64_t)head * a.T + tok] = f.lse;
      }
    } else {
      if (w.first && tid == 0) w.record_open();
      if (valid) {
        const int64_t row = (int64_t)w.slot() * Mt + r;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (c + 8 * i >= groups) break;
          const float v[4] = {acc[i].x, acc[i].y, acc[i].z, acc[i].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int d = 4 * (c + 8 * i) + e;
            if (d < a.hd) a.part_o[row * a.hd + d] = v[e];
          }
        }
        if (c == 0) {
          a.part_ml[2 * row] = m;
          a.part_ml[2 * row + 1] = l;
        }
      }
    }
  }
  wait_kernel_before();  // (also where nothing was joined: the kernels end in order)
}

// ---------------------------------------------------------------------- join ----
// Block (c, y): joins the pieces of the entity that starts in block c, rows 4y .. 4y + 3, a
// warp a row.  Pieces are weighted with 2^(m_i - max m) and added in piece order, eight
// loads in flight.  Bound by latency: most blocks have nothing to join, the others read
// three things one after another (what to join, its statistics, its accumulators).  (Blocks
// of 1024 threads, or four warps a row, took 1.3 to 1.5 times as long.)
constexpr int kJoinRows = 4;

template <typename T, int V>
__global__ void __launch_bounds__(32 * kJoinRows)
paged_join_kernel(const __grid_constant__ Args a, int Mt) {
  start_next_kernel();
  wait_kernel_before();
  const Open op = a.open[blockIdx.x];
  const int lane = threadIdx.x & 31, row = blockIdx.y * kJoinRows + (threadIdx.x >> 5);
  if (op.parts == 0 || row >= op.rows) return;
  constexpr int E = 256 / 32;  // elements per lane, in runs of V
  auto slot_row = [&](int i) {
    const int s = i == 0 ? op.slot : 2 * ((int)blockIdx.x + i);
    return (int64_t)s * Mt + row;
  };
  auto stat = [&](int i) { return *reinterpret_cast<const float2*>(a.part_ml + 2 * slot_row(i)); };
  auto column = [&](int e) { return (e / V) * (32 * V) + lane * V + e % V; };
  float mx = -INFINITY, l = 0.f;
  for (int i = lane; i < op.parts; i += 32) {
    const float2 ml = stat(i);
    if (ml.y != 0.f) mx = fmaxf(mx, ml.x);
  }
  mx = warp_max(mx);
  for (int i = lane; i < op.parts; i += 32) {
    const float2 ml = stat(i);
    l += ml.y == 0.f ? 0.f : exp2f(ml.x - mx) * ml.y;
  }
  l = warp_sum(l);
  float acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma unroll 8
  for (int i = 0; i < op.parts; ++i) {
    const float2 ml = stat(i);
    const float w = ml.y == 0.f ? 0.f : exp2f(ml.x - mx);
    const float* src = a.part_o + slot_row(i) * a.hd;
#pragma unroll
    for (int e = 0; e < E; e += V) {
      if (column(e) >= a.hd) continue;
      float v[V];
      if constexpr (V == 4) {
        const float4 x = *reinterpret_cast<const float4*>(src + column(e));
        v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
      } else {
        v[0] = src[column(e)];
      }
      // (a piece without keys left its accumulator unwritten)
#pragma unroll
      for (int q = 0; q < V; ++q) acc[e + q] += w == 0.f ? 0.f : w * v[q];
    }
  }
  const int rr = op.r0 + row;
  const int tok = op.row0 + rr / a.G, head = op.kvh * a.G + rr % a.G;
  const RowScale f = finish_row(a, tok, head, mx, l);
  const int64_t at = ((int64_t)tok * a.Hq + head) * a.hd;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int d = column(e);
    if (d >= a.hd) continue;
    float x = f.own == 0.f ? 0.f : acc[e] * f.own;
    if (f.pre != 0.f) x += f.pre * a.pre_o[at + d];
    if (a.o32)
      a.o32[at + d] = x;
    else
      static_cast<T*>(a.o)[(int64_t)tok * a.o_ld + (int64_t)head * a.hd + d] = from_f<T>(x);
  }
  if (lane == 0) a.lse[(int64_t)head * a.T + tok] = f.lse;
}

int launch_join(int dtype, const Args& a, int blocks, int Mt, cudaStream_t st) {
  const dim3 grid((unsigned)blocks, (unsigned)ceil_div(Mt, kJoinRows));
  return PE_DISPATCH(dtype, T, [&]() -> int {
    auto kern = a.hd % 4 == 0 ? paged_join_kernel<T, 4> : paged_join_kernel<T, 1>;
    return launch_kernel(kern, grid, 32 * kJoinRows, 0, st, true, a, Mt);
  });
}

int launch_simt(int dtype, const Args& a, int blocks, bool dependent, cudaStream_t st) {
  const int es = dtype == PE_F32 ? 4 : 2;
  const int hdp = (a.hd + 3) / 4 * 4;
  const size_t smem = simt_smem(hdp, es);
  const int vec = a.hd * es % 16 == 0 && (reinterpret_cast<uintptr_t>(a.kc) & 15u) == 0 &&
                  (reinterpret_cast<uintptr_t>(a.vc) & 15u) == 0;
  return PE_DISPATCH(dtype, T, [&]() -> int {
    auto kern = paged_simt_kernel<T>;
    const int rc = allow_smem<paged_simt_kernel<T>>((int)simt_smem(256, sizeof(T)));
    if (rc) return rc;
    return launch_kernel(kern, dim3((unsigned)blocks), kThreads, smem, st, dependent, a, hdp, vec);
  });
}

// ------------------------------------------------------------------ kernel choice ----
enum Kind { kSimt, kFew, kMany };

struct Phase {
  Kind kind;
  int Mt, blocks;
};

Phase simt_phase(int dtype, int hd) {
  // as many blocks as the tiles' shared memory and the registers let an SM hold
  const size_t smem = simt_smem((hd + 3) / 4 * 4, dtype == PE_F32 ? 4 : 2);
  const size_t most = dtype == PE_F32 ? kSimtBlocks<float> : kSimtBlocks<__nv_bfloat16>;
  return {kSimt, kSimtRows,
          sm_count() * (int)std::max<size_t>(1, std::min<size_t>(most, 220 * 1024 / smem))};
}

// Tensor-core kernel for `rows` packed rows (on average) per request and KV head: up to one tile
// of the few-row kernel's largest kind; two of them read every key twice.  Device time of (few,
// many) in us, bf16, requests of the same length:
//   28/4 heads of 128,  8 x 8K:   42 rows 41, 48     63: 43, 49     77: 54, 48    126: 56, 51
//                      64 x 4K:          100, 122       102, 122       174, 121       181, 129
//                      64 x 600:          35, 51         37, 52         57, 51         58, 55
//   40/8 heads of 128,  8 x 8K:   45 rows 59, 71     60: 60, 72     80: 86, 71    125: 89, 74
//   6/6 heads of 64,   64 x 4K:   48 rows 124, 170   64: 127, 160   80: 223, 164
// A single request, whose keys fill no SM for long, would be quicker with the few-row kernel up
// to some hundred rows (1 x 1K, 126 rows: 20, 24), and a mean over requests of very different
// rows fits none of them (requests without rows count in it, too); both are left so.
Phase tc_phase(int64_t rows) {
  if (rows > 64) return {kMany, 256, sm_count()};
  return {kFew, rows <= 16 ? 16 : rows <= 32 ? 32 : 64, sm_count()};
}

bool tc_sizes(int dtype, int hd) { return dtype == PE_BF16 && (hd == 64 || hd == 128); }

// whether the tensor-core kernels take the call's operands
bool tc_operands(const Args& a) {
  auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  return al(a.q) && a.q_ld % 8 == 0 && al(a.kc) && al(a.vc) &&
         a.num_pages * a.Hkv * a.page < (1ll << 31) - 256;
}

// Whether the requests read their common prefix each for itself.  Its pages then come from
// L2 after the first time, and a prefix of its own costs two launches, an fp32 result and a
// second start of the copies.  Device time of (each for itself, once) in us,
// by B * prefix keys * KV heads:
//   bf16, 28/4 heads of 128, 1 row:   131K 22, 30   524K 36, 41   1.05M 57, 48   2.1M 102, 59
//         5 rows:                     131K 28, 43   524K 52, 59   1.05M 85, 66   2.1M 157, 89
//   bf16, 14/2 heads of 64, 5 rows:   131K 27, 41   524K 50, 52   1.05M 83, 58
//   fp32, 4/2 heads of 64, 1 row:      66K 27, 35   131K 37, 44    262K 54, 51    524K 93, 60
//   bf16, 12/3 heads of 80, 1 row:     49K 34, 48   197K 57, 62    393K 96, 72
// With more rows a request than the few-row kernel takes, the prefix's rows of all requests
// fill its tiles better than each request's.
bool prefix_per_request(bool tc, int64_t B, int64_t rows, int64_t keys) {
  if (tc && ceil_div(rows, B) > 64) return false;
  return B * keys <= (tc ? 700000 : 160000);
}

// Whether no entity is cut: requests that cannot be long (the block table's width says so)
// are worth neither partial results nor the join's launch.  Device time of (uncut, cut) in us,
// bf16, requests of up to as many keys, by heads of all requests (B * Hkv):
//   1 row,  28/4 heads of 128:  4  512 keys 11, 13   640 12, 13    768 13, 14   1024 14, 15
//                              64  512 keys 12, 16   640 13, 17    768 14, 17   1024 16, 18
//                             256  512 keys 22, 26   640 24, 28    768 26, 31   1024 32, 35
//   5 rows, 28/4 heads of 128:  4  512 keys 16, 16   640 17, 16    768 18, 16   1024 20, 18
//   (35 packed: 64-row tiles)  16  512 keys 16, 18   640 17, 18    768 18, 19   1024 21, 20
//                              64  512 keys 17, 20   640 18, 21    768 19, 21   1024 22, 23
//   5 rows, 14/2 heads of 64:   2  512 keys 15, 15   640 16, 15    768 17, 15   1024 19, 17
//   (the same)                  8  512 keys 15, 16   640 17, 17    768 18, 17   1024 20, 18
//                              32  512 keys 16, 17   640 17, 19    768 18, 19   1024 20, 19
//   5 rows, 40/8 heads of 128:  8  512 keys 13, 15   640 14, 16    768 15, 16   1024 17, 17
//   (25 packed: 32-row tiles) 128  512 keys 15, 22   640 17, 23    768 18, 24   1024 21, 26
// A 64-row tile takes longer per key, so few heads are cut earlier.  (2048 keys: 21, 19 for 64
// heads of one row; 59, 57 for 256 heads of five.)
bool uncut(const Phase& p, int64_t keys, int64_t heads) {
  if (p.kind != kFew) return false;
  if (heads >= 64) return keys <= 1024;
  return keys <= (p.Mt == 64 && heads < 16 ? 512 : 640);
}

int64_t al256(int64_t x) { return (x + 255) / 256 * 256; }

// bytes of one phase's partial results
int64_t phase_bytes(const Phase& p, int hd) {
  return al256(2ll * p.blocks * p.Mt * hd * 4) + al256(2ll * p.blocks * p.Mt * 2 * 4) +
         al256((int64_t)p.blocks * sizeof(Open));
}

void carve(Args& a, const Phase& p, uint8_t* ws) {
  a.part_o = reinterpret_cast<float*>(ws);
  ws += al256(2ll * p.blocks * p.Mt * a.hd * 4);
  a.part_ml = reinterpret_cast<float*>(ws);
  ws += al256(2ll * p.blocks * p.Mt * 2 * 4);
  a.open = reinterpret_cast<Open*>(ws);
}

int run_phase(int dtype, const Phase& p, const Args& a, bool dependent, cudaStream_t st) {
  const int rc = p.kind == kFew    ? launch_few(a, p.Mt, p.blocks, dependent, st)
                 : p.kind == kMany ? launch_many(a, p.blocks, dependent, st)
                                   : launch_simt(dtype, a, p.blocks, dependent, st);
  if (rc || a.whole) return rc;
  return launch_join(dtype, a, p.blocks, p.Mt, st);
}

}  // namespace
}  // namespace paged
}  // namespace pe

using namespace pe;
using namespace pe::paged;

extern "C" size_t pe_attn_paged_workspace(int dtype, int64_t B, int64_t T, int Hq, int Hkv, int hd,
                                          int64_t shared) {
  if (B < 1 || T < 1 || Hq < 1 || Hkv < 1 || hd < 1) return 0;
  const int64_t G = std::max(Hq / Hkv, 1);
  int64_t bytes = phase_bytes(simt_phase(dtype, hd), hd);  // (operands may rule the tensor cores out)
  if (tc_sizes(dtype, hd)) bytes = std::max(bytes, phase_bytes(tc_phase(ceil_div(T * G, B)), hd));
  if (shared <= 0) return (size_t)bytes;
  int64_t prefix = phase_bytes(simt_phase(dtype, hd), hd);
  if (tc_sizes(dtype, hd)) prefix = std::max(prefix, phase_bytes(tc_phase(T * G), hd));
  return (size_t)(al256(T * Hq * hd * 4) + al256(T * Hq * 4) + prefix + bytes);
}

extern "C" int pe_attn_paged(int dtype, int64_t B, int64_t T, int Hq, int Hkv, int hd,
                             const void* q, int64_t q_ld, const void* k_cache, const void* v_cache,
                             int64_t num_pages, int64_t page, const int32_t* table,
                             int64_t table_ld, int64_t width, const int32_t* lens,
                             const int32_t* cu, int64_t shared, void* o, int64_t o_ld, float* lse,
                             void* workspace, size_t workspace_bytes, int algo, int* status,
                             void* stream) {
  PE_CHECK_ARG(dtype == PE_F32 || dtype == PE_BF16, "attn_paged: unsupported dtype code %d", dtype);
  const bool once = algo & PE_PAGED_PREFIX_ONCE;
  algo &= ~PE_PAGED_PREFIX_ONCE;
  PE_CHECK_ARG(algo == PE_ALGO_AUTO || algo == PE_ALGO_SIMT || algo == PE_ALGO_TCGEN05,
               "attn_paged: unknown algorithm %d", algo);
  PE_CHECK_ARG(Hq >= 1 && Hkv >= 1 && Hq % Hkv == 0 && Hq / Hkv <= 256,
               "attn_paged: %d query heads over %d KV heads", Hq, Hkv);
  PE_CHECK_ARG(hd >= 1 && hd <= 256, "attn_paged: head_dim %d, expected 1 to 256", hd);
  PE_CHECK_ARG(B >= 1 && B < (1 << 20) && T >= 0 && T < (1ll << 31) && T * Hq < (1ll << 31),
               "attn_paged: %lld requests, %lld rows of %d heads", (long long)B, (long long)T, Hq);
  PE_CHECK_ARG(page >= 16 && page % 16 == 0 && page <= (1 << 20),
               "attn_paged: page size %lld is not a multiple of 16", (long long)page);
  PE_CHECK_ARG(num_pages >= 1 && num_pages < (1ll << 31) &&
                   num_pages * page < ceil_div(1ll << 40, Hkv),
               "attn_paged: %lld pages", (long long)num_pages);
  PE_CHECK_ARG(width >= 1 && width <= (1 << 27) / page && table_ld >= width,
               "attn_paged: block table of %lld pages (row stride %lld)", (long long)width,
               (long long)table_ld);
  PE_CHECK_ARG(shared >= 0 && shared % page == 0 && shared / page <= width,
               "attn_paged: %lld shared keys are not whole pages of the table", (long long)shared);
  if (T == 0) return PE_OK;
  PE_CHECK_ARG(q && k_cache && v_cache && table && lens && cu && o && lse,
               "attn_paged: null pointer");
  PE_CHECK_ARG(T == 1 || (q_ld >= (int64_t)Hq * hd && o_ld >= (int64_t)Hq * hd),
               "attn_paged: row strides %lld, %lld below %d x %d", (long long)q_ld,
               (long long)o_ld, Hq, hd);
  const size_t need = pe_attn_paged_workspace(dtype, B, T, Hq, Hkv, hd, shared);
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255u)) {
    set_error("attn_paged: workspace of %zu bytes (256-byte aligned) needed, got %zu", need,
              workspace_bytes);
    return PE_ERR_WORKSPACE;
  }
  const cudaStream_t st = as_stream(stream);
  Args a{};
  a.q = q; a.q_ld = q_ld; a.kc = k_cache; a.vc = v_cache;
  a.num_pages = num_pages; a.page = (int)page;
  a.table = table; a.table_ld = table_ld; a.kmax = width * page;
  a.lens = lens; a.cu = cu;
  a.B = (int)B; a.T = (int)T; a.Hq = Hq; a.Hkv = Hkv; a.hd = hd; a.G = Hq / Hkv;
  a.scale_log2 = 1.4426950408889634f / sqrtf((float)hd);
  a.o = o; a.o_ld = o_ld; a.lse = lse; a.status = status;
  const bool tc = algo != PE_ALGO_SIMT && tc_sizes(dtype, hd) && tc_operands(a);
  if (algo == PE_ALGO_TCGEN05 && !tc) {
    set_error("attn_paged: the tensor-core kernels take bf16, head_dim 64 or 128, 16-byte aligned "
              "rows and pools below 2^31 keys x heads");
    return PE_ERR_UNSUPPORTED;
  }
  if (shared > 0 && !once && prefix_per_request(tc, B, T * a.G, shared * Hkv)) shared = 0;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  if (shared > 0) {
    // the prefix once, all rows of all requests together, into fp32 rows
    float* pre_o = reinterpret_cast<float*>(ws);
    ws += al256(T * Hq * hd * 4);
    float* pre_lse = reinterpret_cast<float*>(ws);
    ws += al256(T * Hq * 4);
    const Phase p = tc ? tc_phase(T * a.G) : simt_phase(dtype, hd);
    Args pa = a;
    pa.all_rows = 1;
    // Alike for a prefix that L2 (126 MB, in two halves) does not keep for all row tiles.  A
    // call among others, sustained under the power cap, in us (equal pieces, aligned), samples
    // of 5 rows:   64, 40/8 heads of 128:   64 MB 192, 199   128 MB 315, 320   256 MB 592, 577
    //                                      512 MB 1129, 1079
    //              64, 28/4 heads of 128:   64 MB 213, 212   128 MB 428, 365   256 MB 790, 686
    //              32, the same:            64 MB 130, 126   128 MB 228, 213   256 MB 419, 384
    // What it saves is the power that HBM takes: a few calls alone gain 5 % at most (28/4 heads)
    // and lose 1 to 9 % (40/8).  (The CUDA-core kernel is bound by other things.)
    pa.align = p.kind != kSimt && 4 * shared * Hkv * hd > (64ll << 20);
    pa.kmax = shared;
    pa.o32 = pre_o;
    pa.lse = pre_lse;
    carve(pa, p, ws);
    ws += phase_bytes(p, hd);
    const int rc = run_phase(dtype, p, pa, false, st);
    if (rc) return rc;
    a.kbeg = shared;
    a.pre_o = pre_o;
    a.pre_lse = pre_lse;
  }
  const Phase p = tc ? tc_phase(ceil_div(T * a.G, B)) : simt_phase(dtype, hd);
  a.whole = uncut(p, a.kmax - a.kbeg, B * Hkv);
  carve(a, p, ws);
  // The requests' own keys start while the prefix ends, unless it takes long (here: some 10
  // ms): nothing is gained then, and a block's bounded waits would run while it waits.
  const bool brief = 4.0 * (double)T * Hq * hd * (double)shared < 1e13;
  return run_phase(dtype, p, a, shared > 0 && brief, st);
}
