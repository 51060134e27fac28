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
// shared memory; 8 threads share a row's scores, statistics and output columns.  It serves
// fp32 (whose products the tensor cores would round) and what the tensor-core kernels do
// not take.  Bound by shared-memory reads: a key's element is read once per 4 rows of a
// warp for the scores and once for the output.
constexpr int kThreads = 128;
constexpr int kSimtRows = 16;
constexpr int kTK = 32;

template <typename T>
__global__ void __launch_bounds__(kThreads)
paged_simt_kernel(const __grid_constant__ Args a, int hdp, int vec) {
  constexpr int Mt = kSimtRows;
  extern __shared__ float sm[];
  const int ldk = hdp + 4;
  float* sQ = sm;                 // [Mt][ldk]
  float* sK = sQ + Mt * ldk;      // [kTK][ldk]
  float* sV = sK + kTK * ldk;     // [kTK][ldk]
  float* sP = sV + kTK * ldk;     // [Mt][kTK]
  __shared__ int64_t scratch[kThreads / 32 + 4];
  const int tid = threadIdx.x, r = tid >> 3, c = tid & 7;
  const T* q = static_cast<const T*>(a.q);
  const T* kc = static_cast<const T*>(a.kc);
  const T* vc = static_cast<const T*>(a.vc);
  const int groups = hdp >> 2;  // float4 columns of the output
  bool joined = false;

  start_next_kernel();
  Sched<Mt, kTK> w(a);
  w.init(scratch);
  if (tid == 0) a.open[blockIdx.x].parts = 0;
  while (w.next()) {
    const int rows = w.tile_rows();
    const int rr = w.rt * Mt + r;  // this thread's packed row
    const bool valid = r < rows;
    const int64_t lim = valid ? w.limit(rr) : 0;
    __syncthreads();  // the tile before is read
    for (int i = tid; i < Mt * hdp; i += kThreads) {
      const int ri = i / hdp, d = i - ri * hdp;
      float x = 0.f;
      if (ri < rows && d < a.hd) {
        const int pr = w.rt * Mt + ri;
        x = to_f(q[(int64_t)(w.rq.row0 + pr / a.G) * a.q_ld +
                   (int64_t)(w.kvh * a.G + pr % a.G) * a.hd + d]);
      }
      sQ[ri * ldk + d] = x;
    }
    float4 acc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    float m = -INFINITY, l = 0.f;
    for (int t = w.t0; t < w.t1; ++t) {
      const int64_t k0 = a.kbeg + (int64_t)t * kTK;
      // keys of the tile -> shared memory (zeros behind the last one)
      {
        const int key = tid >> 2, part = tid & 3;
        const int64_t at = k0 + key;
        const T *kr = nullptr, *vr = nullptr;
        if (at < w.kend) {
          const int64_t pi = at / a.page;
          const int id = w.pages()[pi];
          if (id >= 0 && id < a.num_pages) {
            const int64_t off = (((int64_t)id * a.Hkv + w.kvh) * a.page + (at - pi * a.page)) * a.hd;
            kr = kc + off;
            vr = vc + off;
          }
        }
        float* dk = sK + key * ldk;
        float* dv = sV + key * ldk;
        if (vec) {
          constexpr int N = 16 / sizeof(T);
          for (int u = part; u < hdp / N; u += 4) {
            uint4 ku = make_uint4(0, 0, 0, 0), vu = ku;
            if (kr) {
              ku = reinterpret_cast<const uint4*>(kr)[u];
              vu = reinterpret_cast<const uint4*>(vr)[u];
            }
            const T* kt = reinterpret_cast<const T*>(&ku);
            const T* vt = reinterpret_cast<const T*>(&vu);
#pragma unroll
            for (int e = 0; e < N; ++e) {
              dk[u * N + e] = to_f(kt[e]);
              dv[u * N + e] = to_f(vt[e]);
            }
          }
        } else {
          for (int d = part; d < hdp; d += 4) {
            const bool in = kr && d < a.hd;
            dk[d] = in ? to_f(kr[d]) : 0.f;
            dv[d] = in ? to_f(vr[d]) : 0.f;
          }
        }
      }
      __syncthreads();
      float s[4] = {0.f, 0.f, 0.f, 0.f};
      for (int d = 0; d < hdp; d += 4) {
        const float4 qv = *reinterpret_cast<const float4*>(sQ + r * ldk + d);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float4 kv = *reinterpret_cast<const float4*>(sK + (c + 8 * i) * ldk + d);
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
        sP[r * kTK + c + 8 * i] = p;
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
        const float* vcol = sV + 4 * (c + 8 * i);
#pragma unroll 8
        for (int kk = 0; kk < kTK; ++kk) {
          const float p = sP[r * kTK + kk];
          const float4 v = *reinterpret_cast<const float4*>(vcol + kk * ldk);
          o.x = fmaf(p, v.x, o.x);
          o.y = fmaf(p, v.y, o.y);
          o.z = fmaf(p, v.z, o.z);
          o.w = fmaf(p, v.w, o.w);
        }
        acc[i] = o;
      }
      __syncthreads();
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
// Block (c, y): joins the pieces of the entity that starts in block c, rows 4y .. 4y + 3.
// Pieces are weighted with 2^(m_i - max m) and added in a fixed order.  A warp joins a row;
// when an entity lies in many pieces (a few long requests over all SMs) the four warps
// share each row's pieces instead, as one warp's loads would run one after another.
constexpr int kJoinThreads = 128;
constexpr int kJoinRows = 4;
constexpr int kJoinSplit = 16;  // pieces from which the warps share a row

template <typename T, int V>
__global__ void __launch_bounds__(kJoinThreads)
paged_join_kernel(const __grid_constant__ Args a, int Mt) {
  extern __shared__ float sw[];  // [warps][blocks] weights
  __shared__ float sums[kJoinRows][256];
  start_next_kernel();
  wait_kernel_before();
  const Open op = a.open[blockIdx.x];
  const int row_base = blockIdx.y * kJoinRows;
  if (op.parts == 0 || row_base >= op.rows) return;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int E = 256 / 32;  // elements per lane, in runs of V
  const bool share = op.parts > kJoinSplit;
  float* wgt = sw + warp * gridDim.x;

  for (int k = 0; k < (share ? kJoinRows : 1); ++k) {
    const int row = row_base + (share ? k : warp);
    if (row >= op.rows) break;
    auto slot_row = [&](int i) {
      const int s = i == 0 ? op.slot : 2 * ((int)blockIdx.x + i);
      return (int64_t)s * Mt + row;
    };
    auto column = [&](int e) { return (e / V) * (32 * V) + lane * V + e % V; };
    float mx = -INFINITY;
    for (int i = lane; i < op.parts; i += 32) {
      const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * slot_row(i));
      if (ml.y != 0.f) mx = fmaxf(mx, ml.x);
    }
    mx = warp_max(mx);
    float l = 0.f;
    for (int i = lane; i < op.parts; i += 32) {
      const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * slot_row(i));
      const float w = ml.y == 0.f ? 0.f : exp2f(ml.x - mx);
      wgt[i] = w;
      l += ml.y == 0.f ? 0.f : w * ml.y;
    }
    l = warp_sum(l);
    __syncwarp();
    float acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma unroll 4
    for (int i = share ? warp : 0; i < op.parts; i += share ? kJoinRows : 1) {
      const float w = wgt[i];
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
    if (share) {
      if (k > 0) __syncthreads();  // the row before is read
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (column(e) < a.hd) sums[warp][column(e)] = acc[e];
      __syncthreads();
      if (warp != 0) continue;
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (column(e) < a.hd)
          acc[e] = (sums[0][column(e)] + sums[1][column(e)]) +
                   (sums[2][column(e)] + sums[3][column(e)]);
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
}

int launch_join(int dtype, const Args& a, int blocks, int Mt, cudaStream_t st) {
  const size_t smem = (size_t)blocks * (kJoinThreads / 32) * sizeof(float);
  const dim3 grid((unsigned)blocks, (unsigned)ceil_div(Mt, kJoinRows));
  return PE_DISPATCH(dtype, T, [&]() -> int {
    auto kern = a.hd % 4 == 0 ? paged_join_kernel<T, 4> : paged_join_kernel<T, 1>;
    return launch_kernel(kern, grid, kJoinThreads, smem, st, true, a, Mt);
  });
}

int launch_simt(int dtype, const Args& a, int blocks, bool dependent, cudaStream_t st) {
  const int hdp = (a.hd + 3) / 4 * 4;
  const size_t smem = (size_t)((kSimtRows + 2 * kTK) * (hdp + 4) + kSimtRows * kTK) * sizeof(float);
  const int es = dtype == PE_F32 ? 4 : 2;
  const int vec = a.hd * es % 16 == 0 && (reinterpret_cast<uintptr_t>(a.kc) & 15u) == 0 &&
                  (reinterpret_cast<uintptr_t>(a.vc) & 15u) == 0;
  return PE_DISPATCH(dtype, T, [&]() -> int {
    auto kern = paged_simt_kernel<T>;
    PE_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    return launch_kernel(kern, dim3((unsigned)blocks), kThreads, smem, st, dependent, a, hdp, vec);
  });
}

// ------------------------------------------------------------------ kernel choice ----
enum Kind { kSimt, kFew, kMany };

struct Phase {
  Kind kind;
  int Mt, blocks;
};

Phase simt_phase(int hd) { return {kSimt, kSimtRows, sm_count() * (hd <= 128 ? 4 : 2)}; }

// tensor-core kernel for `rows` packed rows (on average) per request and KV head
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
  if (rc) return rc;
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
  int64_t bytes = phase_bytes(simt_phase(hd), hd);  // (operands may rule the tensor cores out)
  if (tc_sizes(dtype, hd)) bytes = std::max(bytes, phase_bytes(tc_phase(ceil_div(T * G, B)), hd));
  if (shared <= 0) return (size_t)bytes;
  int64_t prefix = phase_bytes(simt_phase(hd), hd);
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
  PE_CHECK_ARG(algo == PE_ALGO_AUTO || algo == PE_ALGO_SIMT || algo == PE_ALGO_TCGEN05,
               "attn_paged: unknown algorithm %d", algo);
  PE_CHECK_ARG(Hq >= 1 && Hkv >= 1 && Hq % Hkv == 0 && Hq / Hkv <= 256,
               "attn_paged: %d query heads over %d KV heads", Hq, Hkv);
  PE_CHECK_ARG(hd >= 1 && hd <= 256, "attn_paged: head_dim %d, expected 1 to 256", hd);
  PE_CHECK_ARG(B >= 1 && B < (1 << 20) && T >= 0 && T * Hq < (1ll << 31),
               "attn_paged: %lld requests, %lld rows of %d heads", (long long)B, (long long)T, Hq);
  PE_CHECK_ARG(page >= 16 && page % 16 == 0 && page <= (1 << 20),
               "attn_paged: page size %lld is not a multiple of 16", (long long)page);
  PE_CHECK_ARG(num_pages >= 1 && num_pages < (1ll << 31) && num_pages * Hkv * page < (1ll << 40),
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
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  if (shared > 0) {
    // the prefix once, all rows of all requests together, into fp32 rows
    float* pre_o = reinterpret_cast<float*>(ws);
    ws += al256(T * Hq * hd * 4);
    float* pre_lse = reinterpret_cast<float*>(ws);
    ws += al256(T * Hq * 4);
    const Phase p = tc ? tc_phase(T * a.G) : simt_phase(hd);
    Args pa = a;
    pa.all_rows = 1;
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
  const Phase p = tc ? tc_phase(ceil_div(T * a.G, B)) : simt_phase(hd);
  carve(a, p, ws);
  return run_phase(dtype, p, a, shared > 0, st);
}
