// The drafter's paged key/value cache: the page plan (block tables, slot maps, pages
// taken from and given back to the free ring) and the append of new rows.
//
// The cache itself is [pages, Hkv, page, hd] for K and for V: one head's keys of one page
// are contiguous, so the attention kernels read whole pages with single copies.  The
// reference keeps no drafter cache: it runs the drafter over the whole context for every
// draft (src/pe/drafter.py:195-236).
#include <limits.h>

#include <algorithm>

#include "common.cuh"

namespace pe {
namespace {

// ---------------------------------------------------------------- page plan ----
// Request b goes from lens[b] cached keys to new_lens[b].  With used = ceil(len / page) and
// need = ceil(new_len / page) pages (neither below the shared ones), need - used pages are
// taken from the ring's head, or used - need are pushed onto its tail, in request order; the
// new rows new_len - len get their positions and slots (page * page_size + offset).
//
// Every block scans all requests by itself (they are a few KB that sit in L2) and then takes
// its share of the three flat index spaces -- new rows, pages taken, pages given back --
// finding an index's request by bisection in shared memory.  A row's page comes straight
// from the ring when this call is the one that takes it, so no block reads what another
// writes and one launch does it all.  A thread describes two rows (one bisection, 16-byte
// stores).  Bound by latency: a scan, then per row a bisection and one dependent read of the
// ring or the table.  Measured: 8 drafts 5.2 us, 512 requests with 788K new rows 11 us.
constexpr int kPlanThreads = 512;
constexpr int kPlanBlocks = 2;    // blocks an SM's registers hold (60 a thread)
constexpr int kPlanBatch = 8192;  // requests whose scan fits the block's shared memory

struct Scan3 {
  int64_t rows;
  int grow, drop;
};

__device__ __forceinline__ Scan3 add3(Scan3 a, Scan3 b) {
  return {a.rows + b.rows, a.grow + b.grow, a.drop + b.drop};
}

// last index i in [0, n) with v[i] <= x (v ascending, v[0] = 0)
__device__ __forceinline__ int find(const int* v, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (v[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kPlanThreads, kPlanBlocks)
plan_kernel(int B, int64_t width, int N, int page, int64_t rows, int sp,
            const int32_t* __restrict__ lens, const int32_t* __restrict__ want,
            int32_t* table, int64_t table_ld, int32_t* ring_pages,
            const int64_t* __restrict__ ring, int64_t* __restrict__ ring_out,
            int32_t* __restrict__ granted, int32_t* __restrict__ cu, int64_t* __restrict__ slots,
            int64_t* __restrict__ pos) {
  extern __shared__ int sm[];
  int* s_cu = sm;                  // [B + 1] first new row
  int* s_grow = s_cu + B + 1;      // [B + 1] pages taken by the requests before
  int* s_drop = s_grow + B + 1;    // [B + 1] pages given back by the requests before
  int* s_used = s_drop + B + 1;    // [B] pages held; -1: the lengths fit no table
  int* s_from = s_used + B;        // [B] keys held
  __shared__ Scan3 s_warp[kPlanThreads / 32];
  __shared__ int s_refused, s_taken, s_given;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) s_refused = s_taken = s_given = 0;
  const int64_t head = ring[0], tail = ring[1];
  // counters that no ring of N pages can have serve nothing
  const bool sane = head >= 0 && tail >= head && tail - head <= N;
  const int avail = sane ? (int)(tail - head) : 0, room = sane ? N - avail : 0;
  const uint32_t head_at = sane ? (uint32_t)(head % N) : 0, tail_at = sane ? (uint32_t)(tail % N) : 0;
  auto ring_at = [&](uint32_t first, uint32_t i) {  // i < N
    const uint32_t x = first + i;
    return x >= (uint32_t)N ? x - (uint32_t)N : x;
  };

  // ---- exclusive scan of (new rows, pages taken, pages given back) over the requests ----
  Scan3 carry{0, 0, 0};
  for (int b0 = 0; b0 < B; b0 += kPlanThreads) {
    const int b = b0 + tid;
    Scan3 v{0, 0, 0};
    if (b < B) {
      const int from = lens[b], to = want[b];
      const int64_t u = ((int64_t)from + page - 1) / page, n = ((int64_t)to + page - 1) / page;
      const int64_t least = (int64_t)sp * page;  // (rows below would land in the shared pages)
      const bool fits = from >= least && to >= least && u <= width && n <= width;
      const int used = max((int)u, sp), need = max((int)n, sp);
      s_from[b] = from;
      s_used[b] = fits ? used : -1;
      // (lengths the table cannot hold still own their rows, without slots)
      v.rows = max((int64_t)0, (int64_t)to - from);
      v.grow = fits ? max(0, need - used) : 0;
      v.drop = fits ? max(0, used - need) : 0;
    }
    Scan3 inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const Scan3 t{__shfl_up_sync(0xffffffffu, inc.rows, o), __shfl_up_sync(0xffffffffu, inc.grow, o),
                    __shfl_up_sync(0xffffffffu, inc.drop, o)};
      if (lane >= o) inc = add3(inc, t);
    }
    if (lane == 31) s_warp[warp] = inc;
    __syncthreads();
    Scan3 base = carry;
    for (int w = 0; w < kPlanThreads / 32; ++w) {
      if (w < warp) base = add3(base, s_warp[w]);
      carry = add3(carry, s_warp[w]);
    }
    if (b < B) {
      s_cu[b] = (int)min(base.rows + inc.rows - v.rows, (int64_t)INT_MAX);  // (only wild lengths)
      s_grow[b] = base.grow + inc.grow - v.grow;
      s_drop[b] = base.drop + inc.drop - v.drop;
    }
    __syncthreads();
  }
  if (tid == 0) {
    s_cu[B] = (int)min(carry.rows, (int64_t)INT_MAX);
    s_grow[B] = carry.grow;
    s_drop[B] = carry.drop;
  }
  __syncthreads();

  // a request is served when its pages are there: growth while the ring's pages last,
  // returns while the ring has room (it always has, unless a page was given back twice)
  auto served = [&](int b) {
    const bool grows = s_grow[b + 1] > s_grow[b], drops = s_drop[b + 1] > s_drop[b];
    return s_used[b] >= 0 && (!grows || s_grow[b + 1] <= avail) && (!drops || s_drop[b + 1] <= room);
  };

  if (blockIdx.x == 0) {
    for (int b = tid; b < B; b += kPlanThreads) {
      const bool ok = served(b);
      granted[b] = ok ? want[b] : s_from[b];
      if (ok && s_grow[b + 1] > s_grow[b]) atomicAdd(&s_taken, s_grow[b + 1] - s_grow[b]);
      if (ok && s_drop[b + 1] > s_drop[b]) atomicAdd(&s_given, s_drop[b + 1] - s_drop[b]);
      if (!ok) atomicAdd(&s_refused, 1);
    }
    for (int b = tid; b <= B; b += kPlanThreads) cu[b] = s_cu[b];
    __syncthreads();
    if (tid == 0) {
      ring_out[0] = head + s_taken;
      ring_out[1] = tail + s_given;
      ring_out[2] = s_refused;
    }
  }

  const int64_t stride = (int64_t)gridDim.x * kPlanThreads, i0 = (int64_t)blockIdx.x * kPlanThreads + tid;
  // ---- new rows, two a thread: position and slot ----
  const int live = s_cu[B];
  const bool wide = ((reinterpret_cast<uintptr_t>(slots) | reinterpret_cast<uintptr_t>(pos)) & 15u) == 0;
  for (int64_t r0 = 2 * i0; r0 < rows; r0 += 2 * stride) {
    int64_t slot[2] = {-1, -1}, p[2] = {0, 0};
    int b = r0 < live ? find(s_cu, B, (int)r0) : 0;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int64_t r = r0 + e;
      if (r >= live) break;
      while (r >= s_cu[b + 1]) ++b;  // (requests without rows)
      p[e] = (int64_t)s_from[b] + ((int)r - s_cu[b]);
      if (!served(b)) continue;
      const uint32_t i = (uint32_t)p[e] / (uint32_t)page;
      const int id = i >= (uint32_t)s_used[b]
                         ? ring_pages[ring_at(head_at, s_grow[b] + i - s_used[b])]
                         : table[(int64_t)b * table_ld + i];
      slot[e] = (int64_t)id * page + ((uint32_t)p[e] - i * (uint32_t)page);
    }
    if (wide && r0 + 1 < rows) {
      *reinterpret_cast<longlong2*>(slots + r0) = make_longlong2(slot[0], slot[1]);
      *reinterpret_cast<longlong2*>(pos + r0) = make_longlong2(p[0], p[1]);
    } else {
      for (int e = 0; e < 2 && r0 + e < rows; ++e) {
        slots[r0 + e] = slot[e];
        pos[r0 + e] = p[e];
      }
    }
  }
  // ---- pages taken: table entries ----
  for (int64_t g = i0; g < min(s_grow[B], avail); g += stride) {
    const int b = find(s_grow, B, (int)g);
    if (served(b))
      table[(int64_t)b * table_ld + s_used[b] + (int)g - s_grow[b]] =
          ring_pages[ring_at(head_at, (uint32_t)g)];
  }
  // ---- pages given back: ring entries ----
  for (int64_t d = i0; d < min(s_drop[B], room); d += stride) {
    const int b = find(s_drop, B, (int)d);
    if (served(b))
      ring_pages[ring_at(tail_at, (uint32_t)d)] =
          table[(int64_t)b * table_ld + s_used[b] - (s_drop[b + 1] - s_drop[b]) + (int)d - s_drop[b]];
  }
}

// ------------------------------------------------------------------- append ----
// Row t of k / v -> its slot in the cache: per head a contiguous run of hd elements.  A
// copy, bound by HBM: one read and one write of each row.  A thread moves kItems pieces
// of K and of V (16 bytes each when rows and cache allow it), with all of its loads
// issued before the first store.  Measured: 16411 rows of 8 x 128 bf16 23.4 us, 5.75 TB/s
// (0.89 of a plain copy); 48 rows 3.4 us.
constexpr int kAppendThreads = 256;
constexpr int kItems = 4;

// I: the type that holds every index (32-bit divisions where the sizes allow them).
template <typename V, typename I>
__global__ void __launch_bounds__(kAppendThreads)
append_kernel(int64_t rows, int per_row, int per_head, int Hkv, const V* __restrict__ k,
              int64_t k_ld, const V* __restrict__ v, int64_t v_ld,
              const int64_t* __restrict__ slots, int64_t num_slots, int page, V* __restrict__ kc,
              V* __restrict__ vc) {
  const I total = (I)rows * per_row;
  const I base = (I)blockIdx.x * (kAppendThreads * kItems) + threadIdx.x;
  V kv[kItems], vv[kItems];
  int64_t dst[kItems];
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const I at = base + (I)(i * kAppendThreads);
    dst[i] = -1;
    if (at >= total) continue;
    const I row = at / (I)per_row;
    const uint32_t j = (uint32_t)(at - row * (I)per_row);
    const int64_t slot = slots[row];
    if (slot < 0 || slot >= num_slots) continue;
    const uint32_t h = j / (uint32_t)per_head;
    const I pg = (I)slot / (I)page;
    const uint32_t off = (uint32_t)((I)slot - pg * (I)page);
    dst[i] = (((int64_t)pg * Hkv + h) * page + off) * per_head + (j - h * (uint32_t)per_head);
    kv[i] = k[(int64_t)row * k_ld + j];
    vv[i] = v[(int64_t)row * v_ld + j];
  }
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    if (dst[i] < 0) continue;
    kc[dst[i]] = kv[i];
    vc[dst[i]] = vv[i];
  }
}

template <typename V>
int append_launch(int64_t rows, int Hkv, int hd_units, const void* k, int64_t k_ld, const void* v,
                  int64_t v_ld, const int64_t* slots, int64_t num_slots, int page, void* kc,
                  void* vc, cudaStream_t st) {
  const int per_row = Hkv * hd_units;
  const int64_t blocks = ceil_div(rows * per_row, kAppendThreads * kItems);
  PE_CHECK_ARG(blocks < (1ll << 31), "cache_append: too many rows for one launch");
  // (the last block's indices run past the total by less than a block)
  const bool small = num_slots < (1ll << 31) &&
                     rows * per_row < (1ll << 32) - kAppendThreads * kItems;
  auto kern = small ? append_kernel<V, uint32_t> : append_kernel<V, uint64_t>;
  kern<<<(unsigned)blocks, kAppendThreads, 0, st>>>(
      rows, per_row, hd_units, Hkv, (const V*)k, k_ld, (const V*)v, v_ld, slots, num_slots, page,
      (V*)kc, (V*)vc);
  PE_LAUNCHED();
  return PE_OK;
}

}  // namespace
}  // namespace pe

using namespace pe;

extern "C" int pe_cache_plan(int64_t B, int64_t width, int64_t num_pages, int64_t page,
                             int64_t rows, int64_t shared, const int32_t* lens,
                             const int32_t* new_lens, int32_t* table, int64_t table_ld,
                             int32_t* free_ring, const int64_t* ring, int64_t* ring_out,
                             int32_t* granted, int32_t* cu, int64_t* slots, int64_t* pos,
                             void* stream) {
  PE_CHECK_ARG(B >= 1 && B <= kPlanBatch, "cache_plan: %lld requests, expected 1 to %d",
               (long long)B, kPlanBatch);
  PE_CHECK_ARG(page >= 1 && page <= (1 << 20), "cache_plan: page size %lld", (long long)page);
  PE_CHECK_ARG(width >= 1 && width < (1ll << 31) && width * page < (1ll << 31) && table_ld >= width,
               "cache_plan: block table of %lld pages (row stride %lld)", (long long)width,
               (long long)table_ld);
  PE_CHECK_ARG(num_pages >= 1 && num_pages < (1ll << 30) && B * width < (1ll << 31),
               "cache_plan: %lld pages", (long long)num_pages);
  PE_CHECK_ARG(rows >= 0 && rows < (1ll << 31), "cache_plan: %lld new rows", (long long)rows);
  PE_CHECK_ARG(shared >= 0 && shared % page == 0 && shared / page <= width,
               "cache_plan: %lld shared keys are not whole pages of the table", (long long)shared);
  PE_CHECK_ARG(lens && new_lens && table && free_ring && ring && ring_out && granted && cu &&
                   (rows == 0 || (slots && pos)),
               "cache_plan: null pointer");
  PE_CHECK_ARG(ring != ring_out && lens != granted && new_lens != granted,
               "cache_plan: ring_out and granted must not alias the inputs");
  const size_t smem = (5 * (size_t)B + 3) * sizeof(int);
  if (smem > 48 * 1024) {
    const int rc = allow_smem<plan_kernel>((5 * kPlanBatch + 3) * (int)sizeof(int));
    if (rc) return rc;
  }
  // a block per 1024 rows (and per 256 requests, whose pages it fills), up to what the SMs hold
  // at once: a row's chain of dependent reads takes the time, so the more in flight the better,
  // but a block that waits for a place starts with a scan of its own (512 prompts, 788K rows:
  // 13.6 us with one an SM, 11.1 with two, 14.0 with three; 96K rows the same with each).
  // Where the scan is long, one an SM: 4000 requests with 302K rows 21.3 us, 25.7 with two.
  const int64_t want = std::max(ceil_div(rows, 2 * kPlanThreads), ceil_div(B, 256));
  const int64_t most = smem > 64 * 1024 ? 1 : kPlanBlocks;
  const int blocks = (int)std::min<int64_t>(std::max<int64_t>(want, 1), most * sm_count());
  plan_kernel<<<blocks, kPlanThreads, smem, as_stream(stream)>>>(
      (int)B, width, (int)num_pages, (int)page, rows, (int)(shared / page), lens, new_lens, table,
      table_ld, free_ring, ring, ring_out, granted, cu, slots, pos);
  PE_LAUNCHED();
  return PE_OK;
}

extern "C" int pe_cache_append(int dtype, int64_t rows, int Hkv, int hd, const void* k,
                               int64_t k_ld, const void* v, int64_t v_ld, const int64_t* slots,
                               int64_t num_pages, int64_t page, void* k_cache, void* v_cache,
                               void* stream) {
  PE_CHECK_ARG(dtype == PE_F32 || dtype == PE_BF16, "cache_append: unsupported dtype code %d",
               dtype);
  PE_CHECK_ARG(rows >= 0 && rows < (1ll << 38) && Hkv >= 1 && hd >= 1 &&
                   (int64_t)Hkv * hd < (1 << 24),
               "cache_append: %lld rows of %d heads of %d", (long long)rows, Hkv, hd);
  PE_CHECK_ARG(num_pages >= 0 && num_pages < (1ll << 31) && page >= 1 && page <= (1 << 20),
               "cache_append: %lld pages of %lld", (long long)num_pages, (long long)page);
  if (rows == 0) return PE_OK;
  PE_CHECK_ARG(k && v && slots && k_cache && v_cache, "cache_append: null pointer");
  PE_CHECK_ARG(rows == 1 || (k_ld >= (int64_t)Hkv * hd && v_ld >= (int64_t)Hkv * hd),
               "cache_append: row strides %lld, %lld below %d x %d", (long long)k_ld,
               (long long)v_ld, Hkv, hd);
  const int es = dtype == PE_F32 ? 4 : 2, per16 = 16 / es;
  auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  const bool wide = hd % per16 == 0 && k_ld % per16 == 0 && v_ld % per16 == 0 && al(k) && al(v) &&
                    al(k_cache) && al(v_cache);
  const cudaStream_t st = as_stream(stream);
  if (wide)
    return append_launch<uint4>(rows, Hkv, hd / per16, k, k_ld / per16, v, v_ld / per16, slots,
                                num_pages * page, (int)page, k_cache, v_cache, st);
  if (es == 4)
    return append_launch<uint32_t>(rows, Hkv, hd, k, k_ld, v, v_ld, slots, num_pages * page,
                                   (int)page, k_cache, v_cache, st);
  return append_launch<uint16_t>(rows, Hkv, hd, k, k_ld, v, v_ld, slots, num_pages * page,
                                 (int)page, k_cache, v_cache, st);
}
