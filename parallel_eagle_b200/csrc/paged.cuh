// Attention that reads the paged key/value cache: the pieces its kernels share.
//
// The work of one launch is a line of cost units: request after request, within a request
// KV head after KV head, within a head one entity per tile of Mt query rows (a row is one
// (new token, query head of the KV head's group) pair; rows of a group share their keys, so
// packing them fills the matrix instructions' row dimension).  An entity's cost is about
// its keys.  Each block takes an equal piece of that line, so a batch of any raggedness
// loads all SMs alike, a lone long request is split over all of them, and no host knowledge
// of the lengths is needed: a block finds its piece from lens and cu alone.
//
// A piece that is a whole entity writes its rows' result.  Otherwise an entity's pieces
// leave partial results (accumulator, running maximum, sum) in per-block slots -- a block
// has at most two incomplete entities, its first and its last -- and the block that holds
// the entity's first piece records how many there are; the join kernel adds them in
// piece order, so results do not depend on timing.  (Where requests are short, no entity is
// cut: a block takes those that start in its piece.)
#pragma once
#include "common.cuh"

namespace pe {
namespace paged {

struct Args {
  const void* q;          // [T, Hq * hd], row stride q_ld
  int64_t q_ld;
  const void *kc, *vc;    // [num_pages, Hkv, page, hd]
  int64_t num_pages;
  int page;
  const int32_t* table;   // [B, width] (row stride table_ld)
  int64_t table_ld;
  int64_t kmax;           // keys a table row can hold: width * page
  const int32_t* lens;    // [B] keys of each request, its new rows among them
  const int32_t* cu;      // [B + 1] first row of each request
  int B, T, Hq, Hkv, hd, G;  // G = Hq / Hkv
  int64_t kbeg;           // first key (the shared prefix, when another launch does it)
  int all_rows;           // 1: one request of cu[B] rows that all see keys [kbeg, kmax)
  int align;              // 1: pieces that cut every entity at the same places (all_rows, and
                          // the piece found by init_warp: the tensor-core kernels)
  int whole;              // 1: a block takes the entities that start in its piece, uncut
  float scale_log2;       // log2(e) / sqrt(hd)
  void* o;                // result rows (the operand type), row stride o_ld
  int64_t o_ld;
  float* lse;             // [Hq, T]
  float* o32;             // when set, results go here instead (fp32 [T, Hq, hd]) with lse
  const float* pre_o;     // a prefix's result [T, Hq, hd] and lse [Hq, T] to join with
  const float* pre_lse;
  float* part_o;          // [2 * blocks, Mt, hd] unnormalised accumulators
  float* part_ml;         // [2 * blocks, Mt, 2] running maximum (log2 units) and sum
  struct Open* open;      // [blocks] incomplete entity that starts in the block
  int* status;
};

// an entity whose first piece block c holds and whose rest the blocks after it hold
struct Open {
  int parts;   // 0: none
  int slot;    // first piece's slot; piece i > 0 lies in slot 2 * (c + i)
  int row0;    // first row of the request
  int r0;      // first packed row (token * G + head in group) of the tile
  int rows;    // packed rows of the tile
  int kvh;
  int pad[2];
};

constexpr float kLn2f = 0.6931471805599453f;

// a / b for a, b >= 0 (the 64-bit division costs several times the 32-bit one, and small
// calls spend their time here)
__device__ __forceinline__ int64_t div_pos(int64_t x, int64_t y) {
  if (((x | y) >> 32) == 0) return (uint32_t)x / (uint32_t)y;
  return x / y;
}

// one request as a launch sees it
struct Req {
  int row0, n;        // first row in q, new rows
  int64_t first;      // keys row 0 sees, kbeg included (row j sees first + j; all_rows: constant)
  int R;              // row tiles
  int64_t A;          // cost model: (A + slope terms), see cost()
};

// A segment as the tensor-core kernels' warps hand it round in shared memory: one warp
// walks the line of work, the others read.
struct Seg {
  int64_t kend;    // keys the tile's last row sees (exclusive end)
  int64_t lim0;    // keys the tile's first row sees
  const int32_t* pages;
  int row0;        // first row of the request
  int r0, rows;    // first packed row of the tile, packed rows in it
  int kvh;
  int t0, t1;      // key tiles
  int slot;        // of the partial result; -1: the segment is its whole entity
  int end;         // 1: no more segments
};

// Mt: packed rows per tile.  TK: keys per tile.  kOver: what a segment's start and end cost
// on top of its keys, in keys (Q rows in, result rows out, the pipeline's filling).  kLeast:
// keys below which no block's piece goes (a small call ends sooner on fewer blocks).
template <int Mt, int TK, int kOver, int kLeast>
struct Sched {
  const Args& a;
  int64_t total, per, pos, end;  // cost units; this block's piece is [pos, end)
  int b;                         // request that holds pos
  int64_t base;                  // its first unit
  Req rq;
  // the current segment: entity (rq, kvh, rt), key tiles [t0, t1) of nt
  int kvh, rt, t0, t1, nt;
  bool first, last;
  int64_t kend;                  // keys the entity's last row sees (exclusive end)
  int seg;                       // segments taken so far

  __device__ __forceinline__ Sched(const Args& args) : a(args) {}

  __device__ __forceinline__ int requests() const { return a.all_rows ? 1 : a.B; }

  __device__ __forceinline__ Req request(int i) const {
    Req r;
    if (a.all_rows) {
      r.row0 = 0;
      r.n = max(0, min(a.cu[a.B], a.T));
      r.first = a.kmax;
      r.A = a.kmax - a.kbeg;
    } else {
      const int c0 = a.cu[i], c1 = a.cu[i + 1];
      r.row0 = max(0, min(c0, a.T));
      r.n = max(0, min(c1, a.T) - r.row0);
      r.first = (int64_t)a.lens[i] - ((int64_t)c1 - c0) + 1;
      r.A = max((int64_t)0, min(r.first, a.kmax) - a.kbeg);
    }
    r.R = (int)(((int64_t)r.n * a.G + Mt - 1) / Mt);
    return r;
  }
  // cost of row tile rt: its keys times G, plus the overhead.  (A last tile that is not full
  // counts like any other: it waits as long for every key tile.)
  __device__ __forceinline__ int64_t cost(const Req& r, int rt) const {
    return (r.A + kOver) * a.G + (a.all_rows ? 0 : (int64_t)(rt + 1) * Mt);
  }
  // ... of the tiles before rt
  __device__ __forceinline__ int64_t cost_before(const Req& r, int64_t rt) const {
    return rt * (r.A + kOver) * a.G + (a.all_rows ? 0 : rt * (rt + 1) / 2 * Mt);
  }
  __device__ __forceinline__ int64_t head_cost(const Req& r) const { return cost_before(r, r.R); }
  __device__ __forceinline__ int64_t req_cost(const Req& r) const {
    return (int64_t)a.Hkv * head_cost(r);
  }

  // The piece of a block whose one warp walks the line, by that warp alone: no barrier, and
  // the lengths' way from memory overlaps the block's other preparations.  (A lane looks at
  // every 32nd part of the requests; from some hundred on the whole block is quicker.)
  static constexpr int kWarpRequests = 128;
  __device__ __forceinline__ void init_warp() {
    const int n = requests(), lane = threadIdx.x & 31;
    const int chunk = (n + 31) / 32, i0 = min(n, lane * chunk), i1 = min(n, i0 + chunk);
    int64_t mine = 0;
    for (int i = i0; i < i1; ++i) mine += req_cost(request(i));
    int64_t inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t t = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += t;
    }
    total = __shfl_sync(0xffffffffu, inc, 31);
    per = max(div_pos(total + gridDim.x - 1, gridDim.x), (int64_t)kLeast * a.G);
    if (a.align) {
      // A piece of a half entity's multiple (within a tenth of an equal share): blocks on the
      // row tiles of one head then walk the same keys at the same time, and a key tile comes
      // from HBM about twice for all of them (L2 has two halves) in place of once for each:
      // seven row tiles over 268 MB of keys and values read 551 MB, 1817 with equal pieces.
      const Req r = request(0);
      const int64_t twice = r.R > 0 ? 2 * cost(r, 0) : 0, halves = div_pos(twice, per);
      if (halves >= 2 && halves * per * 10 >= twice * 9)
        per = div_pos(twice + halves - 1, halves);
    }
    pos = min(total, (int64_t)blockIdx.x * per);
    end = min(total, pos + per);
    seg = 0;
    b = 0;
    base = inc - mine;
    if (pos >= end) return;
    const int owner = __ffs(__ballot_sync(0xffffffffu, pos < inc)) - 1;
    b = __shfl_sync(0xffffffffu, i0, owner);
    base = __shfl_sync(0xffffffffu, base, owner);
    rq = request(b);
    // (next() steps over the owner's requests before pos)
  }

  // all threads of the block; scratch: one int64 per warp plus 4
  __device__ __forceinline__ void init(int64_t* scratch) {
    const int n = requests(), tid = threadIdx.x, nthr = blockDim.x;
    const int lane = tid & 31, warp = tid >> 5, nw = nthr >> 5;
    const int chunk = (n + nthr - 1) / nthr;
    const int i0 = min(n, tid * chunk), i1 = min(n, i0 + chunk);
    int64_t mine = 0;
    for (int i = i0; i < i1; ++i) mine += req_cost(request(i));
    int64_t inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t t = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += t;
    }
    if (lane == 31) scratch[warp] = inc;
    if (tid == 0) scratch[nw] = -1;
    __syncthreads();
    int64_t before = inc - mine, sum = 0;
    for (int w = 0; w < nw; ++w) {
      if (w < warp) before += scratch[w];
      sum += scratch[w];
    }
    total = sum;
    // an equal share each, but none too small
    per = max(div_pos(total + gridDim.x - 1, gridDim.x), (int64_t)kLeast * a.G);
    pos = min(total, (int64_t)blockIdx.x * per);
    end = min(total, pos + per);
    // the thread whose requests hold pos finds the request
    if (pos < end && before <= pos && pos < before + mine) {
      int i = i0;
      int64_t at = before;
      while (true) {
        const int64_t c = req_cost(request(i));
        if (pos < at + c) break;
        at += c;
        ++i;
      }
      scratch[nw] = i;
      scratch[nw + 1] = at;
    }
    __syncthreads();
    b = (int)scratch[nw];
    base = scratch[nw + 1];
    seg = 0;
    if (pos < end) rq = request(b);
    __syncthreads();
  }

  // next segment of the piece; false when there is none.  Same result in every thread.
  __device__ __forceinline__ bool next() {
    while (find()) {
      if (!a.whole || first) return true;
    }
    return false;
  }
  __device__ __forceinline__ bool find() {
    if (pos >= end) return false;
    int64_t rc = req_cost(rq);
    while (pos >= base + rc) {  // (requests without rows cost nothing)
      base += rc;
      if (++b >= requests()) return false;  // (row offsets that make no sense)
      rq = request(b);
      rc = req_cost(rq);
    }
    const int64_t per_head = head_cost(rq);
    int64_t off = pos - base;
    kvh = (int)div_pos(off, per_head);
    off -= kvh * per_head;
    // last row tile that starts at or before off
    int lo = 0, hi = rq.R;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (cost_before(rq, mid) <= off) lo = mid; else hi = mid;
    }
    rt = lo;
    const int64_t c = cost(rq, rt), u0 = off - cost_before(rq, rt);
    const int64_t u1 = a.whole ? c : min(c, u0 + (end - pos));
    // the entity's key tiles, in proportion to its units
    const int rows_end = (int)min((int64_t)rq.n * a.G, (int64_t)(rt + 1) * Mt);
    const int last_tok = (rows_end - 1) / a.G;
    kend = min(a.kmax, a.all_rows ? a.kmax : rq.first + last_tok);
    nt = kend > a.kbeg ? (int)((kend - a.kbeg + TK - 1) / TK) : 0;
    first = u0 == 0;
    last = u1 == c;
    t0 = first ? 0 : (int)div_pos(u0 * nt, c);
    t1 = last ? nt : (int)div_pos(u1 * nt, c);
    entity_end_ = pos - u0 + c;
    pos += u1 - u0;
    ++seg;
    return true;
  }
  __device__ __forceinline__ bool whole() const { return first && last; }
  // slot of the current (incomplete) segment's partial result
  __device__ __forceinline__ int slot() const { return 2 * (int)blockIdx.x + (seg == 1 ? 0 : 1); }
  // pieces of the current entity, for the block that holds its first piece but not its last
  __device__ __forceinline__ int parts() const {
    return (int)div_pos(entity_end_ - 1, per) - (int)blockIdx.x + 1;
  }
  // keys that packed row r (of the whole request) sees, as an exclusive end
  __device__ __forceinline__ int64_t limit(int r) const {
    return min(a.kmax, a.all_rows ? a.kmax : rq.first + r / a.G);
  }
  __device__ __forceinline__ int tile_rows() const {
    return (int)min((int64_t)Mt, (int64_t)rq.n * a.G - (int64_t)rt * Mt);
  }
  // block table row of the current request
  __device__ __forceinline__ const int32_t* pages() const {
    return a.table + (a.all_rows ? 0 : (int64_t)b * a.table_ld);
  }
  __device__ __forceinline__ void describe(Seg& g) const {
    g.kend = kend;
    g.lim0 = limit(rt * Mt);
    g.pages = pages();
    g.row0 = rq.row0;
    g.r0 = rt * Mt;
    g.rows = tile_rows();
    g.kvh = kvh;
    g.t0 = t0;
    g.t1 = t1;
    g.slot = whole() ? -1 : slot();
    g.end = 0;
  }
  // recorded by one thread for a segment that is its entity's first piece but not all of it
  __device__ __forceinline__ void record_open() const {
    Open r{};
    r.parts = parts();
    r.slot = slot();
    r.row0 = rq.row0;
    r.r0 = rt * Mt;
    r.rows = tile_rows();
    r.kvh = kvh;
    a.open[blockIdx.x] = r;
  }

 private:
  int64_t entity_end_;
};

// The kernels of one call (prefix, its join, the requests' own keys, their join) are launched
// as programmatic dependents: each may start while the one before it runs, and waits at
// the point where it reads that one's results.  They share no scratch.
__device__ __forceinline__ void start_next_kernel() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void wait_kernel_before() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// launch, optionally as a dependent of the kernel before it in the stream
template <typename... P, typename... A>
inline int launch_kernel(void (*kern)(P...), dim3 grid, unsigned threads, size_t smem,
                         cudaStream_t st, bool dependent, A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = dependent ? 1 : 0;
  PE_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, P(args)...));
  ++launch_counter();
  return PE_OK;
}

// Block table entries of a segment as its copying warp walks it: a lane holds one entry of
// the 32 in use and one of the 32 behind them, so that no copy waits for the table (a
// lookup per tile took 900 of a tile's 1900 cycles).  All lanes call.
struct PageWalk {
  const int32_t* pages;
  int limit;      // entries that may be read
  int at;         // entry of lane 0's `cur`
  int cur, next;
  __device__ __forceinline__ int load(int i) const { return i < limit ? pages[i] : -1; }
  __device__ __forceinline__ void start(const int32_t* p, int first, int n) {
    const int lane = threadIdx.x & 31;
    pages = p;
    limit = n;
    at = first;
    cur = load(first + lane);
    next = load(first + 32 + lane);
  }
  // first: the lowest entry that is still asked for, the same in all lanes
  __device__ __forceinline__ void advance(int first) {
    if (first < at + 32) return;
    at += 32;
    cur = next;
    next = load(at + 32 + (int)(threadIdx.x & 31));
  }
  // entry i of [at, at + 64); last: the highest one asked for, the same in all lanes
  __device__ __forceinline__ int entry(int i, int last) const {
    const int a = __shfl_sync(0xffffffffu, cur, (i - at) & 31);
    if (last < at + 32) return a;  // (`next` may still be on its way)
    const int b = __shfl_sync(0xffffffffu, next, (i - at) & 31);
    return i - at < 32 ? a : b;
  }
};

// What a finished row's accumulator is multiplied by: o = own * acc + pre * pre_o.
struct RowScale {
  float own, pre, lse;
};

// m (log2 units) and l: running maximum and sum over the row's keys; t, head: the row
__device__ __forceinline__ RowScale finish_row(const Args& a, int t, int head, float m, float l) {
  RowScale s;
  if (!a.pre_lse) {
    s.own = l == 0.f ? 0.f : 1.f / l;
    s.pre = 0.f;
    s.lse = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2f;
    return s;
  }
  const float own = l == 0.f ? -INFINITY : m + log2f(l);
  const float pre = a.pre_lse[(int64_t)head * a.T + t] * (1.f / kLn2f);
  const float top = fmaxf(own, pre);
  if (top == -INFINITY) {
    s.own = s.pre = 0.f;
    s.lse = -INFINITY;
    return s;
  }
  const float wo = exp2f(own - top), wp = exp2f(pre - top), w = wo + wp;
  s.own = l == 0.f ? 0.f : wo / (w * l);
  s.pre = pre == -INFINITY ? 0.f : wp / w;
  s.lse = (top + log2f(w)) * kLn2f;
  return s;
}


// Tensor-core kernels (bf16, head sizes 64 and 128); `rows`: packed rows per tile.
// paged_tc_few.cu: 16, 32 or 64 rows, one block per SM
int launch_few(const Args& a, int rows, int blocks, bool dependent, cudaStream_t st);
// paged_tc_many.cu: 256 rows, one block per SM
int launch_many(const Args& a, int blocks, bool dependent, cudaStream_t st);

}  // namespace paged
}  // namespace pe
