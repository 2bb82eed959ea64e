// Kernels around a paged K/V cache: block tables and slot maps from request lengths, the
// visibility bits of drafted trees, writes of new K/V rows into the page pools, and the move
// of an accepted path's rows.  No counterpart in the reference, whose K/V is contiguous
// (README.md:139-141).
#include "common.cuh"

namespace fa4cp {
namespace {

constexpr int kMaxGrid = 148;  // one CTA per SM: every CTA repeats the scans below

__device__ __forceinline__ int64_t warp_scan_incl(int64_t v, int lane) {
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t o = __shfl_up_sync(0xffffffffu, v, d);
    if (lane >= d) v += o;
  }
  return v;
}

// ---------------------------------------------------------------------------
// block tables and slot maps
// ---------------------------------------------------------------------------
constexpr int kPlanThreads = 1024;

struct PlanParams {
  const int32_t *cached, *fresh, *free_pages, *num_free_dev, *table_in;
  int32_t *table_out, *cu_q, *cu_k, *seq_lens, *pages;
  int64_t* slots;
  int64_t num_tokens;
  int nseq, num_free, page_size, max_pages;
};

__device__ __forceinline__ int to_i32(int64_t v) {
  return int(min(v, int64_t(0x7fffffff)));  // sums past int32 (never valid lengths) saturate
}

// Exclusive block scan of three values at once (kPlanThreads threads); totals in tot[3].
__device__ __forceinline__ void block_scan3(int64_t (&v)[3], int64_t (&tot)[3], int64_t (*ws)[33],
                                            int warp, int lane) {
  int64_t inc[3];
#pragma unroll
  for (int i = 0; i < 3; ++i) inc[i] = warp_scan_incl(v[i], lane);
  __syncthreads();  // ws may still be read by the previous scan
  if (lane == 31) {
#pragma unroll
    for (int i = 0; i < 3; ++i) ws[i][warp] = inc[i];
  }
  __syncthreads();
  if (warp < 3) {
    const int64_t x = ws[warp][lane];
    const int64_t s = warp_scan_incl(x, lane);
    ws[warp][lane] = s - x;
    if (lane == 31) ws[warp][32] = s;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    v[i] = inc[i] - v[i] + ws[i][warp];
    tot[i] = ws[i][32];
  }
}

// Request j's new tokens sit at positions [cached, cached + fresh), on the pages
// [first, end) = [cached / ps, ceil((cached + fresh) / ps)).  The pages that it owns are a
// prefix of its row, so its missing pages are [fm, end) with fm = first negative entry, and
// they take free_pages[rank ...] with rank = the exclusive sum of the missing counts.
//
// Every CTA repeats the scans over all requests (in chunks of kPlanThreads), then fills its
// share of the table and of the slots: one launch with no global hand-over, at the price of
// re-reading 8 bytes a request per CTA from L2.  Bound by the chain lengths, table row, scans,
// free pages: 7.1 us for 256 requests with 513 pages each, 5.9 us for 64 prompts of 4096 tokens.
__global__ void __launch_bounds__(kPlanThreads, 1) plan_kernel(const PlanParams p) {
  __shared__ int s_cached[kPlanThreads], s_cu[kPlanThreads], s_fm[kPlanThreads],
      s_end[kPlanThreads], s_rank[kPlanThreads];
  __shared__ int64_t ws[3][33];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int nfree = max(p.num_free_dev ? min(p.num_free, *p.num_free_dev) : p.num_free, 0);
  int64_t base_q = 0, base_k = 0, base_rank = 0, beyond = 0;
  for (int j0 = 0; j0 < p.nseq; j0 += kPlanThreads) {
    const int j = j0 + tid, nj = min(kPlanThreads, p.nseq - j0);
    int cached = 0, fresh = 0, first = 0, end = 0, lim = 0, fm = 0;
    if (j < p.nseq) {
      cached = max(p.cached[j], 0);
      fresh = min(max(p.fresh[j], 0), 0x7fffffff - cached);
      first = cached / p.page_size;
      end = fresh > 0 ? int((int64_t(cached) + fresh + p.page_size - 1) / p.page_size) : first;
      lim = max(min(end, p.max_pages), first);  // the pages that the row has room for
      fm = first;
    }
    __syncthreads();  // the previous chunk's readers are done with the arrays
    bool wide = false;
    if (p.table_in != nullptr && lim > first) {
      const int32_t* row = p.table_in + int64_t(j) * p.max_pages;
      if (lim - first <= 4) {  // the common step: its few entries at once
        int e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = first + i < lim ? row[first + i] : -1;
        while (fm < lim && e[fm - first] >= 0) ++fm;
      } else {
        wide = true;
      }
    }
    if (tid < nj) { s_fm[tid] = wide ? -1 : fm; s_end[tid] = lim; s_cached[tid] = first; }
    __syncthreads();
    if (p.table_in != nullptr) {  // rows of many pages: a warp narrows [lo, hi) 32-fold a round
      for (int r = warp; r < nj; r += kPlanThreads / 32) {
        if (s_fm[r] >= 0) continue;
        const int32_t* row = p.table_in + int64_t(j0 + r) * p.max_pages;
        int lo = s_cached[r], hi = s_end[r];  // first negative entry is in [lo, hi]
        while (lo < hi) {
          const int step = (hi - lo + 31) / 32;
          const int at = lo + lane * step;
          const unsigned neg = __ballot_sync(0xffffffffu, at >= hi || row[at] < 0);
          if (neg & 1u) { hi = lo; break; }
          const int f = neg ? __ffs(neg) - 1 : 32;  // probe f is negative (or past hi)
          const int nlo = lo + (f - 1) * step + 1;
          hi = min(hi, lo + f * step);
          lo = nlo;
        }
        if (lane == 0) s_fm[r] = hi;
        __syncwarp();
      }
      __syncthreads();
      if (tid < nj) fm = s_fm[tid];
    }
    __syncthreads();
    int64_t v[3] = {fresh, int64_t(cached) + fresh, lim - fm}, tot[3];
    block_scan3(v, tot, ws, warp, lane);
    beyond += end - lim;  // pages past the row's width
    if (tid < nj) {
      s_cached[tid] = cached;
      s_cu[tid] = to_i32(base_q + v[0]);
      s_fm[tid] = fm;
      s_end[tid] = lim;
      s_rank[tid] = to_i32(base_rank + v[2]);
      if (blockIdx.x == 0) {
        p.cu_q[j] = to_i32(base_q + v[0]);
        p.cu_k[j] = to_i32(base_k + v[1]);
        p.seq_lens[j] = cached + fresh;
      }
    }
    __syncthreads();
    base_q += tot[0];
    base_k += tot[1];
    base_rank += tot[2];

    // table rows: one warp per (row, segment of 128 entries)
    const int segs = (p.max_pages + 127) / 128;
    for (int64_t u = int64_t(blockIdx.x) * (kPlanThreads / 32) + warp; u < int64_t(nj) * segs;
         u += int64_t(gridDim.x) * (kPlanThreads / 32)) {
      const int r = int(u / segs), e0 = int(u - int64_t(r) * segs) * 128;
      const int64_t row = int64_t(j0 + r) * p.max_pages;
      const int rfm = s_fm[r], rend = s_end[r], rank = s_rank[r];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = e0 + i * 32 + lane;
        if (e >= p.max_pages) break;
        int val = -1;
        if (e >= rfm && e < rend) {
          const int64_t f = int64_t(rank) + e - rfm;
          if (f < nfree) val = p.free_pages[f];
        } else if (p.table_in != nullptr) {
          val = p.table_in[row + e];
        }
        p.table_out[row + e] = val;
      }
    }
    // slots of the chunk's tokens: the token's request by binary search in s_cu
    const int64_t t_end = min(base_q, p.num_tokens);
    for (int64_t t = int64_t(s_cu[0]) + int64_t(blockIdx.x) * kPlanThreads + tid; t < t_end;
         t += int64_t(gridDim.x) * kPlanThreads) {
      int lo = 0, hi = nj;  // last r with s_cu[r] <= t
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_cu[mid] <= t) lo = mid; else hi = mid;
      }
      const int pos = s_cached[lo] + int(t - s_cu[lo]);
      const int e = pos / p.page_size;
      int page = -1;
      if (e < s_end[lo]) {
        if (e >= s_fm[lo]) {
          const int64_t f = int64_t(s_rank[lo]) + e - s_fm[lo];
          if (f < nfree) page = p.free_pages[f];
        } else {
          page = p.table_in[int64_t(j0 + lo) * p.max_pages + e];
        }
      }
      p.slots[t] = page < 0 ? -1 : int64_t(page) * p.page_size + (pos - e * p.page_size);
    }
    __syncthreads();
  }
  for (int64_t t = base_q + int64_t(blockIdx.x) * kPlanThreads + tid; t < p.num_tokens;
       t += int64_t(gridDim.x) * kPlanThreads)
    p.slots[t] = -1;  // padding behind the last request: paged_kv_write skips it
  if (blockIdx.x == 0) {
    int64_t v[3] = {beyond, 0, 0}, tot[3];
    block_scan3(v, tot, ws, warp, lane);
    if (tid == 0) {
      p.cu_q[p.nseq] = to_i32(base_q);
      p.cu_k[p.nseq] = to_i32(base_k);
      p.pages[0] = int(min(base_rank, int64_t(nfree)));
      p.pages[1] = to_i32(max(base_rank - nfree, int64_t(0)) + tot[0]);
    }
  }
}

// ---------------------------------------------------------------------------
// visibility bits of drafted trees
// ---------------------------------------------------------------------------
constexpr int kMaskThreads = 256;
constexpr int kMaxNodes = 4096;  // parents of one tree in shared memory (16 KB)

// One CTA per (request, share of its words); CTA nseq clears the rows before the first request and
// behind the last.  A tree whose bounds leave the rows is no tree: the rows between them are cleared.
// A thread owns one 64-bit word of one node and walks the node's ancestors in shared memory
// (parents come before children, so the walk descends and ends at the word's first bit).  1.8 us
// for 8 trees of 8 nodes (the launch), 4.5 us for 512 of 200 (the walks; 3.3 MB written).  A thread of
// each word walks the same ancestors, so a chain is the worst: one of 4096 nodes takes 432 us, 8 of
// 1024 84 us.
__global__ void __launch_bounds__(kMaskThreads)
    tree_mask_kernel(const int32_t* __restrict__ parents, const int32_t* __restrict__ cu, int nseq,
                     int64_t total, int max_nodes, int words, int64_t* __restrict__ mask) {
  extern __shared__ int s_par[];
  const int j = blockIdx.x;
  if (j == nseq) {
    const int64_t a = min(max(int64_t(cu[0]), int64_t(0)), total);
    const int64_t b = min(max(int64_t(cu[nseq]), a), total);
    const int64_t n = (a + total - b) * words;
    for (int64_t i = int64_t(blockIdx.y) * kMaskThreads + threadIdx.x; i < n;
         i += int64_t(gridDim.y) * kMaskThreads)
      mask[i < a * words ? i : i - a * words + b * words] = 0;
    return;
  }
  const int64_t a = cu[j], b = cu[j + 1];
  if (a < 0 || b > total) {
    const int64_t lo = max(a, int64_t(0)) * words, hi = min(b, total) * words;
    for (int64_t i = lo + int64_t(blockIdx.y) * kMaskThreads + threadIdx.x; i < hi;
         i += int64_t(gridDim.y) * kMaskThreads)
      mask[i] = 0;
    return;
  }
  if (b <= a) return;
  const int n = int(min(b - a, int64_t(max_nodes)));
  for (int i = threadIdx.x; i < n; i += kMaskThreads) {
    const int par = parents[a + i];
    s_par[i] = par < i ? par : -1;  // a later parent is none: the walk always ends
  }
  __syncthreads();
  for (int64_t u = int64_t(blockIdx.y) * kMaskThreads + threadIdx.x; u < (b - a) * words;
       u += int64_t(gridDim.y) * kMaskThreads) {
    const int i = int(u / words), lo = int(u - int64_t(i) * words) * 64;
    uint64_t bits = 0;
    for (int m = i < n ? i : -1; m >= lo; m = s_par[m])
      if (m < lo + 64) bits |= uint64_t(1) << (m - lo);
    mask[a * words + u] = int64_t(bits);
  }
}

// ---------------------------------------------------------------------------
// writes into the page pools
// ---------------------------------------------------------------------------
struct Pool {
  uint8_t* base;
  int64_t page, row, head;  // strides in bytes
};

struct WriteParams {
  const uint8_t *k, *v;
  int64_t k_stride, v_stride;  // bytes a token
  const float *k_descale, *v_descale;
  Pool kp, vp;
  const int64_t* slots;
  int64_t tokens, num_slots;
  int heads, per_head, page_size;  // per_head: 16-byte pieces of a head's source row
};

// The divisor of a head's values.  Every value needs the rounded quotient x / d, since e4m3 of
// x * (1 / d) would round twice; but the reciprocal is the same for all of them, and a quotient
// from a correctly rounded reciprocal needs one correction (P. Markstein, IBM J. Res. Dev. 34,
// 1990): q = x r, q + r (x - q d).  The remainder is a normal number, or 0, wherever the result
// is not 0 in e4m3, as long as |d| is between 2^-60 and 2^60; other divisors are brought there
// by a power of two, and the values by the same.  (A quotient costs three products, the
// division about ten instructions.)
struct Divisor {
  float d, r, scale;
};

__device__ __forceinline__ Divisor divisor(const float* descale, int head) {
  Divisor v;
  const float d = descale ? descale[head] : 1.f, a = fabsf(d);
  v.scale = a < 0x1p-60f ? 0x1p100f : a > 0x1p60f ? 0x1p-100f : 1.f;
  v.d = d * v.scale;
  v.r = __frcp_rn(v.d);
  if (isinf(d)) v.d = 1.f;  // r = 0: all quotients are 0, those of infinities NaN
  return v;
}

// Eight values, stored as eight bytes.
template <bool BF16>
__device__ __forceinline__ uint2 quant8(const uint4 a, const Divisor& d) {
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
  // with the signs of a product x (-1 / d), which keep that of a zero
  const uint64_t scale = f2pack(-d.scale, -d.scale), r = f2pack(-d.r, -d.r), dd = f2pack(d.d, d.d);
  float q[8], f[8], top[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint64_t x;
    if (BF16) {
      x = f2pack(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
    } else {
      const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x = f2pack(t.x, t.y);
    }
    x = fmul2(x, scale);
    const uint64_t y = fmul2(x, r);
    q[2 * i] = f2lo(y);
    q[2 * i + 1] = f2hi(y);
    const uint64_t c = ffma2(ffma2(y, dd, x), r, y);
    f[2 * i] = f2lo(c);
    f[2 * i + 1] = f2hi(c);
    top[i] = fmaxf(fabsf(q[2 * i]), fabsf(q[2 * i + 1]));
  }
  if (fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) > 4096.f) {
    // what saturates may be infinite, and leave no remainder to add
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = fabsf(q[i]) > 4096.f ? q[i] : f[i];
  }
  return make_uint2(pack_e4m3x4(f[0], f[1], f[2], f[3]), pack_e4m3x4(f[4], f[5], f[6], f[7]));
}

constexpr int kWriteThreads = 256, kWriteBlocks = 4, kWriteBatch = 2;

// A thread owns 16 bytes of the source row's columns, in K and in V, and takes a token out of
// every `gridDim.x` groups of them.  QUANT: 0 copy, 1 bf16 -> e4m3, 2 f16 -> e4m3.  Bound by
// memory: a row's loads do not wait for its slot, which decides on the store alone.  Measured:
// 65536 rows of 8 heads x 128, bf16 into e4m3, 71.5 us = 5.6 TB/s (62.4 us at the rate of a
// copy); loads marked as streaming 73.5 us, a thread a token instead of the loop 93 us, batches of
// 4 at 64 registers (spills) 86 us, at 80 registers (3 blocks) 77 us.  The same rows copied into a bf16
// pool: 93 us = 5.6 TB/s.  64 rows: 2 us, the launch.
template <int QUANT>
__global__ void __launch_bounds__(kWriteThreads, kWriteBlocks) kv_write_kernel(const WriteParams p) {
  const int cols = min(p.heads * p.per_head, kWriteThreads);  // of a block
  const int group = kWriteThreads / cols;                     // its tokens
  const int c = int(blockIdx.y) * cols + int(threadIdx.x) % cols;
  const int in_group = int(threadIdx.x) / cols;
  if (in_group >= group || c >= p.heads * p.per_head) return;
  const int head = c / p.per_head, x = c - head * p.per_head;
  const int64_t step = int64_t(gridDim.x) * group;
  constexpr int OUT = QUANT ? 8 : 16;
  const uint8_t *ks = p.k + int64_t(c) * 16, *vs = p.v + int64_t(c) * 16;
  uint8_t* kd = p.kp.base + head * p.kp.head + x * OUT;
  uint8_t* vd = p.vp.base + head * p.vp.head + x * OUT;
  Divisor dk, dv;
  if (QUANT) {
    dk = divisor(p.k_descale, head);
    dv = divisor(p.v_descale, head);
  }
  for (int64_t t0 = int64_t(blockIdx.x) * group + in_group; t0 < p.tokens; t0 += step * kWriteBatch) {
    uint4 k[kWriteBatch], v[kWriteBatch];
    int64_t slot[kWriteBatch];
#pragma unroll
    for (int i = 0; i < kWriteBatch; ++i) {
      const int64_t t = t0 + i * step;
      slot[i] = -1;
      if (t < p.tokens) {
        slot[i] = p.slots[t];
        k[i] = *reinterpret_cast<const uint4*>(ks + t * p.k_stride);
        v[i] = *reinterpret_cast<const uint4*>(vs + t * p.v_stride);
      }
    }
#pragma unroll
    for (int i = 0; i < kWriteBatch; ++i) {
      if (slot[i] < 0 || slot[i] >= p.num_slots) continue;
      int64_t page, row;
      if (p.num_slots < (int64_t(1) << 32)) {
        const uint32_t g = uint32_t(slot[i]) / uint32_t(p.page_size);
        page = g;
        row = uint32_t(slot[i]) - g * uint32_t(p.page_size);
      } else {
        page = slot[i] / p.page_size;
        row = slot[i] - page * p.page_size;
      }
      uint8_t* ko = kd + page * p.kp.page + row * p.kp.row;
      uint8_t* vo = vd + page * p.vp.page + row * p.vp.row;
      if (QUANT) {
        *reinterpret_cast<uint2*>(ko) = quant8<QUANT == 1>(k[i], dk);
        *reinterpret_cast<uint2*>(vo) = quant8<QUANT == 1>(v[i], dv);
      } else {
        *reinterpret_cast<uint4*>(ko) = k[i];
        *reinterpret_cast<uint4*>(vo) = v[i];
      }
    }
  }
}

// ---------------------------------------------------------------------------
// move of an accepted path's rows
// ---------------------------------------------------------------------------
constexpr int kAcceptThreads = 256;
constexpr int kMaxAccept = 1024;  // accepted nodes of one request (offsets in shared memory)

struct AcceptParams {
  Pool kp, vp;
  const int32_t *table, *cached, *cu, *accepted;
  int32_t* seq_lens;
  int num_pages, page_size, max_pages, max_accept, heads, per_head;  // per_head: 16-byte chunks
};

// CTA = (request, share of the row's 16-byte columns).  The moves (page and row that each comes
// from and goes to) are worked out once, a thread each; then a thread owns a column of K or of V
// through all of them.  The list ascends, so node a_i >= i: a batch of loads followed by its
// stores never overwrites a row that a later batch reads.  Bound by three dependent reads (list,
// table, rows) and, for many requests, by the rows: with the write of 12161 new rows 18 to 20 us for 256
// requests whose 12 rows move over an e4m3 cache (13.5 us of traffic); 26 us when every thread
// worked the moves out for itself.
__global__ void __launch_bounds__(kAcceptThreads) kv_accept_kernel(const AcceptParams p) {
  extern __shared__ int4 s_move[];  // [max_accept]: from (page, row), to (page, row); page -1: stays
  __shared__ int s_n;
  const int j = blockIdx.x, lane = threadIdx.x & 31;
  const int base = max(p.cached[j], 0);
  const int nodes = p.cu[j + 1] - p.cu[j];
  if (threadIdx.x < 32) {
    int n = 0, last = -1;
    for (int i0 = 0; i0 < p.max_accept; i0 += 32) {
      const int i = i0 + lane;
      const int a = i < p.max_accept ? p.accepted[int64_t(j) * p.max_accept + i] : -1;
      int before = __shfl_up_sync(0xffffffffu, a, 1);
      if (lane == 0) before = last;
      const bool good = a > before && a >= 0 && a < nodes;
      const unsigned bad = __ballot_sync(0xffffffffu, !good);
      const int run = bad ? __ffs(bad) - 1 : 32;
      if (lane < run) s_move[i].x = a;
      n += run;
      if (run < 32) break;
      last = __shfl_sync(0xffffffffu, a, 31);
    }
    if (lane == 0) {
      s_n = n;
      if (blockIdx.y == 0) p.seq_lens[j] = base + n;
    }
  }
  __syncthreads();
  const int n = s_n;
  const int32_t* table = p.table + int64_t(j) * p.max_pages;
  for (int i = threadIdx.x; i < n; i += kAcceptThreads) {
    const int a = s_move[i].x;
    auto place = [&](int node, int& page, int& row) {
      const unsigned pos = unsigned(base) + unsigned(node);  // below 2^32
      const unsigned e = pos / unsigned(p.page_size);
      page = e < unsigned(p.max_pages) ? table[e] : -1;
      row = int(pos - e * unsigned(p.page_size));
      if (page >= p.num_pages) page = -1;
    };
    int4 m;
    place(a, m.x, m.y);
    place(i, m.z, m.w);
    if (a == i || m.x < 0 || m.z < 0) m.x = -1;
    s_move[i] = m;
  }
  __syncthreads();
  const int cols = p.heads * p.per_head;
  for (int u = blockIdx.y * kAcceptThreads + threadIdx.x; u < 2 * cols; u += gridDim.y * kAcceptThreads) {
    const Pool pool = u < cols ? p.kp : p.vp;
    const int c = u < cols ? u : u - cols;
    const int head = c / p.per_head;
    uint8_t* col = pool.base + head * pool.head + int64_t(c - head * p.per_head) * 16;
    for (int i0 = 0; i0 < n; i0 += 8) {
      uint4 x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i0 + i >= n) break;
        const int4 m = s_move[i0 + i];
        if (m.x >= 0) x[i] = *reinterpret_cast<const uint4*>(col + m.x * pool.page + m.y * pool.row);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i0 + i >= n) break;
        const int4 m = s_move[i0 + i];
        if (m.x >= 0) *reinterpret_cast<uint4*>(col + m.z * pool.page + m.w * pool.row) = x[i];
      }
    }
  }
}

int check_pool(const char* what, const void* base, int64_t page, int64_t row, int64_t head, int el) {
  FA4CP_CHECK_ARG(base != nullptr, "%s: null pool", what);
  FA4CP_CHECK_ARG((reinterpret_cast<uintptr_t>(base) & 15u) == 0 && page * el % 16 == 0 &&
                      row * el % 16 == 0 && head * el % 16 == 0,
                  "%s: pool pointer and strides must be 16-byte aligned", what);
  return FA4CP_OK;
}

}  // namespace
}  // namespace fa4cp

using namespace fa4cp;

extern "C" int fa4cp_paged_block_tables(const int32_t* cached_lens, const int32_t* new_lens,
                                        int32_t nseq, const int32_t* free_pages, int32_t num_free,
                                        const int32_t* num_free_device, int32_t page_size,
                                        int32_t max_pages, const int32_t* table_in,
                                        int32_t* table_out, int64_t* slot_mapping,
                                        int64_t num_tokens, int32_t* cu_q, int32_t* cu_k,
                                        int32_t* seq_lens, int32_t* pages, void* stream) {
  FA4CP_CHECK_ARG(nseq >= 1 && nseq < (1 << 24), "nseq must be in [1, 2^24)");
  FA4CP_CHECK_ARG(page_size >= 1, "page_size must be positive");
  FA4CP_CHECK_ARG(max_pages >= 1 && num_free >= 0 && num_tokens >= 0, "bad sizes");
  FA4CP_CHECK_ARG(cached_lens && new_lens && table_out && cu_q && cu_k && seq_lens && pages &&
                      (num_free == 0 || free_pages) && (num_tokens == 0 || slot_mapping),
                  "null tensor pointer");
  FA4CP_CHECK_ARG(table_in != table_out, "the new table must not be the old one");
  PlanParams p{};
  p.cached = cached_lens;
  p.fresh = new_lens;
  p.free_pages = free_pages;
  p.num_free_dev = num_free_device;
  p.table_in = table_in;
  p.table_out = table_out;
  p.cu_q = cu_q;
  p.cu_k = cu_k;
  p.seq_lens = seq_lens;
  p.pages = pages;
  p.slots = slot_mapping;
  p.num_tokens = num_tokens;
  p.nseq = nseq;
  p.num_free = num_free;
  p.page_size = page_size;
  p.max_pages = max_pages;
  // enough CTAs for about two table entries and one slot a thread
  const int64_t want = (int64_t(nseq) * max_pages / 2 + num_tokens) / kPlanThreads + 1;
  const int grid = int(want < kMaxGrid ? want : kMaxGrid);
  plan_kernel<<<grid, kPlanThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
  return check_launch("paged_block_tables");
}

extern "C" int fa4cp_paged_tree_mask(const int32_t* parents, const int32_t* cu_q, int32_t nseq,
                                     int64_t total_q, int32_t max_nodes, int64_t* mask,
                                     void* stream) {
  FA4CP_CHECK_ARG(nseq >= 1 && cu_q != nullptr, "cu_seqlens_q must describe >= 1 request");
  FA4CP_CHECK_ARG(max_nodes >= 1 && max_nodes <= kMaxNodes, "max_nodes must be in [1, %d]", kMaxNodes);
  FA4CP_CHECK_ARG(total_q >= 0, "bad sizes");
  if (total_q == 0) return FA4CP_OK;
  FA4CP_CHECK_ARG(parents && mask, "null tensor pointer");
  const int words = (max_nodes + 63) / 64;
  const int64_t want = (int64_t(max_nodes) * words + 4 * kMaskThreads - 1) / (4 * kMaskThreads);
  const dim3 grid(unsigned(nseq) + 1u, unsigned(want));
  tree_mask_kernel<<<grid, kMaskThreads, size_t(max_nodes) * 4, static_cast<cudaStream_t>(stream)>>>(
      parents, cu_q, nseq, total_q, max_nodes, words, mask);
  return check_launch("paged_tree_mask");
}

extern "C" int fa4cp_paged_kv_write(const void* k, const void* v, int64_t k_token_stride,
                                    int64_t v_token_stride, void* k_pages, void* v_pages,
                                    const int64_t* k_strides, const int64_t* v_strides,
                                    int64_t num_pages, int32_t page_size,
                                    const int64_t* slot_mapping, int64_t num_tokens,
                                    int32_t num_heads_kv, int32_t head_dim, int32_t src_dtype,
                                    int32_t pool_dtype, const float* k_descale,
                                    const float* v_descale, void* stream) {
  FA4CP_CHECK_ARG(num_tokens >= 0 && num_pages >= 0 && page_size >= 1 && num_heads_kv >= 1 &&
                      head_dim >= 1, "bad sizes");
  const int se = elem_bytes(src_dtype), pe = elem_bytes(pool_dtype);
  const bool quant = pool_dtype == FA4CP_DTYPE_E4M3 && src_dtype != FA4CP_DTYPE_E4M3;
  FA4CP_CHECK_ARG((src_dtype == pool_dtype && se >= 1 && se <= 2) ||
                      (quant && (src_dtype == FA4CP_DTYPE_BF16 || src_dtype == FA4CP_DTYPE_F16)),
                  "k/v dtype %d cannot be written into a pool of dtype %d", src_dtype, pool_dtype);
  FA4CP_CHECK_ARG(quant || (!k_descale && !v_descale),
                  "descales apply to f16 / bf16 rows written into an e4m3 pool only");
  FA4CP_CHECK_ARG(head_dim * pe % 16 == 0, "a head's row must be a multiple of 16 bytes");
  if (num_tokens == 0 || num_pages == 0) return FA4CP_OK;
  FA4CP_CHECK_ARG(k && v && slot_mapping && k_strides && v_strides, "null tensor pointer");
  FA4CP_CHECK_ARG((reinterpret_cast<uintptr_t>(k) & 15u) == 0 && (reinterpret_cast<uintptr_t>(v) & 15u) == 0 &&
                      k_token_stride * se % 16 == 0 && v_token_stride * se % 16 == 0,
                  "k and v rows must be 16-byte aligned");
  if (int rc = check_pool("k_pages", k_pages, k_strides[0], k_strides[1], k_strides[2], pe)) return rc;
  if (int rc = check_pool("v_pages", v_pages, v_strides[0], v_strides[1], v_strides[2], pe)) return rc;
  WriteParams p{};
  p.k = static_cast<const uint8_t*>(k);
  p.v = static_cast<const uint8_t*>(v);
  p.k_stride = k_token_stride * se;
  p.v_stride = v_token_stride * se;
  p.k_descale = k_descale;
  p.v_descale = v_descale;
  p.kp = Pool{static_cast<uint8_t*>(k_pages), k_strides[0] * pe, k_strides[1] * pe, k_strides[2] * pe};
  p.vp = Pool{static_cast<uint8_t*>(v_pages), v_strides[0] * pe, v_strides[1] * pe, v_strides[2] * pe};
  p.slots = slot_mapping;
  p.tokens = num_tokens;
  p.num_slots = num_pages * page_size;
  p.heads = num_heads_kv;
  p.per_head = head_dim * se / 16;
  p.page_size = page_size;
  const int64_t columns = int64_t(num_heads_kv) * p.per_head;
  FA4CP_CHECK_ARG(columns < (int64_t(1) << 23), "rows of %lld bytes are too long", (long long)columns * 16);
  const int cols = int(columns < kWriteThreads ? columns : kWriteThreads);
  const int64_t groups = (num_tokens + kWriteThreads / cols - 1) / (kWriteThreads / cols);
  const int64_t parts = (columns + cols - 1) / cols;
  // a token a thread while that fills the SMs; beyond it, as many blocks as are resident, since
  // what a thread works out once (its head, the divisor) then serves many tokens
  const int64_t most = (kMaxGrid * kWriteBlocks + parts - 1) / parts;
  const dim3 grid(unsigned(groups < most ? groups : most), unsigned(parts));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (!quant) kv_write_kernel<0><<<grid, kWriteThreads, 0, st>>>(p);
  else if (src_dtype == FA4CP_DTYPE_BF16) kv_write_kernel<1><<<grid, kWriteThreads, 0, st>>>(p);
  else kv_write_kernel<2><<<grid, kWriteThreads, 0, st>>>(p);
  return check_launch("paged_kv_write");
}

extern "C" int fa4cp_paged_kv_accept(void* k_pages, void* v_pages, const int64_t* k_strides,
                                     const int64_t* v_strides, int32_t num_pages,
                                     int32_t page_size, const int32_t* block_table,
                                     int32_t max_pages, const int32_t* cached_lens,
                                     const int32_t* cu_q, int32_t nseq, const int32_t* accepted,
                                     int32_t max_accept, int32_t num_heads_kv, int32_t head_dim,
                                     int32_t dtype, int32_t* seq_lens, void* stream) {
  FA4CP_CHECK_ARG(nseq >= 1, "nseq must be positive");
  FA4CP_CHECK_ARG(num_pages >= 0 && page_size >= 1 && max_pages >= 1 && num_heads_kv >= 1 && head_dim >= 1,
                  "bad sizes");
  FA4CP_CHECK_ARG(max_accept >= 0 && max_accept <= kMaxAccept, "max_accept must be in [0, %d]", kMaxAccept);
  const int pe = elem_bytes(dtype);
  FA4CP_CHECK_ARG(pe == 1 || pe == 2, "pool dtype must be f16, bf16 or e4m3");
  FA4CP_CHECK_ARG(head_dim * pe % 16 == 0, "a head's row must be a multiple of 16 bytes");
  FA4CP_CHECK_ARG(block_table && cached_lens && cu_q && seq_lens && k_strides && v_strides &&
                      (max_accept == 0 || accepted), "null tensor pointer");
  if (num_pages > 0) {
    if (int rc = check_pool("k_pages", k_pages, k_strides[0], k_strides[1], k_strides[2], pe)) return rc;
    if (int rc = check_pool("v_pages", v_pages, v_strides[0], v_strides[1], v_strides[2], pe)) return rc;
  }
  AcceptParams p{};
  p.kp = Pool{static_cast<uint8_t*>(k_pages), k_strides[0] * pe, k_strides[1] * pe, k_strides[2] * pe};
  p.vp = Pool{static_cast<uint8_t*>(v_pages), v_strides[0] * pe, v_strides[1] * pe, v_strides[2] * pe};
  p.table = block_table;
  p.cached = cached_lens;
  p.cu = cu_q;
  p.accepted = accepted;
  p.seq_lens = seq_lens;
  p.num_pages = num_pages;
  p.page_size = page_size;
  p.max_pages = max_pages;
  p.max_accept = max_accept;
  p.heads = num_heads_kv;
  p.per_head = head_dim * pe / 16;
  const int64_t cols = int64_t(2) * p.heads * p.per_head;
  const int64_t want = (cols + kAcceptThreads - 1) / kAcceptThreads;
  const dim3 grid(unsigned(nseq), unsigned(want < 64 ? want : 64));
  kv_accept_kernel<<<grid, kAcceptThreads, size_t(max_accept > 0 ? max_accept : 1) * 16,
                     static_cast<cudaStream_t>(stream)>>>(p);
  return check_launch("paged_kv_accept");
}
