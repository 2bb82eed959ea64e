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
// re-reading 8 bytes a request per CTA from L2.
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

// One CTA per (request, share of its words); CTA nseq clears the rows outside every request.
// A thread owns one 64-bit word of one node and walks the node's ancestors in shared memory
// (parents come before children, so the walk descends and ends at the word's first bit).
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
  if (a < 0 || b > total || b <= a) return;
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
  int heads, per_head, page_size;  // per_head: 16-byte chunks of a stored head row
};

template <bool BF16>
__device__ __forceinline__ uint4 quant16(const uint4 a, const uint4 b, float d) {
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float f[4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t x = w[2 * i + h];
      if (BF16) {
        f[2 * h] = __uint_as_float(x << 16);
        f[2 * h + 1] = __uint_as_float(x & 0xFFFF0000u);
      } else {
        const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&x));
        f[2 * h] = t.x;
        f[2 * h + 1] = t.y;
      }
    }
    // one rounding, of the quotient: a multiplication by 1 / d would round twice
    o[i] = pack_e4m3x4(__fdiv_rn(f[0], d), __fdiv_rn(f[1], d), __fdiv_rn(f[2], d), __fdiv_rn(f[3], d));
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// One thread per 16 bytes stored in K and in V.  QUANT: 0 copy, 1 bf16 -> e4m3, 2 f16 -> e4m3.
template <int QUANT>
__global__ void __launch_bounds__(256) kv_write_kernel(const WriteParams p) {
  const unsigned per_head = unsigned(p.per_head);
  const unsigned per_row = per_head * unsigned(p.heads);
  const int64_t n = p.tokens * per_row;
  for (int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; i < n;
       i += int64_t(gridDim.x) * blockDim.x) {
    const int64_t t = n < (int64_t(1) << 32) ? int64_t(uint32_t(i) / per_row) : i / per_row;
    const unsigned c = unsigned(i - t * per_row);
    const int64_t slot = p.slots[t];
    if (slot < 0 || slot >= p.num_slots) continue;
    const unsigned head = c / per_head, x = c - head * per_head;
    const int64_t page = slot / p.page_size, row = slot - page * p.page_size;
    const uint8_t* ks = p.k + t * p.k_stride + int64_t(c) * (QUANT ? 32 : 16);
    const uint8_t* vs = p.v + t * p.v_stride + int64_t(c) * (QUANT ? 32 : 16);
    uint4 ko, vo;
    if (QUANT) {
      const uint4 k0 = __ldcs(reinterpret_cast<const uint4*>(ks)), k1 = __ldcs(reinterpret_cast<const uint4*>(ks) + 1);
      const uint4 v0 = __ldcs(reinterpret_cast<const uint4*>(vs)), v1 = __ldcs(reinterpret_cast<const uint4*>(vs) + 1);
      ko = quant16<QUANT == 1>(k0, k1, p.k_descale ? p.k_descale[head] : 1.f);
      vo = quant16<QUANT == 1>(v0, v1, p.v_descale ? p.v_descale[head] : 1.f);
    } else {
      ko = __ldcs(reinterpret_cast<const uint4*>(ks));
      vo = __ldcs(reinterpret_cast<const uint4*>(vs));
    }
    *reinterpret_cast<uint4*>(p.kp.base + page * p.kp.page + row * p.kp.row + head * p.kp.head + x * 16) = ko;
    *reinterpret_cast<uint4*>(p.vp.base + page * p.vp.page + row * p.vp.row + head * p.vp.head + x * 16) = vo;
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

// CTA = (request, share of the row's 16-byte columns).  A thread owns a column of K or of V
// through all moved rows.  The list ascends, so node a_i >= i: a batch of loads followed by
// its stores never overwrites a row that a later batch reads.
__global__ void __launch_bounds__(kAcceptThreads) kv_accept_kernel(const AcceptParams p) {
  extern __shared__ int s_pos[];  // [max_accept]: node, or -1 where nothing moves
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
      if (lane < run) s_pos[i] = a;
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
  const int cols = p.heads * p.per_head;
  const int32_t* row = p.table + int64_t(j) * p.max_pages;
  auto offset = [&](const Pool& pool, int node, int64_t& off) -> bool {
    const int64_t pos = int64_t(base) + node;
    const int64_t e = pos / p.page_size;
    if (e >= p.max_pages) return false;
    const int page = row[e];
    if (page < 0 || page >= p.num_pages) return false;
    off = int64_t(page) * pool.page + (pos - e * p.page_size) * pool.row;
    return true;
  };
  for (int u = blockIdx.y * kAcceptThreads + threadIdx.x; u < 2 * cols; u += gridDim.y * kAcceptThreads) {
    const Pool pool = u < cols ? p.kp : p.vp;
    const int c = u < cols ? u : u - cols;
    const int head = c / p.per_head;
    uint8_t* col = pool.base + head * pool.head + int64_t(c - head * p.per_head) * 16;
    for (int i0 = 0; i0 < n; i0 += 8) {
      uint4 x[8];
      bool ok[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        int64_t off = 0;
        ok[i] = i0 + i < n && s_pos[i0 + i] != i0 + i && offset(pool, s_pos[i0 + i], off);
        if (ok[i]) x[i] = *reinterpret_cast<const uint4*>(col + off);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        int64_t off = 0;
        if (ok[i] && offset(pool, i0 + i, off)) *reinterpret_cast<uint4*>(col + off) = x[i];
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
  p.per_head = head_dim * pe / 16;
  p.page_size = page_size;
  const int64_t n = num_tokens * num_heads_kv * p.per_head;
  const int64_t blocks = (n + 255) / 256;
  const unsigned grid = unsigned(blocks < (int64_t(1) << 30) ? blocks : (int64_t(1) << 30));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (!quant) kv_write_kernel<0><<<grid, 256, 0, st>>>(p);
  else if (src_dtype == FA4CP_DTYPE_BF16) kv_write_kernel<1><<<grid, 256, 0, st>>>(p);
  else kv_write_kernel<2><<<grid, 256, 0, st>>>(p);
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
  if (int rc = check_pool("k_pages", k_pages, k_strides[0], k_strides[1], k_strides[2], pe)) return rc;
  if (int rc = check_pool("v_pages", v_pages, v_strides[0], v_strides[1], v_strides[2], pe)) return rc;
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
  kv_accept_kernel<<<grid, kAcceptThreads, size_t(max_accept > 0 ? max_accept : 1) * 4,
                     static_cast<cudaStream_t>(stream)>>>(p);
  return check_launch("paged_kv_accept");
}
