// Attention of drafted tokens over a paged K/V cache (single-token decode is the tree of one
// node).  No counterpart in the reference, whose K/V is contiguous (README.md:139-141).
//
//   O[i] = sum_k softmax_k(scale q_i . K[k]) V[k],  k < ctx, or k one of the request's own new
//   rows that the tree's bits of token i name (ctx = seq_len - n, n new tokens).
//
// The query heads of one K/V head read the same keys, so a request's n tokens x `group` heads
// are packed into rows of one 128-row MMA tile (row = token * group + head of the group), and
// K and V are read once for all of them.  A step is bound by those reads until a request has
// about 250 rows (bf16).
//
// Schedule.  The work is the list of all (request, K/V head, row tile, key tile), in that
// order; every CTA takes an equal share of consecutive key tiles, whatever the lengths are
// (they are only known on the device).  A row tile whose keys several CTAs share leaves one
// partial (O, m, l) each in the workspace, joined by tree_combine_kernel in a fixed order.  A
// CTA has at most two partials (its first and its last row tile), so the workspace does not
// depend on the lengths.
//
// CTA roles (one CTA per SM):
//   warps 0-3  softmax + epilogue, thread t owns row t = TMEM lane t; they load Q, too
//   warp  4    TMA producer: K_0, V_0, K_1, ... into one ring of tiles, a page piece a lane
//   warp  5    TMEM allocator + MMA issuer (one thread)
//   warps 8-15 e4m3 cache only: tiles from the raw ring, widened to f16 into the operand ring
// TMEM: S0 | S1 (BN fp32 columns each) | O (D columns) | Q (D/2 columns of 16-bit pairs).
// Q is the A operand of S = Q K^T straight from TMEM: the shared memory that it would take
// holds K/V tiles in flight instead, and the MMA reads K alone from there.
// MMA order: S0, S1, PV0, S2, PV1, ...; P overwrites its S buffer as in attn_fwd_kernel.
#include <atomic>

#include "common.cuh"

namespace fa4cp {

__device__ int g_tree_status = 0;

int tree_status(int* value, bool clear) {
  FA4CP_CHECK_CUDA(cudaMemcpyFromSymbol(value, g_tree_status, sizeof(int)));
  if (clear) {
    const int z = 0;
    FA4CP_CHECK_CUDA(cudaMemcpyToSymbol(g_tree_status, &z, sizeof(int)));
  }
  return FA4CP_OK;
}

namespace {

constexpr float kNegInf = -__builtin_huge_valf();
constexpr float kRescaleThreshold = 8.0f;  // log2 units: P <= 256
constexpr int BM = 128;

// codes written to the device status word when a bounded wait gives up
enum : int {
  kErrEmpty = 0x401, kErrRawEmpty, kErrRawFull, kErrOpEmpty, kErrQFull, kErrKFull, kErrPFull,
  kErrVFull, kErrOFree, kErrSFull, kErrODone, kErrVFix, kErrDrain
};

struct TreeParams {
  const uint8_t *q, *v;
  int64_t q_stride;               // bytes a token
  int64_t v_page, v_row, v_head;  // strides in bytes (the non-finite pass reads V itself)
  const int32_t *block_table, *cu_q, *seq_lens;
  const uint32_t* mask;  // [total_q, mask_words] 32-bit words, or nullptr: causal
  void* out;
  float* lse;
  const float *q_descale, *k_descale, *v_descale;
  float* part_o;   // [2 * grid][BM][D]
  float2* part_ml; // [2 * grid][BM]: running maximum (log2 units, scaled), sum
  int4* desc;      // [grid][2]: the row tile whose first part a CTA holds
  int64_t total_q;
  int nseq, Hq, Hkv, group, page_size, num_pages, max_pages, mask_words;
  int q_dtype, kv_dtype, out_bf16;
  float scale_log2;
};

template <int D_, int BN_, bool KV8_>
struct TreeTraits {
  static constexpr int D = D_, BN = BN_;
  static constexpr bool KV8 = KV8_;
  static constexpr int NCH = D / 64;                // 128-byte columns of an operand tile
  static constexpr int TILE_BYTES = BN * D * 2;     // one operand tile (K or V)
  static constexpr int CHUNK_BYTES = BN * 128;
  static constexpr int RAW_BYTES = BN * D;          // one e4m3 tile
  static constexpr int RAW_SLOTS = KV8 ? (D == 64 ? 8 : 6) : 0;
  static constexpr int SLOTS = KV8 ? (D == 64 ? 6 : 4) : (D == 64 ? 12 : 7);
  static constexpr int OFF_RAW = SLOTS * TILE_BYTES;
  static constexpr int OFF_BAR = OFF_RAW + RAW_SLOTS * RAW_BYTES;
  // op_full, op_empty [SLOTS]; raw_full, raw_empty [RAW_SLOTS]; s_full[2], p_full[2],
  // o_done[2], q_full, o_free, v_fixed, teardown
  static constexpr int NUM_BARS = 2 * SLOTS + 2 * RAW_SLOTS + 10;
  static constexpr int OFF_MISC = OFF_BAR + NUM_BARS * 8;
  static constexpr int SMEM_BYTES = OFF_MISC + 128 + 1024;
  static constexpr int THREADS = KV8 ? 512 : 192;
  static constexpr int CONV_WARPS = 8;
  static constexpr int TM_S = 0, TM_O = 2 * BN, TM_Q = TM_O + D;
  static_assert(TM_Q + D / 2 <= 512, "TMEM budget");
  static_assert(SMEM_BYTES <= 232448, "shared memory budget");
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void* tmap, int c0, int c1, int c2,
                                            int c3, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void fence_async_shared() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// ---------------------------------------------------------------------------
// schedule
// ---------------------------------------------------------------------------
// One request as the schedule sees it: its rows and key tiles.  Boundaries outside
// [0, total_q] and empty requests give no work; an empty cache gives one tile, all masked, so
// that its rows are written.
struct Request {
  int token0, n, len, mt, kt;  // first token, tokens, cached rows, row tiles, key tiles
};

template <int BN>
__device__ __forceinline__ Request load_request(const TreeParams& p, int j) {
  Request r;
  const int a = p.cu_q[j], b = p.cu_q[j + 1];
  r.token0 = a;
  r.n = (a >= 0 && b > a && b <= p.total_q) ? b - a : 0;
  r.len = max(p.seq_lens[j], 0);
  r.mt = int((int64_t(r.n) * p.group + BM - 1) / BM);
  r.kt = max(int((int64_t(r.len) + BN - 1) / BN), 1);
  return r;
}

// The share of key tiles [t0, t1) of CTA c out of G, and the item that t0 falls into.
struct Share {
  int64_t t0, t1, total;
  int64_t off;  // t0 relative to its request's first tile
  int seq;
};

// All threads of the CTA.  A thread sums a run of requests, a block scan gives its run's first
// tile, and the thread whose run holds t0 finds the request.
template <int BN>
__device__ __forceinline__ Share find_share(const TreeParams& p, int c, int G, int64_t* ws,
                                            int64_t* found) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = blockDim.x >> 5;
  const int per = (p.nseq + int(blockDim.x) - 1) / int(blockDim.x);
  const int j0 = min(tid * per, p.nseq), j1 = min(j0 + per, p.nseq);
  int64_t sum = 0;
  for (int j = j0; j < j1; ++j) {
    const Request r = load_request<BN>(p, j);
    sum += int64_t(p.Hkv) * r.mt * r.kt;
  }
  int64_t inc = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t o = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += o;
  }
  if (lane == 31) ws[warp] = inc;
  __syncthreads();
  int64_t before = 0, total = 0;
  for (int w = 0; w < nw; ++w) {
    if (w < warp) before += ws[w];
    total += ws[w];
  }
  Share s;
  s.total = total;
  const int64_t g = min(int64_t(G), total);  // no CTA has an empty share between others
  s.t0 = c < g ? total * c / g : total;
  s.t1 = c < g ? total * (c + 1) / g : total;
  int64_t first = before + inc - sum;
  if (s.t0 < s.t1 && first <= s.t0 && s.t0 < first + sum) {
    for (int j = j0; j < j1; ++j) {
      const Request r = load_request<BN>(p, j);
      const int64_t tiles = int64_t(p.Hkv) * r.mt * r.kt;
      if (s.t0 < first + tiles) {
        found[0] = j;
        found[1] = s.t0 - first;
        break;
      }
      first += tiles;
    }
  }
  __syncthreads();
  s.seq = int(found[0]);
  s.off = found[1];
  return s;
}

// Walks a CTA's share item by item; every role runs its own copy.
template <int BN>
struct Walk {
  Request r;
  int64_t off, left;
  int seq, kvh, mtile, kt0, nt;  // the current item's K/V head, row tile, first tile, tiles
  __device__ __forceinline__ void start(const TreeParams& p, const Share& s) {
    seq = s.seq;
    off = s.off;
    left = s.t1 - s.t0;
    r = load_request<BN>(p, seq);
    set(p);
  }
  __device__ __forceinline__ void set(const TreeParams&) {
    const int64_t item = off / r.kt;
    kt0 = int(off - item * r.kt);
    kvh = int(item / r.mt);
    mtile = int(item - int64_t(kvh) * r.mt);
    nt = int(min(int64_t(r.kt - kt0), left));
  }
  // to the next item; false at the end of the share
  __device__ __forceinline__ bool next(const TreeParams& p) {
    left -= nt;
    if (left <= 0) return false;
    off += nt;
    if (off >= int64_t(p.Hkv) * r.mt * r.kt) {
      off = 0;
      do {
        r = load_request<BN>(p, ++seq);
      } while (r.n == 0 && seq + 1 < p.nseq);
    }
    set(p);
    return true;
  }
  __device__ __forceinline__ int rows(const TreeParams& p) const {
    return min(BM, r.n * p.group - mtile * BM);
  }
};

// ---------------------------------------------------------------------------
// masks
// ---------------------------------------------------------------------------
// 32 visibility bits of row-token `node` (global token `tok`) for keys [key, key + 32).
__device__ __forceinline__ uint32_t seen32(const TreeParams& p, const Request& r, int64_t tok,
                                           int node, int key) {
  if (key >= r.len) return 0u;
  uint32_t inside = r.len - key >= 32 ? 0xffffffffu : (1u << (r.len - key)) - 1u;
  const int d = key - (r.len - r.n);  // the keys' index among the new rows
  if (d + 31 < 0) return inside;
  uint32_t bits;
  if (p.mask == nullptr) {
    const int last = node - d;  // keys up to the token's own
    bits = last < 0 ? 0u : last >= 31 ? 0xffffffffu : (2u << last) - 1u;
  } else {
    const uint32_t* row = p.mask + tok * p.mask_words;
    const int s = max(d, 0), w = s >> 5;
    const uint32_t lo = w < p.mask_words ? row[w] : 0u;
    const uint32_t hi = w + 1 < p.mask_words ? row[w + 1] : 0u;
    bits = __funnelshift_r(lo, hi, s & 31);
    if (d < 0) bits = (bits << -d) | ((1u << -d) - 1u);  // keys before the new rows
  }
  return bits & inside;
}

__device__ __forceinline__ bool nonfinite16(uint32_t h, bool bf16) {
  const uint32_t e = bf16 ? 0x7F80u : 0x7C00u;
  return (h & e) == e;
}

__device__ __forceinline__ float value16(uint32_t h, bool bf16) {
  if (bf16) return __uint_as_float(h << 16);
  const uint16_t u = uint16_t(h);
  return __half2float(*reinterpret_cast<const __half*>(&u));
}

// ---------------------------------------------------------------------------
// the kernel
// ---------------------------------------------------------------------------
// One 64-element piece of a query row as 32 registers of 16-bit pairs in the operand type.
// f16 operands of an e4m3 cache: x * f with f a power of two (exact unless f16 underflows).
template <bool KV8>
__device__ __forceinline__ void load_q64(const TreeParams& p, const uint8_t* row, int c, float f,
                                         uint32_t (&r)[32]) {
  if (!KV8) {
    const uint4* src = reinterpret_cast<const uint4*>(row + c * 128);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint4 x = src[i];
      r[4 * i] = x.x; r[4 * i + 1] = x.y; r[4 * i + 2] = x.z; r[4 * i + 3] = x.w;
    }
  } else if (p.q_dtype == FA4CP_DTYPE_E4M3) {
    const uint4* src = reinterpret_cast<const uint4*>(row + c * 64);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 x = src[i];
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float a, b, cc, d;
        unpack_e4m3x4(w[k], a, b, cc, d);
        r[8 * i + 2 * k] = pack_f16x2(a * f, b * f);
        r[8 * i + 2 * k + 1] = pack_f16x2(cc * f, d * f);
      }
    }
  } else {
    const bool bf = p.q_dtype == FA4CP_DTYPE_BF16;
    const uint4* src = reinterpret_cast<const uint4*>(row + c * 128);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint4 x = src[i];
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int k = 0; k < 4; ++k)
        r[4 * i + k] = pack_f16x2(value16(w[k] & 0xFFFFu, bf) * f, value16(w[k] >> 16, bf) * f);
    }
  }
}

// Largest magnitude of a query row (e4m3 cache: the row is brought to f16 by a power of two).
template <int D>
__device__ __forceinline__ float q_absmax(const TreeParams& p, const uint8_t* row) {
  float m = 0.f;
  if (p.q_dtype == FA4CP_DTYPE_E4M3) return 448.f;
  const bool bf = p.q_dtype == FA4CP_DTYPE_BF16;
  const uint4* src = reinterpret_cast<const uint4*>(row);
#pragma unroll 8
  for (int i = 0; i < D / 8; ++i) {
    const uint4 x = src[i];
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int k = 0; k < 4; ++k)
      m = fmaxf(m, fmaxf(fabsf(value16(w[k] & 0xFFFFu, bf)), fabsf(value16(w[k] >> 16, bf))));
  }
  return m;
}

// Rows that see a key whose V row is not finite, after the finite part has been written to
// dst: the non-finite values themselves are added (their weight is positive).  Rare; reads V
// again from the pool.
template <int D, class Store>
__device__ __noinline__ void add_nonfinite(const TreeParams& p, const Request& r, int seq, int kvh,
                                           int64_t tok, int node, int key0, int key1, Store dst) {
  const int ctx = max(r.len - r.n, 0);
  for (int key = max(key0, ctx); key < min(key1, r.len); ++key) {
    if (!(seen32(p, r, tok, node, key) & 1u)) continue;
    const int e = key / p.page_size;
    const int page = e < p.max_pages ? p.block_table[int64_t(seq) * p.max_pages + e] : -1;
    if (page < 0 || page >= p.num_pages) continue;
    const uint8_t* row = p.v + page * p.v_page + (key - e * p.page_size) * p.v_row + kvh * p.v_head;
    for (int d = 0; d < D; ++d) {
      float x;
      if (p.kv_dtype == FA4CP_DTYPE_E4M3) {
        if ((row[d] & 0x7F) != 0x7F) continue;
        x = __uint_as_float(0x7FC00000u);
      } else {
        const uint32_t h = reinterpret_cast<const uint16_t*>(row)[d];
        const bool bf = p.kv_dtype == FA4CP_DTYPE_BF16;
        if (!nonfinite16(h, bf)) continue;
        x = value16(h, bf);
      }
      dst.add(d, x);
    }
  }
}

struct AddF32 {
  float* row;
  __device__ __forceinline__ void add(int d, float x) const { row[d] += x; }
};
struct Add16 {
  uint16_t* row;
  int bf16;
  __device__ __forceinline__ void add(int d, float x) const {
    const float y = value16(row[d], bf16) + x;
    row[d] = uint16_t(bf16 ? pack_bf16x2(y, 0.f) : pack_f16x2(y, 0.f));
  }
};

template <class TR>
__global__ void __launch_bounds__(TR::THREADS, 1)
    tree_attn_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                     const TreeParams p) {
  constexpr int D = TR::D, BN = TR::BN, NS = TR::SLOTS, NR = TR::KV8 ? TR::RAW_SLOTS : 1;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cta = int(blockIdx.x), G = int(gridDim.x);

  // the schedule's scratch lies where the ring will be (no copy is in flight yet)
  int64_t* sched = reinterpret_cast<int64_t*>(smem);
  const Share share = find_share<BN>(p, cta, G, sched, sched + 32);
  if (share.t0 >= share.t1) {  // uniform for the CTA
    if (threadIdx.x == 0) p.desc[2 * cta] = make_int4(0, 0, 0, 0);
    return;
  }

  const uint32_t bar0 = smem_u32(smem + TR::OFF_BAR);
  auto BAR = [&](int i) -> uint32_t { return bar0 + 8u * uint32_t(i); };
  auto op_full = [&](int s) { return BAR(s); };
  auto op_empty = [&](int s) { return BAR(NS + s); };
  auto raw_full = [&](int s) { return BAR(2 * NS + s); };
  auto raw_empty = [&](int s) { return BAR(2 * NS + TR::RAW_SLOTS + s); };
  constexpr int B1 = 2 * TR::SLOTS + 2 * TR::RAW_SLOTS;
  auto s_full = [&](int b) { return BAR(B1 + b); };
  auto p_full = [&](int b) { return BAR(B1 + 2 + b); };
  auto o_done = [&](int b) { return BAR(B1 + 4 + b); };
  const uint32_t q_full = BAR(B1 + 6), o_free = BAR(B1 + 7), v_fixed = BAR(B1 + 8),
                 td_bar = BAR(B1 + 9);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + TR::OFF_MISC);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile uint32_t* bad = tmem_slot + 4;  // [2][4]: keys of a tile with a non-finite V row
  int* status = &g_tree_status;

  __syncthreads();  // the schedule's scratch has been read
  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(op_full(s), TR::KV8 ? TR::CONV_WARPS : 1);
      mbar_init(op_empty(s), 1);
    }
    for (int s = 0; s < TR::RAW_SLOTS; ++s) {
      mbar_init(raw_full(s), 1);
      mbar_init(raw_empty(s), TR::CONV_WARPS);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(s_full(b), 1);
      mbar_init(p_full(b), 128);
      mbar_init(o_done(b), 1);
    }
    mbar_init(q_full, 128);
    mbar_init(o_free, 128);
    mbar_init(v_fixed, 4);
    mbar_init(td_bar, 1);
    *abort = 0;
    p.desc[2 * cta] = make_int4(0, 0, 0, 0);  // this thread names the share's split tile at the end
    for (int i = 0; i < 8; ++i) bad[i] = 0;
    fence_mbar_init();
  }
  if (warp == 4 && lane == 0) {
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == 5) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp >= 8) {
    if constexpr (TR::KV8) {
      // ---------------------------------------------------------- e4m3 -> f16
      // e4m3 is a subset of f16: each 16-byte piece becomes two pieces of the swizzled operand
      // tile.  Eight lanes take the 64-byte halves of two rows crosswise (row r from chunk a,
      // row r + 1 from chunk a ^ 1), so neither the reads nor the writes meet in a bank.
      setmaxnreg_dec<104>();
      const int t = threadIdx.x - 256;
      const int sub = t & 7, half = sub >> 2;
      const uint32_t tiles = uint32_t(2 * (share.t1 - share.t0));
      bool ok = true;
      for (uint32_t i = 0; ok && i < tiles; ++i) {
        const int rs = int(i % NR), os = int(i % NS);
        ok = mbar_wait(raw_full(rs), uint32_t(i / NR) & 1, abort, kErrRawFull, status);
        if (ok && i >= NS)
          ok = mbar_wait(op_empty(os), (uint32_t(i / NS) & 1) ^ 1, abort, kErrOpEmpty, status);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const uint8_t* src = smem + TR::OFF_RAW + rs * TR::RAW_BYTES;
        uint8_t* dst = smem + os * TR::TILE_BYTES;
        constexpr int PER = BN * D / 16 / 256;  // 16-byte pieces a thread
        uint4 x[PER];
        int to[PER];
#pragma unroll
        for (int u = 0; u < PER; ++u) {
          const int unit = u * 32 + (t >> 3);
          const int row = unit / TR::NCH * 2 + half;
          const int a = unit % TR::NCH;
          const int ch = TR::NCH > 1 && half ? a ^ 1 : a;
          const int piece = sub & 3;
          x[u] = *reinterpret_cast<const uint4*>(src + row * D + ch * 64 + piece * 16);
          to[u] = ch * TR::CHUNK_BYTES + row * 128 + (((2 * piece) ^ (row & 7)) * 16);
        }
#pragma unroll
        for (int u = 0; u < PER; ++u) {
          const uint32_t w[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
          uint32_t o[8];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(o[2 * k]) : "h"(uint16_t(w[k] & 0xFFFFu)));
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(o[2 * k + 1]) : "h"(uint16_t(w[k] >> 16)));
          }
          *reinterpret_cast<uint4*>(dst + to[u]) = make_uint4(o[0], o[1], o[2], o[3]);
          *reinterpret_cast<uint4*>(dst + (to[u] ^ 16)) = make_uint4(o[4], o[5], o[6], o[7]);
        }
        fence_async_shared();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(raw_empty(rs));
          mbar_arrive(op_full(os));
        }
      }
    }
  } else if (warp >= 4) {
    if constexpr (TR::KV8) setmaxnreg_dec<88>();
    if (warp == 4) {
      // ---------------------------------------------------------- TMA producer
      // a lane copies one (page piece, 128-byte column) of the tile
      constexpr int COLS = TR::KV8 ? 1 : TR::NCH;
      const int box = min(p.page_size, BN);
      const int pieces = BN / box;
      const int piece = lane / COLS, col = lane - piece * COLS;
      const bool mine = piece < pieces;
      constexpr int NSL = TR::KV8 ? NR : NS;
      constexpr int BYTES = TR::KV8 ? TR::RAW_BYTES : TR::TILE_BYTES;
      const uint32_t base = smem_u32(smem + (TR::KV8 ? TR::OFF_RAW : 0)) +
                            uint32_t(TR::KV8 ? piece * box * D
                                             : col * TR::CHUNK_BYTES + piece * box * 128);
      const int c0 = col * 64;
      Walk<BN> w;
      w.start(p, share);
      // the page and row of this lane's piece of a tile; -1 (zeros) where the cache has ended
      auto lookup = [&](int seq, const Request& r, int kt, int& row) -> int {
        const int64_t key = int64_t(kt) * BN + piece * box;
        const int64_t e = key / p.page_size;
        row = int(key - e * p.page_size);
        if (!mine || key >= r.len || e >= p.max_pages) return -1;
        const int page = p.block_table[int64_t(seq) * p.max_pages + e];
        return page >= 0 && page < p.num_pages ? page : -1;
      };
      int row, page = lookup(w.seq, w.r, w.kt0, row);
      uint32_t idx = 0;
      bool ok = true, more = true;
      while (ok && more) {
        const int n = w.nt, kt0 = w.kt0, kvh = w.kvh, seq = w.seq;
        const Request r = w.r;
        more = w.next(p);
        for (int j = 0; ok && j < n; ++j) {
          // the next tile's page is looked up before this one waits for a slot
          int nrow = 0, npage = -1;
          if (j + 1 < n) npage = lookup(seq, r, kt0 + j + 1, nrow);
          else if (more) npage = lookup(w.seq, w.r, w.kt0, nrow);
#pragma unroll
          for (int kv = 0; kv < 2; ++kv, ++idx) {
            const int s = int(idx % NSL);
            const uint32_t ph = uint32_t(idx / NSL) & 1;
            const uint32_t full = TR::KV8 ? raw_full(s) : op_full(s);
            const uint32_t empty = TR::KV8 ? raw_empty(s) : op_empty(s);
            if (idx >= NSL) ok = mbar_wait(empty, ph ^ 1, abort, kErrEmpty, status);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            if (lane == 0) mbar_arrive_expect_tx(full, BYTES);
            __syncwarp();
            if (mine)
              tma_load_4d(base + uint32_t(s * BYTES), kv ? &tmV : &tmK, c0, kvh, row, page, full);
          }
          row = nrow;
          page = npage;
        }
      }
      // every copy that was issued has landed before the CTA ends (on the normal path the
      // consumers have waited for them)
      for (uint32_t i = idx > NSL ? idx - NSL : 0; i < idx; ++i) {
        const int s = int(i % NSL);
        mbar_wait_drain(TR::KV8 ? raw_full(s) : op_full(s), uint32_t(i / NSL) & 1, kErrDrain, status);
      }
    } else if (warp == 5 && lane == 0) {
      // ---------------------------------------------------------- MMA issuer
      const int fmt = p.kv_dtype == FA4CP_DTYPE_BF16 ? 1 : 0;  // an e4m3 cache is attended in f16
      const uint32_t idesc_qk = make_idesc(BM, BN, fmt, fmt, 0, 0);
      const uint32_t idesc_pv = make_idesc(BM, D, fmt, fmt, 0, 1);
      const uint32_t ring = smem_u32(smem);
      Walk<BN> w;
      w.start(p, share);
      uint32_t it = 0;
      int item = 0;
      bool ok = true, more = true;
      auto issue_pv = [&](uint32_t i, bool first) -> bool {
        const int b = int(i & 1), s = int((2 * i + 1) % NS);
        if (!mbar_wait(p_full(b), uint32_t(i >> 1) & 1, abort, kErrPFull, status)) return false;
        if (!mbar_wait(op_full(s), uint32_t((2 * i + 1) / NS) & 1, abort, kErrVFull, status)) return false;
        if (first && item > 0 && !mbar_wait(o_free, uint32_t(item - 1) & 1, abort, kErrOFree, status))
          return false;
        tc_fence_after();
        const uint32_t sV = ring + uint32_t(s * TR::TILE_BYTES);
#pragma unroll
        for (int kk = 0; kk < BN / 16; ++kk) {
          const uint64_t bdesc = make_desc_sw128(sV + kk * 16 * 128, TR::CHUNK_BYTES, 1024);
          mma_f16_ts(tmem + TR::TM_O, tmem + uint32_t(TR::TM_S + b * BN + kk * 8), bdesc, idesc_pv,
                     (!first || kk > 0) ? 1u : 0u);
        }
        tc_commit(o_done(b));
        tc_commit(op_empty(s));
        return true;
      };
      while (ok && more) {
        const int n = w.nt;
        more = w.next(p);
        ok = mbar_wait(q_full, uint32_t(item) & 1, abort, kErrQFull, status);
        tc_fence_after();
        for (int j = 0; ok && j < n; ++j, ++it) {
          const int b = int(it & 1), s = int((2 * it) % NS);
          if (!mbar_wait(op_full(s), uint32_t((2 * it) / NS) & 1, abort, kErrKFull, status)) { ok = false; break; }
          tc_fence_after();
          const uint32_t sK = ring + uint32_t(s * TR::TILE_BYTES);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const int off = kk * 32;  // bytes along D
            const uint64_t bdesc =
                make_desc_sw128(sK + (off / 128) * TR::CHUNK_BYTES + (off % 128), 16, 1024);
            mma_f16_ts(tmem + uint32_t(TR::TM_S + b * BN), tmem + uint32_t(TR::TM_Q + kk * 8), bdesc,
                       idesc_qk, kk > 0 ? 1u : 0u);
          }
          tc_commit(s_full(b));
          tc_commit(op_empty(s));
          if (j > 0 && !issue_pv(it - 1, j == 1)) ok = false;
        }
        if (ok) ok = issue_pv(it - 1, n == 1);
        ++item;
      }
      // every MMA issued above has completed before TMEM is released
      tc_commit(td_bar);
      mbar_wait_drain(td_bar, 0, kErrDrain, status);
    }
  } else {
    // ------------------------------------------------------------ softmax + epilogue
    if constexpr (TR::KV8) setmaxnreg_inc<216>();
    const int t = threadIdx.x;  // 0..127
    const uint32_t t_lane = tmem + (uint32_t(warp * 32) << 16);
    const bool bf16_op = p.kv_dtype == FA4CP_DTYPE_BF16;
    Walk<BN> w;
    w.start(p, share);
    float qf = 1.f;  // the row's power of two (e4m3 cache)

    // Q of item `w` into TMEM.  All S MMAs of the item before are complete (this thread has
    // seen its last s_full).
    auto load_q = [&](const Walk<BN>& x) {
      const int r = x.mtile * BM + t;
      const bool valid = t < x.rows(p);
      if (warp * 32 < x.rows(p)) {  // the warp has rows; the others' lanes are never read
        const int node = r / p.group, head = x.kvh * p.group + (r - node * p.group);
        const uint8_t* row = p.q + (int64_t(x.r.token0) + (valid ? node : 0)) * p.q_stride +
                             int64_t(valid ? head : 0) * D * (p.q_dtype == FA4CP_DTYPE_E4M3 ? 1 : 2);
        if (TR::KV8) {
          // largest magnitude into [2^14, 2^15): f16 then holds the row to 2^-24 of it
          const uint32_t e = __float_as_uint(q_absmax<D>(p, row)) >> 23;
          const int s = e == 0 || e == 255 ? 0 : min(127 + 14 - int(e), 126);
          qf = __uint_as_float(uint32_t(127 + s) << 23);
          if ((p.q_descale ? p.q_descale[x.kvh] : 1.f) * (p.k_descale ? p.k_descale[x.kvh] : 1.f) < 0.f) qf = -qf;
        }
#pragma unroll 1
        for (int c = 0; c < D / 64; ++c) {
          uint32_t reg[32];
          load_q64<TR::KV8>(p, row, c, qf, reg);
          tmem_st32(t_lane + uint32_t(TR::TM_Q + c * 32), reg);
        }
        tmem_wait_st();
      }
      tc_fence_before();
      mbar_arrive(q_full);
    };

    load_q(w);
    uint32_t it = 0, fixes = 0;
    bool aborted = false, more = true;
    while (more && !aborted) {
      const Request r = w.r;
      const int seq = w.seq, kvh = w.kvh, kt0 = w.kt0, n = w.nt, mtile = w.mtile;
      const int rows = w.rows(p);
      const bool active = warp * 32 < rows;
      const int packed = mtile * BM + t;
      const bool valid = t < rows;
      const int node = valid ? packed / p.group : 0;
      const int head = kvh * p.group + (valid ? packed - node * p.group : 0);
      const int64_t tok = int64_t(r.token0) + node;
      const int ctx = r.len - r.n;
      float scale = p.scale_log2, vscale = 1.0f;
      if (TR::KV8) {
        if (p.q_descale) scale *= p.q_descale[kvh];
        if (p.k_descale) scale *= p.k_descale[kvh];
        if (p.v_descale) vscale = p.v_descale[kvh];
        // qf carries the sign of the descales, so the scale is positive; never 0, so that a
        // masked score stays -inf
        scale /= qf;
        scale = scale < 1.17549435e-38f ? 1.17549435e-38f : scale;
      }
      float m = kNegInf, l = 0.f;
      bool sees_bad = false;

      for (int j = 0; j < n; ++j, ++it) {
        const int b = int(it & 1);
        bool ok = mbar_wait(s_full(b), uint32_t(it >> 1) & 1, abort, kErrSFull, status);
        if (!__all_sync(0xffffffffu, ok)) { aborted = true; break; }
        tc_fence_after();
        const int kbase = (kt0 + j) * BN;
        const bool edge = kbase + BN > ctx;  // the tile holds new rows, or the cache's end
        uint32_t vis[BN / 32];
        if (active) {
          uint32_t sr[BN / 32][32];
#pragma unroll
          for (int c = 0; c < BN / 32; ++c) tmem_ld32(t_lane + uint32_t(TR::TM_S + b * BN + c * 32), sr[c]);
          tmem_wait_ld();
#pragma unroll
          for (int c = 0; c < BN / 32; ++c) reg_fence32(sr[c]);
          if (edge) {
#pragma unroll
            for (int c = 0; c < BN / 32; ++c) {
              vis[c] = seen32(p, r, tok, node, kbase + c * 32);
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!((vis[c] >> e) & 1u)) sr[c][e] = __float_as_uint(kNegInf);
            }
          }
          float mx[4] = {kNegInf, kNegInf, kNegInf, kNegInf};
#pragma unroll
          for (int c = 0; c < BN / 32; ++c)
#pragma unroll
            for (int e = 0; e < 32; e += 8)
#pragma unroll
              for (int k = 0; k < 4; ++k)
                mx[k] = fmax3(mx[k], __uint_as_float(sr[c][e + 2 * k]), __uint_as_float(sr[c][e + 2 * k + 1]));
          const float m_new = fmaxf(fmax3(m, mx[0], mx[1]), fmaxf(mx[2], mx[3]));
          if (j == 0) {
            m = m_new;
          } else {
            const bool need = (m_new - m) * scale > kRescaleThreshold;
            if (__any_sync(0xffffffffu, need)) {
              const float f = need ? ex2_approx((m - m_new) * scale) : 1.0f;
              if (need) { l *= f; m = m_new; }
              ok = mbar_wait(o_done(b ^ 1), uint32_t((it - 1) >> 1) & 1, abort, kErrODone, status);
              if (!__all_sync(0xffffffffu, ok)) { aborted = true; break; }
              tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < D / 32; ++c) {
                uint32_t o[32];
                tmem_ld32(t_lane + uint32_t(TR::TM_O + c * 32), o);
                tmem_wait_ld();
                reg_fence32(o);
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                tmem_st32(t_lane + uint32_t(TR::TM_O + c * 32), o);
              }
              tmem_wait_st();
            }
          }
          const float neg_m = (m == kNegInf) ? 0.f : -m * scale;
          const uint64_t scale2 = f2pack(scale, scale), negm2 = f2pack(neg_m, neg_m);
          uint64_t rs[2] = {0ull, 0ull};
#pragma unroll
          for (int hf = 0; hf < BN / 64; ++hf) {
            uint32_t pw[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const int c = hf * 2 + (i >> 4), e = (2 * i) & 31;
              const uint64_t x = ffma2(f2pack(__uint_as_float(sr[c][e]), __uint_as_float(sr[c][e + 1])), scale2, negm2);
              const float x0 = ex2_approx(f2lo(x)), x1 = ex2_approx(f2hi(x));
              rs[i & 1] = fadd2(rs[i & 1], f2pack(x0, x1));
              pw[i] = !TR::KV8 && bf16_op ? pack_bf16x2(x0, x1) : pack_f16x2(x0, x1);
            }
            tmem_st32(t_lane + uint32_t(TR::TM_S + b * BN + hf * 32), pw);
          }
          const uint64_t rsum = fadd2(rs[0], rs[1]);
          l += f2lo(rsum) + f2hi(rsum);
        }
        if (edge) {
          // P is 0 where a row does not look, but 0 * NaN is NaN: V rows behind the cache are
          // cleared, and so are the non-finite values of new rows (a context row is seen by
          // every token, so its values go through as they are).  Thread t has key t.
          const int s = int((2 * it + 1) % NS);
          ok = mbar_wait(op_full(s), uint32_t((2 * it + 1) / NS) & 1, abort, kErrVFix, status);
          if (!__all_sync(0xffffffffu, ok)) { aborted = true; break; }
          const int key = kbase + t;
          uint8_t* vrow = smem + s * TR::TILE_BYTES + t * 128;
          bool mine_bad = false;
          if (t < BN && key >= r.len) {
#pragma unroll 4
            for (int c = 0; c < D / 8; ++c)
              *reinterpret_cast<uint4*>(vrow + (c >> 3) * TR::CHUNK_BYTES + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
          } else if (t < BN && key >= ctx && r.n > 1) {
#pragma unroll 4
            for (int c = 0; c < D / 8; ++c) {
              uint4* at = reinterpret_cast<uint4*>(vrow + (c >> 3) * TR::CHUNK_BYTES + (c & 7) * 16);
              uint32_t x[4] = {at->x, at->y, at->z, at->w};
              bool hit = false;
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                if (nonfinite16(x[k] & 0xFFFFu, bf16_op)) { x[k] &= 0xFFFF0000u; hit = true; }
                if (nonfinite16(x[k] >> 16, bf16_op)) { x[k] &= 0xFFFFu; hit = true; }
              }
              if (hit) {
                *at = make_uint4(x[0], x[1], x[2], x[3]);
                mine_bad = true;
              }
            }
          }
          fence_async_shared();
          if (r.n > 1) {
            // which keys of the tile were cleared: one word a warp, two sets used in turn
            const uint32_t word = __ballot_sync(0xffffffffu, mine_bad);
            volatile uint32_t* set = bad + (fixes & 1) * 4;
            if (lane == 0) {
              set[warp] = word;
              mbar_arrive(v_fixed);
            }
            ok = mbar_wait(v_fixed, fixes & 1, abort, kErrVFix, status);
            if (!__all_sync(0xffffffffu, ok)) { aborted = true; break; }
            ++fixes;
            if (active) {
#pragma unroll
              for (int c = 0; c < BN / 32; ++c) sees_bad |= (set[c] & vis[c]) != 0;
            }
          }
        }
        if (active) tmem_wait_st();
        tc_fence_before();
        mbar_arrive(p_full(b));
      }
      if (aborted) break;

      // the next item's Q goes in before this item's epilogue, so its first S starts meanwhile
      const int64_t left_after = w.left - w.nt;
      const bool whole = kt0 == 0 && n == r.kt;
      const bool begins = kt0 == 0;
      more = w.next(p);
      if (more) load_q(w);

      const uint32_t last = it - 1;
      bool ok = mbar_wait(o_done(int(last & 1)), uint32_t(last >> 1) & 1, abort, kErrODone, status);
      if (!__all_sync(0xffffffffu, ok)) { aborted = true; break; }
      tc_fence_after();
      const int part = 2 * cta + (begins ? 1 : 0);
      const float ms = m == kNegInf ? kNegInf : m * scale;  // log2 units
      const float mult = whole ? (l == 0.f ? 0.f : vscale / l) : vscale;
      const int64_t orow = (tok * p.Hq + head) * D;
      float* prow = p.part_o + (int64_t(part) * BM + t) * D;
      if (active) {
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(t_lane + uint32_t(TR::TM_O + c * 32), o);
          tmem_wait_ld();
          reg_fence32(o);
          if (!valid) continue;
          if (whole) {
            uint4* dst = reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.out) + orow * 2 + c * 64);
#pragma unroll
            for (int v4 = 0; v4 < 4; ++v4) {
              uint32_t x[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float lo = __uint_as_float(o[v4 * 8 + 2 * i]) * mult, hi = __uint_as_float(o[v4 * 8 + 2 * i + 1]) * mult;
                x[i] = p.out_bf16 ? pack_bf16x2(lo, hi) : pack_f16x2(lo, hi);
              }
              dst[v4] = make_uint4(x[0], x[1], x[2], x[3]);
            }
          } else {
            float4* dst = reinterpret_cast<float4*>(prow + c * 32);
#pragma unroll
            for (int v4 = 0; v4 < 8; ++v4)
              dst[v4] = make_float4(__uint_as_float(o[4 * v4]) * mult, __uint_as_float(o[4 * v4 + 1]) * mult,
                                    __uint_as_float(o[4 * v4 + 2]) * mult, __uint_as_float(o[4 * v4 + 3]) * mult);
          }
        }
      }
      tc_fence_before();
      mbar_arrive(o_free);
      if (valid) {
        if (whole) {
          p.lse[tok * p.Hq + head] = l == 0.f ? kNegInf : (ms + lg2_approx(l)) * kLn2;
          if (sees_bad)
            add_nonfinite<D>(p, r, seq, kvh, tok, node, 0, r.len, Add16{static_cast<uint16_t*>(p.out) + orow, p.out_bf16});
        } else {
          p.part_ml[part * BM + t] = make_float2(ms, l);
          if (sees_bad) add_nonfinite<D>(p, r, seq, kvh, tok, node, kt0 * BN, (kt0 + n) * BN, AddF32{prow});
        }
      }
      if (t == 0 && left_after <= 0) {
        // the share's last item: if it began here and goes on, this CTA's descriptor names it
        int4 d0 = make_int4(0, 0, 0, 0), d1 = d0;
        if (begins && !whole) {
          const int64_t end = share.t1 + (r.kt - n);  // one past the item's last tile
          const int64_t g = min(int64_t(G), share.total);
          d0 = make_int4(1, int((end * g - 1) / share.total), rows, mtile * BM);
          d1 = make_int4(r.token0, kvh, 0, 0);
        }
        p.desc[2 * cta] = d0;
        p.desc[2 * cta + 1] = d1;
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 5) tmem_dealloc(tmem, 512);
}

// ---------------------------------------------------------------------------
// join of the parts of split row tiles
// ---------------------------------------------------------------------------
// Block (c, y): the row tile that CTA c began and others went on with, rows y * 8 ...; a warp a
// row.  The parts are CTA c's second partial and the first one of CTAs c + 1 .. last, summed in
// that order.
template <int D>
__global__ void __launch_bounds__(256) tree_combine_kernel(const TreeParams p) {
  const int c = blockIdx.x, lane = threadIdx.x & 31;
  const int4 d0 = p.desc[2 * c];
  if (d0.x == 0) return;
  const int4 d1 = p.desc[2 * c + 1];
  const int parts = d0.y - c + 1;
  auto slot = [&](int i) { return i == 0 ? 2 * c + 1 : 2 * (c + i); };
  for (int row = blockIdx.y * 8 + (threadIdx.x >> 5); row < d0.z; row += gridDim.y * 8) {
    float top = kNegInf;
    for (int i = lane; i < parts; i += 32) top = fmaxf(top, p.part_ml[slot(i) * BM + row].x);
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    constexpr int E = D / 32;
    float acc[E], l = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma unroll 4
    for (int i = 0; i < parts; ++i) {
      const float2 ml = p.part_ml[slot(i) * BM + row];
      const float f = ml.x == kNegInf ? 0.f : ex2_approx(ml.x - top);
      const float* src = p.part_o + (int64_t(slot(i)) * BM + row) * D;
      l = fmaf(ml.y, f, l);
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const float2 x = *reinterpret_cast<const float2*>(src + e * 32 + lane * 2);
        if (ml.x != kNegInf) {
          acc[e] = fmaf(x.x, f, acc[e]);
          acc[e + 1] = fmaf(x.y, f, acc[e + 1]);
        }
      }
    }
    const int packed = d0.w + row, node = packed / p.group;
    const int head = d1.y * p.group + (packed - node * p.group);
    const int64_t o = (int64_t(d1.x) + node) * p.Hq + head;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint32_t* out = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.out) + o * D);
#pragma unroll
    for (int e = 0; e < E; e += 2)
      out[e * 16 + lane] = p.out_bf16 ? pack_bf16x2(acc[e] * inv, acc[e + 1] * inv)
                                      : pack_f16x2(acc[e] * inv, acc[e + 1] * inv);
    if (lane == 0) p.lse[o] = l == 0.f ? kNegInf : (top + lg2_approx(l)) * kLn2;
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
int sm_count(int* out) {
  static std::atomic<int> cached{0};
  int n = cached.load();
  if (n == 0) {
    int dev = 0;
    FA4CP_CHECK_CUDA(cudaGetDevice(&dev));
    FA4CP_CHECK_CUDA(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
    cached.store(n);
  }
  *out = n;
  return FA4CP_OK;
}

constexpr int kMaxGrid = 148;  // B200's SMs: sizes the workspace without a device

int64_t workspace_bytes_for(int D) {
  return int64_t(kMaxGrid) * (2 * (int64_t(BM) * D * 4 + BM * 8) + 32);
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                  const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// Pool view [pages, page_size, heads, D] with a box of (128 bytes | an e4m3 row, 1 head,
// `rows` rows, 1 page).
int make_pool_map(CUtensorMap* map, const void* base, int num_pages, int page_size, int heads, int D,
                  int elem, const int64_t* strides, int rows) {
  static EncodeTiledFn enc = nullptr;
  if (enc == nullptr) {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      enc = reinterpret_cast<EncodeTiledFn>(ptr);
  }
  FA4CP_CHECK_ARG(enc != nullptr, "cuTensorMapEncodeTiled is unavailable");
  const cuuint64_t dims[4] = {cuuint64_t(D), cuuint64_t(heads), cuuint64_t(page_size),
                              cuuint64_t(num_pages > 0 ? num_pages : 1)};
  const cuuint64_t st[3] = {cuuint64_t(strides[2]) * elem, cuuint64_t(strides[1]) * elem,
                            cuuint64_t(strides[0]) * elem};
  const cuuint32_t box[4] = {cuuint32_t(elem == 1 ? D : 64), 1, cuuint32_t(rows), 1};
  const cuuint32_t es[4] = {1, 1, 1, 1};
  const CUresult r = enc(map, elem == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 4,
                         const_cast<void*>(base), dims, st, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         elem == 1 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_last_error("cuTensorMapEncodeTiled (pool) failed (%d)", int(r));
    return FA4CP_ERR_CUDA;
  }
  return FA4CP_OK;
}

template <class TR>
int launch_tree(const void* k_pages, const void* v_pages, const int64_t* ks, const int64_t* vs,
                int max_seqlen_q, const TreeParams& p, cudaStream_t st) {
  static std::atomic<uint64_t> optin{0};
  int dev = 0;
  FA4CP_CHECK_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
  if (bit == 0 || !(optin.load() & bit)) {
    FA4CP_CHECK_CUDA(cudaFuncSetAttribute(tree_attn_kernel<TR>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                          TR::SMEM_BYTES));
    optin.fetch_or(bit);
  }
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  const int grid = sms < kMaxGrid ? sms : kMaxGrid;
  const int rows = p.page_size < TR::BN ? p.page_size : TR::BN;
  const int el = TR::KV8 ? 1 : 2;
  CUtensorMap mk, mv;
  if (int rc = make_pool_map(&mk, p.num_pages ? k_pages : p.q, p.num_pages, p.page_size, p.Hkv, TR::D, el, ks, rows)) return rc;
  if (int rc = make_pool_map(&mv, p.num_pages ? v_pages : p.q, p.num_pages, p.page_size, p.Hkv, TR::D, el, vs, rows)) return rc;
  tree_attn_kernel<TR><<<grid, TR::THREADS, TR::SMEM_BYTES, st>>>(mk, mv, p);
  if (int rc = check_launch("attn_fwd_paged_tree")) return rc;
  const int64_t most = int64_t(max_seqlen_q) * p.group;  // rows of a row tile
  const int blocks = int(((most < BM ? most : BM) + 7) / 8);
  tree_combine_kernel<TR::D><<<dim3(unsigned(grid), unsigned(blocks)), 256, 0, st>>>(p);
  return check_launch("attn_fwd_paged_tree (combine)");
}

}  // namespace
}  // namespace fa4cp

using namespace fa4cp;

extern "C" int64_t fa4cp_attn_paged_tree_workspace_bytes(int32_t num_heads_q, int32_t num_heads_kv,
                                                         int32_t head_dim, int32_t max_seqlen_q) {
  if (num_heads_q < 1 || num_heads_kv < 1 || head_dim < 1 || max_seqlen_q < 0) return -1;
  return workspace_bytes_for(head_dim);
}

extern "C" int fa4cp_attn_fwd_paged_tree(
    const void* q, int64_t q_token_stride, const void* k_pages, const void* v_pages,
    const int64_t* k_strides, const int64_t* v_strides, const int32_t* block_table,
    int32_t page_size, int32_t num_pages, int32_t max_pages, void* out, float* lse,
    const int32_t* cu_q, const int32_t* seq_lens, int32_t nseq, int32_t max_seqlen_q,
    int64_t total_q, int32_t num_heads_q, int32_t num_heads_kv, int32_t head_dim, int32_t q_dtype,
    int32_t kv_dtype, const int64_t* tree_mask, int32_t mask_words, float softmax_scale,
    const float* q_descale, const float* k_descale, const float* v_descale, void* workspace,
    int64_t workspace_bytes, void* stream) {
  FA4CP_CHECK_ARG(nseq >= 1 && cu_q && seq_lens, "cu_seqlens_q and seq_lens must describe >= 1 request");
  FA4CP_CHECK_ARG(num_heads_q > 0 && num_heads_kv > 0 && num_heads_q % num_heads_kv == 0,
                  "H_q=%d not a multiple of H_kv=%d", num_heads_q, num_heads_kv);
  FA4CP_CHECK_ARG(total_q >= 0 && max_seqlen_q >= 0 && num_pages >= 0 && max_pages >= 1, "bad sizes");
  FA4CP_CHECK_ARG(page_size == 16 || page_size == 32 || page_size == 64 ||
                      (page_size > 0 && page_size % 128 == 0),
                  "page_size %d must be 16, 32, 64 or a multiple of 128", page_size);
  const bool q8 = q_dtype == FA4CP_DTYPE_E4M3, kv8 = kv_dtype == FA4CP_DTYPE_E4M3;
  FA4CP_CHECK_ARG(q8 || q_dtype == FA4CP_DTYPE_BF16 || q_dtype == FA4CP_DTYPE_F16,
                  "q dtype must be f16, bf16 or e4m3");
  FA4CP_CHECK_ARG(kv8 || kv_dtype == q_dtype, "K/V dtype must be e4m3 or the dtype of q");
  FA4CP_CHECK_ARG(q8 || !q_descale, "q_descale applies to an e4m3 q only");
  FA4CP_CHECK_ARG(kv8 || (!k_descale && !v_descale), "descales apply to e4m3 K/V only");
  FA4CP_CHECK_ARG(softmax_scale > 0.f, "softmax_scale must be positive");
  FA4CP_CHECK_ARG(tree_mask == nullptr || (mask_words >= 1 && mask_words <= (1 << 24)), "tree_mask needs mask_words >= 1");
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) {
    set_last_error("head_dim %d is not supported", head_dim);
    return FA4CP_ERR_UNSUPPORTED;
  }
  if (total_q == 0 || max_seqlen_q == 0) return FA4CP_OK;
  FA4CP_CHECK_ARG(total_q * int64_t(num_heads_q) < (int64_t(1) << 31), "too many query rows");
  FA4CP_CHECK_ARG(q && out && lse && block_table && k_strides && v_strides && (num_pages == 0 || (k_pages && v_pages)),
                  "null tensor pointer");
  const int qe = q8 ? 1 : 2, ke = kv8 ? 1 : 2;
  auto al = [](const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15u) == 0; };
  FA4CP_CHECK_ARG(al(q) && al(out) && al(k_pages) && al(v_pages) && q_token_stride * qe % 16 == 0,
                  "q rows, out and the pools must be 16-byte aligned");
  for (int i = 0; i < 3; ++i)
    FA4CP_CHECK_ARG(k_strides[i] * ke % 16 == 0 && v_strides[i] * ke % 16 == 0 && k_strides[i] >= 0 && v_strides[i] >= 0,
                    "pool strides must be multiples of 16 bytes");
  FA4CP_CHECK_ARG(workspace_bytes >= workspace_bytes_for(head_dim) && workspace && al(workspace),
                  "workspace too small or not 16-byte aligned: %lld < %lld bytes",
                  (long long)workspace_bytes, (long long)workspace_bytes_for(head_dim));
  TreeParams p{};
  p.q = static_cast<const uint8_t*>(q);
  p.q_stride = q_token_stride * qe;
  p.v = static_cast<const uint8_t*>(v_pages);
  p.v_page = v_strides[0] * ke; p.v_row = v_strides[1] * ke; p.v_head = v_strides[2] * ke;
  p.block_table = block_table;
  p.cu_q = cu_q;
  p.seq_lens = seq_lens;
  p.mask = reinterpret_cast<const uint32_t*>(tree_mask);
  p.out = out;
  p.lse = lse;
  p.q_descale = q_descale;
  p.k_descale = k_descale;
  p.v_descale = v_descale;
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + int64_t(kMaxGrid) * 2 * BM * head_dim);
  p.desc = reinterpret_cast<int4*>(p.part_ml + int64_t(kMaxGrid) * 2 * BM);
  p.total_q = total_q;
  p.nseq = nseq;
  p.Hq = num_heads_q;
  p.Hkv = num_heads_kv;
  p.group = num_heads_q / num_heads_kv;
  p.page_size = page_size;
  p.num_pages = num_pages;
  p.max_pages = max_pages;
  p.mask_words = 2 * mask_words;
  p.q_dtype = q_dtype;
  p.kv_dtype = kv_dtype;
  p.out_bf16 = q_dtype != FA4CP_DTYPE_F16;
  p.scale_log2 = softmax_scale * kLog2e;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto go = [&](auto tr) {
    return launch_tree<decltype(tr)>(k_pages, v_pages, k_strides, v_strides, max_seqlen_q, p, st);
  };
  if (kv8) {
    if (head_dim == 64) return go(TreeTraits<64, 128, true>{});
    if (head_dim == 128) return go(TreeTraits<128, 128, true>{});
    return go(TreeTraits<256, 64, true>{});
  }
  if (head_dim == 64) return go(TreeTraits<64, 128, false>{});
  if (head_dim == 128) return go(TreeTraits<128, 128, false>{});
  return go(TreeTraits<256, 64, false>{});
}
