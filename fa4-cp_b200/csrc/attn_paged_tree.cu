// Attention of drafted tokens over a paged K/V cache (single-token decode is the tree of one
// node).  No counterpart in the reference, whose K/V is contiguous (README.md:139-141).
//
//   O[i] = sum_k softmax_k(scale q_i . K[k]) V[k],  k < ctx, or k one of the request's own new
//   rows that the tree's bits of token i name (ctx = seq_len - n, n new tokens).
//
// The query heads of one K/V head read the same keys, so a request's n tokens x `group` heads
// are packed into rows of one 128-row MMA tile (row = token * group + head of the group), and
// K and V are read once for all of them.
//
// Measured (32/8 heads, head_dim 128; calls of a captured graph).  64 decoding requests of 1K to 32K
// tokens, bf16: 0.68 to 0.72 ms = 6.2 to 6.5 TB/s, the rate of a copy.  32 requests of 1K to 16K
// tokens: bf16 with 1, 8 and 32 new tokens 186, 191 and 206 us (5.6 to 6.1 TB/s); 64 tokens are two
// row tiles, 383 us (620 TFLOP/s).  Over an e4m3 cache 1, 8, 32 and 64 tokens take 139 to 165, 142 to
// 166, 169 and 331 us: a key tile of a CTA takes 1000 to 1100 cycles whatever its bytes, the round
// trip of an S buffer (S 430, softmax 1810, P to PV 210, PV 600, next S 370 cycles) over the three
// buffers that TMEM leaves beside a Q and two O of this layout.  (One token there, and two requests of
// 256K tokens at head_dim 256, 143 to 200 us, run at one of two speeds from call to call.)  One
// request of 100 and 8K tokens: 11 and 17 us, mostly launch and start.
//
// Schedule.  The work is the list of all (request, K/V head, row tile, key tile), in that
// order; every CTA takes an equal share of consecutive key tiles, whatever the lengths are
// (they are only known on the device).  A row tile counts ITEM_COST tiles more than it has, for
// its Q and its result.  A row tile whose keys several CTAs share leaves one partial (O, m, l)
// each in the workspace, joined by tree_combine_kernel in a fixed order.  A CTA has at most two
// partials (its first and its last row tile), so the workspace does not depend on the lengths.
//
// CTA roles (one CTA per SM):
//   warps 0-7   two softmax warpgroups, taking key tiles in turn: thread t of either owns row t
//               = TMEM lane t; each loads half of Q and writes half of the result's columns, too
//   warp  8     the share's items (row tiles) into a ring that the other roles read; TMA producer
//               of K, a page piece a lane, and before an item's first K tile its Q rows
//   warp  10    TMA producer of V (a ring of its own: K runs ahead of V)
//   warp  9     TMEM allocator + issuer of the S MMAs, warp 11 issuer of the PV MMAs (one
//               elected lane each: an issuer is held up while the tensor core is busy, so the
//               waits of one hide behind the other's MMAs)
//   warps 12-15 e4m3 cache only: V tiles from a raw ring, widened to f16
// TMEM: S buffers (64 fp32 columns each, 32 at head_dim 256) | O (D columns, twice up to
// head_dim 128) | Q (D/2).
// P(j) lies over S(j), as 16-bit pairs, and is the A operand of O += P V; S(j + buffers) waits
// for PV(j).  A hand-over between two roles takes 200 to 300 cycles, and a tile has five of
// them, so it is the number of tiles in flight that counts: four of 64 keys ran 1.5 times as
// fast as two of 128.  Q is the A operand of S = Q K^T straight from TMEM, so the MMA reads K
// alone from shared memory; it passes through slots of the K ring, loaded while the item before
// is still worked on.
// An e4m3 cache: K is multiplied as it is, by a Q in two e4m3 terms (hi + lo of q x 2^s, which
// hold a bf16 to 2^-17 of its row's largest value), at twice the rate a term; V is widened to
// f16, because a P in e4m3 would have to be two terms as well, at three conversions a value.
// Up to head_dim 128 the warpgroups work apart, each with an O, a running maximum and a sum of
// its own, joined when the item ends: handing one maximum from tile to tile made every tile wait
// for the one before (e4m3, head_dim 64, 64 tokens: 486 us, apart 324; one token: 203 and 157).
// S and P in buffers of their own, so that S never waits for PV, let the warpgroups fall into step
// and meet at the exponential unit (f16, head_dim 64: 302 us against 250).
// TMEM has no room for that at head_dim 256; there they share one O and one maximum a row, handed
// on through shared memory right after a tile's maximum is known (its exponentials come later).
// What runs once an item is written as small loops: its instructions come from L2 each time.
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
constexpr float kRescaleThreshold = 8.0f;  // log2 units: P <= 256 times the largest at its maximum
// P is rounded to the 16-bit type of the V that it multiplies (f16 for an e4m3 V), by half a step:
// 2^-8 of each weight in bf16, 2^-11 in f16.  (Both operands of an MMA are of one type.  Over a bf16
// cache, 64 requests of 1K to 32K tokens, the result is 0.0023 off the 64-bit one, in norm; with all in
// 32 bits 0.0017, which is the output's own rounding.)  An f16 also ends at the bottom: it is subnormal below
// 2^-14 and 0 below 2^-25, while the sum of the weights is in 32 bits and keeps them all.  So an f16 P
// carries a factor of 2^7, which the sum and O share: the largest weight is between 2^7 and 2^15, and
// what is lost of a weight is below 2^-32 of it.  (It is added to the finished offset: with an fma or a
// product rounded upwards in its place the warpgroups fall into step at head_dim 64, and e4m3 with one
// token takes 162 us instead of 140.)
constexpr float kLiftF16 = 7.0f;
// An offset of 2^22 and more is off by a quarter and more.  The maximum is raised with every larger one
// there, so that this and the threshold do not add up past the end of an f16.
constexpr float kExactBelow = 0x1p22f;
constexpr int BM = 128;

// codes written to the device status word when a bounded wait gives up
enum : int {
  kErrEmpty = 0x401, kErrRawFull, kErrVEmpty, kErrQFull, kErrKFull, kErrPFull,
  kErrVFull, kErrOFree, kErrSFull, kErrSFree, kErrMax, kErrODone, kErrVFix, kErrJoin, kErrItem,
  kErrItemFree, kErrQStaged, kErrDrain
};

constexpr int kItems = 8;     // ring of items

// A CTA's part of a row tile, as the roles of a CTA pass it on (nt == 0: the share has ended).
struct Item {
  int seq, token0, n, len, lim;  // request: first token, tokens, cached rows, those with a page entry
  int kvh, mtile, kt0, nt, kt;   // K/V head, row tile, first key tile, tiles here, tiles in all
  uint32_t k_idx;                // K ring index of its Q; its K tiles follow
  int q_slots;
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
  float2* part_ml; // [2 * grid][BM]: what the exponents are relative to (log2 units), sum
  int4* desc;      // [grid][2]: the row tile whose first part a CTA holds
  int64_t total_q;
  int nseq, Hq, Hkv, group, page_size, num_pages, max_pages, mask_words;
  int q_dtype, kv_dtype, out_bf16;
  float scale_log2;
};

template <int D_, bool KV8_>
struct TreeTraits {
  static constexpr int D = D_, BN = D == 256 ? 32 : 64;  // keys of a tile
  static constexpr bool KV8 = KV8_;
  // key tiles that a row tile's start and end are worth: a tile of an e4m3 cache takes less of a
  // CTA's time (32 requests, 64 tokens: e4m3 D128 352 us with 6, 348 with 9, 341 with 12; bf16 386,
  // 380, 384)
  static constexpr int ITEM_COST = KV8 ? 12 : 8;
  static constexpr int KEL = KV8 ? 1 : 2;             // bytes of a K element
  static constexpr int K_SWZ = D * KEL >= 128 ? 128 : 64;  // bytes of a swizzled row of K
  static constexpr int K_COLS = D * KEL / K_SWZ;
  static constexpr int K_BYTES = BN * D * KEL;
  static constexpr int V_COLS = D / 64;               // 128-byte columns of a V operand tile
  static constexpr int V_CHUNK = BN * 128;
  static constexpr int V_BYTES = BN * D * 2;
  static constexpr int RAW_BYTES = BN * D;            // one e4m3 V tile
  // ring slots: what shared memory holds, 8 at head_dim 64 (e4m3, 64 tokens and one: 273 and 140 us,
  // with 6 276 and 143, with 12 288 and 148)
  static constexpr int KS = D == 64 || (KV8 && D == 256) ? 8 : 6, VS = D == 64 ? 8 : 6, RS = KV8 ? VS : 0;
  static_assert(KS * K_BYTES >= BM * D * 2, "the K ring takes the Q of an item whole");
  static constexpr int OFF_V = KS * K_BYTES;
  static constexpr int OFF_RAW = OFF_V + VS * V_BYTES;
  static constexpr int OFF_ROWS = OFF_RAW + RS * RAW_BYTES;
  // per row: running maximum [BM]; per item parity and warpgroup: maximum, sum, flag [2][2][BM]
  static constexpr int NWG = 2, W0 = 4 * NWG;  // softmax warpgroups, and the first warp behind them
  static constexpr int OFF_ITEMS = OFF_ROWS + BM * 4 + 2 * NWG * BM * 12;
  static constexpr int OFF_BAR = OFF_ITEMS + kItems * 48;
  // k_full, k_empty [KS]; v_full, v_empty [VS]; r_full, r_empty [RS]; s_full, p_full, o_done
  // [NB]; max_known[W0] (warpgroup, warp), v_fixed[NWG], q_full, o_free, joined, teardown;
  // q_staged, item_full, item_free [kItems]
  static constexpr bool APART = D <= 128;
  static constexpr int NB = D == 128 ? 3 : 4;  // S buffers: what TMEM leaves
  static constexpr int NUM_BARS = 2 * (KS + VS + RS) + 3 * NB + 5 * NWG + 4 + 3 * kItems;
  // q_staged(i) is waited for before q_staged(i + kItems) can complete: the items between them
  // take two slots of the K ring each, so the latter needs the former's slots back
  static_assert(KS < 2 * kItems, "Q staging ring");
  static constexpr int OFF_MISC = OFF_BAR + NUM_BARS * 8;
  static constexpr int SMEM_BYTES = OFF_MISC + 128 + 1024;
  // an e4m3 V tile is widened by all four warps, by two at head_dim 64, where it is half as large:
  // their load on the exponential unit then spreads over the SM's quarters, and no softmax warp is
  // later than the others (a warp a tile: D128, 64 tokens and one 347 and 172 us, so 341 and 156)
  static constexpr int CONV_WARPS = KV8 ? 4 : 0, CONV_TEAM = D == 64 ? 2 : 4;
  static constexpr int THREADS = W0 * 32 + 128 + CONV_WARPS * 32;
  // setmaxnreg split, in registers a thread of a warpgroup; the launch gives 512 x 128 or
  // 384 x 168 registers
  static constexpr int REGS_SOFTMAX = KV8 ? 168 : 184, REGS_CONTROL = KV8 ? 80 : 136, REGS_CONV = 96;
  static_assert(128 * (NWG * REGS_SOFTMAX + REGS_CONTROL) + 32 * CONV_WARPS * REGS_CONV <=
                    THREADS * (65536 / THREADS / 8 * 8), "register split exceeds the launch allocation");
  static constexpr int TM_S = 0, TM_O = NB * BN, TM_Q = TM_O + (APART ? NWG : 1) * D;
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
// As make_desc_sw128 with the 64-byte swizzle (mode 4).
__device__ __forceinline__ uint64_t make_desc_sw64(uint32_t saddr, uint32_t lbo_bytes, uint32_t sbo_bytes) {
  return (make_desc_sw128(saddr, lbo_bytes, sbo_bytes) & ~(7ull << 61)) | (4ull << 61);
}
// A ring's current slot and the parity of its fill.
template <int N>
struct Ring {
  uint32_t slot = 0, parity = 0;
  __device__ __forceinline__ void step() {
    if (++slot == uint32_t(N)) { slot = 0; parity ^= 1; }
  }
};
// One lane of a converged warp, chosen by the hardware: code under it stays warp-uniform for the
// compiler, so descriptors and addresses live in uniform registers.
__device__ __forceinline__ bool elect_one() {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok));
  return ok != 0;
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
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
// that its rows are written.  Keys behind the request's table row do not exist.
struct Request {
  int token0, n, len, lim, mt, kt;
};

template <int BN>
__device__ __forceinline__ Request load_request(const TreeParams& p, int j) {
  Request r;
  const int a = p.cu_q[j], b = p.cu_q[j + 1];
  r.token0 = a;
  r.n = (a >= 0 && b > a && b <= p.total_q) ? b - a : 0;
  r.len = max(p.seq_lens[j], 0);
  r.lim = int(min(int64_t(r.len), int64_t(p.max_pages) * p.page_size));
  r.mt = (r.n * p.group + BM - 1) / BM;  // total_q * Hq < 2^31
  r.kt = max(int((int64_t(r.lim) + BN - 1) / BN), 1);
  return r;
}

// Tiles are counted with ITEM_COST more for every row tile: `total` of them, of which CTA c of
// g takes the c-th equal part.
struct Share {
  int64_t t0, t1;        // this CTA's part
  int64_t total, each;   // each = total / g, the first `rest` CTAs take one more
  int g, rest;
  __device__ __forceinline__ int64_t begin(int c) const { return c * each + min(c, rest); }
  __device__ __forceinline__ int owner(int64_t x) const {  // the CTA whose part holds tile x
    const int64_t big = rest * (each + 1);
    return x < big ? int(x / (each + 1)) : rest + int((x - big) / each);
  }
};

// a / b, which are mostly below 2^32 (a 64-bit division takes four times as long).
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  return ((a | b) >> 32) == 0 ? int64_t(uint32_t(a) / uint32_t(b)) : a / b;
}

// Where a share begins: `off` counted tiles into a request.
struct Start {
  Request r;
  int seq;
  int64_t off;
};

// All threads of the CTA.  A thread sums a run of requests, a block scan gives its run's first
// tile, and the thread whose run holds t0 finds the request and leaves it in `found`.  (All this
// is a small batch's latency: each wait for global memory takes 700 cycles or so.)
template <int BN, int COST, int THREADS>
__device__ __forceinline__ Share find_share(const TreeParams& p, int c, int G, int64_t* ws, Start* found) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (p.nseq + THREADS - 1) / THREADS;
  const int j0 = min(tid * per, p.nseq), j1 = min(j0 + per, p.nseq);
  int64_t sum = 0;
  Request r{};
#pragma unroll 1
  for (int j = j0; j < j1; ++j) {
    r = load_request<BN>(p, j);
    sum += int64_t(p.Hkv * r.mt) * (r.kt + COST);
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
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    const int64_t x = ws[w];
    if (w < warp) before += x;
    total += x;
  }
  Share s;
  s.total = total;
  s.g = int(min(int64_t(G), total));  // no CTA has an empty share between others
  s.each = s.g > 0 ? quotient(total, s.g) : 0;
  s.rest = int(total - s.each * s.g);
  s.t0 = c < s.g ? s.begin(c) : total;
  s.t1 = c < s.g ? s.begin(c + 1) : total;
  int64_t first = before + inc - sum;
  if (s.t0 < s.t1 && first <= s.t0 && s.t0 < first + sum) {
#pragma unroll 1
    for (int j = j0; j < j1; ++j) {
      if (per > 1) r = load_request<BN>(p, j);
      const int64_t tiles = int64_t(p.Hkv * r.mt) * (r.kt + COST);
      if (s.t0 < first + tiles) {
        found->r = r;
        found->seq = j;
        found->off = s.t0 - first;
        break;
      }
      first += tiles;
    }
  }
  __syncthreads();
  return s;
}

// Walks a CTA's share item by item (warp 8).
template <int BN, int COST>
struct Walk {
  Request r;
  int64_t left;         // counted tiles left of the share, from the current position on
  int seq, kvh, mtile, at;  // position: `at` counted tiles into the row tile
  int kt0, nt;          // the key tiles of the current row tile that are this CTA's
  __device__ __forceinline__ void start(const Start& f, const Share& s) {
    seq = f.seq;
    left = s.t1 - s.t0;
    r = f.r;
    const int64_t item = quotient(f.off, r.kt + COST);
    at = int(f.off - item * (r.kt + COST));
    kvh = int(item) / r.mt;
    mtile = int(item) - kvh * r.mt;
  }
  // the next row tile with key tiles for this CTA; false at the end of the share
  __device__ __forceinline__ bool next(const TreeParams& p) {
    while (left > 0) {
      if (r.n > 0) {
        const int here = int(min(int64_t(r.kt + COST - at), left));
        kt0 = max(at - COST, 0);
        nt = max(at + here - COST, 0) - kt0;
        left -= here;
        at = 0;
        if (nt > 0) return true;
        advance(p);
      } else {
        if (seq + 1 >= p.nseq) return false;
        r = load_request<BN>(p, ++seq);
      }
    }
    return false;
  }
  __device__ __forceinline__ void advance(const TreeParams& p) {
    if (left <= 0) return;
    if (++mtile < r.mt) return;
    mtile = 0;
    if (++kvh < p.Hkv) return;
    kvh = 0;
    if (seq + 1 < p.nseq) r = load_request<BN>(p, ++seq);
    else left = 0;
  }
};

// ---------------------------------------------------------------------------
// masks
// ---------------------------------------------------------------------------
// 32 visibility bits of row-token `node` (global token `tok`) for keys [key, key + 32).
__device__ __forceinline__ uint32_t seen32(const TreeParams& p, int ctx, int lim, int64_t tok,
                                           int node, int key) {
  if (key >= lim) return 0u;
  const uint32_t inside = lim - key >= 32 ? 0xffffffffu : (1u << (lim - key)) - 1u;
  const int d = key - ctx;  // the keys' index among the new rows
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
// 16 elements of a bf16 query row x f as two e4m3 terms, 4 registers of 4 values each.  With
// the row's largest magnitude brought to [2^7, 2^8) the first term leaves at most half of its
// last place, which the second holds exactly (8 significant bits in all) down to 2^-10.
__device__ __forceinline__ void q16_terms(const uint4 a, const uint4 b, float f, uint32_t (&hi)[4],
                                          uint32_t (&lo)[4]) {
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    float v[4], h[4];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      v[2 * e] = __uint_as_float(w[2 * k + e] << 16) * f;
      v[2 * e + 1] = __uint_as_float(w[2 * k + e] & 0xFFFF0000u) * f;
    }
    hi[k] = pack_e4m3x4(v[0], v[1], v[2], v[3]);
    unpack_e4m3x4(hi[k], h[0], h[1], h[2], h[3]);
    lo[k] = pack_e4m3x4(v[0] - h[0], v[1] - h[1], v[2] - h[2], v[3] - h[3]);
  }
}

// Rows that see a key whose V row is not finite, after the finite part has been written to
// their row of the result (16-bit) or of a partial (fp32): the non-finite values themselves are
// added (their weight is positive): of every STEP blocks of 16 columns the one at `first`.  Rare;
// reads V again from the pool.
template <int D, int STEP>
__device__ __forceinline__ void add_nonfinite(const TreeParams& p, int seq, int kvh, int ctx, int lim,
                                              int64_t tok, int node, int key0, int64_t key1, int first,
                                              uint16_t* out_row, float* part_row) {
  const int end = int(min(key1, int64_t(lim)));
#pragma unroll 1
  for (int key = max(max(key0, ctx), 0); key < end; ++key) {
    if (!(seen32(p, ctx, lim, tok, node, key) & 1u)) continue;
    const int e = key / p.page_size;
    const int page = p.block_table[int64_t(seq) * p.max_pages + e];
    if (page < 0 || page >= p.num_pages) continue;
    const uint8_t* row = p.v + page * p.v_page + (key - e * p.page_size) * p.v_row + kvh * p.v_head;
#pragma unroll 1
    for (int d = first * 16; d < D; d += (d & 15) == 15 ? (STEP - 1) * 16 + 1 : 1) {
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
      if (part_row != nullptr) {
        __stcg(part_row + d, __ldcg(part_row + d) + x);
      } else {
        const float y = value16(out_row[d], p.out_bf16 != 0) + x;
        out_row[d] = uint16_t(p.out_bf16 ? pack_bf16x2(y, 0.f) : pack_f16x2(y, 0.f));
      }
    }
  }
}

template <class TR>
__global__ void __launch_bounds__(TR::THREADS, 1)
    tree_attn_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                     const TreeParams p) {
  constexpr int D = TR::D, BN = TR::BN, NWG = TR::NWG, W0 = TR::W0;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cta = int(blockIdx.x);

  const uint32_t bar0 = smem_u32(smem + TR::OFF_BAR);
  auto BAR = [&](int i) -> uint32_t { return bar0 + 8u * uint32_t(i); };
  auto k_full = [&](uint32_t i) { return BAR(int(i % TR::KS)); };
  auto k_empty = [&](uint32_t i) { return BAR(TR::KS + int(i % TR::KS)); };
  auto v_full = [&](uint32_t i) { return BAR(2 * TR::KS + int(i % TR::VS)); };
  auto v_empty = [&](uint32_t i) { return BAR(2 * TR::KS + TR::VS + int(i % TR::VS)); };
  constexpr int BR = 2 * (TR::KS + TR::VS), NR = TR::KV8 ? TR::RS : 1;
  auto r_full = [&](uint32_t i) { return BAR(BR + int(i % NR)); };
  auto r_empty = [&](uint32_t i) { return BAR(BR + TR::RS + int(i % NR)); };
  // parity of tile i's fill of a ring of n slots
  auto phase = [](uint32_t i, uint32_t n) { return (i / n) & 1u; };
  constexpr int B1 = BR + 2 * TR::RS, NB = TR::NB, B2 = B1 + 3 * NB;
  auto s_full = [&](uint32_t i) { return BAR(B1 + int(i % NB)); };
  auto p_full = [&](uint32_t i) { return BAR(B1 + NB + int(i % NB)); };
  auto o_done = [&](uint32_t i) { return BAR(B1 + 2 * NB + int(i % NB)); };
  auto max_known = [&](int wg, int w4) { return BAR(B2 + wg * 4 + w4); };
  auto v_fixed = [&](int wg) { return BAR(B2 + W0 + wg); };
  constexpr int B3 = B2 + 5 * NWG, B4 = B3 + 4;
  const uint32_t q_full = BAR(B3), o_free = BAR(B3 + 1), joined = BAR(B3 + 2), td_bar = BAR(B3 + 3);
  auto q_staged = [&](int i) { return BAR(B4 + i % kItems); };
  auto item_full = [&](int i) { return BAR(B4 + kItems + i % kItems); };
  auto item_free = [&](int i) { return BAR(B4 + 2 * kItems + i % kItems); };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + TR::OFF_MISC);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile uint32_t* bad = tmem_slot + 4;  // [warpgroups][2][4]: keys with a non-finite V row
  volatile float* row_max = reinterpret_cast<volatile float*>(smem + TR::OFF_ROWS);
  volatile float* end_max = row_max + BM;                // [2 items][warpgroups][BM]
  volatile float* end_sum = end_max + 2 * NWG * BM;
  volatile int* end_bad = reinterpret_cast<volatile int*>(end_sum + 2 * NWG * BM);
  Item* items = reinterpret_cast<Item*>(smem + TR::OFF_ITEMS);
  int* status = &g_tree_status;

  if (threadIdx.x == 32 * W0) {
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    for (int s = 0; s < TR::KS; ++s) {
      mbar_init(k_full(s), 1);
      mbar_init(k_empty(s), 1);
    }
    for (int s = 0; s < TR::VS; ++s) {
      mbar_init(v_full(s), TR::KV8 ? TR::CONV_TEAM : 1);
      mbar_init(v_empty(s), 1);
    }
    for (int s = 0; s < TR::RS; ++s) {
      mbar_init(r_full(s), 1);
      mbar_init(r_empty(s), TR::CONV_TEAM);
    }
    for (int b = 0; b < NB; ++b) {
      mbar_init(s_full(b), 1);
      mbar_init(p_full(b), 4);
      mbar_init(o_done(b), 1);
    }
    for (int g = 0; g < NWG; ++g) mbar_init(v_fixed(g), 4);
    for (int i = 0; i < W0; ++i) mbar_init(max_known(0, i), 1);
    mbar_init(q_full, W0);
    mbar_init(o_free, W0);
    mbar_init(joined, W0);
    mbar_init(td_bar, 2);
    for (int i = 0; i < kItems; ++i) {
      mbar_init(q_staged(i), 32);
      mbar_init(item_full(i), 1);
      mbar_init(item_free(i), W0 + 3 + TR::CONV_WARPS);  // softmax, V, S, PV, converters
    }
    *abort = 0;
    fence_mbar_init();
  }
  if (threadIdx.x == 0) p.desc[2 * cta] = make_int4(0, 0, 0, 0);  // this thread names a split row tile later
  if (warp == W0 + 1) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  // (two __syncthreads; the scratch lies where the K ring will be: warp W0, which reads it last,
  // fills the ring)
  int64_t* sched = reinterpret_cast<int64_t*>(smem);
  Start* found = reinterpret_cast<Start*>(sched + 32);
  const Share share = find_share<BN, TR::ITEM_COST, TR::THREADS>(p, cta, int(gridDim.x), sched, found);
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // The i-th item, for the other roles' warps; false at the end of the share or on give-up.
  auto get_item = [&](int i, Item& x) -> bool {
    const bool ok = mbar_wait(item_full(i), uint32_t(i / kItems) & 1, abort, kErrItem, status);
    if (!__all_sync(0xffffffffu, ok)) return false;
    x = items[i % kItems];
    __syncwarp();
    if (lane == 0) mbar_arrive(item_free(i));
    return x.nt > 0;
  };

  if (share.t0 >= share.t1) {
    // no work (uniform for the CTA): on to the release of TMEM
  } else if (warp >= W0 + 4) {
    if constexpr (TR::KV8) {
      // ---------------------------------------------------------- V: e4m3 -> f16
      // Each 16-byte piece becomes two pieces of the swizzled operand tile.  (Moving the bits with
      // integer instructions instead takes three times as many of them: 423 us against 388, e4m3,
      // head_dim 128, 32 requests of 64 tokens and up to 16K cached.)  Eight lanes take the 64-byte
      // halves of two rows crosswise (row r from chunk a, row r + 1 from chunk a ^ 1), so neither
      // the reads nor the writes meet in a bank.
      setmaxnreg_dec<TR::REGS_CONV>();
      constexpr int TEAM = TR::CONV_TEAM, TEAMS = 4 / TEAM;
      const int team = (warp - W0 - 4) / TEAM, t = (warp - W0 - 4) % TEAM * 32 + lane;
      const int half = (t & 7) >> 2, piece = t & 3, unit = t >> 3;
      const int row0 = unit / TR::V_COLS * 2 + half, a = unit % TR::V_COLS;
      const int ch = TR::V_COLS > 1 && half ? a ^ 1 : a;
      const uint8_t* src0 = smem + TR::OFF_RAW + row0 * D + ch * 64 + piece * 16;
      uint8_t* dst0 = smem + TR::OFF_V + ch * TR::V_CHUNK + row0 * 128;
      constexpr int PIECES = BN * D / 16 / (32 * TEAM);  // 16-byte pieces a thread
      constexpr int STEP = 8 * TEAM / TR::V_COLS;        // rows from one to the next
      uint32_t i = 0;
      Item x;
      for (int item = 0; get_item(item, x); ++item) {
        bool ok = true;
        for (int j = 0; j < x.nt; ++j, ++i) {
          if (int(i % TEAMS) != team) continue;
          ok = mbar_wait(r_full(i), phase(i, NR), abort, kErrRawFull, status) &&
               mbar_wait(v_empty(i), phase(i, TR::VS) ^ 1, abort, kErrVEmpty, status);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          const uint8_t* src = src0 + (i % NR) * TR::RAW_BYTES;
          uint8_t* dst = dst0 + (i % TR::VS) * TR::V_BYTES;
#pragma unroll 1
          for (int u0 = 0; u0 < PIECES; u0 += 4) {
            uint4 in[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) in[u] = *reinterpret_cast<const uint4*>(src + (u0 + u) * STEP * D);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const uint32_t w[4] = {in[u].x, in[u].y, in[u].z, in[u].w};
              uint32_t o[8];
#pragma unroll
              for (int k = 0; k < 4; ++k)
                asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
                    "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
                    : "=r"(o[2 * k]), "=r"(o[2 * k + 1])
                    : "r"(w[k]));
              const int row = row0 + (u0 + u) * STEP;
              uint8_t* to = dst + (u0 + u) * STEP * 128;
              const int at = ((2 * piece) ^ (row & 7)) * 16;
              *reinterpret_cast<uint4*>(to + at) = make_uint4(o[0], o[1], o[2], o[3]);
              *reinterpret_cast<uint4*>(to + (at ^ 16)) = make_uint4(o[4], o[5], o[6], o[7]);
            }
          }
          fence_async_shared();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(r_empty(i));
            mbar_arrive(v_full(i));
          }
        }
        if (!ok) break;
      }
    }
  } else if (warp >= W0) {
    setmaxnreg_dec<TR::REGS_CONTROL>();
    if (warp == W0 || warp == W0 + 2) {
      // ---------------------------------------------------------- producers
      // a lane copies one (page piece, swizzled column) of a tile
      const bool is_v = warp == W0 + 2;
      const int slots = is_v ? (TR::KV8 ? TR::RS : TR::VS) : TR::KS;
      const int bytes = is_v ? (TR::KV8 ? TR::RAW_BYTES : TR::V_BYTES) : TR::K_BYTES;
      const int cols = is_v ? (TR::KV8 ? 1 : TR::V_COLS) : TR::K_COLS;
      const int width = is_v && TR::KV8 ? D : is_v ? 128 : TR::K_SWZ;  // bytes of a column's row
      const int first_full = is_v ? (TR::KV8 ? BR : 2 * TR::KS) : 0;
      const CUtensorMap* map = is_v ? &tmV : &tmK;
      const int box = min(p.page_size, BN);
      const int piece = lane / cols, col = lane - piece * cols;
      const bool mine = piece < BN / box;
      const uint32_t base = smem_u32(smem) + uint32_t(is_v ? (TR::KV8 ? TR::OFF_RAW : TR::OFF_V) : 0) +
                            uint32_t(col * BN * width + piece * box * width);
      const int c0 = col * width / TR::KEL;
      uint32_t idx = 0, slot = 0, ph = 0;
      auto step = [&]() {
        ++idx;
        if (++slot == uint32_t(slots)) { slot = 0; ph ^= 1; }
      };
      auto wait_slot = [&]() -> bool {
        const bool got = idx < uint32_t(slots) ||
                         mbar_wait(BAR(first_full + slots + int(slot)), ph ^ 1, abort, kErrEmpty, status);
        return __all_sync(0xffffffffu, got);
      };
      Walk<BN, TR::ITEM_COST> w;
      bool more = true;
      if (!is_v) {
        w.start(*found, share);
        __syncwarp();
        more = w.next(p);
      }
      bool ok = true;
      for (int item = 0; ok; ++item) {
        Item x;
        int row = 0, page = -1;
        // the page and row of this lane's piece of tile kt; -1 (zeros) where the cache has ended
        auto lookup = [&](int kt, int& row) -> int {
          const int64_t key = int64_t(kt) * BN + piece * box;
          if (!mine || key >= x.lim) { row = 0; return -1; }
          const int e = int(key) / p.page_size;
          row = int(key) - e * p.page_size;
          return p.block_table[int64_t(x.seq) * p.max_pages + e];
        };
        if (is_v) {
          if (!get_item(item, x)) break;
          page = lookup(x.kt0, row);
        } else {
          // publish the item
          if (item >= kItems)
            ok = mbar_wait(item_free(item), (uint32_t(item / kItems) & 1) ^ 1, abort, kErrItemFree, status);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          x.nt = 0;
          int rows = 0;
          constexpr int Q_ROW = D * 2;  // bytes of a bf16 / f16 row (e4m3: half)
          const int q_row = p.q_dtype == FA4CP_DTYPE_E4M3 ? D : Q_ROW;
          if (more) {
            x.seq = w.seq; x.token0 = w.r.token0; x.n = w.r.n; x.len = w.r.len; x.lim = w.r.lim;
            x.kvh = w.kvh; x.mtile = w.mtile; x.kt0 = w.kt0; x.nt = w.nt; x.kt = w.r.kt;
            x.k_idx = idx;
            rows = min(BM, w.r.n * p.group - w.mtile * BM);
            x.q_slots = (rows * q_row + TR::K_BYTES - 1) / TR::K_BYTES;
          }
          if (lane == 0) {
            items[item % kItems] = x;
            mbar_arrive(item_full(item));
          }
          if (!more) break;
          page = lookup(x.kt0, row);  // (read while Q is fetched)
          // its Q rows: 16-byte pieces, swizzled by the row so that a thread a row reads them
          // without bank conflicts
          const int per_row = q_row / 16, rows_step = 32 / per_row;  // per_row: 4 .. 32
          const int per_slot = TR::K_BYTES / q_row;
          const int c = lane & (per_row - 1);
          int q = lane / per_row;
          const int packed = x.mtile * BM + q;
          int node = packed / p.group, g = packed - node * p.group;
          for (int s = 0; ok && s < x.q_slots; ++s) {
            ok = wait_slot();
            if (!ok) break;
            const uint32_t dst = smem_u32(smem) + slot * uint32_t(TR::K_BYTES);
            const int end = min(rows, (s + 1) * per_slot);
#pragma unroll 1
            for (; q < end; q += rows_step) {
              const uint8_t* src = p.q + (int64_t(x.token0) + node) * p.q_stride +
                                   int64_t(x.kvh * p.group + g) * q_row + c * 16;
              const uint32_t to = dst + uint32_t((q - s * per_slot) * q_row + ((c ^ (q & 7 & (per_row - 1))) * 16));
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(src) : "memory");
              g += rows_step;
              while (g >= p.group) { g -= p.group; ++node; }
            }
            if (lane == 0) mbar_arrive(BAR(first_full + int(slot)));  // (Q's arrival is q_staged's)
            step();
          }
          if (!ok) break;
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(q_staged(item)) : "memory");
        }
        for (int j = 0; j < x.nt; ++j) {
          int nrow = 0, npage = -1;  // asked for before this tile waits for its slot
          if (j + 1 < x.nt) npage = lookup(x.kt0 + j + 1, nrow);
          ok = wait_slot();
          if (!ok) break;
          const uint32_t full = BAR(first_full + int(slot));
          if (lane == 0) mbar_arrive_expect_tx(full, uint32_t(bytes));
          __syncwarp();
          const bool inside = page >= 0 && page < p.num_pages;
          if (mine) tma_load_4d(base + slot * uint32_t(bytes), map, c0, x.kvh, row, inside ? page : -1, full);
          step();
          row = nrow;
          page = npage;
        }
        if (!is_v && ok) {
          w.advance(p);
          more = w.next(p);
        }
      }
      // every copy that was issued has landed before the CTA ends (on the normal path the
      // consumers have waited for them)
      asm volatile("cp.async.wait_all;" ::: "memory");
      for (uint32_t i = idx > uint32_t(slots) ? idx - slots : 0; i < idx; ++i)
        mbar_wait_drain(BAR(first_full + int(i % slots)), (i / slots) & 1, kErrDrain, status);
    } else {
      // ---------------------------------------------------------- MMA issuers
      // A warp walks the tiles together and one elected lane issues: descriptors then stay in
      // uniform registers (issuing from one lane's own branch took 1.3 times as long).
      const int fmt = p.kv_dtype == FA4CP_DTYPE_BF16 ? 1 : 0;  // (e4m3 is format 0, and V is f16)
      const uint32_t ring = smem_u32(smem);
      // The loop is what a tile takes here (about 900 cycles when it divided its ring indices), so
      // slots and parities are carried along.  A tile waits for two barriers: one after the other,
      // or, at head_dim 64, by a lane each (e4m3, 64 tokens and one: 282 and 145 us against 300 and
      // 152; at head_dim 128 385 and 175 against 346 and 153).
      auto wait_two = [&](uint32_t bar_a, uint32_t par_a, int code_a, uint32_t bar_b, uint32_t par_b, int code_b) -> bool {
        bool ok;
        if constexpr (D == 64) {
          const bool a = lane == 0;
          ok = mbar_wait(a ? bar_a : bar_b, a ? par_a : par_b, abort, a ? code_a : code_b, status);
        } else {
          ok = mbar_wait(bar_a, par_a, abort, code_a, status) && mbar_wait(bar_b, par_b, abort, code_b, status);
        }
        return __all_sync(0xffffffffu, ok);
      };
      Item x;
      if (warp == W0 + 1) {
        const uint32_t idesc = make_idesc(BM, BN, fmt, fmt, 0, 0);
        const int q_terms = TR::KV8 && p.q_dtype != FA4CP_DTYPE_E4M3 ? 2 : 1;
        // 32 bytes along D a step, then the next swizzled column
        constexpr int STEPS = D * TR::KEL / 32, PER_COL = TR::K_SWZ / 32;
        const uint64_t desc0 = TR::K_SWZ == 128 ? make_desc_sw128(ring, 16, 1024) : make_desc_sw64(ring, 16, 512);
        const uint32_t a = tmem + uint32_t(TR::TM_Q);
        Ring<TR::KS> k;
        Ring<NB> sb;
        for (int item = 0; get_item(item, x); ++item) {
          bool ok = __all_sync(0xffffffffu, mbar_wait(q_full, uint32_t(item) & 1, abort, kErrQFull, status));
          if (!ok) break;
          if (lane < x.q_slots) mbar_arrive(k_empty(x.k_idx + lane));  // Q has been read
          for (int i = 0; i < x.q_slots; ++i) k.step();
          for (int j = 0; j < x.nt; ++j) {
            // the P over the buffer's last S has been multiplied (a buffer's first use waits for a
            // phase that counts as complete), and the K tile is there
            ok = wait_two(BAR(B1 + 2 * NB + int(sb.slot)), sb.parity ^ 1, kErrSFree, BAR(int(k.slot)), k.parity, kErrKFull);
            if (!ok) break;
            tc_fence_after();
            const uint64_t desc = desc0 + uint64_t(k.slot * uint32_t(TR::K_BYTES / 16));
            const uint32_t d = tmem + uint32_t(TR::TM_S) + sb.slot * BN;
            if (elect_one()) {
              if constexpr (TR::KV8) {
#pragma unroll
                for (int kk = 0; kk < STEPS; ++kk)
                  mma_f8_ts(d, a + uint32_t(kk * 8), desc + uint64_t((kk / PER_COL * BN * TR::K_SWZ + kk % PER_COL * 32) / 16),
                            idesc, kk > 0 ? 1u : 0u);
                if (q_terms == 2) {
#pragma unroll
                  for (int kk = 0; kk < STEPS; ++kk)
                    mma_f8_ts(d, a + uint32_t(D / 4 + kk * 8),
                              desc + uint64_t((kk / PER_COL * BN * TR::K_SWZ + kk % PER_COL * 32) / 16), idesc, 1u);
                }
              } else {
#pragma unroll
                for (int kk = 0; kk < STEPS; ++kk)
                  mma_f16_ts(d, a + uint32_t(kk * 8), desc + uint64_t((kk / PER_COL * BN * TR::K_SWZ + kk % PER_COL * 32) / 16),
                             idesc, kk > 0 ? 1u : 0u);
              }
              tc_commit(BAR(B1 + int(sb.slot)));
              tc_commit(BAR(TR::KS + int(k.slot)));
            }
            __syncwarp();
            k.step();
            sb.step();
          }
          if (!ok) break;
        }
      } else {
        const uint32_t idesc = make_idesc(BM, D, fmt, fmt, 0, 1);
        const uint64_t desc0 = make_desc_sw128(ring + TR::OFF_V, TR::V_CHUNK, 1024);
        Ring<TR::VS> v;
        Ring<NB> sb;
        Ring<TR::APART ? NWG : 1> ob;
        for (int item = 0; get_item(item, x); ++item) {
          bool ok = true;
          if (item > 0)
            ok = __all_sync(0xffffffffu, mbar_wait(o_free, uint32_t(item - 1) & 1, abort, kErrOFree, status));
          for (int j = 0; ok && j < x.nt; ++j) {
            ok = wait_two(BAR(2 * TR::KS + int(v.slot)), v.parity, kErrVFull, BAR(B1 + NB + int(sb.slot)), sb.parity, kErrPFull);
            if (!ok) break;
            tc_fence_after();
            const uint64_t desc = desc0 + uint64_t(v.slot * uint32_t(TR::V_BYTES / 16));
            const uint32_t o = tmem + uint32_t(TR::TM_O) + ob.slot * D, a = tmem + uint32_t(TR::TM_S) + sb.slot * BN;
            if (elect_one()) {
#pragma unroll
              for (int kk = 0; kk < BN / 16; ++kk)  // 16 keys: 16 rows of 128 bytes further
                mma_f16_ts(o, a + uint32_t(kk * 8), desc + uint64_t(kk * 16 * 128 / 16), idesc,
                           (j >= (TR::APART ? NWG : 1) || kk > 0) ? 1u : 0u);
              tc_commit(BAR(B1 + 2 * NB + int(sb.slot)));
              tc_commit(BAR(2 * TR::KS + TR::VS + int(v.slot)));
            }
            __syncwarp();
            v.step();
            sb.step();
            ob.step();
          }
          if (!ok) break;
        }
      }
      // every MMA issued above has completed before TMEM is released
      if (elect_one()) tc_commit(td_bar);
      __syncwarp();
      mbar_wait_drain(td_bar, 0, kErrDrain, status);
    }
  } else {
    // ------------------------------------------------------------ softmax + epilogue
    setmaxnreg_inc<TR::REGS_SOFTMAX>();
    const int wg = warp >> 2, w4 = warp & 3;
    const int t = threadIdx.x & 127;  // row of the tile
    const uint32_t t_lane = tmem + (uint32_t(w4 * 32) << 16);
    const uint32_t t_o = t_lane + uint32_t(TR::TM_O + (TR::APART ? wg * D : 0));
    const bool bf16_op = p.kv_dtype == FA4CP_DTYPE_BF16;
    const bool q8 = p.q_dtype == FA4CP_DTYPE_E4M3;
    // One arrival a warp, for its lanes' TMEM (and shared memory) accesses so far.
    auto warp_arrive = [&](uint32_t bar) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    float qf = 1.f;  // the row's factor (e4m3 cache): a power of two, with the descales' sign

    // This warpgroup's half of item `x`'s Q into TMEM.  All S MMAs of the item before are
    // complete (the caller has seen its last s_full).
    auto load_q = [&](const Item& x, int item) -> bool {
      const bool ok = mbar_wait(q_staged(item), uint32_t(item / kItems) & 1, abort, kErrQStaged, status);
      if (!__all_sync(0xffffffffu, ok)) return false;
      const int rows = min(BM, x.n * p.group - x.mtile * BM);
      // Lanes without a row hold zeros (or an older item's rows).  Nothing reads what they give, but
      // decode leaves most of a tile empty, the GPU is at its power limit in it, and MMAs of zeros
      // draw less: 64 requests of 1K to 32K tokens, bf16, in a row: 697 us, with what lay there 737.
      if (w4 * 32 < rows) {  // the warp has rows
        const int row = min(t, rows - 1);
        const int q_row = q8 ? D : 2 * D, per_slot = TR::K_BYTES / q_row;
        const int s = row / per_slot, swz = row & 7 & (q_row / 16 - 1);
        const uint8_t* src = smem + (x.k_idx + s) % TR::KS * TR::K_BYTES + (row - s * per_slot) * q_row;
        auto piece = [&](int c) { return *reinterpret_cast<const uint4*>(src + ((c ^ swz) * 16)); };
        float mul = 1.f;
        if constexpr (TR::KV8) {
          int e = 0;
          bool finite = true;
          if (!q8) {
            uint32_t top = 0;  // largest magnitude, as bits of a bf16
#pragma unroll 4
            for (int c = 0; c < D / 8; ++c) {
              const uint4 v = piece(c);
              top = __vmaxu2(top, __vmaxu2(__vmaxu2(v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu),
                                           __vmaxu2(v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu)));
            }
            const int exp = int(max(top & 0xFFFFu, top >> 16)) >> 7;
            finite = exp != 255;
            if (exp != 0 && finite) e = min(127 + 7 - exp, 126);
          }
          qf = __uint_as_float(uint32_t(127 + e) << 23);
          // a row with infinities or NaN is NaN all over
          mul = finite ? qf : __uint_as_float(0x7FC00000u);
          if ((p.q_descale ? p.q_descale[x.kvh] : 1.f) * (p.k_descale ? p.k_descale[x.kvh] : 1.f) < 0.f) {
            qf = -qf;
            mul = -mul;
          }
        }
#pragma unroll 1
        for (int c = wg; c < D / 32; c += NWG) {  // 32 elements
          if constexpr (TR::KV8) {
            uint32_t hi[8], lo[8];
            if (q8) {
              const uint32_t flip = mul < 0.f ? 0x80808080u : 0u;
              const uint4 a = piece(2 * c), b = piece(2 * c + 1);
              hi[0] = a.x ^ flip; hi[1] = a.y ^ flip; hi[2] = a.z ^ flip; hi[3] = a.w ^ flip;
              hi[4] = b.x ^ flip; hi[5] = b.y ^ flip; hi[6] = b.z ^ flip; hi[7] = b.w ^ flip;
            } else {
              uint32_t h[4], o[4];
              q16_terms(piece(4 * c), piece(4 * c + 1), mul, h, o);
#pragma unroll
              for (int k = 0; k < 4; ++k) { hi[k] = h[k]; lo[k] = o[k]; }
              q16_terms(piece(4 * c + 2), piece(4 * c + 3), mul, h, o);
#pragma unroll
              for (int k = 0; k < 4; ++k) { hi[4 + k] = h[k]; lo[4 + k] = o[k]; }
              if (t >= rows) {
#pragma unroll
                for (int k = 0; k < 8; ++k) lo[k] = 0;
              }
              tmem_st8(t_lane + uint32_t(TR::TM_Q + D / 4 + c * 8), lo);
            }
            if (t >= rows) {
#pragma unroll
              for (int k = 0; k < 8; ++k) hi[k] = 0;
            }
            tmem_st8(t_lane + uint32_t(TR::TM_Q + c * 8), hi);
          } else {
            uint32_t r[16];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint4 v = piece(4 * c + k);
              r[4 * k] = v.x; r[4 * k + 1] = v.y; r[4 * k + 2] = v.z; r[4 * k + 3] = v.w;
            }
            if (t >= rows) {
#pragma unroll
              for (int k = 0; k < 16; ++k) r[k] = 0;
            }
            tmem_st16(t_lane + uint32_t(TR::TM_Q + c * 16), r);
          }
        }
        tmem_wait_st();
      } else if (item == 0) {
        const uint32_t zero[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll 1
        for (int c = wg; c < D / 16; c += NWG) tmem_st8(t_lane + uint32_t(TR::TM_Q + c * 8), zero);
        tmem_wait_st();
      }
      warp_arrive(q_full);
      return true;
    };

    Item x;
    uint32_t it0 = 0, fixes = 0;  // the item's first tile, counted over the share
    int item = 0;
    bool ok = true;
    bool more = get_item(0, x), aborted = false;
    if (more) more = load_q(x, 0);
    while (more) {
      const int n = x.nt;
      const int rows = min(BM, x.n * p.group - x.mtile * BM);
      const bool active = w4 * 32 < rows;
      const bool valid = t < rows;
      const int packed = x.mtile * BM + (valid ? t : 0);
      const int node = packed / p.group;
      const int head = x.kvh * p.group + (packed - node * p.group);
      const int64_t tok = int64_t(x.token0) + node;
      const int ctx = x.len - x.n;
      float scale = p.scale_log2, vscale = 1.0f;
      if (TR::KV8) {
        if (p.q_descale) scale *= p.q_descale[x.kvh];
        if (p.k_descale) scale *= p.k_descale[x.kvh];
        if (p.v_descale) vscale = p.v_descale[x.kvh];
        // qf carries the sign of the descales, so the scale is positive; never 0, so that a
        // masked score stays -inf
        scale /= qf;
        scale = scale < 1.17549435e-38f ? 1.17549435e-38f : scale;
      }
      const float lift = !TR::KV8 && bf16_op ? 0.f : kLiftF16;
      // m: the maximum that this warpgroup's sum l (and its O) are relative to
      float m = kNegInf, l = 0.f;
      bool sees_bad = false;
      for (int j = int((uint32_t(wg) + NWG - it0 % NWG) % NWG); j < n; j += NWG) {
        const uint32_t it = it0 + j;
        ok = mbar_wait(s_full(it), phase(it, NB), abort, kErrSFull, status);
        if (!__all_sync(0xffffffffu, ok)) { aborted = true; break; }
        tc_fence_after();
        const int kbase = (x.kt0 + j) * BN;
        // new rows, or the cache's end (kbase + BN may be 2^31)
        const bool edge = ctx - kbase < BN || x.lim - kbase < BN;
        const uint32_t t_s = t_lane + uint32_t(TR::TM_S) + it % NB * BN;
        constexpr int C = BN / 32;
        uint32_t vis[C];
#pragma unroll
        for (int c = 0; c < C; ++c) vis[c] = 0u;
        // the tile before has settled the maximum (the other warpgroup's tile)
        auto max_settled = [&]() -> bool {
          return it == 0 || __all_sync(0xffffffffu, mbar_wait(max_known((wg + NWG - 1) % NWG, w4), phase(it - 1, NWG), abort,
                                                              kErrMax, status));
        };
        if (active) {
          uint32_t sr[C][32];
#pragma unroll
          for (int c = 0; c < C; ++c) tmem_ld32(t_s + uint32_t(c * 32), sr[c]);
          tmem_wait_ld();
#pragma unroll
          for (int c = 0; c < C; ++c) reg_fence32(sr[c]);
          if (edge) {
#pragma unroll
            for (int c = 0; c < C; ++c) {
              vis[c] = seen32(p, ctx, x.lim, tok, node, kbase + c * 32);
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!((vis[c] >> e) & 1u)) sr[c][e] = __float_as_uint(kNegInf);
            }
          }
          float mx4[4] = {kNegInf, kNegInf, kNegInf, kNegInf};
#pragma unroll
          for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < 32; e += 8)
#pragma unroll
              for (int k = 0; k < 4; ++k)
                mx4[k] = fmax3(mx4[k], __uint_as_float(sr[c][e + 2 * k]), __uint_as_float(sr[c][e + 2 * k + 1]));
          const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
          // the maximum is raised only when it would grow by more than 2^8, or comes to exist
          float so_far = kNegInf;
          if constexpr (TR::APART) {
            so_far = m;
          } else {
            if (!max_settled()) { aborted = true; break; }
            if (j > 0) so_far = row_max[t];
          }
          const bool raise = so_far == kNegInf ? mx != kNegInf
                                               : (mx - so_far) * scale >
                                                     (fabsf(mx) * scale < kExactBelow ? kRescaleThreshold : 0.f);
          const float m_new = raise ? mx : so_far;
          if constexpr (!TR::APART) {
            row_max[t] = m_new;
            __syncwarp();
            if (lane == 0) mbar_arrive(max_known(wg, w4));
          }
          // from here on off the other warpgroup's way
          if (m_new != m) {
            if (m != kNegInf) l *= ex2_approx((m - m_new) * scale);
            m = m_new;
          }
          constexpr int MINE = TR::APART ? NWG : 1;  // PV(it - MINE) was the last one into this O
          if (j >= MINE && __any_sync(0xffffffffu, raise)) {
            const float f = !raise ? 1.f : so_far == kNegInf ? 0.f : ex2_approx((so_far - m_new) * scale);
            ok = mbar_wait(o_done(it - MINE), phase(it - MINE, NB), abort, kErrODone, status);
            if (!__all_sync(0xffffffffu, ok)) { aborted = true; break; }
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D / 16; ++c) {
              uint32_t o[16];
              tmem_ld16(t_o + uint32_t(c * 16), o);
              tmem_wait_ld();
              reg_fence16(o);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st16(t_o + uint32_t(c * 16), o);
            }
          }
          // (P = 0 in a lane without a row, for the same reason)
          const float neg_m = (!valid ? kNegInf : (m == kNegInf) ? 0.f : -m * scale) + lift;
          const uint64_t scale2 = f2pack(scale, scale), negm2 = f2pack(neg_m, neg_m);
          uint64_t rs[2] = {0ull, 0ull};
          uint32_t pw[C][16];
#pragma unroll
          for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const uint64_t y = ffma2(f2pack(__uint_as_float(sr[c][2 * i]), __uint_as_float(sr[c][2 * i + 1])), scale2, negm2);
              const float x0 = ex2_approx(f2lo(y)), x1 = ex2_approx(f2hi(y));
              rs[i & 1] = fadd2(rs[i & 1], f2pack(x0, x1));
              pw[c][i] = !TR::KV8 && bf16_op ? pack_bf16x2(x0, x1) : pack_f16x2(x0, x1);
            }
#pragma unroll
          for (int c = 0; c < C; ++c) tmem_st16(t_s + uint32_t(c * 16), pw[c]);
          const uint64_t rsum = fadd2(rs[0], rs[1]);
          l += f2lo(rsum) + f2hi(rsum);
        } else if (!TR::APART) {
          if (!max_settled()) { aborted = true; break; }
          if (lane == 0) mbar_arrive(max_known(wg, w4));
        }
        if (edge) {
          // P is 0 where a row does not look, but 0 * NaN is NaN: V rows behind the cache are
          // cleared, and so are the non-finite values of new rows that some token may not see (a
          // context row is seen by every token, and one token without a mask sees itself, so
          // their values go through as they are).  Thread t has key t % BN, and its share of the
          // columns.
          const bool hides = x.n > 1 || p.mask != nullptr;
          ok = mbar_wait(v_full(it), phase(it, TR::VS), abort, kErrVFix, status);
          if (!__all_sync(0xffffffffu, ok)) { aborted = true; break; }
          constexpr int PER = D / 8 * BN / 128;  // 16-byte pieces of a thread
          const int key = kbase + (t & (BN - 1));
          uint8_t* vrow = smem + TR::OFF_V + (it % TR::VS) * TR::V_BYTES + (t & (BN - 1)) * 128;
          bool mine_bad = false;
          if (key >= x.lim || (key >= ctx && hides)) {
#pragma unroll 1
            for (int c = t / BN * PER; c < (t / BN + 1) * PER; ++c) {
              uint4* at = reinterpret_cast<uint4*>(vrow + (c >> 3) * TR::V_CHUNK + (c & 7) * 16);
              const uint4 v = *at;
              uint32_t y[4] = {v.x, v.y, v.z, v.w};
              bool hit = key >= x.lim;
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                if (key >= x.lim) y[k] = 0;
                if (nonfinite16(y[k] & 0xFFFFu, bf16_op)) { y[k] &= 0xFFFF0000u; hit = mine_bad = true; }
                if (nonfinite16(y[k] >> 16, bf16_op)) { y[k] &= 0xFFFFu; hit = mine_bad = true; }
              }
              if (hit) *at = make_uint4(y[0], y[1], y[2], y[3]);
            }
          }
          __syncwarp();
          fence_async_shared();
          if (hides) {
            // which keys of the tile were cleared: one word a warp, two sets used in turn
            const uint32_t word = __ballot_sync(0xffffffffu, mine_bad);
            volatile uint32_t* set = bad + wg * 8 + (fixes & 1) * 4;
            if (lane == 0) {
              set[w4] = word;
              mbar_arrive(v_fixed(wg));
            }
            ok = mbar_wait(v_fixed(wg), fixes & 1, abort, kErrVFix, status);
            if (!__all_sync(0xffffffffu, ok)) { aborted = true; break; }
            ++fixes;
#pragma unroll
            for (int i = 0; i < 4; ++i) sees_bad |= active && (set[i] & vis[i % C]) != 0;
          }
        }
        if (active) tmem_wait_st();
        warp_arrive(p_full(it));
      }
      if (aborted) break;

      // what the other warpgroups need to finish the row
      const uint32_t last = it0 + n - 1;
      const int set = (item & 1) * NWG;
      end_max[(set + wg) * BM + t] = m;
      end_sum[(set + wg) * BM + t] = l;
      end_bad[(set + wg) * BM + t] = sees_bad;
      __syncwarp();
      if (lane == 0) mbar_arrive(joined);

      // the next item's Q goes in before this item's epilogue, so its first S starts meanwhile
      ok = mbar_wait(s_full(last), phase(last, NB), abort, kErrSFull, status);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      Item y;
      more = get_item(item + 1, y);
      if (more && !load_q(y, item + 1)) break;

      ok = mbar_wait(joined, uint32_t(item) & 1, abort, kErrJoin, status);
      if (ok) ok = mbar_wait(o_done(last), phase(last, NB), abort, kErrODone, status);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      // Apart: O = f0 O0 + f1 O1.  Shared: O is relative to the last tile's maximum.
      float part_f[NWG];
#pragma unroll
      for (int g = 0; g < NWG; ++g) part_f[g] = end_max[(set + g) * BM + t];
      m = end_max[(set + last % NWG) * BM + t];
      if (TR::APART) {
#pragma unroll
        for (int g = 0; g < NWG; ++g) m = fmaxf(m, part_f[g]);
      }
      l = 0.f;
#pragma unroll
      for (int g = 0; g < NWG; ++g) {
        const float lg = end_sum[(set + g) * BM + t], mg = part_f[g];
        part_f[g] = mg == m ? 1.f : mg == kNegInf ? 0.f : ex2_approx((mg - m) * scale);
        l += mg == kNegInf ? lg : lg * part_f[g];  // (NaN sums have no maximum)
        sees_bad |= end_bad[(set + g) * BM + t] != 0;
      }
      const bool whole = n == x.kt;
      const int part = 2 * cta + (x.kt0 == 0 ? 1 : 0);
      const float mult = whole ? (l == 0.f ? 0.f : vscale / l) : vscale;
      uint16_t* out_row = static_cast<uint16_t*>(p.out) + (tok * p.Hq + head) * D;
      float* prow = p.part_o + (int64_t(part) * BM + t) * D;
      if (active) {
#pragma unroll 1
        for (int c = wg; c < D / 16; c += NWG) {
          uint32_t o[16];
          float f[16];
          const uint32_t from = t_lane + uint32_t(TR::TM_O + c * 16);
          tmem_ld16(from, o);
          if constexpr (TR::APART) {
            uint32_t o1[16];
            tmem_ld16(from + D, o1);
            tmem_wait_ld();
            reg_fence16(o);
            reg_fence16(o1);
            // a warpgroup without a tile of the item left an older item's O
            const bool h0 = n > 1 || last % NWG == 0, h1 = n > 1 || last % NWG == 1;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float y = h0 ? __uint_as_float(o[e]) * part_f[0] : 0.f;
              o[e] = __float_as_uint(h1 ? fmaf(__uint_as_float(o1[e]), part_f[1], y) : y);
            }
          } else {
            tmem_wait_ld();
            reg_fence16(o);
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) f[e] = __uint_as_float(o[e]) * mult;
          if (valid) {
            if (whole) {
              uint32_t h[8];
#pragma unroll
              for (int e = 0; e < 8; ++e)
                h[e] = p.out_bf16 ? pack_bf16x2(f[2 * e], f[2 * e + 1]) : pack_f16x2(f[2 * e], f[2 * e + 1]);
              uint4* dst = reinterpret_cast<uint4*>(out_row + c * 16);
              dst[0] = make_uint4(h[0], h[1], h[2], h[3]);
              dst[1] = make_uint4(h[4], h[5], h[6], h[7]);
            } else {
              float4* dst = reinterpret_cast<float4*>(prow + c * 16);
#pragma unroll
              for (int e = 0; e < 4; ++e) __stcg(dst + e, make_float4(f[4 * e], f[4 * e + 1], f[4 * e + 2], f[4 * e + 3]));
            }
          }
          __syncwarp();  // the next loads from TMEM are the whole warp's
        }
      }
      warp_arrive(o_free);
      if (valid) {
        const float ms = m == kNegInf ? kNegInf : __fmul_rn(m, scale) - lift;
        if (wg == 0) {
          if (whole) p.lse[tok * p.Hq + head] = l == 0.f ? kNegInf : (ms + lg2_approx(l)) * kLn2;
          else __stcg(&p.part_ml[part * BM + t], make_float2(ms, l));
        }
        if (sees_bad)
          add_nonfinite<D, NWG>(p, x.seq, x.kvh, ctx, x.lim, tok, node, x.kt0 * BN, int64_t(x.kt0 + n) * BN, wg,
                                out_row, whole ? nullptr : prow);
      }
      if (threadIdx.x == 0 && !more && x.kt0 == 0 && !whole) {
        // the share's last item began here and goes on: this CTA's descriptor names it, and the
        // CTA that its last tile belongs to
        p.desc[2 * cta] = make_int4(1, share.owner(share.t1 + (x.kt - n) - 1), rows, x.mtile * BM);
        p.desc[2 * cta + 1] = make_int4(x.token0, x.kvh, 0, 0);
      }
      it0 += n;
      ++item;
      x = y;
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == W0 + 1) tmem_dealloc(tmem, 512);
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
  // launched as the attention ends (0.3 to 0.7 us earlier than a plain launch, of 14 to 19 us for
  // one request; letting it come as early as the attention begins cost 1 us): the parts are there
  // from here on
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 d0 = p.desc[2 * c];
  if (d0.x == 0) return;
  const int4 d1 = p.desc[2 * c + 1];
  const int parts = d0.y - c + 1;
  auto slot = [&](int i) { return (i == 0 ? 2 * c + 1 : 2 * (c + i)) * BM; };
  for (int row = blockIdx.y * 8 + (threadIdx.x >> 5); row < d0.z; row += gridDim.y * 8) {
    float top = kNegInf;
    for (int i = lane; i < parts; i += 32) top = fmaxf(top, p.part_ml[slot(i) + row].x);
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    constexpr int E = D / 32;
    float acc[E], l = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma unroll 4
    for (int i = 0; i < parts; ++i) {
      const float2 ml = p.part_ml[slot(i) + row];
      const float f = ml.x == kNegInf ? 0.f : ex2_approx(ml.x - top);
      const float* src = p.part_o + int64_t(slot(i) + row) * D;
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
    const int64_t o = (int64_t(d1.x) + node) * p.Hq + d1.y * p.group + (packed - node * p.group);
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
constexpr int kMaxGrid = 148;  // B200's SMs: sizes the workspace without a device

int64_t workspace_bytes_for(int D) {
  return int64_t(kMaxGrid) * (2 * (int64_t(BM) * D * 4 + BM * 8) + 32);
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                  const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// Pool view [pages, page_size, heads, D] with a box of (`inner` elements, 1 head, `rows` rows,
// 1 page), swizzled over `swizzle` bytes (0: not).
int make_pool_map(CUtensorMap* map, const void* base, int num_pages, int page_size, int heads, int D,
                  int elem, const int64_t* strides, int rows, int inner, int swizzle) {
  static const EncodeTiledFn enc = []() -> EncodeTiledFn {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    const bool found = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
                       q == cudaDriverEntryPointSuccess;
    return found ? reinterpret_cast<EncodeTiledFn>(ptr) : nullptr;
  }();
  FA4CP_CHECK_ARG(enc != nullptr, "cuTensorMapEncodeTiled is unavailable");
  const cuuint64_t dims[4] = {cuuint64_t(D), cuuint64_t(heads), cuuint64_t(page_size),
                              cuuint64_t(num_pages > 0 ? num_pages : 1)};
  const cuuint64_t st[3] = {cuuint64_t(strides[2]) * elem, cuuint64_t(strides[1]) * elem,
                            cuuint64_t(strides[0]) * elem};
  const cuuint32_t box[4] = {cuuint32_t(inner), 1, cuuint32_t(rows), 1};
  const cuuint32_t es[4] = {1, 1, 1, 1};
  const CUresult r = enc(map, elem == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 4,
                         const_cast<void*>(base), dims, st, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         swizzle == 128  ? CU_TENSOR_MAP_SWIZZLE_128B
                         : swizzle == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                         : CU_TENSOR_MAP_SWIZZLE_NONE,
                         // 128: a page's rows of one head may be no longer, and the other heads' rows
                         // between them are another CTA's (f16, head_dim 64: 250 us, 256 took 263)
                         CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
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
  FA4CP_CHECK_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  const int grid = sms < kMaxGrid ? sms : kMaxGrid;
  const int rows = p.page_size < TR::BN ? p.page_size : TR::BN;
  const int el = TR::KV8 ? 1 : 2;
  CUtensorMap mk, mv;
  const void* none = p.q;  // an empty pool: every page is outside, nothing is read
  if (int rc = make_pool_map(&mk, p.num_pages ? k_pages : none, p.num_pages, p.page_size, p.Hkv, TR::D, el, ks,
                             rows, TR::K_SWZ / el, TR::K_SWZ))
    return rc;
  if (int rc = make_pool_map(&mv, p.num_pages ? v_pages : none, p.num_pages, p.page_size, p.Hkv, TR::D, el, vs,
                             rows, TR::KV8 ? TR::D : 64, TR::KV8 ? 0 : 128))
    return rc;
  tree_attn_kernel<TR><<<grid, TR::THREADS, TR::SMEM_BYTES, st>>>(mk, mv, p);
  if (int rc = check_launch("attn_fwd_paged_tree")) return rc;
  const int64_t most = int64_t(max_seqlen_q) * p.group;  // rows of a row tile
  const int blocks = int(((most < BM ? most : BM) + 7) / 8);
  cudaLaunchAttribute overlap{};
  overlap.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  overlap.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(grid), unsigned(blocks));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cfg.attrs = &overlap;
  cfg.numAttrs = 1;
  FA4CP_CHECK_CUDA(cudaLaunchKernelEx(&cfg, tree_combine_kernel<TR::D>, p));
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
  FA4CP_CHECK_ARG(kv_dtype == q_dtype || (kv8 && q_dtype == FA4CP_DTYPE_BF16),
                  "K/V dtype must be the dtype of q, or e4m3 under a bf16 q");
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
    if (head_dim == 64) return go(TreeTraits<64, true>{});
    if (head_dim == 128) return go(TreeTraits<128, true>{});
    return go(TreeTraits<256, true>{});
  }
  if (head_dim == 64) return go(TreeTraits<64, false>{});
  if (head_dim == 128) return go(TreeTraits<128, false>{});
  return go(TreeTraits<256, false>{});
}
