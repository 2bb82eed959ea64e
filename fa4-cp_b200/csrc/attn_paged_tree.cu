// Attention of drafted tokens over a paged K/V cache (single-token decode is the tree of one
// node).  No counterpart in the reference, whose K/V is contiguous (README.md:139-141).
#include "common.cuh"

namespace fa4cp {
namespace {

constexpr float kNegInf = -__builtin_huge_valf();

struct TreeParams {
  const uint8_t* q;
  int64_t q_stride;  // elements a token
  const uint8_t *k, *v;
  int64_t k_page, k_row, k_head, v_page, v_row, v_head;  // strides in bytes
  const int32_t *block_table, *cu_q, *seq_lens;
  const uint64_t* mask;
  void* out;
  float* lse;
  const float *q_descale, *k_descale, *v_descale;
  int64_t total_q;
  int nseq, Hq, Hkv, group, page_size, num_pages, max_pages, words;
  int q_dtype, kv_dtype, out_bf16;
  float scale_log2;
};

__device__ __forceinline__ float load_elem(const uint8_t* p, int dtype, int i) {
  if (dtype == FA4CP_DTYPE_BF16)
    return __uint_as_float(uint32_t(reinterpret_cast<const uint16_t*>(p)[i]) << 16);
  if (dtype == FA4CP_DTYPE_F16) return __half2float(reinterpret_cast<const __half*>(p)[i]);
  float a, b, c, d;
  unpack_e4m3x4(p[i], a, b, c, d);
  return a;
}

// One warp per (token, query head): lanes split the head's elements, keys are walked in order
// with an online softmax.  Reads K and V once per query head; bound by issue and L2.
template <int D>
__global__ void __launch_bounds__(128) tree_simple_kernel(const TreeParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t unit = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (unit >= p.total_q * p.Hq) return;
  const int64_t t = unit / p.Hq;
  const int head = int(unit - t * p.Hq), kvh = head / p.group;
  if (t < p.cu_q[0] || t >= p.cu_q[p.nseq]) return;
  int lo = 0, hi = p.nseq;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.cu_q[mid] <= t) lo = mid; else hi = mid;
  }
  const int node = int(t - p.cu_q[lo]), n = p.cu_q[lo + 1] - p.cu_q[lo];
  const int len = max(p.seq_lens[lo], 0), ctx = len - n;
  constexpr int E = D / 32;
  const int qe = p.q_dtype == FA4CP_DTYPE_E4M3 ? 1 : 2, ke = p.kv_dtype == FA4CP_DTYPE_E4M3 ? 1 : 2;
  float q[E], acc[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    q[i] = load_elem(p.q + (t * p.q_stride + int64_t(head) * D) * qe, p.q_dtype, i * 32 + lane);
    acc[i] = 0.f;
  }
  float scale = p.scale_log2, vscale = 1.f;
  if (p.q_descale) scale *= p.q_descale[kvh];
  if (p.k_descale) scale *= p.k_descale[kvh];
  if (p.v_descale) vscale = p.v_descale[kvh];
  float m = kNegInf, l = 0.f;
  (void)ke;
  for (int key = 0; key < len; ++key) {
    const int d = key - ctx;
    if (d >= 0) {
      bool seen;
      if (p.mask) seen = d < p.words * 64 && ((p.mask[t * p.words + (d >> 6)] >> (d & 63)) & 1);
      else seen = d <= node;
      if (!seen) continue;
    }
    const int e = key / p.page_size, r = key - e * p.page_size;
    const int page = e < p.max_pages ? p.block_table[int64_t(lo) * p.max_pages + e] : -1;
    const bool ok = page >= 0 && page < p.num_pages;  // a page outside the pool reads zeros
    const uint8_t* kr = p.k + (ok ? page * p.k_page + r * p.k_row : 0) + kvh * p.k_head;
    const uint8_t* vr = p.v + (ok ? page * p.v_page + r * p.v_row : 0) + kvh * p.v_head;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) s = fmaf(q[i], ok ? load_elem(kr, p.kv_dtype, i * 32 + lane) : 0.f, s);
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    s *= scale;
    const float mn = fmaxf(m, s);
    const float f = m == kNegInf ? 0.f : exp2f(m - mn), w = exp2f(s - mn);
    m = mn;
    l = fmaf(l, f, w);
#pragma unroll
    for (int i = 0; i < E; ++i)
      acc[i] = fmaf(acc[i], f, w * (ok ? load_elem(vr, p.kv_dtype, i * 32 + lane) : 0.f));
  }
  const float inv = l > 0.f ? vscale / l : 0.f;
  const int64_t o = (t * p.Hq + head) * D;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const float x = l > 0.f ? acc[i] * inv : 0.f;
    if (p.out_bf16) static_cast<__nv_bfloat16*>(p.out)[o + i * 32 + lane] = __float2bfloat16(x);
    else static_cast<__half*>(p.out)[o + i * 32 + lane] = __float2half(x);
  }
  if (lane == 0) p.lse[t * p.Hq + head] = l > 0.f ? (m + log2f(l)) * kLn2 : kNegInf;
}

}  // namespace
}  // namespace fa4cp

using namespace fa4cp;

extern "C" int64_t fa4cp_attn_paged_tree_workspace_bytes(int32_t num_heads_q, int32_t num_heads_kv,
                                                         int32_t head_dim, int32_t max_seqlen_q) {
  if (num_heads_q < 1 || num_heads_kv < 1 || head_dim < 1 || max_seqlen_q < 0) return -1;
  return 16;
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
  FA4CP_CHECK_ARG(tree_mask == nullptr || mask_words >= 1, "tree_mask needs mask_words >= 1");
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) {
    set_last_error("head_dim %d is not supported", head_dim);
    return FA4CP_ERR_UNSUPPORTED;
  }
  if (total_q == 0 || max_seqlen_q == 0) return FA4CP_OK;
  FA4CP_CHECK_ARG(q && out && lse && block_table && k_strides && v_strides && (num_pages == 0 || (k_pages && v_pages)),
                  "null tensor pointer");
  const int qe = q8 ? 1 : 2, ke = kv8 ? 1 : 2;
  auto al = [](const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15u) == 0; };
  FA4CP_CHECK_ARG(al(q) && al(out) && al(k_pages) && al(v_pages) && q_token_stride * qe % 16 == 0,
                  "q rows, out and the pools must be 16-byte aligned");
  for (int i = 0; i < 3; ++i)
    FA4CP_CHECK_ARG(k_strides[i] * ke % 16 == 0 && v_strides[i] * ke % 16 == 0 && k_strides[i] >= 0 && v_strides[i] >= 0,
                    "pool strides must be multiples of 16 bytes");
  TreeParams p{};
  p.q = static_cast<const uint8_t*>(q);
  p.q_stride = q_token_stride;
  p.k = static_cast<const uint8_t*>(k_pages);
  p.v = static_cast<const uint8_t*>(v_pages);
  p.k_page = k_strides[0] * ke; p.k_row = k_strides[1] * ke; p.k_head = k_strides[2] * ke;
  p.v_page = v_strides[0] * ke; p.v_row = v_strides[1] * ke; p.v_head = v_strides[2] * ke;
  p.block_table = block_table;
  p.cu_q = cu_q;
  p.seq_lens = seq_lens;
  p.mask = reinterpret_cast<const uint64_t*>(tree_mask);
  p.out = out;
  p.lse = lse;
  p.q_descale = q_descale;
  p.k_descale = k_descale;
  p.v_descale = v_descale;
  p.total_q = total_q;
  p.nseq = nseq;
  p.Hq = num_heads_q;
  p.Hkv = num_heads_kv;
  p.group = num_heads_q / num_heads_kv;
  p.page_size = page_size;
  p.num_pages = num_pages;
  p.max_pages = max_pages;
  p.words = mask_words;
  p.q_dtype = q_dtype;
  p.kv_dtype = kv_dtype;
  p.out_bf16 = q_dtype != FA4CP_DTYPE_F16;
  p.scale_log2 = softmax_scale * kLog2e;
  (void)workspace;
  (void)workspace_bytes;
  const int64_t units = total_q * num_heads_q;
  const unsigned grid = unsigned((units + 3) / 4);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (head_dim == 64) tree_simple_kernel<64><<<grid, 128, 0, st>>>(p);
  else if (head_dim == 128) tree_simple_kernel<128><<<grid, 128, 0, st>>>(p);
  else tree_simple_kernel<256><<<grid, 128, 0, st>>>(p);
  return check_launch("attn_fwd_paged_tree");
}
