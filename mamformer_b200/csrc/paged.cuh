// Shared by the paged KV cache kernels: of the 8-bit cache (paged_kv.cu, paged_attn.cu, paged_attn_tc.cu) and, in what
// both have alike, of the 4-bit one (paged4.cuh).
//
// One layer's 8-bit cache is four tensors:
//   k, v              (P, G, page, hd) e4m3 codes; the `page` tokens of one KV head are contiguous
//   k_scale, v_scale  (P, G) fp32 powers of two, one for each block of `page` tokens and head
// and a block table (B, W) int32 gives the page of slots [j * page, (j + 1) * page) of a sequence.
// cu (B + 1) int32 are the offsets of the sequences' new tokens in the packed (T, ..) tensors,
// lens (B) int32 the cached lengths with those tokens in: token i of sequence b, of n = cu[b + 1] -
// cu[b], sits in slot lens[b] - n + i.
#pragma once

#include "common.cuh"

#include <cuda_fp8.h>

namespace mamf {
namespace paged {

// What the kernels record; *_error() gives the codes met since they were cleared, code c as bit c.
enum : int { ERR_PAGE = 1, ERR_LENGTH = 2, ERR_POSITION = 3, ERR_WAIT = 4 };

struct Table {
  const int *table, *cu, *lens;
  int P, G, page, shift, W, B, T;        // page = 1 << shift
};
struct Cache : Table {
  uint8_t *k, *v;
  float *ks, *vs;
};

// The block table, offsets and lengths (contiguous, on one GPU) of a cache of P pages of `page` tokens and G heads.
// cu null: an operator that takes no new tokens.
inline Table check_table(const char* what, const at::Tensor& table, const at::Tensor* cu, const at::Tensor& lens, int64_t P,
                         int64_t G, int64_t page, int64_t T) {
  for (const at::Tensor* t : {&table, cu, &lens})
    TORCH_CHECK(!t || t->scalar_type() == at::kInt, what, ": int32 block table, offsets and lengths");
  const int64_t B = lens.numel();
  TORCH_CHECK(table.dim() == 2 && table.size(0) == B && (!cu || cu->numel() == B + 1), what, ": a block table row and an offset for each of ", B, " sequences");
  // slots are counted in 32 bits, and tiles ahead of a sequence's last one too
  TORCH_CHECK(P < (1LL << 31) && G <= 65535 && table.size(1) * page <= (1LL << 31) - (1 << 20) && T < (1LL << 31) && B < (1 << 24), what, ": sizes");
  return Table{table.data_ptr<int>(), cu ? cu->data_ptr<int>() : nullptr, lens.data_ptr<int>(), (int)P, (int)G, (int)page,
               page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : 7, (int)table.size(1), (int)B, (int)T};
}

struct Layer { at::Tensor k, v, ks, vs, table, cu, lens; };

inline Cache check_cache(const char* what, const Layer& l, int64_t T, int64_t hd) {
  const at::Tensor* all[] = {&l.k, &l.v, &l.ks, &l.vs, &l.table, &l.cu, &l.lens};
  for (const at::Tensor* t : all)
    TORCH_CHECK(t->is_cuda() && t->device() == l.k.device() && t->is_contiguous(), what, ": contiguous cache tensors on one GPU");
  TORCH_CHECK(l.k.scalar_type() == at::kFloat8_e4m3fn && l.v.scalar_type() == at::kFloat8_e4m3fn && l.k.dim() == 4 &&
              l.k.sizes() == l.v.sizes(), what, ": k and v pages (P, G, page, hd) in float8_e4m3fn");
  const int64_t P = l.k.size(0), G = l.k.size(1), page = l.k.size(2);
  TORCH_CHECK(l.k.size(3) == hd && (hd == 64 || hd == 128), what, ": head size 64 or 128, got ", l.k.size(3), " in the cache and ", hd);
  TORCH_CHECK(page == 16 || page == 32 || page == 64 || page == 128, what, ": pages of 16, 32, 64 or 128 tokens, got ", page);
  for (const at::Tensor* t : {&l.ks, &l.vs})
    TORCH_CHECK(t->scalar_type() == at::kFloat && t->dim() == 2 && t->size(0) == P && t->size(1) == G, what, ": fp32 scales (P, G)");
  TORCH_CHECK(aligned16(l.k.data_ptr()) && aligned16(l.v.data_ptr()), what, ": 16-byte aligned pages");
  Cache c;
  static_cast<Table&>(c) = check_table(what, l.table, &l.cu, l.lens, P, G, page, T);
  c.k = (uint8_t*)l.k.data_ptr();
  c.v = (uint8_t*)l.v.data_ptr();
  c.ks = l.ks.data_ptr<float>();
  c.vs = l.vs.data_ptr<float>();
  return c;
}

// What the attention kernels of a cache are given.
template <class C> struct AttnOf {
  C c;
  const void *q1, *q2;                 // packed queries (T, H, hd); q2 null: one map
  void* out;                           // (T, H, hd), contiguous
  float* lse;                          // (T, H, maps) log2 of each row's sum of weights, +inf for none; null: not asked for
  const float* lam;
  int64_t st1, sh1, st2, sh2;          // token and head strides of q1, q2 in elements
  int H, rep, maps, window;            // rep = H / G query heads per KV head
  int few;                             // sequences of up to this many rows (n * rep * maps) are the split kernel's
  bool chunked;                        // the chunk kernel takes the others
  float scale_log2;
  long long wait;                      // cycles after which a wait gives up; negative: at once, without a look
};
using Attn = AttnOf<Cache>;

// Cycles of a wait, about 0.25 s, where the longest takes microseconds; paged_attention_wait_limit() sets another number
// for the waits that a test lets run out.
constexpr long long WAIT_CYCLES = 500000000LL;
long long attention_wait_limit();

// csrc/paged_attn_tc.cu: sequences of more than `few` rows (of any number where few is 0, and then rows past
// the last sequence are cleared too)
void paged_chunk_attention(const Attn& p, int hd, bool bf16);
int64_t paged_chunk_error(bool clear);

// The code in a device word, 0 or one of the above, as a bit.
template <typename Word> inline int64_t take_code(Word& word, bool clear) {
  int v = 0, z = 0;
  MAMF_CUDA_CHECK(cudaMemcpyFromSymbol(&v, word, sizeof(int)));
  if (v && clear) MAMF_CUDA_CHECK(cudaMemcpyToSymbol(word, &z, sizeof(int)));
  return v ? 1LL << v : 0;
}

// A tensor whose rows of adjacent values start on 16-byte boundaries: t itself, or a copy of it.
inline at::Tensor rows16(const at::Tensor& t) {
  const int64_t n = 16 / t.element_size();
  if (t.stride(2) == 1 && t.stride(0) % n == 0 && t.stride(1) % n == 0 && aligned16(t.data_ptr())) return t;
  return t.clone(at::MemoryFormat::Contiguous);
}

// bytes -> values
__device__ __forceinline__ float2 dec2(uint16_t c) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(c, __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
__device__ __forceinline__ uint16_t enc2(float a, float b) {
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}

// The sequence that packed token t belongs to: the last b with cu[b] <= t (an empty sequence never
// is), or -1 before the first and past the last one.
__device__ __forceinline__ int sequence_of(const int* cu, int B, int t) {
  if (B == 0 || t < cu[0] || t >= cu[B]) return -1;
  int lo = 0, hi = B - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (cu[mid] <= t) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// Offsets of sequence b that rise and stay within the T packed tokens.
__device__ __forceinline__ bool in_order(const Table& c, int b) { return c.cu[b] >= 0 && c.cu[b] <= c.cu[b + 1] && c.cu[b + 1] <= c.T; }

// The slots of a sequence that the block table has room for.
__device__ __forceinline__ int cached_length(const Table& c, int len) { return max(0, min(len, c.W << c.shift)); }

}  // namespace paged
}  // namespace mamf
