// The paged 4-bit KV cache, shared by its kernels (paged_kv.cu, paged4_kv.cu, paged4_attn.cu, paged4_attn_tc.cu).
//
// One layer's cache is a byte tensor (P, G, page / 16, 18 hd): each block holds 16 tokens of one KV head,
//   key codes (16, hd / 2), key parameters (16, hd / 32) of 16 bits, then the same of the values,
// contiguous, so that a warp fetches a block's keys and values in one copy.  The even one of a byte's two dims is in
// its low half.  Group j of hd / 32 is the 32 dims d with (d / 4) % (hd / 32) == j, a dim and its partner hd / 2 further
// in the same one.  A parameter is the f16 pattern of the group's scale s, of 7 significant bits, with the zero point z in
// the low 4 bits, and a code n stands for s (n - z): 7 bits times 4, exact in f16, which the tensor cores then take as
// they are.  Block table, offsets and lengths are those of paged.cuh.
//
// Runs of 4 dims alternate between groups so that the nibbles i and i + 4 of a 32-bit word (8 dims), which one mask picks
// as the halves of a register, belong to the two groups whose parameters share a 32-bit word: a pair of dims is scaled by
// a pair of scales without a shuffle.
#pragma once

#include "paged.cuh"

namespace mamf {
namespace paged4 {

using namespace paged;

// Constants of the decoding below.  They come with the launch and not with the code, where the compiler would write them
// into a register anew for every use of a pair of constants: an instruction takes one.
struct Base {
  uint32_t one = 0x64006400u;                        // 1024 in both halves
  uint32_t back = 0xF380F380u;                       // -15360
};
struct Cache4 : Table {
  uint8_t* blocks;
  float* mass;                                       // (P, G, page) received weights, or null
  Base base;
};

template <int HD> constexpr int HALF = 9 * HD;        // bytes of a block's keys, or values, with their parameters
template <int HD> constexpr int BLOCK = 18 * HD;
template <int HD> constexpr int PARAMS = 8 * HD;      // where the parameters begin in them

inline Cache4 check_cache4(const char* what, const at::Tensor& blocks, const c10::optional<at::Tensor>& mass,
                           const at::Tensor& table, const at::Tensor* cu, const at::Tensor& lens, int64_t T, int64_t hd) {
  for (const at::Tensor* t : {&blocks, &table, cu, &lens})
    TORCH_CHECK(!t || (t->is_cuda() && t->device() == blocks.device() && t->is_contiguous()), what, ": contiguous cache tensors on one GPU");
  TORCH_CHECK(blocks.scalar_type() == at::kByte && blocks.dim() == 4, what, ": blocks (P, G, page / 16, 18 hd) in uint8");
  TORCH_CHECK((hd == 64 || hd == 128) && blocks.size(3) == 18 * hd, what, ": head size 64 or 128, got ", blocks.size(3) / 18, " in the cache and ", hd);
  const int64_t P = blocks.size(0), G = blocks.size(1), page = 16 * blocks.size(2);
  TORCH_CHECK(page == 16 || page == 32 || page == 64 || page == 128, what, ": pages of 16, 32, 64 or 128 tokens, got ", page);
  TORCH_CHECK(aligned16(blocks.data_ptr()), what, ": 16-byte aligned blocks");
  Cache4 c{};
  static_cast<Table&>(c) = check_table(what, table, cu, lens, P, G, page, T);
  c.blocks = (uint8_t*)blocks.data_ptr();
  c.mass = nullptr;
  if (mass.has_value()) {
    TORCH_CHECK(mass->is_cuda() && mass->device() == blocks.device() && mass->is_contiguous() && mass->scalar_type() == at::kFloat &&
                mass->dim() == 3 && mass->size(0) == P && mass->size(1) == G && mass->size(2) == page, what, ": contiguous fp32 mass (P, G, page)");
    c.mass = mass->data_ptr<float>();
  }
  return c;
}

// The block that slot `slot` of a page lies in.
template <int HD> __device__ __forceinline__ uint8_t* block_of(const Cache4& c, int pg, int g, int slot) {
  return c.blocks + ((((int64_t)pg * c.G + g) << (c.shift - 4)) + ((slot & (c.page - 1)) >> 4)) * BLOCK<HD>;
}

// ---- codes -> f16 ----------------------------------------------------------------------------------
// 0x6400 | n is the f16 1024 + n, and 0x6400 | 16 n is 1024 + 16 n: differences to 1024 + z (1024 + 16 z) are exact, and so
// are their products with s (s / 16).
__device__ __forceinline__ uint32_t hsub(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t hmul(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t hfma(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
// (a & mask) | 1024 in both halves, in one instruction; written as two operators it became two
template <uint32_t MASK> __device__ __forceinline__ uint32_t pick(uint32_t a, uint32_t one) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(a), "n"(MASK), "r"(one));
  return r;
}
// What two groups' parameters give: for codes in the low four bits of a half, and for those in the next four.  The integer
// units are what bounds the decoding, so the second pair comes from the first by f16 arithmetic (exact: 16 (1024 + z) -
// 15360 = 1024 + 16 z).
struct Levels { uint32_t z0, s0, z4, s4; };
__device__ __forceinline__ Levels levels_of(uint32_t params, const Base& base) {
  Levels l;
  l.z0 = pick<0x000F000Fu>(params, base.one);
  l.s0 = params & 0xFFF0FFF0u;
  l.z4 = hfma(l.z0, 0x4C004C00u, base.back);         // 16
  l.s4 = hmul(l.s0, 0x2C002C00u);                    // 1 / 16
  return l;
}
// The 16-bit halves of w hold the codes of two groups, four each: code i of both as the halves of h[i].
__device__ __forceinline__ void decode(uint32_t w, const Levels& l, const Base& base, uint32_t (&h)[4]) {
  const uint32_t u = w >> 8;
  h[0] = hmul(hsub(pick<0x000F000Fu>(w, base.one), l.z0), l.s0);
  h[1] = hmul(hsub(pick<0x00F000F0u>(w, base.one), l.z4), l.s4);
  h[2] = hmul(hsub(pick<0x000F000Fu>(u, base.one), l.z0), l.s0);
  h[3] = hmul(hsub(pick<0x00F000F0u>(u, base.one), l.z4), l.s4);
}

// ---- values -> codes -------------------------------------------------------------------------------
// Scale and zero point of a group with extremes lo <= 0 <= hi.  The scale is a fifteenth of the range rounded up to 7
// significant bits (to a multiple of 2^-20 below 2^-14), so that every value is within half a step of a level.  No level may
// leave f16: the largest scale is 65504 / max(zero, 15 - zero) rounded down to 7 bits, which above 4096 are multiples of
// 64: 64 floor(1023 / max(zero, 15 - zero)).
// It is met only where an extreme is above 60,900; the other end of such a group may then be off by up to a step.
// Elementwise fp32 roundings throughout, so that eager code finds the same codes.
struct Group { float scale, inv; int zero; };
__device__ __forceinline__ Group group_of(float lo, float hi) {
  float s = __fmul_rn(__fsub_rn(hi, lo), 0.06666666f);          // 1/15, rounded down
  if (s < 6.103515625e-5f) s = __fmul_rn(ceilf(__fmul_rn(s, 1048576.f)), 9.5367431640625e-7f);
  else s = __uint_as_float((__float_as_uint(s) + 0x1FFFFu) & ~0x1FFFFu);
  s = fmaxf(s, 9.5367431640625e-7f);
  Group g;
  g.zero = (int)fminf(fmaxf(rintf(__fmul_rn(-lo, __frcp_rn(s))), 0.f), 15.f);
  // 1023 / m for m = 8 .. 15, a byte each: a division cost a single-token append 1 us
  const uint32_t units = __byte_perm(0x5D66717Fu, 0x44494E55u, (uint32_t)max(g.zero, 15 - g.zero) - 8u) & 0xFFu;
  g.scale = fminf(s, 64.f * (float)units);
  g.inv = __frcp_rn(g.scale);
  return g;
}
__device__ __forceinline__ uint32_t param_of(const Group& g) {
  return (uint32_t)__half_as_ushort(__float2half_rn(g.scale)) | (uint32_t)g.zero;
}
__device__ __forceinline__ uint32_t code_of(float x, const Group& g) {
  return (uint32_t)fminf(fmaxf(__fadd_rn(rintf(__fmul_rn(x, g.inv)), (float)g.zero), 0.f), 15.f);
}
// What the cache takes of a value: NaN as 0, anything else within f16.
__device__ __forceinline__ float storable(float x) { return x != x ? 0.f : fminf(fmaxf(x, -65504.f), 65504.f); }

using Attn4 = AttnOf<Cache4>;

// csrc/paged4_attn_tc.cu: sequences of more than `few` rows (of any number where few is 0, and then rows past the last
// sequence are cleared too)
void chunk_attention(const Attn4& p, int hd, bool bf16);
// and the weights that their slots receive, of sequences of more than `kept` rows, from the rows' sums in p.lse
void chunk_weights(const Attn4& p, int kept, int hd, bool bf16);
int64_t chunk_error(bool clear);

}  // namespace paged4
}  // namespace mamf
