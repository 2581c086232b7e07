// Appending keys and values to the paged caches, with the rotation of the keys (and of up to two
// query tensors) on the way.  The reference grows (B, S, G, hd) tensors with torch.cat each step
// (mamformer/layers/attention.py:143-149, kda_diff.py:813-818) and rotates in a pass of its own.
//
//   k' = (k1 cos - k2 sin, k2 cos + k1 sin) at the token's position     (fp32, each product rounded)
//   scale of a block (page, head) = 2^e, the least e with max |finite values| <= 448 * 2^e
//   code = e4m3(value / scale), to nearest even, saturating
//
// A page that already holds tokens of its sequence keeps the larger of its old scale and the new
// tokens' one, and when that grows its old codes are multiplied by old / new.  Scales are powers of two
// so that this changes a code only where it falls below 2^-6 and loses trailing bits.  A page whose first
// slot is among the new tokens starts afresh: what an earlier owner left there does not count.
//
// One CTA owns one (sequence, page, KV head) of K or of V: it reads the page's new tokens once, keeps them
// in registers, reduces their maximum, and writes the codes; no other CTA touches that block, so there are
// no atomics.  Where no sequence has more than one new token, 8 lanes (4 for 64 dims) do that instead of a CTA:
// a step of 200 sequences and 8 heads is then one wave of CTAs.  Pages that take new tokens must belong to one
// sequence only.  Further CTAs rotate the queries in the same launch.
//
// 20,000 prompt tokens, 8 KV heads and two query tensors of 32 heads of 128 (792 MB): 156 us, 5.1 TB/s; the CTAs
// alternate between loads and stores.  One token each of 200 sequences: 10 us, the chain offsets - table -
// scale - rotation and the launch.
#include "paged4.cuh"

namespace mamf {
namespace kva {

using namespace paged;

constexpr int NT = 256;

__device__ int g_err = 0;
__device__ __forceinline__ void record(int code) { atomicCAS(&g_err, 0, code); }

struct Src { const void* p; int64_t st, sh; };       // token and head strides in elements

struct Rows {
  Src k, v, q[2];
  void* qo[2];
  const float *cos, *sin;                            // (n_pos, hd / 2) with row stride rot, null: no rotation
  int64_t rot;
  const int64_t* pos;                                // (T)
  int n_pos, H, nq, units;
};
struct Params : Rows {
  Cache c;
  int per_seq, max_new;
};
struct Params4 : Rows {
  paged4::Cache4 c;
  int max_new;
};

// 8 consecutive values of a token's head as floats
template <typename T> __device__ __forceinline__ void load8(const T* p, float* f) {
  constexpr int N = 16 / sizeof(T);
#pragma unroll
  for (int i = 0; i < 8 / N; ++i) {
    const Vec16<T> v = ld16(p + i * N);
#pragma unroll
    for (int j = 0; j < N; ++j) f[i * N + j] = to_f(v.v[j]);
  }
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float* f) {
  constexpr int N = 16 / sizeof(T);
#pragma unroll
  for (int i = 0; i < 8 / N; ++i) {
    Vec16<T> v;
#pragma unroll
    for (int j = 0; j < N; ++j) v.v[j] = from_f<T>(f[i * N + j]);
    st16(p + i * N, v);
  }
}

// cos and sin of 8 dims at token t's position
struct Turn { float c[8], s[8]; };
template <int HD>
__device__ __forceinline__ Turn turn_of(const Rows& p, int t, int d) {
  int64_t pos = p.pos[t];
  if (pos < 0 || pos >= p.n_pos) { record(ERR_POSITION); pos = pos < 0 ? 0 : p.n_pos - 1; }
  Turn r;
#pragma unroll
  for (int i = 0; i < 8; i += 4) {
    *reinterpret_cast<float4*>(r.c + i) = *reinterpret_cast<const float4*>(p.cos + pos * p.rot + d + i);
    *reinterpret_cast<float4*>(r.s + i) = *reinterpret_cast<const float4*>(p.sin + pos * p.rot + d + i);
  }
  return r;
}
// (a, b) -> (a cos - b sin, b cos + a sin).  Separate roundings, as elementwise operations have them, so
// that a value on the edge between two codes goes the same way.
__device__ __forceinline__ void rotate8(const Turn& r, float* a, float* b) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float x = a[i], y = b[i];
    a[i] = __fsub_rn(__fmul_rn(x, r.c[i]), __fmul_rn(y, r.s[i]));
    b[i] = __fadd_rn(__fmul_rn(y, r.c[i]), __fmul_rn(x, r.s[i]));
  }
}

// e4m3's largest value is 448 = 1.75 * 2^8, so the least e with m * 2^x <= 1.75 * 2^8 * 2^e (m in [1, 2))
// is x - 8, or x - 7 where m > 1.75.
__device__ __forceinline__ float block_scale(float amax) {
  const uint32_t b = __float_as_uint(amax);
  int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  e = max(-100, min(119, amax > 0.f ? e : -100));
  return __uint_as_float((uint32_t)(e + 127) << 23);
}
__device__ __forceinline__ float inverse_pow2(float s) {          // s = 2^e, |e| <= 126
  return __uint_as_float((254u << 23) - __float_as_uint(s));
}

// The codes of a block's first `tokens` tokens, times f (a power of two below 1).
template <int HD>
__device__ __forceinline__ void rescale(uint8_t* codes, int tokens, float f, int first, int step) {
  for (int i = first; i < tokens * HD / 16; i += step) {
    union { uint4 raw; uint16_t c2[8]; } w;
    w.raw = *reinterpret_cast<const uint4*>(codes + i * 16);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float2 v = dec2(w.c2[e]);
      w.c2[e] = enc2(v.x * f, v.y * f);
    }
    *reinterpret_cast<uint4*>(codes + i * 16) = w.raw;
  }
}
// 16 values of a token (8 of each half, from dim d) as codes
template <int HD>
__device__ __forceinline__ void put_codes(uint8_t* token, int d, const float* x, float inv) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    union { uint16_t c2[4]; uint2 raw; } w;
#pragma unroll
    for (int e = 0; e < 4; ++e) w.c2[e] = enc2(x[8 * h + 2 * e] * inv, x[8 * h + 2 * e + 1] * inv);
    *reinterpret_cast<uint2*>(token + h * (HD / 2) + d) = w.raw;
  }
}
// the largest of m and |x|; NaN and infinities do not count
__device__ __forceinline__ float finite_max(const float* x, float m) {
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const float a = fabsf(x[e]);
    m = fmaxf(m, a < INFINITY ? a : 0.f);
  }
  return m;
}

template <typename T, int HD, int NP>
__device__ __forceinline__ void append_block(const Params& p) {
  constexpr int TPT = HD / 16;                 // threads per token: 8 values of each half
  constexpr int TPP = NT / TPT;                // tokens per pass
  const Cache& c = p.c;
  const int tid = threadIdx.x;
  const bool is_v = blockIdx.z != 0;
  const int g = blockIdx.y, u = blockIdx.x;
  int b, j;
  if (p.per_seq > 0) { b = u / p.per_seq; j = u % p.per_seq; }
  else {
    // unit numbers of sequence b start at cu[b] / page + 2 b: with n new tokens it touches at most
    // (n - 1) / page + 2 pages, and the next sequence starts no earlier than that
    int lo = 0, hi = c.B - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (c.cu[mid] / c.page + 2 * mid <= u) lo = mid; else hi = mid - 1;
    }
    b = lo;
    j = u - (c.cu[b] / c.page + 2 * b);
  }
  const int t0 = c.cu[b], n = c.cu[b + 1] - t0, end = c.lens[b], start = end - n;
  if (n <= 0) return;
  const int pages = (end - 1) / c.page - start / c.page + 1;
  if (start < 0 || t0 < 0 || t0 + n > c.T || n > p.max_new) {
    if (tid == 0) record(ERR_LENGTH);
    return;
  }
  if (j < 0 || j >= pages) return;             // below the first unit where the offsets do not start at 0
  const int jp = start / c.page + j;
  const int pg = jp < c.W ? c.table[(int64_t)b * c.W + jp] : -1;
  if (pg < 0 || pg >= c.P) { if (tid == 0) record(ERR_PAGE); return; }
  const int lo = max(start - jp * c.page, 0), hi = min(end - jp * c.page, c.page);   // new slots of the page
  const Src src = is_v ? p.v : p.k;
  const T* in = (const T*)src.p + (int64_t)g * src.sh;
  uint8_t* out = (is_v ? c.v : c.k) + ((int64_t)pg * c.G + g) * c.page * HD;
  float* scale = (is_v ? c.vs : c.ks) + (int64_t)pg * c.G + g;
  const int d = (tid % TPT) * 8;

  float x[NP][16];
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int slot = lo + i * TPP + tid / TPT;
    if (slot < hi) {
      const int t = t0 + jp * c.page + slot - start;
      load8(in + (int64_t)t * src.st + d, x[i]);
      load8(in + (int64_t)t * src.st + HD / 2 + d, x[i] + 8);
      if (!is_v && p.cos) rotate8(turn_of<HD>(p, t, d), x[i], x[i] + 8);
      amax = finite_max(x[i], amax);
    }
  }
  __shared__ float sm_max[NT / 32];
  amax = warp_max(amax);
  if ((tid & 31) == 0) sm_max[tid >> 5] = amax;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NT / 32; ++w) amax = fmaxf(amax, sm_max[w]);
  const float need = block_scale(amax), had = lo > 0 ? *scale : 0.f;
  const float s = fmaxf(need, had), inv = inverse_pow2(s);
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int slot = lo + i * TPP + tid / TPT;
    if (slot < hi) put_codes<HD>(out + slot * HD, d, x[i], inv);
  }
  if (lo > 0 && had != s) rescale<HD>(out, lo, had * inv, tid, NT);
  __syncthreads();                              // every thread has read the old scale
  if (tid == 0 && had != s) *scale = s;
}

// One token per CTA at a time; a thread takes the same 16 dims of its heads in every tensor.  The rows are
// requested before the position, whose load the tables' loads wait for.
template <typename T, int HD>
__device__ __forceinline__ void rotate_queries(const Rows& p, int tokens, int block, int blocks) {
  constexpr int TPT = HD / 16;
  const int d = (threadIdx.x % TPT) * 8;
  for (int t = block; t < tokens; t += blocks)
    for (int h = threadIdx.x / TPT; h < p.H; h += NT / TPT) {
      constexpr int N = 16 / sizeof(T), L = 16 / N;
      Vec16<T> raw[2][L];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (i >= p.nq) break;
        const T* in = (const T*)p.q[i].p + (int64_t)t * p.q[i].st + (int64_t)h * p.q[i].sh + d;
#pragma unroll
        for (int l = 0; l < L; ++l) raw[i][l] = ld16(in + (l < L / 2 ? 0 : HD / 2) + l % (L / 2) * N);
      }
      const Turn turn = turn_of<HD>(p, t, d);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (i >= p.nq) break;
        float x[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = to_f(raw[i][e / N].v[e % N]);
        rotate8(turn, x, x + 8);
        T* out = (T*)p.qo[i] + ((int64_t)t * p.H + h) * HD + d;
        store8(out, x);
        store8(out + HD / 2, x + 8);
      }
    }
}

template <typename T, int HD, int NP>
__global__ void __launch_bounds__(NT, NP == 1 ? 4 : NP == 2 ? 3 : 2) append_kernel(const __grid_constant__ Params p) {
  if ((int)blockIdx.x < p.units) append_block<T, HD, NP>(p);
  else {
    const int qb = gridDim.x - p.units, layer = blockIdx.y + gridDim.y * blockIdx.z;
    rotate_queries<T, HD>(p, p.c.T, (blockIdx.x - p.units) + qb * layer, qb * gridDim.y * gridDim.z);
  }
}

// One new token per sequence at most; a group of TPT lanes does one token of K or V.
template <typename T, int HD>
__global__ void __launch_bounds__(NT, 4) append_one_kernel(const __grid_constant__ Params p) {
  constexpr int TPT = HD / 16;
  if ((int)blockIdx.x >= p.units) {
    rotate_queries<T, HD>(p, p.c.T, blockIdx.x - p.units, gridDim.x - p.units);
    return;
  }
  const Cache& c = p.c;
  const int sub = threadIdx.x % TPT, d = sub * 8;
  const int64_t item = ((int64_t)blockIdx.x * NT + threadIdx.x) / TPT;
  const bool is_v = item & 1;
  const int g = (int)(item / 2 % c.G), t = (int)(item / 2 / c.G);
  bool ok = t < c.T;
  int b = -1, slot = 0, pg = -1;
  if (ok) {
    // the usual step: every sequence has one token
    b = t < c.B && c.cu[t] == t && c.cu[t + 1] == t + 1 ? t : sequence_of(c.cu, c.B, t);
    ok = b >= 0;
  }
  if (ok) {
    const int n = c.cu[b + 1] - c.cu[b];
    slot = c.lens[b] - 1;
    ok = n == 1 && slot >= 0;
    if (!ok && sub == 0) record(ERR_LENGTH);
  }
  if (ok) {
    const int j = slot >> c.shift;
    pg = j < c.W ? c.table[(int64_t)b * c.W + j] : -1;
    ok = pg >= 0 && pg < c.P;
    if (!ok && sub == 0) record(ERR_PAGE);
  }
  const int lo = slot & (c.page - 1);
  const int64_t blk = ok ? (int64_t)pg * c.G + g : 0;
  uint8_t* out = (is_v ? c.v : c.k) + blk * c.page * HD;
  float* scale = (is_v ? c.vs : c.ks) + blk;
  float x[16], had = 0.f;
  if (ok) {
    const Src src = is_v ? p.v : p.k;
    const T* in = (const T*)src.p + (int64_t)t * src.st + (int64_t)g * src.sh + d;
    load8(in, x);
    load8(in + HD / 2, x + 8);
    if (lo > 0) had = *scale;
    if (!is_v && p.cos) rotate8(turn_of<HD>(p, t, d), x, x + 8);
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = 0.f;
  }
  float amax = finite_max(x, 0.f);
#pragma unroll
  for (int o = TPT / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  __syncwarp();                                 // the group's lanes have read the old scale
  if (!ok) return;
  const float s = fmaxf(block_scale(amax), had), inv = inverse_pow2(s);
  put_codes<HD>(out + lo * HD, d, x, inv);
  if (lo > 0 && had != s) rescale<HD>(out, lo, had * inv, sub, TPT);
  if (sub == 0 && had != s) *scale = s;
}

template <typename T, int HD>
void launch(Params& p) {
  const int64_t qblocks = p.nq ? std::min<int64_t>(p.c.T, 1 << 16) : 0;
  if (p.max_new <= 1) {
    p.units = (int)(((int64_t)p.c.T * p.c.G * 2 * (HD / 16) + NT - 1) / NT);
    append_one_kernel<T, HD><<<(unsigned)(p.units + qblocks), NT, 0, stream()>>>(p);
    return;
  }
  // units: (sequence, page) pairs that can take new tokens; the smaller of the two ways to number them
  const int64_t per_seq = ((int64_t)p.max_new + p.c.page - 2) / p.c.page + 1;
  const int64_t even = per_seq * p.c.B, packed = p.c.T / p.c.page + 2LL * p.c.B;
  p.per_seq = even <= packed ? (int)per_seq : 0;
  p.units = (int)std::min(even, packed);
  const dim3 grid((unsigned)(p.units + (qblocks + 2 * p.c.G - 1) / (2 * p.c.G)), (unsigned)p.c.G, 2u);
  // passes over a page's new tokens, which each thread holds 16 values of
  const int np = (int)(((int64_t)std::min(p.max_new, p.c.page) * HD + NT * 16 - 1) / (NT * 16));
  if (np <= 1) append_kernel<T, HD, 1><<<grid, NT, 0, stream()>>>(p);
  else if (np == 2) append_kernel<T, HD, 2><<<grid, NT, 0, stream()>>>(p);
  else append_kernel<T, HD, 4><<<grid, NT, 0, stream()>>>(p);
}

// The inputs' pointers, and room for the rotated queries.  Tensors whose rows are not on 16-byte boundaries are replaced by
// copies.
std::vector<at::Tensor> take_rows(Rows& p, at::Tensor& k, at::Tensor& v, c10::optional<at::Tensor>& cos,
                                  c10::optional<at::Tensor>& sin, c10::optional<at::Tensor>& pos, std::vector<at::Tensor>& queries) {
  const int64_t T = k.size(0), hd = k.size(2);
  auto src = [&](at::Tensor& t) {
    t = rows16(t);
    return Src{t.data_ptr(), t.stride(0), t.stride(1)};
  };
  std::vector<at::Tensor> outs;
  TORCH_CHECK(queries.size() <= 2, "kv_append: at most two query tensors");
  if (cos.has_value()) {
    TORCH_CHECK(sin.has_value() && pos.has_value(), "kv_append: cos, sin and positions go together");
    for (at::Tensor* t : {&*cos, &*sin}) {
      TORCH_CHECK(t->is_cuda() && t->device() == k.device() && t->scalar_type() == at::kFloat && t->dim() == 2 &&
                  t->size(1) == hd / 2 && t->size(0) == cos->size(0) && t->size(0) >= 1, "kv_append: fp32 cos and sin (positions, hd / 2)");
      if (t->stride(1) != 1 || t->stride(0) % 4 != 0 || !aligned16(t->data_ptr())) *t = t->clone(at::MemoryFormat::Contiguous);
    }
    if (cos->stride(0) != sin->stride(0)) { cos = cos->contiguous(); sin = sin->contiguous(); }
    TORCH_CHECK(pos->is_cuda() && pos->device() == k.device() && pos->scalar_type() == at::kLong && pos->is_contiguous() &&
                pos->numel() == T, "kv_append: int64 position of each token");
    TORCH_CHECK(cos->size(0) < (1LL << 31), "kv_append: table length");
    p.cos = cos->data_ptr<float>(); p.sin = sin->data_ptr<float>(); p.pos = pos->data_ptr<int64_t>();
    p.n_pos = (int)cos->size(0);
    p.rot = cos->stride(0);
  } else {
    TORCH_CHECK(queries.empty(), "kv_append: queries are only passed to be rotated");
  }
  for (auto& q : queries) {
    TORCH_CHECK(q.is_cuda() && q.device() == k.device() && q.dim() == 3 && q.size(0) == T && q.size(2) == hd &&
                q.scalar_type() == k.scalar_type() && q.sizes() == queries[0].sizes(), "kv_append: queries (T, H, hd) of k's type");
    outs.push_back(at::empty(q.sizes(), q.options(), at::MemoryFormat::Contiguous));
  }
  p.k = src(k);
  p.v = src(v);
  p.nq = (int)queries.size();
  for (int i = 0; i < p.nq; ++i) { p.q[i] = src(queries[i]); p.qo[i] = outs[i].data_ptr(); }
  p.H = p.nq ? (int)queries[0].size(1) : 0;
  return outs;
}

// ---- the 4-bit cache -------------------------------------------------------------------------------
// 16 values of a token (8 of each half, from dim d) of keys or values: parameters by all lanes of the token together,
// codes and, by one lane or two, the parameters into the block.  Dims d .. d + 3 and d + 4 .. d + 7 are of two groups.
template <int HD>
__device__ __forceinline__ void put_codes4(uint8_t* half_block, int row, int sub, float* x) {
  using namespace paged4;
  constexpr int J = HD / 32;
  float lo[2], hi[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    lo[r] = hi[r] = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float& y = x[8 * h + 4 * r + e];
        y = storable(y);
        lo[r] = fminf(lo[r], y);
        hi[r] = fmaxf(hi[r], y);
      }
  }
  // the lanes whose runs are of the same two groups: every second one of 8 for four groups, all 4 for two
#pragma unroll
  for (int o = HD / 32; o >= J / 2; o >>= 1)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      lo[r] = fminf(lo[r], __shfl_xor_sync(0xffffffffu, lo[r], o));
      hi[r] = fmaxf(hi[r], __shfl_xor_sync(0xffffffffu, hi[r], o));
    }
  const Group g[2] = {group_of(lo[0], hi[0]), group_of(lo[1], hi[1])};
  if (half_block == nullptr) return;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) w |= code_of(x[8 * h + e], g[e / 4]) << (4 * e);
    *reinterpret_cast<uint32_t*>(half_block + row * (HD / 2) + h * (HD / 4) + sub * 4) = w;
  }
  if (sub < J / 2) *reinterpret_cast<uint32_t*>(half_block + PARAMS<HD> + (row * (J / 2) + sub) * 4) = param_of(g[0]) | param_of(g[1]) << 16;
}

// A group of TPT lanes does the keys and values of one token, of every gridDim.y-th head.
template <typename T, int HD>
__global__ void __launch_bounds__(NT, 3) append4_kernel(const __grid_constant__ Params4 p) {
  constexpr int TPT = HD / 16;
  if ((int)blockIdx.x >= p.units) {
    const int qb = gridDim.x - p.units;
    rotate_queries<T, HD>(p, p.c.T, (blockIdx.x - p.units) + qb * blockIdx.y, qb * gridDim.y);
    return;
  }
  const paged4::Cache4& c = p.c;
  if (blockIdx.x + blockIdx.y == 0)
    for (int b = threadIdx.x; b < c.B; b += NT)
      if (!in_order(c, b)) record(ERR_LENGTH);
  const int sub = threadIdx.x % TPT, d = sub * 8;
  const int64_t item = ((int64_t)blockIdx.x * NT + threadIdx.x) / TPT;
  const int t = (int)min(item, (int64_t)c.T);
  bool ok = t < c.T;
  int b = -1, slot = 0, pg = -1;
  if (ok) {
    // the usual step: every sequence has one token
    b = t < c.B && c.cu[t] == t && c.cu[t + 1] == t + 1 ? t : sequence_of(c.cu, c.B, t);
    ok = b >= 0;
  }
  if (ok) {
    const int t0 = c.cu[b], n = c.cu[b + 1] - t0, end = c.lens[b];
    slot = end - n + (t - t0);
    ok = in_order(c, b) && t >= t0 && t - t0 < n && end - n >= 0 && n <= p.max_new;
    if (!ok && sub == 0) record(ERR_LENGTH);
  }
  if (ok) {
    const int j = slot >> c.shift;
    pg = j < c.W ? c.table[(int64_t)b * c.W + j] : -1;
    ok = pg >= 0 && pg < c.P;
    if (!ok && sub == 0) record(ERR_PAGE);
  }
  const bool turn_keys = p.cos != nullptr;
  Turn turn;
  if (ok && turn_keys) turn = turn_of<HD>(p, t, d);
  // all lanes of a warp stay in the loop for its shuffles
  for (int g = blockIdx.y; g < c.G; g += gridDim.y) {
    float x[16], y[16];
    uint8_t* blk = nullptr;
    if (ok) {
      const T* k = (const T*)p.k.p + (int64_t)t * p.k.st + (int64_t)g * p.k.sh + d;
      const T* v = (const T*)p.v.p + (int64_t)t * p.v.st + (int64_t)g * p.v.sh + d;
      load8(k, x);
      load8(k + HD / 2, x + 8);
      load8(v, y);
      load8(v + HD / 2, y + 8);
      if (turn_keys) rotate8(turn, x, x + 8);
      blk = paged4::block_of<HD>(c, pg, g, slot);
      if (c.mass && sub == 0) c.mass[(((int64_t)pg * c.G + g) << c.shift) + (slot & (c.page - 1))] = 0.f;
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] = y[e] = 0.f;
    }
    put_codes4<HD>(blk, slot & 15, sub, x);
    put_codes4<HD>(blk ? blk + paged4::HALF<HD> : nullptr, slot & 15, sub, y);
  }
}

template <typename T, int HD>
void launch4(Params4& p) {
  p.units = (int)(((int64_t)p.c.T * (HD / 16) + NT - 1) / NT);
  const int64_t qblocks = p.nq ? std::min<int64_t>(p.c.T, 1 << 16) : 0;
  // as many ways to share the heads as give every SM some CTAs: the look-ups in front of a token's heads are paid per way
  const int ways = (int)std::max<int64_t>(1, std::min<int64_t>(p.c.G, 8LL * num_sms() / p.units));
  const dim3 grid((unsigned)(p.units + (qblocks + ways - 1) / ways), (unsigned)ways);
  append4_kernel<T, HD><<<grid, NT, 0, stream()>>>(p);
}

}  // namespace kva

// k, v (T, G, hd), queries (T, H, hd): packed new tokens of any strides (rows that are not on 16-byte
// boundaries are copied first).  Writes the cache; returns the rotated queries, contiguous.
std::vector<at::Tensor> kv_append(at::Tensor k, at::Tensor v, at::Tensor ck, at::Tensor cv, at::Tensor ks, at::Tensor vs,
                                  at::Tensor table, at::Tensor cu, at::Tensor lens, int64_t max_new,
                                  c10::optional<at::Tensor> cos, c10::optional<at::Tensor> sin,
                                  c10::optional<at::Tensor> pos, std::vector<at::Tensor> queries) {
  using namespace kva;
  TORCH_CHECK(k.is_cuda() && k.dim() == 3 && v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type() &&
              k.device() == ck.device() && v.device() == ck.device(), "kv_append: k and v (T, G, hd) of one type on the cache's GPU");
  c10::cuda::CUDAGuard guard(k.device());
  const int64_t T = k.size(0), hd = k.size(2);
  Params p{};
  p.c = check_cache("kv_append", Layer{ck, cv, ks, vs, table, cu, lens}, T, hd);
  TORCH_CHECK(k.size(1) == p.c.G, "kv_append: ", p.c.G, " KV heads in the cache, got ", k.size(1));
  TORCH_CHECK(max_new >= 0, "kv_append: max_new must not be negative");
  std::vector<at::Tensor> outs = take_rows(p, k, v, cos, sin, pos, queries);
  if (T == 0 || p.c.B == 0) return outs;
  p.max_new = (int)std::min<int64_t>(max_new, T);
  TORCH_CHECK(T * p.c.G * 2 < (1LL << 31), "kv_append: sizes");
  MAMF_DISPATCH_FLOAT_BF16(k.scalar_type(), "kv_append", [&] {
    if (hd == 128) launch<scalar_t, 128>(p); else launch<scalar_t, 64>(p);
  });
  MAMF_LAUNCH_CHECK();
  return outs;
}

// The same into the 4-bit cache; new slots of `mass` are set to 0.
std::vector<at::Tensor> kv4_append(at::Tensor k, at::Tensor v, at::Tensor blocks, c10::optional<at::Tensor> mass,
                                   at::Tensor table, at::Tensor cu, at::Tensor lens, int64_t max_new,
                                   c10::optional<at::Tensor> cos, c10::optional<at::Tensor> sin,
                                   c10::optional<at::Tensor> pos, std::vector<at::Tensor> queries) {
  using namespace kva;
  TORCH_CHECK(k.is_cuda() && k.dim() == 3 && v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type() &&
              k.device() == blocks.device() && v.device() == blocks.device(), "kv_append: k and v (T, G, hd) of one type on the cache's GPU");
  c10::cuda::CUDAGuard guard(k.device());
  const int64_t T = k.size(0), hd = k.size(2);
  Params4 p{};
  p.c = paged4::check_cache4("kv_append", blocks, mass, table, &cu, lens, T, hd);
  TORCH_CHECK(k.size(1) == p.c.G, "kv_append: ", p.c.G, " KV heads in the cache, got ", k.size(1));
  TORCH_CHECK(max_new >= 0, "kv_append: max_new must not be negative");
  std::vector<at::Tensor> outs = take_rows(p, k, v, cos, sin, pos, queries);
  if (T == 0 || p.c.B == 0) return outs;
  p.max_new = (int)std::min<int64_t>(std::max<int64_t>(max_new, 1), T);      // one token is taken whatever was said, as by the 8-bit kernel
  TORCH_CHECK(T * (hd / 16) < (1LL << 31), "kv_append: sizes");
  MAMF_DISPATCH_FLOAT_BF16(k.scalar_type(), "kv_append", [&] {
    if (hd == 128) launch4<scalar_t, 128>(p); else launch4<scalar_t, 64>(p);
  });
  MAMF_LAUNCH_CHECK();
  return outs;
}

int64_t kv_append_error(bool clear) { return paged::take_code(kva::g_err, clear); }

}  // namespace mamf
