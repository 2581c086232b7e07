// Appending keys and values to the paged 8-bit cache, with the rotation of the keys (and of up to two
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
// no atomics.  Pages that take new tokens must belong to one sequence only.  Further CTAs rotate the queries.
#include "paged.cuh"

namespace mamf {
namespace kva {

using namespace paged;

constexpr int NT = 256;

__device__ int g_err = 0;
__device__ __forceinline__ void record(int code) { atomicCAS(&g_err, 0, code); }

struct Src { const void* p; int64_t st, sh; };       // token and head strides in elements

struct Params {
  Cache c;
  Src k, v, q[2];
  void* qo[2];
  const float *cos, *sin;                            // (n_pos, hd / 2) with row stride rot, null: no rotation
  int64_t rot;
  const int64_t* pos;                                // (T)
  int n_pos, H, units, per_seq, kv_blocks, nq;
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

// (a, b) -> (a cos - b sin, b cos + a sin).  Separate roundings, as elementwise operations have them, so
// that a value on the edge between two codes goes the same way.
template <int HD>
__device__ __forceinline__ void rotate8(const Params& p, int t, int d, float* a, float* b) {
  int64_t pos = p.pos[t];
  if (pos < 0 || pos >= p.n_pos) { record(ERR_POSITION); pos = pos < 0 ? 0 : p.n_pos - 1; }
  float c[8], s[8];
#pragma unroll
  for (int i = 0; i < 8; i += 4) {
    *reinterpret_cast<float4*>(c + i) = *reinterpret_cast<const float4*>(p.cos + pos * p.rot + d + i);
    *reinterpret_cast<float4*>(s + i) = *reinterpret_cast<const float4*>(p.sin + pos * p.rot + d + i);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float x = a[i], y = b[i], cv = c[i], sv = s[i];
    a[i] = __fsub_rn(__fmul_rn(x, cv), __fmul_rn(y, sv));
    b[i] = __fadd_rn(__fmul_rn(y, cv), __fmul_rn(x, sv));
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
  if (start < 0 || t0 < 0 || t0 + n > c.T || (p.per_seq > 0 && j == 0 && pages > p.per_seq)) {
    if (tid == 0) record(ERR_LENGTH);
    if (start < 0 || t0 < 0 || t0 + n > c.T) return;
  }
  if (j >= pages) return;
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
      if (!is_v && p.cos) rotate8<HD>(p, t, d, x[i], x[i] + 8);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float m = fabsf(x[i][e]);
        amax = fmaxf(amax, m < INFINITY ? m : 0.f);        // NaN and infinities do not set the scale
      }
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
    if (slot < hi) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        union { uint16_t c2[4]; uint2 raw; } w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w.c2[e] = enc2(x[i][8 * h + 2 * e] * inv, x[i][8 * h + 2 * e + 1] * inv);
        *reinterpret_cast<uint2*>(out + slot * HD + h * (HD / 2) + d) = w.raw;
      }
    }
  }
  if (lo > 0 && had != s) {
    const float f = had * inv;
    for (int i = tid; i < lo * HD / 16; i += NT) {
      union { uint4 raw; uint16_t c2[8]; } w;
      w.raw = *reinterpret_cast<const uint4*>(out + i * 16);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float2 v = dec2(w.c2[e]);
        w.c2[e] = enc2(v.x * f, v.y * f);
      }
      *reinterpret_cast<uint4*>(out + i * 16) = w.raw;
    }
  }
  __syncthreads();                              // every thread has read the old scale
  if (tid == 0 && had != s) *scale = s;
}

template <typename T, int HD>
__device__ __forceinline__ void rotate_queries(const Params& p, int64_t block, int64_t blocks) {
  constexpr int TPT = HD / 16;
  const int64_t per = (int64_t)p.c.T * p.H * TPT, total = per * p.nq;
  for (int64_t i = block * NT + threadIdx.x; i < total; i += blocks * NT) {
    const int which = i >= per;
    const int64_t r = i - which * per;
    const int d = (int)(r % TPT) * 8, h = (int)(r / TPT % p.H), t = (int)(r / TPT / p.H);
    const T* in = (const T*)p.q[which].p + (int64_t)t * p.q[which].st + (int64_t)h * p.q[which].sh;
    T* out = (T*)p.qo[which] + ((int64_t)t * p.H + h) * HD;
    float x[16];
    load8(in + d, x);
    load8(in + HD / 2 + d, x + 8);
    rotate8<HD>(p, t, d, x, x + 8);
    store8(out + d, x);
    store8(out + HD / 2 + d, x + 8);
  }
}

template <typename T, int HD, int NP>
__global__ void __launch_bounds__(NT) append_kernel(const __grid_constant__ Params p) {
  if ((int)blockIdx.x < p.units) append_block<T, HD, NP>(p);
  else {
    const int64_t qb = gridDim.x - p.units, layer = blockIdx.y + (int64_t)gridDim.y * blockIdx.z;
    rotate_queries<T, HD>(p, (blockIdx.x - p.units) + qb * layer, qb * gridDim.y * gridDim.z);
  }
}

template <typename T, int HD>
void launch(const Params& p, dim3 grid) {
  const int np = std::max(1, p.c.page * HD / (NT * 16));
  if (np == 1) append_kernel<T, HD, 1><<<grid, NT, 0, stream()>>>(p);
  else if (np == 2) append_kernel<T, HD, 2><<<grid, NT, 0, stream()>>>(p);
  else append_kernel<T, HD, 4><<<grid, NT, 0, stream()>>>(p);
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
  if (T == 0 || p.c.B == 0) return outs;
  p.k = src(k);
  p.v = src(v);
  p.nq = (int)queries.size();
  for (int i = 0; i < p.nq; ++i) { p.q[i] = src(queries[i]); p.qo[i] = outs[i].data_ptr(); }
  p.H = p.nq ? (int)queries[0].size(1) : 0;
  // units: (sequence, page) pairs that can take new tokens; the smaller of the two ways to number them
  const int64_t per_seq = max_new == 0 ? 0 : (max_new + p.c.page - 2) / p.c.page + 1;
  const int64_t even = per_seq * p.c.B, packed = T / p.c.page + 2LL * p.c.B;
  if (max_new <= 1 ? true : even <= packed) {
    p.per_seq = max_new <= 1 ? 1 : (int)per_seq;
    p.units = max_new <= 1 ? p.c.B : (int)even;
  } else {
    p.per_seq = 0;
    p.units = (int)packed;
  }
  const int64_t items = T * p.H * (hd / 16) * p.nq;
  const int64_t qblocks = std::min<int64_t>((items + NT - 1) / NT, 8 * num_sms());
  const int64_t qx = (qblocks + 2 * p.c.G - 1) / (2 * p.c.G);
  dim3 grid((unsigned)(p.units + qx), (unsigned)p.c.G, 2u);
  MAMF_DISPATCH_FLOAT_BF16(k.scalar_type(), "kv_append", [&] {
    if (hd == 128) launch<scalar_t, 128>(p, grid); else launch<scalar_t, 64>(p, grid);
  });
  MAMF_LAUNCH_CHECK();
  return outs;
}

int64_t kv_append_error() {
  int v = 0;
  MAMF_CUDA_CHECK(cudaMemcpyFromSymbol(&v, kva::g_err, sizeof(int)));
  if (v) {
    int z = 0;
    MAMF_CUDA_CHECK(cudaMemcpyToSymbol(kva::g_err, &z, sizeof(int)));
  }
  return v;
}

}  // namespace mamf
