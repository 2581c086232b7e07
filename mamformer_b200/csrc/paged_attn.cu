// Attention over the paged 8-bit cache (layout in paged.cuh): one warp per query row.
#include "paged.cuh"

namespace mamf {
namespace pa {

using namespace paged;

constexpr int NT = 128;

__device__ int g_err = 0;

struct Params {
  Cache c;
  const void *q1, *q2;
  void* out;
  const float* lam;
  int64_t st1, sh1, st2, sh2;
  int H, window;
  float scale_log2;
};

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// lane l holds dims [l * D, (l + 1) * D), D = HD / 32
template <typename T, int HD>
__global__ void __launch_bounds__(NT) simple_kernel(Params p) {
  constexpr int D = HD / 32;
  const Cache& c = p.c;
  const int64_t item = (int64_t)blockIdx.x * (NT / 32) + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (item >= (int64_t)c.T * p.H) return;
  const int t = (int)(item / p.H), h = (int)(item % p.H), g = h / (p.H / c.G);
  const int b = sequence_of(c.cu, c.B, t);
  T* out = (T*)p.out + item * HD + lane * D;
  const int maps = p.q2 ? 2 : 1;
  float res[D] = {};
  if (b >= 0) {
    const int n = c.cu[b + 1] - c.cu[b], len = c.lens[b];
    const int at = len - n + t - c.cu[b];                    // the query's slot
    const int first = p.window > 0 ? max(0, at - p.window + 1) : 0;
    for (int map = 0; map < maps; ++map) {
      const T* q = map ? (const T*)p.q2 + t * p.st2 + h * p.sh2 : (const T*)p.q1 + t * p.st1 + h * p.sh1;
      float qv[D], o[D] = {}, m = -INFINITY, l = 0.f;
      for (int i = 0; i < D; ++i) qv[i] = to_f(q[lane * D + i]) * p.scale_log2;
      for (int s = first; s <= min(at, len - 1); ++s) {
        const int j = s / c.page;
        const int pg = j < c.W ? c.table[(int64_t)b * c.W + j] : -1;
        if (pg < 0 || pg >= c.P) { if (lane == 0) atomicCAS(&g_err, 0, (int)ERR_PAGE); continue; }
        const int64_t row = (((int64_t)pg * c.G + g) * c.page + s % c.page) * HD + lane * D;
        const float ks = c.ks[(int64_t)pg * c.G + g], vs = c.vs[(int64_t)pg * c.G + g];
        float dot = 0.f;
        for (int i = 0; i < D; i += 2) {
          const float2 kv = dec2(*reinterpret_cast<const uint16_t*>(c.k + row + i));
          dot = fmaf(qv[i], kv.x, fmaf(qv[i + 1], kv.y, dot));
        }
        dot = warp_sum(dot) * ks;
        const float mn = fmaxf(m, dot), f = m == -INFINITY ? 0.f : ex2(m - mn), e = ex2(dot - mn);
        l = l * f + e;
        for (int i = 0; i < D; i += 2) {
          const float2 vv = dec2(*reinterpret_cast<const uint16_t*>(c.v + row + i));
          o[i] = o[i] * f + e * vs * vv.x;
          o[i + 1] = o[i + 1] * f + e * vs * vv.y;
        }
        m = mn;
      }
      const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
      const float w = maps == 1 ? 1.f : (map ? -p.lam[h] : 1.f) / (1.f - p.lam[h] + 1e-8f);
      for (int i = 0; i < D; ++i) res[i] += o[i] * inv * w;
    }
  }
  for (int i = 0; i < D; ++i) out[i] = from_f<T>(res[i]);
}

}  // namespace pa

// q1, q2 (T, H, hd) bf16 or f16 packed queries -> (T, H, hd)
at::Tensor paged_attention(at::Tensor q1, c10::optional<at::Tensor> q2, c10::optional<at::Tensor> lam, at::Tensor ck,
                           at::Tensor cv, at::Tensor ks, at::Tensor vs, at::Tensor table, at::Tensor cu, at::Tensor lens,
                           int64_t max_new, int64_t window, double scale) {
  using namespace pa;
  TORCH_CHECK(q1.is_cuda() && q1.dim() == 3 && q1.device() == ck.device() && (q1.scalar_type() == at::kBFloat16 || q1.scalar_type() == at::kHalf),
              "paged_attention: bf16 or f16 queries (T, H, hd) on the cache's GPU");
  c10::cuda::CUDAGuard guard(q1.device());
  const int64_t T = q1.size(0), H = q1.size(1), hd = q1.size(2);
  Params p{};
  p.c = check_cache("paged_attention", Layer{ck, cv, ks, vs, table, cu, lens}, T, hd);
  TORCH_CHECK(H >= 1 && p.c.G >= 1 && H % p.c.G == 0, "paged_attention: ", H, " query heads over ", p.c.G, " KV heads");
  TORCH_CHECK(window >= 0 && max_new >= 0, "paged_attention: window and max_new must not be negative");
  q1 = rows16(q1);
  p.q1 = q1.data_ptr(); p.st1 = q1.stride(0); p.sh1 = q1.stride(1);
  if (q2.has_value()) {
    TORCH_CHECK(lam.has_value() && q2->is_cuda() && q2->device() == q1.device() && q2->sizes() == q1.sizes() && q2->scalar_type() == q1.scalar_type(),
                "paged_attention: q2 like q1, with lam");
    TORCH_CHECK(lam->is_cuda() && lam->device() == q1.device() && lam->scalar_type() == at::kFloat && lam->is_contiguous() && lam->numel() == H,
                "paged_attention: fp32 lam (H)");
    q2 = rows16(*q2);
    p.q2 = q2->data_ptr(); p.st2 = q2->stride(0); p.sh2 = q2->stride(1);
    p.lam = lam->data_ptr<float>();
  } else {
    TORCH_CHECK(!lam.has_value(), "paged_attention: lam without q2");
  }
  at::Tensor out = at::empty({T, H, hd}, q1.options());
  if (T == 0) return out;
  p.out = out.data_ptr();
  p.H = (int)H;
  p.window = (int)std::min<int64_t>(window, 1LL << 30);
  p.scale_log2 = (float)(scale * 1.4426950408889634);
  const int64_t blocks = (T * H + NT / 32 - 1) / (NT / 32);
  TORCH_CHECK(blocks < (1LL << 31), "paged_attention: sizes");
  if (q1.scalar_type() == at::kBFloat16) {
    if (hd == 128) simple_kernel<__nv_bfloat16, 128><<<(unsigned)blocks, NT, 0, stream()>>>(p);
    else simple_kernel<__nv_bfloat16, 64><<<(unsigned)blocks, NT, 0, stream()>>>(p);
  } else {
    if (hd == 128) simple_kernel<__half, 128><<<(unsigned)blocks, NT, 0, stream()>>>(p);
    else simple_kernel<__half, 64><<<(unsigned)blocks, NT, 0, stream()>>>(p);
  }
  MAMF_LAUNCH_CHECK();
  return out;
}

int64_t paged_attention_error() {
  int v = 0;
  MAMF_CUDA_CHECK(cudaMemcpyFromSymbol(&v, pa::g_err, sizeof(int)));
  if (v) {
    int z = 0;
    MAMF_CUDA_CHECK(cudaMemcpyToSymbol(pa::g_err, &z, sizeof(int)));
  }
  return v;
}

}  // namespace mamf
