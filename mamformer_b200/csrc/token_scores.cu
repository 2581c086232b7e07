// Scores of given tokens under softmax(logits / T): log probability, entropy and the k most
// likely alternatives, and their gradient.  Used by the policy / reference scoring of GRPO
// (mamformer/model.py:1042-1112 computes log_softmax and gathers) and by rollouts.
//
//   d = x - max(x), S0 = sum exp(d / T), S1 = sum d exp(d / T)
//   log p_j = d_j / T - log S0,   H = log S0 - S1 / (T S0)
//   dx_j = 1/T [ sum_i g_i (j == id_i) - p_j sum_i g_i - gH p_j (log p_j + H) ]
//
// with i over the target and the k alternatives.  Subtracting the maximum before dividing by T keeps
// rows of the type's lowest value finite at every temperature.  A logit of -inf has probability 0 and
// adds nothing to S1 (d is clamped at DMIN, where exp is 0).  A row of -inf only has no distribution:
// its log probabilities are -inf, its entropy and gradient 0.  NaN and +inf make the row NaN.
// Rows whose target is `ignore_index` (or outside the vocabulary) are not read: results 0, ids -1.
#include "common.cuh"

#include <cooperative_groups.h>

namespace mamf {
namespace ts {

constexpr int NT = 512;
constexpr int MAXK = 32;          // alternatives per row
constexpr int CAP = 1024;         // candidates kept in shared memory for the selection
constexpr float DMIN = -1e30f;
constexpr float LOG2E = 1.4426950408889634f;

struct Rows {                     // row r starts at base + (r / n1) * s0 + (r % n1) * s1 elements
  int64_t n1, s0, s1;
  __device__ __forceinline__ int64_t at(int64_t r) const { return (r / n1) * s0 + (r % n1) * s1; }
};

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

struct Stat { float m, s0, s1; };

// Adds b to a.  A side without any logit above -inf has s0 = 0 and is skipped.
__device__ __forceinline__ void merge(Stat& a, const Stat& b, float k2) {
  if (b.m == -INFINITY) return;
  if (a.m == -INFINITY) { a = b; return; }
  const float M = max_nan(a.m, b.m);
  const float da = max_nan(a.m - M, DMIN), db = max_nan(b.m - M, DMIN);
  const float fa = ex2(da * k2), fb = ex2(db * k2);
  a.s1 = fmaf(da, a.s0, a.s1) * fa + fmaf(db, b.s0, b.s1) * fb;
  a.s0 = a.s0 * fa + b.s0 * fb;
  a.m = M;
}

// Order of the alternatives: larger logit first, then the lower index; NaN above everything and
// -0 equal to +0.  0 is below every element.
__device__ __forceinline__ uint32_t order(float x) {
  if (x != x) return 0xFFFFFFFFu;
  const uint32_t b = __float_as_uint(x + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ uint64_t key_of(float x, uint32_t idx) {
  return ((uint64_t)order(x) << 32) | (0xFFFFFFFFu - idx);
}
__device__ __forceinline__ uint32_t key_index(uint64_t k) { return 0xFFFFFFFFu - (uint32_t)k; }
__device__ __forceinline__ uint64_t warp_max_u64(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const uint64_t w = __shfl_xor_sync(0xffffffffu, v, o);
    v = w > v ? w : v;
  }
  return v;
}

struct FwdParams {
  Rows rows;
  const int64_t* target;
  float *lp, *ent, *top_lp, *stats;      // (R), (R), (R, k), (R, 2) = {max, log S0}
  int64_t* top_id;
  int64_t ignore;
  int V, k;
  float inv_t;
};

// One CTA per row.
template <typename T>
__global__ void __launch_bounds__(NT) scores_fwd_kernel(const T* __restrict__ logits, FwdParams p) {
  constexpr int VEC = 16 / sizeof(T);
  __shared__ Stat sm_stat[NT / 32];
  __shared__ Stat sm_all;
  __shared__ uint64_t sm_key[NT / 32];
  __shared__ uint64_t sm_top[MAXK];
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int64_t row = blockIdx.x;
  const int64_t tgt = p.target[row];
  if (tgt == p.ignore || tgt < 0 || tgt >= p.V) {
    if (tid == 0) {
      p.lp[row] = 0.f; p.ent[row] = 0.f;
      p.stats[2 * row] = -INFINITY; p.stats[2 * row + 1] = 0.f;
    }
    if (tid < p.k) { p.top_lp[row * p.k + tid] = 0.f; p.top_id[row * p.k + tid] = -1; }
    return;
  }
  const T* x = logits + p.rows.at(row);
  const float k2 = p.inv_t * LOG2E;
  // elements before the first 16-byte boundary and after the last full vector are taken one by one
  const int head = min(p.V, (int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T)));
  const int nv = (p.V - head) / VEC;
  const int rem = p.V - nv * VEC;
  const T* xv = x + head;

  Stat st{-INFINITY, 0.f, 0.f};
  auto add = [&](const float* v, int n) {
    float cm = v[0];
    for (int i = 1; i < n; ++i) cm = max_nan(cm, v[i]);
    if (!(cm <= st.m) && st.m == st.m) {
      Stat b{cm, 0.f, 0.f};
      if (st.m != -INFINITY) {
        const float d = max_nan(st.m - cm, DMIN), f = ex2(d * k2);
        b.s1 = fmaf(d, st.s0, st.s1) * f;
        b.s0 = st.s0 * f;
      }
      st = b;
    }
    if (st.m == -INFINITY) return;
    for (int i = 0; i < n; ++i) {
      const float d = max_nan(v[i] - st.m, DMIN), e = ex2(d * k2);
      st.s0 += e;
      st.s1 = fmaf(d, e, st.s1);
    }
  };
  for (int i = tid; i < nv; i += NT) {
    const Vec16<T> v = ld16(xv + (int64_t)i * VEC);
    float f[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) f[j] = to_f(v.v[j]);
    add(f, VEC);
  }
  if (tid < rem) {
    const float f = to_f(x[tid < head ? tid : nv * VEC + tid]);
    add(&f, 1);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Stat b{__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s0, o),
           __shfl_xor_sync(0xffffffffu, st.s1, o)};
    merge(st, b, k2);
  }
  if (lane == 0) sm_stat[wid] = st;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < NT / 32; ++w) merge(st, sm_stat[w], k2);
    const bool none = st.m == -INFINITY;
    const float ls = none ? 0.f : logf(st.s0);
    p.lp[row] = none ? -INFINITY : (to_f(x[tgt]) - st.m) * p.inv_t - ls;
    p.ent[row] = none ? 0.f : ls - st.s1 * p.inv_t / st.s0;
    p.stats[2 * row] = st.m;
    p.stats[2 * row + 1] = ls;
    sm_all = Stat{st.m, ls, 0.f};
  }
  // k rounds: the largest element below the last one taken
  uint64_t last = ~0ull;
  for (int r = 0; r < p.k; ++r) {
    uint64_t best = 0;
    for (int i = tid; i < p.V; i += NT) {
      const uint64_t k = key_of(to_f(x[i]), (uint32_t)i);
      if (k < last && k > best) best = k;
    }
    best = warp_max_u64(best);
    __syncthreads();
    if (lane == 0) sm_key[wid] = best;
    __syncthreads();
    best = 0;
    for (int w = 0; w < NT / 32; ++w) best = sm_key[w] > best ? sm_key[w] : best;
    if (tid == 0) sm_top[r] = best;
    last = best;
  }
  __syncthreads();
  if (tid < p.k) {
    const uint32_t id = key_index(sm_top[tid]);
    p.top_id[row * p.k + tid] = id;
    p.top_lp[row * p.k + tid] = sm_all.m == -INFINITY ? -INFINITY : (to_f(x[id]) - sm_all.m) * p.inv_t - sm_all.s0;
  }
}

struct BwdParams {
  Rows rows;
  const int64_t* target;
  const float *stats, *ent;
  const int64_t* top_id;
  const float *g_lp, *g_ent, *g_top;     // any may be null (no gradient)
  int64_t ignore;
  int V, k;
  float inv_t;
};

constexpr int SEG = 16384;               // elements of a row per CTA

// dx_j = p_j (a log p_j + b) with a = -gH / T, b = -(sum g + gH H) / T; the target's and the
// alternatives' elements get their own g on top, written after the rest of the segment.
template <typename T>
__global__ void __launch_bounds__(NT) scores_bwd_kernel(const T* __restrict__ logits, T* __restrict__ out, BwdParams p) {
  constexpr int VEC = 16 / sizeof(T);
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  const int c0 = blockIdx.y * SEG, c1 = min(p.V, c0 + SEG);
  const T* x = logits + p.rows.at(row);
  T* y = out + row * p.V;
  const int64_t tgt = p.target[row];
  const float m = p.stats[2 * row], ls = p.stats[2 * row + 1];
  const bool dead = tgt == p.ignore || tgt < 0 || tgt >= p.V || m == -INFINITY;
  float G = 0.f, a = 0.f, b = 0.f;
  if (!dead) {
    const float gh = p.g_ent ? p.g_ent[row] : 0.f;
    if (p.g_lp) G = p.g_lp[row];
    if (p.g_top) for (int i = 0; i < p.k; ++i) G += p.g_top[row * p.k + i];
    a = -gh * p.inv_t;
    b = -(G + gh * p.ent[row]) * p.inv_t;
  }
  auto grad = [&](float v) {
    const float lp = max_nan(fmaf(v - m, p.inv_t, -ls), DMIN);
    return ex2(lp * LOG2E) * fmaf(a, lp, b);
  };
  // the columns that also have a gradient of their own
  const int extra = dead ? 0 : 1 + (p.g_top ? p.k : 0);
  int col = -1;
  float fix = 0.f;
  if (tid < extra) {
    col = (int)(tid == 0 ? tgt : p.top_id[row * p.k + tid - 1]);
    float own = (p.g_lp && col == tgt) ? p.g_lp[row] : 0.f;
    if (p.g_top)
      for (int i = 0; i < p.k; ++i)
        if (p.top_id[row * p.k + i] == col) own += p.g_top[row * p.k + i];
    if (col < c0 || col >= c1) col = -1;
    else fix = grad(to_f(x[col])) + own * p.inv_t;
  }
  const bool vec = ((reinterpret_cast<uintptr_t>(x + c0) ^ reinterpret_cast<uintptr_t>(y + c0)) & 15) == 0;
  const int head = vec ? min(c1 - c0, (int)(((16 - (reinterpret_cast<uintptr_t>(y + c0) & 15)) & 15) / sizeof(T))) : 0;
  const int nv = vec ? (c1 - c0 - head) / VEC : 0;
  const int rem = c1 - c0 - nv * VEC;
  for (int i = tid; i < nv; i += NT) {
    const int64_t o = c0 + head + (int64_t)i * VEC;
    Vec16<T> v;
    if (dead) v.raw = make_uint4(0, 0, 0, 0);
    else {
      v = ld16(x + o);
#pragma unroll
      for (int j = 0; j < VEC; ++j) v.v[j] = from_f<T>(grad(to_f(v.v[j])));
    }
    st16(y + o, v);
  }
  for (int i = tid; i < rem; i += NT) {
    const int c = c0 + (i < head ? i : nv * VEC + i);
    y[c] = from_f<T>(dead ? 0.f : grad(to_f(x[c])));
  }
  __syncthreads();
  if (col >= 0) y[col] = from_f<T>(fix);
}

// logits as two or three dimensions with adjacent vocabulary entries: a view, or a copy
static at::Tensor as_rows(const at::Tensor& logits) {
  TORCH_CHECK(logits.dim() >= 1 && logits.size(-1) >= 1, "token_scores: logits (.., V)");
  if (logits.dim() >= 2 && logits.dim() <= 3 && logits.stride(-1) == 1) return logits;
  return logits.reshape({-1, logits.size(-1)}).contiguous();
}
static Rows rows_of(const at::Tensor& logits) {
  if (logits.dim() == 2) return Rows{1, logits.stride(0), 0};
  return Rows{std::max<int64_t>(1, logits.size(1)), logits.stride(0), logits.stride(1)};
}

static int64_t check(const at::Tensor& logits, const at::Tensor& target, double temperature, int64_t top_k) {
  TORCH_CHECK(temperature > 0 && std::isfinite(temperature), "token_scores: temperature must be positive and finite, got ", temperature);
  TORCH_CHECK(logits.is_cuda() && target.is_cuda() && logits.device() == target.device(),
              "token_scores: logits and targets on one GPU");
  TORCH_CHECK(target.scalar_type() == at::kLong && target.is_contiguous(), "token_scores: contiguous int64 targets");
  const int64_t V = logits.size(-1);
  TORCH_CHECK(V >= 1 && V < (1LL << 31) - SEG, "token_scores: vocabulary of ", V);
  const int64_t R = logits.numel() / V;
  TORCH_CHECK(target.numel() == R, "token_scores: one target per row (", R, " rows, ", target.numel(), " targets)");
  TORCH_CHECK(R < (1LL << 31), "token_scores: at most 2^31 - 1 rows");
  TORCH_CHECK(top_k >= 0 && top_k <= std::min<int64_t>(MAXK, V), "token_scores: top_k from 0 to ", std::min<int64_t>(MAXK, V), ", got ", top_k);
  return R;
}

}  // namespace ts

// logits (.., V), up to two leading dimensions of any strides without a copy; target (..) int64.
// -> log_probs, entropy (like target, fp32), top_log_probs, top_ids (.., k), stats (R, 2)
std::vector<at::Tensor> token_scores_fwd(at::Tensor logits, at::Tensor target, int64_t ignore_index, double temperature,
                                         int64_t top_k) {
  using namespace ts;
  logits = as_rows(logits);
  const int64_t R = check(logits, target, temperature, top_k);
  c10::cuda::CUDAGuard guard(logits.device());
  auto f32 = logits.options().dtype(at::kFloat);
  at::Tensor lp = at::empty(target.sizes(), f32), ent = at::empty(target.sizes(), f32);
  auto tk = target.sizes().vec();
  tk.push_back(top_k);
  at::Tensor top_lp = at::empty(tk, f32), top_id = at::empty(tk, target.options()), stats = at::empty({R, 2}, f32);
  if (R > 0) {
    FwdParams p{rows_of(logits), target.data_ptr<int64_t>(), lp.data_ptr<float>(), ent.data_ptr<float>(),
                top_lp.data_ptr<float>(), stats.data_ptr<float>(), top_id.data_ptr<int64_t>(), ignore_index,
                (int)logits.size(-1), (int)top_k, (float)(1.0 / temperature)};
    MAMF_DISPATCH_FLOAT_BF16(logits.scalar_type(), "token_scores", [&] {
      scores_fwd_kernel<scalar_t><<<(unsigned)R, NT, 0, stream()>>>((const scalar_t*)logits.data_ptr(), p);
    });
    MAMF_LAUNCH_CHECK();
  }
  return {lp, ent, top_lp, top_id, stats};
}

// -> d logits, contiguous, of the logits' type.  g_* are contiguous fp32 or absent.
at::Tensor token_scores_bwd(at::Tensor logits, at::Tensor target, int64_t ignore_index, double temperature, at::Tensor stats,
                            at::Tensor ent, at::Tensor top_id, c10::optional<at::Tensor> g_lp,
                            c10::optional<at::Tensor> g_ent, c10::optional<at::Tensor> g_top) {
  using namespace ts;
  const int64_t k = top_id.size(-1);
  const auto shape = logits.sizes().vec();
  logits = as_rows(logits);
  const int64_t R = check(logits, target, temperature, k);
  c10::cuda::CUDAGuard guard(logits.device());
  auto ptr = [&](const c10::optional<at::Tensor>& g, int64_t n) -> const float* {
    if (!g.has_value() || n == 0) return nullptr;
    TORCH_CHECK(g->scalar_type() == at::kFloat && g->is_contiguous() && g->numel() == n && g->device() == logits.device(),
                "token_scores: contiguous fp32 gradients");
    return g->data_ptr<float>();
  };
  at::Tensor out = at::empty(shape, logits.options());
  if (R == 0) return out;
  BwdParams p{rows_of(logits), target.data_ptr<int64_t>(), stats.data_ptr<float>(), ent.data_ptr<float>(),
              top_id.data_ptr<int64_t>(), ptr(g_lp, R), ptr(g_ent, R), ptr(g_top, R * k), ignore_index,
              (int)logits.size(-1), (int)k, (float)(1.0 / temperature)};
  MAMF_DISPATCH_FLOAT_BF16(logits.scalar_type(), "token_scores", [&] {
    dim3 grid((unsigned)R, (unsigned)((p.V + SEG - 1) / SEG));
    scores_bwd_kernel<scalar_t><<<grid, NT, 0, stream()>>>((const scalar_t*)logits.data_ptr(), (scalar_t*)out.data_ptr(), p);
  });
  MAMF_LAUNCH_CHECK();
  return out;
}

}  // namespace mamf
