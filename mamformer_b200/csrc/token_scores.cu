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
// Rows whose target is `ignore_index` are not read: results 0, ids -1.  Nor are those of another target outside the
// vocabulary: NaN, ids -1, no gradient, and an error word.
//
// 3686 x 128000 bf16: forward 160 us (5.9 TB/s; with 20 alternatives 210 us), gradient 311-328 us (5.9 TB/s).
// DRAM bounds both, one exponential per logit (the MUFU at 60-70%) comes next.
#include "common.cuh"
#include "f32x2.cuh"

#include <type_traits>

namespace mamf {
namespace ts {

constexpr int MAXK = 32;          // alternatives per row
constexpr int CAP = 1024;         // candidates kept in shared memory for the selection
constexpr float DMIN = -1e30f;
constexpr float LOG2E = 1.4426950408889634f;

__device__ int g_err = 0;         // 1: a target outside the vocabulary

struct Rows {                     // row r starts at base + (r / n1) * s0 + (r % n1) * s1 elements
  int64_t n1, s0, s1;
  __device__ __forceinline__ int64_t at(int64_t r) const { return (r / n1) * s0 + (r % n1) * s1; }
};

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// Good to 2^-22.  With that and the multiplication by a rounded 1 / T, scores of 32000 fp32 logits are 1.2e-7 of their size
// from 64 bits, where torch's exp and a division by T come to 6.6e-8: the pass is next to the MUFU's bound as it is.
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
__device__ __forceinline__ float key_value(uint64_t k) {          // NaN for the NaN key, +0 for both zeros
  const uint32_t o = (uint32_t)(k >> 32);
  return __uint_as_float((o & 0x80000000u) ? o & 0x7FFFFFFFu : ~o);
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
  float *lp, *ent, *top_lp, *stats;      // (R), (R), (R, k), (R, 2) = {max, log S0} or null
  int64_t* top_id;
  int64_t ignore;
  int V, k;
  float inv_t;
};

// maximum of a 16-byte vector, NaN if one is in it
__device__ __forceinline__ float vec_max(const Vec16<float>& v) { return max_nan(max_nan(v.v[0], v.v[1]), max_nan(v.v[2], v.v[3])); }
__device__ __forceinline__ float vec_max(const Vec16<__nv_bfloat16>& v) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v.raw);
  const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
  return max_nan(__bfloat162float(m.x), __bfloat162float(m.y));
}
__device__ __forceinline__ float vec_max(const Vec16<__half>& v) {
  const __half2* h = reinterpret_cast<const __half2*>(&v.raw);
  const __half2 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
  return max_nan(__half2float(m.x), __half2float(m.y));
}

// Raises a thread's running maximum to cm and scales its sums to it.
__device__ __forceinline__ void raise(Stat& st, float cm, float k2) {
  if (cm <= st.m || st.m != st.m) return;                 // a NaN maximum stays, and so do its sums
  if (st.m != -INFINITY) {
    const float d = max_nan(st.m - cm, DMIN), f = ex2(d * k2);
    st.s1 = fmaf(d, st.s0, st.s1) * f;
    st.s0 *= f;
  }
  st.m = cm;
}
template <typename T>
__device__ __forceinline__ void add_vec(const Vec16<T>& v, float m, float k2, uint64_t& s0, uint64_t& s1) {
  constexpr int VEC = 16 / sizeof(T);
  const uint64_t nm = pk(-m, -m), kk = pk(k2, k2);
#pragma unroll
  for (int j = 0; j < VEC; j += 2) {
    float a, b;
    unpk(add2(pk(to_f(v.v[j]), to_f(v.v[j + 1])), nm), a, b);
    const uint64_t d = pk(max_nan(a, DMIN), max_nan(b, DMIN));
    unpk(mul2(d, kk), a, b);
    const uint64_t e = pk(ex2(a), ex2(b));
    s0 = add2(s0, e);
    s1 = fma2(d, e, s1);
  }
}

template <int CL> __device__ __forceinline__ int cluster_rank() {
  if (CL == 1) return 0;
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return (int)r;
}
template <int CL> __device__ __forceinline__ void cluster_sync() {
  if (CL > 1) asm volatile("barrier.cluster.arrive.aligned;\n barrier.cluster.wait.aligned;" ::: "memory");
}
// the same variable of CTA `rank` of the cluster
template <typename V> __device__ __forceinline__ V* in_cta(V* p, int rank) {
  uint64_t r;
  asm volatile("mapa.u64 %0, %1, %2;" : "=l"(r) : "l"(p), "r"(rank));
  return reinterpret_cast<V*>(r);
}

// A row for each cluster of CL CTAs (CL = 1 where there are enough rows to fill the GPU): one pass with a
// running maximum per thread.  The alternatives come from the maxima: at least k threads hold an element no
// smaller than the k-th largest of the threads' maxima, so only threads whose maximum reaches that bound can
// hold an alternative, and only their elements (about k / NT of the row) are read again, by all threads.
template <typename T, int CL, int NT>
__global__ void __launch_bounds__(NT, NT == 512 ? 3 : 5) scores_fwd_kernel(const T* __restrict__ logits, const __grid_constant__ FwdParams p) {
  constexpr int VEC = 16 / sizeof(T), U = 4;
  __shared__ Stat sm_stat[NT / 32], sm_cta;
  __shared__ uint64_t sm_key[NT / 32], sm_top[MAXK], sm_cand[CAP];
  __shared__ uint32_t sm_lo[NT / 32], sm_hi[NT / 32];
  __shared__ int sm_hot[NT], sm_nh, sm_n;
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5, rank = cluster_rank<CL>();
  const int64_t row = blockIdx.x / CL;
  const int64_t tgt = p.target[row];
  if (tgt == p.ignore || tgt < 0 || tgt >= p.V) {
    if (rank > 0) return;
    const float none = tgt == p.ignore ? 0.f : NAN;
    if (tid == 0) {
      if (tgt != p.ignore) g_err = 1;
      p.lp[row] = none; p.ent[row] = none;
      if (p.stats) { p.stats[2 * row] = -INFINITY; p.stats[2 * row + 1] = 0.f; }
    }
    if (tid < p.k) { p.top_lp[row * p.k + tid] = none; p.top_id[row * p.k + tid] = -1; }
    return;
  }
  const T* x = logits + p.rows.at(row);
  const float k2 = p.inv_t * LOG2E;
  // elements before the first 16-byte boundary and after the last full vector are taken one by one by CTA 0
  const int head = min(p.V, (int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T)));
  const int nv = (p.V - head) / VEC, rem = rank == 0 ? p.V - nv * VEC : 0;
  const T* xv = x + head;
  const float x_tgt = rank == 0 && tid == 0 ? to_f(x[tgt]) : 0.f;
  const int g0 = rank * NT + tid;
  auto rem_at = [&](int i) { return i < head ? i : nv * VEC + i; };

  Stat st{-INFINITY, 0.f, 0.f};
  int i = g0;
  for (; i + (U - 1) * CL * NT < nv; i += U * CL * NT) {
    Vec16<T> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = ld16(xv + (int64_t)(i + u * CL * NT) * VEC);
    float cm = vec_max(v[0]);
#pragma unroll
    for (int u = 1; u < U; ++u) cm = max_nan(cm, vec_max(v[u]));
    raise(st, cm, k2);
    if (st.m == -INFINITY) continue;
    uint64_t s0 = pk(st.s0, 0.f), s1 = pk(st.s1, 0.f);
#pragma unroll
    for (int u = 0; u < U; ++u) add_vec(v[u], st.m, k2, s0, s1);
    float a, b;
    unpk(s0, a, b);
    st.s0 = a + b;
    unpk(s1, a, b);
    st.s1 = a + b;
  }
  for (; i < nv; i += CL * NT) {
    const Vec16<T> v = ld16(xv + (int64_t)i * VEC);
    raise(st, vec_max(v), k2);
    if (st.m == -INFINITY) continue;
    uint64_t s0 = pk(st.s0, 0.f), s1 = pk(st.s1, 0.f);
    add_vec(v, st.m, k2, s0, s1);
    float a, b;
    unpk(s0, a, b);
    st.s0 = a + b;
    unpk(s1, a, b);
    st.s1 = a + b;
  }
  if (tid < rem) {
    const float f = to_f(x[rem_at(tid)]);
    raise(st, f, k2);
    if (st.m != -INFINITY) {
      const float d = max_nan(f - st.m, DMIN), e = ex2(d * k2);
      st.s0 += e;
      st.s1 = fmaf(d, e, st.s1);
    }
  }
  const uint32_t mine = (g0 < nv || tid < rem) ? order(st.m) : 0u;     // 0: a thread without elements

#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Stat b{__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s0, o),
           __shfl_xor_sync(0xffffffffu, st.s1, o)};
    merge(st, b, k2);
  }
  if (lane == 0) sm_stat[wid] = st;
  if (p.k > 0) {
    const uint32_t lo = __reduce_min_sync(0xffffffffu, mine), hi = __reduce_max_sync(0xffffffffu, mine);
    if (lane == 0) { sm_lo[wid] = lo; sm_hi[wid] = hi; }
  }
  if (tid == 0) { sm_nh = 0; sm_n = 0; }
  __syncthreads();
  if (wid == 0) {
    st = lane < NT / 32 ? sm_stat[lane] : Stat{-INFINITY, 0.f, 0.f};
#pragma unroll
    for (int o = NT / 64; o > 0; o >>= 1) {
      Stat b{__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s0, o),
             __shfl_xor_sync(0xffffffffu, st.s1, o)};
      merge(st, b, k2);
    }
    if (lane == 0) sm_cta = st;
  }

  if (p.k > 0) {
    // A bound that at least k threads reach: bits that all maxima share, then one bit at a time, until few
    // more than k threads reach it.  Values of the 16-bit types differ in the upper bits only.
    uint32_t lo = ~0u, hi = 0;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) { lo = min(lo, sm_lo[w]); hi = max(hi, sm_hi[w]); }
    constexpr uint32_t LOW = std::is_same<T, float>::value ? 1u : std::is_same<T, __half>::value ? 1u << 13 : 1u << 16;
    uint32_t bit = lo == hi ? 0u : 0x80000000u >> __clz(lo ^ hi);
    uint32_t bound = bit ? lo & ~(2 * bit - 1) : lo & ~(LOW - 1);
    for (; bit >= LOW; bit >>= 1) {
      const int n = __syncthreads_count(mine >= (bound | bit));
      if (n >= p.k) bound |= bit;
      if (n >= p.k && n <= p.k + 4) break;
    }
    if (mine >= bound && mine) sm_hot[atomicAdd(&sm_nh, 1)] = tid;
    __syncthreads();
    const int per = (nv + CL * NT - 1) / (CL * NT), items = sm_nh * per;
    auto offer = [&](float f, int idx) {
      if (order(f) < bound) return;
      const int at = atomicAdd(&sm_n, 1);
      if (at < CAP) sm_cand[at] = key_of(f, (uint32_t)idx);
    };
    for (int it = tid; it < items; it += 4 * NT) {
      Vec16<T> w[4];
      int at[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = it + u * NT;
        at[u] = i < items ? rank * NT + sm_hot[i / per] + i % per * (CL * NT) : nv;
        if (at[u] < nv) w[u] = ld16(xv + (int64_t)at[u] * VEC);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (at[u] >= nv || order(vec_max(w[u])) < bound) continue;
#pragma unroll
        for (int e = 0; e < VEC; ++e) offer(to_f(w[u].v[e]), head + at[u] * VEC + e);
      }
    }
    if (tid < rem) offer(to_f(x[rem_at(tid)]), rem_at(tid));
    __syncthreads();
    const int n = sm_n;
    if (tid < p.k) sm_top[tid] = 0;
    __syncthreads();
    if (n <= CAP) {
      for (int c = tid; c < n; c += NT) {
        const uint64_t me = sm_cand[c];
        int above = 0;
        for (int d = 0; d < n && above < p.k; ++d) above += sm_cand[d] > me;
        if (above < p.k) sm_top[above] = me;
      }
    } else {
      // more equal elements than fit: the largest key below the last one taken, k times
      uint64_t last = ~0ull;
      for (int r = 0; r < p.k; ++r) {
        uint64_t best = 0;
        auto look = [&](float f, int idx) {
          const uint64_t k = key_of(f, (uint32_t)idx);
          if (k < last && k > best) best = k;
        };
        for (int v = g0; v < nv; v += CL * NT) {
          const Vec16<T> w = ld16(xv + (int64_t)v * VEC);
#pragma unroll
          for (int e = 0; e < VEC; ++e) look(to_f(w.v[e]), head + v * VEC + e);
        }
        if (tid < rem) look(to_f(x[rem_at(tid)]), rem_at(tid));
        best = warp_max_u64(best);
        __syncthreads();
        if (lane == 0) sm_key[wid] = best;
        __syncthreads();
        for (int w = 0; w < NT / 32; ++w) best = sm_key[w] > best ? sm_key[w] : best;
        if (tid == 0) sm_top[r] = best;
        last = best;
      }
    }
  }
  __syncthreads();
  cluster_sync<CL>();
  if (rank == 0) {
    // every thread joins the CTAs' sums: it costs less than passing them on
    Stat all = sm_cta;
    for (int r = 1; r < CL; ++r) merge(all, *in_cta(&sm_cta, r), k2);
    const bool none = all.m == -INFINITY;
    const float ls = none ? 0.f : logf(all.s0);
    auto log_p = [&](float f) { return none ? -INFINITY : (f - all.m) * p.inv_t - ls; };
    if (tid == 0) {
      p.lp[row] = log_p(x_tgt);
      p.ent[row] = none ? 0.f : ls - all.s1 * p.inv_t / all.s0;
      if (p.stats) { p.stats[2 * row] = all.m; p.stats[2 * row + 1] = ls; }
    }
    auto write = [&](int at, uint64_t key) {
      p.top_id[row * p.k + at] = key_index(key);
      p.top_lp[row * p.k + at] = log_p(key_value(key));
    };
    if (CL == 1) {
      if (tid < p.k) write(tid, sm_top[tid]);
    } else {
      // CL lists of k, each key in one of them: its rank among all of them
      for (int c = tid; c < CL * p.k; c += NT) sm_cand[c] = *in_cta(&sm_top[c % p.k], c / p.k);
      __syncthreads();
      for (int c = tid; c < CL * p.k; c += NT) {
        const uint64_t me = sm_cand[c];
        int above = 0;
        for (int d = 0; d < CL * p.k && above < p.k; ++d) above += sm_cand[d] > me;
        if (above < p.k && me) write(above, me);
      }
    }
  }
  cluster_sync<CL>();
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

constexpr int NB = 256, BU = 4;          // threads, 16-byte vectors of a thread: a CTA's share of a row is in flight at once
template <typename T> constexpr int seg() { return NB * BU * (16 / (int)sizeof(T)); }

// dx_j = p_j (a log p_j + b) with a = -gH / T, b = -(sum g + gH H) / T; the target's and the
// alternatives' elements get their own g on top, written after the rest of the segment.
template <typename T>
__global__ void __launch_bounds__(NB, 6) scores_bwd_kernel(const T* __restrict__ logits, T* __restrict__ out,
                                                           const __grid_constant__ BwdParams p) {
  constexpr int VEC = 16 / sizeof(T);
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  const int c0 = blockIdx.y * seg<T>(), c1 = min(p.V, c0 + seg<T>());
  const T* x = logits + p.rows.at(row);
  T* y = out + row * p.V;
  const int64_t tgt = p.target[row];
  const float m = p.stats[2 * row], ls = p.stats[2 * row + 1];
  const bool dead = tgt == p.ignore || tgt < 0 || tgt >= p.V || m == -INFINITY;
  // vectors where input and output share their place in a 16-byte line, single elements at the ends
  const bool vec = ((reinterpret_cast<uintptr_t>(x + c0) ^ reinterpret_cast<uintptr_t>(y + c0)) & 15) == 0;
  const int head = vec ? min(c1 - c0, (int)(((16 - (reinterpret_cast<uintptr_t>(y + c0) & 15)) & 15) / sizeof(T))) : 0;
  const int nv = vec ? (c1 - c0 - head) / VEC : 0;
  const int rem = c1 - c0 - nv * VEC;
  Vec16<T> v[BU];
#pragma unroll
  for (int u = 0; u < BU; ++u) {
    v[u].raw = make_uint4(0, 0, 0, 0);
    if (!dead && u * NB + tid < nv) v[u] = ld16(x + c0 + head + (int64_t)(u * NB + tid) * VEC);
  }
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
  const uint64_t nm = pk(-m, -m), it2 = pk(p.inv_t, p.inv_t), nl = pk(-ls, -ls), a2 = pk(a, a), b2 = pk(b, b), l2 = pk(LOG2E, LOG2E);
#pragma unroll
  for (int u = 0; u < BU; ++u) {
    if (u * NB + tid >= nv) break;
    if (!dead) {
#pragma unroll
      for (int j = 0; j < VEC; j += 2) {
        float f0, f1;
        unpk(fma2(add2(pk(to_f(v[u].v[j]), to_f(v[u].v[j + 1])), nm), it2, nl), f0, f1);
        const uint64_t lp = pk(max_nan(f0, DMIN), max_nan(f1, DMIN));
        unpk(mul2(lp, l2), f0, f1);
        unpk(mul2(pk(ex2(f0), ex2(f1)), fma2(a2, lp, b2)), f0, f1);
        v[u].v[j] = from_f<T>(f0);
        v[u].v[j + 1] = from_f<T>(f1);
      }
    }
    st16(y + c0 + head + (int64_t)(u * NB + tid) * VEC, v[u]);
  }
  for (int i = tid; i < rem; i += NB) {
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
  // 1 / T is finite in fp32, and exp(DMIN / T), the weight of a logit of -inf, is 0
  TORCH_CHECK(temperature >= 1e-30 && temperature <= 1e27, "token_scores: temperature from 1e-30 to 1e27, got ", temperature);
  TORCH_CHECK(logits.is_cuda() && target.is_cuda() && logits.device() == target.device(),
              "token_scores: logits and targets on one GPU");
  TORCH_CHECK(target.scalar_type() == at::kLong && target.is_contiguous(), "token_scores: contiguous int64 targets");
  const int64_t V = logits.size(-1);
  TORCH_CHECK(V >= 1 && V < (1LL << 30), "token_scores: vocabulary of ", V);
  const int64_t R = logits.numel() / V;
  TORCH_CHECK(target.numel() == R, "token_scores: one target per row (", R, " rows, ", target.numel(), " targets)");
  TORCH_CHECK(R < (1LL << 28), "token_scores: at most 2^28 rows");
  TORCH_CHECK(top_k >= 0 && top_k <= std::min<int64_t>(MAXK, V), "token_scores: top_k from 0 to ", std::min<int64_t>(MAXK, V), ", got ", top_k);
  return R;
}

// CTAs per row: 8, 4 or 2 where that many per row stay resident at one per SM and each has 16 KB of the row.  Rows of
// 128000 bf16, us with 1, 2, 4 and 8:
//   k = 0     9 rows 14.9, 11.5, 9.1, 8.6    30 rows 16.5, 12.5, 10.5, 10.4   74 rows 16.5, 12.5, 14.4, 18.6
//   k = 20    9 rows 18.8, 16.9, 16.6, 19.0  30 rows 20.7, 18.6, 17.7, 20.7   74 rows 20.8, 18.6, 22.7, 41.2
// from 75 rows on 2 is no better than 1.  The 16 KB edge is flat: 30 rows of 16000 to 64000, k = 0, within 20%.
static int cluster_of(int64_t R, int64_t row_bytes) {
  int cl = 1;
  while (cl < 8 && R * cl * 2 <= num_sms() && row_bytes >= 32768 * cl) cl *= 2;
  return cl;
}
template <typename T, int CL, int NT>
void launch_fwd(const T* x, const FwdParams& p, int64_t R) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(R * CL));
  cfg.blockDim = dim3(NT);
  cfg.stream = stream();
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = CL;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = CL > 1 ? 1 : 0;
  MAMF_CUDA_CHECK(cudaLaunchKernelEx(&cfg, scores_fwd_kernel<T, CL, NT>, x, p));
}
// 512 threads have a row done sooner; 256 waste less at its end, which counts once every SM has three rows, unless the
// search for many alternatives is most of that.  Rows of 128000 bf16, us with 512 / 256 threads:
//   rows      148          443          500          900          3686
//   k = 0     16.7 / 22.8  27.7 / 29.0  35.1 / 34.4  53.5 / 53.5  170 / 159
//   k = 8     20.7 / 26.2  33.0 / 34.0  41.2 / 39.2  62.9 / 64.0  201 / 190
//   k = 12    20.8 / 26.9  33.0 / 35.3  43.0 / 40.8  63.8 / 69.2  211 / 202
//   k = 20    20.8 / 28.9  35.1 / 38.3  45.3 / 43.5  67.8 / 76.2  222 / 231
// So k > 8 is a middle of edges between 4 and 20.  Shorter rows favour 256 earlier, which the rule does not follow: 600
// rows of 16000, k = 8, 24.7 / 16.6.
template <typename T>
void launch_fwd(const T* x, const FwdParams& p, int64_t R) {
  const int cl = cluster_of(R, p.V * (int64_t)sizeof(T));
  if (cl == 8) launch_fwd<T, 8, 512>(x, p, R);
  else if (cl == 4) launch_fwd<T, 4, 512>(x, p, R);
  else if (cl == 2) launch_fwd<T, 2, 512>(x, p, R);
  else if (R < 3 * num_sms() || p.k > 8) launch_fwd<T, 1, 512>(x, p, R);
  else launch_fwd<T, 1, 256>(x, p, R);
}

}  // namespace ts

// 1 where a target was outside the vocabulary since this was cleared
int64_t token_scores_error(bool clear) {
  int v = 0, z = 0;
  MAMF_CUDA_CHECK(cudaMemcpyFromSymbol(&v, ts::g_err, sizeof(int)));
  if (v && clear) MAMF_CUDA_CHECK(cudaMemcpyToSymbol(ts::g_err, &z, sizeof(int)));
  return v;
}

// logits (.., V), up to two leading dimensions of any strides without a copy; target (..) int64.
// -> log_probs, entropy (like target, fp32), top_log_probs, top_ids (.., k), and for the gradient stats (R, 2)
std::vector<at::Tensor> token_scores_fwd(at::Tensor logits, at::Tensor target, int64_t ignore_index, double temperature,
                                         int64_t top_k, bool want_stats) {
  using namespace ts;
  logits = as_rows(logits);
  const int64_t R = check(logits, target, temperature, top_k);
  c10::cuda::CUDAGuard guard(logits.device());
  auto f32 = logits.options().dtype(at::kFloat);
  at::Tensor lp = at::empty(target.sizes(), f32), ent = at::empty(target.sizes(), f32);
  auto tk = target.sizes().vec();
  tk.push_back(top_k);
  at::Tensor top_lp = at::empty(tk, f32), top_id = at::empty(tk, target.options()), stats;
  if (want_stats) stats = at::empty({R, 2}, f32);
  if (R > 0) {
    FwdParams p{rows_of(logits), target.data_ptr<int64_t>(), lp.data_ptr<float>(), ent.data_ptr<float>(),
                top_lp.data_ptr<float>(), want_stats ? stats.data_ptr<float>() : nullptr, top_id.data_ptr<int64_t>(), ignore_index,
                (int)logits.size(-1), (int)top_k, (float)(1.0 / temperature)};
    MAMF_DISPATCH_FLOAT_BF16(logits.scalar_type(), "token_scores", [&] {
      launch_fwd<scalar_t>((const scalar_t*)logits.data_ptr(), p, R);
    });
  }
  if (!want_stats) return {lp, ent, top_lp, top_id};
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
    dim3 grid((unsigned)R, (unsigned)((p.V + seg<scalar_t>() - 1) / seg<scalar_t>()));
    scores_bwd_kernel<scalar_t><<<grid, NB, 0, stream()>>>((const scalar_t*)logits.data_ptr(), (scalar_t*)out.data_ptr(), p);
  });
  MAMF_LAUNCH_CHECK();
  return out;
}

// The operator with its gradient, as a node of torch's graph without Python in it (a small vocabulary's pass is
// mostly that otherwise).
namespace ts {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// The gradient as a node of its own, so that a graph may be kept; differentiating it again is refused.
struct ScoresGrad : torch::autograd::Function<ScoresGrad> {
  static at::Tensor forward(AutogradContext*, at::Tensor logits, at::Tensor target, at::Tensor stats, at::Tensor ent,
                            at::Tensor top_id, c10::optional<at::Tensor> g_lp, c10::optional<at::Tensor> g_ent,
                            c10::optional<at::Tensor> g_top, int64_t ignore_index, double temperature) {
    return token_scores_bwd(logits, target, ignore_index, temperature, stats, ent, top_id, g_lp, g_ent, g_top);
  }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK(false, "token_scores has no second derivative");
  }
};

struct Scores : torch::autograd::Function<Scores> {
  static variable_list forward(AutogradContext* ctx, at::Tensor logits, at::Tensor target, int64_t ignore_index,
                               double temperature, int64_t top_k) {
    auto r = token_scores_fwd(logits, target, ignore_index, temperature, top_k, true);
    ctx->save_for_backward({logits, target, r[4], r[1], r[3]});
    ctx->saved_data["ignore_index"] = ignore_index;
    ctx->saved_data["temperature"] = temperature;
    ctx->mark_non_differentiable({r[3]});
    ctx->set_materialize_grads(false);
    r.pop_back();
    return r;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto v = ctx->get_saved_variables();
    auto plain = [](const at::Tensor& t) {
      return t.defined() ? c10::optional<at::Tensor>(t.to(at::kFloat).contiguous()) : c10::nullopt;
    };
    return {ScoresGrad::apply(v[0], v[1], v[2], v[3], v[4], plain(g[0]), plain(g[1]), plain(g[2]),
                              ctx->saved_data["ignore_index"].toInt(), ctx->saved_data["temperature"].toDouble()),
            at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

// Log probabilities alone, differentiable any number of times: the first gradient is the kernel's, those of the
// gradient are of torch's operations.
struct LogProbsGrad : torch::autograd::Function<LogProbsGrad> {
  static at::Tensor forward(AutogradContext* ctx, at::Tensor logits, at::Tensor target, at::Tensor stats, at::Tensor ent,
                            at::Tensor top_id, at::Tensor g, int64_t ignore_index) {
    ctx->save_for_backward({logits, target, g});
    ctx->saved_data["ignore_index"] = ignore_index;
    return token_scores_bwd(logits, target, ignore_index, 1.0, stats, ent, top_id, g, c10::nullopt, c10::nullopt);
  }
  // dx_j = g (d_jt - p_j): with w the gradient of dx, that of g is w_t - sum p w, that of x_j is -g p_j (w_j - sum p w)
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto v = ctx->get_saved_variables();
    const at::Tensor &logits = v[0], &target = v[1], &g = v[2];
    const int64_t V = logits.size(-1);
    const at::Tensor live = (target != ctx->saved_data["ignore_index"].toInt()) & (target >= 0) & (target < V);
    const at::Tensor w = grads[0].to(at::kFloat), p = at::softmax(logits.to(at::kFloat), -1);
    const at::Tensor away = w - (p * w).sum(-1, true);
    const at::Tensor dg = away.gather(-1, target.clamp(0, V - 1).unsqueeze(-1)).squeeze(-1);
    const at::Tensor dx = -(g * live).unsqueeze(-1) * p * away, none;
    return {dx.to(logits.scalar_type()), none, none, none, none, dg * live, none};
  }
};

struct LogProbs : torch::autograd::Function<LogProbs> {
  static at::Tensor forward(AutogradContext* ctx, at::Tensor logits, at::Tensor target, int64_t ignore_index) {
    const auto r = token_scores_fwd(logits, target, ignore_index, 1.0, 0, true);
    ctx->save_for_backward({logits, target, r[4], r[1], r[3]});
    ctx->saved_data["ignore_index"] = ignore_index;
    return r[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto v = ctx->get_saved_variables();
    return {LogProbsGrad::apply(v[0], v[1], v[2], v[3], v[4], g[0].to(at::kFloat).contiguous(),
                                ctx->saved_data["ignore_index"].toInt()),
            at::Tensor(), at::Tensor()};
  }
};

}  // namespace ts

// -> log probabilities, differentiable in logits as often as needed
at::Tensor token_log_probs(at::Tensor logits, at::Tensor target, int64_t ignore_index) {
  return ts::LogProbs::apply(logits, target, ignore_index);
}

// -> log_probs, entropy, top_log_probs, top_ids, differentiable in logits
std::vector<at::Tensor> token_scores(at::Tensor logits, at::Tensor target, int64_t ignore_index, double temperature,
                                     int64_t top_k) {
  return ts::Scores::apply(logits, target, ignore_index, temperature, top_k);
}

}  // namespace mamf
