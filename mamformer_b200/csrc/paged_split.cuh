// Shared by the attention kernels over the paged caches for few query rows (paged_attn.cu, paged4_attn.cu): the list of
// (sequence, KV head, row tile) items that the CTAs share, the waits, the warp-level products, and the kernel that joins the
// parts of an item.
#pragma once

#include "paged.cuh"
#include "tc5.cuh"

namespace mamf {
namespace split {

using namespace paged;

constexpr int NW = 4, NT = NW * 32, NJ = 512;
constexpr float NONE = -1e30f;                 // maximum of no scores: 2^(score - NONE) is never formed, 2^(NONE - m) is 0

// The file's own words.
static __device__ int g_err = 0, g_wait_err = 0;
__device__ __forceinline__ void record(int code) { atomicCAS(&g_err, 0, code); }

using tc5::ex2;
using tc5::su32;
__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
__device__ __forceinline__ void mma(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// transpose of an 8 x 8 matrix of 16-bit values held as mma fragments
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ bool try_tile(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}\n"
               : "=r"(ok) : "r"(bar), "r"(parity), "r"(1000000u) : "memory");
  return ok != 0;
}
// Waits for the warp's tile, the same answer for all lanes; false after `limit` cycles (recorded).  The record is only
// written: what another warp, or an earlier call, has recorded ends no wait of this one, and a CTA that gives up ends
// after one limit for each of its warps' waits at the same time.
__device__ __forceinline__ bool wait_tile(uint32_t bar, uint32_t parity, long long limit) {
  if (limit >= 0 && __all_sync(0xffffffffu, try_tile(bar, parity))) return true;
  const long long t0 = clock64();
  for (uint32_t n = 1;; ++n) {
    if (limit >= 0 && __all_sync(0xffffffffu, try_tile(bar, parity))) return true;
    if ((n & 63u) == 0) {
      const bool over = clock64() - t0 > limit;
      if (over) atomicCAS(&g_wait_err, 0, (int)ERR_WAIT);
      if (__any_sync(0xffffffffu, over)) return false;
    }
  }
}
// Waits for a copy whose result nobody needs, whatever has been recorded: a CTA's memory may be another's once it ends.
__device__ __forceinline__ void drain_tile(uint32_t bar, uint32_t parity) {
  const long long t0 = clock64();
  while (!try_tile(bar, parity) && clock64() - t0 <= WAIT_CYCLES) {}
}

// One row tile of one KV head of one sequence.
// ROWS: rows of a tile, TILE: tokens of a tile.
struct Item {
  int b, g, rt;
  int t0, n, len;            // first packed token, new tokens, cached length
  int rows;                  // n * rep * maps
  int lo, hi, k0, nt;        // slots [lo, hi) that some row of the tile sees, first tile, tiles (at least 1)
};

template <int ROWS, int TILE, class P>
__device__ __forceinline__ void set_range(const P& p, Item& it) {
  const int per = p.rep * p.maps, first = it.len - it.n;
  const int i0 = it.rt * ROWS / per, i1 = min(it.n - 1, (it.rt * ROWS + ROWS - 1) / per);
  it.hi = max(0, min(it.len, first + i1 + 1));
  it.lo = p.window > 0 ? max(0, first + i0 - p.window + 1) : 0;
  it.k0 = it.lo / TILE;
  it.nt = it.hi > it.lo ? (it.hi + TILE - 1) / TILE - it.k0 : 1;
}
template <int ROWS, int TILE, class P>
__device__ __forceinline__ bool set_sequence(const P& p, Item& it, int b) {
  const Table& c = p.c;
  const int t0 = c.cu[b], t1 = c.cu[b + 1], len = c.lens[b];
  it.b = b;
  it.t0 = t0;
  it.n = t1 - t0;
  if (t0 < 0 || t1 <= t0 || t1 > c.T) return false;             // what does not fit is the join kernel's to report
  it.rows = it.n * p.rep * p.maps;
  if (it.rows > p.few) return false;
  it.len = cached_length(c, len);
  it.g = it.rt = 0;
  set_range<ROWS, TILE>(p, it);
  return true;
}
template <int ROWS, int TILE, class P>
__device__ __forceinline__ void next_item(const P& p, Item& it) {
  if (ROWS > 8 && (it.rt + 1) * ROWS < it.rows) { ++it.rt; set_range<ROWS, TILE>(p, it); return; }
  if (it.g + 1 < p.c.G) { ++it.g; it.rt = 0; set_range<ROWS, TILE>(p, it); return; }
  int b = it.b + 1;
  while (b < p.c.B && !set_sequence<ROWS, TILE>(p, it, b)) ++b;
  it.b = b;
}
template <int ROWS, int TILE, class P>
__device__ __forceinline__ int64_t tiles_of(const P& p, int b) {
  Item it;
  if (!set_sequence<ROWS, TILE>(p, it, b)) return 0;
  int64_t n = 0;
  if constexpr (ROWS == 8) n = it.nt;                           // 8 rows are all there can be
  else
    for (; it.rt * ROWS < it.rows; ++it.rt) {
      set_range<ROWS, TILE>(p, it);
      n += it.nt;
    }
  return n * p.c.G;
}

template <typename T> __device__ __forceinline__ void q_row16(const T* q, float* f) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const Vec16<T> v = ld16(q + 8 * i);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[8 * i + j] = to_f(v.v[j]);
  }
}

// What the split kernel has left out, by one block: offsets or lengths that do not fit are recorded, sequences of more
// tokens than max_new get zeros, and offsets out of order give nothing but zeros.  The look at them needs nothing of that
// kernel and is over before it ends; after it, it cost a short call 1.5 us.
template <typename T, class P>
__device__ __noinline__ void left_out(const P& p, int hd) {
  const Table& c = p.c;
  auto too_many = [&](int b) { return !p.chunked && (int64_t)(c.cu[b + 1] - c.cu[b]) * p.rep * p.maps > p.few; };
  bool broken = false, odd = false;
  for (int b = threadIdx.x; b < c.B; b += NJ) {
    broken = broken || !in_order(c, b);
    odd = odd || too_many(b) || cached_length(c, c.lens[b]) != c.lens[b];
  }
  odd = __syncthreads_or(odd || broken);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (!odd) return;
  broken = __syncthreads_or(broken);
  if (threadIdx.x == 0) record(ERR_LENGTH);
  for (int t = 0; t < c.T; ++t) {
    const int b = broken ? -1 : sequence_of(c.cu, c.B, t);
    if (broken || (b >= 0 && too_many(b))) {
      for (int i = threadIdx.x; i < p.H * hd; i += NJ) ((T*)p.out)[(int64_t)t * p.H * hd + i] = from_f<T>(0.f);
      if (P::SUMS && p.lse)
        for (int i = threadIdx.x; i < p.H * p.maps; i += NJ) p.lse[(int64_t)t * p.H * p.maps + i] = INFINITY;
    }
  }
}

// Joins the parts of an item that ran over several CTAs: block = the CTA in which it ended.
template <typename T, int HD, int NR, class P>
__global__ void __launch_bounds__(NJ, 2) join_kernel(const __grid_constant__ P p) {
  constexpr int ROWS = 8 * NR;
  if (blockIdx.x == 0) {                               // no item ends in the first CTA that began before it
    left_out<T>(p, HD);
    return;
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 j = p.joins[blockIdx.x];
  if (j.x < 0) return;
  const int t0 = j.x, row0 = (j.z >> 16) * ROWS, n_rows = min(ROWS, j.y - row0), g = j.z & 0xffff;
  const int c0 = j.w >> 1, parts = blockIdx.x - c0 + 1, per = p.rep * p.maps;
  // the warps share the rows, and a row's warps its parts, each under a running maximum; the two maps of a head
  // are neighbouring rows
  constexpr int W = NJ / 32, D = HD / 32;
  __shared__ float vals[W][HD];
  __shared__ float2 sums[W];                           // {maximum, sum}
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, r = w % n_rows, gr = w / n_rows, groups = W / n_rows;
  if (gr < groups) {
    float M = NONE, L = 0.f, least = 0.f, a[D] = {};   // least: negative where a part was cut short
    for (int i0 = gr; i0 < parts; i0 += 4 * groups) {   // four parts are on their way at once
      float2 ml[4], v[4][D / 2];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + u * groups;
        ml[u] = make_float2(NONE, 0.f);
#pragma unroll
        for (int d = 0; d < D / 2; ++d) v[u][d] = make_float2(0.f, 0.f);
        if (i < parts) {
          const float* x = p.part + (((int64_t)(c0 + i) * 2 + (i == 0 ? j.w & 1 : 0)) * ROWS + r) * (HD + 2);
          ml[u] = *reinterpret_cast<const float2*>(x + HD);
#pragma unroll
          for (int d = 0; d < D / 2; ++d) v[u][d] = *reinterpret_cast<const float2*>(x + lane * D + 2 * d);
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float mn = fmaxf(M, ml[u].x), f = ex2(M - mn), e = ex2(ml[u].x - mn);
        M = mn;
        least = fminf(least, ml[u].y);
        L = fmaf(L, f, ml[u].y * e);
#pragma unroll
        for (int d = 0; d < D / 2; ++d) {
          a[2 * d] = fmaf(a[2 * d], f, v[u][d].x * e);
          a[2 * d + 1] = fmaf(a[2 * d + 1], f, v[u][d].y * e);
        }
      }
    }
#pragma unroll
    for (int d = 0; d < D; ++d) vals[w][lane * D + d] = a[d];
    if (lane == 0) sums[w] = make_float2(M, least < 0.f ? -1.f : L);
  }
  __syncthreads();
  // a row's value of dim d, and log2 of its sum of weights where `sum` asks for it
  auto value = [&](int row, int d, float* sum) {
    float M = NONE, L = 0.f, x = 0.f;
    float least = 0.f;
    for (int i = row; i < groups * n_rows; i += n_rows) {
      M = fmaxf(M, sums[i].x);
      least = fminf(least, sums[i].y);
    }
    for (int i = row; i < groups * n_rows; i += n_rows) {
      const float e = ex2(sums[i].x - M);
      x = fmaf(vals[i][d], e, x);
      L = fmaf(sums[i].y, e, L);
    }
    const bool none = least < 0.f || L == 0.f;
    if (sum) *sum = none ? INFINITY : M + log2f(L);
    return none ? 0.f : x / L;
  };
  for (int i = threadIdx.x; i < ROWS / p.maps * HD; i += NJ) {
    const int rr = i / HD * p.maps, d = i % HD;
    if (rr >= n_rows) continue;
    const int row = row0 + rr, tok = t0 + row / per, h = g * p.rep + row % per / p.maps;
    float* sums_at = P::SUMS && p.lse && d == 0 ? p.lse + (int64_t)tok * p.H * p.maps + g * per + row % per : nullptr;
    float x = value(rr, d, sums_at);
    if (p.maps == 2) x = (x - p.lam[h] * value(rr + 1, d, sums_at ? sums_at + 1 : nullptr)) / (1.f - p.lam[h] + 1e-8f);
    ((T*)p.out)[((int64_t)tok * p.H + h) * HD + d] = from_f<T>(x);
  }
}

template <typename T, int HD, int NR, class P> void launch_join(const P& p) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(p.ctas);
  cfg.blockDim = dim3(NJ);
  cfg.stream = stream();
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  MAMF_CUDA_CHECK(cudaLaunchKernelEx(&cfg, join_kernel<T, HD, NR, P>, p));
}

}  // namespace split
}  // namespace mamf
